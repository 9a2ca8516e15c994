"""What passes take of the page lists of streams that forget, without a GPU (a C++ program)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_lists_leave_holes_out(tmp_path):
    exe = str(tmp_path / "page_hole_test")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover",
                           os.path.join(HERE, "cpp", "page_hole_test.cpp"), "-o", exe])
    done = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
