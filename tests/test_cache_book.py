"""The paged cache without a GPU: its page bookkeeping and its plans (a C++ program), and what creation refuses."""
import os
import subprocess

import pytest

import gradhip as G

HERE = os.path.dirname(os.path.abspath(__file__))


def test_pages_and_plans(tmp_path):
    exe = str(tmp_path / "page_book_test")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover",
                           os.path.join(HERE, "cpp", "page_book_test.cpp"), "-o", exe])
    done = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr


GOOD = dict(layers=2, heads=4, kv_heads=2, head_dim=64, pages=8)


@pytest.mark.parametrize("change,match", [
    (dict(layers=0), "layers"), (dict(layers=5000), "layers"), (dict(heads=0), "heads"), (dict(heads=2000, kv_heads=2), "heads"),
    (dict(heads=3), "multiple"), (dict(kv_heads=0), "heads"), (dict(head_dim=0), "head_dim"), (dict(head_dim=12), "head_dim"),
    (dict(head_dim=264), "head_dim"), (dict(page_tokens=8), "page_tokens"), (dict(page_tokens=48), "page_tokens"),
    (dict(page_tokens=2048), "page_tokens"), (dict(page_tokens=-1), "page_tokens"), (dict(pages=0), "pages"),
    (dict(pages=2 ** 31 - 1), "pages"), (dict(rope_base=-1.0), "rope_base"), (dict(rope_base=float("nan")), "rope_base"),
    (dict(rope_base=float("inf")), "rope_base"), (dict(dtype="f64"), "type"),
])
def test_creation_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        G.Cache(**{**GOOD, **change})


def test_null_arguments():
    lib = G.load_library()
    assert lib.gh_cache_create(None, None) == G.GH_ERR_INVALID_ARGUMENT
    assert lib.gh_cache_add(None, None) == G.GH_ERR_INVALID_ARGUMENT
    assert lib.gh_cache_extend(None, None, None, 0, None) == G.GH_ERR_INVALID_ARGUMENT
    assert lib.gh_cache_attend(None, 0, None, None, 0.0, 1, 0, None) == G.GH_ERR_INVALID_ARGUMENT
    assert lib.gh_cache_length(None, 0) == -1
    lib.gh_cache_free(None)


def test_creation_without_a_gpu_fails_loudly():
    try:
        G.device_info()
    except G.DeviceError:
        with pytest.raises(G.DeviceError, match="no CPU fallback"):
            G.Cache(**GOOD)
