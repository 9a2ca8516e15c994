"""Sequences that forget and rows that see sinks, without a GPU: the bookkeeping and the plans (a C++ program), and the Python side."""
import os
import subprocess

import pytest

import gradhip as G
from test_cache_python import cache, rows  # noqa: F401  (a cache over a library that accepts everything)

HERE = os.path.dirname(os.path.abspath(__file__))


def test_forgotten_pages_and_plans_with_sinks(tmp_path):
    exe = str(tmp_path / "page_forget_test")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover",
                           os.path.join(HERE, "cpp", "page_forget_test.cpp"), "-o", exe])
    done = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr


def test_null_caches():
    lib = G.load_library()
    assert lib.gh_cache_forget(None, 0, 0, 1) == G.GH_ERR_INVALID_ARGUMENT
    assert lib.gh_cache_attend_sinks(None, 0, None, None, 0.0, 1, 8, 4, None) == G.GH_ERR_INVALID_ARGUMENT


def test_sinks_go_to_the_library(cache):  # noqa: F811
    cache.extend([0], [5])
    cache.attend(0, rows(5, 4), rows(5, 4), window=64, sinks=4)
    name, args = cache._lib.calls[-1]
    assert name == "gh_cache_attend_sinks" and args[5:8] == (1, 64, 4)
    cache.attend(0, rows(5, 4), rows(5, 4), window=64)
    assert cache._lib.calls[-1][0] == "gh_cache_attend"
    before = len(cache._lib.calls)
    for sinks in (2 ** 31, -2 ** 31 - 1, 1.5):
        with pytest.raises((TypeError, ValueError)):
            cache.attend(0, rows(5, 4), rows(5, 4), window=64, sinks=sinks)
    for span in ((0, 2 ** 31), (2 ** 40, 3), (0.5, 2)):
        with pytest.raises((TypeError, ValueError)):
            cache.forget(0, *span)
    assert len(cache._lib.calls) == before
    cache.forget(0, 4, 60)
    assert cache._lib.calls[-1][0] == "gh_cache_forget" and cache._lib.calls[-1][1][1:] == (0, 4, 60)
    assert cache._rows == -1  # the pass is over
