"""fp32 attention of many rows over the paged cache where operands lie far apart: an element next to one many powers of two larger
keeps its digits, whichever of queries, keys, values and probabilities they are in, and whatever shares the pass."""
import pytest

import test_gpu_cache as base
from test_gpu_cache import Rig

pytestmark = pytest.mark.gpu

# (head_dim, heads, kv_heads): each width that has a kernel of its own, and widths between them
WIDTHS = {"64": (64, 2, 1), "128": (128, 2, 2), "40": (40, 1, 1), "96": (96, 2, 1), "256": (256, 1, 1)}


@pytest.fixture(scope="module")
def torch():
    return base._torch()


def _many_rows(torch, width, seed, change):
    """133 cached positions and a chunk of 250 rows onto them; change(k, v) before they are stored.  (rig, sequence, queries)"""
    dim, heads, kv = WIDTHS[width]
    rig = Rig(torch, "f32", heads=heads, kv_heads=kv, dim=dim, page=16, pages=60, seed=seed)
    s = rig.add()
    old = [rig.rand(1, 133, kv, dim), rig.rand(1, 133, kv, dim)]
    new = [rig.rand(1, 250, kv, dim), rig.rand(1, 250, kv, dim)]
    for k, v in (old, new):
        change(k, v)
    rig.grow([s], [133], k=old[0], v=old[1])
    return rig, s, rig.grow([s], [250], k=new[0], v=new[1])


def _check(rig, s, q, what):
    rig.check([s], [250], q, what=what)
    rig.check([s], [250], q, window=60, what=what + ", window")


@pytest.mark.parametrize("size", [1e4, 1e6, 1e8, 1e10, 1e12, 1e20])
@pytest.mark.parametrize("width", WIDTHS)
def test_a_query_element_far_above_the_others(torch, width, size):
    """It meets keys of zero: nothing of it is in the scores, which the other elements decide."""
    def change(k, v):
        k[..., 3] = 0.0
    rig, s, q = _many_rows(torch, width, 41, change)
    q[..., 3] = size
    _check(rig, s, q, f"a query element of {size:g}")


@pytest.mark.parametrize("power", [16, 20, 24, 30, 40, 80])
@pytest.mark.parametrize("width", WIDTHS)
def test_dims_of_values_far_below_the_others(torch, width, power):
    def change(k, v):
        v[..., ::3] *= 2.0 ** -power
    rig, s, q = _many_rows(torch, width, 42, change)
    _check(rig, s, q, f"dims of values by 2^-{power}")


@pytest.mark.parametrize("power", [16, 20, 30, 40])
@pytest.mark.parametrize("width", WIDTHS)
def test_small_key_dims_meet_large_query_dims(torch, width, power):
    def change(k, v):
        k[..., 1::3] *= 2.0 ** -power
    rig, s, q = _many_rows(torch, width, 43, change)
    q[..., 1::3] *= 2.0 ** power
    _check(rig, s, q, f"key dims by 2^-{power}, query dims by 2^{power}")


@pytest.mark.parametrize("power", [20, 35, 60])
@pytest.mark.parametrize("width", WIDTHS)
def test_values_of_zero_where_the_weight_is(torch, width, power):
    """One position takes nearly all of the weight and has zeros in two dims: those outputs are the other positions', whose
    probabilities are near 2^-power."""
    dim = WIDTHS[width][0]

    def change(k, v):
        k[..., 0] = 0.0
        k[:, 5, :, 0] = 1.0
        v[:, 5, :, 2] = 0.0
        v[:, 5, :, 7] = 0.0
    rig, s, q = _many_rows(torch, width, 44, change)
    q[..., 0] = power * 0.6931471805599453 * dim ** 0.5
    _check(rig, s, q, f"weights near 2^-{power}")


@pytest.mark.parametrize("scale", [0.0, 1e-3, 1e-20, 1e-36])
@pytest.mark.parametrize("width", WIDTHS)
def test_queries_and_keys_that_are_both_tiny(torch, width, scale):
    """Scores far below one: every visible position weighs the same, and the others nothing."""
    def change(k, v):
        k *= 2.0 ** -60
    rig, s, q = _many_rows(torch, width, 45, change)
    q *= 2.0 ** -60
    rig.check([s], [250], q, scale=scale, what="tiny")
    rig.check([s], [250], q, scale=scale, window=60, what="tiny, window")


def test_a_row_does_not_depend_on_who_shares_its_pass(torch):
    """Single tokens with far-apart elements, in a pass of their own and beside a chunk of another sequence: right in both."""
    rig = Rig(torch, "f32", heads=4, kv_heads=2, dim=64, page=16, pages=80, seed=46)
    chunk, one = rig.add(), rig.add()
    rig.grow([chunk], [100])
    k, v = rig.rand(1, 300, 2, 64), rig.rand(1, 300, 2, 64)
    k[..., 3] = 0.0
    v[..., 1::2] *= 2.0 ** -36
    rig.grow([one], [300], k=k, v=v)
    for seqs, counts in (([one], [1]), ([chunk, one], [150, 1]), ([one, chunk], [2, 90])):
        rows = sum(counts)
        k, v = rig.rand(1, rows, 2, 64), rig.rand(1, rows, 2, 64)
        k[..., 3] = 0.0
        q = rig.grow(seqs, counts, k=k, v=v)
        q[..., 3] = 1e11
        rig.check(seqs, counts, q, what=f"{counts}")
