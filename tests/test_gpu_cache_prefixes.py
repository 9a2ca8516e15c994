"""Passes whose sequences share prefixes of so many bytes that they meet them in common tiles: several families in one pass, beside
sequences of many rows and of none, under masks that allow sharing and masks that do not."""
import pytest

import test_gpu_cache as base
from test_gpu_cache import HEADS, Rig, TYPES

pytestmark = pytest.mark.gpu

SHARED = 64_000_000  # bytes that a family's members would read of their prefix, each for itself: sharing begins at 40 MiB


@pytest.fixture(scope="module")
def torch():
    return base._torch()


def _family(rig, members, page, longer=0):
    """(prompt, forks of it): prompts as long as `members` forks and the prompt itself need to share them."""
    size = 4 if rig.dtype == "f32" else 2
    n = SHARED // ((members + 1) * 2 * rig.kv_heads * rig.dim * size) // page * page + page + 3 + longer
    return n, members


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", ["mha64", "grouped128", "one-key80", "dim256"])
def test_families_beside_others(torch, dtype, heads):
    h, kv, dim, page = HEADS[heads]
    rig = Rig(torch, dtype, heads=h, kv_heads=kv, dim=dim, page=page, pages=150_000 // page, seed=61)
    a_len, a_kids = _family(rig, 18, page)
    b_len, b_kids = _family(rig, 13, page, longer=page)
    a, b, c, lone, chunk = (rig.add() for _ in range(5))
    rig.grow([a, b, c, lone, chunk], [a_len, b_len, 4 * page + 1, 290, 77])
    firsts = [rig.fork(a) for _ in range(a_kids)]
    seconds = [rig.fork(b, b_len - 2) for _ in range(b_kids)]
    thirds = [rig.fork(c) for _ in range(3)]  # a family too small to share
    rig.grow(firsts[:3] + seconds[:2], [1, 19, 2, 33, 5])
    group = h // kv
    few = max(1, 16 // group)  # rows of a member, at most
    seqs = firsts[:7] + [lone] + seconds + [b, chunk] + thirds + firsts[7:] + [a]
    for counts in ([1] * len(seqs), [1 + i % few if s is not chunk else 1 for i, s in enumerate(seqs)],
                   [90 if s is chunk else 1 for s in seqs],  # rows for tiles of many beside both families
                   [0 if i % 4 == 1 else 45 if i in (2, 9) else 1 for i in range(len(seqs))]):  # members without rows, and with many
        size = 2 * kv * dim * (4 if dtype == "f32" else 2)
        for n, family in ((a_len, firsts + [a]), (b_len - 2, seconds + [b])):
            members = sum(0 < rows * group <= 16 for s, rows in zip(seqs, counts) if s in family)
            assert n // page * page * members * size >= 40 << 20, "a family that shares"
        q = rig.grow(seqs, counts)
        for mask in ({}, {"causal": False}, {"window": 300}, {}):
            out = rig.check(seqs, counts, q, what=f"{mask}", **mask)
            assert torch.equal(out, rig.check(seqs, counts, q, what="again", **mask))
    rig.check_contents([firsts[1], seconds[0], thirds[2]])
