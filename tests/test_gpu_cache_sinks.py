"""Rows that see their sequence's first positions beside a window, and sequences that forget what lies between, on the GPU against the
definition in 64 bits."""
import pytest

import gradhip as G
import test_gpu_cache as base
from test_gpu_cache import HEADS, TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return base._torch()


def attention(R, q, k, v, first, causal, window, sinks, scale, dtype):
    """Row by row over the positions that it sees, which are all that the reference is given; (out, allowance)."""
    import torch
    out, allowed = [], []
    u = torch.arange(k.shape[0])
    for i in range(q.shape[0]):
        seen = torch.ones(k.shape[0], dtype=torch.bool)
        if causal:
            seen &= u <= first + i
        if window:
            seen &= (u > first + i - window) | (u < sinks)
        o, a = R.attention(q[i:i + 1], k[seen], v[seen], int(seen.sum()) - 1, False, 0, scale, dtype)
        out.append(o)
        allowed.append(a)
    return torch.cat(out), torch.cat(allowed)


class Rig(base.Rig):
    def check(self, seqs, counts, q, causal=True, window=0, sinks=0, scale=0.0, what="", stream=0, out=None, rows=None):
        """rows: of each sequence, how many are compared (the first, the last and some between); all if None."""
        torch = self.torch
        out = torch.full_like(q, 7.0) if out is None else out
        for layer in range(self.layers):
            self.cache.attend(layer, q[layer], out[layer], scale=scale, causal=causal, window=window, sinks=sinks, stream=stream)
        torch.cuda.synchronize()
        at = 0
        for s, n in zip(seqs, counts):
            for layer in range(self.layers):
                k, v = self.ref.k[s][layer], self.ref.v[s][layer]
                for i in range(n) if rows is None or rows >= n else sorted({round(j * (n - 1) / (rows - 1)) for j in range(rows)}):
                    want, allowed = attention(self.R, q[layer, at + i:at + i + 1].cpu().double(), k, v, k.shape[0] - n + i, causal, window, sinks, scale, self.dtype)
                    self.R.assert_within(out[layer, at + i:at + i + 1], want, allowed, f"{what} sequence {s} layer {layer} row {i}")
            at += n
        return out


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", TYPES)
def test_sinks_of_ragged_sequences(torch, dtype, heads):
    h, kv, dim, page = HEADS[heads]
    rig = Rig(torch, dtype, heads=h, kv_heads=kv, dim=dim, page=page, pages=4096 // page, seed=103)
    seqs = [rig.add() for _ in range(5)]
    rig.grow(seqs, [1, 33, 0, 150, 402])
    counts = [1, 3, 1, 18, 2]
    q = rig.grow(seqs, counts)
    for window, sinks in ((1, 1), (2, 5), (37, 4), (37, 16), (37, 17), (130, 33), (16, 100), (1000, 3), (20, 2 ** 31 - 1)):
        rig.check(seqs, counts, q, window=window, sinks=sinks, what=f"window {window} sinks {sinks}", rows=4)
    rig.check(seqs, counts, q, causal=False, window=5, sinks=3, what="window ahead", rows=4)
    rig.check(seqs, counts, q, window=40, sinks=4, scale=0.31, what="scale", rows=3)
    counts = [1] * 5
    q = rig.grow(seqs, counts)
    rig.check(seqs, counts, q, window=50, sinks=4, what="single tokens")


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", TYPES)
def test_sinks_of_many_rows_beside_few(torch, dtype, heads):
    h, kv, dim, page = HEADS[heads]
    rig = Rig(torch, dtype, heads=h, kv_heads=kv, dim=dim, page=page, pages=4096 // page, seed=104)
    seqs = [rig.add() for _ in range(4)]
    rig.grow(seqs, [300, 464, 0, 5])
    counts = [200, 1, 131, 70]
    q = rig.grow(seqs, counts)
    rig.check(seqs, counts, q, window=90, sinks=4, what="window 90", rows=9)
    rig.check(seqs, counts, q, window=17, sinks=50, what="window 17", rows=9)
    rig.check(seqs, counts, q, causal=False, window=150, sinks=20, what="window ahead", rows=5)


def test_no_window_and_no_sinks_are_the_calls_that_they_were(torch):
    rig = Rig(torch, "bf16", heads=4, kv_heads=2, dim=64, page=16, pages=64, seed=105)
    s = rig.add()
    rig.grow([s], [500])
    q = rig.grow([s], [40])
    outs = [torch.empty_like(q[0]) for _ in range(4)]
    rig.cache.attend(0, q[0], outs[0])
    rig.cache.attend(0, q[0], outs[1], sinks=9)  # without a window everything is seen
    rig.cache.attend(0, q[0], outs[2], window=33)
    rig.cache.attend(0, q[0], outs[3], window=33, sinks=0)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[2], outs[3]) and not torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("before,new", [(0, 1), (0, 70), (15, 1), (16, 2), (31, 1), (48, 17), (63, 70), (127, 129), (1000, 1), (1500, 5)])
def test_sinks_at_the_edges_of_pages_and_tiles(torch, dtype, before, new):
    rig = Rig(torch, dtype, heads=2, kv_heads=1, dim=64, page=16, pages=160, seed=before + new)
    s = rig.add()
    if before:
        rig.grow([s], [before])
    q = rig.grow([s], [new])
    for window, sinks in ((16, 15), (17, 16), (20, 17), (64, 32), (33, 48), (1, 64)):
        rig.check([s], [new], q, window=window, sinks=sinks, what=f"window {window} sinks {sinks}", rows=6)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_windows_in_many_parts(torch, dtype):
    """One token and a chunk over 20 thousand positions, of which the window and the sinks are cut into parts that are joined; the same
    call gives the same bits."""
    rig = Rig(torch, dtype, heads=4, kv_heads=2, dim=128, page=64, pages=400, seed=106)
    s = rig.add()
    rig.grow([s], [20000])
    for new in (1, 60):
        q = rig.grow([s], [new])
        a = rig.check([s], [new], q, window=9000, sinks=100, what=f"{new} rows", rows=4)
        b = torch.empty_like(q)
        rig.cache.attend(0, q[0], b[0], window=9000, sinks=100)
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 20, 250])
def test_what_lies_between_sinks_and_window_never_reaches_a_row(torch, dtype, new):
    """Infinities and NaN between the sinks and the window, behind the sinks in their own block of 16, and in the window of some rows."""
    for dim, heads, kv in ((64, 2, 1), (128, 3, 1), (24, 1, 1)):
        rig = Rig(torch, dtype, heads=heads, kv_heads=kv, dim=dim, page=16, pages=90, seed=107)
        bad = torch.full((1, 1440, kv, dim), float("nan")).to(rig.R.DTYPES[dtype])
        bad[:, ::2] = float("inf")
        waste = rig.add()
        rig.grow([waste], [1440], k=bad, v=bad)
        rig.drop(waste)  # its pages are handed out again, full of that
        s = rig.add()
        k, v = rig.rand(1, 600, kv, dim), rig.rand(1, 600, kv, dim)
        for t in (5, 9, 15, 40, 300):
            v[0, t, :, 3] = float("inf") if t % 2 else float("nan")
            k[0, t, :, 1] = float("nan")
        v[0, 580, :, 2] = -float("inf")  # in the window of the first rows alone
        rig.grow([s], [600], k=k, v=v)
        k, v = rig.rand(1, new, kv, dim), rig.rand(1, new, kv, dim)
        if new > 4:
            v[0, new - 2, :, 7] = float("inf")
        q = rig.grow([s], [new], k=k, v=v)
        rig.check([s], [new], q, window=30, sinks=5, what="behind the sinks", rows=7)
        rig.check([s], [new], q, window=64, sinks=3, what="seen by some", rows=7)
        rig.check([s], [new], q, window=30, sinks=12, what="a sink of NaN", rows=3)


@pytest.mark.parametrize("dtype", TYPES)
def test_streams_that_forget(torch, dtype):
    """Steps of streams in a pool that holds their windows and not their lengths: rotated, forked, copied, compacted and rewound on the way."""
    page, window, sinks = 16, 40, 5
    rig = Rig(torch, dtype, layers=2, heads=4, kv_heads=2, dim=64, page=page, pages=24, rope=10000.0, seed=108)
    seqs = [rig.add() for _ in range(3)]
    rig.grow(seqs, [3, 50, 20])
    grown = 0
    for step in range(14):
        counts = [(9, 1, 12)[(step + i) % 3] for i in range(3)]
        for s in seqs:
            n = rig.cache.length(s)
            rig.cache.forget(s, sinks, n - window + 1)
        q = rig.grow(seqs, counts)
        grown += sum(counts)
        rig.check(seqs, counts, q, window=window, sinks=sinks, what=f"step {step}", rows=3)
        if step == 5:
            extra = rig.fork(seqs[2])
            rig.cache.forget(extra, sinks, rig.cache.length(extra) - window + 1)
            q = rig.grow([extra, seqs[2]], [1, 2])
            rig.check([extra, seqs[2]], [1, 2], q, window=window, sinks=sinks, what="forked", rows=2)
            rig.drop(extra)
        if step == 8:
            copy = rig.cache.copy(seqs[1])
            rig.ref.fork(seqs[1], copy)
            q = rig.grow([copy], [3])
            rig.check([copy], [3], q, window=window, sinks=sinks, what="copied")
            rig.drop(seqs[1])
            rig.cache.compact()
            seqs[1] = copy
        if step == 11:
            rig.truncate(seqs[0], rig.cache.length(seqs[0]) - 4)
    assert grown > 24 * page - 100  # (more than the pool holds, together with what there was)
    for s in seqs:
        n = rig.cache.length(s)
        k = torch.empty(2, sinks, 2, 64, dtype=rig.R.DTYPES[dtype], device="cuda")
        v = torch.empty_like(k)
        rig.cache.read(s, k, v)
        assert torch.equal(k.cpu().double(), rig.ref.k[s][:, :sinks]) and torch.equal(v.cpu().double(), rig.ref.v[s][:, :sinks])
        tail = n - window
        k = torch.empty(2, window, 2, 64, dtype=rig.R.DTYPES[dtype], device="cuda")
        rig.cache.read(s, k, torch.empty_like(k), start=tail)
        assert torch.equal(k.cpu().double(), rig.ref.k[s][:, tail:])


def test_a_sequence_cut_off_inside_what_it_forgot(torch):
    rig = Rig(torch, "f32", heads=2, kv_heads=1, dim=64, page=16, pages=12, seed=109)
    s = rig.add()
    rig.grow([s], [150])
    rig.cache.forget(s, 4, 120)
    free = rig.cache.pages_free
    rig.truncate(s, 70)  # in the middle of a page that is nobody's
    assert rig.cache.pages_free > free and rig.cache.length(s) == 70
    q = rig.grow([s], [30])
    with pytest.raises(IndexError, match="forgotten positions 4 to 70"):
        rig.cache.attend(0, q[0], torch.empty_like(q[0]), window=31, sinks=4)
    q = rig.grow([s], [2])  # (positions 70 to 99 are there)
    rig.check([s], [2], q, window=31, sinks=4)
    rig.cache.forget(s, 70, 90)
    q = rig.grow([s], [5])
    rig.check([s], [5], q, window=13, sinks=4)


def test_refusals_of_forgetting_and_what_they_leave(torch):
    rig = Rig(torch, "f32", heads=2, kv_heads=2, dim=64, page=16, pages=40, seed=110)
    a, b = rig.add(), rig.add()
    rig.grow([a, b], [200, 30])
    q = rig.grow([a, b], [3, 1])
    for span in ((-1, 5), (10, 204), (300, 301)):
        with pytest.raises(IndexError, match="forgotten of a sequence of 203"):
            rig.cache.forget(a, *span)
    with pytest.raises(IndexError, match="no sequence"):
        rig.cache.forget(7, 0, 1)
    rig.check([a, b], [3, 1], q, what="the pass is still open", rows=2)
    rig.cache.forget(a, 20, 100)
    with pytest.raises(RuntimeError, match="no pass is open"):
        rig.cache.attend(0, q[0], torch.empty_like(q[0]))
    for span in ((102, 110), (0, 19)):
        with pytest.raises(ValueError, match="has to touch"):
            rig.cache.forget(a, *span)
    rig.cache.forget(a, 50, 40)  # nothing
    rig.cache.forget(a, 90, 110)
    assert rig.cache.info.pages_free == 40 - (13 - 4) - 2  # (pages 2 to 5 of a are nobody's)
    q = rig.grow([a, b], [3, 1])
    out = torch.full_like(q[0], 3.0)
    for mask in (dict(), dict(window=96, sinks=20), dict(window=94, sinks=21), dict(window=1000, sinks=5), dict(sinks=20)):
        with pytest.raises(IndexError, match="forgotten positions 20 to 110"):
            rig.cache.attend(0, q[0], out, **mask)
    for mask, match in ((dict(window=-1, sinks=2), "window"), (dict(window=5, sinks=-1), "sinks")):
        with pytest.raises(ValueError, match=match):
            rig.cache.attend(0, q[0], out, **mask)
    assert bool((out == 3.0).all())
    rig.check([a, b], [3, 1], q, window=94, sinks=20, what="all that is left")  # the first row, at 203, sees from 110 on
    rig.check([a, b], [3, 1], q, window=94, what="no sinks")
    kv = torch.empty(30, 2, 64, device="cuda")
    for start in (0, 19, 60, 109):
        with pytest.raises(IndexError, match="forgotten"):
            rig.cache.read(a, kv, torch.empty_like(kv), start=start, layer=0)
    rig.cache.read(a, kv, torch.empty_like(kv), start=110, layer=0)
    # a sequence that forgot takes no part in prefixes that others share
    kids = [rig.fork(b) for _ in range(4)] + [rig.fork(a, 60)]
    q = rig.grow(kids, [1] * 5)
    with pytest.raises(IndexError, match="forgotten positions 20 to 60"):
        rig.cache.attend(0, q[0], torch.empty_like(q[0]), window=20, sinks=10)
    rig.check(kids, [1] * 5, q, window=1, sinks=10)
    rig.drop(kids.pop())
    q = rig.grow(kids, [1] * 4)
    rig.check(kids, [1] * 4, q)


def test_a_context_with_forgotten_positions_is_not_restored(torch):
    from gradhip import synth
    cfg = synth.Config(synth.ARCH_MODERN, 301, 128, 2, 2, 96)
    model = G.Model.from_tensors(cfg, synth.make_weights(cfg, 31, std=0.08, norm_noise=0.1))
    session = G.Session(model)
    ids = synth.uniform_tokens(40, cfg.vocab, 50)
    want = session.prefill(ids)
    cache = G.Cache(2, 2, 2, 64, pages=8, page_tokens=16)
    s = session.store(cache)
    kept = cache.fork(s)
    cache.forget(s, 3, 20)
    with pytest.raises(IndexError, match="forgotten"):
        session.restore(cache, [s], ids)
    import numpy as np
    got = session.restore(cache, [kept], ids)
    assert np.abs(got - want).max() <= 1e-4 * np.abs(want).max()


def test_sinks_on_other_streams_and_strided_rows(torch):
    rig = Rig(torch, "f16", heads=4, kv_heads=2, dim=64, page=16, pages=60, seed=111)
    s = rig.add()
    rig.grow([s], [700])
    n = 9
    q = rig.grow([s], [n])
    wide = torch.full((n, 4, 67), 5.0, dtype=torch.float16, device="cuda")
    wide[:, :, 1:65] = q[0]
    view, back = wide[:, :, 1:65], torch.full((n + 2, 4, 67), 9.0, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    rig.cache.attend(0, view, back[:n, :, 3:], window=100, sinks=7, stream=side.cuda_stream)
    straight = torch.empty_like(q[0])
    rig.cache.attend(0, q[0], straight, window=100, sinks=7)
    torch.cuda.synchronize()
    assert torch.equal(back[:n, :, 3:], straight)
    assert bool((back[:n, :, :3] == 9.0).all()) and bool((back[n:] == 9.0).all())
    rig.check([s], [n], q, window=100, sinks=7)
