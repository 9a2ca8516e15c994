"""Streams that have gone on for millions of positions and forgotten nearly all of them: the same attention, in steps that take no longer."""
import time

import pytest

import gradhip as G
import test_gpu_cache as base
from test_gpu_cache import TYPES

pytestmark = pytest.mark.gpu
CHUNK = 1 << 16


@pytest.fixture(scope="module")
def torch():
    return base._torch()


class Stream:
    """A sequence whose rows see `sinks` first and `window` last positions; those that it has not forgotten are kept here, in 64 bits."""

    def __init__(self, torch, cache, dtype, sinks, window, seed, kv=2, dim=64, heads=4):
        self.torch, self.cache, self.sinks, self.window, self.heads, self.dtype = torch, cache, sinks, window, heads, dtype
        self.gen, self.shape = torch.Generator().manual_seed(seed), (kv, dim)
        self.seq, self.length = cache.add(), 0
        self.places = torch.zeros(0, dtype=torch.int64)
        self.k, self.v = (torch.zeros(0, kv, dim, dtype=torch.float64) for _ in range(2))

    def rows(self, n, heads=None):
        return self.torch.randn(n, heads or self.shape[0], self.shape[1], generator=self.gen).to(base._ref().DTYPES[self.dtype])

    def keep(self, those):
        self.places, self.k, self.v = self.places[those], self.k[those], self.v[those]

    def forget(self):
        end = self.length - self.window + 1
        self.cache.forget(self.seq, self.sinks, end)
        self.keep((self.places < self.sinks) | (self.places >= end))

    def took(self, k, v):
        self.places = self.torch.cat((self.places, self.torch.arange(self.length, self.length + k.shape[0])))
        self.k, self.v = self.torch.cat((self.k, k.double())), self.torch.cat((self.v, v.double()))
        self.length += k.shape[0]

    def skip(self, n):
        """n positions of which nothing is known."""
        self.forget()
        self.cache.extend([self.seq], [n])
        self.length += n
        self.forget()

    def fill(self):
        """A window of positions that are known."""
        self.forget()
        self.cache.extend([self.seq], [self.window])
        k, v = self.rows(self.window), self.rows(self.window)
        self.cache.append(0, k.cuda(), v.cuda())
        self.took(k, v)

    def truncate(self, length):
        self.cache.truncate(self.seq, length)
        self.length = length
        self.keep(self.places < length)

    def fork(self, seed):
        twin = Stream(self.torch, self.cache, self.dtype, self.sinks, self.window, seed)
        self.cache.drop(twin.seq)
        twin.seq, twin.length, twin.places, twin.k, twin.v = self.cache.fork(self.seq), self.length, self.places, self.k, self.v
        return twin


def step(streams, counts, torch, causal=True, forget=True):
    """A pass: rows that are appended and attend; checked row by row."""
    R, first = base._ref(), streams[0]
    for s in streams:
        if forget:
            s.forget()
    first.cache.extend([s.seq for s in streams], counts)
    parts = [(s.rows(n), s.rows(n), s.rows(n, s.heads)) for s, n in zip(streams, counts)]
    k, v, q = (torch.cat([p[i] for p in parts]).cuda() for i in range(3))
    out = torch.full_like(q, 7.0)
    first.cache.append(0, k, v)
    first.cache.attend(0, q, out, causal=causal, window=first.window, sinks=first.sinks)
    torch.cuda.synchronize()
    at = 0
    for s, n, (pk, pv, pq) in zip(streams, counts, parts):
        start = s.length
        s.took(pk, pv)
        for i in sorted({0, n // 2, n - 1}) if n else ():
            t = start + i
            seen = (s.places > t - s.window) | (s.places < s.sinks)
            if causal:
                seen &= s.places <= t
            last = t + 1 if causal else s.length
            assert int(seen.sum()) == min(last, s.sinks) + last - max(min(last, s.sinks), t - s.window + 1)
            want, allowed = R.attention(pq[i:i + 1].double(), s.k[seen], s.v[seen], int(seen.sum()) - 1, False, 0, 0.0, s.dtype)
            R.assert_within(out[at + i:at + i + 1], want, allowed, f"stream of {s.length}, row {i} of {n}")
        at += n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,sinks", [(16, 5), (64, 70), (16, 0), (128, 1)])
def test_far_streams_beside_near_ones(torch, dtype, page, sinks):
    """Pages that are handed out again are full of NaN, which the kernels of many rows take a way of their own with."""
    window = 300
    cache = G.Cache(1, 4, 2, 64, (CHUNK + 4096) // page, dtype=dtype, page_tokens=page)
    waste = cache.add()
    cache.extend([waste], [CHUNK + 2048])
    bad = torch.full((CHUNK + 2048, 2, 64), float("nan"), dtype=base._ref().DTYPES[dtype], device="cuda")
    cache.append(0, bad, bad)
    cache.drop(waste)
    near, far, short = (Stream(torch, cache, dtype, sinks, window, seed) for seed in range(3))
    step([near, far], [400, 90], torch)
    for _ in range(24):
        far.skip(CHUNK - 7)
    assert far.length > 1_500_000
    far.fill()
    for counts in ([1, 1, 1], [2, 5, 30], [0, 200, 3], [150, 1, 0], [3, 140, 130], [1, 1, 1]):
        step([near, far, short], counts, torch)
    step([far, near], [40, 3], torch, causal=False)
    step([far], [1], torch)
    # back to where it was, and a fork that goes its own way
    far.fill()
    far.truncate(far.length - 20)
    twin = far.fork(9)
    step([far, twin, near], [1, 160, 2], torch, forget=False)
    cache.compact()
    step([twin, far], [1, 1], torch)


def test_steps_of_a_far_stream_take_no_longer(torch):
    """A stream at eight million positions has forgotten 500 thousand pages: sent along, they are 2 MB a step."""
    def steps(skips):
        cache = G.Cache(1, 4, 2, 64, (CHUNK + 4096) // 16, dtype="bf16", page_tokens=16)
        seq, length = cache.add(), 2000
        cache.extend([seq], [2000])
        for _ in range(skips):
            cache.forget(seq, 4, length - 999)
            cache.extend([seq], [CHUNK])
            length += CHUNK
        q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda")
        k, out = q[:, :2], torch.empty_like(q)
        best = 1e9
        for _ in range(6):
            torch.cuda.synchronize()
            start = time.perf_counter()
            for _ in range(30):
                cache.forget(seq, 4, length - 999)
                cache.extend([seq], [1])
                length += 1
                cache.append(0, k, k)
                cache.attend(0, q, out, window=1000, sinks=4)
            torch.cuda.synchronize()
            best = min(best, (time.perf_counter() - start) / 30)
        return best * 1e6

    near, far = steps(0), steps(128)
    print(f"{near:.1f} us a step, {far:.1f} at eight million positions")
    assert far < 3 * near, (near, far)
