"""Picks among tens of thousands of equal small weights (gh_sample) on the GPU, against whole-number arithmetic.

A row has a few different logits, each many times.  Its w are taken to 2^-160 and summed as whole numbers, so that cuts and picks are the
definition's; a uniform is left out only where it is within 2^-40 of a border, as the header has it."""
import decimal

import numpy as np
import pytest

import test_gpu_cache as base
from test_gpu_sample import call

pytestmark = pytest.mark.gpu
ONE = 1 << 160


@pytest.fixture(scope="module")
def torch():
    return base._torch()


class Row:
    """The definition for a row of few different logits, one of which is the largest by far or by little."""

    def __init__(self, x, temperature, top_k, top_p):
        self.values = sorted(set(x.tolist()), reverse=True)
        with decimal.localcontext() as ctx:
            ctx.prec = 70
            top, t = decimal.Decimal(self.values[0]), decimal.Decimal(float(np.float32(temperature)))
            self.w = [int(((decimal.Decimal(v) - top) / t).exp() * ONE) for v in self.values]
        counts = [int((x == v).sum()) for v in self.values]
        if top_k:
            left = top_k
            for c, n in enumerate(counts):
                counts[c] = min(n, left)
                left -= counts[c]
        total = sum(n * w for n, w in zip(counts, self.w))
        p, q = float(np.float32(top_p)).as_integer_ratio()  # the first n of a value with sum + (n - 1) w < p / q total
        self.kept, before = [], 0
        for n, w in zip(counts, self.w):
            room = p * total - q * before
            fit = max(0, -(-room // (q * w))) if top_p < 1 else n
            self.kept.append(min(n, fit))
            before += self.kept[-1] * w
        self.kept[0] = max(self.kept[0], 1)
        self.sum = sum(n * w for n, w in zip(self.kept, self.w))
        self.upto = [np.minimum(np.cumsum(x == v), n) for v, n in zip(self.values, self.kept)]  # kept up to an index, by value

    def running(self, i):
        return sum(int(n[i]) * w for n, w in zip(self.upto, self.w)) if i >= 0 else 0

    def pick(self, u):
        """The index; None where u is within 2^-40 of a border."""
        p, q = float(u).as_integer_ratio()
        target = p * self.sum // q
        low, high = 0, len(self.upto[0]) - 1
        while low < high:
            mid = (low + high) // 2
            low, high = (low, mid) if self.running(mid) >= target else (mid + 1, high)
        near = self.sum >> 40
        return low if self.running(low) >= target + near and self.running(low - 1) < target - near else None


def check(torch, x, settings, seed, draws=48):
    rng = np.random.default_rng(seed)
    row = Row(x.double().numpy(), settings.get("temperature", 1.0), settings.get("top_k", 0), settings.get("top_p", 1.0))
    u = (rng.integers(1, 2 ** 24, draws) / 2.0 ** 24).astype(np.float32)
    ids, _ = call(torch, x.cuda().expand(draws, -1), u.tolist(), **settings)
    want = [row.pick(v) for v in u]
    sure = [i for i, v in enumerate(want) if v is not None]
    assert len(sure) > draws * 0.8
    wrong = [(float(u[i]), int(ids[i]), want[i]) for i in sure if ids[i] != want[i]]
    assert not wrong, f"{settings}: {len(wrong)} of {len(sure)}, (uniform, pick, wanted): {wrong[:4]}"
    # the last of what is kept: a uniform of 1 picks it
    last = int(np.flatnonzero(np.diff(sum(row.upto), prepend=0))[-1])
    ids, _ = call(torch, x.cuda().expand(2, -1), [1.0, 1.0], **settings)
    assert list(ids) == [last, last], (settings, list(ids), last)


DTYPE = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("vocab,tail,top_p", [(2 ** 20, -18.03, 0.995), (128000, -20.8, 0.9999), (2 ** 20, -20.79, 0.9995), (50257, -18.03, 0.9999), (2 ** 20, -14.0, 0.6)])
def test_equal_tails(torch, dtype, vocab, tail, top_p):
    """One large logit and equal small ones: the cut falls among them."""
    for at in (0, vocab // 3, vocab - 1):
        x = torch.full((vocab,), tail, dtype=getattr(torch, DTYPE[dtype]))
        x[at] = 0.0
        check(torch, x, dict(top_p=top_p), seed=at)
    check(torch, x, dict(top_k=vocab - 1000, top_p=top_p), seed=1)
    check(torch, x, dict(), seed=2)


@pytest.mark.parametrize("dtype", base.TYPES)
def test_short_tails_behind_equal_ones(torch, dtype):
    """A million equal tokens above the bucket that the cut falls into, which has few; large ones in every stretch of the row."""
    vocab = 2 ** 20
    x = torch.full((vocab,), -15.0, dtype=getattr(torch, DTYPE[dtype]))
    x[::8001] = 0.0
    x[500::1047] = -17.0
    m, n = int((x == 0.0).sum()), int((x == -17.0).sum())
    for share in (0.1, 0.5, 0.9):
        small, rest = float(np.exp(-17.0)) * n, m + float(np.exp(-15.0)) * (vocab - m - n)
        check(torch, x, dict(top_p=(rest + share * small) / (rest + small)), seed=n)


@pytest.mark.parametrize("dtype", base.TYPES)
def test_tails_of_a_few_values_without_a_place_on_the_grid(torch, dtype):
    """Two steps of equal logits, at temperatures for which the buckets of the chunks have no place, and for which all are in one."""
    for vocab in (9001, 262144):
        x = torch.full((vocab,), -1.0, dtype=getattr(torch, DTYPE[dtype]))
        x[::3] = -1.0625
        x[7] = 0.0
        for temperature in (0.0625, 0.0500000007450580596923828125, 1.0, 1000.0):
            check(torch, x, dict(temperature=temperature, top_p=0.8), seed=vocab)
        check(torch, x + 4096 if dtype == "f32" else x, dict(temperature=0.0625, top_p=0.97), seed=vocab)
