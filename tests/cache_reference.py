"""A paged cache's operators by their definitions, in 64 bits, on the CPU; and how far a kernel's outputs may be from them."""
import math

import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {name: torch.finfo(t).eps / 2 for name, t in DTYPES.items()}


def rotated(x, positions, base):
    """x [rows, heads, dim] in double, pairs (2j, 2j + 1) turned by position * base^(-2j / dim)."""
    dim = x.shape[-1]
    angle = torch.as_tensor(positions, dtype=torch.float64)[:, None, None] * float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    a, b = x[..., 0::2], x[..., 1::2]
    out = torch.empty_like(x)
    out[..., 0::2] = a * angle.cos() - b * angle.sin()
    out[..., 1::2] = a * angle.sin() + b * angle.cos()
    return out


def attention(q, k, v, first, causal=True, window=0, scale=0.0, dtype="f32"):
    """Rows q [n, heads, dim] at positions first.. over k, v [len, kv_heads, dim]; all double.  Returns (out, allowance).

    What a row may not see takes no part: it is left out, not multiplied by zero.

    The allowance per element.  Scores: a product of d terms summed in 32 bits, each of the d + 2 roundings at most 2^-23
    of the terms' absolute sum (sums inside the matrix cores may truncate: a whole step, not half), independent, so
    sqrt(d + 2) of them and a factor 4; the exponent's own rounding, 2^-23 of the scores' range.  An error e of a score is a relative
    error e of its probability, which the sum in the denominator can double.  The sum over n positions: sqrt(n + 8) steps of 2^-23,
    factor 4.  Both relative to A = sum p |v| / sum p.  16-bit types: the rounding of p, half a step of the type, relative to A as
    well, and the output's own rounding, half a step of it."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    length = k.shape[0]
    scale = scale or dim ** -0.5
    out, allowed = torch.empty_like(q), torch.empty_like(q)
    u = torch.arange(length)
    for i in range(n):
        t = first + i
        seen = torch.ones(length, dtype=torch.bool)
        if causal:
            seen &= u <= t
        if window:
            seen &= u > t - window
        for h in range(heads):
            kk, vv = k[seen, h // group], v[seen, h // group]
            z = kk @ q[i, h] * scale
            p = torch.softmax(z, 0)
            out[i, h] = (p[:, None] * vv).sum(0)
            absolute = (p[:, None] * vv.abs()).sum(0)
            size = (kk.abs() @ q[i, h].abs()).max() * abs(scale)
            span = z.max() - z.min()
            wrong = 4 * math.sqrt(dim + 2) * 2.0 ** -23 * size + 2.0 ** -23 * (span + z.abs().max())
            of_sum = 4 * math.sqrt(int(seen.sum()) + 8) * 2.0 ** -23
            allowed[i, h] = (2 * wrong + of_sum) * absolute
            if dtype != "f32":
                allowed[i, h] += HALF_STEP[dtype] * (absolute + out[i, h].abs()) * (1 + 2.0 ** -6)
            else:
                allowed[i, h] += 2.0 ** -24 * out[i, h].abs()
    return out, allowed + 1e-30 + (2.0 ** -24 if dtype == "f16" else 0.0)  # (the smallest step of f16)


class Reference:
    """The sequences of a cache as dense rows: the operators' definitions without pages."""

    def __init__(self, layers, kv_heads, dim, dtype):
        self.layers, self.kv_heads, self.dim, self.dtype = layers, kv_heads, dim, dtype
        self.k, self.v = {}, {}

    def add(self, seq):
        self.k[seq] = torch.zeros(self.layers, 0, self.kv_heads, self.dim, dtype=torch.float64)
        self.v[seq] = self.k[seq].clone()

    def fork(self, seq, out, length=-1):
        n = self.k[seq].shape[1] if length == -1 else length
        self.k[out], self.v[out] = self.k[seq][:, :n].clone(), self.v[seq][:, :n].clone()

    def truncate(self, seq, length):
        self.k[seq], self.v[seq] = self.k[seq][:, :length], self.v[seq][:, :length]

    def drop(self, seq):
        del self.k[seq], self.v[seq]

    def extend(self, seq, k, v):
        """k, v [layers, rows, kv_heads, dim], in any type."""
        self.k[seq] = torch.cat((self.k[seq], k.double()), 1)
        self.v[seq] = torch.cat((self.v[seq], v.double()), 1)


def assert_within(got, want, allowed, what=""):
    got = got.detach().cpu().double()
    bad_nan = torch.isnan(got) != torch.isnan(want)
    assert not bad_nan.any(), f"{what}: NaN in {int(bad_nan.sum())} places where it should not be, or missing"
    infinite = torch.isinf(want)
    assert torch.equal(got[infinite], want[infinite]), f"{what}: infinities differ"
    fine = torch.isfinite(want)
    assert torch.isfinite(got[fine]).all(), f"{what}: infinite where it should not be"
    share = ((got[fine] - want[fine]).abs() / allowed[fine]).max() if fine.any() else torch.tensor(0.0)
    assert share <= 1.0, f"{what}: {float(share):.3g} of what is allowed"
