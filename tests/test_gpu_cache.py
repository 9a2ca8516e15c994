"""The paged cache (gh_cache_*) on the GPU against its definitions in 64 bits: attention of chunks and single tokens over
pages, appended rows and their rotation, forks, rewinds, copies and compaction, and what the calls refuse."""
import ctypes

import pytest

import gradhip as G

pytestmark = pytest.mark.gpu


def _torch():
    G.device_info()
    ctypes.CDLL("libamdhip64.so")  # one HIP runtime in the process, whoever loads it first
    return pytest.importorskip("torch")


@pytest.fixture(scope="module")
def torch():
    return _torch()


def _ref():
    import cache_reference
    return cache_reference


class Rig:
    """A cache, the same sequences as dense rows in 64 bits, and inputs from a seed."""

    def __init__(self, torch, dtype, layers=1, heads=4, kv_heads=2, dim=64, page=16, pages=64, rope=0.0, seed=1):
        self.torch, self.R = torch, _ref()
        self.dtype, self.rope = dtype, rope
        self.cache = G.Cache(layers, heads, kv_heads, dim, pages, dtype=dtype, page_tokens=page, rope_base=rope)
        self.ref = self.R.Reference(layers, kv_heads, dim, dtype)
        self.gen = torch.Generator().manual_seed(seed)
        self.layers, self.heads, self.kv_heads, self.dim = layers, heads, kv_heads, dim

    def rand(self, *shape, std=1.0):
        return (self.torch.randn(*shape, generator=self.gen) * std).to(self.R.DTYPES[self.dtype])

    def add(self):
        s = self.cache.add()
        self.ref.add(s)
        return s

    def fork(self, seq, length=-1):
        s = self.cache.fork(seq, length)
        self.ref.fork(seq, s, length)
        return s

    def drop(self, seq):
        self.cache.drop(seq)
        self.ref.drop(seq)

    def truncate(self, seq, length):
        self.cache.truncate(seq, length)
        self.ref.truncate(seq, length)

    def grow(self, seqs, counts, k=None, v=None, stream=0):
        """A pass that appends rows in every layer; checks rotated queries; returns the queries per layer (on the GPU)."""
        torch, rows = self.torch, sum(counts)
        before = [self.cache.length(s) for s in seqs]
        self.cache.extend(seqs, counts, stream=stream)
        k = self.rand(self.layers, rows, self.kv_heads, self.dim) if k is None else k
        v = self.rand(self.layers, rows, self.kv_heads, self.dim) if v is None else v
        q = self.rand(self.layers, rows, self.heads, self.dim, std=2.0)
        kd, vd, qd = k.cuda(), v.cuda(), q.cuda()
        turned = torch.empty_like(qd)
        for layer in range(self.layers):
            self.cache.append(layer, kd[layer], vd[layer], qd[layer], turned[layer], stream=stream)
        at = 0
        positions = [b + i for b, n in zip(before, counts) for i in range(n)]
        if self.rope and rows:
            kept = torch.stack([self.R.rotated(k[layer].double(), positions, self.rope).to(k.dtype) for layer in range(self.layers)])
            want = torch.stack([self.R.rotated(q[layer].double(), positions, self.rope) for layer in range(self.layers)])
            # two products, a sum and the sine's and cosine's own error in 32 bits (four steps of 2^-23 of the pair), then the type's rounding
            pair = q.double().unflatten(-1, (-1, 2)).norm(dim=-1).repeat_interleave(2, -1)
            self.R.assert_within(turned, want, 4 * 2.0 ** -23 * pair + self.R.HALF_STEP[self.dtype] * want.abs() + 2.0 ** -25, "rotated queries")
            # what is kept is the kernel's own rounding: read back and held to the same rule, then taken as it is
            got = torch.empty_like(kd)
            for s, b, n in zip(seqs, before, counts):
                if n:
                    self.cache_read_rows(s, b, got[:, at:at + n], stream)
                at += n
            pair = k.double().unflatten(-1, (-1, 2)).norm(dim=-1).repeat_interleave(2, -1)
            full = torch.stack([self.R.rotated(k[layer].double(), positions, self.rope) for layer in range(self.layers)])
            self.R.assert_within(got, full, 4 * 2.0 ** -23 * pair + self.R.HALF_STEP[self.dtype] * kept.double().abs() * 1.01 + 2.0 ** -25, "rotated keys")
            k = got.cpu()
        elif rows:
            assert torch.equal(turned, qd)
        at = 0
        for s, n in zip(seqs, counts):
            self.ref.extend(s, k[:, at:at + n], v[:, at:at + n])
            at += n
        return turned

    def cache_read_rows(self, seq, start, k_out, stream=0):
        self.cache.read(seq, k_out, self.torch.empty_like(k_out), start=start, stream=stream)

    def check(self, seqs, counts, q, causal=True, window=0, scale=0.0, what="", stream=0, out=None):
        torch = self.torch
        out = torch.full_like(q, 7.0) if out is None else out
        for layer in range(self.layers):
            self.cache.attend(layer, q[layer], out[layer], scale=scale, causal=causal, window=window, stream=stream)
        torch.cuda.synchronize()
        at = 0
        for s, n in zip(seqs, counts):
            for layer in range(self.layers):
                if n:
                    want, allowed = self.R.attention(q[layer, at:at + n].cpu().double(), self.ref.k[s][layer], self.ref.v[s][layer],
                                                     self.ref.k[s].shape[1] - n, causal, window, scale, self.dtype)
                    self.R.assert_within(out[layer, at:at + n], want, allowed, f"{what} sequence {s} layer {layer}")
            at += n
        return out

    def check_contents(self, seqs):
        torch = self.torch
        for s in seqs:
            n = self.cache.length(s)
            assert n == self.ref.k[s].shape[1]
            k = torch.empty(self.layers, n, self.kv_heads, self.dim, dtype=self.R.DTYPES[self.dtype], device="cuda")
            v = torch.empty_like(k)
            if n:
                self.cache.read(s, k, v)
            assert torch.equal(k.cpu().double(), self.ref.k[s]) and torch.equal(v.cpu().double(), self.ref.v[s]), s


TYPES = ("f32", "bf16", "f16")
# (heads, kv_heads, head_dim, page_tokens)
HEADS = {"mha64": (3, 3, 64, 64), "grouped128": (8, 2, 128, 16), "one-key80": (5, 1, 80, 32), "dim8": (2, 2, 8, 16), "dim40": (4, 2, 40, 16),
         "dim96": (6, 2, 96, 128), "dim256": (4, 2, 256, 32), "wide-group64": (34, 2, 64, 16), "dim136": (2, 1, 136, 16)}


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_over_ragged_sequences(torch, dtype, heads):
    h, kv, dim, page = HEADS[heads]
    rig = Rig(torch, dtype, heads=h, kv_heads=kv, dim=dim, page=page, pages=4096 // page, seed=3)
    seqs = [rig.add() for _ in range(5)]
    rig.grow(seqs, [1, 33, 0, 150, 402])
    counts = [1, 3, 1, 18, 2]
    q = rig.grow(seqs, counts)
    rig.check(seqs, counts, q, what="causal")
    rig.check(seqs, counts, q, causal=False, what="all positions")
    for window in (1, 2, 37, 130, 1000):
        rig.check(seqs, counts, q, window=window, what=f"window {window}")
    rig.check(seqs, counts, q, causal=False, window=5, what="window ahead")
    rig.check(seqs, counts, q, scale=0.31, what="scale")
    # single tokens
    counts = [1] * 5
    q = rig.grow(seqs, counts)
    rig.check(seqs, counts, q, what="single tokens")


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_of_many_rows_beside_few(torch, dtype, heads):
    h, kv, dim, page = HEADS[heads]
    rig = Rig(torch, dtype, heads=h, kv_heads=kv, dim=dim, page=page, pages=4096 // page, seed=4)
    seqs = [rig.add() for _ in range(4)]
    rig.grow(seqs, [300, 64, 0, 5])
    counts = [200, 1, 131, 70]
    q = rig.grow(seqs, counts)
    rig.check(seqs, counts, q, what="causal")
    rig.check(seqs, counts, q, window=90, what="window")
    rig.check(seqs, counts, q, causal=False, window=150, what="window ahead")


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_never_see_what_they_may_not(torch, dtype):
    """As below, in chunks of many rows: infinities and NaN in the chunk itself, of values and of keys."""
    for dim, heads, kv in ((64, 2, 2), (128, 3, 1), (24, 1, 1)):
        rig = Rig(torch, dtype, heads=heads, kv_heads=kv, dim=dim, page=16, pages=60, seed=5)
        bad = torch.full((1, 960, kv, dim), float("nan")).to(rig.R.DTYPES[dtype])
        bad[:, ::3] = -float("inf")
        waste = rig.add()
        rig.grow([waste], [960], k=bad, v=bad)
        rig.drop(waste)
        s = rig.add()
        rig.grow([s], [133])
        k, v = rig.rand(1, 250, kv, dim), rig.rand(1, 250, kv, dim)
        v[0, 50, :, 3] = float("inf")
        v[0, 120, :, 3] = -float("inf")
        v[0, 120, 0, 9] = float("nan")
        v[0, 200, :, dim - 1] = -float("inf")
        k[0, 180, :, 1] = float("inf")
        k[0, 230, :, 2] = float("nan")
        q = rig.grow([s], [250], k=k, v=v)
        rig.check([s], [250], q, what="later positions")
        rig.check([s], [250], q, window=40, what="behind the window")


@pytest.mark.parametrize("case", ["huge later values", "huge later keys", "rows far apart", "dims far apart", "large", "tiny", "zeros"])
def test_many_rows_of_any_size(torch, case):
    """fp32 chunks whose operands do not fit one power of two per tile, or just do."""
    for dim, heads, kv in ((64, 2, 1), (128, 2, 2), (40, 1, 1), (256, 1, 1)):
        rig = Rig(torch, "f32", heads=heads, kv_heads=kv, dim=dim, page=16, pages=60, seed=23)
        s = rig.add()
        rig.grow([s], [133])
        k, v = rig.rand(1, 250, kv, dim), rig.rand(1, 250, kv, dim)
        if case == "huge later values":
            v[0, 100:] *= 1e30
        elif case == "huge later keys":
            k[0, 120:] *= 1e12
        elif case == "rows far apart":
            v[0, ::7] *= 2.0 ** -30
            k[0, ::5] *= 2.0 ** -25
        elif case == "dims far apart":
            v[0, :, :, ::3] *= 2.0 ** -14
            k[0, :, :, 1::2] *= 2.0 ** -15
        elif case == "large":
            v *= 2.0 ** 58
            k *= 2.0 ** 40
        elif case == "tiny":
            v *= 2.0 ** -58
            k *= 2.0 ** -40
        else:
            v[0, 30:200] = 0.0
            k[0, 60:] = 0.0
        q = rig.grow([s], [250], k=k, v=v)
        if case == "large":
            q *= 2.0 ** -40
        elif case == "tiny":
            q *= 2.0 ** 40
        elif case == "zeros":
            q[0, 17:90] = 0.0
        rig.check([s], [250], q, what=case)
        rig.check([s], [250], q, window=60, what=case)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("before,new", [(0, 1), (0, 2), (0, 15), (0, 16), (0, 17), (0, 64), (0, 131), (15, 1), (16, 1), (31, 2), (63, 70), (127, 129), (1000, 1), (2047, 5)])
def test_attend_at_the_edges_of_pages_and_tiles(torch, dtype, before, new):
    rig = Rig(torch, dtype, heads=2, kv_heads=1, dim=64, page=16, pages=160, seed=before + new)
    s = rig.add()
    if before:
        rig.grow([s], [before])
    q = rig.grow([s], [new])
    rig.check([s], [new], q)
    rig.check([s], [new], q, window=20)


@pytest.mark.parametrize("dtype", TYPES)
def test_rotated_rows_at_near_and_far_positions(torch, dtype):
    rig = Rig(torch, dtype, layers=2, heads=4, kv_heads=2, dim=64, page=64, pages=64, rope=10000.0, seed=9)
    seqs = [rig.add() for _ in range(3)]
    rig.grow(seqs, [70, 1, 13])
    q = rig.grow(seqs, [2, 5, 1])
    rig.check(seqs, [2, 5, 1], q)


def test_rotation_keeps_its_digits_at_a_million_positions(torch):
    R = _ref()
    cache = G.Cache(1, 2, 1, 64, pages=2100, dtype="f32", page_tokens=1024, rope_base=500000.0)
    s = cache.add()
    cache.extend([s], [2_000_003])  # contents are nobody's business here
    cache.extend([s], [3])
    k, q = torch.randn(3, 1, 64), torch.randn(3, 2, 64)
    turned = torch.empty(3, 2, 64, device="cuda")
    cache.append(0, k.cuda(), k.cuda(), q.cuda(), turned)
    got = torch.empty(3, 1, 64, device="cuda")
    cache.read(s, got, torch.empty_like(got), start=2_000_003, layer=0)
    positions = [2_000_003, 2_000_004, 2_000_005]
    for x, y in ((k, got), (q, turned)):
        pair = x.double().unflatten(-1, (-1, 2)).norm(dim=-1).repeat_interleave(2, -1)
        R.assert_within(y, R.rotated(x.double(), positions, 500000.0), 5 * 2.0 ** -23 * pair, "far rotation")


@pytest.mark.parametrize("dtype", TYPES)
def test_what_a_row_may_not_see_never_reaches_it(torch, dtype):
    """Infinities and NaN in pages' unused places, in later positions, behind the window, in other sequences."""
    for dim, heads, kv in ((64, 2, 1), (128, 4, 2), (24, 1, 1)):
        rig = Rig(torch, dtype, heads=heads, kv_heads=kv, dim=dim, page=16, pages=40, seed=5)
        bad = torch.full((1, 600, kv, dim), float("nan")).to(rig.R.DTYPES[dtype])
        bad[:, ::2] = float("inf")
        waste = rig.add()
        rig.grow([waste], [600], k=bad, v=bad)
        rig.drop(waste)  # its pages are handed out again, full of that
        s = rig.add()
        rig.grow([s], [70])
        k, v = rig.rand(1, 20, kv, dim), rig.rand(1, 20, kv, dim)
        v[0, 9, :, 3] = float("inf")
        v[0, 12, :, 5] = float("nan")
        v[0, 12, :, 3] = -float("inf")
        v[0, 17, 0, dim - 1] = -float("inf")
        k[0, 19, :, 2] = float("nan")
        q = rig.grow([s], [20], k=k, v=v)
        rig.check([s], [20], q, what="later positions")
        rig.check([s], [20], q, window=4, what="behind the window")
        q = rig.grow([s], [1])
        rig.check([s], [1], q, what="seen by all")
        rig.check([s], [1], q, window=2, what="window of two")


def test_rows_whose_scores_are_all_minus_infinity_are_nan(torch):
    cache = G.Cache(1, 1, 1, 64, pages=4, dtype="f32")
    s = cache.add()
    cache.extend([s], [2])
    k = torch.full((2, 1, 64), -float("inf"), device="cuda")
    q = torch.ones(2, 1, 64, device="cuda")
    out = torch.zeros_like(q)
    cache.append(0, k, torch.ones_like(k))
    cache.attend(0, q, out)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_of_the_types_range(torch, dtype):
    """Scores far apart and far from zero: the largest decides, nothing overflows."""
    rig = Rig(torch, dtype, heads=2, kv_heads=2, dim=64, page=16, pages=40, seed=8)
    s = rig.add()
    k = rig.rand(1, 300, 2, 64)
    k[0, 123] *= 100.0
    k[0, 250] *= -100.0
    rig.grow([s], [300], k=k)
    q = rig.grow([s], [3])
    rig.check([s], [3], q)
    rig.check([s], [3], q, scale=3.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_unaligned_rows(torch, dtype):
    rig = Rig(torch, dtype, heads=4, kv_heads=2, dim=64, page=16, pages=40, seed=6)
    s = rig.add()
    rig.grow([s], [50])
    n = 6
    t = rig.R.DTYPES[dtype]
    # one allocation of [rows, q | k | v heads, dim + 3] shifted by one element: nothing is aligned
    wide = rig.rand(n * 8 * 67 + 1).cuda()[1:].view(n, 8, 67)
    q, k, v = wide[:, :4, :64], wide[:, 4:6, :64], wide[:, 6:, 1:65]
    rig.cache.extend([s], [n])
    turned = torch.zeros(4, n + 2, 64, dtype=t, device="cuda").transpose(0, 1)  # heads outermost, two rows more
    rig.cache.append(0, k, v, q, turned)
    assert torch.equal(turned[:n], q) and not turned[n:].any()
    rig.ref.extend(s, k[None].cpu(), v[None].cpu())
    hidden = torch.full((n + 3, 4, 65), 5.0, dtype=t, device="cuda")
    out = hidden[..., 1:]
    rig.cache.attend(0, q, out)
    want, allowed = rig.R.attention(q.cpu().double(), rig.ref.k[s][0], rig.ref.v[s][0], 50, dtype=dtype)
    rig.R.assert_within(out[:n], want, allowed)
    assert (hidden[n:] == 5.0).all() and (hidden[..., 0] == 5.0).all(), "rows and elements beyond are left as they were"
    # the queries' own place for the outputs, and a broadcast key
    own = turned.clone()
    rig.cache.attend(0, own, own)
    rig.R.assert_within(own[:n], want, allowed)
    one = rig.rand(1, 1, 64).cuda().expand(n, 2, 64)
    rig.cache.append(0, one, one)
    got = torch.empty(n, 2, 64, dtype=t, device="cuda")
    rig.cache.read(s, got, torch.empty_like(got), start=50, layer=0)
    assert torch.equal(got, one)


@pytest.mark.parametrize("dtype", TYPES)
def test_forks_share_until_somebody_writes(torch, dtype):
    rig = Rig(torch, dtype, layers=3, heads=4, kv_heads=2, dim=64, page=16, pages=64, seed=12)
    parent = rig.add()
    rig.grow([parent], [40])
    free = rig.cache.pages_free
    kids = [rig.fork(parent) for _ in range(3)] + [rig.fork(parent, 32), rig.fork(parent, 7), rig.fork(parent, 0)]
    assert rig.cache.pages_free == free
    seqs = [kids[0], parent, kids[3], kids[4], kids[1], kids[5]]
    counts = [1, 2, 9, 1, 20, 3]
    q = rig.grow(seqs, counts)
    rig.check(seqs, counts, q)
    rig.check_contents([parent] + kids)
    rig.drop(parent)
    counts = [5, 1]
    q = rig.grow([kids[2], kids[1]], counts)  # kids[2] is the last who holds the parent's last page
    rig.check([kids[2], kids[1]], counts, q)
    for k in kids:
        rig.drop(k) if k in (kids[0], kids[4]) else rig.truncate(k, min(3, rig.cache.length(k)))
    rest = [kids[1], kids[2], kids[3], kids[5]]
    rig.check_contents(rest)
    q = rig.grow(rest, [4, 1, 30, 0])
    rig.check(rest, [4, 1, 30, 0], q)
    rig.check_contents(rest)
    for k in rest:
        rig.drop(k)
    assert rig.cache.pages_free == 64 and rig.cache.info.sequences == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", ["mha64", "grouped128", "one-key80", "dim256"])
def test_many_samples_of_one_prompt(torch, dtype, heads):
    """Sequences that share most of their pages are attended to together: as many as fill several tiles, of lengths of their
    own behind the prompt, beside others that share nothing and two families more."""
    h, kv, dim, page = HEADS[heads]
    rig = Rig(torch, dtype, heads=h, kv_heads=kv, dim=dim, page=page, pages=8192 // page, seed=21)
    a, b, lone = rig.add(), rig.add(), rig.add()
    rig.grow([a, b, lone], [700, 333, 290])
    kids = [rig.fork(a) for _ in range(19)] + [rig.fork(a, 400), rig.fork(a, 150)]
    rig.grow(kids[:5], [3, 70, 1, 12, 30])
    others = [rig.fork(b) for _ in range(2)]
    seqs = kids[:7] + [lone, b] + kids[7:] + others + [a]
    for counts in ([1] * len(seqs), [1 + (i % 3 == 0) for i in range(len(seqs))]):
        q = rig.grow(seqs, counts)
        rig.check(seqs, counts, q, what="shared")
        rig.check(seqs, counts, q, window=200, what="window")
    counts = [40 if i == 4 else 1 for i in range(len(seqs))]  # one of them with many rows
    q = rig.grow(seqs, counts)
    out = rig.check(seqs, counts, q, what="beside a chunk")
    again = rig.check(seqs, counts, q, what="again")
    assert torch.equal(out, again)
    rig.check_contents(kids[:3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", ["mha64", "grouped128", "one-key80", "dim256"])
def test_many_samples_of_a_long_prompt(torch, dtype, heads):
    """Prefixes of so many bytes that they are read for all members together, in several common tiles: 33 samples, among
    them one that only shares a shorter part, beside a sequence of its own."""
    h, kv, dim, page = HEADS[heads]
    size = 4 if dtype == "f32" else 2
    prompt = max(300, 50_000_000 // (33 * 2 * kv * dim * size)) // page * page + 5
    rig = Rig(torch, dtype, heads=h, kv_heads=kv, dim=dim, page=page, pages=(2 * prompt + 40 * 128) // page + 50, seed=31)
    a, lone = rig.add(), rig.add()
    rig.grow([a, lone], [prompt, 290])
    kids = [rig.fork(a) for _ in range(32)] + [rig.fork(a, prompt - page - 7)]
    rig.grow(kids[:3], [3, 17, 1])
    seqs = kids[:20] + [lone] + kids[20:]
    for counts in ([1] * len(seqs), [1 + (i % 3 == 0) for i in range(len(seqs))]):
        q = rig.grow(seqs, counts)
        out = rig.check(seqs, counts, q, what="shared")
        assert torch.equal(out, rig.check(seqs, counts, q, what="again"))
    rig.check_contents(kids[:2])


@pytest.mark.parametrize("dtype", TYPES)
def test_long_contexts_beside_a_chunk(torch, dtype):
    """Single tokens over so much that they get a launch of their own beside the chunk's: with a common prefix (no window)
    and without (a window), and the other way round, a chunk of one of them."""
    rig = Rig(torch, dtype, heads=16, kv_heads=8, dim=128, page=64, pages=180, seed=32)
    a, chunk = rig.add(), rig.add()
    rig.grow([a, chunk], [5500, 70])
    kids = [rig.fork(a) for _ in range(17)]
    for seqs, counts in ((kids[:9] + [chunk] + kids[9:], [1] * 9 + [90] + [1] * 8), ([chunk] + kids, [3, 1, 75] + [1] * 15)):
        q = rig.grow(seqs, counts)
        for window in (0, 5200):
            out = rig.check(seqs, counts, q, window=window, what=f"window {window}")
            assert torch.equal(out, rig.check(seqs, counts, q, window=window, what="again"))


def test_long_lists_of_pages(torch):
    """More pages than a launch's own list takes: copies, reads, compaction."""
    rig = Rig(torch, "bf16", layers=2, heads=1, kv_heads=1, dim=8, page=16, pages=3200, seed=22)
    a, b, c = rig.add(), rig.add(), rig.add()
    rig.grow([a, b, c], [9000, 20000, 10007])
    twin = rig.cache.copy(c)
    rig.ref.fork(c, twin)
    rig.drop(a)
    rig.drop(c)
    rig.cache.compact()
    rig.check_contents([b, twin])
    part = torch.empty(9991, 1, 8, dtype=torch.bfloat16, device="cuda")
    rig.cache.read(twin, part, torch.empty_like(part), start=13, layer=1)
    assert torch.equal(part.cpu().double(), rig.ref.k[twin][1, 13:13 + 9991])


def test_a_rewound_sequence_takes_other_tokens(torch):
    """Drafted tokens of which the first are kept."""
    rig = Rig(torch, "f16", heads=4, kv_heads=4, dim=64, page=16, pages=32, rope=10000.0, seed=13)
    a, b = rig.add(), rig.add()
    rig.grow([a, b], [45, 61])
    for kept in (1, 3, 0, 5):
        before = [rig.cache.length(a), rig.cache.length(b)]
        q = rig.grow([a, b], [5, 5])
        rig.check([a, b], [5, 5], q)
        rig.truncate(a, before[0] + kept)
        rig.truncate(b, before[1] + 5 - kept)
    rig.check_contents([a, b])


@pytest.mark.parametrize("dtype", TYPES)
def test_copies_and_compaction_keep_contents(torch, dtype):
    rig = Rig(torch, dtype, layers=2, heads=2, kv_heads=2, dim=64, page=16, pages=48, seed=14)
    seqs = [rig.add() for _ in range(6)]
    rig.grow(seqs, [5, 40, 16, 100, 33, 1])
    twin = rig.cache.copy(seqs[3])
    rig.ref.fork(seqs[3], twin)
    shared = rig.fork(seqs[4], 30)
    for s in (seqs[1], seqs[0], seqs[3]):
        rig.drop(s)
    rest = [seqs[2], seqs[4], seqs[5], twin, shared]
    used = rig.cache.compact()
    assert used == 48 - rig.cache.pages_free
    rig.check_contents(rest)
    assert rig.cache.compact() == used
    q = rig.grow(rest, [3, 1, 2, 1, 17])
    rig.check(rest, [3, 1, 2, 1, 17], q)
    rig.check_contents(rest)
    # into another cache, larger, with other query heads
    other = G.Cache(2, 4, 2, 64, pages=200, dtype=dtype, page_tokens=16)
    moved = {s: rig.cache.copy(s, to=other) for s in rest}
    for s, t in moved.items():
        n = other.length(t)
        k = torch.empty(2, n, 2, 64, dtype=rig.R.DTYPES[dtype], device="cuda")
        v = torch.empty_like(k)
        other.read(t, k, v)
        assert torch.equal(k.cpu().double(), rig.ref.k[s]) and torch.equal(v.cpu().double(), rig.ref.v[s])
        if n > 4:
            part = torch.empty(n - 4, 2, 64, dtype=k.dtype, device="cuda")
            other.read(t, part, torch.empty_like(part), start=3, layer=1)
            assert torch.equal(part, k[1, 3:n - 1])


def test_pages_beyond_four_gigabytes(torch):
    """Offsets into the pool past 32 bits: the last pages of a pool of 9 GB."""
    rig = Rig(torch, "f32", layers=4, heads=4, kv_heads=4, dim=128, page=256, pages=2300, seed=15)
    assert rig.cache.info.pool_bytes > 9_000_000_000
    filler = rig.cache.add()
    rig.cache.extend([filler], [256 * 2290])
    s, t = rig.add(), rig.add()
    rig.grow([s, t], [300, 270])
    q = rig.grow([s, t], [3, 1])
    rig.check([s, t], [3, 1], q)
    rig.check_contents([s, t])
    twin = rig.cache.copy(s)
    rig.ref.fork(s, twin)
    rig.check_contents([twin])


def test_the_same_call_gives_the_same_bits(torch):
    """Positions dealt to many workgroups, which arrive in any order."""
    rig = Rig(torch, "bf16", heads=8, kv_heads=2, dim=128, page=64, pages=300, seed=16)
    s = rig.add()
    rig.grow([s], [16000])
    q = rig.grow([s], [2])
    first = rig.check([s], [2], q).clone()
    for _ in range(20):
        out = torch.empty_like(first)
        rig.cache.attend(0, q[0], out[0])
        assert torch.equal(out, first)


def test_a_pass_without_rows(torch):
    cache = G.Cache(1, 2, 2, 64, pages=4)
    a = cache.add()
    empty = torch.empty(0, 2, 64, device="cuda")
    for seqs, counts in (([], []), ([a], [0])):
        cache.extend(seqs, counts)
        assert cache.info.pass_rows == 0
        cache.append(0, empty, empty)
        cache.attend(0, empty, empty)
    assert cache.length(a) == 0


def test_calls_on_several_streams_keep_their_order(torch):
    rig = Rig(torch, "f32", heads=4, kv_heads=2, dim=64, page=16, pages=600, seed=17)
    streams = [torch.cuda.Stream() for _ in range(3)]
    s = rig.add()
    rig.grow([s], [4000])
    torch.cuda.synchronize()
    for i in range(6):
        a, b, c = (streams[(i + j) % 3] for j in range(3))
        k, v, q = rig.rand(2, 2, 64), rig.rand(2, 2, 64), rig.rand(2, 4, 64)
        kd, vd, qd = k.cuda(), v.cuda(), q.cuda()
        out = torch.empty_like(qd)
        torch.cuda.synchronize()
        rig.cache.extend([s], [2], stream=a.cuda_stream)
        rig.cache.append(0, kd, vd, stream=b.cuda_stream)
        rig.cache.attend(0, qd, out, stream=c.cuda_stream)
        torch.cuda.synchronize()
        rig.ref.extend(s, k[None], v[None])
        want, allowed = rig.R.attention(q.double(), rig.ref.k[s][0], rig.ref.v[s][0], 4000 + 2 * i)
        rig.R.assert_within(out, want, allowed)


def test_a_stream_may_end_before_the_cache(torch):
    """A call waits for the one before also where that one's stream is gone (as a session's is with the session)."""
    hip = ctypes.CDLL("libamdhip64.so")
    rig = Rig(torch, "f32", heads=4, kv_heads=2, dim=64, page=16, pages=600, seed=19)
    s = rig.add()
    rig.grow([s], [3000])
    for i in range(4):
        k, v, q = rig.rand(2, 2, 64), rig.rand(2, 2, 64), rig.rand(2, 4, 64)
        kd, vd, qd = k.cuda(), v.cuda(), q.cuda()
        out = torch.empty_like(qd)
        torch.cuda.synchronize()
        for call in (lambda st: rig.cache.extend([s], [2], stream=st), lambda st: rig.cache.append(0, kd, vd, stream=st),
                     lambda st: rig.cache.attend(0, qd, out, stream=st)):
            made = ctypes.c_void_p()
            assert hip.hipStreamCreate(ctypes.byref(made)) == 0
            call(made.value)
            assert hip.hipStreamDestroy(made) == 0
        torch.cuda.synchronize()
        rig.ref.extend(s, k[None], v[None])
        want, allowed = rig.R.attention(q.double(), rig.ref.k[s][0], rig.ref.v[s][0], 3000 + 2 * i)
        rig.R.assert_within(out, want, allowed)


def test_two_caches_at_work_beside_each_other(torch):
    rigs = [Rig(torch, t, heads=4, kv_heads=2, dim=64, page=16, pages=600, seed=18) for t in ("f32", "bf16")]
    streams = [torch.cuda.Stream() for _ in rigs]
    passes = []
    for rig in rigs:
        s = rig.add()
        rig.grow([s], [5000])
        passes.append((s, rig.grow([s], [4])))
    torch.cuda.synchronize()
    outs = [torch.empty_like(q) for _, q in passes]
    for _ in range(10):
        for rig, (s, q), out, stream in zip(rigs, passes, outs, streams):
            rig.cache.attend(0, q[0], out[0], stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for rig, (s, q), out in zip(rigs, passes, outs):
        want, allowed = rig.R.attention(q[0].cpu().double(), rig.ref.k[s][0], rig.ref.v[s][0], 5000, dtype=rig.dtype)
        rig.R.assert_within(out[0], want, allowed)


def test_a_stream_under_capture_is_refused(torch):
    cache = G.Cache(1, 2, 2, 64, pages=4)
    s = cache.add()
    cache.extend([s], [1])
    x = torch.zeros(1, 2, 64, device="cuda")
    cache.append(0, x, x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
        y = x + 1
        for call in (lambda: cache.attend(0, x, x, stream=side.cuda_stream), lambda: cache.extend([s], [1], stream=side.cuda_stream),
                     lambda: cache.compact(stream=side.cuda_stream)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert (y == 1).all() and cache.length(s) == 1


def test_refusals(torch):
    cache = G.Cache(2, 4, 2, 64, pages=4, dtype="f32", page_tokens=16)
    a, b = cache.add(), cache.add()
    assert (a, b) == (0, 1)
    q, kv = torch.zeros(8, 4, 64, device="cuda"), torch.zeros(8, 2, 64, device="cuda")
    with pytest.raises(RuntimeError, match="no pass is open"):
        cache.attend(0, q, q)
    with pytest.raises(RuntimeError, match="no pass is open"):
        cache.append(0, kv, kv)
    with pytest.raises(IndexError, match="no sequence 2"):
        cache.extend([2], [1])
    with pytest.raises(IndexError, match="no sequence -1"):
        cache.fork(-1)
    with pytest.raises(ValueError, match="twice"):
        cache.extend([a, a], [1, 1])
    with pytest.raises(ValueError, match="negative"):
        cache.extend([a], [-1])
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.extend([a, b], [33, 17])
    assert cache.length(a) == 0 and cache.length(b) == 0 and cache.pages_free == 4
    cache.extend([a, b], [20, 3])
    with pytest.raises(IndexError, match="no layer 2"):
        cache.attend(2, torch.zeros(23, 4, 64, device="cuda"), torch.zeros(23, 4, 64, device="cuda"))
    for bad, match in ((q, "shape"), (torch.zeros(23, 4, 64, device="cuda", dtype=torch.bfloat16), "bfloat16"), (torch.zeros(23, 4, 64), "cpu"),
                       (torch.zeros(23, 2, 64, device="cuda"), "shape"), (torch.zeros(23, 4, 128, device="cuda")[..., ::2], "dense")):
        with pytest.raises(ValueError, match=match):
            cache.attend(0, bad, torch.zeros(23, 4, 64, device="cuda"))
    fine = torch.zeros(23, 4, 64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        cache.attend(0, fine, torch.zeros(1, 4, 64, device="cuda").expand(23, 4, 64))
    with pytest.raises(ValueError, match="window"):
        cache.attend(0, fine, fine, window=-1)
    for scale in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            cache.attend(0, fine, fine, scale=scale)
    with pytest.raises(ValueError, match="go together"):
        cache.append(0, torch.zeros(23, 2, 64, device="cuda"), torch.zeros(23, 2, 64, device="cuda"), fine)
    with pytest.raises(IndexError, match="fork"):
        cache.fork(b, 4)
    with pytest.raises(IndexError, match="kept"):
        cache.truncate(b, 4)
    with pytest.raises(IndexError, match="positions out of range"):
        cache.read(b, torch.zeros(2, 4, 2, 64, device="cuda"), torch.zeros(2, 4, 2, 64, device="cuda"))
    with pytest.raises(ValueError, match="layer is named"):
        cache.read(b, torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"))
    with pytest.raises(ValueError, match="different"):
        cache.copy(b, to=G.Cache(2, 4, 2, 64, pages=4, dtype="bf16", page_tokens=16))
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.copy(a)
    assert cache.info.sequences == 2
    cache.drop(a)
    with pytest.raises(IndexError, match="no sequence 0"):
        cache.length(a)
    with pytest.raises(RuntimeError, match="no pass is open"):
        cache.attend(0, fine, fine)
    assert cache.add() == a


def test_a_model_of_layers_over_a_serving_run(torch):
    """Requests come, grow by chunks and tokens of their own, are forked, rewound, moved and end; every pass's outputs are right."""
    rig = Rig(torch, "bf16", layers=2, heads=8, kv_heads=2, dim=64, page=16, pages=90, rope=10000.0, seed=20)
    import random
    rng = random.Random(4)
    alive = []
    for step in range(14):
        if len(alive) < 5:
            alive.append(rig.add())
        if step in (4, 8):
            alive.append(rig.fork(rng.choice(alive)))
        if step in (6, 11):
            gone = alive.pop(rng.randrange(len(alive)))
            rig.drop(gone)
            rig.cache.compact()
        if step == 9:
            s = rng.choice(alive)
            rig.truncate(s, rig.cache.length(s) // 2)
        counts = [rng.choice((1, 1, 1, 7, 40)) if rig.cache.length(s) else rng.randint(1, 70) for s in alive]
        q = rig.grow(alive, counts)
        rig.check(alive, counts, q, what=f"step {step}")
    rig.check_contents(alive)
