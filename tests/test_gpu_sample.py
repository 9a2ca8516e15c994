"""Sampling by row (gh_sample) on the GPU against its definition in 64 bits.

Picks are whole numbers and have to be the definition's; the inputs' uniforms are random multiples of 2^-24 and borders are not, but where both are
exact (equal logits).  Probabilities are rounded to 32 bits once: half a step, and 2^-40 for the 64-bit sums."""
import numpy as np
import pytest

import gradhip as G
import sample_reference as R
import test_gpu_cache as base

pytestmark = pytest.mark.gpu
TYPES = base.TYPES


@pytest.fixture(scope="module")
def torch():
    return base._torch()


def call(torch, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, stream=0, probs=True):
    """logits: a tensor on the GPU; settings: None, a number for all rows, or a list."""
    rows = logits.shape[0]

    def put(v, dtype=torch.float32):
        return None if v is None else torch.tensor([v] * rows if np.isscalar(v) else list(v), dtype=dtype).cuda()

    ids = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    p = torch.full((rows,), -7.0, device="cuda") if probs else None
    kind = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[logits.dtype]
    need = G.sample_workspace(rows, logits.shape[1], kind)
    work = torch.empty(need, dtype=torch.uint8, device="cuda").fill_(255) if need else None
    G.sample(logits, put(u), ids, temperature=put(temperature), top_k=put(top_k, torch.int32), top_p=put(top_p), min_p=put(min_p), probs=p, workspace=work,
             stream=stream)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), p.cpu().numpy() if probs else None


def check(torch, logits, u, what="", **settings):
    ids, probs = call(torch, logits, u, **settings)
    x = logits.cpu().double().numpy()
    f32 = lambda v, r: float(np.float32(v if np.isscalar(v) else v[r]))  # noqa: E731
    wrong = []
    for r in range(len(x)):
        mine = {k: (int(v if np.isscalar(v) else v[r]) if k == "top_k" else f32(v, r)) for k, v in settings.items() if v is not None}
        want, p = R.pick(x[r], f32(u, r), **mine)
        if ids[r] != want:
            wrong.append((r, int(ids[r]), want, mine, f32(u, r)))
        else:
            assert abs(probs[r] - p) <= p * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -149, (what, r, probs[r], p)
    assert not wrong, f"{what}: {len(wrong)} of {len(x)} rows, the first ones (row, pick, wanted, settings, uniform): {wrong[:4]}"
    return ids, probs


def rows_of(torch, dtype, rows, vocab, seed, std=2.5, pad=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab + pad, generator=gen) * std
    return x.to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]).cuda()[:, :vocab], \
        (torch.randint(0, 2 ** 24, (rows,), generator=gen).double() / 2 ** 24).tolist()


SETTINGS = {"plain": dict(), "warm": dict(temperature=1.7), "cold": dict(temperature=0.3), "k": dict(top_k=40), "p": dict(top_p=0.9), "m": dict(min_p=0.05),
            "kp": dict(temperature=0.8, top_k=50, top_p=0.95), "km": dict(top_k=100, min_p=0.02), "pm": dict(temperature=1.3, top_p=0.97, min_p=0.001),
            "kpm": dict(temperature=0.9, top_k=300, top_p=0.8, min_p=0.01), "greedy": dict(temperature=0.0), "most": dict(top_p=0.9999)}


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("dtype", TYPES)
def test_settings(torch, dtype, settings):
    for vocab, rows in ((97, 30), (5000, 20), (32003, 8), (128000, 3)):
        x, u = rows_of(torch, dtype, rows, vocab, seed=vocab + len(settings))
        check(torch, x, u, f"vocab {vocab}", **SETTINGS[settings])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 63, 64, 65, 127, 255, 257, 511, 512, 513, 1023, 4095, 4096, 4097, 8191, 8193, 16385, 50257, 65536, 131071, 262144, 2 ** 20])
def test_vocabularies(torch, dtype, vocab):
    rows = 12 if vocab < 20000 else 3
    for pad in (0, 1, 3):
        x, u = rows_of(torch, dtype, rows, vocab, seed=vocab, pad=pad)
        check(torch, x, u, "no filter")
        check(torch, x, u, "all filters", temperature=1.1, top_k=max(1, vocab // 3), top_p=0.93, min_p=0.003)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_row_its_own_settings(torch, dtype):
    rng = np.random.default_rng(11)
    for rows, vocab in ((200, 3001), (64, 40000), (400, 1500)):
        x, u = rows_of(torch, dtype, rows, vocab, seed=rows, std=3.0)
        check(torch, x, u, f"{rows} rows", temperature=rng.choice([0.0, 0.2, 0.7, 1.0, 1.5, float("nan"), -1.0], rows).tolist(),
              top_k=rng.choice([-3, 0, 1, 2, 17, 64, 500, 2999, vocab, vocab + 5, 2 ** 31 - 1], rows).tolist(),
              top_p=rng.choice([-1.0, 0.0, 1e-9, 0.3, 0.9, 0.999, 1.0, 7.0], rows).tolist(),
              min_p=rng.choice([-1.0, 0.0, 1e-6, 0.01, 0.5, 1.0, 3.0], rows).tolist())


@pytest.mark.parametrize("dtype", TYPES)
def test_settings_that_are_not_numbers_are_off(torch, dtype):
    x, u = rows_of(torch, dtype, 50, 700, seed=5)
    nan = float("nan")
    a, pa = call(torch, x, u, top_p=nan, min_p=nan)
    b, pb = call(torch, x, u)
    assert np.array_equal(a, b) and np.array_equal(pa, pb)
    a, _ = call(torch, x, nan)
    b, _ = call(torch, x, 0.0)
    assert np.array_equal(a, b)
    c, pc = call(torch, x, u, temperature=nan)
    assert np.array_equal(c, x.float().argmax(-1).cpu().numpy()) and (pc == 1.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits_go_by_their_index(torch, dtype):
    """Rows of one value, of two, of a few: the cut falls among equals, and whole multiples make borders exact."""
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    for vocab in (10, 1000, 4099, 70001):
        one = torch.full((6, vocab), 1.5, dtype=t, device="cuda")
        for s in (dict(), dict(top_k=7), dict(top_p=0.5), dict(top_k=8, top_p=0.5), dict(min_p=1.0), dict(top_k=5, min_p=0.9), dict(top_p=0.0)):
            check(torch, one, [0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -24, 1.0], f"one value {s}", **s)
        gen = torch.Generator().manual_seed(vocab)
        few = torch.randint(0, 3, (6, vocab), generator=gen).to(t).cuda()
        u = [0.0, 0.1, 0.33, 0.6, 0.99, 1.0 - 2.0 ** -24]
        for s in (dict(top_k=max(1, vocab // 5)), dict(top_p=0.4), dict(top_k=max(1, vocab // 2), top_p=0.7), dict(min_p=0.2), dict(top_k=1), dict()):
            check(torch, few, u, f"few values {s}", **s)
    zeros = torch.zeros(4, 100, dtype=t, device="cuda")
    zeros[:, ::2] = -0.0
    check(torch, zeros, [0.0, 0.3, 0.6, 0.9], "zeros of both signs", top_k=33)
    check(torch, zeros, [0.0, 0.3, 0.6, 0.9], "zeros of both signs", temperature=0.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_with_little_or_nothing_to_pick(torch, dtype):
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    low, inf, nan = torch.finfo(t).min, float("inf"), float("nan")
    for vocab in (5, 900, 33000):
        x = torch.full((12, vocab), -inf, dtype=t)
        x[1] = nan
        x[2, vocab // 2] = 3.0
        x[3] = low
        x[4] = low
        x[4, vocab - 1] = 0.0
        x[5, ::2] = nan
        x[5, 1::2] = 2.0
        x[6] = 1.0
        x[6, 3] = inf
        x[7, 1] = inf
        x[7, 4] = inf
        x[8, 2] = low
        x[9] = torch.finfo(t).max
        x[9, 2] = low
        x[10] = -1.0
        x[10, 4] = nan
        x[11, 0] = nan
        x[11, 1] = -inf
        x[11, 2] = low
        x[11, 3] = 60000.0
        x = x.cuda()
        u = [0.7] * 12
        for s in (dict(), dict(temperature=0.5, top_k=3), dict(top_p=0.5), dict(min_p=0.3), dict(temperature=0.0), dict(top_k=2, top_p=0.9, min_p=0.01)):
            ids, probs = check(torch, x, u, f"{s}", **s)
            assert ids[0] == ids[1] == -1 and probs[0] == probs[1] == 0.0 and ids[2] == vocab // 2 and ids[6] == 3


@pytest.mark.parametrize("dtype", TYPES)
def test_temperatures_of_any_size(torch, dtype):
    x, u = rows_of(torch, dtype, 40, 3000, seed=8)
    for temperature in (1e-45, 1e-38, 1e-6, 0.01, 30.0, 1e6, 1e30, 3e38, float("inf")):
        check(torch, x, u, f"temperature {temperature}", temperature=temperature)
        check(torch, x, u, f"temperature {temperature}, filters", temperature=temperature, top_k=100, top_p=0.7, min_p=0.4)


@pytest.mark.parametrize("dtype", TYPES)
def test_uniforms_at_their_ends(torch, dtype):
    x, _ = rows_of(torch, dtype, 9, 6000, seed=12)
    u = [0.0, -1.0, 2.0 ** -149, 2.0 ** -24, 1.0 - 2.0 ** -24, 1.0, 2.0, float("inf"), 0.5]
    for s in (dict(), dict(top_k=10), dict(top_p=0.9), dict(min_p=0.1)):
        check(torch, x, u, f"{s}", **s)


@pytest.mark.parametrize("vocab", [5000, 20000, 150000])
def test_segments_that_hold_next_to_nothing(torch, vocab):
    # w of 2^-44.5 count as nothing, however large they are beside what stands near them; uniforms that fall where they would be
    x = torch.full((4, vocab), -float("inf"))
    step = float(np.log(2.0))
    x[:, 0:2000:7] = -44.5 * step
    x[0, 4000], x[0, vocab - 1] = -43.0 * step, 0.0  # before the first token that is kept
    x[1, 4000], x[1, 600] = -43.0 * step, 0.0        # behind the only one of its stretch
    x[2, 1000], x[2, vocab - 900:vocab] = 0.0, -44.5 * step  # behind the last
    x[2, vocab - 1300] = -43.0 * step
    x[3, vocab - 1] = 0.0
    for u in (0.0, 2.0 ** -45, 2.0 ** -43, 1 - 2.0 ** -24, 1.0):
        for settings in (dict(), dict(top_p=0.999999), dict(min_p=1e-30)):
            check(torch, x.cuda(), [u] * 4, (u, settings), **settings)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [3, 600, 5207, 31801])
def test_logits_too_close_to_differ(torch, dtype, vocab):
    # w that are all 1 in 64 bits, though the logits differ: min_p = 1 keeps every one
    logits, u = rows_of(torch, dtype, 4, vocab, seed=vocab)
    for temperature in (float("inf"), 1e30):
        for more in (dict(), dict(top_k=500), dict(top_p=0.5)):
            check(torch, logits, u, (temperature, more), temperature=temperature, min_p=1.0, **more)
    check(torch, (logits.float() * 1e-39).to(logits.dtype), u, "close", min_p=1.0)


def test_wide_spreads_and_far_values(torch):
    """Logits over the whole range of fp32, of one sign, next to each other in their last digits."""
    gen = torch.Generator().manual_seed(3)
    exponents = torch.rand(6, 5000, generator=gen) * 250 - 125
    x = torch.exp2(exponents) * torch.where(torch.rand(6, 5000, generator=gen) < 0.5, -1.0, 1.0)
    u = [0.1, 0.3, 0.5, 0.7, 0.9, 0.999]
    for t in (1.0, 1e30, 3e36):
        check(torch, x.cuda(), u, "all exponents", temperature=t, top_k=50, top_p=0.9)
    near = torch.nextafter(torch.full((6, 5000), 1000.0), torch.tensor(2000.0))
    near = near + torch.randint(0, 40, (6, 5000), generator=gen) * 2.0 ** -14
    check(torch, near.cuda(), u, "neighbours", top_k=500, top_p=0.9)
    check(torch, -near.cuda(), u, "neighbours", temperature=1e-4, top_k=500, top_p=0.9)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [2500, 9001, 33000, 140003, 262144, 2 ** 20])
def test_nuclei_of_any_size(torch, dtype, vocab):
    """From one token to most of the row: lists, cuts found among one bucket's tokens, by one workgroup and by several, and by histograms (no
    place on the grid at low temperatures, whole rows in a few buckets at high ones)."""
    rows = 6 if vocab < 200000 else 2
    x, u = rows_of(torch, dtype, rows, vocab, seed=vocab + 1)
    for top_p in (0.01, 0.6, 0.98, 0.99999):
        check(torch, x, u, f"top_p {top_p}", top_p=top_p)
    check(torch, x, u, "and min_p", top_p=0.97, min_p=1e-5)
    check(torch, x, u, "and min_p below", top_p=0.3, min_p=1e-7)
    check(torch, x, u, "min_p alone", min_p=1e-4)
    for temperature in (1e-12, 0.05, 3.0, 50.0, 1e9, float("inf")):
        check(torch, x, u, f"temperature {temperature}", temperature=temperature, top_p=0.7)


@pytest.mark.parametrize("dtype", TYPES)
def test_lists_of_every_length(torch, dtype):
    for vocab in (3000, 8192, 8193, 40000, 150000):
        x, u = rows_of(torch, dtype, 4, vocab, seed=vocab + 2)
        for k in (1, 2, 63, 64, 65, 128, 129, 255, 256, 257, 1000, 2047, 2048, 2049, 2999):
            check(torch, x, u, f"vocab {vocab} top_k {k}", top_k=k)
        check(torch, x, u, "two filters", top_k=300, top_p=0.9)
        for m in (0.5, 0.1, 0.03, 0.005, 0.0004):
            check(torch, x, u, f"vocab {vocab} min_p {m}", min_p=m)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_are_mostly_forbidden(torch, dtype):
    """Whole chunks and groups without a token: all but a few, all but the last, all but one chunk's."""
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    for vocab in (5000, 40001, 140001):
        x, u = rows_of(torch, dtype, 8, vocab, seed=vocab + 3)
        y = torch.full_like(x, -float("inf"))
        y[1] = torch.finfo(t).min
        y[2] = float("nan")
        for r in (0, 1, 2):
            y[r, 17::4999] = x[r, 17::4999]
        y[3, -1] = 0.5
        y[4, vocab // 2:vocab // 2 + 700] = x[4, :700]
        y[5, :3] = x[5, :3]
        y[6, -9:] = x[6, :9]
        y[6, 0] = float("inf")
        y[7, 100:4000] = x[7, 100:4000]
        y[7, 4200] = torch.finfo(t).max
        for s in (dict(), dict(top_k=5), dict(top_k=900), dict(top_p=0.9), dict(top_p=0.9999), dict(min_p=0.01), dict(top_k=50, top_p=0.8, min_p=0.001), dict(temperature=0.0),
                  dict(temperature=20.0, top_p=0.95)):
            check(torch, y, u, f"vocab {vocab} {s}", **s)


@pytest.mark.parametrize("rows", [1, 5, 70, 300, 600])
def test_nuclei_of_many_rows(torch, rows):
    """Chunks of both sizes, rows looked through by one to eight workgroups beside rows that need none."""
    x, u = rows_of(torch, "bf16", rows, 135000, seed=rows)
    rng = np.random.default_rng(rows)
    some = rng.choice(rows, min(rows, 12), replace=False)
    top_p = [0.98 if r % 3 else 0.2 for r in range(rows)]
    temperature = [1.0 if r % 5 else 0.0 for r in range(rows)]
    ids, probs = call(torch, x, u, temperature=temperature, top_p=top_p)
    for r in some:
        want, p = R.pick(x[r].cpu().double().numpy(), float(np.float32(u[r])), temperature=temperature[r], top_p=float(np.float32(top_p[r])))
        assert ids[r] == want and abs(probs[r] - p) <= p * (2.0 ** -24 + 2.0 ** -40), (r, ids[r], want)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_row_of_logits_for_many_draws(torch, dtype):
    """A stride of zero: the draws' shares are the probabilities that are returned."""
    x, _ = rows_of(torch, dtype, 1, 800, seed=21, std=1.5)
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32).tolist()
    ids, probs = call(torch, x.expand(n, 800), u, top_k=30, min_p=0.01)
    for token in np.unique(ids):
        share, p = float((ids == token).mean()), float(probs[ids == token][0])
        assert abs(share - p) <= 1.0 / n + 1e-6 and (probs[ids == token] == probs[ids == token][0]).all()


@pytest.mark.parametrize("rows,vocab", [(1, 5000), (3, 128001), (100, 32000), (300, 1000)])
def test_the_same_call_gives_the_same_bits_on_any_stream(torch, rows, vocab):
    x, u = rows_of(torch, "bf16", rows, vocab, seed=31)
    a = call(torch, x, u, top_p=0.99)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (0, side.cuda_stream, side.cuda_stream, 0):
        b = call(torch, x, u, top_p=0.99, stream=stream)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_no_probabilities_and_what_lies_beside_the_outputs(torch):
    x, u = rows_of(torch, "f32", 5, 300, seed=41)
    ids = torch.full((9,), -5, dtype=torch.int32, device="cuda")
    probs = torch.full((9,), -5.0, device="cuda")
    G.sample(x, torch.tensor(u, device="cuda"), ids[2:7], probs=probs[2:7])
    alone = call(torch, x, u, probs=False)[0]
    torch.cuda.synchronize()
    assert np.array_equal(ids[2:7].cpu().numpy(), alone)
    for t in (ids, probs):
        assert (t[:2] == -5).all() and (t[7:] == -5).all()
    G.sample(x[:0], torch.empty(0, device="cuda"), ids[:0])  # nothing


def test_calls_that_need_a_workspace_refuse_without_one(torch):
    x, u = rows_of(torch, "f32", 1, 262144, seed=43)
    need = G.sample_workspace(1, 262144)
    ids = torch.full((1,), -5, dtype=torch.int32, device="cuda")
    if need:
        for work in (None, torch.empty(need - 1, dtype=torch.uint8, device="cuda")):
            with pytest.raises(ValueError, match="workspace"):
                G.sample(x, torch.tensor(u, device="cuda"), ids, workspace=work)
    assert int(ids[0]) == -5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(300, 8193), (260, 9001), (256, 16384), (129, 16385)])
def test_many_rows_of_one_or_two_chunks(torch, dtype, rows, vocab):
    x, u = rows_of(torch, dtype, rows, vocab, seed=vocab)
    for settings in (dict(), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.02), dict(temperature=0.0)):
        check(torch, x, u, settings, **settings)


@pytest.mark.parametrize("vocab", [9001, 32000, 140003])
def test_a_workspace_of_many_rows_does_for_few(torch, vocab):
    most = 600
    x, u = rows_of(torch, "bf16", most, vocab, seed=47)
    u, p = torch.tensor(u, device="cuda"), torch.full((most,), 0.9, device="cuda")
    work = torch.empty(G.sample_workspace(most, vocab, "bf16"), dtype=torch.uint8, device="cuda").fill_(255)
    ids = [torch.full((most,), -5, dtype=torch.int32, device="cuda") for _ in range(2)]
    G.sample(x, u, ids[0], top_p=p, workspace=work)
    for rows in (511, 255, 127, 85, 64, 27, 1):  # on either side of where other launches are used
        ids[1].fill_(-5)
        G.sample(x[:rows], u[:rows], ids[1][:rows], top_p=p[:rows], workspace=work)
        assert torch.equal(ids[1][:rows], ids[0][:rows]) and (ids[1][rows:] == -5).all(), rows


def test_memory_of_the_host_is_refused(torch):
    import ctypes as C
    host = np.zeros(400, np.float32)
    ok = torch.zeros(4, device="cuda")
    args = G.GhSampleArgs(host.ctypes.data, 100, 0, 4, 100, 0, None, None, None, None, ok.data_ptr(), ok.data_ptr(), None, None, 0)
    assert G.load_library().gh_sample(C.byref(args), None) == G.GH_ERR_INVALID_ARGUMENT
    assert b"device memory" in G.load_library().gh_last_error()


@pytest.mark.parametrize("rows,vocab", [(1, 50257), (40, 9000)])
def test_captured_and_replayed(torch, rows, vocab):
    """A graph of two calls that share a workspace, replayed on other logits and settings, with eager work between."""
    x, u = rows_of(torch, "f32", rows, vocab, seed=51)
    state = {"x": x.clone(), "u": torch.tensor(u, device="cuda"), "t": torch.full((rows,), 0.9, device="cuda"),
             "k": torch.full((rows,), 50, dtype=torch.int32, device="cuda"), "p": torch.full((rows,), 0.9, device="cuda")}
    ids = [torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2)]
    need = G.sample_workspace(rows, vocab)
    work = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None

    def go(stream):
        G.sample(state["x"], state["u"], ids[0], temperature=state["t"], top_k=state["k"], workspace=work, stream=stream)
        G.sample(state["x"], state["u"], ids[1], temperature=state["t"], top_p=state["p"], workspace=work, stream=stream)

    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        go(torch.cuda.current_stream().cuda_stream)
    for turn in range(4):
        x, u = rows_of(torch, "f32", rows, vocab, seed=60 + turn)
        state["x"].copy_(x)
        state["u"].copy_(torch.tensor(u))
        state["t"].fill_((0.7, 0.0, 1.0, 1.4)[turn])
        for t in ids:
            t.fill_(-3)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        t = (0.7, 0.0, 1.0, 1.4)[turn]
        for got, s in zip(ids, (dict(top_k=50), dict(top_p=0.9))):
            want, _ = check(torch, x, u, f"turn {turn}", temperature=t, **s)
            assert np.array_equal(got.cpu().numpy(), want)
