"""Rows whose forbidden tokens hold their type's lowest value instead of minus infinity (gh_sample): the same picks, and as soon."""
import numpy as np
import pytest

import gradhip as G
import sample_reference as R
import test_gpu_cache as base

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return base._torch()


def fastest(torch, go, calls=20, trials=7):
    """us a call, of the trial that was least disturbed."""
    out = []
    for _ in range(trials):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(calls):
            go()
        b.record()
        b.synchronize()
        out.append(a.elapsed_time(b) * 1000 / calls)
    return min(out)


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("settings", [dict(top_k=40), dict(top_k=50, top_p=0.9), dict(top_k=1000, temperature=0.7)])
@pytest.mark.parametrize("forbidden", [0.9, 0.3])
def test_lowest_values_are_as_good_as_minus_infinity(torch, dtype, settings, forbidden):
    """Peaked rows of 50257 tokens.  What decides is whether a list of 2048 tokens holds all that the bound lets through: if not, one workgroup goes through the
    row some ten times, 10 times as long and more."""
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    rows, vocab = 32, 50257
    rng = np.random.default_rng(len(settings))
    ranks = np.stack([rng.permutation(vocab) for _ in range(rows)])
    x = torch.tensor(12 - 1.5 * np.log1p(ranks) + 0.5 * rng.standard_normal((rows, vocab))).to(t)
    u = rng.integers(0, 2 ** 24, rows) / 2.0 ** 24
    mask = torch.tensor(rng.random((rows, vocab)) < forbidden)
    mask[:, 64 * 100:64 * 101] = True  # a group of neighbours without any
    work = torch.empty(G.sample_workspace(rows, vocab, dtype), dtype=torch.uint8, device="cuda")
    put = lambda v, d: torch.full((rows,), v, dtype=d, device="cuda")  # noqa: E731
    more = {k: put(v, torch.int32 if k == "top_k" else torch.float32) for k, v in settings.items()}
    uniforms = torch.tensor(u, dtype=torch.float32, device="cuda")
    picks, times = [], []
    for value in (float("-inf"), torch.finfo(t).min):
        logits = x.masked_fill(mask, value).cuda()
        ids = torch.full((rows,), -5, dtype=torch.int32, device="cuda")

        def go():
            G.sample(logits, uniforms, ids, workspace=work, **more)

        go()
        times.append(fastest(torch, go))
        picks.append(ids.cpu().numpy())
    want = [R.pick(x.masked_fill(mask, float("-inf"))[r].double().numpy(), float(u[r]), **{k: float(np.float32(v)) if k != "top_k" else v for k, v in settings.items()})[0]
            for r in range(rows)]
    assert list(picks[0]) == want and list(picks[1]) == want
    print(dtype, settings, forbidden, times)
    assert times[1] < 2.5 * times[0], times
