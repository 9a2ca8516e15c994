"""Streams that do not end, as a program of its own layers would run them: every step forgets what has left the window, extends, appends and
attends with sinks in two layers, and samples the next tokens from its logits with settings of each stream's own; against the
same model over dense rows in 64 bits."""
import math

import numpy as np
import pytest

import gradhip as G
import sample_reference as R
import test_gpu_cache as base

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, VOCAB, LAYERS, WINDOW, SINKS, BASE = 4, 2, 32, 600, 2, 24, 3, 10000.0
SETTINGS = [dict(), dict(temperature=0.7, top_k=30), dict(temperature=1.3, min_p=0.05), dict(top_p=0.8), dict(temperature=0.0)]


@pytest.fixture(scope="module")
def torch():
    return base._torch()


def weights(torch):
    gen = torch.Generator().manual_seed(7)
    width = HEADS * DIM
    make = lambda *shape: torch.randn(*shape, generator=gen) / math.sqrt(shape[-2])  # noqa: E731
    return {"embed": torch.randn(VOCAB, width, generator=gen), "qkv": make(LAYERS, width, (HEADS + 2 * KV) * DIM), "out": make(LAYERS, width, width),
            "logits": make(width, VOCAB) * 3}


def dense_step(torch, w, history, ids, position):
    """One token of one stream in 64 bits; history: per layer a list of (rotated key, value)."""
    cache_reference = base._ref()
    x = w["embed"][ids].double()
    for layer in range(LAYERS):
        q, k, v = (x @ w["qkv"][layer].double()).view(HEADS + 2 * KV, DIM).split((HEADS, KV, KV))
        turn = lambda t: cache_reference.rotated(t[None], [position], BASE)[0]  # noqa: E731
        history[layer].append((turn(k), v))
        seen = [u for u in range(position + 1) if u > position - WINDOW or u < SINKS]
        keys, values = (torch.stack([history[layer][u][i] for u in seen]) for i in (0, 1))
        q = turn(q)
        heads = []
        for h in range(HEADS):
            z = keys[:, h * KV // HEADS] @ q[h] / math.sqrt(DIM)
            heads.append(torch.softmax(z, 0) @ values[:, h * KV // HEADS])
        x = x + torch.cat(heads) @ w["out"][layer].double()
    return x @ w["logits"].double()


def test_streams_step_by_step(torch):
    w = weights(torch)
    on = {k: t.cuda() for k, t in w.items()}
    n, steps = len(SETTINGS), 70
    # pages for sinks, window and a page of slack each: far fewer than the positions that pass through
    cache = G.Cache(LAYERS, HEADS, KV, DIM, pages=n * 4, page_tokens=16, rope_base=BASE)
    streams = [cache.add() for _ in range(n)]
    uniforms = torch.rand(steps, n, generator=torch.Generator().manual_seed(8))
    put = lambda key, off, kind: torch.tensor([s.get(key, off) for s in SETTINGS], dtype=kind).cuda()  # noqa: E731
    settings = {"temperature": put("temperature", 1.0, torch.float32), "top_k": put("top_k", 0, torch.int32), "top_p": put("top_p", 1.0, torch.float32),
                "min_p": put("min_p", 0.0, torch.float32)}
    tokens = torch.arange(n, dtype=torch.int32, device="cuda") + 10
    ids, probs = torch.empty_like(tokens), torch.empty(n, device="cuda")
    histories = [[[] for _ in range(LAYERS)] for _ in range(n)]
    dense = list(range(10, 10 + n))
    for step in range(steps):
        for s in streams:
            cache.forget(s, SINKS, step - WINDOW + 1)
        cache.extend(streams, [1] * n)
        x = on["embed"][tokens.long()]
        for layer in range(LAYERS):
            rows = (x @ on["qkv"][layer]).view(n, HEADS + 2 * KV, DIM)
            q, k, v = rows[:, :HEADS], rows[:, HEADS:HEADS + KV], rows[:, HEADS + KV:]
            turned, out = torch.empty(n, HEADS, DIM, device="cuda"), torch.empty(n, HEADS, DIM, device="cuda")
            cache.append(layer, k, v, q, turned)
            cache.attend(layer, turned, out, window=WINDOW, sinks=SINKS)
            x = x + out.view(n, -1) @ on["out"][layer]
        logits = x @ on["logits"]
        G.sample(logits, uniforms[step].cuda(), ids, probs=probs, **settings)
        tokens.copy_(ids)
        for i in range(n):
            want = dense_step(torch, w, histories[i], dense[i], step)
            assert (logits[i].cpu().double() - want).abs().max() <= 2e-5 * want.abs().max(), (step, i)
            f32 = {k: (v if k == "top_k" else float(np.float32(v))) for k, v in SETTINGS[i].items()}
            dense[i], _ = R.pick(want.numpy(), float(uniforms[step, i]), **f32)
        assert tokens.cpu().tolist() == dense, step
    assert cache.length(streams[0]) == steps > n * 4 * 16 / n
