"""Work for attention with sinks over the paged cache, streams that forget, and sampling by row, as cases that can be timed.

A long conversation or document is decoded with a sliding window: a token sees the last `window` positions of its sequence
and, besides, its first few (the sinks), which attention leans on whatever they hold.  What lies between the two is
forgotten, and its pages serve others.  The tokens' logits are then sampled from, every request with settings of its own.

A case is a dict of plain values.  Of kind attend, layer or step:
  kind      attend: the attention of one layer alone, its rows already in the cache
            layer:  append (keys and queries rotated to their positions), then attend, in one layer
            step:   a step of streams that do not end, all layers: the last step's rows are taken back (a rejected draft), what has left
                    the window is forgotten, the new rows' places are handed out; then append and attend in every layer
  dtype     f32 | bf16 | f16: queries, keys, values and outputs
  layers, heads, kv_heads, dim, page
  seqs, context, new, spread   sequences in the pass; cached positions before it and new rows of the longest; equal: all like that,
            ragged: each shorter by its own amount, mixed: one with `new` rows, the others with one
  window, sinks   how many positions back a row sees (itself counted), and how many of the first it sees as well
  rope      base of the rotary positions, 0 for none
Of kind sample:
  dtype     f32 | bf16 | f16: of the logits
  rows, vocab, pad    row r begins r * (vocab + pad) elements behind the first
  shape     peaked: falling with the logarithm of a token's rank, as a trained model's; flat: normal, as an early one's;
            masked: peaked, with nine tokens of ten forbidden (minus infinity, or the type's lowest value in every other row)
  temperature, top_k, top_p, min_p   of every row, 1, 0, 1 and 0 for none; or
  mixed     every row has its own, some of them greedy, some without any
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _attend(kind, dtype, layers, heads, kv_heads, dim, page, seqs, context, new, window, sinks, spread="equal", rope=0):
    return {"kind": kind, "dtype": dtype, "layers": layers, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "seqs": seqs,
            "context": context, "new": new, "window": window, "sinks": sinks, "spread": spread, "rope": rope}


def _sample(dtype, rows, vocab, shape, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, pad=0):
    return {"kind": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "shape": shape, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "mixed": mixed, "pad": pad}


def listed():
    def named(name, case):
        return {"name": name, **case}

    return [
        # one token of one conversation beyond its window, the width-512 block's heads: the smallest call
        named("sinks-1-token", _attend("attend", "f32", 1, 8, 8, 64, 64, 1, 700, 1, 256, 4)),
        # batched decoding with a window, requests of their own lengths, the width-768 block in full precision
        named("sinks-64-tokens", _attend("attend", "f32", 1, 12, 12, 64, 64, 64, 2047, 1, 512, 4, "ragged")),
        # serving of long documents, grouped heads and 16-bit pages
        named("sinks-16-long", _attend("attend", "bf16", 1, 32, 8, 128, 64, 16, 32767, 1, 4096, 4, "ragged")),
        # drafted tokens checked together: a few rows per request
        named("layer-5-drafted", _attend("layer", "f16", 1, 16, 8, 64, 16, 24, 1500, 5, 509, 8, rope=10000)),
        # a turn of a conversation among decoding requests, full precision
        named("layer-mixed", _attend("layer", "f32", 1, 12, 12, 64, 64, 13, 4000, 777, 1024, 4, "mixed", rope=10000)),
        # slices of long prompts in 16 bits, grouped heads: the largest attention
        named("sinks-chunks-4x2048", _attend("attend", "bf16", 1, 32, 8, 128, 64, 4, 6144, 2048, 2048, 100)),
        # a decode step of streams that do not end, four layers, memory for the window alone
        named("step-32-streams", _attend("step", "bf16", 4, 16, 4, 128, 64, 32, 6000, 1, 1024, 4, "ragged", rope=500000)),
        # one request, the command-line callers' settings on the small vocabulary: the smallest pick
        named("sample-1", _sample("f32", 1, 5000, "peaked", 0.8, 40, 0.95)),
        # a modest batch of requests, every one with its own settings
        named("sample-13-mixed", _sample("f32", 13, 32000, "peaked", mixed=True)),
        # a batch with a nucleus, tokens forbidden by a grammar, a vocabulary that no vector divides
        named("sample-64-nucleus", _sample("bf16", 64, 50257, "masked", 0.7, 0, 0.9, pad=3)),
        # many requests, a min-p cut at a raised temperature, 16-bit logits of a large vocabulary
        named("sample-256-min-p", _sample("bf16", 256, 128000, "peaked", 1.3, 0, 1.0, 0.02)),
        # evaluation by drawing from the whole of a flat distribution, every token counts: the most arithmetic
        named("sample-100-flat", _sample("f32", 100, 201001, "flat", 1.0, 0, 0.98)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        rows, vocab = _log_int(rng, 1, 512), _log_int(rng, 1000, 262000)
        rows = max(1, min(rows, 25_000_000 // vocab))
        case = _sample(rng.choice(("f32", "bf16", "f16")), rows, vocab, rng.choice(("peaked", "peaked", "flat", "masked")), pad=rng.choice((0, 0, 1, 8, 24)))
        if rng.random() < 0.4:
            return {**case, "mixed": True}
        filters = rng.choice(("k", "p", "m", "kp", "km", "pm", "kpm", ""))
        return {**case, "temperature": round(rng.uniform(0.5, 1.5), 2), "top_k": _log_int(rng, 1, 1000) if "k" in filters else 0,
                "top_p": round(rng.uniform(0.5, 0.99), 3) if "p" in filters else 1.0, "min_p": round(rng.uniform(0.005, 0.2), 3) if "m" in filters else 0.0}
    kind = rng.choice(("attend", "attend", "layer", "layer", "step"))
    kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 5, 8))
    dim, page = rng.choice((32, 64, 64, 64, 80, 96, 128, 128, 256)), rng.choice((16, 32, 64, 64, 128, 256))
    seqs, context = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
    new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 16 if kind == "step" else 2048)
    window, sinks = _log_int(rng, 16, 8192), _log_int(rng, 1, 256)
    layers = rng.randint(2, 4) if kind == "step" else 1
    spread, dtype = rng.choice(("equal", "ragged", "ragged", "mixed")), rng.choice(("f32", "bf16", "f16"))
    rope = 0 if kind == "attend" else rng.choice((0, 10000, 500000))
    while True:
        case = _attend(kind, dtype, layers, heads, kv_heads, dim, page, seqs, context, new, window, sinks, spread, rope)
        held = layers * seqs * (context + new) * kv_heads * dim * 2 * (4 if dtype == "f32" else 2)
        seen = min(context + new, window + new + sinks)
        # no drawn case is larger than the largest listed ones
        if held <= (1 << 31) and 4.0 * seqs * heads * new * min(context + new, window + sinks) * dim * layers <= 2.7e11 and seqs * heads * new * seen <= 1.1e9:
            return case
        if seqs > 1 and (seqs >= 4 or context + new < 64):
            seqs = max(1, seqs * 2 // 3)
        elif new > 64:
            new = new * 2 // 3
        else:
            context = max(1, context * 2 // 3)


# ------------------------------------------------------------------ inputs


def _lengths(case):
    """(cached positions before the pass, new rows) of every sequence: the same for every seed."""
    rng = random.Random(case["seqs"] * 1000003 + case["context"] * 101 + case["new"])
    n, context, new = case["seqs"], case["context"], case["new"]
    if case["spread"] == "equal":
        return [context] * n, [new] * n
    before = [context] + [rng.randint(context // 8, context) for _ in range(n - 1)]
    if case["spread"] == "mixed":
        return before, [new] + [1] * (n - 1)
    return before, [new] + [rng.randint(1, new) for _ in range(n - 1)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows(case, seed):
    """Keys and values that are cached before the pass, and the pass's rows: [layers, rows, heads, dim]."""
    before, news = _lengths(case)
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]

    def normal(rows, heads, std):
        return (torch.randn(case["layers"], rows, heads, case["dim"], generator=gen, device="cuda") * std).to(dtype)

    old, rows = sum(before), sum(news)
    return {"old_k": normal(old, case["kv_heads"], 1.0), "old_v": normal(old, case["kv_heads"], 1.0),
            "k": normal(rows, case["kv_heads"], 1.0), "v": normal(rows, case["kv_heads"], 1.0),
            # queries that look for something: scores of a standard deviation of two
            "q": normal(rows, case["heads"], 2.0)}


def _logits(case, seed):
    """Logits in rows of vocab + pad elements, settings by row and a draw by row."""
    gen, rows, vocab, dtype = _generator(seed), case["rows"], case["vocab"], DTYPES[case["dtype"]]
    noise = torch.randn(rows, vocab, generator=gen, device="cuda")
    if case["shape"] == "flat":
        x = noise * 2.5
    else:
        rank = torch.rand(rows, vocab, generator=gen, device="cuda").argsort(-1) + 1
        x = 12.0 - 1.6 * rank.float().log() + 0.5 * noise
    held = torch.zeros(rows, vocab + case["pad"], dtype=dtype, device="cuda")
    held[:, :vocab] = x.to(dtype)
    if case["shape"] == "masked":
        forbidden = torch.rand(rows, vocab, generator=gen, device="cuda") < 0.9
        held[0::2, :vocab].masked_fill_(forbidden[0::2], -math.inf)
        held[1::2, :vocab].masked_fill_(forbidden[1::2], torch.finfo(dtype).min)
    settings = {"temperature": [case["temperature"]] * rows, "top_k": [case["top_k"]] * rows, "top_p": [case["top_p"]] * rows, "min_p": [case["min_p"]] * rows}
    if case["mixed"]:
        rng = random.Random(seed)
        settings = {"temperature": [rng.choice((0.0, 0.6, 0.7, 0.8, 1.0, 1.0, 1.2)) for _ in range(rows)],
                    "top_k": [rng.choice((0, 0, 20, 40, 50, 200)) for _ in range(rows)],
                    "top_p": [rng.choice((1.0, 1.0, 0.8, 0.9, 0.95)) for _ in range(rows)],
                    "min_p": [rng.choice((0.0, 0.0, 0.02, 0.05, 0.1)) for _ in range(rows)]}
    out = {name: torch.tensor(v, dtype=torch.int32 if name == "top_k" else torch.float32).cuda() for name, v in settings.items()}
    out["uniforms"] = torch.rand(rows, generator=gen, device="cuda")
    out["logits"] = held[:, :vocab]
    return out


# ---------------------------------------------------------------- the state


def _ceil(a, b):
    return -(-a // b)


def _gradhip():
    sys.path.insert(0, os.path.join(os.getcwd(), "grad.cpp_amd"))
    import gradhip
    return gradhip


def prepare(case, seed):
    if case["kind"] == "sample":
        state = {"case": case, **_logits(case, seed), "ids": torch.empty(case["rows"], dtype=torch.int32, device="cuda"),
                 "probs": torch.empty(case["rows"], device="cuda")}
        if own:
            G = _gradhip()
            need = G.sample_workspace(case["rows"], case["vocab"], case["dtype"])
            state.update(G=G, workspace=torch.empty(need, dtype=torch.uint8, device="cuda") if need else None)
        return state
    x = _rows(case, seed)
    before, news = _lengths(case)
    page, layers = case["page"], case["layers"]
    lens = [b + n for b, n in zip(before, news)]
    pages = sum(_ceil(n, page) for n in lens)
    old_k = _rotate(x["old_k"], torch.cat([torch.arange(n, device="cuda") for n in before]), case["rope"])
    state = {"case": case, "q": x["q"], "k": x["k"], "v": x["v"], "out": torch.empty_like(x["q"]), "turned": torch.empty_like(x["q"])}
    if own:
        cache = _gradhip().Cache(layers=layers, heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["dim"], pages=pages,
                                 dtype=case["dtype"], page_tokens=page, rope_base=float(case["rope"]))
        seqs = [cache.add() for _ in before]
        # the context comes from earlier passes, its keys rotated then
        cache.extend(seqs, before)
        for layer in range(layers):
            cache.append(layer, old_k[layer], x["old_v"][layer], rotate=False)
        if case["kind"] != "step":
            cache.extend(seqs, news)
            if case["kind"] == "attend":
                cache.append(0, x["k"][0], x["v"][0], rotate=False)
        state.update(cache=cache, seqs=seqs, before=before, news=news)
        return state
    # the plain form's cache: pool[page, layer, K or V, head, slot, dim], pages handed out in a scrambled order
    order = list(range(pages))
    random.Random(7).shuffle(order)
    order = iter(order)
    pool = torch.zeros(pages, layers, 2, case["kv_heads"], page, case["dim"], dtype=x["q"].dtype, device="cuda")
    tables = [[next(order) for _ in range(_ceil(n, page))] for n in lens]

    def places(starts, ends):
        """Page and slot of the positions from start to end of every sequence, one after the other."""
        t = [torch.arange(a, b) for a, b in zip(starts, ends)]
        p = [torch.tensor(table, dtype=torch.long)[i // page] for table, i in zip(tables, t)]
        return torch.cat(p).cuda(), (torch.cat(t) % page).cuda()

    def fill(starts, ends, k, v):
        p, s = places(starts, ends)
        pool[p, :, 0, :, s] = k.transpose(0, 1)
        pool[p, :, 1, :, s] = v.transpose(0, 1)

    fill([0] * len(before), before, old_k, x["old_v"])
    if case["kind"] == "attend":
        fill(before, lens, x["k"], x["v"])
    p, s = places(before, lens)
    state.update(pool=pool, p=p, s=s, position=torch.cat([torch.arange(b, n) for b, n in zip(before, lens)]).cuda(), groups=[])
    # a prompt's rows among single ones are a group of their own: padding everybody to it would be the most of the work
    every = list(range(len(news)))
    for group in ([every[:1], every[1:]] if case["spread"] == "mixed" and len(news) > 1 else [every]):
        firsts, most = [sum(news[:i]) for i in group], max(news[i] for i in group)
        # what any row of a sequence sees: its sinks, and from the first row's window on
        seen = [_seen(case, before[i], lens[i]) for i in group]
        widest = max(len(u) for u in seen)
        at = torch.full((len(group), widest), 1 << 40, dtype=torch.long)  # (behind everybody where there is none)
        pages_of = torch.zeros(len(group), widest, dtype=torch.long)
        for j, i in enumerate(group):
            at[j, :len(seen[j])] = seen[j]
            pages_of[j, :len(seen[j])] = torch.tensor(tables[i], dtype=torch.long)[seen[j] // page]
        state["groups"].append({
            "at": at.cuda(), "pages": pages_of.cuda(), "slots": (at % page).cuda(),
            # rows as [sequences, most rows of one], short ones repeating a row of theirs, and which of those are the rows
            "rows": torch.tensor([[f + min(r, news[i] - 1) for r in range(most)] for f, i in zip(firsts, group)]).cuda(),
            "back": torch.tensor([j * most + r for j, i in enumerate(group) for r in range(news[i])]).cuda()})
    return state


def _seen(case, first, end):
    start = max(0, first - case["window"] + 1)
    return torch.cat((torch.arange(min(case["sinks"], start)), torch.arange(start, end)))


# ------------------------------------------------------------ the plain forms


def _rotate(x, position, base):
    """Pairs (2j, 2j + 1) of the last dimension turned by position * base ** (-2j / dim); x: [..., rows, heads, dim]."""
    if not base:
        return x
    dim = x.shape[-1]
    speed = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=x.device) / dim)
    angle = position.to(torch.float64)[:, None] * speed
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2).float().to(x.dtype)


def _attention(state, layer, q):
    """Plain attention over the pages of one layer: 32 bits, rounded once at the end."""
    return torch.cat([_group_attention(state, layer, q, group) for group in state["groups"]])


def _group_attention(state, layer, q, members):
    case, pool, at, rows = state["case"], state["pool"], members["at"], members["rows"]
    seqs, most = rows.shape
    kv, dim = case["kv_heads"], case["dim"]
    group = case["heads"] // kv
    # [sequences, positions, K or V, kv heads, dim] -> [K or V, sequences, kv heads, positions, dim]
    held = pool[members["pages"], layer, :, :, members["slots"]].permute(2, 0, 3, 1, 4).float().contiguous()
    wide = q[rows].float().view(seqs, most, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv, most * group, dim)
    scores = torch.matmul(wide, held[0].transpose(-1, -2).contiguous()).view(seqs, kv, most, group, -1) / math.sqrt(dim)
    mine, at = state["position"][rows][:, :, None], at[:, None]
    visible = (at <= mine) & ((at > mine - case["window"]) | (at < case["sinks"]))
    scores = scores.masked_fill(~visible[:, None, :, None, :], -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    scores = scores / scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(seqs, kv, most * group, -1), held[1])
    out = out.view(seqs, kv, most, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs * most, kv * group, dim)
    return out[members["back"]].to(q.dtype)


def _layer(state, layer):
    """Append and attend in one layer, plainly; the rotated queries and the outputs."""
    case, pool = state["case"], state["pool"]
    k, q = (_rotate(state[name][layer], state["position"], case["rope"]) for name in ("k", "q"))
    pool[state["p"], layer, 0, :, state["s"]] = k
    pool[state["p"], layer, 1, :, state["s"]] = state["v"][layer]
    return q, _attention(state, layer, q)


def _pick(state):
    """The definition over the whole vocabulary, in 64 bits (a draw next to a border needs them)."""
    x = state["logits"].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    vocab = x.shape[-1]
    ordered, token = torch.sort(x, dim=-1, descending=True, stable=True)
    top = ordered[:, :1]
    temperature = state["temperature"].double()[:, None]
    greedy = ~(temperature > 0)
    weight = torch.exp((ordered - torch.where(top > -math.inf, top, 0.0)) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(vocab, device=x.device)
    k = state["top_k"][:, None]
    weight = torch.where((k > 0) & (rank >= k), 0.0, weight)
    p = state["top_p"].double()[:, None]
    reached = weight.cumsum(-1)
    # a token is left out if those before it already have the mass
    weight = torch.where((p < 1) & (rank > 0) & (reached - weight >= p * reached[:, -1:]), 0.0, weight)
    weight = torch.where((rank > 0) & (weight < state["min_p"].double()[:, None]), 0.0, weight)
    weight = torch.where(greedy & (rank > 0), 0.0, weight)
    by_token = torch.zeros_like(weight).scatter_(-1, token, weight)
    below = by_token.cumsum(-1)
    total = below[:, -1:]
    hit = (below >= state["uniforms"].double()[:, None] * total) & (by_token > 0)
    ids = hit.to(torch.uint8).argmax(-1)  # (the first of the largest)
    there = top[:, 0] > -math.inf
    probs = (by_token.gather(-1, ids[:, None]) / total)[:, 0]
    return {"ids": torch.where(there, ids, -1).int(), "probs": torch.where(there, probs, 0.0).float()}


# --------------------------------------------------------------------- a pass


def run(state):
    case = state["case"]
    if case["kind"] == "sample":
        if not own:
            return _pick(state)
        state["G"].sample(state["logits"], state["uniforms"], state["ids"], temperature=state["temperature"], top_k=state["top_k"],
                          top_p=state["top_p"], min_p=state["min_p"], probs=state["probs"], workspace=state["workspace"])
        return {"ids": state["ids"], "probs": state["probs"]}
    layers, mask = range(case["layers"]), {"window": case["window"], "sinks": case["sinks"]}
    if not own:
        if case["kind"] == "attend":
            return _attention(state, 0, state["q"][0])[None]
        q, out = zip(*[_layer(state, layer) for layer in layers])
        return {"q": torch.stack(q), "out": torch.stack(out)}
    cache = state["cache"]
    if case["kind"] == "attend":
        cache.attend(0, state["q"][0], state["out"][0], **mask)
        return state["out"]
    if case["kind"] == "step":
        for seq, length in zip(state["seqs"], state["before"]):
            cache.truncate(seq, length)
            cache.forget(seq, case["sinks"], length - case["window"] + 1)
        cache.extend(state["seqs"], state["news"])
    for layer in layers:
        cache.append(layer, state["k"][layer], state["v"][layer], state["q"][layer], state["turned"][layer])
        cache.attend(layer, state["turned"][layer], state["out"][layer], **mask)
    return {"q": state["turned"], "out": state["out"]}


def work(case):
    """Attention: queries, outputs, new rows once; every visible cached position's keys and values once; two products of `dim` terms per
    visible pair and head.  Sampling: the logits once."""
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "sample":
        return {"bytes": float(case["rows"]) * (case["vocab"] * size + 28), "flops": float(case["rows"]) * case["vocab"]}
    cell = 2 * case["kv_heads"] * case["dim"] * size * case["layers"]  # keys and values of a position
    row = case["heads"] * case["dim"] * size * case["layers"]
    pairs = cells = rows = 0
    for b, n in zip(*_lengths(case)):
        rows += n
        pairs += sum(min(t + 1, case["window"]) + min(case["sinks"], max(0, t + 1 - case["window"])) for t in range(b, b + n))
        cells += len(_seen(case, b, b + n)) + (n if case["kind"] != "attend" else 0)  # (written as well as read)
    return {"bytes": float(cell * cells + (2 if case["kind"] == "attend" else 4) * row * rows), "flops": 4.0 * case["dim"] * case["heads"] * case["layers"] * pairs}


# ------------------------------------------------------------- the definitions


def _exact_picks(case, seed):
    """Row by row on the host: tokens in order, cut from the end, and the draw among what is left."""
    x = {name: t.detach().cpu() for name, t in _logits(case, seed).items()}
    setting = {name: x[name].double().numpy() for name in ("temperature", "top_p", "min_p", "uniforms")}
    ids, probs = [], []
    for r in range(case["rows"]):
        logits = x["logits"][r].double().numpy()
        order = np.argsort(-np.where(np.isnan(logits), -np.inf, logits), kind="stable")
        best = logits[order[0]]
        if not best > -np.inf:
            ids.append(-1), probs.append(0.0)
            continue
        if not setting["temperature"][r] > 0:
            ids.append(int(order[0])), probs.append(1.0)
            continue
        k = int(x["top_k"][r])
        order = order[:k] if k > 0 else order
        w = np.exp((logits[order] - best) / setting["temperature"][r])
        if setting["top_p"][r] < 1:
            keep = 1 + int(np.searchsorted(np.cumsum(w), setting["top_p"][r] * math.fsum(w)))
            order, w = order[:keep], w[:keep]
        good = w >= setting["min_p"][r]
        good[0] = True
        order, w = order[good], w[good]
        inward = np.argsort(order)
        order, w = order[inward], w[inward]
        total = math.fsum(w)
        at = min(int(np.searchsorted(np.cumsum(w), setting["uniforms"][r] * total)), len(w) - 1)
        ids.append(int(order[at])), probs.append(w[at] / total)
    return {"ids": torch.tensor(ids, dtype=torch.int32), "probs": torch.tensor(probs, dtype=torch.float64)}


def exact(case, seed):
    """The definitions in 64 bits: attention sequence by sequence and head by head."""
    if case["kind"] == "sample":
        return _exact_picks(case, seed)
    x = _rows(case, seed)
    dtype, dim, base = x["q"].dtype, case["dim"], case["rope"]
    group = case["heads"] // case["kv_heads"]

    def turned(t, position):
        if not base:
            return t
        pairs = torch.view_as_complex(t.double().unflatten(-1, (dim // 2, 2)).contiguous())
        speed = torch.tensor([float(base) ** (-2.0 * j / dim) for j in range(dim // 2)], dtype=torch.float64, device="cuda")
        angle = position.double()[:, None] * speed
        return torch.view_as_real(pairs * torch.polar(torch.ones_like(angle), angle)[:, None]).flatten(-2).float().to(dtype)

    queries, outs = [], []
    for layer in range(case["layers"]):
        got_q, got_o, old, new = [], [], 0, 0
        for b, n in zip(*_lengths(case)):
            position = torch.arange(b + n, device="cuda")
            mine = position[b:]
            nk, q = x["k"][layer, new:new + n], x["q"][layer, new:new + n]
            if case["kind"] != "attend":
                nk, q = turned(nk, mine), turned(q, mine)
            keys = torch.cat((turned(x["old_k"][layer, old:old + b], position[:b]), nk)).double()
            values = torch.cat((x["old_v"][layer, old:old + b], x["v"][layer, new:new + n])).double()
            old, new = old + b, new + n
            # what lies between every row's sinks and windows is left out of the products
            apart = max(0, b - case["window"] + 1)
            take = torch.cat((position[:min(case["sinks"], apart)], position[apart:]))
            keys, values = keys[take], values[take]
            hidden = (take[None] > mine[:, None]) | ((take[None] <= mine[:, None] - case["window"]) & (take[None] >= case["sinks"]))
            heads = []
            for h in range(case["heads"]):
                z = (q[:, h].double() @ keys[:, h // group].T) * dim ** -0.5
                z[hidden] = -math.inf
                heads.append(torch.softmax(z, 1) @ values[:, h // group])
            got_q.append(q)
            got_o.append(torch.stack(heads, 1))
        queries.append(torch.cat(got_q))
        outs.append(torch.cat(got_o))
    if case["kind"] == "attend":
        return torch.stack(outs)
    return {"q": torch.stack(queries), "out": torch.stack(outs)}
