"""Work for the paged cache's operators, as cases that can be timed.

A cache holds keys and values of many sequences in pages of a fixed number of positions.  One
pass over some of its sequences brings new rows (tokens) for each; in every layer the rows'
keys are rotated to their positions and stored with the values (append), and the rows' queries
attend to everything that is cached of their sequence, themselves included (attend).  Sequences
can be forked (pages shared, a shared page copied when somebody writes into it), copied,
compacted and dropped.

A case is a dict of plain values:
  kind      attend | layer | fork | move
              attend: the attention of one layer alone, its rows already in the cache
              layer:  append, then attend, in one layer
              fork:   `seqs` continuations forked off one context, `new` tokens each, all layers
              move:   every sequence copied, every other copy dropped, the pages compacted and
                      the copies that are left read back, all layers
  dtype     f32 | bf16 | f16: queries, keys, values and outputs
  layers, heads, kv_heads, dim, page
  seqs, context, new, spread   sequences in the pass; cached positions before it and new rows of
                      the longest; equal: all like that, ragged: each shorter by its own amount,
                      mixed: one with `new` rows, the others with one
  window    0, or how many positions back a row sees (itself counted)
  causal    whether a row sees the later rows of its sequence
  rope      base of the rotary positions, 0 for none
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _case(kind, dtype, layers, heads, kv_heads, dim, page, seqs, context, new, spread="equal", window=0, causal=True, rope=0):
    return {"kind": kind, "dtype": dtype, "layers": layers, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "seqs": seqs, "context": context, "new": new, "spread": spread, "window": window, "causal": causal, "rope": rope}


def listed():
    def named(name, *a, **k):
        return {"name": name, **_case(*a, **k)}

    return [
        # one token of a short conversation, the width-512 block's heads: the smallest call there is
        named("attend-1-token", "attend", "f32", 1, 8, 8, 64, 64, 1, 96, 1),
        # a decode step's layer for a modest batch of requests of their own lengths, the width-768 block
        named("layer-13-tokens", "layer", "f32", 1, 12, 12, 64, 64, 13, 1023, 1, "ragged", rope=10000),
        # batched decoding over long caches, the width-768 block in full precision
        named("attend-64-tokens", "attend", "f32", 1, 12, 12, 64, 64, 64, 2047, 1, "ragged"),
        # serving with grouped heads and 16-bit pages, tens of thousands of positions per request
        named("attend-16-long", "attend", "bf16", 1, 32, 8, 128, 64, 16, 32767, 1, "ragged"),
        # one very long document, one token at a time
        named("attend-1-long", "attend", "bf16", 1, 16, 4, 128, 128, 1, 131071, 1),
        # drafted tokens checked together: a few rows per request
        named("layer-5-drafted", "layer", "f16", 1, 16, 8, 64, 16, 24, 1500, 5, "equal", rope=10000),
        # a turn of a conversation: a chunk onto a context, the width-768 block in full precision
        named("layer-chunk-397", "layer", "f32", 1, 12, 12, 64, 64, 1, 1602, 397, rope=10000),
        # prompts of many requests from nothing, full precision, evaluation windows' lengths
        named("attend-prompts-16x1024", "attend", "f32", 1, 12, 12, 64, 64, 16, 0, 1024),
        # slices of long prompts in 16 bits, grouped heads: the largest
        named("attend-chunks-4x2048", "attend", "bf16", 1, 32, 8, 128, 64, 4, 6144, 2048),
        # a prompt's slice among decoding requests, a sliding window, heads that share one key
        named("layer-mixed-window", "layer", "f16", 1, 20, 4, 80, 32, 33, 5000, 777, "mixed", window=1024, rope=500000),
        # eight samples of one prompt, their first token, a whole model of eight layers
        named("fork-8-samples", "fork", "f32", 8, 12, 12, 64, 64, 8, 1000, 1, rope=10000),
        # conversations duplicated, half of them ended, the pool made dense, the rest exported
        named("move-6-copies", "move", "f32", 8, 12, 12, 64, 64, 6, 1500, 0, "ragged"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "layer", "layer", "layer", "fork", "move"))
    dtype = rng.choice(("f32", "f32", "bf16", "f16"))
    kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 5, 8))
    dim = rng.choice((32, 64, 64, 64, 80, 96, 128, 128, 256))
    page = rng.choice((16, 32, 64, 64, 128, 256))
    layers = rng.randint(2, 8) if kind in ("fork", "move") else 1
    seqs = _log_int(rng, 1, 64)
    context = _log_int(rng, 1, 32768) if rng.random() < 0.85 else 0
    new = {"move": 0, "fork": _log_int(rng, 1, 16)}.get(kind)
    if new is None:
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 2048)
    if kind in ("fork", "move"):
        context = max(1, context)
    if kind == "move":
        seqs = max(2, seqs)
    spread = "equal" if kind == "fork" else rng.choice(("equal", "ragged")) if kind == "move" else rng.choice(("equal", "ragged", "ragged", "mixed"))
    window = _log_int(rng, 1, context + new) if kind in ("attend", "layer") and rng.random() < 0.25 else 0
    causal = kind not in ("attend", "layer") or rng.random() < 0.9
    rope = rng.choice((0, 10000, 500000)) if kind in ("layer", "fork") else 0
    while True:
        case = _case(kind, dtype, layers, heads, kv_heads, dim, page, seqs, context, new, spread, window, causal, rope)
        size = 4 if dtype == "f32" else 2
        held = (2 if kind == "move" else 1) * layers * seqs * (context + new) * kv_heads * dim * 2 * size
        longest = new if kind != "move" else 1
        # no drawn case is larger than the largest listed ones
        if (held <= (1 << 31) and 4.0 * seqs * heads * longest * (context + new) * dim * layers <= 5e11
                and 4.0 * seqs * heads * longest * (context + new) <= 4e9):
            return case
        if seqs > 1 and (seqs >= 4 or context + new < 64):
            seqs = max(1, seqs * 2 // 3)
        elif new > 64 and kind in ("attend", "layer"):
            new = new * 2 // 3
        else:
            context = max(1, context * 2 // 3)


def _lengths(case):
    """(cached positions before the pass, new rows) of every sequence: the same for every seed."""
    rng = random.Random(case["seqs"] * 1000003 + case["context"] * 101 + case["new"])
    n, context, new = case["seqs"], case["context"], case["new"]
    if case["spread"] == "equal":
        return [context] * n, [new] * n
    before = [context] + [rng.randint(context // 8, context) for _ in range(n - 1)]
    if case["spread"] == "mixed":
        return before, [new] + [min(new, 1)] * (n - 1)
    return before, [new] + [rng.randint(min(new, 1), new) for _ in range(n - 1)]


def _inputs(case, seed):
    """Keys and values that are cached before the pass, and the pass's rows: [layers, rows, heads, dim]."""
    before, news = _lengths(case)
    if case["kind"] == "fork":
        before = before[:1]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, layers, dim = DTYPES[case["dtype"]], case["layers"], case["dim"]

    def normal(rows, heads, std):
        return (torch.randn(layers, rows, heads, dim, generator=gen, device="cuda") * std).to(dtype)

    old, rows = sum(before), sum(news)
    return {"old_k": normal(old, case["kv_heads"], 1.0), "old_v": normal(old, case["kv_heads"], 1.0),
            "k": normal(rows, case["kv_heads"], 1.0), "v": normal(rows, case["kv_heads"], 1.0),
            # queries that look for something: scores of a standard deviation of two
            "q": normal(rows, case["heads"], 2.0)}


def _cache(case, pages):
    sys.path.insert(0, os.path.join(os.getcwd(), "grad.cpp_amd"))
    import gradhip as G
    return G.Cache(layers=case["layers"], heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["dim"], pages=pages,
                   dtype=case["dtype"], page_tokens=case["page"], rope_base=float(case["rope"]))


def _ceil(a, b):
    return -(-a // b)


def prepare(case, seed):
    x = _inputs(case, seed)
    before, news = _lengths(case)
    kind, page = case["kind"], case["page"]
    state = {"case": case, "q": x["q"], "k": x["k"], "v": x["v"]}
    if kind == "move":
        kept = sum(before[1::2])
        state["read"] = [torch.empty(case["layers"], kept, case["kv_heads"], case["dim"], dtype=x["q"].dtype, device="cuda")
                         for _ in range(2)]
    else:
        state["out"] = torch.empty_like(x["q"])
        state["turned"] = torch.empty_like(x["q"])
    parents = before[:1] if kind == "fork" else before
    # pages: what the sequences hold, and what the pass's forks and copies take
    lens = [b + n for b, n in zip(before, news)]
    if kind == "fork":
        pages = _ceil(before[0], page) + sum(_ceil(n, page) - b // page for b, n in zip(before, lens))
    else:
        pages = (2 if kind == "move" else 1) * sum(_ceil(n, page) for n in lens)
    if own:
        cache = _cache(case, pages)
        seqs = [cache.add() for _ in parents]
        if sum(parents):
            # the context comes from earlier passes, its keys rotated then
            old_k = _rotated_old(x["old_k"], case, parents) if kind in ("attend", "layer") else x["old_k"]
            cache.extend(seqs, parents)
            for layer in range(case["layers"]):
                cache.append(layer, old_k[layer], x["old_v"][layer], rotate=False)
        if kind in ("attend", "layer"):
            cache.extend(seqs, news)
            if kind == "attend":
                cache.append(0, x["k"][0], x["v"][0], rotate=False)
        state.update(cache=cache, seqs=seqs, news=news)
        return state
    # the plain form's cache: pool[page, layer, K or V, head, slot, dim], pages handed out in a scrambled order
    order = list(range(pages))
    random.Random(7).shuffle(order)
    order = iter(order)
    pool = torch.zeros(pages, case["layers"], 2, case["kv_heads"], page, case["dim"], dtype=x["q"].dtype, device="cuda")
    tables = [[next(order) for _ in range(_ceil(b if kind in ("fork", "move") else n, page))] for b, n in zip(parents, lens)]

    def index(numbers):
        return torch.as_tensor(numbers, dtype=torch.long).cuda()

    def places(tables, starts, ends):
        """Page and slot of the positions from start to end of every sequence, one after the other."""
        t = [torch.arange(a, b) for a, b in zip(starts, ends)]
        p = [torch.tensor(table, dtype=torch.long)[i // page] for table, i in zip(tables, t)]
        return index(torch.cat(p)), index(torch.cat(t) % page)

    def fill(tables, starts, ends, k, v):
        p, s = places(tables, starts, ends)
        pool[p, :, 0, :, s] = k.transpose(0, 1)
        pool[p, :, 1, :, s] = v.transpose(0, 1)

    fill(tables, [0] * len(parents), parents, _rotated_old(x["old_k"], case, parents) if kind in ("attend", "layer") else x["old_k"], x["old_v"])
    if kind == "move":
        copies = [[next(order) for _ in t] for t in tables]
        kept, ended = copies[1::2], sum(copies[::2], [])
        moved = sum(kept, [])
        n = min(len(moved), len(ended))
        to = dict(zip(moved[:n], ended[:n]))
        p, s = places([[to.get(c, c) for c in t] for t in kept], [0] * len(kept), before[1::2])
        state.update(pool=pool, source=index(sum(tables, [])), copies=index(sum(copies, [])), moved=index(moved[:n]),
                     ended=index(ended[:n]), p=p, s=s)
        return state
    if kind == "fork":
        shared, rest = before[0] // page, before[0] % page
        parent = tables[0]
        tables = [parent[:shared] + [next(order) for _ in range(_ceil(n, page) - shared)] for n in lens]
        state["copies"] = (index([t[shared] for t in tables]), parent[shared]) if rest else None
    if kind == "attend":
        fill(tables, before, lens, x["k"], x["v"])
    p, s = places(tables, before, lens)
    state.update(pool=pool, p=p, s=s, position=index([b + i for b, n in zip(before, news) for i in range(n)]), groups=[])
    # a prompt's rows among single ones are a group of their own: padding everybody to it would be the most of the work
    every = list(range(len(news)))
    for group in ([every[:1], every[1:]] if case["spread"] == "mixed" and len(news) > 1 else [every]):
        widest, most = max(len(tables[i]) for i in group), max(news[i] for i in group)
        firsts = [sum(news[:i]) for i in group]
        state["groups"].append({
            "table": index([tables[i] + [0] * (widest - len(tables[i])) for i in group]), "lens": index([lens[i] for i in group]),
            # rows as [sequences, most rows of one], short ones repeating a row of theirs, and which of those are the rows
            "rows": index([[f + min(r, news[i] - 1) for r in range(most)] for f, i in zip(firsts, group)]),
            "back": index([j * most + r for j, i in enumerate(group) for r in range(news[i])])})
    return state


def _rotated_old(k, case, parents):
    if not case["rope"]:
        return k
    return _rotate(k, torch.cat([torch.arange(n, device="cuda") for n in parents]), case["rope"])


def _rotate(x, position, base):
    """Pairs (2j, 2j + 1) of the last dimension turned by position * base ** (-2j / dim); x: [..., rows, heads, dim]."""
    dim = x.shape[-1]
    speed = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=x.device) / dim)
    angle = position.to(torch.float64)[:, None] * speed
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2).to(x.dtype)


def _attention(state, layer, q):
    """Plain attention over the pages of one layer: 32 bits, rounded once at the end."""
    return torch.cat([_group_attention(state, layer, q, group) for group in state["groups"]])


def _group_attention(state, layer, q, members):
    case, pool, table = state["case"], state["pool"], members["table"]
    seqs, widest = table.shape
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // kv
    held = pool[table, layer].permute(2, 0, 3, 1, 4, 5).reshape(2, seqs, kv, widest * page, dim).float()
    here = torch.arange(widest * page, device="cuda")
    rows = members["rows"]
    most = rows.shape[1]
    # a place that nobody wrote may hold anything
    held = torch.where((here < members["lens"][:, None])[:, None, :, None], held, 0.0)
    wide = q[rows].float().view(seqs, most, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv, most * group, dim)
    scores = torch.matmul(wide, held[0].transpose(-1, -2).contiguous()).view(seqs, kv, most, group, -1) / math.sqrt(dim)
    at = state["position"][rows][:, :, None]
    seen = (here < members["lens"][:, None])[:, None, :].expand(seqs, most, -1)
    if case["causal"]:
        seen = seen & (here <= at)
    if case["window"]:
        seen = seen & (here > at - case["window"])
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    scores = scores / scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(seqs, kv, most * group, -1), held[1])
    out = out.view(seqs, kv, most, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs * most, kv * group, dim)
    return out[members["back"]].to(q.dtype)


def _layer(state, layer):
    """Append and attend in one layer, plainly; the rotated queries and the outputs."""
    case, pool = state["case"], state["pool"]
    k, q = state["k"][layer], state["q"][layer]
    if case["rope"]:
        k, q = _rotate(k, state["position"], case["rope"]), _rotate(q, state["position"], case["rope"])
    pool[state["p"], layer, 0, :, state["s"]] = k
    pool[state["p"], layer, 1, :, state["s"]] = state["v"][layer]
    return q, _attention(state, layer, q)


def _run_own(state):
    case, cache = state["case"], state["cache"]
    kind = case["kind"]
    if kind == "attend":
        cache.attend(0, state["q"][0], state["out"][0], causal=case["causal"], window=case["window"])
        return state["out"]
    if kind == "layer":
        cache.append(0, state["k"][0], state["v"][0], state["q"][0], state["turned"][0])
        cache.attend(0, state["turned"][0], state["out"][0], causal=case["causal"], window=case["window"])
        return {"q": state["turned"], "out": state["out"]}
    if kind == "fork":
        samples = [cache.fork(state["seqs"][0]) for _ in state["news"]]
        cache.extend(samples, state["news"])
        for layer in range(case["layers"]):
            cache.append(layer, state["k"][layer], state["v"][layer], state["q"][layer], state["turned"][layer])
            cache.attend(layer, state["turned"][layer], state["out"][layer])
        for s in samples:
            cache.drop(s)
        return {"q": state["turned"], "out": state["out"]}
    copies = [cache.copy(s) for s in state["seqs"]]
    for s in copies[::2]:
        cache.drop(s)
    cache.compact()
    at = 0
    for s in copies[1::2]:
        n = cache.length(s)
        cache.read(s, state["read"][0][:, at:at + n], state["read"][1][:, at:at + n])
        at += n
        cache.drop(s)
    return {"k": state["read"][0], "v": state["read"][1]}


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    kind = case["kind"]
    if kind == "attend":
        return _attention(state, 0, state["q"][0])[None]
    if kind == "layer":
        q, out = _layer(state, 0)
        return {"q": q[None], "out": out[None]}
    pool = state["pool"]
    if kind == "fork":
        if state["copies"]:
            pool[state["copies"][0]] = pool[state["copies"][1]].clone()
        q, out = zip(*(_layer(state, layer) for layer in range(case["layers"])))
        return {"q": torch.stack(q), "out": torch.stack(out)}
    pool[state["copies"]] = pool[state["source"]]
    pool[state["ended"]] = pool[state["moved"]]
    p, s = state["p"], state["s"]
    return {"k": pool[p, :, 0, :, s].transpose(0, 1).contiguous(), "v": pool[p, :, 1, :, s].transpose(0, 1).contiguous()}


def work(case):
    """Queries, outputs, new rows once; every visible cached position's keys and values once (a shared one once for all who
    share it); two products of `dim` terms per visible pair and head.  Copies: what is moved, read and written."""
    before, news = _lengths(case)
    size = 4 if case["dtype"] == "f32" else 2
    cell = 2 * case["kv_heads"] * case["dim"] * size * case["layers"]  # keys and values of a position
    row = case["heads"] * case["dim"] * size * case["layers"]
    if case["kind"] == "move":
        pages = [_ceil(n, case["page"]) for n in before]
        moved = min(sum(pages[1::2]), sum(pages[::2])) * case["page"]
        return {"bytes": 2.0 * cell * (sum(before) + min(moved, sum(before[1::2])) + sum(before[1::2])), "flops": 0}
    pairs = cells = 0
    window = case["window"] or 1 << 60
    for b, n in zip(before, news):
        end = b + n
        first = [max(0, t - window + 1) for t in range(b, end)]
        last = [t + 1 if case["causal"] else end for t in range(b, end)]
        pairs += sum(e - f for f, e in zip(first, last))
        if n:
            cells += end - first[0]
    rows = sum(news)
    if case["kind"] == "fork":
        cells = before[0] + 2 * case["seqs"] * (before[0] % case["page"]) + 2 * rows
    elif case["kind"] == "layer":
        cells += rows  # written as well as read
    q = 2 * row * rows if case["kind"] != "attend" else 0
    return {"bytes": float(cell * cells + 2 * row * rows + q), "flops": 4.0 * case["dim"] * case["heads"] * case["layers"] * pairs}


def exact(case, seed):
    """The definition, sequence by sequence and head by head in 64 bits."""
    x = _inputs(case, seed)
    before, news = _lengths(case)
    if case["kind"] == "move":
        spans = [(sum(before[:i]), sum(before[:i + 1])) for i in range(1, len(before), 2)]
        pick = [torch.cat([x[name][:, a:b] for a, b in spans], 1) if spans else x[name][:, :0] for name in ("old_k", "old_v")]
        return {"k": pick[0], "v": pick[1]}
    dtype, dim, base = x["q"].dtype, case["dim"], case["rope"]
    group = case["heads"] // case["kv_heads"]

    def turned(t, position):
        if not base:
            return t
        pairs = torch.view_as_complex(t.double().unflatten(-1, (dim // 2, 2)).contiguous())
        speed = torch.tensor([float(base) ** (-2.0 * j / dim) for j in range(dim // 2)], dtype=torch.float64, device="cuda")
        angle = position.double()[:, None] * speed
        return torch.view_as_real(pairs * torch.polar(torch.ones_like(angle), angle)[:, None]).flatten(-2).to(dtype)

    queries, outs = [], []
    for layer in range(case["layers"]):
        got_q, got_o, old, new = [], [], 0, 0
        for b, n in zip(before, news):
            position = torch.arange(b + n, device="cuda")
            ok, ov = x["old_k"][layer, old:old + b], x["old_v"][layer, old:old + b]
            if case["kind"] in ("attend", "layer"):
                ok = turned(ok, position[:b])
                old += b
            mine = position[b:]
            rotates = case["kind"] != "attend"
            nk, q = x["k"][layer, new:new + n], x["q"][layer, new:new + n]
            if rotates:
                nk, q = turned(nk, mine), turned(q, mine)
            keys = torch.cat((ok, nk)).double()
            values = torch.cat((ov, x["v"][layer, new:new + n])).double()
            new += n
            hidden = torch.zeros(n, b + n, dtype=torch.bool, device="cuda")
            if case["causal"]:
                hidden |= position[None] > mine[:, None]
            if case["window"]:
                hidden |= position[None] <= mine[:, None] - case["window"]
            heads = []
            for h in range(case["heads"]):
                g = h // group
                z = (q[:, h].double() @ keys[:, g].T) * dim ** -0.5
                z[hidden] = -math.inf
                heads.append(torch.softmax(z, 1) @ values[:, g])
            got_q.append(q)
            got_o.append(torch.stack(heads, 1))
        queries.append(torch.cat(got_q))
        outs.append(torch.cat(got_o))
    if case["kind"] == "attend":
        return torch.stack(outs)
    return {"q": torch.stack(queries), "out": torch.stack(outs)}
