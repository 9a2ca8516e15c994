"""A session's context in and out of a paged cache: restored sessions go on as the ones that were stored."""
import numpy as np
import pytest

import gradhip as G
from gradhip import synth
from helpers import assert_logits_close

pytestmark = pytest.mark.gpu


def _model(arch, d, heads, max_len=96, vocab=301, layers=2):
    cfg = synth.Config(arch, vocab, d, layers, heads, max_len)
    return cfg, G.Model.from_tensors(cfg, synth.make_weights(cfg, 31, std=0.08, norm_noise=0.1))


def _cache(cfg, pages=40, page=16, **change):
    return G.Cache(**{**dict(layers=cfg.layers, heads=cfg.heads, kv_heads=cfg.heads, head_dim=cfg.d_model // cfg.heads, pages=pages,
                             page_tokens=page), **change})


@pytest.mark.parametrize("arch,d,heads", [(synth.ARCH_GPT2, 128, 2), (synth.ARCH_MODERN, 64, 4), (synth.ARCH_MODERN, 768, 12), (synth.ARCH_GPT2, 512, 8)])
@pytest.mark.parametrize("n", [1, 2, 37])
def test_a_restored_context_goes_on_as_the_stored_one(arch, d, heads, n):
    cfg, model = _model(arch, d, heads)
    ids = synth.uniform_tokens(n, cfg.vocab, 32)
    source = G.Session(model, page_tokens=32)
    logits = source.prefill(ids)[0]
    cache = _cache(cfg)
    kept = source.store(cache)
    assert cache.length(kept) == n
    opt = G.sampling(0.8, 40, 0.9, 1.1)
    u = synth.uniforms(20, 33)
    want = source.decode(20, opt, uniforms=u)[0]
    for batch, engine in ((1, G.ENGINE_AUTO), (1, G.ENGINE_EAGER), (3, G.ENGINE_AUTO), (3, G.ENGINE_GRAPH)):
        session = G.Session(model, batch=batch, engine=engine, page_tokens=64, shuffle_pages=True)
        session.step([5] * batch)  # what it held before is forgotten
        got = session.restore(cache, [kept] * batch, [ids] * batch)
        assert session.position == n
        for b in range(batch):
            assert_logits_close(got[b], logits, what=f"restored {engine} {batch}")
            for layer in range(cfg.layers):
                for kv in (0, 1):
                    for pos in {0, n // 2, max(n - 2, 0)}:
                        if pos < n - 1:
                            assert np.array_equal(session.read_kv(b, layer, kv, pos), source.read_kv(0, layer, kv, pos))
        tokens = session.decode(20, opt, uniforms=np.tile(u, (batch, 1)))
        for b in range(batch):
            assert np.array_equal(tokens[b], want), (engine, batch, b)


def test_sequences_of_a_batch_are_kept_apart_and_grow_in_the_cache():
    cfg, model = _model(synth.ARCH_MODERN, 128, 2)
    ids = np.stack([synth.uniform_tokens(50, cfg.vocab, 40 + b) for b in range(4)])
    source = G.Session(model, batch=4)
    source.prefill(ids)
    cache = _cache(cfg, pages=80)
    kept = [source.store(cache, b) for b in range(4)]
    short = cache.fork(kept[2], 20)
    cache.drop(kept[2])
    cache.compact()
    # the sequences in another order, one of them twice
    order = [kept[3], kept[0], kept[3], kept[1]]
    rows = ids[[3, 0, 3, 1]]
    session = G.Session(model, batch=4)
    got = session.restore(cache, order, rows)
    fresh = G.Session(model, batch=4)
    want = fresh.prefill(rows)
    for b in range(4):
        assert_logits_close(got[b], want[b], what="order")
    # a part of what is kept, and a last token of one's own
    own = np.concatenate([ids[2][:20], [7]]).astype(np.int32)
    one = G.Session(model)
    got = one.restore(cache, [short], [own])
    assert one.position == 21
    want = G.Session(model).prefill(own)
    assert_logits_close(got[0], want[0], what="part")


def test_what_does_not_fit_is_refused():
    cfg, model = _model(synth.ARCH_MODERN, 128, 2, max_len=40)
    session = G.Session(model)
    session.prefill(synth.uniform_tokens(30, cfg.vocab, 50))
    for change in (dict(layers=3), dict(head_dim=32), dict(dtype="bf16"), dict(kv_heads=1)):
        with pytest.raises(ValueError, match="a session's context needs"):
            session.store(_cache(cfg, **change))
    with pytest.raises(RuntimeError, match="out of pages"):
        session.store(_cache(cfg, pages=1))
    cache = _cache(cfg)
    with pytest.raises(IndexError, match="no sequence 1"):
        session.store(cache, 1)
    kept = session.store(cache)
    with pytest.raises(IndexError, match="no sequence 7"):
        session.restore(cache, [7], [[1, 2]])
    with pytest.raises(IndexError, match="positions"):
        session.restore(cache, [kept], [synth.uniform_tokens(32, cfg.vocab, 51)])
    with pytest.raises(RuntimeError, match="max_len"):
        session.restore(cache, [kept], [synth.uniform_tokens(41, cfg.vocab, 51)])
    with pytest.raises(IndexError, match="vocab"):
        session.restore(cache, [kept], [[1, cfg.vocab]])
    with pytest.raises(ValueError, match="one token"):
        session.restore(cache, [kept], np.zeros((1, 0), np.int32))
    assert session.position == 30  # refusals leave the session as it was
    session.restore(cache, [kept], [synth.uniform_tokens(31, cfg.vocab, 52)])
    assert session.position == 31
