"""The paged cache's calls where they meet a limit: what is refused, and what a refusal leaves as it was."""
import pytest

import gradhip as G
import test_gpu_cache as base
from test_gpu_cache import Rig

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return base._torch()


def test_refused_copies_leave_the_open_pass(torch):
    rig = Rig(torch, "f32", heads=4, kv_heads=2, dim=64, page=16, pages=6, seed=53)
    a = rig.add()
    q = rig.grow([a], [50])
    with pytest.raises(RuntimeError, match="out of pages"):
        rig.cache.copy(a)
    assert rig.cache.info.pass_rows == 50 and rig.cache.info.sequences == 1
    rig.check([a], [50], q, what="behind a copy that found no pages")
    full = G.Cache(1, 4, 2, 64, pages=1, page_tokens=16)
    s = full.add()
    full.extend([s], [7])
    with pytest.raises(RuntimeError, match="out of pages"):
        rig.cache.copy(a, to=full)
    assert full.info.pass_rows == 7 and full.info.sequences == 1
    # a copy that is made ends the pass of the cache it goes to, as documented
    rig.truncate(a, 16)
    full.drop(s)
    s = full.add()
    full.extend([s], [0])
    rig.cache.copy(a, to=full)
    assert full.info.pass_rows == -1


def test_a_refused_session_leaves_the_open_pass(torch):
    from gradhip import synth
    cfg = synth.Config(synth.ARCH_MODERN, 301, 128, 2, 2, 96)
    session = G.Session(G.Model.from_tensors(cfg, synth.make_weights(cfg, 31, std=0.08, norm_noise=0.1)))
    session.prefill(synth.uniform_tokens(40, cfg.vocab, 50))
    cache = G.Cache(2, 2, 2, 64, pages=3, page_tokens=16)
    s = cache.add()
    cache.extend([s], [20])
    with pytest.raises(RuntimeError, match="out of pages"):
        session.store(cache)
    assert cache.info.pass_rows == 20 and cache.info.sequences == 1
    rows = torch.zeros(20, 2, 64, device="cuda")
    cache.append(0, rows, rows)
    cache.attend(0, rows, rows)
