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


def test_a_prefix_shared_by_thousands(torch):
    """4096 single tokens behind one prefix, 64 heads of 256: what they would leave for the prefix's joins is more than a workspace
    holds, so each reads the prefix itself."""
    rig = Rig(torch, "bf16", heads=64, kv_heads=64, dim=256, page=16, pages=4200, seed=51)
    parent = rig.add()
    rig.grow([parent], [256])
    kids = [rig.cache.fork(parent) for _ in range(4096)]
    rig.cache.extend(kids, [1] * 4096)
    gen = torch.Generator(device="cuda").manual_seed(52)
    k, v, q = (torch.randn(4096, 64, 256, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(3))
    out = torch.empty_like(q)
    rig.cache.append(0, k, v)
    rig.cache.attend(0, q, out)
    for i in (0, 1, 15, 16, 2047, 4095):
        keys, values = (torch.cat((old, new[i:i + 1].cpu().double())) for old, new in ((rig.ref.k[parent][0], k), (rig.ref.v[parent][0], v)))
        want, allowed = rig.R.attention(q[i:i + 1].cpu().double(), keys, values, 256, dtype="bf16")
        rig.R.assert_within(out[i:i + 1], want, allowed, f"sequence {i}")


@pytest.mark.parametrize("dtype", base.TYPES)
def test_scales_at_the_ends_of_their_range(torch, dtype):
    rig = Rig(torch, dtype, heads=2, kv_heads=1, dim=64, page=16, pages=40, seed=54)
    s = rig.add()
    rig.grow([s], [30])
    q = rig.grow([s], [100])
    q[:] = 0.0
    for scale in (1e-45, 1e-38, 2.3e38):  # scores of zero, whatever they are multiplied by
        rig.check([s], [100], q, scale=scale, what=f"scale {scale:g}")
    for scale in (2.4e38, 3.4e38):  # finite, but not in the base that the exponentials are taken in
        with pytest.raises(ValueError, match="scale"):
            rig.cache.attend(0, q[0], torch.empty_like(q[0]), scale=scale)
