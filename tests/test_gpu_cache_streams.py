"""Calls on one cache run in their order whatever streams they name: streams that end with work under
way, whose handles may come again, and the default stream among others."""
import ctypes

import pytest

import test_gpu_cache as base
from test_gpu_cache import Rig

pytestmark = pytest.mark.gpu

PER_THREAD = 2  # hipStreamPerThread: one handle, a stream of every thread's own


@pytest.fixture(scope="module")
def torch():
    return base._torch()


@pytest.fixture(scope="module")
def hip():
    lib = ctypes.CDLL("libamdhip64.so")
    for name in ("hipStreamCreate", "hipStreamDestroy"):
        getattr(lib, name).argtypes = [ctypes.c_void_p]
    return lib


def _long_pass(torch, seed):
    """A cache whose attention takes a while, in many parts, with a pass of two rows open: (rig, sequence, queries)."""
    rig = Rig(torch, "bf16", heads=8, kv_heads=2, dim=128, page=64, pages=600, seed=seed)
    s = rig.add()
    rig.grow([s], [32000])
    q = rig.grow([s], [2])
    torch.cuda.synchronize()
    return rig, s, q


def test_every_threads_own_stream_is_refused(torch):
    rig = Rig(torch, "f32", heads=2, kv_heads=2, dim=64, page=16, pages=8, seed=71)
    s = rig.add()
    q = rig.grow([s], [5])
    for call in (lambda: rig.cache.attend(0, q[0], q[0], stream=PER_THREAD), lambda: rig.cache.append(0, q[0], q[0], stream=PER_THREAD),
                 lambda: rig.cache.copy(s, stream=PER_THREAD), lambda: rig.cache.compact(stream=PER_THREAD),
                 lambda: rig.cache_read_rows(s, 0, torch.empty_like(q), PER_THREAD)):
        with pytest.raises(ValueError, match="hipStreamPerThread"):
            call()
    assert rig.cache.info.pass_rows == 5 and rig.cache.info.sequences == 1
    rig.check([s], [5], q, what="behind refusals")
    with pytest.raises(ValueError, match="hipStreamPerThread"):
        rig.cache.extend([s], [1], stream=PER_THREAD)
    assert rig.cache.length(s) == 5


def test_streams_that_end_with_work_under_way(torch, hip):
    rig, s, q = _long_pass(torch, 72)
    outs = [torch.empty_like(q) for _ in range(20)]
    torch.cuda.synchronize()
    for out in outs:
        made = ctypes.c_void_p()
        assert hip.hipStreamCreate(ctypes.byref(made)) == 0
        for _ in range(5):
            rig.cache.attend(0, q[0], out[0], stream=made.value)
        assert hip.hipStreamDestroy(made) == 0
    rig.cache.truncate(s, 32000)
    last = rig.grow([s], [2])
    out = torch.empty_like(last)
    rig.cache.attend(0, last[0], out[0])
    torch.cuda.synchronize()
    for other in outs[1:]:
        assert torch.equal(other, outs[0])
    want, allowed = rig.R.attention(last[0].cpu().double(), torch.cat((rig.ref.k[s][0][:32000], rig.ref.k[s][0][-2:])),
                                    torch.cat((rig.ref.v[s][0][:32000], rig.ref.v[s][0][-2:])), 32000, dtype="bf16")
    rig.R.assert_within(out[0], want, allowed)


def test_default_and_other_streams_in_turn(torch):
    rig, s, q = _long_pass(torch, 73)
    side = [torch.cuda.Stream() for _ in range(2)]
    want = torch.empty_like(q)
    rig.cache.attend(0, q[0], want[0])
    outs = [torch.empty_like(q) for _ in range(12)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        for _ in range(3):
            rig.cache.attend(0, q[0], out[0], stream=(0, side[0].cuda_stream, side[1].cuda_stream, side[1].cuda_stream)[i % 4])
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, want)
