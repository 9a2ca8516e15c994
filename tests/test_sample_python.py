"""Sampling by row without a GPU: its definition on rows with known answers, what the calls refuse, the Python side."""
import ctypes as C
import types

import numpy as np
import pytest

import gradhip as G
import sample_reference as R


def test_the_definition():
    x = np.log(np.array([0.1, 0.4, 0.1, 0.3, 0.1]))
    assert [R.pick(x, u)[0] for u in (0.0, 0.099, 0.11, 0.49, 0.51, 0.61, 0.89, 0.91, 1.0)] == [0, 0, 1, 1, 2, 3, 3, 4, 4]
    assert np.flatnonzero(R.kept_weights(x, top_k=3)).tolist() == [0, 1, 3]
    assert np.flatnonzero(R.kept_weights(x, top_p=0.75)).tolist() == [0, 1, 3]
    assert np.flatnonzero(R.kept_weights(x, top_p=0.65)).tolist() == [1, 3]
    assert np.flatnonzero(R.kept_weights(x, top_k=2, top_p=0.58)).tolist() == [1, 3]  # 0.4 of 0.7 is less
    assert np.flatnonzero(R.kept_weights(x, top_k=2, top_p=0.57)).tolist() == [1]
    assert np.flatnonzero(R.kept_weights(x, min_p=0.3)).tolist() == [1, 3]
    assert np.flatnonzero(R.kept_weights(x, temperature=0.0)).tolist() == [1]
    assert R.pick(np.full(4, -np.inf), 0.3) == (-1, 0.0)
    assert R.pick(np.zeros(4), 0.5) == (1, 0.25)


def args(**change):
    a = G.GhSampleArgs(4096, 100, 0, 2, 100, 0, None, None, None, None, 4096, 4096, None, None, 0)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,match", [
    (dict(type=3), b"type"), (dict(type=-1), b"type"), (dict(rows=-1), b"rows"), (dict(rows=2 ** 24 + 1), b"rows"), (dict(vocab=0), b"vocab"),
    (dict(vocab=2 ** 20 + 1), b"vocab"), (dict(row_stride=-1), b"row_stride"), (dict(logits=None), b"null"), (dict(uniforms=None), b"null"),
    (dict(ids=None), b"null"),
])
def test_calls_that_are_refused(change, match):
    lib = G.load_library()
    assert lib.gh_sample(C.byref(args(**change)), None) == G.GH_ERR_INVALID_ARGUMENT
    assert match in lib.gh_last_error()


def test_null_arguments_and_no_rows():
    lib = G.load_library()
    assert lib.gh_sample(None, None) == G.GH_ERR_INVALID_ARGUMENT
    assert lib.gh_sample_workspace(0, 1, 100, None) == G.GH_ERR_INVALID_ARGUMENT
    assert lib.gh_sample(C.byref(args(rows=0, logits=None, uniforms=None, ids=None)), None) == G.GH_OK
    assert C.sizeof(G.GhSampleArgs) == 104 and G.GhSampleArgs.temperature.offset == 32 and G.GhSampleArgs.workspace_bytes.offset == 96


def test_workspaces():
    for dtype in ("f32", "bf16", "f16"):
        assert G.sample_workspace(0, 1, dtype) == 0
        for rows, vocab in ((1, 1), (1, 262144), (300, 5000), (2 ** 24, 2 ** 20)):
            assert G.sample_workspace(rows, vocab, dtype) >= 0
    for bad in ((-1, 10), (1, 0), (1, 2 ** 20 + 1), (2 ** 24 + 1, 5)):
        with pytest.raises(ValueError):
            G.sample_workspace(*bad)
    for bad in ((2 ** 33, 10), (1, 2 ** 32 + 7)):
        with pytest.raises(ValueError, match="beyond 32 bits"):
            G.sample_workspace(*bad)
    with pytest.raises(ValueError, match="type"):
        G.sample_workspace(1, 10, "f64")


def test_a_workspace_does_for_fewer_rows():
    for vocab in (100, 8192, 8193, 16384, 32000, 50257, 131072, 131073, 201001, 2 ** 20):
        needs = [G.sample_workspace(rows, vocab) for rows in range(0, 700)]
        assert needs == sorted(needs), vocab
        assert needs[0] == 0 and (needs[1] > 0) == (vocab > 8192)


def tensor(*shape, dtype="torch.float32", device="cuda:0", stride=None):
    if stride is None:
        stride = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
    kind, index = device.split(":") if ":" in device else (device, None)

    class Device(types.SimpleNamespace):
        def __eq__(self, other):
            return (self.type, self.index) == (other.type, other.index)

    return types.SimpleNamespace(shape=shape, dtype=dtype, device=Device(type=kind, index=index), stride=lambda: tuple(stride), data_ptr=lambda: 4096,
                                 is_contiguous=lambda: True, numel=lambda: int(np.prod(shape)), element_size=lambda: 4)


@pytest.mark.parametrize("change", [
    dict(logits=tensor(4, 50, dtype="torch.float64")), dict(logits=tensor(200)), dict(logits=tensor(4, 50, device="cpu")),
    dict(logits=tensor(4, 50, stride=(1, 4))), dict(uniforms=tensor(3)), dict(uniforms=None), dict(ids=None), dict(ids=tensor(4, dtype="torch.int64")),
    dict(uniforms=tensor(4, dtype="torch.float64")), dict(temperature=tensor(5)), dict(temperature=tensor(4, device="cuda:1")),
    dict(top_k=tensor(4, dtype="torch.int64")), dict(top_p=tensor(4, stride=(2,))), dict(min_p=tensor(4, 1)), dict(probs=tensor(4, dtype="torch.float16")),
    dict(workspace=tensor(9, device="cuda:1")), dict(ids=tensor(4, dtype="torch.int32", device="cpu")),
])
def test_tensors_that_are_refused(change, monkeypatch):
    calls = []

    class Library:
        def gh_sample(self, *a):
            calls.append(a)
            return 0

    monkeypatch.setattr(G, "load_library", Library)
    good = dict(logits=tensor(4, 50), uniforms=tensor(4), ids=tensor(4, dtype="torch.int32"))
    G.sample(**good)
    G.sample(**good, temperature=tensor(4), top_k=tensor(4, dtype="torch.int32"), top_p=tensor(4), min_p=tensor(4), probs=tensor(4), workspace=tensor(9))
    assert len(calls) == 2
    with pytest.raises(ValueError, match="sample: "):
        G.sample(**{**good, **change})
    assert len(calls) == 2
