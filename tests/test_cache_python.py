"""The Python side of the paged cache without a GPU: numbers that the library's 32-bit arguments do not hold, and the rows that a
pass has when a call never reached the library."""
import types

import pytest

import gradhip as G


class Library:
    """Stands in for the library: accepts everything, opens passes, remembers the calls."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def cache(monkeypatch):
    lib = Library()
    monkeypatch.setattr(G, "load_library", lambda: lib)
    cache = G.Cache(layers=2, heads=4, kv_heads=2, head_dim=64, pages=8)
    cache._h = 1
    cache._device = 0
    yield cache
    cache._h = None


def rows(n, heads, dtype="torch.float32"):
    return types.SimpleNamespace(shape=(n, heads, 64), dtype=dtype, device=types.SimpleNamespace(type="cuda", index=0),
                                 stride=lambda: (heads * 64, 64, 1), data_ptr=lambda: 4096)


@pytest.mark.parametrize("seqs,counts", [([0], [1.5]), (["0"], [3]), ([0, None], [1, 1]), ([0], [2 ** 32 + 3]), ([0], [3 - 2 ** 32]), ([2 ** 32], [3]), ([0, 1], [3])])
def test_an_extend_that_never_reached_the_library_leaves_the_pass(cache, seqs, counts):
    """The pass of 20 rows is still open in the library: tensors of fewer rows would be read and written out of range."""
    cache.extend([0, 1], [15, 5])
    before = len(cache._lib.calls)
    with pytest.raises((TypeError, ValueError)):
        cache.extend(seqs, counts)
    assert len(cache._lib.calls) == before
    for n in (0, 2, 19):
        with pytest.raises(ValueError, match="shape"):
            cache.attend(0, rows(n, 4), rows(20, 4))
        with pytest.raises(ValueError, match="shape"):
            cache.attend(0, rows(20, 4), rows(n, 4))
        with pytest.raises(ValueError, match="shape"):
            cache.append(0, rows(20, 2), rows(n, 2))
    cache.attend(0, rows(20, 4), rows(20, 4))
    assert cache._lib.calls[-1][0] == "gh_cache_attend"


def test_numbers_of_other_kinds_are_numbers(cache):
    import numpy as np
    cache.extend(np.array([0, 1]), np.array([15, 5], dtype=np.int16))
    with pytest.raises(ValueError, match="shape"):
        cache.attend(0, rows(19, 4), rows(20, 4))
    cache.attend(np.int64(1), rows(20, 4), rows(20, 4), window=np.int32(7))
    name, args = cache._lib.calls[-1]
    assert name == "gh_cache_attend" and args[1] == 1 and args[6] == 7


@pytest.mark.parametrize("beyond", [2 ** 31, 2 ** 32, 2 ** 32 + 5, -2 ** 31 - 1, -2 ** 32])
def test_numbers_beyond_32_bits_are_refused(cache, beyond):
    """Cut to 32 bits, a length of 2^32 would empty a sequence, a window of 2^32 + 5 show five positions."""
    cache.extend([0], [20])
    before = len(cache._lib.calls)
    k, q = rows(20, 2), rows(20, 4)
    for call in (lambda: cache.fork(beyond), lambda: cache.fork(0, beyond), lambda: cache.copy(beyond), lambda: cache.truncate(beyond, 0),
                 lambda: cache.truncate(0, beyond), lambda: cache.drop(beyond), lambda: cache.length(beyond), lambda: cache.append(beyond, k, k),
                 lambda: cache.attend(beyond, q, q), lambda: cache.attend(0, q, q, window=beyond), lambda: cache.read(beyond, k, k, layer=0),
                 lambda: cache.read(0, k, k, start=beyond, layer=0), lambda: cache.read(0, k, k, layer=beyond),
                 lambda: G.Cache(layers=2, heads=4, kv_heads=2, head_dim=64, pages=beyond), lambda: G.Cache(layers=beyond, heads=4, kv_heads=2, head_dim=64, pages=8)):
        with pytest.raises((ValueError, IndexError), match="32 bits"):
            call()
    assert len(cache._lib.calls) == before


def test_sessions_take_no_such_numbers_either(cache):
    class Session(G.Session):
        def close(self):
            pass

    session = Session.__new__(Session)
    session._h, session.batch, session.vocab = 1, 2, 10
    for seqs in ([0, 2 ** 32], [2 ** 31, 0], [0.5, 1]):
        with pytest.raises((ValueError, TypeError)):
            session.restore(cache, seqs, [[1, 2], [3, 4]])
    for seqs in ([0], [0, 1, 2], 0):
        with pytest.raises(ValueError, match="sequence for each"):
            session.restore(cache, seqs, [[1, 2], [3, 4]])
    with pytest.raises(ValueError, match="32 bits"):
        session.store(cache, 2 ** 32)
    assert not [c for c in cache._lib.calls if c[0].startswith("gh_session")]
    session.restore(cache, [0, 1], [[1, 2], [3, 4]])
    name, args = cache._lib.calls[-1]
    assert name == "gh_session_restore" and list(args[2]) == [0, 1]
