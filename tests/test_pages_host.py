"""What head norms with rotary positions and moves within a cache refuse
before any HIP call, and the books of pages without a device."""

import ctypes
import math

import pytest
import torch

import svdmlp
from svdmlp import _lib, pages

P = ctypes.c_void_p(256)
BAD = _lib.SVDMLP_EINVAL


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _norm_rope(lib, T=4, Hq=4, Hk=2, D=16, rot=16, scale=1.0, eps=1e-5, dtype=1, flags=0, qw=P):
    return lib.svdmlp_norm_rope(P, P, P, P, qw, P, P, P, None, T, Hq, Hk, D, rot, scale, eps, dtype, flags, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=0), b"positive"), (dict(Hq=5), b"no multiple"), (dict(rot=18), b"turned values"), (dict(rot=7), b"turned values"),
    (dict(dtype=2), b"dtype"), (dict(flags=8), b"flags"), (dict(qw=None), b"null"), (dict(scale=math.inf), b"finite"),
    (dict(D=2048, rot=2048), b"head size"), (dict(eps=0.0), b"eps"), (dict(eps=math.inf), b"eps"), (dict(T=1 << 40), b"too many"),
])
def test_norm_rope_refusals(lib, kw, msg):
    assert _norm_rope(lib, **kw) == BAD
    assert msg in lib.svdmlp_last_error()


def test_norm_rope_append_refusals(lib):
    def call(slots=P, v=P, pages=4, page=16, T=4, eps=1e-5):
        return lib.svdmlp_norm_rope_append(P, P, v, P, P, P, P, slots, P, P, P, None, T, pages, page, 4, 2, 16, 16, 1.0, eps, 1, 0, None)

    for kw in (dict(slots=None), dict(v=None), dict(pages=0), dict(page=0), dict(T=-1), dict(page=1 << 40), dict(pages=1 << 62), dict(eps=-1.0)):
        assert call(**kw) == BAD, kw


def _caches(n=2, hole=False):
    return (ctypes.c_void_p * n)(*[None if hole and i == n - 1 else 4096 * (i + 1) for i in range(n)])


@pytest.mark.parametrize("kw,msg", [
    (dict(n=0), b"no caches"), (dict(caches=None), b"no caches"), (dict(caches=_caches(hole=True)), b"null"), (dict(src=None), b"null"),
    (dict(m=0), b"0 pages"), (dict(pages=0), b"positive"), (dict(page=0), b"positive"), (dict(D=0), b"positive"), (dict(dtype=2), b"dtype"),
    (dict(page=1 << 20, D=1 << 20), b"too large"), (dict(strides=(ctypes.c_int64 * 3)(64, -16, 16)), b"negative"), (dict(pages=1 << 31), b"too large"),
    (dict(apart=-8), b"negative"),
])
def test_copy_pages_refusals(lib, kw, msg):
    a = dict(caches=_caches(), n=2, apart=0, strides=None, src=P, dst=P, rows=None, m=3, pages=4, page=16, Hk=2, D=16, dtype=1) | kw
    assert lib.svdmlp_copy_pages(*a.values(), None) == BAD
    assert msg in lib.svdmlp_last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(n=-1), b"no caches"), (dict(table=None), b"null"), (dict(path=None), b"null"), (dict(out=None), b"null"), (dict(B=0), b"positive"),
    (dict(width=0), b"positive"), (dict(width=1 << 40), b"2^31"), (dict(drafts=0), b"1 to 64"), (dict(drafts=65), b"1 to 64"),
    (dict(out=ctypes.c_void_p(P.value - 4)), b"share memory"), (dict(lengths=ctypes.c_void_p(4096), out=ctypes.c_void_p(4100)), b"share memory"),
    (dict(m=5), b"as many"), (dict(m=0), b"as many"), (dict(table_stride=-1), b"negative"), (dict(Hk=0), b"positive"),
])
def test_keep_drafts_refusals(lib, kw, msg):
    a = dict(caches=_caches(), n=2, apart=0, strides=None, table=P, lengths=P, path=P, out=ctypes.c_void_p(4096), table_stride=4, B=2, width=4, m=3, drafts=4, pages=4,
             page=16, Hk=2, D=16, dtype=1) | kw
    assert lib.svdmlp_keep_drafts(*a.values(), None) == BAD
    assert msg in lib.svdmlp_last_error()


def test_python_refusals_before_the_device_is_asked():
    q, k = torch.zeros(4, 4, 16), torch.zeros(4, 2, 16)
    pos, f, w = torch.zeros(4, dtype=torch.int64), torch.ones(8, dtype=torch.float64), torch.ones(16)
    c, i = torch.zeros(4, 6, 4, 2, 8), torch.zeros(2, dtype=torch.int32)
    for fn in (lambda: svdmlp.norm_rope(q, k, pos, f, w, w), lambda: svdmlp.copy_pages(c, i, i), lambda: svdmlp.copy_pages(list(c), i, i),
               lambda: svdmlp.keep_drafts(c, torch.zeros(2, 2, dtype=torch.int32), i, torch.zeros(2, 2, dtype=torch.int32), 3),
               lambda: svdmlp.PagePool(c)):
        with pytest.raises(ValueError, match="ROCm GPU"):
            fn()


class _Books(svdmlp.PagePool):
    """A pool whose caches are on the CPU: copies by indexing."""

    def __init__(self, caches):
        self.caches, (self.pages, self.page), self.device = caches, caches.shape[1:3], torch.device("cpu")
        self._holders, self._free = [0] * self.pages, list(range(self.pages))
        self._held, self._lengths, self._next = {}, {}, 0


def test_books_of_shared_pages(monkeypatch):
    """A shared page that is partly filled is copied by whoever writes behind it first, and only as far as it is filled."""
    calls = []

    def copy(caches, src, dst, rows=None):
        calls.append((src.tolist(), dst.tolist(), None if rows is None else rows.tolist()))

    monkeypatch.setattr(pages, "copy_pages", copy)
    pool = _Books(torch.zeros(2, 8, 4, 1, 2))
    a = pool.add()
    slots, positions, cu = pool.reserve([a], [6])
    assert slots.tolist() == [0, 1, 2, 3, 4, 5] and positions.tolist() == list(range(6)) and cu.tolist() == [0, 6]
    assert pool.alone(a, 6)
    b, c = pool.fork(a), pool.fork(a)
    assert pool.free_pages == 6 and not pool.alone(a, 1) and not pool.alone(c, 6)
    slots, positions, cu = pool.reserve([c, b, a], [1, 0, 3])
    assert calls == [([1, 1], [2, 3], [2, 2])]          # c's copy, then a's, which needs one page more
    assert pool.alone(c, 3) and not pool.alone(c, 4) and pool.alone(c, 0)
    assert slots.tolist() == [10, 14, 15, 16] and positions.tolist() == [6, 6, 7, 8] and cu.tolist() == [0, 1, 1, 4]
    assert pool.table([a, b, c])[0].tolist() == [[0, 3, 4], [0, 1, -1], [0, 2, -1]]
    pool.reserve([b], [1])                              # the last holder: no copy
    assert len(calls) == 1 and pool.free_pages == 3
    pool.trim(a, 4)
    assert pool.free_pages == 5
    pool.free(b)
    assert pool.free_pages == 6 and pool.table([a, c])[0].tolist() == [[0, -1], [0, 2]]
    assert pool.compact() == 2 and calls[1] == ([2], [1], None)
    assert pool.table([c])[0].tolist() == [[0, 1]] and pool.table([])[0].shape == (0, 1)
    pool.free(a), pool.free(c)
    assert pool.free_pages == 8 and pool.compact() == 0


def test_books_copy_after_a_cut_into_a_shared_page(monkeypatch):
    calls = []
    monkeypatch.setattr(pages, "copy_pages", lambda caches, src, dst, rows=None: calls.append((src.tolist(), dst.tolist(), rows.tolist())))
    pool = _Books(torch.zeros(2, 4, 4, 1, 2))
    a = pool.add()
    pool.reserve([a], [8])
    b = pool.fork(a)
    pool.trim(b, 7)
    with pytest.raises(ValueError, match="once"):
        pool.reserve([b, b], [1, 1])
    slots, _, _ = pool.reserve([b], [2])  # a copy, then a page of its own
    assert calls == [([1], [2], [3])] and slots.tolist() == [11, 12] and pool.free_pages == 0
    with pytest.raises(RuntimeError, match="1 pages needed"):
        pool.reserve([a], [1])
