"""Rows moved within a paged cache, and the host's books of its pages.

    copy_pages(caches, src, dst, rows)              pages to other pages
    keep_drafts(caches, block_table, lengths, path, drafts)   accepted drafts' rows
    PagePool(caches)                                which sequence holds which pages

A model has a cache of keys and one of values a layer, and a page has the same
number in all of them: ``caches`` are all of these, (n, pages, page size, Hk, D)
in one tensor or a list of (pages, page size, Hk, D) tensors laid out alike, and
one call moves the rows of all.  bfloat16 or float32 on a ROCm GPU; work goes to
the current stream, and nothing waits for it.
"""

from __future__ import annotations

import ctypes
import heapq

import torch

from . import _lib
from .decoder import (_Strides3, _address, _apart, _bytes, _capturing, _extent, _gradients, _index, _launch, _overlap, _refuse_device,
                      _refuse_dtype, _refuse_grad, _writable)
from .ops import _ACT_CODES


_Pointer = ctypes.c_void_p * 1


def _cache_set(name: str, caches):
    """(shape of a cache, dtype code, all of them, addresses, n, elements apart, device index, strides) of the caches, checked."""
    if isinstance(caches, torch.Tensor):
        shape = caches.shape
        if len(shape) != 5 or 0 in shape:
            raise ValueError(f"caches must have shape (caches, pages, page size, heads, head size), got {tuple(shape)}")
        _check_cache(name, caches)
        st = caches.stride()
        return (shape[1:], _ACT_CODES[caches.dtype], (caches,), _Pointer(caches.data_ptr()), shape[0], st[0] if shape[0] > 1 else 0,
                caches.get_device(), _Strides3(st[1], st[2], st[3]))
    else:
        every = tuple(caches)
        if not every or not all(isinstance(c, torch.Tensor) for c in every):
            raise ValueError("caches must be a tensor or a nonempty list of tensors")
        one, n = every[0], len(every)
        if one.dim() != 4 or not one.numel():
            raise ValueError(f"a cache must have shape (pages, page size, heads, head size), got {tuple(one.shape)}")
        shape, dtype, index, strides = one.shape, one.dtype, one.get_device(), one.stride()
        for c in every:
            if c.shape != shape or c.dtype != dtype or c.get_device() != index or c.stride() != strides:
                raise ValueError("the caches must be alike: shape, dtype, device and strides")
        for c in every if _gradients() else every[:1]:
            _check_cache(name, c)
        pointers = [c.data_ptr() for c in every]
        reach, ends = _extent(one), sorted(pointers)
        if any(b - a < reach for a, b in zip(ends, ends[1:])):  # views of one buffer: exactly
            order = sorted(every, key=torch.Tensor.data_ptr)
            for i, a in enumerate(order):
                for b in order[i + 1:]:
                    if b.data_ptr() - a.data_ptr() >= reach:
                        break
                    if _overlap(a, b):
                        raise ValueError("the caches must not overlap")
    return shape, _ACT_CODES[dtype], every, (ctypes.c_void_p * n)(*pointers), n, 0, index, _Strides3(*strides[:3])


def _check_cache(name: str, c: torch.Tensor) -> None:
    if c.dtype not in _ACT_CODES:
        _refuse_dtype(c.dtype)
    if not c.is_cuda:
        _refuse_device(name, c)
    if _gradients():
        _refuse_grad(name, c)
    _writable("caches", c, c.shape, c)


def _indices_apart(every, *tensors) -> None:
    """No cache shares memory with the index tensors."""
    spans = [_bytes(t) for t in tensors if t is not None and t.numel()]
    for c in every:
        a, b = _bytes(c)
        for p, e in spans:
            if p < b and a < e:
                _apart("caches", c, *(t for t in tensors if t is not None))


def copy_pages(caches, src, dst, rows=None) -> None:
    """Page ``dst[i]`` of every cache becomes page ``src[i]``: all of its rows, or
    the first ``rows[i]``.  src, dst and rows are int32 or int64 tensors on the
    device, one value a pair.  A pair with a page outside the cache, or of a page
    and itself, is skipped.  The pages of dst have to differ from each other and
    from those of src."""
    (pages, page, Hk, D), code, every, pointers, n, apart, index, strides = _cache_set("copy_pages", caches)
    if not isinstance(src, torch.Tensor) or src.dim() != 1:
        raise ValueError("src must hold the pages to copy")
    m = src.shape
    src, dst = _index("src", src, m, torch.int32, index), _index("dst", dst, m, torch.int32, index)
    rows = None if rows is None else _index("rows", rows, m, torch.int32, index)
    if not m[0]:
        return
    _indices_apart(every, src, dst, rows)
    _launch(index, _lib.load().svdmlp_copy_pages, _address(pointers), n, apart, _address(strides), src.data_ptr(), dst.data_ptr(),
            None if rows is None else rows.data_ptr(), m[0], pages, page, Hk, D, code)


def keep_drafts(caches, block_table, lengths, path, drafts: int) -> torch.Tensor:
    """After a tree of drafts has been verified (:func:`svdmlp.cache_attention` with
    ``tree``): the accepted drafts' rows go behind the context, in every cache, and
    the sequences' new lengths are returned (int32).

    The last ``drafts`` (1 to 64) of a sequence's ``lengths[b]`` tokens are its
    drafts.  ``path`` (B, m), m up to ``drafts``, names the accepted ones in
    increasing order, -1 behind the last: draft ``path[b, i]`` becomes the i-th token
    behind the context.  A path ends before the first number that does not
    increase or is no draft.  A sequence of fewer tokens than ``drafts`` keeps
    them and its length.  block_table and lengths are those of
    cache_attention; rows in pages outside the cache are not moved.  A page that
    holds drafts has to be of one sequence alone, as PagePool.reserve leaves it
    (PagePool.alone)."""
    (pages, page, Hk, D), code, every, pointers, n, apart, index, strides = _cache_set("keep_drafts", caches)
    if isinstance(drafts, bool) or not isinstance(drafts, int) or not 1 <= drafts <= 64:
        raise ValueError(f"1 to 64 drafts a sequence, got {drafts}")
    if block_table.dim() != 2 or block_table.shape[1] == 0:
        raise ValueError("block_table must have shape (sequences, pages of the longest)")
    B, width = block_table.shape
    if path.dim() != 2 or path.shape[0] != B or not 1 <= path.shape[1] <= drafts:
        raise ValueError(f"path must have shape ({B}, 1 to {drafts}), got {tuple(path.shape)}")
    path = _index("path", path, path.shape, torch.int32, index)
    if block_table.stride(1) != 1 or block_table.dtype is not torch.int32 or block_table.get_device() != index:
        block_table = _index("block_table", block_table, (B, width), torch.int32, index)
    lengths = _index("lengths", lengths, (B,), torch.int32, index)
    out = lengths.new_empty(B)
    if not B:
        return out
    _indices_apart(every, block_table, lengths, path)
    _launch(index, _lib.load().svdmlp_keep_drafts, _address(pointers), n, apart, _address(strides), block_table.data_ptr(), lengths.data_ptr(),
            path.data_ptr(), out.data_ptr(), block_table.stride(0), B, width, path.shape[1], drafts, pages, page, Hk, D,
            code)
    return out


class PagePool:
    """The host's books of a paged cache: which sequence holds which pages, and how
    many hold each.  Sequences are numbers that :meth:`add` and :meth:`fork` give
    out.  The books are kept on the host, without waiting for the device; the rows
    that they move (:meth:`reserve`, :meth:`compact`) move on the current stream by
    :func:`copy_pages`, so calls on other streams have to be ordered with it.  What
    it gives out is of the moment, and is refused to a stream that is being
    captured.  A refused call changes nothing.  Calls take time by the pages that
    their sequences hold (:meth:`table`: 64 of 4000 tokens in pages of 16 0.9 ms, in pages
    of 64 0.25) and by the tokens asked for (:meth:`reserve`: 8192 2.4 ms)."""

    def __init__(self, caches):
        shape, _, _, _, _, _, index, _ = _cache_set("PagePool", caches)
        self.caches = caches if isinstance(caches, torch.Tensor) else tuple(caches)
        self.pages, self.page = shape[:2]
        self.device = torch.device("cuda", index)
        self._holders = [0] * self.pages
        self._free = list(range(self.pages))  # a heap: the lowest page goes first
        self._held: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        return self._lengths[self._known(sequence)]

    def _known(self, sequence: int) -> int:
        if sequence not in self._held:
            raise KeyError(f"no sequence {sequence}")
        return sequence

    def add(self) -> int:
        """A new sequence, without tokens."""
        self._held[self._next], self._lengths[self._next] = [], 0
        self._next += 1
        return self._next - 1

    def alone(self, sequence: int, tokens: int) -> bool:
        """Whether no other sequence holds the pages of the sequence's last tokens."""
        first = max(self.length(sequence) - tokens, 0) // self.page
        return all(self._holders[p] == 1 for p in self._held[sequence][first:])

    def fork(self, sequence: int) -> int:
        """A new sequence of the same tokens, in the same pages: the last one, partly filled, is copied when one of its holders
        reserves more."""
        held = list(self._held[self._known(sequence)])
        new = self.add()
        self._held[new], self._lengths[new] = held, self._lengths[sequence]
        for p in held:
            self._holders[p] += 1
        return new

    def free(self, sequence: int) -> None:
        """The sequence is gone; pages that no other holds are free."""
        self._release(self._held.pop(self._known(sequence)))
        del self._lengths[sequence]

    def trim(self, sequence: int, length: int) -> None:
        """The sequence's first `length` tokens stay."""
        if not 0 <= length <= self.length(sequence):
            raise ValueError(f"sequence {sequence} has {self.length(sequence)} tokens, cannot be trimmed to {length}")
        held, keep = self._held[sequence], -(-length // self.page)
        self._release(held[keep:])
        del held[keep:]
        self._lengths[sequence] = length

    def _release(self, pages) -> None:
        for p in pages:
            self._holders[p] -= 1
            if not self._holders[p]:
                heapq.heappush(self._free, p)

    def reserve(self, sequences, tokens) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Room for tokens[i] more tokens of sequence sequences[i], each once: (slots,
        positions, cu_seqlens) of the packed new tokens, as the operators take them.
        A partly filled last page that others hold too is copied first."""
        self._uncaptured()
        sequences, tokens = [self._known(s) for s in sequences], [int(t) for t in tokens]
        if len(sequences) != len(tokens) or any(t < 0 for t in tokens):
            raise ValueError("reserve takes a number of tokens, not negative, for each sequence")
        if len(set(sequences)) < len(sequences):
            raise ValueError("reserve takes a sequence once")
        # What it takes: pages behind the last, and copies of shared ones.
        left, need = {}, 0
        for s, t in zip(sequences, tokens):
            length = self._lengths[s]
            if t and length % self.page:
                last = self._held[s][-1]
                holders = left.get(last, self._holders[last])
                if holders > 1:
                    need += 1
                    left[last] = holders - 1
            need += -(-(length + t) // self.page) - -(-length // self.page)
        if need > len(self._free):
            raise RuntimeError(f"{need} pages needed, {len(self._free)} of {self.pages} free")
        slots, positions, cu, copies = [], [], [0], []
        for s, t in zip(sequences, tokens):
            held, length = self._held[s], self._lengths[s]
            if t and length % self.page and self._holders[held[-1]] > 1:
                copies.append((held[-1], self._take(), length % self.page))
                self._holders[held[-1]] -= 1
                held[-1] = copies[-1][1]
            while len(held) * self.page < length + t:
                held.append(self._take())
            for x in range(length, length + t):
                slots.append(held[x // self.page] * self.page + x % self.page)
            positions.extend(range(length, length + t))
            cu.append(cu[-1] + t)
            self._lengths[s] = length + t
        if copies:
            self._copy(*zip(*copies))
        return self._tensor(slots, torch.int64), self._tensor(positions, torch.int64), self._tensor(cu, torch.int32)

    def _uncaptured(self) -> None:
        if self.device.type == "cuda" and _capturing(self.device.index):
            raise RuntimeError("the books of pages are not for a stream that is being captured")

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._holders[p] = 1
        return p

    def _tensor(self, values, dtype) -> torch.Tensor:
        if self.device.type != "cuda":
            return torch.tensor(values, dtype=dtype)
        # (pinned: a copy from other memory waits for the stream)
        return torch.tensor(values, dtype=dtype, pin_memory=True).to(self.device, non_blocking=True)

    def _copy(self, src, dst, rows=None) -> None:
        with torch.no_grad():
            copy_pages(self.caches, self._tensor(src, torch.int32), self._tensor(dst, torch.int32),
                       None if rows is None else self._tensor(rows, torch.int32))

    def table(self, sequences) -> tuple[torch.Tensor, torch.Tensor]:
        """(block_table, lengths) of the sequences, as the operators take them."""
        self._uncaptured()
        held = [self._held[self._known(s)] for s in sequences]
        width = max([1, *map(len, held)])
        return (self._tensor([h + [-1] * (width - len(h)) for h in held], torch.int32).view(len(held), width),
                self._tensor([self._lengths[s] for s in sequences], torch.int32))

    def compact(self) -> int:
        """Moves pages from the end to free ones at the front; returns how many are
        held, all of them now before the free ones.  Block tables from before are
        stale."""
        self._uncaptured()
        used = self.pages - len(self._free)
        dst = sorted(p for p in self._free if p < used)
        src = [p for p in range(used, self.pages) if self._holders[p]]
        if src:
            self._copy(src, dst)
            moved = dict(zip(src, dst))
            for a, b in moved.items():
                self._holders[b], self._holders[a] = self._holders[a], 0
            for s, held in self._held.items():
                self._held[s] = [moved.get(p, p) for p in held]
            self._free = list(range(used, self.pages))
        return used
