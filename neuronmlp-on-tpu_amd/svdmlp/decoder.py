"""The operators around the MLP block of a decoder layer, on MI355X.

    rope(q, k, positions, inv_freq)                 rotary positions
    rope_append(q, k, v, ..., k_cache, v_cache, slots)   ... into a paged cache
    prompt_attention(q, k, v, cu_seqlens)           attention over packed prompts
    cache_attention(q, k_cache, v_cache, table, lengths)  decode, drafted trees
    residual_norm(x, branch, weight)                sum after a block, next norm

With the projections and :func:`svdmlp.svd_mlp` they make a decoder layer
(bench/e2e_block.py:205-278 has its prefill form without positions).  Tensors
are bfloat16 or float32 on a ROCm GPU; queries are (rows, Hq, D), keys and values
(rows, Hk, D) with Hk dividing Hq, caches (pages, page size, Hk, D).  Slices
of a fused projection are read in place (last dimension contiguous, 16-byte
aligned rows); others are copied first.  Work goes to the current stream.

As everywhere in this package the operators are for inference: tensors that
ask for a gradient are refused (wrap the call in ``torch.no_grad()``).
Every call goes to libsvdmlp.so; there is no CPU or PyTorch fallback.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .ops import _ACT_CODES, _on_device, _stream


def _check(name: str, dtype: torch.dtype, *tensors) -> torch.device:
    """All tensors on one GPU; those of the activation's type; none that asks for a gradient."""
    if dtype not in _ACT_CODES:
        raise TypeError("supported dtypes are bfloat16 and float32")
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"{name} runs on a ROCm GPU; got tensors on {dev}")
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t.device != dev:
            raise ValueError("all inputs must be on the same device")
        if grad and t.requires_grad:
            raise ValueError(f"{name} has no gradient: call it under torch.no_grad(), or on detached tensors")
    return dev


def _same_dtype(x, *tensors) -> None:
    for t in tensors:
        if t.dtype != x.dtype:
            raise TypeError("all inputs must have the same dtype")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels can read it in place (last dimension
    contiguous, rows in whole 16-byte pieces), else a contiguous copy."""
    es = t.element_size()
    if t.stride(-1) != 1 and t.shape[-1] != 1 or t.data_ptr() % 16 or any(s * es % 16 for s in t.stride()[:-1]):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _writable(name: str, t: torch.Tensor, shape, like: torch.Tensor) -> None:
    """An output: of the shape, type and device, its elements all apart."""
    if tuple(t.shape) != tuple(shape) or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be a {tuple(shape)} tensor of {like.dtype} on {like.device}")
    reach = 0
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            raise ValueError(f"{name} must not overlap itself")
        reach += stride * (size - 1)
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _aligned(name: str, t: torch.Tensor) -> None:
    es = t.element_size()
    if t.data_ptr() % 16 or any(s * es % 16 for s, n in zip(t.stride()[:-1], t.shape) if n > 1):
        raise ValueError(f"rows of {name} must be 16-byte aligned")


def _extent(t: torch.Tensor, first: int = 0) -> int:
    """Bytes from the first element of dimensions `first` on to the end of their last."""
    return (sum(s * (n - 1) for s, n in zip(t.stride()[first:], t.shape[first:])) + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two nonempty tensors may share memory (slices side by side in the rows of one buffer do not)."""
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + _extent(a) <= pb or pb + _extent(b) <= pa:
        return False
    pitch = a.stride(0) * a.element_size()
    wa, wb = _extent(a, 1), _extent(b, 1)
    if pitch == b.stride(0) * b.element_size() and max(wa, wb) <= pitch:
        d = (pb - pa) % pitch
        return d < wa or d + wb > pitch
    return True


def _apart(name: str, out: torch.Tensor, *tensors, own=()) -> None:
    """out shares no memory with the tensors, and with those of `own` only as the very same elements."""
    if out.numel() == 0:
        return
    for t in tensors:
        if t.numel() and _overlap(out, t) and not any(t is o and out.data_ptr() == t.data_ptr() and out.stride() == t.stride()
                                                      for o in own):
            raise ValueError(f"{name} must not overlap the inputs")


def _index(name: str, t: torch.Tensor, shape, dtype, dev) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an int32 or int64 tensor")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError("all inputs must be on the same device")
    return t.to(dtype).contiguous()


def _heads(q, k, *more) -> tuple[int, int, int, int]:
    """(T, Hq, Hk, D) of q (T, Hq, D) and k, v ... (T, Hk, D)."""
    for t in (q, k, *more):
        if t.dim() != 3:
            raise ValueError(f"expected (tokens, heads, head size), got {tuple(t.shape)}")
    T, Hq, D = q.shape
    Hk = k.shape[1]
    for t in (k, *more):
        if tuple(t.shape) != (T, Hk, D):
            raise ValueError(f"keys and values must have shape {(T, Hk, D)}, got {tuple(t.shape)}")
    if min(Hq, Hk, D) <= 0 or Hq % Hk:
        raise ValueError(f"{Hq} query heads are no multiple of {Hk} key/value heads")
    return T, Hq, Hk, D


def _strides(*values):
    return (ctypes.c_int64 * len(values))(*values)


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------

def rope_frequencies(rot: int, theta: float = 10000.0, *, scaling: dict | None = None,
                     device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq, scale) for :func:`rope`: rot/2 frequencies in float64,
    theta^(-2p/rot), and the factor on cos and sin.  ``scaling`` stretches them
    for contexts longer than the model was trained on:

    * ``{"type": "linear", "factor": f}``: every frequency / f
    * ``{"type": "ntk", "factor": f}``: theta * f^(rot / (rot - 2)), so that
      the lowest frequency is divided by f and the highest kept
    * ``{"type": "llama3", "factor", "low_freq_factor", "high_freq_factor",
      "original_context"}``: wavelengths beyond original_context /
      low_freq_factor are stretched by factor, those below original_context /
      high_freq_factor kept, in between linear in original_context / wavelength
    * ``{"type": "yarn", "factor", "original_context", "beta_fast": 32,
      "beta_slow": 1}``: pairs that turn beta_fast times over original_context
      kept, those that turn beta_slow times divided by factor, linear in the
      pair's number in between; scale 0.1 ln(factor) + 1
    """
    if isinstance(rot, bool) or not isinstance(rot, int) or rot <= 0 or rot % 2:
        raise ValueError(f"rot must be a positive even integer, got {rot}")
    if not theta > 1:
        raise ValueError(f"theta must be over 1, got {theta}")
    half = rot // 2
    kind = "none" if scaling is None else scaling.get("type")
    if kind not in ("none", "linear", "ntk", "llama3", "yarn"):
        raise ValueError(f"unknown scaling {kind!r}")
    if kind != "none" and not float(scaling["factor"]) >= 1:
        raise ValueError(f"the scaling factor must be at least 1, got {scaling['factor']}")
    pair = torch.arange(half, dtype=torch.float64)
    scale = 1.0
    if kind == "ntk" and rot > 2:
        theta = theta * float(scaling["factor"]) ** (rot / (rot - 2))
    freq = float(theta) ** (-pair / half)
    if kind == "linear":
        freq = freq / float(scaling["factor"])
    elif kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not 0 < low < high:
            raise ValueError("high_freq_factor must be over low_freq_factor, and both positive")
        turns = float(scaling["original_context"]) * freq / (2 * math.pi)
        kept = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (kept + (1 - kept) / float(scaling["factor"]))
    elif kind == "yarn":
        context = float(scaling["original_context"])

        def number(turns):  # the pair that turns so many times over the context
            return half * math.log(context / (2 * math.pi * turns)) / math.log(theta)

        first = max(math.floor(number(float(scaling.get("beta_fast", 32)))), 0)
        last = min(math.ceil(number(float(scaling.get("beta_slow", 1)))), rot - 1)
        ramp = ((pair - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        freq = freq * (1 - ramp) + freq / float(scaling["factor"]) * ramp
        scale = 0.1 * math.log(float(scaling["factor"])) + 1.0
    return freq.to(device) if device is not None else freq, scale


def _rope_args(name, q, k, more, positions, inv_freq, scale):
    T, Hq, Hk, D = _heads(q, k, *more)
    _same_dtype(q, k, *more)
    dev = _check(name, q.dtype, q, k, *more)
    if inv_freq.dim() != 1 or not inv_freq.is_floating_point() or inv_freq.device != dev:
        raise ValueError("inv_freq must be a 1-D floating point tensor on the inputs' device")
    rot = 2 * inv_freq.shape[0]
    if not 0 < rot <= D:
        raise ValueError(f"{rot} turned values (two a frequency) of a head of {D}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    positions = _index("positions", positions, (T,), torch.int64, dev)
    return T, Hq, Hk, D, dev, rot, positions, inv_freq.to(torch.float64).contiguous()


def _last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def rope(q, k, positions, inv_freq, *, interleaved: bool = False, scale: float = 1.0,
         out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, k) with the first ``2 * len(inv_freq)`` values of each head turned
    by the tokens' positions: pair p, by positions[t] * inv_freq[p] (in 64 bits),
    is (p, p + rot/2), or (2p, 2p + 1) when ``interleaved``; the rest of the
    head is copied.  ``scale`` multiplies cos and sin (see
    :func:`rope_frequencies`).  q (T, Hq, D), k (T, Hk, D), positions (T,).
    ``out``: the pair of tensors to write, which may be q and k themselves."""
    T, Hq, Hk, D, dev, rot, positions, inv_freq = _rope_args("rope", q, k, (), positions, inv_freq, scale)
    if out is None:
        qo, ko = torch.empty((T, Hq, D), dtype=q.dtype, device=dev), torch.empty((T, Hk, D), dtype=q.dtype, device=dev)
    else:
        qo, ko = out
        _writable("out[0]", qo, (T, Hq, D), q)
        _writable("out[1]", ko, (T, Hk, D), q)
        _apart("out[0]", qo, q, k, ko, own=(q,))
        _apart("out[1]", ko, k, q, own=(k,))
    if T == 0:
        return qo, ko
    q, k = _last(q), _last(k)
    lib = _lib.load()
    st = _strides(q.stride(0), q.stride(1), k.stride(0), k.stride(1), qo.stride(0), qo.stride(1), ko.stride(0), ko.stride(1))
    _lib.check(_on_device(dev, lambda: lib.svdmlp_rope(
        q.data_ptr(), k.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), qo.data_ptr(), ko.data_ptr(),
        ctypes.addressof(st), T, Hq, Hk, D, rot, scale, _ACT_CODES[q.dtype],
        _lib.SVDMLP_ROPE_INTERLEAVED if interleaved else 0, _stream(dev))))
    return qo, ko


def _cache(k_cache, v_cache, q, Hk, D):
    for c in (k_cache, v_cache):
        if c.dim() != 4 or tuple(c.shape[2:]) != (Hk, D) or c.shape[:2] != k_cache.shape[:2] or min(c.shape[:2]) <= 0:
            raise ValueError(f"caches must have shape (pages, page size, {Hk}, {D}), got {tuple(c.shape)}")
    return int(k_cache.shape[0]), int(k_cache.shape[1])


def rope_append(q, k, v, positions, inv_freq, k_cache, v_cache, slots, *, interleaved: bool = False,
                scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`rope` on the way into a paged cache: returns the turned q, and
    writes the turned k and v (T, Hk, D) to row ``slots[t] % page size`` of page
    ``slots[t] // page size`` of the caches (pages, page size, Hk, D).  A token
    whose slot lies outside the cache (-1: padding) is not written.  The slots of
    one call have to differ from each other."""
    T, Hq, Hk, D, dev, rot, positions, inv_freq = _rope_args("rope_append", q, k, (v,), positions, inv_freq, scale)
    _same_dtype(q, k_cache, v_cache)
    _check("rope_append", q.dtype, q, k_cache, v_cache)
    pages, page = _cache(k_cache, v_cache, q, Hk, D)
    _writable("k_cache", k_cache, k_cache.shape, q)
    _writable("v_cache", v_cache, v_cache.shape, q)
    _apart("k_cache", k_cache, v_cache, q, k, v)
    _apart("v_cache", v_cache, q, k, v)
    slots = _index("slots", slots, (T,), torch.int64, dev)
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=dev)
    else:
        _writable("out", out, (T, Hq, D), q)
        _apart("out", out, q, k, v, k_cache, v_cache, own=(q,))
    if T == 0:
        return out
    q, k, v = _last(q), _last(k), _last(v)
    lib = _lib.load()
    st = _strides(q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), out.stride(0), out.stride(1),
                  *k_cache.stride()[:3], *v_cache.stride()[:3])
    _lib.check(_on_device(dev, lambda: lib.svdmlp_rope_append(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), slots.data_ptr(),
        out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), ctypes.addressof(st), T, pages, page, Hq, Hk, D, rot, scale,
        _ACT_CODES[q.dtype], _lib.SVDMLP_ROPE_INTERLEAVED if interleaved else 0, _stream(dev))))
    return out


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def _attention_scale(scale, D: int) -> float:
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _head_size(D: int, dtype: torch.dtype) -> None:
    step = 16 // torch.empty(0, dtype=dtype).element_size()
    if D > 256 or D % step:
        raise ValueError(f"head sizes are multiples of {step} up to 256 for {dtype}, got {D}")


def prompt_attention(q, k, v, cu_seqlens=None, *, causal: bool = True, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of packed sequences, each onto itself: q (T, Hq, D),
    k, v (T, Hk, D); sequence b is rows cu_seqlens[b] to cu_seqlens[b + 1] (int32
    on the device; None: one sequence).  ``causal``: a token sees the keys up to its
    own, else its whole sequence.  ``scale`` defaults to 1/sqrt(D).  Query head
    h reads key/value head h // (Hq // Hk).  Head sizes are multiples of 8 (bf16)
    or 4 (fp32) up to 256.  Rows behind the last sequence are not written."""
    T, Hq, Hk, D = _heads(q, k, v)
    _same_dtype(q, k, v)
    dev = _check("prompt_attention", q.dtype, q, k, v)
    _head_size(D, q.dtype)
    scale = _attention_scale(scale, D)
    B = 1
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2:
            raise ValueError("cu_seqlens must hold the first row of each sequence and the end of the last")
        B = int(cu_seqlens.shape[0]) - 1
        cu_seqlens = _index("cu_seqlens", cu_seqlens, (B + 1,), torch.int32, dev)
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=dev)
    else:
        _writable("out", out, (T, Hq, D), q)
        _aligned("out", out)
        _apart("out", out, q, k, v)
    if T == 0:
        return out
    q, k, v = _rows(q), _rows(k), _rows(v)
    lib = _lib.load()
    st = _strides(q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), out.stride(0), out.stride(1))
    _lib.check(_on_device(dev, lambda: lib.svdmlp_prompt_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), None if cu_seqlens is None else cu_seqlens.data_ptr(), out.data_ptr(),
        ctypes.addressof(st), T, B, Hq, Hk, D, scale, _ACT_CODES[q.dtype], _lib.SVDMLP_CAUSAL if causal else 0,
        _stream(dev))))
    return out


def cache_attention(q, k_cache, v_cache, block_table, lengths, *, tree=None, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the n new tokens of each sequence (q (B, n, Hq, D), n from 1
    to 64) onto its part of a paged cache (pages, page size, Hk, D), in which
    they are the last n of ``lengths[b]`` tokens: key x of sequence b is row
    ``x % page size`` of page ``block_table[b, x // page size]``.  A new token sees
    the context before them and, of the new ones, those that its row of ``tree``
    ((n, n) or (B, n, n) bool) names; without a tree, those up to itself.  n = 1 is
    the decode step.  A token without keys (length 0, or an empty row of a tree
    without context) gets zeros.  Pages outside the cache hold no keys."""
    if q.dim() != 4:
        raise ValueError(f"expected q (sequences, new tokens, heads, head size), got {tuple(q.shape)}")
    B, n, Hq, D = q.shape
    if k_cache.dim() != 4:
        raise ValueError(f"caches must have shape (pages, page size, kv heads, {D}), got {tuple(k_cache.shape)}")
    Hk = int(k_cache.shape[2])
    pages, page = _cache(k_cache, v_cache, q, Hk, D)
    if min(Hq, Hk, D) <= 0 or Hq % Hk:
        raise ValueError(f"{Hq} query heads are no multiple of {Hk} key/value heads")
    if not 1 <= n <= 64:
        raise ValueError(f"1 to 64 new tokens a sequence, got {n}")
    _same_dtype(q, k_cache, v_cache)
    dev = _check("cache_attention", q.dtype, q, k_cache, v_cache)
    _head_size(D, q.dtype)
    scale = _attention_scale(scale, D)
    if block_table.dim() != 2 or block_table.shape[1] == 0:
        raise ValueError("block_table must have shape (sequences, pages of the longest)")
    width = int(block_table.shape[1])
    if block_table.stride(1) != 1 or block_table.dtype != torch.int32:
        block_table = _index("block_table", block_table, (B, width), torch.int32, dev)
    elif block_table.shape[0] != B or block_table.device != dev:
        raise ValueError(f"block_table must have shape ({B}, pages of the longest) on {dev}")
    lengths = _index("lengths", lengths, (B,), torch.int32, dev)
    tree_ptr = tree_b = tree_q = 0
    if tree is not None:
        if tree.dtype not in (torch.bool, torch.uint8) or tuple(tree.shape) not in ((n, n), (B, n, n)):
            raise ValueError(f"tree must be a bool tensor ({n}, {n}) or ({B}, {n}, {n}), got {tree.dtype} {tuple(tree.shape)}")
        if tree.device != dev:
            raise ValueError("all inputs must be on the same device")
        if n > 1 and tree.stride(-1) != 1:
            tree = tree.contiguous()
        tree_ptr, tree_b, tree_q = tree.data_ptr(), tree.stride(0) if tree.dim() == 3 else 0, tree.stride(-2)
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.stride(-1) != 1:
            raise ValueError(f"the last dimension of {name} must be contiguous")
        _aligned(name, c)
    if out is None:
        out = torch.empty((B, n, Hq, D), dtype=q.dtype, device=dev)
    else:
        _writable("out", out, (B, n, Hq, D), q)
        _aligned("out", out)
        _apart("out", out, q, k_cache, v_cache)
    if B == 0:
        return out
    q = _rows(q)
    lib = _lib.load()
    st = _strides(*q.stride()[:3], *k_cache.stride()[:3], *v_cache.stride()[:3], *out.stride()[:3], block_table.stride(0),
                  tree_b, tree_q)

    def call():
        # the partial sums of long contexts: of the call alone, from torch's
        # allocator (of a graph's own pool under capture)
        nbytes = int(lib.svdmlp_cache_attention_workspace_bytes(B, n, page, width, Hq, Hk, D, _ACT_CODES[q.dtype]))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        return lib.svdmlp_cache_attention(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), lengths.data_ptr(), tree_ptr or None,
            out.data_ptr(), ctypes.addressof(st), B, n, pages, page, width, Hq, Hk, D, scale, _ACT_CODES[q.dtype],
            None if ws is None else ws.data_ptr(), nbytes, _stream(dev))

    _lib.check(_on_device(dev, call))
    return out


# ---------------------------------------------------------------------------
# Residual sum and norms
# ---------------------------------------------------------------------------

def _gain(name, w, d, dev):
    if w is None:
        return None
    if w.dim() != 1 or w.shape[0] != d or w.device != dev or not w.is_floating_point():
        raise ValueError(f"{name} must be a ({d},) tensor on x.device")
    return w.to(torch.float32).contiguous()


def residual_norm(x, branch, weight, *, post_weight=None, gate=None, scale: float = 1.0, eps: float = 1e-5,
                  out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The sum after a block of a decoder layer and the norm before the next
    one, (r, n) in x.dtype:

        r = x + scale * gate * b,   b = branch, or RMSNorm(branch) * post_weight
        n = RMSNorm(r) * weight     (of r before its rounding)

    x, branch (T, d); gate (d,) or (T, d) of x.dtype, or None; weight and
    post_weight (d,) gains (any float dtype; used in fp32).  branch None: r is x
    itself (the norm before a model's first block); weight None: n is None (the
    sum after its last).  d up to 32768.  ``out``: (r, n) to write, either may be
    None; they may be x and branch themselves."""
    if x.dim() != 2 or min(x.shape) <= 0:
        raise ValueError(f"expected a nonempty 2D array, got {tuple(x.shape)}")
    T, d = x.shape
    if branch is None and (post_weight is not None or gate is not None or weight is None):
        raise ValueError("without a branch there is only a norm of x")
    tensors = [t for t in (branch, gate) if t is not None]
    _same_dtype(x, *tensors)
    dev = _check("residual_norm", x.dtype, x, *tensors, *(w for w in (weight, post_weight) if w is not None))
    if branch is not None and branch.shape != x.shape:
        raise ValueError(f"branch must have x's shape {tuple(x.shape)}, got {tuple(branch.shape)}")
    if gate is not None and tuple(gate.shape) not in ((d,), (T, d)):
        raise ValueError(f"gate must have shape ({d},) or ({T}, {d}), got {tuple(gate.shape)}")
    if d > 32768:
        raise ValueError(f"rows of {d} values, at most 32768")
    eps, scale = float(eps), float(scale)
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError(f"eps must be positive, got {eps}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    w, pw = _gain("weight", weight, d, dev), _gain("post_weight", post_weight, d, dev)
    x0 = x
    x = _last(x)
    branch = None if branch is None else _last(branch)
    gate = None if gate is None else _last(gate)
    r, n = (None, None) if out is None else out
    for name, t in (("out[0]", r), ("out[1]", n)):
        if t is not None:
            _writable(name, t, (T, d), x)
            inputs = [a for a in (x, branch, gate) if a is not None]
            _apart(name, t, *inputs, own=[a for a in inputs if a.dim() == 2])
    if r is not None and n is not None:
        _apart("out[0]", r, n)
    if branch is not None and r is None:
        r = torch.empty((T, d), dtype=x.dtype, device=dev)
    if w is not None and n is None:
        n = torch.empty((T, d), dtype=x.dtype, device=dev)
    elif w is None:
        n = None
    lib = _lib.load()
    st = _strides(x.stride(0), branch.stride(0) if branch is not None else 0,
                  gate.stride(0) if gate is not None and gate.dim() == 2 else 0,
                  r.stride(0) if r is not None else 0, n.stride(0) if n is not None else 0)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _lib.check(_on_device(dev, lambda: lib.svdmlp_residual_norm(
        x.data_ptr(), ptr(branch), ptr(pw), ptr(gate), ptr(w), ptr(r), ptr(n), ctypes.addressof(st), T, d, scale, eps,
        _ACT_CODES[x.dtype], _stream(dev))))
    return (x0 if r is None else r), n
