"""The operators around the MLP block of a decoder layer, on MI355X.

    rope(q, k, positions, inv_freq)                 rotary positions
    rope_append(q, k, v, ..., k_cache, v_cache, slots)   ... into a paged cache
    norm_rope, norm_rope_append                     both, of normalised heads
    prompt_attention(q, k, v, cu_seqlens)           attention over packed prompts
    cache_attention(q, k_cache, v_cache, table, lengths)  decode, drafted trees
    chunk_attention(q, k_cache, v_cache, table, lengths, cu_seqlens)   chunks of prompts, and decode among them
    residual_norm(x, branch, weight)                sum after a block, next norm

With the projections and :func:`svdmlp.svd_mlp` they make a decoder layer
(bench/e2e_block.py:205-278 has its prefill form without positions).  Tensors
are bfloat16 or float32 on a ROCm GPU; queries are (rows, Hq, D), keys and values
(rows, Hk, D) with Hk dividing Hq, caches (pages, page size, Hk, D).  Slices
of a fused projection are read in place (last dimension contiguous, 16-byte
aligned rows); others are copied first.  Work goes to the current stream.

The operators are for inference: tensors that ask for a gradient, or carry a
forward-mode tangent, are refused (wrap the call in ``torch.no_grad()``, or
detach them).
Every call goes to libsvdmlp.so; there is no CPU or PyTorch fallback.
"""

from __future__ import annotations

import ctypes
import math
import threading

import torch
from torch.autograd import forward_ad as _forward

from . import _lib
from .ops import _ACT_CODES, _PARTIALS_CACHE

# A call at decode shapes takes a few microseconds on the GPU, so the host's
# part is kept short: sizes, types and devices are compared in line (a tensor's
# attribute costs ~0.06 us), what only unusual arguments need (strides that
# overlap, shared memory) is looked at only for them, and the stream is asked
# for without an object around it (0.1 us, 2 us with).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_BF16 = torch.bfloat16


def _refuse_device(name: str, *tensors) -> None:
    """Raises for tensors that are not all on one GPU."""
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError(f"{name} runs on a ROCm GPU; got tensors on {t.device}" if t is tensors[0]
                             else "all inputs must be on the same device")
    raise ValueError("all inputs must be on the same device")


def _refuse_dtype(*dtypes) -> None:
    if any(d != dtypes[0] for d in dtypes):
        raise TypeError("all inputs must have the same dtype")
    raise TypeError("supported dtypes are bfloat16 and float32")


def _gradients() -> bool:
    """Whether a tensor may ask for a gradient here: in grad mode, or where forward-mode tangents live."""
    return torch.is_grad_enabled() or _forward._current_level >= 0


def _refuse_grad(name: str, *tensors) -> None:
    backward, forward = torch.is_grad_enabled(), _forward._current_level >= 0
    for t in tensors:
        if t is None:
            continue
        if backward and t.requires_grad:
            raise ValueError(f"{name} has no gradient: call it under torch.no_grad(), or on detached tensors")
        if forward and _forward.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} has no gradient: call it on tensors without forward-mode tangents")


def _launch(index: int, fn, *args) -> None:
    """fn(*args, stream) on device `index`, its status checked."""
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels can read it in place (last dimension
    contiguous, rows in whole 16-byte pieces), else a contiguous copy.  (The
    stride of a dimension of one element may be anything.)"""
    step = 8 if t.dtype is _BF16 else 4
    st = t.stride()
    if st[-1] == 1 and not t.data_ptr() % 16:
        for s, n in zip(st[:-1], t.shape):
            if s % step and n > 1:
                break
        else:
            return t
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _writable(name: str, t: torch.Tensor, shape, like: torch.Tensor) -> None:
    """An output: of the shape, type and device, its elements all apart."""
    if tuple(t.shape) != tuple(shape) or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be a {tuple(shape)} tensor of {like.dtype} on {like.device}")
    if t.is_contiguous():
        return
    reach = 0
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            raise ValueError(f"{name} must not overlap itself")
        reach += stride * (size - 1)
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _aligned(name: str, t: torch.Tensor) -> None:
    step = 8 if t.dtype is _BF16 else 4
    if t.data_ptr() % 16 or any(s % step for s, n in zip(t.stride()[:-1], t.shape) if n > 1):
        raise ValueError(f"rows of {name} must be 16-byte aligned")


def _extent(t: torch.Tensor, first: int = 0) -> int:
    """Bytes from the first element of dimensions `first` on to the end of their last."""
    return (sum(s * (n - 1) for s, n in zip(t.stride()[first:], t.shape[first:])) + 1) * t.element_size()


def _bytes(t: torch.Tensor) -> tuple[int, int]:
    """The addresses of a nonempty tensor's first byte and behind its last."""
    p, es = t.data_ptr(), t.element_size()
    if t.is_contiguous():
        return p, p + es * t.numel()
    return p, p + _extent(t)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two nonempty tensors may share memory (slices side by side in the rows of one buffer do not)."""
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + _extent(a) <= pb or pb + _extent(b) <= pa:
        return False
    if a.dim() == b.dim() and a.dtype == b.dtype and all(s == t or m == 1 or n == 1 for s, t, m, n in zip(a.stride(), b.stride(), a.shape, b.shape)):
        steps = [(s if m > 1 else t, m, n) for s, t, m, n in zip(a.stride(), b.stride(), a.shape, b.shape) if m > 1 or n > 1]
        steps.sort(reverse=True)
        if all(s > sum(t * (max(m, n) - 1) for t, m, n in steps[i + 1:]) for i, (s, _, _) in enumerate(steps)):
            d, rest = divmod(pb - pa, a.element_size())
            return bool(rest) or _meet(d, steps)
    pitch = a.stride(0) * a.element_size()
    wa, wb = _extent(a, 1), _extent(b, 1)
    if pitch == b.stride(0) * b.element_size() and max(wa, wb) <= pitch:
        d = (pb - pa) % pitch
        return d < wa or d + wb > pitch
    return True


def _meet(d: int, steps) -> bool:
    """Whether an element of a and one of b, `d` elements further on, are the same: d = sum of stride * (index in a - in b),
    each stride beyond what the smaller ones reach."""
    if not steps:
        return d == 0
    s, m, n = steps[0]
    return any(-n < i < m and _meet(d - i * s, steps[1:]) for i in (d // s, d // s + 1))


def _apart(name: str, out: torch.Tensor, *tensors, own=()) -> None:
    """out shares no memory with the tensors, and with those of `own` only as the very same elements."""
    if out.numel() == 0:
        return
    for t in tensors:
        if t.numel() and _overlap(out, t) and not any(t is o and out.data_ptr() == t.data_ptr() and out.stride() == t.stride()
                                                      for o in own):
            raise ValueError(f"{name} must not overlap the inputs")


def _index(name: str, t: torch.Tensor, shape, dtype, device) -> torch.Tensor:
    """An index tensor as the kernels take it: t itself, or a copy of the type and layout (what 32 bits
    do not hold stays beyond every table and row, or negative)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an int32 or int64 tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != device:
        raise ValueError("all inputs must be on the same device")
    if t.dtype is dtype and t.is_contiguous():
        return t
    if dtype is torch.int32 and t.dtype is torch.int64:
        t = t.clamp(-1, 2 ** 31 - 1)
    return t.to(dtype).contiguous()


def _refuse_heads(q, k, *more) -> None:
    for t in (q, k, *more):
        if t.dim() != 3:
            raise ValueError(f"expected (tokens, heads, head size), got {tuple(t.shape)}")
    T, Hq, D = q.shape
    Hk = k.shape[1]
    for t in (k, *more):
        if tuple(t.shape) != (T, Hk, D):
            raise ValueError(f"keys and values must have shape {(T, Hk, D)}, got {tuple(t.shape)}")
    raise ValueError(f"{Hq} query heads are no multiple of {Hk} key/value heads")


_Strides3 = ctypes.c_int64 * 3
_Strides5 = ctypes.c_int64 * 5
_Strides8 = ctypes.c_int64 * 8
_Strides11 = ctypes.c_int64 * 11
_Strides14 = ctypes.c_int64 * 14
_Strides15 = ctypes.c_int64 * 15
_address = ctypes.addressof


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


def _rope_args(name, q, k, v, positions, inv_freq, scale):
    """The checks that rope and rope_append share (v None: rope); (T, Hq, Hk, D, device index, rot, positions, inv_freq)."""
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or ks[0] != qs[0] or ks[2] != qs[2] or not ks[1] or not qs[2] or not qs[1] or qs[1] % ks[1] or (
            v is not None and v.shape != ks):
        _refuse_heads(q, k, *(() if v is None else (v,)))
    T, Hq, D = qs
    dtype, index = q.dtype, q.get_device()
    if k.dtype != dtype or dtype not in _ACT_CODES or (v is not None and v.dtype != dtype):
        _refuse_dtype(dtype, k.dtype, *(() if v is None else (v.dtype,)))
    if index < 0 or k.get_device() != index or (v is not None and v.get_device() != index):
        _refuse_device(name, q, k, v)
    if inv_freq.dim() != 1 or not inv_freq.is_floating_point() or inv_freq.get_device() != index:
        raise ValueError("inv_freq must be a 1-D floating point tensor on the inputs' device")
    if _gradients():
        _refuse_grad(name, q, k, v, inv_freq)
    rot = 2 * inv_freq.shape[0]
    if not 0 < rot <= D:
        raise ValueError(f"{rot} turned values (two a frequency) of a head of {D}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    positions = _index("positions", positions, (T,), torch.int64, index)
    if inv_freq.dtype is not torch.float64 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(torch.float64).contiguous()
    return T, Hq, ks[1], D, index, rot, positions, inv_freq


def rope(q, k, positions, inv_freq, *, interleaved: bool = False, scale: float = 1.0,
         out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, k) with the first ``2 * len(inv_freq)`` values of each head turned
    by the tokens' positions: pair p, by positions[t] * inv_freq[p] (in 64 bits),
    is (p, p + rot/2), or (2p, 2p + 1) when ``interleaved``; the rest of the
    head is copied.  ``scale`` multiplies cos and sin (see
    :func:`rope_frequencies`).  q (T, Hq, D), k (T, Hk, D), positions (T,).
    ``out``: the pair of tensors to write, which may be q and k themselves."""
    T, Hq, Hk, D, index, rot, positions, inv_freq = _rope_args("rope", q, k, None, positions, inv_freq, scale)
    if out is None:
        qo, ko = q.new_empty((T, Hq, D)), q.new_empty((T, Hk, D))
    else:
        qo, ko = out
        if _gradients():
            _refuse_grad("rope", qo, ko)
        _writable("out[0]", qo, (T, Hq, D), q)
        _writable("out[1]", ko, (T, Hk, D), q)
        _apart("out[0]", qo, q, k, ko, positions, inv_freq, own=(q,))
        _apart("out[1]", ko, k, q, positions, inv_freq, own=(k,))
    if T == 0:
        return qo, ko
    q, k = _last(q), _last(k)
    st = _Strides8(*q.stride()[:2], *k.stride()[:2], *qo.stride()[:2], *ko.stride()[:2])
    _launch(index, _lib.load().svdmlp_rope, q.data_ptr(), k.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(),
            qo.data_ptr(), ko.data_ptr(), _address(st), T, Hq, Hk, D, rot, scale, _ACT_CODES[q.dtype], 1 if interleaved else 0)
    return qo, ko


def _refuse_caches(k_cache, v_cache, Hk, D) -> None:
    for c in (k_cache, v_cache):
        if c.dim() != 4 or tuple(c.shape[2:]) != (Hk, D) or c.shape[:2] != k_cache.shape[:2] or min(c.shape[:2]) <= 0:
            raise ValueError(f"caches must have shape (pages, page size, {Hk}, {D}), got {tuple(c.shape)}")


def rope_append(q, k, v, positions, inv_freq, k_cache, v_cache, slots, *, interleaved: bool = False,
                scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`rope` on the way into a paged cache: returns the turned q, and
    writes the turned k and v (T, Hk, D) to row ``slots[t] % page size`` of page
    ``slots[t] // page size`` of the caches (pages, page size, Hk, D).  A token
    whose slot lies outside the cache (-1: padding) is not written.  The slots of
    one call have to differ from each other."""
    T, Hq, Hk, D, index, rot, positions, inv_freq = _rope_args("rope_append", q, k, v, positions, inv_freq, scale)
    cs = k_cache.shape
    if len(cs) != 4 or v_cache.shape != cs or cs[2] != Hk or cs[3] != D or not cs[0] or not cs[1]:
        _refuse_caches(k_cache, v_cache, Hk, D)
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        _refuse_dtype(q.dtype, k_cache.dtype, v_cache.dtype)
    if k_cache.get_device() != index or v_cache.get_device() != index:
        _refuse_device("rope_append", q, k_cache, v_cache)
    if _gradients():
        _refuse_grad("rope_append", k_cache, v_cache, out)
    if not k_cache.is_contiguous():
        _writable("k_cache", k_cache, cs, q)
    if not v_cache.is_contiguous():
        _writable("v_cache", v_cache, cs, q)
    slots = _index("slots", slots, (T,), torch.int64, index)
    if out is not None:
        _writable("out", out, (T, Hq, D), q)
        _apart("out", out, q, k, v, k_cache, v_cache, positions, inv_freq, slots, own=(q,))
    if T == 0:
        return q.new_empty((0, Hq, D)) if out is None else out
    q, k, v = _last(q), _last(k), _last(v)
    a, b, c, kc, vc = q.stride(), k.stride(), v.stride(), k_cache.stride(), v_cache.stride()
    qp, kp, vp, kcp, vcp = q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    # The caches apart from each other and the inputs: by their first and last
    # bytes, exactly where those meet.
    es, n0, n1, n2 = 2 if q.dtype is _BF16 else 4, cs[0] - 1, cs[1] - 1, Hk - 1
    kce, vce = kcp + es * (n0 * kc[0] + n1 * kc[1] + n2 * kc[2] + D), vcp + es * (n0 * vc[0] + n1 * vc[1] + n2 * vc[2] + D)
    low = min(qp, kp, vp)
    high = max(qp + es * (a[0] * (T - 1) + a[1] * (Hq - 1) + D), kp + es * (b[0] * (T - 1) + b[1] * n2 + D),
               vp + es * (c[0] * (T - 1) + c[1] * n2 + D))
    if (kcp < vce and vcp < kce) or (low < kce and kcp < high) or (low < vce and vcp < high):
        _apart("k_cache", k_cache, v_cache, q, k, v)
        _apart("v_cache", v_cache, q, k, v)
    pp, fp, sp = positions.data_ptr(), inv_freq.data_ptr(), slots.data_ptr()
    pe, fe, se = pp + 8 * T, fp + 4 * rot, sp + 8 * T
    if ((pp < kce and kcp < pe) or (sp < kce and kcp < se) or (fp < kce and kcp < fe) or (pp < vce and vcp < pe)
            or (sp < vce and vcp < se) or (fp < vce and vcp < fe)):
        _apart("k_cache", k_cache, positions, inv_freq, slots)
        _apart("v_cache", v_cache, positions, inv_freq, slots)
    if out is None:
        out = q.new_empty((T, Hq, D))
    o = out.stride()
    st = _Strides14(a[0], a[1], b[0], b[1], c[0], c[1], o[0], o[1], kc[0], kc[1], kc[2], vc[0], vc[1], vc[2])
    _launch(index, _lib.load().svdmlp_rope_append, qp, kp, vp, pp, fp, sp,
            out.data_ptr(), kcp, vcp, _address(st), T, cs[0], cs[1], Hq, Hk, D, rot, scale, _ACT_CODES[q.dtype],
            1 if interleaved else 0)
    return out


def _head_gains(name, w, heads, D, index):
    """(gains in fp32, whether each head has its own)."""
    if w.get_device() != index or not w.is_floating_point() or w.shape not in ((D,), (heads, D)):
        raise ValueError(f"{name} must be a ({D},) or ({heads}, {D}) tensor on q.device")
    return w if w.dtype is torch.float32 and w.is_contiguous() else w.to(torch.float32).contiguous(), w.dim() == 2


def _norm_rope_args(name, q, k, q_weight, k_weight, eps, interleaved, D, Hq, Hk, index):
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError(f"eps must be positive, got {eps}")
    qw, q_own = _head_gains("q_weight", q_weight, Hq, D, index)
    kw, k_own = _head_gains("k_weight", k_weight, Hk, D, index)
    if _gradients():
        _refuse_grad(name, q_weight, k_weight)
    flags = ((_lib.SVDMLP_ROPE_INTERLEAVED if interleaved else 0) | (_lib.SVDMLP_Q_HEAD_GAINS if q_own else 0)
             | (_lib.SVDMLP_K_HEAD_GAINS if k_own else 0))
    return qw, kw, flags


def norm_rope(q, k, positions, inv_freq, q_weight, k_weight, *, eps: float = 1e-5, interleaved: bool = False,
              scale: float = 1.0, out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`rope` of heads that are normalised first, in the same pass: each head
    x of q becomes ``q_weight * x / sqrt(mean(x^2) + eps)``, each of k the same
    with ``k_weight``, and is turned before it is rounded.  The gains are (D,) for
    all heads or (heads, D), of any float dtype (used in fp32)."""
    T, Hq, Hk, D, index, rot, positions, inv_freq = _rope_args("norm_rope", q, k, None, positions, inv_freq, scale)
    qw, kw, flags = _norm_rope_args("norm_rope", q, k, q_weight, k_weight, eps, interleaved, D, Hq, Hk, index)
    if out is None:
        qo, ko = q.new_empty((T, Hq, D)), q.new_empty((T, Hk, D))
    else:
        qo, ko = out
        if _gradients():
            _refuse_grad("norm_rope", qo, ko)
        _writable("out[0]", qo, (T, Hq, D), q)
        _writable("out[1]", ko, (T, Hk, D), q)
        _apart("out[0]", qo, q, k, ko, positions, inv_freq, qw, kw, own=(q,))
        _apart("out[1]", ko, k, q, positions, inv_freq, qw, kw, own=(k,))
    if T == 0:
        return qo, ko
    q, k = _last(q), _last(k)
    st = _Strides8(*q.stride()[:2], *k.stride()[:2], *qo.stride()[:2], *ko.stride()[:2])
    _launch(index, _lib.load().svdmlp_norm_rope, q.data_ptr(), k.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), qw.data_ptr(),
            kw.data_ptr(), qo.data_ptr(), ko.data_ptr(), _address(st), T, Hq, Hk, D, rot, scale, eps, _ACT_CODES[q.dtype], flags)
    return qo, ko


def norm_rope_append(q, k, v, positions, inv_freq, q_weight, k_weight, k_cache, v_cache, slots, *, eps: float = 1e-5,
                     interleaved: bool = False, scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`norm_rope` on the way into a paged cache, as :func:`rope_append`:
    returns the turned q, and writes the normalised and turned k, and v as it
    is, to their slots of the caches."""
    name = "norm_rope_append"
    T, Hq, Hk, D, index, rot, positions, inv_freq = _rope_args(name, q, k, v, positions, inv_freq, scale)
    qw, kw, flags = _norm_rope_args(name, q, k, q_weight, k_weight, eps, interleaved, D, Hq, Hk, index)
    cs = k_cache.shape
    if len(cs) != 4 or v_cache.shape != cs or cs[2] != Hk or cs[3] != D or not cs[0] or not cs[1]:
        _refuse_caches(k_cache, v_cache, Hk, D)
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        _refuse_dtype(q.dtype, k_cache.dtype, v_cache.dtype)
    if k_cache.get_device() != index or v_cache.get_device() != index:
        _refuse_device(name, q, k_cache, v_cache)
    if _gradients():
        _refuse_grad(name, k_cache, v_cache, out)
    if not k_cache.is_contiguous():
        _writable("k_cache", k_cache, cs, q)
    if not v_cache.is_contiguous():
        _writable("v_cache", v_cache, cs, q)
    slots = _index("slots", slots, (T,), torch.int64, index)
    if out is not None:
        _writable("out", out, (T, Hq, D), q)
        _apart("out", out, q, k, v, k_cache, v_cache, positions, inv_freq, slots, qw, kw, own=(q,))
    if T == 0:
        return q.new_empty((0, Hq, D)) if out is None else out
    q, k, v = _last(q), _last(k), _last(v)
    # The caches apart from each other and from what is read: by their first and
    # last bytes, exactly where those meet.
    a, b, c, kc, vc = q.stride(), k.stride(), v.stride(), k_cache.stride(), v_cache.stride()
    qp, kp, vp, kcp, vcp = q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    pp, fp, sp, qwp, kwp = positions.data_ptr(), inv_freq.data_ptr(), slots.data_ptr(), qw.data_ptr(), kw.data_ptr()
    es, n0, n1, n2 = 2 if q.dtype is _BF16 else 4, cs[0] - 1, cs[1] - 1, Hk - 1
    kce, vce = kcp + es * (n0 * kc[0] + n1 * kc[1] + n2 * kc[2] + D), vcp + es * (n0 * vc[0] + n1 * vc[1] + n2 * vc[2] + D)
    meet = kcp < vce and vcp < kce
    for p, e in ((min(qp, kp, vp), max(qp + es * (a[0] * (T - 1) + a[1] * (Hq - 1) + D), kp + es * (b[0] * (T - 1) + b[1] * n2 + D),
                                       vp + es * (c[0] * (T - 1) + c[1] * n2 + D))),
                 (pp, pp + 8 * T), (sp, sp + 8 * T), (fp, fp + 4 * rot), (qwp, qwp + 4 * D * Hq), (kwp, kwp + 4 * D * Hk)):
        if (p < kce and kcp < e) or (p < vce and vcp < e):
            meet = True
    if meet:
        _apart("k_cache", k_cache, v_cache, q, k, v, positions, inv_freq, slots, qw, kw)
        _apart("v_cache", v_cache, q, k, v, positions, inv_freq, slots, qw, kw)
    if out is None:
        out = q.new_empty((T, Hq, D))
    o = out.stride()
    st = _Strides14(a[0], a[1], b[0], b[1], c[0], c[1], o[0], o[1], kc[0], kc[1], kc[2], vc[0], vc[1], vc[2])
    _launch(index, _lib.load().svdmlp_norm_rope_append, qp, kp, vp, pp, fp, qwp, kwp, sp, out.data_ptr(), kcp, vcp,
            _address(st), T, cs[0], cs[1], Hq, Hk, D, rot, scale, eps, _ACT_CODES[q.dtype], flags)
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
    step = 8 if dtype is _BF16 else 4
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
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or ks[0] != qs[0] or ks[2] != qs[2] or not ks[1] or not qs[2] or not qs[1] or qs[1] % ks[1] or v.shape != ks:
        _refuse_heads(q, k, v)
    T, Hq, D = qs
    dtype, index = q.dtype, q.get_device()
    if k.dtype != dtype or v.dtype != dtype or dtype not in _ACT_CODES:
        _refuse_dtype(dtype, k.dtype, v.dtype)
    if index < 0 or k.get_device() != index or v.get_device() != index:
        _refuse_device("prompt_attention", q, k, v)
    if _gradients():
        _refuse_grad("prompt_attention", q, k, v, out)
    _head_size(D, dtype)
    scale = _attention_scale(scale, D)
    B, cu = 1, None
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2:
            raise ValueError("cu_seqlens must hold the first row of each sequence and the end of the last")
        B = cu_seqlens.shape[0] - 1
        cu_seqlens = _index("cu_seqlens", cu_seqlens, (B + 1,), torch.int32, index)
        cu = cu_seqlens.data_ptr()
    if out is None:
        out = q.new_empty((T, Hq, D))
    else:
        _writable("out", out, (T, Hq, D), q)
        _aligned("out", out)
        _apart("out", out, q, k, v, *(() if cu is None else (cu_seqlens,)))
    if T == 0:
        return out
    q, k, v = _rows(q), _rows(k), _rows(v)
    if T > 1 and (k.stride(0) > 1 << 23 or v.stride(0) > 1 << 23):  # farther apart than the kernels' offsets reach
        k, v = k.contiguous(), v.contiguous()
    st = _Strides8(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *out.stride()[:2])
    _launch(index, _lib.load().svdmlp_prompt_attention, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu, out.data_ptr(),
            _address(st), T, B, Hq, ks[1], D, scale, _ACT_CODES[dtype], 1 if causal else 0)
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
    qs, cs = q.shape, k_cache.shape
    if len(qs) != 4:
        raise ValueError(f"expected q (sequences, new tokens, heads, head size), got {tuple(qs)}")
    B, n, Hq, D = qs
    if len(cs) != 4 or v_cache.shape != cs or cs[3] != D or not cs[0] or not cs[1]:
        _refuse_caches(k_cache, v_cache, cs[2] if len(cs) == 4 else "kv heads", D)
    pages, page, Hk, _ = cs
    if not Hq or not Hk or not D or Hq % Hk:
        raise ValueError(f"{Hq} query heads are no multiple of {Hk} key/value heads")
    if not 1 <= n <= 64:
        raise ValueError(f"1 to 64 new tokens a sequence, got {n}")
    dtype, index = q.dtype, q.get_device()
    if k_cache.dtype != dtype or v_cache.dtype != dtype or dtype not in _ACT_CODES:
        _refuse_dtype(dtype, k_cache.dtype, v_cache.dtype)
    if index < 0 or k_cache.get_device() != index or v_cache.get_device() != index:
        _refuse_device("cache_attention", q, k_cache, v_cache)
    if _gradients():
        _refuse_grad("cache_attention", q, k_cache, v_cache, out)
    _head_size(D, dtype)
    scale = _attention_scale(scale, D)
    if block_table.dim() != 2 or block_table.shape[1] == 0:
        raise ValueError("block_table must have shape (sequences, pages of the longest)")
    width = block_table.shape[1]
    if block_table.stride(1) != 1 or block_table.dtype is not torch.int32:
        if block_table.dtype is torch.int64:
            block_table = block_table.masked_fill((block_table < 0) | (block_table >= min(pages, 1 << 31)), -1)
        block_table = _index("block_table", block_table, (B, width), torch.int32, index)
    elif block_table.shape[0] != B or block_table.get_device() != index:
        raise ValueError(f"block_table must have shape ({B}, pages of the longest) on {q.device}")
    lengths = _index("lengths", lengths, (B,), torch.int32, index)
    tree_ptr, tree_b, tree_q = None, 0, 0
    if tree is not None:
        if tree.dtype not in (torch.bool, torch.uint8) or tuple(tree.shape) not in ((n, n), (B, n, n)):
            raise ValueError(f"tree must be a bool tensor ({n}, {n}) or ({B}, {n}, {n}), got {tree.dtype} {tuple(tree.shape)}")
        if tree.get_device() != index:
            raise ValueError("all inputs must be on the same device")
        if n > 1 and tree.stride(-1) != 1:
            tree = tree.contiguous()
        tree_ptr, tree_b, tree_q = tree.data_ptr(), tree.stride(0) if tree.dim() == 3 else 0, tree.stride(-2)
    kst, vst, step = k_cache.stride(), v_cache.stride(), 8 if dtype is _BF16 else 4
    if (kst[3] != 1 or vst[3] != 1 or kst[0] % step or kst[1] % step or kst[2] % step or vst[0] % step or vst[1] % step
            or vst[2] % step or k_cache.data_ptr() % 16 or v_cache.data_ptr() % 16):
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            if c.stride(3) != 1:
                raise ValueError(f"the last dimension of {name} must be contiguous")
            _aligned(name, c)
    if out is None:
        out = q.new_empty((B, n, Hq, D))
    else:
        _writable("out", out, (B, n, Hq, D), q)
        _aligned("out", out)
        _apart("out", out, q, k_cache, v_cache, block_table, lengths, *(() if tree is None else (tree,)))
    if B == 0:
        return out
    q = _rows(q)
    lib = _lib.load()
    qst, ost = q.stride(), out.stride()
    st = _Strides15(qst[0], qst[1], qst[2], kst[0], kst[1], kst[2], vst[0], vst[1], vst[2], ost[0], ost[1], ost[2],
                    block_table.stride(0), tree_b, tree_q)
    code = _ACT_CODES[dtype]
    nbytes, counters = _sizes(lib, index, B, n, page, width, Hq, Hk, D, code)
    if nbytes:
        with _partials_lock:  # a call may be two launches: no other thread's between them
            held = _partials(index, nbytes, counters)
            _launch(index, lib.svdmlp_cache_attention, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
                    lengths.data_ptr(), tree_ptr, out.data_ptr(), _address(st), B, n, pages, page, width, Hq, Hk, D, scale, code,
                    held[0].data_ptr(), nbytes, held[1].data_ptr(), counters)
    else:
        _launch(index, lib.svdmlp_cache_attention, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
                lengths.data_ptr(), tree_ptr, out.data_ptr(), _address(st), B, n, pages, page, width, Hq, Hk, D, scale, code,
                None, 0, None, 0)
    return out


def chunk_attention(q, k_cache, v_cache, block_table, lengths, cu_seqlens, *, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed chunks of new tokens onto a paged cache: q (T, Hq, D), rows
    cu_seqlens[b] to cu_seqlens[b + 1] of it are the last of the ``lengths[b]``
    tokens that the cache (pages, page size, Hk, D) holds of sequence b, any number
    of them: one where it generates, a chunk of its prompt where that is being read.
    Each sees the keys of its sequence up to itself.  block_table and lengths as
    :func:`cache_attention`, cu_seqlens as :func:`prompt_attention`.  A token
    without keys (a sequence with more new tokens than its length) gets zeros; pages outside the cache hold
    no keys; rows behind the last sequence are not written.

    Sums and the softmax's statistics are held in 32 bits; of bfloat16, as in the other
    attentions, the weights are rounded to bfloat16 for their product with the values
    (2^-8 of each at most; results are off by 0.0024 rms, 0.0017 of it their own rounding).
    Where every sequence has the same 1 to 64 new tokens :func:`cache_attention` takes them
    too: faster for a few sequences (one of 4097 tokens that generates 13 us, here
    22), slower for many (96 of 4000: 322, here 300)."""
    qs, cs = q.shape, k_cache.shape
    if len(qs) != 3:
        raise ValueError(f"expected q (new tokens, heads, head size), got {tuple(qs)}")
    T, Hq, D = qs
    if len(cs) != 4 or v_cache.shape != cs or cs[3] != D or not cs[0] or not cs[1]:
        _refuse_caches(k_cache, v_cache, cs[2] if len(cs) == 4 else "kv heads", D)
    pages, page, Hk, _ = cs
    if not Hq or not Hk or not D or Hq % Hk:
        raise ValueError(f"{Hq} query heads are no multiple of {Hk} key/value heads")
    dtype, index = q.dtype, q.get_device()
    if k_cache.dtype != dtype or v_cache.dtype != dtype or dtype not in _ACT_CODES:
        _refuse_dtype(dtype, k_cache.dtype, v_cache.dtype)
    if index < 0 or k_cache.get_device() != index or v_cache.get_device() != index:
        _refuse_device("chunk_attention", q, k_cache, v_cache)
    if _gradients():
        _refuse_grad("chunk_attention", q, k_cache, v_cache, out)
    _head_size(D, dtype)
    scale = _attention_scale(scale, D)
    if block_table.dim() != 2 or block_table.shape[1] == 0:
        raise ValueError("block_table must have shape (sequences, pages of the longest)")
    B, width = block_table.shape
    if block_table.stride(1) != 1 or block_table.dtype is not torch.int32:
        if block_table.dtype is torch.int64:
            block_table = block_table.masked_fill((block_table < 0) | (block_table >= min(pages, 1 << 31)), -1)
        block_table = _index("block_table", block_table, (B, width), torch.int32, index)
    elif block_table.get_device() != index:
        raise ValueError("all inputs must be on the same device")
    lengths = _index("lengths", lengths, (B,), torch.int32, index)
    cu_seqlens = _index("cu_seqlens", cu_seqlens, (B + 1,), torch.int32, index)
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.stride(3) != 1:
            raise ValueError(f"the last dimension of {name} must be contiguous")
        _aligned(name, c)
    if out is None:
        out = q.new_empty((T, Hq, D))
    else:
        _writable("out", out, (T, Hq, D), q)
        _aligned("out", out)
        _apart("out", out, q, k_cache, v_cache, block_table, lengths, cu_seqlens)
    if T == 0 or B == 0:
        return out
    q = _rows(q)
    lib, code = _lib.load(), _ACT_CODES[dtype]
    qst, kst, vst, ost = q.stride(), k_cache.stride(), v_cache.stride(), out.stride()
    st = _Strides11(qst[0], qst[1], kst[0], kst[1], kst[2], vst[0], vst[1], vst[2], ost[0], ost[1], block_table.stride(0))

    def launch(room, nbytes):
        _launch(index, lib.svdmlp_chunk_attention, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
                lengths.data_ptr(), cu_seqlens.data_ptr(), out.data_ptr(), _address(st), T, B, pages, page, width, Hq, Hk, D, scale, code,
                room, nbytes)

    key = ("chunk", index, T, B, page, width, Hq, Hk, D, code)
    nbytes = _SIZES.get(key)
    if nbytes is None:
        if len(_SIZES) > 4096:
            _SIZES.clear()
        with torch.cuda.device(index):
            nbytes = _SIZES[key] = int(lib.svdmlp_chunk_attention_workspace_bytes(T, B, page, width, Hq, Hk, D, code))
    if nbytes:
        with _partials_lock:  # a call may be several launches: no other thread's between them
            launch(_partials(index, nbytes, 0)[0].data_ptr(), nbytes)
    else:
        launch(None, 0)
    return out


_SIZES: dict = {}
_partials_lock = threading.Lock()


def _sizes(lib, index, *sizes) -> tuple[int, int]:
    """Workspace bytes and counters of a call's sizes on device `index` (they depend on the sizes and its CUs alone)."""
    key = (index, *sizes)
    plan = _SIZES.get(key)
    if plan is None:
        counters = ctypes.c_int64(0)
        with torch.cuda.device(index):
            nbytes = int(lib.svdmlp_cache_attention_workspace_bytes(*sizes, ctypes.byref(counters)))
        if len(_SIZES) > 4096:
            _SIZES.clear()
        plan = _SIZES[key] = (nbytes, counters.value)
    return plan


def _capturing(index: int) -> bool:
    """Whether device `index`'s current stream is being captured (torch asks for the current device's)."""
    if torch.cuda.current_device() == index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


def _partials(index: int, nbytes: int, counters: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Room for partial sums and zeroed counters.  One pair a (device, stream),
    grown on demand and kept until :func:`svdmlp.clear_workspace_cache`: every
    call leaves the counters zero for the next on its stream.  A captured call
    gets its own from the graph's pool, its counters cleared by the graph."""
    device = f"cuda:{index}"
    if _capturing(index):
        return torch.empty(nbytes, dtype=torch.uint8, device=device), torch.zeros(counters, dtype=torch.int32, device=device)
    key = (index, _raw_stream(index))
    held = _PARTIALS_CACHE.get(key)
    if held is None or held[0].numel() < nbytes or held[1].numel() < counters:
        room, zeros = held or (None, None)  # each grown by itself
        if room is None or room.numel() < nbytes:
            room = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        if zeros is None or zeros.numel() < counters:
            zeros = torch.zeros(max(counters, 4096), dtype=torch.int32, device=device)
        held = _PARTIALS_CACHE[key] = (room, zeros)
    return held


# ---------------------------------------------------------------------------
# Residual sum and norms
# ---------------------------------------------------------------------------

def _gain(name, w, d, index):
    if w.dim() != 1 or w.shape[0] != d or w.get_device() != index or not w.is_floating_point():
        raise ValueError(f"{name} must be a ({d},) tensor on x.device")
    return w if w.dtype is torch.float32 and w.is_contiguous() else w.to(torch.float32).contiguous()


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
    shape, dtype = x.shape, x.dtype
    if len(shape) != 2 or not shape[0] or not shape[1]:
        raise ValueError(f"expected a nonempty 2D array, got {tuple(shape)}")
    T, d = shape
    if branch is None and (post_weight is not None or gate is not None or weight is None):
        raise ValueError("without a branch there is only a norm of x")
    if dtype not in _ACT_CODES or (branch is not None and branch.dtype != dtype) or (gate is not None and gate.dtype != dtype):
        _refuse_dtype(dtype, *(t.dtype for t in (branch, gate) if t is not None))
    index = x.get_device()
    if index < 0 or (branch is not None and branch.get_device() != index) or (gate is not None and gate.get_device() != index):
        _refuse_device("residual_norm", x, branch, gate)
    if _gradients():
        _refuse_grad("residual_norm", x, branch, gate, weight, post_weight, *(out or ()))
    if branch is not None and branch.shape != shape:
        raise ValueError(f"branch must have x's shape {tuple(shape)}, got {tuple(branch.shape)}")
    if gate is not None and tuple(gate.shape) not in ((d,), (T, d)):
        raise ValueError(f"gate must have shape ({d},) or ({T}, {d}), got {tuple(gate.shape)}")
    if d > 32768:
        raise ValueError(f"rows of {d} values, at most 32768")
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError(f"eps must be positive, got {eps}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    w = pw = wp = pwp = bp = gp = rp = n_p = None
    bs = gs = rs = ns = 0
    if weight is not None:
        w = _gain("weight", weight, d, index)
        wp = w.data_ptr()
    if post_weight is not None:
        pw = _gain("post_weight", post_weight, d, index)
        pwp = pw.data_ptr()
    x0, x = x, _last(x)
    if branch is not None:
        branch = _last(branch)
        bp, bs = branch.data_ptr(), branch.stride(0)
    if gate is not None:
        gate = _last(gate)
        gp, gs = gate.data_ptr(), gate.stride(0) if gate.dim() == 2 else 0
    r = n = None
    if out is not None:
        r, n = out
        inputs = [a for a in (x, branch, gate, w, pw) if a is not None]
        for name, t in (("out[0]", r), ("out[1]", n)):
            if t is not None:
                _writable(name, t, (T, d), x)
                _apart(name, t, *inputs, own=[a for a in inputs if a.dim() == 2])
        if r is not None and n is not None:
            _apart("out[0]", r, n)
    if branch is not None and r is None:
        r = x.new_empty((T, d))
    if w is None:
        n = None
    elif n is None:
        n = x.new_empty((T, d))
    if r is not None:
        rp, rs = r.data_ptr(), r.stride(0)
    if n is not None:
        n_p, ns = n.data_ptr(), n.stride(0)
    st = _Strides5(x.stride(0), bs, gs, rs, ns)
    _launch(index, _lib.load().svdmlp_residual_norm, x.data_ptr(), bp, pwp, gp, wp, rp, n_p, _address(st), T, d, scale, eps,
            _ACT_CODES[dtype])
    return (x0 if r is None else r), n
