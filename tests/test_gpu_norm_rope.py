"""Head norms with the rotary positions behind them, against the definition in 64 bits.

Tolerances are bounds, element by element.  u is half a step of the type (bf16
2^-8, fp32 2^-24): the result's rounding.  In 32 bits the sum of a head's squares
takes at most 128 additions in a row, so that its root is off by at most 64
2^-24, and the mean, root, quotient and the products with the gains by a few
2^-24 more: 2^-17 of each value in all.  The turn adds 2^-21 of |a| + |b| for the
cosines and its products.
"""

import math

import pytest
import torch

import svdmlp
from test_gpu_decoder import BF, F32, U, _close, _gen, _qkv, _randn

pytestmark = pytest.mark.gpu


def _ref(x, w, eps, pos, f, interleaved, scale):
    """(result, the size of what went into each value)."""
    x = x.double()
    y = x / (x.square().mean(dim=-1, keepdim=True) + eps).sqrt() * w.double()
    half = f.shape[0]
    ang = pos.double()[:, None] * f.double()
    c, s = (scale * ang.cos())[:, None], (scale * ang.sin())[:, None]
    ia, ib = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = y[..., ia], y[..., ib]
    out, mag = y.clone(), y.abs()
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * abs(scale)
    return out, mag


def _check(got, x, w, eps, pos, f, interleaved=False, scale=1.0):
    out, mag = _ref(x, w, eps, pos, f, interleaved, scale)
    _close(got, out, (U[x.dtype] * out.abs() + (2.0 ** -17 + 2.0 ** -21) * mag) * 1.01 + 1e-38)


def _gains(g, heads, D, own):
    return torch.rand((heads, D) if own else (D,), generator=g) + 0.5


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,K,D,rot,own", [
    (1, 1, 1, 2, 2, False), (3, 4, 2, 16, 16, True), (5, 3, 1, 20, 6, False), (17, 32, 8, 128, 128, False), (1030, 4, 2, 64, 32, True),
    (7, 7, 7, 80, 20, False), (4099, 3, 3, 10, 10, False), (4097, 6, 2, 128, 64, True), (2, 8, 1, 256, 64, False), (9, 64, 8, 128, 64, True),
    (3, 2, 1, 1024, 1024, False), (3, 2, 2, 512, 32, True), (2, 2, 1, 1000, 8, False), (4, 5, 5, 24, 24, False), (6, 12, 4, 96, 96, True),
    (3, 2, 1, 1023, 510, False)])
def test_norm_rope(gpu, dtype, interleaved, T, H, K, D, rot, own):
    g = _gen(T * 31 + D)
    (q, k, _), (qg, kg, _) = _qkv(g, T, H, K, D, dtype, gpu)
    qw, kw = _gains(g, H, D, own), _gains(g, K, D, own)
    pos = torch.randint(0, 200000, (T,), generator=g)
    f, _ = svdmlp.rope_frequencies(rot, 10000.0)
    args = (pos.to(gpu), f.to(gpu), qw.to(gpu), kw.to(gpu))
    oq, ok = svdmlp.norm_rope(qg, kg, *args, eps=1e-3, interleaved=interleaved, scale=1.25)
    _check(oq, q, qw, 1e-3, pos, f, interleaved, 1.25)
    _check(ok, k, kw, 1e-3, pos, f, interleaved, 1.25)
    # in place, with positions in 32 bits, the same bits
    svdmlp.norm_rope(qg, kg, pos.int().to(gpu), *args[1:], eps=1e-3, interleaved=interleaved, scale=1.25, out=(qg, kg))
    assert torch.equal(qg, oq) and torch.equal(kg, ok)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_rope_small_and_large_heads(gpu, dtype):
    """Heads of zeros give zeros, of one value its sign times sqrt(D), of values far over or under 1 what they are beside each other;
    infinities and NaN stay within their head."""
    g = _gen(7)
    T, H, D = 6, 4, 64
    q = _randn(g, T, H, D, dtype=dtype)
    q[0] = 0
    q[1, 0] = 0
    q[1, 0, 5] = -3
    q[2] = (q[2].float() * 1e12).to(dtype)
    q[3] = (q[3].float() * 1e-12).to(dtype)
    bad = q.clone()
    bad[4, 1, 3], bad[4, 2, 60], bad[5, 0, 0] = math.inf, math.nan, -math.inf
    w, pos = torch.ones(D), torch.arange(T)
    f, _ = svdmlp.rope_frequencies(D, 10000.0)
    got, also = svdmlp.norm_rope(bad.to(gpu), q[:, :1].contiguous().to(gpu), *(t.to(gpu) for t in (pos, f, w, w)), eps=1e-6)
    assert torch.isnan(got[4, 1]).any() and torch.isnan(got[4, 2]).all() and torch.isnan(got[5, 0]).any()
    keep = torch.ones(T, H, dtype=torch.bool)
    keep[4, 1] = keep[4, 2] = keep[5, 0] = False
    out, mag = _ref(q, w, 1e-6, pos, f, False, 1.0)
    _close(got.cpu()[keep], out[keep], (U[dtype] * out.abs() + 2.0 ** -16 * mag)[keep] * 1.01 + 1e-38)
    _check(also, q[:, :1], w, 1e-6, pos, f)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,K,D,rot,page,joint", [(1, 4, 2, 64, 64, 16, False), (9, 8, 8, 32, 16, 5, True), (40, 14, 2, 64, 64, 1, False),
                                                    (1100, 2, 1, 128, 128, 64, True), (6, 3, 3, 12, 4, 7, False), (4100, 2, 2, 16, 16, 16, False)])
def test_norm_rope_append(gpu, dtype, T, H, K, D, rot, page, joint):
    g = _gen(T + D)
    (q, k, v), (qg, kg, vg) = _qkv(g, T, H, K, D, dtype, gpu)
    pages = -(-3 * T // page) + 2
    if joint:  # keys and values of a page side by side in one buffer
        pool = _randn(g, pages, 2, page, K, D, dtype=dtype)
        pool_g = pool.to(gpu)
        kc, vc, kcg, vcg = pool[:, 0], pool[:, 1], pool_g[:, 0], pool_g[:, 1]
    else:
        kc, vc = _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
        kcg, vcg = kc.to(gpu), vc.to(gpu)
    v[0, 0, 0], vg[0, 0, 0] = math.nan, math.nan  # values are copied, whatever they are
    pos = torch.randint(0, 5000, (T,), generator=g)
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 5:  # padding, and slots outside the cache: not written
        slots[1], slots[3], slots[4] = -1, pages * page, 2 ** 62
    qw, kw = _gains(g, H, D, False), _gains(g, K, D, True)
    f, _ = svdmlp.rope_frequencies(rot, 10000.0)
    oq = svdmlp.norm_rope_append(qg, kg, vg, pos.to(gpu), f.to(gpu), qw.to(gpu), kw.to(gpu), kcg, vcg, slots.to(gpu))
    _check(oq, q, qw, 1e-5, pos, f)
    keep = (slots >= 0) & (slots < pages * page)
    at = slots[keep]
    pg, row = at // page, at % page
    _check(kcg[pg.to(gpu), row.to(gpu)], k[keep], kw, 1e-5, pos[keep], f)
    assert torch.equal(vcg[pg.to(gpu), row.to(gpu)].cpu().nan_to_num(9.0), v[keep].nan_to_num(9.0))
    other = torch.ones(pages, page, dtype=torch.bool)
    other[pg, row] = False
    assert torch.equal(kcg.cpu()[other], kc[other]) and torch.equal(vcg.cpu()[other], vc[other])
    # the same keys as without a cache
    _, ok = svdmlp.norm_rope(qg, kg, pos.to(gpu), f.to(gpu), qw.to(gpu), kw.to(gpu))
    assert torch.equal(kcg[pg.to(gpu), row.to(gpu)], ok[keep.to(gpu)])


def test_norm_rope_gains_and_strides(gpu):
    """Gains of another type, unaligned or strided; heads outside tokens; outputs with strides of their own."""
    g = _gen(9)
    T, H, K, D = 11, 4, 2, 64
    q, k = _randn(g, H, T, D).transpose(0, 1), _randn(g, T, 1, D).expand(T, K, D)
    pos = torch.arange(T)
    f, _ = svdmlp.rope_frequencies(D, 10000.0)
    qw, kw = (torch.rand(H, D, generator=g) + 0.5).to(BF), torch.rand(D + 1, generator=g) + 0.5
    o = torch.empty(H, T, D, dtype=BF, device=gpu).transpose(0, 1)
    kg = k[:, :1].contiguous().to(gpu).expand(T, K, D)
    oq, ok = svdmlp.norm_rope(q.transpose(0, 1).contiguous().to(gpu).transpose(0, 1), kg, pos.to(gpu), f.to(gpu), qw.to(gpu),
                              kw.to(gpu)[1:], out=(o, torch.empty(T, K, D, dtype=BF, device=gpu)))
    assert oq is o
    _check(oq, q, qw, 1e-5, pos, f)
    _check(ok, k, kw[1:], 1e-5, pos, f)
    none = svdmlp.norm_rope(kg[:0], kg[:0], pos[:0].to(gpu), f.to(gpu), kw.to(gpu)[1:], kw.to(gpu)[1:])
    assert none[0].shape == (0, K, D)


def test_norm_rope_refusals(gpu):
    q, k = torch.zeros(4, 2, 8, device=gpu), torch.zeros(4, 1, 8, device=gpu)
    pos, f, w = torch.arange(4, device=gpu), torch.ones(4, dtype=torch.float64, device=gpu), torch.ones(8, device=gpu)
    c = torch.zeros(2, 4, 1, 8, device=gpu)
    cases = [
        (lambda: svdmlp.norm_rope(q, k, pos, f, w[:4], w), "q_weight"),
        (lambda: svdmlp.norm_rope(q, k, pos, f, w, w.expand(2, 8)), "k_weight"),
        (lambda: svdmlp.norm_rope(q, k, pos, f, w.cpu(), w), "q_weight"),
        (lambda: svdmlp.norm_rope(q, k, pos, f, w.long(), w), "q_weight"),
        (lambda: svdmlp.norm_rope(q, k, pos, f, w, w, eps=0.0), "eps"),
        (lambda: svdmlp.norm_rope(q, k, pos, f, w, w, eps=math.nan), "eps"),
        (lambda: svdmlp.norm_rope(q, k, pos, f, w, w, scale=math.inf), "scale"),
        (lambda: svdmlp.norm_rope(q, k, pos[:3], f, w, w), "positions"),
        (lambda: svdmlp.norm_rope(q, k, pos, torch.ones(5, device=gpu), w, w), "turned values"),
        (lambda: svdmlp.norm_rope(q, k, pos, f, w, w, out=(q.flip(0), q[:, :1])), "overlap"),
        (lambda: svdmlp.norm_rope(q, k, pos, f, q[0, 0], w, out=(q, k)), "overlap"),
        (lambda: svdmlp.norm_rope(q.clone().requires_grad_(), k, pos, f, w, w), "no gradient"),
        (lambda: svdmlp.norm_rope(q, k, pos, f, w.clone().requires_grad_(), w), "no gradient"),
        (lambda: svdmlp.norm_rope_append(q, k, k, pos, f, w, w, c, c, pos), "overlap"),
        (lambda: svdmlp.norm_rope_append(q, k, k, pos, f, c[0, 0, 0], w, c, c.clone(), pos), "overlap"),
        (lambda: svdmlp.norm_rope_append(q, k, k, pos, f, w, w, c, c[:1].clone(), pos), "caches must have shape"),
        (lambda: svdmlp.norm_rope_append(q, k, k, pos, f, w, w, c, c[:1].clone().expand(2, 4, 1, 8), pos), "overlap"),
        (lambda: svdmlp.norm_rope_append(q, k, k, pos, f, w, w, c, c.clone(), pos[:2]), "slots"),
    ]
    for fn, msg in cases:
        with pytest.raises(ValueError, match=msg):
            fn()
    with torch.no_grad():
        svdmlp.norm_rope(q.clone().requires_grad_(), k, pos, f, w, w)
