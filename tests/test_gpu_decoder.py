"""The operators around the MLP block against their definitions in 64 bits.

Tolerances are bounds, element by element.  u is half a step of the type
(bf16 2^-8, fp32 2^-24).  Attention: with A the weighted mean of |v|, rounding
the weights to bf16 moves the result by at most u A, rounding the result by u
|out|; in 32 bits a score of D products is off by (D + 16) 2^-24 of the sum of
their magnitudes (E at most, scaled), exp2 and its argument by 2^-21 more, twice
(numerator and sum), and the sums over n keys by (n + 64) 2^-23.  Rotary: the
result's rounding, and the cosines' and products' in 32 bits, 2^-21 of |a| + |b|.
Norms: sums of squares of 32768 values in 32 bits, in a tree of at most 96
steps: 2^-17 covers them, the root and the products.
"""

import math

import pytest
import torch

import svdmlp
from svdmlp import decoder

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
U = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=BF):
    return torch.randn(shape, generator=g).to(dtype)


def _attend(q, k, v, seen, scale, dtype):
    """(out, tolerance) in 64 bits of one head's q (n, D) on k, v (m, D); seen (n, m)."""
    q, k, v = q.double(), k.double(), v.double()
    s = scale * (q @ k.t())
    s[~seen] = -math.inf
    m = s.amax(dim=1, keepdim=True) if s.shape[1] else torch.full((s.shape[0], 1), -math.inf, dtype=torch.float64)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(dim=1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    vz = torch.nan_to_num(v, 0.0, 0.0, 0.0)  # masked keys have no part, whatever they hold
    out = p @ vz
    A = p @ vz.abs()
    E = (scale * (torch.nan_to_num(q, 0.0, 0.0, 0.0).abs() @ torch.nan_to_num(k, 0.0, 0.0, 0.0).abs().t()))
    E = torch.where(seen, E, 0.0).amax(dim=1, keepdim=True) if s.shape[1] else torch.zeros((s.shape[0], 1))
    off = 2 * ((q.shape[1] + 16) * 2.0 ** -24 * E + 2.0 ** -21) + (k.shape[0] + 64) * 2.0 ** -23
    u = U[dtype]
    tol = A * (off + (u if dtype == BF else 0.0)) * 1.01 + u * out.abs() * 1.01 + 1e-38
    return out, tol


def _prompt_ref(q, k, v, lens, causal, scale, first=0):
    T, H, D = q.shape
    out, tol = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    G = H // k.shape[1]
    at = first
    for n in lens:
        seen = torch.ones(n, n, dtype=torch.bool)
        if causal:
            seen = seen.tril()
        for h in range(H):
            r = slice(at, at + n)
            out[r, h], tol[r, h] = _attend(q[r, h], k[r, h // G], v[r, h // G], seen, scale, q.dtype)
        at += n
    return out, tol


def _close(got, out, tol):
    got = got.double().cpu()
    assert not torch.isnan(got).any()
    excess = ((got - out).abs() / tol).max()
    assert excess <= 1, f"off by {excess:.3g} times the bound"


def _cu(lens, dev, first=0):
    return torch.tensor([first] + [first + sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32, device=dev)


def _qkv(g, T, H, K, D, dtype, dev, fused=True):
    """q, k, v as slices of one buffer (what a fused projection writes), on the CPU and the GPU."""
    flat = _randn(g, T, (H + 2 * K) * D, dtype=dtype)

    def cut(f):
        return f[:, :H * D].view(T, H, D), f[:, H * D:(H + K) * D].view(T, K, D), f[:, (H + K) * D:].view(T, K, D)

    gpu = cut(flat.to(dev))
    return cut(flat), gpu if fused else tuple(t.contiguous() for t in gpu)


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------

def _rope_ref(x, pos, inv_freq, interleaved, scale):
    x = x.double()
    half = inv_freq.shape[0]
    ang = pos.double()[:, None] * inv_freq.double()
    c, s = (scale * ang.cos())[:, None], (scale * ang.sin())[:, None]
    ia, ib = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., ia], x[..., ib]
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * abs(scale)
    return y, mag


def _rope_close(got, x, pos, inv_freq, interleaved, scale):
    y, mag = _rope_ref(x, pos, inv_freq, interleaved, scale)
    tol = (U[x.dtype] * y.abs() + 2.0 ** -21 * mag) * 1.01 + 1e-38
    rot = 2 * inv_freq.shape[0]
    _close(got[..., :rot], y[..., :rot], tol[..., :rot])
    assert torch.equal(got[..., rot:].cpu(), x[..., rot:])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,K,D,rot", [
    (1, 1, 1, 2, 2), (3, 4, 2, 16, 16), (5, 3, 1, 20, 6), (17, 32, 8, 128, 128), (1030, 4, 2, 64, 32), (7, 7, 7, 80, 20),
    (1027, 3, 3, 10, 10), (2, 8, 1, 256, 64), (9, 64, 8, 128, 64)])
def test_rope(gpu, dtype, interleaved, T, H, K, D, rot):
    g = _gen(T * 31 + D)
    (q, k, _), (qg, kg, _) = _qkv(g, T, H, K, D, dtype, gpu)
    pos = torch.randint(0, 200000, (T,), generator=g)
    f, _ = svdmlp.rope_frequencies(rot, 10000.0)
    oq, ok = svdmlp.rope(qg, kg, pos.to(gpu), f.to(gpu), interleaved=interleaved, scale=1.25)
    _rope_close(oq, q, pos, f, interleaved, 1.25)
    _rope_close(ok, k, pos, f, interleaved, 1.25)
    # in place, with positions in 32 bits, the same bits
    svdmlp.rope(qg, kg, pos.int().to(gpu), f.to(gpu), interleaved=interleaved, scale=1.25, out=(qg, kg))
    assert torch.equal(qg, oq) and torch.equal(kg, ok)


def test_rope_far_positions(gpu):
    """Angles of positions near 2^31 keep their fractions (a product in 32 bits is off by whole turns)."""
    g = _gen(5)
    q, k = _randn(g, 6, 2, 64, dtype=F32), _randn(g, 6, 1, 64, dtype=F32)
    pos = torch.tensor([0, 1, 131071, 2 ** 24 + 1, 2 ** 31 - 1, -17])
    f, _ = svdmlp.rope_frequencies(64, 500000.0)
    oq, ok = svdmlp.rope(q.to(gpu), k.to(gpu), pos.to(gpu), f.to(gpu))
    _rope_close(oq, q, pos, f, False, 1.0)
    _rope_close(ok, k, pos, f, False, 1.0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,K,D,rot,page,joint", [(1, 4, 2, 64, 64, 16, False), (9, 8, 8, 32, 16, 5, True), (40, 14, 2, 64, 64, 1, False),
                                                    (1100, 2, 1, 128, 128, 64, True), (6, 3, 3, 12, 4, 7, False)])
def test_rope_append(gpu, dtype, T, H, K, D, rot, page, joint):
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
    pos = torch.randint(0, 5000, (T,), generator=g)
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 5:  # padding, and slots outside the cache: not written
        slots[1], slots[3], slots[4] = -1, pages * page, 2 ** 62
    f, _ = svdmlp.rope_frequencies(rot, 10000.0)
    oq = svdmlp.rope_append(qg, kg, vg, pos.to(gpu), f.to(gpu), kcg, vcg, slots.to(gpu))
    _rope_close(oq, q, pos, f, False, 1.0)
    keep = (slots >= 0) & (slots < pages * page)
    at = slots[keep]
    pg, row = at // page, at % page
    _rope_close(kcg[pg.to(gpu), row.to(gpu)], k[keep], pos[keep], f, False, 1.0)
    assert torch.equal(vcg[pg.to(gpu), row.to(gpu)].cpu(), v[keep])
    other = torch.ones(pages, page, dtype=torch.bool)
    other[pg, row] = False
    assert torch.equal(kcg.cpu()[other], kc[other]) and torch.equal(vcg.cpu()[other], vc[other])


def test_rope_refusals(gpu):
    q, k = torch.zeros(4, 2, 8, device=gpu), torch.zeros(4, 1, 8, device=gpu)
    pos, f = torch.arange(4, device=gpu), torch.ones(4, dtype=torch.float64, device=gpu)
    with pytest.raises(ValueError, match="no gradient"):
        svdmlp.rope(q.clone().requires_grad_(), k, pos, f)
    with torch.no_grad():
        svdmlp.rope(q.clone().requires_grad_(), k, pos, f)
    with pytest.raises(ValueError, match="overlap"):
        svdmlp.rope(q, k, pos, f, out=(q.flip(0), q[:, :1]))
    with pytest.raises(ValueError, match="overlap"):
        svdmlp.rope(q, k, pos, f, out=(q[:1].expand(4, 2, 8), k))
    with pytest.raises(ValueError, match="turned values"):
        svdmlp.rope(q, k, pos, torch.ones(5, device=gpu))
    with pytest.raises(TypeError, match="positions"):
        svdmlp.rope(q, k, pos.float(), f)
    with pytest.raises(ValueError, match="positions"):
        svdmlp.rope(q, k, pos[:3], f)
    with pytest.raises(ValueError, match="same device"):
        svdmlp.rope(q, k.cpu(), pos, f)
    with pytest.raises(ValueError, match="overlap"):
        c = torch.zeros(1, 1, 1, 8, device=gpu).expand(2, 4, 1, 8)
        svdmlp.rope_append(q, k, k, pos, f, c, c, pos)
    e = svdmlp.rope(q[:0], k[:0], pos[:0], f)
    assert e[0].shape == (0, 2, 8) and e[1].shape == (0, 1, 8)


# ---------------------------------------------------------------------------
# Attention over prompts
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,H,K,D", [
    ([1], 1, 1, 8), ([1, 1, 1], 4, 2, 64), ([31, 0, 33], 8, 2, 128), ([64], 4, 4, 64), ([65, 1, 200], 12, 4, 96), ([127], 7, 7, 80),
    ([300], 32, 8, 128), ([129, 128], 8, 1, 256), ([0, 0, 5], 6, 3, 40), ([513], 5, 1, 128), ([70] * 9, 14, 2, 64), ([2, 257], 3, 1, 200),
    ([1025], 2, 1, 128), ([700, 333], 2, 2, 64)])
def test_prompt_attention(gpu, dtype, causal, lens, H, K, D):
    T = sum(lens)
    g = _gen(T * 7 + D)
    (q, k, v), (qg, kg, vg) = _qkv(g, T, H, K, D, dtype, gpu, fused=T % 2 == 1)
    scale = 1 / math.sqrt(D)
    out, tol = _prompt_ref(q, k, v, lens, causal, scale)
    cu = _cu(lens, gpu)
    got = svdmlp.prompt_attention(qg, kg, vg, cu, causal=causal)
    _close(got, out, tol)
    assert torch.equal(got, svdmlp.prompt_attention(qg, kg, vg, cu.long(), causal=causal))
    if len(lens) == 1:
        assert torch.equal(got, svdmlp.prompt_attention(qg, kg, vg, causal=causal))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,H,K,D", [([2100], 32, 8, 128), ([1500, 1, 0, 640], 64, 8, 64), ([1030, 63, 65, 1027], 32, 4, 96), ([4097], 16, 16, 64),
                                        ([900, 1300], 32, 1, 80), ([2113], 40, 8, 128), ([1, 0, 129, 31, 33, 300, 77, 128, 400, 201], 32, 8, 128),
                                        ([33, 250, 64, 2, 391, 460, 7, 193], 32, 4, 96), ([311], 128, 32, 128), ([160, 97], 160, 80, 72)])
def test_prompt_attention_many_rows(gpu, lens, H, K, D, causal):
    g = _gen(sum(lens) + H)
    (q, k, v), dev = _qkv(g, sum(lens), H, K, D, BF, gpu)
    got = svdmlp.prompt_attention(*dev, _cu(lens, gpu), causal=causal).cpu()
    heads = [0, H // 2 + 1, H - 1]
    kv = [h // (H // K) for h in heads]
    out, tol = _prompt_ref(q[:, heads], k[:, kv], v[:, kv], lens, causal, 1 / math.sqrt(D))
    _close(got[:, heads], out, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompt_attention_large_scores_and_scale(gpu, dtype):
    """Scores that grow along the keys by hundreds of powers of two (every tile moves the running maximum) and a scale of one's own."""
    g = _gen(3)
    for T, H, K, D in ((400, 4, 2, 64), (700, 96, 2, 128)):
        q, k, v = (_randn(g, T, n, D, dtype=dtype) for n in (H, K, K))
        q = q.abs()
        k = (k.abs() * torch.linspace(0.0, 4.0, T)[:, None, None]).to(dtype)
        heads = [0, H - 1]
        for causal, scale in ((True, 1.0), (False, 0.37)):
            got = svdmlp.prompt_attention(*(t.to(gpu) for t in (q, k, v)), causal=causal, scale=scale)
            out, tol = _prompt_ref(q[:, heads], k[:, [0, K - 1]], v[:, [0, K - 1]], [T], causal, scale)
            _close(got[:, heads], out, tol)


@pytest.mark.parametrize("H,K,D", [(4, 2, 64), (4, 2, 128), (4, 2, 256), (256, 1, 64), (256, 2, 128), (256, 32, 128)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompt_attention_hidden_keys_have_no_part(gpu, dtype, H, K, D):
    """Infinities and NaN in later tokens, other sequences and rows of no
    sequence; rows of no sequence stay as they were.  A value that a token does
    see reaches it."""
    g = _gen(11)
    lens, first = [150, 90], 3
    T = 260
    q, k, v = (_randn(g, T, n, D, dtype=dtype) for n in (H, K, K))
    out, tol = _prompt_ref(q, k, v, lens, True, 1 / math.sqrt(D), first)
    kb, vb = k.clone(), v.clone()
    for t in (kb, vb):
        t[:first], t[first + 240:] = math.nan, math.inf
        t[first + 149], t[first + 239, :, ::3] = math.nan, -math.inf  # the last token of each sequence
    vb[first + 100, 0, 5], vb[first + 101, 0, 5], vb[first + 102, 0, 6] = math.inf, -math.inf, math.nan
    kept = torch.full((T, H, D), 7.0, dtype=dtype, device=gpu)
    got = svdmlp.prompt_attention(*(t.to(gpu) for t in (q, kb, vb)), _cu(lens, gpu, first), out=kept).cpu()
    assert got.data_ptr() != 0 and (got[:first] == 7).all() and (got[first + 240:] == 7).all()
    clean = torch.ones(T, H, D, dtype=torch.bool)
    clean[:first] = clean[first + 240:] = clean[first + 149] = clean[first + 239] = False
    seen = slice(first + 100, first + 149)
    clean[seen, :H // K, 5:7] = False
    _close(torch.where(clean, got, 0), torch.where(clean, out, 0.0), torch.where(clean, tol, 1.0))
    assert torch.isnan(got[first + 149]).all()
    assert (got[first + 100, :H // K, 5] == math.inf).all()               # +inf alone
    assert torch.isnan(got[first + 101:first + 149, :H // K, 5]).all()    # and -inf with it
    assert torch.isnan(got[first + 102:first + 149, :H // K, 6]).all()


def test_prompt_attention_full_sees_every_value(gpu):
    """Without a causal mask an infinity reaches every token of its sequence, in its column alone."""
    g = _gen(12)
    for T, H in ((70, 2), (1030, 64)):
        q, k, v = (_randn(g, T, H, 64) for _ in range(3))
        v[T - 1, 0, 3], v[5, 1, 4] = math.inf, -math.inf
        got = svdmlp.prompt_attention(*(t.to(gpu) for t in (q, k, v)), causal=False).cpu()
        assert (got[:, 0, 3] == math.inf).all() and (got[:, 1, 4] == -math.inf).all()
        got[:, 0, 3] = got[:, 1, 4] = 0
        assert torch.isfinite(got.float()).all()


def test_prompt_attention_bounds_outside_the_rows(gpu):
    """Sequence bounds that leave the rows or run backwards are cut, not followed."""
    g = _gen(13)
    q, k, v = (_randn(g, 50, 2, 64) for _ in range(3))
    dev = [t.to(gpu) for t in (q, k, v)]
    want = svdmlp.prompt_attention(*dev, _cu([20, 30], gpu))
    cu = torch.tensor([-5, 20, 2 ** 30], dtype=torch.int32, device=gpu)
    assert torch.equal(svdmlp.prompt_attention(*dev, cu), want)
    cu = torch.tensor([0, 20, 10, 50], dtype=torch.int32, device=gpu)  # the second is empty, the third rows 10 to 50
    assert torch.isfinite(svdmlp.prompt_attention(*dev, cu).float()).all()


def test_prompt_attention_many_sequences(gpu):
    """More sequences than a wave looks at at once."""
    g = _gen(14)
    lens = [int(n) for n in torch.randint(0, 40, (200,), generator=g)]
    T = sum(lens)
    q, k, v = (_randn(g, T, n, 64) for n in (4, 2, 2))
    out, tol = _prompt_ref(q, k, v, lens, True, 0.125)
    _close(svdmlp.prompt_attention(*(t.to(gpu) for t in (q, k, v)), _cu(lens, gpu)), out, tol)


def test_prompt_attention_strides(gpu):
    """Heads outside tokens (each head's rows together), a value tensor of unaligned rows (copied), shared keys (stride 0)."""
    g = _gen(15)
    T, H, K, D = 90, 4, 2, 64
    q, k, v = _randn(g, H, T, D).transpose(0, 1), _randn(g, T, 1, D).expand(T, K, D), _randn(g, T, K, D + 1)[..., 1:]
    out, tol = _prompt_ref(q, k, v, [T], True, 0.125)
    qg = q.transpose(0, 1).contiguous().to(gpu).transpose(0, 1)
    kg = k[:, :1].contiguous().to(gpu).expand(T, K, D)
    vg = torch.zeros(T, K, D + 1, dtype=BF, device=gpu)[..., 1:]
    vg.copy_(v)
    o = torch.empty(H, T, D, dtype=BF, device=gpu).transpose(0, 1)
    assert svdmlp.prompt_attention(qg, kg, vg, out=o) is o
    _close(o, out, tol)


def test_prompt_attention_refusals(gpu):
    q, k = torch.zeros(4, 4, 64, dtype=BF, device=gpu), torch.zeros(4, 2, 64, dtype=BF, device=gpu)
    cases = [
        (lambda: svdmlp.prompt_attention(q[..., :12], k[..., :12], k[..., :12]), "head sizes"),
        (lambda: svdmlp.prompt_attention(q, k, k, scale=0.0), "scale"),
        (lambda: svdmlp.prompt_attention(q, k, k, torch.zeros(1, dtype=torch.int32, device=gpu)), "cu_seqlens"),
        (lambda: svdmlp.prompt_attention(q, k, k, torch.zeros(2, dtype=torch.int32)), "same device"),
        (lambda: svdmlp.prompt_attention(q, k, k, out=q), "overlap"),
        (lambda: svdmlp.prompt_attention(q, k, k, out=torch.empty(4, 4, 65, dtype=BF, device=gpu)[..., 1:]), "16-byte"),
        (lambda: svdmlp.prompt_attention(q, k, k, out=torch.empty(4, 4, 64, device=gpu)), "out must be"),
        (lambda: svdmlp.prompt_attention(q.clone().requires_grad_(), k, k), "no gradient"),
    ]
    for fn, msg in cases:
        with pytest.raises(ValueError, match=msg):
            fn()
    assert svdmlp.prompt_attention(q[:0], k[:0], k[:0]).shape == (0, 4, 64)


# ---------------------------------------------------------------------------
# Attention over a paged cache
# ---------------------------------------------------------------------------

def _pages(g, lens, page, spare=3):
    counts = [-(-n // page) for n in lens]
    order = torch.randperm(sum(counts) + spare, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    return table, len(order)


def _cache_ref(q, kc, vc, table, lens, tree, scale):
    B, n, H, D = q.shape
    K, page = kc.shape[2], kc.shape[1]
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.ones(q.shape, dtype=torch.float64) * 1e-30
    for b, length in enumerate(lens):
        keys = torch.arange(length)
        at = table[b].long()[keys // page] * page + keys % page
        k, v = kc.flatten(0, 1)[at], vc.flatten(0, 1)[at]
        draft = keys - (length - n)
        if tree is None:
            seen = draft[None] <= torch.arange(n)[:, None]
        else:
            t = tree if tree.dim() == 2 else tree[b]
            seen = (draft < 0)[None] | t[:, draft.clamp(0, n - 1)]
        for h in range(H):
            out[b, :, h], tol[b, :, h] = _attend(q[b, :, h], k[:, h // (H // K)], v[:, h // (H // K)], seen, scale, q.dtype)
    return out, tol


def _random_tree(g, B, n):
    tree = torch.zeros(B, n, n, dtype=torch.bool)
    for b in range(B):
        for i in range(n):
            if i:
                tree[b, i] = tree[b, int(torch.randint(0, i, (1,), generator=g))]
            tree[b, i, i] = True
    return tree


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,n,H,K,D,page,tree", [
    ([1], 1, 1, 1, 8, 1, None), ([5, 0, 1], 1, 4, 2, 64, 16, None), ([33, 64, 31], 1, 8, 8, 128, 16, None),
    ([1000, 17], 1, 32, 8, 128, 16, None), ([129, 40], 5, 8, 2, 128, 16, None), ([70, 64], 64, 14, 2, 64, 16, "own"),
    ([300, 16, 999], 16, 8, 1, 128, 64, "own"), ([40], 7, 12, 4, 96, 48, "shared"), ([2600], 1, 8, 1, 256, 32, None),
    ([3, 2, 9], 4, 6, 3, 40, 3, None), ([257, 511], 33, 3, 1, 80, 7, "own"), ([5000, 1], 1, 7, 7, 80, 16, None),
    ([4097], 2, 16, 2, 64, 256, "own"), ([700], 12, 5, 1, 200, 16, "shared")])
def test_cache_attention(gpu, dtype, lens, n, H, K, D, page, tree):
    g = _gen(sum(lens) + D + n)
    B = len(lens)
    table, pages = _pages(g, lens, page)
    q = _randn(g, B, n, H, D, dtype=dtype)
    kc, vc = _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    mask = None if tree is None else _random_tree(g, B, n)
    if tree == "shared":
        mask = mask[0]
    scale = 1 / math.sqrt(D)
    out, tol = _cache_ref(q, kc, vc, table, lens, mask, scale)
    # rows behind a sequence's end hold NaN: nobody reads them
    used = torch.zeros(pages * page, dtype=torch.bool)
    for b, length in enumerate(lens):
        keys = torch.arange(length)
        used[table[b].long()[keys // page] * page + keys % page] = True
    kc.view(-1, K, D)[~used] = math.nan
    vc.view(-1, K, D)[~used] = math.inf
    args = [t.to(gpu) for t in (q, kc, vc, table)]
    ln = torch.tensor(lens, device=gpu)
    got = svdmlp.cache_attention(*args, ln, tree=None if mask is None else mask.to(gpu))
    _close(got, out, tol)
    again = svdmlp.cache_attention(*args, ln.int(), tree=None if mask is None else mask.to(gpu).to(torch.uint8))
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype,B,n,H,K,D,page,most", [
    (BF, 40, 1, 8, 2, 64, 16, 4000), (BF, 70, 1, 16, 8, 128, 16, 1500), (BF, 24, 9, 32, 8, 128, 32, 2500), (BF, 33, 3, 8, 8, 256, 64, 900),
    (F32, 64, 1, 8, 4, 64, 16, 2100), (F32, 40, 4, 8, 8, 128, 3, 700), (BF, 90, 20, 8, 4, 64, 128, 1800), (F32, 9, 2, 8, 8, 256, 16, 3000),
    (BF, 1, 1, 8, 1, 128, 1, 60000), (BF, 2, 17, 8, 8, 96, 8, 20000)])
def test_cache_attention_many_keys(gpu, dtype, B, n, H, K, D, page, most):
    """Long caches and many sequences: chunks of every kind, joined by the last block; the counters end where they began."""
    g = _gen(B + most)
    lens = [most, 0, n - 1, n][:B] + [int(x) for x in torch.randint(1, most, (max(B - 4, 0),), generator=g)]
    table, pages = _pages(g, lens, page)
    q = _randn(g, B, n, H, D, dtype=dtype)
    kc, vc = _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    tree = _random_tree(g, B, n) if n > 1 else None
    some = sorted({0, 1 % B, 2 % B, 3 % B, B - 1, B // 2})
    out, tol = _cache_ref(q[some], kc, vc, table[some], [lens[b] for b in some], None if tree is None else tree[some], 1 / math.sqrt(D))
    args = [t.to(gpu) for t in (q, kc, vc, table)]
    ln, tg = torch.tensor(lens, device=gpu), None if tree is None else tree.to(gpu)
    got = svdmlp.cache_attention(*args, ln, tree=tg)
    _close(got[some], out, tol)
    for _ in range(3):
        assert torch.equal(got, svdmlp.cache_attention(*args, ln, tree=tg))
    assert all(int(c.abs().max()) == 0 for _, c in decoder._PARTIALS_CACHE.values())


@pytest.mark.parametrize("dtype,B,n,H,K,D,page,most", [
    (BF, 3, 17, 8, 2, 128, 16, 9000), (BF, 70, 9, 8, 1, 64, 64, 1500), (BF, 2, 64, 16, 2, 40, 7, 3000), (F32, 3, 33, 4, 2, 64, 16, 4000),
    (F32, 67, 17, 4, 1, 24, 32, 700), (BF, 1, 64, 8, 1, 128, 1, 20000), (BF, 2, 64, 2, 1, 96, 48, 513),
    (BF, 300, 9, 8, 1, 32, 16, 1300), (BF, 257, 5, 16, 1, 128, 32, 600)])
def test_cache_attention_many_rows(gpu, dtype, B, n, H, K, D, page, most):
    """Over 64 rows a head: tiles that four waves share, chunks chosen from the lengths, joined by a kernel of its own."""
    g = _gen(B + n)
    lens = [most, 0, n, n - 1][:B] + [int(x) for x in torch.randint(1, most, (max(B - 4, 0),), generator=g)]
    table, pages = _pages(g, lens, page)
    q = _randn(g, B, n, H, D, dtype=dtype)
    kc, vc = _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    for tree in (None, _random_tree(g, B, n)):
        some = sorted({0, 1 % B, 2 % B, 3 % B, B - 1, B // 2})
        out, tol = _cache_ref(q[some], kc, vc, table[some], [lens[b] for b in some], None if tree is None else tree[some], 1 / math.sqrt(D))
        args = [t.to(gpu) for t in (q, kc, vc, table)]
        ln, tg = torch.tensor(lens, device=gpu), None if tree is None else tree.to(gpu)
        got = svdmlp.cache_attention(*args, ln, tree=tg)
        _close(got[some], out, tol)
        assert torch.equal(got, svdmlp.cache_attention(*args, ln, tree=tg))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_cache_attention_hidden_drafts_have_no_part(gpu, dtype):
    """Infinities and NaN in a draft reach its descendants alone; a token whose row of the tree is empty sees the context, or nothing."""
    g = _gen(21)
    lens, n, H, K, D, page = [70, 4], 4, 4, 2, 128, 16
    table, pages = _pages(g, lens, page)
    q, kc, vc = _randn(g, 2, n, H, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    tree = torch.tensor([[1, 0, 0, 0], [1, 1, 0, 0], [1, 0, 1, 0], [0, 0, 0, 0]], dtype=torch.bool)
    out, tol = _cache_ref(q, kc, vc, table, lens, tree, 1 / math.sqrt(D))
    for b, length in enumerate(lens):
        key = length - n + 1  # draft 1: a parent of none
        page_of, row = int(table[b, key // page]), key % page
        kc[page_of, row], vc[page_of, row] = math.nan, math.inf
        key = length - n + 2  # draft 2: its values alone
        vc[int(table[b, key // page]), key % page, 0, 7] = math.inf
    args = [t.to(gpu) for t in (q, kc, vc, table)]
    got = svdmlp.cache_attention(*args, torch.tensor(lens, dtype=torch.int32, device=gpu), tree=tree.to(gpu)).cpu()
    assert torch.isnan(got[:, 1]).all()
    assert (got[:, 2, :H // K, 7] == math.inf).all()
    got[:, 2, :H // K, 7], out[:, 2, :H // K, 7] = 0, 0
    keep = [0, 2, 3]
    _close(got[:, keep], out[:, keep], tol[:, keep] + 1e-30)
    assert (got[1, 3] == 0).all()  # no context, an empty row


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,B", [(64, 1), (128, 1), (256, 1), (128, 300)])
def test_cache_attention_context_values_reach_every_token(gpu, dtype, D, B):
    """An infinity among the context's values is in every row's result, in its column alone."""
    g = _gen(25)
    n, H, K, page, most = 3, 4, 2, 16, 600
    lens = [most] * B
    table, pages = _pages(g, lens, page)
    q, kc, vc = _randn(g, B, n, H, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    vc[table[0, 2].item(), 5, 0, 7], vc[table[0, 20].item(), 0, 1, 9] = math.inf, -math.inf
    vc[table[0, most // page].item(), most % page - n - 1, 1, 3] = math.inf  # the last of the context
    got = svdmlp.cache_attention(*(t.to(gpu) for t in (q, kc, vc, table)), torch.tensor(lens, device=gpu)).cpu()
    assert (got[0, :, :H // K, 7] == math.inf).all() and (got[0, :, H // K:, 9] == -math.inf).all() and (got[0, :, H // K:, 3] == math.inf).all()
    got[0, :, :H // K, 7] = got[0, :, H // K:, 9] = got[0, :, H // K:, 3] = 0
    assert torch.isfinite(got.float()).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,B,n", [(64, 1, 3), (128, 1, 3), (64, 1, 20), (128, 1, 20), (64, 1, 40), (128, 1, 40), (256, 1, 3), (128, 300, 3)])
@pytest.mark.parametrize("page,lost", [(48, False), (16, True)])
def test_cache_attention_context_values_of_any_page(gpu, dtype, D, B, n, page, lost):
    """The same where tiles are not loaded whole: pages of no power of two, and a page outside the cache among the others."""
    g = _gen(26)
    H, K, most = 4, 2, 600
    table, pages = _pages(g, [most] * B, page)
    q, kc, vc = _randn(g, B, n, H, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    for key, head, e, x in ((37, 0, 7, math.inf), (321, 1, 9, -math.inf), (400, 1, 3, math.nan)):
        vc[table[0, key // page].item(), key % page, head, e] = x
    if lost:
        table[:, 10] = pages + 5
    got = svdmlp.cache_attention(*(t.to(gpu) for t in (q, kc, vc, table)), torch.tensor([most] * B, device=gpu)).cpu()
    assert (got[0, :, :H // K, 7] == math.inf).all() and (got[0, :, H // K:, 9] == -math.inf).all() and torch.isnan(got[0, :, H // K:, 3]).all()
    got[0, :, :H // K, 7] = got[0, :, H // K:, 9] = got[0, :, H // K:, 3] = 0
    assert torch.isfinite(got.float()).all()


def test_cache_attention_broken_tables(gpu):
    """Pages outside the cache hold no keys, lengths beyond the table are cut, negative ones empty."""
    g = _gen(22)
    page, K, D = 16, 2, 64
    kc, vc, q = _randn(g, 6, page, K, D), _randn(g, 6, page, K, D), _randn(g, 3, 1, 4, D)
    table = torch.tensor([[0, 99, 1], [2, 3, 4], [5, 5, 5]], dtype=torch.int32)
    lens = [48, 10 ** 9, -3]
    args = [t.to(gpu) for t in (q, kc, vc, table)]
    got = svdmlp.cache_attention(*args, torch.tensor(lens, dtype=torch.int32, device=gpu)).cpu()
    want, tol = _cache_ref(q[:2], kc, vc, torch.tensor([[0, 1, 1], [2, 3, 4]]), [32, 48], None, 0.125)
    _close(got[:2], want, tol)
    assert (got[2] == 0).all()


def test_cache_attention_large_cache(gpu):
    """Pages whose byte offsets pass 2^32, in the wide and the 16-bit type."""
    for dtype, pages in ((BF, 70000), (F32, 35000)):
        page, K, D = 64, 4, 128
        kc = torch.zeros((pages, page, K, D), dtype=dtype, device=gpu)
        vc = torch.zeros_like(kc)
        assert kc.numel() * kc.element_size() > 2 ** 32
        g = _gen(23)
        small = _randn(g, 2, 3, page, K, D, dtype=dtype)
        ids = torch.tensor([[pages - 1, 1, pages - 7]], dtype=torch.int32)
        kc[ids[0].long().to(gpu)], vc[ids[0].long().to(gpu)] = small[0].to(gpu), small[1].to(gpu)
        q = _randn(g, 1, 2, 8, D, dtype=dtype)
        want, tol = _cache_ref(q, small[0], small[1], torch.tensor([[0, 1, 2]]), [190], None, 1 / math.sqrt(D))
        got = svdmlp.cache_attention(q.to(gpu), kc, vc, ids.to(gpu), torch.tensor([190], device=gpu))
        _close(got, want, tol)
        # and written there
        k = _randn(g, 1, K, D, dtype=dtype)
        f = torch.zeros(1, dtype=torch.float64, device=gpu)
        slot = torch.tensor([pages * page - 1], device=gpu)
        svdmlp.rope_append(q[:, 0].to(gpu), k.to(gpu), k.to(gpu), slot, f, kc, vc, slot)
        assert torch.equal(kc[-1, -1].cpu(), k[0]) and torch.equal(vc[-1, -1].cpu(), k[0])
        del kc, vc


def test_cache_attention_joint_pool_and_strided_out(gpu):
    g = _gen(24)
    lens, n, H, K, D, page = [90, 37], 2, 8, 2, 128, 16
    table, pages = _pages(g, lens, page)
    pool = _randn(g, pages, 2, page, K, D)
    q = _randn(g, n, 2, H, D).transpose(0, 1)
    out, tol = _cache_ref(q, pool[:, 0], pool[:, 1], table, lens, None, 0.1)
    pg = pool.to(gpu)
    o = torch.empty(H, n, 2, D, dtype=BF, device=gpu).permute(2, 1, 0, 3)
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table.to(gpu)
    got = svdmlp.cache_attention(q.to(gpu), pg[:, 0], pg[:, 1], wide[:, :table.shape[1]], torch.tensor(lens, device=gpu), scale=0.1, out=o)
    assert got is o
    _close(o, out, tol)


def test_cache_attention_refusals(gpu):
    q = torch.zeros(2, 1, 4, 64, dtype=BF, device=gpu)
    c = torch.zeros(4, 16, 2, 64, dtype=BF, device=gpu)
    t, ln = torch.zeros(2, 2, dtype=torch.int32, device=gpu), torch.ones(2, dtype=torch.int32, device=gpu)
    cases = [
        (lambda: svdmlp.cache_attention(q[:1], c, c, t, ln), "block_table"),
        (lambda: svdmlp.cache_attention(q, c, c, t, ln[:1]), "lengths"),
        (lambda: svdmlp.cache_attention(q, c, c, t[:, :0], ln), "block_table"),
        (lambda: svdmlp.cache_attention(q, c, c, t, ln, tree=torch.ones(2, 2, dtype=torch.bool, device=gpu)), "tree"),
        (lambda: svdmlp.cache_attention(q, c, c, t, ln, tree=torch.ones(1, 1, dtype=torch.bool)), "same device"),
        (lambda: svdmlp.cache_attention(q, c, c.transpose(2, 3).contiguous().transpose(2, 3), t, ln), "contiguous"),
        (lambda: svdmlp.cache_attention(q, c, c, t, ln, out=q), "overlap"),
        (lambda: svdmlp.cache_attention(q, c, c, t, ln, scale=math.inf), "scale"),
        (lambda: svdmlp.cache_attention(q.clone().requires_grad_(), c, c, t, ln), "no gradient"),
    ]
    for fn, msg in cases:
        with pytest.raises(ValueError, match=msg):
            fn()
    assert svdmlp.cache_attention(q[:0], c, c, t[:0], ln[:0]).shape == (0, 1, 4, 64)


# ---------------------------------------------------------------------------
# Residual sum and norms
# ---------------------------------------------------------------------------

def _norm_ref(x, b, w, post, gate, scale, eps):
    rms = lambda t: torch.rsqrt((t * t).mean(dim=1, keepdim=True) + eps)  # noqa: E731
    r, mag = x.double(), x.double().abs()
    if b is not None:
        b = b.double()
        if post is not None:
            b = b * rms(b) * post.double()
        if gate is not None:
            b = b * gate.double()
        r, mag = r + scale * b, mag + abs(scale) * b.abs()
    n = None if w is None else r * rms(r) * w.double()
    nmag = None if w is None else mag * rms(r) * w.double().abs()
    return r, mag, n, nmag


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,d", [(1, 1), (1, 8), (3, 77), (5, 1000), (2, 4096), (9, 2560), (1, 8192), (300, 512), (2, 8191), (2, 32768), (1, 16392), (1, 31111)])
@pytest.mark.parametrize("post,gate", [(False, None), (True, "vector"), (True, "rows"), (False, "rows")])
def test_residual_norm(gpu, dtype, T, d, post, gate):
    g = _gen(T * 131 + d)
    x, b = (3 * torch.randn(T, d, generator=g)).to(dtype), _randn(g, T, d, dtype=dtype)
    w, pw = torch.rand(d, generator=g) + 0.5, torch.rand(d, generator=g) + 0.5 if post else None
    gt = {None: None, "vector": _randn(g, d, dtype=dtype), "rows": _randn(g, T, d, dtype=dtype)}[gate]
    dev = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    r, mag, n, nmag = _norm_ref(x, b, w, pw, gt, 0.7, 1e-5)
    xg, bg = dev(x), dev(b)
    gr, gn = svdmlp.residual_norm(xg, bg, dev(w), post_weight=dev(pw), gate=dev(gt), scale=0.7)
    u = U[dtype]
    _close(gr, r, u * r.abs() * 1.01 + 2.0 ** -17 * mag + 1e-38)
    _close(gn, n, u * n.abs() * 1.01 + 2.0 ** -16 * nmag + 1e-38)
    # in place, the norm over the branch: the same bits
    svdmlp.residual_norm(xg, bg, dev(w), post_weight=dev(pw), gate=dev(gt), scale=0.7, out=(xg, bg))
    assert torch.equal(xg, gr) and torch.equal(bg, gn)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_residual_norm_parts(gpu, dtype):
    """The norm before the first block, the sum after the last, strided rows, gains of another type."""
    g = _gen(31)
    T, d = 6, 256
    x, b, w = _randn(g, T, 2 * d, dtype=dtype)[:, :d], _randn(g, T, d, dtype=dtype), (torch.rand(d, generator=g) + 0.5).to(BF)
    xg = torch.zeros(T, 2 * d, dtype=dtype, device=gpu)[:, :d]
    xg.copy_(x)
    r, mag, n, nmag = _norm_ref(x, None, w, None, None, 1.0, 1e-6)
    gr, gn = svdmlp.residual_norm(xg, None, w.to(gpu), eps=1e-6)
    assert gr is xg
    _close(gn, n, U[dtype] * n.abs() * 1.01 + 2.0 ** -17 * nmag + 1e-38)
    r, mag, _, _ = _norm_ref(x, b, None, None, None, 1.0, 1e-6)
    gr, none = svdmlp.residual_norm(xg, b.to(gpu), None)
    assert none is None
    _close(gr, r, U[dtype] * r.abs() * 1.01 + 2.0 ** -17 * mag + 1e-38)


def test_residual_norm_refusals(gpu):
    x, w = torch.zeros(4, 16, device=gpu), torch.ones(16, device=gpu)
    cases = [
        (lambda: svdmlp.residual_norm(x, x[:3], w), "branch"), (lambda: svdmlp.residual_norm(x, x, w[:8]), "weight"),
        (lambda: svdmlp.residual_norm(x, x, w, gate=w[:8]), "gate"), (lambda: svdmlp.residual_norm(x, x, w, eps=0.0), "eps"),
        (lambda: svdmlp.residual_norm(x, x, w, scale=math.nan), "scale"),
        (lambda: svdmlp.residual_norm(x, x.clone(), w, out=(x, x)), "overlap"),
        (lambda: svdmlp.residual_norm(x[:2], x[2:].clone(), w, out=(x[1:3], None)), "overlap"),
        (lambda: svdmlp.residual_norm(torch.zeros(1, 40000, device=gpu), None, torch.ones(40000, device=gpu)), "at most"),
        (lambda: svdmlp.residual_norm(x.clone().requires_grad_(), x, w), "no gradient"),
    ]
    for fn, msg in cases:
        with pytest.raises(ValueError, match=msg):
            fn()


# ---------------------------------------------------------------------------
# Together, and as a program calls them
# ---------------------------------------------------------------------------

def test_graphs_and_streams(gpu):
    """Each operator captured into a graph: replays with eager work of the same
    stream between them give the eager bits; two graphs of cache attention that
    replay in turn do not share partial sums; and a call on another stream."""
    g = _gen(41)
    T, H, K, D, page = 40, 8, 2, 128, 16
    q, k, v = (_randn(g, T, n, D).to(gpu) for n in (H, K, K))
    f = svdmlp.rope_frequencies(D, 10000.0)[0].to(gpu)
    pos = torch.arange(T, device=gpu)
    lens = [5000, 300]
    table, pages = _pages(g, lens, page)
    kc, vc = _randn(g, pages, page, K, D).to(gpu), _randn(g, pages, page, K, D).to(gpu)
    table, ln = table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu)
    qc, q2 = _randn(g, 2, 1, H, D).to(gpu), _randn(g, 2, 3, H, D).to(gpu)
    x, w = _randn(g, T, 512).to(gpu), torch.ones(512, device=gpu)
    slots = torch.arange(T, device=gpu) + pages * page - T
    calls = [
        lambda: svdmlp.rope(q, k, pos, f),
        lambda: (svdmlp.rope_append(q, k, v, pos, f, kc, vc, slots), kc, vc),
        lambda: (svdmlp.prompt_attention(q, k, v),),
        lambda: (svdmlp.cache_attention(qc, kc, vc, table, ln),),
        lambda: (svdmlp.cache_attention(q2, kc, vc, table, ln),),
        lambda: svdmlp.residual_norm(x, x, w),
    ]
    calls[1]()
    want = [[t.clone() for t in c()] for c in calls]
    torch.cuda.synchronize()
    graphs = []
    for c in calls:
        c()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = c()
        graphs.append((gr, outs))
    for _ in range(3):
        for gr, outs in graphs:
            for o in outs:
                if o is not kc and o is not vc:
                    o.fill_(3.0)
        for gr, _ in graphs:
            gr.replay()
        for c in calls:  # eager work of the same kind between the replays
            c()
        torch.cuda.synchronize()
        for (_, outs), ws in zip(graphs, want):
            for o, e in zip(outs, ws):
                assert torch.equal(o, e)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [[t for t in c()] for c in calls]
    side.synchronize()
    for outs, ws in zip(got, want):
        for o, e in zip(outs, ws):
            assert torch.equal(o, e)


def test_decoder_layer_prefill_and_decode(gpu):
    """Two layers as a model runs them -- norm, projections, rotary positions
    into the cache, attention, sum and norm, SVD MLP -- over a packed prefill
    of three prompts, then one drafted tree a sequence and one more token each,
    against the same tokens in one prefill."""
    g = _gen(51)
    H, K, D, d, ff, r, page, layers = 8, 2, 64, 512, 1024, 256, 16, 2
    mk = lambda *s: (torch.randn(s, generator=g) / math.sqrt(s[0])).to(BF).to(gpu)  # noqa: E731
    ws = [dict(qkv=mk(d, (H + 2 * K) * D), o=mk(H * D, d), n1=torch.ones(d, device=gpu), n2=torch.ones(d, device=gpu),
               mlp=(mk(d, r), mk(r, ff), mk(d, r), mk(r, ff), mk(ff, r), mk(r, d))) for _ in range(layers)]
    f = svdmlp.rope_frequencies(D, 10000.0)[0].to(gpu)
    lens = [37, 5, 80]
    full = [n + 4 for n in lens]
    x_all = _randn(g, sum(full), d).to(gpu)
    ends = [sum(full[:i + 1]) for i in range(3)]
    starts = [e - n for e, n in zip(ends, full)]

    def layer(x, w, pos, attend):
        _, h = svdmlp.residual_norm(x, None, w["n1"])
        qkv = h @ w["qkv"]
        T = x.shape[0]
        q, k, v = (qkv[:, a * D:b * D].view(T, -1, D) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
        o = attend(q, k, v, pos).reshape(T, H * D) @ w["o"]
        x, h = svdmlp.residual_norm(x, o, w["n2"])
        return svdmlp.residual_norm(x, svdmlp.svd_mlp(h, *w["mlp"]), None)[0]

    # the whole of it in one prefill
    pos = torch.cat([torch.arange(n) for n in full]).to(gpu)
    cu = _cu(full, gpu)
    x = x_all
    for w in ws:
        x = layer(x, w, pos, lambda q, k, v, p: svdmlp.prompt_attention(*svdmlp.rope(q, k, p, f), v, cu))
    want = x

    # prefill of the prompts, then three tokens at once (a chain given as a tree), then one
    table, pages = _pages(g, full, page)
    table = table.to(gpu)
    caches = [(torch.zeros(pages, page, K, D, dtype=BF, device=gpu), torch.zeros(pages, page, K, D, dtype=BF, device=gpu)) for _ in ws]

    def step(take, attend_on_cache):
        rows = torch.cat([torch.arange(s + a, s + b) for s, (a, b) in zip(starts, take)]).to(gpu)
        pos = torch.cat([torch.arange(a, b) for a, b in take]).to(gpu)
        seq = torch.cat([torch.full((b - a,), i) for i, (a, b) in enumerate(take)]).to(gpu)
        slots = table[seq, pos // page].long() * page + pos % page
        cu = _cu([b - a for a, b in take], gpu)
        held = torch.tensor([b for _, b in take], dtype=torch.int32, device=gpu)
        n = take[0][1] - take[0][0]
        x = x_all[rows]
        for w, (kc, vc) in zip(ws, caches):
            def attend(q, k, v, p):
                qr = svdmlp.rope_append(q, k, v, p, f, kc, vc, slots)
                if attend_on_cache:
                    tree = torch.ones(n, n, dtype=torch.bool, device=gpu).tril() if n > 1 else None
                    return svdmlp.cache_attention(qr.view(3, n, H, D), kc, vc, table, held, tree=tree)
                kr = svdmlp.rope(q, k, p, f)[1]
                assert torch.equal(kc.view(-1, K, D)[slots], kr)
                return svdmlp.prompt_attention(qr, kr, v, cu)
            x = layer(x, w, pos, attend)
        return rows, x

    for take, cached in (([(0, n) for n in lens], False), ([(n, n + 3) for n in lens], True), ([(n + 3, n + 4) for n in lens], True)):
        rows, x = step(take, cached)
        a, b = x.float(), want[rows].float()
        # the same sums in other orders, rounded to bf16 at every step of two layers: a few times 2^-8
        assert torch.linalg.norm(a - b) / torch.linalg.norm(b) < 1e-2


def test_entry_points_are_exported():
    for name in ("rope", "rope_append", "prompt_attention", "cache_attention", "residual_norm", "rope_frequencies"):
        assert getattr(svdmlp, name) is getattr(decoder, name)


def test_rope_append_refuses_shared_memory(gpu):
    """Caches that are each other, or that hold the inputs; halves of one pool, and inputs beside a cache in one buffer, are fine."""
    pos, f = torch.arange(4, device=gpu), torch.ones(4, dtype=torch.float64, device=gpu)
    pool = torch.zeros(8, 2, 16, 1, 8, device=gpu)
    q, k = torch.randn(4, 2, 8, device=gpu), torch.randn(4, 1, 8, device=gpu)
    svdmlp.rope_append(q, k, k, pos, f, pool[:, 0], pool[:, 1], pos)
    assert torch.equal(pool[0, 1, :4], k)
    for kc, vc, kk in ((pool[:, 0], pool[:, 0], k), (pool[:4, 0], pool[2:6, 0], k), (pool[:, 0], pool[:, 1], pool[0, 0, :4])):
        with pytest.raises(ValueError, match="overlap"):
            svdmlp.rope_append(q, kk, k, pos, f, kc, vc, pos)
    with pytest.raises(ValueError, match="overlap"):
        svdmlp.rope_append(q, k, k, pos, f, pool[:, 0], pool[:, 1], pos, out=pool.view(-1)[:64].view(4, 2, 8))


def _cpu_decoder(x, weights, heads, kv_heads, theta):
    """The decoder's layers in 64 bits: causal, rotary positions of halves, no rounding in between."""
    x = x.double()
    T, H = x.shape
    D = H // heads
    angle = torch.arange(T, dtype=torch.float64)[:, None] * theta ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def norm(t, w):
        return t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w

    def turn(t):
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    for w in weights:
        w = {k: v.double().cpu() for k, v in w.items()}
        n = norm(x, w["norm1_w"])
        q, k, v = (turn((n @ w["wq"]).view(T, heads, D)), turn((n @ w["wk"]).view(T, kv_heads, D)), (n @ w["wv"]).view(T, kv_heads, D))
        k, v = k.repeat_interleave(heads // kv_heads, 1), v.repeat_interleave(heads // kv_heads, 1)
        s = torch.einsum("thd,uhd->htu", q, k) / math.sqrt(D)
        s = s.masked_fill(torch.ones(T, T).triu(1).bool(), -math.inf).softmax(-1)
        x = x + torch.einsum("htu,uhd->thd", s, v).reshape(T, H) @ w["wo"]
        n = norm(x, w["norm2_w"])
        h = torch.nn.functional.silu(n @ w["ug"] @ w["vg"]) * (n @ w["uu"] @ w["vu"])
        x = x + h @ w["ud"] @ w["vd"]
    return x


def test_decoder_model_prompt_and_steps(gpu):
    """The served model's layers against the same in 64 bits: a prompt, then tokens one by one over a page's end.

    Tolerance: per layer some 12 tensors are rounded to bf16 (half a step, at most 2^-8 of a value, 2^-9.8 rms), each of a
    branch that is at most the sum's size, twice over in the worst case: 2 layers * 12 * 2^-9.8 < 0.03 if all errors
    added up, 0.006 as independent ones; 0.02 lies between.
    """
    from svdmlp import e2e_block

    H, I, R, heads, kv = 512, 1024, 256, 8, 2
    gen = torch.Generator(device=gpu)
    gen.manual_seed(5)
    weights = [e2e_block.make_layer_weights(gen, gpu, H, I, R, heads, kv, torch.bfloat16) for _ in range(2)]
    x = (torch.randn((70, H), generator=gen, device=gpu) * 0.02).to(torch.bfloat16)
    want = _cpu_decoder(x.cpu(), weights, heads, kv, 500000.0)
    model = e2e_block.DecoderModel(weights, heads, kv, 70)
    got = [model.prompt(x[:61])] + [model.step(x[t:t + 1], t) for t in range(61, 70)]
    for a, b in ((got[0], want[:61]), *((g, want[t:t + 1]) for t, g in zip(range(61, 70), got[1:]))):
        a = a.double().cpu()
        assert float((a - b).norm() / b.norm()) < 0.02
    with pytest.raises(ValueError, match="positions"):
        model.step(x[:1], 128)


def test_decoder_step_captured(gpu):
    """The served model's step as one graph, replayed after its caches and input changed."""
    from svdmlp import e2e_block

    gen = torch.Generator(device=gpu)
    gen.manual_seed(6)
    weights = [e2e_block.make_layer_weights(gen, gpu, 512, 1024, 256, 8, 2, torch.bfloat16) for _ in range(2)]
    x = (torch.randn((40, 512), generator=gen, device=gpu) * 0.02).to(torch.bfloat16)
    model = e2e_block.DecoderModel(weights, 8, 2, 64)
    model.prompt(x[:39])
    inp = x[39:].clone()
    model.step(inp, 39)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.step(inp, 39)
    for seed in range(3):
        other = x.roll(seed + 1, 0)
        model.prompt(other[:39])
        inp.copy_(other[39:])
        want = model.step(inp, 39).clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_e2e_record_of_the_decoder_arm(gpu):
    import argparse

    from svdmlp import e2e_block

    args = argparse.Namespace(layers=2, model_path=None, compress_ratio=0.8, warmup=1, repeats=2, seed=3, dense_arm=False, decoder_arm=True)
    rec = e2e_block.bench_model(64, dict(hidden=512, intermediate=1024, heads=8, kv_heads=2, layers=2), args)
    assert rec["decoder_step_vs_block_relative_l2"] < 0.02  # as above
    for arm in ("decoder_block", "decoder_step"):
        assert rec[arm]["iterations"] == 2 and 0 < rec[arm]["latency_ms_min"] <= rec[arm]["latency_ms_max"]


def test_cache_attention_two_threads_on_a_stream(gpu):
    """Two threads' calls on one stream, each of two launches that share the stream's room for partial sums."""
    import threading

    g = _gen(31)
    B, n, H, K, D, page = 2, 16, 16, 2, 128, 16
    sets = []
    for lens in ([9000, 4000], [500, 7000]):
        table, pages = _pages(g, lens, page)
        sets.append([t.to(gpu) for t in (_randn(g, B, n, H, D), _randn(g, pages, page, K, D), _randn(g, pages, page, K, D), table, torch.tensor(lens))])
    want = [svdmlp.cache_attention(*s) for s in sets]
    got = [[], []]

    def work(i):
        for _ in range(40):
            got[i].append(svdmlp.cache_attention(*sets[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i]) and len(got[0]) == len(got[1]) == 40


def test_rope_append_into_interleaved_caches(gpu):
    """Keys and values of a head side by side, (pages, page, Hk, 2, D): two views of one buffer that share no element."""
    pos, f = torch.arange(20, device=gpu), torch.ones(4, dtype=torch.float64, device=gpu)
    pool = torch.zeros(3, 16, 2, 2, 8, device=gpu)
    q, k, v = torch.randn(20, 4, 8, device=gpu), torch.randn(20, 2, 8, device=gpu), torch.randn(20, 2, 8, device=gpu)
    svdmlp.rope_append(q, k, v, pos, f, pool[..., 0, :], pool[..., 1, :], pos)
    _, turned = svdmlp.rope(q, k, pos, f)
    assert torch.equal(pool.flatten(0, 1)[:20, :, 0], turned) and torch.equal(pool.flatten(0, 1)[:20, :, 1], v)
    assert (pool.flatten(0, 1)[20:] == 0).all()
    with pytest.raises(ValueError, match="overlap"):
        svdmlp.rope_append(q, k, v, pos, f, pool[..., 0, :], pool[..., 0, :], pos)


def test_cache_attention_graph_with_growing_sequences(gpu):
    """A captured call of many rows, whose chunks follow the lengths: replayed as the sequences grow, with other calls between."""
    g = _gen(51)
    B, n, H, K, D, page = 3, 16, 16, 2, 64, 16
    table, pages = _pages(g, [6000, 5000, 4000], page)
    q, kc, vc = (t.to(gpu) for t in (_randn(g, B, n, H, D), _randn(g, pages, page, K, D), _randn(g, pages, page, K, D)))
    table, lens = table.to(gpu), torch.tensor([30, 16, 700], dtype=torch.int32, device=gpu)
    svdmlp.cache_attention(q, kc, vc, table, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = svdmlp.cache_attention(q, kc, vc, table, lens)
    for now in ([30, 16, 700], [6000, 0, 1], [5999, 5000, 4000], [17, 900, 3999]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(3.0)
        graph.replay()
        want = svdmlp.cache_attention(q, kc, vc, table, lens)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
