"""The operators around the MLP block where layouts, indices and sizes are
unusual: dimensions of one element with any stride, indices beyond 32 bits,
calls of tens of millions of rows, memory shared with what a call reads."""

import math

import pytest
import torch

import svdmlp
from svdmlp import decoder

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _randn(seed, *shape, dtype=BF):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype)


def _laid_out(t, strides, gpu):
    """t's values in a tensor of these strides on the GPU."""
    room = 1 + sum(s * (n - 1) for s, n in zip(strides, t.shape))
    out = torch.zeros(room, dtype=t.dtype, device=gpu).as_strided(t.shape, strides)
    return out.copy_(t)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,K,strides", [
    (1, 1, (132, 130, 1)), (1, 2, (3, 128, 1)), (1, 1, (1 << 24, 128, 1)), (3, 1, (136, 7, 1)), (1, 1, (0, 0, 1))])
def test_prompt_attention_dimensions_of_one(gpu, dtype, T, K, strides):
    """The stride of a dimension of one element says nothing: the same bits as from dense tensors."""
    H, D = 4, 128
    q, k, v = _randn(1, T, H, D, dtype=dtype), _randn(2, T, K, D, dtype=dtype), _randn(3, T, K, D, dtype=dtype)
    want = svdmlp.prompt_attention(*(t.to(gpu) for t in (q, k, v)))
    qs = (strides[0] if T == 1 else H * D, D, 1)
    out = _laid_out(torch.zeros(T, H, D, dtype=dtype), qs, gpu)
    got = svdmlp.prompt_attention(_laid_out(q, qs, gpu), _laid_out(k, strides, gpu), _laid_out(v, strides, gpu), out=out)
    assert got is out and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("pages,page,K,strides", [
    (1, 16, 2, (3, 128, 64, 1)), (5, 1, 2, (128, 7, 64, 1)), (5, 1, 2, (128, 1 << 24, 64, 1)), (3, 16, 1, (1024, 64, 5, 1)), (1, 1, 1, (1, 1, 1, 1))])
def test_cache_attention_dimensions_of_one(gpu, dtype, pages, page, K, strides):
    H, D = 4, 64
    q, kc, vc = _randn(4, 1, 1, H, D, dtype=dtype), _randn(5, pages, page, K, D, dtype=dtype), _randn(6, pages, page, K, D, dtype=dtype)
    table, lens = torch.arange(pages, dtype=torch.int32, device=gpu)[None], torch.tensor([pages * page], dtype=torch.int32, device=gpu)
    want = svdmlp.cache_attention(*(t.to(gpu) for t in (q, kc, vc)), table, lens)
    out = _laid_out(torch.zeros(1, 1, H, D, dtype=dtype), (5, 3, D, 1), gpu)
    got = svdmlp.cache_attention(_laid_out(q, (7, 9, D, 1), gpu), _laid_out(kc, strides, gpu), _laid_out(vc, strides, gpu), table, lens, out=out)
    assert got is out and torch.equal(got, want)
    one = _laid_out(_randn(7, 1, 1, 1, D, dtype=dtype), (1, 1, 1, 1), gpu)  # one head too
    if K == 1:
        assert torch.equal(svdmlp.cache_attention(one, kc.to(gpu), vc.to(gpu), table, lens),
                           svdmlp.cache_attention(one.contiguous().clone(), kc.to(gpu), vc.to(gpu), table, lens))


def test_cache_attention_indices_beyond_32_bits(gpu):
    """Pages of 64 bits that lie outside the cache hold no keys, and lengths are cut at the table, whatever their low 32 bits say."""
    page, K, D, pages = 16, 2, 64, 6
    q, kc, vc = (t.to(gpu) for t in (_randn(8, 4, 1, 4, D), _randn(9, pages, page, K, D), _randn(10, pages, page, K, D)))
    table = torch.tensor([[0, (1 << 32) + 3, 1], [-(1 << 32) + 2, 2, 1 << 31], [3, 4, (1 << 40) + 5], [1, 1, -1]], device=gpu)
    lens = torch.tensor([48, 1 << 31, (1 << 32) + 5, -(1 << 32) + 7], device=gpu)
    inside = torch.where((table >= 0) & (table < pages), table, -1).int()
    want = svdmlp.cache_attention(q, kc, vc, inside, lens.clamp(0, 48).int())
    assert torch.equal(svdmlp.cache_attention(q, kc, vc, table, lens), want)
    assert (want[3] == 0).all() and (want[:3] != 0).any()


def test_prompt_attention_bounds_beyond_32_bits(gpu):
    q, k, v = (_randn(s, 50, 2, 64).to(gpu) for s in (11, 12, 13))
    want = svdmlp.prompt_attention(q, k, v, torch.tensor([0, 20, 50], dtype=torch.int32, device=gpu))
    for cu in ([-(1 << 32) + 9, 20, (1 << 32) + 30], [0, 20, 1 << 31]):
        got = svdmlp.prompt_attention(q, k, v, torch.tensor(cu, device=gpu), out=torch.zeros_like(q))
        assert torch.equal(got, want)


def test_cache_attention_longest_sequence(gpu):
    """A sequence near 2^31 tokens: its last chunk would end beyond (2^25 keys a chunk, 64 of them).  Keys of one page there
    outweigh all others by e^60, so that the result is the mean of their values, all 1.5: sums of up to 2^21 weights of 1
    and values of 1.5 are exact in 32 bits."""
    page, width, D = 2097150, 1024, 8
    kc, vc = torch.zeros((2, page, 1, D), dtype=BF, device=gpu), torch.full((2, page, 1, D), -2.0, dtype=BF, device=gpu)
    kc[1, :, 0, 0], vc[1] = 60.0, 1.5
    q = torch.zeros((1, 1, 1, D), dtype=BF, device=gpu)
    q[..., 0] = 1.0
    table = torch.zeros((1, width), dtype=torch.int32, device=gpu)
    table[0, 1020] = 1
    assert page * 1020 >= 63 * 2 ** 25 and page * width > 2 ** 31 - 8192
    got = svdmlp.cache_attention(q, kc, vc, table, torch.tensor([page * width], device=gpu), scale=1.0)
    assert (got == 1.5).all()


@pytest.mark.parametrize("T,d,dtype", [((1 << 24) + 5, 8, BF), ((1 << 23) + 3, 6, F32)])
def test_residual_norm_of_many_rows(gpu, T, d, dtype):
    """More rows than one launch can have (2^32 threads): the same bits as of the rows alone."""
    x = torch.randn((T, d), device=gpu, dtype=F32).to(dtype)
    b, gate, w = x.flip(0), torch.randn((T, d), device=gpu).to(dtype), torch.rand(d, device=gpu)
    r, n = svdmlp.residual_norm(x, b, w, gate=gate, scale=0.5)
    for at in (0, (1 << 21) - 3, (1 << 22) - 2, (1 << 23) - 4, T - 7):
        s = slice(at, at + 7)
        r1, n1 = svdmlp.residual_norm(x[s], b[s], w, gate=gate[s], scale=0.5)
        assert torch.equal(r[s], r1) and torch.equal(n[s], n1)


def test_rope_of_many_tokens(gpu):
    T = (1 << 26) + 9
    q, k = torch.randn((T, 1, 2), device=gpu, dtype=BF), torch.randn((T, 1, 2), device=gpu, dtype=BF)
    pos, f = torch.arange(T, device=gpu), torch.ones(1, dtype=torch.float64, device=gpu)
    oq, ok = svdmlp.rope(q, k, pos, f)
    kc, vc = torch.zeros((T, 1, 1, 2), device=gpu, dtype=BF), torch.zeros((T, 1, 1, 2), device=gpu, dtype=BF)
    aq = svdmlp.rope_append(q, k, q, pos, f, kc, vc, pos)
    assert torch.equal(aq, oq) and torch.equal(kc[:, 0], ok) and torch.equal(vc[:, 0], q)
    for at in (0, (1 << 24) - 3, (1 << 25) - 3, (1 << 26) - 3, T - 7):
        s = slice(at, at + 7)
        q1, k1 = svdmlp.rope(q[s], k[s], pos[s], f)
        assert torch.equal(oq[s], q1) and torch.equal(ok[s], k1)


def test_attention_of_more_blocks_than_a_launch_has(gpu):
    """Refused, not cut."""
    q = torch.zeros((1, 1, 64), dtype=BF, device=gpu)
    cu = torch.ones((1 << 24) + 2, dtype=torch.int32, device=gpu)
    cu[0] = 0
    with pytest.raises(ValueError, match="one launch"):
        svdmlp.prompt_attention(q, q, q, cu)
    assert torch.equal(svdmlp.prompt_attention(q, q, q, cu[:1 << 20]), q)
    many = torch.zeros((1, 1, 1, 64), dtype=BF, device=gpu).expand((1 << 22) + 2, 1, 16, 64)
    cache = torch.zeros((1, 16, 16, 64), dtype=BF, device=gpu)
    table, lens = torch.zeros(((1 << 22) + 2, 1), dtype=torch.int32, device=gpu), torch.ones((1 << 22) + 2, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError, match="one launch"):
        svdmlp.cache_attention(many, cache, cache, table, lens)


def test_gradients_of_every_tensor_are_refused(gpu):
    """Frequencies, outputs, gains and forward-mode tangents too: nothing that asks for a gradient is used without one."""
    import torch.autograd.forward_ad as fwd

    q, k, pos = torch.randn(4, 2, 8, device=gpu), torch.randn(4, 1, 8, device=gpu), torch.arange(4, device=gpu)
    f, x, w = torch.ones(4, device=gpu), torch.randn(4, 16, device=gpu), torch.ones(16, device=gpu)
    c, qc = torch.zeros(2, 16, 1, 8, device=gpu), q.view(4, 1, 2, 8)
    table, lens = torch.zeros(4, 2, dtype=torch.int32, device=gpu), torch.ones(4, dtype=torch.int32, device=gpu)

    def calls(ask):
        return [
            lambda: svdmlp.rope(ask(q), k, pos, f), lambda: svdmlp.rope(q, k, pos, ask(f)),
            lambda: svdmlp.rope(q, k, pos, f, out=(ask(torch.empty_like(q)), torch.empty_like(k))),
            lambda: svdmlp.rope(q, k, pos, f, out=(torch.empty_like(q), ask(torch.empty_like(k)))),
            lambda: svdmlp.rope_append(q, k, ask(k), pos, f, c.clone(), c.clone(), pos),
            lambda: svdmlp.rope_append(q, k, k, pos, ask(f), c.clone(), c.clone(), pos),
            lambda: svdmlp.rope_append(q, k, k, pos, f, c.clone(), ask(c.clone()), pos),
            lambda: svdmlp.rope_append(q, k, k, pos, f, c.clone(), c.clone(), pos, out=ask(torch.empty_like(q))),
            lambda: svdmlp.prompt_attention(q, ask(k), k), lambda: svdmlp.prompt_attention(q, k, k, out=ask(torch.empty_like(q))),
            lambda: svdmlp.cache_attention(qc, c, ask(c.clone()), table, lens),
            lambda: svdmlp.cache_attention(qc, c, c, table, lens, out=ask(torch.empty_like(qc))),
            lambda: svdmlp.residual_norm(x, x, ask(w)), lambda: svdmlp.residual_norm(x, ask(x), w),
            lambda: svdmlp.residual_norm(x, x, w, post_weight=ask(w)), lambda: svdmlp.residual_norm(x, x, w, gate=ask(w)),
            lambda: svdmlp.residual_norm(x, x, w, out=(ask(torch.empty_like(x)), None)),
            lambda: svdmlp.residual_norm(x, x, w, out=(None, ask(torch.empty_like(x)))),
        ]

    for call in calls(lambda t: t.clone().requires_grad_()):
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    with fwd.dual_level():
        for call in calls(lambda t: fwd.make_dual(t.clone(), torch.ones_like(t))):
            with pytest.raises(ValueError, match="no gradient"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="no gradient"):  # which does not end tangents
                call()
        for call in calls(lambda t: t):
            call()


def test_room_for_partial_sums_does_not_shrink(gpu):
    """Calls of more counters and fewer bytes, and of fewer counters and more bytes, in turn: one pair of buffers serves both."""
    svdmlp.clear_workspace_cache()
    decoder._partials(0, 1 << 22, 10)
    wide = decoder._partials(0, 1 << 10, 9000)
    assert wide[0].numel() >= 1 << 22 and wide[1].numel() >= 9000
    again = decoder._partials(0, 1 << 22, 10)
    assert again[0] is wide[0] and again[1] is wide[1]
    assert (wide[1] == 0).all()
    svdmlp.clear_workspace_cache()


def _equal_values(D, K, T, dtype, gpu):
    """Queries and keys whose weights are 1 and exp(-t), many t, and values alike for all keys."""
    q, k = torch.zeros(T, K, D), torch.zeros(T, K, D)
    q[:, :, 0] = torch.linspace(0.05, 1.4, T)[:, None]
    k[1:, :, 0] = -1.0
    v = _randn(20, 1, K, D, dtype=dtype).expand(T, K, D).contiguous()
    return q.to(dtype).to(gpu), k.to(dtype).to(gpu), v.to(gpu)


@pytest.mark.parametrize("D", [64, 96, 128, 200, 256])
@pytest.mark.parametrize("T,K", [(64, 2), (257, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_weights_are_summed_as_rounded(gpu, D, T, K, causal):
    """Values that all keys share come out as they are: the sum is of the weights as the products take them, rounded to
    bf16.  What is left are sums in 32 bits, T + 8 roundings of at most 2^-23 each: 2^-14 for 257 tokens, less than half a
    step of bf16 (2^-9 of a value at least), so the result rounds to the value itself."""
    q, k, v = _equal_values(D, K, T, BF, gpu)
    assert torch.equal(svdmlp.prompt_attention(q, k, v, causal=causal, scale=1.0), v)
    table, lens = torch.arange(T, dtype=torch.int32, device=gpu)[None], torch.tensor([T], dtype=torch.int32, device=gpu)
    for n in (1, 9):
        got = svdmlp.cache_attention(q[None, -n:], k[:, None], v[:, None], table, lens, scale=1.0)
        assert torch.equal(got[0], v[-n:])


def test_outputs_apart_from_everything_read(gpu):
    """Outputs that share memory with gains, frequencies, positions, slots, bounds, tables, lengths or a tree are refused."""
    room = torch.zeros(4096, device=gpu)
    q, k, v = torch.randn(4, 2, 8, device=gpu), torch.randn(4, 1, 8, device=gpu), torch.randn(4, 1, 8, device=gpu)
    pos, f, slots = torch.arange(4, device=gpu), torch.ones(4, dtype=torch.float64, device=gpu), torch.arange(4, device=gpu)
    whole = room[:64].view(4, 2, 8)
    half = room[64:96].view(4, 1, 8)
    as_i64, as_i32, as_f64, as_u8 = room.view(torch.int64), room.view(torch.int32), room.view(torch.float64), room.view(torch.uint8)
    caches = [torch.zeros(2, 16, 1, 8, device=gpu) for _ in range(2)]
    x, b, w, g = torch.randn(4, 8, device=gpu), torch.randn(4, 8, device=gpu), torch.ones(8, device=gpu), torch.ones(8, device=gpu)
    qc = q.view(4, 1, 2, 8)
    table, lens = torch.zeros(4, 2, dtype=torch.int32, device=gpu), torch.ones(4, dtype=torch.int32, device=gpu)
    tree = torch.ones(4, 1, 1, dtype=torch.bool, device=gpu)
    cases = [
        lambda: svdmlp.rope(q, k, as_i64[:4], f, out=(whole, half)),
        lambda: svdmlp.rope(q, k, as_i64[32:36], f, out=(whole, half)),
        lambda: svdmlp.rope(q, k, pos, as_f64[:4], out=(whole, half)),
        lambda: svdmlp.rope_append(q, k, v, as_i64[:4], f, *caches, slots, out=whole),
        lambda: svdmlp.rope_append(q, k, v, pos, as_f64[:4], *caches, slots, out=whole),
        lambda: svdmlp.rope_append(q, k, v, pos, f, *caches, as_i64[:4], out=whole),
        lambda: svdmlp.rope_append(q, k, v, pos, f, room[:256].view(2, 16, 1, 8), caches[1], as_i64[:4]),
        lambda: svdmlp.rope_append(q, k, v, as_i64[100:104], f, caches[0], room[:256].view(2, 16, 1, 8), slots),
        lambda: svdmlp.rope_append(q, k, v, pos, as_f64[100:104], caches[0], room[:256].view(2, 16, 1, 8), slots),
        lambda: svdmlp.prompt_attention(q, k, v, as_i32[:2], out=whole),
        lambda: svdmlp.cache_attention(qc, *caches, as_i32[:8].view(4, 2), lens, out=whole.view(4, 1, 2, 8)),
        lambda: svdmlp.cache_attention(qc, *caches, table, as_i32[60:64], out=whole.view(4, 1, 2, 8)),
        lambda: svdmlp.cache_attention(qc, *caches, table, lens, tree=as_u8[:4].view(4, 1, 1), out=whole.view(4, 1, 2, 8)),
        lambda: svdmlp.residual_norm(x, b, room[8:16], out=(room[:32].view(4, 8), None)),
        lambda: svdmlp.residual_norm(x, b, w, post_weight=room[8:16], out=(None, room[:32].view(4, 8))),
        lambda: svdmlp.residual_norm(x, b, w, gate=room[8:16], out=(None, room[:32].view(4, 8))),
    ]
    for call in cases:
        with pytest.raises(ValueError, match="overlap"):
            call()
    # beside each other in one buffer they are fine
    svdmlp.rope(q, k, as_i64[512:516], as_f64[600:604], out=(whole, half))
    svdmlp.prompt_attention(q, k, v, as_i32[64:66], out=whole)
    svdmlp.cache_attention(qc, *caches, as_i32[64:72].view(4, 2), as_i32[72:76], tree=as_u8[400:404].view(4, 1, 1), out=whole.view(4, 1, 2, 8))
    svdmlp.residual_norm(x, b, room[128:136], post_weight=room[136:144], gate=room[144:152], out=(whole.view(8, 8)[:4], whole.view(8, 8)[4:]))
    assert torch.equal(g, torch.ones_like(g)) and not tree.logical_not().any()


@pytest.mark.parametrize("dtype,B,n,H,K,D,page,most", [(BF, 24, 64, 8, 1, 256, 16, 3000), (BF, 40, 20, 8, 1, 200, 48, 4000), (F32, 24, 40, 16, 2, 128, 16, 2500)])
def test_cache_attention_many_rows_of_large_heads(gpu, dtype, B, n, H, K, D, page, most):
    """Many row tiles of 32 over longer chunks than 256 keys."""
    import test_gpu_decoder as base

    g = base._gen(B + n)
    lens = [most, 0, n - 1, n] + [int(x) for x in torch.randint(1, most, (B - 4,), generator=g)]
    table, pages = base._pages(g, lens, page)
    q, kc, vc = (base._randn(g, *shape, dtype=dtype) for shape in ((B, n, H, D), (pages, page, K, D), (pages, page, K, D)))
    tree = base._random_tree(g, B, n)
    some = [0, 1, 2, 3, B - 1]
    out, tol = base._cache_ref(q[some], kc, vc, table[some], [lens[b] for b in some], tree[some], 1 / math.sqrt(D))
    args = [t.to(gpu) for t in (q, kc, vc, table)] + [torch.tensor(lens, device=gpu)]
    got = svdmlp.cache_attention(*args, tree=tree.to(gpu))
    base._close(got[some], out, tol)
    assert torch.equal(got, svdmlp.cache_attention(*args, tree=tree.to(gpu)))


def test_svd_mlp_block_of_many_rows(gpu):
    """The block's RMSNorm too: rows beyond a launch's 2^24 come out as in a call of their own.  The two calls may sum in
    other orders: a row's elements are compared as a whole, within 2^-6 of its size (four roundings to bf16 on the way)."""
    T, d, r = (1 << 24) + 300, 64, 64
    g = torch.Generator(device=gpu)
    g.manual_seed(3)
    x = torch.randn((T, d), device=gpu, generator=g).to(BF)
    w = [(torch.randn(s, device=gpu, generator=g) / 8).to(BF) for s in ((d, r), (r, 128), (d, r), (r, 128), (128, r), (r, d))]
    gain = torch.ones(d, device=gpu)
    y = svdmlp.svd_mlp_block(x, gain, *w, eps=1e-5)
    for at in (0, (1 << 23) - 150, T - 300):
        s = slice(at, at + 300)
        a, b = y[s].float(), svdmlp.svd_mlp_block(x[s].contiguous(), gain, *w, eps=1e-5).float()
        assert ((a - b).norm(dim=1) <= 2.0 ** -6 * b.norm(dim=1)).all()
    svdmlp.clear_workspace_cache()


@pytest.mark.parametrize("D", [4, 12, 36, 68, 132, 252])
def test_attention_of_fp32_heads_of_odd_pieces(gpu, D):
    """Heads of an odd number of 16-byte pieces, prompts and cache, one token and many rows."""
    import test_gpu_decoder as base

    g = base._gen(D)
    lens, H, K = [37, 1, 150], 6, 2
    (q, k, v), dev = base._qkv(g, sum(lens), H, K, D, F32, gpu)
    for causal in (True, False):
        base._close(svdmlp.prompt_attention(*dev, base._cu(lens, gpu), causal=causal), *base._prompt_ref(q, k, v, lens, causal, 1 / math.sqrt(D)))
    for page, lens in ((16, [300, 31]), (5, [41, 700])):
        table, pages = base._pages(g, lens, page)
        kc, vc = base._randn(g, pages, page, K, D, dtype=F32), base._randn(g, pages, page, K, D, dtype=F32)
        for n in (1, 7, 30):
            q = base._randn(g, 2, n, H, D, dtype=F32)
            got = svdmlp.cache_attention(*(t.to(gpu) for t in (q, kc, vc, table)), torch.tensor(lens, device=gpu))
            base._close(got, *base._cache_ref(q, kc, vc, table, lens, None, 1 / math.sqrt(D)))
