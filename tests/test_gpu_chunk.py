"""Attention of packed chunks of new tokens onto a paged cache, against its
definition in 64 bits; the bounds are those of the other attentions
(test_gpu_decoder.py), whose arithmetic it has: joining chunks adds products
with exp2 of differences and sums of a few more terms, within the bound's sums."""

import math

import pytest
import torch

import svdmlp
from svdmlp import decoder
from test_gpu_decoder import BF, F32, _attend, _close, _gen, _pages, _randn

pytestmark = pytest.mark.gpu


def _ref(q, kc, vc, table, lens, news, scale, heads=None, lost=()):
    """(out, tolerance) of the given heads; pages in `lost` hold no keys."""
    T, H, D = q.shape
    K, page = kc.shape[2], kc.shape[1]
    heads = range(H) if heads is None else heads
    out, tol = torch.zeros(T, len(heads), D, dtype=torch.float64), torch.full((T, len(heads), D), 1e-30, dtype=torch.float64)
    first = 0
    for b, (length, n) in enumerate(zip(lens, news)):
        keys = torch.arange(length)
        pages = table[b].long()[keys // page]
        there = torch.ones(length, dtype=torch.bool)
        for x in lost:
            there &= pages != x
        keys, pages = keys[there], pages[there]
        at = pages * page + keys % page
        k, v = kc.flatten(0, 1)[at], vc.flatten(0, 1)[at]
        seen = keys[None] <= (length - n + torch.arange(n))[:, None]
        for i, h in enumerate(heads):
            r = slice(first, first + n)
            out[r, i], tol[r, i] = _attend(q[r, h], k[:, h // (H // K)], v[:, h // (H // K)], seen, scale, q.dtype)
        first += n
    return out, tol


def _cu(news, first=0):
    return torch.tensor([first] + [first + sum(news[:i + 1]) for i in range(len(news))], dtype=torch.int32)


def _spoil(kc, vc, table, lens):
    """NaN and infinities in rows that no sequence holds: nobody reads them."""
    page = kc.shape[1]
    used = torch.zeros(kc.shape[0] * page, dtype=torch.bool)
    for b, length in enumerate(lens):
        keys = torch.arange(length)
        used[table[b].long()[keys // page] * page + keys % page] = True
    kc.flatten(0, 1)[~used] = math.nan
    vc.flatten(0, 1)[~used] = math.inf


def _run(g, gpu, dtype, lens, news, H, K, D, page, heads=None, **more):
    table, pages = _pages(g, lens, page)
    q = _randn(g, sum(news), H, D, dtype=dtype)
    kc, vc = _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    scale = 1 / math.sqrt(D)
    out, tol = _ref(q, kc, vc, table, lens, news, scale, heads)
    _spoil(kc, vc, table, lens)
    args = [t.to(gpu) for t in (q, kc, vc, table)]
    ln, cu = torch.tensor(lens, device=gpu), _cu(news).to(gpu)
    got = svdmlp.chunk_attention(*args, ln, cu, **more)
    _close(got if heads is None else got[:, list(heads)], out, tol)
    assert torch.equal(got, svdmlp.chunk_attention(*args[:3], args[3].long(), ln.int(), cu.long(), **more))
    return got


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,news,H,K,D,page", [
    ([1], [1], 1, 1, 8, 1), ([5, 0, 1], [1, 0, 1], 4, 2, 64, 16), ([33, 64, 31], [33, 1, 7], 8, 8, 128, 16), ([1000, 17], [1, 17], 32, 8, 128, 16),
    ([129, 40], [70, 33], 8, 2, 128, 16), ([70, 640], [64, 300], 14, 2, 64, 16), ([300, 16, 999], [40, 16, 512], 8, 1, 128, 64),
    ([40], [7], 12, 4, 96, 48), ([2600], [3], 8, 1, 256, 32), ([300], [129], 8, 1, 256, 32), ([3, 2, 9], [3, 1, 4], 6, 3, 40, 3),
    ([257, 511], [257, 100], 3, 1, 80, 7), ([5000, 1], [1, 1], 7, 7, 80, 16), ([4097], [150], 16, 2, 64, 256), ([700], [200], 5, 1, 200, 16),
    ([65, 64, 63, 128], [65, 64, 63, 128], 8, 2, 128, 64), ([511], [511], 4, 1, 128, 1), ([300], [140], 6, 2, 64, 5), ([200] * 3, [65] * 3, 8, 2, 24, 8)])
def test_chunk_attention(gpu, dtype, lens, news, H, K, D, page):
    _run(_gen(sum(lens) + D), gpu, dtype, lens, news, H, K, D, page)


@pytest.mark.parametrize("dtype,lens,news,H,K,D,page", [
    (BF, [9000], [40], 16, 4, 128, 4), (BF, [20000, 300], [70, 2], 8, 2, 128, 16), (BF, [6000], [90], 4, 2, 64, 1), (BF, [12000, 11000], [300, 1], 4, 1, 96, 8),
    (BF, [5000], [5000], 2, 1, 64, 64), (BF, [30000], [2], 8, 1, 128, 48), (BF, [9000, 100], [140, 90], 2, 1, 256, 16), (F32, [7000], [40], 4, 2, 64, 16),
    (F32, [5000, 64], [3, 64], 4, 1, 128, 3), (F32, [3000], [300], 2, 1, 256, 32), (BF, [70000], [129], 1, 1, 128, 2), (BF, [40000, 3], [1, 3], 2, 2, 64, 16),
    (BF, [7000, 300], [150, 4], 4, 2, 256, 1), (F32, [5000], [70], 2, 1, 256, 1), (BF, [6000, 40], [170, 2], 4, 2, 128, 1)])
def test_chunk_attention_long_contexts(gpu, dtype, lens, news, H, K, D, page):
    """Contexts in several chunks, more pages than lie in LDS at once."""
    _run(_gen(sum(lens) + D), gpu, dtype, lens, news, H, K, D, page, heads=sorted({0, H - 1}))


@pytest.mark.parametrize("dtype,B,most,longest,H,K,D,page", [
    (BF, 200, 900, 3, 8, 2, 128, 16), (BF, 70, 2500, 60, 8, 2, 64, 16), (F32, 130, 300, 9, 4, 2, 64, 32), (BF, 66, 700, 5, 4, 4, 256, 16), (BF, 90, 400, 200, 4, 1, 128, 16),
    (BF, 140, 700, 45, 8, 2, 128, 16), (BF, 260, 500, 90, 3, 1, 64, 16), (BF, 130, 300, 50, 6, 2, 80, 8), (BF, 40, 700, 150, 4, 2, 128, 5)])
def test_chunk_attention_many_sequences(gpu, dtype, B, most, longest, H, K, D, page):
    """More sequences than a wave looks at at once, most with a token or none, some with chunks."""
    g = _gen(B + most)
    lens = [int(x) for x in torch.randint(0, most, (B,), generator=g)]
    news = [min(n, int(x) if i % 7 == 0 else i % 3 % 2) for i, (n, x) in enumerate(zip(lens, torch.randint(1, longest + 1, (B,), generator=g)))]
    _run(g, gpu, dtype, lens, news, H, K, D, page, heads=sorted({0, H - 1}))


def test_chunk_attention_many_rows(gpu):
    """As many row tiles as the card has CUs and more: no chunks; odd group sizes."""
    for H, K, D, lens, news in ((32, 8, 128, [2300, 700], [2100, 700]), (12, 4, 64, [3000, 1], [2990, 1]), (7, 1, 80, [1500, 1200], [900, 1200])):
        _run(_gen(H), gpu, BF, lens, news, H, K, D, 16, heads=sorted({0, H // 2, H - 1}))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_chunk_attention_is_the_other_attentions(gpu, dtype):
    """A prompt on its own is prompt_attention, one token a sequence cache_attention, within the roundings of both."""
    g = _gen(5)
    H, K, D, page = 8, 2, 128, 16
    lens = [300, 77]
    table, pages = _pages(g, lens, page)
    kc, vc = torch.zeros(pages, page, K, D, dtype=dtype), torch.zeros(pages, page, K, D, dtype=dtype)
    q, k, v = (_randn(g, sum(lens), n, D, dtype=dtype) for n in (H, K, K))
    first = 0
    for b, n in enumerate(lens):
        x = torch.arange(n)
        at = table[b].long()[x // page] * page + x % page
        kc.flatten(0, 1)[at], vc.flatten(0, 1)[at] = k[first:first + n], v[first:first + n]
        first += n
    out, tol = _ref(q, kc, vc, table, lens, lens, 1 / math.sqrt(D))
    dev = [t.to(gpu) for t in (q, k, v)]
    args = [t.to(gpu) for t in (kc, vc, table)] + [torch.tensor(lens, device=gpu)]
    got = svdmlp.chunk_attention(dev[0], *args, _cu(lens).to(gpu))
    want = svdmlp.prompt_attention(*dev, _cu(lens).to(gpu))
    _close(got, out, tol)
    _close(got, want.double().cpu(), 2 * tol)
    last = torch.tensor([lens[0] - 1, sum(lens) - 1])
    got = svdmlp.chunk_attention(dev[0][last], *args, _cu([1, 1]).to(gpu))
    _close(got, out[last], tol[last])
    _close(svdmlp.cache_attention(dev[0][last][:, None], *args)[:, 0], out[last], tol[last])


@pytest.mark.parametrize("dtype,H,K,D,news", [(BF, 8, 2, 128, [3, 9]), (BF, 8, 2, 128, [90, 40]), (BF, 8, 2, 64, [150, 4]), (F32, 4, 2, 64, [40, 9]), (BF, 4, 2, 256, [40, 9])])
def test_chunk_attention_more_tokens_than_lengths(gpu, dtype, H, K, D, news):
    """Tokens before the first key get zeros; rows of no sequence, before and behind, stay as they were."""
    g = _gen(6)
    lens, page = [max(1, news[0] // 2), 0], 16
    table, pages = _pages(g, lens, page)
    T = sum(news)
    q, kc, vc = _randn(g, T, H, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    out, tol = _ref(q, kc, vc, table, lens, news, 0.1)
    kept = torch.full((T + 8, H, D), 7.0, dtype=dtype, device=gpu)
    wide = torch.cat([q[:3], q, q[:5]]).to(gpu)
    got = svdmlp.chunk_attention(wide, kc.to(gpu), vc.to(gpu), table.to(gpu), torch.tensor(lens, device=gpu), _cu(news, 3).to(gpu), scale=0.1, out=kept).cpu()
    assert (got[:3] == 7).all() and (got[3 + T:] == 7).all()
    _close(got[3:3 + T], out, tol)
    assert (got[3:3 + news[0] - lens[0]] == 0).all() and (got[3 + news[0]:3 + T] == 0).all()


@pytest.mark.parametrize("dtype,H,K,D", [(BF, 4, 2, 64), (BF, 4, 2, 128), (BF, 4, 2, 256), (F32, 4, 2, 64), (F32, 4, 2, 128), (F32, 2, 2, 256)])
@pytest.mark.parametrize("n", [5, 40, 160])
@pytest.mark.parametrize("page", [16, 48, 6])
def test_chunk_attention_hidden_and_seen_values(gpu, dtype, H, K, D, n, page):
    """Infinities and NaN in later tokens have no part in earlier ones; those of the context reach every token, in their column alone."""
    g = _gen(D + n)
    lens, news = [700, n], [n, n]
    table, pages = _pages(g, lens, page)
    q, kc, vc = _randn(g, 2 * n, H, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    G = H // K

    def put(cache, b, key, head, e, x):
        cache[int(table[b, key // page]), key % page, head, e] = x

    out, tol = _ref(q, kc, vc, table, lens, news, 1 / math.sqrt(D))
    _spoil(kc, vc, table, lens)
    put(vc, 0, 37, 0, 7, math.inf)
    put(vc, 0, 321, 1, 3, -math.inf)
    put(vc, 0, 700 - n - 1, 1, 4, math.nan)       # the last of the context
    for b, length in enumerate(lens):             # the last token of each: keys and values
        kc[int(table[b, (length - 1) // page]), (length - 1) % page] = math.nan
        vc[int(table[b, (length - 1) // page]), (length - 1) % page] = math.inf
        put(vc, b, length - 2, 0, 5, math.inf)    # the last but one: a value
    got = svdmlp.chunk_attention(*(t.to(gpu) for t in (q, kc, vc, table)), torch.tensor(lens, device=gpu), _cu(news).to(gpu)).cpu()
    ends = [n - 1, 2 * n - 1]
    assert torch.isnan(got[ends]).all()
    assert (got[[n - 2, 2 * n - 2], :G, 5] == math.inf).all()
    clean = torch.ones_like(got, dtype=torch.bool)
    clean[ends] = False
    clean[[n - 2, 2 * n - 2], :G, 5] = False
    assert (got[:n - 1, :G, 7] == math.inf).all() and (got[:n - 1, G:, 3] == -math.inf).all() and torch.isnan(got[:n - 1, G:, 4]).all()
    clean[:n, :G, 7] = clean[:n, G:, 3] = clean[:n, G:, 4] = False
    _close(torch.where(clean, got, 0), torch.where(clean, out, 0.0), torch.where(clean, tol, 1.0))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_chunk_attention_large_scores(gpu, dtype):
    """Scores that grow along the keys by hundreds of powers of two: every tile, and every chunk, moves the maximum."""
    g = _gen(3)
    for lens, news, H, K, D in (([1500], [200], 4, 2, 64), ([5000, 40], [60, 3], 8, 2, 128)):
        page = 16
        table, pages = _pages(g, lens, page)
        q = _randn(g, sum(news), H, D, dtype=dtype).abs()
        kc, vc = _randn(g, pages, page, K, D, dtype=dtype).abs(), _randn(g, pages, page, K, D, dtype=dtype)
        for b, length in enumerate(lens):
            x = torch.arange(length)
            at = table[b].long()[x // page] * page + x % page
            kc.flatten(0, 1)[at] = (kc.flatten(0, 1)[at].float() * torch.linspace(0.0, 4.0, length)[:, None, None]).to(dtype)
        for scale in (1.0, 0.05):
            out, tol = _ref(q, kc, vc, table, lens, news, scale, [0, H - 1])
            got = svdmlp.chunk_attention(*(t.to(gpu) for t in (q, kc, vc, table)), torch.tensor(lens, device=gpu), _cu(news).to(gpu), scale=scale)
            _close(got[:, [0, H - 1]], out, tol)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (BF, 256), (F32, 64), (F32, 128), (F32, 256)])
@pytest.mark.parametrize("n", [2, 170])
@pytest.mark.parametrize("page", [16, 3])
def test_chunk_attention_pages_outside_the_cache(gpu, dtype, D, n, page):
    """They hold no keys, whatever page 0 holds; lengths beyond the table are cut, negative ones empty."""
    g = _gen(22)
    H, K = 4, 2
    lens, news = [600, 300], [n, n]
    table, pages = _pages(g, lens, page)
    q, kc, vc = _randn(g, 3 * n, H, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype), _randn(g, pages, page, K, D, dtype=dtype)
    kc[0], vc[0] = math.nan, math.inf
    broken = table.clone()
    for b, i in ((0, 0), (0, 5), (0, 17), (1, 300 // page - 1)):
        broken[b, i] = [-1, pages, 2 ** 31 - 1, -2 ** 31][i % 4]
    for b in range(2):
        for i in range(table.shape[1]):
            if table[b, i] == 0:
                broken[b, i] = -7
    holes = torch.where(broken == table, table, pages + 1)
    big = torch.cat([kc, torch.zeros(2, page, K, D, dtype=dtype)]), torch.cat([vc, torch.zeros(2, page, K, D, dtype=dtype)])
    out, tol = _ref(q[:2 * n], *big, holes, lens, news, 1 / math.sqrt(D), lost=(pages + 1,))
    three = torch.cat([broken, broken[:1]])
    got = svdmlp.chunk_attention(*(t.to(gpu) for t in (q, kc, vc, three)), torch.tensor(lens + [-3], device=gpu), _cu(news + [n]).to(gpu)).cpu()
    _close(got[:2 * n], out, tol)
    assert (got[2 * n:] == 0).all()
    # a length beyond the table is the table's
    full = table.shape[1] * page
    if full > 600:
        return
    one = svdmlp.chunk_attention(*(t.to(gpu) for t in (q[:n], kc, vc, broken[:1])), torch.tensor([10 ** 12], device=gpu), _cu([n]).to(gpu)).cpu()
    _close(one, out[:n], tol[:n])


def test_chunk_attention_bounds_outside_the_rows(gpu):
    """Bounds that leave the rows or run backwards are cut, not followed."""
    g = _gen(13)
    table, pages = _pages(g, [900, 900, 900], 16)
    q = _randn(g, 50, 4, 64).to(gpu)
    kc, vc, table = _randn(g, pages, 16, 1, 64).to(gpu), _randn(g, pages, 16, 1, 64).to(gpu), table.to(gpu)
    ln = torch.tensor([900, 900, 900], device=gpu)
    want = svdmlp.chunk_attention(q, kc, vc, table[:2], ln[:2], torch.tensor([0, 20, 50], device=gpu))
    got = svdmlp.chunk_attention(q, kc, vc, table[:2], ln[:2], torch.tensor([-5, 20, 2 ** 40], device=gpu))
    assert torch.equal(got, want)
    # overlapping and empty sequences: every row is some sequence's or untouched
    got = svdmlp.chunk_attention(q, kc, vc, table, ln, torch.tensor([0, 50, 10, 50], device=gpu), out=torch.zeros_like(q))
    torch.cuda.synchronize()
    assert got.shape == q.shape
    many = torch.tensor([0, 50] * 40, device=gpu)
    svdmlp.chunk_attention(q, kc, vc, table[:1].expand(79, -1), ln[:1].expand(79), many, out=torch.zeros_like(q))
    torch.cuda.synchronize()


def test_chunk_attention_layouts(gpu):
    """Keys and values of a page in one buffer, heads outside rows, caches of different strides, queries of a fused projection, an output with
    strides, a wider table."""
    g = _gen(24)
    lens, news, H, K, D, page = [90, 437], [20, 70], 8, 2, 128, 16
    table, pages = _pages(g, lens, page)
    T = sum(news)
    pool = _randn(g, pages, 2, page, K, D)
    fused = _randn(g, T, (H + 2 * K) * D)
    q = fused[:, :H * D].view(T, H, D)
    out, tol = _ref(q, pool[:, 0], pool[:, 1], table, lens, news, 0.1)
    pg, fg = pool.to(gpu), fused.to(gpu)
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table.to(gpu)
    ln, cu = torch.tensor(lens, device=gpu), _cu(news).to(gpu)
    qg = fg[:, :H * D].view(T, H, D)
    by_head = pg[:, 1].transpose(1, 2).contiguous().transpose(1, 2)
    for vc in (pg[:, 1], by_head, pg[:, 1].contiguous()):
        o = torch.empty(H, T, D, dtype=BF, device=gpu).transpose(0, 1)
        got = svdmlp.chunk_attention(qg, pg[:, 0], vc, wide[:, :table.shape[1]], ln, cu, scale=0.1, out=o)
        assert got is o
        _close(o, out, tol)
    _close(svdmlp.chunk_attention(qg[..., :], pg[:, 0], by_head, table.to(gpu), ln, cu, scale=0.1), out, tol)
    odd = torch.empty(T, H, D + 1, dtype=BF, device=gpu)[..., 1:]
    odd.copy_(qg)  # unaligned rows: copied
    _close(svdmlp.chunk_attention(odd, pg[:, 0], pg[:, 1], table.to(gpu), ln, cu, scale=0.1), out, tol)


def test_chunk_attention_large_cache(gpu):
    """Pages whose byte offsets pass 2^32."""
    pages, page, K, D = 70000, 64, 4, 128
    kc = torch.zeros((pages, page, K, D), dtype=BF, device=gpu)
    vc = torch.zeros_like(kc)
    g = _gen(23)
    small = _randn(g, 2, 3, page, K, D)
    ids = torch.tensor([[pages - 1, 1, pages - 7]], dtype=torch.int32)
    kc[ids[0].long().to(gpu)], vc[ids[0].long().to(gpu)] = small[0].to(gpu), small[1].to(gpu)
    for n in (2, 80):
        q = _randn(g, n, 8, D)
        want, tol = _ref(q, small[0], small[1], torch.tensor([[0, 1, 2]]), [190], [n], 1 / math.sqrt(D))
        _close(svdmlp.chunk_attention(q.to(gpu), kc, vc, ids.to(gpu), torch.tensor([190], device=gpu), _cu([n]).to(gpu)), want, tol)


def test_chunk_attention_graphs_streams_threads(gpu):
    """Two captured calls replayed in turn onto new lengths and bounds, with eager calls between, and threads on streams of their own."""
    import threading

    g = _gen(41)
    H, K, D, page = 8, 2, 128, 16
    table, pages = _pages(g, [6000, 6000, 6000], page)
    kc, vc, table = _randn(g, pages, page, K, D).to(gpu), _randn(g, pages, page, K, D).to(gpu), table.to(gpu)
    T = 120
    q = [_randn(g, T, H, D).to(gpu) for _ in range(2)]
    ln, cu = torch.zeros(3, dtype=torch.int32, device=gpu), torch.zeros(4, dtype=torch.int32, device=gpu)
    outs = [torch.zeros(T, H, D, dtype=BF, device=gpu) for _ in range(2)]

    def call(i):
        return svdmlp.chunk_attention(q[i], kc, vc, table, ln, cu, out=outs[i])

    plans = [([6000, 5000, 1], [0, 1, 100, 101]), ([130, 6000, 2000], [0, 118, 119, 120]), ([64, 0, 4000], [0, 40, 40, 120]), ([5999, 5998, 5997], [0, 40, 80, 120])]
    ln.copy_(torch.tensor(plans[0][0])), cu.copy_(torch.tensor(plans[0][1]))
    graphs = []
    for i in range(2):
        call(i)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call(i)
        graphs.append(gr)
    for lens, bounds in plans * 2:
        ln.copy_(torch.tensor(lens)), cu.copy_(torch.tensor(bounds))
        want = []
        for i in range(2):
            outs[i].fill_(3.0)
            want.append(call(i).clone())
        for o in outs:
            o.fill_(3.0)
        for gr in graphs:
            gr.replay()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    results, errors = [None] * 4, []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(5):
                    r = svdmlp.chunk_attention(q[i % 2], kc, vc, table, ln, cu, out=torch.full((T, H, D), 3.0, dtype=BF, device=gpu))
                s.synchronize()
            results[i] = r
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors and all(torch.equal(r, want[i % 2]) for i, r in enumerate(results))


def test_chunk_attention_room_is_the_streams(gpu):
    """A longer call on the same stream after a shorter one, and the shorter one again: the same bits."""
    g = _gen(17)
    H, K, D, page = 8, 2, 128, 16
    table, pages = _pages(g, [20000, 3000], page)
    kc, vc, table = _randn(g, pages, page, K, D).to(gpu), _randn(g, pages, page, K, D).to(gpu), table.to(gpu)
    small, large = _randn(g, 4, H, D).to(gpu), _randn(g, 700, H, D).to(gpu)
    svdmlp.clear_workspace_cache()
    calls = [lambda: svdmlp.chunk_attention(small, kc, vc, table[:, :200], torch.tensor([3000, 2900], device=gpu), _cu([3, 1]).to(gpu)),
             lambda: svdmlp.chunk_attention(large, kc, vc, table, torch.tensor([20000, 2900], device=gpu), _cu([690, 10]).to(gpu))]
    want = [c() for c in calls]
    assert decoder._PARTIALS_CACHE
    for _ in range(2):
        for c, w in zip(calls, want):
            assert torch.equal(c(), w)


def test_chunk_attention_refusals(gpu):
    q = torch.zeros(5, 4, 64, dtype=BF, device=gpu)
    c = torch.zeros(4, 16, 2, 64, dtype=BF, device=gpu)
    t, ln = torch.zeros(2, 2, dtype=torch.int32, device=gpu), torch.ones(2, dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 2, 5], dtype=torch.int32, device=gpu)
    cases = [
        (lambda: svdmlp.chunk_attention(q[:, None], c, c, t, ln, cu), "expected q"),
        (lambda: svdmlp.chunk_attention(q, c, c[:3], t, ln, cu), "caches must have shape"),
        (lambda: svdmlp.chunk_attention(q[:, :3], c, c, t, ln, cu), "no multiple"),
        (lambda: svdmlp.chunk_attention(q, c, c, t[:1], ln, cu), "lengths"),
        (lambda: svdmlp.chunk_attention(q, c, c, t, ln, cu[:2]), "cu_seqlens"),
        (lambda: svdmlp.chunk_attention(q, c, c, t[:, :0], ln, cu), "block_table"),
        (lambda: svdmlp.chunk_attention(q, c, c, t.cpu(), ln, cu), "same device"),
        (lambda: svdmlp.chunk_attention(q, c, c, t, ln, cu.cpu()), "same device"),
        (lambda: svdmlp.chunk_attention(q, c, c.transpose(2, 3).contiguous().transpose(2, 3), t, ln, cu), "contiguous"),
        (lambda: svdmlp.chunk_attention(q, c, c, t, ln, cu, out=q), "overlap"),
        (lambda: svdmlp.chunk_attention(q, c, c, t, ln, cu, out=c.view(-1)[:5 * 4 * 64].view(5, 4, 64)), "overlap"),
        (lambda: svdmlp.chunk_attention(q, c, c, t, ln, cu, scale=0.0), "scale"),
        (lambda: svdmlp.chunk_attention(q[..., :12], c[..., :12], c[..., :12], t, ln, cu), "head sizes"),
        (lambda: svdmlp.chunk_attention(q.clone().requires_grad_(), c, c, t, ln, cu), "no gradient"),
    ]
    for fn, msg in cases:
        with pytest.raises(ValueError, match=msg):
            fn()
    with pytest.raises(TypeError, match="cu_seqlens"):
        svdmlp.chunk_attention(q, c, c, t, ln, cu.float())
    assert svdmlp.chunk_attention(q[:0], c, c, t, ln, cu).shape == (0, 4, 64)
    untouched = torch.full((5, 4, 64), 2.0, dtype=BF, device=gpu)
    assert (svdmlp.chunk_attention(q, c, c, t[:0], ln[:0], cu[:1], out=untouched) == 2).all()
