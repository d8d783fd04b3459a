"""Attention over chunks where a block takes long tiles by itself: more pages than
their numbers lie in LDS at once (2047 by tiles of 128 rows, 4095 by tiles of 256),
so that a piece is walked in several segments; and where a table is so wide that a
unit of the line is several keys.  Against the definition in 64 bits, with
the bounds of test_gpu_decoder.py."""

import math

import pytest
import torch

import svdmlp
from test_gpu_decoder import BF, F32, _attend, _close, _cu, _gen, _randn

pytestmark = pytest.mark.gpu


def _check(gpu, dtype, lens, news, H, K, D, page, pages, width, rows, heads, lost=(), odd=()):
    """rows: (sequence, its new tokens' numbers) to compare.  Sequences share pages.  lost: (sequence, key) whose page is no page of the cache;
    odd: the same, with infinities in its values, in one column a head."""
    g = _gen(D + len(lens))
    held = [-(-n // page) for n in lens]
    table = torch.full((len(lens), width or max(held)), -1, dtype=torch.int32)
    for b, c in enumerate(held):
        table[b, :c] = torch.randint(0, pages, (c,), generator=g)
    kc, vc = _randn(g, pages + len(odd), page, K, D, dtype=dtype), _randn(g, pages + len(odd), page, K, D, dtype=dtype)
    for i, (b, key) in enumerate(odd):  # pages of their own
        table[b, key // page] = pages + i
        vc[pages + i, key % page, :, i] = math.inf
    for b, key in lost:
        table[b, key // page] = pages + len(odd) + 5
    T = sum(news)
    q = _randn(g, T, H, D, dtype=dtype)
    args = [t.to(gpu) for t in (q, kc, vc, table)] + [torch.tensor(lens, device=gpu), _cu(news, gpu)]
    got = svdmlp.chunk_attention(*args)
    assert torch.equal(got.view(torch.int16 if dtype == BF else torch.int32), svdmlp.chunk_attention(*args).view(torch.int16 if dtype == BF else torch.int32))
    got = got.cpu()
    for b, some in rows:
        keys = torch.arange(lens[b])
        at = table[b].long()[keys // page]
        there = (at >= 0) & (at < pages + len(odd))
        keys, at = keys[there], (at * page + keys % page)[there]
        some = torch.tensor(some)
        seen = keys[None] <= (lens[b] - news[b] + some)[:, None]
        r = sum(news[:b]) + some
        for h in heads:
            k, v = kc.flatten(0, 1)[at, h // (H // K)], vc.flatten(0, 1)[at, h // (H // K)]
            out, tol = _attend(q[r, h], k, v, seen, 1 / math.sqrt(D), dtype)
            mine = got[r, h]
            for i, (bo, key) in enumerate(odd):
                if bo == b:
                    sees = key <= lens[b] - news[b] + some
                    assert (mine[sees, i] == math.inf).all() and not torch.isinf(mine[~sees, i]).any()
                    mine[sees, i], out[sees, i] = 0, 0.0
            _close(mine, out, tol)


@pytest.mark.parametrize("dtype,D", [(BF, 256), (BF, 136), (F32, 136), (F32, 256)])
def test_segments_of_tiles_of_128_rows(gpu, dtype, D):
    """One-token pages: segments of 2016 keys; 520 tiles, of which 256 are blocks of their own."""
    B = 130
    lens, news = [4100 - 7 * (i % 5) for i in range(B)], [40] * B
    # a page lost in the first segment, in the second, in the third; infinities that some rows see, and all
    lost = [(0, 100), (1, 2500), (2, 4060), (3, 0), (3, 2015), (3, 2016)]
    odd = [(64, 4085 - 28), (65, 1000), (66, 2100), (2, 4080)]
    rows = [(b, [0, 1, 17, 31, 32, 39]) for b in (0, 1, 2, 3, 64, 65, 66, B - 1)]
    _check(gpu, dtype, lens, news, 8, 2, D, 1, 5000, 0, rows, (0, 7), lost, odd)


@pytest.mark.parametrize("D,page,H,K", [(128, 4, 32, 4), (96, 4, 32, 4), (64, 8, 16, 2)])
def test_segments_of_tiles_of_256_rows(gpu, D, page, H, K):
    """Segments of 255 tiles of 64 keys (pages of 4) or 511 (of 8); tiles that are blocks of their own, or pieces by themselves."""
    far = 4095 * page // 64 * 64  # keys of a segment
    n = 4200 if K == 4 else 4096 * 2
    lens, news = [2 * far + 4300, far + 4290], [n, n - 11]
    lost = [(0, far + 5000), (1, 77)]
    odd = [(0, 300), (1, lens[1] - 50), (1, far - 1)]
    rows = [(b, [0, 1, 500, 2047, 2048, news[b] - 51, news[b] - 50, news[b] - 2, news[b] - 1]) for b in range(2)]
    _check(gpu, BF, lens, news, H, K, D, page, 3000, 0, rows, (0, H - 1), lost, odd)


@pytest.mark.parametrize("dtype,D,news", [(BF, 64, [3, 1]), (BF, 64, [700, 300]), (BF, 136, [200, 90]), (F32, 64, [5, 90]), (F32, 136, [40, 2])])
def test_units_of_several_keys(gpu, dtype, D, news):
    """A table of 65536 pages of 32752 tokens, of which the sequences have three."""
    lens = [70001, 40000]
    rows = [(b, sorted({0, n // 2, n - 1})) for b, n in enumerate(news)]
    _check(gpu, dtype, lens, news, 4, 2, D, 32752, 3, 65536, rows, (0, 3))
