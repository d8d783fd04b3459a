"""Bounds of chunks that run backwards or overlap: a row is of the first sequence that has it, and the others get none."""

import math

import pytest
import torch

import svdmlp
from test_gpu_chunk import _ref
from test_gpu_decoder import BF, F32, _close, _gen, _pages, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,H,K,D", [(BF, 4, 1, 64), (BF, 32, 4, 128), (BF, 8, 2, 256), (F32, 4, 1, 64), (F32, 4, 2, 136)])
@pytest.mark.parametrize("bounds,owners", [
    ([0, 50, 10, 50], [(0, 0, 50)]), ([3, 20, 3, 40], [(0, 3, 20), (2, 20, 40)]), ([30, 10, 45, 45], [(1, 10, 45)]), ([50, 0, 0, 0], []),
    ([0, 50] * 40, [(0, 0, 50)]), ([0, 0, 7] + [5, 9] * 45, [(1, 0, 7), (3, 7, 9)])])
def test_rows_are_of_the_first_sequence(gpu, dtype, H, K, D, bounds, owners):
    """owners: (sequence, its first row, behind its last).  New tokens of a sequence are those that it has left."""
    g = _gen(D + len(bounds))
    B, T = len(bounds) - 1, 60
    lens = [900 - 3 * (b % 50) for b in range(B)]
    table, pages = _pages(g, lens[:3], 16)
    table = table[torch.arange(B) % 3]
    lens = [min(n, lens[b % 3]) for b, n in enumerate(lens)]
    q, kc, vc = _randn(g, T, H, D, dtype=dtype), _randn(g, pages, 16, K, D, dtype=dtype), _randn(g, pages, 16, K, D, dtype=dtype)
    out = torch.full((T, H, D), 7.0, dtype=dtype, device=gpu)
    svdmlp.chunk_attention(*(t.to(gpu) for t in (q, kc, vc, table)), torch.tensor(lens, device=gpu), torch.tensor(bounds, device=gpu), out=out)
    untouched = torch.ones(T, dtype=torch.bool)
    for b, first, behind in owners:
        want, tol = _ref(q[first:behind], kc, vc, table[b:b + 1], [lens[b]], [behind - first], 1 / math.sqrt(D), heads=(0, H - 1))
        _close(out[first:behind][:, [0, H - 1]], want, tol)
        untouched[first:behind] = False
    assert (out.cpu()[untouched] == 7).all()
