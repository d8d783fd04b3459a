"""Attention over chunks of the longest sequence that it takes, 2^31 - 2^17 tokens: a table
that names one page over and over, and another one at its end.  Queries are zero,
so every weight is 1, and values are 0 or 1: a block's sums are whole numbers below
2^24, exact in fp32, whatever their order.  Roundings are then those of joining up
to 768 pieces (three blocks on each of 256 CUs), one an addition of the weights and
of the values, each at most 2^-24 of the sum; of the inverse and the product, under
4 more; and of the result."""

import pytest
import torch

import svdmlp
from test_gpu_decoder import BF, F32, U, _cu, _gen

pytestmark = pytest.mark.gpu

PAGE, WIDTH, LAST = 32768, 65532, 100  # LAST: entries of the second page
LONGEST = PAGE * WIDTH


def _longest(gpu, dtype, H, D, n):
    assert LONGEST == 0x7ffe0000
    g = _gen(D + n)
    k = torch.zeros(2, PAGE, 1, D, dtype=dtype, device=gpu)
    v = torch.zeros(2, PAGE, 1, D, dtype=dtype)
    v[:, :, :, 1::2] = 1                                                     # every key counts in odd columns
    v[1, :, :, 0::2] = torch.randint(0, 2, (PAGE, 1, D // 2), generator=g).to(dtype)  # and in even ones the far ones do
    table = torch.zeros(1, WIDTH, dtype=torch.int32, device=gpu)
    table[:, -LAST:] = 1
    q = torch.zeros(n, H, D, dtype=dtype, device=gpu)
    got = svdmlp.chunk_attention(q, k, v.to(gpu), table, torch.tensor([LONGEST], device=gpu), _cu([n], gpu))
    rows = v[1, :, 0].double()
    upto = (LAST - 1) * rows.sum(0) + rows.cumsum(0)[PAGE - n:]              # token i sees all but the last n - 1 - i keys
    upto[:, 1::2] = (LONGEST - n + 1 + torch.arange(n, dtype=torch.float64))[:, None]
    want = (upto / (LONGEST - n + 1 + torch.arange(n, dtype=torch.float64))[:, None])[:, None].expand(n, H, D)
    off = ((got.double().cpu() - want).abs() / want).max()
    assert off <= (2 * 768 + 4) * 2.0 ** -24 + U[dtype], float(off)


@pytest.mark.parametrize("dtype,H,D,n", [(F32, 1, 136, 5), (BF, 2, 136, 150)])
def test_longest_sequence_by_tiles_of_128_rows(gpu, dtype, H, D, n):
    _longest(gpu, dtype, H, D, n)


def test_longest_sequence_by_tiles_of_256_rows(gpu):
    _longest(gpu, BF, 1, 128, 300)


@pytest.mark.parametrize("dtype,H,D,n", [(BF, 4, 64, 3), (BF, 2, 128, 9), (F32, 2, 64, 20)])
def test_longest_sequence_by_tiles_of_32_rows(gpu, dtype, H, D, n):
    _longest(gpu, dtype, H, D, n)
