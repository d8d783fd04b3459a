"""Sequences' books where the layers refuse a call."""

import pytest
import torch

from svdmlp import e2e_block
from test_gpu_sequences import HEADS, KV, _weights

pytestmark = pytest.mark.gpu


def test_refused_rows_leave_the_sequences(gpu):
    """Rows of another width or type, or that ask for a gradient: the sequences stay as long as they were, and go on as if nothing had been asked."""
    weights, rows = _weights(gpu, 2, False)
    model, other = (e2e_block.SequenceModel(weights, HEADS, KV, 8) for _ in range(2))
    x = rows(75)
    seqs = [[m.pool.add(), m.pool.add()] for m in (model, other)]
    for m, (a, b) in zip((model, other), seqs):
        m.step(x[:70], [a, b], [60, 10])
    a, b = seqs[0]
    free = model.pool.free_pages
    for bad in (x[:70, :-16].contiguous(), x[:70].double(), x[:70].float().requires_grad_(), x[:70].cpu()):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            model.step(bad, [a, b], [1, 69])
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            model.verify(bad.view(2, 35, -1), [a, b], torch.eye(35, dtype=torch.bool, device=bad.device))
        assert (model.pool.length(a), model.pool.length(b), model.pool.free_pages) == (60, 10, free)
    assert torch.equal(model.step(x[70:], [a, b], [2, 3]), other.step(x[70:], seqs[1], [2, 3]))
