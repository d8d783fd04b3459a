"""Sequences' books where the layers refuse a call, and what the served step's sequences hold."""

import argparse

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


@pytest.mark.parametrize("S,chunk", [(64, 40), (70, 100)])
def test_served_sequences_have_pages_of_their_own(gpu, monkeypatch, S, chunk):
    """The timed step reads as many contexts as it has sequences: no page is of two of them, and each holds the prompt's rows."""
    models, lengths = [], []

    class Model(e2e_block.SequenceModel):
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            models.append(self)

        def step(self, x, sequences, tokens):
            lengths.append([self.pool.length(s) for s in sequences])
            self.last = sequences
            return super().step(x, sequences, tokens)

    monkeypatch.setattr(e2e_block, "SequenceModel", Model)
    weights, rows = _weights(gpu, 4, False)
    args = argparse.Namespace(warmup=1, repeats=2, serve_sequences=3, serve_chunk=chunk)
    rec = e2e_block._serve(torch, weights, HEADS, KV, rows(S), args, None)
    (model,) = models
    assert lengths[-3:] == [[S] * 4] * 3 and rec["sequences"] == 3
    table = model.pool.table(model.last)[0].cpu()
    used = table[table >= 0].tolist()
    assert len(set(used)) == len(used) == 4 * -(-S // model.PAGE)
    last = table[:, -1].tolist()
    held = S - (table.shape[1] - 1) * model.PAGE
    for page in last[1:]:
        assert torch.equal(model.caches[:, :, page, :held], model.caches[:, :, last[0], :held])
    full = table[:, 0].tolist()
    for page in full[1:]:
        assert torch.equal(model.caches[:, :, page], model.caches[:, :, full[0]])
