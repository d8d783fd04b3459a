"""The books of sequences whose layers refuse a call, without a device."""

import pytest
import torch

from svdmlp import e2e_block
from test_pages_host import _Books


class _Pool(_Books):
    def table(self, sequences):
        self.asked = list(sequences)
        return super().table(self.asked)


class _Model(e2e_block.SequenceModel):
    """Its layers refuse rows that are not 8 values."""

    def __init__(self):
        self.pool, self.calls = _Pool(torch.zeros(2, 8, 4, 1, 2)), []

    def _layers(self, x, positions, slots, attend):
        self.calls.append((positions.tolist(), slots.tolist()))
        if x.shape[1] != 8:
            raise ValueError("rows of 8 values")
        return x


def test_refused_rows_leave_the_sequences():
    model = _Model()
    a, b = model.pool.add(), model.pool.add()
    model.step(torch.zeros(7, 8), [a, b], [5, 2])
    free = model.pool.free_pages
    for n in (1, 9):
        with pytest.raises(ValueError, match="8 values"):
            model.step(torch.zeros(n + 1, 6), [b, a], [n, 1])
        with pytest.raises(ValueError, match="8 values"):
            model.verify(torch.zeros(2, n, 6), [a, b], torch.eye(n, dtype=torch.bool))
        assert (model.pool.length(a), model.pool.length(b), model.pool.free_pages) == (5, 2, free)
    model.step(torch.zeros(2, 8), [a, b], [1, 1])
    assert model.calls[-1] == ([5, 2], [5, 10]) and (model.pool.length(a), model.pool.length(b)) == (6, 3)


def test_sequences_from_an_iterator():
    """Both the room and the block table are theirs."""
    model = _Model()
    a, b = model.pool.add(), model.pool.add()
    model.step(torch.zeros(7, 8), (s for s in (b, a)), (t for t in (5, 2)))
    assert model.pool.asked == [b, a] and (model.pool.length(a), model.pool.length(b)) == (2, 5)


def test_captured_stream_of_the_pools_device(monkeypatch):
    """The stream that counts is the pool's device's, whichever device is the current one."""
    now = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.was, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.was

    captured = set()
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] in captured)
    pool = _Books(torch.zeros(2, 8, 4, 1, 2))
    pool._tensor = lambda values, dtype: torch.tensor(values, dtype=dtype)
    pool.device = torch.device("cuda", 1)
    a = pool.add()
    captured.add(0)  # a graph of another device
    pool.reserve([a], [3])
    captured.add(1)
    for current in (0, 1):
        now[0] = current
        for call in (lambda: pool.reserve([a], [1]), lambda: pool.table([a]), pool.compact):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    captured.remove(0)
    now[0] = 0
    with pytest.raises(RuntimeError, match="captured"):
        pool.table([a])
    assert pool.length(a) == 3
