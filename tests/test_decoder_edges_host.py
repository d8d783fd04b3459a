"""The host's part of the operators around the MLP block where a call is
unusual: another device than the current one, large plans."""

import contextlib

import torch

from svdmlp import decoder


def test_partials_of_a_capture_on_another_device(monkeypatch):
    """A call captured on a device that is not the current one gets room of its own, not that of the stream's eager calls."""
    now = [0]

    @contextlib.contextmanager
    def device(index):
        before, now[0] = now[0], index
        yield
        now[0] = before

    empty, zeros = torch.empty, torch.zeros
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == 1)  # device 1's stream is
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))
    monkeypatch.setattr(torch, "zeros", lambda n, dtype, device: zeros(n, dtype=dtype))
    monkeypatch.setattr(decoder, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(decoder, "_PARTIALS_CACHE", {})
    a, b = decoder._partials(1, 64, 4), decoder._partials(1, 64, 4)
    assert a[0] is not b[0] and a[1] is not b[1] and not decoder._PARTIALS_CACHE and now == [0]
    a, b = decoder._partials(0, 64, 4), decoder._partials(0, 64, 4)
    assert a[0] is b[0] and a[1] is b[1] and len(decoder._PARTIALS_CACHE) == 1
