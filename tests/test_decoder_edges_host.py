"""The host's part of the operators around the MLP block where a call is
unusual: another device than the current one, large plans."""

import contextlib
import math
import random

import torch

from svdmlp import _lib, decoder


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


def test_cache_attention_workspace_is_bounded():
    """Partial sums take at most a quarter of the keys and values that the table has room for (D + 2 values a row for D), or
    what four waves of 32 rows on each SIMD of 256 CUs write; and in either case up to one chunk a sequence more."""
    lib, rng = _lib.load(), random.Random(5)
    cases = [(96, 64, 16, 1363, 8, 1, 256, 1), (24, 64, 16, 1363, 8, 1, 256, 0), (63, 64, 16, 1500, 8, 1, 256, 1), (256, 8, 16, 2048, 32, 8, 128, 1)]
    for _ in range(20000):
        heads, kv, D = rng.choice(((32, 8, 128), (64, 8, 128), (24, 8, 128), (16, 16, 64), (14, 2, 64), (12, 4, 96), (8, 1, 256), (7, 7, 80)))
        B, page = round(math.exp(rng.uniform(0, math.log(400)))), rng.choice((16, 32, 48, 64))
        n, width = rng.choice((1, rng.randint(2, 64))), -(-round(math.exp(rng.uniform(0, math.log(32768)))) // page)
        cases.append((B, n, page, width, heads, kv, D, rng.randint(0, 1)))
    for B, n, page, width, heads, kv, D, dtype in cases:
        got = lib.svdmlp_cache_attention_workspace_bytes(B, n, page, width, heads, kv, D, dtype, None)
        room = 2 * B * page * width * kv * D * (2 if dtype == _lib.SVDMLP_BF16 else 4)
        sums = 4 * (D + 2)
        bound = max(room * (D + 2) // D // 4, 4 * 4 * 256 * 32 * sums) + B * n * heads * sums
        assert got <= bound, (B, n, page, width, heads, kv, D, dtype, got, bound)
