"""Registers and waves of the kernels for sequences side by side (attention over
chunks, head norms, moves within a cache), as of the build they were timed on
(``tests/sequence_registers_baseline.json``, rewritten on purpose, with the timing
that justifies it): blocks a CU are planned by them, and the head norms sit on
the last count that leaves seven waves a SIMD."""

import json
from pathlib import Path

from test_kernel_resources import SLACK, _report

BASELINE = Path(__file__).resolve().parent / "sequence_registers_baseline.json"
KERNELS = ("chunk_wave_kernel", "chunk_share_kernel", "chunk_pipe_kernel", "chunk_join_kernel", "head_norm_turn_kernel", "page_copy_kernel",
           "draft_keep_kernel")
WAVES = "Occupancy [waves/SIMD]"


def _ours():
    return {n: {k: int(r[k]) for k in ("VGPRs", "AGPRs", WAVES)} for n, r in _report().items() if any(k in n for k in KERNELS)}


def test_every_kernel_has_its_counts():
    assert sorted(_ours()) == sorted(json.loads(BASELINE.read_text()))
    assert all(any(k in n for n in _ours()) for k in KERNELS)


def test_registers_and_waves_within_the_counts():
    now = _ours()
    worse = {n: (b, now[n]) for n, b in json.loads(BASELINE.read_text()).items()
             if now[n][WAVES] < b[WAVES] or any(now[n][k] > b[k] + SLACK for k in ("VGPRs", "AGPRs"))}
    assert not worse, f"kernels above their recorded registers, or below their waves (recorded, now): {worse}"
