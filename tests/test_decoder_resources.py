"""Register counts of the kernels around the MLP block (attention, rotary
positions, residual norms), as of the build they were timed on: most attention
kernels sit just under a count that costs a wave a SIMD.  The counts
(``tests/decoder_registers_baseline.json``) are rewritten on purpose, with the
timing that justifies it."""

import json
from pathlib import Path

from test_kernel_resources import SLACK, _report

BASELINE = Path(__file__).resolve().parent / "decoder_registers_baseline.json"
KERNELS = ("cache_kernel", "cache_join_kernel", "prompt_kernel", "prompt_pipe_kernel", "rope_kernel", "residual_norm_kernel")


def _ours():
    return {n: {"VGPRs": int(r["VGPRs"]), "AGPRs": int(r["AGPRs"])} for n, r in _report().items() if any(k in n for k in KERNELS)}


def test_every_kernel_has_its_counts():
    assert sorted(_ours()) == sorted(json.loads(BASELINE.read_text()))


def test_registers_within_the_counts():
    now = _ours()
    grown = {n: (b, now[n]) for n, b in json.loads(BASELINE.read_text()).items() if any(now[n][k] > b[k] + SLACK for k in b)}
    assert not grown, f"kernels above their recorded registers (recorded, now): {grown}"
