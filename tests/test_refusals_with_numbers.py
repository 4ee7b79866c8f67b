"""Refusals whose message holds a number end in an exception, not in the end of the process (each in a process of its own)."""

import subprocess
import sys

import pytest

CASES = {
    "too many logical experts: 2400000": "native.PlannerEngine(1, 8, 3, 300000, 1, 0)",
    "malformed IPC handle from rank 1": "e = native.MoeEngine(256, 128, 2, 2, 0, 1, 128, 128, 0); e.alloc(); e.open([b'', b'short'])",
    "workload must have 64 entries, got 63": "planner().solve_probs(torch.zeros(63, dtype=torch.int32, device='cuda'), avail)",
    "indices must live on cuda:0": "planner()._engine.count_idx(torch.zeros(8, 2, dtype=torch.int64), 4)",
}
START = """
import torch
from lplb_b200 import Planner, _native, cube
native = _native.load()
def planner():
    return Planner(cube(), 64 + 16, 64, 8, device="cuda")
avail = torch.zeros(1, dtype=torch.int32, device="cuda") if torch.cuda.is_available() else None
try:
    %s
except (RuntimeError, ValueError) as error:
    print("refused:", error)
"""


def _refused(words):
    run = subprocess.run([sys.executable, "-c", START % CASES[words]], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, (run.returncode, run.stderr[-2000:])
    assert "refused: " in run.stdout and words in run.stdout, run.stdout + run.stderr[-2000:]


def test_a_number_in_a_refusal_without_a_device():
    _refused("too many logical experts: 2400000")


@pytest.mark.gpu
@pytest.mark.parametrize("words", [w for w in CASES if not w.startswith("too many")])
def test_a_number_in_a_refusal(words):
    _refused(words)
