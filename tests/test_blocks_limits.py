"""The block operators at and beyond the sizes that they document."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


def test_the_recurrences_sizes_are_answered_for_any_numbers():
    """0 beyond the limits, however far: asked in a process of its own, which has to end"""
    code = """
from envidr_amd.blocks import _bind
lib = _bind.lib()
for T, N, C in ((1 << 31, 1, 1), (1 << 44, 4, 4), (1 << 46, 4, 4), ((1 << 64) - 1, 4, 4), ((1 << 64) - 1, (1 << 32) - 1, (1 << 32) - 1), (8, 1 << 26, 4), (8, 2, (1 << 19) + 1)):
    assert lib.envidr_ray_recurrence_workspace_bytes(T, N, C) == 0 and lib.envidr_ray_recurrence_saved_floats(T, N, C) == 0, (T, N, C)
for T, N, C in (((1 << 31) - 1, 31 << 20, 1), ((1 << 31) - 1, 1, 1 << 19), (8, 2, 1 << 19), (0, 0, 1), (1, 1, 1)):
    big = lib.envidr_ray_recurrence_workspace_bytes(T, N, C), lib.envidr_ray_recurrence_saved_floats(T, N, C)
    assert (big[0] >= 4 * (T + N) and big[1] >= T * C // 8) if T else big == (0, 0), (T, N, C, big)
print("answered")
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=ROOT)
    assert run.returncode == 0 and "answered" in run.stdout, run.stderr
