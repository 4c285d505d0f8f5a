"""The linear head's losses on tensors of CUDA carriers: autograd, the one-call forms and the module classes, for
both losses, reductions and types.  Each check runs in a process of its own (linear_head_tensors.py), against the host
framework or, where that is not installed, a small stand-in for its tensors."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("check", ["autograd", "one_call", "upstream_placements", "teacher_shapes", "devices"])
def test_tensors(check):
    script = Path(__file__).resolve().parent / "linear_head_tensors.py"
    out = subprocess.run([sys.executable, str(script), check], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
