"""Experiment kernels that are not launched in any build."""
import glob
import os
import re

import pytest

from pytorch_distributed_matmul_benchmark_amd.ops import gemm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("built", [False, True])
@pytest.mark.parametrize("arm", ["x_f32_w4s", "diag_f32_w4s_dbg", 91, 96])
def test_kernels_that_hung_are_refused(monkeypatch, arm, built):
    monkeypatch.setattr(gemm, "experiments_built", lambda: built)
    with pytest.raises(ValueError, match="not launched"):
        gemm._kid(arm)


def test_nothing_launches_them():
    """Neither a script nor the library: no launch of the kernel's function, no call by its name."""
    for pattern in ("*.py", "scripts/**/*.py", "scripts/**/*.sh", "pytorch_distributed_matmul_benchmark_amd/**/*.*"):
        for f in glob.glob(os.path.join(ROOT, pattern), recursive=True):
            if f.endswith((".py", ".sh", ".hip", ".cpp", ".h")) and not f.endswith(os.path.join("ops", "gemm.py")):
                with open(f, errors="replace") as fh:
                    text = fh.read()
                assert not re.search(r"x_f32_w4s|diag_f32_w4s_dbg|LaunchKernelGGL\([^;]*gemm_f32_w4s", text), f
