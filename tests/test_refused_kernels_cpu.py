"""Experiment kernels that are not launched in any build."""
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
    for folder, _, files in os.walk(ROOT):
        if os.path.relpath(folder, ROOT).split(os.sep)[0] in (".git", "_work", "gpurun_out"):
            continue
        for f in files:
            if f.endswith((".py", ".sh", ".hip", ".cpp", ".h")) and f not in ("test_refused_kernels_cpu.py",
                                                                              "test_gemm_gpu.py", "gemm.py"):
                with open(os.path.join(folder, f), errors="replace") as fh:
                    text = fh.read()
                assert not re.search(r"x_f32_w4s|diag_f32_w4s_dbg|LaunchKernelGGL\([^;]*gemm_f32_w4s", text), f
