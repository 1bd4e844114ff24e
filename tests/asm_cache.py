"""One gfx950 compile per (source, build flavour) per test process, shared by
the static assembly checks (test_kernel_asm.py, test_mfma_hazards.py), with the
flags that the library itself is compiled with."""
import functools
import os
import shutil
import subprocess

from pytorch_distributed_matmul_benchmark_amd.ops.build import kernel_flags

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "pytorch_distributed_matmul_benchmark_amd", "ops", "csrc")
HIPCC = "/opt/rocm/bin/hipcc" if os.path.exists("/opt/rocm/bin/hipcc") else shutil.which("hipcc")


def gfx950_asm(src: str, experiments: bool = False) -> str:
    """The device assembly (.s text) of ``csrc/src`` (default build, or with the
    A/B experiment kernels)."""
    return _compile(src, experiments)


@functools.lru_cache(maxsize=None)
def _compile(src: str, experiments: bool) -> str:
    defs = ["-DPDMB_EXPERIMENTS=1"] if experiments else []
    lang = ["-x", "hip"] if src.endswith(".cpp") else []
    r = subprocess.run([HIPCC, *kernel_flags(), *defs, *lang, "-S", "--cuda-device-only", os.path.join(CSRC, src), "-o", "-"],
                       check=True, capture_output=True, text=True, timeout=900)
    return r.stdout
