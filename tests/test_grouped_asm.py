"""Static checks of the grouped and 4-bit kernels' gfx950 code, compiled with the build's own
flags (CPU only: hipcc cross-compiles)."""
import functools
import os
import re
import subprocess

import pytest
import test_mfma_hazards as mfma
import test_sgpr_vmem_hazard as vmem
from asm_cache import CSRC, HIPCC
from test_vmcnt_bound import MAX, peak_outstanding

from pytorch_distributed_matmul_benchmark_amd.ops.build import NO_PACKED_F32

pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")
SOURCES = ["grouped.hip", "grouped_w4.hip", "int4.hip"]


@functools.lru_cache(maxsize=None)
def _asm(src):
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", f"-I{CSRC}", *NO_PACKED_F32, "-S",
                        "--cuda-device-only", os.path.join(CSRC, src), "-o", "-"],
                       check=True, capture_output=True, text=True, timeout=900)
    return r.stdout


@pytest.mark.parametrize("src", SOURCES)
def test_no_packed_fp32_and_no_spills(src):
    s = _asm(src)
    assert not re.search(r"v_pk_(add|mul|fma)_f32", s)
    kernels = re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", s, re.S)
    assert kernels
    for name, kd in kernels:
        assert re.search(r"\.amdhsa_private_segment_fixed_size (\d+)", kd).group(1) == "0", name
        assert int(re.search(r"\.amdhsa_group_segment_fixed_size (\d+)", kd).group(1)) <= 160 * 1024, name


@pytest.mark.parametrize("src", SOURCES)
def test_hazards(src):
    for name, body in mfma._kernels(_asm(src)):
        assert not mfma.hazards(body), name
        assert not vmem.hazards(body), name
        if src == "grouped_w4.hip":  # MFMAs in inline asm, which hipcc does not pad
            assert not mfma.read_hazards(body), name


def test_counted_waits_stay_countable():
    """grouped_w4's K-loop waits on counts of vector-memory operations in flight, at most 63."""
    for name, body in mfma._kernels(_asm("grouped_w4.hip")):
        first = re.search(r"buffer_load_dwordx4 .* lds", body).start()  # all before it has been waited for
        assert "s_waitcnt vmcnt(0)" in body[:first]
        peak = peak_outstanding(body[first:body.rfind("s_waitcnt vmcnt(0)")])
        assert 48 < peak <= MAX, (name, peak)
