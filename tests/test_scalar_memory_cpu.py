"""Static check (CPU): the kernels use scalar memory to read only. Every scalar instruction whose name speaks
of memory has to be one of the reads below, in each source of the library."""
import re

import pytest
from asm_cache import HIPCC, gfx950_asm
from test_grouped_asm import SOURCES, _asm

from pytorch_distributed_matmul_benchmark_amd.ops import build

READS = re.compile(r"s_(buffer_)?load_(dword|dwordx(2|3|4|8|16)|[bu](8|16|32|64|96|128|256|512)|[iu](8|16))|s_mem(real)?time")


def others(asm: str):
    names = set(re.findall(r"^\s*(s_\w+)", asm, re.M))
    return sorted(n for n in names if re.search("load|store|atomic|cache|scratch|buffer|mem", n)
                  and not READS.fullmatch(n))


def test_the_check_sees_a_write():
    assert others("\ts_load_dwordx4 s[0:3], s[4:5], 0x0\n\ts_" + "store_dword s0, s[2:3], 0x0") == ["s_" + "store_dword"]


@pytest.mark.skipif(HIPCC is None, reason="hipcc not available")
@pytest.mark.parametrize("src", build.HIP_SOURCES)
def test_scalar_memory_is_only_read(src):
    asm = _asm(src) if src in SOURCES else gfx950_asm(src)
    assert "s_load_" in asm
    assert not others(asm)
