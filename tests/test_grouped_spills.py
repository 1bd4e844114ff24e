"""Registers of the grouped and 4-bit kernels that did not fit (CPU only: hipcc cross-compiles)."""
import re

import pytest
from asm_cache import HIPCC
from test_grouped_asm import SOURCES, _asm

pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")


@pytest.mark.parametrize("src", SOURCES)
def test_spills(src):
    """Vector registers never; scalar ones, into lanes of a vector register, only in the large tiles' kernels, whose
    loads keep the wait states such a register needs (test_grouped_asm.test_hazards)."""
    found = re.findall(r"\.name:\s+(\S+)\s(?:.*\n)*?\s+\.sgpr_spill_count:\s+(\d+)\s(?:.*\n)*?\s+\.vgpr_spill_count:\s+(\d+)",
                       _asm(src))
    assert len(found) == len(re.findall(r"\.amdhsa_kernel ", _asm(src)))
    for name, scalar, vector in found:
        assert int(vector) == 0, name
        assert int(scalar) <= (47 if "gemm_grouped_w4" in name else 0), (name, scalar)
