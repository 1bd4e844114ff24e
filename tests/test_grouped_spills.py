"""Registers of the grouped and 4-bit kernels that did not fit (CPU only: hipcc cross-compiles)."""
import re

import pytest
from asm_cache import HIPCC, gfx950_asm

pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")


@pytest.mark.parametrize("src", ["grouped.hip", "grouped_w4.hip", "int4.hip"])
def test_spills(src):
    """Vector registers never; scalar ones, into lanes of a vector register, only in the large tiles' kernels, whose
    loads keep the wait states such a register needs (test_grouped_asm.test_hazards)."""
    found = re.findall(r"\.name:\s+(\S+)\s(?:.*\n)*?\s+\.sgpr_spill_count:\s+(\d+)\s(?:.*\n)*?\s+\.vgpr_spill_count:\s+(\d+)",
                       gfx950_asm(src))
    assert len(found) == len(re.findall(r"\.amdhsa_kernel ", gfx950_asm(src)))
    for name, scalar, vector in found:
        assert int(vector) == 0, name
        assert int(scalar) <= (47 if "gemm_grouped_w4" in name else 0), (name, scalar)
