"""The static checks read the code that ships: compiled with the build's own flags (CPU only)."""
import re

import pytest
from asm_cache import HIPCC, gfx950_asm

from pytorch_distributed_matmul_benchmark_amd.ops import build

pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")


def test_checked_code_is_compiled_as_the_library_is():
    """reduce.hip holds packed fp32 arithmetic where the build's flags do not forbid it."""
    assert set(build.NO_PACKED_F32) <= set(build.kernel_flags())
    assert not re.search(r"v_pk_(add|mul|fma)_f32", gfx950_asm("reduce.hip"))
