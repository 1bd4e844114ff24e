"""Compute ops: hand-written gfx950 MFMA GEMM kernels (``csrc/``) + bindings."""
from .autograd import native_grouped_matmul, native_matmul  # noqa: F401
from .gemm import bench_matmul, bmm, kernel_for, matmul  # noqa: F401
from .grouped import grouped_matmul, grouped_weight_grad  # noqa: F401
from .int4 import int4_dequantize, int4_matmul, int4_quantize  # noqa: F401
