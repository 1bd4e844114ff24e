"""``native_matmul`` and ``native_grouped_matmul``: the gfx950 MFMA products as
differentiable ops.

Forward ``C = A @ B`` and both backward GEMMs (``dA = dC @ Bᵀ``,
``dB = Aᵀ @ dC``) run on the native kernels; transposed operands are
materialised row-major first (the kernels take row-major NN operands with a
unit inner stride; the grouped products read a transposed weight in place). Lets the
benchmark GEMM drop into a training step (used by ``__graft_entry__.smoke``).
"""
from __future__ import annotations

import torch

from torch.autograd.function import once_differentiable

from . import gemm, grouped


class _NativeMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, A, B):
        ctx.save_for_backward(A, B)
        return gemm.matmul(A, B)

    @staticmethod
    def backward(ctx, dC):
        A, B = ctx.saved_tensors
        dC = dC.contiguous()
        dA = dB = None
        if ctx.needs_input_grad[0]:
            dA = gemm.matmul(dC, B.transpose(-1, -2).contiguous())
            if A.dim() == 2 and dA.dim() == 3:  # A broadcast over B's batch
                dA = dA.sum(0)
        if ctx.needs_input_grad[1]:
            if A.dim() == 3:
                dB = gemm.matmul(A.transpose(-1, -2).contiguous(), dC)
                if B.dim() == 2:
                    dB = dB.sum(0)
            else:
                dB = gemm.matmul(A.transpose(-1, -2).contiguous(), dC)
        return dA, dB


def native_matmul(A: torch.Tensor, B: torch.Tensor) -> torch.Tensor:
    return _NativeMatmul.apply(A, B)


class _NativeGroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, ends):
        ctx.save_for_backward(x, w, ends)
        return grouped.grouped_matmul(x, w, ends)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, ends = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = grouped.grouped_matmul(dy, w.transpose(1, 2), ends)
        if ctx.needs_input_grad[1]:
            if w.stride(2) != 1 and w.stride(1) == 1:  # column-major weights get a gradient laid out alike
                dw = grouped.grouped_weight_grad(dy, x, ends).transpose(1, 2)
            else:
                dw = grouped.grouped_weight_grad(x, dy, ends)
        return dx, dw, None


def native_grouped_matmul(x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """``grouped.grouped_matmul`` with gradients for ``x`` and ``w``: ``dx[r] = dy[r] @
    w[e]^T`` on the same kernel (the transposed weights are read in place) and
    ``dw[e] = x_e^T @ dy_e`` (``grouped.grouped_weight_grad``). Rows behind the last
    expert's, and experts without rows, get zero gradients. ``ends`` must not
    change between the forward and the backward pass. Under a stream capture an
    operand is refused that is, or was computed from, a leaf whose graph from the default
    stream is still alive."""
    res = grouped._native_call("grouped_node", x, w, ends)
    return _NativeGroupedMatmul.apply(x, w, ends) if res is None else res
