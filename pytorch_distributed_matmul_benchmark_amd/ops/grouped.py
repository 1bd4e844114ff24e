"""Matrix products grouped by expert: ``grouped_matmul`` and the gradient of its
weights, ``grouped_weight_grad`` (differentiable: ``autograd.native_grouped_matmul``).

``x`` holds rows already ordered by expert; ``ends[e]`` is where expert e's rows
end, so that its rows are ``x[ends[e-1]:ends[e]]`` (``ends[-1]`` meaning 0) — the
running sum of the rows each expert has. ``ends`` stays on the GPU: no call
waits for it on the host, so the sizes may change between replays of a captured
graph. Experts may have no rows, and rows may be left behind the last expert's
(a padded batch). ``ends`` must not decrease; values outside [0, T] are held
inside it.

GPU tensors run on ``csrc/grouped.hip`` (bf16 / fp16 with fp32 sums, exact
fp32); CPU tensors use a loop of ``torch.matmul``. As in ``gemm``, a call is
enqueued on the current stream of the tensors' device, and ``out`` must not
overlap the operands.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native
from .gemm import SUPPORTED_DTYPES, _prep


def _native_call(name: str, x, *args):
    """The kernel's result, or None where an argument is not as the kernel takes it (the
    caller then finds out why)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        return None
    try:
        return getattr(_native.load(), name)(x, *args)
    except TypeError:  # an argument that is no tensor
        return None


def _must(res: Optional[torch.Tensor], out: Optional[torch.Tensor], op: str) -> torch.Tensor:
    # (all else that a binding turns down has been checked or copied)
    if res is None:
        raise ValueError(f"{op}: sizes up to 2^30 only" if out is None else
                         f"{op}: out must have contiguous rows that do not overlap, and sizes up to 2^30")
    return res


def _check_ends(ends: torch.Tensor, x: torch.Tensor, experts: int, op: str) -> None:
    if not isinstance(ends, torch.Tensor) or ends.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{op}: ends must be an int32 or int64 tensor")
    if ends.dim() != 1 or ends.shape[0] != experts:
        raise ValueError(f"{op}: ends must have one value for each of the {experts} experts, "
                         f"got shape {tuple(ends.shape)}")
    if ends.device != x.device:
        raise ValueError(f"{op}: ends is on {ends.device}, the rows on {x.device}")


def _check_dtype(t: torch.Tensor, op: str) -> None:
    if t.dtype not in SUPPORTED_DTYPES:
        raise TypeError(f"{op}: unsupported dtype {t.dtype}")


def _check_out(out: torch.Tensor, shape, like: torch.Tensor, op: str) -> None:
    if tuple(out.shape) != tuple(shape) or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{op}: out must be {tuple(shape)} {like.dtype} on {like.device}, got "
                         f"{tuple(out.shape)} {out.dtype} on {out.device}")
    if torch.is_grad_enabled() and out.requires_grad:
        raise RuntimeError(f"{op} records no gradient: out must not require one")
    _no_tangent(op, out)


def _no_grad(op: str, instead: str, *ts: torch.Tensor) -> None:
    # a result without a graph or a tangent would drop the gradients silently
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise RuntimeError(f"{op} records no gradient: {instead}")
    _no_tangent(op, *ts)


def _no_tangent(op: str, *ts: torch.Tensor) -> None:
    if any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError(f"{op} has no forward-mode derivative")


def _ranges(ends: torch.Tensor, rows: int):
    """The row ranges as the kernels take them (host copy; CPU path only)."""
    at = 0
    for e, end in enumerate(ends.tolist()):
        lo, hi = at, max(0, min(int(end), rows))
        yield e, lo, max(lo, hi)
        at = hi


def _prep_weight(w: torch.Tensor) -> torch.Tensor:
    """``w`` as the kernels take it: rows or columns contiguous and not overlapping."""
    K, N = w.shape[1:]
    if (N <= 1 or w.stride(2) == 1) and (K <= 1 or w.stride(1) >= N):
        return w
    if N > 1 and w.stride(2) != 1 and (K <= 1 or w.stride(1) == 1) and w.stride(2) >= K:
        return w
    return w.contiguous()


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[r] = x[r] @ w[e]`` for the rows r of expert e.

    ``x`` [T, K], ``w`` [E, K, N] of the same dtype (float32, float16, bfloat16),
    ``ends`` [E]; returns [T, N]. ``w`` may be row- or column-major (a transposed
    view of [E, N, K] weights is read in place). Rows behind the last expert's
    are zero in a fresh result and left as they were in ``out``."""
    op = "grouped_matmul"
    res = _native_call("grouped_rows", x, w, ends, out)
    if res is not None:
        return res
    if x.dim() != 2 or w.dim() != 3:
        raise ValueError(f"{op}: x must be 2-D and w 3-D")
    if x.shape[1] != w.shape[1]:
        raise ValueError(f"{op}: shape mismatch {tuple(x.shape)} @ {tuple(w.shape)}")
    if w.shape[0] < 1:
        raise ValueError(f"{op}: needs at least one expert")
    _check_dtype(x, op)
    if w.dtype != x.dtype:
        raise TypeError(f"{op}: x is {x.dtype}, w is {w.dtype}")
    if w.device != x.device:
        raise ValueError(f"{op}: w is on {w.device}, x on {x.device}")
    _check_ends(ends, x, w.shape[0], op)
    T, N = x.shape[0], w.shape[2]
    if out is not None:
        _check_out(out, (T, N), x, op)
    _no_grad(op, "use autograd.native_grouped_matmul", x, w)
    if x.device.type != "cuda":
        res = x.new_zeros(T, N) if out is None else out
        for e, lo, hi in _ranges(ends, T):
            if hi > lo:
                res[lo:hi] = torch.matmul(x[lo:hi], w[e])
        return res
    return _must(_native_call("grouped_rows", _prep(x), _prep_weight(w), ends.contiguous(), out), out, op)


def grouped_weight_grad(x: torch.Tensor, dy: torch.Tensor, ends: torch.Tensor,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[e] = x_e^T @ dy_e`` over the rows of expert e: the gradient of
    ``grouped_matmul``'s weights. ``x`` [T, K], ``dy`` [T, N] of one dtype, ``ends``
    [E]; returns [E, K, N], zeros for an expert without rows. The sums are fp32
    and rounded once."""
    op = "grouped_weight_grad"
    res = _native_call("grouped_reduce", x, dy, ends, out)
    if res is not None:
        return res
    if x.dim() != 2 or dy.dim() != 2:
        raise ValueError(f"{op}: x and dy must be 2-D")
    if x.shape[0] != dy.shape[0]:
        raise ValueError(f"{op}: {x.shape[0]} rows of x, {dy.shape[0]} of dy")
    _check_dtype(x, op)
    if dy.dtype != x.dtype:
        raise TypeError(f"{op}: x is {x.dtype}, dy is {dy.dtype}")
    if dy.device != x.device:
        raise ValueError(f"{op}: dy is on {dy.device}, x on {x.device}")
    if not isinstance(ends, torch.Tensor) or ends.dim() != 1 or ends.shape[0] < 1:
        raise ValueError(f"{op}: ends must be a 1-D tensor with one value for each expert")
    _check_ends(ends, x, ends.shape[0], op)
    shape = (ends.shape[0], x.shape[1], dy.shape[1])
    if out is not None:
        _check_out(out, shape, x, op)
    _no_grad(op, "call it under torch.no_grad()", x, dy)
    if x.device.type != "cuda":
        res = x.new_zeros(shape) if out is None else out
        for e, lo, hi in _ranges(ends, x.shape[0]):
            res[e] = torch.matmul(x[lo:hi].t(), dy[lo:hi])
        return res
    return _must(_native_call("grouped_reduce", _prep(x), _prep(dy), ends.contiguous(), out), out, op)
