"""Products of a few rows with 4-bit weights: ``int4_quantize`` lays a weight out
once, ``int4_matmul`` multiplies by it (one weight, or one for each expert).

A weight [K, N] is held by column, as fp8's B operand is: ``q`` [N, K/2] uint8, two
values a byte, the even k in the low half; ``scale`` [N, K/G] in the rows' dtype
and ``zero`` [N, K/G] uint8 (0..15, higher bits are ignored; None: 8 everywhere) for
each group of G values of k:
``W[k, n] = scale[n, k // G] * (q[n, k] - zero[n, k // G])``. G is 32, 64 or a
multiple of 128, and divides K. Expert weights have a leading dimension [E, ...].

GPU tensors run on ``csrc/int4.hip``: the values are multiplied as whole numbers,
each group's fp32 sum is scaled in fp32, and the result is rounded once. They are
made for the rows of a serving batch (100 rows, 4096 x 8192: 22 us); from about a hundred
rows ``matmul`` with a weight kept as ``int4_dequantize`` returns it is faster. CPU
tensors use ``torch.matmul`` on the dequantised weight.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .gemm import _prep
from .grouped import _check_ends, _check_out, _must, _native_call, _no_grad, _ranges

INT4_DTYPES = (torch.float16, torch.bfloat16)
MAX_K = 1 << 23  # of GPU tensors: K, and the distance of two rows that are read in place


def _check_group(K: int, group: int, op: str) -> None:
    if group not in (32, 64) and (group < 128 or group % 128):
        raise ValueError(f"{op}: group of {group} (32, 64 or a multiple of 128 only)")
    if K < 1 or K % group:
        raise ValueError(f"{op}: K = {K} is not a multiple of the group, {group}")


def int4_quantize(w: torch.Tensor, group: int = 128, symmetric: bool = False
                  ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """4-bit copy of ``w`` [K, N] or [E, K, N] (float16 or bfloat16): ``(q, scale, zero)``.

    ``symmetric``: zero is None and the scale maps a group's largest magnitude to 7;
    otherwise a group's range, with 0 inside it, is mapped to 0..15. The scale is
    rounded to ``w``'s dtype before the values are, so a value is off by at most
    half a scale step where the range covers it."""
    op = "int4_quantize"
    if w.dim() not in (2, 3):
        raise ValueError(f"{op}: w must be 2-D or 3-D")
    if w.dtype not in INT4_DTYPES:
        raise TypeError(f"{op}: unsupported dtype {w.dtype}")
    _check_group(w.shape[-2], group, op)
    v = w.detach().transpose(-1, -2).float().unflatten(-1, (-1, group))  # [.., N, K/G, G]
    if symmetric:
        step = v.abs().amax(-1) / 7.0
    else:
        lo, hi = v.amin(-1).clamp(max=0.0), v.amax(-1).clamp(min=0.0)
        step = (hi - lo) / 15.0
    scale = step.to(w.dtype)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)  # an all-zero group
    s = scale.float().unsqueeze(-1)
    if symmetric:
        zero = None
        n = (v / s).round_() + 8.0
    else:
        zero = (-lo / scale.float()).round_().clamp_(0, 15)
        n = (v / s).round_() + zero.unsqueeze(-1)
        zero = zero.to(torch.uint8).contiguous()
    n = n.clamp_(0, 15).to(torch.uint8).flatten(-2)
    q = n[..., 0::2] | (n[..., 1::2] << 4)
    return q.contiguous(), scale.contiguous(), zero


def _check_weight(q, scale, zero, op: str) -> int:
    if q.dtype != torch.uint8 or (zero is not None and zero.dtype != torch.uint8):
        raise TypeError(f"{op}: q and zero must be uint8")
    if q.dim() not in (2, 3) or scale.dim() != q.dim() or scale.shape[:-1] != q.shape[:-1]:
        raise ValueError(f"{op}: q {tuple(q.shape)} and scale {tuple(scale.shape)} do not fit")
    if zero is not None and zero.shape != scale.shape:
        raise ValueError(f"{op}: zero {tuple(zero.shape)} must have scale's shape {tuple(scale.shape)}")
    K, groups = q.shape[-1] * 2, scale.shape[-1]
    if groups < 1 or K % groups:
        raise ValueError(f"{op}: {groups} groups do not divide K = {K}")
    _check_group(K, K // groups, op)
    return K


def int4_dequantize(q: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None
                    ) -> torch.Tensor:
    """The weight that ``(q, scale, zero)`` stand for, float32, [K, N] or [E, K, N] (column-major)."""
    K = _check_weight(q, scale, zero, "int4_dequantize")
    v = torch.stack((q & 15, q >> 4), dim=-1).flatten(-2).float().unflatten(-1, (scale.shape[-1], -1))
    v = v - (8.0 if zero is None else (zero & 15).float().unsqueeze(-1))
    w = (v * scale.float().unsqueeze(-1)).flatten(-2)
    assert w.shape[-1] == K
    return w.transpose(-1, -2)


def _plain(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` with 16-byte aligned rows, which the kernels load 16 bytes at a time (K is a
    multiple of 32, so a copy is aligned), at most 2^23 elements apart (a tile's rows are addressed in 32 bits)."""
    x = _prep(x)
    if x.data_ptr() % 16 or (x.shape[0] > 1 and (x.stride(0) % 8 or x.stride(0) > MAX_K)):
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def int4_matmul(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor,
                zero: Optional[torch.Tensor] = None, ends: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out = x @ W`` with a 4-bit weight (see the module's head).

    ``x`` [M, K] float16 or bfloat16, ``scale`` of x's dtype; returns [M, N]. With
    ``ends`` [E] and a weight for each expert (``q`` [E, N, K/2]) the rows are grouped
    as in ``grouped_matmul``: rows behind the last expert's are zero in a fresh
    result and left as they were in ``out``. The weight is frozen: no gradients
    are recorded.

    Bfloat16 rows are multiplied by ``16 + q`` and ``-(16 + zero)``, whose fp32 sums then
    cancel: their error is relative to ``scale * sum(|x| (32 + q + zero))``, so a value some
    1e5 times as large as the rest of its row leaves noise there even where its weight is zero,
    and a row gives NaN if it holds an infinity or if 31 times the sum of its magnitudes
    over a group passes 3.4e38. (float16 rows are multiplied by ``q - zero``.)"""
    op = "int4_matmul"
    res = _native_call("int4_matmul", x, q, scale, zero, ends, out)
    if res is not None:
        return res
    if x.dim() != 2:
        raise ValueError(f"{op}: x must be 2-D")
    if x.dtype not in INT4_DTYPES:
        raise TypeError(f"{op}: unsupported dtype {x.dtype}")
    K = _check_weight(q, scale, zero, op)
    if scale.dtype != x.dtype:
        raise TypeError(f"{op}: x is {x.dtype}, scale is {scale.dtype}")
    if x.shape[1] != K:
        raise ValueError(f"{op}: x has K = {x.shape[1]}, the weight {K}")
    for name, t in (("q", q), ("scale", scale), ("zero", zero)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{op}: {name} is on {t.device}, x on {x.device}")
    if (q.dim() == 3) != (ends is not None):
        raise ValueError(f"{op}: ends and expert weights [E, N, K/2] go together")
    if ends is not None:
        if q.shape[0] < 1:
            raise ValueError(f"{op}: needs at least one expert")
        _check_ends(ends, x, q.shape[0], op)
    M, N = x.shape[0], q.shape[-2]
    if out is not None:
        _check_out(out, (M, N), x, op)
    _no_grad(op, "4-bit weights are for inference; detach the rows", x, scale)
    if x.device.type != "cuda":
        res = x.new_zeros(M, N) if out is None else out
        w = int4_dequantize(q, scale, zero)
        if ends is None:
            res.copy_(torch.matmul(x.float(), w))
        else:
            for e, lo, hi in _ranges(ends, M):
                if hi > lo:
                    res[lo:hi] = torch.matmul(x[lo:hi].float(), w[e]).to(x.dtype)
        return res
    if K > MAX_K:
        raise ValueError(f"{op}: K = {K} (up to 2^23 on the GPU)")
    return _must(_native_call("int4_matmul", _rows(x), _plain(q), _plain(scale),
                              None if zero is None else _plain(zero),
                              None if ends is None else ends.contiguous(), out), out, op)
