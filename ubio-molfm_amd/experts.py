"""Products grouped by expert: rows sorted by expert, each expert's rows times its own weight, in one launch whose sizes only
the GPU knows (no counterpart in the reference).  ``gemm.gemm_grouped`` joins up to four products of sizes that the host
knows; here the experts' row counts are read from a tensor of offsets by the kernel, so that a router's or a sorted
batch's result (one weight for each element, say) needs no wait and a captured graph takes other counts on replay.

There is no CPU path."""
from __future__ import annotations

import functools
import struct
from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .fp8 import MAX_PITCH, _has_tiles, _on_gpu, _product, _row_operand
from .norms import _TYPES, _address, _call, _first_order, _forward_only, _no_trace, has_tangent

_FORWARD, _ROWS, _WEIGHTS = 0, 1, 2         # E2V2_EXPERT_*
# e2v2_expert_args as bytes
_ARGS = struct.Struct("5Q8q3i4x")


def _matrix(t: torch.Tensor, rows: Optional[int] = None):
    """(t as the kernel reads it, its row stride): consecutive elements in a row."""
    w = t.shape[-1]
    if t.stride(-1) != 1 and w > 1 or t.stride(-2) < w and t.shape[-2] > 1 or t.stride(-2) * t.element_size() > MAX_PITCH:
        t = t.contiguous()
    return t, t.stride(-2) if t.shape[-2] > 1 else w


def _experts_of(name, offsets, experts, dev):
    if (not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] != experts + 1
            or offsets.dtype not in (torch.int32, torch.int64) or offsets.device != dev):
        got = (f"{tuple(offsets.shape)} {offsets.dtype} on {offsets.device}" if isinstance(offsets, torch.Tensor)
               else type(offsets).__name__)
        raise ValueError(f"{name}: offsets [{experts + 1}] int32 or int64 on {dev}, got {got}")
    if offsets.dtype is not torch.int32:
        offsets = offsets.to(torch.int32)
    return offsets if offsets.is_contiguous() else offsets.contiguous()


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(rows: int, n: int, k: int, experts: int) -> int:
    return _lib.load().e2v2_expert_product_workspace(rows, n, k, experts)


def _launch(which, x, w_shape, w, gy, y, offsets, fill):
    experts, n, k = w_shape
    ldx = ldw = ldgy = group = 0
    if x is not None:
        x, ldx = _matrix(x)
    if gy is not None:
        gy, ldgy = _matrix(gy)
    if w is not None:
        w, ldw = _matrix(w)
        group = w.stride(0)
    rows = (gy if x is None else x).shape[0]
    need = _workspace_bytes(rows, n, k, experts) if which == _WEIGHTS else 0
    ws = torch.empty(need // 4, dtype=torch.float32, device=y.device) if need else None
    a = _ARGS.pack(_address(x), _address(w), _address(gy), y.data_ptr(), offsets.data_ptr(), rows, n, k, max(ldx, k),
                   max(ldw, k), max(ldgy, n), y.stride(-2) if y.shape[-2] > 1 else y.shape[-1], group, experts,
                   _TYPES[y.dtype], fill)
    _call("e2v2_expert_product", y.device, a, _lib.i32(which), _lib.vp(_address(ws)), _lib.i64(need))
    return y


class _ExpertLinearFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w, offsets):
        y = torch.empty((x.shape[0], w.shape[1]), dtype=x.dtype, device=x.device)
        need_x, need_w = ctx.needs_input_grad[:2]
        ctx.save_for_backward(x if need_w else None, w if need_x else None, offsets)
        ctx.x_shape, ctx.w_shape = x.shape, w.shape
        return _launch(_FORWARD, x, w.shape, w, None, y, offsets, True) if y.numel() else y

    @staticmethod
    def backward(ctx, gy):
        _first_order("expert_linear", gy)
        x, w, offsets = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        gx = gw = None
        if need_x:
            gx = torch.empty(ctx.x_shape, dtype=gy.dtype, device=gy.device)
            if gx.numel():
                _launch(_ROWS, None, ctx.w_shape, w, gy, gx, offsets, True)
        if need_w:
            gw = torch.empty(ctx.w_shape, dtype=gy.dtype, device=gy.device)
            if ctx.x_shape[0] == 0:
                gw.zero_()
            else:
                _launch(_WEIGHTS, x, ctx.w_shape, None, gy, gw, offsets, True)
        return gx, gw, None


def expert_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = weight[e] x[t] for the rows t = offsets[e] .. offsets[e + 1] - 1 of each expert e.

    x [rows, k] and weight [experts, n, k] in one of fp32, bf16 and fp16; offsets [experts + 1], int32 or int64 on the GPU,
    not decreasing, an expert without rows where two are equal (what lies outside 0 .. rows is clamped; int64 ones are read
    as int32).  Rows of no expert give zeros and take no part in gradients.  Sums are fp32 (fp32 operands are split exactly
    into bf16 pieces, as in ``gemm``: a product with an infinite one is NaN there).  Differentiable once in reverse mode, in x
    and weight.

    out [rows, n]: written instead of a new tensor, rows of no expert left as they were; for calls without gradients.  It may
    not share elements with the operands.  It counts as changed in place: a graph that saved its old elements raises."""
    dev = _on_gpu("expert_linear", x, weight)
    if (x.dim() != 2 or weight.dim() != 3 or weight.shape[2] != x.shape[1] or weight.numel() == 0
            or x.dtype not in _TYPES or weight.dtype != x.dtype):
        raise ValueError("expert_linear: x [rows, k] and weight [experts, n, k] in one of fp32, bf16 and fp16, got "
                         f"{tuple(x.shape)} {x.dtype} and {tuple(weight.shape)} {weight.dtype}")
    offsets = _experts_of("expert_linear", offsets, weight.shape[0], dev)
    if has_tangent(x, weight):
        raise RuntimeError("expert_linear: forward-mode tangents are not supported")
    grads = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)
    if out is None:
        if grads or torch.jit.is_tracing():
            return _ExpertLinearFn.apply(x, weight, offsets)
        y, fill = torch.empty((x.shape[0], weight.shape[1]), dtype=x.dtype, device=dev), True
    else:
        _no_trace("expert_linear with out=")
        _check_out("expert_linear", out, (x.shape[0], weight.shape[1]), x.dtype, dev, grads, x, weight, offsets)
        y, fill = out, False
    if y.numel():
        _launch(_FORWARD, x, weight.shape, weight, None, y, offsets, fill)
        if out is not None:
            increment_version(out)
    return y


def _check_out(name, out, shape, dtype, dev, grads, *operands):
    if grads or (torch.is_grad_enabled() and out.requires_grad):
        raise RuntimeError(f"{name}: out= has no gradients: call it under torch.no_grad()")
    if (out.shape != shape or out.dtype != dtype or out.device != dev or (shape[1] > 1 and out.stride(1) != 1)
            or (shape[0] > 1 and out.stride(0) < shape[1])):
        raise ValueError(f"{name}: out {shape} {dtype} on {dev} with consecutive elements in a row, got "
                         f"{tuple(out.shape)} {out.dtype} on {out.device} with strides {out.stride()}")
    if any(_overlap(out, t) for t in operands):
        raise ValueError(f"{name}: out shares elements with an operand")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether tensors may share elements: their bytes overlap, and they are not matrices with consecutive elements in a
    row that are columns side by side of one table."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.element_size()
                           * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))) for t in (a, b))
    if a1 <= b0 or b1 <= a0:
        return False
    pitch = a.stride(0) * a.element_size()
    if (a.dim() != 2 or b.dim() != 2 or a.stride(1) != 1 or b.stride(1) != 1 or pitch == 0
            or b.stride(0) * b.element_size() != pitch):
        return True
    (lo, wide), (hi, _) = sorted(((a0, a.shape[1] * a.element_size()), (b0, b.shape[1] * b.element_size())))
    between = (hi - lo) % pitch                      # from the lower one's column to the other's, in the table's rows
    return between < wide or between + (b if hi == b0 else a).shape[1] * a.element_size() > pitch


def expert_gemm_fp8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                    offsets: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The product of :func:`expert_linear` in 8 bits (the format of ``fp8``): x [rows, k] with x_scale
    [rows, ceil(k / 128)], weight [experts, n, k] with weight_scale [experts, ceil(n / 128), ceil(k / 128)].  The result is
    fp32, bf16 or fp16 (out's type where it is given).  No gradients: ``fp8.linear`` trains a single weight in 8 bits."""
    dev = _on_gpu("expert_gemm_fp8", x, x_scale, weight, weight_scale)
    dtype = dtype if out is None else out.dtype
    if x.dim() != 2 or weight.dim() != 3 or weight.shape[2] != x.shape[1] or weight.numel() == 0 or dtype not in _TYPES:
        raise ValueError("expert_gemm_fp8: x [rows, k] and weight [experts, n, k], out in fp32, bf16 or fp16, got "
                         f"{tuple(x.shape)}, {tuple(weight.shape)} and {dtype}")
    (rows, k), (experts, n, _) = x.shape, weight.shape
    _has_tiles("expert_gemm_fp8", "x", x, x_scale, tiles=False)
    _has_tiles("expert_gemm_fp8", "weight", weight, weight_scale, rows=False)
    offsets = _experts_of("expert_gemm_fp8", offsets, experts, dev)
    _forward_only("expert_gemm_fp8", x, weight)
    if out is None:
        y, fill = torch.empty((rows, n), dtype=dtype, device=dev), True
    else:
        _check_out("expert_gemm_fp8", out, (rows, n), dtype, dev, False, x, x_scale, weight, weight_scale, offsets)
        y, fill = out, False
    if y.numel() == 0:
        return y
    xr, ldx = _row_operand("expert_gemm_fp8", x)
    w, ldw = _matrix(weight)
    _product(xr, ldx, x_scale, w, ldw, weight_scale, True, y, rows, n, k, offsets, experts, w.stride(0), fill)
    if out is not None:
        increment_version(out)
    return y
