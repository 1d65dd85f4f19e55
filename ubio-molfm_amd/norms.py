"""Layer norm of rows (the reference's nn.LayerNorm, module_utils.py:2151-2178, 2230-2233) as HIP kernels of
libe2v2.so: any width up to 16384, fp32, bf16 or fp16 rows, weight and bias in the rows' type or fp32 or absent,
with the gradients of rows, weight and bias and the derivative of that backward pass (force training differentiates
the forces once more).  Statistics, row sums and the parameters' sums are fp32; each result is rounded once.

The equivariant RMS norm is in ``modules`` / ``second_order``, the fused LayerNorm + SiLU of the radial profiles, and so
every LayerNorm of the models built here, in ``second_order.ln_silu``; ``second_order.run_seq`` calls this one for the
others of a user's net.  There is no CPU path."""
from __future__ import annotations

import struct
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

MAX_WIDTH = 16384
_MAX_PARTS = 1024       # kLnMaxParts of csrc/norm.hip
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else _lib.vp(t.data_ptr())


def _rows(t: torch.Tensor):
    """(t as the kernels read it, its row stride): consecutive elements in a row, rows one stride apart, on the
    boundaries of the element type; a copy where t does not lie so."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.stride(-1) == 1 or t.shape[-1] == 1:
        ld = None
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if ld is None:
                ld, span = stride, size * stride
            elif stride == span:
                span = size * stride
            else:
                break
        else:
            return t, t.shape[-1] if ld is None else ld
    return t.contiguous(), t.shape[-1]


def _will_run(node) -> bool:
    """Whether the running backward needs the gradient flowing into node (False
    only when the engine reports that it will not execute it: autograd.grad of
    other inputs, as the forces' first differentiation)."""
    if node is None:
        return False
    try:
        return bool(torch._C._will_engine_execute_node(node))
    except (AttributeError, RuntimeError):
        return True


# e2v2_layer_norm_args as bytes: packing them is a few times faster than filling a ctypes structure
_ARGS = struct.Struct("10Q4q4if4x")


def _args(x, g, b, stats, eps, gy=None, qx=None, qg=None, qb=None, y=None, gx=None):
    """The kernels' arguments, and the copies that have to live until the call is enqueued."""
    w = x.shape[-1]
    rows, ld = [x, gy, qx], [0, 0, 0]
    for k in range(3):
        if rows[k] is not None:
            rows[k], ld[k] = _rows(rows[k])
    params = [t if t is None or t.is_contiguous() else t.contiguous() for t in (g, b, qg, qb)]
    a = _ARGS.pack(*[0 if t is None else t.data_ptr() for t in (*rows, *params, y, gx, stats)], x.numel() // w, *ld, w,
                   _TYPES[x.dtype], 0 if g is None else _TYPES[g.dtype], 0 if b is None else _TYPES[b.dtype], eps)
    return a, (rows, params)


def _empty_rows(x):
    """A contiguous tensor of x's shape, type and device."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _workspace(x):
    """Room for the parameters' partial sums, as e2v2_layer_norm_workspace says, and its bytes."""
    w = x.shape[-1]
    n = 2 * min(x.numel() // w, _MAX_PARTS) * w
    return x.new_empty(n, dtype=torch.float32), 4 * n


def _call(name, dev, *args):
    if torch.cuda.current_device() == dev.index:
        return _lib.call(name, *args, _lib.stream(dev))
    with torch.cuda.device(dev):
        _lib.call(name, *args, _lib.stream(dev))


def _forward(x, g, b, eps, stats):
    y = _empty_rows(x)
    a, keep = _args(x, g, b, stats, eps, y=y)
    _call("e2v2_layer_norm_fwd", x.device, a)
    return y


def _backward(gy, x, g, b, stats, eps, need_g, need_b):
    gx = _empty_rows(x)
    gg = _empty_rows(g) if need_g else None
    gb = _empty_rows(b) if need_b else None
    ws, n = _workspace(x) if need_g or need_b else (None, 0)
    a, keep = _args(x, g, b, stats, eps, gy=gy, gx=gx)
    _call("e2v2_layer_norm_bwd", x.device, a, _ptr(gg), _ptr(gb), _ptr(ws), _lib.i64(n))
    return gx, gg, gb


class _LayerNormFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, g, b, eps: float, any_order: bool):
        stats = x.new_empty(2 * (x.numel() // x.shape[-1]), dtype=torch.float32)
        y = _forward(x, g, b, eps, stats)
        ctx.save_for_backward(x, g, b, stats)
        ctx.eps, ctx.any_order = eps, any_order
        return y

    @staticmethod
    def backward(ctx, gy):
        x, g, b, stats = ctx.saved_tensors
        need_g, need_b = ctx.needs_input_grad[1:3]
        if _only_torch_takes(ctx.any_order, gy):
            gx, gg, gb = _composed(gy, x, g, b, ctx.eps)
        elif not torch.is_grad_enabled():
            gx, gg, gb = _backward(gy, x, g, b, stats, ctx.eps, need_g, need_b)
        else:
            # the forces' first differentiation asks for neither weight nor bias; their sums come together.
            # next_functions has an entry for each tensor among the inputs
            nodes = iter(ctx.next_functions[1:])
            nodes = [next(nodes)[0] for t in (g, b) if t is not None]
            if not any([_will_run(n) for n in nodes]):
                need_g = need_b = False
            fn = _LayerNormGradAnyFn if ctx.any_order else _LayerNormGradFn
            gx, gg, gb = fn.apply(gy, x, g, b, stats, ctx.eps, need_g, need_b)
        return gx if ctx.needs_input_grad[0] else None, gg, gb, None, None


class _LayerNormGradFn(torch.autograd.Function):
    """(gx, dg, db) of _LayerNormFn given gy; mean and rstd enter as constants, the second-order pass
    differentiates through them by its formulas."""

    @staticmethod
    def forward(ctx, gy, x, g, b, stats, eps, need_g, need_b):
        out = _backward(gy, x, g, b, stats, eps, need_g, need_b)
        ctx.save_for_backward(gy, x, g, b, stats)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, qx, qg, qb):
        _only_torch_takes(False, ctx.saved_tensors[0], qx, qg, qb)
        return _backward2(ctx, qx, qg, qb)


class _LayerNormGradAnyFn(_LayerNormGradFn):
    """The same, differentiable on: where its own backward is to be differentiated (a third derivative of the norm),
    that is composed of torch's operators."""

    @staticmethod
    def backward(ctx, qx, qg, qb):
        gy, x, g, _, _ = ctx.saved_tensors
        if qx is None and qg is None and qb is None or not (torch.is_grad_enabled()
                                                            or _only_torch_takes(True, gy, qx, qg, qb)):
            return _backward2(ctx, qx, qg, qb)
        return (*_composed2(gy, x, g, ctx.eps, qx, qg, qb), None, None, None, None, None)


def _backward2(ctx, qx, qg, qb):
    """The gradients of _LayerNormGradFn's inputs through e2v2_layer_norm_bwd2."""
    gy, x, g, b, stats = ctx.saved_tensors
    if qx is None and qg is None and qb is None:
        return (None,) * 8
    dgy, dx = _empty_rows(x), _empty_rows(x)
    dg = _empty_rows(g) if ctx.needs_input_grad[2] else None
    ws, n = _workspace(x) if dg is not None else (None, 0)
    a, keep = _args(x, g, b, stats, ctx.eps, gy=gy, qx=qx, qg=qg, qb=qb, y=dgy, gx=dx)
    _call("e2v2_layer_norm_bwd2", x.device, a, _ptr(dg), _ptr(ws), _lib.i64(n))
    return dgy, dx, dg, None, None, None, None, None


def _composed(gy, x, g, b, eps):
    """(gx, dg, db) by the formulas at the head of csrc/norm.hip."""
    def mean(t):
        return t.mean(-1, keepdim=True)

    z = x - mean(x)
    r = torch.rsqrt(mean(z * z) + eps)
    h, u, w = z * r, gy if g is None else gy * g, x.shape[-1]
    return (r * (u - mean(u) - h * mean(u * h)), None if g is None else (gy * h).reshape(-1, w).sum(0),
            None if b is None else gy.reshape(-1, w).sum(0))


def _composed2(gy, x, g, eps, qx, qg, qb):
    """(dgy, dx, dg) of the second order by the formulas at the head of csrc/norm.hip."""
    def mean(t):
        return t.mean(-1, keepdim=True)

    z = x - mean(x)
    r = torch.rsqrt(mean(z * z) + eps)
    h, u = z * r, gy if g is None else gy * g
    dgy, t, extra, dg = 0, 0, 0, None
    if qx is not None:
        c, m = mean(u * h), mean(qx * h)
        a = r * (qx - mean(qx) - h * m)
        dgy = a if g is None else a * g
        t = -r * (c * qx + m * u)
        extra = r * h * mean(qx * r * (u - mean(u) - h * c))
        dg = None if g is None else (gy * a).reshape(-1, x.shape[-1]).sum(0)
    if qg is not None:
        dgy, t = dgy + qg * h, t + qg * gy
    if qb is not None:
        dgy = dgy + qb
    dx = None if qx is None and qg is None else r * (t - mean(t) - h * mean(t * h)) - extra
    return dgy.expand_as(gy), dx, dg


def has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a tensor carries a forward-mode tangent."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                                  for t in tensors)


def _only_torch_takes(composed: bool, *tensors: Optional[torch.Tensor]) -> bool:
    """Whether an upstream gradient is one that no kernel reads (batched by is_grads_batched or torch.func, or with a
    tangent); an error unless the pass can be composed of torch's operators."""
    if has_tangent(*tensors) or not all(t is None or torch._C._has_storage(t) for t in tensors):
        if not composed:
            raise RuntimeError("layer_norm: batched gradients and gradients with forward-mode tangents are not supported")
        return True
    return False


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x, as
    torch.nn.functional.layer_norm(x, (w,), weight, bias, eps).

    x: fp32, bf16 or fp16 on the GPU, of any shape with a last dimension of 1 to 16384; read where it lies if its rows
    are consecutive and evenly spaced.  weight, bias: [w], fp32 or x's type, or None.  The result has x's type
    and is contiguous.  Differentiable twice in reverse mode (a third derivative, forward-mode tangents, batched gradients
    and torch.func's transforms raise)."""
    return _layer_norm(x, weight, bias, eps, any_order=False)


def _layer_norm(x, weight, bias, eps: float, any_order: bool) -> torch.Tensor:
    """layer_norm; any_order: differentiable as often as the nn.LayerNorm in whose place it stands, from the third
    derivative on by torch's operators."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("layer_norm runs on the GPU only (HIP library, no CPU path): got "
                           f"{x.device if isinstance(x, torch.Tensor) else type(x).__name__}")
    dtype = x.dtype
    if dtype not in _TYPES or x.dim() == 0:
        raise ValueError(f"layer_norm: rows in fp32, bf16 or fp16, got {tuple(x.shape)} {dtype}")
    w = x.shape[-1]
    if not 1 <= w <= MAX_WIDTH:
        raise ValueError(f"layer_norm: width {w} (1 to {MAX_WIDTH})")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.dim() != 1 or p.shape[0] != w or (p.dtype != dtype and p.dtype != torch.float32)
                              or not p.is_cuda or p.get_device() != x.get_device()):
            raise ValueError(f"layer_norm: {name} [{w}] in fp32 or {dtype} on {x.device}, got {tuple(p.shape)} "
                             f"{p.dtype} on {p.device}")
    if has_tangent(x, weight, bias):
        raise RuntimeError("layer_norm: forward-mode tangents are not supported")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, float(eps), any_order)
    return _forward(x, weight, bias, float(eps), None)
