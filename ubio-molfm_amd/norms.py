"""Norms of rows as HIP kernels of libe2v2.so.

Layer norm (the reference's nn.LayerNorm, module_utils.py:2151-2178, 2230-2233): any width up to 16384, fp32, bf16 or
fp16 rows, weight and bias in the rows' type or fp32 or absent, with the gradients of rows, weight and bias and the
derivative of that backward pass (force training differentiates the forces once more).  Statistics, row sums and the
parameters' sums are fp32; each result is rounded once.

RMS norm (no counterpart in the reference, whose RMS norm is the equivariant one): the same rows, the residual's addition
before it in the same pass, its first gradients; or its output in 8 bits with block scales (``fp8``), for the product
behind it.

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
    index = dev.index                           # a tensor lies there, so that the device is up: the short ways to ask
    if torch._C._cuda_getDevice() == index:
        return _lib.call(name, *args, _lib.vp(torch._C._cuda_getCurrentRawStream(index)))
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
    if torch.jit.is_tracing() or torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, float(eps), any_order)
    return _forward(x, weight, bias, float(eps), None)


# ---------------------------------------------------------------------------------------------
# RMS norm

# e2v2_rms_rows_args as bytes
_RMS_ARGS = struct.Struct("10Q6q3if")
_BLOCK = 128                                # columns that share a scale in 8 bits


def _address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _rms_forward(x, g, eps, res, rstd):
    """(y, h) with rstd written unless None; h is x without a residual."""
    (xr, ldx), w = _rows(x), x.shape[-1]
    rr, ldr = (None, 0) if res is None else _rows(res)
    y = _empty_rows(x)
    h = x if res is None else _empty_rows(x)
    a = _RMS_ARGS.pack(xr.data_ptr(), _address(rr), _address(g), 0 if res is None else h.data_ptr(), y.data_ptr(), 0,
                       _address(rstd), 0, 0, 0, x.numel() // w, ldx, ldr, 0, 0, 0, w, _TYPES[x.dtype],
                       0 if g is None else _TYPES[g.dtype], eps)
    _call("e2v2_rms_rows_fwd", x.device, a)
    return y, h


class _RmsNormFn(torch.autograd.Function):
    """(y, h) of x and a residual, or y of x alone."""

    @staticmethod
    def forward(ctx, x, g, eps: float, res):
        rstd = x.new_empty(x.numel() // x.shape[-1], dtype=torch.float32)
        y, h = _rms_forward(x, g, eps, res, rstd)
        ctx.save_for_backward(h, g, rstd)
        ctx.set_materialize_grads(False)
        return y if res is None else (y, h)

    @staticmethod
    def backward(ctx, gy, gh=None):
        h, g, rstd = ctx.saved_tensors
        _first_order("rms_norm", gy, gh)
        need_x, need_g, _, need_res = ctx.needs_input_grad
        if gy is None:                          # y was not used
            return gh if need_x else None, None, None, gh if need_res else None
        w = h.shape[-1]
        (hr, ldh), (gyr, ldy) = _rows(h), _rows(gy)
        ghr, ldgh = (None, 0) if gh is None else _rows(gh)
        gx = _empty_rows(h)
        gg = ws = None
        n = 0
        if need_g:
            gg = _empty_rows(g)
            n = min(h.numel() // w, _MAX_PARTS) * w
            ws = h.new_empty(n, dtype=torch.float32)
        a = _RMS_ARGS.pack(hr.data_ptr(), 0, _address(g), 0, 0, 0, rstd.data_ptr(), gyr.data_ptr(), _address(ghr),
                           gx.data_ptr(), h.numel() // w, ldh, 0, ldy, ldgh, 0, w, _TYPES[h.dtype],
                           0 if g is None else _TYPES[g.dtype], 0.0)
        _call("e2v2_rms_rows_bwd", h.device, a, _ptr(gg), _ptr(ws), _lib.i64(4 * n))
        return gx if need_x else None, gg, None, gx if need_res else None


def _first_order(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """A backward pass that is to be differentiated itself is refused, and so are upstream gradients that no kernel reads
    (batched, or with a tangent)."""
    if torch.is_grad_enabled():
        raise NotImplementedError(f"{name} is differentiable once: create_graph=True is not supported")
    if has_tangent(*tensors) or not all(t is None or torch._C._has_storage(t) for t in tensors):
        raise RuntimeError(f"{name}: batched gradients and gradients with forward-mode tangents are not supported")


def _no_trace(name: str) -> None:
    """torch.jit.trace records a Function as one call, but of a kernel that is launched here only the empty tensor that it
    writes: what is no Function is refused there."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{name}: torch.jit.trace does not record it")


def _forward_only(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """For calls without gradients: one that would need them (of codes too: those cast from values that need them do) is
    refused instead of losing them, and so is a trace."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} has no gradients: call it under torch.no_grad()")
    if has_tangent(*tensors):
        raise RuntimeError(f"{name} has no gradients: a forward-mode tangent would be lost")
    _no_trace(name)


def _rms_check(name, x, weight, residual):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError(f"{name} runs on the GPU only (HIP library, no CPU path): got "
                           f"{x.device if isinstance(x, torch.Tensor) else type(x).__name__}")
    dtype = x.dtype
    if dtype not in _TYPES or x.dim() == 0:
        raise ValueError(f"{name}: rows in fp32, bf16 or fp16, got {tuple(x.shape)} {dtype}")
    w = x.shape[-1]
    if not 1 <= w <= MAX_WIDTH:
        raise ValueError(f"{name}: width {w} (1 to {MAX_WIDTH})")
    if weight is not None and (weight.dim() != 1 or weight.shape[0] != w or not weight.is_cuda
                               or (weight.dtype != dtype and weight.dtype != torch.float32)
                               or weight.get_device() != x.get_device()):
        raise ValueError(f"{name}: weight [{w}] in fp32 or {dtype} on {x.device}, got {tuple(weight.shape)} "
                         f"{weight.dtype} on {weight.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != dtype or not residual.is_cuda
                                 or residual.get_device() != x.get_device()):
        raise ValueError(f"{name}: residual {tuple(x.shape)} {dtype} on {x.device}, got {tuple(residual.shape)} "
                         f"{residual.dtype} on {residual.device}")
    if has_tangent(x, weight, residual):
        raise RuntimeError(f"{name}: forward-mode tangents are not supported")
    return weight if weight is None or weight.is_contiguous() else weight.contiguous()


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
             residual: Optional[torch.Tensor] = None):
    """h / sqrt(mean(h^2) + eps) * weight over the last dimension, with h = x, or with a residual h = x + residual rounded to
    x's type; returns the norm, with a residual (norm, h).

    x: fp32, bf16 or fp16 on the GPU, of any shape with a last dimension of 1 to 16384, the residual like it; both are read
    where they lie if their rows are consecutive and evenly spaced.  weight: [w], fp32 or x's type, or None.  Results
    have x's type and are contiguous.  The squares' sum is fp32: a row in which it passes 3.4e38 gives zeros.
    Differentiable once in reverse mode (create_graph=True raises)."""
    weight = _rms_check("rms_norm", x, weight, residual)
    if torch.jit.is_tracing() or torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad)
            or (residual is not None and residual.requires_grad)):
        return _RmsNormFn.apply(x, weight, float(eps), residual)
    y, h = _rms_forward(x, weight, float(eps), residual, None)
    return y if residual is None else (y, h)


def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                 residual: Optional[torch.Tensor] = None):
    """rms_norm with its output in 8 bits for ``fp8.gemm`` or ``experts.expert_gemm_fp8``: (codes, scales), with a residual
    (codes, scales, h).  The codes are those of the norm before it is rounded to x's type.  No gradients: call it under
    torch.no_grad(), or with tensors that need none."""
    weight = _rms_check("rms_norm_fp8", x, weight, residual)
    _forward_only("rms_norm_fp8", x, weight, residual)
    w = x.shape[-1]
    n, pitch, blocks = x.numel() // w, (w + 15) // 16 * 16, (w + _BLOCK - 1) // _BLOCK
    (xr, ldx), (rr, ldr) = _rows(x), (None, 0) if residual is None else _rows(residual)
    lead = x.shape[:-1]
    codes = torch.empty((*lead, pitch), dtype=torch.float8_e4m3fn, device=x.device)
    held = torch.empty((blocks, n), dtype=torch.uint8, device=x.device)      # a block's scales side by side
    h = x if residual is None else _empty_rows(x)
    a = _RMS_ARGS.pack(xr.data_ptr(), _address(rr), _address(weight), 0 if residual is None else h.data_ptr(),
                       codes.data_ptr(), held.data_ptr(), 0, 0, 0, 0, n, ldx, ldr, 0, 0, pitch, w, _TYPES[x.dtype],
                       0 if weight is None else _TYPES[weight.dtype], float(eps))
    _call("e2v2_rms_rows_fwd", x.device, a)
    if pitch != w:
        codes = codes[..., :w]
    scales = held.t() if len(lead) == 1 else held.t().view(*lead, blocks)
    return (codes, scales) if residual is None else (codes, scales, h)
