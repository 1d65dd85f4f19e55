"""8-bit floats with block scales: quantising rows and weights, products of them on the matrix units, and a linear layer that
trains with all three of its products in 8 bits (no counterpart in the reference).

Format: e4m3 codes (torch.float8_e4m3fn) and for each block a scale byte s (torch.uint8) that stands for 2^(s - 127), the
smallest power of two (2^-126 at least) with which the block's largest finite value is at most 448.  Blocks are 128
consecutive values of a row (activations, gradients), or tiles of 128 x 128 (weights).  A code is rounded once, to the
nearest, ties to even; what is not finite becomes NaN and has no part in its block's scale.  The matrix units apply such
scales themselves; they add the products of eight values on a grid of 2^-13 of the largest of them, and the rest in fp32.

There is no CPU path."""
from __future__ import annotations

import functools
import struct
from typing import Optional

import torch

from . import _lib
from .norms import _TYPES, _address, _call, _first_order, _forward_only, _rows, has_tangent

BLOCK = 128
CODES = torch.float8_e4m3fn
MAX_PITCH = 1 << 22                         # bytes between rows that the products take
_ROWS, _TILES, _BOTH = 0, 1, 2              # E2V2_QUANT_*

# e2v2_quantize8_args and e2v2_product8_args as bytes
_QUANT_ARGS = struct.Struct("5Q6q3i4x")
_PRODUCT_ARGS = struct.Struct("6Q12q4i")


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _pitch(n: int) -> int:
    return (n + 15) // 16 * 16


def _on_gpu(name: str, *tensors) -> torch.device:
    """The one GPU that all tensors are on."""
    index = None
    for t in tensors:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError(f"{name} runs on the GPU only (HIP library, no CPU path): got "
                               f"{t.device if isinstance(t, torch.Tensor) else type(t).__name__}")
        if index is None:
            index = t.get_device()
        elif t.get_device() != index:
            raise ValueError(f"{name}: operands on {tensors[0].device} and {t.device}")
    return tensors[0].device


def _matrix_codes(rows: int, width: int, dev):
    """Codes of a matrix, rows a multiple of 16 bytes apart, and their pitch."""
    pitch = _pitch(width)
    return torch.empty((rows, pitch), dtype=CODES, device=dev), pitch


def _quantize(x, ldx, mode, codes=None, scales=None, codes_t=None, scales_t=None, n=0, batch=1, x_batch=0):
    """One call of e2v2_quantize8 on x [.., n, width]; codes and codes_t with their padding."""
    a = _QUANT_ARGS.pack(x.data_ptr(), _address(codes), _address(scales), _address(codes_t), _address(scales_t), n,
                         x.shape[-1], ldx, 0 if codes is None else codes.shape[-1],
                         0 if codes_t is None else codes_t.shape[-1], x_batch, batch, _TYPES[x.dtype], mode)
    _call("e2v2_quantize8", x.device, a)


def quantize(x: torch.Tensor, tiles: bool = False):
    """(codes, scales) of x in fp32, bf16 or fp16.

    tiles=False: x [..., w], codes of x's shape, scales [..., ceil(w / 128)] (a view: a block's lie side by side).
    tiles=True: weights [n, k] or [experts, n, k], scales [(experts,) ceil(n / 128), ceil(k / 128)].  Rows of codes lie a
    multiple of 16 bytes apart, so codes are a view where the width is not one.  No gradients."""
    _on_gpu("quantize", x)
    if x.dtype not in _TYPES or x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"quantize: fp32, bf16 or fp16 rows of at least one value, got {tuple(x.shape)} {x.dtype}")
    _forward_only("quantize", x)
    w = x.shape[-1]
    if not tiles:
        xr, ldx = _rows(x)
        lead = x.shape[:-1]
        codes = torch.empty((*lead, _pitch(w)), dtype=CODES, device=x.device)
        scales, held = _block_major(lead, x.numel() // w, _blocks(w), x.device)
        _quantize(xr, ldx, _ROWS, codes, held, n=x.numel() // w)
    else:
        if x.dim() not in (2, 3):
            raise ValueError(f"quantize: weights [n, k] or [experts, n, k], got {tuple(x.shape)}")
        lead, n = x.shape[:-2], x.shape[-2]
        if x.stride(-1) != 1 and w > 1:
            x = x.contiguous()
        codes = torch.empty((*lead, n, _pitch(w)), dtype=CODES, device=x.device)
        scales = torch.empty((*lead, _blocks(n), _blocks(w)), dtype=torch.uint8, device=x.device)
        _quantize(x, x.stride(-2), _TILES, codes, scales, n=n, batch=lead[0] if lead else 1,
                  x_batch=x.stride(0) if lead else 0)
    return (codes if codes.shape[-1] == w else codes[..., :w]), scales


def _has_tiles(name, what, codes, scales, rows=True, tiles=True) -> bool:
    """Whether scales are those of tiles, not of rows; an error where they are of neither that may be."""
    shape, got = tuple(codes.shape), tuple(scales.shape)
    k = _blocks(shape[-1])
    by_row, by_tile = (*shape[:-1], k), (*shape[:-2], _blocks(shape[-2]), k) if len(shape) > 1 else None
    if codes.dtype is CODES and scales.dtype is torch.uint8:
        if rows and got == by_row:
            return False
        if tiles and got == by_tile:
            return True
    raise ValueError(f"{name}: {what} in e4m3 with uint8 scales "
                     f"{' or '.join(str(b) for b, may in ((by_row, rows), (by_tile, tiles)) if may and b)}, got "
                     f"{shape} {codes.dtype} and {got} {scales.dtype}")


def dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that codes and scales stand for, contiguous, in fp32, bf16 or fp16 (exact in the first two, but for values
    outside the type's range).  Whether scales are those of rows or of tiles shows in their shape.  No gradients."""
    dev = _on_gpu("dequantize", codes, scales)
    if dtype not in _TYPES or codes.dim() == 0:
        raise ValueError(f"dequantize: codes {tuple(codes.shape)}, values in fp32, bf16 or fp16, got {dtype}")
    tiles = _has_tiles("dequantize", "codes", codes, scales)
    _forward_only("dequantize", codes)
    out = torch.empty(codes.shape, dtype=dtype, device=dev)
    if out.numel() == 0:
        return out
    w = codes.shape[-1]
    cr, ldc = _rows(codes)
    sr, s_ld = _scale_rows(scales)
    _call("e2v2_values8", dev, _lib.vp(cr.data_ptr()), _lib.i64(ldc), _lib.vp(sr.data_ptr()), _lib.i64(s_ld),
          _lib.i64(sr.stride(-1)), _lib.i32(tiles), _lib.i64(codes.numel() // w), _lib.i64(w),
          _lib.i64(codes.shape[-2] if tiles else 0), _lib.vp(out.data_ptr()), _lib.i32(_TYPES[dtype]))
    return out


def _scale_rows(scales):
    """(scales as the kernels read them, bytes from row to row): rows one stride apart; a copy where they do not lie so."""
    if scales.dim() < 2:
        return scales, 0
    ld = scales.stride(-2) if scales.shape[-2] > 1 else 0
    if scales.dim() > 2:
        span = None
        for size, stride in zip(reversed(scales.shape[:-1]), reversed(scales.stride()[:-1])):
            if size > 1:
                if span is None:
                    ld = stride
                elif stride != span:
                    scales = scales.contiguous()
                    return scales, scales.shape[-1]
                span = size * stride
    return scales, ld


def _block_major(lead, rows: int, blocks: int, dev):
    """Scales [*lead, blocks] of rows that lie side by side block by block (so a tile's are read together), and the tensor
    that the kernels write."""
    held = torch.empty((blocks, rows), dtype=torch.uint8, device=dev)
    return held.t().view(*lead, blocks) if len(lead) != 1 else held.t(), held


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(m: int, n: int, k: int) -> int:
    return _lib.load().e2v2_product8_workspace(m, n, k)


def _product(a, lda, sa, b, ldb, sb, b_tiles, y, m, n, k, offsets=None, groups=0, b_group=0, fill=False):
    """y = a b^T by e2v2_product8; all operands are as the kernel reads them."""
    need = 0 if offsets is not None else _workspace_bytes(m, n, k)
    ws = torch.empty(need // 4, dtype=torch.float32, device=y.device) if need else None
    args = _PRODUCT_ARGS.pack(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), y.data_ptr(), _address(offsets),
                              m, n, k, lda, ldb, y.stride(0) if m > 1 else n, b_group,
                              *sa.stride(), *sb.stride()[-2:], sb.stride(0) if groups else 0, groups, b_tiles,
                              _TYPES[y.dtype], fill)
    _call("e2v2_product8", y.device, args, _lib.vp(_address(ws)), _lib.i64(need))
    return y


def _row_operand(name, codes):
    w = codes.shape[-1]
    if w > MAX_PITCH:
        raise ValueError(f"{name}: rows of {w} bytes (at most {MAX_PITCH})")
    rows, ld = _rows(codes)
    if (ld < w and codes.numel() > w) or ld > MAX_PITCH:        # rows that share bytes or lie too far apart
        rows, ld = rows.contiguous(), w
    return rows, max(ld, w)


def gemm(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
         dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a w^T of 8-bit rows a [..., k] and an 8-bit weight w [n, k]: [..., n] in fp32, bf16 or fp16.

    a_scale [..., ceil(k / 128)]; w_scale [ceil(n / 128), ceil(k / 128)] (tiles) or [n, ceil(k / 128)] (rows).  Any sizes
    (k up to 4,194,304) and alignment; rows that start on multiples of 16 bytes (those of :func:`quantize` do) take the
    faster loads.  No gradients."""
    dev = _on_gpu("gemm", a, a_scale, w, w_scale)
    if a.dim() == 0 or w.dim() != 2 or w.shape[1] != a.shape[-1] or w.shape[1] == 0 or dtype not in _TYPES:
        raise ValueError(f"gemm: a [..., k] and w [n, k], out in fp32, bf16 or fp16; got {tuple(a.shape)}, "
                         f"{tuple(w.shape)} and {dtype}")
    _has_tiles("gemm", "a", a, a_scale, tiles=False)
    tiles = _has_tiles("gemm", "w", w, w_scale)
    _forward_only("gemm", a, w)
    n, k = w.shape
    m = a.numel() // k
    y = torch.empty((m, n), dtype=dtype, device=dev)
    if m:
        (ar, lda), (wr, ldw) = _row_operand("gemm", a), _row_operand("gemm", w)
        _product(ar, lda, a_scale if a.dim() == 2 else a_scale.reshape(m, a_scale.shape[-1]), wr, ldw, w_scale, tiles,
                 y, m, n, k)
    return y if a.dim() == 2 else y.view(*a.shape[:-1], n)


def _linear_forward(x, w, need_x: bool, need_w: bool):
    """(y, and what the gradients of x and w read: the transposed codes and scales of w, and those of x)."""
    n, k = w.shape
    xr, ldx = _rows(x)
    m, dev = x.numel() // k, x.device
    if w.stride(1) != 1 and k > 1:
        w = w.contiguous()
    kb, nb = _blocks(k), _blocks(n)
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=dev)
    wt = wst = xt = xst = None
    if m == 0:
        return y, wt, wst, xt, xst
    wq, _ = _matrix_codes(n, k, dev)
    ws = torch.empty((nb, kb), dtype=torch.uint8, device=dev)
    if need_x:
        wt, wst = _matrix_codes(k, n, dev)[0], torch.empty((kb, nb), dtype=torch.uint8, device=dev)
    _quantize(w, w.stride(0), _TILES, wq, ws, wt, wst, n=n)
    xq, _ = _matrix_codes(m, k, dev)
    xs = torch.empty((kb, m), dtype=torch.uint8, device=dev)
    if need_w:
        xt, xst = _matrix_codes(k, m, dev)[0], torch.empty((_blocks(m), k), dtype=torch.uint8, device=dev)
    _quantize(xr, ldx, _BOTH if need_w else _ROWS, xq, xs, xt, xst, n=m)
    _product(xq, xq.shape[1], xs.t(), wq, wq.shape[1], ws, True, y.view(m, n), m, n, k)
    return y, wt, wst, xt, xst


class _LinearFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w):
        y, *held = _linear_forward(x, w, *ctx.needs_input_grad)
        ctx.sizes, ctx.x_shape, ctx.types = (x.numel() // w.shape[1], *w.shape), x.shape, (x.dtype, w.dtype)
        ctx.save_for_backward(*held)
        return y

    @staticmethod
    def backward(ctx, gy):
        _first_order("linear", gy)
        wt, wst, xt, xst = ctx.saved_tensors
        (m, n, k), dev = ctx.sizes, gy.device
        need_x, need_w = ctx.needs_input_grad
        x_type, w_type = ctx.types
        gx = torch.empty(ctx.x_shape, dtype=x_type, device=dev) if need_x else None
        if m == 0:
            return gx, torch.zeros((n, k), dtype=w_type, device=dev) if need_w else None
        gr, ldg = _rows(gy)
        gq = gs = gt = gst = None
        if need_x:
            gq, gs = _matrix_codes(m, n, dev)[0], torch.empty((_blocks(n), m), dtype=torch.uint8, device=dev)
        if need_w:
            gt, gst = _matrix_codes(n, m, dev)[0], torch.empty((_blocks(m), n), dtype=torch.uint8, device=dev)
        _quantize(gr, ldg, _BOTH if need_w else _ROWS, gq, gs, gt, gst, n=m)
        if need_x:
            _product(gq, gq.shape[1], gs.t(), wt, wt.shape[1], wst, True, gx.view(m, k), m, k, n)
        gw = None
        if need_w:
            gw = torch.empty((n, k), dtype=w_type, device=dev)
            _product(gt, gt.shape[1], gst.t(), xt, xt.shape[1], xst.t(), False, gw, n, k, m)
        return gx, gw


def linear(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """x weight^T with the product, and in the backward pass both gradients' products, in 8 bits.

    x [..., k], weight [n, k], each in fp32, bf16 or fp16; the result and x's gradient have x's type, the weight's gradient
    the weight's.  Rows of x and of the upstream gradient are quantised in blocks of 128 along the reduction of the product
    that they enter (so each has codes along rows and along columns), the weight in tiles of 128 x 128.  The
    gradients are those of the product of the values that the codes stand for; rounding to codes passes them through
    unchanged.  The backward pass keeps the codes, one byte a value, not x.  Differentiable once in reverse mode.  n, k and,
    for the weight's gradient, the rows: 4,194,304 at most."""
    dev = _on_gpu("linear", x, weight)
    if (x.dtype not in _TYPES or weight.dtype not in _TYPES or x.dim() == 0 or weight.dim() != 2
            or weight.shape[1] != x.shape[-1] or weight.numel() == 0):
        raise ValueError(f"linear: x [..., k] and weight [n, k] in fp32, bf16 or fp16, got {tuple(x.shape)} {x.dtype} and "
                         f"{tuple(weight.shape)} {weight.dtype}")
    if has_tangent(x, weight):
        raise RuntimeError("linear: forward-mode tangents are not supported")
    grads = torch.is_grad_enabled()
    # rows of codes: of k and n values, and for the weight's gradient those of the transposes, as long as x has rows
    longest = max(weight.shape[0], weight.shape[1], x.numel() // weight.shape[1] if grads and weight.requires_grad else 0)
    if _pitch(longest) > MAX_PITCH:
        raise ValueError(f"linear: sizes up to {MAX_PITCH}, got {tuple(x.shape)} and {tuple(weight.shape)} on {dev}")
    if torch.jit.is_tracing() or grads and (x.requires_grad or weight.requires_grad):
        return _LinearFn.apply(x, weight)
    return _linear_forward(x, weight, False, False)[0]
