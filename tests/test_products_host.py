"""What the RMS norm, the 8-bit operators and the products grouped by expert refuse, before any kernel or HIP call.  No GPU
needed."""
import ctypes
import struct

import pytest
import torch

from ubio_molfm_amd import _lib, experts, fp8, norms

F8, U8, BF16 = torch.float8_e4m3fn, torch.uint8, torch.bfloat16


class _OnGpu(torch.Tensor):
    """A host tensor that says it lies on the GPU: the checks behind the device's."""
    is_cuda = True


def _gpu(*shape, dtype=torch.float32):
    return torch.zeros(shape).to(dtype).as_subclass(_OnGpu)


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32).as_subclass(_OnGpu)


@pytest.fixture(autouse=True)
def no_kernels(monkeypatch):
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("a kernel was called"))


def test_host_tensors_are_refused():
    x = torch.rand(3, 16)
    for call in (lambda: norms.rms_norm(x), lambda: norms.rms_norm_fp8(x), lambda: norms.rms_norm([1.0]),
                 lambda: fp8.quantize(x), lambda: fp8.linear(x, x), lambda: fp8.linear(x, 3.0),
                 lambda: fp8.dequantize(x.to(F8), torch.zeros(3, 1, dtype=U8)),
                 lambda: fp8.gemm(x.to(F8), torch.zeros(3, 1, dtype=U8), x.to(F8), torch.zeros(3, 1, dtype=U8)),
                 lambda: experts.expert_linear(x, x[None], torch.tensor([0, 3])),
                 lambda: experts.expert_gemm_fp8(x.to(F8), torch.zeros(3, 1, dtype=U8), x[None].to(F8),
                                                 torch.zeros(1, 1, 1, dtype=U8), torch.tensor([0, 3]))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


@pytest.mark.parametrize("fn", [norms.rms_norm, norms.rms_norm_fp8])
@pytest.mark.parametrize("x,kw,match", [
    (lambda: _gpu(3, 8, dtype=torch.float64), {}, "fp32, bf16 or fp16"),
    (lambda: _gpu(), {}, "fp32, bf16 or fp16"),
    (lambda: _gpu(3, 0), {}, "width 0"),
    (lambda: _gpu(1, norms.MAX_WIDTH + 1), {}, "width 16385"),
    (lambda: _gpu(3, 8), dict(weight=torch.ones(8)), "weight"),
    (lambda: _gpu(3, 8), dict(weight=_gpu(7)), "weight"),
    (lambda: _gpu(3, 8), dict(weight=_gpu(8, dtype=BF16)), "weight"),
    (lambda: _gpu(3, 8), dict(residual=_gpu(8)), "residual"),
    (lambda: _gpu(3, 8), dict(residual=_gpu(3, 8, dtype=BF16)), "residual"),
    (lambda: _gpu(3, 8), dict(residual=torch.zeros(3, 8)), "residual"),
])
def test_norm_refusals(fn, x, kw, match):
    with pytest.raises(ValueError, match=match):
        fn(x(), **kw)


def test_8_bit_refusals():
    a, sa, w, sw = _gpu(3, 200, dtype=F8), _gpu(3, 2, dtype=U8), _gpu(130, 200, dtype=F8), _gpu(2, 2, dtype=U8)
    for call, match in (
            (lambda: fp8.quantize(_gpu(3, 8, dtype=torch.float64)), "fp32, bf16 or fp16"),
            (lambda: fp8.quantize(_gpu(3, 0)), "at least one value"),
            (lambda: fp8.quantize(_gpu(3), tiles=True), "weights"),
            (lambda: fp8.gemm(a, sa, w[:, :199], sw), "w \\[n, k\\]"),
            (lambda: fp8.gemm(a, sa, w, sw, dtype=torch.float64), "out in"),
            (lambda: fp8.gemm(a, sa[:, :1], w, sw), "a in e4m3"),
            (lambda: fp8.gemm(a, sa.float(), w, sw), "a in e4m3"),
            (lambda: fp8.gemm(a.float(), sa, w, sw), "a in e4m3"),
            (lambda: fp8.gemm(a, sa, w, sw[:1]), "w in e4m3"),
            (lambda: fp8.dequantize(a, sa[:2]), "codes in e4m3"),
            (lambda: fp8.dequantize(a, sa, torch.float64), "values in"),
            (lambda: fp8.linear(_gpu(3, 8), _gpu(4, 9)), "weight \\[n, k\\]"),
            (lambda: fp8.linear(_gpu(3, 8), _gpu(4, 8, dtype=torch.int32)), "fp32, bf16 or fp16"),
            (lambda: fp8.linear(_gpu(3, 8), _gpu(0, 8)), "weight \\[n, k\\]")):
        with pytest.raises(ValueError, match=match):
            call()


def test_expert_refusals():
    x, w, offs = _gpu(5, 16), _gpu(2, 8, 16), _i32(0, 2, 5)
    for call, match in (
            (lambda: experts.expert_linear(x[0], w, offs), "x \\[rows, k\\]"),
            (lambda: experts.expert_linear(x, w[0], offs), "x \\[rows, k\\]"),
            (lambda: experts.expert_linear(x, w[..., :8], offs), "x \\[rows, k\\]"),
            (lambda: experts.expert_linear(x, w.bfloat16(), offs), "x \\[rows, k\\]"),
            (lambda: experts.expert_linear(x, w[:0], offs[:1]), "x \\[rows, k\\]"),
            (lambda: experts.expert_linear(x, w, offs[:2]), "offsets \\[3\\]"),
            (lambda: experts.expert_linear(x, w, offs.float()), "offsets \\[3\\]"),
            (lambda: experts.expert_linear(x, w, [0, 2, 5]), "offsets \\[3\\]"),
            (lambda: experts.expert_linear(x, w, offs, out=_gpu(5, 9)), "out"),
            (lambda: experts.expert_linear(x, w, offs, out=_gpu(8, 5).t()), "out"),
            (lambda: experts.expert_linear(x, w, offs, out=_gpu(5, 8, dtype=BF16)), "out"),
            (lambda: experts.expert_gemm_fp8(x.to(F8), _gpu(5, 1, dtype=U8), w.to(F8), _gpu(2, 1, 2, dtype=U8), offs),
             "weight in e4m3"),
            (lambda: experts.expert_gemm_fp8(x.to(F8), _gpu(5, 2, dtype=U8), w.to(F8), _gpu(2, 1, 1, dtype=U8), offs),
             "x in e4m3")):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="no gradients"):
        experts.expert_linear(x, torch.nn.Parameter(w.as_subclass(torch.Tensor)).as_subclass(_OnGpu), offs, out=_gpu(5, 8))


def test_out_may_not_share_elements_with_an_operand():
    table = _gpu(12, 40)
    w, offs = _gpu(2, 16, 16), _i32(0, 2, 5)
    x = table[2:7, :16]
    for out in (x, table[2:7, 8:24], table[4:9, :16], table[3:8, 15:31], table.reshape(-1)[30:110].view(5, 16),
                w.reshape(-1)[100:180].view(5, 16), w[1, :5]):
        with pytest.raises(ValueError, match="shares elements"):
            experts.expert_linear(x, w, offs, out=out)
    for out in (table[2:7, 16:32], table[2:7, 24:], table[:5, 16:32], table[4:9, 17:33], table[7:12, :16], _gpu(5, 16)):
        assert not experts._overlap(out, x) and not experts._overlap(out, w)
    one = table[3:4]
    assert experts._overlap(one[:, :16], one[:, 15:31]) and not experts._overlap(one[:, :16], one[:, 16:32])
    assert not experts._overlap(one[:0], one)


def test_packed_arguments_are_the_structures():
    for c, s in ((_lib.RmsRowsArgs, norms._RMS_ARGS), (_lib.Quantize8Args, fp8._QUANT_ARGS),
                 (_lib.Product8Args, fp8._PRODUCT_ARGS), (_lib.ExpertArgs, experts._ARGS)):
        assert ctypes.sizeof(c) == s.size
        fields = [f for f, t in c._fields_]
        values = list(range(1, len(fields) + 1))
        a = c.from_buffer_copy(s.pack(*values))
        assert [int(getattr(a, f) or 0) for f in fields] == values


def test_entry_points_check_on_the_host():
    lib = _lib.load()

    def refused(rc, what):
        assert rc != 0 and what in lib.e2v2_last_error(), lib.e2v2_last_error()

    a = _lib.RmsRowsArgs()
    a.x = a.y = 16
    a.n, a.ldx, a.width = 4, 8, 0
    refused(lib.e2v2_rms_rows_fwd(ctypes.byref(a), None), b"width 0")
    a.width, a.type = 8, 7
    refused(lib.e2v2_rms_rows_fwd(ctypes.byref(a), None), b"types")
    a.type, a.scales, a.ldy = 0, 16, 8
    refused(lib.e2v2_rms_rows_fwd(ctypes.byref(a), None), b"multiple of 16")
    a.scales, a.x = None, 18
    refused(lib.e2v2_rms_rows_fwd(ctypes.byref(a), None), b"misaligned")
    a.x, a.gy, a.gx, a.rstd = 16, 16, 16, 16
    refused(lib.e2v2_rms_rows_bwd(ctypes.byref(a), ctypes.c_void_p(16), None, ctypes.c_int64(0), None), b"workspace")
    assert lib.e2v2_rms_rows_workspace(5, 8) == 160 and lib.e2v2_rms_rows_workspace(0, 8) == 0

    q = _lib.Quantize8Args()
    q.x = q.codes = q.scales = 16
    q.n, q.width, q.ldx, q.ldc, q.batch = 4, 20, 20, 20, 1
    refused(lib.e2v2_quantize8(ctypes.byref(q), None), b"multiple of 16")
    q.ldc, q.mode = 32, 9
    refused(lib.e2v2_quantize8(ctypes.byref(q), None), b"mode 9")
    q.mode, q.codes_t, q.scales_t, q.ldt = 2, 16, 16, 3
    refused(lib.e2v2_quantize8(ctypes.byref(q), None), b"transposed")
    refused(lib.e2v2_values8(ctypes.c_void_p(16), ctypes.c_int64(8), ctypes.c_void_p(16), ctypes.c_int64(1),
                             ctypes.c_int64(1), 1, ctypes.c_int64(9), ctypes.c_int64(8), ctypes.c_int64(4),
                             ctypes.c_void_p(16), 0, None), b"weights of 4")

    p = _lib.Product8Args()
    p.a = p.b = p.sa = p.sb = p.y = 16
    p.m, p.n, p.k, p.lda, p.ldb, p.ldy = 4, 8, 64, 63, 64, 8
    refused(lib.e2v2_product8(ctypes.byref(p), None, ctypes.c_int64(0), None), b"apart")
    p.lda = (1 << 22) + 16
    refused(lib.e2v2_product8(ctypes.byref(p), None, ctypes.c_int64(0), None), b"apart")
    p.lda, p.out_type = 64, 3
    refused(lib.e2v2_product8(ctypes.byref(p), None, ctypes.c_int64(0), None), b"output type")
    p.out_type, p.offsets = 0, 16
    refused(lib.e2v2_product8(ctypes.byref(p), None, ctypes.c_int64(0), None), b"0 experts")
    p.offsets, p.lda, p.ldb, p.m, p.n, p.k = None, 1 << 16, 1 << 16, 100, 128, 1 << 16
    p.ldy = 128
    need = lib.e2v2_product8_workspace(100, 128, 1 << 16)
    assert need > 0
    refused(lib.e2v2_product8(ctypes.byref(p), ctypes.c_void_p(16), ctypes.c_int64(need - 1), None), b"workspace")

    e = _lib.ExpertArgs()
    e.x = e.w = e.gy = e.y = e.offsets = 16
    e.rows, e.n, e.k, e.ldx, e.ldw, e.ldgy, e.ldy = 4, 8, 16, 16, 16, 8, 8
    refused(lib.e2v2_expert_product(ctypes.byref(e), 0, None, ctypes.c_int64(0), None), b"0 experts")
    e.experts, e.type = 2, 5
    refused(lib.e2v2_expert_product(ctypes.byref(e), 0, None, ctypes.c_int64(0), None), b"type 5")
    e.type = 0
    refused(lib.e2v2_expert_product(ctypes.byref(e), 3, None, ctypes.c_int64(0), None), b"pass 3")
    e.ldx = 15
    refused(lib.e2v2_expert_product(ctypes.byref(e), 0, None, ctypes.c_int64(0), None), b"row strides")
    e.ldx, e.x = 16, 18
    refused(lib.e2v2_expert_product(ctypes.byref(e), 0, None, ctypes.c_int64(0), None), b"misaligned")


def test_out_counts_as_changed(monkeypatch):
    """out= is written past torch: autograd is told, so that a graph that saved the old elements raises."""
    x, w, offs = _gpu(5, 16), _gpu(2, 8, 16), _i32(0, 2, 5)
    buf = torch.zeros(5, 8)
    gain = torch.ones(5, 8, requires_grad=True)
    monkeypatch.setattr(experts, "_launch", lambda *a: a[5])
    monkeypatch.setattr(experts, "_product", lambda *a: a[7])
    xq, wq = x.to(F8), w.to(F8)
    for call in (lambda out: experts.expert_linear(x, w, offs, out=out),
                 lambda out: experts.expert_gemm_fp8(xq, _gpu(5, 1, dtype=U8), wq, _gpu(2, 1, 1, dtype=U8), offs, out=out)):
        z = buf * gain
        assert call(buf.as_subclass(_OnGpu)) is not None
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
    with torch.inference_mode():
        out = _gpu(5, 8)
        experts.expert_linear(x, w, offs, out=out)


def test_out_may_not_share_elements_with_offsets_or_scales():
    """Other workgroups still read those while rows are stored."""
    x, w, offs = _gpu(5, 16), _gpu(2, 8, 16), _i32(0, 2, 5)
    store = torch.zeros(4096, dtype=U8)

    def at(first, dtype, *shape):
        n = torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()
        return store[first:first + n].view(dtype).view(shape).as_subclass(_OnGpu)

    out = at(1024, torch.float32, 5, 8)                  # bytes 1024 to 1184
    xq, sx, wq, sw = x.to(F8), _gpu(5, 1, dtype=U8), w.to(F8), _gpu(2, 1, 1, dtype=U8)
    for first in (1016, 1024, 1100, 1180):
        held = at(first, torch.int32, 3)
        held.copy_(offs)
        with pytest.raises(ValueError, match="shares elements"):
            experts.expert_linear(x, w, held, out=out)
        with pytest.raises(ValueError, match="shares elements"):
            experts.expert_gemm_fp8(xq, sx, wq, sw, held, out=out)
    for first in (1020, 1024, 1183):
        with pytest.raises(ValueError, match="shares elements"):
            experts.expert_gemm_fp8(xq, at(first, U8, 5, 1), wq, sw, offs, out=out)
        with pytest.raises(ValueError, match="shares elements"):
            experts.expert_gemm_fp8(xq, sx, wq, at(first + (first == 1020) * 3, U8, 2, 1, 1), offs, out=out)
    assert not experts._overlap(out, at(1012, torch.int32, 3)) and not experts._overlap(out, at(1184, U8, 5, 1))


def test_traces(monkeypatch):
    """A trace gets Functions, which it replays; what is none is refused."""
    x, w, offs = _gpu(5, 16), _gpu(2, 8, 16), _i32(0, 2, 5)
    xq, sx, wq, sw = x.to(F8), _gpu(5, 1, dtype=U8), w.to(F8), _gpu(2, 1, 1, dtype=U8)
    monkeypatch.setattr(torch.jit, "is_tracing", lambda: True)
    for fn in (norms._LayerNormFn, norms._RmsNormFn, fp8._LinearFn, experts._ExpertLinearFn):
        monkeypatch.setattr(fn, "apply", lambda *a, fn=fn: fn)
    assert norms.layer_norm(x) is norms._LayerNormFn and norms.rms_norm(x) is norms._RmsNormFn
    assert norms.rms_norm(x, residual=x) is norms._RmsNormFn and fp8.linear(x, w[0]) is fp8._LinearFn
    assert experts.expert_linear(x, w, offs) is experts._ExpertLinearFn
    for call in (lambda: norms.rms_norm_fp8(x), lambda: fp8.quantize(x), lambda: fp8.dequantize(xq, sx),
                 lambda: fp8.gemm(xq, sx, wq[0], sw[0]), lambda: experts.expert_linear(x, w, offs, out=_gpu(5, 8)),
                 lambda: experts.expert_gemm_fp8(xq, sx, wq, sw, offs)):
        with pytest.raises(RuntimeError, match="torch.jit.trace"):
            call()


def test_codes_with_a_history_are_refused():
    """Codes cast from values that need gradients need them too: their products have none."""
    x = torch.rand(5, 16, requires_grad=True)
    (xq, sx), (wq, sw), offs = (x.to(F8).as_subclass(_OnGpu), _gpu(5, 1, dtype=U8)), (_gpu(8, 16, dtype=F8),
                                                                                    _gpu(1, 1, dtype=U8)), _i32(0, 2, 5)
    wx = torch.rand(2, 8, 16, requires_grad=True).to(F8).as_subclass(_OnGpu)
    calls = [lambda: fp8.dequantize(xq, sx), lambda: fp8.gemm(xq, sx, wq, sw), lambda: fp8.gemm(wq, _gpu(8, 1, dtype=U8), xq, sx),
             lambda: experts.expert_gemm_fp8(xq, sx, wq[None], sw[None], offs[:2]),
             lambda: experts.expert_gemm_fp8(_gpu(5, 16, dtype=F8), sx, wx, _gpu(2, 1, 1, dtype=U8), offs)]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradients"):
            call()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones(5, 16)).to(F8)
        xq = dual.as_subclass(_OnGpu)
        assert norms.has_tangent(xq)
        for call in calls[:2]:
            with pytest.raises(RuntimeError, match="no gradients"):
                call()


def test_linear_takes_many_rows_where_the_weight_needs_no_gradient(monkeypatch):
    """Only the weight's gradient reads codes whose rows are as long as x has rows."""
    monkeypatch.setattr(fp8, "_linear_forward", lambda *a: ("forward",))
    monkeypatch.setattr(fp8._LinearFn, "apply", lambda *a: "function")
    many = fp8.MAX_PITCH + 16
    x, w = _gpu(1, 16).expand(many, 16), _gpu(8, 16)
    trained = torch.nn.Parameter(torch.zeros(8, 16)).as_subclass(_OnGpu)
    assert fp8.linear(x, w) == "forward" and fp8.linear(x.detach().requires_grad_(True), w) == "function"
    with torch.no_grad():
        assert fp8.linear(x, trained) == "forward"
    assert fp8.linear(x[16:], trained) == "function"
    with pytest.raises(ValueError, match="linear: sizes up to"):
        fp8.linear(x, trained)
    for shape in ((many, 16), (16, many)):
        with pytest.raises(ValueError, match="linear: sizes up to"):
            fp8.linear(_gpu(1, 1).expand(1, shape[1]), _gpu(1, 1).expand(*shape))


def test_rows_far_apart_are_copied():
    """Rows of codes further apart than the kernels take."""
    wide = torch.arange(3, dtype=U8)[:, None].expand(3, 96).contiguous()
    far = torch.empty_strided((3, 96), (fp8.MAX_PITCH + 16, 1), dtype=U8).copy_(wide).view(F8)
    rows, ld = fp8._row_operand("gemm", far)
    assert ld == 96 and rows.is_contiguous() and torch.equal(rows.view(U8), wide)
    near = torch.empty_strided((3, 96), (fp8.MAX_PITCH, 1), dtype=U8).view(F8)
    assert fp8._row_operand("gemm", near)[0] is near
    one = torch.zeros(1, 1, dtype=U8).view(F8).expand(2, fp8.MAX_PITCH + 16)
    with pytest.raises(ValueError, match="rows of 4194320"):
        fp8._row_operand("gemm", one)


def test_row_strides_whose_bytes_pass_64_bits_are_refused():
    lib = _lib.load()
    for field, which in (("ldx", 0), ("ldw", 0), ("ldgy", 1), ("ldw", 1), ("ldgy", 2), ("ldx", 2)):
        for far in (1 << 62, (1 << 61) + 16, (1 << 20) + 1):
            e = _lib.ExpertArgs()
            e.x = e.w = e.gy = e.y = e.offsets = 16
            e.rows, e.n, e.k, e.ldx, e.ldw, e.ldgy, e.ldy, e.experts = 4, 16, 16, 16, 16, 16, 16, 2
            setattr(e, field, far)
            assert lib.e2v2_expert_product(ctypes.byref(e), which, None, ctypes.c_int64(0), None) != 0
            assert b"row strides" in lib.e2v2_last_error(), (field, which, far, lib.e2v2_last_error())
