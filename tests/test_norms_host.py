"""What norms.layer_norm and its entry points refuse, before any kernel or HIP call.  No GPU needed."""
import pytest
import torch
from torch.autograd import forward_ad

from ubio_molfm_amd import _lib, norms


def test_host_rows_are_refused(monkeypatch):
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("a kernel was called"))
    with pytest.raises(RuntimeError, match="GPU only"):
        norms.layer_norm(torch.rand(3, 8))
    with pytest.raises(RuntimeError, match="GPU only"):
        norms.layer_norm([1.0, 2.0])


class _OnGpu(torch.Tensor):
    """A host tensor that says it lies on the GPU: the checks behind the device's."""
    is_cuda = True


def _gpu(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(_OnGpu)


@pytest.mark.parametrize("x,kw,match", [
    (lambda: _gpu(3, 8, dtype=torch.float64), {}, "fp32, bf16 or fp16"),
    (lambda: _gpu(3, 8, dtype=torch.int32), {}, "fp32, bf16 or fp16"),
    (lambda: _gpu(), {}, "fp32, bf16 or fp16"),
    (lambda: _gpu(3, 0), {}, "width 0"),
    (lambda: _gpu(1, norms.MAX_WIDTH + 1), {}, "width 16385"),
    (lambda: _gpu(3, 8), dict(weight=torch.ones(7)), "weight"),
    (lambda: _gpu(3, 8), dict(bias=torch.ones(1, 8)), "bias"),
    (lambda: _gpu(3, 8), dict(weight=torch.ones(8, dtype=torch.bfloat16)), "weight"),
    (lambda: _gpu(3, 8, dtype=torch.bfloat16), dict(bias=torch.ones(8, dtype=torch.float16)), "bias"),
    (lambda: _gpu(3, 8), dict(weight=torch.ones(8, device="meta")), "weight"),
])
def test_refusals(x, kw, match, monkeypatch):
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("a kernel was called"))
    with pytest.raises(ValueError, match=match):
        norms.layer_norm(x(), **kw)


@pytest.mark.parametrize("which", ["rows", "weight", "bias"])
def test_forward_mode_tangents_are_refused(which, monkeypatch):
    """A result without the tangent would be a wrong derivative without a word."""
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("a kernel was called"))
    monkeypatch.setattr(norms, "_call", lambda *a: None)
    t = dict(rows=_gpu(3, 8), weight=_gpu(8), bias=_gpu(8))
    monkeypatch.setattr(_OnGpu, "get_device", lambda self: 0, raising=False)
    with forward_ad.dual_level():
        assert norms.layer_norm(t["rows"], t["weight"], t["bias"]).shape == (3, 8)     # no tangent: as ever
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            norms.layer_norm(t["rows"], t["weight"], t["bias"])


@pytest.mark.parametrize("shape,stride,ld", [
    ((4, 8), (8, 1), 8), ((4, 8), (24, 1), 24), ((4, 8), (0, 1), 0), ((2, 3, 8), (24, 8, 1), 8),
    ((2, 3, 8), (48, 16, 1), 16), ((8,), (1,), 8), ((1, 1, 8), (5, 3, 1), 8), ((2, 1, 3, 8), (72, 7, 24, 1), 24),
    ((4, 1), (3, 2), 3)])
def test_rows_that_are_read_where_they_lie(shape, stride, ld):
    t = torch.zeros(512).as_strided(shape, stride)
    u, got = norms._rows(t)
    assert u is t and got == ld


@pytest.mark.parametrize("shape,stride", [((4, 8), (1, 4)), ((4, 8), (16, 2)), ((2, 3, 8), (100, 8, 1)),
                                          ((2, 3, 8), (0, 8, 1))])
def test_rows_that_are_copied(shape, stride):
    t = torch.arange(512.0).as_strided(shape, stride)
    u, ld = norms._rows(t)
    assert u.is_contiguous() and ld == shape[-1] and torch.equal(u, t)


def test_arguments_as_bytes():
    """What _args packs is e2v2_layer_norm_args field by field."""
    x, g, b, st = torch.zeros(3, 8), torch.zeros(8), torch.zeros(8, dtype=torch.bfloat16), torch.zeros(3, 2)
    gy, qx, y, gx = (torch.zeros(3, 8) for _ in range(4))
    gy = torch.zeros(3, 16)[:, :8]
    raw, keep = norms._args(x, g, b, st, 0.5, gy=gy, qx=qx, qg=g, qb=b, y=y, gx=gx)
    assert len(raw) == _lib.C.sizeof(_lib.LayerNormArgs)
    a = _lib.LayerNormArgs.from_buffer_copy(raw)
    want = dict(x=x, gy=gy, qx=qx, g=g, b=b, qg=g, qb=b, y=y, gx=gx, stats=st)
    assert all(getattr(a, k) == t.data_ptr() for k, t in want.items())
    assert (a.n, a.ldx, a.ldgy, a.ldqx, a.w, a.type, a.g_type, a.b_type, a.eps) == (3, 8, 16, 8, 8, 0, 0, 1, 0.5)
    a = _lib.LayerNormArgs.from_buffer_copy(norms._args(x, None, None, None, 0.5)[0])
    assert a.g is None and a.gy is None and a.stats is None and a.ldgy == 0


def test_entry_point_checks():
    lib = _lib.load()
    a = _lib.LayerNormArgs()
    a.n, a.w, a.x, a.y = 4, 16, 64, 64                  # never dereferenced: the checks fail first
    for change, match in ((dict(w=0), b"width 0"), (dict(w=16385), b"width 16385"), (dict(n=-1), b"-1 rows"),
                          (dict(type=3), b"types"), (dict(g_type=-1), b"types"), (dict(ldx=-8), b"stride"),
                          (dict(x=66), b"misaligned"), (dict(stats=68), b"misaligned"), (dict(x=None), b"null")):
        b = _lib.LayerNormArgs.from_buffer_copy(a)
        for k, v in change.items():
            setattr(b, k, v)
        assert lib.e2v2_layer_norm_fwd(_lib.C.byref(b), None) != 0 and match in lib.e2v2_last_error(), change
    assert lib.e2v2_layer_norm_bwd(_lib.C.byref(a), None, None, None, _lib.i64(0), None) != 0
    assert b"null operand" in lib.e2v2_last_error()
    a.gy = a.gx = a.stats = 64
    for rows, w in ((1, 7), (999, 64), (1025, 3), (10 ** 6, 16384)):
        x = torch.empty(rows, w, device="meta")
        ws, n = norms._workspace(x)
        assert n == lib.e2v2_layer_norm_workspace(rows, w) == 4 * ws.numel()
    need = lib.e2v2_layer_norm_workspace(4, 16)
    assert need == 2 * 4 * 16 * 4 and lib.e2v2_layer_norm_workspace(0, 16) == 0
    for fn, args in ((lib.e2v2_layer_norm_bwd, (_lib.vp(64), None, _lib.vp(64))),
                     (lib.e2v2_layer_norm_bwd2, (_lib.vp(64), _lib.vp(64)))):
        assert fn(_lib.C.byref(a), *args, _lib.i64(need - 4), None) != 0 and b"workspace" in lib.e2v2_last_error()


@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("asked", ["xgb", "x", "g", "b", "xb", "gb"])
def test_the_composed_second_order(affine, asked):
    """What a third derivative differentiates, in float64: the second order's values as autograd gives them, and its own
    gradients against differences."""
    g = torch.Generator().manual_seed(3)
    x, gy, q, w, b, qg, qb = (torch.randn(*s, generator=g, dtype=torch.float64)
                              for s in ((2, 3, 5), (2, 3, 5), (2, 3, 5), (5,), (5,), (5,), (5,)))
    if not affine and asked != "x":
        return
    x, gy, w, b = (t.requires_grad_(True) for t in (x, gy, w, b))
    W = w if affine else None
    ups = {"x": q, "g": qg, "b": qb}
    first = torch.autograd.grad(torch.nn.functional.layer_norm(x, (5,), W, b if affine else None, 0.1),
                                [x, *([w, b] if affine else [])], gy, create_graph=True)
    first = dict(zip("xgb", first))
    ref = torch.autograd.grad([first[k] for k in asked], [gy, x, w], [ups[k] for k in asked], allow_unused=True)

    def second(gy, x, w):
        return norms._composed2(gy, x, w if affine else None, 0.1, *(ups[k] if k in asked else None for k in "xgb"))

    got = second(gy, x, w)
    for a, r in zip(got, ref):
        assert (a is None or not a.abs().max()) if r is None else torch.allclose(a, r, rtol=1e-11, atol=1e-12)
    if asked != "b":
        assert torch.autograd.gradcheck(lambda *t: [y for y in second(*t) if y is not None and y.requires_grad],
                                        (gy, x, w) if affine else (gy, x, w.detach()))


class _Emulated:
    """The kernels' three calls by elementary operators on host tensors."""

    def __init__(self, monkeypatch, any_order):
        monkeypatch.setattr(norms, "_forward", lambda x, g, b, eps, stats: self.norm(x, g, b, eps))
        monkeypatch.setattr(norms, "_backward",
                            lambda gy, x, g, b, stats, eps, need_g, need_b: norms._composed(gy, x, g, b, eps))
        monkeypatch.setattr(norms, "_backward2", lambda ctx, *q: (
            *norms._composed2(*ctx.saved_tensors[:3], ctx.eps, *q), *[None] * 5))
        self.any_order = any_order

    @staticmethod
    def norm(x, g, b, eps):
        z = x - x.mean(-1, keepdim=True)
        return z / ((z * z).mean(-1, keepdim=True) + eps).sqrt() * g + b

    def __call__(self, x, g, b):
        return norms._LayerNormFn.apply(x, g, b, 0.1, self.any_order)


def _operands():
    g = torch.Generator().manual_seed(4)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True) for s in ((3, 5), (5,), (5,)))
    return x, w, b, torch.randn(4, 3, 5, generator=g, dtype=torch.float64)


def test_batched_gradients(monkeypatch):
    """is_grads_batched over a module's LayerNorm (jacobians), first and second order; the public one refuses."""
    x, w, b, G = _operands()
    f, ref = _Emulated(monkeypatch, True), lambda x, w, b: _Emulated.norm(x, w, b, 0.1)
    for fn_pair in (((lambda h: h(x, w, b)), G),
                    ((lambda h: torch.autograd.grad(h(x, w, b), x, G[0], create_graph=True)[0]), G)):
        make, up = fn_pair
        got, want = (torch.autograd.grad(make(h), (x, w), up, is_grads_batched=True) for h in (f, ref))
        assert all(torch.allclose(a, r, rtol=1e-11, atol=1e-12) for a, r in zip(got, want))
    y = _Emulated(monkeypatch, False)(x, w, b)
    with pytest.raises(RuntimeError, match="batched"):
        torch.autograd.grad(y, x, G, is_grads_batched=True, retain_graph=True)
    gx, = torch.autograd.grad(y, x, G[0], create_graph=True)
    with pytest.raises(RuntimeError, match="batched"):
        torch.autograd.grad(gx, x, G, is_grads_batched=True)


def test_upstream_gradients_with_tangents(monkeypatch):
    x, w, b, G = _operands()
    f, ref = _Emulated(monkeypatch, True), lambda x, w, b: _Emulated.norm(x, w, b, 0.1)
    own = _Emulated(monkeypatch, False)

    def tangents(h, order):
        y = h(x, w, b)
        if order == 2:
            y, = torch.autograd.grad(y, x, G[2], create_graph=True)
        with forward_ad.dual_level():
            out = torch.autograd.grad(y, (x, w), forward_ad.make_dual(G[0], G[1]))
            return [forward_ad.unpack_dual(t).tangent for t in out]

    for order in (1, 2):
        for a, r in zip(tangents(f, order), tangents(ref, order)):
            assert torch.allclose(a, r, rtol=1e-11, atol=1e-12)
        with pytest.raises(RuntimeError, match="tangents"):
            tangents(own, order)
