"""norms.layer_norm (csrc/norm.hip) against the definition in float64: values, first-order gradients, the gradients
of those gradients, the layouts and sizes at which each kernel variant begins and ends, and the calls around it
(streams, graph replays, the training path's module sequences).

Tolerances.  u = 2^-24 is half a step of fp32, uT half a step of the rows' type.  A row's sum passes at most 16
additions in a lane and 10 across lanes and wavefronts, so a mean is off by at most 26 u of the mean magnitude; with
the subtraction, the square root and the products around it every factor below carries less than 64 u of the
magnitudes that enter it.  A centred element x - <x> is off by 64 u (|x| + <|x|>), absolute: relative to a row's spread
that is the row's condition k = r max|x|, so
    |dxh| <= 64 u (|xh| + k),      |dy| <= |g| |dxh| + 64 u (|g xh| + |b|) + uT |y|,
    |dgx| <= 64 u (1 + k) r (|u| + <|u|> + |xh| <|u xh|> + |xh| <|u|>) + uT |gx|,
and a sum over n rows passes n / 1024 + 96 additions:
    |ddg| <= (n / 1024 + 96 + 64 (1 + k)) u sum (|gy xh| + |gy|) + uT |dg|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
UT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
EPS = 1e-5


def _inputs(n, w, dtype, wdtype, seed, cuda):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, w, generator=g) * 1.5 + 0.3 + torch.randn(n, 1, generator=g)).to(dtype).to(cuda)
    gy = torch.randn(n, w, generator=g).to(dtype).to(cuda)
    wt = (1 + 0.3 * torch.randn(w, generator=g)).to(wdtype).to(cuda)
    b = (0.5 * torch.randn(w, generator=g)).to(wdtype).to(cuda)
    return x, gy, wt, b


def _ref(x, w, b):
    z = x - x.mean(-1, keepdim=True)
    return z / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS) * w + b


def _check_first(x, gy, w, b, y, gx, gg, gb):
    """Every element of the forward and first-order results within the bounds above."""
    n, dt = x.shape[0], x.dtype
    X, G, W, B = (t.detach().double() for t in (x, gy, w, b))
    r = 1 / torch.sqrt(((X - X.mean(-1, keepdim=True)) ** 2).mean(-1, keepdim=True) + EPS)
    xh, u = (X - X.mean(-1, keepdim=True)) * r, G * W
    k = r * X.abs().amax(-1, keepdim=True)

    def mean(t):
        return t.mean(-1, keepdim=True)

    yy = xh * W + B
    tol = W.abs() * 64 * U * (xh.abs() + k) + 64 * U * ((W * xh).abs() + B.abs()) + 1.01 * UT[dt] * yy.abs()
    assert (y.double() - yy).abs().le(tol).all(), "y"
    gxx = r * (u - mean(u) - xh * mean(u * xh))
    tol = (64 * U * (1 + k) * r * (u.abs() + mean(u.abs()) + xh.abs() * mean((u * xh).abs()) + xh.abs() * mean(u.abs()))
           + 1.01 * UT[dt] * gxx.abs())
    assert (gx.double() - gxx).abs().le(tol).all(), "gx"
    kk = float(k.max()) if n else 0.0
    for got, ref, mag in ((gg, (G * xh).sum(0), ((G * xh).abs() + G.abs()).sum(0)), (gb, G.sum(0), G.abs().sum(0))):
        tol = (n / 1024 + 96 + 64 * (1 + kk)) * U * mag + 1.01 * UT[got.dtype] * ref.abs()
        assert (got.double() - ref).abs().le(tol).all(), "parameters"


WIDTHS = [1, 2, 3, 5, 8, 9, 16, 17, 31, 32, 33, 64, 65, 100, 128, 129, 255, 256, 257, 512, 520, 1000, 1024, 1025, 1032,
          2048, 2049, 4096,
          4097, 4104, 5001, 8192, 8193, 16383, 16384]


@pytest.mark.parametrize("w", WIDTHS)
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float32)])
def test_values_and_first_order(pkg, cuda, w, dtype, wdtype):
    from ubio_molfm_amd import norms
    for n in (1, 37):
        x, gy, wt, b = _inputs(n, w, dtype, wdtype, 100 * w + n, cuda)
        with torch.no_grad():
            plain = norms.layer_norm(x, wt, b, EPS)
        leaves = [t.requires_grad_(True) for t in (x, wt, b)]
        y = norms.layer_norm(x, wt, b, EPS)
        assert torch.equal(y, plain) and y.dtype == dtype
        gx, gg, gb = torch.autograd.grad(y, leaves, gy)
        assert gx.dtype == dtype and gg.dtype == gb.dtype == wdtype
        _check_first(x, gy, wt, b, y, gx, gg, gb)


@pytest.mark.parametrize("w", [1, 7, 15, 24, 60, 128, 129, 300, 1000])
def test_many_rows(pkg, cuda, w):
    """More rows than a pass of all workgroups holds: each strides over several."""
    from ubio_molfm_amd import norms
    n = 16 * 1024 + 5003
    x, gy, wt, b = _inputs(n, w, torch.float32, torch.float32, w, cuda)
    leaves = [t.requires_grad_(True) for t in (x, wt, b)]
    y = norms.layer_norm(x, wt, b, EPS)
    one = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    _check_first(x, gy, wt, b, y, *one)
    two = torch.autograd.grad(y, leaves, gy)
    assert all(torch.equal(s, t) for s, t in zip(one, two))          # the sums' order is fixed


def test_second_order(pkg, cuda):
    """L = <gx, R0> + <dg, R1> + <db, R2>, differentiated in x, the weight, the bias and gy.  Five dependent row sums,
    each within 64 u of magnitudes that are at most four times the result's in the 2-norm: 2e-5 relative, plus the
    type's half step for each of two roundings (of gx or its factor, and of the result)."""
    from ubio_molfm_amd import norms
    for w, n, dtype in [(1, 5, torch.float32), (16, 300, torch.float32), (100, 40, torch.float32),
                        (128, 20000, torch.float32), (129, 777, torch.float32), (256, 1, torch.float32),
                        (1000, 33, torch.float32), (1024, 257, torch.float32), (2048, 64, torch.float32),
                        (4097, 19, torch.float32), (8192, 9, torch.float32), (16384, 5, torch.float32),
                        (16383, 3, torch.float32), (129, 65, torch.bfloat16), (512, 65, torch.bfloat16),
                        (2048, 31, torch.float16), (16384, 3, torch.bfloat16)]:
        x, gy, wt, b = _inputs(n, w, dtype, dtype, 7 * w + n, cuda)
        g = torch.Generator().manual_seed(n)
        R = [torch.randn(*s, generator=g).to(dtype).to(cuda) for s in ((n, w), (w,), (w,))]

        def run(f, cast):
            X, G, W, B = (cast(t).detach().requires_grad_(True) for t in (x, gy, wt, b))
            y = f(X, W, B)
            first = torch.autograd.grad(y, (X, W, B), G, create_graph=True)
            second = torch.autograd.grad(first, (X, W, B, G), [cast(r) for r in R], allow_unused=True)
            return [y, *first, *(torch.zeros_like(B) if t is None else t for t in second)]

        got = run(lambda X, W, B: norms.layer_norm(X, W, B, EPS), lambda t: t)
        ref = run(_ref, lambda t: t.double())
        for name, a, r in zip(["y", "gx", "dg", "db", "d2x", "d2g", "d2b", "d2gy"], got, ref):
            if w == 1 and name in ("gx", "dg", "d2x", "d2g"):
                assert a.double().abs().max() < 1e-6      # one element a row: centred it is zero
                continue
            rel = float((a.double() - r).norm() / r.norm()) if r.norm() > 0 else float(a.double().norm())
            assert rel < 2e-5 + (0 if dtype == torch.float32 else 2 * UT[dtype]), (w, n, dtype, name, rel)


def test_gradient_against_differences(pkg, cuda):
    """The gradient along a direction against central differences of the kernel's own forward pass (h = 2^-6).  The
    difference's truncation is taken from the same difference in float64; the kernel's rounding enters with at most
    64 u (2 + k) |R| (|g| + |b|) an element and side, divided by 2 h."""
    from ubio_molfm_amd import norms
    n, w, h = 31, 33, 2.0 ** -6
    x, R, wt, b = _inputs(n, w, torch.float32, torch.float32, 3, cuda)
    d = torch.randn(n, w, generator=torch.Generator().manual_seed(9)).to(cuda)

    def at(f, s, cast):
        return (f(cast(x) + s * cast(d), cast(wt), cast(b)).double() * R.double()).sum()

    x.requires_grad_(True)
    gx, = torch.autograd.grad(norms.layer_norm(x, wt, b, EPS), x, R)
    x = x.detach()
    got = float((gx.double() * d.double()).sum())
    diff = float((at(lambda *a: norms.layer_norm(*a, EPS), h, lambda t: t)
                  - at(lambda *a: norms.layer_norm(*a, EPS), -h, lambda t: t)) / (2 * h))
    x64 = x.double().requires_grad_(True)
    g64, = torch.autograd.grad(_ref(x64, wt.double(), b.double()), x64, R.double())
    diff64 = float((at(_ref, h, lambda t: t.double()) - at(_ref, -h, lambda t: t.double())) / (2 * h))
    trunc = abs(diff64 - float((g64 * d.double()).sum()))
    k = float((x.abs().amax(-1) / x.std(-1)).max()) + 1
    noise = float((64 * U * (2 + k) * R.abs().double() * (wt.abs() + b.abs()).double()).sum()) / h
    assert abs(got - diff) <= 2 * trunc + noise and noise < 0.05 * float(gx.double().norm() * d.double().norm())


@pytest.mark.parametrize("affine", ["none", "weight", "bias"])
def test_absent_parameters(pkg, cuda, affine):
    from ubio_molfm_amd import norms
    x, gy, wt, b = _inputs(50, 96, torch.float32, torch.float32, 11, cuda)
    x.requires_grad_(True)
    W = wt.requires_grad_(True) if affine == "weight" else None
    B = b.requires_grad_(True) if affine == "bias" else None
    y = norms.layer_norm(x, W, B, EPS)
    one, zero = torch.ones_like(wt), torch.zeros_like(b)
    leaves = [t for t in (x, W, B) if t is not None]
    got = torch.autograd.grad(y, leaves, gy, create_graph=True)
    ref_leaves = [t.detach().double().requires_grad_(True) for t in leaves]
    it = iter(ref_leaves)
    X = next(it)
    ref_y = _ref(X, next(it) if W is not None else one.detach().double(),
                 next(it) if B is not None else zero.detach().double())
    ref = torch.autograd.grad(ref_y, ref_leaves, gy.double(), create_graph=True)
    for a, r in zip((y, *got), (ref_y, *ref)):
        assert float((a.double() - r).norm() / r.norm()) < 64 * U
    a, = torch.autograd.grad(got[0].square().sum(), x)
    r, = torch.autograd.grad(ref[0].square().sum(), X)
    assert float((a.double() - r).norm() / r.norm()) < 2e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(pkg, cuda, dtype):
    """Rows of a wider matrix, rows off 16-byte boundaries, every second row, a transposed operand, one row broadcast,
    and upstream gradients that lie in those ways: bitwise the results of contiguous copies, in which the same sums run
    (where the layout takes the elementwise variant, within its bounds)."""
    from ubio_molfm_amd import norms
    n, w = 45, 128
    g = torch.Generator().manual_seed(2)
    big = torch.randn(2 * n + 2, 3 * w, generator=g).to(dtype).to(cuda)
    base = torch.randn(w, n, generator=g).to(dtype).to(cuda)
    wt = torch.randn(w, generator=g).to(cuda)
    b = torch.randn(w, generator=g).to(cuda)
    layouts = {"columns": big[:n, w:2 * w], "shifted": big[:n, 3:3 + w], "every second": big[:2 * n:2, :w],
               "transposed": base.t(), "broadcast": big[:1, :w].expand(n, w),
               "blocks": big[:2 * 20].view(2, 20, -1)[..., :w]}
    for name, x in layouts.items():
        for gy_name in (name, "plain"):
            X = x.detach().clone().requires_grad_(True)
            G = torch.randn(x.shape, generator=g).to(dtype).to(cuda) if gy_name == "plain" else x
            ref_y = norms.layer_norm(X, wt, b)
            ref, = torch.autograd.grad(ref_y, X, G.clone())
            xx = x.detach().requires_grad_(True)
            y = norms.layer_norm(xx, wt, b)
            assert y.is_contiguous()
            got, = torch.autograd.grad(y, xx, G)
            if name == "shifted":
                assert torch.allclose(y.float(), ref_y.float(), atol=1e-4 if dtype == torch.float32 else 0.05)
                rel = float((got.double() - ref.double()).norm() / ref.double().norm())
                assert rel < 64 * U + (0 if dtype == torch.float32 else 2 * UT[dtype]), (name, rel)
            else:
                assert torch.equal(y, ref_y) and torch.equal(got, ref), (name, gy_name)


def test_rows_do_not_mix(pkg, cuda):
    """Constant rows, infinite and NaN elements stay in their rows; constant rows give the bias."""
    from ubio_molfm_amd import norms
    for w in (24, 128, 300, 2048):
        x, gy, wt, b = _inputs(64, w, torch.float32, torch.float32, w, cuda)
        clean = x.clone()
        x[3] = 2.5
        x[7, 1], x[20, 5], x[41] = float("nan"), float("inf"), float("-inf")
        bad = torch.zeros(64, dtype=torch.bool, device=cuda)
        bad[[7, 20, 41]] = True
        X = x.requires_grad_(True)
        y = norms.layer_norm(X, wt, b, EPS)
        gx, = torch.autograd.grad(y, X, gy)
        C = clean.requires_grad_(True)
        y0 = norms.layer_norm(C, wt, b, EPS)
        gx0, = torch.autograd.grad(y0, C, gy)
        assert torch.equal(y[3], b) and gx[3].isfinite().all()
        ok = ~bad
        ok[3] = False
        assert torch.equal(y[ok], y0[ok]) and torch.equal(gx[ok], gx0[ok])
        assert y[bad].isnan().all() and gx[bad].isnan().all()


def test_no_rows(pkg, cuda):
    from ubio_molfm_amd import norms
    x = torch.empty(0, 128, device=cuda, requires_grad=True)
    w = torch.ones(128, device=cuda, requires_grad=True)
    b = torch.ones(128, device=cuda, requires_grad=True)
    y = norms.layer_norm(x, w, b)
    gx, gg, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == gx.shape == (0, 128) and not gg.any() and not gb.any()


def test_streams_and_graph(pkg, cuda):
    """Two streams at once, then a captured step replayed on new inputs with eager work between."""
    from ubio_molfm_amd import norms
    x, gy, wt, b = _inputs(3000, 256, torch.float32, torch.float32, 5, cuda)

    def step(x, gy):
        X, W, B = (t.detach().requires_grad_(True) for t in (x, wt, b))
        y = norms.layer_norm(X, W, B)
        gx, = torch.autograd.grad(y, X, gy, create_graph=True)
        return [y.detach(), gx.detach(), *torch.autograd.grad(gx.square().sum(), (X, W))]

    want = [t.clone() for t in step(x, gy)]
    want2 = [t.clone() for t in step(2 * gy, x)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s, args in zip(streams, ((x, gy), (2 * gy, x))):
        with torch.cuda.stream(s):
            outs.append(step(*args))
    torch.cuda.synchronize()
    for out, ref in zip(outs, (want, want2)):
        assert all(torch.equal(a, r) for a, r in zip(out, ref))
    del outs
    sx, sg = x.clone(), gy.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(sx, sg)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(sx, sg)
    for args, ref in (((x, gy), want), ((2 * gy, x), want2), ((x, gy), want)):
        sx.copy_(args[0])
        sg.copy_(args[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, r) for a, r in zip(res, ref))
        step(gy, x)                                                   # eager work between replays


def test_frozen_parameters_and_third_order(pkg, cuda):
    from ubio_molfm_amd import norms
    x, gy, wt, b = _inputs(20, 64, torch.float32, torch.float32, 6, cuda)
    X = x.requires_grad_(True)
    W = wt.requires_grad_(True)
    gx, = torch.autograd.grad(norms.layer_norm(X, W, b), X, gy, create_graph=True)
    d2, = torch.autograd.grad(gx.square().sum(), X, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d2.sum(), X)
    y = norms.layer_norm(x.detach(), W, b)                            # rows without a gradient
    gg, = torch.autograd.grad(y, W, gy)
    xd = x.detach().double()
    ref = (gy.double() * _ref(xd, 1.0, 0.0)).sum(0)
    assert float((gg.double() - ref).norm() / ref.norm()) < 64 * U


@pytest.mark.parametrize("w,silu", [(128, False), (96, True), (33, True), (640, False)])
def test_run_seq_uses_it(pkg, cuda, w, silu, monkeypatch):
    """A net whose LayerNorm the fused LayerNorm + SiLU is not built for, or that has no SiLU behind it, through the
    training path's run_seq, to second order, against the modules in float64."""
    import copy
    from ubio_molfm_amd import _lib
    from ubio_molfm_amd import second_order as so
    torch.manual_seed(w)
    mods = [torch.nn.Linear(24, w), torch.nn.LayerNorm(w), *([torch.nn.SiLU()] if silu else []), torch.nn.Linear(w, 5)]
    net = torch.nn.Sequential(*mods).to(cuda)
    with torch.no_grad():
        net[1].weight.normal_(1, 0.3)
        net[1].bias.normal_(0, 0.5)
    p = torch.randn(70, 24, device=cuda)
    called = []
    real = _lib.call
    monkeypatch.setattr(_lib, "call", lambda name, *a: (called.append(name), real(name, *a))[1])

    def run(f, net, p):
        p = p.requires_grad_(True)
        e = torch.tanh(f(net, p)).square().sum()
        gp, = torch.autograd.grad(e, p, create_graph=True)
        return [gp, *torch.autograd.grad(gp.square().sum() + e, [p, *net[1].parameters()])]

    got = run(so.run_seq, net, p.clone())
    assert {"e2v2_layer_norm_fwd", "e2v2_layer_norm_bwd", "e2v2_layer_norm_bwd2"} <= set(called)
    ref = run(lambda m, h: m(h), copy.deepcopy(net).double(), p.double())
    for a, r in zip(got, ref):
        # the linears' fp32 products are in it too: the bound of ln_silu's own test
        assert float((a.double() - r).norm() / r.norm()) < 1e-4


def test_run_seq_calls_modules_that_do_more(pkg, cuda):
    """Hooks on a LayerNorm and subclasses of it run as they do in nn.Sequential."""
    from ubio_molfm_amd import second_order as so

    class Scaled(torch.nn.LayerNorm):
        def forward(self, x):
            return 3 * super().forward(x)

    x = torch.randn(7, 24, device=cuda)
    hooked = torch.nn.LayerNorm(24).to(cuda)
    hooked.register_forward_hook(lambda m, i, o: o + 1)
    for net in (torch.nn.Sequential(hooked), torch.nn.Sequential(Scaled(24).to(cuda))):
        assert torch.equal(so.run_seq(net, x), net(x))


@pytest.mark.parametrize("frozen", [True, False])
def test_run_seq_under_transforms(pkg, cuda, frozen):
    """Forward-mode tangents, torch.func's transforms and a trace go through the module, as in nn.Sequential."""
    from torch.autograd import forward_ad
    from ubio_molfm_amd import second_order as so
    torch.manual_seed(5)
    net = torch.nn.Sequential(torch.nn.Linear(6, 24), torch.nn.LayerNorm(24), torch.nn.Linear(24, 3)).to(cuda)
    net.requires_grad_(not frozen)
    x, t = torch.randn(7, 6, device=cuda), torch.randn(7, 6, device=cuda)

    def both(f):
        got, ref = f(lambda v: so.run_seq(net, v)), f(net)
        assert len(got) == len(ref) and all(torch.equal(a, r) for a, r in zip(got, ref))

    def dual(f):
        with forward_ad.dual_level():
            y = forward_ad.unpack_dual(f(forward_ad.make_dual(x, t)))
            assert y.tangent is not None
            return [y.primal.detach().clone(), y.tangent.detach().clone()]

    both(dual)
    both(lambda f: [torch.func.vmap(f)(torch.stack([x, t]))])
    both(lambda f: list(torch.func.jvp(f, (x,), (t,))))
    both(lambda f: [torch.func.grad(lambda v: f(v).square().sum())(x)])
    if frozen:                                     # a trace takes no trainable tensor for a constant
        traced = torch.jit.trace(lambda v: so.run_seq(net, v), (x,))
        assert torch.equal(traced(t), net(t))


@pytest.mark.parametrize("affine", [True, False])
def test_run_seq_to_third_order(pkg, cuda, affine):
    """A LayerNorm in a module sequence is differentiable as often as the module.  Up to the third derivative some 15
    dependent row sums lie behind one another, each within 64 u of magnitudes that are at most four times the result's
    in the 2-norm: 15 * 64 * 4 u = 2.3e-4."""
    import copy
    from ubio_molfm_amd import second_order as so
    torch.manual_seed(8)
    net = torch.nn.Sequential(torch.nn.LayerNorm(40, elementwise_affine=affine)).to(cuda)
    if affine:
        with torch.no_grad():
            net[0].weight.normal_(1, 0.3)
            net[0].bias.normal_(0, 0.5)
    x, R = torch.randn(9, 40, device=cuda), torch.randn(9, 40, device=cuda)

    def run(f, net, x, R):
        x = x.requires_grad_(True)
        leaves = [x, *net.parameters()]
        out = [f(net, x)]
        for k in range(3):
            out += [g for g in torch.autograd.grad((out[-1] * R).square().sum() if k else (out[0] ** 3 * R).sum(), leaves,
                                                   create_graph=True, allow_unused=True) if g is not None][::-1]
        return [t.detach() for t in out]

    got = run(so.run_seq, net, x.clone(), R)
    # by elementary operators: torch's layer_norm holds mean and rstd for constants from the third derivative on (8% off
    # here, in float64)
    ref = run(lambda m, v: _ref(v, *(m[0].weight, m[0].bias) if affine else (1.0, 0.0)), copy.deepcopy(net).double(),
              x.double(), R.double())
    assert len(got) == len(ref)
    for a, r in zip(got, ref):
        assert float((a.double() - r).norm() / r.norm()) < 64 * 60 * U


def test_run_seq_with_hooks_for_all_modules(pkg, cuda):
    from ubio_molfm_amd import second_order as so
    net = torch.nn.Sequential(torch.nn.Linear(8, 24), torch.nn.LayerNorm(24)).to(cuda)
    x = torch.randn(7, 8, device=cuda)
    seen = []
    handle = torch.nn.modules.module.register_module_forward_hook(
        lambda m, i, o: (seen.append(type(m)), 2 * o)[1] if isinstance(m, torch.nn.LayerNorm) else None)
    try:
        assert torch.equal(so.run_seq(net, x), net(x)) and seen == [torch.nn.LayerNorm] * 2
    finally:
        handle.remove()


@pytest.mark.parametrize("which", ["norm hook", "silu hook", "norm subclass", "linear hook", "none"])
def test_run_seq_with_hooks_behind_fused_pairs(pkg, cuda, which):
    """Widths and rows that the fused LayerNorm + SiLU and the Linear over edges take: hooks and subclasses still run."""
    from ubio_molfm_amd import second_order as so

    class Scaled(torch.nn.LayerNorm):
        def forward(self, x):
            return 3 * super().forward(x)

    torch.manual_seed(4)
    net = torch.nn.Sequential(torch.nn.Linear(8, 128), (Scaled if which == "norm subclass" else torch.nn.LayerNorm)(128),
                              torch.nn.SiLU()).to(cuda)
    seen = []
    k = {"linear hook": 0, "norm hook": 1, "silu hook": 2}.get(which)
    if k is not None:
        net[k].register_forward_hook(lambda m, i, o: (seen.append(k), o + 1)[1])
    x = torch.randn(so._EDGE_ROWS, 8, device=cuda)
    with torch.no_grad():
        got, ref = so.run_seq(net, x), net.double()(x.double())
    # a Linear of 8 products, a norm of 128 elements and a SiLU: below 200 u of values below 30
    assert (got.double() - ref).abs().max() < 200 * U * 30 and len(seen) == (0 if k is None else 2)


@pytest.mark.parametrize("w", [3, 24, 100, 129, 500, 1000, 1500, 5001, 8193, 16383])
def test_rows_of_one_value(pkg, cuda, w):
    """They give the bias, whatever the value: a mean off by its sum's rounding (at most 48 u: 32 additions in a lane, 16
    across) is found again with the same relative error, and 48^2 u^2 |x| r |g| is left, r = eps^(-1/2).  Rows between
    them that are not constant, or not in the same way, come out as alone."""
    from ubio_molfm_amd import norms
    values = torch.tensor([0.1, 1000.1, -37.77, 30000.3, 1e-6, 7.0, -0.3], device=cuda)
    x, gy, wt, b = _inputs(40, w, torch.float32, torch.float32, w, cuda)
    plain = norms.layer_norm(x, wt, b, EPS)
    mixed = x.clone()
    mixed[3:38:5] = values[:, None]
    X = mixed.requires_grad_(True)
    y = norms.layer_norm(X, wt, b, EPS)
    rest = torch.ones(40, dtype=torch.bool, device=cuda)
    rest[3:38:5] = False
    assert torch.equal(y[rest], plain[rest])
    r = EPS ** -0.5
    left = 48 ** 2 * U * U * values.abs().double()[:, None] * r
    assert (y[~rest].double() - b.double()).abs().le(left * wt.abs() + U * b.abs()).all()
    gx, = torch.autograd.grad(y, X, gy)
    u = gy[~rest].double() * wt.double()
    ref = r * (u - u.mean(-1, keepdim=True))
    size = u.abs() + u.abs().mean(-1, keepdim=True)
    # the mean is stored in fp32, off by u |x|: xh <u xh> beside it
    xh = left + U * values.abs().double()[:, None] * r
    assert (gx[~rest].double() - ref).abs().le(64 * U * r * size + r * xh * xh * size + U * ref.abs()).all()


def test_rows_far_narrower_than_their_mean(pkg, cuda):
    """A spread of 2^-12 to 2^-6 of the mean on both sides of where the mean is corrected: where it is, y is off by what
    the rounding of x - mean leaves (4 u of the mean, 64 u of the rest), elsewhere by the mean's 48 u."""
    from ubio_molfm_amd import norms
    g = torch.Generator().manual_seed(6)
    for w in (24, 129, 1000, 5001):
        for e in range(6, 13):
            x = (100 + 100 * 2.0 ** -e * torch.randn(50, w, generator=g)).to(cuda)
            y = norms.layer_norm(x, eps=1e-12).double()
            X = x.double()
            z = X - X.mean(-1, keepdim=True)
            ref = z / ((z * z).mean(-1, keepdim=True) + 1e-12).sqrt()
            bound = (4 if e > 8 else 48) * U * 2.0 ** e * 1.5 + 64 * U * (ref.abs() + 1)
            assert (y - ref).abs().le(bound).all(), (w, e, float((y - ref).abs().max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w", [5, 31, 128, 129, 700, 2049])
def test_rows_off_16_byte_boundaries(pkg, cuda, dtype, w):
    """Every start and stride of rows, and of upstream gradients, runs the code of contiguous ones: bitwise its results
    to second order."""
    from ubio_molfm_amd import norms
    x, gy, wt, b = _inputs(37, w, dtype, torch.float32, 3 * w, cuda)
    q = gy.roll(1, 0)

    def run(x, gy, q):
        X, G, W = (t.detach().requires_grad_(True) for t in (x, gy, wt))
        y = norms.layer_norm(X, W, b, EPS)
        gx, gg = torch.autograd.grad(y, (X, W), G, create_graph=True)
        return [y, gx, gg, *torch.autograd.grad(gx, (X, G, W), q)]

    def placed(t, shift, extra):
        buf = torch.full((t.shape[0], w + extra), float("nan"), dtype=dtype, device=cuda).view(-1)
        out = torch.cat([buf, buf[:16]])[shift:shift + buf.numel()].view(t.shape[0], -1)[:, :w]
        return out.copy_(t)

    ref = run(x, gy, q)
    for shift in range(1, 8):
        got = run(placed(x, shift, 3), placed(gy, 8 - shift, 5), placed(q, shift, 8))
        assert all(torch.equal(a, r) for a, r in zip(got, ref)), shift


@pytest.mark.parametrize("w,dtype", [(w, torch.float32) for w in (2, 3, 7, 15, 31, 37, 61, 85, 125, 189, 253, 300, 500,
                                                                  700, 1001, 1500, 3001, 4001, 6001, 12001)]
                         + [(w, torch.bfloat16) for w in (3, 5, 13, 27, 61, 93, 125, 189, 253, 381, 509, 765, 1021,
                                                          1501, 2049, 5001, 8001, 12001)]
                         + [(w, torch.float16) for w in (61, 765, 5001)])
def test_second_order_of_every_shape(pkg, cuda, w, dtype):
    """Each number of lanes and vectors that a row can lie in, the last vector in part; as test_second_order, with its
    bound."""
    from ubio_molfm_amd import norms
    n = 23
    x, gy, wt, b = _inputs(n, w, dtype, dtype, 11 * w, cuda)
    g = torch.Generator().manual_seed(w)
    R = [torch.randn(*s, generator=g).to(dtype).to(cuda) for s in ((n, w), (w,), (w,))]

    def run(f, cast):
        X, G, W, B = (cast(t).detach().requires_grad_(True) for t in (x, gy, wt, b))
        first = torch.autograd.grad(f(X, W, B), (X, W, B), G, create_graph=True)
        return [*first, *torch.autograd.grad(first, (X, W, G), [cast(r) for r in R])]

    got = run(lambda X, W, B: norms.layer_norm(X, W, B, EPS), lambda t: t)
    ref = run(_ref, lambda t: t.double())
    for name, a, r in zip(["gx", "dg", "db", "d2x", "d2g", "d2gy"], got, ref):
        if w == 2 and name in ("gx", "d2x"):
            continue                # two elements: x - <x> is +-d, gx all but cancels; the others see the same sums
        rel = float(((a.double() - r).norm() / r.norm()).detach())
        assert rel < 2e-5 + (0 if dtype == torch.float32 else 2 * UT[dtype]), (name, rel)


def test_run_seq_with_batched_gradients(pkg, cuda):
    """Jacobians in one call (is_grads_batched), of the sequence and of its gradient, and upstream gradients with
    forward-mode tangents: as through the modules."""
    import copy
    from torch.autograd import forward_ad
    from ubio_molfm_amd import norms, second_order as so
    torch.manual_seed(6)
    net = torch.nn.Sequential(torch.nn.Linear(6, 24), torch.nn.LayerNorm(24), torch.nn.Linear(24, 3)).to(cuda)
    ref = copy.deepcopy(net).double()
    x, t = torch.randn(5, 6, device=cuda), torch.randn(5, 3, device=cuda)

    def jacobians(f, x):
        first = torch.autograd.functional.jacobian(f, x, vectorize=True)
        x = x.clone().requires_grad_(True)
        g, = torch.autograd.grad((f(x) ** 2).sum(), x, create_graph=True)
        second, = torch.autograd.grad(g, x, torch.eye(x.numel(), device=cuda, dtype=x.dtype).view(-1, *x.shape),
                                      is_grads_batched=True)
        x = x.detach().requires_grad_(True)
        y = f(x)
        with forward_ad.dual_level():
            up = forward_ad.make_dual(torch.ones_like(y), t.to(y.dtype))
            return first, second, forward_ad.unpack_dual(torch.autograd.grad(y, x, up)[0]).tangent

    for a, r in zip(jacobians(lambda v: so.run_seq(net, v), x), jacobians(ref, x.double())):
        assert float((a.double() - r).norm() / r.norm()) < 1e-4       # as test_run_seq_uses_it
    X = x.clone().requires_grad_(True)
    y = norms.layer_norm(X)
    with pytest.raises(RuntimeError, match="batched"):
        torch.autograd.grad(y, X, torch.ones(2, 5, 6, device=cuda), is_grads_batched=True)
