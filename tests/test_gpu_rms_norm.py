"""norms.rms_norm and norms.rms_norm_fp8 (csrc/rms.hip) against the definition in float64: values, gradients, 8-bit codes,
the widths and layouts at which each kernel variant begins and ends, streams and graph replays.

Tolerances.  u = 2^-24 is half a step of fp32, uT half a step of the rows' type.  h is the rounded sum, compared exactly.
A row's sum of squares passes at most 32 additions in a lane and 16 across lanes and wavefronts, each term positive: it is
off by at most 49 u of itself, its root's reciprocal by half of that and the quotient, root and division by 4 u more; with the
products around it a factor carries less than 32 u:
    |dy| <= 32 u |y| + uT |y|,      |dgx| <= 64 u r (|g| + |hh| <|g hh|>) + 2 u |gh| + uT |gx|   with g = gy w, hh = h r
(the sum <g hh> passes the same additions), and a sum over n rows passes n / 64 + 96 additions at most:
    |dgw| <= (n / 64 + 96 + 64) u sum |gy hh| + uT |gw|.
Below 2^-14 the numbers of fp16 lie 2^-24 apart, and half a step is 2^-25 whatever the value: added for that type.
A code's value is off by half a step of its code (2^-4 of the value, or 2^-10 of the block's scale) and by 32 u |y|."""
import pytest
import torch

from ubio_molfm_amd import fp8, norms

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
UT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
EPS = 1e-5
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _half(dtype, ref):
    """What a rounding of ref to the type may change."""
    return 1.01 * UT[dtype] * ref.abs() + (2.0 ** -25 if dtype == F16 else 0.0)


def _inputs(n, w, dtype, wdtype, seed, cuda):
    g = torch.Generator().manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g)

    x = (rand(n, w) * torch.exp(0.5 * rand(n, 1))).to(dtype).to(cuda)
    res, gy, gh = (rand(n, w).to(dtype).to(cuda) for _ in range(3))
    return x, res, (1 + 0.3 * rand(w)).to(wdtype).to(cuda), gy, gh


def _formulas(h, w, gy, gh):
    h = h.double()
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    hh, w = h * r, torch.ones((), dtype=torch.float64, device=h.device) if w is None else w.double()
    g = gy.double() * w
    m = (g * hh).mean(-1, keepdim=True)
    gx = r * (g - hh * m)
    tol = 64 * U * r * (g.abs() + hh.abs() * (g * hh).abs().mean(-1, keepdim=True))
    if gh is not None:
        gx, tol = gx + gh.double(), tol + 2 * U * gh.double().abs()
    return hh * w, gx, tol, (gy.double() * hh).sum(0), (gy.double() * hh).abs().sum(0)


def _check(x, res, w, gy, gh, y, h, gx, gw):
    n, dt = x.shape[0], x.dtype
    want = x if res is None else (x.detach().float() + res.detach().float()).to(dt)
    assert torch.equal(h, want)
    yy, gxx, tol, gww, mag = _formulas(want, w, gy, gh)
    assert (y.double() - yy).abs().le(32 * U * yy.abs() + _half(dt, yy)).all()
    assert (gx.double() - gxx).abs().le(tol + _half(dt, gxx)).all()
    if gw is not None:
        assert (gw.double() - gww).abs().le((n / 64 + 160) * U * mag + _half(gw.dtype, gww)).all()


WIDTHS = [1, 3, 4, 7, 8, 33, 64, 96, 100, 128, 129, 200, 257, 300, 511, 700, 1000, 1025, 2048, 3001, 5001, 6145, 8192, 9000, 16384]


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("w", WIDTHS)
def test_values_and_gradients(w, dtype, wdtype, cuda):
    n = 1 if w > 9000 else max(3, min(70, 20000 // w))
    x, res, wt, gy, gh = _inputs(n, w, dtype, wdtype, w, cuda)
    for t in (x, res, wt):
        t.requires_grad_(True)
    y, h = norms.rms_norm(x, wt, EPS, residual=res)
    gx, gres, gw = torch.autograd.grad((y, h), (x, res, wt), (gy, gh))
    assert torch.equal(gx, gres) and gw.dtype == wdtype and y.is_contiguous()
    _check(x, res, wt, gy, gh, y, h, gx, gw)
    # without a residual, and with none of the gradients
    y1 = norms.rms_norm(x, wt, EPS)
    gx1, gw1 = torch.autograd.grad(y1, (x, wt), gy)
    _check(x, None, wt, gy, None, y1, x, gx1, gw1)
    with torch.no_grad():
        y2, h2 = norms.rms_norm(x, wt, EPS, residual=res)
    assert torch.equal(y2, y) and torch.equal(h2, h)


@pytest.mark.parametrize("n,w,dtype", [(40000, 40, F32), (3000, 256, BF16), (20011, 129, F32), (700, 4096, BF16)])
def test_many_rows(n, w, dtype, cuda):
    x, res, wt, gy, gh = _inputs(n, w, dtype, dtype, 5, cuda)
    for t in (x, res, wt):
        t.requires_grad_(True)
    y, h = norms.rms_norm(x, wt, EPS, residual=res)
    first = torch.autograd.grad((y, h), (x, wt), (gy, gh), retain_graph=True)
    _check(x, res, wt, gy, gh, y, h, *first)
    again = torch.autograd.grad((y, h), (x, wt), (gy, gh))
    assert all(torch.equal(a, b) for a, b in zip(first, again))          # no order of additions changes


def test_which_gradients(cuda):
    x, res, wt, gy, gh = _inputs(9, 200, F32, F32, 1, cuda)
    xg, rg = x.clone().requires_grad_(True), res.clone().requires_grad_(True)
    y, h = norms.rms_norm(xg, None, EPS, residual=res)                   # no weight, x alone
    gx, = torch.autograd.grad(y, xg, gy, retain_graph=True)
    _check(x, res, None, gy, None, y, h, gx, None)
    only_h, = torch.autograd.grad(h, xg, gh)
    assert torch.equal(only_h, gh)
    y, h = norms.rms_norm(x, wt, EPS, residual=rg)                       # the residual alone
    gr, = torch.autograd.grad((y, h), rg, (gy, gh))
    _check(x, res, wt, gy, gh, y, h, gr, None)
    wg = wt.clone().requires_grad_(True)                                 # the weight alone
    y, h = norms.rms_norm(x, wg, EPS, residual=res)
    gw, = torch.autograd.grad(y, wg, gy)
    _check(x, res, wt, gy, None, y, h, _formulas(h, wt, gy, None)[1].float(), gw)
    # leaves that accumulate: both get the same gradient, in memory of their own
    y, h = norms.rms_norm(xg, wt, EPS, residual=rg)
    torch.autograd.backward((y, h), (gy, gh))
    assert torch.equal(xg.grad, rg.grad) and xg.grad.data_ptr() != rg.grad.data_ptr()


def test_a_tensor_is_its_own_residual(cuda):
    x, _, wt, gy, gh = _inputs(40, 300, F32, F32, 4, cuda)
    xg = x.clone().requires_grad_(True)
    y, h = norms.rms_norm(xg, wt, EPS, residual=xg)
    gx, = torch.autograd.grad((y, h), xg, (gy, gh))
    _check(x, x, wt, gy, gh, y, h, gx / 2, None)     # halving is exact


def test_offsets_past_32_bits(cuda):
    """140,000 rows of 16384 bf16 (4.6 GB): the last ones have the values and gradients that they have alone."""
    n, w = 140_000, 16384
    x, res, wt, gy, gh = _inputs(3, w, BF16, BF16, 5, cuda)
    big, up = torch.zeros(n, w, dtype=BF16, device=cuda), torch.zeros(n, w, dtype=BF16, device=cuda)
    big[-3:], up[-3:] = x, gy
    few = x.clone().requires_grad_(True)
    want = norms.rms_norm(few, wt, EPS)
    gx_want, = torch.autograd.grad(want, few, gy)
    big.requires_grad_(True)
    y = norms.rms_norm(big, wt, EPS)
    gx, = torch.autograd.grad(y, big, up)
    assert torch.equal(y[-3:], want) and torch.equal(gx[-3:], gx_want)
    assert y[:-3].count_nonzero() == 0 and gx[:-3].count_nonzero() == 0
    with torch.no_grad():
        for a, b in zip(norms.rms_norm_fp8(big, wt, EPS), norms.rms_norm_fp8(few, wt, EPS)):
            assert torch.equal(a[-3:].view(torch.uint8), b.view(torch.uint8))


def test_against_differences(cuda):
    """The gradient in a direction against central differences of the definition in float64: their error is of the order of
    step^2 = 1e-8 of third derivatives of the order of 1."""
    x, res, wt, gy, gh = _inputs(4, 50, F32, F32, 3, cuda)
    x.requires_grad_(True), wt.requires_grad_(True)
    y, h = norms.rms_norm(x, wt, EPS, residual=res)
    gx, gw = torch.autograd.grad((y, h), (x, wt), (gy, gh))
    g = torch.Generator().manual_seed(8)
    dx, dw = torch.randn(4, 50, generator=g).double().to(cuda), torch.randn(50, generator=g).double().to(cuda)
    base, w = h.detach().double(), wt.detach().double()      # the sum before it is rounded differs by u |h|

    def f(t):
        v = base + t * dx
        return float(((v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * (w + t * dw)) * gy.double()).sum()
                     + (v * gh.double()).sum())

    d = (f(1e-4) - f(-1e-4)) / 2e-4
    mine = float((gx.double() * dx).sum() + (gw.double() * dw).sum())
    size = float((gx.double() * dx).abs().sum() + (gw.double() * dw).abs().sum())
    assert abs(d - mine) < 1e-5 * size


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(dtype, cuda):
    """Rows inside a wider tensor, on odd boundaries, of several dimensions, transposed: read where they lie or copied."""
    g = torch.Generator().manual_seed(2)
    base = torch.randn(6, 5, 150, generator=g).to(dtype).to(cuda)
    wt = (1 + 0.1 * torch.randn(101, generator=g)).to(dtype).to(cuda)
    for x in (base[..., 3:104], base[::2, :, 7:108], base[:, 1, 2:103], base.transpose(0, 1)[..., :101]):
        y, h = norms.rms_norm(x, wt, EPS, residual=x.flip(0))
        c = x.contiguous()
        y2, h2 = norms.rms_norm(c, wt, EPS, residual=c.flip(0))
        assert torch.equal(y, y2) and torch.equal(h, h2) and y.shape == x.shape
        q, s = norms.rms_norm_fp8(x, wt, EPS)
        q2, s2 = norms.rms_norm_fp8(c, wt, EPS)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2) and q.shape == x.shape
    t = torch.randn(101, 6, generator=g).to(dtype).to(cuda).t()
    assert torch.equal(norms.rms_norm(t, wt), norms.rms_norm(t.contiguous(), wt))
    one = torch.randn(1, 101, generator=g).to(dtype).to(cuda).expand(4, 101)
    assert torch.equal(norms.rms_norm(one, wt), norms.rms_norm(one.contiguous(), wt))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("w", [1, 5, 8, 40, 96, 128, 129, 200, 256, 384, 700, 1000, 1536, 2049, 4096, 5001, 9000])
def test_codes(w, dtype, cuda):
    n = max(2, min(50, 20000 // w))
    x, res, wt, _, _ = _inputs(n, w, dtype, dtype, w + 1, cuda)
    codes, scales, h = norms.rms_norm_fp8(x, wt, EPS, residual=res)
    assert torch.equal(h, (x.float() + res.float()).to(dtype))
    assert codes.shape == x.shape and codes.dtype == torch.float8_e4m3fn
    assert scales.shape == (n, -(-w // 128)) and codes.stride(0) % 16 == 0
    y = _formulas(h, wt, x, None)[0]
    s = torch.exp2(scales.double() - 127).repeat_interleave(128, 1)[:, :w]
    v = fp8.dequantize(codes, scales)
    assert torch.equal(v.double(), codes.double() * s)
    assert (v.double() - y).abs().le(torch.maximum(1.01 * 2.0 ** -4 * y.abs(), s * 2.0 ** -10) + 32 * U * y.abs()).all()
    # each scale is the smallest power of two that holds the block (up to the rounding of its largest value)
    pad = torch.nn.functional.pad(y.abs(), (0, -w % 128)).view(n, -1, 128).amax(-1)
    unit = torch.exp2(scales.double() - 127)
    assert (pad <= 448 * unit * (1 + 32 * U)).all()
    assert ((pad > 224 * unit * (1 - 32 * U)) | (scales == 1)).all()
    if dtype == F32:                            # and those of the norm itself, quantised
        q2, s2 = fp8.quantize(norms.rms_norm(h, wt, EPS))
        assert torch.equal(q2.view(torch.uint8), codes.contiguous().view(torch.uint8)) and torch.equal(s2, scales)


def test_rows_that_are_not_finite_stay_apart(cuda):
    x, res, wt, gy, gh = _inputs(8, 300, F32, F32, 4, cuda)
    bad = x.clone()
    bad[2, 17], bad[5, 0], bad[6] = float("nan"), float("inf"), 0.0
    y, _ = norms.rms_norm(bad, wt, EPS, residual=torch.zeros_like(bad))
    good = norms.rms_norm(x, wt, EPS)
    ok = [0, 1, 3, 4, 7]
    assert torch.equal(y[ok], good[ok]) and y[2].isnan().all() and (y[6] == 0).all()
    codes, scales = norms.rms_norm_fp8(bad, wt, EPS)
    v = fp8.dequantize(codes, scales)
    assert v[2].isnan().all() and (v[6] == 0).all() and v[ok].isfinite().all() and (scales[6] == 1).all()


def test_no_rows(cuda):
    wt = torch.ones(16, device=cuda, requires_grad=True)
    x = torch.empty(0, 16, device=cuda, requires_grad=True)
    y, h = norms.rms_norm(x, wt, residual=torch.empty(0, 16, device=cuda))
    gx, gw = torch.autograd.grad(y, (x, wt), torch.empty(0, 16, device=cuda))
    assert y.shape == h.shape == gx.shape == (0, 16) and torch.equal(gw, torch.zeros(16, device=cuda))
    codes, scales = norms.rms_norm_fp8(torch.empty(0, 3, 16, device=cuda), torch.ones(16, device=cuda))
    assert codes.shape == (0, 3, 16) and scales.shape == (0, 3, 1)


def test_streams_and_graph(cuda):
    x, res, wt, gy, gh = _inputs(64, 1024, BF16, BF16, 6, cuda)

    def step():
        # leaves of its own: a leaf of an eager graph that lives is tied to that graph's stream
        X, W = x.detach().requires_grad_(True), wt.detach().requires_grad_(True)
        y, h = norms.rms_norm(X, W, EPS, residual=res)
        gx, gw = torch.autograd.grad((y, h), (X, W), (gy, gh))
        codes, scales, _ = norms.rms_norm_fp8(x, wt, EPS, residual=res)
        return y.detach(), h.detach(), gx, gw, codes.view(torch.uint8), scales

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        x.mul_(1.5)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k


def test_refused_derivatives(cuda):
    x = torch.randn(4, 32, device=cuda, requires_grad=True)
    y = norms.rms_norm(x)
    with pytest.raises(NotImplementedError, match="create_graph"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(norms.rms_norm(x), x, torch.randn(3, 4, 32, device=cuda), is_grads_batched=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="tangents"):
            norms.rms_norm(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="no gradients"):
        norms.rms_norm_fp8(x)
