"""8-bit floats with block scales (fp8.py; csrc/fp8.hip, csrc/product8.hip) against integer and float64 arithmetic.

Quantisation has one right answer: codes and scale bytes are compared exactly.  A product of two codes has 8 significant bits.
The matrix unit adds products of 8 consecutive values of k on a grid of 2^-13 of the power of two below the largest of
them (a property of the instruction: with one product of 2^16 among them 2^3 is kept and 2^2 is lost), so that each of
the 8 loses less than 2^-13 of the largest, P; what follows is fp32, at most k additions, each off by at most a step, 2^-23,
of the sum of magnitudes M = sum |a b|; and a result is rounded once to its type:
    |dy| <= 7 2^-13 sum over eights of P + k 2^-23 M + uT |y|,  uT half a step of the type."""
import pytest
import torch

from ubio_molfm_amd import fp8

pytestmark = pytest.mark.gpu

UT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F8 = torch.float8_e4m3fn
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _bits(codes):
    return codes.contiguous().view(torch.uint8)


def _held(x, rows):
    """(codes' bits, scale bytes, values) of x [r, c], in float64 from the definition."""
    x = x.detach().double().cpu()
    r, c = x.shape
    nr, nc = -(-r // rows), -(-c // 128)
    full = torch.zeros(nr * rows, nc * 128, dtype=torch.float64)
    full[:r, :c] = x
    b = full.view(nr, rows, nc, 128)
    fin = torch.where(b.isfinite(), b.abs(), 0.0)
    most = fin.amax((1, 3))
    m, e = torch.frexp(most)                         # most = 2 m 2^(e - 1), 448 = 1.75 * 2^8
    e = torch.where(most > 0, e - 9 + (m > 0.875).int(), -126).clamp(min=-126)
    unit = torch.exp2(e.double())[:, None, :, None]
    t = b / unit
    lead = torch.clamp(torch.frexp(t)[1] - 1, min=-6)
    q = torch.round(t / torch.exp2(lead.double() - 3))           # ties to even
    v = q * torch.exp2(lead.double() - 3)
    a = v.abs()
    lead = torch.clamp(torch.frexp(a)[1] - 1, min=-6)
    frac = (a * torch.exp2(3 - lead.double())).long()            # 8..15 for normal codes, 0..7 below 2^-6
    code = torch.where(frac >= 8, (lead + 7) * 8 + frac - 8, frac)
    code = torch.where(torch.signbit(t), code + 128, code)
    ok = b.isfinite()

    def back(t):
        return t.reshape(nr * rows, nc * 128)[:r, :c]

    return back(code), back(ok), e + 127, back(torch.where(ok, v * unit, float("nan")))


def _check_codes(codes, scales, x, rows):
    code, ok, s, v = _held(x, rows)
    got = _bits(codes).cpu().long()
    assert torch.equal(scales.cpu().long(), s.long())
    assert torch.equal(got[ok], code.long()[ok]) and (got[~ok] % 128 == 127).all()
    return v


def _rand(*shape, seed=0, dtype=F32, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(*shape, generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("r,c", [(1, 1), (3, 7), (2, 8), (5, 127), (4, 128), (7, 129), (130, 200), (200, 384), (3, 5001)])
def test_codes_are_those_of_the_definition(r, c, dtype, cuda):
    x = _rand(r, c, seed=c, dtype=dtype).to(cuda)
    for tiles in (False, True):
        codes, scales = fp8.quantize(x, tiles=tiles)
        v = _check_codes(codes, scales, x, 128 if tiles else 1)
        for dt in (F32, BF16):
            assert torch.equal(fp8.dequantize(codes, scales, dt).double().cpu(), v.to(dt).double())


def test_ties_borders_and_extremes(cuda):
    row = torch.zeros(12, 128)
    row[0, :16] = torch.tensor([448.0] + [k + 0.5 for k in range(15)]) / 2 ** 9      # ties of subnormal codes
    row[1, :9] = torch.tensor([17.0, 19.0, 21.0, 23.0, 25.0, 27.0, 29.0, 31.0, 448.0])   # ties between codes of 2^4
    row[2, 0] = 448.0
    row[3, 0] = 448.0 * (1 + 2 ** -20)
    row[4, 0], row[4, 1] = torch.finfo(F32).max, -1e30
    row[5, 0], row[5, 1] = 1e-45, -1.2e-38
    row[6, 3] = -0.0
    row[7, 0], row[7, 1], row[7, 2] = float("inf"), 2.0, -float("inf")
    row[8, 0], row[8, 1] = float("nan"), -3.0
    row[9] = float("nan")
    row[10, 0] = 2.0 ** -126
    row[11] = torch.linspace(-500, 500, 128)
    x = row.to(cuda)
    codes, scales = fp8.quantize(x)
    v = _check_codes(codes, scales, x, 1)
    s = scales.cpu()[:, 0].tolist()
    assert s[2] == 127 and s[3] == 128 and s[5] == s[6] == s[9] == 1 and s[4] == 127 + 120
    assert torch.equal(fp8.dequantize(codes, scales).cpu().nan_to_num(7e30), v.float().nan_to_num(7e30))
    _check_codes(*fp8.quantize(x, tiles=True), x, 128)


def test_quantised_layouts(cuda):
    base = _rand(6, 5, 300, seed=3).to(cuda)
    for x in (base[..., 1:202], base[::2, :, 3:], base[0, 0], base.transpose(0, 1)[..., :200]):
        codes, scales = fp8.quantize(x)
        c2, s2 = fp8.quantize(x.contiguous())
        assert codes.shape == x.shape and scales.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        assert torch.equal(_bits(codes), _bits(c2)) and torch.equal(scales, s2)
        w = x.shape[-1]
        assert torch.equal(_bits(codes).view(-1, w), _bits(fp8.quantize(x.reshape(-1, w))[0]))
    wts = _rand(3, 140, 260, seed=4).to(cuda)
    codes, scales = fp8.quantize(wts, tiles=True)
    assert scales.shape == (3, 2, 3)
    for e in range(3):
        v = _check_codes(codes[e], scales[e], wts[e], 128)
        assert torch.equal(fp8.dequantize(codes, scales)[e].double().cpu(), v)
    turned = wts.transpose(1, 2)
    _check_codes(*(t[1] for t in fp8.quantize(turned, tiles=True)), turned[1], 128)


def _product(cuda, m, n, k, seed, tiles=True):
    a, w = _rand(m, k, seed=seed, spread=0.7), _rand(n, k, seed=seed + 1, spread=0.7) / k ** 0.5
    (aq, sa), (wq, sw) = fp8.quantize(a.to(cuda)), fp8.quantize(w.to(cuda), tiles=tiles)
    return aq, sa, wq, sw


def _largest_of_8(t):
    """The largest magnitude of each 8 consecutive values of a row."""
    return torch.nn.functional.pad(t.abs(), (0, -t.shape[1] % 8)).view(t.shape[0], -(-t.shape[1] // 8), 8).amax(-1)


def _check_product(y, a, w, k):
    """y against the product of the values a and w."""
    a, w = a.double(), w.double()
    want, mag = a @ w.T, a.abs() @ w.abs().T
    tol = 7 * 2.0 ** -13 * (_largest_of_8(a) @ _largest_of_8(w).T) + k * 2.0 ** -23 * mag + 1.01 * UT[y.dtype] * want.abs()
    if y.dtype == F16:
        tol = tol + 2.0 ** -25                       # half a step of fp16 below its normal numbers
    assert (y.double() - want).abs().le(tol).all()


SIZES = [(1, 1, 1), (1, 16, 16), (2, 3, 130), (5, 128, 128), (16, 64, 257), (17, 200, 384), (33, 127, 1000), (100, 100, 100),
         (128, 128, 2048), (129, 257, 512), (300, 500, 640), (1000, 136, 4096), (64, 4096, 4096), (1, 5000, 2000),
         (13, 1000, 8192), (16, 96, 16), (7, 130, 120), (2048, 2304, 256), (5000, 2500, 144)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("tiles", [True, False])
def test_products(m, n, k, tiles, cuda):
    aq, sa, wq, sw = _product(cuda, m, n, k, m + n, tiles)
    for dt in (F32, BF16, F16):
        y = fp8.gemm(aq, sa, wq, sw, dtype=dt)
        _check_product(y, fp8.dequantize(aq, sa), fp8.dequantize(wq, sw), k)
        assert torch.equal(y, fp8.gemm(aq, sa, wq, sw, dtype=dt))


@pytest.mark.parametrize("m,n,k", [(1, 40, 100), (20, 130, 131), (200, 300, 515), (3, 64, 128), (16, 200, 1000)])
def test_products_on_any_boundary(m, n, k, cuda):
    """Codes packed without padding and starting on every byte of a dword; surroundings of NaN codes stay out."""
    aq, sa, wq, sw = _product(cuda, m, n, k, 7)
    want = fp8.gemm(aq, sa, wq, sw, dtype=F32)
    for skew in range(4):
        def moved(q):
            r, c = q.shape
            flat = torch.full((r * (c + skew) + 40,), 0x7F, dtype=torch.uint8, device=cuda)
            view = flat[skew:skew + r * (c + skew)].view(r, c + skew)[:, :c]
            view.copy_(_bits(q))
            return view.view(torch.float8_e4m3fn)
        a2, w2 = moved(aq), moved(wq)
        y = fp8.gemm(a2, sa, w2, sw, dtype=F32)
        _check_product(y, fp8.dequantize(aq, sa), fp8.dequantize(wq, sw), k)
    # rows padded with NaN codes, on boundaries of 16
    pitch = -(-k // 16) * 16 + 16
    pad = torch.full((m, pitch), 0x7F, dtype=torch.uint8, device=cuda)
    pad[:, :k] = _bits(aq)
    assert torch.equal(fp8.gemm(pad[:, :k].view(torch.float8_e4m3fn), sa, wq, sw, dtype=F32), want)
    # columns apart, leading dimensions
    assert torch.equal(fp8.gemm(aq.t().contiguous().t(), sa, wq, sw, dtype=F32), want)
    assert torch.equal(fp8.gemm(aq.view(1, m, k) if aq.is_contiguous() else aq[None], sa[None], wq, sw, dtype=F32)[0], want)


def test_rows_that_share_bytes(cuda):
    """A row repeated by expand() and overlapping windows are read where they are, not past their end."""
    aq, sa, wq, sw = _product(cuda, 1, 40, 256, 3)
    one = fp8.gemm(aq, sa, wq, sw, dtype=F32)
    assert torch.equal(fp8.gemm(aq.expand(130, 256), sa.expand(130, 2), wq, sw, dtype=F32), one.expand(130, 40))
    wide = _bits(_product(cuda, 1, 8, 1024, 4)[0]).view(-1)
    windows = wide.as_strided((7, 256), (128, 1)).view(torch.float8_e4m3fn)
    s7 = torch.full((7, 2), 127, dtype=torch.uint8, device=cuda)
    assert torch.equal(fp8.gemm(windows, s7, wq, sw, dtype=F32), fp8.gemm(windows.contiguous(), s7, wq, sw, dtype=F32))
    x = torch.randn(1, 64, device=cuda)
    w = torch.randn(24, 64, device=cuda)
    assert torch.equal(fp8.linear(x.expand(9, 64), w), fp8.linear(x, w).expand(9, 24))


def test_products_keep_nan_to_their_row(cuda):
    aq, sa, wq, sw = _product(cuda, 40, 50, 300, 9)
    want = fp8.gemm(aq, sa, wq, sw, dtype=F32)
    _bits_view = aq.view(torch.uint8) if aq.is_contiguous() else aq.contiguous().view(torch.uint8)
    bad = _bits_view.clone()
    bad[3, 299] = 0x7F
    y = fp8.gemm(bad.view(torch.float8_e4m3fn), sa, wq, sw, dtype=F32)
    rows = [r for r in range(40) if r != 3]
    assert y[3].isnan().all() and torch.equal(y[rows], want[rows])


def test_extreme_scales(cuda):
    """Scale bytes from 1 to 247 in one product: its range is fp32's."""
    a = torch.ones(3, 256, device=cuda)
    a[0] *= 2.0 ** 60
    a[1, 128:] *= 2.0 ** -60
    w = torch.ones(130, 256, device=cuda) * 2.0 ** -50
    w[:, 128:] *= 2.0 ** 40
    (aq, sa), (wq, sw) = fp8.quantize(a), fp8.quantize(w)
    y = fp8.gemm(aq, sa, wq, sw, dtype=F32)
    assert torch.equal(y, (a.double() @ w.double().T).float())


@pytest.mark.parametrize("m,n,k,dtype,wdtype", [(1, 1, 1, F32, F32), (5, 40, 72, F32, F32), (200, 130, 300, BF16, BF16),
                                               (129, 256, 128, BF16, F32), (64, 64, 1000, F16, F16),
                                               (1000, 384, 256, BF16, BF16), (3000, 100, 120, F32, F32)])
def test_linear(m, n, k, dtype, wdtype, cuda):
    x = (_rand(m, k, seed=1, spread=0.7)).to(dtype).to(cuda).requires_grad_(True)
    w = (_rand(n, k, seed=2, spread=0.5) / k ** 0.5).to(wdtype).to(cuda).requires_grad_(True)
    gy = _rand(m, n, seed=3, spread=0.7).to(dtype).to(cuda)
    y = fp8.linear(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), gy, retain_graph=True)

    def held(t, rows=1):
        return _held(t, rows)[3].to(cuda)

    _check_product(y, held(x), held(w, 128), k)
    _check_product(gx, held(gy), held(w, 128).T, n)
    _check_product(gw, held(gy.T), held(x.T), m)
    assert y.dtype == gx.dtype == dtype and gw.dtype == wdtype
    # one gradient alone, and the product by hand, are bitwise the same
    assert torch.equal(torch.autograd.grad(fp8.linear(x, w.detach()), x, gy)[0], gx)
    assert torch.equal(torch.autograd.grad(fp8.linear(x.detach(), w), w, gy)[0], gw)
    with torch.no_grad():
        assert torch.equal(fp8.linear(x, w), y)
        by_hand = fp8.gemm(*fp8.quantize(x.float()), *fp8.quantize(w.float(), tiles=True), dtype=dtype)
        assert torch.equal(by_hand, y)
    # leading dimensions and strided operands
    x3 = x.detach().view(1, m, k).expand(2, m, k)
    assert torch.equal(fp8.linear(x3, w)[1], fp8.linear(x3.contiguous(), w)[1])
    assert torch.equal(fp8.linear(x, w.detach().t().contiguous().t()), y)
    # a weight changed in place after the forward pass: the gradients are those of the product that was taken
    with torch.no_grad():
        w.mul_(2.0)
    assert torch.equal(torch.autograd.grad(y, x, gy)[0], gx)


def test_empty(cuda):
    w = torch.randn(24, 40, device=cuda, requires_grad=True)
    x = torch.empty(0, 40, device=cuda, requires_grad=True)
    y = fp8.linear(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty(0, 24, device=cuda))
    assert y.shape == (0, 24) and gx.shape == (0, 40) and torch.equal(gw, torch.zeros_like(w))
    codes, scales = fp8.quantize(torch.empty(0, 40, device=cuda))
    assert fp8.dequantize(codes, scales).shape == (0, 40)
    wq, sw = fp8.quantize(w.detach(), tiles=True)
    assert fp8.gemm(codes, scales, wq, sw).shape == (0, 24)


def test_streams_and_graph(cuda):
    x = _rand(150, 256, seed=1).to(BF16).to(cuda)
    w = _rand(200, 256, seed=2).to(BF16).to(cuda)
    gy = _rand(150, 200, seed=3).to(BF16).to(cuda)
    deep = _rand(40, 4096, seed=5).to(cuda)                  # a product whose reduction is cut
    dq, ds = fp8.quantize(deep)

    def step():
        # leaves of its own: a leaf of an eager graph that lives is tied to that graph's stream
        X, W = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = fp8.linear(X, W)
        gx, gw = torch.autograd.grad(y, (X, W), gy)
        codes, scales = fp8.quantize(x)
        one = fp8.gemm(codes[:1], scales[:1], *fp8.quantize(w, tiles=True))
        return y.detach(), gx, gw, one, fp8.gemm(dq, ds, dq, ds), fp8.dequantize(codes, scales)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.cuda.graph(other):
        held2 = step()
    for _ in range(3):
        x.mul_(-1.5)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, held, held2))


def test_offsets_past_32_bits(cuda):
    """Codes of 2.2 GB: rows past 2^31 and 2^32 bytes' offsets are read where they lie."""
    m, k, n = 1_100_000, 2048, 16
    a = torch.zeros(m, k, dtype=torch.uint8, device=cuda)
    a[::100_003] = 0x38                              # 1.0
    a[-1] = 0x40                                     # 2.0
    sa = torch.full((m, k // 128), 127, dtype=torch.uint8, device=cuda)
    w = torch.full((n, k), 0x38, dtype=torch.uint8, device=cuda)
    sw = torch.full((1, k // 128), 127, dtype=torch.uint8, device=cuda)
    y = fp8.gemm(a.view(torch.float8_e4m3fn), sa, w.view(torch.float8_e4m3fn), sw, dtype=F32)
    want = torch.zeros(m, device=cuda)
    want[::100_003] = k
    want[-1] = 2 * k
    assert torch.equal(y, want[:, None].expand(m, n))


def test_quantised_past_32_bits(cuda):
    """140,000 x 16384 bf16 (4.6 GB): blocks past 2^31 elements, along rows, in tiles and along columns."""
    n, w = 140_000, 16384
    x = torch.zeros(n, w, dtype=BF16, device=cuda)
    x[-1, -2:] = torch.tensor([3.0, -448.0], dtype=BF16)
    codes, scales = fp8.quantize(x)
    assert fp8.dequantize(codes[-1:], scales[-1:])[0, -2:].tolist() == [3.0, -448.0]
    assert codes[:-1].view(torch.uint8).count_nonzero() == 0 and scales[-1, -1] == 127 and (scales[:-1] == 1).all()
    back = fp8.dequantize(codes, scales, BF16)
    assert torch.equal(back, x)
    del codes, scales, back
    codes, scales = fp8.quantize(x, tiles=True)
    assert scales[-1, -1] == 127 and (scales.view(-1)[:-1] == 1).all()
    assert torch.equal(fp8.dequantize(codes, scales, BF16), x)
    del codes, scales
    turned = torch.empty((w, n), dtype=F8, device=cuda)
    by_column = torch.empty((-(-n // 128), w), dtype=torch.uint8, device=cuda)
    codes, by_row = torch.empty((n, w), dtype=F8, device=cuda), torch.empty((w // 128, n), dtype=torch.uint8, device=cuda)
    fp8._quantize(x, w, fp8._BOTH, codes, by_row, turned, by_column, n=n)
    assert torch.equal(fp8.dequantize(codes, by_row.t(), BF16), x)
    assert torch.equal(fp8.dequantize(turned, by_column.t(), BF16), x.t())


def test_refused_derivatives(cuda):
    x = torch.randn(4, 32, device=cuda, requires_grad=True)
    w = torch.randn(8, 32, device=cuda, requires_grad=True)
    with pytest.raises(NotImplementedError, match="create_graph"):
        torch.autograd.grad(fp8.linear(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradients"):
        fp8.quantize(x)


def test_codes_with_a_history_are_refused(cuda):
    x = torch.randn(4, 32, device=cuda, requires_grad=True)
    codes, s = x.to(F8), torch.full((4, 1), 127, dtype=torch.uint8, device=cuda)
    for call in (lambda: fp8.dequantize(codes, s), lambda: fp8.gemm(codes, s, codes.detach(), s)):
        with pytest.raises(RuntimeError, match="no gradients"):
            call()
        with torch.no_grad():
            call()


def test_linear_with_many_rows(cuda):
    """More rows than a row of codes may have bytes: x's gradient and calls without gradients have no such rows."""
    m, n, k = (1 << 22) + 37, 24, 140
    x = _rand(1000, k, seed=1, spread=0.7).to(BF16).to(cuda).repeat(-(-m // 1000), 1)[:m].requires_grad_(True)
    w = (_rand(n, k, seed=2, spread=0.5) / k ** 0.5).to(BF16).to(cuda)
    gy = _rand(1000, n, seed=3, spread=0.7).to(BF16).to(cuda).repeat(-(-m // 1000), 1)[:m]
    y = fp8.linear(x, w)
    gx, = torch.autograd.grad(y, x, gy)
    short = x.detach()[:1000].requires_grad_(True)
    y0 = fp8.linear(short, w)
    g0, = torch.autograd.grad(y0, short, gy[:1000])
    last = m // 1000 * 1000
    for got, want in ((y, y0), (gx, g0)):
        assert torch.equal(got[:1000], want) and torch.equal(got[last:], want[:m - last])
        assert (got[:last].view(-1, 1000, got.shape[1]) == want).all()
    with torch.no_grad():
        assert torch.equal(fp8.linear(x, w.requires_grad_(True)), y)
    with pytest.raises(ValueError, match="linear: sizes up to"):
        fp8.linear(x, w)


def test_rows_far_apart(cuda):
    aq, sa, wq, sw = _product(cuda, 3, 40, 200, 11)

    def far(q):
        t = torch.empty_strided(tuple(q.shape), (fp8.MAX_PITCH + 16, 1), dtype=torch.uint8, device=cuda)
        return t.copy_(_bits(q)).view(F8)

    for y in (fp8.gemm(far(aq), sa, wq, sw, dtype=F32), fp8.gemm(aq, sa, far(wq), sw, dtype=F32)):
        _check_product(y, fp8.dequantize(aq, sa), fp8.dequantize(wq, sw), 200)


@pytest.mark.parametrize("m,n,k", [(65, 64, 8191), (200, 300, 4100), (33, 130, 6001), (100, 700, 2049), (3000, 5000, 145)])
def test_long_and_many_tiles_on_any_boundary(m, n, k, cuda):
    """Codes packed without padding, where k is cut into parts and where a workgroup takes several tiles."""
    aq, sa, wq, sw = _product(cuda, m, n, k, 17)
    assert k % 16 and (m <= 64 or k < 4096 or fp8._workspace_bytes(m, n, k) > 0) and (m < 3000 or -(-m // 128) * -(-n // 128) > 512)
    av, wv = fp8.dequantize(aq, sa), fp8.dequantize(wq, sw)
    for skew in (0, 1, 2, 3):
        def moved(q):
            r, c = q.shape
            flat = torch.full((r * c + 40,), 0x7F, dtype=torch.uint8, device=cuda)
            view = flat[skew:skew + r * c].view(r, c)
            view.copy_(_bits(q))
            return view.view(F8)
        y = fp8.gemm(moved(aq), sa, moved(wq), sw, dtype=F32)
        _check_product(y, av, wv, k)
        assert torch.equal(y, fp8.gemm(moved(aq), sa, moved(wq), sw, dtype=F32))
