"""Products grouped by expert (experts.py; csrc/experts.hip, csrc/product8.hip, csrc/mm.h) against float64.

Tolerances.  M = sum |a b| of a result, r the length of its reduction, uT half a step of its type.  Products of 16-bit
operands are exact in fp32 and a result passes at most r additions, each off by at most a step of fp32:
    |dy| <= r 2^-23 M + uT |y|;   for 8-bit operands + 7 2^-13 sum over eights of the largest product (test_gpu_fp8.py).
fp32 operands are split exactly into three bf16 pieces, of which the products of order 3 and above are left out, at most
4 2^-24 |a b| each, and the others make six additions for each of the r: |dy| <= (6 r + 4) 2^-23 M + uT |y|."""
import pytest
import torch

from ubio_molfm_amd import experts, fp8, norms

pytestmark = pytest.mark.gpu

UT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _close(y, want, mag, r, operand=None, extra=0.0):
    r = 6 * r + 4 if (operand or y.dtype) == F32 else r
    tol = extra + r * 2.0 ** -23 * mag + 1.01 * UT[y.dtype] * want.abs() + (2.0 ** -25 if y.dtype == F16 else 0.0)
    assert (y.double() - want).abs().le(tol).all()


def _largest_of_8(t):
    return torch.nn.functional.pad(t.abs(), (0, -t.shape[1] % 8)).view(t.shape[0], -(-t.shape[1] // 8), 8).amax(-1)


def _inputs(sizes, spare, n, k, dtype, seed, cuda, before=0):
    g = torch.Generator().manual_seed(seed)
    rows = before + sum(sizes) + spare
    x = torch.randn(rows, k, generator=g).to(dtype).to(cuda)
    w = (torch.randn(len(sizes), n, k, generator=g) / k ** 0.5).to(dtype).to(cuda)
    gy = torch.randn(rows, n, generator=g).to(dtype).to(cuda)
    offs = torch.tensor([before] + sizes).cumsum(0).to(torch.int32).to(cuda)
    return x, w, gy, offs


def _check(x, w, gy, offs, y, gx=None, gw=None):
    x, w, gy = x.detach(), w.detach(), gy.detach()
    o = offs.tolist()
    E, n, k = w.shape
    inside = torch.zeros(x.shape[0], dtype=torch.bool, device=x.device)
    for e in range(E):
        s = slice(o[e], o[e + 1])
        inside[s] = True
        xd, wd, gd = x[s].double(), w[e].double(), gy[s].double()
        _close(y[s], xd @ wd.T, xd.abs() @ wd.abs().T, k, x.dtype)
        if gx is not None:
            _close(gx[s], gd @ wd, gd.abs() @ wd.abs(), n)
        if gw is not None:
            _close(gw[e], gd.T @ xd, gd.abs().T @ xd.abs(), max(1, o[e + 1] - o[e]))
    assert (y[~inside] == 0).all() and (gx is None or (gx[~inside] == 0).all())


CASES = [([1], 0, 1, 1), ([0, 3, 0, 2, 0], 2, 16, 16), ([5, 130, 0, 17], 3, 64, 128), ([128, 128], 0, 128, 64),
         ([300, 1, 0, 0, 77], 0, 100, 72), ([40, 90], 9, 33, 65), ([0, 0], 5, 40, 24), ([700], 0, 256, 512),
         ([20] * 70 + [0] * 3 + [200], 11, 96, 48), ([3] * 140, 0, 65, 40), ([1500, 900, 2500], 0, 256, 256),
         ([260, 513, 0, 31], 4, 200, 264)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes,spare,n,k", CASES)
def test_products_and_gradients(sizes, spare, n, k, dtype, cuda):
    x, w, gy, offs = _inputs(sizes, spare, n, k, dtype, 1, cuda)
    # what belongs to no expert is not looked at
    if spare:
        x[-spare:], gy[-spare:] = float("nan"), float("inf")
    x.requires_grad_(True), w.requires_grad_(True)
    y = experts.expert_linear(x, w, offs)
    gx, gw = torch.autograd.grad(y, (x, w), gy, retain_graph=True)
    _check(x, w, gy, offs, y, gx, gw)
    empty = [e for e, s in enumerate(sizes) if s == 0]
    assert (gw[empty] == 0).all()
    assert torch.equal(torch.autograd.grad(y, x, gy, retain_graph=True)[0], gx)
    assert torch.equal(torch.autograd.grad(y, w, gy)[0], gw)
    with torch.no_grad():
        assert torch.equal(experts.expert_linear(x, w, offs.long()), y)


# sizes at which tiles of 256 x 256 begin, in each pass
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes,spare,n,k", [([6000, 0, 5001, 7000], 77, 1024, 1000), ([257, 1300, 900], 0, 4360, 4104)])
def test_large_tiles(sizes, spare, n, k, dtype, cuda):
    x, w, gy, offs = _inputs(sizes, spare, n, k, dtype, 2, cuda)
    x.requires_grad_(True), w.requires_grad_(True)
    y = experts.expert_linear(x, w, offs)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    _check(x, w, gy, offs, y, gx, gw)


def test_against_differences(cuda):
    """The gradients in a direction against differences of the product in float64, which is bilinear: central differences
    are exact but for rounding."""
    x, w, gy, offs = _inputs([7, 0, 12], 1, 20, 30, F32, 3, cuda)
    x.requires_grad_(True), w.requires_grad_(True)
    gx, gw = torch.autograd.grad(experts.expert_linear(x, w, offs), (x, w), gy)
    g = torch.Generator().manual_seed(4)
    dx, dw = torch.randn(x.shape, generator=g).double().to(cuda), torch.randn(w.shape, generator=g).double().to(cuda)

    def f(t):
        total, o = 0.0, offs.tolist()
        for e in range(3):
            s = slice(o[e], o[e + 1])
            total += float((((x[s].double() + t * dx[s]) @ (w[e].double() + t * dw[e]).T) * gy[s].double()).sum())
        return total

    d = (f(0.5) - f(-0.5)) / 1.0
    mine = float((gx.double() * dx).sum() + (gw.double() * dw).sum())
    assert abs(d - mine) < 1e-5 * float((gx.double() * dx).abs().sum() + (gw.double() * dw).abs().sum())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(dtype, cuda):
    x, w, gy, offs = _inputs([30, 0, 45], 2, 40, 72, dtype, 5, cuda, before=6)
    want = experts.expert_linear(x, w, offs)
    _check(x, w, gy, offs, want)

    def wide(t, left):
        out = torch.full((*t.shape[:-1], t.shape[-1] + 11), float("nan"), dtype=dtype, device=cuda)
        v = out[..., left:left + t.shape[-1]]
        v.copy_(t)
        return v

    def near(got, ref):
        tol = 2 * (6 * 72 + 4) * 2.0 ** -23 * 20 + 2.02 * UT[dtype] * ref.double().abs()
        assert (got.double() - ref.double()).abs().le(tol).all()

    for left in (0, 1, 3, 8):
        near(experts.expert_linear(wide(x, left), w, offs), want)
        near(experts.expert_linear(x, wide(w, left), offs), want)
    assert torch.equal(experts.expert_linear(x.t().contiguous().t(), w, offs), want)
    assert torch.equal(experts.expert_linear(x, w.transpose(1, 2).contiguous().transpose(1, 2), offs), want)
    row = x[:1].expand(x.shape[0], -1)
    assert torch.equal(experts.expert_linear(row, w, offs), experts.expert_linear(row.contiguous(), w, offs))
    one = w[:1].expand(3, -1, -1)
    assert torch.equal(experts.expert_linear(x, one, offs), experts.expert_linear(x, one.contiguous(), offs))
    xg, wg = wide(x, 1).requires_grad_(True), wide(w, 3).requires_grad_(True)
    gx, gw = torch.autograd.grad(experts.expert_linear(xg, wg, offs), (xg, wg), wide(gy, 5))
    _check(x, w, gy, offs, want, gx, gw)


def test_out_leaves_other_rows(cuda):
    x, w, gy, offs = _inputs([9, 0, 140], 8, 48, 64, BF16, 6, cuda, before=5)
    buf = torch.full((162, 60), 7.0, dtype=BF16, device=cuda)
    y = experts.expert_linear(x, w, offs, out=buf[:, 3:51])
    assert y.data_ptr() == buf[:, 3:51].data_ptr()
    want = experts.expert_linear(x, w, offs)
    assert torch.equal(y[5:154], want[5:154]) and (y[:5] == 7).all() and (y[154:] == 7).all()
    assert (buf[:, :3] == 7).all() and (buf[:, 51:] == 7).all() and (want[:5] == 0).all()
    codes, scales = fp8.quantize(x.float())
    wq, ws = fp8.quantize(w.float(), tiles=True)
    out = torch.full((162, 48), 7.0, device=cuda)
    experts.expert_gemm_fp8(codes, scales, wq, ws, offs, out=out)
    assert (out[:5] == 7).all() and (out[154:] == 7).all()
    assert torch.equal(out[5:154], experts.expert_gemm_fp8(codes, scales, wq, ws, offs, dtype=F32)[5:154])


def test_offsets_outside_the_rows_are_clamped(cuda):
    x, w, gy, _ = _inputs([50, 50], 0, 32, 40, BF16, 7, cuda)
    inside = torch.tensor([0, 60, 100], dtype=torch.int32, device=cuda)
    want = experts.expert_linear(x, w, inside)
    for far in ([-5, 60, 2 ** 31 - 1], [-2 ** 31, 60, 101]):
        got = experts.expert_linear(x, w, torch.tensor(far, dtype=torch.int32, device=cuda))
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [100, 3000])
def test_offsets_that_decrease_stay_inside(rows, cuda):
    """Rows that two experts claim hold the one's or the other's products; all others are right."""
    a, b, c = rows // 5, rows // 2, rows
    x, w, gy, _ = _inputs([a, b - a, c - b], 0, 256, 320, BF16, 8, cuda)
    table = torch.full((rows + 64, 256), 7.0, dtype=BF16, device=cuda)
    offs = torch.tensor([0, b, a, c], dtype=torch.int32, device=cuda)
    y = experts.expert_linear(x, w, offs, out=table[32:-32])
    first = experts.expert_linear(x, w, torch.tensor([0, b, b, b], dtype=torch.int32, device=cuda))
    third = experts.expert_linear(x, w, torch.tensor([0, 0, a, c], dtype=torch.int32, device=cuda))
    assert torch.equal(y[:a], first[:a]) and torch.equal(y[b:], third[b:])
    assert ((y[a:b] == first[a:b]) | (y[a:b] == third[a:b])).all()
    assert (table[:32] == 7).all() and (table[-32:] == 7).all()


def test_offsets_past_32_bits(cuda):
    """Weights of 6.4 GB, and 70,001 rows of 4.6 GB: what lies past 2^31 elements and bytes is read and written in its place."""
    w = torch.zeros(3, 32768, 32768, dtype=BF16, device=cuda)
    w[2, 32767, ::3] = 1.5
    w[2, 3] = 0.25
    x = torch.ones(300, 32768, dtype=BF16, device=cuda)
    y = experts.expert_linear(x, w, torch.tensor([0, 1, 1, 300], dtype=torch.int32, device=cuda))
    want = torch.zeros(300, 32768, dtype=BF16, device=cuda)
    want[1:, 32767], want[1:, 3] = 16384.0, 8192.0   # 10,923 terms of 1.5 (16384.5, rounded) and 32,768 of 0.25
    assert torch.equal(y, want)
    del w, x, y, want
    rows, k, n = 70_001, 32768, 16
    x = torch.zeros(rows, k, dtype=BF16, device=cuda)
    x[-1, -1] = 2.0
    w = torch.zeros(2, n, k, dtype=BF16, device=cuda)
    w[1, :, -1] = 3.0
    offs = torch.tensor([0, 60_000, rows], dtype=torch.int32, device=cuda)
    xg, wg = x.requires_grad_(True), w.requires_grad_(True)
    gy = torch.zeros(rows, n, dtype=BF16, device=cuda)
    gy[-1] = 0.5
    y = experts.expert_linear(xg, wg, offs)
    gx, gw = torch.autograd.grad(y, (xg, wg), gy)
    assert (y[-1] == 6).all() and (y[:-1] == 0).all()
    assert gx[-1, -1] == 1.5 * n and gx.count_nonzero() == 1
    assert (gw[1, :, -1] == 1).all() and gw.count_nonzero() == n


@pytest.mark.parametrize("sizes,spare,n,k", CASES + [([600, 0, 500, 701], 9, 2560, 512),
                                                     ([1500, 0, 1300, 900, 1296], 40, 2560, 1000)])
def test_8_bits(sizes, spare, n, k, cuda):
    x, w, gy, offs = _inputs(sizes, spare, n, k, F32, 8, cuda)
    (xq, sx), (wq, sw) = fp8.quantize(x), fp8.quantize(w, tiles=True)
    xv, wv = fp8.dequantize(xq, sx), fp8.dequantize(wq, sw)
    for dt in (F32, BF16, F16):
        y = experts.expert_gemm_fp8(xq, sx, wq, sw, offs, dtype=dt)
        o = offs.tolist()
        for e in range(len(sizes)):
            a, b = xv[o[e]:o[e + 1]].double(), wv[e].double()
            grid = 7 * 2.0 ** -13 * (_largest_of_8(a) @ _largest_of_8(b).T)
            _close(y[o[e]:o[e + 1]], a @ b.T, a.abs() @ b.abs().T, k, BF16, grid)
        assert (y[o[-1]:] == 0).all()


def test_no_rows(cuda):
    w = torch.randn(3, 8, 16, device=cuda, requires_grad=True)
    x = torch.empty(0, 16, device=cuda, requires_grad=True)
    offs = torch.zeros(4, dtype=torch.int32, device=cuda)
    y = experts.expert_linear(x, w, offs)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty(0, 8, device=cuda))
    assert y.shape == (0, 8) and gx.shape == (0, 16) and torch.equal(gw, torch.zeros_like(w))


def test_graph_with_other_counts_and_streams(cuda):
    x, w, gy, offs = _inputs([100, 20, 0, 60], 20, 72, 128, BF16, 9, cuda)
    (xq, sx), (wq, sw) = fp8.quantize(x), fp8.quantize(w, tiles=True)

    def step():
        # leaves of its own: a leaf of an eager graph that lives is tied to that graph's stream
        X, W = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = experts.expert_linear(X, W, offs)
        gx, gw = torch.autograd.grad(y, (X, W), gy)
        return y.detach(), gx, gw, experts.expert_gemm_fp8(xq, sx, wq, sw, offs)

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
    for sizes in ([0, 0, 0, 200], [50, 50, 50, 50], [1, 0, 3, 2]):
        offs.copy_(torch.tensor([0] + sizes).cumsum(0))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), sizes
        _check(x, w, gy, offs, *held[:3])


def test_feed_forward_of_experts(cuda):
    """The operators together, as a block of experts uses them: norm with the residual, rows sorted by a router's choice, two
    products with an activation between them, rows back in their order; in 16 bits with gradients, in 8 bits for serving."""
    g = torch.Generator().manual_seed(11)
    rows, c, hidden, E = 500, 256, 384, 6

    def rand(*s):
        return torch.randn(*s, generator=g)

    branch, res = rand(rows, c).to(BF16).to(cuda).requires_grad_(True), rand(rows, c).to(BF16).to(cuda)
    gain = (1 + 0.1 * rand(c)).to(BF16).to(cuda).requires_grad_(True)
    w1 = (rand(E, hidden, c) / 16).to(BF16).to(cuda).requires_grad_(True)
    w2 = (rand(E, c, hidden) / 20).to(BF16).to(cuda).requires_grad_(True)
    chosen = torch.randint(0, E, (rows,), generator=g).to(cuda)
    chosen[chosen == 3] = 2                          # an expert without rows
    order = torch.argsort(chosen, stable=True)
    back = torch.argsort(order)
    offs = torch.searchsorted(chosen[order], torch.arange(E + 1, device=cuda)).to(torch.int32)

    y, h = norms.rms_norm(branch, gain, residual=res)
    a = torch.nn.functional.silu(experts.expert_linear(y[order], w1, offs))
    out = h + experts.expert_linear(a, w2, offs)[back]
    up = rand(rows, c).to(BF16).to(cuda)
    grads = torch.autograd.grad(out, (branch, gain, w1, w2), up)

    # the same in float64, from the same inputs
    b2, gain2, w12, w22 = (t.detach().double().requires_grad_(True) for t in (branch, gain, w1, w2))
    hd = b2 + res.double()
    yd = hd / torch.sqrt((hd * hd).mean(-1, keepdim=True) + 1e-5) * gain2
    ad = torch.nn.functional.silu((w12[chosen] @ yd[:, :, None])[:, :, 0])
    outd = hd + (w22[chosen] @ ad[:, :, None])[:, :, 0]
    want = torch.autograd.grad(outd, (b2, gain2, w12, w22), up.double())

    def off(t, ref):
        return float((t.detach().double() - ref.detach()).norm() / ref.detach().norm())

    # some eight roundings to bf16 on the way, 2^-9 rms each at most, and of independent signs
    assert off(out, outd) < 8 * 2.0 ** -9
    assert all(off(t, ref) < 8 * 2.0 ** -9 for t, ref in zip(grads, want))
    assert (grads[2][3] == 0).all() and (grads[3][3] == 0).all()

    with torch.no_grad():
        codes, scales, h8 = norms.rms_norm_fp8(branch, gain, residual=res)
        q1, s1 = fp8.quantize(w1, tiles=True)
        q2, s2 = fp8.quantize(w2, tiles=True)
        a8 = torch.nn.functional.silu(experts.expert_gemm_fp8(codes.view(torch.uint8)[order].view(torch.float8_e4m3fn),
                                                              scales[order], q1, s1, offs))
        out8 = h8 + experts.expert_gemm_fp8(*fp8.quantize(a8), q2, s2, offs)[back]
    assert torch.equal(h8, h)
    # four operands rounded to 3 bits, 2^-4 / sqrt(3) rms each at most, on the branch alone
    assert float((out8.double() - outd).norm()) < 4 * 2.0 ** -4 / 3 ** 0.5 * float((outd - hd).norm())


def test_out_counts_as_changed(cuda):
    """A graph that saved out's old elements, also those of a view, raises instead of taking the new ones."""
    x, w, gy, offs = _inputs([9, 0, 140], 8, 48, 64, BF16, 12, cuda)
    codes, scales = fp8.quantize(x)
    wq, ws = fp8.quantize(w, tiles=True)
    buf = torch.zeros(x.shape[0], 60, dtype=BF16, device=cuda)
    gain = torch.ones_like(buf, requires_grad=True)
    for call in (lambda out: experts.expert_linear(x, w, offs, out=out),
                 lambda out: experts.expert_gemm_fp8(codes, scales, wq, ws, offs, out=out)):
        z = buf * gain
        call(buf[:, 3:51])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
        torch.autograd.grad((buf * gain).sum(), gain)
    with torch.inference_mode():
        out = torch.empty(x.shape[0], 48, dtype=BF16, device=cuda)
        assert torch.equal(experts.expert_linear(x, w, offs, out=out)[:149], experts.expert_linear(x, w, offs)[:149])


@pytest.mark.parametrize("sizes,n,k", [([9, 0, 40], 48, 64), ([300, 513, 0, 31], 200, 264), ([40, 90], 33, 65), ([3, 2], 16, 40)])
def test_largest_fp32_operands(sizes, n, k, cuda):
    """Operands that bf16 rounds to infinity, up to fp32's largest, have finite pieces as all others have.  First pieces are
    cut, so that second ones are below 2^-7 and third ones at most 2^-16 of an operand: the products left out stay
    within the 4 2^-24 |a b| of the tolerance (2 2^-7 2^-16; where both come that near, |a b| is 2^-6 larger than its power
    of two, more than the 2^-32 of the product of third pieces)."""
    x, w, gy, offs = _inputs(sizes, 0, n, k, F32, 13, cuda)
    top = torch.finfo(F32).max
    gy *= 1e-3
    x[::4, 3], x[1::4, 3] = 3.3962e38, -top
    w[:, :, 3] *= 0.1
    w[:, 1, 2], w[:, 2, 2] = top, -3.4e38
    x[:, 2] *= 1e-3
    gy[2, 5], gy[3, 5] = top, -3.3962e38
    x[2:4] *= 1e-3
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = experts.expert_linear(xg, wg, offs)
    gx, gw = torch.autograd.grad(y, (xg, wg), gy)
    assert y.isfinite().all() and gx.isfinite().all() and gw.isfinite().all()
    _check(x, w, gy, offs, y, gx, gw)
    # what is not finite stays in its row
    x[1, 0], x[0, 0] = float("inf"), float("nan")
    bad = experts.expert_linear(x, w, offs)
    assert not bad[:2].isfinite().any() and torch.equal(bad[2:], y[2:])


@pytest.mark.parametrize("sizes,spare,n,k", [([1], 0, 1, 1), ([5, 130, 0, 17], 3, 64, 131), ([3, 0, 2, 1], 2, 40, 515),
                                             ([20] * 70 + [0] * 3 + [200], 11, 96, 33), ([700, 0, 513], 5, 130, 257),
                                             ([3000, 0, 2500, 1300], 40, 1500, 145)])
def test_8_bits_on_any_boundary(sizes, spare, n, k, cuda):
    """Codes packed without padding, starting on every byte of a dword, with NaN codes around and in rows of no expert."""
    x, w, gy, offs = _inputs(sizes, spare, n, k, F32, 14, cuda)
    (xq, sx), (wq, sw) = fp8.quantize(x), fp8.quantize(w, tiles=True)
    xv, wv = fp8.dequantize(xq, sx), fp8.dequantize(wq, sw)
    o = offs.tolist()
    for skew in range(4):
        def moved(q):
            flat = torch.full((q.numel() + 40,), 0x7F, dtype=torch.uint8, device=cuda)
            view = flat[skew:skew + q.numel()].view(q.shape)
            view.copy_(q.contiguous().view(torch.uint8))
            return view
        xs, ws = moved(xq), moved(wq)
        xs[o[-1]:] = 0x7F
        y = experts.expert_gemm_fp8(xs.view(torch.float8_e4m3fn), sx, ws.view(torch.float8_e4m3fn), sw, offs, dtype=F32)
        for e in range(len(sizes)):
            a, b = xv[o[e]:o[e + 1]].double(), wv[e].double()
            grid = 7 * 2.0 ** -13 * (_largest_of_8(a) @ _largest_of_8(b).T)
            _close(y[o[e]:o[e + 1]], a @ b.T, a.abs() @ b.abs().T, k, BF16, grid)
        assert (y[o[-1]:] == 0).all()


# the weights' gradient in parts of the rows; more tiles than workgroups in every pass
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes,spare,n,k", [([5000, 0, 3001], 7, 131, 203), ([9000], 3, 65, 257), ([4000, 0, 3500, 2900], 9, 1027, 1301)])
def test_odd_widths_with_many_rows(sizes, spare, n, k, dtype, cuda):
    x, w, gy, offs = _inputs(sizes, spare, n, k, dtype, 15, cuda)
    x[-spare:], gy[-spare:] = float("nan"), float("inf")
    cut = experts._workspace_bytes(x.shape[0], n, k, len(sizes)) > 0
    tiles = [sum(-(-s // 128) for s in sizes) * -(-n // 128), len(sizes) * -(-n // 128) * -(-k // 128)]
    assert cut or min(tiles) > 256 and tiles[0] > 512
    x.requires_grad_(True), w.requires_grad_(True)
    y = experts.expert_linear(x, w, offs)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    _check(x, w, gy, offs, y, gx, gw)


def test_more_experts_tiles_than_workgroups_on_odd_widths(cuda):
    """The weights' gradient with several tiles of different experts in turn for a workgroup."""
    x, w, gy, offs = _inputs([37, 0, 300, 5, 64, 129, 1, 200] * 8, 3, 387, 519, BF16, 16, cuda)
    x.requires_grad_(True), w.requires_grad_(True)
    y = experts.expert_linear(x, w, offs)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    _check(x, w, gy, offs, y, gx, gw)
