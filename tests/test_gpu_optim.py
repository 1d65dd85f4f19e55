"""optim.AdamW, clip_grad_norm_ and grad_norm (csrc/optim.hip) against their formulas in float64, one step at a time
from the kernel's own state, so that errors do not compound.

Tolerances (u = 2^-24, half a step of fp32): a moment is two products and a sum of numbers that carry a scaled
gradient's two roundings: 6 u of the two terms' magnitudes.  The update's factor has an expm1 of a rounded argument (4
u), two quotients, two roots and three products: 24 u of its magnitude, besides the moments' errors (the root halves
v's).  A parameter adds one subtraction and its type's rounding uT."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
UT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SHAPES = [(1,), (3,), (63,), (64,), (65,), (37, 129), (0,), (4096,), (4097,), (2, 5, 8191), (31,), (32,), (33,),
          (20001,)]


def _params(shapes, dtype, cuda, seed, shift=0):
    """Parameters with gradients; ``shift``: that many elements off an allocation's start."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for k, s in enumerate(shapes):
        n = math.prod(s)
        p = torch.empty(n + shift, dtype=dtype, device=cuda)[shift:].view(s)
        p.copy_(0.1 * torch.randn(s, generator=g))
        p.requires_grad_(True)
        gr = torch.empty(n + shift, dtype=dtype, device=cuda)[shift:].view(s)
        gr.copy_(10.0 ** (k % 4 - 3) * torch.randn(s, generator=g))
        p.grad = gr
        out.append(p)
    return out


def _step64(p, g, m, v, t, lr, b1, b2, eps, wd):
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    up = lr / (1 - b1 ** t) * m2 / ((v2 / (1 - b2 ** t)).sqrt() + eps)
    return p - lr * wd * p - up, m2, v2, up


def _check_step(p, p0, g, m0, v0, m, v, t, hyper, bits=32):
    """One parameter's step within the bounds above (all float64 but p)."""
    lr, b1, b2, eps, wd = hyper
    P, M, V, up = _step64(p0, g, m0, v0, t, *hyper)
    em = 6 * U * ((b1 * m0).abs() + ((1 - b1) * g).abs())
    ev = 6 * U * V
    if bits == 32:
        assert (m - M).abs().le(em + 1e-42).all() and (v - V).abs().le(ev + 1e-42).all()
    den = (V / (1 - b2 ** t)).sqrt() + eps
    eu = lr / (1 - b1 ** t) * em / den + (24 + 3) * U * up.abs() + lr * wd * 4 * U * p0.abs()
    tol = 1.01 * eu + (U + 1.01 * UT[p.dtype]) * P.abs() + (2.0 ** -25 if p.dtype == torch.float16 else 1e-42)
    assert (p.double() - P).abs().le(tol).all(), float(((p.double() - P).abs() / tol).max())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,shift", [(torch.float32, 0), (torch.float32, 1), (torch.bfloat16, 0),
                                         (torch.bfloat16, 3), (torch.float16, 0), (torch.float16, 1)])
def test_steps(pkg, cuda, dtype, shift, bits):
    """Several steps with new gradients, two groups with their own values, clipped."""
    from ubio_molfm_amd import optim
    ps = _params(SHAPES, dtype, cuda, 1, shift)
    hyper = [(3e-3, 0.9, 0.999, 1e-8, 0.01), (1e-3, 0.5, 0.95, 1e-6, 0.0)]
    groups = [dict(params=ps[k::2], lr=h[0], betas=h[1:3], eps=h[3], weight_decay=h[4]) for k, h in enumerate(hyper)]
    opt = optim.AdamW(groups, state_bits=bits, max_norm=0.5, seed=3)
    order = ps[0::2] + ps[1::2]
    g = torch.Generator().manual_seed(8)
    for t in range(1, 5):
        before = [p.detach().double().clone() for p in order]
        m0, v0 = (x.double().clone() for x in opt.moments())
        grads = [p.grad.double().clone() for p in order]
        opt.step()
        norm = math.sqrt(sum(float(x.square().sum()) for x in grads))
        assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        c = min(1.0, 0.5 / (norm + 1e-6))
        m, v = (x.double() for x in opt.moments())
        off = 0
        for k, (p, p0, gr) in enumerate(zip(order, before, grads)):
            n = p.numel()
            cut = [x[off:off + n].view(p.shape) for x in (m0, v0, m, v)]
            off += -(-n // 64) * 64
            assert torch.equal(p.grad.double(), gr)                   # left as they were
            st = opt.state[p]
            assert int(st["step"]) == (t if n else 0)
            _check_step(p.detach(), p0, c * gr, *cut, t, hyper[0 if k < len(ps[0::2]) else 1], bits)
        assert off == m.numel()
        for p in ps:
            p.grad = (10.0 ** (t % 3 - 2) * torch.randn(p.shape, generator=g)).to(dtype).to(cuda)


def _hash(x):
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _grid(x, bits):
    """The step of the codes at x (float64), runs of 32 along the last dimension of the flat x."""
    signed = bits == 4
    top = x.abs().view(-1, 32).amax(1)
    e = torch.where(top > 0, torch.frexp(top)[1].double() - 1, -200.0)
    e = torch.where(top > (1.875 if signed else 1.75) * torch.exp2(e), e + 1, e).repeat_interleave(32)
    low = e - (2 ** bits - 2)
    return torch.exp2(torch.maximum(torch.where(x != 0, torch.frexp(x.abs())[1].double() - 1, -2000.0), low) - 3)


def test_eight_bit_codes(pkg, cuda):
    """The stored moments: each is the float64 result rounded down or up to a code as the hash of seed, step and
    element says, but where fp32 rounding (2^-18 of a step at most: 6 u of a value of at most 16 steps, and the move
    into place) takes the sum of fraction and random part across one."""
    from ubio_molfm_amd import optim
    ps = _params([(5000,), (96,), (33,)], torch.float32, cuda, 4)
    opt = optim.AdamW(ps, lr=1e-3, state_bits=8, seed=77)
    for t in range(1, 6):
        m0, v0 = (x.double() for x in opt.moments())
        opt.step()
        m, v = (x.double() for x in opt.moments())
        g = torch.zeros_like(m)
        off = 0
        for p in ps:
            g[off:off + p.numel()] = p.grad.double()
            off += -(-p.numel() // 64) * 64
        _, M, V, _ = _step64(0.0, g, m0, v0, t, 1e-3, 0.9, 0.999, 1e-8, 0.0)
        key = _hash((_hash(77) + t * 0x9E3779B9) & 0xFFFFFFFF)
        u = _hash(torch.arange(m.numel(), device=cuda) ^ key)
        for got, ref, bits, r in ((m, M, 4, u & 0xFFFF), (v, V, 5, u >> 16)):
            step = _grid(ref, bits)
            f = ref.abs() / step + (16 * r + 8).double() / 2 ** 20
            want = torch.sign(ref) * torch.floor(f) * step
            if bits == 5:
                want = torch.where(ref > 0, torch.maximum(want, step), want)
            near = (f - torch.round(f)).abs() < 2.0 ** -18
            assert torch.equal(got[~near], want[~near]) and near.sum() < 3
            assert (got - ref).abs().le(1.001 * step).all()
        for p in ps:
            p.grad = p.grad.roll(7) * (1.5 - 0.2 * t)


def test_eight_bit_moments_follow_the_mean(pkg, cuda):
    """Constant gradients, 500 steps.  A step moves v by 0.1% of its distance: the nearest code, 6% to 12% apart, would
    never be left.  Stochastically rounded, v's mean is that of the recursion; a step's rounding has variance at most
    (0.001 + 0.001) v^2 / 8 with memory 1/0.002, 0.35 v over one element and 0.0055 v over 4,096: five of those, and
    likewise m (0.1 / 8 and 1/0.19)."""
    from ubio_molfm_amd import optim
    p = torch.zeros(4096, device=cuda, requires_grad=True)
    p.grad = torch.full_like(p, 0.7)
    opt = optim.AdamW([p], lr=1e-6, state_bits=8)
    for _ in range(500):
        opt.step()
    m, v = (x.double().mean().item() for x in opt.moments())
    ev = 0.49 * (1 - 0.999 ** 500)
    assert abs(v - ev) < 5 * 0.0055 * ev * 1.3 and abs(m - 0.7) < 5 * 0.7 * math.sqrt(0.1 / 8 / 0.19 / 4096)


@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite_stay_with_their_element(pkg, cuda, bits):
    from ubio_molfm_amd import optim
    ps = _params([(200,)], torch.float32, cuda, 6)
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    bad = torch.zeros(200, dtype=torch.bool, device=cuda)
    bad[[3, 70, 71, 199]] = True
    g = ps[0].grad.clone()
    qs[0].grad = torch.where(bad, 0.0, g)
    ps[0].grad = torch.where(bad, torch.tensor(float("nan"), device=cuda), g)
    ps[0].grad[70] = float("inf")
    a, b = (optim.AdamW(x, lr=1e-3, state_bits=bits) for x in (ps, qs))
    for _ in range(3):
        a.step(), b.step()
    assert ps[0][bad].isnan().all() and torch.equal(ps[0][~bad], qs[0][~bad])
    for x, y in zip(a.moments(), b.moments()):
        assert torch.equal(x[:200][~bad], y[:200][~bad]) and not x[:200][bad].isfinite().any()


def test_many_tensors(pkg, cuda):
    """More tensors than a norm launch (256) and a step launch (384) take; one is large, some have no gradient."""
    from ubio_molfm_amd import optim
    shapes = [(k % 97 + 1,) for k in range(900)] + [(300, 1001)]
    ps = _params(shapes, torch.float32, cuda, 2)
    for p in ps[5::7]:
        p.grad = None
    opt = optim.AdamW(ps, lr=1e-3, max_norm=1e9)
    before = [p.detach().double().clone() for p in ps]
    opt.step()
    grads = [p.grad for p in ps if p.grad is not None]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    assert abs(float(optim.grad_norm(grads)) - norm) <= 2 * U * norm
    for p, p0 in zip(ps, before):
        st = opt.state[p]
        if p.grad is None:
            assert torch.equal(p.double(), p0) and int(st["step"]) == 0 and not st["exp_avg"].any()
        else:
            z = torch.zeros_like(p0)
            _check_step(p.detach(), p0, p.grad.double(), z, z, st["exp_avg"].double(), st["exp_avg_sq"].double(), 1,
                        (1e-3, 0.9, 0.999, 1e-8, 0.01))
    for p in ps[5::7]:
        p.grad = torch.ones_like(p)
    opt.step()
    assert {int(opt.state[p]["step"]) for p in ps[5::7]} == {1} and int(opt.state[ps[0]]["step"]) == 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("max_norm", [0.3, 1e6])
def test_clip(pkg, cuda, dtype, max_norm):
    from ubio_molfm_amd import optim
    ps = _params(SHAPES, dtype, cuda, 5, shift=1) + _params([(70, 40)], dtype, cuda, 9)
    ps.append(_params([(40, 70)], dtype, cuda, 10)[0])
    ps[-1].grad = ps[-2].grad.clone().t()                                 # strides of a transposed matrix
    assert not ps[-1].grad.is_contiguous()
    grads = [p.grad.double().clone() for p in ps]
    versions = [p.grad._version for p in ps]
    norm = math.sqrt(sum(float(g.square().sum()) for g in grads))
    got = optim.clip_grad_norm_(ps, max_norm)
    assert got.shape == () and got.dtype == torch.float32 and abs(float(got) - norm) <= 2 * U * norm
    c = min(1.0, max_norm / (norm + 1e-6))
    for p, g, v in zip(ps, grads, versions):
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
        assert (p.grad.double() - c * g).abs().le((3 * U + 1.01 * UT[dtype]) * (c * g).abs() + tiny).all()
        assert p.grad._version > v
    assert torch.equal(optim.clip_grad_norm_(ps[:0], 1.0).cpu(), torch.zeros(()))


def test_norms_at_the_edges(pkg, cuda):
    """Squares that overflow fp32 or vanish in it, elements that are not finite, empty lists."""
    from ubio_molfm_amd import optim
    big = torch.full((3, 5), 1e30, device=cuda)
    assert abs(float(optim.grad_norm(big)) / (1e30 * math.sqrt(15)) - 1) < 4 * U
    small = torch.full((4,), 1e-30, device=cuda)
    assert abs(float(optim.grad_norm([small])) / 2e-30 - 1) < 4 * U
    assert float(optim.grad_norm([])) == 0 and float(optim.grad_norm([torch.empty(0, device=cuda)])) == 0
    mixed = [torch.ones(3, device=cuda), torch.ones(6, device=cuda).bfloat16(), torch.ones(7, device=cuda).half()]
    assert float(optim.grad_norm(mixed)) == 4.0
    p = torch.zeros(4, device=cuda, requires_grad=True)
    p.grad = torch.tensor([1.0, float("inf"), 2.0, -3.0], device=cuda)
    assert float(optim.clip_grad_norm_([p], 1.0)) == math.inf
    assert p.grad[1].isnan() and (p.grad[[0, 2, 3]] == 0).all()
    p.grad = torch.tensor([1.0, float("nan"), 2.0, -3.0], device=cuda)
    assert math.isnan(float(optim.clip_grad_norm_([p], 1.0))) and p.grad.isnan().all()


@pytest.mark.parametrize("bits", [32, 8])
def test_skipped_steps(pkg, cuda, bits):
    from ubio_molfm_amd import optim
    ps = _params(SHAPES, torch.float32, cuda, 3)
    opt = optim.AdamW(ps, lr=1e-2, state_bits=bits, skip_nonfinite=True)
    opt.step()
    good = ps[4].grad.clone()
    keep = [p.detach().clone() for p in ps] + [x.clone() for x in opt.moments()]
    for bad in (float("nan"), float("inf")):
        ps[4].grad[64] = bad
        opt.step()
        assert all(torch.equal(a, b) for a, b in zip(keep, [p.detach() for p in ps] + list(opt.moments())))
        assert not opt.grad_norm.isfinite()
    assert int(opt.skipped) == 2 and int(opt.state[ps[0]]["step"]) == 1
    ps[4].grad.copy_(good)
    opt.step()
    assert int(opt.skipped) == 2 and int(opt.state[ps[0]]["step"]) == 2 and not torch.equal(ps[0].detach(), keep[0])


@pytest.mark.parametrize("bits,dtype", [(32, torch.float32), (32, torch.bfloat16), (8, torch.float32),
                                        (8, torch.bfloat16)])
def test_state_goes_on(pkg, cuda, bits, dtype):
    """A saved and loaded state, a copied optimizer, parameters that moved, and one more group: each goes on bitwise as
    the first."""
    from ubio_molfm_amd import optim

    def fresh(src):
        qs = [p.detach().clone().requires_grad_(True) for p in src]
        for p, q in zip(src, qs):
            q.grad = p.grad.clone()
        return qs

    ps = _params(SHAPES, dtype, cuda, 7)
    a = optim.AdamW(ps, lr=1e-3, state_bits=bits, seed=5, max_norm=2.0)
    for _ in range(2):
        a.step()
    qs = fresh(ps)
    b = optim.AdamW(qs, lr=0.5, state_bits=bits, seed=5, max_norm=2.0)
    sd = {k: copy.deepcopy(v) for k, v in a.state_dict().items()}
    sd["state"] = {i: {k: t.cpu() for k, t in e.items()} for i, e in sd["state"].items()}
    b.load_state_dict(sd)
    assert b.param_groups[0]["lr"] == 1e-3 and b.state[qs[0]]["exp_avg"].is_cuda
    rs = copy.deepcopy((a, ps))
    c, ts = rs
    for p, t in zip(ps, ts):
        t.grad = p.grad.clone()
    assert c.param_groups[0]["params"][3] is ts[3]
    for step in range(2):
        for o in (a, b, c):
            o.step()
        for p in qs:
            p.data = p.data.clone()                               # other memory from here on
    for p, q, t in zip(ps, qs, ts):
        assert torch.equal(p, q) and torch.equal(p, t) and int(a.state[p]["step"]) == int(b.state[q]["step"])
    for x, y, z in zip(a.moments(), b.moments(), c.moments()):
        assert torch.equal(x, y) and torch.equal(x, z)
    extra = _params([(50,)], dtype, cuda, 12)
    m0 = a.moments()[0].clone()
    a.add_param_group(dict(params=extra, lr=1e-2))
    a.step()
    assert int(a.state[extra[0]]["step"]) == 1 and int(a.state[ps[0]]["step"]) == 5
    assert a.moments()[0].numel() == m0.numel() + 64


def test_takes_a_torch_checkpoint(pkg, cuda):
    from ubio_molfm_amd import optim
    ps = _params(SHAPES, torch.float32, cuda, 13)
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = p.grad
    a = torch.optim.AdamW(qs, lr=1e-3)
    for _ in range(3):
        a.step()
    for p, q in zip(ps, qs):
        p.data.copy_(q.data)
    b = optim.AdamW(ps, lr=1e-3)
    b.load_state_dict({"state": a.state_dict()["state"], "param_groups": b.state_dict()["param_groups"]})
    before, m0, v0 = [p.detach().double().clone() for p in ps], *(x.double().clone() for x in b.moments())
    b.step()
    off = 0
    for p, p0 in zip(ps, before):
        n = p.numel()
        st = b.state[p]
        _check_step(p.detach(), p0, p.grad.double(), m0[off:off + n].view(p.shape), v0[off:off + n].view(p.shape),
                    st["exp_avg"].double(), st["exp_avg_sq"].double(), 4, (1e-3, 0.9, 0.999, 1e-8, 0.01))
        off += -(-n // 64) * 64
    with pytest.raises(ValueError, match="exp_avg_scale"):
        optim.AdamW(ps, state_bits=8).load_state_dict(
            {"state": a.state_dict()["state"], "param_groups": b.state_dict()["param_groups"]})


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_and_streams(pkg, cuda, bits):
    """A captured step with a learning rate on the device, replayed on new gradients with eager work between, against
    eager steps; and a step on a stream of its own."""
    from ubio_molfm_amd import optim
    ps, qs = (_params(SHAPES, torch.float32, cuda, 21) for _ in range(2))
    lr_a, lr_b = (torch.tensor(1e-3, device=cuda) for _ in range(2))
    a, b = (optim.AdamW(x, lr=lr, state_bits=bits, max_norm=0.4, skip_nonfinite=True, seed=1)
            for x, lr in ((ps, lr_a), (qs, lr_b)))
    with pytest.raises(RuntimeError, match="captured"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    other = _params([(1000,)], torch.float32, cuda, 30)
    o = optim.AdamW(other)
    for k in range(4):
        for p, q in zip(ps, qs):
            g = torch.randn(p.shape, generator=torch.Generator().manual_seed(k)).to(cuda)
            if k == 2 and p.numel():
                g.view(-1)[0] = float("inf")
            p.grad.copy_(g)
            q.grad.copy_(g)
        lr_a.mul_(0.7)
        lr_b.mul_(0.7)
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        o.step()
        optim.clip_grad_norm_(other, 0.1)
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), k
        assert all(torch.equal(x, y) for x, y in zip(a.moments(), b.moments()))
        assert torch.equal(a.grad_norm, b.grad_norm) or k == 2
    assert int(a.skipped) == int(b.skipped) == 1 and int(a.state[ps[0]]["step"]) == 4


def test_clip_in_a_graph(pkg, cuda):
    from ubio_molfm_amd import optim
    ps = _params(SHAPES, torch.float32, cuda, 22)
    optim.clip_grad_norm_(ps, 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = optim.clip_grad_norm_(ps, 0.5)
    for k in range(3):
        qs = _params(SHAPES, torch.float32, cuda, 40 + k)
        for p, q in zip(ps, qs):
            p.grad.copy_(q.grad)
        graph.replay()
        torch.cuda.synchronize()
        want = optim.clip_grad_norm_(qs, 0.5)
        assert torch.equal(norm, want) and all(torch.equal(p.grad, q.grad) for p, q in zip(ps, qs))


def test_refusals(pkg, cuda):
    from ubio_molfm_amd import optim
    p = torch.zeros(4, 6, device=cuda).t().requires_grad_(True)
    p.grad = torch.zeros_like(p)
    with pytest.raises(ValueError, match="contiguous"):
        optim.AdamW([p]).step()
    d = torch.zeros(4, device=cuda, dtype=torch.float64, requires_grad=True)
    d.grad = torch.zeros_like(d)
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        optim.AdamW([d]).step()
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        optim.clip_grad_norm_([d], 1.0)
    s = torch.zeros(4, 3, device=cuda, requires_grad=True)
    s.grad = torch.sparse_coo_tensor([[1], [0]], [1.0], (4, 3), device=cuda)
    with pytest.raises(ValueError, match="sparse"):
        optim.AdamW([s]).step()
    with pytest.raises(ValueError, match="sparse"):
        optim.clip_grad_norm_([s], 1.0)
    with pytest.raises(RuntimeError, match="GPU only"):
        optim.grad_norm([torch.ones(3, device=cuda), torch.ones(3)])


def test_gradients_that_are_not_contiguous(pkg, cuda):
    from ubio_molfm_amd import optim
    p, q = (torch.ones(30, 50, device=cuda, requires_grad=True) for _ in range(2))
    g = torch.randn(50, 30, generator=torch.Generator().manual_seed(1)).to(cuda)
    p.grad, q.grad = g.t(), g.t().contiguous()
    a, b = optim.AdamW([p], max_norm=1.0), optim.AdamW([q], max_norm=1.0)
    a.step(), b.step()
    assert torch.equal(p, q)
    p.grad, q.grad = g[:1].t()[:, :1].expand(30, 50), g[:1].t()[:, :1].expand(30, 50).contiguous()
    a.step(), b.step()
    assert torch.equal(p, q) and torch.equal(a.grad_norm, b.grad_norm)


def test_scheduler_and_closure(pkg, cuda):
    from ubio_molfm_amd import optim
    p = torch.full((10,), 2.0, device=cuda, requires_grad=True)
    opt = optim.AdamW([p], lr=1e-2, weight_decay=0.0)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.5 ** k)

    def closure():
        opt.zero_grad()
        loss = p.square().sum()
        loss.backward()
        return loss

    seen = [float(opt.step(closure))]
    sched.step()
    seen.append(float(opt.step(closure)))
    # both steps are lr times a sign, within the effect of eps and of the second step's slightly smaller gradient
    assert seen[0] == 40.0 and abs(float(p[0]) - (2.0 - 1e-2 - 0.5e-2)) < 1e-4 and opt.param_groups[0]["lr"] == 5e-3


def test_training_run(pkg, cuda):
    """The operators as they are used: a net with layer norms whose loss holds a gradient (forces), clipped AdamW
    steps; against torch's modules, clipping and AdamW in float64.  Each of five steps moves a parameter by at most
    about lr = 1e-3; the gradients agree to 1e-5, the steps' directions where sqrt(v) is not small against that: 1e-3
    of the distance travelled, in the 2-norm."""
    from ubio_molfm_amd import optim
    from ubio_molfm_amd import second_order as so
    torch.manual_seed(3)
    net = torch.nn.Sequential(torch.nn.Linear(12, 96), torch.nn.LayerNorm(96), torch.nn.SiLU(), torch.nn.Linear(96, 48),
                              torch.nn.LayerNorm(48), torch.nn.Linear(48, 1)).to(cuda)
    ref = copy.deepcopy(net).double()
    start = [p.detach().double().clone() for p in net.parameters()]
    a = optim.AdamW(net.parameters(), lr=1e-3, max_norm=1.0)
    b = torch.optim.AdamW(ref.parameters(), lr=1e-3)
    x = torch.randn(200, 12, device=cuda)

    def loss(f, net, x):
        x = x.clone().requires_grad_(True)
        e = f(net, x).sum()
        gx, = torch.autograd.grad(e, x, create_graph=True)
        return (gx - 1).square().mean() + e.square() / 200

    for _ in range(5):
        a.zero_grad(), b.zero_grad()
        loss(so.run_seq, net, x).backward()
        loss(lambda m, h: m(h), ref, x.double()).backward()
        # the last layers' biases that force training does not reach have no gradient on either side
        assert [p.grad is None for p in net.parameters()] == [p.grad is None for p in ref.parameters()]
        n64 = torch.nn.utils.clip_grad_norm_(ref.parameters(), 1.0)
        a.step(), b.step()
        assert abs(float(a.grad_norm) / float(n64) - 1) < 1e-4
    for p, q, s in zip(net.parameters(), ref.parameters(), start):
        assert float((p.double() - q).norm()) <= 1e-3 * float((q - s).norm()) + 1e-9


def test_model_sees_the_new_weights(pkg, cuda):
    """What the model keeps per weight version (packed weights, distance tables) is made anew after a step: its
    energies are bitwise those of a new model with the same weights."""
    from ubio_molfm_amd import model, optim, systems
    torch.manual_seed(0)
    m = model.MolfmAtomic(model.default_args()).to(cuda)
    sysd = systems.small_water(8, 6.2, seed=3)
    pos, Z = (torch.as_tensor(sysd[k], device=cuda) for k in ("pos", "Z"))

    def energy(m):
        return m.eval().energy_forces_flat(pos, Z, sysd["graph_ptr"], sysd["cell"], sysd["pbc"])[0].detach().clone()

    e0 = energy(m)
    g = torch.Generator().manual_seed(1)
    ps = [p for p in m.parameters() if p.requires_grad]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g).to(cuda)
    optim.AdamW(ps, lr=1e-3).step()
    e1 = energy(m)
    other = model.MolfmAtomic(model.default_args()).to(cuda)
    other.load_state_dict(m.state_dict())
    assert not torch.equal(e0, e1) and torch.equal(e1, energy(other))


def test_parameters_without_gradients_of_any_kind(pkg, cuda):
    """A model's constants stand in the groups: whole numbers, transposed and host tensors, none with a gradient."""
    from ubio_molfm_amd import optim
    ps = _params([(40,)], torch.float32, cuda, 1)
    odd = [torch.nn.Parameter(t, requires_grad=t.is_floating_point())
           for t in (torch.arange(5, device=cuda), torch.zeros(4, 6, device=cuda).t(), torch.zeros(3))]
    opt = optim.AdamW(odd[:2] + ps + odd[2:], lr=1e-3)
    opt.step()
    assert int(opt.state[ps[0]]["step"]) == 1 and not any(p in opt.state for p in odd)
    sd = opt.state_dict()
    assert list(sd["state"]) == [2]
    opt.load_state_dict(sd)
    odd[1].grad = torch.ones_like(odd[1])
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    empty = optim.AdamW(odd[:1])
    empty.step()
    assert empty.moments()[0].numel() == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_goes_on_after_load_state_dict(pkg, cuda, bits):
    """A loaded state goes into the buffers that are there: a step captured before takes up the new state."""
    from ubio_molfm_amd import optim
    ps, qs = (_params(SHAPES, torch.float32, cuda, 51) for _ in range(2))
    a, b = (optim.AdamW(x, lr=1e-3, state_bits=bits, seed=2) for x in (ps, qs))
    a.step(), b.step()
    saved = copy.deepcopy(a.state_dict())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    graph.replay()
    torch.cuda.synchronize()
    ptr = a.state[ps[3]]["exp_avg"].data_ptr()
    a.load_state_dict(saved)
    assert a.state[ps[3]]["exp_avg"].data_ptr() == ptr and int(a.state[ps[3]]["step"]) == 1
    for p, q in zip(ps, qs):
        p.data.copy_(q.data)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    a.param_groups[0]["lr"] = 0.0                                    # the groups are the loaded ones
    before = ps[3].detach().clone()
    a.step()
    assert torch.equal(ps[3], before) and int(a.state[ps[3]]["step"]) == 4


def test_states_that_are_taken_out_start_anew(pkg, cuda):
    from ubio_molfm_amd import optim
    ps = _params([(100,), (5000,)], torch.float32, cuda, 52)
    opt = optim.AdamW(ps, lr=1e-3)
    for _ in range(3):
        opt.step()
    kept = opt.state[ps[1]]["exp_avg"].clone()
    del opt.state[ps[0]]
    opt.step()
    assert int(opt.state[ps[0]]["step"]) == 1 and int(opt.state[ps[1]]["step"]) == 4
    assert not torch.equal(opt.state[ps[1]]["exp_avg"], kept)
    opt.state.clear()
    opt.step()
    assert {int(opt.state[p]["step"]) for p in ps} == {1}


def test_what_cannot_be_updated_is_refused(pkg, cuda):
    """Memory that two parameters or two gradients share would be written by two workgroups at once; a checkpoint of
    another method would go on as this one."""
    from ubio_molfm_amd import optim
    flat = torch.zeros(100, device=cuda)
    a, b = flat[:60].requires_grad_(True), flat[50:].requires_grad_(True)
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    with pytest.raises(ValueError, match="share memory"):
        optim.AdamW([a, b]).step()
    optim.AdamW([flat[:50].requires_grad_(True), flat[50:].requires_grad_(True)]).step()
    with pytest.raises(ValueError, match="twice"):
        optim.clip_grad_norm_([a, a], 1.0)
    p = torch.zeros(3, device=cuda, requires_grad=True)
    p.grad = torch.ones_like(p)
    for other, match in ((torch.optim.AdamW([p], amsgrad=True), "amsgrad"),
                         (torch.optim.AdamW([p], maximize=True), "maximize"),
                         (torch.optim.Adam([p], weight_decay=0.1), "decay")):
        other.step()
        opt = optim.AdamW([p], lr=0.25)
        with pytest.raises(ValueError, match=match):
            opt.load_state_dict(other.state_dict())
        assert opt.param_groups[0]["lr"] == 0.25
    good = torch.optim.Adam([p], lr=2e-3)
    good.step()
    opt = optim.AdamW([p])
    opt.load_state_dict(good.state_dict())
    assert opt.param_groups[0]["lr"] == 2e-3 and int(opt.state[p]["step"]) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_loading_its_own_state_changes_nothing(pkg, cuda, bits):
    """state_dict refers to the state itself; loading it back keeps it, and parameters that a checkpoint leaves out
    start anew."""
    from ubio_molfm_amd import optim
    ps = _params(SHAPES, torch.float32, cuda, 53)
    opt = optim.AdamW(ps, lr=1e-3, state_bits=bits)
    opt.step(), opt.step()
    before = [x.clone() for x in opt.moments()]
    sd = opt.state_dict()
    opt.load_state_dict(sd)
    assert all(torch.equal(x, y) for x, y in zip(before, opt.moments())) and int(opt.state[ps[5]]["step"]) == 2
    sd = copy.deepcopy(sd)
    del sd["state"][5]
    opt.load_state_dict(sd)
    assert int(opt.state[ps[5]]["step"]) == 0 and not opt.state[ps[5]]["exp_avg"].any()
    assert int(opt.state[ps[8]]["step"]) == 2
    opt.step()
    assert int(opt.state[ps[5]]["step"]) == 1 and int(opt.state[ps[8]]["step"]) == 3


def test_tiny_gradients_without_eps(pkg, cuda):
    """Second moments below the smallest normal number (g^2 (1 - b2) from 1e-43 on) still scale the update: against the
    formula in float64 from the moments that the kernel stored, with the update's factor as above."""
    from ubio_molfm_amd import optim
    p = torch.zeros(4100, device=cuda).requires_grad_(True)
    p.grad = torch.logspace(-20, -12, 4100, device=cuda) * (1 - 2 * (torch.arange(4100, device=cuda) % 2))
    opt = optim.AdamW([p], lr=1e-3, eps=0.0, weight_decay=0.0)
    opt.step()
    m, v = (opt.state[p][k].double() for k in ("exp_avg", "exp_avg_sq"))
    assert (v > 0).all() and v.min() < 1e-42
    want = -1e-3 / (1 - 0.9) * m / (v / (1 - 0.999)).sqrt()
    assert (p.detach().double() - want).abs().le((24 + 3) * U * want.abs()).all()
    # eps on both sides of 2^-38 / (1 - b2)^(1/2): second moments that still count beside it, and that round away
    for eps in (2e-21, 1.1e-10, 1.2e-10, 1e-8):
        p.data.zero_()
        opt = optim.AdamW([p], lr=1e-3, eps=eps, weight_decay=0.0)
        opt.step()
        m, v = (opt.state[p][k].double() for k in ("exp_avg", "exp_avg_sq"))
        want = -1e-3 / (1 - 0.9) * m / ((v / (1 - 0.999)).sqrt() + eps)
        assert (p.detach().double() - want).abs().le((24 + 3) * U * want.abs() + 1e-42).all()
    q = torch.ones(5, device=cuda).requires_grad_(True)
    q.grad = torch.zeros(5, device=cuda)
    optim.AdamW([q], eps=1e-42, weight_decay=0.0).step()
    assert torch.equal(q.detach(), torch.ones(5, device=cuda))


def test_groups_that_are_changed_by_hand(pkg, cuda):
    """A group or a parameter taken out stays as it is, one put in its place or added is updated, the others go on."""
    from ubio_molfm_amd import optim
    ps = _params([(70,), (64,), (4100,), (9,)], torch.float32, cuda, 4)
    ref = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, r in zip(ps, ref):
        r.grad = p.grad.clone()
    kw = dict(lr=1e-2, weight_decay=0.1)
    opts = [cls([dict(params=q[:2]), dict(params=[q[2]], lr=2e-2)], **kw)
            for cls, q in ((optim.AdamW, ps), (torch.optim.AdamW, ref))]

    def check():
        for o in opts:
            o.step()
        for p, r in zip(ps, ref):
            # each of up to 4 steps: 27 u of an update below 2 lr, and the sums' roundings, on both sides
            assert (p - r).abs().max() <= 4 * 2 * (27 * U * 4e-2 + 3 * U * float(r.detach().abs().max()))

    check()
    for o in opts:
        o.param_groups.pop()
    check()
    for o, q in zip(opts, (ps, ref)):
        o.param_groups[0]["params"][1] = q[3]
    check()
    for o, q in zip(opts, (ps, ref)):
        o.param_groups[0]["params"].append(q[2])
    check()


def test_parameters_whose_memory_is_cut_turned_or_brought(pkg, cuda):
    """.data that starts where it did with fewer elements or other strides, gradients of another size, a parameter that
    comes to the GPU after a step: each is seen before the launch."""
    from ubio_molfm_amd import optim
    p = torch.ones(5000, device=cuda).requires_grad_(True)
    whole = p.detach()
    host = torch.ones(6).requires_grad_(True)
    opt = optim.AdamW([p, host], lr=1e-2, weight_decay=0.0)
    p.grad = torch.ones(5000, device=cuda)
    opt.step()
    p.grad = None
    p.data = whole[:100]
    p.grad = torch.ones(100, device=cuda)
    del opt.state[p]
    after = whole.clone()
    opt.step()
    assert (whole[:100] < after[:100]).all() and torch.equal(whole[100:], after[100:])
    host.data = host.data.to(cuda)
    host.grad = torch.ones(6, device=cuda)
    opt.step()
    assert (host.detach() < 1).all()
    p.data = whole[:200]                       # the gradient is still that of 100 elements
    del opt.state[p]
    with pytest.raises(ValueError, match="other sizes"):
        opt.step()

    q = torch.ones(8, 8, device=cuda).requires_grad_(True)
    opt = optim.AdamW([q])
    q.grad = torch.ones(8, 8, device=cuda)
    opt.step()
    q.data = q.data.t()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()


@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_gradients_left_behind_on_the_host(pkg, cuda, max_norm):
    """A parameter brought to the GPU by .data keeps its host gradient, and a gradient can be moved by its own .data:
    the step refuses both and goes on once they are together."""
    from ubio_molfm_amd import optim
    p, q = torch.ones(6).requires_grad_(True), torch.ones(5, device=cuda).requires_grad_(True)
    p.grad, q.grad = torch.ones(6), torch.ones(5, device=cuda)
    p.data = p.data.to(cuda)
    opt = optim.AdamW([q, p], lr=1e-2, max_norm=max_norm)
    with pytest.raises(RuntimeError, match="gradients on"):
        opt.step()
    p.grad = p.grad.to(cuda)
    opt.step()
    after = p.detach().clone()
    assert (after < 1).all() and int(opt.state[p]["step"]) == 1
    p.grad.data = p.grad.data.cpu()
    with pytest.raises(RuntimeError, match="gradients on"):
        opt.step()
    assert torch.equal(p.detach(), after) and int(opt.state[q]["step"]) == 1


def test_a_captured_rate_after_load_state_dict(pkg, cuda):
    """A step captured with its learning rate on the device takes the loaded rate, and what is written to it later."""
    from ubio_molfm_amd import optim
    ps, qs = (_params(SHAPES, torch.float32, cuda, 54) for _ in range(2))
    a, b = (optim.AdamW(x, lr=torch.tensor(1e-3, device=cuda)) for x in (ps, qs))
    a.step(), b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    saved = copy.deepcopy(b.state_dict())
    for rate in (torch.tensor(4e-3), 2e-3):
        saved["param_groups"][0]["lr"] = rate
        a.load_state_dict(saved)
        b.load_state_dict(saved)
        for p, q in zip(ps, qs):
            p.data.copy_(q.data)
        junk = [torch.full((), 1e3, device=cuda) for _ in range(64)]      # takes memory that was let go
        for k in range(3):
            graph.replay()
            torch.cuda.synchronize()
            b.step()
            assert all(torch.equal(p, q) for p, q in zip(ps, qs)), (rate, k)
            for o in (a, b):
                o.param_groups[0]["lr"].mul_(0.5)
        del junk


@pytest.mark.parametrize("kind", ["group", "type", "list"])
def test_the_norm_of_a_step_behind_empty_tensors(pkg, cuda, kind):
    """A group, a type or a whole launch of parameters without elements comes first: the norm is this step's all the
    same, and steps left out are counted."""
    from ubio_molfm_amd import optim
    empty = torch.zeros(0, device=cuda, dtype=torch.float16 if kind == "type" else torch.float32, requires_grad=True)
    empties = [empty] + [torch.zeros(0, device=cuda, requires_grad=True) for _ in range(400 if kind == "list" else 0)]
    ps = _params([(30,), (5000,)], torch.float32, cuda, 55)
    for p in empties:
        p.grad = torch.zeros_like(p)
    groups = [dict(params=empties), dict(params=ps)] if kind == "group" else [dict(params=empties + ps)]
    opt = optim.AdamW(groups, max_norm=0.5, skip_nonfinite=True)
    for scale in (1.0, 3.0):
        for p in ps:
            p.grad.mul_(scale)
        opt.step()
        norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps))
        assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    ps[1].grad[7] = float("nan")
    opt.step()
    assert int(opt.skipped) == 1 and opt.grad_norm.isnan() and int(opt.state[ps[0]]["step"]) == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_gaps_stay_zero_under_a_nan_factor(pkg, cuda, bits):
    """One NaN gradient makes the clipping factor NaN, and so all moments; the gaps between tensors are none, and a good
    checkpoint loaded in place brings everything back."""
    from ubio_molfm_amd import optim
    ps = _params(SHAPES, torch.float32, cuda, 56)
    opt = optim.AdamW(ps, state_bits=bits, max_norm=0.5)
    opt.step()
    good = copy.deepcopy(opt.state_dict())
    want = [x.clone() for x in opt.moments(torch.float32)]
    inside = torch.zeros(want[0].numel(), dtype=torch.bool, device=cuda)
    off = 0
    for p in ps:
        inside[off:off + p.numel()] = True
        off += -(-p.numel() // 64) * 64
    ps[5].grad[3, 4] = float("nan")
    opt.step()
    for x in opt.moments(torch.float32):
        assert x[inside].isnan().all() and not x[~inside].any()
    opt.load_state_dict(good)
    assert all(torch.equal(x, y) for x, y in zip(opt.moments(torch.float32), want))


def test_entries_taken_out_behind_others(pkg, cuda):
    """Entries left over from a group that was popped, and empty ones that reading the state makes, do not hide one that
    was taken out; a captured step goes on in the same buffers."""
    from ubio_molfm_amd import optim
    ps = _params([(100,), (5000,), (70,)], torch.float32, cuda, 57)
    opt = optim.AdamW([dict(params=ps[:2]), dict(params=ps[2:])], lr=1e-3)
    opt.step(), opt.step()
    opt.param_groups.pop()
    opt.step()
    steps = lambda: [int(opt.state[p]["step"]) for p in ps[:2]]
    assert steps() == [3, 3] and ps[2] in opt.state
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    m = opt.state[ps[0]]["exp_avg"]
    del opt.state[ps[0]]
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step()
    assert steps() == [1, 4] and opt.state[ps[0]]["exp_avg"] is m
    assert torch.equal(m, _first_moments(ps[0].grad, 1))
    del opt.state[ps[0]]
    assert opt.state[ps[0]] == {}                                    # reading makes an entry
    opt.step()
    assert steps() == [1, 5]
    graph.replay()
    torch.cuda.synchronize()
    assert steps() == [2, 6] and torch.allclose(m, _first_moments(ps[0].grad, 2))
    del opt.state[ps[1]]
    assert not opt.moments()[1][128:].any() and opt.moments()[1][:100].any() and int(opt.state[ps[1]]["step"]) == 0


def _first_moments(g, steps):
    """First moments after steps with the same gradient, each rounding as the kernel's."""
    b1, one_b1 = (torch.tensor(x, dtype=torch.float32) for x in (0.9, 1 - 0.9))
    m = torch.zeros_like(g)
    for _ in range(steps):
        m = (one_b1.double().item() * g.double() + (b1.to(g.device) * m).double()).float()
    return m


def test_entries_put_in_by_hand(pkg, cuda):
    from ubio_molfm_amd import optim
    ps = _params([(100,), (5000,)], torch.float32, cuda, 58)
    opt = optim.AdamW(ps, lr=1e-3)
    opt.step()
    saved = {k: t.clone() for k, t in opt.state[ps[1]].items()}
    params = ps[1].detach().clone()
    opt.step()
    after = ps[1].detach().clone()
    ps[1].data.copy_(params)
    opt.state[ps[1]] = saved
    opt.step()
    assert torch.equal(ps[1], after) and int(opt.state[ps[1]]["step"]) == 2 and int(opt.state[ps[0]]["step"]) == 3
    for broken in ({"step": 1}, {**saved, "exp_avg": saved["exp_avg"][:5]}):
        opt.state[ps[1]] = broken
        with pytest.raises(ValueError, match="exp_avg"):
            opt.step()
    assert torch.equal(ps[1], after)


def test_tensors_put_into_entries(pkg, cuda, tmp_path):
    """A moment and a step count put into an entry are the next step's; a saved state is made of plain dicts."""
    from ubio_molfm_amd import optim
    (p,), (q,) = (_params([(9001,)], torch.float32, cuda, 59) for _ in range(2))
    a, b = optim.AdamW([p], lr=1e-3), optim.AdamW([q], lr=1e-3)
    for _ in range(3):
        a.step()
    b.step()
    for k in ("exp_avg", "exp_avg_sq", "step"):
        b.state[q][k] = a.state[p][k].clone()
    q.data.copy_(p.data)
    a.step(), b.step()
    assert torch.equal(p, q) and int(b.state[q]["step"]) == 4 and torch.equal(a.moments()[1], b.moments()[1])
    torch.save(a.state_dict(), tmp_path / "a.pt")
    sd = torch.load(tmp_path / "a.pt", weights_only=True)
    assert type(a.state_dict()["state"][0]) is dict
    b.load_state_dict(sd)
    a.step(), b.step()
    assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16, torch.int64])
def test_a_rate_on_the_gpu_in_another_type(pkg, cuda, dtype):
    """It is taken to fp32 there: a step reads nothing back, and a captured one follows the tensor."""
    from ubio_molfm_amd import optim
    (p,), (q,) = (_params([(5000,)], torch.float32, cuda, 60) for _ in range(2))
    lr = torch.tensor(1 if dtype == torch.int64 else 0.0625 if dtype == torch.bfloat16 else 1e-3, dtype=dtype, device=cuda)
    a, b = optim.AdamW([p], lr=lr), optim.AdamW([q], lr=lr.item())
    a.step(), b.step()
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        a.step()
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    b.step()
    assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for rate in (2.0, 4.0, 1.0):
        lr.fill_(rate)
        b.param_groups[0]["lr"] = rate
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        assert torch.equal(p, q)


def test_step_counts_are_loaded_together(pkg, cuda, monkeypatch):
    """Step counts of a checkpoint in host memory (tensors, numbers, torch's floating ones) go to the GPU in one copy,
    into every chunk of their tensors."""
    from ubio_molfm_amd import optim
    ps = _params([(k % 5 * 3000 + k % 2,) for k in range(200)], torch.float32, cuda, 61)
    opt = optim.AdamW(ps)
    opt.step()
    sd = copy.deepcopy(opt.state_dict())
    for k, e in sd["state"].items():
        e["step"] = (torch.tensor(float(k)), k, torch.tensor([k], dtype=torch.int64))[k % 3]
    copies = []
    real = torch.Tensor.to
    monkeypatch.setattr(torch.Tensor, "to", lambda t, *a, **k: (copies.append(t.is_cuda), real(t, *a, **k))[1])
    opt.load_state_dict(sd)
    monkeypatch.undo()
    assert copies.count(False) <= 3, len(copies)
    for k, p in enumerate(ps):
        st = opt.state[p]
        assert int(st["step"]) == k and (st.steps == k).all() and st.steps.numel() == -(-p.numel() // 4096)
    sd["state"][3]["step"] = torch.tensor(50, device=cuda)               # some of them on the GPU
    opt.load_state_dict(sd)
    assert int(opt.state[ps[3]]["step"]) == 50 and int(opt.state[ps[4]]["step"]) == 4


def test_clipping_of_gradients_that_share_memory(pkg, cuda):
    """Their elements would be scaled by two workgroups at once, or twice: refused, and left as they were."""
    from ubio_molfm_amd import optim
    flat = torch.ones(10000, device=cuda)

    def params(*grads):
        out = []
        for g in grads:
            p = torch.zeros(g.shape, dtype=g.dtype, device=cuda, requires_grad=True)
            p.grad = g
            out.append(p)
        return out

    turned = params(flat.view(100, 100).t())[0]
    row = params(flat[:50].expand(30, 50))[0]
    for ps, match in ((params(flat[:6000], flat[5000:]), "share"), (params(flat, flat[3:4]), "share"),
                      (params(flat[:100], flat[40:100].view(torch.float16)), "share"), ([turned, turned], "twice"),
                      ([row], "share"), (params(flat[:50], flat[60:90].expand(3, 30)), "share")):
        with pytest.raises(ValueError, match=match):
            optim.clip_grad_norm_(ps, 0.1)
        assert (flat == 1).all()
    one = params(torch.ones(1, 30, 50, device=cuda).as_strided((1, 30, 50), (0, 1, 30)))
    optim.clip_grad_norm_(params(flat[:100], flat[100:100], flat[100:]) + one, 1.0)
    assert torch.allclose(flat, torch.full_like(flat, 1 / math.sqrt(11500))) and (one[0].grad < 0.01).all()


def test_clipping_gradients_with_a_history(pkg, cuda):
    """Gradients of a backward pass with create_graph: scaled as without, outside of their history."""
    from ubio_molfm_amd import optim
    x = torch.randn(40, 30, device=cuda)
    ps = [torch.nn.Parameter(torch.randn(30, 40, device=cuda)) for _ in range(2)]
    ((ps[0] @ x).square().sum() + (ps[1].t() @ x.t()).pow(3).sum()).backward(create_graph=True)
    ps[1].grad = ps[1].grad.t().contiguous().t()
    want = [p.grad.detach().double().clone() for p in ps]
    norm = math.sqrt(sum(float(g.square().sum()) for g in want))
    own = [ps[0].grad, ps[1].grad._base]                                 # the second is a view
    fns = [g.grad_fn for g in own]
    assert all(fns) and not ps[1].grad.is_contiguous()
    assert abs(float(optim.clip_grad_norm_(ps, 0.5)) - norm) <= 2 * U * norm
    assert all(g.grad_fn is fn for g, fn in zip(own, fns))
    for p, g in zip(ps, want):
        c = 0.5 / (norm + 1e-6)
        assert (p.grad.double() - c * g).abs().le(4 * U * (c * g).abs()).all()


@pytest.mark.parametrize("before,after", [(torch.float32, torch.bfloat16), (torch.float16, torch.bfloat16)])
def test_parameters_that_take_another_type_in_place(pkg, cuda, before, after):
    """.data of another type at the same address with as many elements: updated as what it is now."""
    from ubio_molfm_amd import optim
    p, q = (torch.ones(5000, dtype=t, device=cuda, requires_grad=True) for t in (before, after))
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt, ref = optim.AdamW([p], lr=1e-2), optim.AdamW([q], lr=1e-2)
    opt.step()
    p.grad = None
    p.data = p.data.view(after)[:5000].fill_(1.0)
    p.grad = torch.ones(5000, dtype=after, device=cuda)
    opt.state[p] = {"step": 0, "exp_avg": torch.zeros(5000), "exp_avg_sq": torch.zeros(5000)}
    opt.step(), ref.step()
    assert torch.equal(p, q) and (p < 1).all()


@pytest.mark.parametrize("how", ["load", "state"])
@pytest.mark.parametrize("bits", [32, 8])
def test_states_that_change_places(pkg, cuda, bits, how):
    """An optimizer's own states loaded back in another order, or exchanged in place: none is read after it is written."""
    from ubio_molfm_amd import optim
    ps = _params([(5000,), (5000,), (5000,)], torch.float32, cuda, 62)
    opt = optim.AdamW(ps, state_bits=bits)
    opt.step()
    opt.state[ps[1]]["step"] = 5
    before = [{k: t.clone() for k, t in opt.state[p].items()} for p in ps]
    if how == "load":
        sd = opt.state_dict()
        sd["state"] = {0: sd["state"][1], 1: sd["state"][2], 2: sd["state"][0]}
        opt.load_state_dict(sd)
    else:
        opt.state[ps[0]], opt.state[ps[1]], opt.state[ps[2]] = (opt.state[ps[k]] for k in (1, 2, 0))
        opt.moments()
    for p, k in zip(ps, (1, 2, 0)):
        assert all(torch.equal(t, before[k][name]) for name, t in opt.state[p].items())
    assert [int(opt.state[p]["step"]) for p in ps] == [5, 1, 1]
