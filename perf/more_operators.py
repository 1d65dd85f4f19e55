"""RMS norm with the residual's addition, products in 8 bits with block scales, and products grouped by expert, as
measurable cases.

Families (``kind``):

* ``norm_train``    h = x + residual and the RMS norm of h, forward and backward: output, h, gradients of the rows (those
                    of x and of the residual are one tensor) and of the weight;
* ``norm_fp8``      the same forward pass with its output in 8 bits: the values it stands for, and h;
* ``fp8``           the product of 8-bit rows and an 8-bit weight, out in 16 bits;
* ``fp8_train``     a linear layer whose three products run in 8 bits: output, gradients of rows and weight;
* ``experts``       rows sorted by expert times their expert's weight, forward only;
* ``experts_train`` the same with the gradients of rows and weights;
* ``experts_fp8``   the forward pass on 8-bit rows and weights.

8 bits: e4m3 codes, and a scale byte s for each block that stands for 2^(s - 127), the smallest power of two with which
the block's largest finite value is at most 448 (2^-126 at least).  Blocks are 128 consecutive values of a row, or
tiles of 128 x 128 of a weight.  Codes are rounded to the nearest, ties to even; what is not finite becomes NaN.

Experts: rows offsets[e] to offsets[e + 1] belong to expert e; rows behind the last one belong to none and give zeros."""
import importlib
import math
import random

import torch

own = False

_PKG = "ubio-molfm_amd"
EPS = 1e-5
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def _mod(name):
    return importlib.import_module(f"{_PKG}.{name}")


# --------------------------------------------------------------------------- the cases

def listed():
    return [
        # node features of a 10,000-atom system in training, fp32
        dict(name="norm_train_nodes", kind="norm_train", rows=10000, width=256, dtype="fp32"),
        # bf16 hidden states of a long batch in training
        dict(name="norm_train_bf16", kind="norm_train", rows=32768, width=2048, dtype="bf16"),
        # one token between two layers while serving
        dict(name="norm_fp8_token", kind="norm_fp8", rows=1, width=4096, dtype="bf16"),
        # the rows of a long prompt, quantised for the next product
        dict(name="norm_fp8_long", kind="norm_fp8", rows=16384, width=4096, dtype="bf16"),
        # one token through a weight: the weight's bytes are all there is
        dict(name="fp8_token", kind="fp8", m=1, n=4096, k=4096, dtype="bf16"),
        # an odd number of nodes through a feed-forward block's first layer
        dict(name="fp8_nodes", kind="fp8", m=10007, n=768, k=256, dtype="bf16"),
        # a long prompt through a large layer
        dict(name="fp8_long", kind="fp8", m=8192, n=8192, k=4096, dtype="bf16"),
        # a training step's layer in 8 bits
        dict(name="fp8_train", kind="fp8_train", m=16384, n=4096, k=2048, dtype="bf16"),
        # a few tokens, each through an expert of its own
        dict(name="experts_tokens", kind="experts", rows=13, spare=0, experts=64, n=1024, k=2048, dtype="bf16"),
        # one weight for each element, over the nodes of a 10,000-atom system, fp32 training
        dict(name="experts_elements", kind="experts_train", rows=10000, spare=0, experts=6, n=256, k=256, dtype="fp32"),
        # a training batch routed to 32 experts, rows kept free for a fuller one
        dict(name="experts_train_bf16", kind="experts_train", rows=16384, spare=509, experts=32, n=1408, k=2048,
             dtype="bf16"),
        # a prompt routed to 64 experts, in 8 bits
        dict(name="experts_fp8", kind="experts_fp8", rows=32768, spare=0, experts=64, n=2048, k=1408, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width over the range: as it comes, or a multiple of 16 or 128."""
    w = _log(rng, lo, hi)
    step = rng.choice([1, 16, 128, 128])
    return max(min(step, hi), w // step * step)


def draw(rng):
    kind = rng.choice(["norm_train", "norm_train", "norm_fp8", "norm_fp8", "fp8", "fp8", "fp8_train", "experts",
                       "experts_train", "experts_fp8"])
    half = rng.choice(["bf16", "bf16", "fp16"])
    dtype = rng.choice([half, half, "fp32"])
    if kind.startswith("norm"):
        width = _width(rng, 32, 8192)
        return dict(kind=kind, rows=_log(rng, 1, max(16, min(200_000, 60_000_000 // width))), width=width, dtype=dtype)
    n, k = _width(rng, 64, 8192), _width(rng, 64, 8192)
    if kind.startswith("fp8"):
        most = 2.5e11 if kind == "fp8" else 1.2e11
        return dict(kind=kind, m=_log(rng, 1, max(16, min(32768, int(most / (n * k))))), n=n, k=k, dtype=half)
    n, k, experts = min(n, 4096), min(k, 4096), _log(rng, 1, 128)
    experts = min(experts, max(1, 200_000_000 // (n * k)))
    rows = _log(rng, 1, max(16, min(32768, int((9e10 if kind != "experts_train" else 4.5e10) / (n * k)))))
    if dtype == "fp32":
        rows = max(1, rows // 4)
    return dict(kind=kind, rows=rows, spare=rng.choice([0, 0, rng.randint(1, 300)]), experts=experts, n=n, k=k,
                dtype=half if kind == "experts_fp8" else dtype)


def _sizes(case):
    """Rows of each expert: uneven as a router's or a molecule's elements are, some experts without any."""
    rng = random.Random(case["rows"] * 1000003 + case["experts"] * 4099 + case["n"])
    e = case["experts"]
    share = [math.exp(0.6 * rng.gauss(0, 1)) * (e < 8 or rng.random() > 0.1) for _ in range(e)]
    if case["rows"] <= e:
        sizes = [0] * e
        for _ in range(case["rows"]):
            sizes[rng.randrange(e)] += 1
        return sizes
    total = sum(share) or 1.0
    sizes = [int(case["rows"] * s / total) for s in share]
    sizes[max(range(e), key=lambda i: share[i])] += case["rows"] - sum(sizes)
    return sizes


def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind.startswith("norm"):
        n = case["rows"] * case["width"]
        if kind == "norm_fp8":      # x, residual in; h, the codes and the values they stand for out
            return {"bytes": (3 * size + 1 + 1 / 128 + 2) * n, "flops": 12 * n}
        # forward: x, residual in, h, y out; backward: gradients of y and h in, the rows' gradient out
        return {"bytes": 7 * size * n + 2 * size * case["width"], "flops": 16 * n}
    if kind == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + size * m * n, "flops": 2.0 * m * n * k}
    if kind == "fp8_train":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * size * (m * k + n * k + m * n), "flops": 6.0 * m * n * k}
    live = sum(s > 0 for s in _sizes(case))
    rows, every, n, k = case["rows"], case["rows"] + case["spare"], case["n"], case["k"]
    one = 1 if kind == "experts_fp8" else size
    moved = one * (rows * k + live * n * k) + size * every * n
    if kind == "experts_train":
        moved += size * (rows * n + every * k + case["experts"] * n * k)
    return {"bytes": moved, "flops": (6.0 if kind == "experts_train" else 2.0) * rows * n * k}


# --------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, kind = DTYPES[case["dtype"]], case["kind"]

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    st = dict(kind=kind, dtype=dt)
    if kind.startswith("norm"):
        n, w = case["rows"], case["width"]
        # a branch's output on hidden states whose rows have sizes of their own
        st["x"], st["res"] = rand(n, w).to(dt), rand(n, w).mul_(torch.exp(0.5 * rand(n, 1))).to(dt)
        st["w"] = (1 + 0.3 * rand(w)).to(dt)
        if kind == "norm_train":
            st["gy"], st["gh"] = rand(n, w).to(dt), rand(n, w).to(dt)
            for name in ("x", "res", "w"):
                st[name].requires_grad_(True)
        return st
    if kind.startswith("fp8"):
        m, n, k = case["m"], case["n"], case["k"]
        # rows as a norm leaves them, with a few wide channels
        x, w = rand(m, k) * torch.exp(0.7 * rand(k)), rand(n, k) / math.sqrt(k)
        if kind == "fp8":
            st["a"], st["sa"] = _quantize(x, tiles=False)
            st["w"], st["sw"] = _quantize(w, tiles=True)
        else:
            st["x"], st["w"] = x.to(dt).requires_grad_(True), w.to(dt).requires_grad_(True)
            st["gy"] = (1e-3 * rand(m, n) * torch.exp(0.5 * rand(m, 1))).to(dt)
        return st
    e, n, k, every = case["experts"], case["n"], case["k"], case["rows"] + case["spare"]
    sizes = _sizes(case)
    sizes = sizes[seed % e:] + sizes[:seed % e]
    st["most"] = max(sizes)
    st["offsets"] = torch.tensor([0] + sizes, device="cuda").cumsum(0).to(torch.int32)
    x, w = rand(every, k), rand(e, n, k).div_(math.sqrt(k))
    if kind == "experts_fp8":
        st["x"], st["sx"] = _quantize(x, tiles=False)
        st["w"], st["sw"] = _quantize(w, tiles=True)
        return st
    st["x"], st["w"] = x.to(dt), w.to(dt)
    if kind == "experts_train":
        st["x"].requires_grad_(True), st["w"].requires_grad_(True)
        st["gy"] = rand(every, n).to(dt)
    return st


# --------------------------------------------------------------------------- one pass

def run(st):
    kind = st["kind"]
    if kind == "norm_train":
        return _norm_train_own(st) if own else _norm_train(st)
    if kind == "norm_fp8":
        return _norm_fp8_own(st) if own else _norm_fp8(st)
    if kind == "fp8":
        return _fp8_own(st) if own else _fp8(st)
    if kind == "fp8_train":
        return _fp8_train_own(st) if own else _fp8_train(st)
    if kind == "experts_fp8":
        return _experts_fp8_own(st) if own else _experts_fp8(st)
    if kind == "experts":
        return _experts_own(st) if own else _experts(st)
    return _experts_train_own(st) if own else _experts_train(st)


def _norm_train_own(st):
    y, h = _mod("norms").rms_norm(st["x"], st["w"], EPS, residual=st["res"])
    gx, gres, gw = torch.autograd.grad((y, h), (st["x"], st["res"], st["w"]), (st["gy"], st["gh"]))
    return y, h, gx, gw


def _norm_fp8_own(st):
    codes, scales, h = _mod("norms").rms_norm_fp8(st["x"], st["w"], EPS, residual=st["res"])
    return _mod("fp8").dequantize(codes, scales, torch.bfloat16), h


def _fp8_own(st):
    return _mod("fp8").gemm(st["a"], st["sa"], st["w"], st["sw"], dtype=st["dtype"])


def _fp8_train_own(st):
    y = _mod("fp8").linear(st["x"], st["w"])
    return (y, *torch.autograd.grad(y, (st["x"], st["w"]), st["gy"]))


def _experts_own(st):
    return _mod("experts").expert_linear(st["x"], st["w"], st["offsets"])


def _experts_train_own(st):
    y = _mod("experts").expert_linear(st["x"], st["w"], st["offsets"])
    return (y, *torch.autograd.grad(y, (st["x"], st["w"]), st["gy"]))


def _experts_fp8_own(st):
    return _mod("experts").expert_gemm_fp8(st["x"], st["sx"], st["w"], st["sw"], st["offsets"], dtype=st["dtype"])


def _normed(st):
    """h in the rows' type, and in 32 bits h scaled to a mean square of one, and the scale."""
    h = (st["x"].detach().float() + st["res"].detach().float()).to(st["dtype"])
    f = h.float()
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    return h, f * r, r


def _norm_train(st):
    h, hh, r = _normed(st)
    w, gy, dt = st["w"].detach().float(), st["gy"].float(), st["dtype"]
    u = gy * w
    gx = r * (u - hh * (u * hh).mean(-1, keepdim=True)) + st["gh"].float()
    return (hh * w).to(dt), h, gx.to(dt), (gy * hh).sum(0).to(dt)


def _norm_fp8(st):
    h, hh, _ = _normed(st)
    codes, scales = _quantize(hh * st["w"].float(), tiles=False)
    return _values(codes, scales, tiles=False).to(torch.bfloat16), h


def _fp8(st):
    return torch.mm(_values(st["a"], st["sa"], False), _values(st["w"], st["sw"], True).t()).to(st["dtype"])


def _fp8_train(st):
    def held(t, tiles=False):
        return _values(*_quantize(t, tiles), tiles)

    x, w, gy, dt = st["x"].detach().float(), held(st["w"].detach().float(), True), st["gy"].float(), st["dtype"]
    return (torch.mm(held(x), w.t()).to(dt), torch.mm(held(gy), w).to(dt),
            torch.mm(held(gy.t().contiguous()), held(x.t().contiguous()).t()).to(dt))


def _places(st, rows):
    """For each row whether it has an expert, and its place in a grid of experts times the largest one's rows."""
    at = torch.arange(rows, device="cuda")
    offs = st["offsets"].long()
    e = torch.bucketize(at, offs[1:], right=True)
    inside = e < offs.numel() - 1
    e = torch.where(inside, e, 0)
    return inside, e, torch.where(inside, e * st["most"] + at - offs[e], offs.numel() * st["most"])


def _grid(x, place, experts, most):
    """The rows of x at their places, zeros elsewhere."""
    grid = x.new_zeros((experts + 1) * most + 1, x.shape[1])
    grid[place] = x
    return grid[:experts * most].view(experts, most, x.shape[1])


def _rows_of(grid, place, inside):
    flat = grid.reshape(-1, grid.shape[-1])
    return flat[torch.where(inside, place, 0)] * inside[:, None]


def _expert_products(st, x, w):
    inside, e, place = _places(st, x.shape[0])
    if x.shape[0] <= w.shape[0]:       # fewer rows than experts: each row with its weight
        return (torch.bmm(w[e], x[:, :, None])[:, :, 0] * inside[:, None]).to(st["dtype"])
    y = torch.bmm(_grid(x, place, w.shape[0], st["most"]), w.transpose(1, 2))
    return _rows_of(y, place, inside).to(st["dtype"])


def _experts(st):
    if st["x"].shape[0] <= st["w"].shape[0]:
        inside, e, _ = _places(st, st["x"].shape[0])
        y = torch.bmm(st["w"][e].float(), st["x"].float()[:, :, None])[:, :, 0]
        return (y * inside[:, None]).to(st["dtype"])
    return _expert_products(st, st["x"].float(), st["w"].float())


def _experts_train(st):
    x, w, gy, dt = st["x"].detach().float(), st["w"].detach().float(), st["gy"].float(), st["dtype"]
    inside, _, place = _places(st, x.shape[0])
    xg, gg = (_grid(t, place, w.shape[0], st["most"]) for t in (x, gy))
    y, gx = torch.bmm(xg, w.transpose(1, 2)), torch.bmm(gg, w)
    gw = torch.bmm(gg.transpose(1, 2), xg)
    return _rows_of(y, place, inside).to(dt), _rows_of(gx, place, inside).to(dt), gw.to(dt)


def _experts_fp8(st):
    return _expert_products(st, _values(st["x"], st["sx"], False), _values(st["w"], st["sw"], True))


# --------------------------------------------------------------------------- 8 bits

def _blocked(x, tiles):
    """x [..., r, c] filled up with zeros to whole blocks, as [..., blocks of rows, their rows, blocks of columns, 128]."""
    r, c = x.shape[-2:]
    rb = 128 if tiles else 1
    x = torch.nn.functional.pad(x, (0, -c % 128, 0, -r % rb))
    return x.reshape(*x.shape[:-2], -(-r // rb), rb, -(-c // 128), 128)


def _quantize(x, tiles):
    """e4m3 codes of x [..., r, c] in 32 bits and the scale bytes of its blocks."""
    b = _blocked(x, tiles)
    top = torch.where(b.isfinite(), b.abs(), 0).amax((-3, -1)).contiguous().view(torch.int32)
    # the exponent of the smallest power of two that brings the mantissa 1.75 to 448 at most
    s = torch.clamp((top + 0x1FFFFF >> 23) - 8, min=1)
    t = x * torch.exp2(127.0 - _spread(s, x.shape, tiles))
    return torch.where(x.isfinite(), t, math.nan).to(torch.float8_e4m3fn), s.to(torch.uint8)


def _spread(s, shape, tiles):
    s = s.float().repeat_interleave(128, -1)[..., :shape[-1]]
    return s.repeat_interleave(128, -2)[..., :shape[-2], :] if tiles else s


def _values(codes, s, tiles):
    """What codes and scales stand for, in 32 bits."""
    return codes.float() * torch.exp2(_spread(s, codes.shape, tiles) - 127.0)


# --------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("norm"):
        # h is a rounded sum that the norm starts from
        h = (st["x"].detach().double() + st["res"].detach().double()).to(st["dtype"])
        z, w = h.double().requires_grad_(True), st["w"].detach().double().requires_grad_(True)
        y = z / (z.square().sum(-1, keepdim=True) / case["width"] + EPS).sqrt() * w
        if kind == "norm_fp8":
            return _held(y.detach(), 1), h.double()
        gx, gw = torch.autograd.grad(y, (z, w), st["gy"].double())
        return y.detach(), h.double(), gx + st["gh"].double(), gw
    if kind == "fp8":
        return _stood(st["a"], st["sa"], 1) @ _stood(st["w"], st["sw"], 128).T
    if kind == "fp8_train":
        x, w, gy = st["x"].detach().double(), _held(st["w"].detach().double(), 128), st["gy"].double()
        return _held(x, 1) @ w.T, _held(gy, 1) @ w, _held(gy.T, 1) @ _held(x.T, 1).T
    if kind == "experts_fp8":
        x, w = _stood(st["x"], st["sx"], 1), torch.stack([_stood(c, s, 128) for c, s in zip(st["w"], st["sw"])])
    else:
        x, w = st["x"].detach().double(), st["w"].detach().double()
    ends = st["offsets"].tolist()
    y = x.new_zeros(x.shape[0], w.shape[1])
    gx, gw = torch.zeros_like(x), torch.zeros_like(w)
    gy = st["gy"].double() if kind == "experts_train" else None
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        y[lo:hi] = x[lo:hi] @ w[e].T
        if gy is not None:
            gx[lo:hi] = gy[lo:hi] @ w[e]
            gw[e] = gy[lo:hi].T @ x[lo:hi]
    return y if gy is None else (y, gx, gw)


def _stood(codes, s, rows):
    """What codes and scales stand for, in 64 bits, from the codes' bits."""
    c = codes.view(torch.uint8).long()
    e, f = c // 8 % 16, (c % 8).double()
    v = torch.where(e > 0, (1 + f / 8) * torch.exp2(e.double() - 7), f * 2.0 ** -9)
    v = torch.where(c % 128 == 127, math.nan, torch.where(c > 127, -v, v))
    i = torch.arange(c.shape[0], device=c.device) // rows
    j = torch.arange(c.shape[1], device=c.device) // 128
    return v * torch.exp2(s.double()[i][:, j] - 127)


def _held(x, rows):
    """x [r, c] in 64 bits, rounded as its blocks of `rows` x 128 are held."""
    r, c = x.shape
    full = x.new_zeros(-(-r // rows) * rows, -(-c // 128) * 128)
    full[:r, :c] = x
    b = full.view(full.shape[0] // rows, rows, -1, 128)
    most = b.abs().amax((1, 3), keepdim=True)
    unit = torch.exp2(torch.clamp(torch.ceil(torch.log2(most / 448)), min=-126.0))
    unit = torch.where(most > 448 * unit, 2 * unit, torch.where(most <= 224 * unit, unit / 2, unit))
    unit = torch.clamp(unit, min=2.0 ** -126)
    t = b / unit
    step = torch.exp2(torch.clamp(torch.frexp(t)[1] - 1, min=-6).double() - 3)
    return (torch.round(t / step) * step * unit).view_as(full)[:r, :c]
