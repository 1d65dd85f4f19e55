"""The parameter update of force training and the layer norm, as measurable cases.

Families (``kind``):

* ``norm``        layer norm of rows, forward only (no gradients: evaluation);
* ``norm_train``  its forward and backward pass: output, gradients of the rows, the weight and the bias;
* ``norm_force``  the second order of force training: output, the rows' first gradient, and the gradients of
                  a function of that gradient in the rows, the upstream gradient and the weight;
* ``adamw``       one AdamW step over the parameters of a model, states in 32 or 8 bits, with or without
                  clipping by the gradients' global norm;
* ``clip``        scaling of all gradients by their global norm, in place.

8-bit states: runs of 32 consecutive elements of a parameter share a scale byte s; 2^(s - 127) is the top binade of
the run's codes.  First moments: sign, 4 exponent and 3 mantissa bits (with subnormals; code 0x80 is NaN).  Second
moments: 5 exponent and 3 mantissa bits (code 255 is NaN; a value above zero keeps a code above zero).  Values
are rounded stochastically, by bits that are a hash of the seed, the step and the element's position.

The parameters, their moments and (in these cases) their gradients lie in flat buffers, each tensor from a multiple
of 64 elements on."""
import importlib
import math

import torch

own = False

_PKG = "ubio-molfm_amd"
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM = 1e-4, 0.9, 0.999, 1e-8, 0.01, 10.0
LN_EPS = 1e-5
STEP = 1000                      # steps taken before the measured one
SEED = 20251
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def _mod(name):
    return importlib.import_module(f"{_PKG}.{name}")


# --------------------------------------------------------------------------- the cases

def listed():
    return [
        # node features of one small molecule in an evaluation: a launch is all there is
        dict(name="norm_rows24", kind="norm", rows=24, width=256, dtype="fp32", weights="fp32"),
        # wide rows in bf16 with a width that no vector divides
        dict(name="norm_bf16_5001", kind="norm", rows=6007, width=5001, dtype="bf16", weights="bf16"),
        # the hidden rows of a radial profile over the edges of a 1,500-atom system, training
        dict(name="norm_train_edges", kind="norm_train", rows=127113, width=128, dtype="fp32", weights="fp32"),
        # an odd width on a ragged batch of molecules
        dict(name="norm_train_odd", kind="norm_train", rows=3318, width=129, dtype="fp32", weights="fp32"),
        # bf16 rows with fp32 weights, the wide generic case
        dict(name="norm_train_bf16", kind="norm_train", rows=32768, width=2048, dtype="bf16", weights="fp32"),
        # force training: the radial profiles' rows of a 10,000-atom system, differentiated twice
        dict(name="norm_force_edges", kind="norm_force", rows=853991, width=128, dtype="fp32", weights="fp32"),
        # fine-tuning the energy head alone: six small tensors
        dict(name="adamw_head", kind="adamw", layers=0, channels=256, dtype="fp32", bits=32, clip=False),
        # the default model's 240 trained tensors, clipped
        dict(name="adamw_model", kind="adamw", layers=4, channels=256, dtype="fp32", bits=32, clip=True),
        # a large model kept in bf16
        dict(name="adamw_large_bf16", kind="adamw", layers=12, channels=480, dtype="bf16", bits=32, clip=False),
        # the default model with states in 8 bits, clipped
        dict(name="adamw8_model", kind="adamw", layers=4, channels=256, dtype="fp32", bits=8, clip=True),
        # a large model with states in 8 bits
        dict(name="adamw8_large", kind="adamw", layers=12, channels=480, dtype="fp32", bits=8, clip=False),
        # clipping for another optimizer: the default model's gradients
        dict(name="clip_model", kind="clip", layers=4, channels=256, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "norm_train", "norm_force", "adamw", "adamw", "adamw", "clip"])
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    if kind.startswith("norm"):
        width = _log(rng, 8, 8192)
        width = width if rng.random() < 0.4 else max(8, width // 64 * 64)
        dtype = "fp32" if kind == "norm_force" else dtype
        rows = _log(rng, 1, max(16, min(1_000_000, 100_000_000 // width)))
        return dict(kind=kind, rows=rows, width=width, dtype=dtype, weights=rng.choice(["fp32", dtype]))
    layers, channels = rng.randint(0, 8), 8 * _log(rng, 4, 64) + rng.choice([0, 0, 1, 3])
    if kind == "clip":
        return dict(kind=kind, layers=layers, channels=channels, dtype=dtype)
    return dict(kind=kind, layers=layers, channels=channels, dtype=dtype, bits=rng.choice([32, 8]),
                clip=rng.random() < 0.5)


def _shapes(layers, c):
    """The trained tensors of the backbone and its energy head with c channels (no layers: the head alone)."""
    head = [(c, c), (c,), (c, c), (c,), (1, c), (1,)]
    if not layers:
        return head

    def profile(k):
        return [(128, k), (128,), (128,), (128,), (128, 128), (128,), (128,), (128,), (c, 128), (c,)]

    def scalars(k):
        return [(3, 2 * c, k), (1, 1, 2 * c), (3, 2 * c, k), (2 * c, 6 * c), (2 * c,), (2 * c,), (2 * c,),
                (4 * c, 2 * c), (4 * c,)]

    first = [(256, c), (30, c), (30, c), (c, 2 * c), (c,), (c, c), (c,), (256, c), (c, 128), (c,)]
    degree = 3 * profile(768) + [(300, 256), (300, 256), (3, c, 2 * c), (c,)]
    block = ([(3, c), (c,), (256, 128), (256, 128)] + profile(512) + 2 * scalars(c) + [(3, c, c), (c,)]
             + [(c, c), (c, 3 * c), (c, 2 * c), (3, c, c), (c,)]
             + [(3, c), (c,), (3, c, c), (c,), (3 * c, c), (3 * c,), (3, c, c), (c,)])
    return first + degree + layers * block + [(3, c), (c,)] + head


def _layout(layers, c):
    """Shapes, offsets and the length of the flat buffer."""
    shapes = _shapes(layers, c)
    ends, off = [], 0
    for s in shapes:
        ends.append(off)
        off += -(-math.prod(s) // 64) * 64
    return shapes, ends, off


def work(case):
    if case["kind"].startswith("norm"):
        n, w = case["rows"] * case["width"], case["width"]
        moved = {"norm": 2, "norm_train": 4, "norm_force": 7}[case["kind"]]
        flops = {"norm": 8, "norm_train": 20, "norm_force": 45}[case["kind"]]
        return {"bytes": moved * n * SIZE[case["dtype"]] + 2 * w * SIZE[case["weights"]], "flops": flops * n}
    n = sum(math.prod(s) for s in _shapes(case["layers"], case["channels"]))
    size = SIZE[case["dtype"]]
    if case["kind"] == "clip":
        return {"bytes": 2 * size * n, "flops": 3 * n}
    # 8 bits: codes in and out, two scale bytes in and out for 32 elements, the moments' values given back in bf16
    states = 16 if case["bits"] == 32 else 4 + 4 / 32 + 4
    return {"bytes": (3 * size + states) * n, "flops": (18 if case["bits"] == 32 else 60) * n}


# --------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["kind"].startswith("norm"):
        n, w = case["rows"], case["width"]
        wd = DTYPES[case["weights"]]
        # rows as a Linear leaves them: an offset and a spread of their own
        x = rand(n, w).mul_(torch.exp(0.5 * rand(n, 1))).add_(rand(n, 1)).to(dt)
        st = dict(kind=case["kind"], x=x, w=(1 + 0.3 * rand(w)).to(wd), b=(0.5 * rand(w)).to(wd))
        if case["kind"] != "norm":
            st["gy"] = rand(n, w).to(dt)
        if case["kind"] == "norm_force":
            st["q"] = rand(n, w)
        if case["kind"] != "norm":
            st["x"].requires_grad_(True), st["w"].requires_grad_(True), st["b"].requires_grad_(True)
            st["gy"].requires_grad_(case["kind"] == "norm_force")
        return st
    shapes, offs, total = _layout(case["layers"], case["channels"])
    sizes = [math.prod(s) for s in shapes]
    # each tensor's gradients have a size of their own; padding stays zero
    reps = torch.tensor([-(-k // 64) * 64 for k in sizes], device="cuda")
    scale = torch.repeat_interleave(10 ** (2 * torch.rand(len(sizes), device="cuda", generator=g) - 3), reps,
                                    output_size=total)
    inside = torch.arange(total, device="cuda") - torch.repeat_interleave(torch.tensor(offs, device="cuda"), reps,
                                                                          output_size=total)
    scale *= inside < torch.repeat_interleave(torch.tensor(sizes, device="cuda"), reps, output_size=total)
    del inside
    grad = (rand(total) * scale).to(dt)
    if case["kind"] == "clip":
        st = dict(kind="clip", grad=grad, params=[])
        for s, o, k in zip(shapes, offs, sizes):
            p = torch.empty(s, device="cuda", dtype=dt).requires_grad_(True)
            p.grad = grad[o:o + k].view(s)
            st["params"].append(p)
        return st
    st = dict(kind="adamw", bits=case["bits"], clip=case["clip"], step=STEP, grad=grad,
              flat=(0.05 * rand(total) * (scale > 0)).to(dt))
    m = 0.25 * rand(total) * scale
    v = (scale * (0.3 + torch.rand(total, device="cuda", generator=g))) ** 2
    del scale
    if case["bits"] == 32:
        st["m"], st["v"] = m, v
    else:
        u = torch.randint(0, 65536, (total,), device="cuda", generator=g)
        st["mc"], st["ms"] = _encode(m, u, signed=True)
        u = torch.randint(0, 65536, (total,), device="cuda", generator=g)
        st["vc"], st["vs"] = _encode(v, u, signed=False)
    if own:
        _optimizer(st, shapes, offs, sizes)
    return st


def _optimizer(st, shapes, offs, sizes):
    """The optimizer that a training program keeps, its states those of the middle of a run."""
    st["params"] = []
    for s, o, k in zip(shapes, offs, sizes):
        p = st["flat"][o:o + k].view(s).requires_grad_(True)
        p.grad = st["grad"][o:o + k].view(s)
        st["params"].append(p)
    st["opt"] = _mod("optim").AdamW(st["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                    state_bits=st["bits"], max_norm=MAX_NORM if st["clip"] else None, seed=SEED)
    sd = st["opt"].state_dict()
    for i, (s, o, k) in enumerate(zip(shapes, offs, sizes)):
        e = {"step": torch.tensor(STEP)}
        if st["bits"] == 32:
            e["exp_avg"], e["exp_avg_sq"] = st["m"][o:o + k].view(s), st["v"][o:o + k].view(s)
        else:
            lo, hi = o // 32, o // 32 + -(-k // 32)
            e["exp_avg"], e["exp_avg_scale"] = st["mc"][o:o + k].view(s), st["ms"][lo:hi]
            e["exp_avg_sq"], e["exp_avg_sq_scale"] = st["vc"][o:o + k].view(s), st["vs"][lo:hi]
        sd["state"][i] = e
    st["opt"].load_state_dict(sd)


# --------------------------------------------------------------------------- one pass

def run(st):
    if st["kind"] == "norm":
        return _norm_own(st) if own else _norm(st)
    if st["kind"] == "norm_train":
        return _norm_train_own(st) if own else _norm_train(st)
    if st["kind"] == "norm_force":
        return _norm_force_own(st) if own else _norm_force(st)
    if st["kind"] == "clip":
        return _clip_own(st) if own else _clip(st)
    return _adamw_own(st) if own else _adamw(st)


def _norm_own(st):
    return _mod("norms").layer_norm(st["x"], st["w"], st["b"], LN_EPS)


def _norm_train_own(st):
    y = _mod("norms").layer_norm(st["x"], st["w"], st["b"], LN_EPS)
    return (y, *torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["gy"]))


def _norm_force_own(st):
    y = _mod("norms").layer_norm(st["x"], st["w"], st["b"], LN_EPS)
    gx, = torch.autograd.grad(y, st["x"], st["gy"], create_graph=True)
    return (y, gx, *torch.autograd.grad(gx, (st["x"], st["gy"], st["w"]), st["q"]))


def _adamw_own(st):
    st["opt"].step()
    if st["bits"] == 32:
        return st["flat"], *st["opt"].moments()
    return st["flat"], *st["opt"].moments(dtype=torch.bfloat16)


def _clip_own(st):
    return _mod("optim").clip_grad_norm_(st["params"], MAX_NORM), st["grad"]


def _normed(x):
    """The rows in 32 bits, centred and scaled, and the scale."""
    x = x.detach().float()
    x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + LN_EPS)
    return x * r, r


def _norm(st):
    xh, _ = _normed(st["x"])
    return (xh * st["w"].detach().float() + st["b"].detach().float()).to(st["x"].dtype)


def _norm_train(st):
    xh, r = _normed(st["x"])
    w, gy = st["w"].detach().float(), st["gy"].float()
    y = xh * w + st["b"].detach().float()
    u = gy * w
    gx = r * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))
    return (y.to(st["x"].dtype), gx.to(st["x"].dtype), (gy * xh).sum(0).to(st["w"].dtype),
            gy.sum(0).to(st["b"].dtype))


def _norm_force(st):
    def mean(t):
        return t.mean(-1, keepdim=True)

    xh, r = _normed(st["x"])
    w, gy, q = st["w"].detach().float(), st["gy"].detach().float(), st["q"]
    y = xh * w + st["b"].detach().float()
    u = gy * w
    c, m = mean(u * xh), mean(q * xh)
    gx = r * (u - mean(u) - xh * c)
    a = r * (q - mean(q) - xh * m)
    t = -r * (c * q + m * u)
    dx = r * (t - mean(t) - xh * mean(t * xh)) - r * mean(q * gx) * xh
    return (y.to(st["x"].dtype), gx.to(st["x"].dtype), dx.to(st["x"].dtype), (w * a).to(st["x"].dtype),
            (gy * a).sum(0).to(st["w"].dtype))


def _norm_of(grad):
    return grad.double().square().sum().sqrt()


def _clip(st):
    norm = _norm_of(st["grad"])
    c = torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0).float()
    st["grad"].copy_(st["grad"].float() * c)
    return norm.float(), st["grad"]


def _adamw(st):
    st["step"] += 1
    t = st["step"]
    p, g = st["flat"].float(), st["grad"].float()
    if st["clip"]:
        g = g * torch.clamp(MAX_NORM / (_norm_of(st["grad"]) + 1e-6), max=1.0).float()
    if st["bits"] == 32:
        m, v = st["m"], st["v"]
    else:
        m, v = _decode(st["mc"], st["ms"], signed=True), _decode(st["vc"], st["vs"], signed=False)
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = p * (1 - LR * DECAY) - LR / (1 - BETA1 ** t) * m / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    st["flat"].copy_(p)
    if st["bits"] == 32:
        st["m"], st["v"] = m, v
        return st["flat"], m, v
    u = _random_bits(p.numel(), t)
    st["mc"], st["ms"] = _encode(m, u & 0xFFFF, signed=True)
    st["vc"], st["vs"] = _encode(v, u >> 16, signed=False)
    return (st["flat"], _decode(st["mc"], st["ms"], signed=True).to(torch.bfloat16),
            _decode(st["vc"], st["vs"], signed=False).to(torch.bfloat16))


# --------------------------------------------------------------------------- states in 8 bits

_MASK, _GOLDEN, _ROOT2, _ROOT3 = 0xFFFFFFFF, 0x9E3779B9, 0x6A09E667, 0xBB67AE85


def _mix(x):
    """A 32-bit hash of whole numbers (of Python, or tensors of 64 bits)."""
    x = ((x ^ (x >> 16)) * _ROOT2) & _MASK
    x = ((x ^ (x >> 15)) * _ROOT3) & _MASK
    return x ^ (x >> 16)


def _random_bits(n, step):
    """32 random bits for each of the first n positions at a step; beyond 2^32 positions the key would change."""
    key = _mix((_mix(SEED & _MASK) + step * _GOLDEN) & _MASK)
    return _mix(torch.arange(n, device="cuda") ^ key)


def _encode(x, u, signed):
    """Codes and scale bytes of x, rounded up where the 16 random bits u reach its distance to the next code."""
    runs = x.abs().view(-1, 32)
    top = torch.where(runs.isfinite(), runs, 0).amax(1).view(torch.int32)
    # the binade in which the largest value stays below the last code
    s = (top + (0x0FFFFF if signed else 0x1FFFFF)) >> 23
    # moved so that the exponent fields of 32-bit numbers are those of the codes
    t = (runs.double() * torch.exp2((15 if signed else 31) - s.double()).view(-1, 1)).float().view(-1)
    code = (t.view(torch.int32) + (u.int() << 4) + 8) >> 20
    if signed:
        code = torch.where(code > 0, code + torch.where(x < 0, 128, 0), 0)
    else:
        code = torch.maximum(code, (x > 0).int())
    code = torch.where(x.isfinite(), code, 128 if signed else 255)
    return code.to(torch.uint8), s.to(torch.uint8)


def _decode(code, s, signed):
    c = code.int()
    t = ((c & 127 if signed else c) << 20).view(torch.float32).view(-1, 32)
    x = (t.double() * torch.exp2(s.double() - (15 if signed else 31)).view(-1, 1)).float().view(-1)
    if signed:
        x = torch.where(c > 127, -x, x)
    return torch.where(c == (128 if signed else 255), math.nan, x)


# --------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"].startswith("norm"):
        x, w, b = (st[k].detach().double().requires_grad_(True) for k in ("x", "w", "b"))
        z = x - x.sum(-1, keepdim=True) / x.shape[-1]
        y = z / ((z ** 2).sum(-1, keepdim=True) / x.shape[-1] + LN_EPS).sqrt() * w + b
        if case["kind"] == "norm":
            return y.detach()
        gy = st["gy"].detach().double().requires_grad_(True)
        if case["kind"] == "norm_train":
            return (y.detach(), *torch.autograd.grad(y, (x, w, b), gy))
        gx, = torch.autograd.grad(y, x, gy, create_graph=True)
        return (y.detach(), gx.detach(), *torch.autograd.grad(gx, (x, gy, w), st["q"].double()))
    g = st["grad"].double()
    norm = torch.linalg.vector_norm(g)
    c = min(1.0, MAX_NORM / (float(norm) + 1e-6))
    if case["kind"] == "clip":
        return norm, g * c
    g = g * c if case["clip"] else g
    if case["bits"] == 32:
        m, v = st["m"].double(), st["v"].double()
    else:
        m, v = _value(st["mc"], st["ms"], 4, True), _value(st["vc"], st["vs"], 5, False)
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g ** 2 - v)
    t = STEP + 1
    mhat, vhat = m / -math.expm1(t * math.log(BETA1)), v / -math.expm1(t * math.log(BETA2))
    p = st["flat"].double()
    p = p - LR * (DECAY * p + mhat / (vhat.sqrt() + EPS))
    if case["bits"] == 32:
        return p, m, v
    u = _random_bits(m.numel(), t)
    return p, _rounded(m, u & 0xFFFF, 4, True), _rounded(v, u >> 16, 5, False)


def _value(code, s, bits, signed):
    """What codes of 3 mantissa and `bits` exponent bits stand for, in 64 bits."""
    c = code.long()
    sign = torch.where(c > 127, -1.0, 1.0) if signed else 1.0
    c = c % 128 if signed else c
    e, f = c // 8, (c % 8).double()
    lead = (e > 0).double()
    top = s.double().repeat_interleave(32) - 127
    return sign * (lead + f / 8) * torch.exp2(top - (2 ** bits - 1) + torch.clamp(e, min=1))


def _rounded(x, u, bits, signed):
    """x at the code below or above it, in 64 bits: above where the random part of a step reaches it."""
    a = x.abs()
    most = a.view(-1, 32).amax(1)
    e = torch.frexp(most)[1] - 1.0
    last = 1.875 if signed else 1.75
    e = torch.where(most > last * torch.exp2(e), e + 1, e).repeat_interleave(32)
    low = e - (2 ** bits - 1) + 1                  # the lowest binade; its step holds below it too
    step = torch.exp2(torch.maximum(torch.frexp(a)[1] - 1.0, low) - 3)
    q = torch.floor(a / step + (16 * u + 8).double() / 2 ** 20)
    q = q if signed else torch.maximum(q, (a > 0).double())
    return torch.where(a > 0, torch.sign(x) * q * step, 0.0)
