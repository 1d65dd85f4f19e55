"""What optim refuses and checks without a GPU, and the entry points' checks of their arguments."""
import copy
import pickle
from types import SimpleNamespace

import pytest
import torch

from ubio_molfm_amd import _lib, optim


@pytest.fixture(autouse=True)
def _no_kernels(monkeypatch):
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("a kernel was called"))


def _p(*shape):
    p = torch.zeros(shape, requires_grad=True)
    p.grad = torch.ones(shape)
    return p


@pytest.mark.parametrize("kw,match", [
    (dict(lr=-1.0), "lr"), (dict(lr=float("nan")), "lr"), (dict(lr=torch.zeros(2)), "lr"),
    (dict(betas=(1.0, 0.9)), "betas"),
    (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=-1e-8), "eps"), (dict(weight_decay=-0.1), "weight_decay"),
    (dict(state_bits=16), "16 bits"), (dict(max_norm=0.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm")])
def test_constructor_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        optim.AdamW([_p(3)], **kw)


def test_group_values_are_checked():
    opt = optim.AdamW([_p(3)])
    with pytest.raises(ValueError, match="lr"):
        opt.add_param_group(dict(params=[_p(4)], lr=-2.0))
    assert len(opt.param_groups) == 1


def test_host_tensors_are_refused():
    for call in (lambda: optim.AdamW([_p(3)]).step(), lambda: optim.AdamW([_p(3)]).moments(),
                 lambda: optim.clip_grad_norm_([_p(3)], 1.0), lambda: optim.grad_norm([torch.ones(3)]),
                 lambda: optim.grad_norm(torch.ones(3))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_([_p(3)], -1.0)


def test_entry_point_checks():
    lib, C = _lib.load(), _lib.C
    ptrs, numel = (_lib.vp * 2)(64, 128), (_lib.i64 * 2)(5, 1 << 33)
    assert lib.e2v2_grad_norm_parts(numel, 2) == 1024 and lib.e2v2_grad_norm_parts(numel, 0) == 0
    many = (_lib.i64 * 600)(*([7] * 600))
    assert lib.e2v2_grad_norm_parts(many, 600) == 3 * 1024
    count = C.c_int(0)

    def norm(n=2, type=0, parts=64, cap=0):
        return lib.e2v2_grad_norm(ptrs, numel, n, type, _lib.vp(parts), cap, C.byref(count), None)

    assert norm(n=-1) != 0 and b"-1 tensors" in lib.e2v2_last_error()
    assert norm(type=5) != 0 and b"type 5" in lib.e2v2_last_error()
    assert norm(parts=None) != 0 and b"null operand" in lib.e2v2_last_error()
    assert norm() != 0 and b"room for 0" in lib.e2v2_last_error() and count.value == 0
    ptrs[1] = 66
    assert norm() != 0 and b"tensor 1" in lib.e2v2_last_error()
    ptrs[1], numel[0] = 128, -1
    assert norm() != 0 and b"tensor 0 of -1" in lib.e2v2_last_error()
    assert lib.e2v2_grad_scale(ptrs, numel, 2, 0, None, 0, _lib.f32(1), None, None) != 0
    assert lib.e2v2_grad_norm_value(None, 1, _lib.vp(64), None) != 0
    a = _lib.AdamWArgs()
    a.n_chunks, a.n_tensors, a.bits = 1, 1, 32
    a.chunks = a.steps = a.grads = a.m = a.v = C.addressof(ptrs)
    a.m = a.v = 64
    a.beta1 = a.beta2 = 0.9
    ptrs[0] = 64
    for change, match in ((dict(n_tensors=385), b"385"), (dict(n_chunks=-1), b"-1 chunks"), (dict(bits=4), b"4 bits"),
                          (dict(type=3), b"type 3"), (dict(bits=8), b"null operand"), (dict(m=None), b"null operand"),
                          (dict(m=72), b"16-byte"), (dict(n_parts=2), b"null operand"),
                          (dict(skip_nonfinite=1), b"null operand"), (dict(beta2=1.0), b"betas")):
        b = _lib.AdamWArgs.from_buffer_copy(a)
        for k, v in change.items():
            setattr(b, k, v)
        assert lib.e2v2_adamw(C.byref(b), None) != 0 and match in lib.e2v2_last_error(), change
    ptrs[0] = 66
    assert lib.e2v2_adamw(C.byref(a), None) != 0 and b"misaligned gradient 0" in lib.e2v2_last_error()
    v = _lib.vp(64)
    assert lib.e2v2_moments(v, v, v, v, v, v, 0, _lib.i64(33), None) != 0
    assert lib.e2v2_moments(v, v, _lib.vp(68), v, v, v, 0, _lib.i64(32), None) != 0
    assert lib.e2v2_moments(v, None, v, v, v, v, 0, _lib.i64(32), None) != 0


def test_chunk_table():
    """Every element of every tensor in one chunk, in order, in the layout of e2v2_opt_chunk."""
    sizes, ptrs = [5, 0, 4096, 4097, 20000], [1 << 40, 64, 128, 256, 512]
    offs = [0, 64, 64, 4160, 8320]
    t, first = optim._chunk_table(ptrs, offs, sizes)
    assert first == [0, 1, 1, 2, 4] and len(t) == 9 and t.dtype.itemsize == _lib.C.sizeof(_lib.OptChunk) == 32
    rows = (_lib.OptChunk * len(t)).from_buffer_copy(t.tobytes())
    got = [(r.p, r.at, r.off, r.n, r.tensor) for r in rows]
    assert got == [(ptrs[k], at, offs[k] + at, min(4096, n - at), k) for k, n in enumerate(sizes)
                   for at in range(0, n, 4096)]
    assert [len(x) for x in optim._chunk_table([], [], [])] == [0, 0]


class _OnGpu1(torch.Tensor):
    """A host tensor that says it lies on the second GPU."""

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        return 1 if func is torch.Tensor.get_device else super().__torch_function__(func, types, args, kwargs or {})


@pytest.mark.parametrize("device,second", [(0, torch.Tensor), (1, torch.Tensor), (1, _OnGpu1), (0, _OnGpu1)])
def test_gradients_that_lie_elsewhere(device, second):
    """.data moves a parameter, or a gradient, without the other: the step sees it before it takes an address."""
    grads = [torch.ones(4).as_subclass(_OnGpu1 if device else torch.Tensor), torch.ones(6).as_subclass(second)]
    launch = SimpleNamespace(device=device, dtype=torch.float32, nbytes=[16, 24])
    if device and second is _OnGpu1:
        assert optim._matching(grads, launch, True) is grads
        return
    with pytest.raises(RuntimeError, match="gradients on"):
        optim._matching(grads, launch, True)
    with pytest.raises(RuntimeError, match="gradients on"):
        optim._matching(grads[1:], launch, [False, True])


@pytest.mark.parametrize("loaded", [0.25, torch.tensor(0.25), torch.tensor([0.25], dtype=torch.float64)])
def test_rates_that_are_tensors_stay(loaded, monkeypatch):
    """load_state_dict writes the loaded learning rate into the tensor that a captured step (and a scheduler) holds."""
    monkeypatch.setattr(optim, "_Plan", lambda opt: None)
    lr = torch.tensor(1e-3)
    opt = optim.AdamW([dict(params=[_p(3)], lr=lr), dict(params=[_p(2)], lr=0.5)])
    sd = opt.state_dict()
    for g, value in zip(sd["param_groups"], (loaded, 0.125)):
        g["lr"] = value
    opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.25 and opt.param_groups[1]["lr"] == 0.125
    opt.load_state_dict(opt.state_dict())
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.25


def test_one_rate_for_groups_that_are_loaded_with_two(monkeypatch):
    monkeypatch.setattr(optim, "_Plan", lambda opt: None)
    lr = torch.tensor(1e-3)
    opt = optim.AdamW([dict(params=[_p(3)]), dict(params=[_p(2)])], lr=lr)
    assert opt.param_groups[1]["lr"] is lr
    sd = opt.state_dict()
    sd["param_groups"][0]["lr"], sd["param_groups"][1]["lr"] = 0.25, torch.tensor(0.5)
    opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] is lr and [float(g["lr"]) for g in opt.param_groups] == [0.25, 0.5]


def test_what_is_put_into_an_entry():
    """Tensors put in the place of an entry's own are copied into the buffers that the step reads."""
    m, v, steps = torch.zeros(6), torch.zeros(6, dtype=torch.uint8), torch.zeros(3, dtype=torch.int32)
    e = optim._Entry({"step": steps[0], "exp_avg": m.view(2, 3), "exp_avg_sq": v.view(2, 3)}, steps)
    own = dict(e)
    for k in list(e):
        e[k] = e[k]                                           # as a loop that moves a state to a device does
    e["exp_avg"] = torch.arange(6.0, dtype=torch.float64).view(2, 3)
    e.update(step=torch.tensor(7.0), exp_avg_sq=torch.full((2, 3), 9, dtype=torch.uint8))
    e |= {"exp_avg": e["exp_avg"] + 1}
    assert m.tolist() == [1, 2, 3, 4, 5, 6] and steps.tolist() == [7] * 3 and v.tolist() == [9] * 6
    assert all(e[k] is own[k] for k in own)
    for k, t in (("exp_avg", torch.zeros(6)), ("exp_avg", torch.zeros(2, 3, dtype=torch.int32)),
                 ("exp_avg_sq", torch.zeros(2, 3))):
        with pytest.raises(ValueError, match=k):
            e[k] = t
    with pytest.raises(KeyError, match="max_exp_avg_sq"):
        e["max_exp_avg_sq"] = m
    for change in (lambda: e.pop("step"), lambda: e.clear(), lambda: e.__delitem__("step")):
        with pytest.raises(TypeError, match="stay"):
            change()
    for plain in (copy.deepcopy(e), copy.copy(e), e.copy(), pickle.loads(pickle.dumps(e))):
        assert type(plain) is dict and plain.keys() == own.keys() and torch.equal(plain["exp_avg"], e["exp_avg"])


def test_memory_that_tensors_share():
    buf = torch.zeros(100)

    def overlap(*ts):
        return optim._overlap(optim._by_type(ts, {t.dtype for t in ts}))

    assert torch.zeros(0).data_ptr() == buf[50:50].data_ptr() == 0      # those without elements lie nowhere
    assert not overlap(buf[60:], buf[:50], buf[50:60], buf[50:50], torch.zeros(0), buf.new_zeros(5))
    assert not overlap(buf) and not overlap(torch.zeros(0), torch.zeros(0))
    for ts in ((buf, buf), (buf[:51], buf[50:]), (buf, buf[7:8]), (buf[50:], torch.zeros(9), buf[:99]),
               (buf, buf[40:].view(torch.bfloat16)[3:5])):
        assert overlap(*ts) and overlap(*ts[::-1])
    assert not overlap(buf[:50], buf[50:].view(torch.float16))


def test_hooks_of_loading(monkeypatch):
    """They see the whole state and may change it; what belongs to no parameter is kept."""
    plans = []
    monkeypatch.setattr(optim, "_Plan", lambda opt: plans.append(dict(opt.state)))
    monkeypatch.setattr(optim, "_usable", lambda p: True)
    p = _p(3)
    opt = optim.AdamW([p], lr=0.5)
    entry = {"step": 4, "exp_avg": torch.ones(3), "exp_avg_sq": torch.ones(3)}
    given = {"state": {0: entry, "run": [1, 2]}, "param_groups": opt.state_dict()["param_groups"]}
    seen = []

    def double(o, sd):
        seen.append(list(sd["state"]))
        return {**sd, "state": {**sd["state"], 0: {**entry, "exp_avg": 2 * entry["exp_avg"]}}}

    opt.register_load_state_dict_pre_hook(double)
    opt.register_load_state_dict_post_hook(lambda o: seen.append(len(plans)))
    for _ in range(2):
        opt.load_state_dict(given)
    assert seen == [[0, "run"], 1, [0, "run"], 2] and list(given["state"]) == [0, "run"]
    assert plans[0][p]["exp_avg"].tolist() == [2, 2, 2] and plans[0]["run"] == [1, 2]
    with pytest.raises(ValueError, match="parameter groups"):
        opt.load_state_dict({"state": {}, "param_groups": given["param_groups"] * 2})
    assert len(opt._optimizer_load_state_dict_pre_hooks) == len(opt._optimizer_load_state_dict_post_hooks) == 1
