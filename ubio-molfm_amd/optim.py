"""The parameter update of training over many tensors at once (HIP kernels of libe2v2.so, csrc/optim.hip):
``AdamW`` with moments in 32 or in 8 bits, ``clip_grad_norm_`` and ``grad_norm``.

One launch updates all tensors of a parameter group (two with clipping: the norm's sums, then the update, which applies
the clipping factor to each gradient as it reads it), whatever their number and sizes; nothing is read back to
the host.  The reference's trainer calls torch's counterparts (src/molfm/pipeline/trainer.py:114-662).  There is no
CPU path."""
from __future__ import annotations

import ctypes as C
import math
from array import array
from collections import OrderedDict
from contextlib import nullcontext
from itertools import chain, compress
from operator import attrgetter, is_
from typing import Iterable, Optional, Tuple, Union

import numpy as np
import torch

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_CHUNK = 4096           # E2V2_OPT_CHUNK
_LIST = 384             # tensors of one step launch
_ALIGN = 64             # a tensor's moments start at a multiple of this many elements
_RUN = 32               # elements that share a scale byte
_NBYTES = attrgetter("nbytes")


class _Lists:
    """Dense tensors of one type as the library takes them: their addresses (0: left out) and sizes."""

    def __init__(self, dtype, ptrs, numels):
        self.type, self.itemsize = _lib.i32(_TYPES[dtype]), dtype.itemsize
        self.numel = array("q", numels)
        self.n = _lib.i32(len(self.numel))
        self.set(ptrs)

    def set(self, ptrs):
        self.ptrs = array("Q", ptrs)

    def address(self) -> int:
        return self.ptrs.buffer_info()[0]

    def parts(self) -> int:
        return int(_lib.load().e2v2_grad_norm_parts(_lib.vp(self.numel.buffer_info()[0]), self.n))

    def norm(self, parts, count, st):
        _lib.call("e2v2_grad_norm", _lib.vp(self.address()), _lib.vp(self.numel.buffer_info()[0]), self.n, self.type,
                  _lib.vp(parts.data_ptr()), _lib.i32(parts.numel()), C.byref(count), st)

    def scale(self, parts, count, max_norm, norm, st):
        _lib.call("e2v2_grad_scale", _lib.vp(self.address()), _lib.vp(self.numel.buffer_info()[0]), self.n, self.type,
                  _lib.vp(parts.data_ptr()), count, _lib.f32(max_norm), _lib.vp(norm.data_ptr()), st)


def _dense(ts, what: str):
    """The tensors in known types and contiguous (copies where they are not), and their types.  A few hundred pass here
    every step: each property is read in one sweep."""
    types = {t.dtype for t in ts}
    try:
        contiguous = all(map(torch.Tensor.is_contiguous, ts))
    except RuntimeError:                       # sparse tensors do not answer
        contiguous = False
    if not contiguous or not types <= _TYPES.keys():
        layouts = {t.layout for t in ts} - {torch.strided}
        if layouts or not types <= _TYPES.keys():
            raise ValueError(f"{what}: dense fp32, bf16 or fp16 tensors, got {', '.join(map(str, [*layouts, *types]))}")
        ts = [t.contiguous() for t in ts]
    return types, ts


def _check(ts, what: str):
    """As _dense, for tensors that have to lie on one GPU, which comes first."""
    devices = set(map(torch.Tensor.get_device, ts))
    if -1 in devices:
        raise RuntimeError(f"{what} runs on the GPU only (HIP library, no CPU path): got a tensor on "
                           f"{next(t.device for t in ts if not t.is_cuda)}")
    if len(devices) > 1:
        raise ValueError(f"{what}: tensors on the GPUs {sorted(devices)}")
    return ts[0].device, *_dense(ts, what)


def _by_type(ts, types):
    """The tensors' lists."""
    lists = []
    for d in sorted(types, key=_TYPES.get):
        of = ts if len(types) == 1 else [t for t in ts if t.dtype == d]
        lists.append(_Lists(d, map(torch.Tensor.data_ptr, of), map(torch.Tensor.numel, of)))
    return lists


def _norm_parts(lists, dev, st):
    """The partial sums of the norm of all lists, and how many there are."""
    parts = torch.empty(max(1, sum([l.parts() for l in lists])), dtype=torch.float64, device=dev)
    count = C.c_int(0)
    for l in lists:
        l.norm(parts, count, st)
    return parts, count


def _overlap(lists) -> bool:
    """Whether tensors of the lists share memory."""
    at, size = ([f(l) for l in lists] for f in (lambda l: np.frombuffer(l.ptrs, np.int64),
                                                lambda l: np.frombuffer(l.numel, np.int64) * l.itemsize))
    at, size = (x[0] if len(x) == 1 else np.concatenate(x) for x in (at, size))
    order = at.argsort()
    at, end = at[order], (at + size)[order]
    return bool((end[:-1] > at[1:]).any())


def _on(dev):
    """A context with dev as the current device."""
    return nullcontext() if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def grad_norm(tensors: Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all elements of the tensors (dense, fp32, bf16 or fp16, one device), as an fp32 tensor of one
    element on that device; the squares are summed in fp64.  An empty list has norm 0 (on the current device)."""
    ts = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not ts:
        return torch.zeros((), device="cuda")
    dev, types, ts = _check(ts, "grad_norm")
    out = torch.empty((), dtype=torch.float32, device=dev)
    with _on(dev):
        st = _lib.stream(dev)
        lists = _by_type(ts, types)
        parts, count = _norm_parts(lists, dev, st)
        _lib.call("e2v2_grad_norm_value", _lib.vp(parts.data_ptr()), count, _lib.vp(out.data_ptr()), st)
    return out


def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """Scales the parameters' gradients in place by min(1, max_norm / (norm + 1e-6)), norm their global 2-norm, which
    is returned (an fp32 tensor of one element), as torch.nn.utils.clip_grad_norm_.  Contiguous gradients that share
    memory, and the same one twice, are refused.  A norm that is not finite scales by what the quotient gives (0, or
    NaN); nothing is read back to the host."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_grad_norm_: max_norm {max_norm}")
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return torch.zeros((), device="cuda" if torch.cuda.is_available() else None)
    dev, types, dense = _check(grads, "clip_grad_norm_")
    lists = _by_type(dense, types)
    if _overlap(lists):
        raise ValueError("clip_grad_norm_: the same gradient twice, or gradients that share memory")
    if dense is not grads:
        if len(set(map(id, grads))) < len(grads):
            raise ValueError("clip_grad_norm_: the same gradient twice")
        if any(step == 0 and n > 1 for g in grads for step, n in zip(g.stride(), g.shape)):
            raise ValueError("clip_grad_norm_: a gradient whose elements share memory")
    out = torch.zeros((), dtype=torch.float32, device=dev)
    with _on(dev):
        st = _lib.stream(dev)
        parts, count = _norm_parts(lists, dev, st)
        for l in lists:
            l.scale(parts, count, max_norm, out, st)
    if dense is not grads:
        with torch.no_grad():
            for g, d in zip(grads, dense):
                if d is not g:
                    g.copy_(d)
    torch.autograd.graph.increment_version(grads)
    return out


def _usable(p) -> bool:
    return p.is_cuda and p.layout == torch.strided and p.dtype in _TYPES and p.is_contiguous()


def _refuse(params):
    """Parameters that a step cannot take: an error if one has a gradient."""
    for p in params:
        if p.grad is None:
            continue
        if not p.is_cuda:
            raise RuntimeError(f"AdamW runs on the GPU only (HIP library, no CPU path): got a parameter on {p.device}")
        raise ValueError("AdamW: contiguous parameters in fp32, bf16 or fp16, got "
                         f"{tuple(p.shape)} {p.dtype} with strides {p.stride()}")


class _Launch:
    """One step launch: up to _LIST parameters of one group and type, and their chunks of the table."""

    def __init__(self, group, dtype, params, first_tensor, chunk0, n_chunks):
        self.group, self.dtype, self.params = group, dtype, params
        self.first_tensor, self.chunk0, self.n_chunks = first_tensor, chunk0, n_chunks
        self.device = params[0].get_device()
        self.grads = _Lists(dtype, [0] * len(params), [p.numel() for p in params])
        self.nbytes = [p.nbytes for p in params]
        self.args = _lib.AdamWArgs()


class _OtherTypes(Exception):
    """The parameters were given another type in place."""


def _matching(grads, launch, which):
    """The gradients of the launch's parameters (of those that ``which`` says; True: all), contiguous: on their device, of
    their types and sizes.  torch checks a gradient where it is set, but .data moves a parameter or a gradient alone."""
    if set(map(torch.Tensor.get_device, grads)) != {launch.device}:
        raise RuntimeError(f"AdamW: gradients on {sorted({str(g.device) for g in grads})} for parameters on "
                           f"cuda:{launch.device}")
    sizes = launch.nbytes if which is True else list(compress(launch.nbytes, which))
    try:
        # bytes that agree leave the type open only between the two of 16 bits
        if (all(map(torch.Tensor.is_contiguous, grads)) and list(map(_NBYTES, grads)) == sizes
                and (launch.dtype == torch.float32 or {g.dtype for g in grads} == {launch.dtype})):
            return grads
    except RuntimeError:                       # sparse tensors do not answer
        pass
    types, grads = _dense(grads, "AdamW")
    if types != {launch.dtype}:
        if any(p.dtype != launch.dtype for p in launch.params):
            raise _OtherTypes
        raise ValueError(f"AdamW: gradients of type {types} for parameters in {launch.dtype}")
    if list(map(_NBYTES, grads)) != sizes:
        raise ValueError("AdamW: gradients of other sizes than their parameters")
    return grads


def _chunk_table(ptrs, offs, sizes):
    """The e2v2_opt_chunk table of tensors at ptrs whose moments start at offs, and each tensor's first chunk."""
    counts = np.array([-(-n // _CHUNK) for n in sizes], np.int64)
    first = np.cumsum(counts) - counts
    which = np.repeat(np.arange(len(sizes)), counts)
    t = np.zeros(len(which), np.dtype([("p", np.uint64), ("at", np.int64), ("off", np.int64), ("n", np.int32),
                                       ("tensor", np.int32)]))
    t["p"] = np.array(ptrs, np.uint64)[which]
    t["at"] = (np.arange(len(which)) - first[which]) * _CHUNK
    t["off"] = np.array(offs, np.int64)[which] + t["at"]
    t["n"] = np.minimum(np.array(sizes, np.int64)[which] - t["at"], _CHUNK)
    t["tensor"] = which
    return t, first.tolist()


class _Entry(dict):
    """A parameter's state: views of the plan's buffers, and its step count in every chunk.  A tensor that is put in a
    view's place is copied into it; copies and pickles are plain dicts."""

    def __init__(self, views, steps):
        super().__init__(views)
        self.steps = steps

    def __setitem__(self, k, t):
        if k not in self:
            raise KeyError(f"AdamW: the state has no {k}")
        own = self[k]
        if t is own:
            return
        t = torch.as_tensor(t).detach()
        if k == "step":
            t = t.clone().view(())
            own.copy_(t)
            self.steps.copy_(t)
            return
        if t.shape != own.shape or not (t.is_floating_point() if own.is_floating_point() else t.dtype == own.dtype):
            raise ValueError(f"AdamW: {k} of {tuple(t.shape)} {t.dtype}, not {tuple(own.shape)} {own.dtype}")
        own.copy_(t)

    def update(self, *args, **kw):
        for k, t in dict(*args, **kw).items():
            self[k] = t

    def __ior__(self, other):
        self.update(other)
        return self

    def _stay(self, *args):
        raise TypeError("AdamW: the tensors of a state stay; take the parameter's whole entry out")

    __delitem__ = pop = popitem = clear = _stay

    def __reduce__(self):
        return dict, (dict(self),)


class _Plan:
    """What stays from step to step: moments and step counts of all parameters, the chunks' table, the launches."""

    @torch.no_grad()
    def __init__(self, opt: "AdamW"):
        groups = opt.param_groups
        every = [p for g in groups for p in g["params"]]
        # the others may stand in the groups as long as they have no gradient (a model's constants)
        self.every, self.split = every, [len(g["params"]) for g in groups]
        params = [p for p in every if _usable(p)]
        self.outside = [p for p in every if not _usable(p)]
        _refuse(self.outside)
        for p in params:
            if p.device != params[0].device:
                raise ValueError(f"AdamW: parameters on {params[0].device} and {p.device}")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("AdamW: parameters that share memory")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the first step, and the one after a change of parameters or groups, cannot be "
                               "captured: take it before the capture")
        self.device = dev = params[0].device if params else torch.device("cuda", torch.cuda.current_device())
        self.ptrs, self.nbytes = [p.data_ptr() for p in params], [p.nbytes for p in params]
        self.params = params
        bits = opt.state_bits
        sizes = [p.numel() for p in params]
        ends = np.cumsum([0] + [-(-n // _ALIGN) * _ALIGN for n in sizes]).tolist()
        self.total = ends[-1]
        place = dict(zip(params, ends))
        dt = torch.float32 if bits == 32 else torch.uint8
        self.m, self.v = (torch.zeros(self.total, dtype=dt, device=dev) for _ in range(2))
        self.ms, self.vs = ((torch.zeros(self.total // _RUN, dtype=torch.uint8, device=dev) for _ in range(2))
                            if bits == 8 else (None, None))
        self.launches, order, chunks = [], [], 0
        for k_group, group in enumerate(groups):
            by_type = {}
            for p in group["params"]:
                if p in place:
                    by_type.setdefault(p.dtype, []).append(p)
            for dtype, ps in by_type.items():
                for k in range(0, len(ps), _LIST):
                    part = ps[k:k + _LIST]
                    n = sum([-(-p.numel() // _CHUNK) for p in part])
                    self.launches.append(_Launch(k_group, dtype, part, len(order), chunks, n))
                    order += part
                    chunks += n
        table, first = _chunk_table([p.data_ptr() for p in order], [place[p] for p in order],
                                    [p.numel() for p in order])
        self.chunks = torch.from_numpy(table.view(np.uint8)).to(dev)
        self.steps = torch.zeros(max(len(table), 1), dtype=torch.int32, device=dev)
        first = dict(zip(order, first))
        self.parts = torch.empty(max(1, sum(l.grads.parts() for l in self.launches)), dtype=torch.float64, device=dev)
        self.norm = torch.zeros((), dtype=torch.float32, device=dev)
        for l in self.launches:
            a = l.args
            a.chunks = self.chunks.data_ptr() + l.chunk0 * C.sizeof(_lib.OptChunk)
            a.steps = self.steps.data_ptr() + l.chunk0 * 4
            a.m, a.v = self.m.data_ptr(), self.v.data_ptr()
            if bits == 8:
                a.ms, a.vs = self.ms.data_ptr(), self.vs.data_ptr()
            a.n_chunks, a.n_tensors, a.first_tensor = l.n_chunks, len(l.params), l.first_tensor
            a.type, a.bits, a.seed = _TYPES[l.dtype], bits, opt.seed & 0xFFFFFFFF
        self.first = first
        self.state = {p: self._views(p, place[p], first[p]) for p in params}
        if opt._skipped is None or opt._skipped.device != dev:
            opt._skipped = torch.zeros((), dtype=torch.int32, device=dev)
        self.fill({p: opt._entry(p, opt.state[p], f"a parameter {tuple(p.shape)}") for p in params if opt.state.get(p)})
        opt.state.update(self.state)
        self.entries = list(opt.state.values())

    @torch.no_grad()
    def fill(self, entries):
        """Takes over the states in entries (of the plan's parameters)."""
        if not entries:
            return
        dev = self.device
        steps = [torch.as_tensor(e["step"]) for e in entries.values()]
        if any(t.is_cuda for t in steps):
            steps = torch.stack([t.to(dev, torch.int32).view(()) for t in steps])
        else:
            steps = torch.tensor([int(t) for t in steps], dtype=torch.int32).to(dev)      # one copy for all
        counts = np.array([-(-p.numel() // _CHUNK) for p in entries])
        ends = np.cumsum(counts)
        where = np.arange(ends[-1]) + np.repeat(np.array([self.first[p] for p in entries]) - (ends - counts), counts)
        which = np.repeat(np.arange(len(entries)), counts)
        where, which = torch.from_numpy(np.stack([where, which])).to(dev)
        self.steps[where] = steps[which]
        for p, step in zip(entries, steps):
            if not p.numel():
                self.state[p]["step"].copy_(step)
        pairs = [(t, e[k]) for p, e in entries.items() for k, t in self.state[p].items() if k != "step"]
        # another parameter's views of these buffers may be written before they are read
        buffers = {t.untyped_storage().data_ptr() for t in (self.m, self.v, self.ms, self.vs) if t is not None}
        pairs = [(d, o.clone() if o.untyped_storage().data_ptr() in buffers and o.data_ptr() != d.data_ptr() else o)
                 for d, o in pairs]
        torch._foreach_copy_([d for d, _ in pairs], [o for _, o in pairs])

    def clear(self, params):
        """Zero states for some of the plan's parameters."""
        for p in params:
            self.state[p].steps.zero_()
            for t in self.state[p].values():
                t.zero_()

    def _views(self, p, o, chunk):
        """The parameter's state: views of the plan's buffers."""
        n = p.numel()
        st = {"step": self.steps[chunk] if n else torch.zeros((), dtype=torch.int32, device=p.device)}
        for k, t, s in (("exp_avg", self.m, self.ms), ("exp_avg_sq", self.v, self.vs)):
            st[k] = t[o:o + n].view(p.shape)
            if s is not None:
                st[k + "_scale"] = s[o // _RUN:o // _RUN + -(-n // _RUN)]
        return _Entry(st, self.steps[chunk:chunk - (-n // _CHUNK)])


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay; Adam for weight_decay=0) over all parameters at once.

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

    params: contiguous fp32, bf16 or fp16 parameters on one GPU (others only without a gradient), or groups of them
    with their own lr, betas, eps and weight_decay (lr may be a tensor of one element on that GPU, read by the step
    itself).  Parameters without a gradient are left out of a step, as in torch.  Arithmetic and 32-bit moments
    are fp32 whatever the parameters' type, which are rounded to nearest once a step.

    state_bits=8 keeps both moments in 8 bits (runs of 32 elements share a power-of-two scale; 3 mantissa bits, rounded
    stochastically by a hash of ``seed``, step and element, so that runs repeat): 2.1 bytes a parameter instead of 8.
    ``state[p]`` then holds codes ("exp_avg", "exp_avg_sq") and scale bytes ("..._scale"); ``moments`` gives values.

    max_norm scales the gradients by min(1, max_norm / (norm + 1e-6)), norm their global 2-norm over all groups, as
    they are read (they stay as they were); skip_nonfinite leaves parameters, moments and step counts as they were
    where that norm is not finite and counts such steps in ``skipped``.  ``grad_norm`` is the last step's norm (None
    without either).

    A step after the first can be captured into a graph and replayed: step counts are on the device.  Such a graph goes
    on after load_state_dict (numbers among a group's values are those of the capture; a learning rate that is a tensor
    is the loaded one); parameters that move and groups that are added void it.  As with any graph torch does not
    see that a replay changed the parameters: torch.autograd.graph.increment_version(parameters) says so to what is
    kept per weight version (the evaluation path's packed weights and tables).  ``state`` entries are views of flat
    buffers: moments can be written in place, and what is put in an entry's place or in that of one of its tensors (step
    counts only so) is copied into the buffers that are there; an entry that is taken out starts anew.  Entries are looked
    over by steps that are not captured."""

    _plan: Optional[_Plan] = None
    _OPTIONS = ("state_bits", "max_norm", "skip_nonfinite", "seed")

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 max_norm: Optional[float] = None, skip_nonfinite: bool = False, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: moments of {state_bits} bits (8 or 32)")
        if max_norm is not None and not float(max_norm) > 0:
            raise ValueError(f"AdamW: max_norm {max_norm}")
        self.state_bits, self.seed = int(state_bits), int(seed)
        self.max_norm = None if max_norm is None else float(max_norm)
        self.skip_nonfinite = bool(skip_nonfinite)
        self._skipped = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    @staticmethod
    def _check_group(g):
        lr, (b1, b2) = g["lr"], g["betas"]
        for k in ("amsgrad", "maximize", "differentiable"):
            if g.get(k):
                raise ValueError(f"AdamW: {k} is not supported")
        if not g.get("decoupled_weight_decay", True) and g["weight_decay"]:
            raise ValueError("AdamW: weight decay as a part of the gradient is not supported")
        if not isinstance(lr, torch.Tensor) and not 0.0 <= lr < math.inf:
            raise ValueError(f"AdamW: lr {lr}")
        if isinstance(lr, torch.Tensor) and lr.numel() != 1:
            raise ValueError(f"AdamW: lr of {lr.numel()} elements")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: betas {g['betas']}")
        if not g["eps"] >= 0.0 or not g["weight_decay"] >= 0.0:
            raise ValueError(f"AdamW: eps {g['eps']}, weight_decay {g['weight_decay']}")

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            self._check_group(self.param_groups[-1])
        except ValueError:
            self.param_groups.pop()
            raise
        self._plan = None

    def __getstate__(self):
        return {**super().__getstate__(), **{k: getattr(self, k) for k in self._OPTIONS}, "_skipped": self._skipped}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plan = None

    @property
    def grad_norm(self) -> Optional[torch.Tensor]:
        """The global norm of the last step's gradients (before scaling); None where no step computes it."""
        if self._plan is None or (self.max_norm is None and not self.skip_nonfinite):
            return None
        return self._plan.norm

    @property
    def skipped(self) -> Optional[torch.Tensor]:
        """Steps left out because the norm was not finite (an int32 tensor of one element); None without
        skip_nonfinite."""
        return self._skipped if self.skip_nonfinite else None

    def _entry(self, p, e, name):
        """What belongs to the parameter's state of a loaded or hand-made entry."""
        names = ["step", "exp_avg", "exp_avg_sq"]
        if self.state_bits == 8:
            names += ["exp_avg_scale", "exp_avg_sq_scale"]
        for k in names:
            if k not in e:
                raise ValueError(f"AdamW: the state of {name} has no {k} (moments of {self.state_bits} bits)")
        for k in names[1:]:
            size = (-(-p.numel() // _RUN),) if k.endswith("scale") else tuple(p.shape)
            right = e[k].is_floating_point() if self.state_bits == 32 else e[k].dtype == torch.uint8
            if tuple(e[k].shape) != size or not right:
                raise ValueError(f"AdamW: {k} of {name} is {tuple(e[k].shape)} {e[k].dtype}, not {size} "
                                 f"{'in a floating type' if self.state_bits == 32 else torch.uint8}")
        return {k: e[k] for k in names}

    def state_dict(self):
        """As torch's; the entries refer to the state itself."""
        sd = super().state_dict()
        sd["state"] = {k: dict(e) if type(e) is _Entry else e for k, e in sd["state"].items()}
        return sd

    def load_state_dict(self, state_dict):
        """As torch's, with moments kept in their own types: fp32, or codes and scale bytes.  Learning rates that are
        tensors stay and take the loaded values (one tensor for several groups where these agree; the others get the
        loaded ones, which a step captured before does not read)."""
        pre, post = self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks
        state_dict = state_dict.copy()
        for hook in pre.values():                                 # they see the whole state, which torch's part does not
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        self._load(state_dict)
        for hook in post.values():
            hook(self)

    def _load(self, state_dict):
        """load_state_dict without hooks; torch's part gets the groups and what belongs to no parameter."""
        groups = state_dict["param_groups"]
        saved, new = dict(state_dict["state"]), {}
        for i, p in zip(chain.from_iterable(g["params"] for g in groups),
                        chain.from_iterable(g["params"] for g in self.param_groups)):
            e = saved.pop(i, None)
            if not e:
                continue
            if not _usable(p):
                raise ValueError(f"AdamW: state for parameter {i}, which is not contiguous in fp32, bf16 or fp16 on "
                                 "the GPU")
            new[p] = self._entry(p, e, f"parameter {i}")
        for g in groups:
            self._check_group(g)
        plan = self._plan if self._valid() else None
        rates = [g["lr"] for g in self.param_groups]
        hooks = self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks
        self._optimizer_load_state_dict_pre_hooks = self._optimizer_load_state_dict_post_hooks = OrderedDict()
        try:                                                      # refuses groups of other sizes
            super().load_state_dict({**state_dict, "state": saved})
        finally:
            self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks = hooks
        values = {}
        for g, lr in zip(self.param_groups, rates):               # captured steps read the rates that are there
            if isinstance(lr, torch.Tensor):
                value = float(g["lr"])
                if values.setdefault(id(lr), value) == value:     # else one tensor for groups of several rates
                    with torch.no_grad():
                        lr.fill_(value)
                    g["lr"] = lr
        if plan is None:
            self.state.update(new)
            self._plan = _Plan(self)
        else:                                                     # in place: captured steps go on with the new state
            plan.fill(new)                                        # new may be the plan's own state
            plan.clear([p for p in plan.params if p not in new])
            self.state.update(plan.state)
            plan.entries = list(self.state.values())
            self._plan = plan

    def moments(self, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(m, v) of all parameters in the order of the groups, flat, each parameter's from a multiple of 64 elements on
        (the gaps are zero).  32 bits without a dtype: the state itself; else values in dtype (fp32, bf16, fp16;
        8-bit moments are exact in each as long as they are normal there)."""
        if dtype not in (None, *_TYPES):
            raise ValueError(f"AdamW.moments: {dtype}")
        plan = self._with_entries(self._plan) if self._same_groups() else self._current()
        if self.state_bits == 32:
            return (plan.m, plan.v) if dtype is None else (plan.m.to(dtype), plan.v.to(dtype))
        dtype = dtype or torch.float32
        m, v = (torch.empty(plan.total, dtype=dtype, device=plan.device) for _ in range(2))
        with _on(plan.device):
            _lib.call("e2v2_moments", *(_lib.vp(t.data_ptr()) for t in (plan.m, plan.ms, plan.v, plan.vs, m, v)),
                      _lib.i32(_TYPES[dtype]), _lib.i64(plan.total), _lib.stream(plan.device))
        return m, v

    def _same_groups(self) -> bool:
        """Whether the plan is that of the groups' parameters, in their order."""
        plan = self._plan
        if plan is None:
            return False
        groups = [g["params"] for g in self.param_groups]
        return list(map(len, groups)) == plan.split and all(map(is_, chain.from_iterable(groups), plan.every))

    def _valid(self) -> bool:
        """Whether the plan holds for a step: the same groups, and no parameter was moved, cut, turned or given a type of
        another size (of one of that size, the gradients' types tell)."""
        plan = self._plan
        return (self._same_groups() and list(map(torch.Tensor.data_ptr, plan.params)) == plan.ptrs
                and list(map(_NBYTES, plan.params)) == plan.nbytes
                and all(map(torch.Tensor.is_contiguous, plan.params)) and not any(map(_usable, plan.outside)))

    def _with_entries(self, plan: _Plan) -> _Plan:
        """The plan, with the states of entries that were taken out or put in their place by hand: zeros, or what they
        hold, written into the buffers that are there, so that captured steps go on."""
        state = self.state
        if len(state) == len(plan.entries) and all(map(is_, state.values(), plan.entries)):
            return plan
        changed = {p: state.get(p) for p in plan.params if state.get(p) is not plan.state[p]}
        if changed:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: the first step after a change of the states cannot be captured: take it "
                                   "before the capture")
            new = {p: self._entry(p, e, f"a parameter {tuple(p.shape)}") for p, e in changed.items() if e}
            plan.fill(new)
            plan.clear([p for p in changed if p not in new])
            state.update({p: plan.state[p] for p in changed})
        plan.entries = list(state.values())
        return plan

    def _current(self) -> _Plan:
        if not self._valid():
            self._plan = _Plan(self)
        return self._with_entries(self._plan)

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        plan = self._current()
        try:
            with _on(plan.device):
                self._launch(plan)
        except _OtherTypes:
            self._plan = plan = _Plan(self)
            with _on(plan.device):
                self._launch(plan)
        return loss

    def _launch(self, plan: _Plan):
        st = _lib.stream(plan.device)
        normed = self.max_norm is not None or self.skip_nonfinite
        _refuse(plan.outside)
        count = C.c_int(0)
        keep, updated = [], []
        for l in plan.launches:
            grads = [p.grad for p in l.params]
            try:
                dense = _matching(grads, l, True)
                updated += l.params
                l.grads.set(list(map(torch.Tensor.data_ptr, dense)))
            except TypeError:                  # some parameters have none
                there = [g is not None for g in grads]
                dense = list(compress(grads, there))
                dense = _matching(dense, l, there) if dense else []
                updated += compress(l.params, there)
                it = iter(dense)
                l.grads.set([next(it).data_ptr() if t else 0 for t in there])
            keep.append(dense)
            if normed:
                l.grads.norm(plan.parts, count, st)
        if normed and not count.value:
            plan.norm.zero_()                  # no gradient at all
        norm = plan.norm.data_ptr()
        for l in plan.launches:
            a, g = l.args, self.param_groups[l.group]
            a.grads = l.grads.address()
            lr = g["lr"]
            if isinstance(lr, torch.Tensor) and lr.is_cuda:
                lr = lr.to(plan.device, torch.float32)     # itself, or on the GPU: nothing is read back
                keep.append(lr)
                a.lr_dev, a.lr = lr.data_ptr(), 0.0
            else:
                a.lr_dev, a.lr = None, float(lr)
            a.beta1, a.beta2 = g["betas"]
            a.eps, a.weight_decay = g["eps"], g["weight_decay"]
            a.parts, a.n_parts = plan.parts.data_ptr(), count.value
            a.max_norm = math.inf if self.max_norm is None else self.max_norm
            a.norm = norm if l.n_chunks else None      # one launch writes it; without chunks there is none
            norm = None if l.n_chunks else norm
            a.skip_nonfinite = int(self.skip_nonfinite)
            a.skipped = self._skipped.data_ptr()
            _lib.call("e2v2_adamw", C.byref(a), st)
        # what is kept per weight version (packed weights, radial tables) is made anew
        torch.autograd.graph.increment_version(updated)
