"""torch.jit.trace over the norms, the 8-bit operators and the products by expert: a trace replays the kernels on other
inputs, or the call is refused; it never returns the empty tensor that a launch outside of a Function leaves in it."""
import pytest
import torch

from ubio_molfm_amd import experts, fp8, norms

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore")]


def _rand(*shape, seed, cuda):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(cuda)


def _all(o):
    return o if isinstance(o, tuple) else (o,)


def _replays(f, make, grads):
    """The trace of f on make(1) gives f's bits on make(2) and make(3), with gradients and without."""
    args = make(1)
    args[0].requires_grad_(grads)
    traced = torch.jit.trace(f, args, check_trace=False)
    for seed in (2, 3):
        args = make(seed)
        with torch.no_grad():
            want, got = _all(f(*args)), _all(traced(*args))
        assert len(want) == len(got) and all(torch.equal(a, b) for a, b in zip(got, want))
        leaf = args[0].detach().clone().requires_grad_(True)
        grads = [torch.autograd.grad([t for t in _all(g(leaf, *args[1:])) if t.requires_grad][0].float().sum(), leaf)[0]
                 for g in (f, traced)]
        assert torch.equal(*grads)


@pytest.mark.parametrize("grads", [False, True])
def test_traces_replay(grads, cuda):
    gain = _rand(64, seed=0, cuda=cuda)
    w = _rand(40, 64, seed=1, cuda=cuda)
    each = _rand(3, 40, 64, seed=2, cuda=cuda)

    def rows(seed):
        return (_rand(9, 64, seed=seed, cuda=cuda),)

    def two(seed):
        return rows(seed) + rows(seed + 10)

    def sorted_rows(seed):
        return rows(seed) + (torch.tensor([0, seed, 5, 9], dtype=torch.int32, device=cuda),)

    _replays(lambda x: norms.layer_norm(x, gain), rows, grads)
    _replays(lambda x: norms.rms_norm(x, gain), rows, grads)
    _replays(lambda x: norms.rms_norm(x), rows, grads)
    _replays(lambda x, r: norms.rms_norm(x, gain, residual=r), two, grads)
    _replays(lambda x: fp8.linear(x, w), rows, grads)
    _replays(lambda x, o: experts.expert_linear(x, each, o), sorted_rows, grads)


def test_what_a_trace_would_lose_is_refused(cuda):
    x, w = _rand(9, 64, seed=1, cuda=cuda), _rand(2, 40, 64, seed=2, cuda=cuda)
    offs = torch.tensor([0, 4, 9], dtype=torch.int32, device=cuda)
    (xq, sx), (wq, sw) = fp8.quantize(x), fp8.quantize(w, tiles=True)
    out = torch.zeros(9, 40, device=cuda)
    for f in (lambda t: norms.rms_norm_fp8(t)[1], lambda t: fp8.quantize(t)[1],
              lambda t: fp8.dequantize(xq, sx) + t, lambda t: fp8.gemm(xq, sx, wq[0], sw[0]) + t[:, :40],
              lambda t: experts.expert_linear(t, w, offs, out=out),
              lambda t: experts.expert_gemm_fp8(xq, sx, wq, sw, offs) + t[:, :40]):
        f(x)
        with pytest.raises(RuntimeError, match="torch.jit.trace"):
            torch.jit.trace(f, (x,), check_trace=False)
