"""Forward-mode derivatives of the layer operators are refused: a tangent that the kernels do not see would read as zero."""
import pytest
import torch
from torch.autograd import forward_ad

from i8muon_b200 import layer_norm, linear, quantise_activation

CALLS = {
    "linear x": lambda t, p: linear(t, p["w"]),
    "linear weight": lambda t, p: linear(p["x"], t),
    "linear bias": lambda t, p: linear(p["x"], p["w"], t),
    "linear residual": lambda t, p: linear(p["x"], p["w"], residual=t),
    "layer_norm x": lambda t, p: layer_norm(t, p["b"]),
    "layer_norm weight": lambda t, p: layer_norm(p["x"], t),
    "layer_norm bias": lambda t, p: layer_norm(p["x"], None, t),
    "quantise_activation": lambda t, p: quantise_activation(t),
}


def arguments(device="cpu"):
    gen = torch.Generator().manual_seed(1)
    return {k: torch.randn(s, generator=gen).bfloat16().to(device) for k, s in dict(x=(3, 8), w=(8, 8), b=(8,)).items()}


def primal_of(call, p):
    return p["w"] if call == "linear weight" else p["b"] if call.split()[-1] in ("weight", "bias") else p["x"]


def dual_of(call, p, requires_grad=False):
    t = primal_of(call, p)
    return forward_ad.make_dual(t.clone().requires_grad_(requires_grad), torch.ones_like(t))


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("call", CALLS)
def test_a_tangent_is_refused(call, requires_grad):
    p = arguments()
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            CALLS[call](dual_of(call, p, requires_grad), p)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            CALLS[call](dual_of(call, p, requires_grad), p)
        with pytest.raises(ValueError, match="needs CUDA"):       # tensors without one are as good as ever
            CALLS[call](primal_of(call, p), p)


@pytest.mark.gpu
@pytest.mark.parametrize("call", CALLS)
def test_a_tangent_is_refused_on_the_device(cuda_device, call):
    p = arguments(cuda_device)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            CALLS[call](dual_of(call, p), p)
        CALLS[call](primal_of(call, p), p)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: CALLS[call](t, p), (primal_of(call, p),), (torch.ones_like(primal_of(call, p)),))


@pytest.mark.gpu
@pytest.mark.parametrize("make", [lambda x, p: linear(x, p["w"], activation="silu"), lambda x, p: layer_norm(x, p["b"])])
def test_a_tangent_of_the_results_gradient_is_refused(cuda_device, make):
    p = arguments(cuda_device)
    x = p["x"].clone().requires_grad_()
    y = make(x, p)
    dy = torch.ones_like(y)
    want, = torch.autograd.grad(y, x, dy, retain_graph=True)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.autograd.grad(y, x, forward_ad.make_dual(dy, dy.clone()), retain_graph=True)
        got, = torch.autograd.grad(y, x, dy)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_a_residuals_gradient_alone_keeps_its_tangent(cuda_device):
    """It is the result's gradient itself: nothing is computed that could lose one."""
    p = arguments(cuda_device)
    r = p["x"].clone().requires_grad_()
    y = linear(p["x"], p["w"], residual=r)
    dy = torch.ones_like(y)
    with forward_ad.dual_level():
        got, = torch.autograd.grad(y, r, forward_ad.make_dual(dy, 2 * dy))
        primal, tangent = forward_ad.unpack_dual(got)
        assert torch.equal(primal, dy) and torch.equal(tangent, 2 * dy)
