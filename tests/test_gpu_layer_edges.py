"""The layer operators where values leave a type or a range."""
import pytest
import torch

from i8muon_b200 import check_status, linear

pytestmark = pytest.mark.gpu
BEYOND = {       # dtype: (x, magnitude of W, magnitude of the bias); z = 64 x W + bias is exact and no longer a number of the type
    "fp16 7e4": (torch.float16, 128.0, 8.5, 0.0),                                        # 69632
    "fp16 1e6": (torch.float16, 128.0, 122.0, 0.0),                                      # 999424
    "bf16 max": (torch.bfloat16, 2.0 ** 60, 0.75 * 2.0 ** 54, 255 * 2.0 ** 120),         # 255.75 2^120, below 2^128
}


@pytest.mark.parametrize("checkpoint", [None, "int8", "fp8"])
@pytest.mark.parametrize("act", ["relu", "relu2", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("outer", [16, 17])
@pytest.mark.parametrize("beyond", BEYOND)
def test_slopes_at_a_pre_activation_beyond_its_type(cuda_device, beyond, outer, act, checkpoint):
    """A pre-activation that FP32 holds is kept as an infinity of its type, or as a code that may stand for one: the slopes are
    0 and 1 there, and every gradient is a sum of few equal terms, exact in the type.  (relu2's slope on the right is twice the
    pre-activation, which leaves the type itself.)"""
    dtype, x_value, w_value, b_value = BEYOND[beyond]
    rows, inner = 3, 64
    sign = torch.ones(outer, dtype=torch.float64, device=cuda_device)
    if act == "relu2":
        sign[:] = -1
    else:
        sign[1::2] = -1
    x = torch.full((rows, inner), x_value, dtype=dtype, device=cuda_device).requires_grad_()
    w = (sign * w_value).to(dtype)[:, None].repeat(1, inner).requires_grad_()
    b = (sign * b_value).to(dtype).requires_grad_()
    # brings the results on the right back into the type where it can
    r = (sign.clamp_min(0) * (-2.0 ** 14 if dtype == torch.float16 else -2.0 ** 126)).to(dtype).expand(rows, outer)
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    assert (z.abs() < torch.finfo(torch.float32).max).all() and torch.isinf(z.to(dtype)).all()
    y = linear(x, w, b, activation=act, residual=r, checkpoint=checkpoint)
    assert torch.equal(y.detach(), (z.clamp_min(0) + r.double()).to(dtype))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    check_status()
    dz = (z > 0).double()
    assert torch.equal(dx.double(), dz @ w.detach().double())
    assert torch.equal(dw.double(), dz.t() @ x.detach().double())
    assert torch.equal(db.double(), dz.sum(0))
