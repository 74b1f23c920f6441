"""The layer operators where values leave a type or a range."""
import math

import pytest
import torch

import layer_reference as ref
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


EPS, FLUSH = 2.0 ** -24, 2.0 ** -126
# the exponential's instruction is good to 2^-22 of its result, the reciprocal's to 2^-23; results below 2^-126 become zero
EX2, RCP = 4 * EPS, 2 * EPS


def activation_in_double(z, act):
    """(value, slope, what FP32 may lose of either) in 64 bits; the lower tail of the normal distribution from erfc, which does
    not cancel."""
    a = z.abs()
    if act == "gelu":
        tail, density = 0.5 * torch.erfc(a / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        # exponent -a^2 / 2: a constant and two products, each rounded; the polynomial's 5e-7 holds a reciprocal and FP32 sums
        exponential = 3 * EPS * z * z / 2 + EX2
        lost = exponential + 5e-7 + 2 * EPS
        cdf = torch.where(z < 0, tail, 1 - tail)
        return (z * cdf, cdf + z * density, lost * a * tail + FLUSH * a,
                lost * tail + (exponential + 4 * EPS) * a * density + 2 * EPS * cdf + FLUSH * (1 + a))
    if act == "silu":
        v, dv, loss = z, torch.ones_like(z), 2 * EPS * a
    else:
        c = 2 * math.sqrt(2 / math.pi)
        v, dv = c * (z + 0.044715 * z ** 3), c * (1 + 3 * 0.044715 * z * z)
        loss = 6 * EPS * v.abs()               # two constants, a square, a cubic and the product with z
    s, rest = torch.sigmoid(v), torch.sigmoid(-v)
    off = s * rest * (loss + EX2) + s * (RCP + EPS) + FLUSH
    y, slope = z * s, s + z * dv * s * rest
    return y, slope, a * off + EPS * y.abs(), off * (1 + a * dv) + 8 * EPS * (s + a * dv * s * rest)


@pytest.mark.parametrize("act, far", [("gelu", 12.9), ("gelu_tanh", 12.0), ("silu", 100.0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_activations_and_slopes_over_their_tails(cuda_device, act, far, dtype):
    """z is the bias alone, every number of the type up to ``far`` (of FP16 every third): relative to the value, also where
    that is 1e-37."""
    bits = torch.arange(0, 1 << 15, dtype=torch.int32).to(torch.int16)
    z = bits.view(dtype)
    z = z[torch.isfinite(z) & (z <= far) & (z >= 2.0 ** -12)][::1 if dtype == torch.bfloat16 else 3]
    z = torch.cat((z, -z)).to(cuda_device).requires_grad_()
    x, w = torch.zeros(1, 8, dtype=dtype, device=cuda_device), torch.zeros(z.numel(), 8, dtype=dtype, device=cuda_device)
    y = linear(x, w, z, activation=act)
    got, = torch.autograd.grad(y, z, torch.ones_like(y))
    check_status()
    want, slope, off, off_slope = activation_in_double(z.detach().double(), act)
    ref.assert_within(y[0].detach(), want, off + ref.half_step(want.abs() + off, dtype), "value")
    ref.assert_within(got, slope, off_slope + ref.half_step(slope.abs() + off_slope, dtype), "slope")
