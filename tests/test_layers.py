"""Refusals of the layer operators, checked without a GPU: arguments are looked at before the device is."""
import pytest
import torch

from i8muon_b200 import QuantisedActivation, layer_norm, linear, native, quantise_activation, restore_activation
from i8muon_b200.build import build


@pytest.fixture(scope="module", autouse=True)
def library():
    build()


X, H, W = torch.zeros(3, 40), torch.zeros(3, 40).half(), torch.zeros(8, 40).half()


@pytest.mark.parametrize("call, message", [
    (lambda: quantise_activation(X, None), "'int8' or 'fp8'"),
    (lambda: quantise_activation(X, "int4"), "'int8' or 'fp8'"),
    (lambda: quantise_activation(X, ["int8"]), "'int8' or 'fp8'"),
    (lambda: quantise_activation(X.double()), "float32 or float16 or bfloat16"),
    (lambda: quantise_activation(torch.zeros(())), "at least one dimension"),
    (lambda: quantise_activation(torch.zeros(3, 0)), "must not be empty"),
    (lambda: quantise_activation(X), "needs CUDA"),
    (lambda: restore_activation(X), "what quantise_activation returned"),
    (lambda: layer_norm(X, checkpoint="int4"), "checkpoint must be"),
    (lambda: layer_norm(X.long()), "float32 or float16 or bfloat16"),
    (lambda: layer_norm(X, torch.zeros(39)), "weight must be a vector of 40"),
    (lambda: layer_norm(X, torch.zeros(1, 40)), "weight must be a vector of 40"),
    (lambda: layer_norm(X, bias=torch.zeros(40).half()), "bias must be a vector of 40"),
    (lambda: layer_norm(X, eps=-1e-5), "eps must be >= 0"),
    (lambda: layer_norm(X, eps=float("nan")), "eps must be >= 0"),
    (lambda: layer_norm(torch.zeros(2, 0)), "must not be empty"),
    (lambda: layer_norm(X, torch.zeros(40)), "needs CUDA"),
    (lambda: linear(X, torch.zeros(8, 40)), "float16 or bfloat16"),
    (lambda: linear(H, torch.zeros(8, 40)), "40 columns of the input's type"),
    (lambda: linear(H, W.t()), "40 columns"),
    (lambda: linear(H, W[None]), "40 columns"),
    (lambda: linear(H, W[:0]), "40 columns"),
    (lambda: linear(H, W, torch.zeros(7).half()), "bias must be a vector of 8"),
    (lambda: linear(H, W, torch.zeros(8)), "bias must be a vector of 8"),
    (lambda: linear(H, W, activation="tanh"), "activation must be"),
    (lambda: linear(H, W, activation=1), "activation must be"),
    (lambda: linear(H, W, residual=torch.zeros(8).half()), "shape and type of the result"),
    (lambda: linear(H, W, residual=torch.zeros(3, 8)), "shape and type of the result"),
    (lambda: linear(H, W, checkpoint="bf16"), "checkpoint must be"),
    (lambda: linear(torch.zeros(3, 0).half(), torch.zeros(8, 0).half()), "must not be empty"),
    (lambda: linear(H, W), "needs CUDA"),
])
def test_refusals(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_codes_that_do_not_belong_to_their_tensor_are_refused():
    codes, exponents = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3, 2, dtype=torch.uint8)
    good = QuantisedActivation(codes, exponents, torch.Size((3, 40)), torch.float32, "int8")
    with pytest.raises(ValueError, match="needs CUDA"):
        restore_activation(good)
    for bad in (good._replace(shape=torch.Size((3, 65))), good._replace(shape=torch.Size((4, 40))),
                good._replace(codes=codes[:, :32]), good._replace(exponents=exponents[:, :1]),
                good._replace(codes=codes.to(torch.uint8)), good._replace(checkpoint="fp8"),
                good._replace(exponents=exponents.to(torch.int8))):
        with pytest.raises(ValueError, match="do not belong"):
            restore_activation(bad)
    for bad in (good._replace(shape=torch.Size(())), good._replace(dtype=torch.float64),
                good._replace(shape=torch.Size((3, 0)))):
        with pytest.raises(ValueError, match="not a quantised activation"):
            restore_activation(bad)
    with pytest.raises(ValueError, match="checkpoint must be"):
        restore_activation(good._replace(checkpoint="int4"))


def test_native_argument_errors_are_codes():
    lib = native.library()
    assert lib.i8m_activation_quant(None, 0, 1, 1, 0, None, None, None) == -1
    assert lib.i8m_activation_quant(16, 0, 0, 1, 0, 16, 16, None) == -1
    assert lib.i8m_activation_quant(16, 7, 1, 1, 0, 16, 16, None) == -1
    assert lib.i8m_activation_quant(16, 0, 1, 1, -1, 16, 16, None) == -1
    assert lib.i8m_activation_quant(16, 0, 1, (1 << 24) + 1, 0, 16, 16, None) == -4
    assert lib.i8m_activation_restore(16, 16, 1 << 31, 8, 0, 16, 0, None) == -4
    assert lib.i8m_activation_quant(16, 0, 1, 1, 0, 24, 16, None) == -1        # codes on 16 bytes
    assert lib.i8m_layer_norm(16, None, None, 16, None, None, 24, 16, 0, 1, 8, 0, 1e-5, None) == -1
    assert lib.i8m_layer_norm(16, None, None, None, None, None, None, None, -1, 1, 8, 0, 1e-5, None) == -1
    assert lib.i8m_layer_norm(16, None, None, 16, None, None, None, None, 0, 1, 8, 0, 1e-5, None) == -1
    assert lib.i8m_layer_norm(16, None, None, 16, None, None, None, None, 2, 1, 8, 0, 1e-5, None) == -1
    backward = lambda *, x=16, mean=16, dx=16, dw=None, scratch=None, size=0: lib.i8m_layer_norm_backward(  # noqa: E731
        16, x, mean, 16, None, None, -1, None, dx, dw, None, 4, 8, 0, scratch, size, None)
    assert backward(x=None) == -1 and backward(mean=None) == -1 and backward(dx=None) == -1
    need = native.layer_norm_scratch_bytes(4, 8)
    assert need >= 2 * 8 * 4
    assert backward(dw=16) == -2 and backward(dw=16, scratch=16, size=need - 1) == -2


def test_native_linear_argument_errors_are_codes():
    lib = native.library()
    p = 1 << 20      # 16-byte aligned, never dereferenced: every call is refused before a launch

    def forward(*, x=p, w=p, y=p, z=None, codes=None, exponents=None, fmt=-1, act=0, rows=4, inner=16, outer=8, dtype=2, ws=None,
                size=0, status=p):
        return lib.i8m_linear(x, w, None, None, y, z, codes, exponents, fmt, act, rows, inner, outer, dtype, ws, size, status, None)
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(status=None), dict(rows=0), dict(inner=0), dict(outer=0),
                dict(dtype=0), dict(act=6), dict(act=-1), dict(fmt=2), dict(fmt=0, codes=p), dict(z=p + 8), dict(fmt=0, codes=p + 4, exponents=p)):
        assert forward(**bad) == -1, bad
    assert forward(inner=(1 << 24) + 8) == -4
    assert forward(rows=(1 << 31) - 1) == -4
    assert forward(inner=17) == -2 and forward(x=p + 2) == -2
    need = native.linear_workspace_bytes(p, p, 4, 17, 8)
    assert need >= (4 + 8) * 24 * 2
    assert forward(inner=17, ws=p, size=need - 1) == -2
    assert native.linear_workspace_bytes(p, p, 4, 16, 8) == 0
    assert native.linear_workspace_bytes(p + 2, p, 4, 16, 8) >= 4 * 16 * 2

    def backward(*, dy=p, x=p, codes=None, w=p, z=None, z_codes=None, fmt=-1, act=0, dx=p, dw=None, db=None, outer=8, ws=None, size=0):
        return lib.i8m_linear_backward(dy, x, codes, codes, w, z, z_codes, z_codes, fmt, act, dx, dw, db, 4, 16, outer, 2, ws, size, p, None)
    for bad in (dict(dy=None), dict(dx=None), dict(w=None), dict(x=None, dw=p), dict(fmt=0, dw=p), dict(act=3), dict(act=3, fmt=0),
                dict(act=3, z=p + 2)):
        assert backward(**bad) == -1, bad
    assert backward(act=3, z=p) == -2            # dz needs room
    assert backward(outer=9) == -2               # dy's rows start anywhere: a copy
    assert backward(dx=None, db=p) == -2         # partial sums
    assert backward(dx=None, db=p, ws=p + 16, size=1 << 20) == -1 and forward(inner=17, ws=p + 8, size=1 << 20) == -1
    # a long sum into few tiles takes FP32 parts, up to 64 MB of them
    assert 0 < native.linear_backward_workspace_bytes(p, p, p, 65536, 512, 512, 0, -1, 0, 1, 0) <= 64 << 20
    assert native.linear_backward_workspace_bytes(p, p, p, 4, 16, 8, 0, -1, 1, 1, 0) == 0
    assert native.linear_backward_workspace_bytes(p, p, p, 4, 16, 8, 0, 0, 0, 1, 0) >= 4 * 16 * 2
