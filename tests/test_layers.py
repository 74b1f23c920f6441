"""Refusals of the layer operators, checked without a GPU: arguments are looked at before the device is."""
import pytest
import torch

from i8muon_b200 import QuantisedActivation, layer_norm, native, quantise_activation, restore_activation
from i8muon_b200.build import build


@pytest.fixture(scope="module", autouse=True)
def library():
    build()


X = torch.zeros(3, 40)


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
    assert lib.i8m_layer_norm(16, None, None, None, None, None, None, None, -1, 1, 8, 0, 1e-5, None) == -1
    assert lib.i8m_layer_norm(16, None, None, 16, None, None, None, None, 0, 1, 8, 0, 1e-5, None) == -1
    assert lib.i8m_layer_norm(16, None, None, 16, None, None, None, None, 2, 1, 8, 0, 1e-5, None) == -1
    backward = lambda *, x=16, mean=16, dx=16, dw=None, scratch=None, size=0: lib.i8m_layer_norm_backward(  # noqa: E731
        16, x, mean, 16, None, None, -1, None, dx, dw, None, 4, 8, 0, scratch, size, None)
    assert backward(x=None) == -1 and backward(mean=None) == -1 and backward(dx=None) == -1
    need = native.layer_norm_scratch_bytes(4, 8)
    assert need == 4 * 2 * 8 * 4
    assert backward(dw=16) == -2 and backward(dw=16, scratch=16, size=need - 1) == -2
