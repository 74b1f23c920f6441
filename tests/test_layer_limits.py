"""Extents beyond 32 bits and beyond the layers' limits, without a GPU: refused by the arguments' checks before anything is
allocated, and by the C ABI under the value that was passed."""
import pytest
import torch

from i8muon_b200 import QuantisedActivation, layer_norm, linear, native, quantise_activation, restore_activation
from i8muon_b200.build import build

WRAPS = (1 << 32) + 8        # 8 in 32 bits
ONE, HALF = torch.zeros(1), torch.zeros(1, dtype=torch.float16)


@pytest.fixture(scope="module", autouse=True)
def library():
    build()


def rows_of(rows, width=1, like=ONE):
    """A tensor of any extents over a single element."""
    return like.expand(rows, width)


def codes_of(rows, width):
    return QuantisedActivation(rows_of(rows, width, ONE.char()), rows_of(rows, width // 32, ONE.byte()), torch.Size((rows, width)),
                               torch.float32, "int8")


@pytest.mark.parametrize("call", [
    lambda: quantise_activation(rows_of(1, WRAPS)),
    lambda: quantise_activation(rows_of(1, (1 << 24) + 1)),
    lambda: quantise_activation(rows_of(WRAPS)),
    lambda: quantise_activation(ONE.expand(WRAPS)),
    lambda: restore_activation(codes_of(1, WRAPS + 24)),
    lambda: restore_activation(codes_of(WRAPS, 32)),
    lambda: layer_norm(rows_of(1, WRAPS)),
    lambda: layer_norm(rows_of(WRAPS)),
    lambda: layer_norm(ONE.expand(1 << 16, 1 << 16, 1 << 16)),
    lambda: linear(rows_of(WRAPS, 1, HALF), rows_of(8, 1, HALF)),
    lambda: linear(rows_of((1 << 31) - 1024, 1, HALF), rows_of(8, 1, HALF)),
    lambda: linear(rows_of(3, WRAPS, HALF), rows_of(8, WRAPS, HALF)),
    lambda: linear(rows_of(3, 8, HALF), rows_of(WRAPS, 8, HALF)),
    lambda: linear(rows_of(3, 8, HALF), rows_of((1 << 24) + 1, 8, HALF)),
])
def test_extents_beyond_the_limits_are_refused(call):
    with pytest.raises(ValueError, match="above the limits"):
        call()


@pytest.mark.parametrize("call", [
    lambda: quantise_activation(rows_of(1, 1 << 24)),
    lambda: layer_norm(rows_of((1 << 31) - 1025)),
    lambda: linear(rows_of((1 << 31) - 1025, 1, HALF), rows_of(1 << 24, 1, HALF)),
])
def test_extents_at_the_limits_are_not(call):
    with pytest.raises(ValueError, match="needs CUDA"):
        call()


def test_the_c_abi_sees_the_extents_that_were_passed():
    lib, p = native.library(), 1 << 20      # never dereferenced: every call is refused before a launch
    over = native.MAX_LAYER_WIDTH + 1
    for width in (WRAPS, over, 1 << 33):
        assert lib.i8m_activation_quant(p, 0, 1, width, 0, p, p, None) == -4
        assert lib.i8m_activation_restore(p, p, 1, width, 0, p, 0, None) == -4
        assert lib.i8m_layer_norm(p, None, None, p, None, None, None, None, -1, 1, width, 0, 1e-5, None) == -4
        assert lib.i8m_layer_norm_backward(p, p, p, p, None, None, -1, None, p, None, None, 1, width, 0, None, 0, None) == -4
        with pytest.raises(native.NativeError, match=str(width)):
            native.layer_norm_scratch_bytes(4, width)
    for rows, inner, outer in ((WRAPS, 16, 8), (4, WRAPS, 8), (4, 16, WRAPS), (native.MAX_LAYER_ROWS + 1, 16, 8), (4, over, 8), (4, 16, over)):
        assert lib.i8m_linear(p, p, None, None, p, None, None, None, -1, 0, rows, inner, outer, 2, None, 0, p, None) == -4
        assert lib.i8m_linear_backward(p, p, None, None, p, None, None, None, -1, 0, p, None, None, rows, inner, outer, 2, None, 0, p,
                                       None) == -4
        with pytest.raises(native.NativeError, match="above the limits"):
            native.linear_workspace_bytes(p, p, rows, inner, outer)
        with pytest.raises(native.NativeError, match="above the limits"):
            native.linear_backward_workspace_bytes(p, p, p, rows, inner, outer, 0, -1, 1, 1, 1)
    # what is not above the limits is asked for in full
    assert native.linear_workspace_bytes(p, p, 1 << 30, 17, 8) >= (1 << 30) * 24 * 2
    assert native.layer_norm_scratch_bytes(4, native.MAX_LAYER_WIDTH) == 4 * 2 * native.MAX_LAYER_WIDTH * 4


def test_every_extent_is_bound_as_a_64_bit_number():
    """The header's parameters and the binding's, one by one: an int here and a long long there would pass garbage."""
    import re
    from ctypes import c_float, c_int, c_longlong, c_size_t
    from pathlib import Path
    text = (Path(__file__).resolve().parents[1] / "include" / "i8muon_b200.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    scalars = {"int": c_int, "long long": c_longlong, "float": c_float, "size_t": c_size_t}
    names = [n for n in native.EXPORTED_SYMBOLS if n.startswith(("i8m_linear", "i8m_layer_norm", "i8m_activation"))]
    assert len(names) == 9 and native.library().i8m_version() >= 101
    for name in names:
        declared = re.search(rf"\bint {name}\(([^)]*)\)", text).group(1).split(",")
        bound = native._SIGNATURES[name][1]
        assert len(declared) == len(bound), name
        for parameter, kind in zip(declared, bound):
            words = parameter.split()
            if "*" in parameter or words[0] == "i8m_stream_t":
                assert kind not in scalars.values(), (name, parameter)
            else:
                assert kind is scalars[" ".join(words[:-1])], (name, parameter)
                if words[-1] in ("rows", "inner", "outer", "width"):
                    assert kind is c_longlong, (name, parameter)
