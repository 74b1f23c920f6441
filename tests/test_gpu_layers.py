"""The layer operators against their formulas in 64 bits (layer_reference.py), through the public entry points."""
import math
import pathlib
import subprocess
import sys

import pytest
import torch

import layer_reference as ref
from i8muon_b200 import QuantisedActivation, check_status, layer_norm, linear, quantise_activation, restore_activation

pytestmark = pytest.mark.gpu
TYPES = (torch.bfloat16, torch.float16, torch.float32)
FORMATS = ("int8", "fp8")


def normal(shape, seed, dtype, device, std=1.0, mean=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * std + mean).to(dtype).to(device)


# ------------------------------------------------------------- eight-bit format
@pytest.mark.parametrize("rows, width", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 127), (4, 128), (1000, 96), (33, 1531), (129, 4096),
                                         (1, 20000)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("checkpoint", FORMATS)
def test_codes_stand_for_the_nearest_values_exactly(cuda_device, rows, width, dtype, checkpoint):
    x = normal((rows, width), rows + width, torch.float64, "cpu")
    x = (x * torch.exp2(torch.randint(-12, 6, (rows, width), generator=torch.Generator().manual_seed(3)).double())).to(dtype)
    q = quantise_activation(x.to(cuda_device), checkpoint)
    groups = -(-width // 32)
    e, _ = ref.exponents_of(x.double(), checkpoint)
    assert torch.equal(q.exponents.cpu().double(), e + 127)
    assert q.codes.shape == (rows, 32 * groups) and q.exponents.shape == (rows, groups)
    assert not q.codes.view(torch.uint8)[:, width:].any()
    got = restore_activation(q)
    assert got.dtype == dtype and got.shape == x.shape
    assert torch.equal(got.cpu().double(), ref.kept(x.double(), checkpoint))   # a power of two: nothing is rounded twice


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("checkpoint", FORMATS)
def test_groups_at_the_ends_of_the_range(cuda_device, dtype, checkpoint):
    info = torch.finfo(dtype)
    tiny = 2 * ref.TINY[dtype]
    most = 127.0 if checkpoint == "int8" else 448.0
    tops = [0.0, tiny, 3 * tiny, info.tiny, info.tiny * (2 - 2 * info.eps), most * 2.0 ** -10, most * 2.0 ** -10 * (1 + info.eps),
            most / 2 * (1 + info.eps), info.max, info.max / 2, 1.0, 2.0 - info.eps * 2]
    rows = torch.zeros(len(tops), 32, dtype=torch.float64)
    for i, top in enumerate(tops):
        rows[i] = torch.linspace(-1, 1, 32, dtype=torch.float64) * top
        rows[i, 7] = -top
    x = rows.to(dtype)
    assert torch.isfinite(x).all()
    got = restore_activation(quantise_activation(x.to(cuda_device), checkpoint)).cpu()
    assert torch.isfinite(got).all()
    want = ref.kept(x.double(), checkpoint, dtype=dtype)
    assert torch.equal(got.double(), want)
    # half a step: top / 127 of the group for INT8, 2^-4 of the value or 2^-10 of the scale for E4M3, 2^-128 at the lowest
    # scale; a whole step where the code below is taken
    off, top = (got.double() - x.double()).abs(), x.double().abs().amax(1, keepdim=True)
    bound = top / 127 if checkpoint == "int8" else torch.maximum(x.double().abs() * 2.0 ** -4, top / 224 * 2.0 ** -10)
    whole = 1 + (top > info.max / 2).double()
    assert (off <= bound * whole + 2.0 ** -128).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("checkpoint", FORMATS)
@pytest.mark.parametrize("width", [64, 97])
def test_a_group_that_is_not_finite_reads_back_as_nan(cuda_device, dtype, checkpoint, width):
    x = normal((4, width), 5, dtype, cuda_device)
    x[0, 3], x[1, 40], x[2, 63] = math.inf, -math.inf, math.nan
    got = restore_activation(quantise_activation(x, checkpoint))
    want = torch.zeros_like(x, dtype=torch.bool)
    want[0, :32] = want[1, 32:64] = want[2, 32:64] = True
    assert torch.equal(torch.isnan(got), want)
    clean = torch.where(want, torch.zeros_like(x), x).cpu().double()
    assert torch.equal(got.cpu().double()[~want.cpu()], ref.kept(clean, checkpoint)[~want.cpu()])


def test_shapes_strides_and_offsets(cuda_device):
    base = normal((6, 5, 70), 7, torch.bfloat16, cuda_device)
    for x in (base, base.transpose(0, 1), base[..., 1:], base[:, ::2, 3:67], base.reshape(-1)[1:2001].view(20, 100), base[0, 0],
              base[:, :0], base[0, 0, :1].expand(9, 64)):
        got = restore_activation(quantise_activation(x, "int8"))
        want = ref.kept(x.reshape(-1, x.shape[-1]).cpu().double(), "int8").reshape(x.shape)
        assert got.shape == x.shape and torch.equal(got.cpu().double(), want)
    x = base.clone().requires_grad_()
    assert not quantise_activation(x, "fp8").exponents.requires_grad


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_start_at_any_element(cuda_device, dtype):
    """Every offset from a 16-byte boundary, widths around whole octets and warps: quantised, restored and normalised."""
    flat = normal((40000,), 3, dtype, cuda_device)
    dyflat = normal((40000,), 4, dtype, cuda_device)
    for width in (1, 3, 7, 8, 9, 31, 33, 39, 64, 65, 255, 257, 265, 1000, 1029, 2055):
        rows = min(9, 16000 // width)
        for offset in (0, 1, 2, 3, 5, 7):
            x = flat[offset:offset + rows * width].view(rows, width)
            q = quantise_activation(x)
            assert torch.equal(restore_activation(q).double(), ref.kept(x.double(), "int8"))
            w, b = flat[offset + 1:offset + 1 + width], flat[100 + offset:100 + offset + width]
            leaf = x.detach().requires_grad_()
            y = layer_norm(leaf, w, b)
            want, tol, u, tol_u, rstd, rel = ref.layer_norm(x.double(), w.double(), b.double(), 1e-5, dtype)
            ref.assert_within(y, want, tol, (width, offset))
            dy = dyflat[2 * offset:2 * offset + rows * width].view(rows, width)
            dx, = torch.autograd.grad(y, leaf, dy)
            ref.assert_within(dx, *ref.layer_norm_gradients(dy.double(), u, tol_u, rstd, rel, w.double(), dtype)["dx"], (width, offset))
    moved = QuantisedActivation(torch.zeros(97, dtype=torch.int8, device=cuda_device)[1:].copy_(q.codes[0, :96]).view(1, 96),
                                q.exponents[:1, :3].contiguous(), torch.Size((1, 96)), dtype, "int8")
    assert torch.equal(restore_activation(moved)[0], restore_activation(q)[0, :96])


# ------------------------------------------------------------------ layer norm
WIDTHS = [1, 2, 31, 33, 96, 128, 768, 1000, 1024, 1531, 2048, 4096, 6144, 8192, 8200, 16384, 20001]


def norm_inputs(rows, width, dtype, device, affine, shift):
    x = normal((rows, width), width, dtype, device, 1.0, shift)
    w = normal((width,), 1, dtype, device, 0.1, 1.0) if affine[0] else None
    b = normal((width,), 2, dtype, device, 0.1) if affine[1] else None
    return x, w, b, normal((rows, width), 3, dtype, device)


def double(t):
    return None if t is None else t.detach().double()


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, affine, shift", [(5, (True, True), 0.0), (301, (True, False), 3.0), (1, (False, False), -0.5)])
def test_layer_norm_and_its_gradients(cuda_device, width, dtype, rows, affine, shift):
    eps = 1e-5
    x, w, b, dy = norm_inputs(rows, width, dtype, cuda_device, affine, shift)
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = layer_norm(x, w, b, eps)
    got = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y)        # the same values where nothing is kept
    want, tol, u, tol_u, rstd, rel = ref.layer_norm(double(x), double(w), double(b), eps, dtype)
    ref.assert_within(y, want, tol, "y")
    wants = ref.layer_norm_gradients(double(dy), u, tol_u, rstd, rel, double(w), dtype)
    for name, g in zip([n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None], got):
        assert g.dtype == dtype
        ref.assert_within(g, *wants[name], name)


@pytest.mark.parametrize("rows, width", [(1, 1), (40, 33), (300, 768), (17, 1531), (64, 4096), (9, 8192), (5, 16384), (3, 20001)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("checkpoint", FORMATS)
def test_layer_norm_gradients_at_rows_kept_in_eight_bits(cuda_device, rows, width, dtype, checkpoint):
    eps = 1e-5
    x, w, b, dy = norm_inputs(rows, width, dtype, cuda_device, (True, True), 1.0 if width > 1 else 0.0)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = layer_norm(x, w, b, eps, checkpoint=checkpoint)
    got = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y, layer_norm(x, w, b, eps))
    _, _, u, tol_u, rstd, rel = ref.layer_norm(double(x), double(w), double(b), eps, dtype)
    kept, off = ref.kept_with_slack(u, tol_u, checkpoint)
    wants = ref.layer_norm_gradients(double(dy), kept, off, rstd, rel, double(w), dtype)
    for name, g in zip(("dx", "dw", "db"), got):
        ref.assert_within(g, *wants[name], name)


def test_layer_norm_gradients_against_differences(cuda_device):
    """Central differences of the formula in 64 bits: (f(t + h) - f(t - h)) / 2h is off by h^2 f''' / 6 and by the
    rounding of f over h, both below 1e-6 here; the FP32 gradients by their own bounds, a few 1e-6."""
    x, w, b, dy = norm_inputs(3, 40, torch.float32, cuda_device, (True, True), 0.5)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(layer_norm(x, w, b, 1e-3), leaves, dy)

    def f(*ts):
        x, w, b = ts
        c = x - x.mean(1, keepdim=True)
        return ((c / torch.sqrt(c.square().mean(1, keepdim=True) + 1e-3) * w + b) * double(dy)).sum()
    args = [double(t) for t in leaves]
    h = 1e-4
    for k, t in enumerate(args):
        for i in range(0, t.numel(), 7):
            side = []
            for sign in (1, -1):
                moved = [a.clone() for a in args]
                moved[k].view(-1)[i] += sign * h
                side.append(f(*moved).item())
            assert abs((side[0] - side[1]) / (2 * h) - got[k].reshape(-1)[i].item()) < 1e-5


def test_layer_norm_takes_any_strides_and_leading_dimensions(cuda_device):
    base = normal((4, 6, 70), 1, torch.bfloat16, cuda_device)
    for x in (base.transpose(0, 1), base[..., 1:65], base[:, ::3], base[0, 0], base.reshape(-1)[3:3 + 640].view(10, 64),
              base[0, :1].expand(5, 70)):
        w = normal((2 * x.shape[-1],), 2, torch.bfloat16, cuda_device)[::2]
        leaf = x.detach().requires_grad_()
        y = layer_norm(leaf, w)
        flat = x.reshape(-1, x.shape[-1]).double()
        want, tol, u, tol_u, rstd, rel = ref.layer_norm(flat, double(w), None, 1e-5, torch.bfloat16)
        assert y.shape == x.shape
        ref.assert_within(y.reshape(flat.shape), want, tol, "y")
        dy = normal(tuple(reversed(y.shape)), 3, torch.bfloat16, cuda_device).permute(*reversed(range(y.ndim)))
        dx, = torch.autograd.grad(y, leaf, dy)
        wants = ref.layer_norm_gradients(dy.reshape(flat.shape).double(), u, tol_u, rstd, rel, double(w), torch.bfloat16)
        ref.assert_within(dx.reshape(flat.shape), *wants["dx"], "dx")


def test_layer_norm_edges(cuda_device):
    # no rows: empty result, zero gradients of the vectors
    w, b = torch.ones(8, device=cuda_device, requires_grad=True), torch.zeros(8, device=cuda_device, requires_grad=True)
    x = torch.zeros(0, 8, device=cuda_device, requires_grad=True)
    for checkpoint in (None, "int8"):
        dx, dw, db = torch.autograd.grad(layer_norm(x, w, b, checkpoint=checkpoint).sum(), (x, w, b))
        assert dx.shape == (0, 8) and not dw.any() and not db.any()
    # constant rows: variance zero
    x = torch.full((2, 8), 3.0, device=cuda_device, requires_grad=True)
    y = layer_norm(x, w, b)
    assert not y.any()
    dx, = torch.autograd.grad(y, x, torch.randn(2, 8, device=cuda_device))
    assert torch.isfinite(dx).all()
    # a row that is not finite spoils itself alone
    x = normal((3, 64), 1, torch.float32, cuda_device)
    x[1, 5] = math.inf
    y = layer_norm(x)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2]).all()
    # values far from zero: the variance is taken around the mean
    x = normal((4, 1024), 2, torch.float32, cuda_device, 1.0, 1000.0)
    want, tol, *_ = ref.layer_norm(x.double(), None, None, 1e-5, torch.float32)
    ref.assert_within(layer_norm(x), want, tol, "y")
    # only what is asked for is computed, and the backward pass is differentiable once
    x = normal((3, 64), 1, torch.float32, cuda_device).requires_grad_()
    w = torch.ones(64, device=cuda_device, requires_grad=True)
    dw, = torch.autograd.grad(layer_norm(x.detach(), w).sum(), w)
    assert dw.shape == (64,)
    dx, = torch.autograd.grad(layer_norm(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


# ---------------------------------------------------------------------- linear
ACTS = (None, "relu", "relu2", "gelu", "gelu_tanh", "silu")


def linear_inputs(rows, inner, outer, dtype, device, bias=True, residual=True, seed=0):
    x = normal((rows, inner), seed + 1, dtype, device)
    w = normal((outer, inner), seed + 2, dtype, device, inner ** -0.5)
    b = normal((outer,), seed + 3, dtype, device, 0.3) if bias else None
    r = normal((rows, outer), seed + 4, dtype, device) if residual else None
    return x, w, b, r, normal((rows, outer), seed + 5, dtype, device)


def check_linear(x, w, b, r, dy, act, checkpoint=None):
    dtype = x.dtype
    leaves = {name: t.detach().requires_grad_() for name, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None}
    y = linear(leaves["x"], leaves["w"], leaves.get("b"), activation=act, residual=leaves.get("r"), checkpoint=checkpoint)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    assert torch.equal(linear(x, w, b, activation=act, residual=r), y)      # the same values where nothing is kept
    check_status()
    want, tol, z, tol_z = ref.linear(double(x), double(w), double(b), double(r), act, dtype)
    ref.assert_within(y, want, tol, "y")
    if checkpoint is None:
        kept, off = ref.rounded_with_slack(z, tol_z, dtype)
        kept_x = double(x)
    else:
        kept, off = ref.kept_with_slack(z, tol_z, checkpoint)
        kept_x = ref.kept(double(x), checkpoint)
    wants = ref.linear_gradients(double(dy), kept_x, double(w), kept, off, act, dtype)
    for name in ("x", "w", "b"):
        if name in got:
            assert got[name].dtype == dtype
            ref.assert_within(got[name], *wants["d" + name], "d" + name)
    if r is not None:
        assert torch.equal(got["r"], dy)


LINEAR_SHAPES = [(1, 1, 1), (1, 8, 8), (2, 7, 5), (1, 64, 128), (3, 4096, 64), (16, 1000, 200), (17, 72, 1001), (33, 129, 130), (64, 256, 512),
                 (65, 513, 384), (128, 128, 128), (129, 264, 257), (200, 1001, 333), (257, 768, 640), (1000, 96, 1000), (2050, 320, 72)]


@pytest.mark.parametrize("shape", LINEAR_SHAPES)
@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("act", ACTS)
def test_linear_and_its_gradients(cuda_device, shape, dtype, act):
    extras = sum(shape) % 4
    check_linear(*linear_inputs(*shape, dtype, cuda_device, bias=extras != 1, residual=extras >= 2), act)


@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 33, 5), (16, 1000, 200), (65, 96, 384), (130, 264, 257), (300, 768, 640)])
@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("checkpoint", FORMATS)
def test_linear_gradients_at_what_was_kept_in_eight_bits(cuda_device, shape, dtype, act, checkpoint):
    check_linear(*linear_inputs(*shape, dtype, cuda_device), act, checkpoint)


@pytest.mark.parametrize("shape", [(4096, 512, 1024), (300, 8192, 256), (12000, 256, 256), (2, 2048, 9000)])
def test_linear_over_many_tiles_and_long_sums(cuda_device, shape):
    check_linear(*linear_inputs(*shape, torch.bfloat16, cuda_device), "gelu")


@pytest.mark.parametrize("shape", [(5003, 72, 2056), (5003, 80, 2057), (2600, 40, 4328)])
@pytest.mark.parametrize("checkpoint", (None, "int8"))
def test_linear_units_at_the_edges(cuda_device, shape, checkpoint):
    """Products in units of 256 x 256 whose last units reach beyond the rows and the columns."""
    from i8muon_b200 import native
    from i8muon_b200.engine import status_word
    rows, inner, outer = shape
    x, w, b, r, dy = linear_inputs(*shape, torch.float16, cuda_device)
    check_linear(x, w, b, r, dy, "silu", checkpoint)
    # nothing behind the last row of y and of the kept pre-activation is written, and nothing in front
    pitch = -(-outer // 8) * 8
    y = torch.full((rows * outer + 1024,), 77, dtype=torch.float16, device=cuda_device)
    z = torch.full((rows * pitch + 1024,), 77, dtype=torch.float16, device=cuda_device)
    size = native.linear_workspace_bytes(x.data_ptr(), w.data_ptr(), rows, inner, outer)
    work = torch.empty(size, dtype=torch.uint8, device=cuda_device)
    native.call("i8m_linear", x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(), y[512:].data_ptr(), z[512:].data_ptr(), None, None, -1, 5, rows,
                inner, outer, native.F16, work.data_ptr(), size, status_word(cuda_device).data_ptr(), torch.cuda.current_stream().cuda_stream)
    check_status()
    for t, count in ((y, rows * outer), (z, rows * pitch)):
        assert (t[:512] == 77).all() and (t[512 + count:] == 77).all()
    assert torch.equal(y[512:512 + rows * outer].view(rows, outer), linear(x, w, b, activation="silu", residual=r))


@pytest.mark.parametrize("shape, checkpoint", [((16384, 768, 768), None), ((20000, 520, 513), None), ((16384, 256, 300), "fp8"), ((300, 768, 16384), None)])
def test_linear_sums_in_parts(cuda_device, shape, checkpoint):
    """Gradients that are long sums into few units: cut along the sum."""
    check_linear(*linear_inputs(*shape, torch.bfloat16, cuda_device, residual=False), None, checkpoint)


def test_linear_takes_any_strides_and_leading_dimensions(cuda_device):
    dtype = torch.bfloat16
    base, wbase = normal((4, 6, 80), 1, dtype, cuda_device), normal((50, 160), 2, dtype, cuda_device, 0.1)
    for x, w in ((base.transpose(0, 1), wbase[:, :80]), (base[..., 1:65], wbase[:, 3:67]), (base[:, ::3], wbase[:, ::2]), (base[0, 0], wbase[5:, 80:]),
                 (base.reshape(-1)[3:3 + 640].view(10, 64), wbase.reshape(-1)[1:1 + 640].view(10, 64)),
                 (base[0, :1].expand(5, 80), wbase[:1, :80].expand(7, 80)),
                 (base[..., :50], wbase.t()[7:11, :])):
        b = normal((2 * w.shape[0],), 3, dtype, cuda_device)[1::2]
        r = normal((w.shape[0], *x.shape[:-1]), 4, dtype, cuda_device).movedim(0, -1)
        dy = normal((w.shape[0], *x.shape[:-1]), 5, dtype, cuda_device).movedim(0, -1)
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = linear(leaves[0], leaves[1], leaves[2], activation="silu", residual=leaves[3])
        got = torch.autograd.grad(y, leaves, dy)
        flat = [t.reshape(-1, t.shape[-1]) for t in (x, r, dy)]
        want, tol, z, tol_z = ref.linear(flat[0].double(), w.double(), b.double(), flat[1].double(), "silu", dtype)
        assert y.shape == (*x.shape[:-1], w.shape[0]) and y.is_contiguous()
        ref.assert_within(y.reshape(want.shape), want, tol, "y")
        wants = ref.linear_gradients(flat[2].double(), flat[0].double(), w.double(), *ref.rounded_with_slack(z, tol_z, dtype), "silu", dtype)
        for name, g, t in zip(("dx", "dw", "db"), got, leaves):
            assert g.shape == t.shape
            ref.assert_within(g.reshape(wants[name][0].shape), *wants[name], name)
        assert torch.equal(got[3], dy)


def test_linear_gradients_against_differences(cuda_device):
    """Central differences of the formula in 64 bits with h = 1e-4: off by less than 1e-6 from the derivative, the kernels'
    gradients by their rounding to FP16 (2^-11 each for dz and the result, values below 4) and FP32 sums."""
    x, w, b, r, dy = linear_inputs(5, 24, 16, torch.float16, cuda_device)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    for act in ("gelu", "gelu_tanh", "silu"):
        got = torch.autograd.grad(linear(x, w, b, activation=act, residual=r), leaves, dy)
        args = [double(t) for t in leaves]
        for k, t in enumerate(args):
            for i in range(0, t.numel(), 11):
                side = []
                for sign in (1, -1):
                    moved = [a.clone() for a in args]
                    moved[k].view(-1)[i] += sign * 1e-4
                    side.append((ref.activation(moved[0] @ moved[1].t() + moved[2], act)[0] * double(dy)).sum().item())
                # dz's roundings add up over at most 16 products, z was kept in FP16 (2^-11 of z times the slope's change)
                assert abs((side[0] - side[1]) / 2e-4 - got[k].reshape(-1)[i].item()) < 2.0 ** -11 * 3 * 4 * 4


@pytest.mark.parametrize("act", ["relu", "relu2", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype, z", [(torch.float16, 6e4), (torch.bfloat16, 6e4), (torch.bfloat16, 1e20), (torch.bfloat16, 3e38)])
def test_derivatives_far_out(cuda_device, act, dtype, z):
    """z is the bias alone.  The slopes there are 1 and 0 to the last bit, and 2 z for relu2 (rounded once: half a step)."""
    bias = torch.tensor([z, -z] * 8, dtype=dtype, device=cuda_device).requires_grad_()
    x, w = (torch.zeros(s, dtype=dtype, device=cuda_device) for s in ((1, 64), (16, 64)))
    y = linear(x, w, bias, activation=act)
    got, = torch.autograd.grad(y, bias, torch.ones_like(y))
    slope = 2 * bias.detach().double() if act == "relu2" else torch.ones(16, dtype=torch.float64, device=cuda_device)
    want = torch.where(bias > 0, slope, 0.0).to(dtype)
    assert torch.equal(got, want)
    top = bias.detach().double() ** (2 if act == "relu2" else 1)
    assert torch.equal(y[0].detach(), torch.where(bias > 0, top, 0.0).to(dtype))
    check_status()


def test_linear_edges(cuda_device):
    dtype = torch.bfloat16
    w, b = normal((8, 16), 1, dtype, cuda_device).requires_grad_(), normal((8,), 2, dtype, cuda_device).requires_grad_()
    # no rows
    x = torch.zeros(0, 3, 16, dtype=dtype, device=cuda_device, requires_grad=True)
    for checkpoint in (None, "fp8"):
        y = linear(x, w, b, activation="gelu", checkpoint=checkpoint)
        dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
        assert y.shape == (0, 3, 8) and dx.shape == x.shape and not dw.any() and not db.any()
    # a vector is a row
    x = normal((16,), 3, dtype, cuda_device).requires_grad_()
    y = linear(x, w, b)
    assert y.shape == (8,)
    assert torch.autograd.grad(y.sum(), x)[0].shape == (16,)
    # an element that is not finite spoils its own row, and nothing else
    x = normal((200, 16), 4, dtype, cuda_device)
    x[130, 5] = math.nan
    for act in ACTS:
        y = linear(x, w, b, activation=act)
        assert torch.isnan(y[130]).all() and torch.isfinite(y[:130]).all() and torch.isfinite(y[131:]).all()
    # each gradient alone
    x = normal((40, 16), 5, dtype, cuda_device).requires_grad_()
    r = normal((40, 8), 6, dtype, cuda_device).requires_grad_()
    dy = normal((40, 8), 7, dtype, cuda_device)
    for checkpoint in (None, "int8"):
        def y():
            return linear(x, w, b, activation="silu", residual=r, checkpoint=checkpoint)
        together = torch.autograd.grad(y(), (x, w, b, r), dy)
        for t, g in zip((x, w, b, r), together):
            others = [s for s in (x, w, b, r) if s is not t]
            for s in others:
                s.requires_grad_(False)
            assert torch.equal(torch.autograd.grad(y(), t, dy)[0], g)
            for s in others:
                s.requires_grad_(True)
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(linear(x, w).float().square().sum(), x, create_graph=True)
        g.float().sum().backward()


# ------------------------------------------------------------- together, and as programs call them
def block(x, p, checkpoint):
    """A pre-norm block: norm, widening product with GELU, narrowing product onto the residual stream."""
    u = layer_norm(x, p["nw"], p["nb"], checkpoint=checkpoint)
    h = linear(u, p["w1"], p["b1"], activation="gelu", checkpoint=checkpoint)
    return linear(h, p["w2"], p["b2"], residual=x, checkpoint=checkpoint)


def block_parameters(width, dtype, device):
    p = dict(nw=normal((width,), 1, dtype, device, 0.1, 1.0), nb=normal((width,), 2, dtype, device, 0.1),
             w1=normal((4 * width, width), 3, dtype, device, width ** -0.5), b1=normal((4 * width,), 4, dtype, device, 0.1),
             w2=normal((width, 4 * width), 5, dtype, device, (4 * width) ** -0.5), b2=normal((width,), 6, dtype, device, 0.1))
    return {k: torch.nn.Parameter(v) for k, v in p.items()}


def block_in_double(x, p, dy):
    """The same block in 64 bits through torch's own graph: (y, gradients by name)."""
    leaves = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    xd = x.detach().double().requires_grad_()
    u = torch.nn.functional.layer_norm(xd, (x.shape[-1],), leaves["nw"], leaves["nb"])
    h = torch.nn.functional.gelu(u @ leaves["w1"].t() + leaves["b1"])
    y = h @ leaves["w2"].t() + leaves["b2"] + xd
    g = torch.autograd.grad(y, [xd, *leaves.values()], dy.double())
    return y, dict(zip(["x", *leaves], g))


def relative(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("rows, width", [(1, 64), (33, 200), (700, 256)])
@pytest.mark.parametrize("checkpoint, loss", [(None, 0.0), ("int8", 2.0 ** -7), ("fp8", 2.0 ** -4)])
def test_a_block_and_its_optimizer_step(cuda_device, rows, width, checkpoint, loss):
    """Roundings on the way: the two intermediate results and the gradients between the layers are rounded to BF16, half a
    step being 2^-8 of a value, at most six times between an input and a gradient, each of which the next product passes on
    with its own norm; what is kept in eight bits adds up to half a step of its format (2^-7 of the group's largest value for
    INT8, 2^-4 for E4M3) in each of the three layers."""
    from i8muon_b200 import FusedAdamW, Muon
    p = block_parameters(width, torch.bfloat16, cuda_device)
    x = normal((rows, width), 9, torch.bfloat16, cuda_device).requires_grad_()
    dy = normal((rows, width), 10, torch.bfloat16, cuda_device)
    y = block(x, p, checkpoint)
    want, wants = block_in_double(x, p, dy)
    assert relative(y, want) < 3 * 2.0 ** -8
    y.backward(dy)
    for name, g in wants.items():
        got = x.grad if name == "x" else p[name].grad
        assert relative(got, g) < 6 * 2.0 ** -8 + 3 * loss, name
    before = {k: v.detach().clone() for k, v in p.items()}
    vectors = [p[k] for k in ("nw", "nb", "b1", "b2")]
    Muon([p["w1"], p["w2"]], lr=0.02, precision="bfloat16", scalar_optimizer=FusedAdamW(vectors, lr=1e-2)).step()
    check_status()
    for k, v in p.items():
        assert torch.isfinite(v).all() and not torch.equal(v, before[k]), k


@pytest.mark.parametrize("rows, width", [(3, 64), (300, 200), (1500, 512)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_same_bits_twice_on_another_stream_and_replayed(cuda_device, rows, width, checkpoint):
    dtype = torch.bfloat16
    p = block_parameters(width, dtype, cuda_device)
    xs = [normal((rows, width), 20 + i, dtype, cuda_device) for i in range(3)]
    dys = [normal((rows, width), 30 + i, dtype, cuda_device) for i in range(3)]

    def step(x, dy):
        leaf = x.detach().requires_grad_()
        y = block(leaf, p, checkpoint)
        return [y.detach(), *torch.autograd.grad(y, [leaf, *p.values()], dy)]
    want = [step(x, dy) for x, dy in zip(xs, dys)]
    for a, b in zip(want[0], step(xs[0], dys[0])):
        assert torch.equal(a, b)
    # two streams at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([step(xs[i], dys[i]) for _ in range(5)])
    for i, s in enumerate(streams):
        torch.cuda.current_stream().wait_stream(s)
        for result in got[i]:
            for a, b in zip(want[i], result):
                assert torch.equal(a, b)
    # captured, and replayed over other inputs in the same memory, beside an eager call
    x, dy = xs[0].clone(), dys[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, dy)
    for i in (1, 2, 0):
        x.copy_(xs[i])
        dy.copy_(dys[i])
        graph.replay()
        eager = step(xs[(i + 1) % 3], dys[(i + 1) % 3])
        for a, b, c, d in zip(out, want[i], eager, want[(i + 1) % 3]):
            assert torch.equal(a, b) and torch.equal(c, d)
    check_status()


def test_offsets_beyond_32_bits(cuda_device):
    """More than 2^31 elements: the last rows of a tall tensor are what the same rows give alone."""
    rows, width = (1 << 20) + 3, 2080
    x = torch.zeros((rows, width), dtype=torch.bfloat16, device=cuda_device)
    tail = normal((5, width), 1, torch.bfloat16, cuda_device)
    x[-5:] = tail
    assert torch.equal(restore_activation(quantise_activation(x))[-5:], restore_activation(quantise_activation(tail)))
    leaf = x.requires_grad_()
    y = layer_norm(leaf)
    assert torch.equal(y[-5:], layer_norm(tail))
    dy = torch.zeros_like(y)
    dy[-5:] = normal((5, width), 2, torch.bfloat16, cuda_device)
    dx, = torch.autograd.grad(y, leaf, dy)
    small = tail.clone().requires_grad_()
    want, = torch.autograd.grad(layer_norm(small), small, dy[-5:])
    assert torch.equal(dx[-5:], want) and not dx[:-5].any()
    del y, dx, leaf, x
    # a product with so tall a result, and its gradient
    x = torch.zeros((rows, 64), dtype=torch.bfloat16, device=cuda_device)
    x[-5:] = tail[:, :64]
    w = normal((width, 64), 3, torch.bfloat16, cuda_device, 0.125).requires_grad_()
    y = linear(x, w, activation="relu", checkpoint="int8")
    want, tol, *_ = ref.linear(tail[:, :64].double(), w.detach().double(), None, None, "relu", torch.bfloat16)
    ref.assert_within(y[-5:].detach(), want, tol, "y")
    assert not y[:-5].any()
    dw, = torch.autograd.grad(y, w, dy)
    small = linear(x[-5:], w, activation="relu", checkpoint="int8")
    dw_small, = torch.autograd.grad(small, w, dy[-5:])
    # zero rows add nothing; the two calls add up in another order and may cut the sum elsewhere
    slack = 2 * (ref.product_slack(dy[-5:].double().t(), x[-5:].double().t()) + ref.half_step(dw_small.double(), torch.bfloat16))
    ref.assert_within(dw, dw_small.double(), slack, "dw")


def test_only_what_belongs_to_a_tensor_is_written(cuda_device):
    """Through the C ABI into larger buffers: a pattern around every output stays."""
    from i8muon_b200 import native
    from i8muon_b200.engine import status_word
    dtype = torch.bfloat16
    stream = torch.cuda.current_stream().cuda_stream

    def guarded(count, kind):
        flat = torch.full((count + 512,), 77, dtype=kind, device=cuda_device)
        return flat, flat[256:256 + count]

    def intact(flat, count):
        return bool((flat[:256] == 77).all() and (flat[256 + count:] == 77).all())
    for rows, width, outer in ((1, 33, 7), (5, 1001, 130), (130, 72, 257), (300, 264, 513)):
        groups, zgroups, zp = -(-width // 32), -(-outer // 32), -(-outer // 8) * 8
        x, w = normal((rows, width), 1, dtype, cuda_device), normal((outer, width), 2, dtype, cuda_device, 0.1)
        dy, dyx = normal((rows, outer), 3, dtype, cuda_device), normal((rows, width), 4, dtype, cuda_device)
        sizes = dict(codes=(rows * groups * 32, torch.uint8), exps=(rows * groups, torch.uint8), back=(rows * width, dtype), y=(rows * width, dtype),
                     dx=(rows * width, dtype), nw=(width, dtype), nb=(width, dtype), rstd=(rows, torch.float32), mean=(rows, torch.float32),
                     ly=(rows * outer, dtype), z=(rows * zp, dtype), zcodes=(rows * zgroups * 32, torch.uint8), zexps=(rows * zgroups, torch.uint8),
                     ldx=(rows * width, dtype), ldw=(outer * width, dtype), ldb=(outer, dtype))
        g = {k: guarded(*v) for k, v in sizes.items()}
        at = {k: v[1].data_ptr() for k, v in g.items()}
        status = status_word(cuda_device).data_ptr()
        native.call("i8m_activation_quant", x.data_ptr(), native.BF16, rows, width, 0, at["codes"], at["exps"], stream)
        native.call("i8m_activation_restore", at["codes"], at["exps"], rows, width, 0, at["back"], native.BF16, stream)
        native.call("i8m_layer_norm", x.data_ptr(), None, None, at["y"], at["mean"], at["rstd"], None, None, -1, rows, width, native.BF16, 1e-5, stream)
        size = native.layer_norm_scratch_bytes(rows, width)
        scratch = guarded(size, torch.uint8)
        native.call("i8m_layer_norm_backward", dyx.data_ptr(), x.data_ptr(), at["mean"], at["rstd"], None, None, -1, None, at["dx"], at["nw"], at["nb"],
                    rows, width, native.BF16, scratch[1].data_ptr(), size, stream)
        fsize = native.linear_workspace_bytes(x.data_ptr(), w.data_ptr(), rows, width, outer)
        fwork = guarded(fsize, torch.uint8)
        for z, zc, ze, fmt in ((at["z"], None, None, -1), (None, at["zcodes"], at["zexps"], 1)):
            native.call("i8m_linear", x.data_ptr(), w.data_ptr(), None, None, at["ly"], z, zc, ze, fmt, 5, rows, width, outer, native.BF16,
                        fwork[1].data_ptr(), fsize, status, stream)
        bsize = native.linear_backward_workspace_bytes(dy.data_ptr(), x.data_ptr(), w.data_ptr(), rows, width, outer, 5, -1, 1, 1, 1)
        bwork = guarded(bsize, torch.uint8)
        native.call("i8m_linear_backward", dy.data_ptr(), x.data_ptr(), None, None, w.data_ptr(), at["z"], None, None, -1, 5, at["ldx"], at["ldw"],
                    at["ldb"], rows, width, outer, native.BF16, bwork[1].data_ptr(), bsize, status, stream)
        torch.cuda.synchronize()
        check_status()
        for k, (count, _) in sizes.items():
            assert intact(g[k][0], count), (k, rows, width, outer)
        assert intact(scratch[0], size) and intact(fwork[0], fsize) and intact(bwork[0], bsize)
        assert torch.equal(g["y"][1].view(rows, width), layer_norm(x))
        assert torch.equal(g["ly"][1].view(rows, outer), linear(x, w, activation="silu"))


@pytest.mark.parametrize("rows, inner, outer", [(3, 64, 64), (3, 1024, 512), (1100, 512, 1024)])
def test_bounded_waits_run_out_and_report(cuda_device, rows, inner, outer):
    """The failure path of both product kernels, in the one way that leaves nothing in flight: the producers issue no copy,
    every other role's wait runs out after about two seconds, the status word holds a timeout code, and the same call without
    the flag is then correct."""
    from i8muon_b200 import native
    x, w = normal((rows, inner), 1, torch.bfloat16, cuda_device), normal((outer, inner), 2, torch.bfloat16, cuda_device, 0.1)
    want = linear(x, w)
    check_status()
    try:
        native.call("i8m_set_debug_core", 2)
        linear(x, w)
        with pytest.raises(native.NativeError, match="timed out"):
            check_status()
    finally:
        native.call("i8m_set_debug_core", 0)
    assert torch.equal(linear(x, w), want)
    check_status()


def test_a_first_call_on_a_device_is_not_captured(cuda_device, monkeypatch):
    from i8muon_b200 import layers
    x, w = normal((3, 64), 1, torch.bfloat16, cuda_device), normal((64, 64), 2, torch.bfloat16, cuda_device)
    monkeypatch.setattr(layers, "_STATUS_ADDRESSES", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        linear(x, w)


FRESH_THREADS = """
import threading
import torch
from i8muon_b200 import check_status, linear
x, w = (torch.full(s, 0.125, dtype=torch.bfloat16, device="cuda", requires_grad=True) for s in ((128, 256), (192, 256)))
dy = torch.ones(128, 192, dtype=torch.bfloat16, device="cuda")
spare = [torch.empty(1 << 16, device="cuda") for _ in range(8)]   # what the threads allocate is there already
y = linear(x, w)
del spare
dx, dw = torch.autograd.grad(y, (x, w), dy)        # the first work of autograd's thread of this device
assert (dx == 24).all() and (dw == 16).all() and (y == 4).all()
seen = []
def forward():
    seen.append(linear(x.detach(), w.detach()))    # the first work of a thread of the user's
thread = threading.Thread(target=forward)
thread.start()
thread.join()
torch.cuda.synchronize()
assert len(seen) == 1 and torch.equal(seen[0], y)
check_status()
"""


def test_the_first_work_of_a_thread(cuda_device):
    """A new thread has no current context before its first runtime call: a child process, for threads that are new."""
    root = pathlib.Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", FRESH_THREADS], cwd=root, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr


CAPTURED_AT_FIRST = """
import torch
from i8muon_b200 import check_status, layer_norm, linear
one = torch.ones(1, 8, dtype=torch.bfloat16, device="cuda")
linear(one, one)                                   # the device's status word; no kernel of the sizes below has run
gen = torch.Generator(device="cuda").manual_seed(1)
def leaf(*shape, std=1.0):
    return torch.randn(shape, device="cuda", generator=gen).mul_(std).bfloat16().requires_grad_()
leaves = h, nw, w1, w2 = leaf(3000, 640), leaf(640), leaf(1280, 640, std=0.04), leaf(640, 1280, std=0.03)
dy = torch.randn(3000, 640, device="cuda", generator=gen).bfloat16()
def step():
    y = linear(linear(layer_norm(h, nw, checkpoint="fp8"), w1, activation="silu", checkpoint="int8"), w2, residual=h)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
side = torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.graph(graph, stream=side):
    captured = step()
graph.replay()
torch.cuda.synchronize()
check_status()
for a, b in zip(captured, step()):
    assert torch.equal(a, b)
"""


def test_first_calls_of_kernels_under_capture(cuda_device):
    root = pathlib.Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", CAPTURED_AT_FIRST], cwd=root, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr
