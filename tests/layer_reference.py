"""The layer operators from their formulas, in 64 bits, with bounds on what 32-bit evaluation may add.

Every function works on the device of its inputs.  ``EPS`` is half a step of FP32; HALF[dtype] half a step of a type,
relative to a value.  Bounds count roundings along the longest chain of additions a kernel may use."""
import math

import torch

EPS = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half the distance between the smallest numbers of a type, which is what rounding may add near zero
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
GROUP = 32


def half_step(value, dtype):
    return value.abs() * HALF[dtype] + TINY[dtype]


def chain(width):
    """Additions behind one another in a sum over a row: what a thread adds up alone and the tree above it."""
    return width / 128 + 32


def row_chain(rows):
    """The same for sums over rows: a band of rows, the block's lanes, the bands."""
    return rows / 200 + 64


# ------------------------------------------------------------- eight-bit format
def exponents_of(x, checkpoint):
    """Exponent of every group of rows ``x`` (64 bits), by counting up from -127."""
    most = 127.0 if checkpoint == "int8" else 448.0
    pad = torch.nn.functional.pad(x, (0, -x.shape[1] % GROUP)).reshape(x.shape[0], -(-x.shape[1] // GROUP), GROUP)
    top = pad.abs().amax(-1)
    _, guess = torch.frexp(top / most)
    e = guess.double().clamp(-127, 200)
    for _ in range(3):
        e = torch.where(top > most * torch.exp2(e), e + 1, e)
    for _ in range(3):
        e = torch.where((e > -127) & (top <= most * torch.exp2(e - 1)), e - 1, e)
    return e, pad


def round_code(v, checkpoint):
    if checkpoint == "int8":
        return torch.round(v)
    _, exponent = torch.frexp(v)
    unit = torch.exp2((exponent - 1).clamp_min(-6).double() - 3)
    return torch.round(v / unit) * unit


def kept(x, checkpoint, exponent=None, dtype=torch.float32):
    """Values that the format keeps of the rows ``x`` of type ``dtype``; ``exponent`` overrides the groups' own."""
    e, pad = exponents_of(x, checkpoint)
    scale = torch.exp2(e if exponent is None else exponent).unsqueeze(-1)
    v = round_code(pad / scale, checkpoint) * scale
    below = (63.0 if checkpoint == "int8" else 240.0) * scale      # the code under the one that leaves the type
    v = torch.where(v.abs() > torch.finfo(dtype).max, torch.sign(v) * below, v)
    bad = ~torch.isfinite(pad).all(-1, keepdim=True)
    v = torch.where(bad, torch.full_like(v, math.nan), v)
    return v.reshape(x.shape[0], pad.shape[1] * GROUP)[:, :x.shape[1]]


def kept_with_slack(x, slack, checkpoint):
    """What is kept of ``x``, and how far what is kept of values up to ``slack`` away may be from that: rounding is
    monotone, so the ends of the interval decide, at the exponents that the group's largest magnitude may have."""
    v, off = kept(x, checkpoint), torch.zeros_like(x)
    for e in (exponents_of((x.abs() - slack).clamp_min(0), checkpoint)[0], exponents_of(x, checkpoint)[0],
              exponents_of(x.abs() + slack, checkpoint)[0]):
        for end in (x - slack, x + slack):
            off = torch.maximum(off, (kept(end, checkpoint, e) - v).abs())
    return v, off


# ------------------------------------------------------------------ layer norm
def layer_norm(x, w, b, eps, dtype):
    """(y, tolerance, u, tolerance of u, 1 / sigma, relative tolerance of it)."""
    n = x.shape[1]
    d = chain(n)
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    u = (x - mean) * rstd
    # the mean loses d roundings of the sum of magnitudes, the variance as many of itself and the mean's error squared
    off_mean = (d + 2) * EPS * x.abs().mean(1, keepdim=True)
    rel_rstd = (d + 6) * EPS + (off_mean * rstd).square()
    tol_u = off_mean * rstd + u.abs() * (rel_rstd + 3 * EPS)
    one, zero = torch.ones(n, dtype=x.dtype, device=x.device), torch.zeros(n, dtype=x.dtype, device=x.device)
    w, b = one if w is None else w, zero if b is None else b
    y = u * w + b
    tol = tol_u * w.abs() + 2 * EPS * ((u * w).abs() + b.abs())
    return y, tol + half_step(y.abs() + tol, dtype), u, tol_u, rstd, rel_rstd


def layer_norm_gradients(dy, u, tol_u, rstd, rel_rstd, w, dtype):
    """{name: (gradient, tolerance)} at the rows ``u`` known to ``tol_u``."""
    n, d, dr = u.shape[1], chain(u.shape[1]), row_chain(u.shape[0])
    g = dy if w is None else dy * w
    mg, mu = g.mean(1, keepdim=True), (g * u).mean(1, keepdim=True)
    off_g = (d + 3) * EPS * g.abs().mean(1, keepdim=True)
    off_u = (d + 4) * EPS * (g * u).abs().mean(1, keepdim=True) + (g.abs() * tol_u).mean(1, keepdim=True)
    raw = (g - mg - u * mu) * rstd
    tol = rstd * (off_g + (u.abs() + tol_u) * off_u + tol_u * mu.abs() + 4 * EPS * (g.abs() + mg.abs() + (u * mu).abs()))
    tol = tol + raw.abs() * (rel_rstd + 2 * EPS)
    dw, db = (dy * u).sum(0), dy.sum(0)
    tol_dw = (dr + 3) * EPS * (dy * u).abs().sum(0) + (dy.abs() * tol_u).sum(0)
    tol_db = (dr + 3) * EPS * dy.abs().sum(0)
    return {name: (v, t + half_step(v.abs() + t, dtype)) for name, v, t in
            (("dx", raw, tol), ("dw", dw, tol_dw), ("db", db, tol_db))}


def assert_within(got, want, tol, what):
    got = got.double()
    off = (got - want).abs()
    bad = ~(off <= tol)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, off / tol.clamp_min(1e-300), torch.zeros_like(off)).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst at {i}: got "
                             f"{got.flatten()[i].item():.9g}, want {want.flatten()[i].item():.9g} +- {tol.flatten()[i].item():.3g}")
