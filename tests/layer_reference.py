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


# ---------------------------------------------------------------------- linear
def activation(z, name):
    """The activation, its derivative and (a bound on) the slope of that."""
    zero, one = torch.zeros_like(z), torch.ones_like(z)
    if name is None:
        return z, one, zero
    if name == "relu":
        return z.clamp_min(0), (z > 0).double(), zero
    if name == "relu2":
        return z.clamp_min(0).square(), 2 * z.clamp_min(0), 2 * one
    if name == "silu":
        s = torch.sigmoid(z)
        ds = s * (1 - s)
        return z * s, s + z * ds, 2 * ds + z * ds * (1 - 2 * s)
    if name == "gelu":
        cdf, pdf = torch.special.ndtr(z), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf, pdf * (2 - z * z)
    c, k = math.sqrt(2 / math.pi), 0.044715
    u, du, ddu = c * (z + k * z ** 3), c * (1 + 3 * k * z * z), 6 * c * k * z
    t = torch.tanh(u)
    dt = (1 - t * t) * du
    return z * (1 + t) / 2, (1 + t) / 2 + z * dt / 2, dt + z / 2 * ((1 - t * t) * ddu - 2 * t * dt * du)


def activation_slack(z, name):
    """What evaluating an activation and its derivative in FP32 may lose: a few roundings, an exponential whose argument is
    no larger than 1 + z^2 and rounded relative to itself, a quotient, and a published approximation's last places - 32
    roundings per unit of the argument, of the terms that are added up."""
    y, d1, _ = activation(z, name)
    if name is None:
        return torch.zeros_like(z), torch.zeros_like(z)
    gate = torch.where(z == 0, torch.full_like(z, 0.5), y / z)
    unit = 32 * EPS * (1 + z * z)
    return unit * y.abs(), unit * (gate.abs() + d1.abs())


def product_slack(a, b):
    """What a product a b^T with FP32 accumulation of 16 terms at a time may lose: each instruction's sum is truncated,
    two units in the last place of at most the sum of magnitudes; splitting the sum adds a few roundings."""
    return (a.shape[1] / 16 + 24) * 4 * EPS * (a.abs() @ b.abs().t())


def linear(x, w, b, r, name, dtype):
    """(y, tolerance, z, tolerance of z)."""
    z = x @ w.t() + (0 if b is None else b)
    tol_z = product_slack(x, w) + 2 * EPS * z.abs()
    y, d1, _ = activation(z, name)
    # the derivatives are bounded over the interval by their values and the next derivative's change
    slope = d1.abs() + 3 * tol_z
    if name == "relu":
        slope = torch.ones_like(z)
    tol = tol_z * slope + activation_slack(z, name)[0]
    if r is not None:
        tol = tol + 2 * EPS * (y.abs() + r.abs())
        y = y + r
    return y, tol + half_step(y.abs() + tol, dtype), z, tol_z


def rounded_with_slack(z, slack, dtype):
    """z rounded to a type, and how far the rounding of values up to ``slack`` away may be from that."""
    v = z.to(dtype).double()
    return v, torch.maximum((z + slack).to(dtype).double() - v, v - (z - slack).to(dtype).double())


def linear_gradients(dy, x, w, kept_z, off_z, name, dtype):
    """{name: (gradient, tolerance)} at the kept rows x and a kept pre-activation known to ``off_z``."""
    _, d1, d2 = activation(kept_z, name)
    dz = dy * d1
    if name is None:
        off = torch.zeros_like(dz)
        exact = dz
    else:
        # relu's derivative may differ where z is on either side of zero
        flip = ((kept_z.abs() <= off_z) & (off_z > 0)).double() if name == "relu" else 0
        off = dy.abs() * (activation_slack(kept_z, name)[1] + off_z * (d2.abs() + 3 * off_z) + flip)
        exact = dz
        off_rounded = off + half_step(dz.abs() + off, dtype)
    rounded = off if name is None else off_rounded
    dx, dw, db = exact @ w, exact.t() @ x, exact.sum(0)
    tol_dx = rounded @ w.abs() + product_slack(exact.abs() + rounded, w.t())
    tol_dw = rounded.t() @ x.abs() + product_slack((exact.abs() + rounded).t(), x.t())
    tol_db = off.sum(0) + (row_chain(dy.shape[0]) + 3) * EPS * exact.abs().sum(0)
    return {key: (v, t + half_step(v.abs() + t, dtype)) for key, v, t in
            (("dx", dx, tol_dx), ("dw", dw, tol_dw), ("db", db, tol_db))}


def assert_within(got, want, tol, what):
    got = got.double()
    off = (got - want).abs()
    bad = ~(off <= tol)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, off / tol.clamp_min(1e-300), torch.zeros_like(off)).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst at {i}: got "
                             f"{got.flatten()[i].item():.9g}, want {want.flatten()[i].item():.9g} +- {tol.flatten()[i].item():.3g}")
