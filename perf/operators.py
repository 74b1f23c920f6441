"""The layers around the matrices that Muon steps, as cases that can be timed and compared.

Three operators, each through its public entry point:

  linear   y = act(x W^T + b) + r, and with ``train`` the gradients of x, W and b.  What the backward pass reads of the
           forward pass - x, and the pre-activation z where there is an activation - is kept in the type of x, or in
           eight bits where the case names a checkpoint format
  norm     layer norm y = (x - mean) / sqrt(var + eps) * w + b, and with ``train`` the gradients of x, w and b; with a
           checkpoint format the normalised rows are kept in eight bits and x is not kept at all
  quant    an activation written in eight bits and read back

Eight-bit format: groups of 32 consecutive elements of a row share one exponent e, the smallest integer with
max|x| <= M 2^e (M = 127 for INT8, 448 for E4M3, e >= -127); a code is x 2^-e rounded to the nearest integer or E4M3
value, ties to even, and stands for code 2^e, which every type of x holds exactly.

Sizes are those of this repository's benchmark configurations and cases, or generic ones.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
GROUP = 32
LN_EPS = 1e-5
MOST_FLOPS = 2.9e12
MOST_BYTES = 1.1e9


def _linear(name, rows, inner, outer, dtype, train=False, activation="none", bias=True, residual=False, checkpoint="none"):
    case = dict(kind="linear", rows=rows, inner=inner, outer=outer, dtype=dtype, train=train, activation=activation, bias=bias,
                residual=residual, checkpoint=checkpoint)
    return dict(case, name=name) if name else case


def _norm(name, rows, width, dtype, train=False, checkpoint="none", shift=0.0):
    case = dict(kind="norm", rows=rows, width=width, dtype=dtype, train=train, checkpoint=checkpoint, shift=shift)
    return dict(case, name=name) if name else case


def _quant(name, rows, width, dtype, checkpoint):
    case = dict(kind="quant", rows=rows, width=width, dtype=dtype, checkpoint=checkpoint)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token through a projection of an 8B-shaped model: reading the weights is all there is
        _linear("linear-token-bf16", 1, 4096, 4096, "bf16", bias=False),
        # a handful of sequences, one token each, through the widening projection of the same model
        _linear("linear-tokens-fp16", 16, 4096, 14336, "fp16", activation="gelu_tanh"),
        # evaluation of a 1.3B-shaped model on a batch of prompts
        _linear("linear-prompt-bf16", 8192, 2048, 8192, "bf16", activation="gelu"),
        # a training step of a 768-wide block on one short sequence: launches and tails count
        _linear("linear-train-768-bf16", 1024, 768, 768, "bf16", train=True, activation="silu"),
        # sizes that fit no tile (a pruned or factorised layer), residual in the epilogue
        _linear("linear-train-ragged-fp16", 333, 1001, 517, "fp16", train=True, activation="gelu", residual=True),
        # an attention output projection in training: residual, input kept in E4M3
        _linear("linear-train-fp8-bf16", 4096, 2048, 2048, "bf16", train=True, residual=True, checkpoint="fp8"),
        # the widening projection of an 8B-shaped model in training, input and pre-activation kept in INT8: the largest
        _linear("linear-train-int8-bf16", 8192, 4096, 14336, "bf16", train=True, activation="relu2", bias=False,
                checkpoint="int8"),
        # one token of a small model: the smallest call
        _norm("norm-token-bf16", 1, 768, "bf16"),
        # a training batch of an 8B-shaped model
        _norm("norm-train-bf16", 16384, 4096, "bf16", train=True),
        # rows that fit no vector, normalised rows kept in INT8, values far from zero
        _norm("norm-train-ragged-int8-fp16", 3001, 1531, "fp16", train=True, checkpoint="int8", shift=4.0),
        # a training batch's activations through the eight-bit format
        _quant("quant-int8-bf16", 16384, 4096, "bf16", "int8"),
        # full precision, rows that fit no vector
        _quant("quant-ragged-fp8-fp32", 1000, 3001, "fp32", "fp8"),
    ]


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def _size(rng, low, high):
    """A size of the range: a multiple of 64 as models have them, or (one in three) whatever it is."""
    v = _log_uniform(rng, low, high)
    return max(low, min(high, int(v) if rng.random() < 1 / 3 else 64 * max(1, round(v / 64))))


def draw(rng):
    while True:
        kind = rng.random()
        if kind < 0.6:
            train = rng.random() < 0.6
            case = _linear("", int(_log_uniform(rng, 1, 16384)), _size(rng, 32, 8192), _size(rng, 32, 14336),
                           rng.choice(("bf16", "bf16", "fp16")), train=train,
                           activation=rng.choice(("none", "none", "relu", "relu2", "gelu", "gelu_tanh", "silu")),
                           bias=rng.random() < 0.6, residual=rng.random() < 0.4,
                           checkpoint=rng.choice(("none", "int8", "fp8")) if train else "none")
        elif kind < 0.85:
            train, dtype = rng.random() < 0.7, rng.choice(("bf16", "bf16", "fp16", "fp32"))
            # codes of normalised rows: a last-place difference of a row's mean moves some value across a border between two
            # codes, which no 32-bit evaluation can be held to at the precision of FP32 gradients
            checkpoint = rng.choice(("none", "int8", "fp8")) if train and dtype != "fp32" else "none"
            case = _norm("", int(_log_uniform(rng, 1, 32768)), _size(rng, 16, 16384), dtype, train=train, checkpoint=checkpoint,
                         shift=rng.choice((0.0, 0.0, 0.5, 4.0)))
        else:
            case = _quant("", int(_log_uniform(rng, 1, 32768)), _size(rng, 16, 16384), rng.choice(("bf16", "fp16", "fp32")),
                          rng.choice(("int8", "fp8")))
        cost = work(case)
        if cost["flops"] <= MOST_FLOPS and cost["bytes"] <= MOST_BYTES:
            return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(shape, std, mean=0.0):
        return torch.randn(shape, device="cuda", generator=gen).mul_(std).add_(mean).to(dtype)

    def activations(rows, width, shift=0.0):
        """Unit rows in which some channels are ten times larger, as the residual stream of a trained model has them."""
        channel = torch.rand(width, device="cuda", generator=gen).lt_(0.01).mul_(9.0).add_(1.0)
        return torch.randn((rows, width), device="cuda", generator=gen).mul_(channel).add_(shift).to(dtype)

    state = dict(case=case)
    if case["kind"] == "quant":
        return dict(state, x=activations(case["rows"], case["width"]))
    if case["kind"] == "norm":
        rows, width = case["rows"], case["width"]
        state.update(x=activations(rows, width, case["shift"]), w=normal((width,), 0.1, 1.0), b=normal((width,), 0.1),
                     dy=normal((rows, width), 1e-2) if case["train"] else None)
    else:
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        state.update(x=normal((rows, inner), 1.0), w=normal((outer, inner), inner ** -0.5),
                     b=normal((outer,), 0.1) if case["bias"] else None,
                     r=normal((rows, outer), 1.0) if case["residual"] else None,
                     dy=normal((rows, outer), 1e-2) if case["train"] else None)
    if case["train"]:
        for name in ("x", "w", "b"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# ----------------------------------------------------------------- plain forms
def _activation(z, name):
    """The activation and its derivative at z."""
    if name == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if name == "relu2":
        p = z.clamp_min(0)
        return p * p, 2 * p
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        phi = torch.erfc(z * -(0.5 ** 0.5)) * 0.5
        return z * phi, phi + z * torch.exp(z * z * -0.5) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        s = torch.sigmoid(2 * c * (z + 0.044715 * z * z * z))
        return z * s, s + z * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _power(e):
    """2^e as a float, exactly, for -127 <= e <= 127."""
    normal = ((e.clamp_min(-126) + 127) << 23).to(torch.int32).view(torch.float32)
    return torch.where(e < -126, normal * 0.5, normal)


def _kept(v, checkpoint):
    """The values that the eight-bit format keeps of the rows v (32 bits)."""
    rows, width = v.shape
    groups = -(-width // GROUP)
    p = torch.zeros((rows, groups * GROUP), dtype=v.dtype, device=v.device)
    p[:, :width] = v
    p = p.view(rows, groups, GROUP)
    most, bits = (127.0, 7) if checkpoint == "int8" else (448.0, 9)
    mantissa, exponent = torch.frexp(p.abs().amax(2, keepdim=True))
    e = (exponent - bits + (mantissa > most / 2 ** bits)).clamp_min(-127)
    e = torch.where(mantissa == 0, torch.full_like(e, -127), e)
    scaled = p * _power(-e)
    codes = scaled.round() if checkpoint == "int8" else scaled.to(torch.float8_e4m3fn).to(v.dtype)
    return (codes * _power(e)).view(rows, -1)[:, :width]


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["w"].detach().float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    y = _activation(z, case["activation"])[0]
    if s["r"] is not None:
        y = y + s["r"].float()
    out = dict(y=y.to(dtype))
    if case["train"]:
        dz = s["dy"].float()
        if case["activation"] != "none":
            kept = z.to(dtype).float() if case["checkpoint"] == "none" else _kept(z, case["checkpoint"])
            dz = dz * _activation(kept, case["activation"])[1]
        kept = x if case["checkpoint"] == "none" else _kept(x, case["checkpoint"])
        out.update(dx=(dz @ w).to(dtype), dw=(dz.t() @ kept).to(dtype))
        if s["b"] is not None:
            out["db"] = dz.sum(0).to(dtype)
    return out


def _plain_norm(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["w"].detach().float()
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + LN_EPS)
    unit = centred * rstd
    out = dict(y=(unit * w + s["b"].detach().float()).to(dtype))
    if case["train"]:
        if case["checkpoint"] != "none":
            unit = _kept(unit, case["checkpoint"])
        dy = s["dy"].float()
        g = dy * w
        dx = (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True)) * rstd
        out.update(dx=dx.to(dtype), dw=(dy * unit).sum(0).to(dtype), db=dy.sum(0).to(dtype))
    return out


def run(state):
    case = state["case"]
    if not own:
        if case["kind"] == "quant":
            return _kept(state["x"].float(), case["checkpoint"]).to(state["x"].dtype)
        return _plain_linear(state) if case["kind"] == "linear" else _plain_norm(state)
    from i8muon_b200 import layer_norm, linear, quantise_activation, restore_activation
    if case["kind"] == "quant":
        return restore_activation(quantise_activation(state["x"], case["checkpoint"]))
    checkpoint = None if case["checkpoint"] == "none" else case["checkpoint"]
    if case["kind"] == "norm":
        y = layer_norm(state["x"], state["w"], state["b"], LN_EPS, checkpoint=checkpoint)
    else:
        y = linear(state["x"], state["w"], state["b"], activation=None if case["activation"] == "none" else case["activation"],
                   residual=state["r"], checkpoint=checkpoint)
    if not case["train"]:
        return dict(y=y)
    names = [name for name in ("x", "w", "b") if state[name] is not None]
    gradients = torch.autograd.grad(y, [state[name] for name in names], state["dy"])
    return dict(y=y.detach(), **{"d" + name: g for name, g in zip(names, gradients)})


# ------------------------------------------------------- the definition in 64 bits
def _two_to(e):
    """2^e in 64 bits, by its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_rounded(v, checkpoint):
    """Nearest eight-bit value by definition: magnitudes in units of the last place, ties to even."""
    if checkpoint == "int8":
        return torch.round(v)
    _, exponent = torch.frexp(v)                              # |v| in [2^(exponent-1), 2^exponent)
    unit = _two_to((exponent - 1).clamp_min(-6) - 3)          # three mantissa bits, subnormals below 2^-6
    return torch.round(v / unit) * unit


def _exact_kept(v, checkpoint):
    most = 127.0 if checkpoint == "int8" else 448.0
    kept = torch.nn.functional.pad(v, (0, -v.shape[1] % GROUP)).reshape(v.shape[0], -1, GROUP)
    e = torch.ceil(torch.log2(kept.abs().amax(-1) / most)).clamp(-127, 127)
    scale = _two_to(torch.where(torch.isfinite(e), e, torch.full_like(e, -127.0))).unsqueeze(-1)
    top = kept.abs().amax(-1, keepdim=True)
    scale = torch.where(top > most * scale, 2 * scale, scale)           # the logarithm may be off by a rounding
    scale = torch.where((top <= most * scale / 2) & (scale > 2.0 ** -127), scale / 2, scale)
    return (_exact_rounded(kept / scale, checkpoint) * scale).reshape(v.shape[0], -1)[:, :v.shape[1]]


def _exact_act(z, name):
    if name == "none":
        return z, None
    if name in ("relu", "relu2"):
        p = torch.relu(z)
        return (p, torch.heaviside(z, torch.zeros_like(z))) if name == "relu" else (p ** 2, 2 * p)
    if name == "gelu":
        cdf, pdf = torch.special.ndtr(z), torch.exp(-0.5 * z ** 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf
    if name == "silu":
        gate = 1 / (1 + torch.exp(-z))
        return z * gate, gate + z * gate * (1 - gate)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t ** 2) * k * (1 + 0.134145 * z ** 2)


def exact(case, seed):
    s = prepare(case, seed)
    dtype = s["x"].dtype
    with torch.no_grad():
        x = s["x"].double()
        if case["kind"] == "quant":
            return _exact_kept(x, case["checkpoint"])
        w, b = s["w"].double(), None if s["b"] is None else s["b"].double()
        if case["kind"] == "norm":
            var, mean = torch.var_mean(x, dim=1, keepdim=True, correction=0)
            sigma = torch.sqrt(var + LN_EPS)
            unit = (x - mean) / sigma
            out = dict(y=unit * w + b)
            if case["train"]:
                if case["checkpoint"] != "none":
                    unit = _exact_kept(unit, case["checkpoint"])
                dy = s["dy"].double()
                width = x.shape[1]
                dunit = dy * w
                inner = dunit.sum(1, keepdim=True) + unit * (dunit * unit).sum(1, keepdim=True)
                out.update(dx=(width * dunit - inner) / (width * sigma), dw=(dy * unit).sum(0), db=dy.sum(0))
            return out
        z = torch.nn.functional.linear(x, w, b)
        y = _exact_act(z, case["activation"])[0]
        out = dict(y=y if s["r"] is None else y + s["r"].double())
        if case["train"]:
            dz = s["dy"].double()
            eight = case["checkpoint"] != "none"
            if case["activation"] != "none":
                z = _exact_kept(z, case["checkpoint"]) if eight else z.to(dtype).double()
                dz = dz * _exact_act(z, case["activation"])[1]
            out.update(dx=torch.mm(dz, w), dw=torch.mm(dz.t(), _exact_kept(x, case["checkpoint"]) if eight else x))
            if b is not None:
                out["db"] = dz.sum(0)
        return out


def work(case):
    """Flops: the products, one forward and two backward.  Bytes: every input and every output once, and what the
    forward pass keeps written once and read once."""
    size = SIZES[case["dtype"]]
    eight = 1.0 + 1.0 / GROUP          # bytes of an element in the eight-bit format
    if case["kind"] == "quant":
        n = float(case["rows"]) * case["width"]
        return {"bytes": n * (2 * size + 2 * eight), "flops": 2 * n}
    if case["kind"] == "norm":
        n = float(case["rows"]) * case["width"]
        total, flops = n * 2 * size + 2.0 * size * case["width"], 8 * n
        if case["train"]:
            # dy in, dx out, dw and db out; the backward pass reads x again, or the codes that the forward pass wrote
            total += n * 2 * size + 2.0 * size * case["width"] + n * (size if case["checkpoint"] == "none" else 2 * eight)
            flops += 14 * n
        return {"bytes": total, "flops": flops}
    rows, inner, outer = float(case["rows"]), float(case["inner"]), float(case["outer"])
    total = size * (rows * inner + outer * inner + rows * outer * (2 if case["residual"] else 1) + (outer if case["bias"] else 0))
    flops = 2 * rows * inner * outer
    if case["train"]:
        kept = size if case["checkpoint"] == "none" else eight
        # dy and W in, dx, dW and db out; the kept input is read (and written, unless it is x itself), and z is written and read
        total += size * (rows * outer + 2 * outer * inner + rows * inner + (outer if case["bias"] else 0))
        total += rows * inner * (kept if case["checkpoint"] == "none" else 2 * kept)
        total += 2 * rows * outer * kept if case["activation"] != "none" else 0.0
        flops *= 3
    return {"bytes": total, "flops": flops}
