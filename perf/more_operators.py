"""Measured cases of the 8-bit operators of a decoder layer.

Four operators that together run a layer's projections in 8-bit integers, with
one scale per token and one per output channel:

  norm     residual addition and root-mean-square norm, written as 8-bit
           integers with a scale per token; the sum is kept in 16 bits
  silu     silu(gate) * up, written as 8-bit integers with a scale per token
  quantize a 16-bit tensor (the attention's output) as 8-bit integers with a
           scale per token
  linear   matrix product of such tokens with 8-bit weights, scaled by token
           and channel

The scale of a row is its largest magnitude / 127, an element's integer the
nearest to 127 times it over that magnitude (halves to even).  What is held in 8 bits is
returned as the values it stands for, in the inputs' type (the framework's
kernel for that is part of the pass).

A case is a dict of plain values.  ``run`` computes the operators in their
plain form, or calls the framework's when ``own`` is set.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5


def listed():
    return [
        # decode step of one request: launch latency
        dict(name="norm 1 token", kind="norm", tokens=1, k=4096, residual=True, dtype="bf16"),
        # a full prefill step
        dict(name="norm prompt", kind="norm", tokens=8192, k=5120, residual=True, dtype="bf16"),
        # the first layer's norm (nothing to add), a ragged step, rows that end inside every vector
        dict(name="norm odd", kind="norm", tokens=333, k=2047, residual=False, dtype="fp16"),
        # a decode batch: the halves of a merged gate and up projection
        dict(name="silu batch", kind="silu", tokens=48, k=13824, dtype="bf16"),
        # a full prefill step
        dict(name="silu prompt", kind="silu", tokens=8192, k=14336, dtype="bf16"),
        # attention output of a decode batch
        dict(name="quantize batch", kind="quantize", tokens=64, k=4096, dtype="bf16"),
        # attention output of a full prefill step
        dict(name="quantize prompt", kind="quantize", tokens=16384, k=5120, dtype="fp16"),
        # queries, keys and values of one request's token: launch latency and the weights' bytes
        dict(name="linear 1 token", kind="linear", tokens=1, k=4096, n=6144, bias=False, dtype="bf16"),
        # gate and up of a decode batch: the weights' bytes
        dict(name="linear batch", kind="linear", tokens=64, k=5120, n=27648, bias=False, dtype="bf16"),
        # a mixed step of prompts' chunks and decodes, a ragged number of tokens
        dict(name="linear mixed", kind="linear", tokens=306, k=5120, n=5120, bias=True, dtype="fp16"),
        # gate and up of a full prefill step: the tensor cores
        dict(name="linear prompt", kind="linear", tokens=8192, k=4096, n=28672, bias=False, dtype="bf16"),
        # logits of a decode batch over a large vocabulary
        dict(name="linear logits", kind="linear", tokens=16, k=4096, n=128256, bias=False, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, int(lo * math.exp(rng.random() * math.log((hi + 1) / lo))))


def draw(rng):
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["kind"], {"bytes": 0.0, "flops": 0.0})
        for k in m:
            m[k] = max(m[k], w[k])
    while True:
        kind = rng.choice(["norm", "silu", "quantize", "linear", "linear", "linear"])
        c = dict(kind=kind, tokens=_log(rng, 1, 16384), dtype=rng.choice(["bf16", "bf16", "fp16"]))
        # widths of all kinds: whole vectors and blocks, and odd ones
        unit = rng.choice([1, 8, 16, 128, 128])
        c["k"] = unit * max(1, _log(rng, 64, 16384) // unit)
        if kind == "norm":
            c["residual"] = rng.random() < 0.7
        if kind == "linear":
            unit = rng.choice([1, 8, 64, 128, 128])
            c.update(n=unit * max(1, _log(rng, 64, 131072) // unit), bias=rng.random() < 0.3,
                     dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        w = work(c)
        if all(w[k] <= most[kind][k] for k in w):
            return c


def work(c):
    t, k, el = c["tokens"], c["k"], BYTES[c["dtype"]]
    if c["kind"] == "norm":
        # in: x, the norm's weights, the residual; out: the values, the scales, the sum
        return {"bytes": float(t * k * el * (4 if c["residual"] else 2) + k * el + 4 * t), "flops": 8.0 * t * k}
    if c["kind"] == "silu":
        return {"bytes": float(3 * t * k * el + 4 * t), "flops": 9.0 * t * k}
    if c["kind"] == "quantize":
        return {"bytes": float(2 * t * k * el + 4 * t), "flops": 3.0 * t * k}
    n = c["n"]
    return {"bytes": float(t * k + n * k + 4 * (t + n) + t * n * el + (n * el if c["bias"] else 0)),
            "flops": 2.0 * t * k * n}


# ------------------------------------------------------------------- inputs
def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rows(x):
    """The rows of x (32 bits) as 8-bit integers, and their scales."""
    s = x.abs().amax(1) / 127
    return (x / s[:, None]).round().to(torch.int8), s


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, k, dt = c["tokens"], c["k"], DTYPES[c["dtype"]]
    s = dict(c=c)
    # activations: tokens of different size, and a few channels that stand out
    size = 0.5 + torch.rand(t, 1, generator=g, device=DEV)
    loud = torch.where(torch.rand(k, generator=g, device=DEV) < 0.005, 12.0, 1.0)
    if c["kind"] == "norm":
        s["x"] = (_rand(g, t, k) * size).to(dt)
        s["residual"] = (_rand(g, t, k) * size * loud).to(dt) if c["residual"] else None
        s["weight"] = (1 + 0.1 * _rand(g, k)).to(dt)
    elif c["kind"] == "silu":
        # the halves of one projection's output: strided views
        s["merged"] = (_rand(g, t, 2 * k) * size).to(dt)
        s["gate"], s["up"] = s["merged"][:, :k], s["merged"][:, k:]
    elif c["kind"] == "quantize":
        s["x"] = (_rand(g, t, k) * size * loud).to(dt)
    else:
        s["q"], s["scales"] = _rows(_rand(g, t, k) * size * loud)
        s["weight_q"] = torch.empty(c["n"], k, dtype=torch.int8, device=DEV)
        s["weight_scales"] = torch.empty(c["n"], device=DEV)
        for i in range(0, c["n"], 16384):
            s["weight_q"][i:i + 16384], s["weight_scales"][i:i + 16384] = _rows(
                _rand(g, min(16384, c["n"] - i), k) * 0.02)
        s["bias"] = (0.1 * _rand(g, c["n"])).to(dt) if c["bias"] else None
    if own:
        _handle(s)
    return s


def _handle(s):
    """What a program keeps of a projection's weights."""
    from kunserve_b200 import ops
    if "weight_q" in s:
        s["handle"] = ops.Int8Weight(s["weight_q"], s["weight_scales"])


# ------------------------------------------------------------- plain forms
def _through_8_bits(y, dt):
    """The values that the rows of y (32 bits) stand for in 8 bits, and the scales."""
    top = y.abs().amax(1, keepdim=True)
    scale = top / 127
    q = torch.round(127 * y / torch.where(top > 0, top, 1.0))     # the product first: halves stay halves
    return (q * scale).to(dt), scale[:, 0]


def _norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"].float()
    out = _through_8_bits(y, s["x"].dtype)
    return out if s["residual"] is None else out + (h.to(s["x"].dtype),)


def _silu(s):
    g = s["gate"].float()
    return _through_8_bits(g / (1 + torch.exp(-g)) * s["up"].float(), s["gate"].dtype)


def _quantize(s):
    return _through_8_bits(s["x"].float(), s["x"].dtype)


def _linear(s):
    y = s["q"].float() @ s["weight_q"].float().t() * s["scales"][:, None] * s["weight_scales"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["c"]["dtype"]])


PLAIN = {"norm": _norm, "silu": _silu, "quantize": _quantize, "linear": _linear}


# --------------------------------------------------------- the framework's
def _own(s):
    from kunserve_b200 import ops
    kind, dt = s["c"]["kind"], DTYPES[s["c"]["dtype"]]
    if kind == "linear":
        return ops.int8_linear(s["q"], s["scales"], s["handle"], bias=s["bias"], dtype=dt)
    if kind == "norm":
        q, scales, total = ops.add_rms_norm_int8(s["x"], s["weight"], EPS, residual=s["residual"])
        out = ops.dequantize_int8(q, scales, dt), scales
        return out if s["residual"] is None else out + (total,)
    if kind == "silu":
        q, scales = ops.silu_mul_int8(s["gate"], s["up"])
    else:
        q, scales = ops.quantize_int8(s["x"])
    return ops.dequantize_int8(q, scales, dt), scales


def run(s):
    if own:
        return _own(s)
    return PLAIN[s["c"]["kind"]](s)


# ------------------------------------------------------------------- exact
def exact(c, seed):
    """What ``run`` returns, in 64 bits from the definitions."""
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    f64 = torch.float64
    if c["kind"] == "linear":
        y = torch.einsum("tk,nk->tn", s["q"].to(f64), s["weight_q"].to(f64))
        y.mul_(torch.outer(s["scales"].to(f64), s["weight_scales"].to(f64)))
        return y if s["bias"] is None else y.add_(s["bias"].to(f64))
    total = None
    if c["kind"] == "norm":
        total = s["x"].to(f64) if s["residual"] is None else torch.add(s["x"].to(f64), s["residual"].to(f64))
        y = s["weight"].to(f64) * total / torch.sqrt(total.square().sum(1) / c["k"] + EPS).unsqueeze(1)
    elif c["kind"] == "silu":
        y = s["up"].to(f64) * s["gate"].to(f64) * torch.special.expit(s["gate"].to(f64))
    else:
        y = s["x"].to(f64)
    top = torch.maximum(y.max(1).values, -y.min(1).values).unsqueeze(1)
    step = top / 127
    values = torch.where(top > 0, y.mul(127).div_(top).round_() * step, 0.0)
    if c["kind"] == "norm" and s["residual"] is not None:
        return values, step[:, 0], total
    return values, step[:, 0]
