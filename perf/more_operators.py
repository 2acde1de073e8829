"""Performance cases of the linear layers of a generating transformer in 8-bit floating point (e4m3, fp32 scales a block of 128).

Kinds
  norm     root-mean-square norm of a row plus its residual; the result in 8 bits with a scale for every 128 channels, or in 16
  rows     rows (or silu(gate) * up of them) to 8 bits with a scale for every 128 channels; weights to 8 bits with a scale for every 128 x 128
  linear   product of such rows with such weights

`listed()` names twelve of them, `draw()` gives more over the same ranges, odd sizes among them.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
BLOCK = 128
TOP = 448.0              # the largest e4m3
LEAST = 2.0 ** -126      # the smallest scale
EPS = 1e-6


def listed():
    return [
        # one new token in front of a projection: the latency of a call
        dict(name="norm_bf16_one", kind="norm", dtype="bf16", tokens=1, channels=4096, residual=True, f8=True),
        # a long prompt in front of a projection
        dict(name="norm_bf16_prompt", kind="norm", dtype="bf16", tokens=8191, channels=4096, residual=True, f8=True),
        # the last norm of a batch, in front of 16-bit consumers, a width that 128 does not divide
        dict(name="norm_f16_ragged", kind="norm", dtype="f16", tokens=300, channels=5000, residual=True, f8=False),
        # what stands between the two products of a feed-forward layer, in a decoding step
        dict(name="rows_bf16_gated_step", kind="rows", form="gated", dtype="bf16", tokens=32, channels=11008),
        # the same for a prompt
        dict(name="rows_bf16_gated_prompt", kind="rows", form="gated", dtype="bf16", tokens=4001, channels=11008),
        # attention's result in front of the output projection
        dict(name="rows_f16_prompt", kind="rows", form="plain", dtype="f16", tokens=8192, channels=4096),
        # weights of a model that is being loaded
        dict(name="rows_f32_weights", kind="rows", form="weights", dtype="f32", tokens=11008, channels=4096),
        # q, k and v of one new token: 32 + 8 + 8 heads of 128
        dict(name="linear_bf16_one", kind="linear", dtype="bf16", rows=1, outputs=6144, channels=4096, bias=True),
        # gate and up of a decoding batch
        dict(name="linear_bf16_b32", kind="linear", dtype="bf16", rows=32, outputs=22016, channels=4096, bias=False),
        # logits of a few sequences: an odd number of words, a width that 128 does not divide
        dict(name="linear_f32_logits", kind="linear", dtype="f32", rows=5, outputs=32003, channels=4000, bias=False),
        # the second product of a feed-forward layer, a short prompt
        dict(name="linear_f16_b300", kind="linear", dtype="f16", rows=300, outputs=4096, channels=11008, bias=False),
        # gate and up of a long prompt
        dict(name="linear_bf16_prompt", kind="linear", dtype="bf16", rows=8192, outputs=22016, channels=4096, bias=False),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):      # most widths are multiples of 128, some of 8, some of nothing
        n, step = spread(lo, hi), rng.choice([128, 128, 128, 8, 1])
        return max(1, n // step) * step

    kind = rng.choice(["norm", "rows", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    while True:
        if kind == "norm":
            c = dict(kind=kind, dtype=dtype, tokens=spread(1, 16384), channels=width(64, 16384), residual=rng.random() < 0.7, f8=rng.random() < 0.7)
            if c["tokens"] * c["channels"] <= 8192 * 4096:
                return c
        elif kind == "rows":
            c = dict(kind=kind, form=rng.choice(["plain", "gated", "weights"]), dtype=dtype, tokens=spread(1, 22016), channels=width(64, 22016))
            if c["tokens"] * c["channels"] <= 4096 * 11008:
                return c
        else:
            c = dict(kind=kind, dtype=dtype, rows=spread(1, 8192), outputs=width(64, 32768), channels=width(64, 16384), bias=rng.random() < 0.3)
            if c["rows"] * c["outputs"] * c["channels"] <= 8192 * 22016 * 4096 and c["outputs"] * c["channels"] <= 22016 * 8192:
                return c


def _blocks(n):
    return -(-n // BLOCK)


def _f8_tensor(x, scale):
    """e4m3 of x / scale in rows that lie a multiple of 16 bytes apart"""
    rows, n = x.shape
    q = torch.zeros((rows, -(-n // 16) * 16), dtype=F8, device="cuda")[:, :n]
    q.copy_((x / scale).clamp(-TOP, TOP))
    return q


def _spread_out(scale, rows, n, tall):
    """a scale for each element: [rows, n] of [.., blocks]"""
    scale = scale.repeat_interleave(BLOCK, 1)[:, :n]
    return scale.repeat_interleave(BLOCK, 0)[:rows] if tall else scale


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    n = c["channels"]
    size = torch.exp(0.5 * randn(n)) * torch.where(torch.rand(n, generator=g, device="cuda") < 0.005, 20.0, 1.0)   # channels differ, a few stand out
    s = dict(c=c)
    if c["kind"] == "norm":
        dtype = DTYPES[c["dtype"]]
        s["x"] = (randn(c["tokens"], n) * size).to(dtype)
        s["residual"] = (2.0 * randn(c["tokens"], n) * size).to(dtype) if c["residual"] else None
        s["weight"] = 0.5 + torch.rand(n, generator=g, device="cuda")
    elif c["kind"] == "rows":
        dtype = DTYPES[c["dtype"]]
        if c["form"] == "weights":
            s["x"] = (0.02 * randn(c["tokens"], n)).to(dtype)
        elif c["form"] == "gated":     # the rows of one product: gate, then up
            s["x"] = (randn(c["tokens"], 2 * n) * torch.cat([size.clamp(max=4.0), size])).to(dtype)
        else:
            s["x"] = (randn(c["tokens"], n) * size).to(dtype)
    else:
        x = randn(c["rows"], n) * size
        scale = torch.nn.functional.pad(x.abs(), (0, -n % BLOCK)).unflatten(1, (-1, BLOCK)).amax(-1) / TOP
        s["a"], s["a_scale"] = _f8_tensor(x, _spread_out(scale, c["rows"], n, False)), scale.contiguous()
        w = 0.02 * randn(c["outputs"], n)
        tall = torch.nn.functional.pad(w.abs(), (0, -n % BLOCK, 0, -c["outputs"] % BLOCK)).unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK)).amax((1, 3)) / TOP
        s["w"], s["w_scale"] = _f8_tensor(w, _spread_out(tall, c["outputs"], n, True)), tall.contiguous()
        s["bias"] = 0.1 * randn(c["outputs"]) if c["bias"] else None
    return s


# ---- the operators as a user of the framework calls them ----------------------------------------------------------

def _run_own(s):
    from onenew_amd import hip
    c = s["c"]
    if c["kind"] == "norm":
        return hip.rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"], f8=c["f8"])
    if c["kind"] == "rows":
        if c["form"] == "weights":
            return hip.f8_from_weights(s["x"])
        return hip.f8_from_rows(s["x"], gated=c["form"] == "gated")
    return hip.linear_f8(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"], dtype=DTYPES[c["dtype"]])


# ---- the plain form: elementary operations in 32 bits --------------------------------------------------------------

def _plain_f8(y, tall=False):
    """y [rows, n] in 32 bits -> e4m3 values and the scales of blocks of 128, or of 128 x 128"""
    rows, n = y.shape
    wide = torch.nn.functional.pad(y.abs(), (0, -n % BLOCK, 0, -rows % BLOCK if tall else 0)).unflatten(1, (-1, BLOCK))
    top = wide.unflatten(0, (-1, BLOCK)).amax((1, 3)) if tall else wide.amax(-1)
    scale = (top / TOP).clamp(min=LEAST)
    return (y / _spread_out(scale, rows, n, tall)).clamp(-TOP, TOP).to(F8), scale


def _plain_norm(s):
    c = s["c"]
    h = s["x"].float()
    if c["residual"]:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"]
    out = _plain_f8(y) if c["f8"] else (y.to(s["x"].dtype),)
    out = out + ((h.to(s["x"].dtype),) if c["residual"] else ())
    return out if len(out) > 1 else out[0]


def _plain_rows(s):
    c = s["c"]
    x = s["x"].float()
    if c["form"] == "gated":
        gate, up = x[:, :c["channels"]], x[:, c["channels"]:]
        x = gate * torch.sigmoid(gate) * up
    return _plain_f8(x, c["form"] == "weights")


def _plain_linear(s):
    c = s["c"]
    a = s["a"].float() * _spread_out(s["a_scale"], c["rows"], c["channels"], False)
    w = s["w"].float() * _spread_out(s["w_scale"], c["outputs"], c["channels"], True)
    y = torch.matmul(a, w.t())
    if c["bias"]:
        y = y + s["bias"]
    return y.to(DTYPES[c["dtype"]])


def run(state):
    if own:
        return _run_own(state)
    kind = state["c"]["kind"]
    if kind == "norm":
        return _plain_norm(state)
    if kind == "rows":
        return _plain_rows(state)
    return _plain_linear(state)


def work(case):
    c = case
    n = c["channels"]
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "norm":
        values = c["tokens"] * n
        out = values + 4 * c["tokens"] * _blocks(n) if c["f8"] else values * size
        return {"bytes": values * size * (3 if c["residual"] else 1) + out + 4 * n, "flops": 8 * values}
    if c["kind"] == "rows":
        values = c["tokens"] * n
        scales = _blocks(c["tokens"]) * _blocks(n) if c["form"] == "weights" else c["tokens"] * _blocks(n)
        return {"bytes": values * size * (2 if c["form"] == "gated" else 1) + values + 4 * scales, "flops": (12 if c["form"] == "gated" else 4) * values}
    m, f = c["rows"], c["outputs"]
    return {"bytes": m * n + 4 * m * _blocks(n) + f * n + 4 * _blocks(f) * _blocks(n) + m * f * size + (4 * f if c["bias"] else 0), "flops": 2 * m * f * n}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def _exact_f8(y, height):
    """y [rows, n] in 64 bits, a block of columns at a time: the nearest e4m3 of y / scale (steps of 2^(e - 3), 2^-9 at least; ties to even), and the scales"""
    rows, n = y.shape
    q = torch.empty_like(y)
    scales = torch.empty((-(-rows // height), _blocks(n)), dtype=torch.float64, device=y.device)
    group = torch.arange(rows, device=y.device) // height
    for b in range(_blocks(n)):
        part = y[:, b * BLOCK:(b + 1) * BLOCK]
        top = torch.zeros(scales.shape[0], dtype=torch.float64, device=y.device).scatter_reduce(0, group, part.abs().amax(1), "amax")
        scales[:, b] = torch.maximum(top / TOP, torch.tensor(LEAST, dtype=torch.float64, device=y.device))
        z = part / scales[:, b][group][:, None]
        exponent = torch.frexp(z)[1] - 1
        step = torch.exp2(exponent.clamp(min=-6).double() - 3)
        q[:, b * BLOCK:(b + 1) * BLOCK] = (torch.round(z / step) * step).clamp(-TOP, TOP)
    return q, scales


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["kind"] == "norm":
        h = s["x"].double()
        if c["residual"]:
            h += s["residual"].double()
        root = torch.sqrt((h * h).sum(1) / c["channels"] + EPS)
        y = h * s["weight"].double()[None] / root[:, None]
        out = list(_exact_f8(y, 1)) if c["f8"] else [y]
        if c["residual"]:
            out.append(h)
        return tuple(out) if len(out) > 1 else out[0]
    if c["kind"] == "rows":
        y = s["x"].double()
        if c["form"] == "gated":
            y = y[:, :c["channels"]] / (1.0 + torch.exp(-y[:, :c["channels"]])) * y[:, c["channels"]:]
        return _exact_f8(y, BLOCK if c["form"] == "weights" else 1)
    out = torch.zeros((c["rows"], c["outputs"]), dtype=torch.float64, device="cuda")
    column = torch.arange(c["outputs"], device="cuda") // BLOCK
    for b in range(_blocks(c["channels"])):      # the definition: a sum of blocks, each with its two scales
        k = slice(b * BLOCK, (b + 1) * BLOCK)
        part = torch.matmul(s["a"][:, k].double(), s["w"][:, k].double().t())
        out += part.mul_(s["a_scale"][:, b].double()[:, None]).mul_(s["w_scale"][:, b].double()[column][None])
    return out if s["bias"] is None else out + s["bias"].double()
