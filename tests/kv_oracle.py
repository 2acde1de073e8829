"""The operators around the paged key-value cache in 64 bits, from their definitions, and the bounds that the kernels' roundings give."""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative


def attention(q, k, v, seen, scale=1.0, cap=0.0, slopes=None, distance=None):
    """q [h, n, d], k and v [hkv, t, d] (any type), seen [n, t], slopes [h], distance [n, t] -> out and the bound of its error, both [h, n, d]

    Error: half a step of the type for each rounded probability and for the result; a probability also has twice (once in the weight, once in
    the sum) its score's error: d additions of products in fp32 and four roundings on its way into the exponential, which itself is off by
    two units; the sum has t additions.  A capped score: tanh from an exponential and a reciprocal, eight units of the cap.  fp16 probabilities are
    at least 2^7 at their largest and lose 2^-25 below 2^-14, and a result below fp16's normal numbers 2^-25."""
    half = HALF[q.dtype]
    group = q.shape[0] // k.shape[0]
    out, bound = [], []
    for h in range(q.shape[0]):
        a, b, c = q[h].double(), k[h // group].double(), v[h // group].double()
        s = (a @ b.t()) * scale
        size = (a.abs() @ b.abs().t()) * abs(scale)
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s - slopes[h].double() * distance.double()
            size = size + slopes[h].double() * distance.double()
        s = torch.where(seen, s, -math.inf)
        alive = seen.any(1, keepdim=True)
        p = torch.where(alive, torch.softmax(torch.where(alive, s, 0.0), 1), 0.0)
        c0 = torch.where(seen.any(0)[:, None], c, 0.0)   # values that nobody sees may be anything
        o = p @ c0
        mass = p @ c0.abs()
        top = float(torch.where(seen, size, 0.0).max()) if seen.numel() else 0.0
        score = 2 * ((q.shape[2] + 8) * top + 8 * cap + 16 + k.shape[1]) * 2.0 ** -24
        tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
        out.append(o)
        bound.append(half * o.abs() + (half + score) * (1 + half) * mass + tiny * (1 + 2.0 ** -7 * c0.abs().sum(0)))
    return torch.stack(out), torch.stack(bound)


def seen_by(tq, tk, causal, window, q_offset, ranges=None):
    """[tq, tk] truth values and the distances"""
    place, key = torch.arange(tq)[:, None] + q_offset, torch.arange(tk)[None]
    away = place - key
    seen = torch.ones((tq, tk), dtype=torch.bool)
    if causal:
        seen &= away >= 0
    if window:
        seen &= away < window
    if ranges is not None:
        seen &= (key >= ranges[:, :1]) & (key < ranges[:, 1:])
    return seen, away.abs()


def turned(x, weight, positions, freq, eps, interleaved):
    """norm and rotation of x [tokens, heads, d] in 64 bits, and the bound of an fp32 computation's error"""
    d = x.shape[-1]
    x = x.double()
    rel = 0.0
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
        rel = (d / 2 + 8) * 2.0 ** -24   # the sum's additions count half in a square root
    y, size = x.clone(), x.abs().clone()
    if freq is not None:
        r = freq.numel()
        angle = positions.double()[:, None, None] * freq.double()
        cs, sn = torch.cos(angle), torch.sin(angle)
        one, two = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved else (slice(0, r), slice(r, 2 * r))
        a, b = x[..., one], x[..., two]
        y[..., one], y[..., two] = a * cs - b * sn, b * cs + a * sn
        size[..., one] = size[..., two] = a.abs() + b.abs()
    # cosine and sine: their argument's rounding (2^-25 of a half revolution, times pi) and two units; three roundings of the turn
    return y, size * (rel + 10 * 2.0 ** -24)


def rows(cache, scale, table, n):
    """rows 0 .. n - 1 of one sequence: [kv_heads, n, d] in 64 bits"""
    page = cache.shape[2]
    at = torch.arange(n)
    x = cache[table.long()[at // page], :, at % page].double()
    if scale is not None:
        x = x * scale[table.long()[at // page], :, at % page].double().unsqueeze(-1)
    return x.permute(1, 0, 2)
