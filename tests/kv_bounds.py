"""Attention of one new token over a cache in 64 bits, with the bound that its probabilities' own rounding gives, apart from the result's."""
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative


def weight_bits(dtype, int8):
    """how far a probability (times its value's scale) may be off, relative: two bf16 parts, of which the first is cut (a step, 2^-7, is left at most) and the second
    rounded (half a step of that), or one fp16, rounded"""
    return HALF[torch.float16] if dtype == torch.float16 and not int8 else 2.0 ** -7 * HALF[torch.bfloat16]


def attention(q, k, v, scale, weight):
    """q [h, d], k and v [t, d] in 64 bits -> out and the bound of its error [h, d]; the result is rounded to q's type.

    Probabilities: `weight` each, on values and (where the rounded ones are summed) on the sum.  Scores: d additions of products, the products with a scale and with
    log2(e), the difference to the reference point, and the exponential, two units: on the weight and on the sum.  The sum's t additions; a product of the weight with
    a value's scale, the quotient.  A part of a result below the type's normal numbers: 2^-25 in fp16, whose probabilities are at least 2^7 at their largest and
    lose 2^-25 below 2^-14."""
    a = q.double()
    s = (a @ k.t()) * scale
    top = float((a.abs() @ k.abs().t()).max()) * abs(scale)
    p = torch.softmax(s, 1)
    out, mass = p @ v, p @ v.abs()
    fp32 = (2 * ((q.shape[1] + 8) * top + 16) + 2 * k.shape[0] + 4) * 2.0 ** -24
    low = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    half = HALF[q.dtype]
    return out, half * out.abs() + (1 + half) * (weight + fp32) * (mass + out.abs()) + low * (1 + 2.0 ** -7 * (v.abs().sum(0) + k.shape[0] * out.abs()))
