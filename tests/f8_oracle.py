"""e4m3 rows with scales for blocks of 128, their product and the norm in front of it, in 64 bits, with bounds of what 32 bits may be off."""
import torch

BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -126
F8 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative
LOW = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half of the smallest step


def blocks(n):
    return -(-n // BLOCK)


def spread(scale, rows, n, tall=False):
    """a scale for each element"""
    scale = scale.repeat_interleave(BLOCK, 1)[:, :n]
    return scale.repeat_interleave(BLOCK, 0)[:rows] if tall else scale


def tops(y, tall=False):
    """the largest magnitude of each block, NaN passed over"""
    rows, n = y.shape
    y = torch.nn.functional.pad(y.abs().nan_to_num(nan=0.0, posinf=torch.inf), (0, -n % BLOCK, 0, -rows % BLOCK if tall else 0)).unflatten(1, (-1, BLOCK))
    return y.unflatten(0, (-1, BLOCK)).amax((1, 3)) if tall else y.amax(-1)


def to_f8(y, tall=False):
    """y in fp32, as the rule has it in fp32: scales and bytes"""
    assert y.dtype == torch.float32
    scale = (tops(y, tall) / TOP).clamp(min=LEAST)
    return (y / spread(scale, *y.shape, tall)).to(F8), scale


def values(q, scale, tall=False):
    return q.double() * spread(scale.double(), *q.shape, tall)


def check_f8(q, scale, y, off, tall=False):
    """q and scale against y in 64 bits, of which fp32 may be `off` (a tensor like y): the scale, and half a step of e4m3 from the value: 2^-4 of it, or 2^-10
    scales where the steps are 2^-9 (the quotient's own rounding is 2^-24 of it)"""
    want = (tops(y, tall) / TOP).clamp(min=LEAST)
    far = tops(off, tall) / TOP
    assert bool(((scale.double() - want).abs() <= far + 2.0 ** -24 * want * (1 + 2.0 ** -20)).all())
    got = values(q, scale, tall)
    each = spread(scale.double(), *y.shape, tall)
    half = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * each)
    assert bool(((got - y).abs() <= half * (1 + 2.0 ** -20) + 2 * off + spread(far, *y.shape, tall) * TOP).all())


def silu_gated(x):
    """fp32's bound: the exponential off by |g| 2^-24 and two units, five roundings"""
    g, u = x.double().chunk(2, 1)
    y = g / (1 + torch.exp(-g)) * u
    return y, (g.abs() + 10) * 2.0 ** -24 * y.abs()


def norm(x, residual, weight, eps):
    """h, y and what y may be off in fp32: h rounded, the sum's additions (a lane has n / 64 of them at most, six steps between lanes and sixteen between
    wavefronts), half of that under the root, and eight roundings"""
    h = x.double() + (0 if residual is None else residual.double())
    n = h.shape[1]
    y = h / torch.sqrt((h * h).sum(1, keepdim=True) / n + eps) * (1 if weight is None else weight.double())
    return h, y, ((n / 64 + 22 + 2) / 2 + 10) * 2.0 ** -24 * y.abs()


def linear(a, a_scale, w, w_scale, bias=None, cut=False):
    """the product and what it may be off in fp32: the scales' product, a block's 128 additions (each off by a unit of the magnitudes' sum at most, however the matrix
    instruction orders and cuts them), the fused sums over blocks, the bias.

    cut: sums of eight products with 13 bits below the power of two of the largest: a product of two e4m3 has 8 bits, so the largest is whole, and each of the seven others loses
    less than 2^-13 of the largest, which is at most the eight magnitudes' sum: 7 2^-13 of the magnitudes' sum over all channels."""
    x, y = values(a, a_scale), values(w, w_scale, True)
    out, mass = x @ y.t(), x.abs() @ y.abs().t()
    far = (128 + blocks(a.shape[1]) + 4) * 2.0 ** -23 * mass + (7 * 2.0 ** -13 * mass if cut else 0)
    if bias is not None:
        out, far = out + bias.double(), far + 2.0 ** -23 * (mass + bias.double().abs())
    return out, far


def cuts(m, dtype):
    """whether a product of m rows may sum with 13 bits: more than 32 rows with a result in 16 bits"""
    return m > 32 and dtype != torch.float32


def check(got, ref, off):
    half = HALF[got.dtype]
    assert got.shape == ref.shape
    far = (got.double() - ref).abs() - (half * ref.abs() + (1 + half) * off + LOW[got.dtype])
    assert bool((far <= 0).all()), float(far.max())
