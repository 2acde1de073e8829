"""Gated rows over the whole range of a gate: silu(g) = g / (1 + e^-g) is a normal number of fp32 down to g = -91.9, below which e^g is no longer one from g = -87.34 on, and a large
factor takes it back into the range from much further down."""
import math

import pytest
import torch

import f8_oracle as o
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def gated(x):
    """silu(g) u in 64 bits and what fp32 may be off: the exponent g log2(e) by 2^-24 of its rounding and 2^-26 of the constant's (1.25 |g| 2^-24 of the result), three exponentials by an
    ulp each (6 2^-24), six products and the quotient's two steps; a subnormal number on the way by half of its step, times factors of 2 at most"""
    g, u = x.double().chunk(2, 1)
    y = torch.where(g < 0, g * torch.exp(g) / (1 + torch.exp(g)), g / (1 + torch.exp(-g))) * u
    return y, (1.25 * g.abs() + 14) * 2.0 ** -24 * y.abs() + 2.0 ** -148


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("power", [0, 10, 100, 126])
def test_low_gates(dtype, power):
    """a block for each range of gates, so that its scale is of their size; factors up to 2^power"""
    if dtype == "f16" and power > 10:
        pytest.skip("out of fp16's range")
    hip.init(0)
    rows = 24
    g = torch.Generator().manual_seed(power)
    low = torch.tensor([0.0, -60.0, -80.0, -86.0, -88.0, -92.0, -100.0, -120.0, -150.0, -172.0, -176.0, -200.0]).repeat_interleave(128)
    n = low.numel()
    gate = low - 6.0 * torch.rand((rows, n), generator=g)
    up = torch.randn((rows, n), generator=g).clamp(-3.0, 3.0) * 2.0 ** power / (4.0 if power == 126 else 1.0)
    x = torch.cat([gate, up], 1).to(DT[dtype]).cuda()
    y, off = gated(x)
    o.check_f8(*hip.f8_from_rows(x, gated=True), y, off)


@pytest.mark.parametrize("dtype", DT)
def test_one_low_gate_among_others(dtype):
    """one lane's gates are low, the others' of a block are not, on rows of an odd length"""
    hip.init(0)
    g = torch.Generator().manual_seed(3)
    rows, n = 16, 333
    gate, up = torch.randn((rows, n), generator=g) * 3.0, torch.randn((rows, n), generator=g)
    for i in range(rows):
        gate[i, 8 * i + i % 8] = -84.0 - i
        up[i, 8 * i + i % 8] = 30000.0
    x = torch.cat([gate, up], 1).to(DT[dtype]).cuda()
    y, off = gated(x)
    o.check_f8(*hip.f8_from_rows(x, gated=True), y, off)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_the_ends_of_the_range(dtype):
    """gates whose exponential is zero for every factor, and infinite ones"""
    hip.init(0)
    top = float(torch.finfo(DT[dtype]).max)
    gate = torch.tensor([-300.0, -1000.0, -1e30, -top, top / 4, math.inf, -math.inf, math.nan]).repeat_interleave(128)
    x = torch.cat([gate, torch.full_like(gate, 2.0)])[None].to(DT[dtype]).cuda()
    x[0, -1] = 1.0
    q, scale = hip.f8_from_rows(x, gated=True)
    q, scale = q.cpu().float()[0], scale.cpu()[0]
    assert not q[:512].any() and bool((scale[:4] == 2.0 ** -126).all())
    assert bool((q[512:640] == 448.0).all()) and scale[5] == math.inf and bool(q[640:].isnan().all())
