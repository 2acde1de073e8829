"""The weights of attention over the paged cache: they sum to one wherever they are rounded, and a key that has none does not take bits from the others."""
import math

import numpy as np
import pytest
import torch

import kv_oracle
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _rounded_up(scale):
    """d in (4, 5) for which 2^d scale lies a little above the middle of two numbers of eleven bits, so that rounding adds all but half a step"""
    frac = math.frexp(scale)[0] * 2.0
    for k in range(1024):
        target = 1.0 + (k + 0.55) * 2.0 ** -10
        if target > frac:
            return 4.0 + math.log2(target / frac)
    raise AssertionError


@pytest.mark.parametrize("hd", [64, 128])
def test_largest_values_of_fp16(hd):
    """of one value everywhere, the largest: 256 keys at a score of 0, where the reference point stays, and 768 whose probability rounds up by 0.4 of a step of
    eleven bits.  Weights that sum to at most 1 + 1024 2^-24 (additions in fp32) give at most 65508, which rounds to 65504."""
    hip.init(0)
    q, k = torch.zeros((1, 3, hd), dtype=torch.float16), torch.zeros((64, 1, 16, hd), dtype=torch.float16)
    q[..., 0] = 1.0
    k.view(-1, hd)[256:, 0] = 1.0
    v = torch.full_like(k, 65504.0)
    table, n = torch.arange(64, dtype=torch.int32).view(1, 64), torch.tensor([1024], dtype=torch.int32)
    got = hip.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), n.cuda(), scale=_rounded_up(1.0) * math.log(2.0))
    torch.cuda.synchronize()
    assert bool((got == 65504.0).all()), got.flatten()[0]


@pytest.mark.parametrize("hd", [64, 128])
def test_largest_values_of_int8(hd):
    """the same with 127 times a scale: a probability times its scale keeps sixteen bits, 2^-15 at most, and 65506 rounds to 65504"""
    hip.init(0)
    scale = float(np.float32(65504.0 / 127.0))
    q, k = torch.zeros((1, 3, hd), dtype=torch.float16), torch.zeros((64, 1, 16, hd), dtype=torch.int8)
    q[..., 0] = 1.0
    k.view(-1, hd)[256:, 0] = 1
    v = torch.full_like(k, 127)
    ks, vs = torch.ones((64, 1, 16)), torch.full((64, 1, 16), scale)
    table, n = torch.arange(64, dtype=torch.int32).view(1, 64), torch.tensor([1024], dtype=torch.int32)
    got = hip.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), n.cuda(), scale=_rounded_up(scale) * math.log(2.0), k_scale=ks.cuda(), v_scale=vs.cuda())
    torch.cuda.synchronize()
    assert bool((got == 65504.0).all()), got.flatten()[0]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("ratio", [2.0 ** -10, 2.0 ** -20, 2.0 ** -30, 2.0 ** -60])
def test_a_large_scale_without_weight(dtype, page, ratio):
    """a key whose value is large and whose probability is below e^-100 next to keys with small values: the result is theirs.  fp16 results need small values of at
    least 2^-14 to be more than a few bits, so there the large one has the factor."""
    hip.init(0)
    hd, lengths = 64, [40, 700]
    g = torch.Generator().manual_seed(page)
    per = -(-700 // page)
    shape = (2 * per, 2, page, hd)
    k, v = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2))
    k[..., 0] = 0
    table = torch.randperm(2 * per, generator=g).view(2, per).int()
    ks, vs = 0.001 + 0.01 * torch.rand(shape[:3], generator=g), (0.01 + 0.01 * torch.rand(shape[:3], generator=g)) * (ratio if dtype == "bf16" else 1.0)
    for b, n in enumerate(lengths):
        for at in (1, n // 2):
            page_at, row = int(table[b, at // page]), at % page
            k[page_at, :, row] = 0
            k[page_at, :, row, 0] = -127
            ks[page_at, :, row] = 1.0
            vs[page_at, :, row] = 0.02 if dtype == "bf16" else 0.02 / ratio
    q = torch.randn((2, 4, hd), generator=g).to(DT[dtype])
    q[..., 0] = 10.0
    n = torch.tensor(lengths, dtype=torch.int32)
    got = hip.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), n.cuda(), scale=0.2, k_scale=ks.cuda(), v_scale=vs.cuda())
    torch.cuda.synchronize()
    for b, m in enumerate(lengths):
        kr, vr = kv_oracle.rows(k, ks, table[b], m), kv_oracle.rows(v, vs, table[b], m)
        keep = torch.ones((1, m), dtype=torch.bool)
        keep[0, [1, m // 2]] = False     # their scores are 250 below the others'
        ref, bound = kv_oracle.attention(q[b][:, None], kr, vr, keep, 0.2)
        err = (got[b].double().cpu() - ref[:, 0]).abs()
        assert bool((err <= 1.1 * bound[:, 0]).all()), (b, float((err / bound[:, 0]).max()))   # the products with the scales, one more rounding each


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_scales_of_either_sign_and_zero(dtype):
    """a value is int8 times its scale"""
    hip.init(0)
    hd, n = 64, 300
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randint(-127, 128, (20, 1, 16, hd), generator=g, dtype=torch.int8) for _ in range(2))
    ks, vs = 0.01 * torch.randn((20, 1, 16), generator=g), torch.randn((20, 1, 16), generator=g)
    vs.view(-1)[::7] = 0.0
    vs.view(-1)[3::7] = -0.0
    table, q = torch.randperm(20, generator=g).view(1, 20).int(), torch.randn((1, 4, hd), generator=g).to(DT[dtype])
    lengths = torch.tensor([n], dtype=torch.int32)
    run = lambda: hip.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lengths.cuda(), scale=0.1, slopes=torch.full((4,), 3.0, device="cuda"), k_scale=ks.cuda(), v_scale=vs.cuda())  # noqa: E731
    got = run()
    away = (n - 1 - torch.arange(n))[None]
    ref, bound = kv_oracle.attention(q[0][:, None], kv_oracle.rows(k, ks, table[0], n), kv_oracle.rows(v, vs, table[0], n), away >= 0, 0.1, 0.0, torch.full((4,), 3.0), away)
    assert bool(((got[0].double().cpu() - ref[:, 0]).abs() <= 1.1 * bound[:, 0]).all())
    # a scale that is an infinity: of the sign of its int8 where that is not 0
    at = n - 2
    page, row = int(table[0, at // 16]), at % 16
    vs[page, 0, row] = math.inf
    v[page, 0, row, :3] = torch.tensor([5, -5, 0], dtype=torch.int8)
    got = run().float()
    assert bool((got[..., 0] == math.inf).all()) and bool((got[..., 1] == -math.inf).all()) and bool(got[..., 2].isnan().all())
