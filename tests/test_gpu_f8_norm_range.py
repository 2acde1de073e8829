"""The norm of rows whose squares leave fp32's range, which it takes again scaled by a power of two, against 64 bits."""
import pytest
import torch

import f8_oracle as o
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _check(x, weight, eps, f8, residual=None):
    """o.norm's bound and, for subnormal numbers, half of fp32's smallest step in front of a weight of at most 2, and behind it"""
    eps = float(torch.tensor(eps, dtype=torch.float32))
    got = hip.rms_norm(x, weight, eps=eps, residual=residual, f8=f8)
    _, y, off = o.norm(x, residual, weight, eps)
    off = off + 3 * 2.0 ** -150
    if f8:
        o.check_f8(got[0], got[1], y, off)
    else:
        o.check(got if residual is None else got[0], y, off)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("n", [256, 1000, 4096, 20000])
@pytest.mark.parametrize("power", [-125, -100, -75, -60, -45, 50, 62, 100, 120])
def test_far_from_one(dtype, f8, n, power):
    """rows of one size, with no eps, one far below the squares, one near them and one far above, and beside ordinary rows"""
    hip.init(0)
    g = torch.Generator().manual_seed(n + power)
    x = torch.randn((5, n), generator=g).clamp(-4, 4)
    x[1:4] *= 2.0 ** power
    x = x.to(DT[dtype]).cuda()
    w = 0.5 + torch.rand(n, generator=g).cuda()
    for eps in (0.0, 1e-38, 1e-30, 1e-24, 1e-6):
        _check(x, w, eps, f8)
    _check(x, None, 0.0, f8, residual=x.flip(1).contiguous())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("n", [256, 4096, 20000])
@pytest.mark.parametrize("high,low", [(66, -56), (66, -40), (100, -20), (126, 0), (-60, -100), (-51, -110)])
def test_small_beside_large(dtype, f8, n, high, low):
    """every 128th value large, the others small: results near fp32's smallest normal numbers keep their bits"""
    hip.init(0)
    g = torch.Generator().manual_seed(n)
    x = torch.randn((3, n), generator=g).clamp(-1.9, 1.9) * 2.0 ** low
    x[:, ::128] = torch.randn((3, x[:, ::128].shape[1]), generator=g).clamp(-1.9, 1.9) * 2.0 ** high
    x = x.to(DT[dtype]).cuda()
    _check(x, None, 0.0, f8)
    _check(x, 0.5 + torch.rand(n, generator=g).cuda(), 0.0, f8)
