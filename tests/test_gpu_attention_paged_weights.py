"""The weights of attention over the paged cache: they sum to one wherever they are rounded."""
import math

import pytest
import torch

from onenew_amd import hip

pytestmark = pytest.mark.gpu


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
