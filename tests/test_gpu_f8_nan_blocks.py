"""Blocks without a value that is a number: the largest magnitude passes over every NaN, so that such a block has the smallest scale, as one of zeros has, and its bytes are NaN."""
import math

import pytest
import torch

import f8_oracle as o
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIGNALS = {"bf16": (torch.int16, 0x7f81), "f16": (torch.int16, 0x7c01), "f32": (torch.int32, 0x7f800001)}


def _check(q, scale, nan, blocks):
    """q is NaN exactly in `nan`, the scales of `blocks` (a mask like them) are 2^-126 and the others above"""
    assert torch.equal(q.float().isnan(), nan)
    assert bool((scale[blocks] == o.LEAST).all()) and bool((scale[~blocks] > o.LEAST).all()) and bool(scale.isfinite().all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [40, 128, 300, 520])
@pytest.mark.parametrize("kind", ["plain", "gated", "weights"])
def test_rows(kind, n, dtype):
    """the first block and the last, which may be short, of some rows are NaN, quiet or signalling, of either sign"""
    hip.init(0)
    rows, tall = 5 if kind != "weights" else 300, kind == "weights"
    g = torch.Generator().manual_seed(n)
    x = (torch.randn((rows, n), generator=g) + 3.0).to(DT[dtype])
    last = (n - 1) // 128
    nan = torch.zeros((rows, n), dtype=torch.bool)
    some = slice(128, 256) if tall else slice(1, 4)
    nan[some, :128] = True
    nan[some, last * 128:] = True
    x[nan] = math.nan
    x[some, 0] = -math.nan
    bits, signal = SIGNALS[dtype]
    x.view(bits)[some, last * 128] = signal
    blocks = torch.zeros((o.blocks(rows) if tall else rows, o.blocks(n)), dtype=torch.bool)
    which = slice(1, 2) if tall else some
    blocks[which, 0] = blocks[which, last] = True
    if kind == "gated":   # a NaN in the gate or in what it goes to
        up = (torch.randn((rows, n), generator=g) + 3.0).to(DT[dtype])
        for both in (torch.cat([x, up], 1), torch.cat([up, x], 1)):
            q, scale = hip.f8_from_rows(both.cuda(), gated=True)
            _check(q.cpu(), scale.cpu(), nan, blocks)
        return
    q, scale = (hip.f8_from_weights if tall else hip.f8_from_rows)(x.cuda())
    _check(q.cpu(), scale.cpu(), nan, blocks)
    assert torch.equal(scale.cpu(), o.to_f8(x.float(), tall)[1])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [40, 300, 4096, 20000])
def test_norm(n, dtype):
    """a NaN of a row is all of its row"""
    hip.init(0)
    g = torch.Generator().manual_seed(n)
    x = (torch.randn((6, n), generator=g) + 3.0).to(DT[dtype])
    x[2, n // 2], x[5, 0] = math.nan, math.nan
    q, scale, _ = hip.rms_norm(x.cuda(), residual=torch.ones_like(x).cuda(), f8=True)
    nan = torch.zeros((6, n), dtype=torch.bool)
    nan[[2, 5]] = True
    _check(q.cpu(), scale.cpu(), nan, nan[:, :o.blocks(n)])
