"""Rows, gated rows and weights as e4m3 with scales for blocks of 128: the bytes that the rule gives in fp32, and 64 bits."""
import math

import pytest
import torch

import f8_oracle as o
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = [(1, 1), (1, 128), (3, 7), (2, 129), (5, 1000), (16, 256), (129, 40), (257, 384), (33, 2056), (1, 11008), (300, 5000), (128, 16384), (1000, 127)]


def _rows(rows, n, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, n), generator=g) * torch.exp(2 * torch.randn(n, generator=g))
    x[torch.rand((rows, n), generator=g) < 0.05] = 0.0
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("rows,n", SIZES)
def test_bytes(dtype, tall, rows, n):
    hip.init(0)
    x = _rows(rows, n, DT[dtype], rows + n)
    q, scale = (hip.f8_from_weights if tall else hip.f8_from_rows)(x)
    want, want_scale = o.to_f8(x.float().cpu(), tall)
    assert q.dtype == o.F8 and q.shape == (rows, n) and q.stride(0) % 16 == 0
    assert torch.equal(scale.cpu(), want_scale)
    assert torch.equal(q.cpu().contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,n", SIZES)
def test_gated(dtype, rows, n):
    hip.init(0)
    x = _rows(rows, 2 * n, DT[dtype], rows + n)
    x[:, :n].clamp_(-60, 60)
    q, scale = hip.f8_from_rows(x, gated=True)
    y, off = o.silu_gated(x)
    assert q.shape == (rows, n)
    o.check_f8(q, scale, y, off)


def test_ties():
    """quotients in the middle of two e4m3 go to the even one: a block's largest value 448 2^e, the others at every middle, and a unit beside it"""
    hip.init(0)
    low = torch.arange(0, 126, dtype=torch.uint8).view(o.F8).float()
    high = torch.arange(1, 127, dtype=torch.uint8).view(o.F8).float()
    middle = (low + high) / 2
    x = torch.zeros((9, 128))
    for i, e in enumerate((-20, -1, 0, 1, 40)):
        x[i, :126] = middle * 2.0 ** e
        x[i, 126] = 448.0 * 2.0 ** e
    x[5, :126], x[6, :126] = middle * (1 + 2.0 ** -23), middle * (1 - 2.0 ** -23)
    x[5:7, 126] = 448.0
    x[7, :126], x[7, 126] = middle * (1 / 3), 448.0 / 3      # a scale that is not a power of two
    x[8] = torch.linspace(-1, 1, 128)
    q, scale = hip.f8_from_rows(x.cuda())
    want, want_scale = o.to_f8(x)
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("tall", [False, True])
def test_out_of_the_ordinary(tall):
    """zeros, subnormal numbers, the largest ones; NaN stays in its place, an infinity takes its block"""
    hip.init(0)
    x = torch.randn((128 * 6 if tall else 6, 256))
    step = 128 if tall else 1
    x[0] = 0.0
    x[0:step, :128] = 0.0
    x[step:2 * step] *= 2.0 ** -130
    x[2 * step:3 * step] = torch.finfo(torch.float32).max
    x[3 * step, 5] = math.nan
    x[4 * step, 130] = -math.inf
    q, scale = (hip.f8_from_weights if tall else hip.f8_from_rows)(x.cuda())
    want, want_scale = o.to_f8(x, tall)
    v = o.values(q.cpu(), scale.cpu(), tall)
    assert torch.equal(scale.cpu(), want_scale)
    keep = torch.ones_like(x, dtype=torch.bool)
    keep[4 * step:5 * step, 128:] = False
    assert bool(v[~keep].isnan().all())
    assert torch.equal(q.cpu().float()[keep].isnan(), x[keep].isnan())
    good = keep & ~x.isnan()
    assert torch.equal(q.cpu().float()[good], want.float()[good])
    assert not v[0].any() and scale[0, 0] == 2.0 ** -126


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("form", ["plain", "gated", "weights"])
def test_strides(dtype, form):
    """slices of wider rows, at an odd element, broadcast rows, results and scales with strides, and nothing written beside them"""
    hip.init(0)
    rows, n = 37, 300
    wide = _rows(rows, 2 * n + 40, DT[dtype], 3)
    call = {"plain": hip.f8_from_rows, "gated": lambda x, **k: hip.f8_from_rows(x, gated=True, **k), "weights": hip.f8_from_weights}[form]
    take = 2 * n if form == "gated" else n
    scale_rows = 1 if form == "weights" else rows
    for x in (wide[:, :take], wide[:, 16:16 + take], wide[:, 3:3 + take], wide[:1, :take].expand(rows, take)):
        want, want_scale = call(x.contiguous())
        q = torch.full((rows, 352), 7, dtype=torch.uint8, device="cuda").view(o.F8)
        scale = torch.full((3, scale_rows + 2), 5.0, device="cuda").t()
        got = call(x, out=q[:, 16:16 + n], scale_out=scale[:scale_rows])
        assert got[0].data_ptr() == q.data_ptr() + 16
        assert torch.equal(q[:, 16:16 + n].contiguous().view(torch.uint8), want.contiguous().view(torch.uint8)) and torch.equal(scale[:scale_rows], want_scale)
        left = q.view(torch.uint8)
        assert bool((left[:, :16] == 7).all()) and bool((left[:, 16 + n:] == 7).all()) and bool((scale[scale_rows:] == 5.0).all())


def test_no_rows():
    hip.init(0)
    x = torch.zeros((0, 256), device="cuda")
    assert [tuple(t.shape) for t in hip.f8_from_rows(x)] == [(0, 256), (0, 2)] and [tuple(t.shape) for t in hip.f8_from_rows(x, gated=True)] == [(0, 128), (0, 1)]
    assert [tuple(t.shape) for t in hip.f8_from_weights(x)] == [(0, 256), (0, 2)]


def test_far_rows():
    """operands and results past 2^32 bytes"""
    hip.init(0)
    rows, n = 3, 300
    store = torch.zeros((2 << 30) + 4096, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((rows, n), (1 << 30, 1))
    x.copy_(_rows(rows, n, torch.bfloat16, 1))
    far = torch.zeros((5 << 30) + 4096, dtype=torch.uint8, device="cuda").view(o.F8).as_strided((rows, n), (5 << 29, 1))
    q, scale = hip.f8_from_rows(x, out=far)
    want, want_scale = o.to_f8(x.float().cpu())
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(q.cpu().contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


@pytest.mark.parametrize("form", ["rows", "weights", "norm"])
def test_many_rows(form):
    """more workgroups than a launch's first dimension takes: every row, all alike, is written"""
    hip.init(0)
    rows, n = {"rows": ((1 << 25) + 40, 16), "weights": ((1 << 28) + 130, 16), "norm": ((1 << 21) + 3, 528)}[form]
    x = _rows(1, n, torch.bfloat16, 7).expand(rows, n)
    q = torch.full((rows, n), 0x55, dtype=torch.uint8, device="cuda").view(o.F8)
    print(form, rows, n, flush=True)
    if form == "norm":
        q, scale = hip.rms_norm(x, f8=True, out=q)
        first = hip.rms_norm(x[:1], f8=True)
    else:
        q, scale = (hip.f8_from_weights if form == "weights" else hip.f8_from_rows)(x, out=q)
        first = (hip.f8_from_weights if form == "weights" else hip.f8_from_rows)(x[:1])
    q = q.view(torch.uint8)
    assert scale.shape[0] == (-(-rows // 128) if form == "weights" else rows) and bool((scale == first[1]).all())
    for at in range(0, rows, 1 << 24):
        assert bool((q[at:at + (1 << 24)] == first[0].view(torch.uint8)).all())
