"""The root-mean-square norm of rows plus their residuals against 64 bits."""
import math

import pytest
import torch

import f8_oracle as o
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = [(1, 1), (1, 4096), (2, 64), (5, 127), (7, 512), (6, 513), (3, 1000), (9, 2048), (4, 2049), (300, 4096), (3, 5000), (2, 8192), (2, 8200), (3, 16384), (2, 16385), (2, 40000)]


def _rows(rows, n, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn((rows, n), generator=g) + 0.1) * torch.exp(0.5 * torch.randn(n, generator=g))).to(dtype).cuda()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,n", SIZES)
def test_norm(dtype, f8, rows, n):
    hip.init(0)
    x, r = _rows(rows, n, DT[dtype], n), _rows(rows, n, DT[dtype], n + 1)
    w = 0.5 + torch.rand(n, generator=torch.Generator().manual_seed(2)).cuda()
    for residual, weight in ((r, w), (None, w), (r, None)):
        got = hip.rms_norm(x, weight, eps=1e-5, residual=residual, f8=f8)
        got = got if isinstance(got, tuple) else (got,)
        h, y, off = o.norm(x, residual, weight, 1e-5)
        if f8:
            assert got[0].dtype == o.F8 and got[0].stride(0) % 16 == 0
            o.check_f8(got[0], got[1], y, off)
        else:
            o.check(got[0], y, off)
        assert len(got) == 1 + f8 + (residual is not None)
        if residual is not None:
            assert torch.equal(got[-1], (x.float() + r.float()).to(DT[dtype]))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [300, 4096, 20000])
def test_in_place(dtype, n):
    """the residual's sum in its place or x's, a result in the other one's; slices at odd elements; nothing beside them"""
    hip.init(0)
    rows = 11
    wide = [_rows(rows, n + 9, DT[dtype], i) for i in range(2)]
    w = torch.rand(n, device="cuda")
    for first in (0, 1, 8):
        x, r = (t[:, first:first + n] for t in wide)
        want, total = hip.rms_norm(x.contiguous(), w, residual=r.contiguous())
        q, scale, _ = hip.rms_norm(x.contiguous(), w, residual=r.contiguous(), f8=True)
        for places in ("rx", "xr", "r-", "-r", "-x"):
            one, two = (t.clone() for t in wide)
            at = {"x": one[:, first:first + n], "r": two[:, first:first + n], "-": None}
            got = hip.rms_norm(at["x"], w, residual=at["r"], sum_out=at[places[0]], out=at[places[1]])
            assert torch.equal(got[0], want) and torch.equal(got[1], total), places
            for t, name, was in ((one, "x", wide[0]), (two, "r", wide[1])):
                t, was = t.clone(), was.clone()
                if name in places:
                    t[:, first:first + n] = was[:, first:first + n] = 0
                assert torch.equal(t, was)
        two = wide[1].clone()
        got = hip.rms_norm(x, w, residual=two[:, first:first + n], sum_out=two[:, first:first + n], f8=True)
        assert torch.equal(got[0].contiguous().view(torch.uint8), q.contiguous().view(torch.uint8)) and torch.equal(got[1], scale) and torch.equal(two[:, first:first + n], total)


def test_strides():
    """broadcast operands, an unaligned weight, results in wider rows"""
    hip.init(0)
    rows, n = 9, 260
    x, w = _rows(1, n, torch.float16, 5).expand(rows, n), torch.rand(n + 1, device="cuda")[1:]
    r = _rows(rows, n, torch.float16, 6)
    q = torch.full((rows, 304), 9, dtype=torch.uint8, device="cuda").view(o.F8)
    scale, total = torch.full((4, rows), 5.0, device="cuda").t(), torch.full((rows, n + 3), 4.0, dtype=torch.float16, device="cuda")
    hip.rms_norm(x, w, residual=r, f8=True, out=q[:, 32:32 + n], scale_out=scale[:, :3], sum_out=total[:, 1:1 + n])
    h, y, off = o.norm(x, r, w, 1e-6)
    o.check_f8(q[:, 32:32 + n], scale[:, :3], y, off)
    assert torch.equal(total[:, 1:1 + n], h.half()) and bool((total[:, 0] == 4.0).all()) and bool((total[:, 1 + n:] == 4.0).all())
    assert bool((q.view(torch.uint8)[:, :32] == 9).all()) and bool((q.view(torch.uint8)[:, 32 + n:] == 9).all()) and bool((scale[:, 3] == 5.0).all())


def test_out_of_the_ordinary():
    """rows of zeros (with and without eps), one with a NaN, one with an infinity, values whose squares leave 16 bits; no rows"""
    hip.init(0)
    x = _rows(6, 256, torch.bfloat16, 1)
    x[0] = 0.0
    x[1, 3] = math.nan
    x[2, 4] = math.inf
    x[3] *= 2.0 ** 60
    x[4] *= 2.0 ** -60
    y = hip.rms_norm(x, eps=1e-6)
    assert not y[0].any() and bool(y[1].isnan().all())
    assert bool(y[2, 4].isnan()) and not y[2, :4].any()      # the infinity over an infinite root, finite ones over it
    _, want, off = o.norm(x[3:], None, None, 1e-6)
    o.check(y[3:], want, off)
    assert bool(hip.rms_norm(x[:1], eps=0.0).isnan().all())   # 0 / 0
    q, scale = hip.rms_norm(x, eps=1e-6, f8=True)
    assert not q[0].float().any() and bool((scale[0] == 2.0 ** -126).all()) and bool(q[1].float().isnan().all())
    assert [tuple(t.shape) for t in hip.rms_norm(x[:0], residual=x[:0], f8=True)] == [(0, 256), (0, 2), (0, 256)]
