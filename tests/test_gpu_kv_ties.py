"""Rows written into an int8 cache: rint(x 127 / max|x|), ties to even, also where the quotient lies in the middle of two whole numbers."""
import pytest
import torch

from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _written(x):
    """x [tokens, 1, hd] as v of a cache without norm and rotation"""
    tokens, _, hd = x.shape
    pages = -(-tokens // 16)
    k, v = (torch.zeros((pages, 1, 16, hd), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((pages, 1, 16), device="cuda") for _ in range(2))
    xd = x.cuda()
    hip.cache_append(xd, xd, xd, None, torch.arange(tokens, dtype=torch.int32, device="cuda"), k, v, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    for t in (k, v):
        yield t.view(-1, hd)[:tokens].cpu()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_halves_of_a_step(dtype, hd):
    """a row's largest value is 127 units, the others n and a half: sizes of a unit over the type's range"""
    hip.init(0)
    rows = []
    for power in range(-124, 119) if dtype == "bf16" else range(-16, 9):
        for first in range(0, 127, hd - 1):
            row = torch.full((hd,), 127.0, dtype=torch.float64)
            n = first + torch.arange(hd - 1)
            row[1:] = torch.where(n < 127, n + 0.5, 0.0) * (1 - 2 * (n % 3 == 0).double())
            rows.append(row * 2.0 ** power)
    x = torch.stack(rows).to(DT[dtype])
    keep = x.double() == torch.stack(rows)      # what the type holds exactly
    want = torch.round(x.double() * 127 / x.double().abs().amax(1, keepdim=True))
    for got in _written(x[:, None]):
        assert torch.equal(got.double()[keep], want[keep])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_any_row(dtype):
    """values of the 16-bit type times 127 are whole numbers of at most 18 bits, and fp32's quotient of two such is in the middle of two steps or 2^-19 of it away"""
    hip.init(0)
    g = torch.Generator().manual_seed(4)
    x = torch.randn((4000, 128), generator=g).to(DT[dtype])
    top = x.abs().amax(1)
    x[:, 1], x[:, 2], x[:, 3] = top / 2, -top / 2, top / 4     # 63.5, -63.5, 31.75
    want = torch.round(x.double() * 127 / x.double().abs().amax(1, keepdim=True))
    for got in _written(x[:, None]):
        assert torch.equal(got.double(), want)
