"""Parts of the keys joined: a value that is no number stays in the result however little its part weighs, as it does where one workgroup has all keys."""
import math

import pytest
import torch

from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _values(dtype, keys, hd, g):
    v = torch.randn((keys, hd), generator=g).to(DT[dtype])
    v[3, 0], v[5, 1], v[7, 2] = math.nan, math.inf, -math.inf
    return v


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("keys,queries,heads", [(100, 4, 1), (3000, 4, 1), (70000, 1, 1), (4000, 500, 32)])
def test_prompts(dtype, hd, keys, queries, heads):
    """the first half of the keys is 2^-400 of the second"""
    hip.init(0)
    print(dtype, hd, keys, queries, heads, flush=True)
    g = torch.Generator().manual_seed(keys)
    q, k = torch.zeros((1, heads, queries, hd), dtype=DT[dtype]), torch.zeros((1, 1, keys, hd), dtype=DT[dtype])
    q[..., 0] = 1.0
    k[0, 0, : keys // 2, 0] = -280.0
    v = _values(dtype, keys, hd, g)[None, None]
    got = hip.attention_masked(q.cuda(), k.cuda(), v.cuda(), causal=True, merged_out=False).float().cpu()
    assert bool(got[..., 0].isnan().all()) and not bool(got[..., 1:3].isfinite().any()) and bool(got[..., 3:].isfinite().all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("keys,batch", [(100, 1), (1000, 1), (5000, 1), (5000, 100), (70000, 1)])
def test_the_next_token(dtype, hd, keys, batch):
    hip.init(0)
    print(dtype, hd, keys, batch, flush=True)
    g = torch.Generator().manual_seed(keys)
    per = -(-keys // 16)
    k, v = (torch.zeros((per, 1, 16, hd), dtype=DT[dtype]) for _ in range(2))
    k.view(-1, hd)[: keys // 2, 0] = -280.0
    v.view(-1, hd)[:keys] = _values(dtype, keys, hd, g)
    q = torch.zeros((batch, 2, hd), dtype=DT[dtype])
    q[..., 0] = 1.0
    table = torch.arange(per, dtype=torch.int32).expand(batch, per).contiguous()
    got = hip.attention_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.full((batch,), keys, dtype=torch.int32, device="cuda")).float().cpu()
    assert bool(got[..., 0].isnan().all()) and not bool(got[..., 1:3].isfinite().any()) and bool(got[..., 3:].isfinite().all())
