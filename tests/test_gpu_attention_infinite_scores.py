"""Rows whose every seen score is minus infinity: a softmax that is no number, as by the definition, and not the zeros of a row that sees nothing.  Beside
finite scores such keys have no weight."""
import math

import pytest
import torch

import kv_oracle
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}

# workgroups of 64 rows, the same in parts of the keys, of 128 rows, of 256, of 256 in parts
SHAPES = [(1, 2, 1, 100, 100, 64), (2, 3, 1, 90, 200, 128), (1, 2, 1, 20, 2000, 64), (2, 4, 2, 7, 3000, 128), (300, 1, 1, 33, 70, 64), (9, 32, 32, 129, 129, 128), (56, 8, 8, 250, 300, 128),
          (1, 32, 8, 500, 4000, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bias,causal", [(False, True), (True, True), (True, False)])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_prompts(dtype, bias, causal, i):
    hip.init(0)
    b, hq, hkv, tq, tk, hd = SHAPES[i]
    print(dtype, bias, causal, SHAPES[i], flush=True)
    g = torch.Generator().manual_seed(i)
    q, k, v = (torch.randn((b, h, t, hd), generator=g).to(DT[dtype]) for h, t in ((hq, tq), (hkv, tk), (hkv, tk)))
    q[..., 0] = 1.0
    cut = tk - tq + tq // 2            # rows whose place is below see no finite score
    low = k.clone()
    low[:, :, :cut, 0] = -math.inf
    place = torch.arange(tq) + tk - tq
    ranges = torch.stack([torch.zeros(tq), place + 1], 1).int().expand(b, tq, 2).contiguous()
    ranges[:, 3] = 5                   # a row that sees nothing
    slopes = 2.0 ** -torch.arange(1, hq + 1).float() if bias else None
    got = hip.attention_masked(q.cuda(), low.cuda(), v.cuda(), scale=hd ** -0.5, causal=causal, slopes=None if slopes is None else slopes.cuda(), ranges=ranges.cuda(), merged_out=False)
    torch.cuda.synchronize()
    got = got.double().cpu()
    none, empty = place < cut, torch.arange(tq) == 3
    assert bool(got[:, :, none & ~empty].isnan().all())
    assert not got[:, :, empty].any()
    for n in range(0, b, max(1, b // 4)):
        seen, away = kv_oracle.seen_by(tq, tk, True, 0, tk - tq, ranges[n])
        seen[:, :cut] = False          # no weight
        ref, bound = kv_oracle.attention(q[n], k[n], v[n], seen, hd ** -0.5, 0.0, slopes, away)
        assert bool(((got[n] - ref).abs() <= bound)[:, ~none].all())
    if not bias and causal:            # by the interval of the causal mask alone
        got = hip.attention_masked(q.cuda(), low.cuda(), v.cuda(), scale=hd ** -0.5, causal=True, merged_out=False)
        torch.cuda.synchronize()
        assert bool(got[:, :, none.cuda()].isnan().all()) and bool(got[:, :, ~none.cuda()].isfinite().all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("longest", [300, 5000])
def test_the_next_token(dtype, int8, hd, page, longest):
    """one part, and parts that a second launch joins"""
    hip.init(0)
    print(dtype, int8, hd, page, longest, flush=True)
    lengths = [longest, longest, 1, 0, 33, longest - 1]
    per = -(-longest // page)
    g = torch.Generator().manual_seed(hd + page)
    shape = (len(lengths) * per, 2, page, hd)
    table = torch.randperm(shape[0], generator=g).view(len(lengths), per).int()
    q = torch.zeros((len(lengths), 4, hd)).to(DT[dtype])
    q[..., 0] = 1.0
    if int8:
        k, v = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2))
        k[..., 0] = -1
        ks, vs = (0.01 * torch.rand(shape[:3], generator=g) for _ in range(2))
        low = lambda b, at: ks[int(table[b, at // page]), :, at % page].fill_(math.inf)  # noqa: E731
    else:
        k, v = (torch.randn(shape, generator=g).to(DT[dtype]) for _ in range(2))
        ks = vs = None
        low = lambda b, at: k[int(table[b, at // page]), :, at % page, 0].fill_(-math.inf)  # noqa: E731
    for b, n in enumerate(lengths):
        for at in range(n):
            if b in (0, 2, 4) or (b == 1 and at != n // 2) or (b == 5 and at != 2):    # of two sequences one key is finite
                low(b, at)
    dev = lambda x: None if x is None else x.cuda()  # noqa: E731
    got = hip.attention_paged(dev(q), dev(k), dev(v), dev(table), torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale=0.1, k_scale=dev(ks), v_scale=dev(vs))
    torch.cuda.synchronize()
    got = got.double().cpu()
    assert bool(got[[0, 2, 4]].isnan().all()) and not got[3].any()
    for b, at in ((1, longest // 2), (5, 2)):
        ref = kv_oracle.rows(v, vs, table[b], lengths[b])[:, at].repeat_interleave(2, dim=0)
        assert bool(((got[b] - ref).abs() <= 2 * kv_oracle.HALF[DT[dtype]] * ref.abs() + (2.0 ** -24 if dtype == "f16" else 0.0)).all())   # a rounded weight, a rounded result
