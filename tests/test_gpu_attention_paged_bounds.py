"""How many bits the probabilities of attention over the paged cache have: with few keys, whose values largely cancel, a result is off by more than its own
rounding allows wherever they are rounded to one bf16 (16-bit caches of bf16) or to fp16 (int8 caches, with a result in fp16)."""
import pytest
import torch

import kv_bounds

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
HQ, HKV, PAGE = 4, 2, 16


def _case(dtype, int8, hd, seed):
    """40 sequences of 2 to 41 keys; scores of about one"""
    g = torch.Generator().manual_seed(seed)
    lengths = torch.arange(2, 42, dtype=torch.int32)
    shape = (len(lengths) * 3, HKV, PAGE, hd)
    table = torch.randperm(shape[0], generator=g).view(-1, 3).int()
    q = (0.3 * torch.randn((len(lengths), HQ, hd), generator=g)).to(DT[dtype])
    if int8:
        kv = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2)] + [0.005 + 0.01 * torch.rand(shape[:3], generator=g) for _ in range(2)]
    else:
        kv = [torch.randn(shape, generator=g).to(DT[dtype]) for _ in range(2)] + [None, None]
    return q, kv, table, lengths


def _rows(kv, i, table, head, n):
    at = torch.arange(n)
    page = table.long()[at // PAGE]
    x = kv[i][page, head, at % PAGE].double()
    return x if kv[2] is None else x * kv[2 + i][page, head, at % PAGE].double().unsqueeze(-1)


def _worst(got, q, kv, table, lengths, scale, weight):
    """the largest error in units of its bound"""
    most = 0.0
    for b, n in enumerate(lengths.tolist()):
        for h in range(HKV):
            heads = slice(h * HQ // HKV, (h + 1) * HQ // HKV)
            ref, bound = kv_bounds.attention(q[b, heads], _rows(kv, 0, table[b], h, n), _rows(kv, 1, table[b], h, n), scale, weight)
            most = max(most, float(((got[b, heads].double() - ref).abs() / bound).max()))
    return most


KINDS = [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,int8", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_the_kernels(dtype, int8, hd):
    from onenew_amd import hip
    hip.init(0)
    for seed in range(3):
        q, kv, table, lengths = _case(dtype, int8, hd, seed)
        k, v, ks, vs = (None if t is None else t.cuda() for t in kv)
        got = hip.attention_paged(q.cuda(), k, v, table.cuda(), lengths.cuda(), scale=hd ** -0.5, k_scale=ks, v_scale=vs)
        torch.cuda.synchronize()
        assert _worst(got.cpu(), q, kv, table, lengths, hd ** -0.5, kv_bounds.weight_bits(DT[dtype], int8)) <= 1.0


def _rounded(x, dtype):
    return x.to(dtype).double()


@pytest.mark.parametrize("dtype,int8", KINDS)
def test_the_bound(dtype, int8):
    """weights in 64 bits with the kernels' roundings, and with a coarser one, which the bound has to find: bf16 for two bf16 parts, with a result in fp16 also fp16"""
    hd = 64
    q, kv, table, lengths = _case(dtype, int8, hd, 0)
    scale, t = hd ** -0.5, DT[dtype]

    def result(parts):
        out = torch.empty(q.shape, dtype=t)
        for b, n in enumerate(lengths.tolist()):
            for h in range(HQ):
                k, v = (_rows(kv, i, table[b], h * HKV // HQ, n) for i in range(2))
                s = (q[b, h].double() @ k.t()) * scale
                e = 128 * torch.exp(s - s.max())
                step = _rows([torch.ones_like(x) for x in kv[:2]] + [kv[2], kv[3]], 1, table[b], h * HKV // HQ, n)[:, 0] if int8 else torch.ones(n, dtype=torch.float64)
                w = e * step
                first = _rounded(w, parts[0])
                w = first + (_rounded(w - first, parts[1]) if len(parts) > 1 else 0.0)
                total = w.sum() if t == torch.float16 and not int8 else e.sum()
                out[b, h] = ((w[:, None] * (v / step[:, None])).sum(0) / total).to(t)
        return out

    worst = lambda *parts: _worst(result(parts), q, kv, table, lengths, scale, kv_bounds.weight_bits(t, int8))  # noqa: E731
    assert worst(torch.float64) <= 1.0
    assert worst(*([torch.float16] if dtype == "f16" and not int8 else [torch.bfloat16] * 2)) <= 1.0
    assert worst(torch.bfloat16) > 2.0
    if int8 and dtype == "f16":
        assert worst(torch.float16) > 1.0
