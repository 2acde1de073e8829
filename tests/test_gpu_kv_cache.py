"""Norm, rotation and the write into the paged cache, and the cache read back, against 64 bits."""
import math

import pytest
import torch

import kv_oracle
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _cache(pages, heads, page, hd, dtype, int8):
    shape = (pages, heads, page, hd)
    if int8:
        kv = [torch.full(shape, 77, dtype=torch.int8, device="cuda") for _ in range(2)]
        return kv + [torch.full(shape[:3], 3.0, device="cuda") for _ in range(2)]
    return [torch.full(shape, 7.0, dtype=dtype, device="cuda") for _ in range(2)] + [None, None]


CASES = [  # tokens, q heads, kv heads, head dim, page, pairs, interleaved, norms, first position
    (1, 1, 1, 64, 1, 32, False, "qk", 0), (3, 4, 2, 128, 16, 64, False, "qk", 100), (5, 3, 1, 64, 8, 16, True, "", 1000000), (33, 6, 3, 128, 2, 32, False, "q", 2 ** 31 - 40),
    (17, 5, 5, 128, 64, 64, True, "k", -9), (300, 32, 8, 128, 16, 64, False, "qk", 0), (700, 12, 12, 64, 32, 0, False, "qk", 0), (2, 40, 1, 64, 1024, 8, False, "", 7),
    (400, 7, 2, 64, 16, 32, True, "qk", 131000)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_append(dtype, int8, i):
    hip.init(0)
    tokens, hq, hkv, hd, page, pairs, interleaved, norms, first = CASES[i]
    print(dtype, int8, CASES[i], flush=True)
    g = torch.Generator().manual_seed(i)
    x = torch.randn((tokens, hq + 2 * hkv, hd), generator=g).to(DT[dtype])
    pages = (tokens + page - 1) // page + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens].int()
    gone = torch.zeros(tokens, dtype=torch.bool)
    if tokens > 2:    # padding, and slots that do not exist
        gone[[0, tokens // 2]] = True
        slots[0], slots[tokens // 2] = -1, pages * page
    positions = (first + torch.arange(tokens)).int()
    freq = (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))).float() if pairs else None
    qw, kw = (torch.rand(hd, generator=g) + 0.5 if n in norms else None for n in "qk")
    k, v, ks, vs = _cache(pages, hkv, page, hd, DT[dtype], int8)
    before = [None if t is None else t.cpu().clone() for t in (k, v, ks, vs)]
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    xd = x.cuda()
    q = hip.cache_append(xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], dev(positions), dev(slots), k, v, inv_freq=dev(freq), q_weight=dev(qw), k_weight=dev(kw),
                         eps=1e-5, interleaved=interleaved, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    half, low = kv_oracle.HALF[DT[dtype]], 2.0 ** -25 if dtype == "f16" else 0.0
    ref, off = kv_oracle.turned(x[:, :hq], qw, positions, freq, 1e-5, interleaved)
    assert bool(((q.double().cpu() - ref).abs() <= half * ref.abs() + (1 + half) * off + low).all())
    kref, koff = kv_oracle.turned(x[:, hq:hq + hkv], kw, positions, freq, 1e-5, interleaved)
    vref = x[:, hq + hkv:].double()
    keep = (~gone).nonzero()[:, 0]
    at = slots[keep].long()
    for cache, scale, was, was_scale, ref, off in ((k, ks, before[0], before[2], kref, koff), (v, vs, before[1], before[3], vref, torch.zeros_like(vref))):
        got = cache.cpu()[at // page, :, at % page].double()
        ref, off = ref[keep], off[keep]
        if int8:
            step = scale.cpu()[at // page, :, at % page].double()
            top = ref.abs().amax(-1)
            far = off.amax(-1)
            assert bool(((step * 127 - top).abs() <= far + 4 * 2.0 ** -24 * top).all())
            # half a step, what the value is off, and the roundings of the product with 127 / max (at most 127 steps, three of them and the scale's)
            assert bool(((got * step[..., None] - ref).abs() <= (step * (0.5 + 127 * 6 * 2.0 ** -24) + 2 * far)[..., None]).all())
            was_scale[at // page, :, at % page] = scale.cpu()[at // page, :, at % page]
            assert torch.equal(was_scale, scale.cpu())
        else:
            assert bool(((got - ref).abs() <= half * ref.abs() + (1 + half) * off + low).all())
        was[at // page, :, at % page] = cache.cpu()[at // page, :, at % page]
        assert torch.equal(was, cache.cpu())    # every other row as it was


def test_nothing_but_the_write():
    """no norm, no rotation, no positions; no tokens"""
    hip.init(0)
    x = torch.randn((5, 4, 128), device="cuda").bfloat16()
    k, v, _, _ = _cache(2, 1, 4, 128, torch.bfloat16, False)
    slots = torch.tensor([7, 0, 3, 5, 1], dtype=torch.int32, device="cuda")
    q = hip.cache_append(x[:, :2], x[:, 2:3], x[:, 3:], None, slots, k, v)
    torch.cuda.synchronize()
    assert torch.equal(q, x[:, :2])
    for cache, y in ((k, x[:, 2]), (v, x[:, 3])):
        assert torch.equal(cache[slots.long() // 4, 0, slots.long() % 4], y) and bool((cache[[0, 1, 1], 0, [2, 0, 2]] == 7.0).all())
    assert hip.cache_append(x[:0, :2], x[:0, 2:3], x[:0, 3:], None, slots[:0], k, v).shape == (0, 2, 128)
    with pytest.raises(hip.OnhipError):
        hip.cache_append(x[:, :2], x[:, 2:3], x[:, 3:], None, slots, k, v, inv_freq=torch.ones(64, device="cuda"))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_int8_rows_out_of_the_ordinary(dtype):
    hip.init(0)
    x = torch.randn((6, 3, 64)).to(DT[dtype])
    x[0, 1:] = 0.0
    x[1, 1:, 5] = math.inf
    x[2, 1:, 9] = math.nan
    x[3, 1:] *= 2.0 ** -126 if dtype == "bf16" else 2.0 ** -20
    x[4, 1:] = torch.finfo(DT[dtype]).max
    k, v, ks, vs = _cache(1, 1, 8, 64, DT[dtype], True)
    xd = x.cuda()
    hip.cache_append(xd[:, :1], xd[:, 1:2], xd[:, 2:], torch.zeros(6, dtype=torch.int32, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda"), k, v, k_scale=ks, v_scale=vs)
    table, lengths = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.full((1,), 6, dtype=torch.int32, device="cuda")
    back = [t[0, 0].double().cpu() for t in hip.cache_read(k, v, table, lengths, 6, k_scale=ks, v_scale=vs, dtype=DT[dtype])]
    for i, (scale, y) in enumerate(zip((ks, vs), back)):
        s, ref = scale[0, 0].cpu(), x[:, 1 + i].double()
        assert s[0] == 0 and bool(s[1:3].isnan().all()) and not y[0].any() and bool(y[1:3].isnan().all())
        for row in (3, 4, 5):
            top = float(ref[row].abs().max())
            step = top / 127
            # half a step of 127, half a step of the type; the smallest rows' scales are denormal: a unit of 2^-149, 127 times
            assert bool(((y[row] - ref[row]).abs() <= step * 0.501 + kv_oracle.HALF[DT[dtype]] * ref[row].abs() * 1.01 + 128 * 2.0 ** -149 + (2.0 ** -25 if dtype == "f16" else 2.0 ** -134)).all()), row


def test_in_place_and_strides():
    hip.init(0)
    t, hq, hkv, hd = 20, 4, 2, 64
    g = torch.Generator().manual_seed(3)
    rows = torch.randn((t, (hq + 2 * hkv) * hd + 24), generator=g).half().cuda()
    q, k, v = (rows[:, a * hd:b * hd].unflatten(1, (b - a, hd)) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    # a cache stored [pages, page_tokens, heads, dim], int8, scales with the heads last
    kc, vc = (torch.zeros((4, 8, hkv, hd), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((4, 8, hkv), device="cuda") for _ in range(2))
    view = lambda x: x.transpose(1, 2)  # noqa: E731
    slots, positions = torch.arange(t, dtype=torch.int32, device="cuda"), torch.arange(t, dtype=torch.int32, device="cuda")
    freq = torch.rand(32, device="cuda")
    plain = _cache(4, hkv, 8, hd, torch.float16, True)
    want = hip.cache_append(q, k, v, positions, slots, plain[0], plain[1], inv_freq=freq, k_scale=plain[2], v_scale=plain[3])
    left = rows[:, hq * hd:].clone()
    got = hip.cache_append(q, k, v, positions, slots, view(kc), view(vc), inv_freq=freq, k_scale=view(ks), v_scale=view(vs), q_out=q)
    torch.cuda.synchronize()
    assert got.data_ptr() == rows.data_ptr() and torch.equal(got, want) and torch.equal(rows[:, hq * hd:], left)
    for a, b in ((view(kc), plain[0]), (view(vc), plain[1]), (view(ks), plain[2]), (view(vs), plain[3])):
        assert torch.equal(a.reshape(4, hkv, 8, -1)[:2], b.reshape(4, hkv, 8, -1)[:2]) and torch.equal(a.reshape(4, hkv, 8, -1)[2, :, :4], b.reshape(4, hkv, 8, -1)[2, :, :4])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("batch,heads,hd,page,tokens", [(1, 1, 64, 1, 1), (3, 2, 128, 8, 100), (5, 3, 64, 16, 333), (2, 8, 128, 64, 129), (70, 1, 64, 2, 9)])
def test_read(dtype, int8, batch, heads, hd, page, tokens):
    hip.init(0)
    print(dtype, int8, batch, heads, hd, page, tokens, flush=True)
    g = torch.Generator().manual_seed(tokens)
    per = (tokens + page - 1) // page
    pages = batch * per + 1
    shape = (pages, heads, page, hd)
    if int8:
        cache = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2)] + [torch.rand(shape[:3], generator=g) * 0.02 for _ in range(2)]
    else:
        cache = [torch.randn(shape, generator=g).to(DT[dtype]) for _ in range(2)] + [None, None]
    table = torch.randperm(pages, generator=g)[: batch * per].view(batch, per).int()
    lengths = torch.randint(0, tokens + 1, (batch,), generator=g).int()
    lengths[0] = tokens
    if batch > 2:
        lengths[1], lengths[2] = -5, tokens + 50     # more than asked for: the rest is not
        table[2, 0] = pages                           # a page that does not exist
    dev = [None if t is None else t.cuda() for t in cache]
    outs = [torch.full((batch, heads, tokens + 3, hd + 8), 7.0, dtype=DT[dtype], device="cuda") for _ in range(2)]
    got = hip.cache_read(dev[0], dev[1], table.cuda(), lengths.cuda(), tokens, k_scale=dev[2], v_scale=dev[3], k_out=outs[0][:, :, :tokens, :hd], v_out=outs[1][:, :, :tokens, :hd])
    torch.cuda.synchronize()
    for o in outs:
        assert bool((o[:, :, tokens:] == 7.0).all()) and bool((o[..., hd:] == 7.0).all())
    for i, x in enumerate(got):
        for b in range(batch):
            n = min(max(int(lengths[b]), 0), tokens)
            y = x[b].double().cpu()
            assert not y[:, n:].any()
            bad = b == 2 and batch > 2
            t = table[b].clone()
            if bad:
                t[0] = 0
            ref = kv_oracle.rows(cache[i], cache[2 + i], t, n)
            if bad:
                assert bool(y[:, : min(page, n)].isnan().all())
                y, ref = y[:, page:n], ref[:, page:]
            else:
                y = y[:, :n]
            low = 2.0 ** -25 if dtype == "f16" else 0.0
            assert bool(((y - ref).abs() <= (kv_oracle.HALF[DT[dtype]] * 1.01 * ref.abs() + low if int8 else 0.0)).all())


def test_read_past_the_table():
    hip.init(0)
    k, v, _, _ = _cache(4, 1, 8, 64, torch.float16, False)
    table, lengths = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2), torch.full((1,), 20, dtype=torch.int32, device="cuda")
    a, b = hip.cache_read(k, v, table, lengths, 24)
    torch.cuda.synchronize()
    for x in (a, b):
        assert bool((x[0, 0, :16] == 7.0).all()) and bool(x[0, 0, 16:20].isnan().all()) and not x[0, 0, 20:].any()


def test_refusals():
    hip.init(0)
    k, v, _, _ = _cache(4, 2, 8, 64, torch.float16, False)
    i8 = _cache(4, 2, 8, 64, torch.float16, True)
    x = torch.zeros((3, 6, 64), dtype=torch.float16, device="cuda")
    ints = torch.zeros(3, dtype=torch.int32, device="cuda")
    q, kk, vv = x[:, :2], x[:, 2:4], x[:, 4:]
    bad = [(q.float(), kk, vv, ints, ints, k, v), (q, kk.bfloat16(), vv, ints, ints, k, v), (q, kk[:, :1], vv, ints, ints, k, v), (q, kk, vv, ints.long(), ints, k, v),
           (q, kk, vv, ints[:2], ints, k, v), (q, kk, vv, ints, ints.cpu(), k, v), (q, kk, vv, ints, ints, k, v[:2]), (q, kk, vv, ints, ints, i8[0], i8[1]),
           (q, kk, vv, ints, ints, k, i8[1]), (q.transpose(0, 2), kk, vv, ints, ints, k, v), (q, kk, vv, torch.stack([ints, ints], 1)[:, 0], ints, k, v)]
    for args in bad:
        with pytest.raises(hip.OnhipError):
            hip.cache_append(*args)
    for kw in (dict(k_scale=i8[2], v_scale=i8[3]), dict(q_weight=torch.ones(32, device="cuda")), dict(inv_freq=torch.ones(12, device="cuda")), dict(inv_freq=torch.ones(32, device="cuda").double()),
               dict(q_out=torch.zeros((3, 2, 64), device="cuda")), dict(q_out=torch.zeros((1, 2, 64), device="cuda").half().expand(3, 2, 64))):
        with pytest.raises(hip.OnhipError):
            hip.cache_append(q, kk, vv, ints, ints, k, v, **kw)
    table = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    for args in ((k, v, table.long(), ints, 4), (k, v, table, ints[:2], 4), (k, v, table.t(), ints[:2], 4), (i8[0], i8[1], table, ints, 4)):
        with pytest.raises(hip.OnhipError):
            hip.cache_read(*args)
    with pytest.raises(hip.OnhipError):
        hip.cache_read(i8[0], i8[1], table, ints, 4, k_scale=i8[2], v_scale=i8[3])     # in which type?
