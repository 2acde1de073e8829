"""Attention of prompts against 64 bits: lengths around the tiles of 32 and 64 keys and of 128 rows, shared heads, masks that leave rows empty, capped and
biased scores, values that are no numbers in unseen places, strides, parts of the keys, streams and graphs."""
import math

import pytest
import torch

import kv_oracle
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _inputs(b, hq, hkv, tq, tk, hd, dtype, seed=0):
    g = torch.Generator().manual_seed(1000 * tq + tk + seed)
    q = torch.randn((b, tq, hq, hd), generator=g).to(dtype)
    k, v = (torch.randn((b, tk, hkv, hd), generator=g).to(dtype) for _ in range(2))
    return [x.permute(0, 2, 1, 3) for x in (q, k, v)]


def _check(q, k, v, got, scale, causal, window, cap, slopes, q_offset, ranges):
    b, hq, tq, hd = q.shape
    got = got.double().cpu().view(b, tq, hq, hd).permute(0, 2, 1, 3)
    for i in range(b):
        seen, away = kv_oracle.seen_by(tq, k.shape[2], causal, window, q_offset, None if ranges is None else ranges[i])
        ref, bound = kv_oracle.attention(q[i], k[i], v[i], seen, scale, cap, slopes, away)
        err = (got[i] - ref).abs()
        assert bool((err <= bound).all()), (i, float((err / bound.clamp(min=1e-30)).max()))
        assert not got[i][:, ~seen.any(1)].any()


def _run(dtype, b, hq, hkv, tq, tk, hd, scale=None, causal=True, window=0, cap=0.0, bias=False, q_offset=None, ranges=None):
    hip.init(0)
    scale = hd ** -0.5 if scale is None else scale
    print(dtype, b, hq, hkv, tq, tk, hd, scale, causal, window, cap, bias, q_offset, flush=True)
    q, k, v = _inputs(b, hq, hkv, tq, tk, hd, DT[dtype])
    slopes = 2.0 ** (-torch.arange(1, hq + 1).float()) if bias else None
    dev = lambda x: None if x is None else x.cuda()  # noqa: E731
    got = hip.attention_masked(dev(q), dev(k), dev(v), scale=scale, causal=causal, window=window, softcap=cap, slopes=dev(slopes), ranges=dev(ranges), q_offset=q_offset)
    torch.cuda.synchronize()
    _check(q, k, v, got, scale, causal, window, cap, slopes, tk - tq if q_offset is None else q_offset, ranges)


SHAPES = [(1, 1, 1, 1, 1), (2, 3, 1, 1, 63), (1, 4, 2, 31, 32), (2, 2, 2, 32, 33), (1, 6, 2, 33, 64), (1, 5, 1, 43, 65), (2, 3, 3, 127, 127), (1, 2, 1, 128, 129),
          (1, 8, 8, 129, 200), (1, 12, 4, 200, 321), (3, 1, 1, 257, 257), (1, 16, 1, 17, 1111), (1, 7, 1, 3, 5000), (8, 2, 1, 300, 300)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("b,hq,hkv,tq,tk", SHAPES)
def test_causal(dtype, hd, b, hq, hkv, tq, tk):
    _run(dtype, b, hq, hkv, tq, tk, hd)


# more than one workgroup a compute unit: 128 rows each, heads divided among the XCDs and not
MANY = [(33, 16, 8, 130, 200, 64), (37, 14, 7, 70, 65, 128), (300, 1, 1, 33, 70, 64), (9, 32, 32, 129, 129, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("i", range(len(MANY)))
def test_many_rows(dtype, i):
    b, hq, hkv, tq, tk, hd = MANY[i]
    _run(dtype, b, hq, hkv, tq, tk, hd)
    _run(dtype, b, hq, hkv, tq, tk, hd, window=40, cap=20.0, bias=i % 2 == 0)
    g = torch.Generator().manual_seed(i)
    edge = torch.randint(-20, tk + 20, (b, tq, 2), generator=g, dtype=torch.int32)
    _run(dtype, b, hq, hkv, tq, tk, hd, causal=i % 2 == 0, ranges=edge, q_offset=tk // 2)


# workgroups of 256 rows: a block of heads of one key-value head that is (nearly) 256 rows, and 448 to 512 or 1792 to 2048 of them
WIDE = [(56, 8, 8, 250, 300), (61, 16, 8, 128, 77), (4, 32, 8, 1001, 1001), (30, 30, 15, 128, 400), (120, 16, 16, 256, 70)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("i", range(len(WIDE)))
def test_blocks_of_256_rows(dtype, i):
    b, hq, hkv, tq, tk = WIDE[i]
    _run(dtype, b, hq, hkv, tq, tk, 128, causal=i % 2 == 0)
    if i == 2:
        _run(dtype, b, hq, hkv, tq, tk, 128, bias=True)
        return
    _run(dtype, b, hq, hkv, tq, tk, 128, window=40, cap=20.0, bias=i % 2 == 0)
    _run(dtype, b, hq, hkv, tq, tk, 128, bias=True, window=0 if i else 90)
    g = torch.Generator().manual_seed(i)
    edge = torch.randint(-20, tk + 20, (b, tq, 2), generator=g, dtype=torch.int32)
    _run(dtype, b, hq, hkv, tq, tk, 128, causal=i % 2 == 0, ranges=edge, q_offset=tk // 2)


# the last tokens of a long prompt: 256 rows a workgroup, keys in parts that a group of lanes joins by itself
CHUNKS = [(1, 32, 8, 500, 4000), (1, 16, 8, 256, 6000), (2, 8, 1, 130, 11000), (1, 32, 8, 700, 4300)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("i", range(len(CHUNKS)))
def test_chunks_behind_many_keys(dtype, i):
    b, hq, hkv, tq, tk = CHUNKS[i]
    _run(dtype, b, hq, hkv, tq, tk, 128)
    _run(dtype, b, hq, hkv, tq, tk, 128, bias=True, causal=i % 2 == 0)
    _run(dtype, b, hq, hkv, tq, tk, 128, window=tk - 600, cap=20.0)
    edge = torch.randint(-20, tk + 20, (b, tq, 2), generator=torch.Generator().manual_seed(i), dtype=torch.int32)
    _run(dtype, b, hq, hkv, tq, tk, 128, causal=False, ranges=edge)


def test_scores_above_half_of_the_cap():
    """capped by a polynomial below, by an exponential above"""
    for scale in (0.05, 0.3, 1.0, 5.0, -2.0):
        _run("f16", 1, 2, 1, 64, 130, 64, scale=scale, cap=6.0)
        _run("bf16", 60, 16, 8, 100, 130, 128, scale=scale, cap=6.0, causal=False)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_cap_far_above_the_scores(dtype):
    """is no cap: s - cap tanh(s / cap) = s^3 / (3 cap^2) is 10^-8 at most here, and the polynomial's 2.4 10^-6 |s| are within the bound's allowance
    for a score, hd 2^-24 sum |q k| scale"""
    hip.init(0)
    q, k, v = _inputs(2, 4, 2, 50, 200, 64, DT[dtype])
    for cap in (1e6, 1e25):
        got = hip.attention_masked(q.cuda(), k.cuda(), v.cuda(), scale=0.125, causal=True, softcap=cap)
        torch.cuda.synchronize()
        _check(q, k, v, got, 0.125, True, 0, 0.0, None, 150, None)


@pytest.mark.parametrize("hq,hkv", [(2, 2), (16, 4)])
def test_a_rows_bits_are_its_own(hq, hkv):
    """whatever the scores of the rows beside it are"""
    hip.init(0)
    q, k, v = (x.cuda() for x in _inputs(1, hq, hkv, 100, 300, 64, torch.bfloat16))
    more = q.clone()
    more[:, 1::2] *= 40
    more[:, :, 1::2] *= 40
    for cap in (0.0, 8.0):
        a, b = (hip.attention_masked(x, k, v, scale=0.125, causal=True, softcap=cap, merged_out=False) for x in (q, more))
        torch.cuda.synchronize()
        assert torch.equal(a[:, ::2, ::2], b[:, ::2, ::2]) and not torch.equal(a, b)


@pytest.mark.parametrize("scale", [1e-5, 1e-7, -0.02, 30.0])
@pytest.mark.parametrize("causal", [True, False])
def test_biases_next_to_small_and_large_scales(causal, scale):
    for dtype, hd in (("bf16", 64), ("f16", 128)):
        _run(dtype, 2, 4, 2, 200, 300, hd, scale=scale, causal=causal, bias=True, window=150)
        _run(dtype, 3, 16, 16, 700, 700, hd, scale=scale, causal=causal, bias=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_slopes_that_leave_one_key(dtype):
    """with slopes from 200 on a key's probability is below 2^-280 of the next one's (scores differ by less than 10): the row's own place alone"""
    hip.init(0)
    q, k, v = _inputs(1, 4, 2, 90, 90, 64, DT[dtype])
    slopes = torch.tensor([200.0, 1e10, 1e30, 3e37])
    got = hip.attention_masked(q.cuda(), k.cuda(), v.cuda(), scale=0.01, causal=True, slopes=slopes.cuda(), merged_out=False)
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), v.repeat_interleave(2, dim=1))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,merged", [(100, 1), (100, 30)])
def test_scores_of_any_size(dtype, tokens, merged):
    """a row's largest score lies 10^9 above the next one: its own key alone, beside rows of ordinary scores"""
    hip.init(0)
    q, k, v = _inputs(merged, 16, 8, tokens, tokens, 64, DT[dtype])
    q[:, ::2] = 0.0
    q[:, ::2, :, 0] = 60000.0
    k[..., 0] = torch.arange(tokens) * 512.0    # a number of seven bits
    q[:, 1::2, :, 0] = 0.0
    for bias in (None, torch.full((16,), 1.0)):
        got = hip.attention_masked(q.cuda(), k.cuda(), v.cuda(), scale=40.0, causal=True, slopes=None if bias is None else bias.cuda(), merged_out=False)
        torch.cuda.synchronize()
        assert torch.equal(got[:, ::2].cpu(), v)
        assert bool(got.isfinite().all())
        even = torch.arange(0, 16, 2)
        seen, away = kv_oracle.seen_by(tokens, tokens, True, 0, 0)
        ref, bound = kv_oracle.attention(q[0, even + 1], k[0], v[0], seen, 40.0, 0.0, None if bias is None else bias[even + 1], away)
        assert bool(((got[0, even + 1].double().cpu() - ref).abs() <= bound).all())


def test_scores_a_step_of_fp32_apart():
    """the next number above a score may be farther away than a probability's room above the reference point"""
    hip.init(0)
    q, k, v = (torch.zeros((1, n, 192, 64), dtype=torch.float16) for n in (2, 1, 1))
    v += torch.randn(v.shape, generator=torch.Generator().manual_seed(1)).half()
    q[..., 0], q[..., 1] = 2048.0, 8.0
    k[:, :, 64:128, 1], k[:, :, 128:, 1] = 1.0, 3.0
    for at in range(30016, 60000, 1504):
        k[..., 0] = at
        for slopes in (None, torch.zeros(2).cuda()):
            got = hip.attention_masked(q.cuda(), k.cuda(), v.cuda(), scale=1.0, causal=slopes is not None, slopes=slopes)
            torch.cuda.synchronize()
            assert bool((got.abs().cpu() <= v.abs().max()).all()), at


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_many_parts(dtype):
    _run(dtype, 1, 1, 1, 1, 70000, 64)
    _run(dtype, 1, 2, 1, 5, 33333, 128, window=20000)


def test_no_keys():
    hip.init(0)
    q = torch.randn((2, 4, 9, 64), device="cuda").half()
    k = torch.empty((2, 2, 0, 64), device="cuda", dtype=torch.float16)
    got = hip.attention_masked(q, k, k, causal=True)
    torch.cuda.synchronize()
    assert got.shape == (2, 9, 256) and not got.any()
    for empty in (q[:0], q[:, :, :0]):
        assert hip.attention_masked(empty, q[: empty.shape[0], :2], q[: empty.shape[0], :2]).numel() == 0


MORE = [dict(causal=False), dict(scale=0.0), dict(scale=-0.3, causal=False), dict(window=1), dict(window=37), dict(window=64, causal=False), dict(cap=3.0), dict(cap=50.0, window=100),
        dict(bias=True), dict(bias=True, causal=False), dict(bias=True, cap=5.0, window=90), dict(q_offset=-20), dict(q_offset=0), dict(q_offset=500, window=300),
        dict(q_offset=1000, window=100), dict(q_offset=-400), dict(scale=3.0)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("i", range(len(MORE)))
def test_masks_caps_and_biases(dtype, i):
    _run(dtype, 2, 4, 2, 150, 210, 64 if i % 2 else 128, **MORE[i])
    _run(dtype, 1, 2, 1, 20, 1500, 128 if i % 2 else 64, **MORE[i])   # in parts


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tq,tk,causal", [(90, 200, False), (260, 260, True), (40, 2500, False)])
def test_ranges(dtype, tq, tk, causal):
    g = torch.Generator().manual_seed(tq)
    edge = torch.randint(-20, tk + 20, (2, tq, 2), generator=g, dtype=torch.int32)   # a third or so of the rows see nothing
    edge[0, 5] = torch.tensor([-2 ** 31, 2 ** 31 - 1])
    edge[0, 6] = torch.tensor([2 ** 31 - 1, -2 ** 31])
    edge[1, : tq // 2] = 7   # begin == end: half of the rows, whole wavefronts of them
    _run(dtype, 2, 4, 2, tq, tk, 64, causal=causal, ranges=edge)
    _run(dtype, 2, 3, 1, tq, tk, 128, causal=causal, ranges=edge, cap=4.0, bias=True)
    documents = torch.tensor([0, 1, 2, 40, 41, 105, tk])
    at = torch.searchsorted(documents, torch.arange(tq) + tk - tq, right=True)
    packed = torch.stack([documents[at - 1], documents[at.clamp(max=6)]], -1).int().expand(2, tq, 2).contiguous()
    _run(dtype, 2, 2, 2, tq, tk, 128, causal=True, ranges=packed)
    _run(dtype, 2, 2, 2, tq, tk, 64, causal=False, ranges=torch.zeros_like(packed))   # nobody sees anything


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tq,tk,b", [(100, 100, 1), (20, 2000, 1), (100, 150, 300), (125, 190, 460), (125, 5200, 32)])
def test_unseen_values(dtype, hd, tq, tk, b):
    """what a row does not see leaves its bits alone, infinities and NaN of k and v included; what it sees does not"""
    hip.init(0)
    print(dtype, hd, tq, tk, b, flush=True)
    q, k, v = [x.cuda() for x in _inputs(b, 2, 1, tq, tk, hd, DT[dtype])]
    if b > 1:
        q, k, v = (x[:1].expand(b, -1, -1, -1) for x in (q, k, v))
    cut = tk - tq // 2      # rows whose place is below see nothing from here on
    clean = hip.attention_masked(q, k, v, causal=True, scale=0.1)[-1].view(tq, 2, hd)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, cut + 1], k2[:, :, cut + 2, 3] = math.nan, math.inf
    v2[:, :, cut, 0], v2[:, :, cut, 1], v2[:, :, cut, 2] = math.inf, -math.inf, math.nan
    v2[:, :, cut + 3, 1] = math.inf
    got = hip.attention_masked(q, k2, v2, causal=True, scale=0.1)[-1].view(tq, 2, hd)
    torch.cuda.synchronize()
    first = cut - (tk - tq)   # the first row that sees key `cut`
    assert torch.equal(got[:first], clean[:first])
    row = got[first].float()
    assert bool((row[:, 0] == math.inf).all()) and bool((row[:, 1] == -math.inf).all()) and bool(row[:, 2].isnan().all())
    err = (row[:, 3:] - clean[first, :, 3:].float()).abs()
    assert float(err.max()) == 0.0          # its k is clean, so the other channels are
    assert bool(got[first + 1:].float().isnan().all())   # a score that is NaN
    # the same with k clean: infinities of both signs in one channel are no number
    got = hip.attention_masked(q, k, v2, causal=True, scale=0.1)[-1].view(tq, 2, hd).float()
    torch.cuda.synchronize()
    assert bool((got[first:first + 3, :, 1] == -math.inf).all()) and bool(got[first + 3:, :, 1].isnan().all())
    assert bool((got[first:, :, 0] == math.inf).all()) and bool(got[first:, :, 2].isnan().all())
    assert torch.equal(got[first:, :, 3:], clean[first:, :, 3:].float())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_largest_values(dtype):
    hip.init(0)
    big = float(torch.finfo(DT[dtype]).max) * 0.98
    q, k = (torch.zeros((1, 1, 700, 64), dtype=DT[dtype], device="cuda") for _ in range(2))
    v = torch.full((1, 1, 700, 64), big, dtype=DT[dtype], device="cuda")
    q[0, 0, :, 0] = 1.0
    k[0, 0, :, 0] = torch.arange(700) / 100.0    # a maximum that moves on slowly
    got = hip.attention_masked(q, k, v, causal=True).float()
    torch.cuda.synchronize()
    assert torch.allclose(got, torch.full_like(got, big), rtol=2e-2)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_strides(dtype):
    hip.init(0)
    b, hq, hkv, t, hd = 2, 6, 2, 77, 64
    g = torch.Generator().manual_seed(9)
    rows = torch.randn((b, t, (hq + 2 * hkv) * hd + 8), generator=g).to(DT[dtype])     # one projection's rows with a pitch
    dev = rows.cuda()
    cut = lambda x, first, n: x[..., first * hd:(first + n) * hd].unflatten(-1, (n, hd)).permute(0, 2, 1, 3)  # noqa: E731
    q, k, v = cut(dev, 0, hq), cut(dev, hq, hkv), cut(dev, hq + hkv, hkv)
    out = torch.full((b, t, hq * hd + 16), 7.0, dtype=DT[dtype], device="cuda")
    assert hip.attention_masked(q, k, v, causal=True, out=out) is out
    torch.cuda.synchronize()
    assert bool((out[..., hq * hd:] == 7.0).all())
    cq, ck, cv = cut(rows, 0, hq), cut(rows, hq, hkv), cut(rows, hq + hkv, hkv)
    _check(cq, ck, cv, out[..., :hq * hd].contiguous(), 1.0, True, 0, 0.0, None, 0, None)
    # heads first, and keys that all heads and sequences share through strides of zero
    out2 = torch.empty((b, hq, t, hd), dtype=DT[dtype], device="cuda")
    ke, ve = (x[:1, :1].expand(b, hkv, t, hd) for x in (k, v))
    hip.attention_masked(q.contiguous(), ke, ve, causal=True, out=out2, merged_out=False)
    torch.cuda.synchronize()
    _check(cq, ck[:1, :1].expand(b, hkv, t, hd), cv[:1, :1].expand(b, hkv, t, hd), out2.permute(0, 2, 1, 3).reshape(b, t, hq * hd), 1.0, True, 0, 0.0, None, 0, None)


def test_far_rows():
    """keys 2 MB apart: offsets that pass 32 bits"""
    hip.init(0)
    q, k, v = _inputs(1, 2, 1, 2600, 2600, 64, torch.bfloat16)
    wide = torch.empty((2600, (1 << 20) + 8), dtype=torch.bfloat16, device="cuda")
    wide[:, :64], wide[:, 64:128] = k[0, 0].cuda(), v[0, 0].cuda()
    got = hip.attention_masked(q.cuda(), wide[None, None, :, :64], wide[None, None, :, 64:128], causal=True, scale=0.125)
    torch.cuda.synchronize()
    _check(q, k, v, got, 0.125, True, 0, 0.0, None, 0, None)


def test_streams_and_graphs():
    hip.init(0)
    sets = [[x.cuda() for x in _inputs(1, 4, 2, 24, 3000, 128, torch.bfloat16, seed=s)] for s in range(2)]   # in parts: each call has its workspace
    call = lambda s: hip.attention_masked(*s, causal=True, scale=0.1)  # noqa: E731
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            outs.append(call(sets[i]))
    for n in range(3):
        for i in range(2):
            for x in sets[i]:
                x.copy_(torch.roll(x, 1, 2))
        graphs[0].replay()
        with torch.cuda.stream(streams[1]):
            streams[1].wait_stream(torch.cuda.default_stream())
            graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], call(sets[i])) for i in range(2))


def test_refusals():
    hip.init(0)
    q, k, v = (x.cuda() for x in _inputs(1, 2, 1, 8, 8, 64, torch.float16))
    for bad in (dict(k=k.bfloat16()), dict(v=v[:, :, :4]), dict(q=q.float()), dict(q=q.cpu()), dict(slopes=torch.zeros(3, device="cuda")),
                dict(slopes=torch.zeros(2, device="cuda").double()), dict(ranges=torch.zeros((1, 8, 2), device="cuda")), dict(ranges=torch.zeros((1, 7, 2), device="cuda", dtype=torch.int32)),
                dict(out=torch.zeros((1, 8, 64), device="cuda").half()), dict(out=torch.zeros((1, 8, 128), device="cuda")), dict(q=q.transpose(2, 3)), dict(q=q[:, :1].expand(1, 3, 8, 64)[:, :3])):
        args = dict(q=q, k=k, v=v)
        kw = {n: x for n, x in bad.items() if n not in args}
        args.update({n: x for n, x in bad.items() if n in args})
        if "q" in bad and bad["q"].shape[1] == 3:   # three query heads for two key-value heads
            args.update(k=k.expand(1, 2, 8, 64), v=v.expand(1, 2, 8, 64))
        with pytest.raises(hip.OnhipError):
            hip.attention_masked(args["q"], args["k"], args["v"], **kw)
