"""Attention of one new token over the paged cache against 64 bits: lengths around tiles, parts and pages, shared heads, windows, caps and biases, int8 caches,
pages that do not exist, values that are no numbers behind the last row, far offsets, streams and graphs; and the operators of a decoder one after the other."""
import math

import pytest
import torch

import kv_oracle
from onenew_amd import hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _case(lengths, hq, hkv, hd, page, dtype, int8, seed=0, spare=0):
    g = torch.Generator().manual_seed(seed + 7 * len(lengths) + hd + page)
    per = max(1, max((max(n, 0) + page - 1) // page for n in lengths)) + spare
    pages = len(lengths) * per + 1
    shape = (pages, hkv, page, hd)
    if int8:
        cache = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2)] + [0.001 + 0.02 * torch.rand(shape[:3], generator=g) for _ in range(2)]
    else:
        cache = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)] + [None, None]
    table = torch.randperm(pages, generator=g)[: len(lengths) * per].view(len(lengths), per).int()
    q = torch.randn((len(lengths), hq, hd), generator=g).to(dtype)
    return q, cache, table, torch.tensor(lengths, dtype=torch.int32)


def _dev(*x):
    return [None if t is None else t.cuda() for t in x]


def _check(got, q, cache, table, lengths, scale, window=0, cap=0.0, slopes=None):
    for b, n in enumerate(lengths.tolist()):
        if n <= 0:
            assert not got[b].any()
            continue
        k, v = (kv_oracle.rows(cache[i], cache[2 + i], table[b], n) for i in range(2))
        away = (n - 1 - torch.arange(n))[None]
        seen = away < window if window else away >= 0
        ref, bound = kv_oracle.attention(q[b][:, None], k, v, seen, scale, cap, slopes, away)
        if cache[2] is not None:   # the scores' and the probabilities' products with the scales, one more rounding each
            bound = bound * 1.1
        err = (got[b].double().cpu() - ref[:, 0]).abs()
        assert bool((err <= bound[:, 0]).all()), (b, n, float((err / bound[:, 0].clamp(min=1e-30)).max()))


def _run(dtype, int8, lengths, hq, hkv, hd, page, scale=None, window=0, cap=0.0, bias=False, spare=0):
    hip.init(0)
    scale = hd ** -0.5 if scale is None else scale
    print(dtype, int8, lengths, hq, hkv, hd, page, scale, window, cap, bias, flush=True)
    q, cache, table, n = _case(lengths, hq, hkv, hd, page, DT[dtype], int8, spare=spare)
    slopes = 2.0 ** (-torch.arange(1, hq + 1).float() / 2) if bias else None
    k, v, ks, vs = _dev(*cache)
    got = hip.attention_paged(q.cuda(), k, v, table.cuda(), n.cuda(), scale=scale, window=window, softcap=cap, slopes=_dev(slopes)[0], k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    _check(got, q, cache, table, n, scale, window, cap, slopes)


SHAPES = [([1], 1, 1, 1), ([0, 1, 2], 2, 1, 1), ([31, 32, 33, 0, -7], 3, 3, 2), ([15, 16, 17, 127, 128, 129], 6, 2, 4), ([500], 8, 1, 8), ([777, 3], 16, 1, 16),
          ([1000, 1, 513], 34, 2, 32), ([64, 4097], 40, 1, 64), ([2000] * 3, 4, 4, 1024), ([300] * 40, 12, 12, 16), ([9000, 100], 5, 5, 128),
          ([70001], 1, 1, 256), ([33000, 1, 12345], 2, 1, 8)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lengths,hq,hkv,page", SHAPES)
def test_lengths(dtype, int8, hd, lengths, hq, hkv, page):
    _run(dtype, int8, lengths, hq, hkv, hd, page)


MORE = [dict(scale=0.0), dict(scale=-0.4), dict(scale=2.0), dict(window=1), dict(window=33), dict(window=1000), dict(window=100000), dict(cap=3.0), dict(cap=30.0, window=200),
        dict(bias=True), dict(bias=True, cap=10.0, window=150), dict(spare=300)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("i", range(len(MORE)))
def test_windows_caps_and_biases(dtype, int8, i):
    _run(dtype, int8, [0, 1, 32, 70, 333, 1500], 6, 2, 128 if i % 2 else 64, [4, 16, 64][i % 3], **MORE[i])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("int8", [False, True])
def test_a_cap_far_above_the_scores(dtype, int8):
    """is no cap: s - cap tanh(s / cap) = s^3 / (3 cap^2) is 10^-8 at most here, and the polynomial's 2.4 10^-6 |s| are within the bound's allowance
    for a score, hd 2^-24 sum |q k| scale; and a head's bits do not depend on the scores of the heads beside it"""
    hip.init(0)
    q, cache, table, n = _case([1, 70, 1500], 6, 2, 64, 16, DT[dtype], int8)
    k, v, ks, vs = _dev(*cache)
    run = lambda q, cap: hip.attention_paged(q.cuda(), k, v, table.cuda(), n.cuda(), scale=0.125, softcap=cap, k_scale=ks, v_scale=vs)
    for cap in (1e6, 1e25):
        got = run(q, cap)
        torch.cuda.synchronize()
        _check(got, q, cache, table, n, 0.125)
    more = q.clone()
    more[:, 1::2] *= 40
    a, b = run(q, 8.0), run(more, 8.0)
    torch.cuda.synchronize()
    assert torch.equal(a[:, ::2], b[:, ::2]) and not torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_slopes_that_leave_one_key(dtype):
    """with slopes from 200 on a key's probability is below 2^-280 of the next one's (scores differ by less than 10): the new token's alone"""
    hip.init(0)
    q, cache, table, n = _case([1, 70, 1500], 6, 2, 64, 16, DT[dtype], False)
    k, v = _dev(*cache[:2])
    slopes = torch.tensor([200.0, 1e10, 1e30, 3e37, 3e38, 300.0])
    got = hip.attention_paged(q.cuda(), k, v, table.cuda(), n.cuda(), scale=0.01, slopes=slopes.cuda())
    torch.cuda.synchronize()
    for b, m in enumerate(n.tolist()):
        assert torch.equal(got[b].double().cpu(), kv_oracle.rows(cache[1], None, table[b], m)[:, -1].repeat_interleave(3, dim=0))


def test_scores_a_step_of_fp32_apart():
    """the next number above a score may be farther away than a probability's room above the reference point"""
    hip.init(0)
    q, cache, table, n = _case([1000], 2, 1, 64, 16, torch.float16, False)
    k, v = _dev(*cache[:2])
    q.zero_()
    q[..., 0], q[..., 1] = 2048.0, 8.0
    for at in range(30016, 60000, 1504):
        k.zero_()
        k[..., 0] = at
        k[..., 1] = torch.arange(k.shape[0], device="cuda")[:, None, None] % 7    # a page's rows alike
        got = hip.attention_paged(q.cuda(), k, v, table.cuda(), n.cuda(), scale=1.0)
        torch.cuda.synchronize()
        assert bool((got.abs() <= v.abs().max() * (1 + 2.0 ** -10)).all()), at   # probabilities rounded to fp16 over a sum that is not


def test_no_pages():
    hip.init(0)
    q, cache, _, _ = _case([5, 5], 4, 2, 64, 16, torch.float16, False)
    k, v, _, _ = _dev(*cache)
    table, n = torch.empty((2, 0), dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    got = hip.attention_paged(q.cuda(), k, v, table, n)
    a, b = hip.cache_read(k, v, table, n, 4)
    torch.cuda.synchronize()
    assert not got[0].any() and bool(got[1].isnan().all())
    for x in (a, b):
        assert not x[0].any() and bool(x[1, :, :3].isnan().all()) and not x[1, :, 3:].any()
    assert hip.attention_paged(q.cuda()[:0], k, v, table[:0], n[:0]).numel() == 0


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("page", [2, 16, 64])
def test_pages_that_do_not_exist(int8, page):
    hip.init(0)
    print(int8, page, flush=True)
    q, cache, table, n = _case([100, 100, 100, 1000, 900, 100], 4, 2, 64, page, torch.float16, int8)
    want_table = table.clone()
    pages = cache[0].shape[0]
    table[1, 0], table[2, 99 // page], table[3, 500 // page] = -1, pages, 2 ** 31 - 1
    table[4, (n[4] + page - 1) // page:] = -2 ** 31    # behind the last row: not looked at
    n[5] = 16 * table.shape[1] * page                   # longer than its table
    k, v, ks, vs = _dev(*cache)
    got = hip.attention_paged(q.cuda(), k, v, table.cuda(), n.cuda(), scale=0.1, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert bool(got[[1, 2, 3, 5]].float().isnan().all())
    keep = [0, 4]
    _check(got[keep], q[keep], cache, want_table[keep], n[keep], 0.1)
    # outside of the window, pages are not looked at either
    got = hip.attention_paged(q.cuda(), k, v, table.cuda(), n.cuda(), scale=0.1, window=30, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert bool(got[[2, 5]].float().isnan().all())
    keep = [0, 1, 3, 4]
    _check(got[keep], q[keep], cache, want_table[keep], n[keep], 0.1, window=30)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("page", [4, 32])
def test_rows_behind_the_last(int8, page):
    """rows that no sequence has yet, and rows before the window, may hold anything"""
    hip.init(0)
    q, cache, table, n = _case([5, 45, 1000], 4, 2, 128, page, torch.bfloat16, int8)
    k, v, ks, vs = _dev(*cache)
    run = lambda w: hip.attention_paged(q.cuda(), k, v, table.cuda(), n.cuda(), scale=0.1, window=w, k_scale=ks, v_scale=vs)  # noqa: E731
    want = [run(0), run(20)]
    for b in range(3):
        for at in range(int(n[b]), (int(n[b]) + page - 1) // page * page):
            for t in (ks, vs) if int8 else (k, v):
                t[int(table[b, at // page]), :, at % page] = math.nan if at % 2 else math.inf
    got = run(0)
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    for b in range(3):
        for at in range(0, int(n[b]) - 20):
            for t in (ks, vs) if int8 else (k, v):
                t[int(table[b, at // page]), :, at % page] = math.nan if at % 2 else -math.inf
    got = run(20)
    torch.cuda.synchronize()
    assert torch.equal(got, want[1])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_out_of_the_ordinary(dtype):
    hip.init(0)
    q, cache, table, n = _case([200], 2, 1, 64, 16, DT[dtype], False)
    k, v, _, _ = _dev(*cache)
    big = float(torch.finfo(DT[dtype]).max) * 0.98
    run = lambda: hip.attention_paged(q.cuda(), k, v, table.cuda(), n.cuda(), scale=0.1).float()  # noqa: E731
    v[:] = big
    got = run()
    assert torch.allclose(got, torch.full_like(got, big), rtol=2e-2)
    v[:] = 1.0
    page = int(table[0, 3])
    v[page, 0, 1, 0], v[page, 0, 2, 1], v[page, 0, 3, 2] = math.inf, -math.inf, math.nan
    got = run()
    assert bool((got[..., 0] == math.inf).all()) and bool((got[..., 1] == -math.inf).all()) and bool(got[..., 2].isnan().all()) and torch.allclose(got[..., 3:], torch.ones_like(got[..., 3:]), rtol=1e-2)
    k[page, 0, 5, 7] = math.nan
    assert bool(run().isnan().all())


def test_small_scales_in_fp16():
    """scales of 10^-6 and of 30 next to each other: a probability times its scale keeps eleven bits"""
    hip.init(0)
    for least, most in ((1e-6, 2e-6), (1e-6, 30.0), (0.0, 1e-6)):
        q, cache, table, n = _case([700, 40], 4, 2, 64, 16, torch.float16, True)
        cache[3] = least + (most - least) * torch.rand(cache[3].shape) ** 4
        k, v, ks, vs = _dev(*cache)
        got = hip.attention_paged(q.cuda(), k, v, table.cuda(), n.cuda(), scale=0.1, k_scale=ks, v_scale=vs)
        torch.cuda.synchronize()
        _check(got, q, cache, table, n, 0.1)


def test_strides_and_far_pages():
    """pages 8 GB apart, the heads inside the rows, a table with a pitch, results with one"""
    hip.init(0)
    hq, hkv, hd, page = 4, 2, 128, 16
    lengths = [100, 40]
    q, cache, table, n = _case(lengths, hq, hkv, hd, page, torch.bfloat16, False)
    pages = cache[0].shape[0]
    room = torch.empty((pages, 1 << 30), dtype=torch.bfloat16, device="cuda")   # 2 GB a page
    views = []
    for i in range(2):
        x = room[:, i * (1 << 20): i * (1 << 20) + page * hkv * hd].unflatten(1, (page, hkv, hd)).transpose(1, 2)
        x.copy_(cache[i].cuda())
        views.append(x)
    wide = torch.full((2, table.shape[1] + 5), 10 ** 9, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table.cuda()
    out = torch.full((2, hq, hd + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    qd = torch.zeros((2, hq + 3, hd + 8), dtype=torch.bfloat16, device="cuda")
    qd[:, :hq, :hd] = q.cuda()
    hip.attention_paged(qd[:, :hq, :hd], views[0], views[1], wide[:, : table.shape[1]], n.cuda(), scale=0.1, out=out[..., :hd])
    torch.cuda.synchronize()
    assert bool((out[..., hd:] == 7.0).all())
    _check(out[..., :hd], q, cache, table, n, 0.1)


def test_streams_and_graphs():
    hip.init(0)
    sets = [_case([3000, 17, 2900], 8, 2, 128, 16, torch.bfloat16, False, seed=s) for s in range(2)]
    dev = [(q.cuda(), *_dev(*cache)[:2], table.cuda(), n.cuda()) for q, cache, table, n in sets]
    call = lambda i: hip.attention_paged(*dev[i], scale=0.1)  # noqa: E731
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    for step in range(3):
        for i in range(2):
            dev[i][4].copy_(torch.tensor([2500 + step, 40 * step, 2999 - 700 * step]))     # a replay reads the lengths as they are then
        graphs[0].replay()
        with torch.cuda.stream(streams[1]):
            streams[1].wait_stream(torch.cuda.default_stream())
            graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], call(i)) for i in range(2))


def test_refusals():
    hip.init(0)
    q, cache, table, n = _case([10, 20], 4, 2, 64, 16, torch.float16, False)
    k, v, _, _ = _dev(*cache)
    q, table, n = q.cuda(), table.cuda(), n.cuda()
    for args in ((q.float(), k, v, table, n), (q.bfloat16(), k, v, table, n), (q[..., :32], k, v, table, n), (q[:1], k, v, table, n), (q, k, v, table.long(), n), (q, k, v, table, n.long()),
                 (q, k, v, table, n.cpu()), (q[:, :3], k, v, table, n), (q, k[..., :32], v[..., :32], table, n)):
        with pytest.raises(hip.OnhipError):
            hip.attention_paged(*args)
    for kw in (dict(slopes=torch.zeros(3, device="cuda")), dict(out=torch.zeros((2, 4, 64), device="cuda")), dict(window=-1), dict(softcap=-1.0), dict(softcap=math.nan)):
        with pytest.raises(hip.OnhipError):
            hip.attention_paged(q, k, v, table, n, **kw)


@pytest.mark.parametrize("dtype,int8", [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)])
def test_a_decoder(dtype, int8):
    """one attention layer of a decoder: two prompts of 70 and 33 tokens, a second chunk of the first one on its cached keys, then five steps of both, every
    result against the whole sequence's attention in 64 bits"""
    hip.init(0)
    hq, hkv, hd, page, total = 6, 2, 64, 16, (100, 33)
    g = torch.Generator().manual_seed(5)
    steps = 5
    x = [torch.randn((n + steps, hq + 2 * hkv, hd), generator=g).to(DT[dtype]) for n in total]
    qw, kw = (torch.rand(hd, generator=g) + 0.5 for _ in range(2))
    freq = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float()
    per = 8
    table = torch.randperm(2 * per, generator=g).view(2, per).int()
    shape = (2 * per, hkv, page, hd)
    if int8:
        k, v = (torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2))
        scales = dict(k_scale=torch.zeros(shape[:3], device="cuda"), v_scale=torch.zeros(shape[:3], device="cuda"))
    else:
        k, v = (torch.zeros(shape, dtype=DT[dtype], device="cuda") for _ in range(2))
        scales = {}
    qwd, kwd, fd, td = qw.cuda(), kw.cuda(), freq.cuda(), table.cuda()

    def append(pieces):      # (sequence, first, last) one behind the other
        rows = torch.cat([x[s][a:b] for s, a, b in pieces]).cuda()
        place = torch.cat([torch.arange(a, b) for _, a, b in pieces])
        slots = torch.cat([table[s].long()[torch.arange(a, b) // page] * page + torch.arange(a, b) % page for s, a, b in pieces])
        return hip.cache_append(rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:], place.int().cuda(), slots.int().cuda(), k, v, inv_freq=fd, q_weight=qwd, k_weight=kwd, **scales)

    results = [[], []]
    # the prompts' first chunks in one packed batch: documents
    q = append([(0, 0, 70), (1, 0, 33)])
    lengths = torch.tensor([70, 33], dtype=torch.int32, device="cuda")
    kk, vv = hip.cache_read(k, v, td, lengths, 70, dtype=DT[dtype], **scales)
    packed_k, packed_v = (torch.cat([t[0, :, :70], t[1, :, :33]], 1)[None] for t in (kk, vv))
    ranges = torch.tensor([[0, 70]] * 70 + [[70, 103]] * 33, dtype=torch.int32, device="cuda")[None]
    o = hip.attention_masked(q.permute(1, 0, 2)[None], packed_k, packed_v, scale=hd ** -0.5, causal=True, ranges=ranges).view(103, hq, hd)
    results[0].append(o[:70])
    results[1].append(o[70:])
    # the second chunk of the first prompt
    q = append([(0, 70, 100)])
    kk, vv = hip.cache_read(k, v, td[:1], torch.full((1,), 100, dtype=torch.int32, device="cuda"), 100, dtype=DT[dtype], **scales)
    results[0].append(hip.attention_masked(q.permute(1, 0, 2)[None], kk, vv, scale=hd ** -0.5, causal=True).view(30, hq, hd))
    for step in range(steps):
        q = append([(s, total[s] + step, total[s] + step + 1) for s in range(2)])
        lengths = torch.tensor([total[s] + step + 1 for s in range(2)], dtype=torch.int32, device="cuda")
        o = hip.attention_paged(q, k, v, td, lengths, scale=hd ** -0.5, **scales)
        for s in range(2):
            results[s].append(o[s:s + 1])
    torch.cuda.synchronize()
    half = kv_oracle.HALF[DT[dtype]]
    for s in range(2):
        n = total[s] + steps
        place = torch.arange(n)
        ref_q, _ = kv_oracle.turned(x[s][:, :hq], qw, place, freq, 1e-6, False)
        ref_k, _ = kv_oracle.turned(x[s][:, hq:hq + hkv], kw, place, freq, 1e-6, False)
        ref_v = x[s][:, hq + hkv:].double()
        seen, away = kv_oracle.seen_by(n, n, True, 0, 0)
        got = torch.cat(results[s]).double().cpu()
        for h in range(hq):
            a, b, c = ref_q[:, h], ref_k[:, h // 3], ref_v[:, h // 3]
            p = torch.softmax(torch.where(seen, (a @ b.t()) * hd ** -0.5, -math.inf), 1)
            ref, mass = p @ c, p @ c.abs()
            # what q and k are off (half a step of the type each; in an int8 cache half of 1 / 127 of the row's largest value, then half a step where it is read
            # back) moves a score by their products with the other, and the probabilities' weights by twice that; then the roundings of attention itself
            kb = half * b.abs() + ((0.5 / 127 * b.abs().amax(1, keepdim=True)) * (1 + half) if int8 else 0.0)
            vb = (0.5 / 127 * c.abs().amax(1, keepdim=True) * (1 + half) + half * c.abs()) if int8 else 0.0 * c
            move = torch.where(seen, ((half * a.abs()) @ b.abs().t() + (a.abs() * (1 + half)) @ kb.t()) * hd ** -0.5, 0.0).amax(1, keepdim=True)
            bound = half * ref.abs() + (torch.expm1(2 * move) + half + 2.0 ** -12) * 1.01 * (mass + p @ vb) + p @ vb + (2.0 ** -24 if dtype == "f16" else 0.0)
            err = (got[:, h] - ref).abs()
            assert bool((err <= bound).all()), (s, h, float((err / bound).max()))
