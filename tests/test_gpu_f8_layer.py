"""A decoder layer with its linear layers in 8 bits, as a generating program calls it: norm, q k v, the cache, attention, the output product, norm, gate and up, down.  Every
step against 64 bits on what it was given, a prompt and then single tokens; a step captured into a graph; two layers on two streams."""
import pytest
import torch

import f8_oracle as o
from onenew_amd import hip

pytestmark = pytest.mark.gpu
HQ, HKV, HD, HIDDEN, INNER, PAGE, EPS = 8, 2, 64, 512, 1400, 16, 1e-5


def _layer(seed, dtype):
    g = torch.Generator().manual_seed(seed)
    f8 = lambda n, k: hip.f8_from_weights((torch.randn((n, k), generator=g) * k ** -0.5).to(dtype).cuda())  # noqa: E731
    return dict(qkv=f8((HQ + 2 * HKV) * HD, HIDDEN), out=f8(HIDDEN, HQ * HD), up=f8(2 * INNER, HIDDEN), down=f8(HIDDEN, INNER), norms=[(torch.rand(HIDDEN, generator=g) + 0.5).cuda() for _ in range(2)],
                bias=(0.1 * torch.randn((HQ + 2 * HKV) * HD, generator=g)).cuda(), freq=(10000.0 ** (-torch.arange(HD // 2) / (HD // 2))).cuda())


def _cache(dtype, pages=8):
    return [torch.zeros((pages, HKV, PAGE, HD), dtype=dtype, device="cuda") for _ in range(2)]


def _step(p, cache, x, residual, positions, slots, attend, seen=None):
    """x [tokens, hidden] and the residual in front of the layer -> the same behind it; `seen` collects (name, operands, results)"""
    note = (lambda *a: None) if seen is None else (lambda *a: seen.append(a))
    t = x.shape[0]
    q, s, h = hip.rms_norm(x, p["norms"][0], eps=EPS, residual=residual, f8=True)
    note("norm", x, residual, p["norms"][0], q, s, h)
    qkv = hip.linear_f8(q, s, *p["qkv"], bias=p["bias"], dtype=x.dtype)
    note("linear", q, s, p["qkv"], p["bias"], qkv)
    rows = qkv.view(t, HQ + 2 * HKV, HD)
    turned = hip.cache_append(rows[:, :HQ], rows[:, HQ:HQ + HKV], rows[:, HQ + HKV:], positions, slots, *cache, inv_freq=p["freq"])
    y = attend(turned, rows)
    q, s = hip.f8_from_rows(y.view(t, HQ * HD))
    note("rows", y.view(t, HQ * HD), q, s)
    x = hip.linear_f8(q, s, *p["out"], dtype=x.dtype)
    note("linear", q, s, p["out"], None, x)
    q, s, h2 = hip.rms_norm(x, p["norms"][1], eps=EPS, residual=h, f8=True)
    note("norm", x, h, p["norms"][1], q, s, h2)
    gate = hip.linear_f8(q, s, *p["up"], dtype=x.dtype)
    note("linear", q, s, p["up"], None, gate)
    q, s = hip.f8_from_rows(gate, gated=True)
    note("gated", gate, q, s)
    x = hip.linear_f8(q, s, *p["down"], dtype=x.dtype)
    note("linear", q, s, p["down"], None, x)
    return x, h2


def _check(seen):
    for name, *v in seen:
        if name == "norm":
            x, r, w, q, s, h = v
            _, y, off = o.norm(x, r, w, EPS)
            o.check_f8(q, s, y, off)
            assert torch.equal(h, (x.float() + r.float()).to(x.dtype))
        elif name == "linear":
            q, s, (w, sw), bias, y = v
            o.check(y, *o.linear(q, s, w, sw, bias, o.cuts(q.shape[0], y.dtype)))
        elif name == "rows":
            o.check_f8(v[1], v[2], v[0].double(), torch.zeros_like(v[0].double()))
        else:
            o.check_f8(v[1], v[2], *o.silu_gated(v[0]))


def _rows(t, g, dtype):
    return torch.randn((t, HIDDEN), generator=g).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prompt", [1, 50, 77])
def test_prompt_and_tokens(dtype, prompt):
    hip.init(0)
    g = torch.Generator().manual_seed(prompt)
    p, cache = _layer(1, dtype), _cache(dtype)
    table = torch.randperm(8, generator=g).view(1, 8).int().cuda()
    slot = lambda i: (table[0, i // PAGE] * PAGE + i % PAGE).view(-1)  # noqa: E731
    seen = []
    positions = torch.arange(prompt, dtype=torch.int32, device="cuda")
    slots = (table[0].long()[positions.long() // PAGE] * PAGE + positions % PAGE).int()

    def prompt_attention(q, rows):
        k, v = hip.cache_read(*cache, table, torch.tensor([prompt], dtype=torch.int32, device="cuda"), prompt)
        return hip.attention_masked(q.view(1, prompt, HQ, HD).transpose(1, 2), k, v, scale=HD ** -0.5, causal=True)

    _step(p, cache, _rows(prompt, g, dtype), _rows(prompt, g, dtype), positions, slots, prompt_attention, seen)
    for i in range(prompt, prompt + 3):
        lengths = torch.tensor([i + 1], dtype=torch.int32, device="cuda")
        _step(p, cache, _rows(1, g, dtype), _rows(1, g, dtype), lengths - 1, slot(i), lambda q, rows: hip.attention_paged(q, *cache, table, lengths, scale=HD ** -0.5), seen)
    torch.cuda.synchronize()
    _check(seen)


@pytest.mark.parametrize("batch", [1, 5, 40])
def test_a_captured_step(batch):
    """replayed with other rows and a cache that grows, every replay against the calls one by one"""
    hip.init(0)
    dtype, steps = torch.bfloat16, 6
    g = torch.Generator().manual_seed(batch)
    p, caches = _layer(2, dtype), [_cache(dtype, batch) for _ in range(2)]
    table = torch.randperm(batch, generator=g).view(batch, 1).int().cuda()
    x, r = _rows(batch, g, dtype), _rows(batch, g, dtype)
    positions, slots, lengths = (torch.zeros(batch, dtype=torch.int32, device="cuda") for _ in range(3))

    def step(cache):
        return _step(p, cache, x, r, positions, slots, lambda q, rows: hip.attention_paged(q, *cache, table, lengths, scale=HD ** -0.5))

    lengths.fill_(1)
    slots.copy_(table[:, 0] * PAGE)
    step(_cache(dtype, batch))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    for n in range(steps):
        x.copy_(_rows(batch, g, dtype))
        r.copy_(_rows(batch, g, dtype))
        positions.fill_(n)
        lengths.fill_(n + 1)
        slots.copy_(table[:, 0] * PAGE + n)
        graph.replay()
        want = step(caches[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(*caches)), n


def test_two_streams():
    """two layers at once on streams of their own: the bits of one behind the other"""
    hip.init(0)
    g = torch.Generator().manual_seed(5)
    layers = [_layer(i, torch.bfloat16) for i in range(2)]
    rows = [[_rows(t, g, torch.bfloat16) for _ in range(2)] for t in (3, 300)]
    want, got = [], [None, None]

    def both(p, x, r):
        q, s, h = hip.rms_norm(x, p["norms"][0], residual=r, f8=True)
        q, s = hip.f8_from_rows(hip.linear_f8(q, s, *p["up"]), gated=True)
        return hip.linear_f8(q, s, *p["down"]), h

    for p, (x, r) in zip(layers, rows):
        want.append(both(p, x, r))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = both(layers[i], *rows[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
