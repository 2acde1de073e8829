"""A decoding step captured into a graph, append, attention over 16-bit and int8 caches, the cache read back and attention of its rows, and replayed while the
cache grows over pages: every replay against the same calls one by one."""
import pytest
import torch

from onenew_amd import hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("table_pages", [3, 300])
def test_a_captured_step(dtype, table_pages):
    """a table as wide as its sequences, and one whose width calls for parts and a workspace"""
    hip.init(0)
    hq, hkv, hd, page, batch, steps = 8, 2, 128, 16, 5, 40
    g = torch.Generator().manual_seed(3)
    caches = [[torch.zeros((15, hkv, page, hd), dtype=t, device="cuda") for _ in range(2)] for t in (dtype, torch.int8)]
    scales = [torch.zeros((15, hkv, page), device="cuda") for _ in range(2)]
    eager = [[t.clone() for t in kv] for kv in caches], [t.clone() for t in scales]
    table = torch.full((batch, table_pages), -1, dtype=torch.int32, device="cuda")
    table[:, :3] = torch.randperm(15, generator=g).view(batch, 3).int().cuda()
    x = torch.zeros((batch, hq + 2 * hkv, hd), dtype=dtype, device="cuda")
    positions, slots, lengths = (torch.zeros(batch, dtype=torch.int32, device="cuda") for _ in range(3))
    freq, weight = (10000.0 ** (-torch.arange(64) / 64)).cuda(), torch.rand(hd, generator=g).cuda() + 0.5

    def step(caches, scales):
        out = []
        for i, (k, v) in enumerate(caches):
            s = dict(k_scale=scales[0], v_scale=scales[1]) if i else {}
            q = hip.cache_append(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], positions, slots, k, v, inv_freq=freq, q_weight=weight, k_weight=weight, **s)
            out.append(hip.attention_paged(q, k, v, table, lengths, scale=hd ** -0.5, **s))
            rows = hip.cache_read(k, v, table, lengths, steps, dtype=dtype, **s)
            ranges = torch.stack([torch.zeros_like(lengths), lengths], -1)[:, None].contiguous()
            out += [*rows, hip.attention_masked(q[:, :, None], *rows, scale=hd ** -0.5, ranges=ranges)]
        return out

    lengths.fill_(1)
    slots.copy_(table[:, 0] * page)
    step([[t.clone() for t in kv] for kv in caches], [t.clone() for t in scales])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches, scales)
    for n in range(steps):
        x.copy_(torch.randn(x.shape, generator=g).to(dtype))
        positions.fill_(n)
        lengths.fill_(n + 1)
        slots.copy_(table[:, n // page] * page + n % page)
        graph.replay()
        want = step(*eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n
        assert all(torch.equal(a, b) for kv, other in zip(caches, eager[0]) for a, b in zip(kv, other)) and all(torch.equal(a, b) for a, b in zip(scales, eager[1])), n
