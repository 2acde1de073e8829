"""Products of up to 32 rows on every form that they have: 8, 16 or 32 rows a workgroup, and 16 or 32 outputs with eight or four wavefronts, by the number of outputs (up to 4096, to 16384 and
above).  onhip_linear_f8_way is 0 for all of them.  Against 64 bits."""
import pytest
import torch

import f8_oracle as o
from onenew_amd import hip
from test_gpu_f8_linear import operand

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# rows that are whole lines of 128 bytes apart and not, scales of four blocks at a time and of one, a last block of channels that is short, a last workgroup that is
SIZES = [(5, 32003, 4000), (1, 16384, 640), (1, 16385, 640), (8, 16385, 640), (8, 20000, 130), (9, 16384, 300), (9, 16385, 1024), (13, 20001, 1000), (16, 17000, 2048), (16, 4097, 1100),
         (17, 4096, 640), (17, 4097, 640), (17, 16384, 520), (17, 16385, 768), (24, 6144, 2056), (32, 22016, 520), (32, 16390, 4096), (31, 16401, 136), (32, 4096, 11008), (32, 4100, 16)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(dtype, m, n, k):
    hip.init(0)
    print(dtype, m, n, k, flush=True)
    (a, sa), (w, sw) = operand(m, k, m + k), operand(n, k, n + k + 1, True)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(4)).cuda()
    ref, off = o.linear(a, sa, w, sw)
    got = hip.linear_f8(a, sa, w, sw, dtype=DT[dtype])
    o.check(got, ref, off)
    # with a bias, scales whose blocks do not lie side by side, results at an odd element of wider rows; nothing beside them
    wide = torch.full((m, n + 5), 3.0, dtype=DT[dtype], device="cuda")
    hip.linear_f8(a, sa.t().contiguous().t(), w, sw.t().contiguous().t(), bias=bias, out=wide[:, 3:3 + n])
    o.check(wide[:, 3:3 + n], *o.linear(a, sa, w, sw, bias))
    assert bool((wide[:, :3] == 3.0).all()) and bool((wide[:, 3 + n:] == 3.0).all())
    # rows further apart than they are long, NaN in between
    far = torch.full((n, (k + 15) // 16 * 16 + 48), 0x7f, dtype=torch.uint8, device="cuda").view(o.F8)
    far[:, :k] = w
    o.check(hip.linear_f8(a, sa, far[:, :k], sw, dtype=DT[dtype]), ref, off)


@pytest.mark.parametrize("m,n,k", [(5, 32003, 4000), (13, 20001, 1024), (32, 22016, 520)])
def test_repeats(m, n, k):
    """the same bits each time"""
    hip.init(0)
    (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 2, True)
    want = hip.linear_f8(a, sa, w, sw, dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(hip.linear_f8(a, sa, w, sw, dtype=torch.float32), want)
