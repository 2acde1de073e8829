"""The product of e4m3 rows and weights with scales for blocks of 128 against 64 bits."""
import ctypes as C

import pytest
import torch

import f8_oracle as o
from onenew_amd import abi, hip

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def operand(rows, n, seed, tall=False, pad=0, low=-3.0):
    """e4m3 bytes of every kind, NaN behind a row's end, scales over six powers of two"""
    g = torch.Generator().manual_seed(seed)
    q = torch.full((rows, (n + 15) // 16 * 16 + pad), 0x7f, dtype=torch.uint8).view(o.F8)
    x = torch.randn((rows, n), generator=g) * torch.exp2(6 * torch.rand((rows, n), generator=g) - 2)
    q[:, :n] = x.clamp(-448, 448).to(o.F8)
    scale = torch.exp2(6 * torch.rand((o.blocks(rows) if tall else rows, o.blocks(n)), generator=g) + low) * 0.01
    return q.cuda()[:, :n], scale.cuda()


SIZES = [(1, 1, 1), (1, 128, 128), (2, 5, 16), (3, 130, 129), (1, 1000, 4096), (7, 33, 1000), (16, 64, 256), (17, 257, 300), (32, 96, 4000), (33, 640, 143), (48, 1025, 512), (64, 1000, 1000), (65, 384, 640),
         (100, 31, 2000), (127, 129, 127), (128, 128, 1024), (129, 511, 2049), (192, 256, 384), (200, 300, 136), (256, 512, 128), (300, 1280, 1152), (257, 513, 8192), (511, 1100, 640), (1000, 1000, 1000), (1, 4096, 16384),
         (5, 128, 20000)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(dtype, m, n, k):
    hip.init(0)
    print(dtype, m, n, k, flush=True)
    (a, sa), (w, sw) = operand(m, k, m + k), operand(n, k, n + k + 1, True)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(4)).cuda()
    for b in (None, bias):
        got = hip.linear_f8(a, sa, w, sw, bias=b, dtype=DT[dtype])
        torch.cuda.synchronize()
        o.check(got, *o.linear(a, sa, w, sw, b, o.cuts(m, DT[dtype])))


# one and more of every kernel, whole and ragged at each edge, one block of channels and several, an odd number of workgroups for the XCDs
WAYS = [(0, 40, 500, 900), (0, 64, 2048, 128), (0, 100, 300, 2056), (1, 200, 4090, 1500), (1, 130, 4096, 4096), (1, 200, 3000, 1000), (2, 300, 4090, 2056), (2, 200, 6100, 1500), (2, 40, 20000, 300),
        (3, 400, 4096, 1025), (3, 512, 4000, 700), (4, 64, 40000, 520), (4, 333, 6000, 130), (4, 700, 4096, 640), (4, 128, 20000, 520), (5, 1000, 4096, 640), (5, 333, 10007, 130),
        (6, 600, 10000, 300), (6, 1999, 4090, 1100), (7, 4000, 4096, 4104), (7, 4090, 4090, 1030), (7, 8170, 8150, 640), (7, 8161, 4085, 777)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("i", range(len(WAYS)))
def test_every_kernel(dtype, i):
    """the kernel that onhip_linear_f8_way names, for bf16 results (fp32 ones take none of 256 x 256, and 128 x 128 in pairs alone)"""
    hip.init(0)
    way, m, n, k = WAYS[i]
    print(dtype, WAYS[i], flush=True)
    pitch = (k + 15) // 16 * 16
    d = abi.F8LinearDesc(m, n, k, abi.COMPUTE_BF16, pitch, pitch, n)
    assert hip.load().onhip_linear_f8_way(C.byref(d)) == way
    (a, sa), (w, sw) = operand(m, k, i), operand(n, k, i + 1, True)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(4)).cuda() if i % 2 else None
    got = hip.linear_f8(a, sa, w, sw, bias=bias, dtype=DT[dtype])
    o.check(got, *o.linear(a, sa, w, sw, bias, o.cuts(m, DT[dtype])))
    # scales with the blocks first, which do not lie side by side; results at an odd element; nothing beside them
    wide = torch.full((m, n + 5), 3.0, dtype=DT[dtype], device="cuda")
    hip.linear_f8(a, sa.t().contiguous().t(), w, sw.t().contiguous().t(), bias=bias, out=wide[:, 3:3 + n])
    assert torch.equal(wide[:, 3:3 + n], got) and bool((wide[:, :3] == 3.0).all()) and bool((wide[:, 3 + n:] == 3.0).all())
    # rows at a multiple of 16 bytes, behind whose ends nothing is written
    wide = torch.full((m, (n + 7) // 8 * 8 + 16), 3.0, dtype=DT[dtype], device="cuda")
    hip.linear_f8(a, sa, w, sw, bias=bias, out=wide[:, 8:8 + n])
    assert torch.equal(wide[:, 8:8 + n], got) and bool((wide[:, :8] == 3.0).all()) and bool((wide[:, 8 + n:] == 3.0).all())


@pytest.mark.parametrize("m,n,k", [(200, 4096, 4096), (512, 4096, 4096), (2048, 4096, 4096), (8192, 8192, 1024)])
def test_how_exact(m, n, k):
    """ordinary rows, results in fp16: what sums of eight with 13 bits leave out is small next to the result's own rounding.

    A product's cut is uniform in 0 .. 2^-13 of the power of two of the largest of eight, at most a third of the eight's root of summed squares on average, towards zero: with
    signs as they come, its variance is at most 2^-26 / 3 / 2 of the eight products' summed squares' mean largest, for each of 7: below (2^-13)^2 of the summed squares.  So the error's root
    mean square is below 2^-13 of the results' (sums of products with random signs have the summed squares as their variance), on top of 2^-11 / sqrt(12) 2 of the rounding."""
    hip.init(0)
    g = torch.Generator(device="cuda").manual_seed(3)
    a, sa = hip.f8_from_rows(torch.randn((m, k), generator=g, device="cuda"))
    w, sw = hip.f8_from_weights(torch.randn((n, k), generator=g, device="cuda"))
    ref, _ = o.linear(a, sa, w, sw)
    size = float(ref.square().mean().sqrt())
    off = [float((hip.linear_f8(a, sa, w, sw, dtype=t).double() - ref).square().mean().sqrt()) / size for t in (torch.float16, torch.float32)]
    assert off[0] <= 2.0 ** -13 + 2.0 ** -11 and off[1] <= 2.0 ** -20, off


@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_strides(m):
    """wider rows, scales with their blocks first or the same for all rows, results in wider rows at an odd element: nothing beside them"""
    hip.init(0)
    n, k = 300, 520
    (a, sa), (w, sw) = operand(m, k, 1, pad=48), operand(n, k, 2, True, pad=32)
    ref, off = o.linear(a, sa, w, sw, cut=o.cuts(m, torch.bfloat16))
    turned = [t.t().contiguous().t() for t in (sa, sw)]
    for first in (0, 1, 4):
        wide = torch.full((m, n + 12), 3.0, dtype=torch.bfloat16, device="cuda")
        got = hip.linear_f8(a, turned[0], w, turned[1], out=wide[:, first:first + n])
        o.check(got, ref, off)
        assert bool((wide[:, :first] == 3.0).all()) and bool((wide[:, first + n:] == 3.0).all())
    one = sa[:1].expand(m, -1)
    o.check(hip.linear_f8(a, one, w, sw, dtype=torch.float32), *o.linear(a, one, w, sw))
    single = sa[:1, :1].expand(m, sa.shape[1])
    o.check(hip.linear_f8(a, single, w, sw[:1, :1].expand(sw.shape), dtype=torch.float32), *o.linear(a, single, w, sw[:1, :1].expand(sw.shape)))


@pytest.mark.parametrize("m,n", [(1, 200), (40, 200), (200, 200)])
def test_nan_stays_in_its_row(m, n):
    """a NaN of a row is in all of that row's results and in no other's, one of the weights in its column; an infinite and a NaN scale likewise"""
    hip.init(0)
    k = 400
    (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 2, True)
    a[m // 2, 399] = float("nan")
    w[150, 3] = float("nan")
    got = hip.linear_f8(a, sa, w, sw, dtype=torch.float32)
    want = torch.zeros((m, n), dtype=torch.bool, device="cuda")
    want[m // 2], want[:, 150] = True, True
    assert torch.equal(got.isnan(), want)
    (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 2, True)
    sa[0, 1], sw[1, 2] = float("inf"), float("nan")
    got = hip.linear_f8(a, sa, w, sw, dtype=torch.float32)
    assert not got[0].isfinite().any() and bool(got[:, 128:].isnan().all()) and bool(got[1:, :128].isfinite().all())


def test_no_rows():
    hip.init(0)
    (a, sa), (w, sw) = operand(3, 128, 1), operand(5, 128, 2, True)
    assert hip.linear_f8(a[:0], sa[:0], w, sw).shape == (0, 5) and hip.linear_f8(a, sa, w[:0], sw[:0]).shape == (3, 0)
    with pytest.raises(hip.OnhipError):
        hip.linear_f8(a[:, :0], sa[:, :0], w[:, :0], sw[:, :0])


def test_far_results():
    """results past 2^32 bytes, weights 2^22 bytes apart"""
    hip.init(0)
    m, n, k = 70001, 32768, 16
    (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 2, True)
    got = hip.linear_f8(a, sa, w, sw)
    for rows in (slice(0, 130), slice(65500, 65600), slice(m - 130, m)):
        o.check(got[rows], *o.linear(a[rows], sa[rows], w, sw, cut=True))
    del got
    n, k = 1100, 300
    (a, sa), (w, sw) = operand(150, k, 1), operand(n, k, 2, True)
    far = torch.zeros((n - 1 << 22) + 4096, dtype=torch.uint8, device="cuda").view(o.F8).as_strided((n, k), (1 << 22, 1))
    far.copy_(w)
    for rows in (1, 30, 150):
        o.check(hip.linear_f8(a[:rows], sa[:rows], far, sw), *o.linear(a[:rows], sa[:rows], w, sw, cut=o.cuts(rows, torch.bfloat16)))


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (32, 4096, 4096), (300, 4096, 11008), (1024, 4096, 4096)])
def test_repeats(m, n, k):
    """the same bits each time, whatever order workgroups run in"""
    hip.init(0)
    (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 2, True)
    want = hip.linear_f8(a, sa, w, sw)
    o.check(want, *o.linear(a, sa, w, sw, cut=o.cuts(m, torch.bfloat16)))
    for _ in range(5):
        assert torch.equal(hip.linear_f8(a, sa, w, sw), want)
