"""NaN and infinities in rows, weights and scales of a product with 16-bit results, on every kernel that those have: they take the results that depend on them and leave the others' bits."""
import ctypes as C

import pytest
import torch

from onenew_amd import abi, hip
from test_gpu_f8_linear import operand

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
# (what onhip_linear_f8_way names for bf16 results, rows, outputs, channels)
WAYS = [(0, 5, 300, 400), (0, 20, 17000, 640), (0, 40, 500, 900), (1, 200, 3000, 1000), (2, 300, 4090, 2056), (3, 512, 4000, 700), (4, 700, 4096, 640), (5, 1000, 4096, 640), (6, 1999, 4090, 1100),
        (7, 4090, 4090, 1030), (7, 8170, 8150, 640)]


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("way,m,n,k", WAYS)
def test_what_they_take(way, m, n, k, dtype, exact):
    hip.init(0)
    print(dtype, way, m, n, k, exact, flush=True)
    pitch = (k + 15) // 16 * 16
    assert hip.load().onhip_linear_f8_way(C.byref(abi.F8LinearDesc(m, n, k, abi.COMPUTE_BF16, pitch, pitch, n))) == way
    (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 2, True)
    sa = sa * 2.0 ** -6      # within fp16
    run = lambda a, sa, w, sw: hip.linear_f8(a, sa, w, sw, dtype=DT[dtype], exact=exact)  # noqa: E731
    clean = run(a, sa, w, sw)
    assert bool(clean.isfinite().all())

    def check(got, taken, kind):
        assert torch.equal(got[~taken], clean[~taken]) and bool(kind(got[taken]).all())

    nan, none = torch.isnan, lambda t: ~t.isfinite()
    rows, columns = torch.zeros((2, m, n), dtype=torch.bool, device="cuda")
    rows[m // 2], rows[m - 1], columns[:, n // 3], columns[:, n - 1] = True, True, True, True
    one, other = a.clone(), w.clone()      # clones of rows that are not contiguous are: give them their pitch again
    one, other = (torch.nn.functional.pad(t.view(torch.uint8), (0, pitch - k)).view(t.dtype)[:, :k] for t in (one, other))
    one[m // 2, k - 1], one[m - 1, 0] = float("nan"), -float("nan")
    other[n // 3, k // 2], other[n - 1, k - 1] = float("nan"), float("nan")
    check(run(one, sa, w, sw), rows, nan)
    check(run(a, sa, other, sw), columns, nan)
    check(run(one, sa, other, sw), rows | columns, nan)
    # scales: of a row's first and last block, of the last 128 outputs
    for bad, kind in ((float("nan"), nan), (float("inf"), none)):
        scale = sa.clone()
        scale[m // 2, 0], scale[m - 1, -1] = bad, bad
        check(run(a, scale, w, sw), rows, kind)
        scale = sw.clone()
        scale[-1, scale.shape[1] // 2] = bad
        last = torch.zeros_like(rows)
        last[:, (n - 1) // 128 * 128:] = True
        check(run(a, sa, w, scale), last, kind)
