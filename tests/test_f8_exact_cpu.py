"""Exact sums of a product of e4m3 rows: which kernels they run on, what is refused, and what the Python call hands over.  No GPU is needed."""
import ctypes as C

import pytest
import torch

from onenew_amd import abi, hip
from test_f8_calls_cpu import _operands, stub  # noqa: F401
from test_f8_refusals_cpu import _desc, _linear, _refused


def test_refused():
    for exact in (-1, 2):
        _refused(_linear(exact=exact), "exact")
        assert hip.load().onhip_linear_f8_way(C.byref(_desc(exact=exact))) < 0


@pytest.mark.parametrize("compute", [abi.COMPUTE_BF16, abi.COMPUTE_F16])
def test_the_kernels_of_fp32_results(compute):
    def way(m, n, k, **more):
        return hip.load().onhip_linear_f8_way(C.byref(_desc(rows=m, outputs=n, channels=k, a_stride=k, w_stride=k, out_stride=n, **more)))

    for m in (1, 32, 33, 200, 300, 700, 2048, 8192):
        for n in (300, 4096, 6144, 22016):
            for k in (128, 1024, 4096):
                assert way(m, n, k, compute=compute, exact=1) == way(m, n, k, compute=abi.COMPUTE_F32) == way(m, n, k, compute=abi.COMPUTE_F32, exact=1)


def test_what_the_call_hands_over(stub):  # noqa: F811
    a, sa, w, sw = _operands()
    for exact in (False, True, torch.tensor(True), 0):
        hip.linear_f8(a, sa, w, sw, exact=exact)
    hip.linear_f8(a, sa, w, sw)
    assert [g[0].exact for g in stub.got] == [0, 1, 1, 0, 0]
