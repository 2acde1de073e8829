"""How the Python calls on e4m3 rows describe themselves to the library: the entry points are stubbed, so no GPU is needed."""
import ctypes as C

import pytest
import torch

from onenew_amd import abi, hip

F8 = torch.float8_e4m3fn
ENTRIES = ("onhip_rms_norm", "onhip_f8_from_rows", "onhip_linear_f8")


class _Stub:
    """the library, whose entry points keep a copy of the descriptions that they are handed"""

    def __init__(self, lib):
        self.lib, self.got = lib, []

    def __getattr__(self, name):
        if name not in ENTRIES:
            return getattr(self.lib, name)

        def call(*args):
            kept = []
            for x in args:
                x = getattr(x, "_obj", x)
                kept.append(type(x).from_buffer_copy(x) if isinstance(x, C.Structure) else x)
            self.got.append(kept)
            return 0
        return call


@pytest.fixture
def stub(monkeypatch):
    s = _Stub(hip.load())
    monkeypatch.setattr(hip, "_lib", s)
    monkeypatch.setattr(hip, "load", lambda: s)
    monkeypatch.setattr(hip, "_device", lambda: -1)
    monkeypatch.setattr(hip, "_stream", lambda: 0)
    monkeypatch.setattr(hip, "_plans", {})
    monkeypatch.setattr(hip, "_last", {})
    return s


def _f8(rows, n):
    return torch.zeros((rows, (n + 15) // 16 * 16), dtype=torch.uint8).view(F8)[:, :n]


def _operands(m=3, n=130, k=300):
    return _f8(m, k), torch.ones((m, 3)), _f8(n, k), torch.ones((2, 3))


@pytest.mark.parametrize("dtype,compute", [(torch.float32, abi.COMPUTE_F32), (torch.bfloat16, abi.COMPUTE_BF16), (torch.float16, abi.COMPUTE_F16)])
def test_descriptions(stub, dtype, compute):
    x = torch.zeros((3, 340), dtype=dtype)[:, :300]
    out = hip.rms_norm(x, torch.ones(300), eps=1e-5, residual=x[:1].expand(3, 300), f8=True)
    d, at = stub.got[-1][0], stub.got[-1][1:]
    assert (d.rows, d.channels, d.compute, d.f8, d.x_stride, d.residual_stride, d.sum_stride, d.out_stride, list(d.scale_strides)) == (3, 300, compute, 1, 340, 0, 300, 304, [3, 1])
    assert abs(d.eps - 1e-5) < 1e-12 and [t.dtype for t in out] == [F8, torch.float32, dtype] and [tuple(t.shape) for t in out] == [(3, 300), (3, 3), (3, 300)]
    assert at[3] == out[0].data_ptr() and at[4] == out[1].data_ptr() and at[5] == out[2].data_ptr()
    y = hip.rms_norm(x)
    assert y.dtype == dtype and stub.got[-1][0].f8 == 0 and stub.got[-1][2:4] == [None, None] and stub.got[-1][5:7] == [None, None]
    for call, form, shape, scales in ((hip.f8_from_rows, abi.F8_ROWS, (3, 300), (3, 3)), (lambda t: hip.f8_from_rows(t, gated=True), abi.F8_GATED, (3, 150), (3, 2)), (hip.f8_from_weights, abi.F8_WEIGHTS, (3, 300), (1, 3))):
        q, s = call(x)
        d = stub.got[-1][0]
        assert (d.rows, d.channels, d.compute, d.form, d.x_stride) == (3, shape[1], compute, form, 340) and q.dtype == F8 and tuple(q.shape) == shape and tuple(s.shape) == scales and d.q_stride == q.stride(0)
    a, sa, w, sw = _operands()
    got = hip.linear_f8(a, sa.t().contiguous().t(), w, sw, dtype=dtype)
    d = stub.got[-1][0]
    assert (d.rows, d.outputs, d.channels, d.compute, d.a_stride, d.w_stride, d.out_stride, list(d.a_scale_strides), list(d.w_scale_strides)) == (3, 130, 300, compute, 304, 304, 130, [1, 3], [3, 1])
    assert got.dtype == dtype and tuple(got.shape) == (3, 130)


def test_numbers_are_read_when_they_are_given(stub):
    """eps as a tensor that changes in place, flags as anything with a truth"""
    x, eps = torch.zeros((2, 128)), torch.tensor(1e-5)
    hip.rms_norm(x, eps=eps)
    eps.fill_(0.5)
    hip.rms_norm(x, eps=eps)
    assert [round(g[0].eps, 6) for g in stub.got] == [1e-5, 0.5]
    hip.rms_norm(x, f8=1)
    hip.f8_from_rows(x, gated=torch.tensor(True))
    assert stub.got[-2][0].f8 == 1 and stub.got[-1][0].form == abi.F8_GATED
    with pytest.raises(hip.OnhipError, match="eps"):
        hip.rms_norm(x, eps="small")


def test_a_call_behind_another_is_its_own(stub):
    """the description that is kept from one call is not the next one's where a type, shape, stride or result differs"""
    a, sa, w, sw = _operands()
    hip.linear_f8(a, sa, w, sw)
    hip.linear_f8(a, sa, w, sw, out=torch.zeros((3, 140), dtype=torch.float16)[:, :130])
    hip.linear_f8(a, sa[:1].expand(3, 3), w, sw)
    hip.linear_f8(a[:2], sa[:2], w, sw)
    assert [(g[0].rows, g[0].compute, g[0].out_stride, g[0].a_scale_strides[0]) for g in stub.got] == [(3, 1, 130, 3), (3, 2, 140, 3), (3, 1, 130, 0), (2, 1, 130, 3)]
    for bias in (torch.zeros(130, dtype=torch.float16), torch.zeros((130, 1)), torch.zeros(260)[::2]):
        with pytest.raises(hip.OnhipError, match="bias"):
            hip.linear_f8(a, sa, w, sw, bias=bias)


def test_refusals(stub):
    x, w = torch.zeros((3, 300), dtype=torch.bfloat16), torch.ones(300)
    a, sa, b, sb = _operands()
    bad = [
        (lambda: hip.rms_norm(x.double()), "none of"), (lambda: hip.rms_norm(x[0]), "dimensions|values|unpack"), (lambda: hip.rms_norm(x.t()), "contiguous"),
        (lambda: hip.rms_norm(x, w.half()), "weight"), (lambda: hip.rms_norm(x, w[:299]), "weight"), (lambda: hip.rms_norm(x, torch.ones(600)[::2]), "weight"),
        (lambda: hip.rms_norm(x, residual=x[:2]), "residual"), (lambda: hip.rms_norm(x, residual=x.half()), "residual"), (lambda: hip.rms_norm(x, sum_out=x), "sum_out"),
        (lambda: hip.rms_norm(x, out=x.float()), "out"), (lambda: hip.rms_norm(x, out=x[:, :299]), "out"), (lambda: hip.rms_norm(x, scale_out=sa), "scales"),
        (lambda: hip.rms_norm(x, f8=True, out=x), "out"), (lambda: hip.rms_norm(x, f8=True, scale_out=sa.half()), "scale"), (lambda: hip.rms_norm(x, f8=True, scale_out=sa[:, :2]), "scale"),
        (lambda: hip.rms_norm(x[:, :0]), "without channels"), (lambda: hip.f8_from_rows(x[:, :0]), "without channels"), (lambda: hip.f8_from_rows(x[:, :299], gated=True), "two halves"),
        (lambda: hip.f8_from_rows(x.int()), "none of"), (lambda: hip.f8_from_rows(x, out=_f8(3, 301)), "out"), (lambda: hip.f8_from_weights(x, scale_out=torch.ones((3, 3))), "scale"),
        (lambda: hip.linear_f8(a.view(torch.uint8), sa, b, sb), "float8"), (lambda: hip.linear_f8(a, sa, b[:, :299], sb), "channels"), (lambda: hip.linear_f8(a, sa[:, :2], b, sb), "a_scale"),
        (lambda: hip.linear_f8(a, sa.double(), b, sb), "a_scale"), (lambda: hip.linear_f8(a, sa, b, sb[:1]), "w_scale"), (lambda: hip.linear_f8(a, sa, b, sb, dtype=torch.float64), "none of"),
        (lambda: hip.linear_f8(a, sa, b, sb, out=torch.zeros((3, 129), dtype=torch.bfloat16)), "out"), (lambda: hip.linear_f8(a, sa, b, sb, dtype=torch.float32, out=torch.zeros((3, 130), dtype=torch.bfloat16)), "out"),
        (lambda: hip.linear_f8(a, sa, b.t(), sb), "contiguous|channels")]
    for call, word in bad:
        with pytest.raises((hip.OnhipError, ValueError), match=word):
            call()
    assert not stub.got
