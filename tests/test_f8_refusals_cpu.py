"""What the entry points on e4m3 rows refuse, and which kernel a product takes: every check comes before any device work, so no GPU is needed."""
import ctypes as C

import pytest

from onenew_amd import abi, hip

A = 1 << 30   # addresses that are never used
B, S, D, E = (A + (i << 24) for i in range(1, 5))


def _refused(rc, word):
    assert rc == -1, (rc, hip.load().onhip_last_error())
    assert word in hip.load().onhip_last_error().decode(), hip.load().onhip_last_error()


def _norm(x=A, residual=None, weight=None, out=B, scale=S, total=None, **more):
    f = dict(rows=5, channels=300, compute=abi.COMPUTE_BF16, f8=1, x_stride=304, residual_stride=304, sum_stride=304, out_stride=304, scale_strides=(3, 1), eps=1e-6)
    f.update(more)
    d = abi.NormDesc(**{n: v for n, v in f.items() if n != "scale_strides"})
    d.scale_strides[:] = f["scale_strides"]
    return hip.load().onhip_rms_norm(C.byref(d), x, residual, weight, out, scale, total, None)


def _rows(x=A, q=B, scale=S, **more):
    f = dict(rows=5, channels=300, compute=abi.COMPUTE_BF16, form=abi.F8_ROWS, x_stride=304, q_stride=304, scale_strides=(3, 1))
    f.update(more)
    d = abi.F8RowsDesc(**{n: v for n, v in f.items() if n != "scale_strides"})
    d.scale_strides[:] = f["scale_strides"]
    return hip.load().onhip_f8_from_rows(C.byref(d), x, q, scale, None)


def _desc(**more):
    f = dict(rows=5, outputs=200, channels=300, compute=abi.COMPUTE_BF16, a_stride=304, w_stride=304, out_stride=200, a_scale_strides=(3, 1), w_scale_strides=(3, 1))
    f.update(more)
    d = abi.F8LinearDesc(**{n: v for n, v in f.items() if not n.endswith("scale_strides")})
    d.a_scale_strides[:], d.w_scale_strides[:] = f["a_scale_strides"], f["w_scale_strides"]
    return d


def _linear(a=A, a_scale=S, w=B, w_scale=D, bias=None, out=E, **more):
    return hip.load().onhip_linear_f8(C.byref(_desc(**more)), a, a_scale, w, w_scale, bias, out, None)


def test_norm():
    L = hip.load()
    _refused(L.onhip_rms_norm(None, A, None, None, B, S, None, None), "shape")
    for more in (dict(rows=0), dict(rows=-3), dict(channels=0)):
        _refused(_norm(**more), "shape")
    _refused(_norm(channels=(1 << 30) + 1, x_stride=1 << 31, out_stride=1 << 31), "channels")
    for compute in (-1, 3, 9):
        _refused(_norm(compute=compute), "type")
    _refused(_norm(f8=2), "f8")
    for eps in (-1e-6, float("nan")):
        _refused(_norm(eps=eps), "eps")
    _refused(_norm(total=D), "without a residual")
    for name in ("x", "out", "scale"):
        _refused(_norm(**{name: None}), "null")
    _refused(_norm(out=None, f8=0), "null")
    _refused(_norm(x=A + 1), "misaligned")
    _refused(_norm(residual=D + 1), "misaligned")
    _refused(_norm(weight=D + 2), "misaligned")
    _refused(_norm(scale=S + 2), "misaligned")
    _refused(_norm(residual=D, total=E + 1), "misaligned")
    for name in ("x_stride", "residual_stride"):
        _refused(_norm(residual=D, **{name: -1}), "stride")
        _refused(_norm(residual=D, **{name: (1 << 40) + 1}), "stride")
    _refused(_norm(residual=D, total=E, sum_stride=299), "stride")
    _refused(_norm(f8=0, out_stride=299), "stride")
    _refused(_norm(out=B + 8), "16-byte")
    _refused(_norm(out_stride=308), "16-byte")
    for strides in ((0, 1), (3, 0), (-3, 1), ((1 << 40) + 1, 1)):
        _refused(_norm(scale_strides=strides), "scale strides")
    _refused(_norm(scale_strides=(2, 1)), "overlap")
    # one memory for two results, or for a result and an operand that it may not take the place of
    _refused(_norm(scale=B + 304), "two results")
    _refused(_norm(residual=D, total=B), "two results")
    _refused(_norm(residual=D, total=S - 2), "two results")
    _refused(_norm(out=A), "operand")
    _refused(_norm(scale=A + 600), "operand")
    _refused(_norm(weight=B, out=B), "operand")
    _refused(_norm(f8=0, out=A + 2), "operand")
    _refused(_norm(f8=0, out=A, out_stride=305), "operand")
    _refused(_norm(residual=D, total=D + 608, sum_stride=304), "operand")
    _refused(_norm(residual=A, total=A, x_stride=0, residual_stride=304), "operand")


def test_rows():
    L = hip.load()
    _refused(L.onhip_f8_from_rows(None, A, B, S, None), "shape")
    for more in (dict(rows=0), dict(channels=0), dict(rows=-1)):
        _refused(_rows(**more), "shape")
    _refused(_rows(compute=3), "type")
    for form in (-1, 3):
        _refused(_rows(form=form), "form")
    for name in ("x", "q", "scale"):
        _refused(_rows(**{name: None}), "null")
    _refused(_rows(x=A + 1), "misaligned")
    _refused(_rows(q=B + 4), "16-byte")
    _refused(_rows(q_stride=299), "stride")
    _refused(_rows(q_stride=310), "16-byte")
    _refused(_rows(x_stride=-304), "stride")
    _refused(_rows(scale_strides=(2, 1)), "overlap")
    _refused(_rows(rows=1 << 30, channels=1024, x_stride=1024, q_stride=1024, scale_strides=(8, 1), q=A + (1 << 44), scale=A + (1 << 46)), "too many")
    _refused(_rows(q=A), "results lie over")
    _refused(_rows(scale=A + 4), "results lie over")
    _refused(_rows(scale=B + 300), "results lie over")
    _refused(_rows(form=abi.F8_GATED, x_stride=608, q=A + 608), "results lie over")


def test_linear():
    L = hip.load()
    _refused(L.onhip_linear_f8(None, A, S, B, D, None, E, None), "shape")
    for name in ("rows", "outputs", "channels"):
        for n in (0, -1):
            _refused(_linear(**{name: n}), "shape")
    _refused(_linear(compute=4), "type")
    for more in (dict(rows=(1 << 27) + 1), dict(outputs=(1 << 27) + 1, out_stride=1 << 31), dict(channels=(1 << 22) + 1)):
        _refused(_linear(**more), "up to")
    for name in ("a_stride", "w_stride"):
        for n in (-304, 288, 305, 312, (1 << 22) + 16):
            _refused(_linear(**{name: n}), "apart")
    _refused(_linear(out_stride=199), "apart")
    for name in ("a", "a_scale", "w", "w_scale", "out"):
        _refused(_linear(**{name: None}), "null")
    for name in ("a", "w"):
        _refused(_linear(**{name: A + 8}), "16-byte")
    for more in (dict(a_scale=S + 2), dict(w_scale=S + 1), dict(bias=E + 3), dict(out=E + 1), dict(out=E + 2, compute=abi.COMPUTE_F32)):
        _refused(_linear(**more), "misaligned")
    for name in ("a_scale_strides", "w_scale_strides"):
        for strides in ((-1, 1), (3, -1), (1 << 41, 1)):
            _refused(_linear(**{name: strides}), "scale strides")
    for more in (dict(out=A), dict(out=B + 304 * 150), dict(out=S - 4), dict(out=D), dict(bias=E + 400), dict(out=A - 1998)):
        _refused(_linear(**more), "over an operand")


def test_which_kernel():
    """few rows, tiles in between and many; a row stride past 2^22 bytes and fp32 results leave the largest tiles out"""
    def way(m, n, k, **more):
        k16 = (k + 15) // 16 * 16
        return hip.load().onhip_linear_f8_way(C.byref(_desc(rows=m, outputs=n, channels=k, a_stride=k16, w_stride=k16, out_stride=more.pop("out_stride", n), **more)))

    assert [way(m, 4096, 4096) for m in (1, 32, 33, 64)] == [0, 0, 0, 0]
    assert {way(m, n, 4096) for m in (200, 300, 512, 700, 1024, 2048) for n in (4096, 6144, 22016)} <= set(range(1, 8))
    assert way(8192, 22016, 4096) == 7 and way(8192, 22016, 4096, compute=abi.COMPUTE_F32) == 6 and way(8192, 22016, 4096, out_stride=(1 << 21) + 8) == 6
    assert way(1 << 27, 1, 1) in range(1, 8)      # more groups of rows than a grid's second dimension has
    sizes = [1 << i for i in range(5, 15)] + [5 << i for i in range(4, 12)]
    for compute, ways in ((abi.COMPUTE_F32, {0, 1, 2, 3, 4, 6}), (abi.COMPUTE_F16, set(range(8)))):
        assert {way(m, n, k, compute=compute) for m in sizes for n in sizes + [40000] for k in (128, 1024, 4096)} == ways
    assert way(0, 4096, 4096) < 0 and way(5, 200, 300, compute=7) < 0
    assert hip.load().onhip_linear_f8_way(None) < 0
