"""Results and caches whose rows share memory are refused: two wavefronts would write one row, and which one is last is a matter of time."""
import ctypes as C

import pytest

from onenew_amd import abi, hip
from test_kv_refusals_cpu import A, B, _append, _cache, _refused, _rows


@pytest.mark.parametrize("strides", [(64, 64), (64, 128), (192, 64), (64, 72), (128, 64)])
def test_append_results(strides):
    """4 heads of 64 channels, 3 tokens"""
    _refused(_append(_cache(), _rows(out_strides=strides)), "overlap")


CACHES = [dict(k_strides=(64, 64, 64)), dict(v_strides=(1024, 1024, 64)), dict(k_strides=(1024, 512, 64)), dict(v_strides=(2048, 1024, 128)), dict(k_strides=(64, 448, 1024)),
          dict(k_strides=(2048, 1024, 8192))]
SCALES = [(16, 16, 1), (32, 8, 1), (1, 2, 1), (1, 8, 15)]


@pytest.mark.parametrize("i", range(len(CACHES)))
def test_caches_that_are_written(i):
    """8 pages of 16 rows, 2 heads of 64 channels"""
    _refused(_append(_cache(**CACHES[i]), _rows()), "overlap")


@pytest.mark.parametrize("strides", SCALES)
def test_scales_that_are_written(strides):
    _refused(_append(_cache(quantised=1, scale_strides=strides), _rows(), memory=(A, A, A, A)), "overlap")


@pytest.mark.parametrize("strides", [(64, 64, 64), (1024, 1024, 64), (64, 128, 192), (640, 256, 64)])
@pytest.mark.parametrize("which", range(2))
def test_read_results(strides, which):
    """2 sequences, 2 heads, 5 tokens"""
    c, three = _cache(), lambda x: (C.c_longlong * 3)(*x)
    fine = (4096, 1024, 64)
    _refused(hip.load().onhip_cache_read(C.byref(c), A, A, None, None, A, 4, 4, A, 2, 5, B, three(fine if which else strides), 2 * B, three(strides if which else fine), None), "overlap")


@pytest.mark.parametrize("strides", [(64, 64), (128, 64), (64, 128), (192, 64), (128, 256)])
def test_paged_results(strides):
    """3 sequences, 4 heads"""
    d = abi.PagedAttentionDesc(3, 4, 4, 0, 4, (256, 64), strides, 1.0, 0.0)
    c = _cache()
    _refused(hip.load().onhip_attention_paged(C.byref(c), A, A, None, None, C.byref(d), A, A, A, None, B, None, 0, None), "overlap")


@pytest.mark.parametrize("strides", [(64, 64, 64), (2048, 64, 64), (2048, 64, 128), (256, 64, 256), (2048, 64, 192), (1024, 128, 256), (1 << 60, 64, 192)])
def test_masked_results(strides):
    """2 sequences of 8 tokens, 4 heads"""
    d = abi.MaskedAttentionDesc(2, 4, 2, 8, 8, 64, (2048, 64, 256), (1024, 64, 128), (1024, 64, 128), strides, 1.0, 0.0, 1, 0, 0, abi.COMPUTE_F16)
    _refused(hip.load().onhip_attention_masked(C.byref(d), A, A, A, None, None, B, None, 0, None), "overlap")


@pytest.mark.parametrize("strides", [(4 * 8 * 64, 64, 256), (4 * 8 * 64, 8 * 64, 64), (256, 64, 512), (64, 1024, 128), (1 << 62, 64, 256), (4 * 8 * 128, 64, 512)])
def test_layouts_that_are_not_refused(strides):
    """any order of the extents, and gaps between them: the next check, of the workspace, is what refuses (2 sequences of 8 tokens, 4 heads; many keys)"""
    d = abi.MaskedAttentionDesc(2, 4, 2, 8, 5000, 64, (2048, 64, 256), (1 << 20, 64, 128), (1 << 20, 64, 128), strides, 1.0, 0.0, 1, 0, 0, abi.COMPUTE_F16)
    _refused(hip.load().onhip_attention_masked(C.byref(d), A, A, A, None, None, B, None, 0, None), "workspace", -3)


def test_one_memory_for_two():
    """keys and values in one place, and results in the cache's"""
    _refused(_append(_cache(), _rows(), memory=(A, A, None, None)), "one memory")
    _refused(_append(_cache(quantised=1), _rows(), memory=(A, 2 * A, 3 * A, 3 * A)), "one memory")
    for memory in ((B, A, None, None), (A, B, None, None)):
        _refused(_append(_cache(), _rows(), memory=memory), "one memory")
    c, three = _cache(), (C.c_longlong * 3)(4096, 1024, 64)
    d = abi.PagedAttentionDesc(1, 4, 4, 0, 4, (256, 64), (256, 64), 1.0, 0.0)
    for memory in ((B, A), (A, B)):
        for k, v in ((B, 2 * B), (2 * B, B)):
            _refused(hip.load().onhip_cache_read(C.byref(c), *memory, None, None, A, 4, 4, A, 2, 5, k, three, v, three, None), "one memory")
        _refused(hip.load().onhip_attention_paged(C.byref(c), *memory, None, None, C.byref(d), A, A, A, None, B, None, 0, None), "one memory")
