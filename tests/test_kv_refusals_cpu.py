"""What the entry points around the paged key-value cache refuse: every check comes before any device work, so no GPU is needed."""
import ctypes as C

import pytest

from onenew_amd import abi, hip

A = 1 << 20   # an address that is never used


def _cache(**more):
    f = dict(pages=8, page_tokens=16, kv_heads=2, head_dim=64, compute=abi.COMPUTE_BF16, quantised=0)
    f.update({n: x for n, x in more.items() if n not in ("k", "v", "k_scale", "v_scale")})
    d = abi.CacheDesc(**{n: x for n, x in f.items() if not n.endswith("strides")})
    rows = f["page_tokens"] * f["head_dim"]
    d.k_strides[:] = f.get("k_strides", (2 * rows, rows, f["head_dim"]))
    d.v_strides[:] = f.get("v_strides", (2 * rows, rows, f["head_dim"]))
    d.scale_strides[:] = f.get("scale_strides", (2 * f["page_tokens"], f["page_tokens"], 1))
    return d


BAD_CACHES = [dict(pages=0), dict(pages=-1), dict(kv_heads=0), dict(page_tokens=0), dict(page_tokens=12), dict(page_tokens=2048), dict(head_dim=96), dict(head_dim=32),
              dict(compute=abi.COMPUTE_F32), dict(compute=7), dict(quantised=2), dict(quantised=1), dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 2),
              dict(pages=1 << 30), dict(k_strides=(2048, 1024, 60)), dict(v_strides=(2048, 1024, 68)), dict(k_strides=(-2048, 1024, 64)), dict(k_strides=(2048, 0, 64)),
              dict(v_strides=(2048, 1024, 1 << 30)), dict(quantised=1, k_scale=A, v_scale=None), dict(quantised=1, k_scale=A + 1, v_scale=A),
              dict(quantised=1, k_scale=A, v_scale=A, scale_strides=(32, 16, 0)), dict(quantised=1, k_scale=A, v_scale=A, k_strides=(2048, 1024, 72))]


def _refused(rc, word, code=-1):
    assert rc == code, (rc, hip.load().onhip_last_error())
    assert word in hip.load().onhip_last_error().decode()


def _memory(more):
    return [more.get(n, at) for n, at in (("k", A), ("v", A), ("k_scale", None), ("v_scale", None))]


B = A + (1 << 16)   # of results


def _append(c, r, q=A, k=A, v=A, positions=A, slots=A, inv_freq=A, qw=None, kw=None, out=B, memory=(A, A, None, None)):
    return hip.load().onhip_cache_append(None if c is None else C.byref(c), *memory, None if r is None else C.byref(r), q, k, v, positions, slots, inv_freq, qw, kw, out, None)


def _rows(**more):
    f = dict(tokens=3, q_heads=4, pairs=32, interleaved=0, eps=1e-6, q_strides=(512, 64), k_strides=(512, 64), v_strides=(512, 64), out_strides=(256, 64))
    f.update(more)
    r = abi.CacheRowsDesc(**{n: x for n, x in f.items() if not n.endswith("strides")})
    for n in ("q_strides", "k_strides", "v_strides", "out_strides"):
        getattr(r, n)[:] = f[n]
    return r


@pytest.mark.parametrize("i", range(len(BAD_CACHES)))
def test_caches(i):
    c, memory = _cache(**BAD_CACHES[i]), _memory(BAD_CACHES[i])
    _refused(_append(c, _rows(), memory=memory), "cache append")
    three = (C.c_longlong * 3)(4096, 1024, 64)
    _refused(hip.load().onhip_cache_read(C.byref(c), *memory, A, 4, 4, A, 1, 5, A, three, B, three, None), "cache read")
    d = abi.PagedAttentionDesc(1, 4, 4, 0, 4, (256, 64), (256, 64), 1.0, 0.0)
    _refused(hip.load().onhip_attention_paged(C.byref(c), *memory, C.byref(d), A, A, A, None, B, None, 0, None), "paged attention")
    if not set(BAD_CACHES[i]) & {"k", "v", "k_scale"}:
        assert hip.load().onhip_attention_paged_workspace(C.byref(c), C.byref(d)) == 0


def test_append():
    c = _cache()
    _refused(_append(None, _rows()), "null")
    _refused(_append(c, None), "shape")
    for name in ("q", "k", "v", "slots", "out"):
        _refused(_append(c, _rows(), **{name: None}), "null")
    for name in ("q", "k", "v", "out"):
        _refused(_append(c, _rows(), **{name: B + 8}), "aligned")
    _refused(_append(c, _rows(), positions=None), "positions")
    _refused(_append(c, _rows(), inv_freq=None), "frequencies")
    for more in (dict(tokens=0), dict(q_heads=0), dict(tokens=-4)):
        _refused(_append(c, _rows(**more)), "shape")
    for pairs in (-8, 4, 12, 40):
        _refused(_append(c, _rows(pairs=pairs)), "pairs")
    for name in ("q_strides", "k_strides", "v_strides", "out_strides"):
        _refused(_append(c, _rows(**{name: (512, 60)})), "multiples of 8")
        _refused(_append(c, _rows(**{name: (-512, 64)})), "non-negative")
    _refused(_append(c, _rows(out_strides=(256, 0))), "overlap")
    for name in ("k", "v"):
        _refused(_append(c, _rows(), **{name: B}), "q alone")
    _refused(_append(c, _rows(), q=B), "strides")
    for eps in (-1.0, float("nan")):
        _refused(_append(c, _rows(eps=eps), qw=A), "eps")


def test_read():
    c, lib = _cache(), hip.load()
    three = lambda *x: (C.c_longlong * 3)(*x)  # noqa: E731

    def read(table=A, stride=4, pages=4, lengths=A, batch=2, tokens=5, k=A, ks=three(4096, 1024, 64), v=B, vs=three(4096, 1024, 64)):
        return lib.onhip_cache_read(C.byref(c), A, A, None, None, table, stride, pages, lengths, batch, tokens, k, ks, v, vs, None)

    for more in (dict(table=None), dict(lengths=None), dict(k=None), dict(v=None), dict(ks=None), dict(vs=None)):
        _refused(read(**more), "null")
    for more in (dict(batch=0), dict(tokens=0), dict(pages=-1), dict(stride=-1)):
        _refused(read(**more), "shape")
    for more in (dict(ks=three(4096, 1024, 60)), dict(vs=three(4096, 0, 64)), dict(ks=three(-8, 1024, 64))):
        _refused(read(**more), "strides")
    _refused(read(k=A + 2), "aligned")
    _refused(read(batch=40000), "sequences")
    _refused(read(tokens=(1 << 30) + 1), "tokens")


def test_paged():
    c, lib = _cache(), hip.load()

    def paged(q=A, table=A, lengths=A, out=B, ws=None, nbytes=0, **more):
        f = dict(batch=1, q_heads=4, table_pages=4, window=0, table_stride=4, q_strides=(256, 64), out_strides=(256, 64), scale=1.0, softcap=0.0)
        f.update(more)
        d = abi.PagedAttentionDesc(*f.values())
        return lib.onhip_attention_paged(C.byref(c), A, A, None, None, C.byref(d), q, table, lengths, None, out, ws, nbytes, None)

    for more in (dict(q=None), dict(table=None), dict(lengths=None), dict(out=None)):
        _refused(paged(**more), "null")
    for more in (dict(batch=0), dict(q_heads=0), dict(table_pages=-1), dict(table_stride=-1)):
        _refused(paged(**more), "shape")
    _refused(paged(q_heads=3), "query heads")
    _refused(paged(window=-1), "window")
    _refused(paged(batch=1 << 21), "sequences")
    _refused(paged(table_pages=1 << 27), "table")
    for more in (dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(scale=float("inf")), dict(scale=float("nan"))):
        _refused(paged(**more), "finite")
    for more in (dict(softcap=1e30), dict(softcap=1e-31), dict(scale=1e-10, softcap=1e25), dict(scale=-1e30)):
        _refused(paged(**more), "quotient")
    for more in (dict(q_strides=(256, 60)), dict(out_strides=(256, -64)), dict(q_strides=(100, 64), batch=2)):
        _refused(paged(**more), "multiples of 8")
    _refused(paged(out_strides=(256, 0)), "overlap")
    _refused(paged(q=A + 8), "aligned")
    _refused(paged(q=B), "operand")
    # a long table: parts, hence a workspace
    d = abi.PagedAttentionDesc(1, 4, 400, 0, 400, (256, 64), (256, 64), 1.0, 0.0)
    need = lib.onhip_attention_paged_workspace(C.byref(c), C.byref(d))
    assert need > 0
    for ws, nbytes in ((None, need), (A, need - 1), (A + 8, need)):
        _refused(paged(table_pages=400, table_stride=400, ws=ws, nbytes=nbytes), "workspace", -3)


def test_masked():
    lib = hip.load()

    def masked(q=A, k=A, v=A, ranges=None, out=B, ws=None, nbytes=0, size=False, **more):
        f = dict(batch=1, q_heads=4, kv_heads=2, q_tokens=8, k_tokens=8, head_dim=64, q_strides=(2048, 64, 256), k_strides=(1024, 64, 128), v_strides=(1024, 64, 128),
                 out_strides=(2048, 64, 256), scale=1.0, softcap=0.0, causal=1, window=0, q_offset=0, compute=abi.COMPUTE_F16)
        f.update(more)
        d = abi.MaskedAttentionDesc(*f.values())
        return lib.onhip_attention_masked_workspace(C.byref(d)) if size else lib.onhip_attention_masked(C.byref(d), q, k, v, ranges, None, out, ws, nbytes, None)

    assert lib.onhip_attention_masked(None, A, A, A, None, None, B, None, 0, None) == -1
    for more in (dict(q=None), dict(k=None), dict(v=None), dict(out=None)):
        _refused(masked(**more), "null")
    for more in (dict(batch=0), dict(q_heads=0), dict(kv_heads=0), dict(q_tokens=0), dict(k_tokens=-1)):
        _refused(masked(**more), "shape")
    _refused(masked(q_heads=3), "query heads")
    _refused(masked(compute=abi.COMPUTE_F32), "neither")
    _refused(masked(head_dim=32), "head dimension")
    for w in (-1, (1 << 29) + 1):
        _refused(masked(window=w), "window")
    for more in (dict(k_tokens=(1 << 29) + 1), dict(q_offset=(1 << 29) + 1), dict(q_offset=-(1 << 29) - 1)):
        _refused(masked(**more), "2^29")
    _refused(masked(q_tokens=1 << 29, q_heads=8), "too many rows")
    for more in (dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(scale=float("inf")), dict(scale=float("nan"))):
        _refused(masked(**more), "finite")
    for more in (dict(softcap=1e30), dict(softcap=1e-31), dict(scale=1e-10, softcap=1e25), dict(scale=-1e30)):
        _refused(masked(**more), "quotient")
    for name in ("q_strides", "k_strides", "v_strides", "out_strides"):
        _refused(masked(**{name: (2048, 64, 252)}), "multiples of 8")
        _refused(masked(batch=2, **{name: (-2048, 64, 256)}), "non-negative")
    _refused(masked(out_strides=(2048, 64, 0)), "overlap")
    _refused(masked(k_strides=(1024, 64, 1 << 23)), "token strides")
    for more in (dict(q=A + 8), dict(out=B + 2)):
        _refused(masked(**more), "aligned")
    for more in (dict(q=B), dict(k=B), dict(v=B)):
        _refused(masked(**more), "operand")
    _refused(masked(ranges=A + 4), "ranges")
    need = masked(size=True, k_tokens=5000)
    assert need > 0 and masked(size=True) == 0 and masked(size=True, batch=0) == 0
    for ws, nbytes in ((None, need), (A, need - 1), (A + 8, need)):
        _refused(masked(k_tokens=5000, ws=ws, nbytes=nbytes), "workspace", -3)


def test_layouts(tmp_path):
    """the ctypes mirrors against the header's structures"""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pairs = {"onhip_cache_desc_t": abi.CacheDesc, "onhip_cache_rows_desc_t": abi.CacheRowsDesc, "onhip_paged_attention_desc_t": abi.PagedAttentionDesc,
             "onhip_masked_attention_desc_t": abi.MaskedAttentionDesc}
    lines = [f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for f, _ in t._fields_) for n, t in pairs.items()]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include "onenew_hip.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    exe = tmp_path / "t"
    subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)])
    want = [x for t in pairs.values() for x in [C.sizeof(t)] + [getattr(t, f).offset for f, _ in t._fields_]]
    assert [int(x) for x in subprocess.check_output([str(exe)]).split()] == want
