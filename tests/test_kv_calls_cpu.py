"""How the Python calls around the paged key-value cache describe themselves to the library: the entry points are stubbed, so no GPU is needed."""
import ctypes as C

import pytest
import torch

from onenew_amd import abi, hip

ENTRIES = ("onhip_cache_append", "onhip_cache_read", "onhip_attention_paged", "onhip_attention_masked")


class _Stub:
    """the library, whose four entry points keep a copy of the descriptions that they are handed"""

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


def _cache():
    return [torch.zeros((8, 2, 16, 64), dtype=torch.bfloat16) for _ in range(2)]


def _masked(**kw):
    q, k = torch.zeros((1, 4, 5, 64), dtype=torch.bfloat16), torch.zeros((1, 2, 9, 64), dtype=torch.bfloat16)
    return hip.attention_masked(q, k, k.clone(), **kw)


def _paged(**kw):
    k, v = _cache()
    return hip.attention_paged(torch.zeros((3, 4, 64), dtype=torch.bfloat16), k, v, torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32), **kw)


def _append(**kw):
    k, v = _cache()
    x = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    return hip.cache_append(x[:, :4], x[:, 4:6], x[:, 6:], None, torch.zeros(3, dtype=torch.int32), k, v, **kw)


def _read(tokens):
    k, v = _cache()
    return hip.cache_read(k, v, torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32), tokens)


def _said(stub, kind, field):
    return getattr(next(x for x in stub.got[-1] if isinstance(x, kind)), field)


NUMBERS = [(_masked, abi.MaskedAttentionDesc, "scale", 0.5), (_masked, abi.MaskedAttentionDesc, "softcap", 3.0), (_paged, abi.PagedAttentionDesc, "scale", 0.5),
           (_paged, abi.PagedAttentionDesc, "softcap", 3.0), (_append, abi.CacheRowsDesc, "eps", 0.25), (_masked, abi.MaskedAttentionDesc, "window", 3),
           (_masked, abi.MaskedAttentionDesc, "q_offset", 5), (_paged, abi.PagedAttentionDesc, "window", 7), (_masked, abi.MaskedAttentionDesc, "causal", True),
           (_append, abi.CacheRowsDesc, "interleaved", True)]


@pytest.mark.parametrize("i", range(len(NUMBERS)))
@pytest.mark.parametrize("wrap", [torch.tensor, lambda x: torch.nn.Parameter(torch.tensor(x), requires_grad=False)])
def test_a_number_that_changes_in_place(stub, i, wrap):
    """is the one of the call that it is handed to"""
    call, kind, field, value = NUMBERS[i]
    x = wrap(value)
    for now in (value, type(value)(0), value):
        x.fill_(now)
        call(**{field: x})
        assert _said(stub, kind, field) == now
    call(**{field: value})
    assert _said(stub, kind, field) == value
    assert not any(isinstance(part, torch.Tensor) for _, key in hip._plans for part in key)   # nothing of a caller's is kept alive


def test_a_length_that_changes_in_place(stub):
    n = torch.tensor(5)
    for now in (5, 9, 5):
        n.fill_(now)
        k, v = _read(n)
        assert k.shape == v.shape == (3, 2, now, 64) and stub.got[-1][10] == now


@pytest.mark.parametrize("call,field,bad", [(_masked, "scale", "1"), (_masked, "scale", torch.zeros(2)), (_paged, "softcap", [1.0]), (_append, "eps", None), (_masked, "window", 2.0),
                                            (_masked, "q_offset", torch.tensor(1.0)), (_paged, "window", "2"), (_paged, "window", 2.0)])
def test_what_is_no_number(stub, call, field, bad):
    for again in (False, True):   # also behind a call whose number compares equal
        if again:
            call(**{field: 2 if field in ("window", "q_offset") else 1.0})
        with pytest.raises(hip.OnhipError, match=field):
            call(**{field: bad})


def _arrays():
    """calls by one array's shape: the right one, and the same number of elements in another"""
    q, cache = torch.zeros((3, 4, 64), dtype=torch.bfloat16), _cache()
    x = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    row = lambda **kw: hip.cache_append(x[:, :4], x[:, 4:6], x[:, 6:], **{**dict(positions=ints(3), slots=ints(3), k_cache=cache[0], v_cache=cache[1], inv_freq=torch.zeros(32)), **kw})  # noqa: E731
    return {
        "masked slopes": (lambda s: _masked(slopes=torch.zeros(s)), (4,), (2, 2)),
        "paged slopes": (lambda s: _paged(slopes=torch.zeros(s)), (4,), (4, 1)),
        "paged lengths": (lambda s: hip.attention_paged(q, *cache, ints(3, 2), ints(*s)), (3,), (3, 1)),
        "read lengths": (lambda s: hip.cache_read(*cache, ints(3, 2), ints(*s), 5), (3,), (1, 3)),
        "positions": (lambda s: row(positions=ints(*s)), (3,), (3, 1)),
        "slots": (lambda s: row(slots=ints(*s)), (3,), (1, 3)),
        "q_weight": (lambda s: row(q_weight=torch.zeros(s)), (64,), (8, 8)),
        "k_weight": (lambda s: row(k_weight=torch.zeros(s)), (64,), (64, 1)),
    }


@pytest.mark.parametrize("name", sorted(_arrays()))
def test_a_shape_is_refused_whatever_was_called_before(stub, name):
    call, right, wrong = _arrays()[name]
    for _ in range(2):
        with pytest.raises(hip.OnhipError, match="shape"):
            call(wrong)
        call(right)


BIG = 1 << 32


@pytest.mark.parametrize("call,field", [(_masked, "window"), (_masked, "q_offset"), (_paged, "window")])
@pytest.mark.parametrize("value", [BIG + 5, -BIG + 3, 1 << 31, -(1 << 31) - 1, 10 ** 30])
def test_numbers_past_32_bits(stub, call, field, value):
    """are refused, not cut to their lower half"""
    for _ in range(2):
        with pytest.raises(hip.OnhipError, match=field):
            call(**{field: value})
    assert not stub.got


def test_extents_past_32_bits(stub):
    """views may have them"""
    one = torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16)
    long = one.expand(1, 1, BIG + 1, 64)
    for args in ((one, long, long), (long, one, one), (one.expand(BIG + 1, 1, 1, 64),) * 3, (one.expand(1, BIG + 1, 1, 64), one, one)):
        with pytest.raises(hip.OnhipError, match="2\\^31"):
            hip.attention_masked(*args, out=torch.zeros((1, 1, 64), dtype=torch.bfloat16))
    table, n = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    many = one.expand(BIG + 1, 1, 1, 64)
    with pytest.raises(hip.OnhipError, match="contiguous rows"):
        hip.attention_paged(one[0], one, one, table.expand(1, BIG + 1), n)
    for call in (lambda: hip.attention_paged(one[0], many, many, table, n),
                 lambda: hip.cache_read(many, many, table, n, 1), lambda: hip.cache_read(one, one, table, n, BIG + 1, k_out=one, v_out=one),
                 lambda: hip.cache_append(one[0], one[0], one[0], None, n, many, many), lambda: hip.cache_append(one[0].expand(1, BIG + 1, 64), one[0], one[0], None, n, one, one.clone())):
        with pytest.raises(hip.OnhipError, match="2\\^31"):
            call()
    assert not stub.got
