"""Performance cases of the operators around a generating transformer's key-value cache.

Kinds
  masked   attention of a prompt: causal, sliding window, key ranges (packed documents, prefixes), capped scores, distance bias
  paged    attention of one new token a sequence over a paged cache, 16-bit or int8
  append   norms of q and k, position rotation and the write into the paged cache; an int8 cache is read back, as the values it stands for
  read     the cache's rows back in sequence order

`listed()` names twelve of them, `draw()` gives more over the same ranges, odd sizes among them.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
THETA = 10000.0


def listed():
    return [
        # a short prompt of one user: the latency of a call
        dict(name="masked_f16_short", kind="masked", dtype="f16", batch=1, q_heads=12, kv_heads=12, dim=64, q_tokens=77, k_tokens=77,
             causal=True, window=0, cap=0.0, bias=False, mask="none"),
        # a long document in one piece, eight key-value heads for 32 query heads
        dict(name="masked_bf16_8k", kind="masked", dtype="bf16", batch=1, q_heads=32, kv_heads=8, dim=128, q_tokens=8192, k_tokens=8192,
             causal=True, window=0, cap=0.0, bias=False, mask="none"),
        # capped scores in a sliding window, a length that no tile divides
        dict(name="masked_f16_capped_window", kind="masked", dtype="f16", batch=2, q_heads=16, kv_heads=8, dim=128, q_tokens=4001, k_tokens=4001,
             causal=True, window=1024, cap=50.0, bias=False, mask="none"),
        # documents packed one behind the other, scores that fall with the distance
        dict(name="masked_bf16_documents", kind="masked", dtype="bf16", batch=2, q_heads=16, kv_heads=16, dim=64, q_tokens=4096, k_tokens=4096,
             causal=True, window=0, cap=0.0, bias=True, mask="documents"),
        # the next token of one conversation: latency
        dict(name="paged_bf16_one", kind="paged", dtype="bf16", int8=False, batch=1, q_heads=32, kv_heads=8, dim=128, longest=777, page=16,
             window=0, cap=0.0, bias=False),
        # the next token of a serving batch of ragged lengths
        dict(name="paged_bf16_b32", kind="paged", dtype="bf16", int8=False, batch=32, q_heads=32, kv_heads=8, dim=128, longest=4096, page=16,
             window=0, cap=0.0, bias=False),
        # few long contexts in an int8 cache: the work is split over the length
        dict(name="paged_int8_long", kind="paged", dtype="bf16", int8=True, batch=4, q_heads=32, kv_heads=8, dim=128, longest=65536, page=64,
             window=0, cap=0.0, bias=False),
        # many short ones, a key-value head for each query head, capped and biased scores
        dict(name="paged_f16_b64_capped", kind="paged", dtype="f16", int8=False, batch=64, q_heads=16, kv_heads=16, dim=64, longest=2000, page=32,
             window=0, cap=30.0, bias=True),
        # the rows of one decoding step
        dict(name="append_bf16_step", kind="append", dtype="bf16", int8=False, tokens=32, q_heads=32, kv_heads=8, dim=128, page=16, pairs=64,
             interleaved=False, norm=True),
        # a prompt of ragged sequences into an int8 cache
        dict(name="append_int8_prompt", kind="append", dtype="bf16", int8=True, tokens=8191, q_heads=32, kv_heads=8, dim=128, page=16, pairs=64,
             interleaved=False, norm=True),
        # the cache of one short sequence read back
        dict(name="read_f16_one", kind="read", dtype="f16", int8=False, batch=1, kv_heads=16, dim=64, longest=333, page=16),
        # a batch's int8 cache read back for the next chunk of its prompts
        dict(name="read_int8_b8", kind="read", dtype="bf16", int8=True, batch=8, kv_heads=8, dim=128, longest=8192, page=16),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["masked", "masked", "paged", "paged", "append", "read"])
    dtype, dim = rng.choice(["bf16", "f16"]), rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    q_heads = kv_heads * rng.choice([1, 2, 4, 8])
    page = rng.choice([8, 16, 32, 64, 128])
    biased = dict(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.random() < 0.3)
    while True:
        if kind == "masked":
            q_tokens = spread(1, 8192)
            k_tokens = q_tokens if rng.random() < 0.6 else q_tokens + spread(1, 16384)
            c = dict(kind=kind, dtype=dtype, batch=spread(1, 8), q_heads=q_heads, kv_heads=kv_heads, dim=dim, q_tokens=q_tokens, k_tokens=k_tokens,
                     causal=True, window=rng.choice([0, 0, spread(16, 4096)]), mask=rng.choice(["none", "none", "documents", "prefix"]), **biased)
            if c["mask"] == "prefix":
                c["causal"] = False
            if c["batch"] * q_heads * q_tokens * k_tokens <= 32 * 8192 * 8192 // 2:
                return c
        elif kind == "paged":
            c = dict(kind=kind, dtype=dtype, int8=rng.random() < 0.4, batch=spread(1, 128), q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                     longest=spread(1, 65536), page=page, window=rng.choice([0, 0, 0, spread(16, 4096)]), **biased)
            if c["batch"] * kv_heads * dim * c["longest"] <= 4 * 8 * 128 * 65536:
                return c
        elif kind == "append":
            return dict(kind=kind, dtype=dtype, int8=rng.random() < 0.4, tokens=spread(1, 8192), q_heads=min(q_heads, 32), kv_heads=min(kv_heads, 8) if q_heads > 32 else kv_heads,
                        dim=dim, page=page, pairs=rng.choice([dim // 2, dim // 2, dim // 4]), interleaved=rng.random() < 0.4, norm=rng.random() < 0.7)
        else:
            c = dict(kind=kind, dtype=dtype, int8=rng.random() < 0.5, batch=spread(1, 32), kv_heads=kv_heads, dim=dim, longest=spread(1, 16384), page=page)
            if c["batch"] * kv_heads * dim * c["longest"] <= 8 * 8 * 128 * 8192:
                return c


def _cache(c, pages, g):
    """a cache that earlier steps have filled, and its scales"""
    shape = (pages, c["kv_heads"], c["page"], c["dim"])
    s = {}
    for name in ("k", "v"):
        if c["int8"]:
            s[name] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
            s[name + "_scale"] = 0.005 + 0.02 * torch.rand(shape[:3], generator=g, device="cuda")
        else:
            s[name] = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(DTYPES[c["dtype"]])
            s[name + "_scale"] = None
    return s


def _sequences(c, g):
    """lengths between half of the longest and the longest, pages handed out in no order"""
    longest, page, batch = c["longest"], c["page"], c["batch"]
    lengths = torch.randint((longest + 1) // 2, longest + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    lengths[0] = longest
    per = -(-longest // page)
    table = torch.randperm(batch * per, generator=g, device="cuda").to(torch.int32).view(batch, per)
    return lengths, table


def _ranges(c, g):
    """[batch, q_tokens, 2]: the keys that each query may see, for documents one behind the other or for prefixes"""
    tq, tk, batch = c["q_tokens"], c["k_tokens"], c["batch"]
    place = torch.arange(tq, device="cuda") + (tk - tq)
    if c["mask"] == "documents":   # about nine of them, cut at random places
        cuts = torch.sort(torch.randint(0, tk, (batch, 8), generator=g, device="cuda"), dim=1).values
        edges = torch.cat([torch.zeros_like(cuts[:, :1]), cuts, torch.full_like(cuts[:, :1], tk)], 1).contiguous()
        at = torch.searchsorted(edges, place.expand(batch, tq).contiguous(), right=True)
        begin, end = edges.gather(1, at - 1), edges.gather(1, at.clamp(max=9))
    else:                            # a prefix that everyone sees, then causal
        prefix = torch.randint(0, tk + 1, (batch, 1), generator=g, device="cuda")
        end = torch.maximum((place + 1).expand(batch, tq), prefix)
        begin = torch.zeros_like(end)
    return torch.stack([begin, end], -1).to(torch.int32).contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = dict(c=c)
    slopes = lambda: torch.exp2(-8.0 * torch.arange(1, c["q_heads"] + 1, device="cuda", dtype=torch.float32) / c["q_heads"])  # noqa: E731
    if c["kind"] == "masked":
        b, hq, hkv, d = c["batch"], c["q_heads"], c["kv_heads"], c["dim"]
        # projections' rows: [batch, tokens, heads, dim], seen as [batch, heads, tokens, dim]
        s["q"] = randn(b, c["q_tokens"], hq, d).permute(0, 2, 1, 3)
        s["k"], s["v"] = (randn(b, c["k_tokens"], hkv, d).permute(0, 2, 1, 3) for _ in range(2))
        s["slopes"] = slopes() if c["bias"] else None
        s["ranges"] = None if c["mask"] == "none" else _ranges(c, g)
    elif c["kind"] == "paged":
        s["lengths"], s["table"] = _sequences(c, g)
        s.update(_cache(c, s["table"].numel(), g))
        s["q"] = randn(c["batch"], c["q_heads"], c["dim"])
        s["slopes"] = slopes() if c["bias"] else None
    elif c["kind"] == "append":
        t, hq, hkv, d = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"]
        pages = -(-t // c["page"]) + 3
        s["qkv"] = randn(t, hq + 2 * hkv, d)     # the rows of one projection
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        s["table"] = order[: -(-t // c["page"])].view(1, -1).contiguous()
        place = torch.arange(t, device="cuda")
        s["slots"] = (s["table"][0].long()[place // c["page"]] * c["page"] + place % c["page"]).to(torch.int32)
        s["lengths"] = torch.full((1,), t, device="cuda", dtype=torch.int32)
        s["positions"] = (place + torch.randint(0, 100000, (1,), generator=g, device="cuda")).to(torch.int32)
        s.update(_cache(c, pages, g))
        s["inv_freq"] = (THETA ** (-torch.arange(c["pairs"], device="cuda", dtype=torch.float64) / c["pairs"])).float()
        s["q_weight"], s["k_weight"] = (0.5 + torch.rand(d, generator=g, device="cuda") if c["norm"] else None for _ in range(2))
    else:
        s["lengths"], s["table"] = _sequences(c, g)
        s.update(_cache(c, s["table"].numel(), g))
    return s


# ---- the operators as a user of the framework calls them ----------------------------------------------------------

def _run_own(s):
    from onenew_amd import hip
    c = s["c"]
    if c["kind"] == "masked":
        return hip.attention_masked(s["q"], s["k"], s["v"], scale=c["dim"] ** -0.5, causal=c["causal"], window=c["window"], softcap=c["cap"],
                                    slopes=s["slopes"], ranges=s["ranges"])
    if c["kind"] == "paged":
        return hip.attention_paged(s["q"], s["k"], s["v"], s["table"], s["lengths"], scale=c["dim"] ** -0.5, window=c["window"], softcap=c["cap"],
                                   slopes=s["slopes"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if c["kind"] == "append":
        hq, hkv = c["q_heads"], c["kv_heads"]
        x = s["qkv"]
        q = hip.cache_append(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], s["positions"], s["slots"], s["k"], s["v"], inv_freq=s["inv_freq"],
                             q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, interleaved=c["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        if not c["int8"]:
            return q, s["k"], s["v"]
        return (q,) + tuple(hip.cache_read(s["k"], s["v"], s["table"], s["lengths"], c["tokens"], k_scale=s["k_scale"], v_scale=s["v_scale"], dtype=DTYPES[c["dtype"]]))
    return tuple(hip.cache_read(s["k"], s["v"], s["table"], s["lengths"], c["longest"], k_scale=s["k_scale"], v_scale=s["v_scale"], dtype=DTYPES[c["dtype"]]))


# ---- the plain form: elementary operations in 32 bits --------------------------------------------------------------

def _softmax_times(scores, seen, v):
    """softmax over the seen keys (zeros where there are none) and its product with v"""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return torch.matmul(e, v) / torch.where(total == 0, 1.0, total)


def _plain_masked(s):
    c = s["c"]
    b, hq, hkv, d, tq, tk = c["batch"], c["q_heads"], c["kv_heads"], c["dim"], c["q_tokens"], c["k_tokens"]
    group = hq // hkv
    q = s["q"].float().reshape(b, hkv, group * tq, d)
    k, v = s["k"].float(), s["v"].float().contiguous()
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(b, hkv, group, tq, tk) * d ** -0.5
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    place, key = torch.arange(tq, device="cuda").view(tq, 1) + (tk - tq), torch.arange(tk, device="cuda").view(1, tk)
    if c["bias"]:
        scores = scores - s["slopes"].view(1, hkv, group, 1, 1) * (place - key).abs().float()
    seen = torch.ones((tq, tk), dtype=torch.bool, device="cuda")
    if c["causal"]:
        seen = seen & (key <= place)
    if c["window"]:
        seen = seen & (place - key < c["window"])
    seen = seen.view(1, 1, 1, tq, tk)
    if s["ranges"] is not None:
        begin, end = (s["ranges"][..., i].view(b, 1, 1, tq, 1) for i in range(2))
        seen = seen & (key >= begin) & (key < end)
    out = _softmax_times(scores.view(b, hkv, group * tq, tk), seen.expand(b, 1, group, tq, tk).reshape(b, 1, group * tq, tk), v)
    return out.view(b, hq, tq, d).permute(0, 2, 1, 3).reshape(b, tq, hq * d).to(DTYPES[c["dtype"]])


def _rows(s, name, tokens):
    """[batch, kv_heads, tokens, dim] of the cache in 32 bits, through the table"""
    c = s["c"]
    per = -(-tokens // c["page"])
    at = s["table"][:, :per].long()

    def in_order(x):
        y = x[at].transpose(1, 2)
        return y.reshape(y.shape[0], y.shape[1], per * c["page"], *y.shape[4:])[:, :, :tokens]

    x = in_order(s[name]).float()
    return x * in_order(s[name + "_scale"]).unsqueeze(-1) if c["int8"] else x


def _plain_paged(s):
    c = s["c"]
    b, hq, hkv, d, t = c["batch"], c["q_heads"], c["kv_heads"], c["dim"], c["longest"]
    group = hq // hkv
    k, v = _rows(s, "k", t), _rows(s, "v", t)
    scores = torch.matmul(s["q"].float().view(b, hkv, group, d), k.transpose(-1, -2).contiguous()) * d ** -0.5
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    behind = s["lengths"].view(b, 1, 1, 1) - 1 - torch.arange(t, device="cuda").view(1, 1, 1, t)
    if c["bias"]:
        scores = scores - s["slopes"].view(1, hkv, group, 1) * behind.float()
    seen = behind >= 0
    if c["window"]:
        seen = seen & (behind < c["window"])
    return _softmax_times(scores, seen, v).view(b, hq, d).to(DTYPES[c["dtype"]])


def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _rotated(x, cos, sin, c):
    r = c["pairs"]
    if c["interleaved"]:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :r], x[..., r:2 * r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * r:]], -1)


def _plain_read(s, tokens):
    c = s["c"]
    there = torch.arange(tokens, device="cuda").view(1, 1, tokens, 1) < s["lengths"].view(-1, 1, 1, 1)
    return tuple(torch.where(there, _rows(s, name, tokens), 0.0).to(DTYPES[c["dtype"]]) for name in ("k", "v"))


def _plain_append(s):
    c = s["c"]
    hq, hkv = c["q_heads"], c["kv_heads"]
    x = s["qkv"].float()
    angle = s["positions"].double().view(-1, 1, 1) * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _rotated(_normed(x[:, :hq], s["q_weight"]), cos, sin, c)
    k = _rotated(_normed(x[:, hq:hq + hkv], s["k_weight"]), cos, sin, c)
    page, row = s["slots"].long() // c["page"], s["slots"].long() % c["page"]
    out = q.to(DTYPES[c["dtype"]])
    if c["int8"]:
        for name, y in (("k", k), ("v", x[:, hq + hkv:])):
            top = y.abs().amax(-1, keepdim=True)
            s[name][page, :, row] = torch.round(y * (127.0 / torch.where(top == 0, 1.0, top))).to(torch.int8)
            s[name + "_scale"][page, :, row] = top.squeeze(-1) / 127.0
        return (out,) + _plain_read(s, c["tokens"])
    s["k"][page, :, row] = k.to(s["k"].dtype)
    s["v"][page, :, row] = s["qkv"][:, hq + hkv:]
    return out, s["k"], s["v"]


def run(state):
    if own:
        return _run_own(state)
    kind = state["c"]["kind"]
    if kind == "masked":
        return _plain_masked(state)
    if kind == "paged":
        return _plain_paged(state)
    if kind == "append":
        return _plain_append(state)
    return _plain_read(state, state["c"]["longest"])


def work(case):
    c = case
    size = 1 if c.get("int8") else 2
    if c["kind"] == "masked":
        tq, tk = c["q_tokens"], c["k_tokens"]
        place = [i + tk - tq for i in range(tq)]
        seen = [p + 1 if c["causal"] else tk for p in place]
        if c["mask"] == "documents":      # nine documents of even length
            span = max(1, tk // 9)
            seen = [min(n, p % span + 1) for n, p in zip(seen, place)]
        elif c["mask"] == "prefix":       # half of the keys for everyone
            seen = [max(p + 1, tk // 2) for p in place]
        if c["window"]:
            seen = [min(n, c["window"]) for n in seen]
        pairs = c["batch"] * c["q_heads"] * sum(seen)
        rows = c["batch"] * c["dim"] * 2 * (2 * c["q_heads"] * tq + 2 * c["kv_heads"] * tk)
        return {"bytes": rows + (0 if c["mask"] == "none" else 8 * c["batch"] * tq), "flops": 4 * c["dim"] * pairs}
    if c["kind"] == "paged":
        tokens = (c["longest"] + (c["batch"] - 1) * 0.75 * c["longest"]) if not c["window"] else c["batch"] * min(c["window"], 0.75 * c["longest"])
        rows = tokens * c["kv_heads"]
        return {"bytes": rows * 2 * (c["dim"] * size + (4 if c["int8"] else 0)) + 4 * c["batch"] * c["q_heads"] * c["dim"] + 4 * c["batch"] * c["longest"] / c["page"],
                "flops": 4 * tokens * c["q_heads"] * c["dim"]}
    if c["kind"] == "append":
        heads = c["q_heads"] + 2 * c["kv_heads"]
        read = c["tokens"] * heads * c["dim"] * 2
        written = c["tokens"] * (c["q_heads"] * c["dim"] * 2 + 2 * c["kv_heads"] * (c["dim"] * size + (4 if c["int8"] else 0)))
        back = c["tokens"] * 2 * c["kv_heads"] * (3 * c["dim"] + 4) if c["int8"] else 0
        return {"bytes": read + written + back, "flops": 10 * c["tokens"] * heads * c["dim"]}
    there = (c["longest"] + (c["batch"] - 1) * 0.75 * c["longest"]) * c["kv_heads"]
    return {"bytes": 2 * (there * (c["dim"] * size + (4 if c["int8"] else 0)) + c["batch"] * c["longest"] * c["kv_heads"] * c["dim"] * 2),
            "flops": 2 * there * c["dim"]}


# ---- the definitions in 64 bits, a sequence (and a head) at a time ------------------------------------------------

def _exact_attention(q, k, v, scale, cap, slope, distance, seen):
    """q [n, d], k and v [t, d], distance and seen [n, t]"""
    z = (q @ k.t()) * scale
    if cap:
        z = cap * torch.tanh(z / cap)
    if slope is not None:
        z = z - slope * distance.double()
    z = z.masked_fill(~seen, -math.inf)
    alive = seen.any(1, keepdim=True)
    z = torch.softmax(z.masked_fill(~alive, 0.0), 1)
    return torch.where(alive, z @ v, 0.0)


def _exact_row(s, name, b, h, t):
    """rows 0 .. t - 1 of sequence b, head h in 64 bits"""
    c = s["c"]
    at = torch.arange(t, device="cuda")
    page, row = s["table"][b].long()[at // c["page"]], at % c["page"]
    x = s[name][page, h, row].double()
    return x * s[name + "_scale"][page, h, row].double().unsqueeze(-1) if c["int8"] else x


def _exact_turned(x, weight, positions, freq, c):
    """one head of every token: x [tokens, d]"""
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * weight.double()
    x = x.clone()
    r = c["pairs"]
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None] * freq.double()[None])
    one, two = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if c["interleaved"] else (slice(0, r), slice(r, 2 * r))
    y = torch.complex(x[:, one].contiguous(), x[:, two].contiguous()) * z
    x[:, one], x[:, two] = y.real, y.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["kind"] == "masked":
        tq, tk, group = c["q_tokens"], c["k_tokens"], c["q_heads"] // c["kv_heads"]
        out = torch.empty((c["batch"], tq, c["q_heads"], c["dim"]), dtype=torch.float64, device="cuda")
        key = torch.arange(tk, device="cuda")[None]
        for b in range(c["batch"]):
            for first in range(0, tq, 2048):
                rows = torch.arange(first, min(tq, first + 2048), device="cuda")
                away = rows[:, None] + (tk - tq) - key
                seen = (away >= 0) if c["causal"] else torch.ones_like(away, dtype=torch.bool)
                if c["window"]:
                    seen &= away < c["window"]
                if s["ranges"] is not None:
                    seen &= (key >= s["ranges"][b, rows, :1]) & (key < s["ranges"][b, rows, 1:])
                for h in range(c["q_heads"]):
                    out[b, rows, h] = _exact_attention(s["q"][b, h, rows].double(), s["k"][b, h // group].double(), s["v"][b, h // group].double(), c["dim"] ** -0.5,
                                                       c["cap"], s["slopes"][h].double() if c["bias"] else None, away.abs(), seen)
        return out.view(c["batch"], tq, -1)
    if c["kind"] == "paged":
        group = c["q_heads"] // c["kv_heads"]
        out = torch.zeros((c["batch"], c["q_heads"], c["dim"]), dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lengths"].tolist()):
            away = (n - 1 - torch.arange(n, device="cuda"))[None]
            seen = away < c["window"] if c["window"] else away >= 0
            for h in range(c["kv_heads"]):
                k, v = _exact_row(s, "k", b, h, n), _exact_row(s, "v", b, h, n)
                heads = slice(h * group, (h + 1) * group)
                out[b, heads] = _exact_attention(s["q"][b, heads].double(), k, v, c["dim"] ** -0.5, c["cap"],
                                                 s["slopes"][heads].double()[:, None] if c["bias"] else None, away.expand(group, n), seen.expand(group, n))
        return out
    if c["kind"] == "append":
        hq, hkv = c["q_heads"], c["kv_heads"]
        x = s["qkv"].double()
        turned = [_exact_turned(x[:, h], s["q_weight"] if h < hq else s["k_weight"], s["positions"], s["inv_freq"], c) for h in range(hq + hkv)]
        q = torch.stack(turned[:hq], 1)
        rows = {"k": torch.stack(turned[hq:], 1), "v": x[:, hq + hkv:]}
        if c["int8"]:
            for name, y in rows.items():
                step = y.abs().amax(-1, keepdim=True) / 127
                rows[name] = torch.round(y / torch.where(step == 0, 1.0, step)) * step
            return q, rows["k"].permute(1, 0, 2)[None], rows["v"].permute(1, 0, 2)[None]
        cache = {name: s[name].double() for name in ("k", "v")}
        for name, y in rows.items():
            cache[name].permute(0, 2, 1, 3)[s["slots"].long() // c["page"], s["slots"].long() % c["page"]] = y
        return q, cache["k"], cache["v"]
    got = []
    for name in ("k", "v"):
        y = torch.zeros((c["batch"], c["kv_heads"], c["longest"], c["dim"]), dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lengths"].tolist()):
            for h in range(c["kv_heads"]):
                y[b, h, :n] = _exact_row(s, name, b, h, n)
        got.append(y)
    return tuple(got)
