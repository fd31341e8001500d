"""The operators of a decode step over a 4-bit cache, as measurable cases: every one in its plain form and as the framework's calls.

The cases stand for (`op`):

  append  a step's tokens: the queries and keys rotated by their positions, the keys and values into the 4-bit cache
  attn    attention of the step's query tokens over that cache
  adapt   low-rank adapters, each request its own, beside a projection that all share: out = y + scale (x A^T) B^T

The cache holds a token of one head in groups of 64 numbers with a bf16 scale each, [pages, kv_heads, page_size, D / 64].
Of a group's numbers m is the one of largest magnitude (of two, the positive one); the scale is -m / 8 with five
significant bits, to nearest even, and 0 if |m| < 2^-90; a code is the fp32 quotient by the scale, to nearest even, in
-8..7.  (Code times scale is a bf16 number.)  Eight codes + 8 lie in a 32-bit word's nibbles 0, 4, 1, 5, 2, 6, 3, 7 in
this order.  K pages [pages, kv_heads, page_size, D / 2 bytes]: of D / 64 groups, word (D / 64) 2 g + 2 G + j of a token
holds the group G's numbers 16 g + 8 j + 0..7.  V pages [pages, kv_heads, page_size / 16, D, 8 bytes]: word h of a d
holds tokens 8 h + 0..7 of the 16.

The rotation turns the pair (x1, x2) of the angle position * inv_freq[i]: numbers i and i + rot / 2, or 2 i and 2 i + 1
where pairs are interleaved.  Angles, their sines and the rotated keys are taken in 64 bits, keys then rounded to fp32.
Codes come back as the bytes that hold them and have to be equal.

Lengths are fixed by the case (spread evenly between its bounds); values and page orders come from the seed.
"""
import math

import torch

own = False

WORKSPACE = 256 << 20  # one scratch buffer for every operator of the program's stream


def listed():
    return [
        # one chat's next token: the smallest step, where only latency counts
        {"name": "append_decode_1", "op": "append", "b": 1, "pos_lo": 900, "pos_hi": 900, "new": 1, "hq": 32, "hkv": 8, "d": 128,
         "page": 16, "rot": 128, "inter": False},
        # one token of each of 64 sequences, some of them far along
        {"name": "append_decode_64", "op": "append", "b": 64, "pos_lo": 3, "pos_hi": 100000, "new": 1, "hq": 32, "hkv": 8, "d": 128,
         "page": 16, "rot": 128, "inter": False},
        # five draft tokens for each of 16 sequences, head size 64, half of it rotated, in interleaved pairs
        {"name": "append_draft_16", "op": "append", "b": 16, "pos_lo": 1000, "pos_hi": 3000, "new": 5, "hq": 16, "hkv": 16, "d": 64,
         "page": 32, "rot": 32, "inter": True},
        # five prompts of about 1600 tokens, some behind a cached beginning, in larger pages
        {"name": "append_prefill_8000", "op": "append", "b": 5, "pos_lo": 0, "pos_hi": 75, "new": 1600, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "rot": 128, "inter": False},
        # one sequence of 2000 tokens, one new token: latency
        {"name": "attn_decode_1x2000", "op": "attn", "b": 1, "hq": 32, "hkv": 8, "d": 128, "page": 16, "new": 1,
         "ctx_lo": 2000, "ctx_hi": 2000},
        # 64 sequences of very different lengths, one new token each: bound by reading the cache
        {"name": "attn_decode_64x8000", "op": "attn", "b": 64, "hq": 32, "hkv": 8, "d": 128, "page": 16, "new": 1,
         "ctx_lo": 90, "ctx_hi": 8000},
        # five draft tokens for each of 16 sequences, head size 64, heads of their own
        {"name": "attn_draft_16x3000", "op": "attn", "b": 16, "hq": 16, "hkv": 16, "d": 64, "page": 32, "new": 5,
         "ctx_lo": 1000, "ctx_hi": 3000},
        # a prompt in pieces: 700 tokens of each of four sequences over what is cached of them: bound by the products
        {"name": "attn_chunk_4x700", "op": "attn", "b": 4, "hq": 32, "hkv": 8, "d": 128, "page": 64, "new": 700,
         "ctx_lo": 1100, "ctx_hi": 4100},
        # one request's token beside a 4096 -> 4096 projection
        {"name": "adapt_decode_1", "op": "adapt", "b": 1, "new": 1, "n": 4096, "k": 4096, "rank": 16, "loaded": 8, "every": 0},
        # 64 requests' tokens and 40 adapters, every fifth request without one, beside a 4096 -> 11008 projection
        {"name": "adapt_decode_64", "op": "adapt", "b": 64, "new": 1, "n": 11008, "k": 4096, "rank": 16, "loaded": 40, "every": 5},
        # draft tokens, small layers and a size that is no multiple of anything
        {"name": "adapt_draft_20x5", "op": "adapt", "b": 20, "new": 5, "n": 1001, "k": 2056, "rank": 8, "loaded": 20, "every": 4},
        # five prompts of 400 tokens with adapters of rank 64
        {"name": "adapt_prefill_2000", "op": "adapt", "b": 5, "new": 400, "n": 11008, "k": 4096, "rank": 64, "loaded": 6, "every": 0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw(rng, op):
    if op == "append":
        hkv, d, page = rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([64, 128]), rng.choice([16, 16, 32, 64, 128])
        if rng.random() < 0.6:
            b, new = _log(rng, 1, 300), rng.choice([1, 1, 1, 2, 5])
        else:
            b, new = _log(rng, 1, 16), _log(rng, 20, 4000)
        lo = _log(rng, 1, 200000) - 1
        return {"op": op, "b": b, "pos_lo": lo, "pos_hi": lo + rng.randint(0, 5000), "new": new,
                "hq": hkv * rng.choice([1, 1, 2, 4, 7, 8]), "hkv": hkv, "d": d, "page": page,
                "rot": rng.choice([d, d, d // 2, d // 4]), "inter": rng.random() < 0.3}
    if op == "attn":
        hkv, d, page = rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([64, 128]), rng.choice([16, 16, 32, 64, 128])
        new = rng.choice([1, 1, 1, 2, 5, _log(rng, 8, 1000)])
        hi = new + _log(rng, 1, 16000)
        return {"op": op, "b": _log(rng, 1, 100), "hq": hkv * rng.choice([1, 1, 2, 4, 7, 8]), "hkv": hkv, "d": d, "page": page,
                "new": new, "ctx_lo": rng.randint(new, hi), "ctx_hi": hi}
    b, new = (_log(rng, 1, 200), rng.choice([1, 1, 1, 2, 5])) if rng.random() < 0.6 else (_log(rng, 1, 16), _log(rng, 6, 1500))
    return {"op": op, "b": b, "new": new, "n": _log(rng, 100, 12000), "k": 8 * _log(rng, 32, 1376),
            "rank": rng.choice([8, 16, 16, 32, 64]), "loaded": _log(rng, 1, 64), "every": rng.choice([0, 0, 3, 10])}


def draw(rng):
    op = rng.choice([c["op"] for c in listed()])
    costs = [work(c) for c in listed() if c["op"] == op]
    most = {key: max(c[key] for c in costs) for key in ("bytes", "flops")}
    while True:
        case = _draw(rng, op)
        cost = work(case)
        if cost["bytes"] <= most["bytes"] and cost["flops"] <= most["flops"]:
            return case


# ── lengths ─────────────────────────────────────────────────────────────────


def _spread(low, high, n):
    """n lengths over [low, high], the longest first met neither first nor last."""
    return [low + int((high - low) * ((0.5 + 0.6180339887 * i) % 1) + 0.5) if n > 1 else high for i in range(n)]


def _pages(length, page):
    return -(-length // page)


def _append_lengths(case):
    """(position of the first new token, new tokens) of every sequence."""
    return (_spread(case["pos_lo"], case["pos_hi"], case["b"]),
            [case["new"] + (i % 3 if case["new"] > 8 else 0) for i in range(case["b"])])


def _contexts(case):
    return _spread(case["ctx_lo"], case["ctx_hi"], case["b"])


def _requests(case):
    """(adapter or -1, tokens) of every request."""
    every = case["every"]
    return [(-1 if every and i % every == every - 1 else (7 * i + 3) % case["loaded"],
             case["new"] + (i % 3 if case["new"] > 8 else 0)) for i in range(case["b"])]


# ── what the program holds ──────────────────────────────────────────────────


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _five_bits(x):
    """fp32 with five significant bits, to nearest even."""
    u = x.contiguous().view(torch.int32)
    return ((u + 0x3FFFF + ((u >> 19) & 1)) & ~0x7FFFF).view(torch.float32)


def _random_codes(shape, gen):
    """Bytes of two codes each, normally distributed."""
    c = torch.randn((*shape, 2), generator=gen, device="cuda").mul_(2.9).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    return (c[..., 0] | (c[..., 1] << 4)).view(torch.int8)


def _random_scales(shape, gen):
    sign = torch.randint(0, 2, shape, generator=gen, device="cuda") * 2 - 1
    return _five_bits((torch.rand(shape, generator=gen, device="cuda") * 0.6 + 0.7) / 2.9 * sign).bfloat16()


def _random_cache(pages, case, gen):
    h, d, page = case["hkv"], case["d"], case["page"]
    return {"k_cache": _random_codes((pages, h, page, d // 2), gen), "v_cache": _random_codes((pages, h, page // 16, d, 8), gen),
            "k_scale": _random_scales((pages, h, page, d // 64), gen), "v_scale": _random_scales((pages, h, page, d // 64), gen)}


def _inputs_append(case, gen):
    hkv, d, page = case["hkv"], case["d"], case["page"]
    first, new = _append_lengths(case)
    tokens = sum(new)
    # the pool holds the pages that the new tokens lie in, in random order
    counts = [_pages(p + n, page) - p // page for p, n in zip(first, new)]
    pages = sum(counts)
    order = torch.randperm(pages, generator=gen, device="cuda")
    base = [sum(counts[:i]) - p // page for i, p in enumerate(first)]
    at = torch.tensor([p + i for p, n in zip(first, new) for i in range(n)], device="cuda")
    row = torch.tensor([x for x, n in zip(base, new) for _ in range(n)], device="cuda")
    slots = order[row + at // page] * page + at % page
    # keys have channels that stand out
    wide = 1 + 5 * (torch.rand(hkv, d, generator=gen, device="cuda") < 0.03)
    made = {"q": torch.randn(tokens, case["hq"], d, generator=gen, device="cuda").bfloat16(),
            "k": (torch.randn(tokens, hkv, d, generator=gen, device="cuda") * wide).bfloat16(),
            "v": torch.randn(tokens, hkv, d, generator=gen, device="cuda").bfloat16(),
            "positions": at.to(torch.int32), "slots": slots.to(torch.int32)}
    made["inv_freq"] = 10000.0 ** (-torch.arange(case["rot"] // 2, device="cuda") * 2 / case["rot"])
    made.update(_random_cache(pages, case, gen))
    return made


def _inputs_attn(case, gen):
    b, d, page, new = case["b"], case["d"], case["page"], case["new"]
    ctx = _contexts(case)
    counts = [_pages(n, page) for n in ctx]
    pages, width = sum(counts) + 3, max(counts)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None] < _ints(counts)[:, None]] = order[:sum(counts)]
    q = torch.randn(b * new, case["hq"], d, generator=gen, device="cuda").bfloat16()
    return {"q": q, **_random_cache(pages, case, gen), "block_table": table, "context_lens": _ints(ctx),
            "q_starts": _ints([new * i for i in range(b + 1)])}


def _inputs_adapt(case, gen):
    n, k, rank, loaded = case["n"], case["k"], case["rank"], case["loaded"]
    ids = [a for a, count in _requests(case) for _ in range(count)]
    m = len(ids)
    return {"x": torch.randn(m, k, generator=gen, device="cuda").bfloat16(),
            "a": (torch.randn(loaded, rank, k, generator=gen, device="cuda") / math.sqrt(k)).bfloat16(),
            "b": (torch.randn(loaded, n, rank, generator=gen, device="cuda") * 0.3).bfloat16(),
            "scale": torch.rand(loaded, generator=gen, device="cuda") * 1.5 + 0.25,
            "adapters": _ints(ids), "y": torch.randn(m, n, generator=gen, device="cuda").bfloat16()}


_INPUTS = {"append": _inputs_append, "attn": _inputs_attn, "adapt": _inputs_adapt}


def _inputs(case, seed):
    return _INPUTS[case["op"]](case, torch.Generator(device="cuda").manual_seed(seed))


def _results(case, made):
    """bf16 outputs that the program keeps: {name: shape}."""
    name, like = {"append": ("q_out", "q"), "attn": ("o", "q"), "adapt": ("out", "y")}[case["op"]]
    return {name: made[like].shape}


class _Array:
    """A framework buffer as torch sees it (no copy; keeps the buffer alive)."""

    def __init__(self, buf):
        self.buf = buf
        kind = {"f32": "<f4", "bf16": "<i2", "i8": "|i1", "i32": "<i4"}[buf.dtype.name]
        self.__cuda_array_interface__ = {"shape": buf.shape, "typestr": kind, "data": (buf.ptr, False), "version": 3}


def _buffer(dev, shape, dtype):
    """(the framework's buffer, torch's view of it)."""
    name = {torch.float32: "f32", torch.bfloat16: "bf16", torch.int8: "i8", torch.int32: "i32"}[dtype]
    buf = dev.buffer(name, tuple(shape))
    view = torch.as_tensor(_Array(buf), device="cuda")
    return buf, view.view(torch.bfloat16) if dtype == torch.bfloat16 else view


def prepare(case, seed):
    made = _inputs(case, seed)
    state = {"case": case, "in": made}
    if own:  # the same inputs in the framework's buffers, and the workspace that its program attached at its start
        import teenygrad_amd as tg
        from teenygrad_amd.runtime import NULL_STREAM

        dev = tg.open(0)
        if NULL_STREAM._workspace is None:
            NULL_STREAM.set_workspace(dev.buffer(tg.i8, (WORKSPACE,)))
        state["kernels"], state["in"], state["view"] = tg.kernels, {}, {}
        for name, t in made.items():
            state["in"][name], state["view"][name] = _buffer(dev, t.shape, t.dtype)
            state["view"][name].copy_(t)
        for name, shape in _results(case, made).items():
            state["in"][name], state["view"][name] = _buffer(dev, shape, torch.bfloat16)
    return state


# ── one pass ────────────────────────────────────────────────────────────────


def _own_append(K, case, i):
    K.kv4_cache_append(i["q"], i["k"], i["v"], i["positions"], i["slots"], i["inv_freq"], i["k_cache"], i["v_cache"],
                       i["k_scale"], i["v_scale"], interleaved=case["inter"], q_out=i["q_out"])


def _own_attn(K, case, i):
    K.kv4_cache_attention(i["q"], i["k_cache"], i["v_cache"], i["k_scale"], i["v_scale"], i["block_table"], i["context_lens"],
                          i["q_starts"], max_q_len=case["new"], max_context=case["ctx_hi"], o=i["o"])


def _own_adapt(K, case, i):
    K.adapter_add(i["x"], i["a"], i["b"], i["adapters"], i["y"], scale=i["scale"], out=i["out"])


_NIBBLES = (0, 4, 1, 5, 2, 6, 3, 7)


def _rotated(x, i, inter):
    """x [T, H, D] in 64 bits, its first numbers rotated."""
    half = i["inv_freq"].numel()
    angle = (i["positions"].double()[:, None] * i["inv_freq"].double())[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    x = x.double()
    x1, x2 = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if inter else (x[..., :half], x[..., half:2 * half])
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    both = torch.stack([y1, y2], -1).flatten(-2) if inter else torch.cat([y1, y2], -1)
    return torch.cat([both, x[..., 2 * half:]], -1)


def _plain_codes(x):
    """x [T, H, D] fp32 -> (codes + 8 [T, H, D] int32, scales [T, H, D / 64])."""
    t, h, d = x.shape
    x = x.reshape(t, h, d // 64, 64)
    high, low = x.amax(-1), x.amin(-1)
    most = torch.where(high >= -low, high, low)
    scale = torch.where(most.abs() < 2.0 ** -90, 0.0, _five_bits(most / -8))
    codes = torch.where(scale[..., None] == 0, 0.0, x / scale[..., None]).round().clamp(-8, 7).to(torch.int32) + 8
    return codes.reshape(t, h, d), scale.bfloat16()


def _plain_append(case, i):
    d, page = case["d"], case["page"]
    slots = i["slots"].long()
    where, off = slots // page, slots % page
    shift = torch.tensor([4 * p for p in _NIBBLES], dtype=torch.int32, device=slots.device)
    codes, scale = _plain_codes(_rotated(i["k"], i, case["inter"]).float())
    words = (codes.reshape(-1, case["hkv"], d // 64, 4, 2, 8) << shift).sum(-1, dtype=torch.int32)
    i["k_cache"].view(torch.int32)[where, :, off] = words.transpose(2, 3).flatten(2)
    i["k_scale"][where, :, off] = scale
    codes, scale = _plain_codes(i["v"].float())
    v_words = i["v_cache"].view(torch.int32)
    for o in range(16):  # tokens that share a word one after the other
        mine = torch.nonzero(off % 16 == o)[:, 0]
        at = where[mine], slice(None), off[mine] // 16, slice(None), o // 8
        place = 4 * _NIBBLES[o % 8]
        keep = ~(15 << place) if place < 28 else 0x0FFFFFFF
        v_words[at] = (v_words[at] & keep) | (codes[mine] << place)
    i["v_scale"][where, :, off] = scale
    return {"q_out": _rotated(i["q"], i, case["inter"]).float().bfloat16(),
            **{n: i[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}}


def _plain_values(i, pages, d):
    """K and V fp32 [..., page_size, D] of the given pages' heads."""
    shift = torch.tensor([4 * p for p in _NIBBLES], dtype=torch.int32, device=pages.device)
    k = ((i["k_cache"].view(torch.int32)[pages][..., None] >> shift) & 15) - 8  # [..., page, words, 8]
    k = k.unflatten(-2, (4, d // 64, 2)).transpose(-4, -3).flatten(-4)
    v = ((i["v_cache"].view(torch.int32)[pages][..., None] >> shift) & 15) - 8  # [..., page / 16, d, 2, 8]
    v = v.flatten(-2).transpose(-2, -1).flatten(-3, -2)
    return (k.float() * i["k_scale"][pages].float().repeat_interleave(64, -1),
            v.float() * i["v_scale"][pages].float().repeat_interleave(64, -1))


def _plain_attn(case, i):
    b, new, hq, hkv, d, page = (case[n] for n in ("b", "new", "hq", "hkv", "d", "page"))
    group = hq // hkv
    pages = i["block_table"][:, :_pages(case["ctx_hi"], page)].clamp(min=0).long()
    k, v = _plain_values(i, pages, d)  # [b, w, h, page, d]
    k, v = (x.transpose(1, 2).reshape(b * hkv, -1, d) for x in (k, v))
    q = i["q"].float().reshape(b, new, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b * hkv, group * new, d)
    s = torch.bmm(q, k.mT.contiguous()) * (1 / math.sqrt(d))
    key = torch.arange(s.shape[-1], device=s.device)
    last = i["context_lens"][:, None] - new + torch.arange(new, device=s.device)  # [b, new]
    hidden = (key > last[..., None])[:, None, None]
    s = s.reshape(b, hkv, group, new, -1).masked_fill_(hidden, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.bmm(p.reshape(b * hkv, group * new, -1), v)
    return {"o": o.reshape(b, hkv, group, new, d).permute(0, 3, 1, 2, 4).reshape(b * new, hq, d).bfloat16()}


def _plain_adapt(case, i):
    x, y = i["x"].float(), i["y"].float()
    if case["new"] <= 8:  # every token its own copy of its adapter
        ids = i["adapters"].long()
        of = ids.clamp(min=0)
        h = torch.bmm(i["a"][of].float(), x[..., None]) * i["scale"][of][:, None, None]
        more = torch.bmm(i["b"][of].float(), h)[..., 0]
        return {"out": (y + torch.where(ids[:, None] >= 0, more, 0.0)).bfloat16()}
    at = 0
    for adapter, count in _requests(case):
        if adapter >= 0:
            h = x[at:at + count] @ i["a"][adapter].float().T * i["scale"][adapter]
            y[at:at + count] += h @ i["b"][adapter].float().T
        at += count
    return {"out": y.bfloat16()}


_OUTPUTS = {"append": ("q_out", "k_cache", "v_cache", "k_scale", "v_scale"), "attn": ("o",), "adapt": ("out",)}
_OWN = {"append": _own_append, "attn": _own_attn, "adapt": _own_adapt}
_PLAIN = {"append": _plain_append, "attn": _plain_attn, "adapt": _plain_adapt}


def run(state):
    op = state["case"]["op"]
    if own:
        _OWN[op](state["kernels"], state["case"], state["in"])
        return {n: state["view"][n] for n in _OUTPUTS[op]}
    return _PLAIN[op](state["case"], state["in"])


# ── what a pass cannot do without ───────────────────────────────────────────


def work(case):
    op = case["op"]
    if op == "append":
        tokens, hq, hkv, d = sum(_append_lengths(case)[1]), case["hq"], case["hkv"], case["d"]
        held = d // 2 + 2 * (d // 64)
        # q in and out, k and v in, codes and scales out, positions and slots, the frequencies
        return {"bytes": tokens * (4 * hq * d + 4 * hkv * d + 2 * hkv * held + 8) + 2 * case["rot"],
                "flops": tokens * (3 * (hq + hkv) * case["rot"] + 2 * hkv * d * 6)}
    if op == "attn":
        b, new, hq, hkv, d, page = (case[n] for n in ("b", "new", "hq", "hkv", "d", "page"))
        ctx = _contexts(case)
        pairs = sum(new * c - new * (new - 1) // 2 for c in ctx)
        cache = sum(2 * hkv * c * (d // 2 + 2 * (d // 64)) + 4 * _pages(c, page) for c in ctx)
        return {"bytes": cache + 2 * 2 * b * new * hq * d, "flops": 4 * hq * pairs * d}
    asked = _requests(case)
    n, k, rank = case["n"], case["k"], case["rank"]
    m, with_one = sum(c for _, c in asked), sum(c for a, c in asked if a >= 0)
    used = len({a for a, _ in asked if a >= 0})
    return {"bytes": 2 * with_one * k + 4 * m * n + 2 * used * rank * (k + n) + 4 * m + 4 * used,
            "flops": 2 * with_one * rank * (k + n)}


# ── the same in 64 bits ─────────────────────────────────────────────────────


def _exact_turn(x, t, inter):
    """x [T, H, D] rotated, as complex numbers times exp(i angle)."""
    half = t["inv_freq"].numel()
    x = x.double()
    pairs = x[..., :2 * half].unflatten(-1, (half, 2) if inter else (2, half))
    re, im = pairs.unbind(-1 if inter else -2)
    angle = torch.outer(t["positions"].double(), t["inv_freq"].double())[:, None]
    turned = torch.complex(re, im) * torch.polar(torch.ones_like(angle), angle)
    out = x.clone()
    out[..., :2 * half] = torch.view_as_real(turned).flatten(-2) if inter else torch.cat([turned.real, turned.imag], -1)
    return out


def _exact_scales(old, x, slots, page):
    t, h, d = x.shape
    groups = x.reshape(t, h, d // 64, 64).double()
    # a positive number counts a little more than a negative one of the same magnitude
    place = (groups.abs() * (1 + (groups > 0).double() * 2.0 ** -40)).argmax(-1, keepdim=True)
    most = groups.gather(-1, place)[..., 0]
    part, power = torch.frexp(most / -8)
    scale = torch.ldexp((part * 32).round(), power - 5)
    new = old.double().clone()
    new[slots.long() // page, :, slots.long() % page] = torch.where(most.abs() < 2.0 ** -90, 0.0, scale)
    return new


def _exact_append(case, t):
    k = _exact_turn(t["k"], t, case["inter"]).float()  # keys are held by their fp32 values
    return {"q_out": _exact_turn(t["q"], t, case["inter"]), "k_cache": None, "v_cache": None,  # the codes are whole numbers
            "k_scale": _exact_scales(t["k_scale"], k, t["slots"], case["page"]),
            "v_scale": _exact_scales(t["v_scale"], t["v"], t["slots"], case["page"])}


def _exact_nibbles(cache):
    """Bytes [..., 4 w] -> codes [..., 8 w] in 64 bits."""
    raw = cache.view(torch.uint8).unflatten(-1, (-1, 4)).to(torch.int16)
    both = torch.stack([raw & 15, raw >> 4], -1).flatten(-2)  # nibbles 0..7 of each word
    return both[..., list(_NIBBLES)].flatten(-2).double() - 8


def _exact_attn(case, t):
    new, hkv, group, d, page = case["new"], case["hkv"], case["hq"] // case["hkv"], case["d"], case["page"]
    # numbers 64 G + 16 g + e of a K row lie at 16 (D / 64) g + 16 G + e
    n = torch.arange(d, device="cuda")
    place = 16 * (d // 64) * (n % 64 // 16) + 16 * (n // 64) + n % 16
    outs = []
    for b, ctx in enumerate(_contexts(case)):
        pages = t["block_table"][b, :_pages(ctx, page)].long()
        k = _exact_nibbles(t["k_cache"][pages])[..., place]  # [w, h, page, d]
        v = _exact_nibbles(t["v_cache"][pages]).transpose(-1, -2).reshape(k.shape)
        k, v = (x.unflatten(-1, (-1, 64)) * s[pages].double()[..., None] for x, s in ((k, t["k_scale"]), (v, t["v_scale"])))
        k, v = (x.transpose(0, 1).reshape(hkv, -1, d)[:, :ctx].repeat_interleave(group, 0) for x in (k, v))
        s = t["q"][b * new:(b + 1) * new].double().transpose(0, 1) @ k.mT.contiguous() / math.sqrt(d)
        seen = torch.ones(new, ctx, dtype=torch.bool, device=s.device).tril(ctx - new)
        outs.append((torch.softmax(s.where(seen, -math.inf), -1) @ v).transpose(0, 1))
    return {"o": torch.cat(outs)}


def _exact_adapt(case, t):
    out, at = t["y"].double(), 0
    for adapter, count in _requests(case):
        if adapter >= 0:
            both = t["b"][adapter].double() @ t["a"][adapter].double() * t["scale"][adapter].double()  # [n, k]
            out[at:at + count] += t["x"][at:at + count].double() @ both.T.contiguous()
        at += count
    return {"out": out}


def exact(case, seed):
    t = _inputs(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "adapt": _exact_adapt}[case["op"]](case, t)
