"""The operators of a quantized decode step, as measurable cases: every one in its plain form and as the framework's calls.

The cases stand for (`op`):

  plan    the start of a step: pages for the tokens that each request adds, pages of ended requests back, and the
          slots, positions and row starts that the other operators of the step read
  write   the step's K and V into the 8-bit cache, one scale for each page and head
  attn    attention of the step's query tokens over that cache
  w4      a linear layer with 4-bit weights and group scales, for one token, a few, or whole prompts

The cache: K pages [pages, kv_heads, page_size, head_dim], V pages transposed, [pages, kv_heads, head_dim, page_size],
int8, with fp32 scales [pages, kv_heads].  Codes come back as the int8 numbers they are and have to be equal.

4-bit weights [N, K]: rows padded to whole chunks of 128, 64 bytes each.  In a chunk the 32-bit word 4 g + c holds
k = 32 c + 8 g + 0..7, code + 8 in the nibbles 0, 4, 1, 5, 2, 6, 3, 7 in this order.

Lengths are fixed by the case (spread evenly between its bounds); values and page orders come from the seed.
"""
import math
import random

import torch

own = False

WORKSPACE = 256 << 20  # one scratch buffer for every operator of the program's stream


def listed():
    return [
        # eight chats, one token each: the smallest step, where only latency counts
        {"name": "plan_decode_8", "op": "plan", "b": 8, "seq_lo": 40, "seq_hi": 900, "prompts": 0, "prompt": 0, "ended": 0,
         "page": 16, "width": 64},
        # a busy server's step: 512 requests, most of them decoding, some new prompts, some that end
        {"name": "plan_mixed_512", "op": "plan", "b": 512, "seq_lo": 1, "seq_hi": 8000, "prompts": 9, "prompt": 1500,
         "ended": 17, "page": 16, "width": 640},
        # one token of each of 64 sequences, 8 K/V heads
        {"name": "write_decode_64", "op": "write", "b": 64, "before_lo": 3, "before_hi": 400, "new": 1, "h": 8, "d": 128,
         "page": 16},
        # five prompts of about 1600 tokens, one of them behind a cached beginning, in larger pages
        {"name": "write_prefill_8000", "op": "write", "b": 5, "before_lo": 0, "before_hi": 75, "new": 1600, "h": 8, "d": 128,
         "page": 64},
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
        # one token through a 4096 -> 11008 layer
        {"name": "w4_decode_1", "op": "w4", "m": 1, "n": 11008, "k": 4096, "group": 128, "zero": False, "act": ""},
        # 16 tokens, small groups with zero points
        {"name": "w4_decode_16_zp", "op": "w4", "m": 16, "n": 4096, "k": 4096, "group": 32, "zero": True, "act": ""},
        # an ordinary batch, with the activation behind it
        {"name": "w4_batch_50", "op": "w4", "m": 50, "n": 5504, "k": 2048, "group": 64, "zero": False, "act": "silu"},
        # prompts of 2000 tokens together: bound by the products
        {"name": "w4_prefill_2000", "op": "w4", "m": 2000, "n": 11008, "k": 4096, "group": 128, "zero": False, "act": ""},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw(rng, op):
    if op == "plan":
        b, page, width = _log(rng, 1, 700), rng.choice([16, 16, 32, 64, 128]), _log(rng, 4, 700)
        hi = _log(rng, 1, page * width)
        return {"op": op, "b": b, "seq_lo": min(hi, _log(rng, 1, 400)), "seq_hi": hi, "prompts": rng.randint(0, b // 16),
                "prompt": rng.randint(1, 2000), "ended": rng.randint(0, b // 8), "page": page, "width": width}
    if op == "write":
        page, h, d = rng.choice([16, 16, 32, 64, 128]), rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([64, 128])
        if rng.random() < 0.5:
            return {"op": op, "b": _log(rng, 1, 200), "before_lo": 0, "before_hi": rng.randint(0, 600), "new": rng.choice([1, 1, 1, 2, 5]),
                    "h": h, "d": d, "page": page}
        return {"op": op, "b": _log(rng, 1, 16), "before_lo": 0, "before_hi": rng.randint(0, 300), "new": _log(rng, 20, 4000),
                "h": h, "d": d, "page": page}
    if op == "attn":
        hkv, d, page = rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([64, 128]), rng.choice([16, 16, 32, 64, 128])
        hq = hkv * rng.choice([1, 1, 2, 4, 7, 8])
        new = rng.choice([1, 1, 1, 2, 5, _log(rng, 8, 1000)])
        hi = new + _log(rng, 1, 16000)
        return {"op": op, "b": _log(rng, 1, 100), "hq": hq, "hkv": hkv, "d": d, "page": page, "new": new,
                "ctx_lo": rng.randint(new, hi), "ctx_hi": hi}
    k = 8 * round(_log(rng, 256, 11008) / 8)
    if rng.random() < 0.7:
        k = max(256, 128 * round(k / 128))
    return {"op": op, "m": rng.choice([1, 1, _log(rng, 1, 64), _log(rng, 1, 2000)]), "n": _log(rng, 100, 12000), "k": k,
            "group": rng.choice([32, 64, 128, 128]), "zero": rng.random() < 0.4, "act": rng.choice(["", "", "silu", "gelu"])}


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


def _plan_lengths(case):
    """(cached tokens, tokens to add: -1 ends the request) of every request; what does not fit a row is cut."""
    b, most = case["b"], case["page"] * case["width"]
    seq = [min(x, most - 1) for x in _spread(case["seq_lo"], case["seq_hi"], b)]
    new = [1] * b
    order = list(range(b))
    random.Random(b).shuffle(order)
    for i in order[:case["prompts"]]:
        seq[i], new[i] = 0, min(most, case["prompt"] + i)
    for i in order[case["prompts"]:case["prompts"] + case["ended"]]:
        new[i] = -1
    return seq, new


def _plan_pages(case):
    seq, new = _plan_lengths(case)
    held = sum(_pages(s, case["page"]) for s in seq)
    return held, held + sum(_pages(max(n, 0), case["page"]) + 1 for n in new)


def _write_lengths(case):
    before = _spread(case["before_lo"], case["before_hi"], case["b"])
    return before, [case["new"] + (i % 3 if case["new"] > 8 else 0) for i in range(case["b"])]


def _contexts(case):
    return _spread(case["ctx_lo"], case["ctx_hi"], case["b"])


# ── what the program holds ──────────────────────────────────────────────────


def _ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _table(lengths, page, width, pages, gen):
    """A block table whose pages lie in random order: (table [b, width], -1 behind each row's pages; the other pages)."""
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    counts = torch.tensor([_pages(n, page) for n in lengths], device="cuda")
    held = torch.arange(width, device="cuda")[None] < counts[:, None]
    used = int(counts.sum())
    table[held] = order[:used]
    return table, order[used:]


def _inputs_plan(case, gen):
    seq, new = _plan_lengths(case)
    held, pages = _plan_pages(case)
    table, free = _table(seq, case["page"], case["width"], pages, gen)
    stack = torch.zeros(pages, dtype=torch.int32, device="cuda")
    stack[:free.numel()] = free
    return {"new_lens": _ints(new), "seq_lens": _ints(seq), "block_table": table, "free_list": stack,
            "free_count": _ints([free.numel()])}


def _inputs_write(case, gen):
    h, d, page = case["h"], case["d"], case["page"]
    before, new = _write_lengths(case)
    after = [a + n for a, n in zip(before, new)]
    width = max(_pages(n, page) for n in after)
    pages = sum(_pages(n, page) for n in after)
    table, _ = _table(after, page, width, pages, gen)
    tokens = sum(new)
    at = torch.tensor([a + i for a, n in zip(before, new) for i in range(n)], device="cuda")
    row = torch.tensor([i for i, n in enumerate(new) for _ in range(n)], device="cuda")
    slots = table[row, at // page] * page + at % page
    # keys have channels that stand out; the tokens cached before are a little smaller, so that some scales grow
    wide = 1 + 5 * (torch.rand(h, d, generator=gen, device="cuda") < 0.03)
    k = (torch.randn(tokens, h, d, generator=gen, device="cuda") * wide).bfloat16()
    v = torch.randn(tokens, h, d, generator=gen, device="cuda").bfloat16()
    codes = {n: torch.randint(-127, 128, s, generator=gen, device="cuda", dtype=torch.int8)
             for n, s in (("k_cache", (pages, h, page, d)), ("v_cache", (pages, h, d, page)))}
    scales = {n: torch.rand(pages, h, generator=gen, device="cuda") * t + t
              for n, t in (("k_scale", 0.05), ("v_scale", 0.012))}
    return {"k": k, "v": v, "slots": slots.to(torch.int32), **codes, **scales}


def _inputs_attn(case, gen):
    b, hkv, d, page, new = case["b"], case["hkv"], case["d"], case["page"], case["new"]
    ctx = _contexts(case)
    width = max(_pages(n, page) for n in ctx)
    pages = sum(_pages(n, page) for n in ctx) + 3
    table, _ = _table(ctx, page, width, pages, gen)
    q = torch.randn(b * new, case["hq"], d, generator=gen, device="cuda").bfloat16()
    codes = {n: torch.randn(s, generator=gen, device="cuda").mul_(38).round_().clamp_(-127, 127).to(torch.int8)
             for n, s in (("k_cache", (pages, hkv, page, d)), ("v_cache", (pages, hkv, d, page)))}
    scales = {n: (torch.rand(pages, hkv, generator=gen, device="cuda") * 0.4 + 0.8) / 38 for n in ("k_scale", "v_scale")}
    return {"q": q, **codes, **scales, "block_table": table, "context_lens": _ints(ctx),
            "q_starts": _ints([new * i for i in range(b + 1)])}


_NIBBLES = (0, 4, 1, 5, 2, 6, 3, 7)


def _pack(codes):
    """[N, K] int codes in -8..7 -> [N, ceil(K / 128) * 64] bytes."""
    n, k = codes.shape
    chunks = _pages(k, 128)
    full = torch.full((n, chunks * 128), 8, dtype=torch.int64, device=codes.device)
    full[:, :k] = codes.to(torch.int64) + 8
    words = full.reshape(n, chunks, 4, 4, 8).transpose(2, 3)  # [n, chunk, g, c, 8]
    shift = torch.tensor([4 * p for p in _NIBBLES], device=codes.device)
    words = (words << shift).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    return words.reshape(n, -1).contiguous().view(torch.int8)


def _inputs_w4(case, gen):
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    groups = _pages(k, group)
    x = torch.randn(m, k, generator=gen, device="cuda").bfloat16()
    w = torch.zeros(n, groups * group, device="cuda")
    w[:, :k] = torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k)
    w = w.reshape(n, groups, group)
    made = {"x": x}
    if case["zero"]:
        low, high = w.amin(-1).clamp_(max=0), w.amax(-1).clamp_(min=0)
        scale = (high - low) / 15
        zero = (-8 - low / scale).round_().clamp_(-8, 7)
        made["zero_point"] = zero.to(torch.int32)
        codes = (w / scale[..., None] + zero[..., None]).round_().clamp_(-8, 7)
    else:
        scale = w.abs().amax(-1) / 7
        codes = (w / scale[..., None]).round_().clamp_(-7, 7)
    made["scale"] = scale.contiguous()
    made["qweight"] = _pack(codes.reshape(n, -1)[:, :k])
    made["bias"] = torch.randn(n, generator=gen, device="cuda") * 0.02
    return made


_INPUTS = {"plan": _inputs_plan, "write": _inputs_write, "attn": _inputs_attn, "w4": _inputs_w4}


def _inputs(case, seed):
    return _INPUTS[case["op"]](case, torch.Generator(device="cuda").manual_seed(seed))


def _step_tokens(case):
    """Tokens that a step has room for: those of the case and a few rows of padding, as a captured step has."""
    return sum(max(n, 0) for n in _plan_lengths(case)[1]) + 3


def _results(case):
    """Outputs that the program keeps: {name: (shape, torch dtype)}."""
    if case["op"] == "plan":
        t, b = (_step_tokens(case),), (case["b"],)
        return {n: (s, torch.int32) for n, s in (("slots", t), ("positions", t), ("q_starts", (case["b"] + 1,)),
                                                 ("context_lens", b), ("granted", b), ("free_after", (1,)))}
    if case["op"] == "attn":
        return {"o": ((case["b"] * case["new"], case["hq"], case["d"]), torch.bfloat16)}
    if case["op"] == "w4":
        return {"y": ((case["m"], case["n"]), torch.bfloat16)}
    return {}


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
        for name, (shape, dtype) in _results(case).items():
            state["in"][name], state["view"][name] = _buffer(dev, shape, dtype)
    return state


# ── one pass ────────────────────────────────────────────────────────────────


def _own_plan(K, case, i):
    K.kv_cache_plan(i["new_lens"], i["seq_lens"], i["block_table"], i["free_list"], i["free_count"], case["page"],
                    slots=i["slots"], positions=i["positions"], q_starts=i["q_starts"], context_lens=i["context_lens"],
                    granted=i["granted"], free_after=i["free_after"])


def _own_write(K, case, i):
    K.kv_cache_write(i["k"], i["v"], i["slots"], i["k_cache"], i["v_cache"], i["k_scale"], i["v_scale"])


def _own_attn(K, case, i):
    K.kv_cache_attention(i["q"], i["k_cache"], i["v_cache"], i["k_scale"], i["v_scale"], i["block_table"], i["context_lens"],
                         i["q_starts"], max_q_len=case["new"], max_context=case["ctx_hi"], o=i["o"])


def _own_w4(K, case, i):
    K.w4a16_linear(i["x"], i["qweight"], i["scale"], case["group"], zero_point=i.get("zero_point"), bias=i["bias"],
                   act=case["act"] or None, y=i["y"])


def _plain_plan(case, i):
    page, width = case["page"], case["width"]
    new, seq, table, stack, free = (i[n] for n in ("new_lens", "seq_lens", "block_table", "free_list", "free_count"))
    tokens = _step_tokens(case)
    add = new.clamp(min=0).long()
    end = add.cumsum(0)
    start = end - add
    held = (seq + page - 1) // page
    col = torch.arange(width, device=new.device)[None]
    # pages of ended requests, in order, on top of the stack
    back = torch.where(new < 0, held, 0).long()
    avail = free.long() + back.sum()
    ended = col < back[:, None]
    stack[(free + back.cumsum(0) - back)[:, None].add(col)[ended]] = table[ended]
    # pages from its top, in order; what does not fit is refused
    fits = (new > 0) & (seq + new <= page * width) & (end <= tokens)
    need = torch.where(fits, (seq + new + page - 1) // page - held, 0).long()
    upto = need.cumsum(0)
    given = fits & ((upto <= avail) | (need == 0))
    number = col - held[:, None]
    mine = given[:, None] & (number >= 0) & (number < need[:, None])
    top = (avail - 1 - (upto - need)[:, None] - number).clamp(0, stack.numel() - 1)
    table.copy_(torch.where(mine, stack[top], table))
    granted = torch.where(given, new, 0)
    context = torch.where(new < 0, 0, seq + granted)
    t = torch.arange(tokens, device=new.device)
    row = torch.searchsorted(end, t, right=True).clamp(max=case["b"] - 1)
    at = seq[row] + t - start[row]
    fine = (t < end[-1]) & given[row]
    slots = torch.where(fine, table[row, (at // page).clamp(0, width - 1)] * page + at % page, -1)
    starts = torch.cat([torch.zeros_like(end[:1]), end])
    left = avail - torch.where(given, need, 0).sum()
    return {"slots": slots.int(), "positions": torch.where(fine, at, -1).int(), "q_starts": starts.int(),
            "context_lens": context.int(), "granted": granted.int(), "free_after": left.int(), "block_table": table,
            "free_list": stack}


def _plain_store(x, slots, cache, scale, page, tokens_last):
    """Tokens x [T, H, D] into the pages of one cache (V's pages have the tokens last)."""
    slots = slots.long()
    at = torch.nonzero(slots >= 0)[:, 0]
    where, off = slots[at] // page, slots[at] % page
    x = x[at].float()
    most = torch.zeros_like(scale).index_reduce_(0, where, x.abs().amax(-1), "amax")
    first = torch.full((scale.shape[0],), page, device=x.device).index_reduce_(0, where, off, "amin")
    lead = torch.nonzero(off == first[where])[:, 0]
    pages = where[lead]
    old = torch.where((first[pages] > 0)[:, None], scale[pages], 0.0)
    now = torch.maximum(old, most[pages] / torch.full((1,), 127.0, device=x.device))
    ratio = torch.where(now > 0, old / now, 1.0)
    kept = torch.arange(page, device=x.device)[None] < first[pages][:, None]
    codes = cache[pages]
    kept = kept[:, None, None, :] if tokens_last else kept[:, None, :, None]
    again = (codes.float() * ratio[:, :, None, None]).round().to(torch.int8)
    cache[pages] = torch.where(kept, again, codes)
    scale[pages] = now
    mine = scale[where][..., None]
    fresh = torch.where(mine > 0, x / mine, 0.0).round().clamp(-127, 127).to(torch.int8)
    if tokens_last:
        cache[where, :, :, off] = fresh
    else:
        cache[where, :, off] = fresh


def _plain_write(case, i):
    page = case["page"]
    _plain_store(i["k"], i["slots"], i["k_cache"], i["k_scale"], page, False)
    _plain_store(i["v"], i["slots"], i["v_cache"], i["v_scale"], page, True)
    return {n: i[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _plain_attn(case, i):
    b, new, hq, hkv, d, page = (case[n] for n in ("b", "new", "hq", "hkv", "d", "page"))
    group, longest = hq // hkv, case["ctx_hi"]
    pages = i["block_table"][:, :_pages(longest, page)].clamp(min=0).long()
    k = i["k_cache"][pages].float() * i["k_scale"][pages][..., None, None]  # [b, w, h, page, d]
    v = i["v_cache"][pages].float() * i["v_scale"][pages][..., None, None]  # [b, w, h, d, page]
    k = k.transpose(1, 2).reshape(b * hkv, -1, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(b * hkv, -1, d)
    q = i["q"].float().reshape(b, new, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b * hkv, group * new, d)
    s = torch.bmm(q, k.mT) * (1 / math.sqrt(d))
    key = torch.arange(s.shape[-1], device=s.device)
    last = i["context_lens"][:, None] - new + torch.arange(new, device=s.device)  # [b, new]
    hidden = (key > last[..., None])[:, None, None]
    s = s.reshape(b, hkv, group, new, -1).masked_fill_(hidden, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.bmm(p.reshape(b * hkv, group * new, -1), v)
    return {"o": o.reshape(b, hkv, group, new, d).permute(0, 3, 1, 2, 4).reshape(b * new, hq, d).bfloat16()}


def _codes(qweight, k):
    """The inverse of _pack."""
    n = qweight.shape[0]
    words = qweight.view(torch.int32).reshape(n, -1, 4, 4, 1)
    shift = torch.tensor([4 * p for p in _NIBBLES], dtype=torch.int32, device=qweight.device)
    return (((words >> shift) & 15) - 8).transpose(2, 3).reshape(n, -1)[:, :k]


def _plain_w4(case, i):
    n, k, group = case["n"], case["k"], case["group"]
    w = _codes(i["qweight"], k).float()
    if "zero_point" in i:
        w = w - i["zero_point"].float().repeat_interleave(group, 1)[:, :k]
    w = w * i["scale"].repeat_interleave(group, 1)[:, :k]
    y = i["x"].float() @ w.T + i["bias"]
    if case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif case["act"] == "gelu":
        y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return {"y": y.bfloat16()}


_OUTPUTS = {"plan": ("slots", "positions", "q_starts", "context_lens", "granted", "free_after", "block_table", "free_list"),
            "write": ("k_cache", "v_cache", "k_scale", "v_scale"), "attn": ("o",), "w4": ("y",)}
_OWN = {"plan": _own_plan, "write": _own_write, "attn": _own_attn, "w4": _own_w4}
_PLAIN = {"plan": _plain_plan, "write": _plain_write, "attn": _plain_attn, "w4": _plain_w4}


def run(state):
    op = state["case"]["op"]
    if own:
        _OWN[op](state["kernels"], state["case"], state["in"])
        return {n: state["view"][n] for n in _OUTPUTS[op]}
    return _PLAIN[op](state["case"], state["in"])


# ── what a pass cannot do without ───────────────────────────────────────────


def work(case):
    op = case["op"]
    if op == "plan":
        seq, new = _plan_lengths(case)
        page = case["page"]
        tokens = _step_tokens(case)
        moved = sum(_pages(s, page) if n < 0 else _pages(s + n, page) - _pages(s, page) for s, n in zip(seq, new))
        # lengths in; starts, contexts and grants out; a slot and a position of each token; each moved page read and written
        return {"bytes": 4 * (2 * case["b"] + 3 * case["b"] + 2 * tokens + 2 * moved), "flops": 10 * (case["b"] + tokens)}
    if op == "write":
        before, new = _write_lengths(case)
        tokens, h, d, page = sum(new), case["h"], case["d"], case["page"]
        pages = sum(_pages(a + n, page) - a // page for a, n in zip(before, new))
        # bf16 in and int8 out for K and V, the slots, the scales of the pages
        return {"bytes": 2 * tokens * h * d * 3 + 4 * tokens + 2 * 8 * pages * h, "flops": 2 * tokens * h * d * 6}
    if op == "attn":
        b, new, hq, hkv, d, page = (case[n] for n in ("b", "new", "hq", "hkv", "d", "page"))
        ctx = _contexts(case)
        pairs = sum(new * c - new * (new - 1) // 2 for c in ctx)
        cache = sum(2 * hkv * (c * d + 4 * _pages(c, page)) + 4 * _pages(c, page) for c in ctx)
        return {"bytes": cache + 2 * 2 * b * new * hq * d, "flops": 4 * hq * pairs * d}
    m, n, k = case["m"], case["n"], case["k"]
    groups = _pages(k, case["group"])
    return {"bytes": n * k // 2 + (8 if case["zero"] else 4) * n * groups + 2 * m * k + 2 * m * n + 4 * n,
            "flops": 2 * m * n * k}


# ── the same in 64 bits ─────────────────────────────────────────────────────


def _exact_scales(x, slots, old, page):
    """Every page's scale after the tokens x: the largest magnitude of what it holds over 127, never less than before."""
    big = x.double().abs().amax(-1)
    scale = old.double().clone()
    fresh = {}
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            fresh.setdefault(s // page, []).append((t, s % page))
    pages = sorted(fresh)
    first = torch.tensor([min(o for _, o in fresh[p]) for p in pages], device=x.device)
    most = torch.stack([big[[t for t, _ in fresh[p]]].amax(0) for p in pages]) / 127
    held = torch.where(first[:, None] > 0, scale[pages], torch.zeros_like(most))
    scale[pages] = torch.maximum(held, most)
    return scale


def _exact_attn(case, t):
    new, group, d, page = case["new"], case["hq"] // case["hkv"], case["d"], case["page"]
    outs = []
    for b, ctx in enumerate(_contexts(case)):
        pages = t["block_table"][b, :_pages(ctx, page)].long()
        k = (t["k_cache"][pages].double() * t["k_scale"][pages].double()[..., None, None]).transpose(0, 1)
        v = (t["v_cache"][pages].double() * t["v_scale"][pages].double()[..., None, None]).permute(1, 0, 3, 2)
        k, v = (x.reshape(case["hkv"], -1, d)[:, :ctx].repeat_interleave(group, 0) for x in (k, v))
        s = t["q"][b * new:(b + 1) * new].double().transpose(0, 1) @ k.mT.contiguous() / math.sqrt(d)
        seen = torch.ones(new, ctx, dtype=torch.bool, device=s.device).tril(ctx - new)
        outs.append((torch.softmax(s.where(seen, -math.inf), -1) @ v).transpose(0, 1))
    return {"o": torch.cat(outs)}


def _exact_w4(case, t):
    n, k, group = case["n"], case["k"], case["group"]
    raw = t["qweight"].view(torch.uint8).reshape(n, -1, 4, 4, 4).to(torch.int64)  # [n, chunk, g, c, byte]
    both = torch.stack([raw & 15, raw >> 4], -1).flatten(-2)  # nibbles 0..7 of each word
    both = both[..., list(_NIBBLES)].double() - 8
    w = both.permute(0, 1, 3, 2, 4).reshape(n, -1)[:, :k]
    at = torch.arange(k, device=w.device) // group
    if "zero_point" in t:
        w = w - t["zero_point"].double()[:, at]
    y = t["x"].double() @ (w * t["scale"].double()[:, at]).T.contiguous() + t["bias"].double()
    if case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"] == "gelu":
        y = torch.nn.functional.gelu(y, approximate="tanh")
    return {"y": y}


def exact(case, seed):
    op = case["op"]
    t = _inputs(case, seed)
    if op == "plan":  # whole numbers only
        return None
    if op == "write":  # the codes are whole numbers
        return {"k_cache": None, "v_cache": None, "k_scale": _exact_scales(t["k"], t["slots"], t["k_scale"], case["page"]),
                "v_scale": _exact_scales(t["v"], t["slots"], t["v_scale"], case["page"])}
    return _exact_attn(case, t) if op == "attn" else _exact_w4(case, t)
