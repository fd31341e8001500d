"""Plain numpy forms of the 8-bit cache's operators and of the 4-bit linear
layer, and the arithmetic bounds that their GPU tests use.

Bounds count roundings: half a step of a type is ``2^-8`` (bf16) or ``2^-24``
(fp32) of the value, and an fp32 sum of n terms is off by at most n such
halves of the sum of magnitudes, whatever its order."""
import math

import numpy as np

H16, H32 = 2.0 ** -8, 2.0 ** -24


def pages_of(n, page):
    return -(-n // page)


def plan(new, seq, table, free_list, free_count, page, tokens):
    """The plan request by request.  Returns the outputs and the new table and stack."""
    table, stack = table.copy(), free_list.copy()
    width, held = table.shape[1], int(free_count)
    for b, n in enumerate(new):
        if n < 0:
            for i in range(pages_of(min(max(int(seq[b]), 0), width * page), page)):
                stack[held] = table[b, i]
                held += 1
    starts, slots, positions = [0], np.full(tokens, -1, np.int32), np.full(tokens, -1, np.int32)
    granted, context = np.zeros(len(new), np.int32), np.array(seq, np.int32)
    need_all, avail = 0, held
    for b, n in enumerate(int(x) for x in new):
        s = int(seq[b])
        first, end = starts[-1], starts[-1] + max(n, 0)
        starts.append(min(end, tokens))
        if n < 0:
            context[b] = 0
        if n <= 0 or s < 0 or s + n > width * page or end > tokens:
            continue
        need = pages_of(s + n, page) - pages_of(s, page)
        need_all += need
        if need and need_all > avail:
            continue
        for i in range(need):
            held -= 1
            table[b, pages_of(s, page) + i] = stack[held]
        for i in range(n):
            positions[first + i] = s + i
            slots[first + i] = table[b, (s + i) // page] * page + (s + i) % page
        granted[b], context[b] = n, s + n
    return {"slots": slots, "positions": positions, "q_starts": np.array(starts, np.int32), "context_lens": context,
            "granted": granted, "free_after": np.array([held], np.int32)}, table, stack


def write(x, slots, cache, scale, page, tokens_last):
    """Tokens x fp32 [T, H, D] into the pages of one cache, in fp32 steps (as the kernel's); new codes and scales."""
    cache, scale = cache.copy(), scale.copy()
    view = cache.transpose(0, 1, 3, 2) if tokens_last else cache  # [pages, heads, page, d]
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= cache.shape[0] * page:
            t += 1
            continue
        where, old = divmod(int(slots[t]), page)
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and old + n < page:
            n += 1
        for h in range(cache.shape[1]):
            new = x[t:t + n, h].astype(np.float32)
            before = scale[where, h] if old else np.float32(0)
            with np.errstate(all="ignore"):
                s = np.maximum(before, np.float32(np.abs(new).max() if not np.isnan(new).any() else np.nan) / np.float32(127))
                fine = s > 0 and np.isfinite(s)
                ratio = np.float32(before) / s if fine else np.float32(0)
                kept = view[where, h, :old].astype(np.float32)
                if not s == before:
                    view[where, h, :old] = np.rint(kept * ratio).astype(np.int8) if fine else 0
                view[where, h, old:old + n] = np.rint(np.clip(new / s, -127, 127)).astype(np.int8) if fine else 0
            scale[where, h] = s
        t += n
    return cache, scale


def attention(q, kc, vc, ks, vs, table, ctx, starts, scale, causal):
    """(o, lse, bound on o's error, bound on lse's) in 64 bits; q fp32 [T, Hq, D].  Rows of no sequence hold NaN.

    The bound: the scores are fp32 sums of D products, and their fp32 exponents are off by as much; a probability
    times its V scale is rounded to bf16 (of the sum of p |v|), and so is the output."""
    t, hq, d = q.shape
    pages, hkv, page, _ = kc.shape
    group, width = hq // hkv, table.shape[1]
    o, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    lse, ltol = np.full((t, hq), np.nan), np.full((t, hq), np.nan)
    for b in range(len(ctx)):
        first, end = int(starts[b]), int(starts[b + 1])
        n_ctx = min(max(int(ctx[b]), 0), width * page)
        tok = np.arange(n_ctx)
        where = table[b, tok // page].astype(np.int64) if n_ctx else np.zeros(0, np.int64)
        there = (where >= 0) & (where < pages)
        where, off = where[there], (tok % page)[there]
        for i in range(end - first):
            seen = min(max(n_ctx - (end - first) + 1 + i, 0), n_ctx) if causal else n_ctx
            use = tok[there] < seen
            w, f = where[use], off[use]
            for h in range(hq):
                kh = h // group
                if not len(w):
                    o[first + i, h], tol[first + i, h], lse[first + i, h], ltol[first + i, h] = 0, 0, -np.inf, 0
                    continue
                k = kc[w, kh, f].astype(np.float64) * ks[w, kh].astype(np.float64)[:, None]
                v = vc[w, kh, :, f].astype(np.float64) * vs[w, kh].astype(np.float64)[:, None]
                qq = q[first + i, h].astype(np.float64)
                s = k @ qq * scale
                m = s.max()
                p = np.exp(s - m)
                den = p.sum()
                o[first + i, h] = p @ v / den
                lse[first + i, h] = m + math.log(den)
                off_s = ((d + 8) * H32 * (np.abs(k) @ np.abs(qq)).max() * abs(scale) + 8 * H32 * (np.abs(s).max() + 16))
                mag = p @ np.abs(v) / den
                tol[first + i, h] = mag * (H16 + 2 * off_s + 4 * (len(w) + 64) * H32) * 1.01 + np.abs(o[first + i, h]) * H16 * 1.01 + 1e-30
                ltol[first + i, h] = 2 * off_s + (len(w) + 64) * H32 + 8 * H32 * abs(lse[first + i, h])
    return o, lse, tol, ltol


NIBBLES = (0, 4, 1, 5, 2, 6, 3, 7)


def pack(codes):
    """[N, K] codes in -8..7 -> packed bytes, word by word as the header says."""
    n, k = codes.shape
    out = np.zeros((n, pages_of(k, 128) * 16), np.uint32)
    for chunk in range(pages_of(k, 128)):
        for g in range(4):
            for c in range(4):
                for j in range(8):
                    at = 128 * chunk + 32 * c + 8 * g + j
                    code = codes[:, at].astype(np.int64) + 8 if at < k else np.full(n, 8)
                    out[:, 16 * chunk + 4 * g + c] |= (code << (4 * NIBBLES[j])).astype(np.uint32)
    return out.view(np.int8)


def act64(y, act):
    if act == "relu":
        return np.maximum(y, 0)
    if act == "silu":
        return y / (1 + np.exp(-y))
    if act == "gelu":
        return y / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def w4_linear(x, codes, scale, zero, bias, group, act, copy):
    """(y in 64 bits, bound).  The streaming kernel sums x (16 + code + 8) / 16 over a group in fp32 (128 products deep
    at most, then the chunks and the waves), takes the offset off and scales; the copy rounds each weight to bf16."""
    k = x.shape[1]
    at = np.arange(k) // group
    x = x.astype(np.float64)
    s = scale.astype(np.float64)[:, at]
    z = zero.astype(np.float64)[:, at] if zero is not None else np.zeros_like(s)
    w = (codes.astype(np.float64) - z) * s
    y = x @ w.T + (bias.astype(np.float64) if bias is not None else 0)
    if copy:
        off = np.abs(x) @ np.abs(w).T * (H16 + (k + 64) * 2 * H32)
    else:
        off = np.abs(x) @ (16 * s * (3.5 + np.abs(z) / 16)).T * (128 + k / 128 + 24) * 2 * H32
    # the activations' slopes are at most 1.13
    return act64(y, act), 1.13 * off + np.abs(act64(y, act)) * (H16 + 2.0 ** -18) + 2.0 ** -18 * np.abs(y) + 1e-30
