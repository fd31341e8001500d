"""Plain numpy forms of the 4-bit cache's operators and of the low-rank adapters in 64 bits, and the arithmetic bounds
that their GPU tests use (counted as in kv_cases.py: half a step of bf16 is 2^-8 of the value, of fp32 2^-24)."""
import math

import numpy as np

from kv_cases import H16, H32, NIBBLES


def rotate(x, positions, inv_freq, interleaved):
    """x [T, H, D] in 64 bits with its first 2 len(inv_freq) numbers rotated."""
    out = x.astype(np.float64)
    half = len(inv_freq)
    first = np.arange(half) * 2 if interleaved else np.arange(half)
    second = first + 1 if interleaved else first + half
    angle = positions.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = out[..., first].copy(), out[..., second].copy()
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    return out


def five_bits(x):
    """Five significant bits, to nearest even."""
    with np.errstate(invalid="ignore"):
        part, power = np.frexp(x.astype(np.float64))
        return np.ldexp(np.rint(part * 32), power - 5)


def quantize(x):
    """fp32 [..., D] -> (codes [..., D] in -8..7, scales [..., D / 64])."""
    x = np.asarray(x, np.float32)
    groups = x.reshape(*x.shape[:-1], -1, 64)
    with np.errstate(all="ignore"):
        high, low = groups.max(-1), groups.min(-1)
        most = np.where(high >= -low, high, low)
        fine = np.isfinite(groups).all(-1)
        scale = np.where(np.abs(most) < 2.0 ** -90, 0, five_bits(np.where(fine, most, 0) / -8)).astype(np.float32)
        q = np.where(scale[..., None] != 0, groups / scale[..., None], np.float32(0))
        codes = np.where(fine[..., None], np.clip(np.rint(q), -8, 7), 0).astype(np.int8)
    return codes.reshape(x.shape), np.where(fine, scale, np.float32(np.nan))


def k_place(d, n):
    """(word of a K row, its code) of number n of a head."""
    group, g, j, e = n // 64, n % 64 // 16, n % 16 // 8, n % 8
    return d // 64 * 2 * g + 2 * group + j, e


def put(words, at, code, value):
    """The code in nibbles of uint32 words[at]."""
    shift = np.uint32(4 * NIBBLES[code])
    words[at] = (words[at] & ~(np.uint32(15) << shift)) | ((value.astype(np.int64) + 8).astype(np.uint32) << shift)


def get(words, code):
    return ((words >> np.uint32(4 * NIBBLES[code])) & np.uint32(15)).astype(np.int8) - 8


def append(k, v, slots, cache):
    """Tokens k, v (fp32 [T, H, D]; k rotated) into copies of (k_cache, v_cache, k_scale, v_scale): int8 and fp32 arrays."""
    kc, vc, ks, vs = (a.copy() for a in cache)
    pages, heads, page, _ = kc.shape
    d = 2 * kc.shape[3]
    kw, vw = kc.view(np.uint32), vc.view(np.uint32)
    (kq, ksc), (vq, vsc) = quantize(k), quantize(v)
    for t, slot in enumerate(slots):
        if not 0 <= slot < pages * page:
            continue
        where, off = divmod(int(slot), page)
        for n in range(d):
            word, code = k_place(d, n)
            put(kw, (where, slice(None), off, word), code, kq[t, :, n])
        put(vw, (where, slice(None), off // 16, slice(None), off % 16 // 8), off % 8, vq[t])
        ks[where, :, off], vs[where, :, off] = ksc[t], vsc[t]
    return kc, vc, ks, vs


def codes_of(kc, vc):
    """The caches' codes [pages, heads, page_size, D] of both."""
    pages, heads, page, row = kc.shape
    d = 2 * row
    kw, vw = kc.view(np.uint32), vc.view(np.uint32)
    kq, vq = (np.empty((pages, heads, page, d), np.int8) for _ in range(2))
    for n in range(d):
        word, code = k_place(d, n)
        kq[..., n] = get(kw[..., word], code)
    for t in range(page):
        vq[:, :, t] = get(vw[:, :, t // 16, :, t % 16 // 8], t % 8)
    return kq, vq


def attention(q, kc, vc, ks, vs, table, ctx, starts, scale, causal):
    """(o, lse, bound on o's error, bound on lse's) in 64 bits; q fp32 [T, Hq, D].  Rows of no sequence hold NaN.

    The bound: a group's scores are an fp32 sum of 64 products of q and 24 + code (16 to 31) and of 24 times q's sum, which
    the scale multiplies; where q is held as the sum of two fp8 numbers (its largest between 128 and 256, the second's last
    bit 2^-9), it is off by 2^-10, so by 2^-17 of the largest; the exponents are off by as much and a few roundings; a probability times its V scale is rounded
    to bf16 (of the sum of p |v|), multiplies 24 + code in an fp32 sum over the tokens, less 24 times its own sum; the
    output is rounded to bf16.  A code times its scale is a bf16 number (scales of five bits): kernels may multiply that."""
    t, hq, d = q.shape
    pages, hkv, page, _ = kc.shape
    group, width = hq // hkv, table.shape[1]
    o, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    lse, ltol = np.full((t, hq), np.nan), np.full((t, hq), np.nan)
    kq, vq = codes_of(kc, vc)
    for b in range(len(ctx)):
        first, end = int(starts[b]), int(starts[b + 1])
        n_ctx = min(max(int(ctx[b]), 0), width * page)
        tok = np.arange(n_ctx)
        where = table[b, tok // page].astype(np.int64) if n_ctx else np.zeros(0, np.int64)
        there = (where >= 0) & (where < pages)
        where, off = where[there], (tok % page)[there]
        for kh in range(hkv):
            steps = [np.repeat(s[where, kh, off].astype(np.float64), 64, axis=-1) for s in (ks, vs)]
            k_all, v_all = kq[where, kh, off] * steps[0], vq[where, kh, off] * steps[1]
            for i in range(end - first):
                seen = min(max(n_ctx - (end - first) + 1 + i, 0), n_ctx) if causal else n_ctx
                n = int((tok[there] < seen).sum())  # tokens are in order
                rows = first + i, slice(kh * group, (kh + 1) * group)
                if n == 0:
                    o[rows], tol[rows], lse[rows], ltol[rows] = 0, 0, -np.inf, 0
                    continue
                k, v = k_all[:n], v_all[:n]
                qq = q[rows].astype(np.float64)
                s = qq @ k.T * scale
                m = s.max(-1, keepdims=True)
                p = np.exp(s - m)
                den = p.sum(-1, keepdims=True)
                o[rows] = p @ v / den
                lse[rows] = (m + np.log(den))[:, 0]
                # 2.4375 = 39 / 16: the largest operand, with that of the sum beside it
                made = (np.abs(qq) @ (39 * np.abs(steps[0][:n]) + np.abs(k)).T).max(-1, keepdims=True) * abs(scale)
                made = made * (64 + 16) * H32 + np.abs(qq).max(-1, keepdims=True) * np.abs(k).sum(-1).max() * 2.0 ** -17 * abs(scale)
                off_s = made + 8 * H32 * (np.abs(s).max(-1, keepdims=True) + 16)
                mag, held = p @ np.abs(v) / den, p @ (39 * np.abs(steps[1][:n])) / den
                tol[rows] = (mag * (H16 + 2 * off_s) + (mag + held) * (n + 64) * 2 * H32) * 1.01 + np.abs(o[rows]) * H16 * 1.01 + 1e-30
                # (the rounded probabilities also multiply the offset, whose sum is taken off exactly: the same rounded ones)
                ltol[rows] = (2 * off_s + (n + 64) * H32 + 8 * H32 * np.abs(lse[rows])[:, None])[:, 0]
    return o, lse, tol, ltol


def adapter(x, a, b, ids, scale, y):
    """(out in 64 bits, bound): fp32 sums of K and of rank products, the first one's result in two bf16 parts (2^-17)."""
    out, tol = y.astype(np.float64), np.zeros(y.shape)
    for m, i in enumerate(ids):
        if 0 <= i < len(a):
            s = 1.0 if scale is None else float(scale[i])
            aa, bb, xx = a[i].astype(np.float64), b[i].astype(np.float64), x[m].astype(np.float64)
            h = s * (aa @ xx)
            out[m] += bb @ h
            made = abs(s) * (np.abs(aa) @ np.abs(xx)) * (x.shape[1] + 16) * H32 + np.abs(h) * 2.0 ** -16
            tol[m] = np.abs(bb) @ made + (np.abs(bb) @ np.abs(h)) * (2 * a.shape[1] + 16) * H32
    return out, tol * 1.01 + np.abs(out) * (H16 + 2 * H32) * 1.01 + np.abs(y) * 2 * H32 + 1e-30
