"""The 4-bit paged K/V cache on the GPU: appends, attention, and a step of them with plan, 4-bit layers and adapters,
against the plain forms of kv4_cases.py."""
import contextlib
import math

import numpy as np
import pytest

import kv4_cases as kv4
import kv_cases as kv
from gpu_util import stream_workspace
from kv_cases import H16, H32
from teenygrad_amd import kernels as K
from teenygrad_amd._lib import check, lib
from teenygrad_amd.dtypes import bf16, from_bf16, to_bf16
from teenygrad_amd.runtime import NULL_STREAM, Stream
from test_gpu_kv_cache import ATTN, ints, make_table

pytestmark = pytest.mark.gpu


def rounded(a):
    return from_bf16(to_bf16(np.asarray(a, np.float32)))


def up(dev, a):
    return dev.upload(to_bf16(np.asarray(a, np.float32)), bf16)


def random_cache(rng, pages, heads, page, d, low=0.005, high=0.03):
    def scales():
        s = rng.uniform(low, high, (pages, heads, page, d // 64)) * rng.choice([-1, 1], (pages, heads, page, d // 64))
        return kv4.five_bits(s).astype(np.float32)
    return [rng.integers(-128, 128, (pages, heads, page, d // 2)).astype(np.int8),
            rng.integers(-128, 128, (pages, heads, page // 16, d, 8)).astype(np.int8), scales(), scales()]


def up_cache(dev, cache):
    return [dev.upload(a) if a.dtype == np.int8 else up(dev, a) for a in cache]


def down_cache(bufs):
    return [b.to_host() if b.dtype.name == "i8" else from_bf16(b.to_host()) for b in bufs]


def freqs(rot, base=10000.0):
    return (base ** (-np.arange(rot // 2) * 2.0 / max(rot, 1))).astype(np.float32)


# ── append ──────────────────────────────────────────────────────────────────


def append_case(rng, before, new, hq, hkv, d, page, pad=0, far=0):
    """Tokens of sequences with `before` cached ones; positions further along by `far`; pad rows of no token between them."""
    after = [a + n for a, n in zip(before, new)]
    table, pages, _ = make_table(rng, after, page, max(1, max(kv.pages_of(n, page) for n in after)), extra=2)
    slots, pos = [], []
    for b, (a, n) in enumerate(zip(before, new)):
        slots += [table[b, (a + i) // page] * page + (a + i) % page for i in range(n)] + [-1] * pad
        pos += [a + i + far for i in range(n)] + [-1] * pad
    t = len(slots)
    wide = 1 + 4 * (rng.random((1, 1, d)) < 0.05)
    x = {"q": rounded(rng.standard_normal((t, hq, d))), "k": rounded(rng.standard_normal((t, hkv, d)) * wide),
         "v": rounded(rng.standard_normal((t, hkv, d)) * (1 + 3 * rng.random((t, hkv, 1))))}
    return x, np.array(slots, np.int32), np.array(pos, np.int32), random_cache(rng, pages, hkv, page, d)


def check_append(dev, x, slots, pos, cache, freq, inter=False, in_place=False):
    bufs, q = up_cache(dev, cache), up(dev, x["q"])
    out = q if in_place else up(dev, np.full(x["q"].shape, 123.0))
    K.kv4_cache_append(q, up(dev, x["k"]), up(dev, x["v"]), ints(dev, pos), ints(dev, slots), dev.upload(freq) if len(freq) else None, *bufs,
                       interleaved=inter, q_out=out)
    got = down_cache(bufs)
    k = kv4.rotate(x["k"], pos, freq, inter).astype(np.float32)
    want = kv4.append(k, x["v"], np.where(pos < 0, -1, slots), cache)
    for g, r, n in zip(got, want, ("k codes", "v codes", "k scales", "v scales")):
        np.testing.assert_array_equal(g, r, err_msg=n)
    ref = kv4.rotate(x["q"], pos, freq, inter)
    o, live = from_bf16(out.to_host()), pos >= 0
    assert (o[~live] == (x["q"][~live] if in_place else 123.0)).all(), "rows of no token were written"
    # two fp32 products of fp32 cosines and sines, added, and the rounding to bf16
    size = np.abs(kv4.rotate(np.abs(x["q"]), np.zeros_like(pos), freq, inter)).max(-1, keepdims=True)
    assert (np.abs(o[live] - ref[live]) <= np.abs(ref[live]) * H16 * 1.01 + 8 * H32 * size[live]).all()
    return got


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("d,rot,inter", [(128, 128, False), (64, 64, False), (128, 32, True), (64, 48, False), (128, 128, True)])
@pytest.mark.parametrize("before,new,hq,hkv", [
    ([0], [1], 1, 1), ([15, 16, 17, 0, 127, 900], [1] * 6, 8, 2), ([3, 100], [13, 200], 3, 3), ([0, 1, 31, 63, 70], [129, 5, 1, 66, 0], 4, 1),
    (list(range(40, 110)), [1] * 70, 2, 2)])
def test_append(dev, page, d, rot, inter, before, new, hq, hkv):
    rng = np.random.default_rng(sum(before) + sum(new) + page + d + rot)
    check_append(dev, *append_case(rng, before, new, hq, hkv, d, page), freqs(rot), inter)


def test_append_many_tokens(dev):
    """More tokens than the rows of one form: 600 tokens in pieces of odd lengths, two of them padded behind."""
    rng = np.random.default_rng(1)
    check_append(dev, *append_case(rng, [5, 0, 77], [301, 18, 333], 5, 2, 64, 32, pad=3), freqs(64))
    check_append(dev, *append_case(rng, [9, 0], [1100, 7], 4, 1, 128, 16, pad=1), freqs(128))


def test_append_without_rotation(dev):
    rng = np.random.default_rng(2)
    for d in (64, 128):
        check_append(dev, *append_case(rng, [5, 0], [30, 3], 2, 2, d, 16, pad=2), freqs(0))


@pytest.mark.parametrize("far", [1 << 17, (1 << 24) + 1, (1 << 31) - 200])
def test_append_far_positions(dev, far):
    """Angles of far positions: in fp32 they would be off by many turns' parts."""
    rng = np.random.default_rng(3)
    check_append(dev, *append_case(rng, [0, 3], [50, 60], 4, 2, 128, 16, far=far), freqs(128))


@pytest.mark.parametrize("inter", [False, True])
def test_append_in_place(dev, inter):
    rng = np.random.default_rng(4)
    check_append(dev, *append_case(rng, [5, 0, 40], [70, 1, 3], 6, 2, 128, 16, pad=2), freqs(64), inter, in_place=True)


def test_append_without_queries(dev):
    rng = np.random.default_rng(5)
    x, slots, pos, cache = append_case(rng, [5, 0], [30, 3], 1, 2, 64, 16)
    bufs, f = up_cache(dev, cache), freqs(64)
    assert K.kv4_cache_append(None, up(dev, x["k"]), up(dev, x["v"]), ints(dev, pos), ints(dev, slots), dev.upload(f), *bufs) is None
    for g, r in zip(down_cache(bufs), kv4.append(kv4.rotate(x["k"], pos, f, False).astype(np.float32), x["v"], slots, cache)):
        np.testing.assert_array_equal(g, r)


def test_append_skips_and_bounds(dev):
    """Padding among the rows, slots past the cache, rows of queries alone."""
    rng = np.random.default_rng(6)
    x, slots, pos, cache = append_case(rng, [4, 20, 0], [9, 9, 40], 2, 2, 64, 16)
    slots, pos = slots.copy(), pos.copy()
    slots[3:9] = -1                     # a run breaks off; queries are rotated all the same
    limit = cache[0].shape[0] * 16
    slots[12:15] = [limit, limit + 1, 2 ** 31 - 1]
    slots[15:18] = -5
    pos[40:] = -1                       # no token at all, whatever the slot says
    pos[39] = -2 ** 31
    check_append(dev, x, slots, pos, cache, freqs(64))


@pytest.mark.parametrize("d", [64, 128])
def test_append_special_values(dev, d):
    """Zeros, infinities, NaN, ties between signs, the largest and the smallest numbers."""
    rng = np.random.default_rng(d)
    x, slots, pos, cache = append_case(rng, [5, 0, 18], [12, 3, 40], 2, 2, d, 16)
    for n in "kv":
        a = x[n]
        a[0:2] = 0
        a[2, 0, 7], a[3, 0, 60], a[4, 1, 9] = np.inf, -np.inf, np.nan
        a[5] = rounded(2e-38)
        a[6] = rounded(2.0 ** -90)
        a[7] = -rounded(2.0 ** -91)
        a[8] = rounded(np.where(np.arange(d) % 2, 3.0, -3.0))
        a[9] = rounded(3.0e38 * np.sign(rng.standard_normal((2, d))))
        a[10] = -0.0
        a[12:14] = rounded(np.rint(rng.uniform(-8, 8, (2, 2, d)) * 2) / 2)  # quotients at a half
        a[12:14, :, ::64] = -8
    x["q"][0, 0, 3], x["q"][1, 0, 5] = np.inf, np.nan
    for freq in (freqs(0), freqs(d)):
        with np.errstate(all="ignore"):
            bufs, q = up_cache(dev, cache), up(dev, x["q"])
            o = K.kv4_cache_append(q, up(dev, x["k"]), up(dev, x["v"]), ints(dev, pos), ints(dev, slots),
                                   dev.upload(freq) if len(freq) else None, *bufs)
            k = kv4.rotate(x["k"], pos, freq, False).astype(np.float32)
            for g, r, n in zip(down_cache(bufs), kv4.append(k, x["v"], slots, cache), ("k codes", "v codes", "k scales", "v scales")):
                np.testing.assert_array_equal(g, r, err_msg=n)
        o, ref = from_bf16(o.to_host()), kv4.rotate(x["q"], pos, freq, False)
        np.testing.assert_array_equal(np.isfinite(o), np.isfinite(ref))


@pytest.mark.parametrize("d", [64, 128])
def test_append_over_all_exponents(dev, d):
    """Groups of every magnitude that bf16 has, each significand for the largest number, and quotients at a half."""
    rng = np.random.default_rng(d)
    exps = np.repeat(np.arange(-100, 128), 7)
    x, slots, pos, cache = append_case(rng, [0], [len(exps)], 1, 1, d, 64)
    for n in "kv":
        m = rng.uniform(-1, 1, x[n].shape)
        m[:, 0, ::64] = -rng.integers(128, 256, (len(exps), d // 64)) / 256
        m[::7] = rng.integers(-16, 16, m[::7].shape) / 32  # half steps of the scale 1 / 16
        m[::7, 0, ::64] = -0.5
        x[n] = rounded(np.ldexp(m, exps[:, None, None]))
    check_append(dev, x, slots, pos, cache, freqs(0))


def test_append_rounds_any_quotient(dev):
    """Rotated keys have all of fp32's bits: codes are those of the fp32 quotient, a million of them."""
    rng = np.random.default_rng(8)
    check_append(dev, *append_case(rng, [0], [512], 1, 16, 128, 128), freqs(128))


def test_append_strides(dev):
    """q, k and v as parts of one projection's rows, over the C entry point; the rest of the rows stays."""
    rng = np.random.default_rng(9)
    hq, hkv, d, page = 4, 2, 64, 16
    x, slots, pos, cache = append_case(rng, [3, 0], [20, 5], hq, hkv, d, page)
    t, row = len(slots), (hq + 2 * hkv) * d + 8
    both = np.full((t, row), 9.0, np.float32)
    at = {"q": 0, "k": hq * d, "v": (hq + hkv) * d}
    for n, o in at.items():
        both[:, o:o + x[n][0].size] = x[n].reshape(t, -1)
    qkv, bufs, out = up(dev, both), up_cache(dev, cache), dev.buffer(bf16, (t, hq, d))
    p, s, f = ints(dev, pos), ints(dev, slots), dev.upload(freqs(d))
    check(lib.teeny_kv4_cache_append(*[qkv.ptr + 2 * at[n] for n in "qkv"], p.ptr, s.ptr, f.ptr, out.ptr, *[b.ptr for b in bufs], t, hq, hkv, d, d,
                                     cache[0].shape[0], page, row, row, row, 0, None))
    want = kv4.append(kv4.rotate(x["k"], pos, freqs(d), False).astype(np.float32), x["v"], slots, cache)
    for g, r in zip(down_cache(bufs), want):
        np.testing.assert_array_equal(g, r)
    ref = kv4.rotate(x["q"], pos, freqs(d), False)
    assert (np.abs(from_bf16(out.to_host()) - ref) <= np.abs(ref) * H16 * 1.01 + 8 * H32 * np.abs(x["q"]).max()).all()
    np.testing.assert_array_equal(qkv.to_host(), to_bf16(both))


def test_append_over_refused_tokens(dev):
    """Drafts are appended, some are refused, and others take their slots: every other token keeps its codes."""
    rng = np.random.default_rng(10)
    x, _, _, cache = append_case(rng, [0], [32], 2, 2, 64, 16)
    slots = np.arange(16, 48, dtype=np.int32)
    cache = check_append(dev, x, slots, slots, [np.concatenate([a, a]) for a in cache], freqs(64))
    for first, n in ((21, 3), (30, 4), (47, 1), (16, 16)):
        part = {m: a[:n] * 2 for m, a in x.items()}
        cache = check_append(dev, part, np.arange(first, first + n, dtype=np.int32), np.arange(n, dtype=np.int32), cache, freqs(64))


# ── attention ───────────────────────────────────────────────────────────────


def attn_case(rng, ctx, new, hq, hkv, d, page, extra=2, low=0.02, high=0.12):
    table, pages, _ = make_table(rng, ctx, page, max(1, max(kv.pages_of(n, page) for n in ctx)) + 1, extra=extra)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = rounded(rng.standard_normal((int(starts[-1]), hq, d)))
    return dict(q=q, cache=random_cache(rng, pages, hkv, page, d, low, high), table=table, ctx=np.array(ctx, np.int32), starts=starts)


def run_attn(dev, c, scale=None, causal=True, hint=None, pad=0, stream=None, starts=True):
    t, hq, d = c["q"].shape
    q = np.concatenate([c["q"], np.ones((pad, hq, d), np.float32)])
    o = up(dev, np.full(q.shape, 123.0))
    lse = dev.upload(np.full((t + pad, hq), 55.0, np.float32))
    K.kv4_cache_attention(up(dev, q), *up_cache(dev, c["cache"]), dev.upload(c["table"]), ints(dev, c["ctx"]),
                          ints(dev, c["starts"]) if starts else None, *(hint or (None, None)), softmax_scale=scale, causal=causal, o=o, lse=lse,
                          stream=stream)
    if stream is not None:
        stream.synchronize()
    return from_bf16(o.to_host()), lse.to_host()


def oracle(c, scale=None, causal=True):
    d = c["q"].shape[2]
    return kv4.attention(c["q"], *c["cache"], c["table"], c["ctx"], c["starts"], 1 / math.sqrt(d) if scale is None else scale, causal)


def check_attn(c, got, scale=None, causal=True, ref=None):
    t = c["q"].shape[0]
    o, lse, tol, ltol = oracle(c, scale, causal) if ref is None else ref
    go, gl = got[0].astype(np.float64), got[1].astype(np.float64)
    assert (go[t:] == 123.0).all() and (gl[t:] == 55.0).all(), "rows past the last sequence were written"
    np.testing.assert_array_equal(np.isneginf(gl[:t]), np.isneginf(lse))
    err = np.abs(go[:t] - o)
    assert (err <= tol).all(), f"o: worst {np.nanmax(err - tol)} over the bound, error {np.nanmax(err)}"
    fin = np.isfinite(lse)
    assert (np.abs(gl[:t][fin] - lse[fin]) <= ltol[fin]).all(), np.max(np.abs(gl[:t][fin] - lse[fin]) - ltol[fin])


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ctx,new,hq,hkv", ATTN)
def test_attention(dev, ctx, new, hq, hkv, d, page):
    rng = np.random.default_rng(sum(ctx) + 7 * sum(new) + hq + d + page)
    c = attn_case(rng, ctx, new, hq, hkv, d, page)
    check_attn(c, run_attn(dev, c, hint=(max(new), max(ctx)), pad=3))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ctx,new,hq,hkv", [([2100, 5, 900], [1, 1, 1], 8, 2), ([1500, 1030], [9, 2], 6, 2), ([1300, 40], [70, 40], 4, 2)])
def test_attention_splits(dev, ctx, new, hq, hkv, causal):
    """With a workspace the tokens are shared out; hints that are wrong change nothing but the speed."""
    rng = np.random.default_rng(sum(ctx))
    c = attn_case(rng, ctx, new, hq, hkv, 128, 16)
    t, ref = int(c["starts"][-1]), oracle(c, causal=causal)
    for hint in ((max(new), max(ctx)), (1, 1100), (100, 1 << 20), (max(new), 1), None):
        most = hint or (t, c["table"].shape[1] * 16)
        size = max(K.kv4_cache_attention_workspace_size(t, len(ctx), hq, hkv, 128, most[0], m) for m in (most[1], max(ctx) + 48))
        with stream_workspace(dev, size):
            check_attn(c, run_attn(dev, c, causal=causal, hint=hint), ref=ref)
        with stream_workspace(dev, 1024):  # too small: none is used
            check_attn(c, run_attn(dev, c, causal=causal, hint=hint), ref=ref)


@pytest.mark.parametrize("ctx,new", [(2000, 1), (2000, 7), (4500, 40)])
def test_attention_workspace_size(dev, ctx, new):
    """The size that is asked for is enough: the results are those of any larger workspace."""
    c = attn_case(np.random.default_rng(ctx + new), [ctx], [new], 8, 2, 64, 16)
    c["table"] = c["table"][:, :kv.pages_of(ctx, 16)]
    size = K.kv4_cache_attention_workspace_size(new, 1, 8, 2, 64, new, 1 << 15)
    assert 0 < size < 32 << 20
    got = []
    for n, hint in ((K.kv4_cache_attention_workspace_size(new, 1, 8, 2, 64, new, ctx), ctx), (size, 1 << 15), (64 << 20, 1 << 15)):
        ws = dev.upload(np.full(n, 77, np.int8))
        NULL_STREAM.set_workspace(ws)
        try:
            got.append(run_attn(dev, c, hint=(new, hint)))
        finally:
            NULL_STREAM.set_workspace(None)
        assert (ws.to_host() != 77).any()  # it was used
    for o, lse in got[1:]:
        np.testing.assert_array_equal(o, got[0][0])
        np.testing.assert_array_equal(lse, got[0][1])
    check_attn(c, got[0])


@pytest.mark.parametrize("ctx,new,hq,hkv", [([4500], 1, 8, 2), ([3000, 700], 7, 8, 2), ([5000, 60], 40, 4, 2)])
@pytest.mark.parametrize("part", [0.9, 0.4])
def test_attention_in_part_of_its_workspace(dev, ctx, new, hq, hkv, part):
    """A workspace that does not hold all the parts that were planned holds fewer; nothing outside of it is written."""
    c = attn_case(np.random.default_rng(ctx[0]), ctx, [new] * len(ctx), hq, hkv, 64, 16)
    c["table"] = c["table"][:, :kv.pages_of(ctx[0], 16)]
    size = K.kv4_cache_attention_workspace_size(new * len(ctx), len(ctx), hq, hkv, 64, new, ctx[0])
    assert size > 0
    small = int(size * part) // 256 * 256
    ws = dev.upload(np.full(size, 77, np.int8))
    check(lib.teeny_hip_stream_set_workspace(None, ws.ptr, small))
    try:
        got = run_attn(dev, c, hint=(new, ctx[0]))
    finally:
        NULL_STREAM.set_workspace(None)
    assert (ws.to_host()[small:] == 77).all()
    check_attn(c, got)


@pytest.mark.parametrize("new,batch", [(1, 150), (5, 150), (20, 150), (1, 300), (20, 300), (1, 4500)])
def test_attention_of_many_sequences(dev, new, batch):
    """More sequences than lanes: one, a few and many query rows, some sequences without any, with and without splits."""
    rng = np.random.default_rng(70 + new)
    lens = rng.integers(0, 200 if batch < 1000 else 30, batch)
    lens[[3, 77, batch - 1]] = 1500, 0, 2000
    c = attn_case(rng, [int(n) for n in lens], [int(n) for n in rng.integers(new == 1, new + 1, batch)], 8, 2, 64, 16)
    t, hint, ref = int(c["starts"][-1]), (new, 2000), oracle(c)
    check_attn(c, run_attn(dev, c, hint=hint, pad=2), ref=ref)
    with stream_workspace(dev, K.kv4_cache_attention_workspace_size(t + 2, batch, 8, 2, 64, *hint)):
        check_attn(c, run_attn(dev, c, hint=hint, pad=2), ref=ref)


@pytest.mark.parametrize("d,batch,hkv,new,causal", [(64, 40, 16, 1, True), (128, 40, 16, 1, True), (64, 64, 9, 3, False), (64, 24, 16, 20, True),
                                                    (128, 24, 16, 20, False)])
def test_attention_of_many_parts(dev, d, batch, hkv, new, causal):
    """Up to 64 sequences with more parts than the device takes at once, which go out longest first: empty contexts, sequences
    without queries, contexts past all splits and rows past the hinted ones among them."""
    rng = np.random.default_rng(batch + hkv + new)
    ctx, lens = rng.integers(0, 900, batch), rng.integers(0, new + 1, batch)
    ctx[[0, 5, 17, batch - 1]], lens[[0, 3, 5, batch - 1]] = [0, 5000, 1290, 2100], [new, 0, new, new]
    if new == 1:
        lens[:] = 1
    c = attn_case(rng, [int(n) for n in ctx], [int(n) for n in lens], 2 * hkv, hkv, d, 16)
    t, ref = int(c["starts"][-1]), oracle(c, causal=causal)
    block = 32 if new > 8 else 16
    walk = min(t * 2 // block + batch, batch * -(-2 * new // block))
    assert walk * hkv > 2 * dev.info()["compute_units"], "few parts go out in the sequences' order"
    for hint in ((new, 5000), (new, 2100), (1, 2100), (new, 1)):
        check_attn(c, run_attn(dev, c, causal=causal, hint=hint, pad=2), ref=ref)
        size = K.kv4_cache_attention_workspace_size(t + 2, batch, 2 * hkv, hkv, d, *hint)
        assert (size > 0) == (hint[1] > 1)
        with stream_workspace(dev, max(size, 4096)):
            check_attn(c, run_attn(dev, c, causal=causal, hint=hint, pad=2), ref=ref)


def test_attention_of_many_sequences_in_tiles(dev):
    """5000 sequences of 32 heads of their own under a hint of many queries: near the limit of rows."""
    rng = np.random.default_rng(71)
    batch, heads = 5000, 32
    c = attn_case(rng, [int(n) for n in rng.integers(0, 40, batch)], [1] * batch, heads, heads, 64, 16)
    o, lse = run_attn(dev, c, hint=(100, 40), pad=2)
    assert (o[:batch] != 123.0).all() and (o[batch:] == 123.0).all() and (lse[batch:] == 55.0).all()
    some = np.concatenate([[0, batch - 1], rng.choice(batch, 40, replace=False)])  # for the oracle
    table = c["table"][some]
    pages = np.unique(table[table >= 0])
    table = np.where(table >= 0, np.searchsorted(pages, table), -1)
    part = dict(q=c["q"][some], cache=[a[pages] for a in c["cache"]], table=table, ctx=c["ctx"][some], starts=np.arange(len(some) + 1))
    check_attn(part, (o[some], lse[some]))


@pytest.mark.parametrize("new", [1, 30, 90])
def test_attention_rows_of_no_sequence(dev, new):
    """Rows before the first sequence stay as they were, as those past the last one do."""
    rng = np.random.default_rng(new)
    c = attn_case(rng, [70, 200], [new, new], 8, 2, 128, 32)
    before = 5
    moved = dict(c, starts=c["starts"] + before, q=np.concatenate([np.ones((before, 8, 128), np.float32), c["q"]]))
    o, lse = run_attn(dev, moved, hint=(new, 200), pad=1)
    assert (o[:before] == 123.0).all() and (lse[:before] == 55.0).all()
    check_attn(c, (o[before:], lse[before:]))


def test_attention_not_causal(dev):
    rng = np.random.default_rng(2)
    for d in (64, 128):
        c = attn_case(rng, [70, 0, 19], [9, 4, 33], 6, 3, d, 32)
        check_attn(c, run_attn(dev, c, causal=False), causal=False)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.7])
def test_attention_scales(dev, scale):
    rng = np.random.default_rng(3)
    for new in ([3, 20], [2, 1], [70, 30]):
        c = attn_case(rng, [90, 133], new, 4, 2, 64, 16)
        c["cache"][2][c["table"][0, 1]] = 0
        c["cache"][3][c["table"][0, 2]] = 0
        check_attn(c, run_attn(dev, c, scale=scale), scale=scale)


def test_attention_without_starts(dev):
    rng = np.random.default_rng(4)
    c = attn_case(rng, [90, 33, 0, 700], [1] * 4, 4, 2, 64, 64)
    check_attn(c, run_attn(dev, c, starts=False))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 20, 80])
def test_attention_unseen_tokens(dev, new, d):
    """What a query does not see does not reach it: scales that hold NaN or infinities, page numbers that are none."""
    rng = np.random.default_rng(new)
    c = attn_case(rng, [200, 130], [new, new], 4, 2, d, 16, extra=6)
    used = np.unique(c["table"][c["table"] >= 0])
    ks, vs = c["cache"][2:]
    spare = np.setdiff1d(np.arange(len(ks)), used)
    ks[spare], vs[spare] = np.nan, np.inf
    ks[c["table"][0, 12], :, 8:], vs[c["table"][0, 12], :, 8:] = np.nan, np.nan  # behind the context, in its last page
    ks[c["table"][1, 8], :, 2:], vs[c["table"][1, 8], :, 2:] = np.inf, -np.inf
    c["table"][0, 13:] = spare[0]
    c["table"][0, 2], c["table"][0, 5], c["table"][1, 0], c["table"][1, 4] = -1, len(ks), 2 ** 31 - 1, -2 ** 31
    check_attn(c, run_attn(dev, c))
    # the last token holds NaN, in one group of one head: the last query sees it, the others do not
    c = attn_case(rng, [201], [new], 4, 2, d, 16)
    ks, vs = c["cache"][2:]
    page = c["table"][0, 12]
    clean = {n: [a.copy() for a in x] if n == "cache" else x for n, x in c.items()}
    vs[page, 0, 8, 0] = np.nan
    o, _ = run_attn(dev, c)
    assert np.isnan(o[-1, :2, :64]).all() and np.isfinite(o[-1, 2:]).all() and np.isfinite(o[:-1]).all() and np.isfinite(o[-1, :, 64:]).all()
    ks[page, 1, 8, 0] = np.nan
    o, _ = run_attn(dev, c)
    assert np.isnan(o[-1, 2:]).all() and np.isfinite(o[:-1]).all()
    ref, _, tol, _ = oracle(clean)
    assert (np.abs(o - ref)[:-1] <= tol[:-1]).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 20, 80])
def test_attention_of_scales_that_are_no_numbers(dev, new, d):
    """An infinite scale counts as NaN; a token that a row sees counts however little it weighs, early or late in the context."""
    rng = np.random.default_rng(new)
    for where in (3, 90, 195):
        for value in (np.nan, np.inf, -np.inf):
            c = attn_case(rng, [300], [new], 4, 2, d, 16)
            c["q"][...] = 30.0  # the token's score lies some hundreds below the others'
            ks, vs = c["cache"][2:]
            page, at = c["table"][0, where // 16], where % 16
            k_codes = c["cache"][0]
            k_codes[page, 0, at] = 0x11  # codes of -7
            ks[page, 0, at] = 0.5
            vs[page, 0, at, 0] = value
            o, _ = run_attn(dev, c)
            assert np.isnan(o[:, :2, :64]).all() and np.isfinite(o[:, :2, 64:]).all() and np.isfinite(o[:, 2:]).all()
            ks[page, 1, at, 0] = value
            o, _ = run_attn(dev, c)
            assert np.isnan(o[:, 2:]).all() and np.isfinite(o[:, :2, 64:]).all()


def test_attention_of_infinite_queries(dev):
    """An infinity or NaN in one row and head of q reaches that one alone."""
    rng = np.random.default_rng(5)
    for new in (1, 9, 70):
        c = attn_case(rng, [150, 90], [new, new], 4, 2, 128, 16)
        ref, _, tol, _ = oracle(c)
        q = c["q"].copy()
        q[0, 1, 5], q[-1, 2, 99] = np.inf, np.nan
        o, _ = run_attn(dev, dict(c, q=q))
        bad = np.zeros(o.shape[:2], bool)
        bad[0, 1] = bad[-1, 2] = True
        assert np.isnan(o[bad]).all() and (np.abs(o - ref)[~bad] <= tol[~bad]).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 20, 80])
def test_attention_of_infinite_queries_whose_scores_are_all_low(dev, new, d):
    """An infinity is NaN also where every token that the row sees gives -inf: nothing tells it from a row that sees none."""
    rng = np.random.default_rng(new + d)
    for ctx, causal in ((3, False), (new, True)):
        c = attn_case(rng, [ctx], [new], 4, 2, d, 16)
        c["cache"][0][...] = 0x33  # codes of -5
        c["cache"][2] = np.abs(c["cache"][2])
        ref, lse, tol, ltol = oracle(c, causal=causal)
        for scale, value in ((None, np.inf), (-1 / math.sqrt(d), -np.inf)):
            q = c["q"] * (1 if scale is None else -1)
            q[0, 1, 5] = value
            o, low = run_attn(dev, dict(c, q=q), scale=scale, causal=causal)
            bad = np.zeros(o.shape[:2], bool)
            bad[0, 1] = True
            assert np.isnan(o[bad]).all() and np.isnan(low[bad]).all()
            assert (np.abs(o - ref)[~bad] <= tol[~bad]).all() and (np.abs(low - lse)[~bad] <= ltol[~bad]).all()


@pytest.mark.parametrize("space", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 20, 80])
def test_attention_of_vast_values(dev, new, d, space):
    """V scales near bf16's largest number, of all tokens, of late ones, of one: outputs are finite, so is every sum on the way.
    The bounds are relative (a power of two on V's scales changes no rounding)."""
    rng = np.random.default_rng(new + d)
    hint = (new, 2100)
    for tokens in (slice(None), slice(700, None), slice(1203, 1204), slice(40, 60)):
        c = attn_case(rng, [2100, 130], [new, new], 4, 2, d, 16)
        vs = c["cache"][3]
        at = np.arange(2100)[tokens]
        where = c["table"][0, at // 16], slice(None), at % 16, 0
        vs[where] = np.abs(vs[where]) * np.float32(2.0 ** 126)  # below 0.12 * 2^126, so the values below 2^126
        ref = oracle(c)
        with stream_workspace(dev, K.kv4_cache_attention_workspace_size(2 * new, 2, 4, 2, d, *hint)) if space else contextlib.nullcontext():
            check_attn(c, run_attn(dev, c, hint=hint), ref=ref)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 20, 80])
def test_attention_of_vast_keys(dev, new, d):
    """K scales near bf16's largest number and small queries: scores of ordinary size."""
    rng = np.random.default_rng(new + d)
    for tokens in (slice(None), slice(700, None), slice(1203, 1204)):
        c = attn_case(rng, [1500, 130], [new, new], 4, 2, d, 16, low=1.0, high=1.9)
        c["q"] *= np.float32(2.0 ** -117)
        ks = c["cache"][2]
        at = np.arange(1500)[tokens]
        ks[c["table"][0, at // 16], :, at % 16] *= np.float32(2.0 ** 124)
        check_attn(c, run_attn(dev, c, scale=2.0 ** -8), scale=2.0 ** -8)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 20, 80])
def test_attention_of_vast_keys_under_a_scale_of_zero(dev, new, d):
    """Every token that a row sees counts alike, whatever its keys."""
    rng = np.random.default_rng(new + d)
    c = attn_case(rng, [700, 130], [new, new], 4, 2, d, 16, low=1.0, high=1.9)
    c["q"] *= np.float32(0.25)
    clean = oracle(c, scale=0.0)
    c["cache"][2] *= np.float32(2.0 ** 124)
    check_attn(c, run_attn(dev, c, scale=0.0), ref=clean)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 20, 80])
def test_attention_of_small_values_beside_unseen_vast_ones(dev, new, d):
    """Scales behind the context and on pages that are none change no bit, however large."""
    rng = np.random.default_rng(new + d)
    c = attn_case(rng, [200, 130], [new, new], 4, 2, d, 16, extra=6)
    ks, vs = c["cache"][2:]
    vs *= np.float32(2.0 ** -86)
    c["table"][0, 2] = -1
    spare = np.setdiff1d(np.arange(len(ks)), c["table"])
    want = run_attn(dev, c)
    assert (want[0] != 0).any()
    for value in (2.0 ** 120, np.inf):
        for s in (ks, vs):
            s[spare] = value
            s[c["table"][0, 12], :, 8:], s[c["table"][1, 8], :, 2:] = value, -value
        for g, w in zip(run_attn(dev, c), want):
            np.testing.assert_array_equal(g, w)


def test_attention_empty_tables(dev):
    """No page at all, and tables of unfilled rows."""
    rng = np.random.default_rng(6)
    c = attn_case(rng, [40, 40], [1, 1], 2, 2, 64, 16)
    c["table"][:] = -1
    o, lse = run_attn(dev, c)
    assert (o == 0).all() and np.isneginf(lse).all()
    q, out, ctx = up(dev, c["q"]), up(dev, np.ones_like(c["q"])), ints(dev, [4, 4])
    check(lib.teeny_kv4_cache_attention(q.ptr, None, None, None, None, None, ctx.ptr, None, out.ptr, None, 2, 2, 2, 2,
                                        64, 0, 16, 0, 1, 40, 128, 0.1, 1, None))
    assert (from_bf16(out.to_host()) == 0).all()


def test_attention_query_stride(dev):
    rng = np.random.default_rng(8)
    for new in ([4, 1], [90, 31]):
        c = attn_case(rng, [100, 31], new, 4, 2, 64, 16)
        t, hq, d = c["q"].shape
        wide = np.full((t, hq * d + 24), 7.0, np.float32)
        wide[:, 16:16 + hq * d] = c["q"].reshape(t, -1)
        qb, o, lse = up(dev, wide), dev.buffer(bf16, c["q"].shape), dev.buffer("f32", (t, hq))
        cache = up_cache(dev, c["cache"]) + [dev.upload(c["table"]), ints(dev, c["ctx"]), ints(dev, c["starts"])]
        check(lib.teeny_kv4_cache_attention(qb.ptr + 32, *[b.ptr for b in cache], o.ptr, lse.ptr, t, 2, hq, 2, d, len(c["cache"][0]), 16,
                                            c["table"].shape[1], max(new), 100, hq * d + 24, 1 / math.sqrt(d), 1, None))
        check_attn(c, (from_bf16(o.to_host()), lse.to_host()))


def test_attention_of_any_scale(dev):
    """Scales of all of bf16's bits, not five: codes times scales are rounded where there are many rows (2^-8 of each)."""
    rng = np.random.default_rng(7)
    for new in (1, 5, 90):
        c = attn_case(rng, [300, 120], [new, new], 4, 2, 128, 32)
        for i in (2, 3):
            c["cache"][i] = rounded(c["cache"][i] * rng.uniform(0.9, 1.1, c["cache"][i].shape))
        o, lse, tol, ltol = oracle(c)
        kq, vq = kv4.codes_of(*c["cache"][:2])
        most = [np.abs(x * np.repeat(s, 64, -1)).max() for x, s in ((kq, c["cache"][2]), (vq, c["cache"][3]))]
        off = np.abs(c["q"]).sum(-1) / math.sqrt(128) * most[0] * H16  # of a score
        check_attn(c, run_attn(dev, c), ref=(o, lse, tol + most[1] * (2 * off[..., None] + H16), ltol + 2 * off))


@pytest.mark.parametrize("new", [1, 20, 80])
def test_attention_repeats(dev, new):
    """The same call gives the same bits, split or not, also where scales are vast or no numbers."""
    rng = np.random.default_rng(new)
    c = attn_case(rng, [2100, 130], [new, new], 8, 2, 128, 16)
    for value in (None, 2.0 ** 120, np.nan):
        if value is not None:
            c["cache"][3][c["table"][0, 70], 0, 3:9, 1] = value
        for size in (4096, K.kv4_cache_attention_workspace_size(2 * new, 2, 8, 2, 128, new, 2100)):
            with stream_workspace(dev, size):
                runs = [run_attn(dev, c, hint=(new, 2100)) for _ in range(4)]
            for o, lse in runs[1:]:
                np.testing.assert_array_equal(o, runs[0][0])
                np.testing.assert_array_equal(lse, runs[0][1])


# ── together ────────────────────────────────────────────────────────────────


def test_two_streams(dev):
    """Calls on two streams at once, each with its own workspace: split attention, shared tiles and few rows."""
    rng = np.random.default_rng(14)
    streams = [Stream.create(), Stream.create()]
    jobs = []
    for i, (ctx, new) in enumerate([([3000, 40, 700], [1, 1, 1]), ([1500, 300], [60, 90]), ([900, 2100], [9, 5]), ([2500], [1])]):
        c = attn_case(rng, ctx, new, 8, 2, 128, 16)
        bufs = [up(dev, c["q"]), *up_cache(dev, c["cache"]), dev.upload(c["table"]), ints(dev, c["ctx"]), ints(dev, c["starts"])]
        t = c["q"].shape[0]
        jobs.append((c, streams[i % 2], bufs, (max(new), max(ctx)), dev.buffer(bf16, c["q"].shape), dev.buffer("f32", (t, 8)),
                     K.kv4_cache_attention_workspace_size(t, len(ctx), 8, 2, 128, max(new), max(ctx))))
    dev.synchronize()
    most = max(j[-1] for j in jobs)
    with stream_workspace(dev, most, streams[0]), stream_workspace(dev, most, streams[1]):
        for _ in range(5):
            for c, s, bufs, hint, o, lse, _ in jobs:
                K.kv4_cache_attention(*bufs, *hint, o=o, lse=lse, stream=s)
        for s in streams:
            s.synchronize()
        for c, s, bufs, hint, o, lse, _ in jobs:
            check_attn(c, (from_bf16(o.to_host()), lse.to_host()))


def test_large_cache(dev):
    """Pages whose bytes lie past 2^32: the same tokens at the pool's start and end."""
    rng = np.random.default_rng(13)
    hkv, d, page, pages = 8, 128, 128, 72000  # 4.7 GB each for K and V
    kc, vc = dev.buffer("i8", (pages, hkv, page, d // 2)), dev.buffer("i8", (pages, hkv, page // 16, d, 8))
    ks, vs = dev.buffer(bf16, (pages, hkv, page, 2)), dev.buffer(bf16, (pages, hkv, page, 2))
    n = 150
    k, v = (up(dev, rng.standard_normal((n, hkv, d))) for _ in range(2))
    q, q1 = up(dev, rng.standard_normal((2, 16, d))), up(dev, rng.standard_normal((90, 16, d)))
    pos, f, outs = ints(dev, np.arange(n)), dev.upload(freqs(d)), []
    for table in ([[0, 1]], [[pages - 2, pages - 1]]):
        slots = np.array([table[0][t // page] * page + t % page for t in range(n)], np.int32)
        K.kv4_cache_append(None, k, v, pos, ints(dev, slots), f, kc, vc, ks, vs)
        rest = [ints(dev, np.array(table)), ints(dev, [n])]
        outs.append([K.kv4_cache_attention(a, kc, vc, ks, vs, *rest, ints(dev, [0, m])).to_host() for a, m in ((q, 2), (q1, 90))])
    for a, b in zip(*outs):
        np.testing.assert_array_equal(a, b)
        assert np.isfinite(from_bf16(a)).all() and from_bf16(a).any()
    for b in (kc, vc):
        b.free()


class Layer:
    """A decoder layer's attention half as a server runs it: a 4-bit projection to q, k and v with adapters beside it, the
    append, attention, and a 4-bit projection back, with adapters."""

    def __init__(self, dev, rng, batch, rows, pages, width, stream=None):
        self.dev, self.stream, self.page = dev, stream, 16
        self.hq, self.hkv, self.d, self.hidden, self.rank, loaded = 4, 2, 64, 256, 8, 3
        hq, hkv, d, hidden = self.hq, self.hkv, self.d, self.hidden
        self.n = (hq + 2 * hkv) * d
        self.w, self.parts = {}, {}
        for name, n, k in (("qkv", self.n, hidden), ("out", hidden, hq * d)):
            codes, scale = rng.integers(-8, 8, (n, k)).astype(np.int8), rng.uniform(0.005, 0.02, (n, k // 64)).astype(np.float32)
            a, b = rounded(rng.standard_normal((loaded, 8, k)) / 16), rounded(rng.standard_normal((loaded, n, 8)) * 0.2)
            s = rng.uniform(0.5, 2, loaded).astype(np.float32)
            self.w[name] = codes, scale, a, b, s
            self.parts[name] = K.pack_int4(dev.upload(codes)), dev.upload(scale), up(dev, a), up(dev, b), dev.upload(s)
        self.freq = freqs(d)
        self.f = dev.upload(self.freq)
        self.cache = up_cache(dev, random_cache(rng, pages, hkv, self.page, d))
        self.seq, self.table = ints(dev, np.zeros(batch)), dev.upload(np.full((batch, width), -1, np.int32))
        self.stack, self.count, self.new = ints(dev, rng.permutation(pages)), ints(dev, [pages]), ints(dev, np.zeros(batch))
        self.x, self.ids = dev.buffer(bf16, (rows, hidden)), ints(dev, np.zeros(rows))
        self.buf = {n: dev.buffer(bf16, (rows, m)) for n, m in (("qkv", self.n), ("y", hidden))}
        self.q, self.o = (dev.buffer(bf16, (rows, hq, d)) for _ in range(2))
        self.o2 = dev.buffer(bf16, (rows, hq * d))
        self.at = {n: dev.buffer("i32", (m,)) for n, m in (("slots", rows), ("pos", rows), ("starts", batch + 1), ("granted", batch))}
        self.rows, self.pages, self.width = rows, pages, width

    def step(self, longest):
        s, at, dev = self.stream, self.at, self.dev
        K.kv_cache_plan(self.new, self.seq, self.table, self.stack, self.count, self.page, slots=at["slots"], positions=at["pos"],
                        q_starts=at["starts"], context_lens=self.seq, granted=at["granted"], free_after=self.count, stream=s)
        qw, qs, a, b, scale = self.parts["qkv"]
        K.w4a16_linear(self.x, qw, qs, 64, y=self.buf["qkv"], stream=s)
        K.adapter_add(self.x, a, b, self.ids, self.buf["qkv"], scale=scale, out=self.buf["qkv"], stream=s)
        p, hd = self.buf["qkv"].ptr, 2 * self.d
        check(lib.teeny_kv4_cache_append(p, p + self.hq * hd, p + (self.hq + self.hkv) * hd, at["pos"].ptr, at["slots"].ptr, self.f.ptr, self.q.ptr,
                                         *[c.ptr for c in self.cache], self.rows, self.hq, self.hkv, self.d, self.d, self.pages, self.page,
                                         self.n, self.n, self.n, 0, s.handle if s else None))
        K.kv4_cache_attention(self.q, *self.cache, self.table, self.seq, at["starts"], max_q_len=longest, max_context=self.width * self.page,
                              o=self.o, stream=s)
        check(lib.teeny_hip_memcpy_d2d(self.o2.ptr, self.o.ptr, self.o.nbytes, s.handle if s else None))
        qw, qs, a, b, scale = self.parts["out"]
        K.w4a16_linear(self.o2, qw, qs, 64, y=self.buf["y"], stream=s)
        K.adapter_add(self.o2, a, b, self.ids, self.buf["y"], scale=scale, out=self.buf["y"], stream=s)


def test_steps_together(dev):
    """Prompts, then single tokens, with requests that end and pages that are used again: each operator of a step against
    its plain form on what the operator before it gave."""
    rng = np.random.default_rng(11)
    batch, rows, width, pages = 4, 200, 12, 40
    net = Layer(dev, rng, batch, rows, pages, width)
    net.q.to_device(to_bf16(np.full(net.q.shape, 123.0, np.float32)))
    held = np.zeros(batch, int)
    for new in [[50, 7, 0, 90], [1, 1, 33, 1], [1, 1, 1, -1], [1, -1, 1, 100], [1, 20, 1, 1]] + [[1, 1, 1, 1]] * 6:
        n = sum(max(i, 0) for i in new)
        x = rounded(rng.standard_normal((rows, net.hidden)))
        ids = rng.integers(-1, 4, batch)  # of three: the fourth is none
        net.x.to_device(to_bf16(x))
        net.ids.to_device(np.array([i for b, m in enumerate(new) for i in [ids[b]] * max(m, 0)] + [-1] * (rows - n), np.int32))
        net.new.to_device(np.array(new, np.int32))
        before = down_cache(net.cache)
        net.step(max(new))
        held = np.array([0 if m < 0 else h + m for h, m in zip(held, new)])
        assert net.seq.to_host().tolist() == held.tolist()
        slots, pos, starts = (net.at[m].to_host() for m in ("slots", "pos", "starts"))
        ids = net.ids.to_host()

        def projected(name, x):
            codes, scale, a, b, s = net.w[name]
            y, off = kv.w4_linear(x, codes, scale, None, None, 64, None, False)
            # the layer's output is rounded to bf16 before the adapter's is added to it
            out, tol = kv4.adapter(x, a, b, ids, s, y.astype(np.float32))
            return out, tol + off + np.abs(y) * H16

        qkv = from_bf16(net.buf["qkv"].to_host())
        ref, tol = projected("qkv", x)
        assert (np.abs(qkv - ref) <= tol).all()
        q, k, v = (a.reshape(rows, -1, net.d) for a in np.split(qkv, [net.hq * net.d, (net.hq + net.hkv) * net.d], axis=1))
        cache = down_cache(net.cache)
        for g, r in zip(cache, kv4.append(kv4.rotate(k, pos, net.freq, False).astype(np.float32), v, slots, before)):
            np.testing.assert_array_equal(g, r)
        turned = from_bf16(net.q.to_host())
        assert (turned[n:] == 123.0).all() or n < 140  # rows of earlier steps' prompts stay
        ref = kv4.rotate(q, pos, net.freq, False)
        assert (np.abs(turned - ref)[:n] <= np.abs(ref[:n]) * H16 * 1.01 + 8 * H32 * np.abs(q[:n]).max()).all()
        c = dict(q=turned[:n], cache=cache, table=net.table.to_host(), ctx=held, starts=starts)
        o = from_bf16(net.o.to_host())
        ref, _, tol, _ = oracle(c)
        assert (np.abs(o[:n] - ref) <= tol).all()
        ref, tol = projected("out", o.reshape(rows, -1))
        y = from_bf16(net.buf["y"].to_host())
        assert (np.abs(y - ref) <= tol)[:n].all()


def test_step_in_a_graph(dev):
    """A step captured once and replayed while requests grow: every replay equals the eager step."""
    batch, width, pages = 3, 40, 90
    streams = [Stream.create(), Stream.create()]
    nets = [Layer(dev, np.random.default_rng(12), batch, batch, pages, width, s) for s in streams]
    rng = np.random.default_rng(13)
    lens, table = [30, 500, 15], np.full((batch, width), -1, np.int32)
    order, at = rng.permutation(pages).astype(np.int32), 0
    for b, n in enumerate(lens):
        used = kv.pages_of(n, 16)
        table[b, :used] = order[at:at + used]
        at += used
    stack = np.zeros(pages, np.int32)
    stack[:pages - at] = order[at:]
    for net in nets:
        net.seq.to_device(np.array(lens, np.int32))
        net.table.to_device(table)
        net.stack.to_device(stack)
        net.count.to_device(np.array([pages - at], np.int32))
        net.new.to_device(np.ones(batch, np.int32))
        net.ids.to_device(np.array([2, -1, 0], np.int32))
    dev.synchronize()
    size = K.kv4_cache_attention_workspace_size(batch, batch, nets[0].hq, nets[0].hkv, nets[0].d, 1, width * 16)
    with stream_workspace(dev, size + (1 << 20), streams[0]), stream_workspace(dev, size + (1 << 20), streams[1]):
        streams[0].begin_capture()
        nets[0].step(1)
        graph = streams[0].end_capture()
        for i in range(20):
            x = to_bf16(rng.standard_normal((batch, nets[0].hidden)).astype(np.float32))
            for net in nets:
                net.x.to_device(x)
            dev.synchronize()
            graph.launch(streams[0])
            nets[1].step(1)
            for s in streams:
                s.synchronize()
            for a, b in zip([*nets[0].cache, nets[0].o, nets[0].q, nets[0].seq, nets[0].table, *nets[0].buf.values()],
                            [*nets[1].cache, nets[1].o, nets[1].q, nets[1].seq, nets[1].table, *nets[1].buf.values()]):
                np.testing.assert_array_equal(a.to_host(), b.to_host(), err_msg=f"replay {i}")
        assert nets[0].seq.to_host().tolist() == [n + 20 for n in lens]
        graph.destroy()


class WideLayer(Layer):
    """Adapters of a rank that takes two launches, the ranks' products by way of the workspace that the step's other operators use."""

    def __init__(self, dev, rng, *args):
        super().__init__(dev, rng, *args)
        loaded, rank = 3, 128
        for name, (codes, scale, _, _, s) in list(self.w.items()):
            n, k = codes.shape
            a, b = rounded(rng.standard_normal((loaded, rank, k)) / 16), rounded(rng.standard_normal((loaded, n, rank)) * 0.05)
            self.w[name] = codes, scale, a, b, s
            self.parts[name] = *self.parts[name][:2], up(dev, a), up(dev, b), self.parts[name][4]

    def workspace(self, longest):
        """The largest of the step's operators'."""
        context = self.width * self.page
        adapters = [K.adapter_add_workspace_size(self.rows, c.shape[0], c.shape[1], 128) for c, *_ in self.w.values()]
        attention = K.kv4_cache_attention_workspace_size(self.rows, self.seq.numel, self.hq, self.hkv, self.d, longest, context)
        layers = [K.w4a16_linear_workspace_size(self.rows, *c.shape, 64) for c, *_ in self.w.values()]
        assert min(adapters) > 0
        return max(*adapters, *layers, attention)


def test_steps_with_one_workspace(dev, monkeypatch):
    """The steps of test_steps_together, with prompts: the adapters' two launches and the 4-bit layers on one workspace."""
    monkeypatch.setitem(globals(), "Layer", WideLayer)
    with stream_workspace(dev, WideLayer(dev, np.random.default_rng(0), 4, 200, 40, 12).workspace(100)):
        test_steps_together(dev)


def test_step_with_one_workspace_in_a_graph(dev, monkeypatch):
    """The replays of test_step_in_a_graph, with those adapters and split attention: its workspace holds every operator's part."""
    monkeypatch.setitem(globals(), "Layer", WideLayer)
    net = WideLayer(dev, np.random.default_rng(0), 3, 3, 90, 40)
    size = K.kv4_cache_attention_workspace_size(3, 3, net.hq, net.hkv, net.d, 1, 40 * 16)
    assert size > 0 and net.workspace(1) <= size + (1 << 20)
    test_step_in_a_graph(dev)
