"""The 8-bit paged K/V cache on the GPU: plan, writes, attention, and the three
in a row, against the plain forms of kv_cases.py."""
import ctypes
import math

import numpy as np
import pytest

import kv_cases as kv
from gpu_util import stream_workspace
from teenygrad_amd import _lib
from teenygrad_amd import kernels as K
from teenygrad_amd._lib import check, lib
from teenygrad_amd.dtypes import bf16, from_bf16, to_bf16
from teenygrad_amd.runtime import NULL_STREAM, Stream

pytestmark = pytest.mark.gpu

NAMES = ("slots", "positions", "q_starts", "context_lens", "granted", "free_after")


def ints(dev, a):
    return dev.upload(np.asarray(a, np.int32).reshape(-1) if np.ndim(a) < 2 else np.asarray(a, np.int32))


def make_table(rng, lens, page, width, extra=0):
    """A block table with pages in random order; (table, pages, unused pages)."""
    counts = [kv.pages_of(n, page) for n in lens]
    order = rng.permutation(sum(counts) + extra).astype(np.int32)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table, len(order), order[at:]


# ── plan ────────────────────────────────────────────────────────────────────


def plan_case(rng, batch, page, width, tokens, free=None):
    seq = rng.integers(0, width * page + 1, batch)
    new = np.where(rng.random(batch) < 0.15, -1, np.where(rng.random(batch) < 0.2, rng.integers(0, 3 * page, batch), 1))
    table, pages, spare = make_table(rng, seq, page, width, extra=batch * 3 if free is None else free)
    stack = np.zeros(pages, np.int32)
    stack[:len(spare)] = spare
    return new.astype(np.int32), seq.astype(np.int32), table, stack, len(spare), tokens


@pytest.mark.parametrize("batch,page,width,tokens,free", [
    (1, 16, 1, 1, None), (3, 16, 4, 40, None), (8, 128, 3, 8, None), (64, 32, 9, 500, None), (65, 16, 20, 3000, None),
    (300, 64, 5, 4000, 10), (300, 16, 30, 1000, None), (257, 16, 7, 260, 0), (2000, 16, 6, 9000, 500), (4096, 32, 3, 20000, 50)])
def test_plan(dev, batch, page, width, tokens, free):
    rng = np.random.default_rng(batch * 131 + tokens)
    new, seq, table, stack, count, tokens = plan_case(rng, batch, page, width, tokens, free)
    ref, ref_table, ref_stack = kv.plan(new, seq, table, stack, count, page, tokens)
    bufs = [ints(dev, a) for a in (new, seq)] + [dev.upload(table), ints(dev, stack), ints(dev, [count])]
    out = dict(zip(NAMES, K.kv_cache_plan(*bufs, page, n_tokens=tokens)))
    for n in NAMES:
        np.testing.assert_array_equal(out[n].to_host(), ref[n], err_msg=n)
    np.testing.assert_array_equal(bufs[2].to_host(), ref_table)
    # below the old and the new count: entries above both are free to hold anything
    top = max(count, int(ref["free_after"][0]))
    np.testing.assert_array_equal(bufs[3].to_host()[:top], ref_stack[:top])
    # in place: the same numbers over the inputs
    bufs = [ints(dev, a) for a in (new, seq)] + [dev.upload(table), ints(dev, stack), ints(dev, [count])]
    K.kv_cache_plan(*bufs, page, n_tokens=tokens, context_lens=bufs[1], granted=bufs[0], free_after=bufs[4])
    for n, b in (("granted", 0), ("context_lens", 1), ("free_after", 4)):
        np.testing.assert_array_equal(bufs[b].to_host(), ref[n], err_msg=n)
    np.testing.assert_array_equal(bufs[2].to_host(), ref_table)


def test_plan_odd_lengths(dev):
    """Lengths that cannot be: the request is refused and nothing is read or written out of place."""
    page, width, pages = 16, 4, 10
    big = 2 ** 31 - 1
    new = np.array([big, 1, 5, -1, 3, 1, big, -7], np.int32)
    seq = np.array([0, -5, 62, big, 0, 64, big, -3], np.int32)
    table = np.zeros((8, width), np.int32)
    stack = np.arange(pages, dtype=np.int32)
    bufs = [ints(dev, a) for a in (new, seq)] + [dev.upload(table), ints(dev, stack), ints(dev, [2])]
    out = dict(zip(NAMES, K.kv_cache_plan(*bufs, page, n_tokens=30)))
    # the first request fills the step, so every later one lies past its end
    assert out["granted"].to_host().tolist() == [0] * 8
    assert out["q_starts"].to_host().tolist() == [0] + [30] * 8
    assert (out["slots"].to_host() == -1).all() and (out["positions"].to_host() == -1).all()
    assert out["context_lens"].to_host().tolist() == [0, -5, 62, 0, 0, 64, big, 0]
    assert out["free_after"].to_host().tolist() == [6]  # the longest row's four pages came back
    for count in (-3, 100):  # a free count that cannot be is the nearest that can
        bufs = [ints(dev, [1]), ints(dev, [0]), dev.upload(np.full((1, 4), -1, np.int32)), ints(dev, stack), ints(dev, [count])]
        out = dict(zip(NAMES, K.kv_cache_plan(*bufs, page, n_tokens=1)))
        assert out["free_after"].to_host().tolist() == [0 if count < 0 else pages - 1]
        assert out["granted"].to_host().tolist() == [0 if count < 0 else 1]


def test_plan_of_nothing(dev):
    stack, count, slots, positions, starts, left = (ints(dev, a) for a in ([0, 1, 2], [3], [7, 7], [0, 0], [9], [0]))
    check(lib.teeny_kv_cache_plan(None, None, None, stack.ptr, count.ptr, starts.ptr, slots.ptr, positions.ptr, None, None,
                                  left.ptr, 0, 0, 3, 16, 2, None))
    assert starts.to_host().tolist() == [0] and slots.to_host().tolist() == [-1, -1] and left.to_host().tolist() == [3]


# ── write ───────────────────────────────────────────────────────────────────


def write_case(rng, before, new, heads, d, page, pad=0):
    after = [a + n for a, n in zip(before, new)]
    table, pages, _ = make_table(rng, after, page, max(1, max(kv.pages_of(n, page) for n in after)), extra=2)
    slots = [table[b, (a + i) // page] * page + (a + i) % page for b, (a, n) in enumerate(zip(before, new)) for i in range(n)]
    slots = np.array(slots + [-1] * pad, np.int32)
    t = len(slots)
    x = {n: from_bf16(to_bf16(rng.standard_normal((t, heads, d)).astype(np.float32) * (1 + 3 * rng.random((t, heads, 1)).astype(np.float32))))
         for n in "kv"}
    kc = rng.integers(-127, 128, (pages, heads, page, d)).astype(np.int8)
    vc = rng.integers(-127, 128, (pages, heads, d, page)).astype(np.int8)
    ks, vs = (rng.uniform(0.01, 0.06, (pages, heads)).astype(np.float32) for _ in range(2))
    return x, slots, kc, vc, ks, vs


def run_write(dev, x, slots, kc, vc, ks, vs):
    bufs = [dev.upload(a) for a in (kc, vc, ks, vs)]
    K.kv_cache_write(dev.upload(to_bf16(x["k"]), bf16), dev.upload(to_bf16(x["v"]), bf16), ints(dev, slots), *bufs)
    return [b.to_host() for b in bufs]


def check_write(dev, x, slots, kc, vc, ks, vs):
    page = kc.shape[2]
    got = run_write(dev, x, slots, kc, vc, ks, vs)
    k_ref = kv.write(x["k"], slots, kc, ks, page, False)
    v_ref = kv.write(x["v"], slots, vc, vs, page, True)
    for g, r, n in zip(got, (k_ref[0], v_ref[0], k_ref[1], v_ref[1]), ("k codes", "v codes", "k scales", "v scales")):
        np.testing.assert_array_equal(g, r, err_msg=n)
    return got


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("before,new,heads", [
    ([0], [1], 1), ([15, 16, 17, 0, 127], [1, 1, 1, 1, 1], 5), ([3, 100], [13, 200], 2), ([0, 1, 31, 63], [129, 5, 1, 66], 3),
    (list(range(0, 70)), [1] * 70, 2), ([7, 0], [1100, 90], 1)])
def test_write(dev, page, d, before, new, heads):
    rng = np.random.default_rng(sum(before) + sum(new) + page + d)
    check_write(dev, *write_case(rng, before, new, heads, d, page, pad=3))


def test_write_skips_and_bounds(dev):
    """Padding among the rows, slots past the cache, and a pool where only one page is meant."""
    rng = np.random.default_rng(5)
    x, slots, *cache = write_case(rng, [4, 20], [9, 9], 2, 64, 16)
    slots = slots.copy()
    slots[3] = -1  # a run breaks here and goes on in the same page: keep them in pages of their own
    slots[4:9] = -1
    pages = cache[0].shape[0]
    slots[12:15] = [pages * 16, pages * 16 + 1, 2 ** 31 - 1]
    slots[15:] = -5
    check_write(dev, x, slots, *cache)


@pytest.mark.parametrize("page", [16, 64])
def test_write_special_values(dev, page):
    """Zeros, infinities, NaN, values whose scale is tiny, and pages that were begun anew after them."""
    rng = np.random.default_rng(page)
    x, slots, kc, vc, ks, vs = write_case(rng, [5, 5, 5, 5, 0, 5, 2], [2, 2, 2, 2, 3, 2, 1], 2, 128, page)
    for n in "kv":
        a = x[n]
        a[0:2] = 0
        a[2, 0, 7] = np.inf
        a[4, 1, 90] = np.nan
        a[6:8] = from_bf16(to_bf16(np.float32(2e-38)))
        a[8:11, 0] = 0
        a[8:11, 1] = from_bf16(to_bf16(np.float32(2e-38)))  # a scale below the normal numbers
        a[12, 0, 0] = -np.inf
    first = slots[0] // page
    ks[first] = 0  # held nothing but zeros
    last = slots[-1] // page
    ks[last], vs[last] = np.nan, np.inf  # held NaN: stays so
    got = check_write(dev, x, slots, kc, vc, ks, vs)
    assert np.isnan(got[2][last]).all() and np.isinf(got[3][last]).all()
    # the same pages from their first slot: clean again
    x2 = {n: np.abs(rng.standard_normal((1, 2, 128))).astype(np.float32) for n in "kv"}
    x2 = {n: from_bf16(to_bf16(a)) for n, a in x2.items()}
    again = check_write(dev, x2, np.array([last * page], np.int32), *got)
    assert np.isfinite(again[2][last]).all() and np.isfinite(again[3][last]).all()


@pytest.mark.parametrize("d", [64, 128])
def test_write_over_all_exponents(dev, d):
    """Codes are rint of the fp32 quotient exactly: pages of every magnitude that bf16 has, and quotients at a half."""
    rng = np.random.default_rng(d)
    exps = np.arange(-133, 128)  # 2^-133: the smallest bf16 number
    x, slots, *cache = write_case(rng, [0] * len(exps), [7] * len(exps), 1, d, 16)
    for n in "kv":
        m = np.ldexp(rng.uniform(-1, 1, x[n].shape), np.repeat(exps, 7)[:, None, None])
        m[3::7] = np.sign(m[3::7]) * np.ldexp((rng.integers(0, 127, m[3::7].shape) + 0.5) / 127, np.repeat(exps, 1)[:, None, None])
        m[0::7, 0, 0] = np.ldexp(1.0, exps)  # the largest: the half steps above are halves of its scale
        x[n] = from_bf16(to_bf16(m.astype(np.float32)))
    check_write(dev, x, slots, *cache)


def test_write_token_strides(dev):
    """K and V as parts of one projection's rows: strides over the C entry point."""
    rng = np.random.default_rng(9)
    heads, d, page = 2, 64, 16
    x, slots, kc, vc, ks, vs = write_case(rng, [3, 0], [20, 5], heads, d, page)
    t, hd = len(slots), heads * d
    row = 3 * hd + 8
    both = np.zeros((t, row), np.float32)
    both[:, hd:2 * hd], both[:, 2 * hd:3 * hd] = x["k"].reshape(t, hd), x["v"].reshape(t, hd)
    qkv = dev.upload(to_bf16(both), bf16)
    bufs, at = [dev.upload(a) for a in (kc, vc, ks, vs)], ints(dev, slots)
    check(lib.teeny_kv_cache_write(qkv.ptr + 2 * hd, qkv.ptr + 4 * hd, at.ptr, *[b.ptr for b in bufs], t, heads, d,
                                   kc.shape[0], page, row, row, None))
    want = kv.write(x["k"], slots, kc, ks, page, False), kv.write(x["v"], slots, vc, vs, page, True)
    for b, r in zip(bufs, (want[0][0], want[1][0], want[0][1], want[1][1])):
        np.testing.assert_array_equal(b.to_host(), r)


# ── attention ───────────────────────────────────────────────────────────────


def attn_case(rng, ctx, new, hq, hkv, d, page, extra=2):
    table, pages, _ = make_table(rng, ctx, page, max(1, max(kv.pages_of(n, page) for n in ctx)) + 1, extra=extra)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = from_bf16(to_bf16(rng.standard_normal((int(starts[-1]), hq, d)).astype(np.float32)))
    kc = rng.integers(-127, 128, (pages, hkv, page, d)).astype(np.int8)
    vc = rng.integers(-127, 128, (pages, hkv, d, page)).astype(np.int8)
    ks, vs = (rng.uniform(0.005, 0.03, (pages, hkv)).astype(np.float32) for _ in range(2))
    return dict(q=q, kc=kc, vc=vc, ks=ks, vs=vs, table=table, ctx=np.array(ctx, np.int32), starts=starts)


def run_attn(dev, c, scale=None, causal=True, hint=None, pad=0, stream=None, starts=True):
    t, hq, d = c["q"].shape
    q = np.concatenate([c["q"], np.ones((pad, hq, d), np.float32)])
    o = dev.upload(to_bf16(np.full(q.shape, 123.0, np.float32)), bf16)
    lse = dev.upload(np.full((t + pad, hq), 55.0, np.float32))
    K.kv_cache_attention(dev.upload(to_bf16(q), bf16), dev.upload(c["kc"]), dev.upload(c["vc"]), dev.upload(c["ks"]), dev.upload(c["vs"]),
                         dev.upload(c["table"]), ints(dev, c["ctx"]), ints(dev, c["starts"]) if starts else None,
                         *(hint or (None, None)), softmax_scale=scale, causal=causal, o=o, lse=lse, stream=stream)
    if stream is not None:
        stream.synchronize()
    return from_bf16(o.to_host()), lse.to_host()


def check_attn(c, got, scale=None, causal=True):
    t, hq, d = c["q"].shape
    o, lse, tol, ltol = kv.attention(c["q"], c["kc"], c["vc"], c["ks"], c["vs"], c["table"], c["ctx"], c["starts"],
                                     1 / math.sqrt(d) if scale is None else scale, causal)
    go, gl = got[0].astype(np.float64), got[1].astype(np.float64)
    assert (go[t:] == 123.0).all() and (gl[t:] == 55.0).all(), "rows past the last sequence were written"
    np.testing.assert_array_equal(np.isneginf(gl[:t]), np.isneginf(lse))
    err = np.abs(go[:t] - o)
    assert (err <= tol).all(), f"o: worst {np.max(err - tol)} over the bound, error {np.max(err)}"
    fin = np.isfinite(lse)
    assert (np.abs(gl[:t][fin] - lse[fin]) <= ltol[fin]).all(), np.max(np.abs(gl[:t][fin] - lse[fin]) - ltol[fin])


ATTN = [
    ([1], [1], 1, 1), ([5, 16, 17, 64, 65, 130], [1] * 6, 8, 2), ([0, 3, 200], [1, 1, 1], 7, 1), ([1000, 30, 515], [1, 1, 1], 16, 2),
    ([40, 7, 300], [5, 7, 2], 4, 4), ([33, 90], [16, 3], 4, 2), ([129, 20, 64], [40, 20, 0], 8, 2), ([300, 0, 140], [130, 0, 140], 4, 1),
    ([10, 70], [12, 70], 2, 2),  # more queries than context: the first see nothing
    ([700], [513], 2, 1),
]


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
    t = int(c["starts"][-1])
    for hint in ((max(new), max(ctx)), (1, 1100), (100, 1 << 20), (max(new), 1), None):
        most = hint or (t, c["table"].shape[1] * 16)
        size = max(K.kv_cache_attention_workspace_size(t, len(ctx), hq, hkv, 128, most[0], m) for m in (most[1], max(ctx) + 48))
        with stream_workspace(dev, size):
            check_attn(c, run_attn(dev, c, causal=causal, hint=hint), causal=causal)
        with stream_workspace(dev, 1024):  # too small: none is used
            check_attn(c, run_attn(dev, c, causal=causal, hint=hint), causal=causal)


@pytest.mark.parametrize("ctx,new", [(2000, 1), (2000, 7), (4500, 40)])
def test_attention_workspace_size(dev, ctx, new):
    """The size that is asked for is enough: the results are those of any larger workspace."""
    c = attn_case(np.random.default_rng(ctx + new), [ctx], [new], 8, 2, 64, 16)
    c["table"] = c["table"][:, :kv.pages_of(ctx, 16)]
    size = K.kv_cache_attention_workspace_size(new, 1, 8, 2, 64, new, 1 << 15)
    assert 0 < size < 32 << 20
    got = []
    for n, hint in ((K.kv_cache_attention_workspace_size(new, 1, 8, 2, 64, new, ctx), ctx), (size, 1 << 15), (64 << 20, 1 << 15)):
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


@pytest.mark.parametrize("new,batch", [(1, 150), (5, 150), (20, 150), (1, 300), (5, 300), (20, 300), (1, 4500)])
def test_attention_of_many_sequences(dev, new, batch):
    """More sequences than lanes: one, a few and many query rows, some sequences without any, with and without splits."""
    rng = np.random.default_rng(70 + new)
    lens = rng.integers(0, 200 if batch < 1000 else 30, batch)
    lens[[3, 77, batch - 1]] = 1500, 0, 2000
    c = attn_case(rng, [int(n) for n in lens], [int(n) for n in rng.integers(new == 1, new + 1, batch)], 8, 2, 64, 16)
    t, hint = int(c["starts"][-1]), (new, 2000)
    check_attn(c, run_attn(dev, c, hint=hint, pad=2))
    with stream_workspace(dev, K.kv_cache_attention_workspace_size(t + 2, batch, 8, 2, 64, *hint)):
        check_attn(c, run_attn(dev, c, hint=hint, pad=2))


@pytest.mark.parametrize("new", [1, 30])
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
    c = attn_case(rng, [90, 33], [3, 20], 4, 2, 64, 16)
    c["ks"][c["table"][0, 1]] = 0
    c["vs"][c["table"][0, 2]] = 0
    check_attn(c, run_attn(dev, c, scale=scale), scale=scale)


def test_attention_without_starts(dev):
    rng = np.random.default_rng(4)
    c = attn_case(rng, [90, 33, 0, 700], [1] * 4, 4, 2, 64, 64)
    check_attn(c, run_attn(dev, c, starts=False))


@pytest.mark.parametrize("new", [1, 20, 80])
def test_attention_unseen_pages(dev, new):
    """What a query does not see does not reach it: scales that hold NaN or infinities, page numbers that are none."""
    rng = np.random.default_rng(new)
    c = attn_case(rng, [200, 130], [new, new], 4, 2, 128, 16, extra=6)
    used = np.unique(c["table"][c["table"] >= 0])
    spare = np.setdiff1d(np.arange(c["kc"].shape[0]), used)
    c["ks"][spare], c["vs"][spare] = np.nan, np.inf
    c["table"][0, 13:] = spare[0]  # behind the context
    c["table"][0, 2], c["table"][0, 5], c["table"][1, 0], c["table"][1, 4] = -1, c["kc"].shape[0], 2 ** 31 - 1, -2 ** 31
    check_attn(c, run_attn(dev, c))
    if new > 1:  # the last page holds NaN: its own queries see it, the others do not
        c = attn_case(rng, [208], [new], 4, 2, 128, 16)
        page = c["table"][0, 12]
        c["ks"][page], c["vs"][page] = np.nan, np.nan
        o, lse = run_attn(dev, c)
        sees = 208 - new + np.arange(new) >= 192
        assert np.isnan(o[sees]).all() and np.isfinite(o[~sees]).all()
        ref, _, tol, _ = kv.attention(*[c[m] for m in ("q", "kc", "vc", "ks", "vs", "table", "ctx", "starts")], 1 / math.sqrt(128), True)
        assert (np.abs(o - ref)[~sees] <= tol[~sees]).all()


def test_attention_empty_tables(dev):
    """No page at all, and tables of unfilled rows."""
    rng = np.random.default_rng(6)
    c = attn_case(rng, [40, 40], [1, 1], 2, 2, 64, 16)
    c["table"][:] = -1
    o, lse = run_attn(dev, c)
    assert (o == 0).all() and np.isneginf(lse).all()
    q, out, ctx = dev.upload(to_bf16(c["q"]), bf16), dev.upload(to_bf16(np.ones_like(c["q"])), bf16), ints(dev, [4, 4])
    check(lib.teeny_kv_cache_attention(q.ptr, None, None, None, None, None, ctx.ptr, None, out.ptr, None, 2, 2, 2, 2,
                                       64, 0, 16, 0, 1, 40, 128, 0.1, 1, None))
    assert (from_bf16(out.to_host()) == 0).all()


def test_attention_query_stride(dev):
    rng = np.random.default_rng(8)
    c = attn_case(rng, [100, 31], [4, 1], 4, 2, 64, 16)
    t, hq, d = c["q"].shape
    wide = np.full((t, hq * d + 24), 7.0, np.float32)
    wide[:, 16:16 + hq * d] = c["q"].reshape(t, -1)
    qb, o, lse = dev.upload(to_bf16(wide), bf16), dev.buffer(bf16, c["q"].shape), dev.buffer("f32", (t, hq))
    cache = [dev.upload(c[n]) for n in ("kc", "vc", "ks", "vs", "table")] + [ints(dev, c["ctx"]), ints(dev, c["starts"])]
    check(lib.teeny_kv_cache_attention(qb.ptr + 32, *[b.ptr for b in cache], o.ptr, lse.ptr, t, 2, hq, 2, d, c["kc"].shape[0], 16, c["table"].shape[1], 4, 100,
                                       hq * d + 24, 1 / math.sqrt(d), 1, None))
    check_attn(c, (from_bf16(o.to_host()), lse.to_host()))


# ── together ────────────────────────────────────────────────────────────────


def test_steps_together(dev):
    """Prompts, then single tokens, on one cache: plan, write and attention as a server's step runs them, with
    requests that end and pages that are used again, against attention over the unquantized tokens."""
    rng = np.random.default_rng(11)
    hq, hkv, d, page, width, pages, batch = 8, 2, 64, 16, 12, 40, 4
    kc, vc = dev.buffer("i8", (pages, hkv, page, d)), dev.buffer("i8", (pages, hkv, d, page))
    ks, vs = dev.buffer("f32", (pages, hkv)), dev.buffer("f32", (pages, hkv))
    for b in (kc, vc):
        b.to_device(rng.integers(-128, 128, b.shape).astype(np.int8))
    for b in (ks, vs):
        b.to_device(np.full(b.shape, np.nan, np.float32))  # pages that were never begun
    seq, table = ints(dev, np.zeros(batch)), dev.upload(np.full((batch, width), -1, np.int32))
    stack, count = ints(dev, rng.permutation(pages)), ints(dev, [pages])
    said = [[] for _ in range(batch)]  # (k, v) of each request's tokens
    steps = [[50, 7, 0, 90], [1, 1, 33, 1], [1, 1, 1, -1], [1, -1, 1, 100]] + [[1, 20, 1, 1]] + [[1, 1, 1, 1]] * 20
    for new in steps:
        n = sum(max(x, 0) for x in new)
        k, v, q = (from_bf16(to_bf16(rng.standard_normal((n, h, d)).astype(np.float32))) for h in (hkv, hkv, hq))
        slots, _, starts, _, granted, _ = K.kv_cache_plan(ints(dev, new), seq, table, stack, count, page, n_tokens=n, context_lens=seq,
                                                          free_after=count)
        assert granted.to_host().tolist() == [max(x, 0) for x in new]
        K.kv_cache_write(dev.upload(to_bf16(k), bf16), dev.upload(to_bf16(v), bf16), slots, kc, vc, ks, vs)
        o = K.kv_cache_attention(dev.upload(to_bf16(q), bf16), kc, vc, ks, vs, table, seq, starts, max_q_len=max(new), max_context=160)
        at = 0
        got = from_bf16(o.to_host())
        codes = dict(q=q, kc=kc.to_host(), vc=vc.to_host(), ks=ks.to_host(), vs=vs.to_host(), table=table.to_host(),
                     ctx=seq.to_host(), starts=starts.to_host())
        ref, _, tol, _ = kv.attention(*[codes[m] for m in ("q", "kc", "vc", "ks", "vs", "table", "ctx", "starts")], 1 / math.sqrt(d), True)
        assert (np.abs(got - ref) <= tol).all()
        for b, x in enumerate(new):
            if x < 0:
                said[b] = []
            for i in range(max(x, 0)):
                said[b].append((k[at + i], v[at + i]))
            if said[b]:
                # what the cache stands for: a code is off by half a step, and by half a step of each later, larger
                # scale; the scales of a page grow by its running maximum, 16 times at most
                keys, vals = (np.stack([s[j] for s in said[b]]).astype(np.float64) for j in (0, 1))
                for t in range(len(keys)):
                    pg = codes["table"][b, t // page]
                    for x_, c_, s_ in ((keys, codes["kc"][pg, :, t % page], codes["ks"][pg]), (vals, codes["vc"][pg, :, :, t % page], codes["vs"][pg])):
                        assert (np.abs(c_ * s_[:, None].astype(np.float64) - x_[t]) <= 8.01 * s_[:, None]).all()
            at += max(x, 0)
        assert codes["ctx"].tolist() == [len(s) for s in said]


def test_step_in_a_graph(dev):
    """A step captured once and replayed while requests grow: every replay equals the eager step."""
    rng = np.random.default_rng(12)
    hq, hkv, d, page, width, batch = 8, 2, 128, 16, 40, 3
    lens = [30, 500, 15]
    table0, _, _ = make_table(rng, lens, page, width, extra=30)
    pages = sum(kv.pages_of(n, page) for n in lens) + 30
    spare = np.setdiff1d(np.arange(pages), table0[table0 >= 0])
    cache0 = [rng.integers(-127, 128, (pages, hkv, page, d)).astype(np.int8), rng.integers(-127, 128, (pages, hkv, d, page)).astype(np.int8),
              rng.uniform(0.01, 0.02, (pages, hkv)).astype(np.float32), rng.uniform(0.01, 0.02, (pages, hkv)).astype(np.float32)]

    def program(stream):
        b = {n: dev.upload(a) for n, a in zip(("kc", "vc", "ks", "vs"), cache0)}
        stack = np.zeros(pages, np.int32)
        stack[:len(spare)] = spare
        b.update(seq=ints(dev, lens), table=dev.upload(table0), stack=ints(dev, stack), count=ints(dev, [len(spare)]), new=ints(dev, [1] * batch),
                 **{n: dev.buffer(bf16, (batch, h, d)) for n, h in (("k", hkv), ("v", hkv), ("q", hq), ("o", hq))},
                 **{n: dev.buffer("i32", (s,)) for n, s in (("slots", batch), ("pos", batch), ("starts", batch + 1), ("granted", batch))})

        def step():
            K.kv_cache_plan(b["new"], b["seq"], b["table"], b["stack"], b["count"], page, slots=b["slots"], positions=b["pos"],
                            q_starts=b["starts"], context_lens=b["seq"], granted=b["granted"], free_after=b["count"], stream=stream)
            K.kv_cache_write(b["k"], b["v"], b["slots"], b["kc"], b["vc"], b["ks"], b["vs"], stream=stream)
            K.kv_cache_attention(b["q"], b["kc"], b["vc"], b["ks"], b["vs"], b["table"], b["seq"], b["starts"], max_q_len=1, o=b["o"],
                                 stream=stream)
        return b, step

    graphed, eager = Stream.create(), Stream.create()
    gb, gstep = program(graphed)
    eb, estep = program(eager)
    size = K.kv_cache_attention_workspace_size(batch, batch, hq, hkv, d, 1, width * page)
    with stream_workspace(dev, size, graphed), stream_workspace(dev, size, eager):
        graphed.begin_capture()
        gstep()
        graph = graphed.end_capture()
        for i in range(20):
            for n, h in (("k", hkv), ("v", hkv), ("q", hq)):
                x = to_bf16(rng.standard_normal((batch, h, d)).astype(np.float32))
                gb[n].to_device(x)
                eb[n].to_device(x)
            dev.synchronize()
            graph.launch(graphed)
            estep()
            graphed.synchronize()
            eager.synchronize()
            for n in ("o", "kc", "vc", "ks", "vs", "table", "seq", "count", "slots"):
                np.testing.assert_array_equal(gb[n].to_host(), eb[n].to_host(), err_msg=f"{n}, replay {i}")
        assert gb["seq"].to_host().tolist() == [n + 20 for n in lens]
        graph.destroy()


def test_two_streams(dev):
    """Calls on two streams at once, each with its own workspace: split attention, shared tiles and few rows."""
    rng = np.random.default_rng(14)
    streams = [Stream.create(), Stream.create()]
    jobs = []
    for i, (ctx, new) in enumerate([([3000, 40, 700], [1, 1, 1]), ([1500, 300], [60, 90]), ([900, 2100], [9, 5]), ([2500], [1])]):
        c = attn_case(rng, ctx, new, 8, 2, 128, 16)
        bufs = [dev.upload(to_bf16(c["q"]), bf16)] + [dev.upload(c[n]) for n in ("kc", "vc", "ks", "vs", "table")]
        bufs += [ints(dev, c["ctx"]), ints(dev, c["starts"])]
        t = c["q"].shape[0]
        jobs.append((c, streams[i % 2], bufs, (max(new), max(ctx)), dev.buffer(bf16, c["q"].shape), dev.buffer("f32", (t, 8)),
                     K.kv_cache_attention_workspace_size(t, len(ctx), 8, 2, 128, max(new), max(ctx))))
    dev.synchronize()
    most = max(j[-1] for j in jobs)
    with stream_workspace(dev, most, streams[0]), stream_workspace(dev, most, streams[1]):
        for _ in range(5):
            for c, s, bufs, hint, o, lse, _ in jobs:
                K.kv_cache_attention(*bufs, *hint, o=o, lse=lse, stream=s)
        for s in streams:
            s.synchronize()
        for c, s, bufs, hint, o, lse, _ in jobs:
            check_attn(c, (from_bf16(o.to_host()), lse.to_host()))


def test_large_cache(dev):
    """Pages whose bytes lie past 2^32: the same tokens at the pool's start and end."""
    rng = np.random.default_rng(13)
    hkv, d, page, pages = 8, 128, 128, 36000  # 4.7 GB each for K and V
    kc, vc = dev.buffer("i8", (pages, hkv, page, d)), dev.buffer("i8", (pages, hkv, d, page))
    ks, vs = dev.buffer("f32", (pages, hkv)), dev.buffer("f32", (pages, hkv))
    n = 150
    k, v = (dev.upload(to_bf16(rng.standard_normal((n, hkv, d)).astype(np.float32)), bf16) for _ in range(2))
    q = dev.upload(to_bf16(rng.standard_normal((2, 16, d)).astype(np.float32)), bf16)
    outs = []
    for table in ([[0, 1]], [[pages - 2, pages - 1]]):
        slots = np.array([table[0][t // page] * page + t % page for t in range(n)], np.int32)
        K.kv_cache_write(k, v, ints(dev, slots), kc, vc, ks, vs)
        outs.append(K.kv_cache_attention(q, kc, vc, ks, vs, ints(dev, np.array(table)), ints(dev, [n]), ints(dev, [0, 2])).to_host())
    np.testing.assert_array_equal(outs[0], outs[1])
    assert np.isfinite(from_bf16(outs[0])).all() and from_bf16(outs[0]).any()
    for b in (kc, vc):
        b.free()


def test_attention_of_the_largest_launch(dev):
    """Short sequences of many heads under a very large max_context, with the workspace that it asks for (35 GB): as
    many parts as a launch takes, nearly all of them empty."""
    rng = np.random.default_rng(15)
    batch, heads, d, most = 1024, 64, 64, 1 << 19
    c = attn_case(rng, [int(n) for n in rng.integers(0, 40, batch)], [1] * batch, heads, heads, d, 16)
    c["table"] = np.pad(c["table"], ((0, 0), (0, most // 16 - c["table"].shape[1])), constant_values=-1)
    c["ctx"][7], c["table"][7, [300, 700, 1023]] = 1 << 14, [0, 1, 2]  # a few pages, far apart
    size = K.kv_cache_attention_workspace_size(batch, batch, heads, heads, d, 1, most)
    assert size > 1 << 35
    with stream_workspace(dev, size):
        check_attn(c, run_attn(dev, c, hint=(1, most)))


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d", [64, 128])
def test_write_over_refused_tokens(dev, page, d):
    """Drafts are written, some are refused, and others take their slots: what is before them takes the page's scale,
    what is behind them keeps its codes, and attention over the tokens that count reads none of it."""
    rng = np.random.default_rng(page + d)
    heads, slots = 2, np.arange(page, 2 * page - 2, dtype=np.int32)  # the second page, but for two slots
    cache = [np.zeros((2, heads, page, d), np.int8), np.zeros((2, heads, d, page), np.int8)] + [np.zeros((2, heads), np.float32)] * 2

    def tokens(n, most):
        return {m: from_bf16(to_bf16((most * rng.uniform(-1, 1, (n, heads, d))).astype(np.float32))) for m in "kv"}

    first, second = tokens(len(slots), 1.0), tokens(3, 9.0)
    cache = check_write(dev, first, slots, *cache)
    after = check_write(dev, second, slots[5:8], *cache)
    assert (after[2][1] > 5 * cache[2][1]).all()  # a larger scale
    np.testing.assert_array_equal(after[0][1, :, 8:], cache[0][1, :, 8:])
    np.testing.assert_array_equal(after[1][1, :, :, 8:], cache[1][1, :, :, 8:])
    for codes, scale, name in ((after[0][1], after[2][1], "k"), (after[1][1].transpose(0, 2, 1), after[3][1], "v")):
        want = np.concatenate([first[name][:5], second[name]]).transpose(1, 0, 2)
        # half a step of the old scale, at most a fifth of the new one, and half of the new one
        assert (np.abs(codes[:, :8] * scale[:, None, None] - want) <= 0.61 * scale[:, None, None]).all()
    c = dict(q=from_bf16(to_bf16(rng.standard_normal((1, heads, d)).astype(np.float32))), kc=after[0], vc=after[1], ks=after[2], vs=after[3],
             table=np.array([[1]], np.int32), ctx=np.array([8], np.int32), starts=np.array([0, 1], np.int32))
    check_attn(c, run_attn(dev, c, hint=(1, page)))


def test_plan_after_refused_tokens(dev):
    """Five drafts a step, some taken back: within a page nothing else is to do, pages past the new end go back on the
    stack, and over many steps none is lost or held twice."""
    rng = np.random.default_rng(16)
    batch, page, width, pages = 6, 16, 20, 100
    table, stack, count, seq = np.full((batch, width), -1, np.int32), rng.permutation(pages).astype(np.int32), pages, np.zeros(batch, np.int32)
    for step in range(60):
        new = np.where(seq > 250, -1, np.where(seq == 0, rng.integers(1, 40, batch), 5)).astype(np.int32)
        bufs = [ints(dev, new), ints(dev, seq), dev.upload(table), ints(dev, stack), ints(dev, [count])]
        slots, _, starts, context, granted, left = [b.to_host() for b in K.kv_cache_plan(*bufs, page, n_tokens=int(new.clip(0).sum()))]
        ref, table, stack = kv.plan(new, seq, table, stack, count, page, len(slots))
        np.testing.assert_array_equal(granted, new.clip(0))
        for name, got in (("slots", slots), ("context_lens", context), ("free_after", left)):
            np.testing.assert_array_equal(got, ref[name], err_msg=name)
        np.testing.assert_array_equal(bufs[2].to_host(), table)
        seq, count = context, int(left[0])
        back = np.where(new == 5, rng.integers(0, 6, batch), 0)
        for b in range(batch):
            for i in range(kv.pages_of(seq[b] - back[b], page), kv.pages_of(seq[b], page)):
                stack[count] = table[b, i]
                count += 1
        seq = (seq - back).astype(np.int32)
        held = [table[b, i] for b in range(batch) for i in range(kv.pages_of(seq[b], page))]
        assert sorted(held + stack[:count].tolist()) == list(range(pages))
    assert step == 59 and (seq > 0).any()


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("growth", ["none", "slow", "twice"])
def test_write_rounds_at_every_growth(dev, page, growth):
    """A page filled token by token.  A code is rounded when it is written and whenever its page's scale grows: a token is
    off by at most half the sum of the scales that its page has had since."""
    rng = np.random.default_rng(page)
    heads, d = 2, 64
    bufs = [dev.upload(a) for a in (np.zeros((1, heads, page, d), np.int8), np.zeros((1, heads, d, page), np.int8),
                                    np.zeros((1, heads), np.float32), np.zeros((1, heads), np.float32))]
    said = {n: np.zeros((heads, page, d)) for n in "kv"}
    since = {n: np.zeros((heads, page)) for n in "kv"}  # the sum of the scales since the token was written
    last = {n: np.zeros(heads) for n in "kv"}
    for t in range(page):
        most = 2.0 ** (t % 100 - 50) if growth == "twice" else 1.004 ** t if growth == "slow" else 1.0
        x = {n: from_bf16(to_bf16((most * np.sign(rng.uniform(-1, 1, (1, heads, d))) * (rng.uniform(0, 1, (1, heads, d)) if growth == "none" else 1))
                                  .astype(np.float32))) for n in "kv"}
        K.kv_cache_write(dev.upload(to_bf16(x["k"]), bf16), dev.upload(to_bf16(x["v"]), bf16), ints(dev, [t]), *bufs)
        kc, vc, ks, vs = [b.to_host()[0].astype(np.float64) for b in bufs]
        for n, codes, scale in (("k", kc, ks), ("v", vc.transpose(0, 2, 1), vs)):
            said[n][:, t] = x[n][0]
            grown = scale > last[n]
            since[n][:, :t] += np.where(grown, scale, 0)[:, None]
            since[n][:, t] = scale
            last[n] = scale
            # (codes are at most 127: their fp32 quotients and ratios are off by less than 2^-15)
            off = np.abs(codes[:, :t + 1] * scale[:, None, None] - said[n][:, :t + 1])
            assert (off <= ((0.5 + 2.0 ** -15) * since[n][:, :t + 1])[..., None]).all()


@pytest.mark.parametrize("batch,ended", [(40, 36), (256, 200), (400, 390)])
def test_plan_of_many_endings(dev, batch, ended):
    """A step of few tokens in which nearly all requests end, with long rows: their pages in request and row order."""
    rng = np.random.default_rng(batch)
    page, width = 16, 120
    seq = rng.integers(60 * page, width * page - 1, batch).astype(np.int32)
    new = np.ones(batch, np.int32)
    new[rng.permutation(batch)[:ended]] = -1
    table, pages, spare = make_table(rng, seq, page, width, extra=3)
    stack = np.zeros(pages, np.int32)
    stack[:len(spare)] = spare
    tokens = batch - ended
    ref, ref_table, ref_stack = kv.plan(new, seq, table, stack, len(spare), page, tokens)
    for in_place in (False, True):
        bufs = [ints(dev, new), ints(dev, seq), dev.upload(table), ints(dev, stack), ints(dev, [len(spare)])]
        over = dict(context_lens=bufs[1], granted=bufs[0], free_after=bufs[4]) if in_place else {}
        out = dict(zip(NAMES, K.kv_cache_plan(*bufs, page, n_tokens=tokens, **over)))
        for n in NAMES:
            np.testing.assert_array_equal(out[n].to_host(), ref[n], err_msg=n)
        np.testing.assert_array_equal(bufs[2].to_host(), ref_table)
        left = int(ref["free_after"][0])
        np.testing.assert_array_equal(bufs[3].to_host()[:left], ref_stack[:left])


def test_attention_of_a_mixed_step(dev):
    """Prompts and single tokens: in one call under either hint, and in a call each over its part of the sequences and the
    whole of q and o."""
    rng = np.random.default_rng(17)
    ctx, new = [900, 260, 30, 1200, 77, 0, 515, 64, 700], [300, 130, 1, 1, 1, 1, 1, 1, 1]
    hq, hkv, d, page = 8, 2, 128, 16
    c = attn_case(rng, ctx, new, hq, hkv, d, page)
    t, b = int(c["starts"][-1]), len(ctx)
    size = max(K.kv_cache_attention_workspace_size(t, b, hq, hkv, d, n, 1200) for n in (300, 48, 1))
    for hint in ((300, 1200), (1, 1200), None):
        with stream_workspace(dev, size):
            check_attn(c, run_attn(dev, c, hint=hint, pad=2))
    bufs = [dev.upload(to_bf16(c["q"]), bf16)] + [dev.upload(c[n]) for n in ("kc", "vc", "ks", "vs", "table")]
    lens, starts = ints(dev, c["ctx"]), ints(dev, c["starts"])
    o, lse = dev.upload(to_bf16(np.full(c["q"].shape, 123.0, np.float32)), bf16), dev.upload(np.full((t, hq), 55.0, np.float32))
    width = c["table"].shape[1]
    with stream_workspace(dev, size):
        for first, n, longest in ((0, 2, 300), (2, b - 2, 1)):
            check(lib.teeny_kv_cache_attention(*[x.ptr for x in bufs[:5]], bufs[5].ptr + 4 * width * first, lens.ptr + 4 * first,
                                               starts.ptr + 4 * first, o.ptr, lse.ptr, t, n, hq, hkv, d, c["kc"].shape[0], page, width, longest,
                                               1200, hq * d, 1 / math.sqrt(d), 1, None))
            got = from_bf16(o.to_host())
            if first == 0:
                assert (got[430:] == 123.0).all() and (got[:430] != 123.0).any()
    check_attn(c, (got, lse.to_host()))


@pytest.mark.parametrize("ctx,new,hq,hkv", [([4500], 1, 8, 2), ([3000, 700], 7, 8, 2), ([9000, 60], 40, 4, 2)])
@pytest.mark.parametrize("part", [0.9, 0.4])
def test_attention_in_part_of_its_workspace(dev, ctx, new, hq, hkv, part):
    """A workspace that does not hold all the parts that were planned holds fewer; nothing outside of it is written."""
    c = attn_case(np.random.default_rng(ctx[0]), ctx, [new] * len(ctx), hq, hkv, 64, 16)
    c["table"] = c["table"][:, :kv.pages_of(ctx[0], 16)]
    size = K.kv_cache_attention_workspace_size(new * len(ctx), len(ctx), hq, hkv, 64, new, ctx[0])
    assert size > 0
    small = int(size * part) // 256 * 256
    ws = dev.upload(np.full(size, 77, np.int8))
    check(lib.teeny_hip_stream_set_workspace(None, ws.ptr, small))
    try:
        got = run_attn(dev, c, hint=(new, ctx[0]))
    finally:
        NULL_STREAM.set_workspace(None)
    held = ws.to_host()
    assert (held[:small] != 77).any() and (held[small:] == 77).all()
    check_attn(c, got)
