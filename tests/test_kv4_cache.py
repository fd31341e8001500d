"""The 4-bit cache's operators and the low-rank adapters without a GPU: refusals, shape rules, and the layout."""
import ctypes

import numpy as np
import pytest

import kv4_cases as kv4
from teenygrad_amd import _lib
from teenygrad_amd import kernels as K
from teenygrad_amd._lib import lib

FAKE, FAKE_ODD = 0x100000, 0x100002
BIG = 1 << 31


def expect(status, code):
    assert status == code, (status, code, _lib.last_error())
    assert _lib.last_error() != ""


def append_args(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, positions=FAKE, slots=FAKE, inv_freq=FAKE, q_out=FAKE, k_cache=FAKE, v_cache=FAKE, k_scale=FAKE,
             v_scale=FAKE, n_tokens=4, q_heads=8, kv_heads=2, head_dim=128, rotary_dim=128, num_pages=8, page_size=16, q_stride=1024,
             k_stride=256, v_stride=256, interleaved=0)
    assert set(kw) <= set(a)
    return [*{**a, **kw}.values(), None]


@pytest.mark.parametrize("kw,code", [
    *[(dict([(n, -1)]), _lib.ERR_SHAPE_MISMATCH) for n in ("n_tokens", "q_heads", "kv_heads", "num_pages", "rotary_dim")],
    (dict(head_dim=96), _lib.ERR_UNSUPPORTED), (dict(head_dim=0), _lib.ERR_UNSUPPORTED), (dict(head_dim=256), _lib.ERR_UNSUPPORTED),
    (dict(page_size=8), _lib.ERR_UNSUPPORTED), (dict(page_size=256), _lib.ERR_UNSUPPORTED),
    (dict(rotary_dim=144), _lib.ERR_UNSUPPORTED), (dict(rotary_dim=24), _lib.ERR_UNSUPPORTED), (dict(rotary_dim=8), _lib.ERR_UNSUPPORTED),
    (dict(num_pages=BIG // 16), _lib.ERR_SHAPE_MISMATCH), (dict(n_tokens=(1 << 24) + 1), _lib.ERR_SHAPE_MISMATCH),
    (dict(q_heads=65536, q_stride=1 << 24), _lib.ERR_SHAPE_MISMATCH), (dict(kv_heads=65536, k_stride=1 << 24, v_stride=1 << 24), _lib.ERR_SHAPE_MISMATCH),
    (dict(n_tokens=1 << 24, kv_heads=128, k_stride=1 << 14, v_stride=1 << 14), _lib.ERR_SHAPE_MISMATCH),  # more workgroups than a launch has
    (dict(q_stride=1016), _lib.ERR_SHAPE_MISMATCH), (dict(k_stride=248), _lib.ERR_SHAPE_MISMATCH), (dict(v_stride=0), _lib.ERR_SHAPE_MISMATCH),
    (dict(q_stride=1028), _lib.ERR_MISALIGNED), (dict(k_stride=260), _lib.ERR_MISALIGNED), (dict(v_stride=257), _lib.ERR_MISALIGNED),
    *[(dict([(n, FAKE_ODD)]), _lib.ERR_MISALIGNED) for n in ("q", "k", "v", "q_out", "k_cache", "v_cache")],
    (dict(q_stride=2048), _lib.ERR_INVALID_ARGUMENT),  # q_out is q, whose rows are not dense
    *[(dict([(n, None)]), _lib.ERR_NULL_POINTER) for n in (
        "q", "k", "v", "positions", "slots", "inv_freq", "q_out", "k_cache", "v_cache", "k_scale", "v_scale")]])
def test_append_refusals(kw, code):
    expect(lib.teeny_kv4_cache_append(*append_args(**kw)), code)


@pytest.mark.parametrize("tokens,kv_heads", [(1024, 65535), (961, 65535), (4000, 65535), (1 << 20, 247), (1 << 24, 7), (513, 65535), (1, 65535)])
def test_append_within_the_limit(tokens, kv_heads):
    """Calls within the documented limit are not refused for their size: the one thing that is wrong with these, and found
    later, is the cache's address."""
    assert tokens / 4 + tokens / 32 * kv_heads < 1 << 23
    row = kv_heads * 64
    a = dict(n_tokens=tokens, kv_heads=kv_heads, head_dim=64, rotary_dim=64, k_stride=row, v_stride=row, v_cache=FAKE_ODD)
    expect(lib.teeny_kv4_cache_append(*append_args(**a)), _lib.ERR_MISALIGNED)
    a.update(n_tokens=1 << 24, kv_heads=65535, k_stride=1 << 23, v_stride=1 << 23)
    expect(lib.teeny_kv4_cache_append(*append_args(**a)), _lib.ERR_SHAPE_MISMATCH)


def test_nothing_to_append():
    none = dict(q=None, k=None, v=None, positions=None, slots=None, inv_freq=None, q_out=None)
    assert lib.teeny_kv4_cache_append(*append_args(n_tokens=0, **none)) == _lib.OK
    assert lib.teeny_kv4_cache_append(*append_args(q_heads=0, kv_heads=0, **none)) == _lib.OK
    assert lib.teeny_kv4_cache_append(*append_args(q_heads=0, num_pages=0, k_cache=None, v_cache=None, **none)) == _lib.OK


def attn_args(**kw):
    a = dict(q=FAKE, k_cache=FAKE, v_cache=FAKE, k_scale=FAKE, v_scale=FAKE, block_table=FAKE, context_lens=FAKE,
             q_starts=FAKE, o=FAKE, l=None, n_tokens=4, batch=4, q_heads=8, kv_heads=2, head_dim=128, num_pages=32,
             page_size=16, max_pages=8, max_q_len=1, max_context=128, q_stride=1024, scale=0.1, causal=1)
    assert set(kw) <= set(a)
    return [*{**a, **kw}.values(), None]


@pytest.mark.parametrize("kw,code", [
    *[(dict([(n, -1)]), _lib.ERR_SHAPE_MISMATCH) for n in (
        "n_tokens", "batch", "q_heads", "kv_heads", "num_pages", "max_pages", "max_q_len", "max_context")],
    (dict(head_dim=32), _lib.ERR_UNSUPPORTED), (dict(head_dim=256), _lib.ERR_UNSUPPORTED),
    (dict(page_size=48), _lib.ERR_UNSUPPORTED), (dict(kv_heads=3), _lib.ERR_SHAPE_MISMATCH),
    (dict(kv_heads=0), _lib.ERR_SHAPE_MISMATCH), (dict(q_starts=None, n_tokens=5), _lib.ERR_SHAPE_MISMATCH),
    (dict(q_stride=1000), _lib.ERR_SHAPE_MISMATCH), (dict(q_stride=1025), _lib.ERR_MISALIGNED),
    *[(dict([(n, FAKE_ODD)]), _lib.ERR_MISALIGNED) for n in ("q", "o", "k_cache", "v_cache", "k_scale", "v_scale")],
    (dict(n_tokens=BIG), _lib.ERR_SHAPE_MISMATCH), (dict(n_tokens=1 << 29), _lib.ERR_SHAPE_MISMATCH),
    (dict(max_context=BIG), _lib.ERR_SHAPE_MISMATCH), (dict(max_pages=BIG // 16), _lib.ERR_SHAPE_MISMATCH),
    (dict(num_pages=1 << 26, kv_heads=8), _lib.ERR_SHAPE_MISMATCH),
    *[(dict([(n, None)]), _lib.ERR_NULL_POINTER) for n in (
        "q", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "context_lens", "o")]])
def test_attention_refusals(kw, code):
    expect(lib.teeny_kv4_cache_attention(*attn_args(**kw)), code)


def test_attention_without_queries():
    assert lib.teeny_kv4_cache_attention(*attn_args(n_tokens=0, q=None, o=None)) == _lib.OK
    assert lib.teeny_kv4_cache_attention(*attn_args(batch=0, context_lens=None, block_table=None)) == _lib.OK


def test_attention_workspace_refusals():
    n = ctypes.c_size_t(7)
    f = lib.teeny_kv4_cache_attention_workspace_size
    expect(f(4, 4, 8, 2, 128, 1, 128, None), _lib.ERR_NULL_POINTER)
    expect(f(4, 4, 8, 3, 128, 1, 128, ctypes.byref(n)), _lib.ERR_SHAPE_MISMATCH)
    expect(f(4, 4, 8, 2, 80, 1, 128, ctypes.byref(n)), _lib.ERR_UNSUPPORTED)
    expect(f(-4, 4, 8, 2, 128, 1, 128, ctypes.byref(n)), _lib.ERR_SHAPE_MISMATCH)
    assert n.value == 0
    assert f(0, 4, 8, 2, 128, 1, 128, ctypes.byref(n)) == _lib.OK and n.value == 0
    sizes = []
    for longest in (40, 1 << 40, (1 << 63) - 1):  # no sequence has more queries than there are rows
        assert f(40, 2, 8, 2, 128, longest, 9000, ctypes.byref(n)) == _lib.OK
        sizes.append(n.value)
    assert sizes[0] > 0 and len(set(sizes)) == 1


@pytest.mark.parametrize("batch,hq,hkv,d,longest,context", [(4096, 8, 8, 64, 1, 1 << 20), (2000, 32, 32, 128, 1, (1 << 31) - 5000),
                                                            (3000, 16, 4, 64, 4, 1 << 26), (1, 8, 2, 128, 1, 1 << 30)])
def test_attention_splits_fit_a_launch(batch, hq, hkv, d, longest, context):
    tokens, rows = batch * longest, hq // hkv * longest
    block = 128 if rows > 64 else 32 if rows > 16 else 16
    units = (tokens * (hq // hkv) // block + batch) * hkv
    assert units * block < 1 << 25, "within the documented limit of rows"
    n = ctypes.c_size_t(0)
    assert lib.teeny_kv4_cache_attention_workspace_size(tokens, batch, hq, hkv, d, longest, context, ctypes.byref(n)) == _lib.OK
    splits = n.value // (units * block * (d + 2) * 4)
    assert splits > 1 and units * splits < (1 << 31) // 256


@pytest.mark.parametrize("tokens,batch,hq,hkv,d,longest,context", [
    ((1 << 22) - 1000, 1, 8, 1, 128, 10, 1 << 30), ((1 << 20) - 1000, 1, 32, 2, 64, 8, 1 << 28), (1 << 19, 2, 32, 1, 64, 3, 1 << 29)])
def test_attention_splits_of_tiles_fit_a_launch(tokens, batch, hq, hkv, d, longest, context):
    """Many more rows than the hint stands for: as many splits as a launch of 512 threads a workgroup holds."""
    assert hq // hkv * longest > 64, "shared tiles, of 256 rows"
    units = (tokens * (hq // hkv) // 256 + batch) * hkv
    n = ctypes.c_size_t(0)
    assert lib.teeny_kv4_cache_attention_workspace_size(tokens, batch, hq, hkv, d, longest, context, ctypes.byref(n)) == _lib.OK
    splits = n.value // (units * 256 * (d + 2) * 4)
    assert n.value == splits * units * 256 * (d + 2) * 4
    most = ((1 << 31) // 512 - 1) // units
    assert 1 < splits <= most
    assert splits == most, "the launch is what bounds it"


LIMIT = 1 << 25  # of n_tokens * q_heads + 128 * batch * kv_heads


@pytest.mark.parametrize("tokens,batch,hq,hkv,longest", [
    (5000, 5000, 32, 32, 100), (LIMIT // 8 - 200, 1, 8, 1, 100), (LIMIT // 32 // 129 - 1, LIMIT // 32 // 129 - 1, 32, 32, 65),
    (LIMIT // 136 - 1, LIMIT // 136 - 1, 8, 1, 1), (LIMIT // 160 - 1, LIMIT // 160 - 1, 32, 1, 1)])
def test_attention_rows_within_the_limit(tokens, batch, hq, hkv, longest):
    """Calls within the documented limit are not refused for their rows, whichever form they take: the one thing that is wrong
    with these, and found later, are their scales' addresses.  32 times the rows are refused."""
    assert tokens * hq + 128 * batch * hkv < LIMIT
    a = dict(n_tokens=tokens, batch=batch, q_heads=hq, kv_heads=hkv, max_q_len=longest, q_stride=hq * 128, k_scale=FAKE_ODD)
    expect(lib.teeny_kv4_cache_attention(*attn_args(**a)), _lib.ERR_MISALIGNED)
    a.update(n_tokens=32 * tokens, batch=32 * batch if batch > 1 else 1)
    expect(lib.teeny_kv4_cache_attention(*attn_args(**a)), _lib.ERR_SHAPE_MISMATCH)


def adapter_args(**kw):
    a = dict(x=FAKE, a=FAKE, b=FAKE, adapters=FAKE, scale=None, y=FAKE, out=2 * FAKE, M=4, N=100, K=64, rank=16, num_adapters=3, x_stride=64,
             y_stride=100, out_stride=100)
    assert set(kw) <= set(a)
    return [*{**a, **kw}.values(), None]


@pytest.mark.parametrize("kw,code", [
    *[(dict([(n, -1)]), _lib.ERR_SHAPE_MISMATCH) for n in ("M", "N", "K", "rank", "num_adapters")],
    (dict(M=(1 << 24) + 1), _lib.ERR_SHAPE_MISMATCH), (dict(N=(1 << 24) + 1, y_stride=1 << 25, out_stride=1 << 25), _lib.ERR_SHAPE_MISMATCH),
    (dict(K=1 << 25, x_stride=1 << 25), _lib.ERR_SHAPE_MISMATCH), (dict(num_adapters=BIG), _lib.ERR_SHAPE_MISMATCH),
    (dict(K=60), _lib.ERR_SHAPE_MISMATCH), (dict(rank=12), _lib.ERR_UNSUPPORTED), (dict(rank=136), _lib.ERR_UNSUPPORTED),
    (dict(x_stride=(1 << 24) + 8), _lib.ERR_SHAPE_MISMATCH), (dict(x_stride=56), _lib.ERR_SHAPE_MISMATCH), (dict(y_stride=99), _lib.ERR_SHAPE_MISMATCH), (dict(out_stride=99), _lib.ERR_SHAPE_MISMATCH),
    (dict(x_stride=68), _lib.ERR_MISALIGNED), *[(dict([(n, FAKE_ODD)]), _lib.ERR_MISALIGNED) for n in "xab"],
    (dict(out=FAKE, out_stride=108), _lib.ERR_INVALID_ARGUMENT),
    *[(dict([(n, None)]), _lib.ERR_NULL_POINTER) for n in ("x", "a", "b", "adapters", "y", "out")]])
def test_adapter_refusals(kw, code):
    expect(lib.teeny_adapter_add(*adapter_args(**kw)), code)


def test_adapter_workspace_refusals():
    n = ctypes.c_size_t(7)
    f = lib.teeny_adapter_add_workspace_size
    expect(f(4, 32, 256, 16, None), _lib.ERR_NULL_POINTER)
    expect(f(-4, 32, 256, 16, ctypes.byref(n)), _lib.ERR_SHAPE_MISMATCH)
    expect(f(4, 32, 256, 20, ctypes.byref(n)), _lib.ERR_UNSUPPORTED)
    expect(f(4, 32, BIG, 16, ctypes.byref(n)), _lib.ERR_SHAPE_MISMATCH)
    assert n.value == 0
    assert f(4, 32, 0, 16, ctypes.byref(n)) == _lib.OK and n.value == 0
    assert f(4, 32, 256, 16, ctypes.byref(n)) == _lib.OK and n.value == 0  # one launch
    assert f(4, 32, 2048, 16, ctypes.byref(n)) == _lib.OK and n.value > 0


def test_nothing_to_adapt():
    assert lib.teeny_adapter_add(*adapter_args(M=0, x=None, y=None, out=None, adapters=None)) == _lib.OK
    assert lib.teeny_adapter_add(*adapter_args(N=0, b=None)) == _lib.OK


def test_shape_rules():
    good = [(9, 2, 32, 64), (9, 2, 2, 128, 8), (9, 2, 32, 2), (9, 2, 32, 2)]
    assert K.kv4_cache_dims(*good) == (9, 2, 32, 128)
    assert K.kv4_cache_dims((9, 2, 16, 32), (9, 2, 1, 64, 8), (9, 2, 16, 1), (9, 2, 16, 1)) == (9, 2, 16, 64)
    for i, bad in ((0, (9, 2, 32, 60)), (0, (9, 2, 40, 64)), (0, (9, 2, 2048)), (1, (9, 2, 2, 128, 16)), (1, (9, 2, 128, 2, 8)), (2, (9, 2, 32)),
                   (3, (9, 2, 32, 1)), (3, (9, 2, 64))):
        with pytest.raises(ValueError):
            K.kv4_cache_dims(*[bad if j == i else s for j, s in enumerate(good)])
    good = [(5, 64), (3, 16, 64), (3, 100, 16), 5, (5, 100), (3,)]
    assert K.adapter_dims(*good) == (5, 100, 64, 16, 3)
    for i, bad in ((0, (5, 72)), (0, (320,)), (1, (3, 8, 64)), (1, (2, 16, 64)), (2, (3, 16, 100)), (3, 4), (4, (5, 104)), (4, (4, 100)), (5, (2,))):
        with pytest.raises(ValueError):
            K.adapter_dims(*[bad if j == i else s for j, s in enumerate(good)])


def test_layout():
    """The words that single codes lie in."""
    for d, n, word, nibble in ((64, 0, 0, 0), (64, 9, 1, 4), (64, 63, 7, 7), (128, 17, 4, 4), (128, 64, 2, 0), (128, 64 + 16 + 10, 7, 1),
                               (128, 127, 15, 7)):
        zero = [np.zeros((1, 1, 16, d // 2), np.int8), np.zeros((1, 1, 1, d, 8), np.int8), *[np.zeros((1, 1, 16, d // 64), np.float32)] * 2]
        k = np.zeros((1, 1, d), np.float32)
        k[0, 0, n] = 4.0  # the largest: code -8, held as 0
        kc, vc, ks, vs = kv4.append(k, k, [11], zero)
        words = kc.view(np.uint32)[0, 0, 11]
        assert words[word] == 0x88888888 - (8 << (4 * nibble)) and (np.delete(words, word) == 0x88888888).all()
        assert (kc[0, 0, np.arange(16) != 11] == 0).all()
        words = vc.view(np.uint32)[0, 0, 0]  # token 11 of 16: word 1, code 3, nibble 5
        assert words[n].tolist() == [0, 0] and (np.delete(words, n, 0) == [0, 8 << 20]).all()
        assert ks[0, 0, 11, n // 64] == vs[0, 0, 11, n // 64] == -0.5 and np.count_nonzero(ks) == 1
        kq, vq = kv4.codes_of(kc, vc)
        assert kq[0, 0, 11, n] == vq[0, 0, 11, n] == -8 and np.count_nonzero(kq[0, 0, 11]) == 1


def test_quantize_oracle():
    """Scales by hand: a tie between signs goes to the positive number, five bits to nearest even, small groups are zero."""
    x = np.zeros((6, 64), np.float32)
    x[0, :2] = 8, -8
    x[1, :2] = -8, 7.5
    x[2, 0] = 8 * (1 + 1 / 32)     # half-way between 16 and 17 sixteenths: the even one
    x[3, 0] = 8 * (1 + 3 / 32)     # half-way between 17 and 18
    x[4, 0] = 2.0 ** -91
    x[5, 5] = np.inf
    codes, scale = kv4.quantize(x)
    assert scale[:5, 0].tolist() == [-1, 1, -1, -1.125, 0] and np.isnan(scale[5, 0])
    assert codes[0, :2].tolist() == [-8, 7] and codes[1, :2].tolist() == [-8, 7] and codes[2, 0] == -8 and (codes[4:] == 0).all()


def test_quantize_bound():
    """Half a step, or 1.25 of them for numbers of the other sign; and a code times its scale is a bf16 number."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((4000, 64)).astype(np.float32) * np.exp(rng.uniform(-30, 30, (4000, 1))).astype(np.float32)
    codes, scale = kv4.quantize(x)
    value = codes.astype(np.float64) * scale
    off = np.abs(value - x) / np.abs(scale)
    q = x / scale
    assert (off[q <= 7.5] <= 0.5 + 2.0 ** -20).all() and (off <= 1.25 + 2.0 ** -20).all()
    assert (value.astype(np.float32).view(np.uint32) & 0xFFFF == 0).all() and (value == value.astype(np.float32)).all()
    assert 0.09 < np.sqrt(np.mean((off * np.abs(scale) / x.std(-1, keepdims=True)) ** 2)) < 0.1
