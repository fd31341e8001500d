"""The 8-bit cache's operators and the 4-bit linear layer without a GPU: refusals, and the packed layout."""
import ctypes

import numpy as np
import pytest

import kv_cases as kv
from teenygrad_amd import _lib
from teenygrad_amd import kernels as K
from teenygrad_amd._lib import lib

FAKE, FAKE_ODD = 0x100000, 0x100002
BIG = 1 << 31


def expect(status, code):
    assert status == code, (status, code, _lib.last_error())
    assert _lib.last_error() != ""


def plan_args(**kw):
    a = dict(new_lens=FAKE, seq_lens=FAKE, block_table=FAKE, free_list=FAKE, free_count=FAKE, q_starts=FAKE, slots=FAKE,
             positions=FAKE, context_lens=FAKE, granted=FAKE, free_after=FAKE, batch=4, max_pages=8, num_pages=32,
             page_size=16, n_tokens=64)
    assert set(kw) <= set(a)
    return [*{**a, **kw}.values(), None]


@pytest.mark.parametrize("kw,code", [
    (dict(batch=-1), _lib.ERR_SHAPE_MISMATCH), (dict(n_tokens=-1), _lib.ERR_SHAPE_MISMATCH),
    (dict(max_pages=-1), _lib.ERR_SHAPE_MISMATCH), (dict(num_pages=-1), _lib.ERR_SHAPE_MISMATCH),
    (dict(batch=4097), _lib.ERR_SHAPE_MISMATCH), (dict(page_size=0), _lib.ERR_UNSUPPORTED),
    (dict(page_size=24), _lib.ERR_UNSUPPORTED), (dict(page_size=256), _lib.ERR_UNSUPPORTED),
    (dict(num_pages=BIG // 16), _lib.ERR_SHAPE_MISMATCH), (dict(max_pages=BIG // 16), _lib.ERR_SHAPE_MISMATCH),
    (dict(n_tokens=BIG), _lib.ERR_SHAPE_MISMATCH), (dict(n_tokens=(1 << 30) + 1), _lib.ERR_SHAPE_MISMATCH),
    *[(dict([(n, None)]), _lib.ERR_NULL_POINTER) for n in (
        "new_lens", "seq_lens", "block_table", "free_list", "free_count", "q_starts", "slots", "positions",
        "context_lens", "granted", "free_after")]])
def test_plan_refusals(kw, code):
    expect(lib.teeny_kv_cache_plan(*plan_args(**kw)), code)


def write_args(**kw):
    a = dict(k=FAKE, v=FAKE, slots=FAKE, k_cache=FAKE, v_cache=FAKE, k_scale=FAKE, v_scale=FAKE, n_tokens=4, kv_heads=2,
             head_dim=128, num_pages=8, page_size=16, k_stride=256, v_stride=256)
    assert set(kw) <= set(a)
    return [*{**a, **kw}.values(), None]


@pytest.mark.parametrize("kw,code", [
    (dict(n_tokens=-1), _lib.ERR_SHAPE_MISMATCH), (dict(kv_heads=-1), _lib.ERR_SHAPE_MISMATCH),
    (dict(num_pages=-1), _lib.ERR_SHAPE_MISMATCH), (dict(head_dim=96), _lib.ERR_UNSUPPORTED),
    (dict(head_dim=0), _lib.ERR_UNSUPPORTED), (dict(page_size=8), _lib.ERR_UNSUPPORTED),
    (dict(num_pages=BIG // 16), _lib.ERR_SHAPE_MISMATCH), (dict(kv_heads=65536, k_stride=1 << 24, v_stride=1 << 24), _lib.ERR_SHAPE_MISMATCH),
    (dict(n_tokens=BIG), _lib.ERR_SHAPE_MISMATCH), (dict(n_tokens=(1 << 27) + 1), _lib.ERR_SHAPE_MISMATCH),
    (dict(k_stride=255), _lib.ERR_SHAPE_MISMATCH),
    (dict(v_stride=128), _lib.ERR_SHAPE_MISMATCH), (dict(k_stride=260), _lib.ERR_MISALIGNED),
    (dict(v_stride=257), _lib.ERR_MISALIGNED), (dict(k=FAKE_ODD), _lib.ERR_MISALIGNED),
    (dict(v=FAKE_ODD), _lib.ERR_MISALIGNED), (dict(k_cache=FAKE_ODD), _lib.ERR_MISALIGNED),
    (dict(v_cache=FAKE_ODD), _lib.ERR_MISALIGNED),
    *[(dict([(n, None)]), _lib.ERR_NULL_POINTER) for n in ("k", "v", "slots", "k_cache", "v_cache", "k_scale", "v_scale")]])
def test_write_refusals(kw, code):
    expect(lib.teeny_kv_cache_write(*write_args(**kw)), code)


def test_nothing_to_write():
    assert lib.teeny_kv_cache_write(*write_args(n_tokens=0, k=None, v=None, slots=None)) == _lib.OK
    assert lib.teeny_kv_cache_write(*write_args(num_pages=0, k_cache=None, v_cache=None)) == _lib.OK


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
    (dict(q=FAKE_ODD), _lib.ERR_MISALIGNED), (dict(o=FAKE_ODD), _lib.ERR_MISALIGNED),
    (dict(k_cache=FAKE_ODD), _lib.ERR_MISALIGNED), (dict(v_cache=FAKE_ODD), _lib.ERR_MISALIGNED),
    (dict(n_tokens=BIG), _lib.ERR_SHAPE_MISMATCH), (dict(n_tokens=1 << 29), _lib.ERR_SHAPE_MISMATCH),
    (dict(max_context=BIG), _lib.ERR_SHAPE_MISMATCH), (dict(max_pages=BIG // 16), _lib.ERR_SHAPE_MISMATCH),
    *[(dict([(n, None)]), _lib.ERR_NULL_POINTER) for n in (
        "q", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "context_lens", "o")]])
def test_attention_refusals(kw, code):
    expect(lib.teeny_kv_cache_attention(*attn_args(**kw)), code)


def test_attention_without_queries():
    assert lib.teeny_kv_cache_attention(*attn_args(n_tokens=0, q=None, o=None)) == _lib.OK
    assert lib.teeny_kv_cache_attention(*attn_args(batch=0, context_lens=None, block_table=None)) == _lib.OK


def test_attention_workspace_refusals():
    n = ctypes.c_size_t(7)
    f = lib.teeny_kv_cache_attention_workspace_size
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


def w4_args(**kw):
    a = dict(x=FAKE, qweight=FAKE, scale=FAKE, zero=None, bias=None, y=FAKE, m=4, n=32, k=256, group=128, act=0)
    assert set(kw) <= set(a)
    return [*{**a, **kw}.values(), None]


@pytest.mark.parametrize("kw,code", [
    *[(dict([(n, -1)]), _lib.ERR_SHAPE_MISMATCH) for n in "mnk"], *[(dict([(n, BIG)]), _lib.ERR_SHAPE_MISMATCH) for n in "mnk"],
    (dict(k=252), _lib.ERR_SHAPE_MISMATCH), *[(dict(group=g), _lib.ERR_INVALID_GROUP_SIZE) for g in (0, -32, 16, 96, 100, 192)],
    (dict(act=9), _lib.ERR_INVALID_ARGUMENT), (dict(act=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(x=FAKE_ODD), _lib.ERR_MISALIGNED), (dict(qweight=FAKE_ODD), _lib.ERR_MISALIGNED),
    *[(dict([(n, None)]), _lib.ERR_NULL_POINTER) for n in ("x", "qweight", "scale", "y")]])
def test_w4_refusals(kw, code):
    expect(lib.teeny_w4a16_linear_forward(*w4_args(**kw)), code)


def test_w4_helpers_refuse():
    n = ctypes.c_size_t(7)
    expect(lib.teeny_w4a16_linear_workspace_size(4, 32, 256, 48, ctypes.byref(n)), _lib.ERR_INVALID_GROUP_SIZE)
    expect(lib.teeny_w4a16_linear_workspace_size(4, 32, 256, 32, None), _lib.ERR_NULL_POINTER)
    assert lib.teeny_w4a16_linear_workspace_size(4, 32, 256, 32, ctypes.byref(n)) == _lib.OK and n.value == 0
    expect(lib.teeny_pack_int4(None, FAKE, 4, 8, None), _lib.ERR_NULL_POINTER)
    expect(lib.teeny_pack_int4(FAKE, None, 4, 8, None), _lib.ERR_NULL_POINTER)
    expect(lib.teeny_pack_int4(FAKE, FAKE_ODD, 4, 8, None), _lib.ERR_MISALIGNED)
    expect(lib.teeny_pack_int4(FAKE, FAKE, -4, 8, None), _lib.ERR_SHAPE_MISMATCH)
    assert lib.teeny_pack_int4(None, None, 0, 8, None) == _lib.OK


def test_shape_rules():
    assert K.kv_cache_dims((9, 2, 16, 64), (9, 2, 64, 16), (9, 2), (9, 2)) == (9, 2, 16, 64)
    for bad in ([(9, 2, 16, 64), (9, 2, 16, 64), (9, 2), (9, 2)], [(9, 2, 16, 64), (9, 2, 64, 16), (9, 1), (9, 2)],
                [(9, 2, 16, 64), (9, 2, 64, 16), (9, 2), (18,)], [(9, 2, 1024), (9, 2, 64, 16), (9, 2), (9, 2)]):
        with pytest.raises(ValueError):
            K.kv_cache_dims(*bad)
    assert K.w4a16_dims((3, 200), (7, 128), (7, 7), 32, (49,), (7,)) == (3, 7, 200)
    for bad in ([(3, 200), (7, 100), (7, 7), 32], [(3, 200), (7, 128), (7, 6), 32], [(3, 200), (7, 128), (7, 7), 48],
                [(3, 200), (7, 128), (7, 7), 32, (7,)], [(3, 200), (7, 128), (7, 7), 32, None, (6,)], [(200,), (7, 128), (7, 7), 32]):
        with pytest.raises(ValueError):
            K.w4a16_dims(*bad)


def test_w4_runtime_op():
    op = K.W4A16LinearRuntimeOp(64, use_zero_point=True, use_bias=True, act="silu")
    shapes = op.param_shapes([[5, 200]], [5, 24])
    assert shapes == [[24, 128], [24, 4], [24, 4], [24]]
    assert op.param_names() == ("qweight", "scale", "zero_point", "bias")
    assert op.const_generics() == (1, _lib.ACT_SILU, 64) and op.entry_point_name() == "w4a16_linear_forward_entry_point"
    rec = K.RecordingVisitor()
    op.pack_args([(1, [5, 200])], [2, 3, 4, 5], 6, [5, 24], 24, rec)
    assert rec.args == [("ptr", 1), ("ptr", 2), ("ptr", 3), ("ptr", 4), ("ptr", 5), ("ptr", 6), ("i32", 5), ("i32", 24), ("i32", 200)]
    rec = K.RecordingVisitor()
    K.W4A16LinearRuntimeOp(64).pack_args([(1, [5, 200])], [2, 3], 6, [5, 24], 24, rec)
    assert [a[1] for a in rec.args[:6]] == [1, 2, 3, None, None, 6]


def test_packed_words():
    codes = np.zeros((1, 136), np.int8)
    codes[0, 32 * 2 + 8 * 3 + 1] = 7  # word 4 g + c = 14, second code: nibble 4
    codes[0, 129] = -8
    words = kv.pack(codes).view(np.uint32).reshape(-1)
    assert len(words) == 32 and words[14] == 0x888F8888 and words[16] == 0x88808888
    assert all(w == 0x88888888 for i, w in enumerate(words) if i not in (14, 16))


def test_plan_oracle():
    """The plain plan on a case small enough to follow by eye."""
    table = np.array([[5, -1], [7, 2], [-1, -1]], np.int32)
    out, table, stack = kv.plan([2, -1, 17], [15, 20, 0], table, np.array([4, 0, 0, 0, 0, 0, 0, 0], np.int32), 1, 16, 20)
    assert table.tolist() == [[5, 2], [7, 2], [7, 4]] and stack[:3].tolist() == [4, 7, 2]
    assert out["slots"].tolist() == [95, 32] + [112 + i for i in range(16)] + [64, -1]
    assert out["q_starts"].tolist() == [0, 2, 2, 19] and out["context_lens"].tolist() == [17, 0, 17]
    assert out["granted"].tolist() == [2, 0, 17] and out["free_after"].tolist() == [0]


@pytest.mark.parametrize("batch,hq,hkv,d,longest,context", [(4096, 8, 8, 64, 1, 1 << 20), (2000, 32, 32, 128, 1, (1 << 31) - 5000),
                                                            (3000, 16, 4, 64, 4, 1 << 26), (1, 8, 2, 128, 1, 1 << 30)])
def test_attention_splits_fit_a_launch(batch, hq, hkv, d, longest, context):
    """A large max_context asks for no more parts than a launch of 2^31 threads has workgroups for, in which case the
    call would be refused."""
    tokens, rows = batch * longest, hq // hkv * longest
    block = 128 if rows > 64 else 32 if rows > 16 else 16
    units = (tokens * (hq // hkv) // block + batch) * hkv
    assert units * block < 1 << 25, "within the documented limit of rows"
    n = ctypes.c_size_t(0)
    assert lib.teeny_kv_cache_attention_workspace_size(tokens, batch, hq, hkv, d, longest, context, ctypes.byref(n)) == _lib.OK
    splits = n.value // (units * block * (d + 2) * 4)
    assert splits > 1 and units * splits < (1 << 31) // 256


@pytest.mark.parametrize("group", [(1 << 63), (1 << 64) + 32, (1 << 64) + 128, 3 << 64])
def test_w4_group_size_beyond_64_bits(group):
    """Cut to 64 bits it would be another group size, whose scales the buffers do not hold."""
    with pytest.raises(ValueError):
        K.w4a16_dims((3, 264), (7, 192), (7, 1), group)
    with pytest.raises(ValueError):
        K.W4A16LinearRuntimeOp(group)
    assert K.w4a16_dims((3, 264), (7, 192), (7, 1), (1 << 63) - 128) == (3, 7, 264)


@pytest.mark.parametrize("batch,hq,hkv,d,context,splits", [
    (64, 32, 8, 128, 5000, 1), (64, 32, 8, 128, 5200, 1), (64, 32, 8, 128, 7600, 1), (64, 32, 8, 128, 8000, 3), (128, 32, 8, 128, 6400, 2),
    (48, 32, 8, 128, 6400, 2), (56, 32, 8, 128, 6400, 1), (80, 32, 8, 128, 6400, 2),
    (1, 64, 64, 128, 30000, 8), (1, 64, 32, 128, 60000, 16), (4, 32, 8, 128, 60000, 23)])
def test_attention_splits_of_long_contexts(batch, hq, hkv, d, context, splits):
    """Contexts that may differ in length get a split for each 2560 tokens, but not two of them where the unsplit call just fills
    two workgroups a CU, and no more than the device holds where there is one sequence."""
    n = ctypes.c_size_t(0)
    assert lib.teeny_kv_cache_attention_workspace_size(batch, batch, hq, hkv, d, 1, context, ctypes.byref(n)) == _lib.OK
    units = (batch * (hq // hkv) // 16 + batch) * hkv
    assert n.value == (units * splits * 16 * (d + 2) * 4 if splits > 1 else 0)
