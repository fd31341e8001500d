"""The 4-bit linear layer on the GPU: packing, few rows, many rows through the bf16 copy, and the quantizer before it."""
import numpy as np
import pytest

import kv_cases as kv
from gpu_util import stream_workspace
from teenygrad_amd import kernels as K
from teenygrad_amd._lib import check as check_status
from teenygrad_amd._lib import lib
from teenygrad_amd.dtypes import bf16, from_bf16, to_bf16
from teenygrad_amd.runtime import Stream

pytestmark = pytest.mark.gpu


def case(rng, m, n, k, group, zero):
    groups = kv.pages_of(k, group)
    x = from_bf16(to_bf16(rng.standard_normal((m, k)).astype(np.float32)))
    codes = rng.integers(-8 if zero else -7, 8, (n, k)).astype(np.int8)
    scale = rng.uniform(0.004, 0.02, (n, groups)).astype(np.float32)
    zp = rng.integers(-8, 8, (n, groups)).astype(np.int32) if zero else None
    return x, codes, scale, zp, rng.standard_normal(n).astype(np.float32)


def run(dev, x, codes, scale, zp, bias, group, act, stream=None):
    y = K.w4a16_linear(dev.upload(to_bf16(x), bf16), K.pack_int4(dev.upload(codes)), dev.upload(scale), group,
                       zero_point=dev.upload(zp) if zp is not None else None,
                       bias=dev.upload(bias) if bias is not None else None, act=act, stream=stream)
    if stream is not None:
        stream.synchronize()
    return from_bf16(y.to_host())


def check(got, x, codes, scale, zp, bias, group, act, copy):
    ref, tol = kv.w4_linear(x, codes, scale, zp, bias, group, act, copy)
    err = np.abs(got.astype(np.float64) - ref)
    assert (err <= tol).all(), f"worst {np.max(err - tol)} over the bound, error {np.max(err)}"
    if not copy:  # all that is rounded is the output: half a step of bf16, and what fp32 sums add
        assert np.linalg.norm(err) <= 1.13 * (kv.H16 + 2.0 ** -12) * np.linalg.norm(ref)


@pytest.mark.parametrize("n,k", [(1, 8), (16, 128), (17, 136), (5, 120), (100, 1000), (3, 4104)])
def test_pack(dev, n, k):
    codes = np.random.default_rng(n + k).integers(-8, 8, (n, k)).astype(np.int8)
    np.testing.assert_array_equal(K.pack_int4(dev.upload(codes)).to_host(), kv.pack(codes))


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (1, 1, 8), (2, 33, 264), (16, 100, 1024), (17, 48, 520), (33, 70, 2048), (64, 31, 384),
                                   (65, 40, 256), (200, 17, 136), (4, 20, 8200), (7, 40, 8192), (13, 17, 8456), (5, 100, 640), (130, 1100, 256), (64, 8200, 128), (40, 4200, 200), (11, 12300, 128)])
def test_linear(dev, m, n, k, group, zero):
    rng = np.random.default_rng(m + 3 * n + k + group)
    c = case(rng, m, n, k, group, zero)
    check(run(dev, *c, group, None), *c, group, None, False)


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("m", [3, 40, 150])
def test_linear_epilogue(dev, m, act):
    rng = np.random.default_rng(m)
    c = case(rng, m, 90, 320, 64, True)
    check(run(dev, *c, 64, act), *c, 64, act, False)
    check(run(dev, *c[:4], None, 64, act), *c[:4], None, 64, act, False)


@pytest.mark.parametrize("m,n,k,group,zero,act", [(65, 40, 256, 32, True, None), (100, 256, 512, 128, False, "silu"),
                                                  (300, 1000, 1032, 64, True, "gelu"), (513, 264, 2048, 256, False, None),
                                                  (1050, 1000, 1032, 64, True, "silu"), (200, 5300, 256, 32, False, None),
                                                  (4100, 264, 512, 512, True, None), (460, 1720, 136, 128, True, None),
                                                  (500, 2000, 264, 32, False, "relu")])
def test_linear_copy(dev, m, n, k, group, zero, act):
    """Many rows with a workspace: the weights as bf16, each rounded once."""
    rng = np.random.default_rng(m + k)
    c = case(rng, m, n, k, group, zero)
    with stream_workspace(dev, K.w4a16_linear_workspace_size(m, n, k, group)):
        check(run(dev, *c, group, act), *c, group, act, True)
    with stream_workspace(dev, 512):  # too small
        check(run(dev, *c, group, act), *c, group, act, False)


def test_linear_of_nothing(dev):
    x, w = dev.buffer(bf16, (0, 128)), dev.buffer("i8", (16, 64))
    assert K.w4a16_linear(x, w, dev.buffer("f32", (16, 1)), 128).shape == (0, 16)


@pytest.mark.parametrize("group", [384, 1 << 20, 1 << 40, (1 << 63) - 128])
def test_linear_of_one_group(dev, group):
    rng = np.random.default_rng(7)
    c = case(rng, 5, 20, 264, 384, True)
    check(run(dev, *c, group, None), *c, 384, None, False)


def test_linear_without_k(dev):
    """K = 0: the bias and the activation."""
    bias = np.array([-1.0, 0.5, 3.0], np.float32)
    y, b = dev.buffer(bf16, (2, 3)), dev.upload(bias)
    check_status(lib.teeny_w4a16_linear_forward(None, None, None, None, b.ptr, y.ptr, 2, 3, 0, 128, K.ACTS["relu"], None))
    np.testing.assert_array_equal(from_bf16(y.to_host()), np.tile(np.maximum(bias, 0), (2, 1)))


def test_linear_ignores_what_pads_k(dev):
    """The last chunk's codes past K and groups past the last one count for nothing, whatever they hold."""
    rng = np.random.default_rng(21)
    c = case(rng, 4, 20, 200, 64, True)
    packed = kv.pack(np.concatenate([c[1], rng.integers(-8, 8, (20, 56)).astype(np.int8)], 1))
    y = K.w4a16_linear(dev.upload(to_bf16(c[0]), bf16), dev.upload(packed), dev.upload(c[2]), 64, zero_point=dev.upload(c[3]),
                       bias=dev.upload(c[4]))
    check(from_bf16(y.to_host()), *c, 64, None, False)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize_pack_multiply(dev, orc, symmetric, group):
    """teeny-quant's 4-bit groups, packed and multiplied, against the oracle's dequantized weights."""
    rng = np.random.default_rng(group)
    n, k, m = 48, 416, 5
    w = rng.normal(0, 0.05, (n, k)).astype(np.float32)
    q, scales, zps, _ = K.quantize_affine(dev.upload(w), [n, k], "group", 1, group, symmetric=symmetric, bits=4)
    qo, so, zo, _ = orc.quantize_affine(w, [n, k], "group", 1, group, symmetric=symmetric, bits=4)
    np.testing.assert_array_equal(q.to_host().reshape(-1), qo)
    x = from_bf16(to_bf16(rng.standard_normal((m, k)).astype(np.float32)))
    y = K.w4a16_linear(dev.upload(to_bf16(x), bf16), K.pack_int4(q), scales, group, zero_point=None if symmetric else zps)
    ref, tol = kv.w4_linear(x, qo.reshape(n, k), so.reshape(n, -1), None if symmetric else zo.reshape(n, -1), None, group, None, False)
    wd = orc.dequantize_affine(qo, so, zo, [n, k], "group", 1, group).reshape(n, k).astype(np.float64)
    np.testing.assert_allclose(x.astype(np.float64) @ wd.T, ref, rtol=1e-5, atol=1e-5)
    assert (np.abs(from_bf16(y.to_host()) - ref) <= tol).all()


def test_runtime_op(dev):
    """The dispatch entry point computes what the typed one does."""
    rng = np.random.default_rng(31)
    x, codes, scale, zp, bias = case(rng, 6, 40, 256, 32, True)
    op = K.W4A16LinearRuntimeOp(32, use_zero_point=True, use_bias=True, act="gelu")
    xb, y = dev.upload(to_bf16(x), bf16), dev.buffer(bf16, (6, 40))
    params = [K.pack_int4(dev.upload(codes)), dev.upload(scale), dev.upload(zp), dev.upload(bias)]
    op.launch([(xb, [6, 256])], params, y, [6, 40], bf16)
    np.testing.assert_array_equal(from_bf16(y.to_host()), run(dev, x, codes, scale, zp, bias, 32, "gelu"))


def test_linear_in_a_graph(dev):
    """Both forms captured once and replayed over new inputs, eager work of another stream between."""
    rng = np.random.default_rng(41)
    for m, n in ((4, 96), (1030, 1024)):
        x, codes, scale, zp, bias = case(rng, m, n, 512, 64, False)
        s = Stream.create()
        xb, y = dev.buffer(bf16, (m, 512)), dev.buffer(bf16, (m, n))
        w, sc, bb = K.pack_int4(dev.upload(codes)), dev.upload(scale), dev.upload(bias)
        dev.synchronize()
        with stream_workspace(dev, K.w4a16_linear_workspace_size(m, n, 512, 64), s):
            s.begin_capture()
            K.w4a16_linear(xb, w, sc, 64, bias=bb, y=y, stream=s)
            graph = s.end_capture()
            for _ in range(4):
                x = from_bf16(to_bf16(rng.standard_normal((m, 512)).astype(np.float32)))
                xb.to_device(to_bf16(x))
                dev.synchronize()
                graph.launch(s)
                s.synchronize()
                check(from_bf16(y.to_host()), x, codes, scale, None, bias, 64, None, m > 64)
            graph.destroy()


@pytest.mark.parametrize("m", [5, 460])
def test_linear_rows_that_are_not_finite(dev, m):
    """An infinity or NaN stays in its row.  There the streaming form gives NaN, the one through the copy what the
    products add up to."""
    rng = np.random.default_rng(51)
    n, k, group = 1720, 136, 128
    x, *w = case(rng, m, n, k, group, True)
    sound = np.setdiff1d(np.arange(m), [1, 3])
    x[1, 130], x[3, 5] = np.nan, -np.inf

    def check_rows(copy):
        got = run(dev, x, *w, group, None)
        assert np.isnan(got[1]).all()
        check(got[sound], x[sound], *w, group, None, copy)
        return got[3]

    size = K.w4a16_linear_workspace_size(m, n, k, group)
    assert (size > 0) == (m > 448)
    with stream_workspace(dev, 256):
        assert np.isnan(check_rows(False)).all()
    if size:
        with stream_workspace(dev, size):
            got = check_rows(True)
        sign = np.sign(w[0][:, 5] - w[2][:, 0])
        np.testing.assert_array_equal(got, np.where(sign == 0, np.nan, -np.inf * np.where(sign == 0, 1, sign)))


def check_some(got, c, rows, cols, group, act, copy):
    """The chosen rows and columns: an output needs no other row of x or of the weights."""
    x, codes, scale, zp, bias = c
    part = x[rows], codes[cols], scale[cols], zp[cols] if zp is not None else None, bias[cols]
    check(got[np.ix_(rows, cols)], *part, group, act, copy)


@pytest.mark.parametrize("m,n,k,group,zero,act", [
    (256, 1024, 36000, 128, True, "gelu"),  # K in slices, whose sums lie behind the copy
    (200, 11501, 4096, 128, True, "silu"), (450, 1749, 520, 64, False, None),  # rows of y at odd offsets
    (300, 8003, 4000, 32, False, "relu"), (4096, 4099, 1024, 64, True, "silu"), (4096, 4104, 1032, 32, False, "gelu"),
    (500, 1600, 264, 256, True, None)])
def test_linear_through_the_copy(dev, m, n, k, group, zero, act):
    rng = np.random.default_rng(m + n + k)
    c = case(rng, m, n, k, group, zero)
    size = K.w4a16_linear_workspace_size(m, n, k, group)
    assert size >= 2 * n * k, "this shape takes the copy"
    assert (size > 2 * n * k + 256) == (k == 36000)
    rows = np.unique(np.concatenate([np.arange(4), m - 1 - np.arange(4), rng.integers(0, m, 200)]))
    with stream_workspace(dev, size):
        check_some(run(dev, *c, group, act), c, rows, np.arange(n), group, act, True)


def test_linear_of_a_million_rows(dev):
    """More rows than a launch has workgroups for along one axis, in both forms."""
    rng = np.random.default_rng(61)
    m = 65535 * 16 + 17
    c = case(rng, m, 8, 8, 32, True)
    rows, cols = np.concatenate([np.arange(100), np.arange(65535 * 16 - 40, m)]), np.arange(8)
    check_some(run(dev, *c, 32, None), c, rows, cols, 32, None, False)  # no workspace: 256 bytes would hold the copy
    with stream_workspace(dev, K.w4a16_linear_workspace_size(m, 8, 8, 32)):
        check_some(run(dev, *c, 32, None), c, rows, cols, 32, None, True)


def test_linear_of_many_columns(dev):
    """More columns than one launch takes."""
    rng = np.random.default_rng(62)
    n = (1 << 25) + 21
    c = case(rng, 3, n, 8, 32, True)
    cols = np.concatenate([np.arange(100), np.arange((1 << 25) - 40, n)])
    check_some(run(dev, *c, 32, "relu"), c, np.arange(3), cols, 32, "relu", False)
