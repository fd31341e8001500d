"""Low-rank adapters of many requests on the GPU, against the plain form of kv4_cases.py."""
import contextlib

import numpy as np
import pytest

import kv4_cases as kv4
from gpu_util import stream_workspace
from teenygrad_amd import kernels as K
from teenygrad_amd._lib import check, lib
from teenygrad_amd.dtypes import bf16, from_bf16, to_bf16
from teenygrad_amd.runtime import Stream

pytestmark = pytest.mark.gpu


def rounded(a):
    return from_bf16(to_bf16(np.asarray(a, np.float32)))


def up(dev, a):
    return dev.upload(to_bf16(np.asarray(a, np.float32)), bf16)


def case(rng, ids, n, k, rank, adapters):
    m = len(ids)
    return dict(x=rounded(rng.standard_normal((m, k))), a=rounded(rng.standard_normal((adapters, rank, k)) / np.sqrt(max(k, 1))),
                b=rounded(rng.standard_normal((adapters, n, rank)) * 0.4), ids=np.array(ids, np.int32),
                scale=rng.uniform(0.3, 2, adapters).astype(np.float32), y=rounded(rng.standard_normal((m, n))))


def run(dev, c, scale=True, in_place=False, stream=None):
    y = up(dev, c["y"])
    out = K.adapter_add(up(dev, c["x"]), up(dev, c["a"]), up(dev, c["b"]), dev.upload(c["ids"]), y, scale=dev.upload(c["scale"]) if scale else None,
                        out=y if in_place else None, stream=stream)
    if stream is not None:
        stream.synchronize()
    return from_bf16(out.to_host())


def check_run(c, got, scale=True):
    ref, tol = kv4.adapter(c["x"], c["a"], c["b"], c["ids"], c["scale"] if scale else None, c["y"])
    err = np.abs(got - ref)
    assert (err <= tol).all(), f"worst {np.nanmax(err - tol)} over the bound"
    none = (c["ids"] < 0) | (c["ids"] >= len(c["a"]))
    np.testing.assert_array_equal(got[none], c["y"][none])


def size_of(c):
    return K.adapter_add_workspace_size(len(c["ids"]), c["y"].shape[1], c["x"].shape[1], c["a"].shape[1])


def space_for(dev, c, space):
    return stream_workspace(dev, size_of(c)) if space else contextlib.nullcontext()


IDS = {
    "one": [1], "none": [-1] * 3, "all of one": [2] * 37, "each its own": list(range(40)), "runs": [0] * 5 + [3] * 30 + [-1] * 4 + [1] + [0] * 21,
    "mixed": [3, 1, 3, 0, -1, 1, 1, 0, 3, 2, 77, 0, 1, 2, 3, 0, 1, 2, -5, 2 ** 31 - 1, 3], "long": [1] * 130 + [2] * 70 + [0] * 9,
}


@pytest.mark.parametrize("space", [False, True])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 64, 104, 128])
@pytest.mark.parametrize("ids", list(IDS))
def test_adapters(dev, ids, rank, space):
    """Odd numbers of columns and sizes of K, rows in any order; small products are one launch, with or without a workspace."""
    rng = np.random.default_rng(rank + len(ids))
    for n, k in ((4, 8), (100, 264), (333, 1032), (4, 2056)):
        c = case(rng, IDS[ids], n, k, rank, 40 if ids == "each its own" else 4)
        with space_for(dev, c, space):
            check_run(c, run(dev, c))


@pytest.mark.parametrize("space", [False, True])
@pytest.mark.parametrize("m,n,k,rank,adapters", [(1, 4096, 4096, 16, 3), (64, 1001, 2056, 16, 20), (300, 520, 4096, 64, 5), (17, 11008, 512, 32, 9)])
def test_larger(dev, m, n, k, rank, adapters, space):
    rng = np.random.default_rng(m + n)
    c = case(rng, np.sort(rng.integers(-1, adapters, m)) if m > 100 else rng.integers(-1, adapters, m), n, k, rank, adapters)
    if m == 1:
        c["ids"][:] = 1
    with space_for(dev, c, space):
        check_run(c, run(dev, c))
        check_run(c, run(dev, c, scale=False), scale=False)
        check_run(c, run(dev, c, in_place=True))


@pytest.mark.parametrize("space", [False, True])
@pytest.mark.parametrize("ordered", [False, True])
@pytest.mark.parametrize("m,n,k,rank", [(257, 70, 264, 16), (400, 130, 520, 16), (777, 130, 520, 16), (513, 333, 40, 32), (601, 36, 1032, 64), (1025, 300, 520, 8), (1090, 66, 136, 128)])
def test_many_rows(dev, m, n, k, rank, ordered, space):
    """Tiles of several adapters, more of them than workgroups take at once, and a last tile that is not whole."""
    rng = np.random.default_rng(m)
    ids = rng.integers(-1, 9, m)
    c = case(rng, np.sort(ids) if ordered else ids, n, k, rank, 9)
    with space_for(dev, c, space):
        check_run(c, run(dev, c))
        check_run(c, run(dev, c, in_place=True))


@pytest.mark.parametrize("space", [False, True])
def test_rows_are_apart(dev, space):
    """What a row of x holds reaches that row alone, an adapter's numbers its own rows, and infinities follow the products."""
    rng = np.random.default_rng(3)
    c = case(rng, [0, 1, 0, 2, -1, 1, 0], 70, 1064 if space else 40, 16, 3)
    assert (size_of(c) > 0) == space
    clean = kv4.adapter(c["x"], c["a"], c["b"], c["ids"], c["scale"], c["y"])
    c["x"][2, 5], c["x"][4, 1], c["a"][2, 3, 7], c["b"][1, 11, 4] = np.nan, np.inf, np.inf, np.nan
    c["x"][3] = 1.0
    with space_for(dev, c, space):
        got = run(dev, c)
    assert np.isnan(got[2]).all() and np.isnan(got[[1, 5], 11]).all() and np.isinf(got[3]).all()
    rows = np.ones(got.shape, bool)
    rows[[2, 3]] = rows[[1, 5], 11] = False
    assert (np.abs(got - clean[0]) <= clean[1])[rows].all()
    np.testing.assert_array_equal(got[4], c["y"][4])


@pytest.mark.parametrize("space", [False, True])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(7, 70, 1064), (9, 333, 40), (300, 520, 264), (600, 130, 264)])
def test_infinities_in_b(dev, m, n, k, rank, space):
    """An infinity in B gives the infinity or NaN of the formula, whatever the sign and size of the ranks' second part."""
    rng = np.random.default_rng(m + rank)
    c = case(rng, np.sort(rng.integers(-1, 3, m)) if m > 9 else [0, 1, 0, 2, -1, 1, 0, 2, 2][:m], n, k, rank, 3)
    # each product of the ranks is one number of x times one of A: its sign is in no doubt, and some have a second part of 0
    c["x"][:, 1:] = 0
    c["x"][:, 0] = np.where(np.arange(m) % 2, 2.0 ** rng.integers(-3, 4, m), rounded(rng.uniform(0.5, 2, m))) * rng.choice([-1, 1], m)
    c["a"][:, ::2, 0] = 1
    c["scale"][0] = 1
    c["b"][0, 11, 4], c["b"][0, 12, 7], c["b"][1, 3, 5], c["b"][2, 69, 6] = np.inf, -np.inf, np.inf, np.inf
    c["b"][0, 20, :2] = np.inf, -np.inf
    c["b"][1, 40, 1] = np.nan
    with np.errstate(all="ignore"):
        ref, tol = kv4.adapter(c["x"], c["a"], c["b"], c["ids"], c["scale"], c["y"])
    with space_for(dev, c, space):
        got = run(dev, c)
    fin = np.isfinite(ref)
    assert np.isinf(ref).any() and np.isnan(ref).any()
    np.testing.assert_array_equal(got[~fin], ref[~fin].astype(np.float32))
    assert (np.abs(got[fin] - ref[fin]) <= tol[fin]).all()


@pytest.mark.parametrize("space", [False, True])
def test_strides(dev, space):
    """Rows of x, y and out inside wider ones, the aligned and the odd kind; nothing between them is written."""
    rng = np.random.default_rng(4)
    for n, first, row in ((64, 16, 96), (61, 3, 67), (64, 2, 70)):
        k = 1072 if space else 48
        c = case(rng, [0, 2, -1, 1, 1], n, k, 8, 3)
        m = 5
        x, y, out = (np.full((m, w), 5.0, np.float32) for w in (k + 16, row, row + 4))
        x[:, 8:k + 8], y[:, first:first + n] = c["x"], c["y"]
        xb, yb, ob, a, b = (up(dev, z) for z in (x, y, out, c["a"], c["b"]))
        ids, s = dev.upload(c["ids"]), dev.upload(c["scale"])
        with space_for(dev, c, space):
            check(lib.teeny_adapter_add(xb.ptr + 16, a.ptr, b.ptr, ids.ptr, s.ptr, yb.ptr + 2 * first, ob.ptr + 2 * first, m, n, k, 8, 3,
                                        k + 16, row, row + 4, None))
            got = from_bf16(ob.to_host())
        check_run(c, got[:, first:first + n])
        assert (np.delete(got, np.s_[first:first + n], axis=1) == 5.0).all()


def test_without_adapters(dev):
    """No adapter, no rank, no K: the output is y."""
    rng = np.random.default_rng(5)
    c = case(rng, [0, 1, -1], 33, 16, 8, 2)
    y, out, ids = up(dev, c["y"]), dev.buffer(bf16, (3, 33)), dev.upload(c["ids"])
    x, a = up(dev, c["x"]), up(dev, c["a"])
    for rank, k, count in ((8, 16, 0), (0, 16, 2), (8, 0, 2)):
        out.to_device(np.zeros((3, 33), np.uint16))
        check(lib.teeny_adapter_add(x.ptr, a.ptr, a.ptr, ids.ptr, None, y.ptr, out.ptr, 3, 33, k, rank, count, 16, 33, 33, None))
        np.testing.assert_array_equal(out.to_host(), y.to_host())


def test_two_streams_and_a_graph(dev):
    """Two streams at once, each with its own workspace, one of them replaying a captured call with new inputs."""
    rng = np.random.default_rng(6)
    streams = [Stream.create(), Stream.create()]
    ids = [[0] * 40 + [2, 1, -1] * 9, [1, 0, 2, 2, -1]]
    cases = [case(rng, i, 300, 2048, 16, 3) for i in ids]
    bufs = [(up(dev, c["x"]), up(dev, c["a"]), up(dev, c["b"]), dev.upload(c["ids"]), up(dev, c["y"])) for c in cases]
    scales, outs = [dev.upload(c["scale"]) for c in cases], [dev.buffer(bf16, c["y"].shape) for c in cases]
    with stream_workspace(dev, size_of(cases[0]), streams[0]), stream_workspace(dev, size_of(cases[1]), streams[1]):
        streams[0].begin_capture()
        K.adapter_add(*bufs[0], scale=scales[0], out=outs[0], stream=streams[0])
        graph = streams[0].end_capture()
        for _ in range(5):
            for c, b in zip(cases, bufs):
                c["x"] = rounded(rng.standard_normal(c["x"].shape))
                b[0].to_device(to_bf16(c["x"]))
            dev.synchronize()
            graph.launch(streams[0])
            for _ in range(3):
                K.adapter_add(*bufs[1], scale=scales[1], out=outs[1], stream=streams[1])
            for s in streams:
                s.synchronize()
            for c, o in zip(cases, outs):
                check_run(c, from_bf16(o.to_host()))
        graph.destroy()


def test_results_repeat(dev):
    """The same call gives the same bits."""
    rng = np.random.default_rng(7)
    c = case(rng, rng.integers(0, 4, 50), 600, 2048, 16, 4)
    with stream_workspace(dev, size_of(c)):
        first = run(dev, c)
        for _ in range(4):
            np.testing.assert_array_equal(run(dev, c), first)
