"""GPU: the maps of a step's rows and the pages that groups share, whole numbers against the host."""
import numpy as np
import pytest

import step_ref
from brasa_amd import Kernels
from brasa_amd.device import DeviceBuffer, Graph, Stream, synchronize
from test_gpu_paged import ints

pytestmark = pytest.mark.gpu
PAGE = step_ref.PAGE
NAMES = ("cu", "lk", "seq", "pos", "slot")


def _table(rng, n, width, pages):
    return rng.integers(-1, pages, (n, width)).astype(np.int32)


def _bufs(n, tokens):
    return {name: ints(np.full(size, 77)) for name, size in zip(NAMES, (n + 1, n, tokens, tokens, tokens))}


def _check(out, want, only=NAMES):
    for name, w in zip(NAMES, want):
        got = out[name].download(np.int32)[:len(w)]
        if name in only:
            assert np.array_equal(got, w), (name, np.flatnonzero(got != w)[:5], got[:8], w[:8])
        else:
            assert (got == 77).all(), name


@pytest.mark.parametrize("n,most,tokens", [(1, 1, 1), (1, 300, 200), (64, 1, 64), (64, 1, 100), (5, 700, 4000),
                                           (1000, 9, 6000), (1024, 3, 3000), (1025, 3, 3000), (3000, 40, 70000),
                                           (65536, 1, 70000), (2500, 0, 5)])
def test_rows(n, most, tokens):
    print("rows", n, most, tokens, flush=True)
    rng = np.random.default_rng(n + tokens)
    width, pages = 7, 50
    add = rng.integers(-1 if most else 0, most + 1, n).astype(np.int32)
    lens = rng.integers(-1, width * PAGE + 20, n).astype(np.int32)
    table = _table(rng, n, width, pages + 3)  # (ids past the pool among them)
    out = _bufs(n, tokens)
    Kernels().kv_rows(ints(add), ints(lens), ints(table), n, width, pages, tokens, **out)
    synchronize()
    _check(out, step_ref.rows(add, lens, table, pages, tokens))


def test_rows_extremes():
    """Counts and lengths at the ends of their type; sums past it."""
    top = 2 ** 31 - 1
    for add, lens in (([top, top, 5], [0, 3, 9]), ([3, top], [top, top - 1]), ([-top - 1, 4], [5, -top - 1]), ([0, 0], [top, 0])):
        n = len(add)
        table = np.arange(2 * n, dtype=np.int32).reshape(n, 2)
        for tokens in (1, 6, 3000):
            out = _bufs(n, tokens)
            Kernels().kv_rows(ints(add), ints(lens), ints(table), n, 2, 100, tokens, **out)
            synchronize()
            _check(out, step_ref.rows(add, lens, table, 100, tokens))


def test_rows_some_outputs():
    add, lens, table = np.array([2, 3], np.int32), np.array([5, 100], np.int32), np.array([[4, 1], [0, 3]], np.int32)
    want = step_ref.rows(add, lens, table, 9, 8)
    for only in (("cu",), ("pos", "slot"), ("lk", "seq"), ("slot",), ()):
        out = _bufs(2, 8)
        Kernels().kv_rows(ints(add), ints(lens), ints(table), 2, 2, 9, 8, **{k: out[k] for k in only})
        synchronize()
        _check(out, want, only)
    out = _bufs(2, 8)  # no rows are asked for, and a table without columns
    Kernels().kv_rows(ints(add), ints(lens), None, 2, 0, 9, 8, **out)
    synchronize()
    _check(out, step_ref.rows(add, lens, np.zeros((2, 0), np.int32), 9, 8))


@pytest.mark.parametrize("n,width,groups", [(2, 3, 1), (64, 130, 2), (64, 130, 64), (300, 700, 5), (2000, 9, 700)])
def test_shared(n, width, groups):
    print("shared", n, width, groups, flush=True)
    rng = np.random.default_rng(n + width)
    pages = 3000
    bounds = np.sort(rng.integers(0, n + 1, groups + 1)).astype(np.int32)
    bounds[0] = 0
    table = _table(rng, n, width, pages)
    lens = rng.integers(0, width * PAGE + 1, n).astype(np.int32)
    for a, b in zip(bounds, bounds[1:]):
        lead = rng.integers(0, pages, width)
        for i in range(a, b):
            same = rng.integers(0, width + 1)
            table[i, :same] = lead[:same]
            if rng.random() < 0.7:
                lens[i] = rng.integers(lens[i], width * PAGE + 1)
            if rng.random() < 0.1:
                lens[i] = rng.integers(-1, 1)
    out = ints(np.full(groups + 1, 77))
    Kernels().kv_pages_shared(ints(table), ints(lens), ints(bounds), groups, n, width, pages, out)
    synchronize()
    got = out.download(np.int32)
    assert np.array_equal(got[:-1], step_ref.shared(table, lens, bounds, pages)) and got[-1] == 77
    assert got[:-1].any() or n == 2  # (the small case has nothing to share)


def test_shared_edges():
    """Rows alike to the last page, ids that are no pages, bounds out of range and of order."""
    table = np.array([[1, 2, 3, 4], [1, 2, 3, 4], [1, 2, -1, 4], [1, 2, -1, 4], [1, 20, 3, 4], [1, 20, 3, 4]], np.int32)
    lens = np.full(6, 256, np.int32)
    lens[1] = 255
    group = np.array([0, 2, 4, 6, 6, 9, -3, 2], np.int32)
    out = ints(np.full(7, 77))
    Kernels().kv_pages_shared(ints(table), ints(lens), ints(group), 7, 6, 4, 10, out)
    synchronize()
    assert list(out.download(np.int32)) == [192, 128, 64, 0, 0, 0, 192]
    Kernels().kv_pages_shared(None, ints(lens), ints(group), 7, 6, 0, 10, out)
    synchronize()
    assert not out.download(np.int32).any()


def test_maps_in_a_graph():
    """A captured step is replayed while lengths, counts and tables change."""
    n, width, pages, tokens = 40, 20, 500, 300
    rng, kern, stream = np.random.default_rng(2), Kernels(), Stream()
    ga, gl, gt, gg = ints(np.zeros(n)), ints(np.zeros(n)), ints(np.zeros((n, width))), ints([0, 10, 40])
    out, prefix = _bufs(n, tokens), ints([0, 0])
    synchronize()
    with Graph.capture(stream) as g:
        kern.kv_rows(ga, gl, gt, n, width, pages, tokens, stream=stream, **out)
        kern.kv_pages_shared(gt, gl, gg, 2, n, width, pages, prefix, stream=stream)
    for _ in range(4):
        add, lens = rng.integers(-1, 12, n).astype(np.int32), rng.integers(-2, width * PAGE, n).astype(np.int32)
        table = _table(rng, n, width, pages)
        table[:, :3] = table[0, :3]
        for buf, x in ((ga, add), (gl, lens), (gt, table)):
            buf.upload(x)
        g.launch(stream)
        stream.synchronize()
        _check(out, step_ref.rows(add, lens, table, pages, tokens))
        assert np.array_equal(prefix.download(np.int32), step_ref.shared(table, lens, [0, 10, 40], pages))
