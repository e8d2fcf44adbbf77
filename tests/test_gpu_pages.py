"""GPU: forking, reserving and compacting the pages of the cache, and a run of all the paged
operators together, against the same one step after another on the host."""
import numpy as np
import pytest

import oracle
import paged_ref as ref
from brasa_amd import (AttnShape, Kernels, KvPool, KvType, decode_paged_workspace_len, kv_pages_workspace_len)
from brasa_amd.device import DeviceBuffer, Graph, Stream, synchronize
from test_gpu_paged import assert_pool, ints, random_table, upload_pool

pytestmark = pytest.mark.gpu
PAGE = ref.PAGE


def down(buf, like):
    return buf.download(np.int32).reshape(like.shape)


class State:
    """Sequences of `lens` positions on random pages of a pool with random bytes."""

    def __init__(self, lens, pages, hkv=2, layers=2, width=None, seed=0, shared=0):
        rng = np.random.default_rng(seed)
        self.rng, self.lens = rng, np.array(lens, np.int32)
        counts = [-(-n // PAGE) for n in lens]
        self.width = width or max(max(counts), 1) + 1
        self.pool = ref.Pool(layers, pages, hkv, rng)
        self.table = random_table(rng, counts, pages, self.width)
        self.ref = np.bincount(self.table[self.table >= 0], minlength=pages).astype(np.int32)
        n = len(lens)
        for _ in range(shared):
            self.fork_host([int(x) for x in rng.integers(-1, n, n)])
        self.dev = upload_pool(self.pool)
        self.wlen = kv_pages_workspace_len(pages, n, self.width)
        self.ws = DeviceBuffer(max(self.wlen, 1))
        self.ws.fill(0xA5)
        self.gt, self.gl, self.gr = ints(self.table), ints(self.lens), ints(self.ref)
        self.status = ints([77, 77])

    def fork_host(self, parent):
        self.table, self.lens, self.ref = ref.fork(parent, self.table, self.lens, self.ref)

    def fork(self, parent, in_place, stream=None):
        n, pages = len(self.lens), len(self.ref)
        t2, l2 = ints(np.full_like(self.table, 99)), ints(np.full_like(self.lens, 99))
        r2 = self.gr if in_place else ints(np.full_like(self.ref, 99))
        Kernels().kv_pages_fork(ints(parent), self.gt, self.gl, self.gr, t2, l2, r2, n, self.width, pages, stream)
        synchronize()
        self.fork_host(parent)
        self.gt, self.gl, self.gr = t2, l2, r2
        self.check()

    def reserve(self, add, in_place, stream=None):
        t2 = self.gt if in_place else ints(np.full_like(self.table, 99))
        r2 = self.gr if in_place else ints(np.full_like(self.ref, 99))
        Kernels().kv_pages_reserve(self.dev, ints(add), self.gt, self.gl, self.gr, t2, r2, self.status,
                                   len(self.lens), self.width, self.ws, self.wlen, stream)
        synchronize()
        self.table, self.ref, want = ref.reserve(self.pool, add, self.table, self.lens, self.ref)
        self.gt, self.gr = t2, r2
        assert np.array_equal(self.status.download(np.int32), want), (self.status.download(np.int32), want)
        self.check()
        return want

    def compact(self, in_place, stream=None):
        t2 = self.gt if in_place else ints(np.full_like(self.table, 99))
        r2 = self.gr if in_place else ints(np.full_like(self.ref, 99))
        Kernels().kv_pages_compact(self.dev, self.gt, self.gr, t2, r2, self.status, len(self.lens), self.width,
                                   self.ws, self.wlen, stream)
        synchronize()
        self.table, self.ref, live = ref.compact(self.pool, self.table, self.ref)
        self.gt, self.gr = t2, r2
        assert self.status.download(np.int32)[0] == live
        self.check()

    def check(self):
        assert np.array_equal(down(self.gt, self.table), self.table)
        assert np.array_equal(down(self.gl, self.lens), self.lens)
        assert np.array_equal(down(self.gr, self.ref), self.ref)
        assert_pool(self.dev, self.pool)
        n = np.bincount(self.table[self.table >= 0], minlength=len(self.ref))
        assert np.array_equal(n, self.ref)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("parent", [[0, 1, 2, 3], [-1, -1, -1, -1], [3, 2, 1, 0], [1, 1, 1, 1], [2, 9, -7, 2]],
                         ids=str)
def test_fork(parent, in_place):
    print("fork", parent, in_place, flush=True)
    State([100, 0, 64, 300], 12).fork(parent, in_place)


@pytest.mark.parametrize("n,pages", [(1, 40), (130, 900), (700, 40000)])
def test_fork_sizes(n, pages):
    """One row, and more entries or pages than the one-workgroup kernel takes."""
    rng = np.random.default_rng(n)
    s = State([int(x) for x in rng.integers(0, 8 * PAGE if n < 700 else 3 * PAGE, n)], pages, hkv=1, layers=1,
              width=40, seed=n)
    for in_place in (False, True):
        print("fork", n, pages, in_place, flush=True)
        s.fork([int(x) for x in rng.integers(-1, n, n)], in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("shared", [0, 1, 2])
@pytest.mark.parametrize("add", [1, 64, 130])
def test_reserve(add, shared, in_place):
    print("reserve", add, shared, in_place, flush=True)
    s = State([100, 0, 64, 300, 63, 1, 129], 60, seed=add, width=9, shared=shared)
    want = s.reserve(np.array([add, 0, add, 1, -3, add, 2], np.int32), in_place)
    assert want[1] == 0


def test_reserve_every_owner_of_a_page():
    """Rows that share a partly filled page and all reserve: the first keeps it."""
    for parent in ([0, 0, 0, 0], [1, 1, 2, 2], [3, 0, 3, 3]):
        s = State([100, 70, 64, 300], 30, seed=1, width=7)
        s.fork(parent, False)
        s.reserve(np.array([1, 1, 1, 1], np.int32), False)
    s = State([100, 70, 64, 300], 30, seed=1, width=7)
    s.fork([0, 0, 0, 0], False)
    s.reserve(np.array([0, 1, 1, 1], np.int32), False)  # row 0 keeps its page without asking


def test_reserve_too_few_pages_changes_nothing():
    s = State([100, 70], 6, seed=2, width=9)
    before = s.table.copy()
    want = s.reserve(np.array([300, 10], np.int32), False)
    assert want[0] == 0 and want[1] > 0 and np.array_equal(s.table, before)
    assert list(s.reserve(np.array([29, 58], np.int32), True)) == [1, 0]     # 129 positions: one more page
    assert list(s.reserve(np.array([2000, 1], np.int32), False)) == [0, -1]  # past the table's width
    assert list(s.reserve(np.array([92, 100], np.int32), False)) == [1, 0]   # the last page, for the second row
    assert s.reserve(np.array([0, 300], np.int32), True)[1] > 0


def test_reserve_many_rows():
    """More rows and more claims than one round of the workgroup takes."""
    rng = np.random.default_rng(3)
    n = 1500
    s = State([int(x) for x in rng.integers(0, 200, n)], 9000, hkv=1, layers=1, width=8, seed=3, shared=1)
    assert s.reserve(rng.integers(-1, 200, n).astype(np.int32), False)[1] == 0
    s.compact(False)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,pages", [([100, 0, 64, 300], 12), ([], 5), ([1], 1), ([64 * 5], 5), ([100] * 9, 200),
                                        ([500] * 40, 3000)], ids=str)
def test_compact(lens, pages, in_place):
    print("compact", len(lens), pages, in_place, flush=True)
    if not lens:
        lens = [0]
    State(lens, pages, seed=pages, hkv=3, layers=2).compact(in_place)


def test_pages_replay():
    """A captured fork and reserve, replayed on other parents, beside work on another stream."""
    s, kern, n = Stream(), Kernels(), 6
    st = State([100, 64, 300, 63, 1, 129], 80, seed=5, width=8)
    other = State([100, 64, 300], 40, seed=6)
    parent, add = ints([0] * n), ints([1] * n)
    tm, t2 = ints(np.zeros_like(st.table)), ints(np.zeros_like(st.table))
    l2, rm, r2 = ints(np.zeros_like(st.lens)), ints(np.zeros_like(st.ref)), ints(np.zeros_like(st.ref))
    with Graph.capture(s) as g:
        kern.kv_pages_fork(parent, st.gt, st.gl, st.gr, tm, l2, rm, n, st.width, 80, s)
        kern.kv_pages_reserve(st.dev, add, tm, l2, rm, t2, r2, st.status, n, st.width, st.ws, st.wlen, s)
    for p in ([0, 1, 2, 3, 4, 5], [2, 2, 2, -1, 4, 4], [5, 5, 0, 0, 0, 1]):
        parent.upload(np.array(p, np.int32))
        g.launch(s)
        s.synchronize()
        other.compact(False)
        table, lens, counts = ref.fork(p, st.table, st.lens, st.ref)
        table, counts, want = ref.reserve(st.pool, [1] * n, table, lens, counts)
        assert np.array_equal(st.status.download(np.int32), want)
        assert np.array_equal(down(t2, table), table) and np.array_equal(down(r2, counts), counts)
        assert np.array_equal(down(l2, lens), lens)
        assert_pool(st.dev, st.pool)


def test_serving_run():
    """Prompts arrive packed, fill the cache, fork, decode several tokens, end, and the pool is compacted:
    each step's output against the host, with the host's own copy of the cache beside it."""
    rng, kern = np.random.default_rng(11), Kernels()
    hq, hkv, n, width, pages = 8, 2, 5, 8, 40
    lens = np.array([70, 1, 200, 64], np.int32)
    rows = int(lens.sum())
    cu = np.r_[0, np.cumsum(lens)].astype(np.int32)
    pool = ref.Pool(1, pages, hkv, rng)
    dev = upload_pool(pool)
    table, counts = np.full((n, width), -1, np.int32), np.zeros(pages, np.int32)
    have = np.zeros(n, np.int32)
    st = State([0], pages)  # (its workspace is of another shape: one of the right size below)
    wlen = kv_pages_workspace_len(pages, n, width)
    ws, dws = DeviceBuffer(wlen), DeviceBuffer(decode_paged_workspace_len(hq, hkv))
    dws.fill(0)
    status = st.status
    gt, gl, gr = ints(table), ints(have), ints(counts)
    # room for the prompts; the last row stays empty
    add = np.r_[lens, 0].astype(np.int32)
    kern.kv_pages_reserve(dev, ints(add), gt, gl, gr, gt, gr, status, n, width, ws, wlen)
    table, counts, _ = ref.reserve(pool, add, table, have, counts)
    q, k, v = (rng.standard_normal((rows, h, 128)).astype(np.float32) for h in (hq, hkv, hkv))
    gq, gk, gv = (DeviceBuffer.from_array(x) for x in (q, k, v))
    o = DeviceBuffer(q.nbytes)
    from brasa_amd import PrefillPrecision
    kern.flash_attention_packed(gq, gk, gv, o, ints(cu), 4, AttnShape(rows, hq, hkv, 128, 0, KvType.F32),
                                PrefillPrecision.F32)
    kern.store_kv_paged(dev, 0, gk, gv, ints(np.r_[cu, rows]), gl, gt, n, width, rows)
    synchronize()
    ref.store(pool, 0, k, v, np.r_[cu, rows], have, table)
    assert_pool(dev, pool)
    got = o.download(np.float32).reshape(q.shape)
    for a, b in zip(cu, cu[1:]):
        want, av, top = ref.attend(q[a:b], k[a:b].astype(np.float64), v[a:b].astype(np.float64), True)
        assert np.all(np.abs(got[a:b] - want) <= av * (top * 2.0 ** -15 + 2.0 ** -14))
    have = np.r_[lens, 0].astype(np.int32)
    gl = ints(have)
    for step, parent in enumerate([[0, 1, 2, 2, 2], [0, 3, 2, 4, -1], [0, 1, 2, 3, 0], [4, 1, -1, 3, 4]]):
        print("step", step, flush=True)
        t2, l2 = ints(table), ints(have)
        kern.kv_pages_fork(ints(parent), gt, gl, gr, t2, l2, gr, n, width, pages)
        table, have, counts = ref.fork(parent, table, have, counts)
        gt, gl = t2, l2
        new = (have > 0).astype(np.int32)
        kern.kv_pages_reserve(dev, ints(new), gt, gl, gr, gt, gr, status, n, width, ws, wlen)
        table, counts, want = ref.reserve(pool, new, table, have, counts)
        r = int(new.sum())
        q, k, v = (rng.standard_normal((m, h, 128)).astype(np.float32) for m, h in ((n, hq), (r, hkv), (r, hkv)))
        c1 = np.r_[0, np.cumsum(new)].astype(np.int32)
        bufs = [DeviceBuffer.from_array(x) for x in (q, k, v)]
        kern.store_kv_paged(dev, 0, bufs[1], bufs[2], ints(c1), gl, gt, n, width, r)
        ref.store(pool, 0, k, v, c1, have, table)
        have = have + new
        gl = ints(have)
        o = DeviceBuffer(q.nbytes)
        kern.decode_attention_paged(bufs[0], dev, 0, gt, gl, n, width, dws, dws.nbytes, o, hq)
        if step == 2:
            kern.kv_pages_compact(dev, gt, gr, gt, gr, status, n, width, ws, wlen)
        synchronize()
        got = o.download(np.float32).reshape(q.shape)
        for i, lk in enumerate(have):
            kk, vv = ref.rows_of(pool, 0, table[i, :-(-lk // PAGE)], lk)
            o64, av, top = (x[0] for x in ref.attend(q[i:i + 1], kk, vv, False))
            assert np.all(np.abs(got[i] - o64) <= av * (top * 2.0 ** -15 + 2.0 ** -14) + 1e-37), (step, i)
        if step == 2:
            table, counts, _ = ref.compact(pool, table, counts)
        assert np.array_equal(down(gt, table), table) and np.array_equal(down(gr, counts), counts)
        assert_pool(dev, pool)
