"""GPU: calls of the paged cache at the ends of what they allow: tables whose entries name free pages, and
the most workgroups that a write can ask for."""
import numpy as np
import pytest

import paged_ref as ref
from brasa_amd import Kernels
from brasa_amd.device import DeviceBuffer, synchronize
from test_gpu_paged import assert_pool, ints, upload_pool
from test_gpu_pages import State, down

pytestmark = pytest.mark.gpu
PAGE = ref.PAGE


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,pages", [([100, 0, 64, 300], 12), ([500] * 40 + [0], 3000)], ids=["12", "3000"])
def test_compact_leaves_entries_of_free_pages(lens, pages, in_place):
    """Entries that name a page nobody owns (a row left behind by its sequence) stay as they are, whatever
    the workspace holds; ids out of range do too."""
    print("stale entries", pages, in_place, flush=True)
    s = State(lens, pages, seed=pages)
    row, live = lens.index(0), int((s.ref > 0).sum())
    free = np.flatnonzero(s.ref <= 0)
    picked = np.r_[free[free < live][:2], free[free >= live][-2:]]
    assert (picked < live).any() and (picked >= live).any()
    s.table[row, :len(picked)] = picked
    s.table[row, len(picked)] = pages
    s.gt.upload(s.table)
    t2, r2 = (s.gt, s.gr) if in_place else (ints(np.full_like(s.table, 99)), ints(np.full_like(s.ref, 99)))
    Kernels().kv_pages_compact(s.dev, s.gt, s.gr, t2, r2, s.status, len(lens), s.width, s.ws, s.wlen)
    synchronize()
    table, counts, _ = ref.compact(s.pool, s.table, s.ref)
    assert np.array_equal(table[row], s.table[row])
    assert np.array_equal(down(t2, table), table) and np.array_equal(down(r2, counts), counts)
    assert_pool(s.dev, s.pool)


def test_store_of_most_workgroups():
    """8200 sequences of two rows that cross a page, 1024 heads: more than 2^24 workgroups of 256 threads,
    past what one launch takes. All but a few sequences have no page (their rows are dropped and
    never read); of the few, some are the last ones."""
    n, hkv, per = 8200, 1024, 2
    some = [0, 1, 4095, 4096, n - 2, n - 1]
    rng = np.random.default_rng(12)
    pool = ref.Pool(1, 2 * len(some), hkv, rng)
    pool.k_exp[:], pool.v_exp[:] = 110, 111
    table = np.full((n, 2), -1, np.int32)
    table[some] = rng.permutation(2 * len(some)).reshape(-1, 2)
    cu, pos = np.arange(0, per * n + 1, per, dtype=np.int32), np.full(n, PAGE - 1, np.int32)
    row = hkv * 128 * 4
    bufs, new = [], []
    for _ in range(2):
        x = rng.standard_normal((per * len(some), hkv, 128)).astype(np.float32)
        b = DeviceBuffer(per * n * row)
        for j, i in enumerate(some):
            b.upload(x[per * j:per * (j + 1)], per * i * row)
        bufs.append(b)
        new.append(x)
    dev = upload_pool(pool)
    print("store of", n, "sequences,", hkv, "heads", flush=True)
    Kernels().store_kv_paged(dev, 0, *bufs, ints(cu), ints(pos), ints(table), n, 2, per * n)
    synchronize()
    ref.store(pool, 0, *new, np.arange(0, per * len(some) + 1, per), pos[some], table[some])
    assert_pool(dev, pool)


def test_fill_past_4_gib():
    """Clearing a pool or a workspace of more than 2^32 bytes writes all of it."""
    b = DeviceBuffer((1 << 32) + 300)
    at = [0, 511, 512, (1 << 31) - 1, 1 << 31, (1 << 32) - 1, 1 << 32, b.nbytes - 1]
    for value in (0x5A, 0x11):
        print("fill", value, flush=True)
        b.fill(value)
        synchronize()
        assert [int(b.download(np.uint8, 1, i)[0]) for i in at] == [value] * len(at)
