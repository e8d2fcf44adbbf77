"""GPU: calls of the paged cache at the ends of what they allow: tables whose entries name free pages."""
import numpy as np
import pytest

import paged_ref as ref
from brasa_amd import Kernels
from brasa_amd.device import synchronize
from test_gpu_paged import assert_pool, ints
from test_gpu_pages import State, down

pytestmark = pytest.mark.gpu


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
