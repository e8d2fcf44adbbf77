"""GPU: the fused paged writer where the sequences' bounds are out of order."""
import numpy as np
import pytest

import paged_ref as ref
import step_ref
from brasa_amd import Kernels, RopeAxes, RopeTable
from brasa_amd.device import DeviceBuffer, synchronize
from test_gpu_paged import ints, random_table, upload_pool

pytestmark = pytest.mark.gpu
PAGE, DIM = ref.PAGE, ref.DIM


def _both(given, raised, pos, hq=4, hkv=2, seed=0):
    """The call with the bounds as given and with them in order: the same k and the same pages."""
    rng, kern, n = np.random.default_rng(seed), Kernels(), len(pos)
    lens = np.array(pos) + np.diff(raised)
    counts = [-(-int(x) // PAGE) for x in lens]
    width, pages, tokens = max(counts), sum(counts) + 2, int(raised[-1]) + 3
    pool = ref.Pool(1, pages, hkv, rng)
    pool.k_exp[:] = pool.v_exp[:] = 118
    table = random_table(rng, counts, pages, width)
    rope_pos = rng.integers(0, 300, (1, tokens))
    x = [rng.standard_normal((tokens, h, DIM)).astype(np.float32) for h in (hq, hkv, hkv)]
    one = DeviceBuffer.from_array(np.ones(DIM, np.float32))
    out = []
    for cu in (given, raised):
        dev, bufs = upload_pool(pool), [DeviceBuffer.from_array(a) for a in x]
        kern.qk_norm_rope_store_paged(dev, 0, bufs, (one, one), 1e-6, RopeTable(1e6, DIM, 300), RopeAxes([64]), ints(rope_pos),
                                      ints(cu), ints(pos), ints(table), n, width, tokens, hq)
        synchronize()
        out.append([b.download(np.uint8) for b in (bufs[1], dev.k, dev.v, dev.k_exp, dev.v_exp)])
    assert not np.array_equal(out[1][0], x[1].view(np.uint8).ravel())
    for a, b in zip(*out):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("cu,tokens", [([0, 5, 2, 8], 8), ([3, 70, 1, 0, 90, 80, 200], 200), ([0, 200, 100, 150], 203), ([-7, 4, -1, 9], 9)],
                         ids=str)
def test_bounds_out_of_order(cu, tokens):
    """No row of k is turned twice: a bound below an earlier one is raised to it."""
    print("bounds", cu, flush=True)
    raised = step_ref.raised(cu, tokens)
    rng = np.random.default_rng(len(cu))
    _both(np.array(cu), raised, rng.integers(0, 150, len(cu) - 1), seed=len(cu))


def test_bounds_out_of_order_in_later_rounds():
    """More sequences than a wave has lanes, with bounds below those of an earlier round."""
    rng = np.random.default_rng(5)
    cu = np.cumsum(rng.integers(0, 3, 300))
    for at in (60, 64, 65, 130, 191, 192, 299):
        cu[at] -= 40
    cu[140:200] = 20
    raised = step_ref.raised(cu, int(cu.max()))
    _both(cu, raised, rng.integers(0, 100, 299), hkv=1)
