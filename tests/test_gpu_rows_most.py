"""GPU: the maps of the most rows a call takes: two full counts add up to 2^31 before they are cut off."""
import numpy as np
import pytest

from brasa_amd import Kernels
from brasa_amd.device import synchronize
from test_gpu_paged import ints

pytestmark = pytest.mark.gpu
MOST = 1 << 30


@pytest.mark.parametrize("add", [[MOST, MOST], [MOST, 3, MOST], [5, MOST, 0, MOST] * 400, [2 ** 31 - 1] * 1500], ids=lambda a: str(a[:4]))
def test_most_rows(add):
    n = len(add)
    print("most rows", n, flush=True)
    lens = np.arange(n)
    cu, lk = ints(np.full(n + 1, 77)), ints(np.full(n, 77))
    Kernels().kv_rows(ints(add), ints(lens), None, n, 0, 9, MOST, cu=cu, lk=lk)
    synchronize()
    want = np.minimum(np.r_[0, np.cumsum(np.array(add, np.int64))], MOST)
    assert np.array_equal(cu.download(np.int32), want)
    assert np.array_equal(lk.download(np.int32), lens + np.diff(want))
