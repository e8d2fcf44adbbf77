"""CPU: the short form of attention over the paged cache is for f16 results, and for that call only."""
import pytest

from brasa_amd import BrasaError, Kernels, KvPool, OutDType
from brasa_amd.kernels import OUT_F16_SHORT

P = 4096  # an address that passes the checks of null and alignment; never followed here


def _refused(code, call):
    with pytest.raises(BrasaError) as e:
        call()
    assert e.value.code == code, str(e.value)


def test_short_is_for_f16_results():
    pool = KvPool.view(P, P, P, P, 1, 8, 8)
    _refused(5, lambda: Kernels().attention_paged(P, pool, 0, P, 2, 4, 5, P, 1 << 40, P, 32, OutDType.F32, short=True))
    # (no rows: the output's type passes)
    Kernels().attention_paged(0, pool, 0, 0, 2, 4, 0, 0, 1 << 40, 0, 32, OutDType.F16, short=True)
    _refused(5, lambda: Kernels().decode_attention_paged(P, pool, 0, P, 4, P, 2, P, 1 << 40, P, 32, OUT_F16_SHORT))


def test_short_overlaps():
    base = 1 << 40
    pool = KvPool.view(P, P, P, P, 1, 8, 8)
    _refused(5, lambda: Kernels().attention_paged(base + 2 * 5 * 32 * 128 - 16, pool, 0, P, 2, 4, 5, P, 1 << 36, base, 32,
                                                  OutDType.F16, short=True))
