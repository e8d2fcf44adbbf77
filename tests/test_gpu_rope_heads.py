"""GPU: the fused paged writer with head counts whose rows of q take several workgroups, or a last wave with few heads.

A workgroup takes 32 heads of a token, a wave 8: more than 32 heads, one more than 32, 8 and 4.
"""
import pytest

from test_gpu_rope_axes import _writer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv", [(40, 8), (33, 1), (12, 4), (128, 8), (65, 5), (1024, 2), (9, 9)])
@pytest.mark.parametrize("new,old", [([1], [5]), ([70, 1, 9], [0, 200, 63])], ids=str)
def test_writer_heads(new, old, hq, hkv):
    print("writer heads", new, hq, hkv, flush=True)
    _writer(hq + len(new), new, old, hq, hkv)
