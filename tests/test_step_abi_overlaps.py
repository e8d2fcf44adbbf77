"""CPU: arrays of a step's calls that overlap what the call writes are refused before the device is touched."""
import pytest

from brasa_amd import BrasaError, Kernels, KvPool, OutDType, attention_paged_workspace_len

P = 4096  # an address that passes the checks of null and alignment; never followed here
ARG = 5


def _refused(call):
    with pytest.raises(BrasaError) as e:
        call()
    assert e.value.code == ARG, str(e.value)


@pytest.mark.parametrize("groups", [1, 3, 64, 5000])
def test_attention_inside_a_grouped_workspace(groups):
    """q or o in the part of the workspace that only a plan with groups takes."""
    n, tokens, hq, hkv, base = 64, 64, 32, 8, 1 << 40
    alone, size = (attention_paged_workspace_len(n, g, tokens, hq, hkv) for g in (0, groups))
    assert size > alone + (2 << 20)
    for at in (alone, alone + 1024, size - 256):
        for q, o in ((base + at, P), (P, base + at)):
            _refused(lambda: Kernels().attention_paged(q, KvPool.view(P, P, P, P, 1, 8, hkv), 0, P, n, 4, tokens, base, size, o, hq,
                                                       OutDType.F32))


@pytest.mark.parametrize("name,size", [("cu", 4 * 65), ("pos", 4 * 64), ("group", 16), ("prefix", 12)])
def test_plan_inputs_inside_the_workspace(name, size):
    n, groups, tokens, hq, hkv, base = 64, 3, 64, 32, 8, 1 << 40
    need = attention_paged_workspace_len(n, groups, tokens, hq, hkv)
    for at in (base, base + 4096, base + need - 4, base - size + 4):
        a = {**dict(cu=P, pos=P, group=P, prefix=P), name: at}
        _refused(lambda: Kernels().attention_paged_plan(**a, groups=groups, n=n, width=4, tokens=tokens, hq=hq, hkv=hkv,
                                                        workspace=base, workspace_len=need))
