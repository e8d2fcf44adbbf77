"""CPU: arrays of a step's calls that overlap what the call writes are refused before the device is touched."""
import pytest

from brasa_amd import BrasaError, Kernels, KvPool, OutDType, RopeAxes, RopeTable, attention_paged_workspace_len

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


@pytest.mark.parametrize("out,size", [(OutDType.F32, 4), (OutDType.F16, 2)])
def test_attention_over_its_table(out, size):
    n, width, tokens, hq, base, ws = 3, 5, 7, 32, 1 << 40, 1 << 36
    need = attention_paged_workspace_len(n, 0, tokens, hq, 8)
    for table in (base, base - 4 * n * width + 4, base + size * tokens * hq * 128 - 4, ws + 4096, ws + need - 4):
        _refused(lambda: Kernels().attention_paged(P, KvPool.view(P, P, P, P, 1, 8, 8), 0, table, n, width, tokens, ws, need, base, hq, out))


@pytest.mark.parametrize("name,size", [("rope_pos", 4 * 2 * 9), ("cu", 4 * 4), ("pos", 4 * 3), ("pages", 4 * 3 * 5), ("qn", 512), ("kn", 512),
                                       ("cos", 4 * 64 * 10), ("sin", 4 * 64 * 10)])
def test_writer_over_its_inputs(name, size):
    n, width, tokens, hq, hkv, q, k = 3, 5, 9, 32, 8, 1 << 40, 1 << 41
    for at in (q, q - size + 4, q + 4 * tokens * hq * 128 - 4, k, k - size + 4, k + 4 * tokens * hkv * 128 - 4):
        a = {**dict(rope_pos=P, cu=P, pos=P, pages=P, qn=P, kn=P, cos=P, sin=P), name: at}
        _refused(lambda: Kernels().qk_norm_rope_store_paged(
            KvPool.view(P, P, P, P, 1, 8, hkv), 0, (q, k, 1 << 42), (a["qn"], a["kn"]), 1e-6, RopeTable.view(a["cos"], a["sin"], 128, 10),
            RopeAxes([60, 4]), a["rope_pos"], a["cu"], a["pos"], a["pages"], n, width, tokens, hq))


@pytest.mark.parametrize("name,size", [("pos", 4 * 2 * 9), ("cos", 4 * 36 * 10), ("sin", 4 * 36 * 10)])
def test_rotation_over_its_inputs(name, size):
    tokens, heads, dim, x = 9, 3, 72, 1 << 40
    for at in (x, x - size + 4, x + 4 * tokens * heads * dim - 4):
        a = {**dict(pos=P, cos=P, sin=P), name: at}
        _refused(lambda: Kernels().rope_axes(x, RopeTable.view(a["cos"], a["sin"], dim, 10), RopeAxes([30, 6]), a["pos"], tokens, heads, dim))
