"""CPU: the calls of a step's maps, rotary axes and attention of new rows refuse bad arguments before they
touch the device; sizes and axis maps; their host references against hand-made values."""
import numpy as np
import pytest

import step_ref
from brasa_amd import (BrasaError, Kernels, KvPool, OutDType, RopeAxes, RopeTable, attention_paged_workspace_len)

P = 4096  # an address that passes the checks of null and alignment; never followed here
ARG, SHAPE, SCRATCH = 5, 1, 2


def _refused(code, call):
    with pytest.raises(BrasaError) as e:
        call()
    assert e.value.code == code, str(e.value)


@pytest.mark.parametrize("code,over", [
    (SHAPE, {"n": 65537}), (SHAPE, {"n": 0}), (SHAPE, {"width": 1 << 25}), (SHAPE, {"pages": 0}),
    (SHAPE, {"pages": 1 << 25}), (SHAPE, {"tokens": (1 << 30) + 1}), (ARG, {"add": 0}), (ARG, {"lens": 0}),
    (ARG, {"table": 0}), (ARG, {"lk": P}), (ARG, {"cu": P + 64}),
])
def test_rows_refusals(code, over):
    a = {**dict(add=P + 64, lens=P, table=P, n=2, width=3, pages=9, tokens=5, cu=P + 128, lk=P + 192, slot=P + 256), **over}
    _refused(code, lambda: Kernels().kv_rows(**a))


@pytest.mark.parametrize("code,over", [
    (SHAPE, {"n": 65537}), (SHAPE, {"groups": 65537}), (SHAPE, {"pages": 0}), (ARG, {"group": 0}), (ARG, {"prefix": 0}),
    (ARG, {"table": 0}), (ARG, {"lens": 0}),
])
def test_shared_refusals(code, over):
    a = {**dict(table=P, lens=P, group=P, groups=1, n=2, width=3, pages=9, prefix=P), **over}
    _refused(code, lambda: Kernels().kv_pages_shared(**a))


def test_nothing_to_do():
    k, t = Kernels(), RopeTable.view(P, P, 128, 10)
    pool = KvPool.view(P, P, P, P, 1, 8, 8)
    k.kv_pages_shared(0, 0, 0, 0, 2, 3, 9, 0)
    for tokens, heads in ((0, 4), (4, 0)):
        k.rope_axes(0, t, RopeAxes([64]), 0, tokens, heads, 128)
    for n, tokens in ((0, 3), (3, 0)):
        k.qk_norm_rope_store_paged(pool, 0, (0, 0, 0), (0, 0), 1e-6, t, RopeAxes([64]), 0, 0, 0, 0, n, 4, tokens, 32)
        k.attention_paged(0, pool, 0, 0, n, 4, tokens, 0, 1 << 40, 0, 32)


@pytest.mark.parametrize("code,over", [
    (SHAPE, {"dim": 64}), (SHAPE, {"heads": 1025}), (SHAPE, {"tokens": (1 << 30) + 1}), (ARG, {"x": 0}), (ARG, {"pos": 0}),
    (ARG, {"x": P + 2}), (ARG, {"table": RopeTable.view(0, P, 128, 10)}), (SHAPE, {"axes": RopeAxes.of_pairs([0] * 64, 5)}),
    (SHAPE, {"axes": RopeAxes.of_pairs([0] * 64, 0)}), (ARG, {"axes": RopeAxes.of_pairs([0] * 63 + [2], 2)}),
    (SHAPE, {"axes": RopeAxes([63])}), (SHAPE, {"table": RopeTable.view(P, P, 258, 10), "dim": 258}),
])
def test_rope_refusals(code, over):
    a = {**dict(x=P, table=RopeTable.view(P, P, 128, 10), axes=RopeAxes([24, 20, 20]), pos=P, tokens=3, heads=2, dim=128), **over}
    _refused(code, lambda: Kernels().rope_axes(**a))


@pytest.mark.parametrize("code,over", [
    (SHAPE, {"layer": 2}), (SHAPE, {"n": 65537}), (SHAPE, {"tokens": 1 << 26}), (SHAPE, {"hq": 1025}),
    (SHAPE, {"table": RopeTable.view(P, P, 64, 10)}), (SHAPE, {"table": RopeTable.view(P, P, 128, 0)}),
    (ARG, {"qkv": (0, P, P)}), (ARG, {"qkv": (P, 0, P)}), (ARG, {"qkv": (P, P, 0)}), (ARG, {"qkv": (P, P + 4, P)}),
    (ARG, {"norms": (P, 0)}), (ARG, {"rope_pos": 0}), (ARG, {"cu": 0}), (ARG, {"pos": 0}), (ARG, {"pages": 0}),
    (SHAPE, {"axes": RopeAxes([32])}),
])
def test_writer_refusals(code, over):
    a = {**dict(pool=KvPool.view(P, P, P, P, 2, 8, 8), layer=1, qkv=(P, P, P), norms=(P, P), eps=1e-6,
                table=RopeTable.view(P, P, 128, 10), axes=RopeAxes([64]), rope_pos=P, cu=P, pos=P, pages=P, n=2,
                width=3, tokens=5, hq=32), **over}
    _refused(code, lambda: Kernels().qk_norm_rope_store_paged(**a))


@pytest.mark.parametrize("code,over", [
    (SHAPE, {"n": 65537}), (SHAPE, {"groups": 65537}), (SHAPE, {"hq": 30}), (SHAPE, {"hq": 0}), (SHAPE, {"hkv": 0}),
    (SHAPE, {"hq": 2048}), (SHAPE, {"tokens": 1 << 25}), (SHAPE, {"n": 1 << 15, "width": 1 << 16}), (SCRATCH, {"workspace_len": 1000}),
    (ARG, {"workspace": 0}), (ARG, {"workspace": P + 16}), (ARG, {"cu": 0}), (ARG, {"pos": 0}), (ARG, {"group": 0}), (ARG, {"prefix": 0}),
])
def test_plan_refusals(code, over):
    a = {**dict(cu=P, pos=P, group=P, prefix=P, groups=1, n=2, width=4, tokens=5, hq=32, hkv=8, workspace=P,
                workspace_len=1 << 40), **over}
    _refused(code, lambda: Kernels().attention_paged_plan(**a))


@pytest.mark.parametrize("code,over", [
    (SHAPE, {"n": 65537}), (SHAPE, {"layer": 1}), (SHAPE, {"hq": 30}), (SHAPE, {"tokens": 1 << 25}), (SCRATCH, {"workspace_len": 1000}),
    (ARG, {"workspace": 0}), (ARG, {"workspace": P + 16}), (ARG, {"q": 0}), (ARG, {"o": 0}), (ARG, {"table": 0}), (ARG, {"q": P + 4}),
    (ARG, {"o": P + 8}), (ARG, {"out": 7}),
])
def test_attention_refusals(code, over):
    a = {**dict(q=P, pool=KvPool.view(P, P, P, P, 1, 8, 8), layer=0, table=P, n=2, width=4, tokens=5, workspace=P,
                workspace_len=1 << 40, o=P, hq=32, out=OutDType.F32), **over}
    _refused(code, lambda: Kernels().attention_paged(**a))


@pytest.mark.parametrize("over", [
    {"lk": P + 4}, {"cu": P + 68}, {"cu": P - 8}, {"lk": P + 64}, {"seq": P + 60}, {"slot": P + 512}, {"pos": P + 512 + 20},
    {"slot": P + 192}, {"seq": P + 256, "pos": P + 272}], ids=str)
def test_rows_overlaps(over):
    a = {**dict(add=P + 64, lens=P, table=P + 512, n=2, width=3, pages=9, tokens=5, cu=P + 128, lk=P + 192, slot=P + 256), **over}
    _refused(ARG, lambda: Kernels().kv_rows(**a))


@pytest.mark.parametrize("prefix", [P, P + 4, P + 68, P + 140, P - 4])
def test_shared_overlaps(prefix):
    _refused(ARG, lambda: Kernels().kv_pages_shared(table=P + 128, lens=P + 64, group=P, groups=2, n=2, width=3, pages=9,
                                                   prefix=prefix))


@pytest.mark.parametrize("qkv", [(P, P, 1 << 30), (1 << 30, P, P), (P, 1 << 30, P), (P, P + 5 * 32 * 512 - 16, 1 << 30),
                                 (1 << 30, P, P + 5 * 8 * 512 - 16)])
def test_writer_overlaps(qkv):
    _refused(ARG, lambda: Kernels().qk_norm_rope_store_paged(
        KvPool.view(P, P, P, P, 2, 8, 8), 1, qkv, (P, P), 1e-6, RopeTable.view(P, P, 128, 10), RopeAxes([64]), P, P, P, P, 2, 3, 5, 32))


@pytest.mark.parametrize("out,size", [(OutDType.F32, 4), (OutDType.F16, 2)])
def test_attention_overlaps(out, size):
    base, values = 1 << 40, 5 * 32 * 128
    need = attention_paged_workspace_len(2, 0, 5, 32, 8)
    for q, o, ws in ((base, base, P), (base, base + 4 * values - 16, P), (base + size * values - 16, base, P),
                     (P, base, base), (base, P, base + 1024), (base + need - need % 16 - 16, P, base)):
        _refused(ARG, lambda: Kernels().attention_paged(q, KvPool.view(P, P, P, P, 1, 8, 8), 0, P, 2, 4, 5, ws, need, o, 32, out))


def test_workspace_len():
    assert attention_paged_workspace_len(2, 0, 4, 30, 8) == 0
    for n, groups, tokens, hq, hkv in ((1, 0, 1, 32, 8), (64, 3, 64, 32, 8), (3, 1, 9000, 8, 8), (100, 2, 100, 128, 1)):
        size = attention_paged_workspace_len(n, groups, tokens, hq, hkv)
        assert size % 256 == 0 and size >= attention_paged_workspace_len(n, 0, tokens, hq, hkv)
        assert attention_paged_workspace_len(n, groups, tokens + 50, hq, hkv) >= size


def test_axes():
    a = RopeAxes([24, 20, 20], interleaved=True)
    assert list(a.c(128).of[:64]) == [0, 1, 2] * 20 + [0] * 4
    assert list(RopeAxes([3, 0, 2]).c(10).of[:5]) == [0, 0, 0, 2, 2]
    assert RopeAxes.of_pairs([1, 0]).axes == 2
    with pytest.raises(BrasaError):
        RopeAxes([200])
    with pytest.raises(BrasaError):
        RopeAxes([5, -1])


def test_references():
    """The host references on values made by hand."""
    table = np.array([[3, 5], [7, -1]])
    cu, lk, seq, pos, slot = step_ref.rows([2, 3], [63, 62], table, 8, 6)
    assert list(cu) == [0, 2, 5] and list(lk) == [65, 65] and list(seq) == [0, 0, 1, 1, 1, -1]
    assert list(pos) == [63, 64, 62, 63, 64, -1] and list(slot) == [3 * 64 + 63, 5 * 64, 7 * 64 + 62, 7 * 64 + 63, -1, -1]
    assert list(step_ref.shared(np.array([[1, 2, 3], [1, 2, 4], [9, 9, 9]]), [200, 130, 0], [0, 3], 10)) == [128]
    x = np.array([[[1.0, 2.0, 3.0, 4.0]]])
    cos, sin = np.array([[1.0, 1.0], [0.0, 0.5]]), np.array([[0.0, 0.0], [1.0, 0.25]])
    y = step_ref.rope(x, cos, sin, [0, 1], np.array([[1], [0]]))
    assert np.array_equal(y, [[[-3.0, 2.0, 1.0, 4.0]]])
    q = np.zeros((2, 1, 128))
    v = np.arange(3.0)[:, None, None] * np.ones((3, 1, 128))
    o, _, _ = step_ref.attend(q, np.zeros((3, 1, 128)), v, 1)
    assert np.allclose(o[:, 0, 0], [0.5, 1.0])
