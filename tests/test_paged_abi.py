"""CPU: the packed and paged entry points refuse bad calls before they touch the device, and the
sizes they publish; the reference's own e4m3 against its definition."""
import numpy as np
import pytest

import paged_ref as ref
from brasa_amd import (AttnShape, BrasaError, Kernels, KvPool, KvType, OutDType, PrefillPrecision,
                       decode_paged_workspace_len, kv_pages_workspace_len, kv_pool_bytes)

P = 4096  # an address that passes the checks of null and alignment; never followed here
POOL = dict(k=P, v=P, k_exp=P, v_exp=P, layers=2, pages=8, hkv=8)
ARG, SHAPE, SCRATCH, UNSUPPORTED = 5, 1, 2, 3


def _pool(**over):
    return KvPool.view(**{**POOL, **over})


def _refused(code, call):
    with pytest.raises(BrasaError) as e:
        call()
    assert e.value.code == code, str(e.value)


@pytest.mark.parametrize("code,over", [
    (UNSUPPORTED, {"kv": KvType.Q8_0}), (SHAPE, {"dim": 64}), (SHAPE, {"hkv": 5}), (SHAPE, {"hkv": 0}),
    (SHAPE, {"hq": 0}), (SHAPE, {"pos0": 1}), (SHAPE, {"tokens": 1 << 30}), (SHAPE, {"n": 65537}),
    (ARG, {"precision": 7}), (ARG, {"kv": 9}), (ARG, {"q": 0}), (ARG, {"k": 0}), (ARG, {"v": 0}),
    (ARG, {"o": 0}), (ARG, {"cu": 0}), (ARG, {"q": P + 4}), (ARG, {"o": P + 8}),
])
def test_packed_refusals(code, over):
    a = {**dict(q=P, k=P, v=P, o=P, cu=P, n=2, tokens=5, hq=32, hkv=8, dim=128, pos0=0, kv=KvType.F16,
                precision=PrefillPrecision.F16), **over}
    shape = AttnShape(a["tokens"], a["hq"], a["hkv"], a["dim"], a["pos0"], a["kv"])
    _refused(code, lambda: Kernels().flash_attention_packed(a["q"], a["k"], a["v"], a["o"], a["cu"], a["n"],
                                                            shape, a["precision"]))


def test_packed_nothing_to_do():
    for tokens, n in ((0, 3), (5, 0)):
        Kernels().flash_attention_packed(0, 0, 0, 0, 0, n, AttnShape(tokens, 32, 8, 128, 0, KvType.F16))


@pytest.mark.parametrize("code,pool,over", [
    (SHAPE, {"dim": 64}, {}), (SHAPE, {"hkv": 0}, {}), (SHAPE, {"hkv": 2000}, {}), (SHAPE, {"pages": 0}, {}),
    (SHAPE, {"layers": 0}, {}), (SHAPE, {"pages": 1 << 25}, {}), (SHAPE, {"layers": 1 << 40}, {}),
    (SHAPE, {}, {"layer": 2}), (ARG, {"k": 0}, {}), (ARG, {"v_exp": 0}, {}), (ARG, {"v": P + 8}, {}),
    (SHAPE, {}, {"n": 65537}), (SHAPE, {}, {"width": 1 << 25}), (SHAPE, {}, {"n": 1 << 15, "width": 1 << 16}),
])
def test_pool_refusals(code, pool, over):
    a = {**dict(layer=0, n=2, width=4), **over}
    p, k = _pool(**pool), Kernels()
    _refused(code, lambda: k.store_kv_paged(p, a["layer"], P, P, P, P, P, a["n"], a["width"], 5))
    _refused(code, lambda: k.decode_attention_paged(P, p, a["layer"], P, P, a["n"], a["width"], P, 1 << 30,
                                                    P, 32))
    if "layer" not in over:
        _refused(code, lambda: k.kv_pages_reserve(p, P, P, P, P, P, P, P, a["n"], a["width"], P, 1 << 40))
        _refused(code, lambda: k.kv_pages_compact(p, P, P, P, P, P, a["n"], a["width"], P, 1 << 40))


def test_store_refusals():
    k, p = Kernels(), _pool()
    for i in range(5):
        args = [P] * 5
        args[i] = 0
        _refused(ARG, lambda: k.store_kv_paged(p, 0, *args, 2, 4, 5))
    _refused(ARG, lambda: k.store_kv_paged(p, 0, P + 4, P, P, P, P, 2, 4, 5))
    _refused(SHAPE, lambda: k.store_kv_paged(p, 0, P, P, P, P, P, 2, 4, 1 << 29))
    k.store_kv_paged(p, 0, 0, 0, 0, 0, 0, 0, 4, 5)
    k.store_kv_paged(p, 0, 0, 0, 0, 0, 0, 2, 4, 0)


def test_decode_refusals():
    k, p, w = Kernels(), _pool(), decode_paged_workspace_len(32, 8)
    call = lambda **o: k.decode_attention_paged(*[{**dict(  # noqa: E731
        q=P, pool=p, layer=0, table=P, lk=P, n=2, width=4, ws=P, wlen=w, o=P, hq=32,
        out=OutDType.F32), **o}[x] for x in ("q", "pool", "layer", "table", "lk", "n", "width", "ws", "wlen",
                                             "o", "hq", "out")])
    for name in ("q", "table", "lk", "ws", "o"):
        _refused(ARG, lambda: call(**{name: 0}))
    _refused(ARG, lambda: call(out=3))
    _refused(ARG, lambda: call(ws=P + 16))
    _refused(ARG, lambda: call(q=P + 4))
    _refused(ARG, lambda: call(o=P + 8))
    _refused(SCRATCH, lambda: call(wlen=w - 1))
    _refused(SHAPE, lambda: call(hq=30))
    _refused(SHAPE, lambda: call(hq=0))
    _refused(SHAPE, lambda: call(hq=2048))
    call(n=0, q=0, table=0, lk=0, ws=0, o=0)


def test_pages_refusals():
    k, p = Kernels(), _pool()
    w = kv_pages_workspace_len(8, 2, 4)
    for i in range(7):
        args = [P, P, P, P, 2 * P, 2 * P, P]
        args[i] = 0
        _refused(ARG, lambda: k.kv_pages_fork(*args, 2, 4, 8))
    _refused(ARG, lambda: k.kv_pages_fork(P, P, P, P, P, 2 * P, P, 2, 4, 8))
    _refused(ARG, lambda: k.kv_pages_fork(P, P, P, P, 2 * P, P, P, 2, 4, 8))
    _refused(SHAPE, lambda: k.kv_pages_fork(P, P, P, P, 2 * P, 2 * P, P, 2, 4, 0))
    _refused(SHAPE, lambda: k.kv_pages_fork(P, P, P, P, 2 * P, 2 * P, P, 2, 0, 8))
    for i in range(7):
        args = [P] * 7
        args[i] = 0
        _refused(ARG, lambda: k.kv_pages_reserve(p, *args, 2, 4, P, w))
    _refused(SCRATCH, lambda: k.kv_pages_reserve(p, *[P] * 7, 2, 4, P, w - 1))
    _refused(ARG, lambda: k.kv_pages_reserve(p, *[P] * 7, 2, 4, 0, w))
    _refused(ARG, lambda: k.kv_pages_reserve(p, *[P] * 7, 2, 4, P + 8, w))
    for i in range(5):
        args = [P] * 5
        args[i] = 0
        _refused(ARG, lambda: k.kv_pages_compact(p, *args, 2, 4, P, w))
    _refused(SCRATCH, lambda: k.kv_pages_compact(p, *[P] * 5, 2, 4, P, w - 1))


def test_sizes():
    assert kv_pool_bytes(3, 5, 8) == 3 * 5 * 8 * 64 * 128
    assert _pool().bytes() == 2 * (kv_pool_bytes(2, 8, 8) + 2 * 8 * 8)
    assert decode_paged_workspace_len(32, 8) > 0 and decode_paged_workspace_len(30, 8) == 0
    assert kv_pages_workspace_len(1 << 25, 1, 1) == 0


def test_reference_codes():
    """The reference's encoder against every code, every midpoint and what lies next to one."""
    codes = np.r_[np.arange(127), np.arange(128, 255)].astype(np.uint8)
    assert np.array_equal(ref.encode(ref.E4M3[codes]), codes)
    a, b = ref.E4M3[:126], ref.E4M3[1:127]
    mid = (a + b) / 2
    even = np.where(np.arange(126) % 2 == 0, np.arange(126), np.arange(1, 127))
    assert np.array_equal(ref.encode(mid), even)
    assert np.array_equal(ref.encode(np.nextafter(mid, 0)), np.arange(126))
    assert np.array_equal(ref.encode(np.nextafter(mid, 1e3)), np.arange(1, 127))
    assert list(ref.encode(np.array([np.nan, np.inf, -np.inf]))) in ([127, 127, 255], [255, 127, 255])
    assert [ref.scale_byte(x) for x in (0.0, 448.0, 448.01, 1.0, 1.75, 1.76)] == [0, 127, 128, 119, 119, 120]
