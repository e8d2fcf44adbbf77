"""GPU: packed prompts in calls of more than 256 workgroups, which the three-stage kernel serves, and
in calls of a few longer prompts, which the kernel of four key groups serves. Inputs, tolerances (element by
element, against 64 bits) and the check of the rows outside are test_gpu_packed.py's.

Which kernel a call takes goes by its rows, its number of prompts and its heads alone; `workgroups` counts as
the call does, and each case says on which side of the border it stands, so that a border that
moves shows here.
"""
import numpy as np
import pytest

from brasa_amd import Kernels, KvType, PrefillPrecision
from brasa_amd.device import Graph, Stream, synchronize
from test_gpu_packed import Case, _run

pytestmark = pytest.mark.gpu
F16, F32, PF32 = PrefillPrecision.F16, PrefillPrecision.F32, PrefillPrecision.F16_PF32

# prompts of several stages (32 keys each), tiles past the first, one row, none, and one of more than
# 1024 rows: from there on its eighth, not 128 rows, sets where P goes down to one half
LENS = [311, 45, 128, 0, 64, 97, 501, 23, 1, 260, 1100, 77, 333, 190, 32, 33]


def workgroups(c):
    """Workgroups of the call: a bound of the query tiles, times the head groups."""
    hw = next(x for x in (4, 2, 1) if (c.hq // c.hkv) % x == 0)
    tpw = 128 // hw
    tiles = (c.tokens + min(len(c.lens), c.tokens) * (tpw - 1)) // tpw
    return tiles * (c.hq // hw)


def batch(hq, hkv, precision, seed, lens=LENS, before=3, behind=5):
    c = Case(lens, hq, hkv, KvType.F16, precision, seed, before=before, behind=behind)
    assert workgroups(c) > 256  # the three-stage kernel's side
    return c


@pytest.mark.parametrize("precision", [F16, PF32])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (16, 2), (16, 8), (18, 3), (12, 12), (15, 5)])
def test_batches(hq, hkv, precision):
    """Four, two and one head of a group in a workgroup."""
    _run(batch(hq, hkv, precision, hq), f"batch {hq} {hkv} {precision}")


@pytest.mark.parametrize("precision", [F16, PF32])
def test_batches_large_scores(precision):
    """Weights that peak, and a maximum that moves from stage to stage."""
    c = Case(LENS, 16, 4, KvType.F16, precision, 3, before=3, behind=5, q_scale=40.0)
    assert workgroups(c) > 256
    _run(c, f"large scores {precision}")


def _leaks(c, rows, say):
    """NaN and infinities in `rows` of q, k and v leave the bits of all others."""
    print(say, flush=True)
    c.upload()
    c.call(Kernels())
    synchronize()
    c.check()
    clean = c.raw().reshape(c.tokens, -1)
    keep = np.setdiff1d(np.arange(c.tokens), rows)
    for bad in (np.nan, np.inf):
        k, v, q = c.k_raw.copy(), c.v_raw.copy(), c.q.copy()
        k[rows] = v[rows] = q[rows] = bad
        for dev, x in zip(c.dev, (q, k, v)):
            dev.upload(x)
        c.o.upload(c.mark)
        c.call(Kernels())
        synchronize()
        assert np.array_equal(c.raw().reshape(c.tokens, -1)[keep], clean[keep]), bad
    inside = np.intersect1d(rows, np.arange(c.cu[0], c.cu[-1]))
    got = c.raw().reshape(c.tokens, -1)[inside]
    assert inside.size == 0 or not np.array_equal(got, clean[inside])  # (the rows were read at all)


@pytest.mark.parametrize("precision", [F16, PF32])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (16, 8), (12, 12)])
def test_batches_do_not_leak(hq, hkv, precision):
    """Every second prompt, and the rows before and behind all of them, not finite."""
    c = batch(hq, hkv, precision, 8, before=20, behind=70)
    every = [np.arange(c.cu[i], c.cu[i + 1]) for i in range(1, len(c.lens), 2)]
    _leaks(c, np.concatenate([np.arange(20), np.arange(c.cu[-1], c.tokens)] + every), f"leaks {hq} {hkv} {precision}")


@pytest.mark.parametrize("precision", [F16, PF32])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (12, 12)])
def test_batches_repeat_and_replay(hq, hkv, precision):
    """The same bits every time: eager, another stream, a captured call whose cu changes between replays,
    with eager calls between these."""
    k, s, other = Kernels(), Stream(), Stream()
    a = batch(hq, hkv, precision, 9)
    b = batch(hq, hkv, precision, 9, lens=LENS[::-1])
    assert a.tokens == b.tokens and np.array_equal(a.q, b.q)
    want = {}
    for name, c in (("a", a), ("b", b)):
        c.upload()
        c.call(k, other)
        other.synchronize()
        c.check()
        want[name] = c.raw()
    for _ in range(8):
        a.o.upload(a.mark)
        a.call(k, other)
        other.synchronize()
        assert np.array_equal(a.raw(), want["a"])
    with Graph.capture(s) as g:
        a.call(k, s)
    for name in "abba":
        a.dev[3].upload((a if name == "a" else b).cu)
        a.o.upload(a.mark)
        g.launch(s)
        s.synchronize()
        assert np.array_equal(a.raw(), want[name]), name
        b.call(k, other)
        other.synchronize()
        assert np.array_equal(b.raw(), want["b"])


def test_batches_of_more_prompts_than_lanes():
    """150 prompts of 0 to 90 rows: tiles past the first in the second and third 64 prompts."""
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.integers(0, 91, 150)]
    for hq, hkv in ((8, 2), (4, 2), (3, 3)):
        _run(batch(hq, hkv, F16, 4, lens=lens), f"150 prompts {hq} {hkv}")


# ---- f32 accuracy: four key groups of two column blocks -------------------------------------------
def few(hq, hkv, kv, seed, lens, precision=F32, before=3, behind=29):
    c = Case(lens, hq, hkv, kv, precision, seed, before=before, behind=behind)
    assert workgroups(c) <= 192 and c.tokens // 100 >= len(lens)  # the four key groups' side
    return c


@pytest.mark.parametrize("kv,precision", [(KvType.F16, F32), (KvType.F32, F32), (KvType.F32, F16), (KvType.F32, PF32)])
@pytest.mark.parametrize("hq,hkv", [(16, 8), (8, 8), (8, 2), (6, 2)])
def test_few_long_prompts(hq, hkv, kv, precision):
    _run(few(hq, hkv, kv, 5, [130, 257, 1, 600], precision), f"few {hq} {hkv} {kv} {precision}")


@pytest.mark.parametrize("kv", [KvType.F16, KvType.F32])
@pytest.mark.parametrize("hq,hkv", [(16, 8), (8, 8), (8, 2)])
def test_few_long_prompts_do_not_leak(hq, hkv, kv):
    c = few(hq, hkv, kv, 6, [150, 37, 190], before=20, behind=70)
    _leaks(c, np.r_[0:20, 170:207, 397:467], f"few leaks {hq} {hkv} {kv}")
