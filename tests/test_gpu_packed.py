"""GPU: causal attention over packed prompts against 64 bits.

Tolerances, by element. A score errs by at most A * e_s, A its row's largest sum of |q k| / sqrt(128):
e_s is half a step of the f16 rounding of q / sqrt(128) (2^-11) where the precision rounds it, and 2^-21
where it keeps hi + lo halves (2^-22) of both factors, plus 128 + 4 roundings of f32 sums and products
(2^-24 each). A weight errs by that, by 2^-11 where it is rounded to f16, and by a few f32 roundings;
numerator and denominator both carry it, so o errs by twice that times the weighted sum of |v|. Sums over
lk keys in f32 add at most lk * 2^-24 of it (a lane adds its keys one by one). f16 rows of v are exact,
f32 rows of v in two halves 2^-21. An f16 result adds half a step, 2^-11 of it (2^-25 below f16's normal
range). A weight below f16's normal range errs by half of f16's smallest step, 2^-25, where the row's
largest weight is at least 1: o by 2^-25 of the sum of |v|. The halves have the same floor: the lo half of an
f32 value x errs by 2^-22 |x| or, where it is below f16's normal range, by 2^-25 (x = hi + lo + e with
|lo| <= 2^-11 |x|, and f16 steps by 2^-24 below 2^-14). That is 2^-25 in every v (o errs by as much, the
weights' sum being 1), in every k (a score by 2^-25 of the sum of |q| / sqrt(128)) and in every
q / sqrt(128) (a score by 2^-25 of the largest sum of |k|).
"""
import numpy as np
import pytest

import oracle
import paged_ref as ref
from brasa_amd import AttnShape, Kernels, KvType, PrefillPrecision
from brasa_amd.device import DeviceBuffer, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu
F16, F32, PF32 = PrefillPrecision.F16, PrefillPrecision.F32, PrefillPrecision.F16_PF32


def _rows(rng, kv, tokens, hkv, scale=1.0):
    x = (scale * rng.standard_normal((tokens, hkv, 128))).astype(np.float32)
    if kv == KvType.F16:
        h = x.astype(np.float16)
        return h.astype(np.float32), h
    return x, x


class Case:
    def __init__(self, lens, hq, hkv, kv, precision, seed, before=0, behind=0, q_scale=1.0):
        rng = np.random.default_rng(seed)
        self.lens, self.hq, self.hkv, self.kv, self.precision = lens, hq, hkv, kv, precision
        self.tokens = before + sum(lens) + behind
        self.cu = (before + np.r_[0, np.cumsum(lens)]).astype(np.int32)
        self.q = (q_scale * rng.standard_normal((self.tokens, hq, 128))).astype(np.float32)
        self.k, self.k_raw = _rows(rng, kv, self.tokens, hkv)
        self.v, self.v_raw = _rows(rng, kv, self.tokens, hkv)
        self.f32_out = precision == F32

    def upload(self):
        self.dev = [DeviceBuffer.from_array(x) for x in (self.q, self.k_raw, self.v_raw, self.cu)]
        kind = np.float32 if self.f32_out else np.uint16
        self.mark = np.full(self.tokens * self.hq * 128, 7 if self.f32_out else 0x4700, kind)
        self.o = DeviceBuffer.from_array(self.mark)

    def shape(self):
        return AttnShape(self.tokens, self.hq, self.hkv, 128, 0, self.kv)

    def call(self, kernels, stream=None):
        q, k, v, cu = self.dev
        kernels.flash_attention_packed(q, k, v, self.o, cu, len(self.lens), self.shape(), self.precision,
                                       stream)

    def raw(self):
        return self.o.download(np.float32 if self.f32_out else np.uint16)

    def check(self, raw=None):
        raw = self.raw() if raw is None else raw
        got = raw if self.f32_out else oracle.f16_to_f32(raw)
        got = got.astype(np.float64).reshape(self.tokens, self.hq, 128)
        f16 = self.precision != F32
        e_s = (2.0 ** -11 if f16 else 0) + 2.0 ** -21 + 132 * 2.0 ** -24
        e_p = (2.0 ** -11 if self.precision == F16 else 2.0 ** -21) + 8 * 2.0 ** -24
        worst = 0.0
        for a, b in zip(self.cu, self.cu[1:]):
            if a == b:
                continue
            o, av, top = ref.attend(self.q[a:b], self.k[a:b].astype(np.float64),
                                    self.v[a:b].astype(np.float64), True)
            tol = av * (2 * (top * e_s + e_p) + 2.0 ** -21 + (b - a + 64) * 2.0 ** -24) + 1e-30
            tol += 2.0 ** -25 * np.abs(self.v[a:b].astype(np.float64)).sum(0).repeat(self.hq // self.hkv, 0)
            floor = np.abs(self.q[a:b]).sum(-1, keepdims=True) / np.sqrt(128.0) + \
                np.abs(self.k[a:b]).sum(-1).max()
            tol += 2.0 ** -25 * (2 * floor * av + 1)
            if f16:
                tol += np.abs(o) * 2.0 ** -11 + 2.0 ** -25
            err = np.abs(got[a:b] - o)
            worst = max(worst, float((err / tol).max()))
            assert np.all(err <= tol), (a, b, float((err / tol).max()))
        outside = np.r_[0:self.cu[0], self.cu[-1]:self.tokens].astype(int)
        rows = raw.reshape(self.tokens, -1)[outside]
        assert np.array_equal(rows, self.mark.reshape(self.tokens, -1)[outside]), "rows outside were written"
        return worst


LENS = [[1], [0, 1, 0], [65, 64, 63], [129, 1, 300, 0, 2, 31, 33], [700], [32] * 5, [256, 257, 255]]


def _run(c, say):
    print(say, flush=True)
    c.upload()
    c.call(Kernels())
    synchronize()
    print("  worst error / tolerance", c.check(), flush=True)


@pytest.mark.parametrize("precision,kv", [(F16, KvType.F16), (PF32, KvType.F16), (F32, KvType.F16),
                                          (F32, KvType.F32), (F16, KvType.F32), (PF32, KvType.F32)])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
def test_packed(lens, precision, kv):
    _run(Case(lens, 8, 2, kv, precision, len(lens), before=3, behind=5), f"{lens} {precision} {kv}")


@pytest.mark.parametrize("precision,kv", [(F16, KvType.F16), (F32, KvType.F32)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (4, 2), (16, 2), (6, 2), (5, 1), (7, 1), (24, 2)])
def test_packed_heads(hq, hkv, precision, kv):
    _run(Case([70, 1, 140], hq, hkv, kv, precision, hq), f"heads {hq} {hkv}")


@pytest.mark.parametrize("precision,kv", [(F16, KvType.F16), (F32, KvType.F32)])
def test_packed_many_short(precision, kv):
    """More prompts than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(1)
    _run(Case([int(x) for x in rng.integers(0, 9, 333)], 4, 2, kv, precision, 5), "333 short prompts")


@pytest.mark.parametrize("precision,kv", [(F16, KvType.F16), (F32, KvType.F32)])
def test_packed_most_prompts(precision, kv):
    """As many prompts as a call takes, of one row each: more query tiles than one grid holds. Each
    row's result is its own v, weight 1."""
    n = 65536
    c = Case([1] * n, 1, 1, kv, precision, 11)
    c.upload()
    c.call(Kernels())
    synchronize()
    raw = c.raw()
    got = (raw if c.f32_out else oracle.f16_to_f32(raw)).reshape(n, 128)
    # f32 rows: two halves, 2^-22 of the value or 2^-25; f16 rows are exact
    assert np.all(np.abs(got - c.v[:, 0]) <= (0 if kv == KvType.F16 else 2.0 ** -22 * np.abs(c.v[:, 0]) + 2.0 ** -25))


@pytest.mark.parametrize("precision,kv", [(F16, KvType.F16), (F32, KvType.F32)])
def test_packed_long(precision, kv):
    _run(Case([1500, 40, 2100], 4, 1, kv, precision, 6), "long")


@pytest.mark.parametrize("precision,kv", [(F16, KvType.F16), (F32, KvType.F16)])
def test_packed_large_scores(precision, kv):
    """Peaked weights: scores of hundreds, whose maximum moves from key to key."""
    _run(Case([200, 333], 4, 1, kv, precision, 7, q_scale=40.0), "large scores")


@pytest.mark.parametrize("kv", [KvType.F16, KvType.F32])
@pytest.mark.parametrize("precision", [F16, F32])
def test_packed_neighbours_do_not_leak(kv, precision):
    """NaN and infinities in the rows before, behind and of another prompt leave the others' bits."""
    c = Case([50, 37, 90], 8, 2, kv, precision, 8, before=20, behind=70)
    c.upload()
    c.call(Kernels())
    synchronize()
    clean = c.raw().reshape(c.tokens, -1)
    for bad in (np.nan, np.inf):
        k, v, q = c.k_raw.copy(), c.v_raw.copy(), c.q.copy()
        rows = np.r_[0:20, 70:107, 197:267]
        k[rows] = v[rows] = q[rows] = bad
        for dev, x in zip(c.dev, (q, k, v)):
            dev.upload(x)
        c.o.upload(c.mark)
        c.call(Kernels())
        synchronize()
        got = c.raw().reshape(c.tokens, -1)
        keep = np.r_[0:70, 107:267]
        assert np.array_equal(got[keep], clean[keep]), bad


@pytest.mark.parametrize("precision,kv", [(F16, KvType.F16), (F32, KvType.F32)])
def test_packed_repeats_and_replays(precision, kv):
    """The same bits every time: eager, another stream, a graph whose cu changes between replays."""
    k, s, other = Kernels(), Stream(), Stream()
    a = Case([300, 20, 511], 8, 2, kv, precision, 9)
    b = Case([100, 700, 31], 8, 2, kv, precision, 9)
    assert a.tokens == b.tokens and np.array_equal(a.q, b.q)
    want = {}
    for name, c in (("a", a), ("b", b)):
        c.upload()
        c.call(k, other)
        other.synchronize()
        c.check()
        want[name] = c.raw()
    a.o.upload(a.mark)
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
    for _ in range(3):
        g.launch(s)
    s.synchronize()
    assert np.array_equal(a.raw(), want["a"])


def test_packed_clamps_cu():
    """Row numbers past the rows are clamped: the prompt ends with the arrays."""
    for kv, precision in ((KvType.F16, F16), (KvType.F32, F32)):
        c = Case([40, 61], 8, 2, kv, precision, 10)
        c.upload()
        c.dev[3].upload(np.array([-5, 40, 1 << 30], np.int32))
        c.call(Kernels())
        synchronize()
        c.check()
