"""GPU: the paged 8-bit cache's writer (bytes for bytes) and its decode attention (against 64 bits).

The decode's tolerance, by element: a score errs by at most A * e_s, A its row's largest sum of
|q k| / sqrt(128): q / sqrt(128) * log2 e in two f16 halves (2^-22), its f32 rounding and product
(2 * 2^-24), 128 + 2 roundings of f32 sums, exp2 and its argument (|s| * 2^-24 with |s| <= A); a weight
in two halves adds 2^-22 and a few roundings; numerator and denominator both carry it. Sums over lk keys
in f32: a chain of at most lk / 16 + 200 additions. An f16 result adds 2^-11 of itself.
A weight below f16's normal range has an absolute error instead: its lo half errs by half of f16's
smallest step, 2^-25, where the row's largest weight is at least 2^7 (a weight is
2^(s - m + 7) with m one of the row's scores, so at most the largest). Relative to that largest weight
it is 2^-32, and the denominator is at least the largest weight: o errs by at most 2^-32 times the
sum of |v|, which is more than all the rest where the largest weights meet values near 0.
"""
import numpy as np
import pytest

import oracle
import paged_ref as ref
from brasa_amd import Kernels, KvPool, OutDType, decode_paged_workspace_len
from brasa_amd.device import DeviceBuffer, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu
PAGE = ref.PAGE


def ints(x):
    return DeviceBuffer.from_array(np.asarray(x, np.int32))


def upload_pool(pool: ref.Pool) -> KvPool:
    return KvPool.view(*(DeviceBuffer.from_array(a) for a in pool.arrays()), pool.layers, pool.pages, pool.hkv)


def pool_bytes(dev: KvPool, like: ref.Pool):
    return [b.download(np.uint8).reshape(a.shape) for b, a in zip((dev.k, dev.v, dev.k_exp, dev.v_exp),
                                                                  like.arrays())]


def assert_pool(dev: KvPool, want: ref.Pool):
    for name, got, w in zip(("k", "v", "k_exp", "v_exp"), pool_bytes(dev, want), want.arrays()):
        assert np.array_equal(got, w), (name, np.argwhere(got != w)[:5].tolist())


def random_table(rng, counts, pages, width):
    ids = rng.permutation(pages)[:sum(counts)]
    table = np.full((len(counts), width), -1, np.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = ids[at:at + c]
        at += c
    return table


# ---- store --------------------------------------------------------------------------------------
def _store(rng, new, old, hkv, layers=1, layer=0, spare=3, spoil=None, x=None):
    """One call on random pages; new, old: rows per sequence and positions before them."""
    counts = [-(-(a + b) // PAGE) for a, b in zip(new, old)]
    width, pages = max(max(counts), 1), sum(counts) + spare
    pool = ref.Pool(layers, pages, hkv, rng)
    pool.k_exp[:], pool.v_exp[:] = rng.integers(100, 130, pool.k_exp.shape), rng.integers(100, 130, pool.v_exp.shape)
    table = random_table(rng, counts, pages, width)
    rows = sum(new)
    cu = np.r_[0, np.cumsum(new)].astype(np.int32)
    if x is None:
        x = [(rng.standard_normal((rows, hkv, 128)) * 2.0 ** rng.integers(-12, 12, (rows, hkv, 1))).astype(np.float32)
             for _ in range(2)]
    pos = np.array(old, np.int32)
    if spoil:
        spoil(table, pos, cu, pages)
    dev = upload_pool(pool)
    Kernels().store_kv_paged(dev, layer, *(DeviceBuffer.from_array(a) for a in x), ints(cu), ints(pos),
                             ints(table), len(new), width, rows)
    synchronize()
    ref.store(pool, layer, *x, cu, pos, table)
    assert_pool(dev, pool)


@pytest.mark.parametrize("hkv", [1, 3, 8])
@pytest.mark.parametrize("new,old", [
    ([1], [0]), ([1], [63]), ([1], [64]), ([1, 1, 1, 1], [5, 200, 64, 127]), ([64], [0]), ([65], [63]),
    ([200, 0, 3, 64], [0, 10, 70, 31]), ([0, 0, 1], [3, 0, 2]), ([130], [1]), ([4, 4], [61, 125]),
], ids=str)
def test_store(new, old, hkv):
    print("store", new, old, hkv, flush=True)
    _store(np.random.default_rng(hkv + sum(new)), new, old, hkv)


def test_store_layers_and_many_sequences():
    rng = np.random.default_rng(3)
    _store(rng, [int(a) for a in rng.integers(0, 3, 300)], [int(a) for a in rng.integers(0, 130, 300)], 2,
           layers=3, layer=1)


def test_store_odd_values():
    """Zeros, subnormals, the largest floats, values next to a change of scale, NaN and infinities."""
    rng = np.random.default_rng(4)
    for k, values in enumerate([[0.0, -0.0], [1e-45, -1e-40], [3.4e38, 1.0], [448.0, 448.0001, -3.0],
                                [1.75, 1.7500001], [2.0 ** -130, 2.0 ** -140], [np.nan, 1.0, np.inf, -np.inf, -5.0],
                                [np.nan, np.inf]]):
        print("values", values, flush=True)
        x = [rng.choice(np.array(values, np.float32), (70, 2, 128)) for _ in range(2)]
        _store(np.random.default_rng(k), [70], [30], 2, x=x)
        _store(np.random.default_rng(k), [70], [0], 2, x=x)


def test_store_rounds_as_e4m3():
    """Every code and every midpoint between two, at a block's own scale."""
    pos = ref.E4M3[:127]
    vals = np.r_[pos, (pos[1:] + pos[:-1]) / 2, np.nextafter(((pos[1:] + pos[:-1]) / 2).astype(np.float32), 0)]
    x = np.zeros((64, 1, 128), np.float32)
    x.reshape(-1)[:len(vals)] = vals
    x.reshape(-1)[1000:1000 + len(vals)] = -vals
    _store(np.random.default_rng(5), [64], [0], 1, x=[x, x * np.float32(2.0 ** -9)])


def test_store_drops_rows_without_a_page():
    def no_page(table, pos, cu, pages):
        table[0, 1] = -1
        table[1, 0] = pages
        table[2, 0] = 1 << 30

    def bad_positions(table, pos, cu, pages):
        pos[0], pos[1], pos[2] = -1, table.shape[1] * PAGE, table.shape[1] * PAGE - 2

    def bad_rows(table, pos, cu, pages):
        cu[-1] = cu[-2]  # the last sequence has none

    for spoil in (no_page, bad_positions, bad_rows):
        print(spoil.__name__, flush=True)
        _store(np.random.default_rng(6), [150, 70, 9], [3, 0, 60], 2, spoil=spoil)


def test_store_grows_token_by_token():
    """A block written one row at a time, each larger than all before it."""
    rng, hkv = np.random.default_rng(7), 2
    pool = ref.Pool(1, 3, hkv, rng)
    table = np.array([[2, 0]], np.int32)
    dev, kern = upload_pool(pool), Kernels()
    gt, gcu = ints(table), ints([0, 1])
    for p in range(80):
        x = [(rng.standard_normal((1, hkv, 128)) * 1.2 ** p).astype(np.float32) for _ in range(2)]
        bufs = [DeviceBuffer.from_array(a) for a in x]
        kern.store_kv_paged(dev, 0, *bufs, gcu, ints([p]), gt, 1, 2, 1)
        synchronize()
        ref.store(pool, 0, *x, np.array([0, 1]), np.array([p]), table)
    assert_pool(dev, pool)


# ---- decode -------------------------------------------------------------------------------------
class Decode:
    def __init__(self, lens, hq, hkv, seed, layers=1, layer=0, out=OutDType.F32, exps=(110, 122), q_scale=1.0,
                 width=None):
        rng = np.random.default_rng(seed)
        counts = [-(-n // PAGE) for n in lens]
        self.width = width or max(max(counts), 1)
        pool = ref.Pool(layers, sum(counts) + 2, hkv, rng)
        live = lambda a: np.where((a & 127) == 127, a - 1, a)  # noqa: E731
        pool.k, pool.v = live(pool.k), live(pool.v)
        pool.k_exp[:] = rng.integers(*exps, pool.k_exp.shape)
        pool.v_exp[:] = rng.integers(*exps, pool.v_exp.shape)
        self.table = random_table(rng, counts, pool.pages, self.width)
        for i, n in enumerate(lens):  # what stands behind the last position is NaN
            if n % PAGE:
                pool.k[:, self.table[i, n // PAGE], :, n % PAGE:] = 127
                pool.v[:, self.table[i, n // PAGE], :, n % PAGE:] = 255
        self.pool, self.lens, self.hq, self.layer, self.out = pool, lens, hq, layer, out
        self.q = (q_scale * rng.standard_normal((len(lens), hq, 128))).astype(np.float32)
        self.dev = upload_pool(pool)
        self.gq, self.gt, self.gl = DeviceBuffer.from_array(self.q), ints(self.table), ints(lens)
        self.wlen = decode_paged_workspace_len(hq, hkv)
        self.ws = DeviceBuffer(self.wlen)
        self.ws.fill(0)
        self.o = DeviceBuffer(self.q.size * (4 if out == OutDType.F32 else 2))

    def call(self, stream=None, ws=None):
        ws = ws or self.ws
        Kernels().decode_attention_paged(self.gq, self.dev, self.layer, self.gt, self.gl, len(self.lens),
                                         self.width, ws, ws.nbytes, self.o, self.hq, self.out, stream)

    def raw(self):
        return self.o.download(np.float32 if self.out == OutDType.F32 else np.uint16)

    def check(self, raw=None, nan=()):
        raw = self.raw() if raw is None else raw
        got = (raw if self.out == OutDType.F32 else oracle.f16_to_f32(raw)).astype(np.float64).reshape(self.q.shape)
        worst = 0.0
        for i, lk in enumerate(self.lens):
            if i in nan:
                assert np.isnan(got[i]).all(), i
                continue
            k, v = ref.rows_of(self.pool, self.layer, self.table[i, :-(-lk // PAGE)], lk)
            o, av, top = (x[0] for x in ref.attend(self.q[i:i + 1], k, v, False))
            tol = av * (2 * (top * (2.0 ** -22 + 136 * 2.0 ** -24) + 2.0 ** -22 + 8 * 2.0 ** -24)
                        + (lk / 16 + 200) * 2.0 ** -24) + 1e-37
            tol += 2.0 ** -32 * np.abs(v).sum(0).repeat(self.hq // self.pool.hkv, 0)
            if self.out == OutDType.F16:
                tol += np.abs(o) * 2.0 ** -11 + 2.0 ** -25
            err = np.abs(got[i] - o)
            assert np.all(err <= tol), (i, lk, float((err / tol).max()))
            worst = max(worst, float((err / tol).max()))
        return worst


def _decode(say, **kw):
    print(say, flush=True)
    d = Decode(**kw)
    d.call()
    synchronize()
    print("  worst error / tolerance", d.check(), flush=True)
    return d


@pytest.mark.parametrize("lens", [[1], [0], [63, 64, 65], [257], [0, 1, 128, 0, 700], [513, 512, 511], [3000],
                                  [2, 5000, 1, 90]], ids=str)
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8)])
def test_decode(lens, hq, hkv):
    _decode(f"decode {lens} {hq} {hkv}", lens=lens, hq=hq, hkv=hkv, seed=sum(lens))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 1), (8, 1), (16, 1), (3, 1), (10, 2), (20, 1), (33, 1), (64, 2),
                                    (6, 3), (4, 4)])
def test_decode_heads(hq, hkv):
    _decode(f"heads {hq} {hkv}", lens=[700, 65, 1], hq=hq, hkv=hkv, seed=hq)


@pytest.mark.parametrize("lens", [[1, 70, 300], [2000]], ids=str)
def test_decode_f16_out(lens):
    _decode("f16 out", lens=lens, hq=8, hkv=2, seed=1, out=OutDType.F16)


def test_decode_layers():
    for layer in (0, 2):
        _decode("layer", lens=[100, 300], hq=8, hkv=2, seed=2, layers=3, layer=layer)


def test_decode_many_sequences():
    """More sequences than a wave has lanes, of very different lengths; runs hold several."""
    rng = np.random.default_rng(8)
    lens = [int(x) for x in np.r_[rng.integers(0, 200, 290), 4000, rng.integers(0, 64, 9)]]
    _decode("many", lens=lens, hq=4, hkv=2, seed=3)


@pytest.mark.parametrize("exps,q_scale", [((0, 3), 1.0), ((1, 20), 1e30), ((60, 200), 1e-30), ((118, 122), 50.0),
                                          ((90, 123), 1.0)])
def test_decode_scales(exps, q_scale):
    """Scales far apart from page to page, and scores that peak."""
    if exps == (60, 200):  # scores within f32, values too
        exps = (100, 160)
    _decode(f"scales {exps} {q_scale}", lens=[700, 90], hq=4, hkv=1, seed=4, exps=exps, q_scale=q_scale)


def test_decode_bad_tables():
    """A length out of range, or a page that is not there, gives NaN in that sequence alone."""
    d = Decode(lens=[300, 900, 128, 64, 77, 2000], hq=8, hkv=2, seed=5)
    t, n = d.table.copy(), list(d.lens)
    t[0, 2], t[1, 14], t[5, 20] = -1, d.pool.pages, 1 << 30
    n[2], n[4] = -1, d.width * PAGE + 1
    d.gt.upload(t)
    d.gl.upload(np.array(n, np.int32))
    d.call()
    synchronize()
    d.check(nan=(0, 1, 2, 4, 5))
    d.gt.upload(d.table)
    d.gl.upload(np.array(d.lens, np.int32))
    d.call()
    synchronize()
    d.check()


def test_decode_nan_codes_spoil_their_sequence_only():
    d = Decode(lens=[300, 400, 500], hq=8, hkv=2, seed=6)
    d.pool.k[0, d.table[1, 3], 0, 10] = 127
    dev = upload_pool(d.pool)
    d.dev = dev
    d.call()
    synchronize()
    got = d.raw().reshape(d.q.shape)
    assert np.isnan(got[1, :4]).all() and not np.isnan(got[1, 4:]).any() and not np.isnan(got[[0, 2]]).any()


def test_decode_one_workspace_for_many_shapes():
    """Calls of other lengths, counts and heads in turn leave the workspace's counters at zero."""
    ds = [Decode(lens=l, hq=32, hkv=8, seed=i) for i, l in enumerate([[5000], [64] * 70, [900, 1, 2000], [3]])]
    first = []
    for d in ds + ds[::-1] + ds:
        d.call(ws=ds[0].ws)
        synchronize()
        first.append(d.raw())
    for d, a, b, c in zip(ds, first, first[4:8][::-1], first[8:]):
        d.check(a)
        assert np.array_equal(a, b) and np.array_equal(a, c)


def test_decode_one_workspace_for_many_heads():
    """Calls of other heads take turns on one workspace, each splitting its sequences."""
    ds = [Decode(lens=[3000, 700], hq=hq, hkv=hkv, seed=hq) for hq, hkv in ((32, 8), (4, 1), (40, 1), (6, 3))]
    ds.append(Decode(lens=[900], hq=1024, hkv=1024, seed=1))
    ws = DeviceBuffer(max(d.wlen for d in ds))
    ws.fill(0)
    for d in ds + ds[::-1] + ds:
        d.call(ws=ws)
        synchronize()
        d.check()


def test_decode_replays_with_other_lengths():
    """A captured step whose lengths grow, on its own workspace, beside eager calls on another stream."""
    s, other = Stream(), Stream()
    d = Decode(lens=[2100, 64, 700], hq=32, hkv=8, seed=9)
    ws2 = DeviceBuffer(d.wlen)
    ws2.fill(0)
    with Graph.capture(s) as g:
        d.call(stream=s)
    for lens in ([2100, 64, 700], [1, 0, 650], [2050, 33, 7], [2100, 64, 700]):
        d.gl.upload(np.array(lens, np.int32))
        g.launch(s)
        s.synchronize()
        got = d.raw()
        d.call(stream=other, ws=ws2)
        other.synchronize()
        assert np.array_equal(d.raw(), got), lens
    for _ in range(4):
        g.launch(s)
    s.synchronize()
    assert np.array_equal(d.raw(), got)
    d.check(got)


def test_decode_two_streams_at_once():
    a, b = (Decode(lens=l, hq=32, hkv=8, seed=i) for i, l in ((10, [9000]), (11, [4000, 5000])))
    sa, sb = Stream(), Stream()
    for _ in range(6):
        a.call(stream=sa)
        b.call(stream=sb)
    sa.synchronize()
    sb.synchronize()
    a.check()
    b.check()
