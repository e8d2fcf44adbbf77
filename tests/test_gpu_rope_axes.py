"""GPU: rotary positions with several axes, and the paged cache's writer fused with the norms and the rotation.

Tolerance of a rotation: two products and their sum, each rounded to f32 (half a step, 2^-24 of each term's
size): 2^-22 (|a| + |b|). With one axis the bits are rope_neox's. The fused call's q has the bits of rms_norm and
rope_axes in sequence; its k is computed in 64 bits (at most 2^-40 of a term with the root's, far more than its 20
roundings of 2^-53 and a Newton step from 2^-26) and rounded once, half a step of 2^-24; and its pages have the
bits of store_kv_paged on that k.
"""
import numpy as np
import pytest

import paged_ref as ref
import step_ref
from brasa_amd import Kernels, RopeAxes, RopeTable, rope_table
from brasa_amd.device import DeviceBuffer, Graph, Stream, synchronize
from test_gpu_paged import assert_pool, ints, random_table, upload_pool

pytestmark = pytest.mark.gpu
PAGE, DIM = ref.PAGE, ref.DIM
bits = lambda x: np.ascontiguousarray(x, np.float32).view(np.uint32)  # noqa: E731


def _f32(x):
    return DeviceBuffer.from_array(np.asarray(x, np.float32))


@pytest.mark.parametrize("dim", [2, 6, 22, 64, 72, 80, 128, 250, 256])
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (3, 5), (131, 4), (64, 33)])
def test_rope_axes(dim, axes, tokens, heads):
    print("rope_axes", dim, axes, tokens, heads, flush=True)
    rng = np.random.default_rng(dim + axes)
    of = rng.integers(0, axes, dim // 2)
    cos, sin = rope_table(1e6, dim, 97)
    t = RopeTable(1e6, dim, 97)
    pos = rng.integers(0, 97, (axes, tokens)).astype(np.int32)
    pos[rng.integers(axes), ::7] = -1
    pos[rng.integers(axes), 3::11] = 97
    x = rng.standard_normal((tokens + 1, heads, dim)).astype(np.float32)
    buf = _f32(x)
    Kernels().rope_axes(buf, t, RopeAxes.of_pairs(of, axes), ints(pos), tokens, heads, dim)
    synchronize()
    got = buf.download(np.float32).reshape(x.shape)
    assert np.array_equal(bits(got[tokens]), bits(x[tokens]))  # behind the last row
    got, x = got[:tokens], x[:tokens]
    want = step_ref.rope(x, cos, sin, of, pos)
    left = (pos < 0).any(0)
    assert np.array_equal(bits(got[left]), bits(x[left]))
    past = (pos >= 97).any(0) & ~left
    assert np.isnan(got[past]).all()
    on = ~left & ~past
    size = np.abs(x[..., :dim // 2]) + np.abs(x[..., dim // 2:])
    err = np.abs(got - want)[on]
    assert np.all(err <= 2.0 ** -22 * np.concatenate([size, size], -1)[on])


@pytest.mark.parametrize("dim,offset", [(128, 0), (128, 4), (72, 0), (22, 0)])
def test_one_axis_is_rope_neox(dim, offset):
    """Bit for bit, at an address that is not 16-byte aligned too."""
    rng, t, kern = np.random.default_rng(dim), RopeTable(1e4, dim, 200), Kernels()
    x = rng.standard_normal(50 * 6 * dim).astype(np.float32)
    a, b = DeviceBuffer(x.nbytes + 16), DeviceBuffer(x.nbytes + 16)
    for buf in (a, b):
        buf.upload(x, offset)
    kern.rope_neox((a, offset), t, 50, 6, dim, 31)
    kern.rope_axes((b, offset), t, RopeAxes([dim // 2]), ints(np.arange(31, 81)), 50, 6, dim)
    synchronize()
    assert np.array_equal(a.download(np.uint32, x.size, offset), b.download(np.uint32, x.size, offset))


@pytest.mark.parametrize("dim,heads,tokens,offset", [(128, 33, 2100, 0), (72, 37, 3200, 0), (128, 33, 2100, 4)])
def test_many_rows(dim, heads, tokens, offset):
    """A call over more than 2^23 values gives the bits of its rows in pieces."""
    assert tokens * heads * dim > 1 << 23
    rng, t, kern = np.random.default_rng(dim), RopeTable(1e4, dim, 200), Kernels()
    x = rng.standard_normal(tokens * heads * dim).astype(np.float32)
    pos = rng.integers(-2, 202, (3, tokens)).astype(np.int32)
    a, b, axes = DeviceBuffer(x.nbytes + 16), DeviceBuffer(x.nbytes + 16), RopeAxes.of_pairs(rng.integers(0, 3, dim // 2), 3)
    for buf in (a, b):
        buf.upload(x, offset)
    kern.rope_axes((a, offset), t, axes, ints(pos), tokens, heads, dim)
    for i in range(0, tokens, 700):
        n = min(700, tokens - i)
        kern.rope_axes((b, offset + 4 * i * heads * dim), t, axes, ints(pos[:, i:i + n]), n, heads, dim)
    synchronize()
    assert np.array_equal(a.download(np.uint32, x.size, offset), b.download(np.uint32, x.size, offset))


def test_gradient_of_a_rotation():
    """A rotation is linear: the differences of its values are the rotation of the differences, and the rotation
    by the opposite angles (its transpose) undoes it."""
    rng, kern, dim = np.random.default_rng(3), Kernels(), 128
    cos, sin = rope_table(1e6, dim, 50)
    t, back = RopeTable(1e6, dim, 50), RopeTable.view(_f32(cos), _f32(-sin), dim, 50)
    axes, pos = RopeAxes([24, 20, 20], True), ints(rng.integers(0, 50, (3, 40)))
    x = rng.standard_normal((40, 3, dim)).astype(np.float32)
    buf = _f32(x)
    kern.rope_axes(buf, t, axes, pos, 40, 3, dim)
    kern.rope_axes(buf, back, axes, pos, 40, 3, dim)
    synchronize()
    size = np.abs(x[..., :64]) + np.abs(x[..., 64:])
    # two rotations' roundings, and c^2 + s^2 of a table rounded to f32: 2^-23 more
    assert np.all(np.abs(buf.download(np.float32).reshape(x.shape) - x) <= 2.0 ** -20 * np.concatenate([size, size], -1))


# ---- the writer ---------------------------------------------------------------------------------
def _writer(seed, new, old, hq, hkv, axes=3, layers=1, layer=0, spoil=None, stream=None):
    """One fused call against rms_norm, rope_axes and store_kv_paged in sequence: the same bits everywhere."""
    rng, kern = np.random.default_rng(seed), Kernels(stream)
    counts = [-(-(a + b) // PAGE) for a, b in zip(new, old)]
    n, width, pages, tokens = len(new), max(max(counts), 1), sum(counts) + 3, sum(new) + 2
    pool = ref.Pool(layers, pages, hkv, rng)
    pool.k_exp[:], pool.v_exp[:] = rng.integers(100, 130, pool.k_exp.shape), rng.integers(100, 130, pool.v_exp.shape)
    table = random_table(rng, counts, pages, width)
    first = 1  # a row before the first sequence's, and one behind the last's
    cu, pos = (first + np.r_[0, np.cumsum(new)]).astype(np.int32), np.array(old, np.int32)
    rope_pos = rng.integers(0, 300, (axes, tokens)).astype(np.int32)
    x = [(rng.standard_normal((tokens, h, DIM)) * rng.uniform(0.1, 9, (tokens, 1, 1))).astype(np.float32)
         for h in (hq, hkv, hkv)]
    if spoil:
        spoil(table, pos, cu, rope_pos, x)
    w = [rng.uniform(0.5, 1.5, DIM).astype(np.float32) for _ in range(2)]
    axis = rng.integers(0, axes, 64)
    t, of = RopeTable(1e6, DIM, 300), RopeAxes.of_pairs(axis, axes)
    gcu, gpos, gt, gr = ints(cu), ints(pos), ints(table), ints(rope_pos)
    gw = [_f32(a) for a in w]
    one, two = upload_pool(pool), upload_pool(pool)
    a, b = [_f32(v) for v in x], [_f32(v) for v in x]
    kern.qk_norm_rope_store_paged(one, layer, a, gw, 1e-6, t, of, gr, gcu, gpos, gt, n, width, tokens, hq)
    kern.rms_norm(b[0], gw[0], b[0], tokens * hq, DIM, 1e-6)
    kern.rope_axes(b[0], t, of, gr, tokens, hq, DIM)
    if stream:
        stream.synchronize()
    kern.store_kv_paged(two, layer, a[1], b[2], gcu, gpos, gt, n, width, tokens)
    if stream:
        stream.synchronize()
    synchronize()
    for c, d in zip((one.k, one.v, one.k_exp, one.v_exp), (two.k, two.v, two.k_exp, two.v_exp)):
        assert np.array_equal(c.download(np.uint8), d.download(np.uint8))
    inside = np.zeros(tokens, bool)
    inside[cu[0]:cu[-1]] = True
    stored = np.zeros(tokens, bool)
    for i in range(n):
        for j in range(cu[i + 1] - cu[i]):
            p = int(pos[i]) + j
            stored[cu[i] + j] = pos[i] >= 0 and p < width * PAGE and 0 <= table[i, p // PAGE] < pages
    q, seq = (buf.download(np.float32).reshape(x[0].shape) for buf in (a[0], b[0]))
    same = (bits(q) == bits(seq)) | (np.isnan(q) & np.isnan(seq))
    assert same[inside].all() and np.array_equal(bits(q[~inside]), bits(x[0][~inside]))
    got, given = a[1].download(np.float32).reshape(x[1].shape), x[1].astype(np.float64)
    assert np.array_equal(bits(got[~stored]), bits(x[1][~stored]))
    with np.errstate(invalid="ignore"):
        norm = given / np.sqrt((given ** 2).mean(-1, keepdims=True) + np.float64(np.float32(1e-6))) * w[1]
        want = step_ref.rope(norm, *rope_table(1e6, DIM, 300), axis, rope_pos)
        size = np.abs(norm[..., :64]) + np.abs(norm[..., 64:])
        tol = 2.0 ** -24 * np.abs(want) + 2.0 ** -40 * np.concatenate([size, size], -1) + 2.0 ** -150
        close = (np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want))
    assert close[stored].all()
    return got


@pytest.mark.parametrize("new,old", [([1], [0]), ([1], [63]), ([1], [64]), ([64], [0]), ([130, 1, 0, 70], [5, 700, 9, 0]),
                                     ([1] * 70, list(range(0, 700, 10))), ([300], [37])], ids=str)
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8), (3, 1)])
def test_writer(new, old, hq, hkv):
    print("writer", new[:4], hq, hkv, flush=True)
    _writer(len(new), new, old, hq, hkv)


@pytest.mark.parametrize("axes", [1, 2, 4])
def test_writer_axes_and_layers(axes):
    _writer(axes, [70, 3], [10, 127], 16, 2, axes=axes, layers=3, layer=1)


def test_writer_many_rows():
    """More rows of q than waves at once (four rows a wave), and a stream of its own."""
    _writer(9, [250, 37, 1], [0, 64, 200], 32, 4, stream=Stream())


def test_writer_bad_rows():
    def no_page(table, pos, cu, rope_pos, x):
        table[0, 1], table[2, 0] = -1, 1 << 30

    def bad_positions(table, pos, cu, rope_pos, x):
        pos[0], pos[1], pos[2] = -1, table.shape[1] * PAGE, table.shape[1] * PAGE - 2

    def not_finite(table, pos, cu, rope_pos, x):
        x[0][5], x[1][7, 0, 3], x[1][9, :, 4], x[2][11] = np.nan, np.inf, np.nan, -np.inf

    def past_the_table(table, pos, cu, rope_pos, x):
        rope_pos[1, 4], rope_pos[0, 60:70] = 300, 1 << 30

    for spoil in (no_page, bad_positions, not_finite, past_the_table):
        print(spoil.__name__, flush=True)
        _writer(6, [150, 70, 9], [3, 0, 60], 4, 2, spoil=spoil)


def test_writer_negative_rotary_position():
    """NaN in that row of q and k, and NaN codes; the others as ever."""
    rng, kern = np.random.default_rng(8), Kernels()
    pool = ref.Pool(1, 2, 1, rng)
    dev = upload_pool(pool)
    q, k, v = (rng.standard_normal((3, 1, DIM)).astype(np.float32) for _ in range(3))
    bufs, one = [_f32(x) for x in (q, k, v)], _f32(np.ones(DIM))
    kern.qk_norm_rope_store_paged(dev, 0, bufs, (one, one), 1e-6, RopeTable(1e6, DIM, 50), RopeAxes([64]), ints([0, -1, 2]),
                                  ints([0, 3]), ints([0]), ints([[1]]), 1, 1, 3, 1)
    synchronize()
    for buf in bufs[:2]:
        got = buf.download(np.float32).reshape(3, DIM)
        assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2]]).all()
    codes = dev.k.download(np.uint8).reshape(2, PAGE, DIM)[1, :3] & 127
    assert (codes[1] == 127).all() and (codes[[0, 2]] != 127).all()


def test_writer_in_a_graph():
    """A captured decode step is replayed while the sequences grow; every replay against the host."""
    rng, kern, stream = np.random.default_rng(4), Kernels(), Stream()
    n, hq, hkv, width = 5, 8, 2, 6
    pool = ref.Pool(1, n * width, hkv, rng)
    pool.k_exp[:] = pool.v_exp[:] = 100
    dev, table = upload_pool(pool), rng.permutation(n * width).astype(np.int32).reshape(n, width)
    lens = np.array([0, 62, 63, 64, 200], np.int32)
    gl, gt, gadd = ints(lens), ints(table), ints(np.ones(n))
    gcu, grp = ints(np.zeros(n + 1)), ints(np.full(n, 7))
    t, of, one = RopeTable(1e6, DIM, 400), RopeAxes([64]), _f32(np.ones(DIM))
    bufs = [DeviceBuffer(4 * n * h * DIM) for h in (hq, hkv, hkv)]
    synchronize()
    with Graph.capture(stream) as g:
        kern.kv_rows(gadd, gl, gt, n, width, n * width, n, cu=gcu, pos=grp, stream=stream)
        kern.qk_norm_rope_store_paged(dev, 0, bufs, (one, one), 1e-6, t, of, grp, gcu, gl, gt, n, width, n, hq, stream)
    for _ in range(4):
        x = [rng.standard_normal((n, h, DIM)).astype(np.float32) for h in (hq, hkv, hkv)]
        for buf, a in zip(bufs, x):
            buf.upload(a)
        gl.upload(lens)
        g.launch(stream)
        stream.synchronize()
        k = bufs[1].download(np.float32).reshape(x[1].shape)
        norm = x[1] / np.sqrt((x[1].astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-6)
        want = step_ref.rope(norm, *rope_table(1e6, DIM, 400), [0] * 64, lens[None])
        assert np.all(np.abs(k - want) <= 2.0 ** -19 * np.abs(norm).max())
        ref.store(pool, 0, k, x[2], np.arange(n + 1), lens, table)
        assert_pool(dev, pool)
        lens += 1
