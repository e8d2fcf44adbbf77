"""GPU: attention of new rows over the paged cache, with and without a shared prefix, against 64 bits.

The tolerance, by element, is that of the paged decode (test_gpu_paged.py): a score errs by at most A * e_s, A its
row's largest sum of |q k| / sqrt(128): q / sqrt(128) * log2 e in two f16 halves (2^-22), its f32 rounding and product
(2 * 2^-24), 128 + 2 roundings of f32 sums, exp2 and its argument; a weight in two halves adds 2^-22 and a few
roundings; numerator and denominator both carry it. Sums over keys in f32: a lane adds every second key of its
wave's pages, so at most lk / 2 additions in a chain, and 300 for the parts and their joining. A weight below f16's
normal range errs by 2^-32 of the largest one, times |v| of its key. An f16 result adds 2^-11 of itself, and its call
keeps less of q and the weights: q's f16 value errs by 2^-11 of it, and the e4m3 code of what is left by 2^-4 of
that, or by half the least code, 2^-10 / 2^11 where the row's largest |q| is at least 2^8: 2^-15 of each q, and 2^-29
of the largest times the key's sum of |k|; a weight errs by 2^-11 of itself.
"""
import numpy as np
import pytest

import oracle
import paged_ref as ref
import step_ref
from brasa_amd import Kernels, OutDType, attention_paged_workspace_len
from brasa_amd.device import DeviceBuffer, Graph, Stream, synchronize
from test_gpu_paged import ints, upload_pool

pytestmark = pytest.mark.gpu
PAGE, DIM = ref.PAGE, ref.DIM


class Step:
    """Sequences of `held` positions with `new` rows each; groups: (sequences, prefix) one after another."""

    def __init__(self, new, held, hq=8, hkv=2, groups=(), seed=0, layers=1, layer=0, out=OutDType.F32, exps=(110, 122),
                 q_scale=1.0, extra=0, behind=2, before=1):
        rng = self.rng = np.random.default_rng(seed)
        self.new, self.held, self.hq, self.hkv, self.layer, self.out = list(new), list(held), hq, hkv, layer, out
        n = len(new)
        lens = [a + b for a, b in zip(new, held)]
        counts = [-(-x // PAGE) for x in lens]
        self.width = max(max(counts), 1) + extra
        self.group, self.prefix = [0], []
        for size, prefix in groups:
            self.group.append(self.group[-1] + size)
            self.prefix.append(prefix)
        pool = self.pool = ref.Pool(layers, sum(counts) + 2, hkv, rng)
        live = lambda a: np.where((a & 127) == 127, a - 1, a)  # noqa: E731
        pool.k, pool.v = live(pool.k), live(pool.v)
        pool.k_exp[:], pool.v_exp[:] = rng.integers(*exps, pool.k_exp.shape), rng.integers(*exps, pool.v_exp.shape)
        ids = iter(rng.permutation(pool.pages))
        self.table = np.full((n, self.width), -1, np.int32)
        for i, c in enumerate(counts):
            self.table[i, :c] = [next(ids) for _ in range(c)]
        for g, prefix in enumerate(self.prefix):  # the pages of the group's first sequence that has them
            pages = prefix // PAGE
            mine = [i for i in range(self.group[g], self.group[g + 1]) if held[i] >= pages * PAGE]
            for i in mine[1:]:
                self.table[i, :pages] = self.table[mine[0], :pages]
        for i, x in enumerate(lens):  # what stands behind the last position is NaN
            if x % PAGE:
                pool.k[:, self.table[i, x // PAGE], :, x % PAGE:] = 127
                pool.v[:, self.table[i, x // PAGE], :, x % PAGE:] = 255
        self.cu = (before + np.r_[0, np.cumsum(new)]).astype(np.int32)
        self.tokens = int(self.cu[-1]) + behind
        self.q = (q_scale * rng.standard_normal((self.tokens, hq, DIM))).astype(np.float32)
        self.pos = np.array(held, np.int32)

    def upload(self):
        self.dev, self.gq, self.gt = upload_pool(self.pool), DeviceBuffer.from_array(self.q), ints(self.table)
        self.gcu, self.gpos, self.gg, self.gp = ints(self.cu), ints(self.pos), ints(self.group), ints(self.prefix or [0])
        self.wlen = attention_paged_workspace_len(len(self.new), len(self.prefix), self.tokens, self.hq, self.hkv)
        self.ws = DeviceBuffer(self.wlen)
        self.ws.fill(0xC3)
        self.o = DeviceBuffer(self.q.size * (4 if self.out == OutDType.F32 else 2))
        self.o.fill(0x3C)
        return self

    def plan(self, stream=None, ws=None):
        ws = ws or self.ws
        Kernels().attention_paged_plan(self.gcu, self.gpos, self.gg, self.gp, len(self.prefix), len(self.new), self.width,
                                       self.tokens, self.hq, self.hkv, ws, ws.nbytes, stream)

    def call(self, stream=None, ws=None):
        ws = ws or self.ws
        Kernels().attention_paged(self.gq, self.dev, self.layer, self.gt, len(self.new), self.width, self.tokens, ws,
                                  ws.nbytes, self.o, self.hq, self.out, stream)

    def raw(self):
        return self.o.download(np.float32 if self.out == OutDType.F32 else np.uint16)

    def check(self, raw=None, nan=(), only=None):
        """nan: sequences whose rows are all NaN. Where the values seen are not finite, NaN in the same places."""
        raw = self.raw() if raw is None else raw
        got = (raw if self.out == OutDType.F32 else oracle.f16_to_f32(raw)).astype(np.float64).reshape(self.q.shape)
        words = raw.view(np.uint8).reshape(self.tokens, -1)
        assert (words[:self.cu[0]] == 0x3C).all() and (words[self.cu[-1]:] == 0x3C).all()  # rows outside
        worst = 0.0
        for i, (a, b) in enumerate(zip(self.cu, self.cu[1:])):
            if a == b or (only is not None and i not in only):
                continue
            if i in nan:
                assert np.isnan(got[a:b]).all(), i
                continue
            lk = self.held[i] + int(b - a)
            k, v = ref.rows_of(self.pool, self.layer, self.table[i, :-(-lk // PAGE)], lk)
            o, av, top = step_ref.attend(self.q[a:b], k, v, self.held[i])
            e_q, e_p, rest = 2.0 ** -22, 2.0 ** -22, 0.0
            if self.out == OutDType.F16:
                e_q, e_p = 2.0 ** -15, 2.0 ** -11
                most = np.abs(np.nan_to_num(k)).sum(-1).max(0).repeat(self.hq // self.hkv)[None, :, None]
                rest = 2.0 ** -29 * np.abs(np.nan_to_num(self.q[a:b])).max(-1, keepdims=True) * most / np.sqrt(DIM)
            tol = av * (2 * (top * (e_q + 136 * 2.0 ** -24) + rest + e_p + 8 * 2.0 ** -24)
                        + (lk / 2 + 300) * 2.0 ** -24) + 1e-37
            tol += 2.0 ** -32 * np.abs(np.nan_to_num(v)).sum(0).repeat(self.hq // self.hkv, 0)
            if self.out == OutDType.F16:
                tol += np.abs(o) * 2.0 ** -11 + 2.0 ** -25
            assert np.array_equal(np.isnan(got[a:b]), np.isnan(o)), (i, np.argwhere(np.isnan(got[a:b]) != np.isnan(o))[:4])
            err = np.where(np.isnan(o), 0.0, np.abs(got[a:b] - o))
            tol = np.where(np.isnan(o), 1.0, tol)
            assert np.all(err <= tol), (i, lk, float((err / tol).max()), np.argwhere(err > tol)[:4])
            worst = max(worst, float((err / tol).max()))
        return worst


def _run(say, **kw):
    print(say, flush=True)
    s = Step(**kw).upload()
    s.plan()
    s.call()
    synchronize()
    print("  worst error / tolerance", s.check(), flush=True)
    return s


@pytest.mark.parametrize("new,held", [([1], [0]), ([1], [63]), ([1], [64]), ([1], [256]), ([3], [30]), ([64], [0]), ([65], [0]),
                                      ([1, 0, 1, 1], [5, 9, 128, 700]), ([33, 1, 70], [100, 2000, 63]), ([300], [0]),
                                      ([200], [1000]), ([1], [3000]), ([7, 2], [61, 4100])], ids=str)
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8), (16, 2), (3, 1)])
def test_rows_alone(new, held, hq, hkv):
    _run(("alone", new, held, hq, hkv), new=new, held=held, hq=hq, hkv=hkv, seed=len(new) + hq)


@pytest.mark.parametrize("new,held,groups", [
    ([1, 1], [64, 64], [(2, 64)]), ([1] * 4, [700, 650, 645, 800], [(4, 640)]), ([1] * 40, [130 + 7 * i for i in range(40)], [(40, 128)]),
    ([1, 2, 0, 5, 1], [200, 300, 250, 193, 700], [(5, 192)]), ([3, 40, 1, 60], [128, 140, 300, 128], [(4, 128)]),
    ([1] * 6, [100, 300, 63, 64, 1000, 130], [(3, 64), (3, 64)]), ([1] * 7, [500] * 7, [(2, 448), (1, 448), (4, 64)]),
    ([1, 1, 1], [100, 500, 600], [(3, 448)]), ([2] * 5, [4200, 4100, 4097, 4300, 4500], [(5, 4096)]),
    ([1, 1], [90, 70], [(2, 63)]), ([9, 9], [90, 70], [(0, 64), (2, 64), (0, 64)])], ids=str)
@pytest.mark.parametrize("hq,hkv", [(32, 8), (4, 4), (16, 1)])
def test_shared_prefix(new, held, groups, hq, hkv):
    """Forks and prompts behind a prefix; some with rows below it or too many of them, which go alone."""
    _run(("shared", new[:5], groups, hq, hkv), new=new, held=held, groups=groups, hq=hq, hkv=hkv, seed=len(new) + hq)


@pytest.mark.parametrize("hq,hkv", [(128, 1), (160, 1), (300, 2), (1024, 8), (5, 1), (64, 64)])
def test_head_counts(hq, hkv):
    """Groups of more heads than a tile has columns, and of odd ones."""
    _run(("heads", hq, hkv), new=[1, 2, 1], held=[130, 70, 200], groups=[(3, 64)], hq=hq, hkv=hkv, seed=hq)


@pytest.mark.parametrize("new,held,groups", [
    ([1], [0], []), ([1], [256], []), ([65], [0], []), ([33, 1, 70], [100, 2000, 63], []), ([1] * 6, [100, 300, 63, 64, 1000, 130], [(3, 64), (3, 64)]),
    ([2] * 5, [4200, 4100, 4097, 4300, 4500], [(5, 4096)])], ids=str)
@pytest.mark.parametrize("hq,hkv", [(32, 8), (4, 4), (16, 1), (128, 1)])
def test_f16_results(new, held, groups, hq, hkv):
    _run(("f16", new[:5], groups, hq, hkv), new=new, held=held, groups=groups, hq=hq, hkv=hkv, out=OutDType.F16, seed=len(new) + hq)


@pytest.mark.parametrize("out", list(OutDType))
def test_f16_and_layers(out):
    _run(("layer", out), new=[1, 50, 1, 200], held=[500, 448, 449, 20], groups=[(3, 448)], hq=16, hkv=4, layers=3, layer=1, out=out)


@pytest.mark.parametrize("exps,q_scale,out", [((60, 200), 1.0, OutDType.F32), ((0, 3), 1e-3, OutDType.F32), ((100, 140), 1e-30, OutDType.F32),
                                              ((127, 135), 3.0, OutDType.F32), ((105, 121), 1e-2, OutDType.F16), ((110, 114), 50.0, OutDType.F16)])
def test_scales_far_apart(exps, q_scale, out):
    """V's scale jumps between pages, and the scores are large or tiny."""
    _run(("scales", exps, q_scale), new=[1, 40, 3], held=[700, 64, 200], groups=[(3, 64)], exps=exps, q_scale=q_scale, out=out, seed=5)


def test_first_keys_small():
    """The running maximum grows with every page, by more than the lazy reference point allows."""
    s = Step(new=[2, 100], held=[900, 500], seed=6)
    for i in range(2):
        for b, page in enumerate(s.table[i]):
            if page >= 0:
                s.pool.k_exp[0, page] = 112 + b
    s.upload()
    s.plan()
    s.call()
    synchronize()
    s.check()


def test_many_sequences():
    """More sequences, tiles and groups than one round of the plan's workgroup takes."""
    rng = np.random.default_rng(7)
    n = 2300
    held = [int(x) for x in 64 + rng.integers(0, 100, n)]
    s = Step(new=[int(x) for x in rng.integers(0, 3, n)], held=held, groups=[(2, 64)] * 1100 + [(50, 0)], hq=2, hkv=1, seed=7).upload()
    s.plan()
    s.call()
    synchronize()
    s.check()


@pytest.mark.parametrize("n,hq", [(250, 2), (257, 2), (300, 16), (900, 16)])
def test_rounds_of_the_plan(n, hq):
    """Each size of the plan's workgroup, with tiles for one round of it or more: few and many columns of a sequence
    in a prefix that crosses tiles, and one group whose rows are not packed behind each other."""
    new = [1] * n
    new[n // 2] = 40
    held = [64 + (7 * i) % 90 for i in range(n)]
    _run(("rounds", n, hq), new=new, held=held, groups=[(n // 3, 64), (n - n // 3, 64)], hq=hq, hkv=1, seed=n)


@pytest.mark.parametrize("out", list(OutDType))
def test_values_that_are_not_finite(out):
    """NaN keys and values reach the rows that see them, in their places, and no others."""
    s = Step(new=[50, 1, 1, 9], held=[70, 200, 130, 128], groups=[(4, 64)], hq=8, hkv=2, out=out, seed=8)
    s.pool.v[0, s.table[0, 1], 1, 20, 5] = 127    # position 84, below some of sequence 0's rows only
    s.pool.v[0, s.table[0, 1], 0, 55, :] = 255    # position 119, its last row's own
    s.pool.k[0, s.table[1, 3], 0, 3, 7] = 127     # position 195: sequence 1 sees it
    s.pool.v[0, s.table[2, 1], 1, 0, 127] = 127   # a page all see whole
    s.pool.v[0, s.table[3, 2], 0, 4, 64] = 255    # position 132
    s.q[s.cu[1] - 3] = np.nan
    s.upload()
    s.plan()
    s.call()
    synchronize()
    s.check()


def test_bad_sequences():
    """Positions and pages that are not there: NaN in the rows that need them."""
    s = Step(new=[1, 3, 1, 2, 70], held=[100, 64, 128, 300, 190], groups=[(3, 64)], hq=8, hkv=2, seed=9)
    s.pos[0] = -1
    s.table[2, 1] = s.pool.pages
    s.table[4, 3] = -1  # positions 192 and on: all but its first two rows
    s.upload()
    s.plan()
    s.call()
    synchronize()
    s.check(only=[1, 3])
    got = s.raw().reshape(s.q.shape)
    assert np.isnan(got[s.cu[0]:s.cu[1]]).all() and np.isnan(got[s.cu[2]:s.cu[3]]).all()
    assert np.isfinite(got[s.cu[4]:s.cu[4] + 2]).all() and np.isnan(got[s.cu[4] + 2:s.cu[5]]).all()
    # rows past the table's width, and a position past it
    s = Step(new=[6, 1, 1], held=[60, 5, 63], hq=4, hkv=2, seed=10)
    s.width, s.table = 1, s.table[:, :1].copy()
    s.pos[2] = 64
    s.upload()
    s.plan()
    s.call()
    synchronize()
    s.check(only=[1])
    got = s.raw().reshape(s.q.shape)
    assert np.isfinite(got[s.cu[0]:s.cu[0] + 4]).all() and np.isnan(got[s.cu[0] + 4:s.cu[1]]).all()
    assert np.isnan(got[s.cu[2]:s.cu[3]]).all()


@pytest.mark.parametrize("out", list(OutDType))
def test_table_without_columns(out):
    """No position has a page: NaN in every row of a sequence, as many as there are."""
    s = Step(new=[1, 40, 0, 3], held=[5, 0, 7, 200], groups=[(4, 64)], hq=8, hkv=2, seed=17, out=out)
    s.width = 0
    s.upload()
    s.plan()
    s.call()
    synchronize()
    s.check(nan=(0, 1, 3))


def test_bounds_out_of_order():
    """cu and group are raised to the largest before them: no row of o outside is touched."""
    s = Step(new=[4, 3, 5, 2], held=[70, 80, 64, 90], groups=[(2, 64), (2, 64)], hq=4, hkv=1, seed=11)
    given = s.cu.copy()
    s.cu[2], s.group[1] = given[2] - 5, 9
    s.upload()
    s.plan()
    s.call()
    synchronize()
    raised = step_ref.raised(s.cu, s.tokens)
    assert list(raised[:3]) == [given[0], given[1], given[1]]
    s.table[3, 0] = s.table[0, 0]  # group 0 is now all four sequences, whose first page is sequence 0's
    s.check(only=[0, 3])


def test_without_a_plan():
    """A workspace without a plan, or with that of other sizes: NaN throughout, whatever it holds."""
    for out in OutDType:
        s = Step(new=[1, 1], held=[100, 90], hq=4, hkv=2, seed=12, out=out).upload()
        other = Step(new=[1, 1, 1], held=[100, 90, 80], hq=4, hkv=2, seed=12, out=out).upload()
        big = DeviceBuffer(max(s.wlen, other.wlen))
        for fill in (0, 0x61, None):
            if fill is None:
                other.plan(ws=big)
            else:
                big.fill(fill)
            s.o.fill(0)
            s.call(ws=big)
            synchronize()
            raw = s.raw()
            assert np.isnan(raw if out == OutDType.F32 else oracle.f16_to_f32(raw)).all()


def test_same_bits_again():
    """Two calls, another stream and a workspace with other contents: the same bits."""
    s = Step(new=[1] * 20 + [90], held=[600 + 13 * i for i in range(20)] + [700], groups=[(21, 576)], hq=32, hkv=8, seed=13).upload()
    s.plan()
    s.call()
    synchronize()
    first = s.raw()
    s.check(first)
    stream, ws = Stream(), DeviceBuffer(s.wlen + 512)
    ws.fill(0x55)
    synchronize()
    s.plan(stream, ws)
    for _ in range(2):
        s.o.fill(0x3C, stream)
        s.call(stream, ws)
        stream.synchronize()
        assert np.array_equal(s.raw().view(np.uint8), first.view(np.uint8))


def test_two_streams_at_once():
    """Steps in flight together, each on a workspace of its own."""
    steps = [Step(new=[1] * 9, held=[300 + 50 * i for i in range(9)], groups=[(9, 256)], seed=20 + i).upload() for i in range(2)]
    streams = [Stream(), Stream()]
    synchronize()
    for _ in range(5):
        for s, stream in zip(steps, streams):
            s.plan(stream)
            s.call(stream)
    synchronize()
    for s in steps:
        s.check()


def test_captured_step():
    """A captured plan and two layers are replayed while lengths, rows, tables and prefixes change."""
    n, hq, hkv, width, tokens = 6, 8, 2, 20, 90
    stream, kern, rng = Stream(), Kernels(), np.random.default_rng(14)
    pool = ref.Pool(2, 150, hkv, rng)
    pool.k, pool.v = (np.where((x & 127) == 127, x - 1, x) for x in (pool.k, pool.v))
    pool.k_exp[:], pool.v_exp[:] = 112, 120
    dev = upload_pool(pool)
    wlen = attention_paged_workspace_len(n, 2, tokens, hq, hkv)
    ws = DeviceBuffer(wlen)
    gcu, gpos, gg, gp, gt = ints(np.zeros(n + 1)), ints(np.zeros(n)), ints([0, 4, 6]), ints([0, 0]), ints(np.zeros((n, width)))
    gq, o = DeviceBuffer(2 * 4 * tokens * hq * DIM), DeviceBuffer(2 * 4 * tokens * hq * DIM)
    half = 4 * tokens * hq * DIM
    synchronize()
    with Graph.capture(stream) as g:
        kern.attention_paged_plan(gcu, gpos, gg, gp, 2, n, width, tokens, hq, hkv, ws, wlen, stream)
        for layer in range(2):
            kern.attention_paged((gq, layer * half), dev, layer, gt, n, width, tokens, ws, wlen, (o, layer * half), hq, stream=stream)
    for step in range(5):
        new = [int(x) for x in rng.integers(0, 16, n)]
        held = [int(x) for x in rng.integers(0, 17 * PAGE, n)]
        s = Step(new=new, held=held, hq=hq, hkv=hkv, seed=step, before=0, behind=tokens - sum(new))
        s.pool, s.width = pool, width
        s.table = rng.integers(0, 150, (n, width)).astype(np.int32)
        s.table[:4, :6], s.table[4:, :6] = s.table[0, :6], s.table[4, :6]
        prefix = [int(x) for x in rng.integers(0, 6 * PAGE + 1, 2)]
        q2 = rng.standard_normal((2, tokens, hq, DIM)).astype(np.float32)
        for buf, x in ((gcu, s.cu), (gpos, s.pos), (gp, np.array(prefix, np.int32)), (gt, s.table), (gq, q2)):
            buf.upload(x)
        o.fill(0x3C)
        synchronize()
        g.launch(stream)
        stream.synchronize()
        raw = o.download(np.float32).reshape(2, -1)
        for layer in range(2):
            s.layer, s.q = layer, q2[layer]
            s.check(raw[layer])


@pytest.mark.parametrize("new,held,groups,hq,hkv", [
    ([1], [16384], [], 32, 8), ([1] * 64, [8192 + 11 * i for i in range(64)], [(64, 8192)], 8, 2),
    ([700, 5, 300], [4096, 4096, 4100], [(3, 4096)], 4, 1), ([2500], [600], [], 4, 1)], ids=lambda x: str(x)[:20])
def test_long(new, held, groups, hq, hkv):
    _run(("long", new[:3], held[:3], hq, hkv), new=new, held=held, groups=groups, hq=hq, hkv=hkv, seed=15)


def test_a_servers_steps():
    """The operators as a server calls them: requests behind one system prompt are forked from it, their
    prompts arrive packed, then drafts and single tokens: maps, shared pages, the fused writer, plan and attention, each
    step against the host's own copy."""
    from brasa_amd import RopeAxes, RopeTable, kv_pages_workspace_len, rope_table
    rng, kern = np.random.default_rng(16), Kernels()
    hq, hkv, n, width, pages, tokens, layers = 8, 2, 4, 10, 40, 150, 2
    pool = ref.Pool(layers, pages, hkv, rng)
    dev = upload_pool(pool)
    t, of, (cos, sin) = RopeTable(1e6, DIM, 2000), RopeAxes([24, 20, 20], True), rope_table(1e6, DIM, 2000)
    axis = [0, 1, 2] * 20 + [0] * 4
    plen, wlen = kv_pages_workspace_len(pages, n, width), attention_paged_workspace_len(n, 1, tokens, hq, hkv)
    pws, ws, status = DeviceBuffer(plen), DeviceBuffer(wlen), ints([0, 0])
    table, lens, counts = np.full((n, width), -1, np.int32), np.zeros(n, np.int32), np.zeros(pages, np.int32)
    gt, gl, gr, gg, gp = ints(table), ints(lens), ints(counts), ints([0, n]), ints([7])
    out = {name: ints(np.zeros(size)) for name, size in (("cu", n + 1), ("lk", n), ("seq", tokens), ("pos", tokens), ("slot", tokens))}
    weights = [rng.uniform(0.5, 1.5, DIM).astype(np.float32) for _ in range(2)]
    gw = [DeviceBuffer.from_array(w) for w in weights]
    steps = [([140, 0, 0, 0], None), ([3, 90, 20, 1], [0, 0, 0, 0]), ([4, 1, 5, 2], None), ([1, 1, 1, 1], [0, 1, 3, 3])]
    for add, parent in steps:
        print("step", add, flush=True)
        if parent:
            t2, l2 = ints(table), ints(lens)
            kern.kv_pages_fork(ints(parent), gt, gl, gr, t2, l2, gr, n, width, pages)
            gt, gl = t2, l2
            table, lens, counts = ref.fork(parent, table, lens, counts)
        ga = ints(add)
        kern.kv_pages_reserve(dev, ga, gt, gl, gr, gt, gr, status, n, width, pws, plen)
        table, counts, want = ref.reserve(pool, add, table, lens, counts)
        assert want[1] == 0
        kern.kv_rows(ga, gl, gt, n, width, pages, tokens, **out)
        kern.kv_pages_shared(gt, gl, gg, 1, n, width, pages, gp)
        kern.attention_paged_plan(out["cu"], gl, gg, gp, 1, n, width, tokens, hq, hkv, ws, wlen)
        cu, lk, seq, pos, slot = step_ref.rows(add, lens, table, pages, tokens)
        rope_pos = np.stack([pos, np.where(pos >= 0, pos // 3, -1), np.where(pos >= 0, pos % 50, -1)]).astype(np.int32)
        grp = ints(rope_pos)
        s = Step(new=add, held=lens.tolist(), hq=hq, hkv=hkv, before=0, behind=tokens - sum(add))
        for layer in range(layers):
            x = [rng.standard_normal((tokens, h, DIM)).astype(np.float32) for h in (hq, hkv, hkv)]
            bufs = [DeviceBuffer.from_array(a) for a in x]
            o = DeviceBuffer(x[0].nbytes)
            o.fill(0x3C)
            kern.qk_norm_rope_store_paged(dev, layer, bufs, gw, 1e-6, t, of, grp, out["cu"], gl, gt, n, width, tokens, hq)
            kern.attention_paged(bufs[0], dev, layer, gt, n, width, tokens, ws, wlen, o, hq)
            synchronize()
            rows = int(cu[-1])
            now = [b.download(np.float32).reshape(a.shape) for b, a in zip(bufs, x)]
            for got, given, w in zip(now[:2], x, weights):
                y = given.astype(np.float64)
                y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + 1e-6) * w
                y = step_ref.rope(y, cos, sin, axis, rope_pos)
                assert np.all(np.abs(got[:rows] - y[:rows]) <= 2.0 ** -19 * np.abs(y[:rows]).max())
                assert np.array_equal(got[rows:], given[rows:])
            ref.store(pool, layer, now[1], x[2], cu, lens, table)
            s.pool, s.table, s.layer, s.q = pool, table, layer, now[0]
            s.check(o.download(np.float32))
        for name, w in zip(("cu", "lk", "seq", "pos", "slot"), (cu, lk, seq, pos, slot)):
            assert np.array_equal(out[name].download(np.int32), w), name
        assert list(gp.download(np.int32)) == list(step_ref.shared(table, lens, [0, n], pages))
        from test_gpu_paged import assert_pool
        assert_pool(dev, pool)
        lens = lk.copy()
        gl = ints(lens)
    assert list(step_ref.shared(table, lens, [0, n], pages)) == [128]
