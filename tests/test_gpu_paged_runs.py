"""GPU: paged decode whose workgroups hold long runs of pages over several sequences, a pool that owns its
buffers, and what the calls on packed prompts and pages allocate. Tolerances: test_gpu_paged.py's."""
import numpy as np
import pytest

import paged_ref as ref
from brasa_amd import (AttnShape, Kernels, KvPool, KvType, OutDType, PrefillPrecision, decode_paged_workspace_len,
                       kv_pages_workspace_len)
from brasa_amd.device import DeviceBuffer, mem_info, synchronize
from test_gpu_paged import Decode, assert_pool, ints, upload_pool

pytestmark = pytest.mark.gpu
PAGE = ref.PAGE
SLOTS, SHORT = 512, 8  # workgroups of a launch; pages of a run that is not long


def run_size(d):
    """Pages of a workgroup's run, as the call counts them (several sequences, none cut by itself)."""
    hq, hkv, n = d.hq, d.pool.hkv, len(d.lens)
    chunks = -(-(hq // hkv) // 8)
    runs = max(SLOTS // (hkv * chunks), 1)
    assert n > 64 or n > runs // 4
    return -(-sum(max(-(-x // PAGE), 1) for x in d.lens) // runs)


@pytest.mark.parametrize("out", [OutDType.F32, OutDType.F16])
@pytest.mark.parametrize("hq,hkv,n,most", [(32, 8, 40, 4000), (32, 32, 30, 1500), (64, 4, 100, 2000),
                                           (16, 16, 150, 700)])
def test_decode_long_runs(hq, hkv, n, most, out):
    """Runs of more pages than a short one that end inside sequences: a run's first segment, whole sequences
    and its last, lengths of 0 and 1 among them, and the same bits from call to call."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(2, most, n)]
    lens[3], lens[n // 2], lens[-2] = 0, 1, most
    d = Decode(lens=lens, hq=hq, hkv=hkv, seed=n, out=out)
    size = run_size(d)
    print(f"long runs {hq} {hkv} {n}: {size} pages", flush=True)
    assert size > SHORT
    first = None
    for _ in range(3):
        d.call()
        synchronize()
        first = d.raw() if first is None else first
        assert np.array_equal(d.raw(), first)
    print("  worst error / tolerance", d.check(), flush=True)


def test_pool_of_its_own():
    """A KvPool that owns its buffers, cleared, written and read like one over the caller's."""
    rng = np.random.default_rng(3)
    layers, pages, hkv, hq, lens = 2, 7, 2, 8, [130, 64]
    dev, like = KvPool(layers, pages, hkv), ref.Pool(layers, pages, hkv)
    assert dev.bytes() == sum(a.nbytes for a in like.arrays())
    for b, a in zip((dev.k, dev.v, dev.k_exp, dev.v_exp), like.arrays()):
        assert b.nbytes == a.nbytes
        b.fill(0)
    rows, n, width = sum(lens), len(lens), 3
    table = rng.permutation(pages)[:n * width].reshape(n, width).astype(np.int32)
    cu = np.r_[0, np.cumsum(lens)].astype(np.int32)
    x = [rng.standard_normal((rows, hkv, 128)).astype(np.float32) for _ in range(2)]
    q = rng.standard_normal((n, hq, 128)).astype(np.float32)
    kern, ws = Kernels(), DeviceBuffer(decode_paged_workspace_len(hq, hkv))
    ws.fill(0)
    gq, o = DeviceBuffer.from_array(q), DeviceBuffer(q.nbytes)
    bufs = [DeviceBuffer.from_array(a) for a in x]
    kern.store_kv_paged(dev, 1, *bufs, ints(cu), ints([0] * n), ints(table), n, width, rows)
    kern.decode_attention_paged(gq, dev, 1, ints(table), ints(lens), n, width, ws, ws.nbytes, o, hq)
    synchronize()
    ref.store(like, 1, *x, cu, np.zeros(n, int), table)
    assert_pool(dev, like)
    got = o.download(np.float32).reshape(q.shape)
    for i, lk in enumerate(lens):
        want, av, top = (a[0] for a in ref.attend(q[i:i + 1], *ref.rows_of(like, 1, table[i, :-(-lk // PAGE)], lk),
                                                  False))
        # (the looser bound that test_serving_run takes: 2^-15 of the scores, 2^-14 of the weights)
        assert np.all(np.abs(got[i] - want) <= av * (top * 2.0 ** -15 + 2.0 ** -14))


def test_calls_allocate_nothing():
    """Device memory in use stays the same over every call on packed prompts and pages, larger calls
    after smaller ones (the first calls load the code objects)."""
    rng, kern = np.random.default_rng(4), Kernels()
    hq, hkv, layers, pages, width = 8, 2, 2, 400, 40

    def inputs(n, most):
        lens = rng.integers(1, most, n)
        rows = int(lens.sum())
        cu = np.r_[0, np.cumsum(lens)].astype(np.int32)
        rnd = lambda *s: DeviceBuffer.from_array(rng.standard_normal(s).astype(np.float32))  # noqa: E731
        z = dict(n=n, rows=rows, cu=ints(cu), q=rnd(rows, hq, 128), k=rnd(rows, hkv, 128), v=rnd(rows, hkv, 128),
                 o=DeviceBuffer(rows * hq * 128 * 4), pos=ints([0] * n), lens=ints(lens), one=ints([1] * n),
                 parent=ints(np.arange(n)), table=ints(np.full((n, width), -1)), ref=ints([0] * pages))
        z["len0"] = ints([0] * n)
        z["t2"], z["l2"] = ints(np.full((n, width), -1)), ints([0] * n)
        z["ws"] = DeviceBuffer(kv_pages_workspace_len(pages, n, width))
        z["status"] = ints([0, 0])
        return z

    dev = upload_pool(ref.Pool(layers, pages, hkv))
    dws = DeviceBuffer(decode_paged_workspace_len(hq, hkv))
    dws.fill(0)

    def step(z):
        n = z["n"]
        for kv, precision in ((KvType.F16, PrefillPrecision.F16), (KvType.F16, PrefillPrecision.F16_PF32),
                              (KvType.F16, PrefillPrecision.F32), (KvType.F32, PrefillPrecision.F32)):
            kern.flash_attention_packed(z["q"], z["k"], z["v"], z["o"], z["cu"], n,
                                        AttnShape(z["rows"], hq, hkv, 128, 0, kv), precision)
        kern.kv_pages_reserve(dev, z["lens"], z["table"], z["len0"], z["ref"], z["table"], z["ref"], z["status"],
                              n, width, z["ws"], z["ws"].nbytes)
        kern.store_kv_paged(dev, 0, z["k"], z["v"], z["cu"], z["pos"], z["table"], n, width, z["rows"])
        kern.decode_attention_paged(z["q"], dev, 0, z["table"], z["lens"], n, width, dws, dws.nbytes, z["o"], hq)
        kern.kv_pages_fork(z["parent"], z["table"], z["lens"], z["ref"], z["t2"], z["l2"], z["ref"], n, width, pages)
        kern.kv_pages_reserve(dev, z["one"], z["t2"], z["l2"], z["ref"], z["t2"], z["ref"], z["status"], n, width,
                              z["ws"], z["ws"].nbytes)
        kern.kv_pages_compact(dev, z["t2"], z["ref"], z["t2"], z["ref"], z["status"], n, width, z["ws"],
                              z["ws"].nbytes)
        synchronize()

    few, two, many = inputs(2, 40), inputs(60, 200), inputs(90, 250)
    for z in (few, two):  # both sides of every choice of a kernel
        step(z)
        step(z)
    free, _ = mem_info()
    for z in (many, two, many):
        print("step of", z["n"], "sequences", flush=True)
        step(z)
        assert mem_info()[0] == free
