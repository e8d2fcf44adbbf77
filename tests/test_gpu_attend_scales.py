"""GPU: attention of new rows over pages whose V scales lie far apart, where the pages of the large scale have small
weights: the other pages' values keep their bits.

The tolerance, by element. A score errs by e_s of its key's sum A_j of |q k| / sqrt(128) (the bound of test_gpu_attend.py: 2^-22,
or 2^-15 for the short form, and 136 * 2^-24), a weight by e_p of itself (2^-22 or 2^-11) and 8 roundings; the numerator and the
denominator carry both: sum w |v| A e_s + (sum w |v|) (sum w A) e_s, and (sum w |v|) (2 e_p + 16 * 2^-24). Sums in f32: lk / 2
additions in a chain, and 300. A weight below f16's normal range errs by 2^-25 of units in which the largest part of the sum, a
weight times its page's V scale, is at least 2^7: 2^-32 of that part times the key's code. An f16 result adds half a step.
"""
import numpy as np
import pytest

import oracle
import paged_ref as ref
from brasa_amd import Kernels, OutDType
from brasa_amd.device import synchronize
from test_gpu_attend import Step

pytestmark = pytest.mark.gpu
PAGE, DIM = ref.PAGE, ref.DIM
BASE = 118


class Far(Step):
    """Every fifth page from the `first` on has V values 2^gap times as large, and scores 2^down log2 units lower."""

    def __init__(self, gap, down, first, short=False, **kw):
        super().__init__(exps=(BASE, BASE + 1), **kw)
        self.short, pool, (layer, rng) = short, self.pool, (self.layer, self.rng)
        pool.k[..., 0] = np.where((pool.k[..., 0] & 127) == 127, pool.k[..., 0], 0)
        self.q[..., 0] = np.sqrt(DIM) * np.log(2.0)
        for i, row in enumerate(self.table):
            for b in range(first, (self.new[i] + self.held[i]) // PAGE, 5):
                pool.k[layer, row[b]] = 0
                pool.k[layer, row[b], :, :, 0] = 0xB8  # -1
                pool.k_exp[layer, row[b]] = 127 + down
                pool.v_exp[layer, row[b]] = BASE + gap

    def call(self, stream=None, ws=None):
        Kernels().attention_paged(self.gq, self.dev, self.layer, self.gt, len(self.new), self.width, self.tokens, self.ws,
                                  self.wlen, self.o, self.hq, self.out, stream, short=self.short)

    def check_far(self):
        raw = self.raw()
        got = (raw if self.out == OutDType.F32 else oracle.f16_to_f32(raw)).astype(np.float64).reshape(self.q.shape)
        e_s, e_p = (2.0 ** -15, 2.0 ** -11) if self.short else (2.0 ** -22, 2.0 ** -22)
        e_s += 136 * 2.0 ** -24
        worst = 0.0
        for i, (a, b) in enumerate(zip(self.cu, self.cu[1:])):
            lk = self.held[i] + int(b - a)
            ids = self.table[i, :-(-lk // PAGE)]
            k, v = ref.rows_of(self.pool, self.layer, ids, lk)
            unit = np.repeat(2.0 ** (self.pool.v_exp[self.layer, ids].astype(np.float64) - 127), PAGE, 0)[:lk]
            for r in range(int(b - a)):
                n = self.held[i] + r + 1
                for h in range(self.hq):
                    kh = h // (self.hq // self.hkv)
                    q, kk, vv = self.q[a + r, h].astype(np.float64), k[:n, kh], v[:n, kh]
                    s, size = kk @ q / np.sqrt(DIM), np.abs(kk) @ np.abs(q) / np.sqrt(DIM)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    o, av = w @ vv, w @ np.abs(vv)
                    tol = e_s * ((w * size) @ np.abs(vv) + av * (w @ size)) + av * (2 * e_p + (16 + n / 2 + 300) * 2.0 ** -24)
                    tol += 2.0 ** -32 * (w * unit[:n, kh]).max() * (np.abs(vv) / unit[:n, kh, None]).sum(0)
                    if self.out == OutDType.F16:
                        tol += np.abs(o) * 2.0 ** -11 + 2.0 ** -25
                    err = np.abs(got[a + r, h] - o) / tol
                    assert err.max() <= 1, (i, r, h, float(err.max()))
                    worst = max(worst, float(err.max()))
        return worst


def _run(**kw):
    s = Far(**kw).upload()
    s.plan()
    s.call()
    synchronize()
    print("  worst error / tolerance", s.check_far(), flush=True)


@pytest.mark.parametrize("first", [0, 3])
@pytest.mark.parametrize("gap,down", [(3, 8), (14, 4), (20, 2), (20, 5), (30, 5), (30, 8), (40, 6), (100, 8), (120, 3)])
def test_large_scale_with_small_weights(gap, down, first):
    """Long runs of few waves: each holds pages of both kinds, the large ones first or behind others."""
    print("far", gap, down, first, flush=True)
    _run(gap=gap, down=down, first=first, new=[1, 2], held=[1500, 900], hq=256, hkv=256, behind=0, seed=gap + down)


@pytest.mark.parametrize("out,short", [(OutDType.F16, False), (OutDType.F16, True)])
@pytest.mark.parametrize("gap,down", [(14, 4), (30, 5), (30, 8)])
def test_f16_results(gap, down, out, short):
    print("far f16", gap, down, short, flush=True)
    _run(gap=gap, down=down, first=0, new=[1, 2], held=[1500, 900], hq=256, hkv=256, behind=0, out=out, short=short, seed=gap)


@pytest.mark.parametrize("gap,down", [(30, 5), (40, 6)])
def test_shared_prefix(gap, down):
    """Columns of several sequences in one tile, each with reference points of its own."""
    print("far shared", gap, down, flush=True)
    _run(gap=gap, down=down, first=1, new=[1, 3, 1], held=[700, 660, 900], groups=[(3, 640)], hq=128, hkv=64, behind=0, seed=gap)


def test_scales_that_grow_and_shrink():
    """Each page's V scale is drawn anew; the weights follow the scores."""
    for seed in range(3):
        s = Far(gap=0, down=0, first=99, new=[1, 2], held=[1500, 900], hq=256, hkv=256, behind=0, seed=seed)
        s.pool.v_exp[:] = s.rng.integers(BASE - 25, BASE + 25, s.pool.v_exp.shape)
        s.q *= np.float32(8.0)
        s.upload()
        s.plan()
        s.call()
        synchronize()
        print("  worst error / tolerance", s.check_far(), flush=True)
