"""GPU: the bits that attention of new rows over the paged cache keeps of its operands.

f16 results are the f32 results rounded: both calls contract q and the weights as two f16 halves, in the same order. The last
product, a sum times 1 / l, is rounded to f32 (half a step, 2^-24 of it) in the one call, and to f16 with or without that step in
the other: the two differ by half a step of f16 and 2^-24. The short form's tolerance is the one written in test_gpu_attend.py
for f16 results.
"""
import numpy as np
import pytest

import oracle
from brasa_amd import Kernels, OutDType
from brasa_amd.device import synchronize
from test_gpu_attend import Step

pytestmark = pytest.mark.gpu

CASES = [([1], [0], []), ([1], [256], []), ([65], [0], []), ([33, 1, 70], [100, 2000, 63], []),
         ([1] * 6, [100, 300, 63, 64, 1000, 130], [(3, 64), (3, 64)]), ([2] * 5, [4200, 4100, 4097, 4300, 4500], [(5, 4096)]),
         ([300, 9], [900, 3000], [])]
HEADS = [(32, 8), (4, 4), (16, 1), (128, 1)]


class Short(Step):
    def call(self, stream=None, ws=None):
        ws = ws or self.ws
        Kernels().attention_paged(self.gq, self.dev, self.layer, self.gt, len(self.new), self.width, self.tokens, ws,
                                  ws.nbytes, self.o, self.hq, self.out, stream, short=True)


def _result(kind, out, **kw):
    s = kind(out=out, **kw).upload()
    s.plan()
    s.call()
    synchronize()
    return s, s.raw()[s.cu[0] * s.hq * 128:s.cu[-1] * s.hq * 128]


@pytest.mark.parametrize("new,held,groups", CASES, ids=str)
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_f16_results_are_f32_results_rounded(new, held, groups, hq, hkv):
    print("rounded", new[:5], groups, hq, hkv, flush=True)
    kw = dict(new=new, held=held, groups=groups, hq=hq, hkv=hkv, seed=len(new) + hq)
    s, exact = _result(Step, OutDType.F32, **kw)
    s.check()
    got = oracle.f16_to_f32(_result(Step, OutDType.F16, **kw)[1]).astype(np.float64)
    exact = exact.astype(np.float64)
    step = 2.0 ** np.maximum(np.frexp(exact)[1] - 11, -24)  # of f16: 11 bits, 2^-24 at least
    assert np.all(np.abs(got - exact) <= step / 2 + 2.0 ** -24 * np.abs(exact))


@pytest.mark.parametrize("new,held,groups", CASES, ids=str)
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_short(new, held, groups, hq, hkv):
    print("short", new[:5], groups, hq, hkv, flush=True)
    kw = dict(new=new, held=held, groups=groups, hq=hq, hkv=hkv, seed=len(new) + hq)
    s, got = _result(Short, OutDType.F16, **kw)
    s.check()
    if sum(held) > 2000:  # (a form of its own)
        assert not np.array_equal(got, _result(Step, OutDType.F16, **kw)[1])


def test_short_values_that_are_not_finite():
    s = Short(new=[50, 1, 9], held=[70, 200, 128], groups=[(3, 64)], hq=8, hkv=2, out=OutDType.F16, seed=8)
    s.pool.v[0, s.table[0, 1], 1, 20, 5] = 127    # position 84, below some of sequence 0's rows only
    s.pool.k[0, s.table[1, 3], 0, 3, 7] = 127     # position 195: sequence 1 sees it
    s.q[s.cu[1] - 3] = np.nan
    s.upload()
    s.plan()
    s.call()
    synchronize()
    s.check()


def test_short_without_a_plan():
    s = Short(new=[1, 1], held=[100, 90], hq=4, hkv=2, seed=12, out=OutDType.F16).upload()
    s.o.fill(0)
    s.call()
    synchronize()
    assert np.isnan(oracle.f16_to_f32(s.raw())).all()
