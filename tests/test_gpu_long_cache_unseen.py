"""Keys that only later rows of a call see: earlier rows' results differ from those without them by
rounding at most, whatever they hold (they may send a block of rows another way).

Tolerances: either result is within 2e-5 of max |v|, or of a key's weight, of the exact one
(test_gpu_kv4.py, test_gpu_attention_weights.py), so two are within twice that of each other."""
import numpy as np
import pytest

import long_cache_reference as ref
from test_gpu_attention_weights import run
from test_gpu_kv4 import TOL, attend, cache_of, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("qrows,keys,window", [(2, 70, 0), (12, 320, 0), (45, 320, 130), (140, 2100, 0)])
def test_a_4_bit_key_that_the_last_row_sees(g4, hd, qrows, keys, window):
    rng = np.random.default_rng([hd, qrows])
    q, k, v = inputs(rng, qrows, 8, hd, keys)
    pk, pv = ref.pack(k), ref.pack(v)
    want, _ = attend(g4, cache_of(g4, pk, pv, hd), q, keys, keys - qrows, window)
    for fill in (0x7fc0, 0x7f80, 0xff80, 0x7f7f, 0x0001, 0):  # NaN, infinities, the largest, the least, zero
        for at in ((0,), (1,), (0, 1)):
            odd = [(c, s.copy()) for c, s in (pk, pv)]
            for i in at:
                odd[i][1][-1] = fill
            got, w = attend(g4, cache_of(g4, *odd, hd), q, keys, keys - qrows, window, True)
            assert np.abs(got[:-1] - want[:-1]).max() <= 2 * TOL * np.abs(v).max()
            # rows before the last one give the last key nothing, it its own weight of the last row at most
            assert not w[-1] > 8 * (1 + TOL)


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("qrows,keys", [(2, 70), (45, 333), (140, 2100)])
@pytest.mark.parametrize("odd", [500.0, 1e30, 2.0 ** -30])
def test_an_fp32_key_that_the_last_row_sees(g4, hd, qrows, keys, odd):
    # q is 0 in the key's one other value, so that all weights are what they are without it
    rng = np.random.default_rng([hd, qrows, 1])
    q, k, _ = inputs(rng, qrows, 8, hd, keys)
    q[:, :, 0] = 0
    k[-1] = 0
    want = run(g4, q, k, keys, keys - qrows, 0)
    k[-1, 0] = odd
    got = run(g4, q, k, keys, keys - qrows, 0)
    assert (np.abs(got - want) <= 2 * TOL * want).all()


@pytest.mark.parametrize("qrows", [45, 140])
def test_small_fp32_keys_under_a_small_q(g4, qrows):
    # k of 2^-28 .. 2^-20 is held to 2^-33 where q is below 16, a score to 512 * 16 * 2^-33 < 10^-6: the
    # weights stay within their tolerance, beside keys of usual size and alone
    hd, keys = 512, 333
    rng = np.random.default_rng([qrows, 2])
    q, k = np.clip(rng.standard_normal((qrows, 8, hd)) * 6, -15.9, 15.9).astype(np.float32), np.zeros((keys, hd), np.float32)
    k[:] = rng.standard_normal((keys, hd)) * np.exp2(rng.integers(-28, -19, (keys, 1)))
    for usual in (0, 100):
        k[:usual] = rng.standard_normal((usual, hd)) * 0.05
        want = ref.weights(q, k, keys, keys - qrows).sum((0, 1))
        got = run(g4, q, k, keys, keys - qrows, 0)
        assert (np.abs(got - want) <= TOL * want).all()
