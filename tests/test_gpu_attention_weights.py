"""g4_attention_weights against its definition in 64 bits.

Tolerance: a score is a sum of at most 512 products with sum |q k| < 33, q and k as they are or as
sums of FP16 or BF16 values that hold them to 2^-22, so off by less than 33 * 2^-21 = 1.6e-5 in the
worst case and 1e-6 in general; a weight by the same relative amount: 2e-5 of it."""
import numpy as np
import pytest

import long_cache_reference as ref

pytestmark = pytest.mark.gpu
TOL = 2e-5


def inputs(rng, qrows, heads, hd, keys):
    at = 1.5 / hd ** 0.25
    return ((rng.standard_normal((qrows, heads, hd)) * at).astype(np.float32),
            (rng.standard_normal((keys, hd)) * at).astype(np.float32))


def run(g4, q, k, keys, qpos0, window, before=None):
    w = g4.Buffer.from_array(np.full(keys, np.nan, np.float32))
    b = g4.Buffer.from_array(before) if before is not None else None
    g4.attention_weights(g4.Buffer.from_array(q), g4.Buffer.from_array(k), len(q), q.shape[1], q.shape[2], keys,
                         qpos0, window > 0, window, w, b)
    return w.download(np.float32)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("qrows,heads,keys,qpos0,window", [
    (1, 8, 1, 0, 0), (1, 1, 2, 1, 0), (1, 8, 15, 14, 0), (1, 8, 17, 16, 0), (1, 7, 300, 299, 0), (2, 8, 64, 62, 0),
    (3, 5, 65, 62, 0), (4, 8, 127, 120, 16), (1, 8, 2000, 1999, 512), (1, 3, 600, 599, 1), (5, 8, 5, 0, 0),
    (17, 8, 17, 0, 0), (33, 8, 90, 57, 0), (64, 8, 700, 636, 64), (70, 1, 200, 130, 0), (129, 2, 400, 200, 33),
    (1, 8, 500, 100, 0), (9, 8, 100, 50, 3), (1, 8, 5000, 4999, 0), (40, 8, 3333, 3293, 0)])
def test_shapes(g4, hd, qrows, heads, keys, qpos0, window):
    print("weights", hd, qrows, heads, keys, qpos0, window, flush=True)
    rng = np.random.default_rng([hd, qrows, heads, keys])
    q, k = inputs(rng, qrows, heads, hd, keys)
    before = (rng.random(keys) * qrows * heads / keys).astype(np.float32) if keys % 2 else None
    want = ref.weights(q, k, keys, qpos0, window).sum((0, 1)) + (0 if before is None else before)
    assert (np.abs(run(g4, q, k, keys, qpos0, window, before) - want) <= TOL * want).all()


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_long_cache(g4, hd):
    rng = np.random.default_rng(hd)
    q, k = inputs(rng, 2, 8, hd, 30007)
    want = ref.weights(q, k, 30007, 30005).sum((0, 1))
    assert (np.abs(run(g4, q, k, 30007, 30005, 0) - want) <= TOL * want).all()


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("qrows", [1, 20])
def test_unseen_rows_have_no_influence(g4, hd, qrows):
    rng = np.random.default_rng([hd, 2])
    q, k = inputs(rng, qrows, 8, hd, 300)
    want = run(g4, q, k, 300, 200, 50)
    for fill in (np.nan, np.inf, -np.inf, 3.4e38):
        k[:151], k[200 + qrows:] = fill, fill
        np.testing.assert_array_equal(run(g4, q, k, 300, 200, 50), want)
    assert (want[:151] == 0).all() and (want[200 + qrows:] == 0).all() and (want[151:200 + qrows] > 0).all()


@pytest.mark.parametrize("hd", [64, 512])
def test_a_key_without_numbers_reaches_the_rows_that_see_it(g4, hd):
    rng = np.random.default_rng([hd, 3])
    q, k = inputs(rng, 20, 4, hd, 120)
    k[110, 7] = np.nan
    got = run(g4, q, k, 120, 100, 12)
    assert np.isnan(got[110 - 11:]).all()
    want = ref.weights(q, np.where(np.isnan(k), 0, k), 120, 100, 12)[:10].sum((0, 1))
    assert (np.abs(got[:99] - want[:99]) <= TOL * want[:99]).all()


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("exp", [-100, -30, 30, 100])
def test_value_ranges(g4, hd, exp):
    rng = np.random.default_rng([hd, 4])
    q, k = inputs(rng, 4, 8, hd, 200)
    want = ref.weights(q, k, 200, 196).sum((0, 1))
    got = run(g4, q * np.float32(2.0 ** -exp), k * np.float32(2.0 ** exp), 200, 196, 0)
    assert (np.abs(got - want) <= TOL * want).all()


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_values_of_very_different_sizes_in_a_row(g4, hd):
    # a large k meets a small q and the other way round, so that all products are alike
    rng = np.random.default_rng([hd, 5])
    q, k = inputs(rng, 4, 8, hd, 200)
    e = rng.integers(-8, 9, hd)
    want = ref.weights(q, k, 200, 196).sum((0, 1))
    got = run(g4, q * np.exp2(-e).astype(np.float32), k * np.exp2(e).astype(np.float32), 200, 196, 0)
    assert (np.abs(got - want) <= TOL * want).all()


def test_in_place_over_calls(g4):
    rng = np.random.default_rng(6)
    q, k = inputs(rng, 30, 8, 256, 500)
    w, kb = g4.Buffer.from_array(np.full(500, 0.5, np.float32)), g4.Buffer.from_array(k)
    for i in range(3):
        g4.attention_weights(g4.Buffer.from_array(q[10 * i:10 * i + 10]), kb, 10, 8, 256, 480 + 10 * i, 470 + 10 * i,
                             False, 0, w, w)
    want = 0.5 + ref.weights(q, k, 500, 470).sum((0, 1))
    assert (np.abs(w.download(np.float32) - want) <= TOL * want).all()


def test_equal_to_those_of_a_4_bit_cache(g4):
    # of the same values: the sums of g4_attention_kv4
    rng = np.random.default_rng(7)
    q, k = inputs(rng, 3, 8, 256, 700)
    c, x = g4.Kv4Cache(700, 256), g4.Buffer.from_array(k)
    c.append(x, x, 700, 0)
    c.read(0, 700, x, None)
    w, y = g4.Buffer(2800), g4.Buffer(q.nbytes)
    c.attention(g4.Buffer.from_array(q), 3, 8, 700, 697, False, 0, y, w)
    got = run(g4, q, x.download(np.float32).reshape(k.shape), 700, 697, 0)
    np.testing.assert_allclose(got, w.download(np.float32), rtol=2 * TOL)


def test_refuses_short_buffers(g4):
    q, k, w = g4.Buffer(2 * 8 * 64 * 4), g4.Buffer(50 * 64 * 4), g4.Buffer(50 * 4)
    small = g4.Buffer(49 * 4)
    g4.attention_weights(q, k, 2, 8, 64, 50, 48, False, 0, w)
    for args in ((q, k, 2, 8, 64, 51, 49, False, 0, w), (q, k, 3, 8, 64, 50, 47, False, 0, w),
                 (q, k, 2, 8, 64, 50, 48, False, 0, small), (q, k, 2, 8, 64, 50, 48, False, 0, w, small),
                 (None, k, 2, 8, 64, 50, 48, False, 0, w), (q, None, 2, 8, 64, 50, 48, False, 0, w),
                 (q, k, 2, 8, 64, 50, 48, False, 0, None)):
        with pytest.raises(g4.G4Error):
            g4.attention_weights(*args)
    g4.attention_weights(None, k, 0, 8, 64, 50, 50, False, 0, w)
    np.testing.assert_array_equal(w.download(np.float32), 0)
