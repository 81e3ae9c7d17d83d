"""Caches of 4 bits: rows written and read to the bit, and g4_attention_kv4 against its definition
in 64 bits on the values that the cache holds.

Tolerance: a q enters as two FP16 values, off by at most 2^-22 of it (two roundings of half a step
of 2^-11 each), the cache's values as they are; sum |q k| is about 1.43 sqrt(hd) <= 33 here, so a
score is off by less than 33 * 2^-22 = 8e-6 and the sums' rounding (FP32, far less), a weight by the
same relative amount, as a weight's own two FP16 values, 2^-22.  The output is off by no more than
twice that of the largest value: 2e-5 of max |v|; a key's weight by 2e-5 of it."""
import numpy as np
import pytest

import long_cache_reference as ref

pytestmark = pytest.mark.gpu
TOL = 2e-5


def inputs(rng, qrows, heads, hd, keys):
    at = 1.5 / hd ** 0.25
    q = (rng.standard_normal((qrows, heads, hd)) * at).astype(np.float32)
    k = (rng.standard_normal((keys, hd)) * at).astype(np.float32)
    v = rng.standard_normal((keys, hd)).astype(np.float32)
    return q, k, v


def cache_of(g4, packed_k, packed_v, hd):
    b = [g4.Buffer.from_array(a) for a in packed_k + packed_v]
    return g4.Kv4Cache(len(packed_k[0]), hd, b)


def attend(g4, cache, q, keys, qpos0, window, weights=False, before=None):
    y = g4.Buffer(q.nbytes)
    w = g4.Buffer.from_array(np.full(keys, np.nan, np.float32)) if weights else None
    b = g4.Buffer.from_array(before) if before is not None else None
    cache.attention(g4.Buffer.from_array(q), len(q), q.shape[1], keys, qpos0, window > 0, window, y, w, b)
    return y.download(np.float32).reshape(q.shape), w.download(np.float32) if weights else None


def check(g4, rng, qrows, heads, hd, keys, qpos0, window, weights):
    print("kv4", qrows, heads, hd, keys, qpos0, window, weights, flush=True)
    q, k, v = inputs(rng, qrows, heads, hd, keys)
    pk, pv = ref.pack(k), ref.pack(v)
    before = (rng.random(keys) * qrows * heads / keys).astype(np.float32) if weights == "added" else None
    y, w = attend(g4, cache_of(g4, pk, pv, hd), q, keys, qpos0, window, bool(weights), before)
    p = ref.weights(q, ref.unpack(*pk), keys, qpos0, window)
    want = p @ ref.unpack(*pv)
    assert np.abs(y - want).max() <= TOL * np.abs(v).max()
    if weights:
        want = p.sum((0, 1))
        if before is not None:
            want = want + before
        assert (np.abs(w - want) <= TOL * want).all()
    return y, w


# ---- rows -------------------------------------------------------------------------

@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("n,at,cap", [(1, 0, 1), (1, 1900, 2000), (5, 3, 8), (63, 1, 100), (1000, 7, 1100)])
def test_rows_to_the_bit(g4, hd, n, at, cap):
    rng = np.random.default_rng([hd, n])
    old = [rng.integers(0, 2 ** 32, (cap, hd // 8), dtype=np.uint32),
           rng.integers(0, 2 ** 16, (cap, hd // 32), dtype=np.uint16)]
    c = cache_of(g4, tuple(old), tuple(old), hd)
    x = [(rng.standard_normal((n, hd)) * np.exp(3 * rng.standard_normal((n, 1)))).astype(np.float32)
         for _ in range(2)]
    c.append(g4.Buffer.from_array(x[0]), g4.Buffer.from_array(x[1]), n, at)
    back = [g4.Buffer(x[0].nbytes) for _ in range(2)]
    c.read(at, n, back[0], back[1])
    for a, codes, scales, b in zip(x, (c.k, c.v), (c.k_scales, c.v_scales), back):
        want = [p.copy() for p in old]
        want[0][at:at + n], want[1][at:at + n] = ref.pack(a)
        np.testing.assert_array_equal(codes.download(np.uint32).reshape(want[0].shape), want[0])
        np.testing.assert_array_equal(scales.download(np.uint16).reshape(want[1].shape), want[1])
        got = b.download(np.float32).reshape(a.shape)
        np.testing.assert_array_equal(got, ref.unpack(*ref.pack(a)))  # 4 bits times 8: exact


def test_values_beside_the_borders_of_codes(g4):
    # x = (code + 1/2) scale, an ulp above and below it, for scales all over the exponents
    rng = np.random.default_rng(9)
    rows = []
    for e in list(range(-130, 124, 7)) + [-133, -128, -127, -126, -125]:
        s = np.float32(ref.wide(np.array([rng.integers(0x3f80, 0x4000)], np.uint16))[0]) * 2.0 ** e
        s = ref.wide(ref.bf16(np.array([s], np.float32)))[0]
        half = ((np.arange(-7, 7) + 0.5) * np.float64(s)).astype(np.float32)
        x = np.concatenate([half, np.nextafter(half, np.float32(np.inf)), [np.float32(7 * np.float64(s)), 0, 0, 0]])
        y = np.concatenate([half, np.nextafter(half, np.float32(-np.inf)), [np.float32(-7 * np.float64(s)), -0.0, 0, s]])
        rows.append(np.concatenate([x, y]))
    x = np.array(rows, np.float32)
    c = g4.Kv4Cache(len(x), 64)
    b = g4.Buffer.from_array(x)
    c.append(b, b, len(x), 0)
    codes, scales = ref.pack(x)
    np.testing.assert_array_equal(c.v_scales.download(np.uint16, scales.size).reshape(scales.shape), scales)
    np.testing.assert_array_equal(c.k.download(np.uint32, codes.size).reshape(codes.shape), codes)


def test_groups_of_zeros_and_of_no_numbers(g4):
    x = np.zeros((6, 128), np.float32)
    x[1, 40] = np.nan
    x[1, 3] = 5.0
    x[2, 64] = np.inf
    x[3, 127] = -np.inf
    x[4, :] = -0.0
    x[5, 0], x[5, 32], x[5, 64], x[5, 96] = 1e-45, -1e-42, 3.4e38, 1.2e-38
    c = g4.Kv4Cache(6, 128)
    b = g4.Buffer.from_array(x)
    y = g4.Buffer(x.nbytes)
    c.append(b, b, 6, 0)
    c.read(0, 6, None, y)
    got = y.download(np.float32).reshape(x.shape)
    want = ref.unpack(*ref.pack(x))
    np.testing.assert_array_equal(got, want.astype(np.float32))
    assert np.isnan(got[1, 32:64]).all() and np.isnan(got[2, 64:96]).all() and np.isnan(got[3, 96:]).all()
    assert np.isfinite(got).sum() == x.size - 96


def test_other_rows_stay_and_nothing_to_do(g4):
    rng = np.random.default_rng(1)
    c = g4.Kv4Cache(10, 64)
    x = g4.Buffer.from_array(rng.standard_normal((10, 64)).astype(np.float32))
    c.append(x, x, 10, 0)
    before = [b.download(np.uint8) for b in (c.k, c.k_scales, c.v, c.v_scales)]
    c.append(x, x, 0, 10)
    c.append(x, x, 1, 4)
    for b, old in zip((c.k, c.k_scales, c.v, c.v_scales), before):
        new = b.download(np.uint8)
        per = old.size // 10
        np.testing.assert_array_equal(np.delete(new.reshape(10, per), 4, 0), np.delete(old.reshape(10, per), 4, 0))
    c.read(3, 0, None, None)
    with pytest.raises(g4.G4Error) as e:
        c.append(x, x, 2, 9)
    assert e.value.code == g4.G4_E_ARG


def test_refuses_short_buffers(g4):
    x, small = g4.Buffer(4 * 64 * 4), g4.Buffer(3 * 64 * 4)
    c = g4.Kv4Cache(8, 64)
    short = g4.Kv4Cache(8, 64, [g4.Buffer(7 * 32), c.k_scales, c.v, c.v_scales])
    none = g4.Kv4Cache(8, 64, [c.k, None, c.v, c.v_scales])
    w = g4.Buffer(7 * 4)
    for call in (lambda: c.append(small, x, 4, 0), lambda: c.append(x, small, 4, 0), lambda: c.append(None, x, 4, 0),
                 lambda: c.read(0, 4, small, x), lambda: short.append(x, x, 4, 4), lambda: none.append(x, x, 4, 0),
                 lambda: short.attention(x, 1, 4, 8, 7, False, 0, x), lambda: none.attention(x, 1, 4, 8, 7, False, 0, x),
                 lambda: c.attention(small, 1, 4, 8, 7, False, 0, x), lambda: c.attention(x, 1, 4, 8, 7, False, 0, small),
                 lambda: c.attention(x, 1, 4, 8, 7, False, 0, x, w), lambda: c.attention(x, 1, 4, 8, 7, False, 0, None)):
        with pytest.raises(g4.G4Error):
            call()
    c.attention(x, 1, 4, 7, 6, False, 0, g4.Buffer(1024), w)


# ---- attention ---------------------------------------------------------------------

@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("qrows,heads,keys,qpos0,window", [
    (1, 8, 1, 0, 0), (1, 1, 2, 1, 0), (1, 8, 31, 30, 0), (1, 8, 32, 31, 0), (1, 8, 33, 32, 0), (1, 7, 300, 299, 0),
    (2, 8, 64, 62, 0), (3, 5, 65, 62, 0), (4, 8, 127, 120, 16), (1, 8, 2000, 1999, 512), (1, 3, 600, 599, 1),
    (5, 8, 5, 0, 0), (17, 8, 17, 0, 0), (33, 8, 90, 57, 0), (64, 8, 700, 636, 64), (70, 1, 200, 130, 0),
    (129, 2, 400, 200, 33), (1, 8, 500, 100, 0), (9, 8, 100, 50, 3), (1, 8, 5000, 4999, 0)])
def test_shapes(g4, hd, qrows, heads, keys, qpos0, window):
    rng = np.random.default_rng([hd, qrows, heads, keys])
    check(g4, rng, qrows, heads, hd, keys, qpos0, window, [None, "written", "added"][(qrows + keys) % 3])


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("qrows,keys,qpos0,window", [(1, 5003, 5002, 0), (1, 3000, 2999, 512), (20, 333, 313, 0),
                                                     (100, 1000, 900, 200), (2, 40, 38, 0)])
@pytest.mark.parametrize("weights", ["written", "added"])
def test_weights(g4, hd, qrows, keys, qpos0, window, weights):
    check(g4, np.random.default_rng([hd, qrows, keys, 7]), qrows, 8, hd, keys, qpos0, window, weights)


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_long_cache(g4, hd):
    check(g4, np.random.default_rng(hd), 1, 8, hd, 40011, 40010, 0, "added")
    check(g4, np.random.default_rng(hd), 3, 5, hd, 20011, 20008, 0, None)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("qrows", [1, 6, 40])
def test_unseen_rows_have_no_influence(g4, hd, qrows):
    rng = np.random.default_rng([hd, qrows, 3])
    keys, qpos0, window = 300, 200, 50
    q, k, v = inputs(rng, qrows, 8, hd, keys)
    pk, pv = ref.pack(k), ref.pack(v)
    want, ww = attend(g4, cache_of(g4, pk, pv, hd), q, keys, qpos0, window, True)
    for fill in (0x7fc0, 0x7f80, 0xff80, 0x7f7f):  # NaN, infinities, the largest number
        for p in (pk, pv):
            p[1][:qpos0 - window + 1] = fill
            p[1][qpos0 + qrows:] = fill
            p[0][:qpos0 - window + 1] = 0xffffffff
            p[0][qpos0 + qrows:] = 0
        y, w = attend(g4, cache_of(g4, pk, pv, hd), q, keys, qpos0, window, True)
        np.testing.assert_array_equal(y, want)
        np.testing.assert_array_equal(w, ww)
    seen = np.zeros(keys, bool)
    seen[qpos0 - window + 1:qpos0 + qrows] = True
    assert (ww[~seen] == 0).all() and (ww[seen] > 0).all()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_a_row_without_numbers_reaches_those_that_see_it(g4, hd):
    rng = np.random.default_rng([hd, 4])
    qrows, keys, qpos0 = 40, 140, 100
    q, k, v = inputs(rng, qrows, 8, hd, keys)
    pk, pv = ref.pack(k), ref.pack(v)
    want, _ = attend(g4, cache_of(g4, pk, pv, hd), q, keys, qpos0, 0)
    bad, group = 117, hd // 32 - 1
    for fill in (0x7fc0, 0x7f80):
        s = pv[1].copy()
        s[bad, group] = fill
        got, _ = attend(g4, cache_of(g4, pk, (pv[0], s), hd), q, keys, qpos0, 0)
        np.testing.assert_allclose(got[:bad - qpos0], want[:bad - qpos0], rtol=0, atol=TOL * np.abs(v).max())
        rest = got[bad - qpos0:]
        assert not np.isfinite(rest[:, :, 32 * group:]).any()
        np.testing.assert_allclose(rest[:, :, :32 * group], want[bad - qpos0:, :, :32 * group], rtol=0,
                                   atol=TOL * np.abs(v).max())
        s = pk[1].copy()
        s[bad, group] = fill
        got, w = attend(g4, cache_of(g4, (pk[0], s), pv, hd), q, keys, qpos0, 0, True)
        np.testing.assert_allclose(got[:bad - qpos0], want[:bad - qpos0], rtol=0, atol=TOL * np.abs(v).max())
        assert np.isnan(got[bad - qpos0:]).all() and np.isnan(w[:bad + 1]).all()


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_a_query_without_numbers_is_alone(g4, hd):
    rng = np.random.default_rng([hd, 5])
    q, k, v = inputs(rng, 9, 4, hd, 80)
    c = cache_of(g4, ref.pack(k), ref.pack(v), hd)
    want, _ = attend(g4, c, q, 80, 71, 0)
    q[3, 2, 5] = np.nan
    got, w = attend(g4, c, q, 80, 71, 0, True)
    assert np.isnan(got[3, 2]).all()
    got[3, 2] = want[3, 2]
    np.testing.assert_array_equal(got, want)
    assert np.isnan(w[:75]).all() and np.isfinite(w[75:]).all()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("kexp,vexp", [(-110, 0), (100, 0), (0, -90), (0, 110), (-40, 60), (30, -30)])
def test_value_ranges(g4, hd, kexp, vexp):
    # q takes back what k is scaled by; the values' size is the output's
    rng = np.random.default_rng([hd, 6])
    q, k, v = inputs(rng, 5, 8, hd, 333)
    q, k, v = (q * np.float32(2.0 ** -kexp)).astype(np.float32), k * np.float32(2.0 ** kexp), v * np.float32(2.0 ** vexp)
    pk, pv = ref.pack(k), ref.pack(v)
    y, w = attend(g4, cache_of(g4, pk, pv, hd), q, 333, 328, 0, True)
    p = ref.weights(q, ref.unpack(*pk), 333, 328)
    assert np.abs(y - p @ ref.unpack(*pv)).max() <= TOL * np.abs(v).max()
    want = p.sum((0, 1))
    assert (np.abs(w - want) <= TOL * want).all()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("seed", range(4))
def test_rows_of_very_different_sizes(g4, hd, seed):
    # v rows from 2^-40 to 2^40, the large ones with small weights, so that all matter
    rng = np.random.default_rng([hd, 7, seed])
    qrows, keys = (1, 12)[seed % 2], 260
    q, k, v = inputs(rng, qrows, 4, hd, keys)
    e = rng.integers(-40, 41, keys)
    u = np.zeros(hd, np.float32)
    u[0] = 1
    q[:, :, :32] = 0
    q[:, :, 0] = 1
    k[:, :32] = 0
    k[:, 0] = -e * np.log(2)  # a group of its own: the code is 7 or -7, times a BF16 scale
    v = (v * np.exp2(e.astype(np.float64))[:, None]).astype(np.float32)
    pk, pv = ref.pack(k), ref.pack(v)
    y, _ = attend(g4, cache_of(g4, pk, pv, hd), q, keys, keys - qrows, 0)
    p = ref.weights(q, ref.unpack(*pk), keys, keys - qrows)
    vv = ref.unpack(*pv)
    # scores of up to 60: off by 60 * 2^-22 more; each contribution by that, relative
    assert (np.abs(y - p @ vv) <= 2 * TOL * (p @ np.abs(vv)).max(-1, keepdims=True)).all()


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_large_scores(g4, hd):
    # scores in the hundreds: off by 2^-22 * sum |q k| < 2e-3, the weights alike
    rng = np.random.default_rng([hd, 8])
    q, k, v = inputs(rng, 6, 8, hd, 400)
    q *= 50
    pk, pv = ref.pack(k), ref.pack(v)
    y, w = attend(g4, cache_of(g4, pk, pv, hd), q, 400, 394, 0, True)
    p = ref.weights(q, ref.unpack(*pk), 400, 394)
    assert np.abs(y - p @ ref.unpack(*pv)).max() <= 2e-3 * np.abs(v).max()
    assert np.abs(w - p.sum((0, 1))).max() <= 2e-3 * 48
    assert abs(float(w.astype(np.float64).sum()) - 48) <= 48 * 1e-5


@pytest.mark.parametrize("hd", [64, 512])
def test_negative_scales_and_the_code_of_minus_eight(g4, hd):
    # what no append writes, but the format holds
    rng = np.random.default_rng([hd, 9])
    q, k, v = inputs(rng, 3, 8, hd, 200)
    pk, pv = ref.pack(k), ref.pack(v)
    for codes, scales in (pk, pv):
        codes[...] = rng.integers(0, 2 ** 32, codes.shape, dtype=np.uint32)
        scales[rng.random(scales.shape) < 0.5] ^= 0x8000
        scales[rng.random(scales.shape) < 0.1] = 0
    y, _ = attend(g4, cache_of(g4, pk, pv, hd), q, 200, 197, 0)
    kk, vv = ref.unpack(*pk), ref.unpack(*pv)
    p = ref.weights(q, kk, 200, 197)
    # sum |q k| is twice that of normal rows' codes
    assert np.abs(y - p @ vv).max() <= 2 * TOL * np.abs(vv).max()


def test_weights_in_place_and_over_chunks_of_rows(g4):
    # sums over several calls, in place, equal one sum to rounding
    rng = np.random.default_rng(12)
    q, k, v = inputs(rng, 30, 8, 128, 500)
    pk, pv = ref.pack(k), ref.pack(v)
    c = cache_of(g4, pk, pv, 128)
    w = g4.Buffer.from_array(np.full(500, 0.25, np.float32))
    y = g4.Buffer(q[:10].nbytes)
    for i in range(3):
        c.attention(g4.Buffer.from_array(q[10 * i:10 * i + 10]), 10, 8, 470 + 10 * i + 10, 470 + 10 * i, False, 0, y, w, w)
    want = 0.25 + ref.weights(q, ref.unpack(*pk), 500, 470).sum((0, 1))
    got = w.download(np.float32)
    assert (np.abs(got - want) <= TOL * want).all()


def test_no_rows(g4):
    c = g4.Kv4Cache(40, 64)
    w, b = g4.Buffer.from_array(np.full(40, 3, np.float32)), g4.Buffer.from_array(np.arange(40, dtype=np.float32))
    c.attention(None, 0, 8, 40, 40, False, 0, None, w, b)
    np.testing.assert_array_equal(w.download(np.float32), np.arange(40))
    c.attention(None, 0, 8, 40, 40, False, 0, None, w)
    np.testing.assert_array_equal(w.download(np.float32), 0)
    c.attention(None, 0, 8, 0, 0, False, 0, None, w)
