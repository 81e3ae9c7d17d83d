"""The attention kernels of long caches where they change their way or their offsets grow: many rows
of which some need another kernel, recordings of such calls, sums over several chunks of scores,
caches past 4 GiB.

Tolerances as in test_gpu_kv4.py and test_gpu_attention_weights.py, 2e-5 of max |v| and of a key's
weight, unless a test says otherwise."""
import numpy as np
import pytest

import long_cache_reference as ref
from test_gpu_kv4 import TOL, attend, cache_of, inputs

pytestmark = pytest.mark.gpu
HEADS = 8


def odd_rows(rng, what, hd, qrows, keys):
    """Inputs of which some rows are unlike the others."""
    q, k, v = inputs(rng, qrows, HEADS, hd, keys)
    if what == "zero q":
        q[::3] = 0
    elif what == "tiny q":
        q[qrows // 9:qrows // 5 + 1] *= np.float32(2.0 ** -104)
    elif what == "tiny k":
        k[100:140] *= np.float32(2.0 ** -20)  # scales below 2^-18
        k[3] *= np.float32(2.0 ** -90)
    elif what == "large v":
        v[50:60] *= 1024  # scales above 2^7
        v[7, :64] = 0   # scales of 1
    elif what == "one late key":
        v[-1] *= 2048     # seen by the last row alone
    return q, k, v


ODD = ["zero q", "tiny q", "tiny k", "large v", "one late key"]


@pytest.mark.parametrize("hd,qrows,keys,window", [(hd, 45, 333, window) for hd in (64, 128, 256, 512) for window in (0, 130)] +
                         [(512, 140, 2100, 0), (512, 200, 2100, 1500), (256, 140, 2100, 0)])
@pytest.mark.parametrize("what", ODD)
def test_some_rows_unlike_the_others(g4, hd, qrows, keys, window, what):
    rng = np.random.default_rng([hd, window, len(what)])
    q, k, v = odd_rows(rng, what, hd, qrows, keys)
    pk, pv = ref.pack(k), ref.pack(v)
    y, w = attend(g4, cache_of(g4, pk, pv, hd), q, keys, keys - qrows, window, True)
    p = ref.weights(q, ref.unpack(*pk), keys, keys - qrows, window)
    # (of each row's own largest: a v that a row does not see has no part in it)
    vv = ref.unpack(*pv)
    for r in range(qrows):
        end = keys - qrows + r + 1
        seen = np.abs(vv[max(0, end - window) if window else 0:end]).max()
        assert np.abs(y[r] - p[r] @ vv).max() <= TOL * seen
    want = p.sum((0, 1))
    assert (np.abs(w - want) <= TOL * want).all()


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("window", [0, 130])
@pytest.mark.parametrize("what", ["zero q", "tiny q", "tiny k", "large k", "large q", "large q, tiny k"])
@pytest.mark.parametrize("qrows", [45, 4, 1])
def test_fp32_keys_unlike_the_others(g4, hd, window, what, qrows):
    rng = np.random.default_rng([hd, window, len(what), 1])
    keys = 333
    q, k, _ = odd_rows(rng, what, hd, qrows, keys)
    if what == "large k":
        q[:, :, 0], k[:, 0] = 0, 0
        k[20:22, 0] = 500  # of no weight, but for the whole row's split into two values
    if what.startswith("large q"):
        q[:, :, 1], k[:, 1] = 0, 0
        q[qrows // 4:qrows // 4 + 2, :, 1] = 400
    if what == "large q, tiny k":
        k[60:70] *= np.float32(2.0 ** -14)
        k[60:70, 1] = np.float32(2.0 ** -14)  # 0.024 of those rows' scores
    want = ref.weights(q, k, keys, keys - qrows, window).sum((0, 1))
    w = g4.Buffer.from_array(np.full(keys, np.nan, np.float32))
    g4.attention_weights(g4.Buffer.from_array(q), g4.Buffer.from_array(k), qrows, HEADS, hd, keys, keys - qrows,
                         window > 0, window, w)
    got = w.download(np.float32)
    assert (np.abs(got - want) <= TOL * want).all()


@pytest.mark.parametrize("hd,qrows,keys", [(512, 45, 700), (512, 140, 2100), (512, 2100, 2200), (256, 45, 700),
                                           (256, 2200, 2300)])
def test_recordings_whose_rows_change_their_kernel(g4, hd, qrows, keys):
    """Replays equal eager calls to the bit, whatever the replay before needed."""
    rng = np.random.default_rng([hd, qrows])
    c = g4.Kv4Cache(keys, hd)
    q, y = (g4.Buffer(qrows * HEADS * hd * 4) for _ in range(2))
    w, w2 = g4.Buffer(keys * 4), g4.Buffer(keys * 4)
    k = g4.Buffer(keys * hd * 4)
    heavy = qrows > 1000

    def call():
        c.attention(q, qrows, HEADS, keys, keys - qrows, False, 0, y, None if heavy else w)
        if not heavy:
            g4.attention_weights(q, k, qrows, HEADS, hd, keys, keys - qrows, False, 0, w2)

    def fill(what):
        x = odd_rows(rng, what, hd, qrows, keys)
        if what == "large k":
            x[0][:, :, 0] = 0
            x[1][:, 0] = 300
        kb, vb = (g4.Buffer.from_array(a) for a in x[1:])
        c.append(kb, vb, keys, 0)
        k.upload(x[1])
        q.upload(x[0])
        return x

    outs = (y,) if heavy else (y, w, w2)
    fill("")
    call()
    with g4.Encoder() as enc:
        call()
    plain = fill("")
    call()
    first = [b.download(np.uint32) for b in outs]
    for what in ("", "large v", "large k", "tiny k", "", "tiny q", ""):
        fill(what)
        call()
        want = [b.download(np.uint32) for b in outs]
        for b in outs:
            b.upload(np.full(b.nbytes // 4, np.nan, np.float32))
        enc.cmdbuf.submit()
        for b, a in zip(outs, want):
            np.testing.assert_array_equal(b.download(np.uint32), a)
        # and the plain inputs give what they gave at first
        kb, vb = (g4.Buffer.from_array(a) for a in plain[1:])
        c.append(kb, vb, keys, 0)
        k.upload(plain[1])
        q.upload(plain[0])
        enc.cmdbuf.submit()
        for b, a in zip(outs, first):
            np.testing.assert_array_equal(b.download(np.uint32), a)


@pytest.mark.parametrize("hd", [64, 512])
@pytest.mark.parametrize("window", [0, 9000])
def test_scores_in_several_chunks(g4, hd, window):
    """More scores than are kept at once: 512 * 8 rows over 20011 keys."""
    rng = np.random.default_rng([hd, window, 2])
    qrows, keys = 512, 20011
    q, k, v = inputs(rng, qrows, HEADS, hd, keys)
    pk, pv = ref.pack(k), ref.pack(v)
    kk, vv = ref.unpack(*pk), ref.unpack(*pv)
    before = rng.random(keys).astype(np.float32)
    y, w = attend(g4, cache_of(g4, pk, pv, hd), q, keys, keys - qrows, window, True, before)
    w2 = g4.Buffer.from_array(before)
    g4.attention_weights(g4.Buffer.from_array(q), g4.Buffer.from_array(kk.astype(np.float32)), qrows, HEADS, hd, keys,
                         keys - qrows, window > 0, window, w2, w2)
    want = before.astype(np.float64)
    for r in range(0, qrows, 64):
        p = ref.weights(q[r:r + 64], kk, keys, keys - qrows + r, window)
        assert np.abs(y[r:r + 64] - p @ vv).max() <= TOL * np.abs(v).max()
        want = want + p.sum((0, 1))
    for got in (w, w2.download(np.float32)):
        assert (np.abs(got - want) <= TOL * want).all()


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("qrows", [1, 30])
def test_a_window_longer_than_any_cache(g4, hd, qrows):
    rng = np.random.default_rng([hd, qrows, 3])
    q, k, v = inputs(rng, qrows, HEADS, hd, 200)
    c = cache_of(g4, ref.pack(k), ref.pack(v), hd)
    want = attend(g4, c, q, 200, 200 - qrows, 0, True)
    qb, kb, w = g4.Buffer.from_array(q), g4.Buffer.from_array(k), [g4.Buffer(800) for _ in range(2)]
    for i, window in enumerate((0, 0x7fffffff)):
        g4.attention_weights(qb, kb, qrows, HEADS, hd, 200, 200 - qrows, window > 0, window, w[i])
    for window in (200, 0x7fffffff):
        for a, b in zip(attend(g4, c, q, 200, 200 - qrows, window, True), want):
            np.testing.assert_allclose(a, b, rtol=2 * TOL, atol=2 * TOL)
    np.testing.assert_allclose(w[0].download(np.float32), w[1].download(np.float32), rtol=2 * TOL)


@pytest.mark.parametrize("hd", [64, 512])
def test_the_most_splits(g4, hd):
    """131149 keys, and the first 65537 of them."""
    rng = np.random.default_rng([hd, 4])
    keys = 131149
    q, k, v = inputs(rng, 1, HEADS, hd, keys)
    pk, pv = ref.pack(k), ref.pack(v)
    kk, vv = ref.unpack(*pk), ref.unpack(*pv)
    c = cache_of(g4, pk, pv, hd)
    for n in (keys, 65537):
        y, w = attend(g4, c, q, n, n - 1, 0, True)
        p = ref.weights(q, kk, n, n - 1)
        assert np.abs(y - p @ vv[:n]).max() <= TOL * np.abs(v).max()
        want = p.sum((0, 1))
        assert (np.abs(w - want) <= TOL * want).all()


def test_many_light_keys_beside_a_heavy_one(g4):
    """2^18 keys whose weights are all 2^-18.03 of the heaviest, about half of the output: their weights
    are held to 2^-38 of that, so to 2^-20 of themselves in the same direction."""
    hd, keys = 256, 1 << 18
    k, v, q = np.zeros((keys, hd), np.float32), np.ones((keys, hd), np.float32), np.zeros((1, HEADS, hd), np.float32)
    k[77, :32] = 7
    q[0, :, 0] = 12.5 / 7
    v[77] = 0.25
    v[:, ::2] *= -1
    pk, pv = ref.pack(k), ref.pack(v)
    y, w = attend(g4, cache_of(g4, pk, pv, hd), q, keys, keys - 1, 0, True)
    p = ref.weights(q, ref.unpack(*pk), keys, keys - 1)
    assert np.abs(y - p @ ref.unpack(*pv)).max() <= TOL
    want = p.sum((0, 1))
    assert (np.abs(w - want) <= TOL * want).all()


def test_a_cache_past_4_gib(g4):
    """17000000 rows of 512: planes of 4.35 GB.  All zeros (scales too) but a few rows, so that the
    sums are known: the others weigh 1 each."""
    hd, rows = 512, 17000000
    rng = np.random.default_rng(5)
    c = g4.Kv4Cache(rows, hd)
    at = [0, 5, 8388607, 16777215, 16777216, rows - 40, rows - 2, rows - 1]
    x = rng.standard_normal((len(at), hd)).astype(np.float32)
    v = rng.standard_normal((len(at), hd)).astype(np.float32)
    for i, a in enumerate(at):
        c.append(g4.Buffer.from_array(x[i:i + 1]), g4.Buffer.from_array(v[i:i + 1]), 1, a)
    back = g4.Buffer(2 * hd * 4)
    c.read(rows - 2, 2, None, back)
    vv, kk = ref.unpack(*ref.pack(v)), ref.unpack(*ref.pack(x))
    np.testing.assert_array_equal(back.download(np.float32).reshape(2, hd), vv[-2:])
    c.read(16777215, 2, back, None)
    np.testing.assert_array_equal(back.download(np.float32).reshape(2, hd), kk[3:5])
    # scores of about 14 for these keys, so that they weigh as much as all the others
    q = np.zeros((3, HEADS, hd), np.float32)
    for r in range(3):
        for h in range(HEADS):
            i = (HEADS * r + h) % len(at)
            q[r, h] = kk[i] * (15 / (kk[i] @ kk[i]))
    for qrows in (1, 3):
        pos = rows - qrows + np.arange(qrows)
        y, w = attend(g4, c, q[:qrows], rows, rows - qrows, 0, True)
        total = np.zeros(len(at))
        light = 0.0
        for r in range(qrows):
            seen = np.array(at) <= pos[r]
            e = np.where(seen, np.exp(q[r].astype(np.float64) @ kk.T), 0)
            s = (e.sum(1) + (pos[r] + 1 - seen.sum()))[:, None]
            # sum |q k| <= 15 |k|^2 / |k|^2: scores off by 15 * 2^-21 at most
            assert np.abs(y[r] - e / s @ vv).max() <= TOL * np.abs(v).max()
            total += (e / s).sum(0)
            light += (1 / s).sum()
        assert (np.abs(w[at] - total) <= TOL * total).all()
        some = w[1000:rows - 50:4999]
        some = some[~np.isin(np.arange(1000, rows - 50, 4999), at)]
        assert (np.abs(some - light) <= TOL * light).all()
    # a window of the last rows only
    y, w = attend(g4, c, q, rows, rows - 3, 41, True)
    p = np.zeros((3, HEADS, len(at)))
    for r in range(3):
        pos = rows - 3 + r
        seen = (np.array(at) <= pos) & (np.array(at) > pos - 41)
        e = np.where(seen, np.exp(q[r].astype(np.float64) @ kk.T), 0)
        p[r] = e / (e.sum(1) + 41 - seen.sum())[:, None]
        assert np.abs(y[r] - p[r] @ vv).max() <= TOL * np.abs(v).max()
    assert (np.abs(w[at] - p.sum((0, 1))) <= TOL * p.sum((0, 1))).all()
    assert (w[:rows - 43] == 0).sum() == rows - 43


def test_fp32_keys_past_4_gib(g4):
    """17000000 rows of 64 in FP32: 4.35 GB, zeros but a few."""
    hd, rows = 64, 17000000
    rng = np.random.default_rng(6)
    k = g4.Buffer(rows * hd * 4)
    at = np.array([0, 8388608, 16777215, 16777216, rows - 9, rows - 1])
    x = rng.standard_normal((len(at), hd)).astype(np.float32)
    for i, a in enumerate(at):
        k.upload(x[i], int(a) * hd * 4)
    q = np.zeros((2, HEADS, hd), np.float32)
    for r in range(2):
        for h in range(HEADS):
            i = (3 * r + h) % len(at)
            q[r, h] = x[i] * (15 / (x[i] @ x[i]))
    w = g4.Buffer(rows * 4)
    g4.attention_weights(g4.Buffer.from_array(q), k, 2, HEADS, hd, rows, rows - 2, False, 0, w)
    got = w.download(np.float32)
    want, light = np.zeros(len(at)), 0.0
    for r in range(2):
        pos = rows - 2 + r
        e = np.where(at <= pos, np.exp(q[r].astype(np.float64) @ x.T.astype(np.float64)), 0)
        s = e.sum(1) + pos + 1 - (at <= pos).sum()
        want += (e / s[:, None]).sum(0)
        light += (1 / s).sum()
    # sums of 17e6 terms in FP32, in parts: the scores' tolerance covers them
    assert (np.abs(got[at] - want) <= TOL * want).all()
    some = np.setdiff1d(np.arange(3, rows - 2, 3001), at)
    assert (np.abs(got[some] - light) <= TOL * light).all()
