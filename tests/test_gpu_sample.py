"""g4_sample against its definition in 64 bits: equal tokens, and probabilities to 1e-6
relative (FP32's half step 2^-24 and what 64-bit sums of 10^5 exponentials may differ by,
far below).  A token could differ only where u lies within about 1e-12 of a border."""
import numpy as np
import pytest

import draft_reference as ref

pytestmark = pytest.mark.gpu


def run(g4, x, u, stride=None, **cuts):
    rows, vocab = x.shape
    stride = vocab if stride is None else stride
    wide = np.full((rows, stride), 1e9, np.float32)
    wide[:, :vocab] = x
    tok, pr = g4.Buffer.from_array(np.full(rows, -7, np.int32)), g4.Buffer(rows * 4)
    g4.sample(g4.Buffer.from_array(wide), rows, vocab, g4.Buffer.from_array(np.asarray(u, np.float32)),
              tok, pr, stride, **cuts)
    return tok.download(np.int32), pr.download(np.float32)


def check(g4, x, u, stride=None, **cuts):
    print("sample", x.shape, cuts, flush=True)
    tok, pr = run(g4, x, u, stride, **cuts)
    for r in range(x.shape[0]):
        t, p = ref.sample(x[r], np.float32(u[r]), **cuts)
        assert tok[r] == t, (r, tok[r], t)
        assert abs(pr[r] - p) <= 1e-6 * p, (r, pr[r], p)


def logits(rng, rows, vocab, spread=3.0):
    x = rng.standard_normal((rows, vocab)) * spread
    for r in range(rows):
        x[r, rng.integers(0, vocab, 6)] += 4 * spread
    return (30 * np.tanh(x / 30)).astype(np.float32)


CUTS = [dict(), dict(temperature=0.7), dict(temperature=2.5, top_k=1), dict(top_k=50),
        dict(top_p=0.9), dict(min_p=0.02), dict(temperature=0.8, top_k=100, top_p=0.95),
        dict(temperature=1.3, top_k=500, top_p=0.8, min_p=0.001), dict(top_p=0.3, min_p=0.5),
        dict(top_p=1e-6), dict(min_p=1.0), dict(temperature=0.0, top_k=9), dict(top_k=10 ** 9),
        dict(temperature=1e-3), dict(temperature=1e3, top_p=0.5)]


@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 2), (3, 63), (4, 1000), (2, 4096), (5, 4097),
                                        (2, 16384), (3, 30011), (1, 65536), (3, 262144), (2, 300001)])
def test_shapes_and_cuts(g4, rows, vocab):
    rng = np.random.default_rng([rows, vocab])
    x = logits(rng, rows, vocab)
    for cuts in CUTS:
        check(g4, x, rng.random(rows), stride=vocab + 3 * rows, **cuts)


@pytest.mark.parametrize("rows,vocab", [(40, 5000), (64, 70000), (200, 300)])
def test_many_rows(g4, rows, vocab):
    rng = np.random.default_rng([rows, vocab])
    x = logits(rng, rows, vocab, spread=1.5)
    for cuts in CUTS[:9]:
        check(g4, x, rng.random(rows), **cuts)


@pytest.mark.parametrize("vocab", [1900, 3000, 4096, 8191])
def test_ties_in_rows_of_one_slice(g4, vocab):
    # 8191 equal logits are more than the tokens listed near by
    rng = np.random.default_rng(vocab)
    x = rng.integers(-8, 4, (4, vocab)).astype(np.float32)
    x[1] = 1.25
    x[2] = rng.integers(0, 2, vocab) * 0.125
    x[3] = logits(rng, 1, vocab, 0.3)[0]
    for cuts in CUTS + [dict(top_k=vocab // 2), dict(top_k=vocab // 3, top_p=0.77),
                        dict(top_k=17, top_p=0.5, min_p=0.3)]:
        check(g4, x, rng.random(4), **cuts)


@pytest.mark.parametrize("rows,vocab", [(130, 70000), (300, 9000)])
def test_many_rows_of_several_slices(g4, rows, vocab):
    # 130 rows: enough for long slices; 300 rows: more than one launch takes
    rng = np.random.default_rng([rows, vocab])
    x = logits(rng, rows, vocab, spread=1.5)
    x[1] = 0.5  # more equal logits than a list holds
    x[2] = rng.integers(-3, 2, vocab)
    x[3] = rng.integers(-9, 2, vocab)
    x[rows - 1, ::3] = -np.inf
    x[rows - 2] = np.nan
    for cuts in [dict(), dict(temperature=0.7), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.02),
                 dict(top_k=vocab // 5), dict(temperature=1.3, top_k=vocab // 4, top_p=0.8, min_p=0.001)]:
        check(g4, x, rng.random(rows), **cuts)


def test_the_largest_vocabulary(g4):
    vocab = 1 << 22
    rng = np.random.default_rng(22)
    x = logits(rng, 2, vocab)
    x[1] = rng.integers(-2, 3, vocab)
    for cuts in [dict(), dict(temperature=0.8, top_k=100, top_p=0.95), dict(top_k=vocab // 3),
                 dict(top_p=0.9), dict(min_p=0.02)]:
        check(g4, x, rng.random(2), **cuts)


def test_rows_far_apart(g4):
    # the second row starts past 2^31 values
    vocab, stride = 10001, 2 ** 31 + 12
    rng = np.random.default_rng(23)
    x, u = logits(rng, 2, vocab), rng.random(2).astype(np.float32)
    b = g4.Buffer((stride + vocab) * 4)
    for r in range(2):
        b.upload(x[r], r * stride * 4)
    bu, tok, pr = g4.Buffer.from_array(u), g4.Buffer(8), g4.Buffer(8)
    for cuts in (dict(), dict(top_k=50, top_p=0.9)):
        g4.sample(b, 2, vocab, bu, tok, pr, stride, **cuts)
        want = [ref.sample(x[r], u[r], **cuts) for r in range(2)]
        assert tok.download(np.int32).tolist() == [w[0] for w in want]
        np.testing.assert_allclose(pr.download(np.float32), [w[1] for w in want], rtol=1e-6)


@pytest.mark.parametrize("vocab", [257, 20000, 150000])
def test_ties_go_to_the_lowest_index(g4, vocab):
    # logits of few values: every cut falls among equal ones
    rng = np.random.default_rng(vocab)
    x = rng.integers(-8, 4, (4, vocab)).astype(np.float32)
    x[1] = 1.25  # all equal
    x[2] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)  # zeros are equal
    x[3, 1:] = np.minimum(x[3, 1:], 2.0)
    for cuts in CUTS + [dict(top_k=vocab // 2), dict(top_k=vocab // 3, top_p=0.77),
                        dict(top_k=17, top_p=0.5, min_p=0.3)]:
        check(g4, x, rng.random(4), **cuts)


def test_exact_borders(g4):
    # eight equal logits: token k from u = k / 8 on
    x = np.zeros((8, 8), np.float32)
    u = np.arange(8, dtype=np.float32) / 8
    assert run(g4, x, u)[0].tolist() == list(range(8))
    assert run(g4, x, np.nextafter(u, np.float32(-1)))[0].tolist() == [0] + list(range(7))
    # half of the mass is four tokens, whatever lies behind
    assert run(g4, x, u, top_p=0.5)[0].tolist() == [0, 0, 1, 1, 2, 2, 3, 3]
    assert run(g4, x, u, top_k=2)[0].tolist() == [0] * 4 + [1] * 4


@pytest.mark.parametrize("vocab", [50, 9000, 262144])
def test_random_numbers_at_the_ends(g4, vocab):
    rng = np.random.default_rng(vocab)
    x = np.repeat(logits(rng, 1, vocab, 1.0), 7, 0)
    u = np.array([0.0, -0.0, -3.0, np.nan, 1 - 2.0 ** -24, 1.0, np.inf], np.float32)
    ids, _ = ref.kept(x[0], top_k=40)
    tok, _ = run(g4, x, u, top_k=40)
    assert tok.tolist() == [ids[0]] * 4 + [ids[-1]] * 3
    check(g4, x[:5], u[:5])
    check(g4, x[:1], np.array([1e-30], np.float32), temperature=0.9)


@pytest.mark.parametrize("vocab", [5, 3000, 100003])
def test_only_finite_logits_take_part(g4, vocab):
    rng = np.random.default_rng(vocab)
    x = logits(rng, 5, vocab)
    x[0, rng.random(vocab) < 0.7] = -np.inf
    x[0, vocab // 2] = 1.0
    x[1, rng.random(vocab) < 0.7] = np.nan
    x[1, vocab - 1] = 1.0
    x[2, ::2] = np.inf
    x[3] = [-np.inf, np.inf, np.nan][vocab % 3]
    x[4] = -np.inf
    x[4, vocab - 2] = -3e38
    for cuts in CUTS:
        check(g4, x, rng.random(5), **cuts)
    assert run(g4, x, np.zeros(5))[0][3] == -1


def test_largest_and_lowest_logits(g4):
    x = np.array([[3.4e38, -3.4e38, 3.4e38, 0], [-3.4e38, -3.4e38, -3.4e38, -3.4e38],
                  [1e-45, 0, -1e-45, 0]], np.float32)
    for cuts in CUTS:
        check(g4, x, np.array([0.6, 0.3, 0.9]), **cuts)


def test_temperature_zero_is_the_argmax(g4):
    rng = np.random.default_rng(2)
    x = logits(rng, 3, 262144)
    x[1, [77, 200000]] = 29.9
    tok, pr = run(g4, x, rng.random(3), temperature=0.0, top_p=0.5, min_p=0.1)
    for r in range(3):
        o = g4.Buffer(4)
        g4.argmax(g4.Buffer.from_array(x[r]), x.shape[1], o)
        assert tok[r] == o.download(np.int32)[0]
    assert (pr == 1).all()


def test_a_flat_row_follows_its_distribution(g4):
    # 4096 evenly spread numbers over 16 tokens of known probabilities
    p = np.arange(1, 17) / np.arange(1, 17).sum()
    x = np.log(p).astype(np.float32)[None].repeat(4096, 0)
    tok, pr = run(g4, x, (np.arange(4096) + 0.5) / 4096)
    counts = np.bincount(tok, minlength=16)
    assert np.abs(counts - 4096 * p).max() <= 1.01  # the two borders of each token
    np.testing.assert_allclose(pr, p[tok], rtol=1e-6)


def test_probabilities_are_optional(g4):
    x = g4.Buffer.from_array(np.zeros(10, np.float32))
    u, t = g4.Buffer.from_array(np.array([0.35], np.float32)), g4.Buffer(4)
    g4.sample(x, 1, 10, u, t)
    assert t.download(np.int32)[0] == 3


def test_refuses_short_buffers(g4):
    x, u, t = g4.Buffer(400), g4.Buffer(8), g4.Buffer(8)
    for args in ((x, 1, 101, u, t), (x, 2, 50, u, t, None, 51), (x, 3, 20, u, t), (x, 2, 20, u, None)):
        with pytest.raises(g4.G4Error):
            g4.sample(*args)
