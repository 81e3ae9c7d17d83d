"""g4_cache_evict: the rows to the index, the kept weights to the bit."""
import numpy as np
import pytest

import long_cache_reference as ref

pytestmark = pytest.mark.gpu


def run(g4, w, keep, first, recent, n=None, place=False, kept=True):
    """w [sets, stride]; caches of n rows."""
    sets, stride = w.shape
    n = stride if n is None else n
    wb = g4.Buffer.from_array(w)
    rows = g4.Buffer.from_array(np.full(sets * keep + 3, -7, np.int32))
    kb = wb if place else g4.Buffer.from_array(np.full(w.shape, 9, np.float32)) if kept else None
    g4.cache_evict(wb, sets, n, keep, first, recent, rows, kb, stride)
    got = rows.download(np.int32)
    assert (got[sets * keep:] == -7).all()
    if not place:
        np.testing.assert_array_equal(wb.download(np.uint32), w.view(np.uint32).ravel())
    return got[:sets * keep].reshape(sets, keep), kb.download(np.float32).reshape(w.shape) if kb else None


def check(g4, w, keep, first, recent, n=None, place=False):
    print("evict", w.shape, keep, first, recent, n, place, flush=True)
    n = w.shape[1] if n is None else n
    rows, kept = run(g4, w, keep, first, recent, n, place)
    for s in range(len(w)):
        r, k = ref.evict(w[s, :n], keep, first, recent)
        np.testing.assert_array_equal(rows[s], r)
        np.testing.assert_array_equal(kept[s, :n].view(np.uint32), k.view(np.uint32))
        rest = w[s, n:] if place else np.full(w.shape[1] - n, 9, np.float32)
        np.testing.assert_array_equal(kept[s, n:].view(np.uint32), rest.view(np.uint32))


def weights(rng, sets, n):
    w = np.exp(2.5 * rng.standard_normal((sets, n)) - 3).astype(np.float32)
    w[rng.random(w.shape) < 0.05] = 0
    return w


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("sets,n,keep,first,recent", [
    (1, 1, 1, 0, 0), (1, 1, 0, 0, 0), (1, 2, 1, 0, 0), (1, 2, 1, 1, 0), (1, 2, 1, 0, 1), (2, 63, 20, 4, 8),
    (1, 64, 64, 0, 0), (3, 65, 12, 4, 8), (1, 1000, 999, 0, 0), (1, 1023, 500, 4, 128), (2, 1024, 1000, 0, 0),
    (15, 1025, 600, 3, 64), (1, 2112, 2048, 4, 128), (3, 2112, 2048, 4, 128), (5, 4097, 1, 0, 0), (3, 4096, 100, 1, 1), (2, 8192, 5000, 4, 30),
    (2, 8193, 5000, 4, 30),    (1, 16384, 4096, 4, 512), (2, 16385, 16000, 4, 512), (1, 40000, 39999, 0, 0), (1, 32768, 0, 0, 0),
    (3, 33000, 8000, 16, 300), (1, 131072, 32768, 4, 512), (2, 100003, 50001, 0, 1), (7, 20000, 19000, 9000, 9000)])
def test_shapes(g4, sets, n, keep, first, recent, place):
    check(g4, weights(np.random.default_rng([sets, n, keep]), sets, n), keep, first, recent, place=place)


@pytest.mark.parametrize("n", [50, 3000, 17000, 70000])
def test_equal_weights(g4, n):
    rng = np.random.default_rng(n)
    for w in (np.zeros((2, n)), np.full((2, n), 0.125), rng.integers(0, 3, (2, n)), rng.integers(0, 40, (2, n)) / 64,
              np.where(rng.random((2, n)) < 0.5, 0.0, -0.0)):
        w = w.astype(np.float32)
        check(g4, w, n // 3, 2, 5)
        check(g4, w, n - 1, 0, 0, place=True)


@pytest.mark.parametrize("n", [40, 5000, 66000])
def test_any_numbers(g4, n):
    rng = np.random.default_rng([n, 1])
    w = rng.integers(0, 2 ** 32, (3, n), dtype=np.uint32).view(np.float32).copy()  # NaN of both signs among them
    w[0, ::7], w[1, ::5], w[2, ::3] = np.nan, -np.inf, np.inf
    for keep in (n // 10, n // 2, n - 2):
        check(g4, w, keep, 1, 2)
        check(g4, w, keep, 0, 0, place=True)
    w[:] = np.nan
    check(g4, w, n // 2, 0, 0)


@pytest.mark.parametrize("n", [40, 5000, 66000])
def test_weights_that_differ_in_their_last_bits(g4, n):
    rng = np.random.default_rng([n, 2])
    w = (np.uint32(0x3f800000) + rng.integers(0, 700, (2, n), dtype=np.uint32)).view(np.float32)
    check(g4, w, n // 2, 3, 3)
    w = np.nextafter(np.float32(1), np.arange(2 * n, dtype=np.float32).reshape(2, n) % 3)
    check(g4, w, n // 2, 0, 0)


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("n,stride", [(100, 128), (1000, 1001), (20000, 20480), (70000, 131072)])
def test_strides(g4, n, stride, place):
    check(g4, weights(np.random.default_rng([n, stride]), 3, stride), n // 2, 4, n // 8, n, place)


def test_sorted_weights(g4):
    for n in (3000, 50000):
        w = np.sort(weights(np.random.default_rng(n), 2, n), axis=1)
        check(g4, w, n // 2, 4, 100)
        check(g4, np.ascontiguousarray(w[:, ::-1]), n // 2, 4, 100, place=True)


def test_without_kept_weights(g4):
    for n in (500, 60000):
        w = weights(np.random.default_rng(n), 2, n)
        rows, _ = run(g4, w, n // 2, 4, 9, kept=False)
        for s in range(2):
            np.testing.assert_array_equal(rows[s], ref.evict(w[s], n // 2, 4, 9)[0])


def test_most_sets_and_most_rows(g4):
    check(g4, weights(np.random.default_rng(3), 256, 300), 100, 4, 20)
    w = np.random.default_rng(4).random((1, 1 << 24), np.float32)
    check(g4, w, 1 << 20, 4, 512, place=True)


def test_refuses_short_buffers(g4):
    w, rows = g4.Buffer(2 * 100 * 4), g4.Buffer(2 * 50 * 4)
    g4.cache_evict(w, 2, 100, 50, 0, 0, rows, w)
    for args in ((w, 2, 101, 50, 0, 0, rows), (w, 3, 100, 10, 0, 0, rows), (w, 2, 100, 51, 0, 0, rows),
                 (w, 2, 100, 50, 0, 0, rows, rows), (w, 2, 100, 50, 0, 0, None), (None, 2, 100, 50, 0, 0, rows)):
        with pytest.raises(g4.G4Error):
            g4.cache_evict(*args)
    g4.cache_evict(w, 0, 100, 50, 0, 0, None)
    g4.cache_evict(w, 2, 0, 0, 0, 0, None)
