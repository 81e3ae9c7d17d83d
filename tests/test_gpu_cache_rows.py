"""g4_cache_rows: copied bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def planes(g4, rng, widths, cap, extra=0):
    a = [rng.standard_normal((cap, w)).astype(np.float32) for w in widths]
    return a, [g4.Buffer.from_array(p) for p in a]


def idx(g4, rows):
    return g4.Buffer.from_array(np.asarray(rows, np.int32))


def want_rows(a, rows):
    ok = (np.asarray(rows) >= 0) & (np.asarray(rows) < len(a))
    got = a[np.where(ok, rows, 0)].copy()
    got[~ok] = np.nan
    return got


@pytest.mark.parametrize("widths", [[256, 512], [4], [1, 3, 7], [64] * 128, [255, 256], [516, 2048]])
@pytest.mark.parametrize("n,at,cap", [(1, 0, 1), (3, 5, 20), (16, 40, 64), (17, 3, 64), (33, 20, 90),
                                      (64, 0, 64), (65, 10, 200), (300, 100, 777)])
def test_in_place(g4, widths, n, at, cap):
    rng = np.random.default_rng([len(widths), n])
    print("in place", widths[:3], n, at, cap, flush=True)
    for rows in (np.sort(rng.choice(np.arange(at, cap), n, replace=False)) if cap - at >= n else
                 np.sort(rng.integers(0, cap, n)),
                 rng.integers(0, cap, n),                       # any order, twice the same
                 np.arange(at + n - 1, at - 1, -1)):            # reversed onto itself
        a, b = planes(g4, rng, widths, cap)
        g4.CachePlanes(b, b, widths).rows(idx(g4, rows), n, at, cap)
        for p, buf in zip(a, b):
            w = p.copy()
            w[at:at + n] = want_rows(p, rows)
            np.testing.assert_array_equal(buf.download(np.float32).reshape(p.shape), w)


@pytest.mark.parametrize("widths", [[256, 512], [5, 1], [1024]])
@pytest.mark.parametrize("n,at", [(1, 0), (40, 7), (1000, 0), (3001, 50)])
def test_into_another_cache(g4, widths, n, at):
    rng = np.random.default_rng([n, at])
    cap = 3100
    a, src = planes(g4, rng, widths, cap)
    c, dst = planes(g4, rng, widths, at + n + 3)
    rows = rng.integers(0, cap, n)
    g4.CachePlanes(dst, src, widths).rows(idx(g4, rows), n, at, cap)
    for p, old, d, s in zip(a, c, dst, src):
        old[at:at + n] = p[rows]
        np.testing.assert_array_equal(d.download(np.float32).reshape(old.shape), old)
        np.testing.assert_array_equal(s.download(np.float32).reshape(p.shape), p)


def test_planes_side_by_side_in_one_buffer(g4):
    # shifted pointers (not 16-byte aligned) into one allocation; some in place, some not
    rng = np.random.default_rng(5)
    a = rng.standard_normal(1 + 60 * 8 + 60 * 8 + 60 * 8).astype(np.float32)
    b = g4.Buffer.from_array(a)
    p = [b.at(4 * (1 + 480 * i)) for i in range(3)]
    rows = np.array([50, 49, 3, 3, 59, 0])
    g4.CachePlanes([p[0], p[2]], [p[0], p[1]], [8, 8]).rows(idx(g4, rows), 6, 2, 60)
    w = a.copy()
    v = [w[1 + 480 * i:1 + 480 * (i + 1)].reshape(60, 8) for i in range(3)]
    first, second = v[0][rows].copy(), v[1][rows].copy()
    v[0][2:8], v[2][2:8] = first, second
    np.testing.assert_array_equal(b.download(np.float32), w)


@pytest.mark.parametrize("n", [5, 70])
@pytest.mark.parametrize("place", [True, False])
def test_rows_outside_the_source_are_nan(g4, n, place):
    rng = np.random.default_rng(n)
    a, src = planes(g4, rng, [256, 12], 100)
    dst = src if place else [g4.Buffer(100 * w * 4) for w in (256, 12)]
    rows = rng.integers(0, 100, n)
    rows[[0, n // 2, n - 1]] = [-1, 100, 2 ** 31 - 1]
    g4.CachePlanes(dst, src, [256, 12]).rows(idx(g4, rows), n, 20, 100)
    for p, d in zip(a, dst):
        np.testing.assert_array_equal(d.download(np.float32).reshape(p.shape)[20:20 + n],
                                      want_rows(p, rows))


def test_nothing_to_do(g4):
    a, b = planes(g4, np.random.default_rng(1), [16], 4)
    g4.CachePlanes(b, b, [16]).rows(idx(g4, [0]), 0, 0, 4)
    np.testing.assert_array_equal(b[0].download(np.float32).reshape(4, 16), a[0])


def test_refuses_rows_outside_the_planes(g4):
    _, b = planes(g4, np.random.default_rng(1), [16, 16], 10)
    small = g4.Buffer(9 * 16 * 4)
    for dst, src, n, at, cap in (([b[0], small], b, 5, 5, 10), (b, [b[0], small], 5, 5, 10),
                                 (b, b, 6, 5, 10), (b, b, 2, 0, 11)):
        with pytest.raises(g4.G4Error) as e:
            g4.CachePlanes(dst, src, [16, 16]).rows(idx(g4, range(6)), n, at, cap)
        assert e.value.code == g4.G4_E_RANGE
    with pytest.raises(g4.G4Error):
        g4.CachePlanes(b, b, [16, 16]).rows(idx(g4, [0]), 2, 0, 10)


@pytest.mark.parametrize("shift", [4, 1, 8, 64, 260, 512])
@pytest.mark.parametrize("n", [7, 64, 100])
def test_planes_that_overlap_at_any_shift(g4, shift, n):
    # dst begins `shift` values behind src: whole rows of 256 or not
    rng = np.random.default_rng([shift, n])
    w, cap, at = 256, 200, 30
    a = rng.standard_normal(cap * w + shift).astype(np.float32)
    rows = rng.integers(0, cap, n)
    for d, s in ((shift, 0), (0, shift)):
        b = g4.Buffer.from_array(a)
        g4.CachePlanes([b.at(4 * d)], [b.at(4 * s)], [w]).rows(idx(g4, rows), n, at, cap)
        want = a.copy()
        want[d + at * w:d + (at + n) * w] = a[s:s + cap * w].reshape(cap, w)[rows].ravel()
        np.testing.assert_array_equal(b.download(np.float32), want)


def test_a_cache_past_32_bits(g4):
    w, cap = 512, 2 ** 22 + 500  # the last rows lie past 2^31 values
    rng = np.random.default_rng(7)
    b, near = g4.Buffer(cap * w * 4), rng.standard_normal((300, w)).astype(np.float32)
    for n in (40, 200):
        b.upload(near, (cap - 300) * w * 4)
        rows = np.sort(rng.choice(300, n, False))
        g4.CachePlanes([b], [b], [w]).rows(idx(g4, cap - 300 + rows), n, cap - 300, cap)
        got = b.download(np.float32, 300 * w, (cap - 300) * w * 4).reshape(300, w)
        np.testing.assert_array_equal(got[:n], near[rows])
        np.testing.assert_array_equal(got[n:], near[n:])
