"""g4_bf16_head_rows against x . E^T and the cap in 64 bits.

Tolerance: the products are exact to 2^-23 and summed in FP32; a sum of K of them in any
order is off by a few times 2^-24 sqrt(K) of their absolute sum's mean step: 2^-24 *
(8 + sqrt(K)) * sum |x E| bounds what is seen by far.  The cap's slope is at most 1, its
tanh off by a few ulps: 4 * 2^-23 of the cap's output."""
import numpy as np
import pytest

import synthetic as syn

pytestmark = pytest.mark.gpu


def case(rng, n, rows, k):
    x = rng.standard_normal((n, k)).astype(np.float32)
    x[0] *= 30
    E = syn.bf16_rne((rng.standard_normal((rows, k)) * 0.05).astype(np.float32))
    return x, E


def run(g4, x, E, stride=None, scale=1.0, softcap=30.0):
    n, k = x.shape
    rows = E.shape[0]
    stride = rows if stride is None else stride
    out = g4.Buffer.from_array(np.full((n, stride), 7.0, np.float32))
    g4.bf16_head_rows(g4.Buffer.from_array(x), n, g4.Buffer.from_array(E), rows, k, out, stride,
                      scale, softcap)
    return out.download(np.float32).reshape(n, stride)


def check(got, x, E, scale=1.0, softcap=30.0):
    e = syn.bf16_to_f32(E).astype(np.float64)
    x64 = x.astype(np.float64)
    z = scale * (x64 @ e.T)
    want = softcap * np.tanh(z / softcap) if softcap > 0 else z
    off = 2.0 ** -24 * (8 + np.sqrt(x.shape[1])) * abs(scale) * (np.abs(x64) @ np.abs(e).T)
    assert (np.abs(got - want) <= off + 4 * 2.0 ** -23 * np.abs(want) + 1e-37).all()


@pytest.mark.parametrize("n,rows,k", [
    (1, 100, 1536), (2, 1, 8), (2, 257, 1536), (3, 4096, 1536), (5, 1000, 64), (8, 333, 40),
    (15, 515, 1528), (16, 64, 256), (17, 129, 1536), (31, 700, 2048), (33, 255, 520),
    (48, 1025, 1536), (63, 130, 4096), (64, 4096, 1536), (65, 300, 1536), (130, 77, 104),
    # many rows: the table's tiles, one and several per block
    (5, 50001, 1536), (16, 66001, 72), (20, 25003, 1528), (40, 17002, 520), (64, 13001, 1536),
    (64, 150007, 64), (130, 13003, 104)])
def test_shapes(g4, n, rows, k):
    print("head rows", n, rows, k, flush=True)
    x, E = case(np.random.default_rng([n, rows, k]), n, rows, k)
    check(run(g4, x, E), x, E)


@pytest.mark.parametrize("n", [2, 20, 70])
@pytest.mark.parametrize("rows,stride", [(301, 333), (50001, 50020)])
def test_scale_without_cap_and_stride(g4, n, rows, stride):
    x, E = case(np.random.default_rng(n), n, rows, 128)
    got = run(g4, x, E, stride=stride, scale=-0.37, softcap=0.0)
    check(got[:, :rows], x, E, scale=-0.37, softcap=0.0)
    assert (got[:, rows:] == 7.0).all()  # the rest of a row stays


def test_one_state_has_the_single_head_s_bits(g4):
    x, E = case(np.random.default_rng(4), 1, 1000, 1536)
    out, xb, eb = g4.Buffer(4000), g4.Buffer.from_array(x), g4.Buffer.from_array(E)
    g4.bf16_head(xb.ptr, eb.ptr, 1000, 1536, out.ptr)
    np.testing.assert_array_equal(run(g4, x, E)[0], out.download(np.float32))


@pytest.mark.parametrize("n,rows", [(4, 500), (64, 500), (4, 50000), (64, 13000)])
def test_a_state_s_logits_do_not_depend_on_the_others(g4, n, rows):
    x, E = case(np.random.default_rng(n), n, rows, 256)
    a = run(g4, x, E)
    y = x.copy()
    y[1:] = np.nan
    y[2] = np.inf
    np.testing.assert_array_equal(run(g4, y, E)[0], a[0])
    b = run(g4, y, E)
    assert np.isnan(b[1]).all() and not np.isnan(b[0]).any()


@pytest.mark.parametrize("rows", [200, 50003])
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_sizes_of_the_states(g4, size, rows):
    x, E = case(np.random.default_rng(8), 6, rows, 264)
    x = (x * np.float32(size)).astype(np.float32)
    check(run(g4, x, E, scale=1.0, softcap=0.0), x, E, softcap=0.0)


def test_a_largest_finite_state(g4):
    x, E = case(np.random.default_rng(9), 3, 64, 256)
    x[1] = 0.0
    x[1, 7] = 3.4e38  # rounds to infinity in BF16
    E[:, 7] = syn.bf16_rne(np.full(64, 1e-30, np.float32))
    check(run(g4, x, E, softcap=0.0), x, E, softcap=0.0)


def test_refuses_short_buffers(g4):
    x, e, o = g4.Buffer(4 * 64 * 4), g4.Buffer(10 * 64 * 2), g4.Buffer(4 * 10 * 4)
    for args in ((x, 5, e, 10, 64, o), (x, 4, e, 11, 64, o), (x, 4, e, 10, 64, o, 11),
                 (x, 4, None, 10, 64, o)):
        with pytest.raises(g4.G4Error):
            g4.bf16_head_rows(*args)


def test_a_table_past_32_bits(g4):
    # 2.3e9 values, the last 40 rows checked
    rows, k, n = 1100003, 2048, 3
    E = g4.Buffer(rows * k * 2)
    g4.fill_random(E, rows * k, g4.RAND_BF16_NORMAL, 11, 0.05)
    x = np.random.default_rng(8).standard_normal((n, k)).astype(np.float32)
    out = g4.Buffer(n * rows * 4)
    g4.bf16_head_rows(g4.Buffer.from_array(x), n, E, rows, k, out, rows, 1.0, 30.0)
    got = out.download(np.float32).reshape(n, rows)[:, -40:]
    check(got, x, E.download(np.uint16, 40 * k, (rows - 40) * k * 2).reshape(40, k))
