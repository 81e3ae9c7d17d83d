"""Calls of the drafted-token operators that one launch cannot hold: a grid has less than 2^32
threads per dimension, so these take several, and a row of the second one has its own result."""
import numpy as np
import pytest

import draft_reference as ref
import synthetic as syn

pytestmark = pytest.mark.gpu


def test_sample_rows_of_more_than_one_grid(g4):
    # 2^23 blocks of 512 threads are 2^32
    rows, vocab = 2 ** 23 + 3, 4
    rng = np.random.default_rng(1)
    kinds = rng.standard_normal((64, vocab)).astype(np.float32)
    us = rng.random(64).astype(np.float32)
    at = np.arange(rows) % 64
    x, u = g4.Buffer.from_array(kinds[at]), g4.Buffer.from_array(us[at])
    tok, pr = g4.Buffer.from_array(np.full(rows, -7, np.int32)), g4.Buffer(rows * 4)
    for cuts in (dict(temperature=0.7), dict(top_k=3, top_p=0.8)):
        g4.sample(x, rows, vocab, u, tok, pr, **cuts)
        want = [ref.sample(kinds[i], us[i], **cuts) for i in range(64)]
        np.testing.assert_array_equal(tok.download(np.int32), np.array([w[0] for w in want], np.int32)[at])
        # FP32's half step, and 64-bit sums of four exponentials: far below 1e-6
        np.testing.assert_allclose(pr.download(np.float32), np.array([w[1] for w in want])[at], rtol=1e-6)


@pytest.mark.parametrize("place", [False, True])
def test_cache_rows_of_more_than_one_grid(g4, place):
    # 2^24 blocks of 256 threads are 2^32; a block takes 16 rows of one value
    n, at, cap = 2 ** 28 + 37, 5, 1009
    a = np.random.default_rng(2).standard_normal(cap).astype(np.float32)
    rows = np.arange(n, dtype=np.int32) % cap
    idx, dst = g4.Buffer.from_array(rows), g4.Buffer((at + n + 3) * 4)
    src = dst if place else g4.Buffer.from_array(a)
    if place:  # the source's rows lie where the first ones go
        dst.upload(a)
    g4.CachePlanes([dst], [src], [1]).rows(idx, n, at, cap)
    got = dst.download(np.float32)
    np.testing.assert_array_equal(got[:at], a[:at] if place else 0)
    np.testing.assert_array_equal(got[at:at + n], a[rows])
    assert not got[at + n:].any()


def test_head_of_one_state_of_more_than_one_grid(g4):
    # 2^24 blocks of 256 threads are 2^32; a block takes 32 rows of the table
    rows, k = 2 ** 29 + 45, 8
    E, out = g4.Buffer(rows * k * 2), g4.Buffer(rows * 4)
    g4.fill_random(E, rows * k, g4.RAND_BF16_NORMAL, 11, 0.5)
    x = np.random.default_rng(3).standard_normal((1, k)).astype(np.float32)
    xb = g4.Buffer.from_array(x)
    g4.bf16_head_rows(xb, 1, E, rows, k, out, rows, 1.0, 30.0)
    part = g4.Buffer(4 * 500)
    for at in (0, 2 ** 28 - 250, rows - 500):  # the last 500 lie around 2^29
        # the bits of a call of these rows alone, and 30 tanh(x . E / 30): a sum of 8 exact
        # products' FP32 roundings and tanh's few ulps
        g4.bf16_head(xb.ptr, E.at(at * k * 2), 500, k, part.ptr)
        got = out.download(np.float32, 500, at * 4)
        np.testing.assert_array_equal(got, part.download(np.float32))
        e = syn.bf16_to_f32(E.download(np.uint16, 500 * k, at * k * 2).reshape(500, k)).astype(np.float64)
        z = e @ x[0].astype(np.float64)
        off = 8 * 2.0 ** -24 * (np.abs(e) @ np.abs(x[0]).astype(np.float64)) + 2.0 ** -21 * np.abs(z)
        assert (np.abs(got - 30 * np.tanh(z / 30)) <= off).all()
