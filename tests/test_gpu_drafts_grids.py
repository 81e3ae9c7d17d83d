"""Calls of the drafted-token operators that one launch cannot hold: a grid has less than 2^32
threads per dimension, so these take several, and a row of the second one has its own result."""
import numpy as np
import pytest

import draft_reference as ref

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
