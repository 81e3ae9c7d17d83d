"""g4_sample where the cuts lie among more tokens than are listed: flat rows, high temperatures
and many equal logits, against the definition in 64 bits."""
import numpy as np
import pytest

from test_gpu_sample import check

pytestmark = pytest.mark.gpu

FLAT = [dict(temperature=1.5, top_p=0.75), dict(temperature=1.5, top_k=131072),
        dict(temperature=1.5, top_k=131072, top_p=0.9), dict(temperature=2.5, top_p=0.6, min_p=0.05),
        dict(temperature=4.0, top_k=200000, top_p=0.5), dict(temperature=30.0, top_k=1000),
        dict(temperature=30.0, top_k=99999, top_p=0.999), dict(temperature=4.0, top_k=99999, min_p=0.3),
        dict(temperature=1e30, top_p=0.41)]


@pytest.mark.parametrize("rows,vocab", [(2, 8191), (3, 30011), (2, 131073), (3, 262144), (20, 262144),
                                        (3, 300001)])
def test_flat_rows(g4, rows, vocab):
    rng = np.random.default_rng([rows, vocab])
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    x[1] *= np.float32(0.1)
    x[1, ::5] = -np.inf
    x[1, 3::7] = np.nan
    x[rows - 1] = np.round(x[rows - 1] * 16) / 16  # equal logits among all of them
    for cuts in FLAT:
        check(g4, x, rng.random(rows), **cuts)


@pytest.mark.parametrize("vocab", [8192, 50000, 262144])
def test_rows_of_equal_logits(g4, vocab):
    rng = np.random.default_rng(vocab)
    x = np.zeros((3, vocab), np.float32)
    x[1, 1::2] = -np.inf
    x[2, vocab // 3:] = 0.125
    for cuts in (dict(top_k=1000), dict(top_p=0.3), dict(top_k=vocab // 2, top_p=0.5), dict(min_p=0.9),
                 dict(top_k=vocab // 2 + 1, min_p=0.5)):
        check(g4, x, rng.random(3), **cuts)
