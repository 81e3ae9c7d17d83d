"""g4_attention_kv4 where a few values of the cache are far larger or smaller than the others: what
one group of a row holds has no part in the outputs' other dims.

Tolerance as in test_gpu_kv4.py, 2e-5, here of the largest |v| that the row sees in each 32 dims by
themselves: an output's error is that of the weights (1e-5 relative, or 2^-39 of the row's largest for
at most 400 keys, 8e-10), times these values."""
import numpy as np
import pytest

import long_cache_reference as ref
from test_gpu_kv4 import TOL, attend, cache_of, inputs

pytestmark = pytest.mark.gpu


def check_groups(g4, q, pk, pv, keys, qpos0, window):
    hd = q.shape[2]
    y, _ = attend(g4, cache_of(g4, pk, pv, hd), q, keys, qpos0, window)
    kk, vv = ref.unpack(*pk), ref.unpack(*pv)
    p = ref.weights(q, kk, keys, qpos0, window)
    for r in range(len(q)):
        end = qpos0 + r + 1
        seen = np.abs(vv[max(0, end - window) if window else 0:end]).reshape(-1, hd // 32, 32).max((0, 2))
        err = np.abs(y[r] - p[r] @ vv).reshape(-1, hd // 32, 32).max((0, 2))
        assert (err <= TOL * seen).all(), (r, err / seen)


# splits joined by a block per row, and by a thread per 16 bytes (64 rows and more, up to 16 splits)
@pytest.mark.parametrize("hd,qrows,keys", [(64, 3, 2000), (512, 3, 2000), (512, 64, 2000), (256, 40, 2000), (512, 1, 300)])
@pytest.mark.parametrize("exp", [118, 123])
def test_all_values_near_the_largest_number(g4, hd, qrows, keys, exp):
    # of one sign, so that the outputs are as large; rows of zeros weigh all keys alike
    rng = np.random.default_rng([hd, exp])
    q, k, v = inputs(rng, qrows, 8, hd, keys)
    q[::2] = 0
    v = (np.clip(np.abs(v), 0, 4) * np.float32(2.0 ** exp)).astype(np.float32)
    check_groups(g4, q, ref.pack(k), ref.pack(v), keys, keys - qrows, 0)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("qrows", [1, 2, 12, 45])
@pytest.mark.parametrize("b", [12, 28, 40, 50, 90, -40, -90])
def test_one_group_of_one_row(g4, hd, qrows, b):
    rng = np.random.default_rng([hd, qrows, b + 100])
    keys = 320
    q, k, v = inputs(rng, qrows, 8, hd, keys)
    group = rng.integers(0, hd // 32)
    v[77, 32 * group:32 * group + 32] *= np.float32(2.0 ** b)
    check_groups(g4, q, ref.pack(k), ref.pack(v), keys, keys - qrows, 0)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("qrows", [1, 12, 45])
@pytest.mark.parametrize("window", [0, 130])
def test_groups_of_any_size(g4, hd, qrows, window):
    # every group of every row 2^-45 to 2^45 times the usual
    rng = np.random.default_rng([hd, qrows, window])
    keys = 333
    q, k, v = inputs(rng, qrows, 8, hd, keys)
    e = np.repeat(rng.integers(-45, 46, (keys, hd // 32)), 32, axis=1)
    check_groups(g4, q, ref.pack(k), ref.pack((v * np.exp2(e)).astype(np.float32)), keys, keys - qrows, window)


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("qrows", [1, 40])
def test_the_largest_values_beside_small_ones(g4, hd, qrows):
    # 2^122 and 2^-70 in different dims, the large ones in the first, a middle and the last row
    rng = np.random.default_rng([hd, qrows, 5])
    keys = 300
    q, k, v = inputs(rng, qrows, 8, hd, keys)
    v[:, 32:64] *= np.float32(2.0 ** -70)
    v[0, :32] *= np.float32(2.0 ** 122)
    v[150, :32] *= np.float32(2.0 ** 115)
    v[keys - 1, :32] *= np.float32(2.0 ** 122)
    check_groups(g4, q, ref.pack(k), ref.pack(v), keys, keys - qrows, 0)


@pytest.mark.parametrize("hd", [64, 512])
@pytest.mark.parametrize("exp", [-124, -118])
def test_all_values_near_the_smallest_number(g4, hd, exp):
    rng = np.random.default_rng([hd, exp + 200])
    q, k, v = inputs(rng, 3, 8, hd, 2000)
    check_groups(g4, q, ref.pack(k), ref.pack((v * np.float32(2.0 ** exp)).astype(np.float32)), 2000, 1997, 0)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("qrows", [1, 12, 40])
def test_the_largest_q_and_small_k(g4, hd, qrows):
    # scores of up to 2^27, 2^25 and more apart: each row's weight is on one key
    keys = 300
    rng = np.random.default_rng([hd, qrows, 6])
    q, k, v = inputs(rng, qrows, 8, hd, keys)
    q[:], k[:] = 0, 0
    q[:, :, 0] = np.float32(2.0 ** 124)
    k[:, 0], k[:, 1] = np.float32(2.0 ** -100), np.float32(7 * 2.0 ** -100)  # (the second one for the scale)
    k[37, 0] = np.float32(5 * 2.0 ** -100)
    k[keys - 1, 0] = np.float32(7 * 2.0 ** -100)
    check_groups(g4, q, ref.pack(k), ref.pack(v), keys, keys - qrows, 0)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("qrows", [1, 12, 45])
@pytest.mark.parametrize("what", ["zeros", "large", "any"])
def test_small_k_beside_large_ones(g4, hd, qrows, what):
    # the scores come from one group of k, 2^-40 times the usual; the others hold zeros, whose scale is 1,
    # values 2^30 times the usual that q does not look at, or ones of any size in each key
    keys = 320
    rng = np.random.default_rng([hd, qrows, len(what)])
    q, k, v = inputs(rng, qrows, 8, hd, keys)
    group = rng.integers(0, hd // 32)
    mine = np.arange(hd) // 32 == group
    q[:, :, ~mine] = 0
    q[:, :, mine] *= np.float32(2.0 ** 40)
    k[:, mine] *= np.float32(2.0 ** -40)
    if what == "any":
        k[:, ~mine] *= np.repeat(np.exp2(rng.integers(-60, 61, (keys, hd // 32 - 1))), 32, axis=1).astype(np.float32)
    else:
        k[:, ~mine] *= np.float32(0 if what == "zeros" else 2.0 ** 30)
    check_groups(g4, q, ref.pack(k), ref.pack(v), keys, keys - qrows, 0)
