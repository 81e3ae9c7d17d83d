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
