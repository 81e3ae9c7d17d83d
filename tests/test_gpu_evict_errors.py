"""An eviction that ends with an error between its launches leaves nothing to the next one."""
import ctypes

import numpy as np
import pytest

import long_cache_reference as ref
from test_gpu_evict import check, weights

pytestmark = pytest.mark.gpu


def leave_an_error():
    """An error of another HIP call, which the library's check after its next launch reports."""
    hip = ctypes.CDLL("libamdhip64.so")
    assert hip.hipSetDevice(9999) != 0


@pytest.mark.parametrize("sets,n", [(1, 20000), (3, 9000), (1, 131072)])
def test_a_call_after_a_failed_one(g4, sets, n):
    rng = np.random.default_rng([sets, n])
    check(g4, weights(rng, sets, n), n // 2, 4, 100)
    for turn in range(3):
        w = np.exp(rng.standard_normal((sets, n))).astype(np.float32)  # other bins than the next call's
        wb, rows = g4.Buffer.from_array(w), g4.Buffer(sets * n * 4)
        leave_an_error()
        with pytest.raises(g4.G4Error) as e:
            g4.cache_evict(wb, sets, n, 3 * n // 4, 0, 0, rows)
        assert e.value.code == g4.G4_E_HIP
        check(g4, weights(rng, sets, n), n // 2, 4, 100, place=turn == 1)


def test_a_replay_after_a_failed_call(g4):
    rng = np.random.default_rng(3)
    n, keep = 30000, 9000
    w, rows, kept = g4.Buffer(n * 4), g4.Buffer(keep * 4), g4.Buffer(n * 4)
    w.upload(weights(rng, 1, n))
    g4.cache_evict(w, 1, n, keep, 4, 64, rows, kept)
    with g4.Encoder() as enc:
        g4.cache_evict(w, 1, n, keep, 4, 64, rows, kept)
    for _ in range(3):
        leave_an_error()
        with pytest.raises(g4.G4Error):
            g4.cache_evict(w, 1, n, n // 2, 0, 0, g4.Buffer(n * 2))
        x = weights(rng, 1, n)
        w.upload(x)
        enc.cmdbuf.submit()
        r, k = ref.evict(x[0], keep, 4, 64)
        np.testing.assert_array_equal(rows.download(np.int32), r)
        np.testing.assert_array_equal(kept.download(np.uint32), k.view(np.uint32))
