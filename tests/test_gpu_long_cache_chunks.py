"""Keys' weights of more scores than are kept at once: how many chunks of query rows a call takes, and
that each adds to the keys that its rows see and to no others.

Tolerance as in test_gpu_attention_weights.py, 2e-5 of a key's weight."""
import ctypes

import numpy as np
import pytest

import long_cache_reference as ref

pytestmark = pytest.mark.gpu
TOL, HEADS = 2e-5, 8


def launches(enc):
    """Nodes of a recording: a cmdbuf starts with its HIP graph."""
    hip = ctypes.CDLL("libamdhip64.so")
    graph = ctypes.cast(enc.cmdbuf.ptr, ctypes.POINTER(ctypes.c_void_p))[0]
    n = ctypes.c_size_t()
    assert hip.hipGraphGetNodes(ctypes.c_void_p(graph), None, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("op", ["attention", "weights"])
@pytest.mark.parametrize("qrows,keys,window,chunks", [
    # r rows of 8 heads see at most window + r keys of which 2^26 scores are kept: 2652 rows of a window
    # of 512, whatever the prompt's length; 419 rows of 20000 keys, of which 2019 lie behind the last row
    (16384, 16384, 512, 7), (16384, 40000, 512, 7), (3000, 3000, 512, 2), (400, 20000, 0, 1), (2000, 2000, 0, 1),
    (900, 20000, 0, 3)])
def test_chunks(g4, op, qrows, keys, window, chunks):
    hd = 64
    q, y = (g4.Buffer(qrows * HEADS * hd * 4) for _ in range(2))
    c, k, w = g4.Kv4Cache(keys, hd), g4.Buffer(keys * hd * 4), g4.Buffer(keys * 4)
    at = keys - qrows if keys < 40000 else 100

    def call():
        if op == "attention":
            c.attention(q, qrows, HEADS, keys, at, window > 0, window, y, w)
        else:
            g4.attention_weights(q, k, qrows, HEADS, hd, keys, at, window > 0, window, w)

    call()
    with g4.Encoder() as enc:
        call()
    # scores, at most, the join of the splits, the sums of each 32 rows and the sums of these
    assert launches(enc) <= 4 * chunks


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("at,window", [(0, 100), (70, 100), (70, 0)])
def test_sums_of_several_chunks(g4, place, at, window):
    # q and k of zeros: a row weighs the keys that it sees alike, so the sums are known for any size
    qrows, keys, hd = 6000, 6200, 64
    q, y = (g4.Buffer(qrows * HEADS * hd * 4) for _ in range(2))
    c, k = g4.Kv4Cache(keys, hd), g4.Buffer(keys * hd * 4)
    rng = np.random.default_rng(3)
    before = rng.random(keys).astype(np.float32)
    pos = at + np.arange(qrows)
    first = np.maximum(0, pos - window + 1) if window else np.zeros(qrows, int)
    want = np.zeros(keys + 1)
    np.add.at(want, first, HEADS / (pos + 1 - first))
    np.add.at(want, pos + 1, -HEADS / (pos + 1 - first))
    want = before + np.cumsum(want)[:keys]
    for op in range(2):
        b = g4.Buffer.from_array(before)
        w = b if place else g4.Buffer.from_array(np.full(keys, np.nan, np.float32))
        if op == 0:
            c.attention(q, qrows, HEADS, keys, at, window > 0, window, y, w, b)
        else:
            g4.attention_weights(q, k, qrows, HEADS, hd, keys, at, window > 0, window, w, b)
        got = w.download(np.float32)
        assert (np.abs(got - want) <= TOL * want).all()
        np.testing.assert_array_equal(got[at + qrows:], before[at + qrows:])
