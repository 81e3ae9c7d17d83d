"""Refusals of the operators of long caches: arguments are checked before the device is needed,
so these run without a GPU."""
import ctypes

import pytest

import g4hip


def refused(rc, *words):
    assert rc == g4hip.G4_E_ARG
    msg = g4hip.lib().g4_last_error().decode()
    for w in words:
        assert w in msg, msg


def cache(rows=100, hd=256, k=16, v=16, ks=16, vs=16):
    return ctypes.byref(g4hip.Kv4(k, v, ks, vs, rows, hd))


@pytest.mark.parametrize("c,n,at", [
    (cache(hd=96), 1, 0), (cache(hd=0), 1, 0), (cache(hd=1024), 1, 0), (cache(rows=-1), 0, 0),
    (cache(), -1, 0), (cache(), 1, -1), (cache(), 101, 0), (cache(), 1, 100), (cache(), 50, 51),
    (cache(), 0x7fffffff, 1), (cache(), 1, 0x7fffffff), (cache(k=8), 1, 0), (cache(v=20), 1, 0),
    (cache(ks=18), 1, 0), (cache(vs=24), 1, 0), (None, 1, 0)])
def test_kv4_rows(c, n, at):
    refused(g4hip.lib().g4_kv4_append(c, 16, 16, n, at), "g4_kv4_append")
    refused(g4hip.lib().g4_kv4_read(c, at, n, 16, 16), "g4_kv4_read")


@pytest.mark.parametrize("k,v", [(8, 16), (16, 4)])
def test_unaligned_rows(k, v):
    refused(g4hip.lib().g4_kv4_append(cache(), k, v, 1, 0), "aligned")
    refused(g4hip.lib().g4_kv4_read(cache(), 0, 1, k, v), "aligned")


MASKS = [(-1, 8, 50, 0, 0, 0), ((1 << 20) + 1, 8, 50, 0, 0, 0), (4, 0, 50, 0, 0, 0), (4, 9, 50, 0, 0, 0),
         (4, 8, -1, 0, 0, 0), (4, 8, 50, -1, 0, 0), (4, 8, 50, 47, 0, 0), (51, 8, 50, 0, 0, 0),
         (4, 8, 50, 0x7fffffff, 0, 0), (4, 8, 50, 10, 1, 0), (4, 8, 50, 10, 1, -3)]


@pytest.mark.parametrize("qrows,heads,keylen,qpos0,sliding,window", MASKS)
def test_attention_masks(qrows, heads, keylen, qpos0, sliding, window):
    L = g4hip.lib()
    refused(L.g4_attention_kv4(16, cache(), qrows, heads, keylen, qpos0, sliding, window, 16, None, 16),
            "g4_attention_kv4")
    refused(L.g4_attention_weights(16, 16, qrows, heads, 256, keylen, qpos0, sliding, window, None, 16),
            "g4_attention_weights")


def test_attention_kv4_operands():
    L = g4hip.lib()
    call = lambda q=16, c=cache(), keys=50, y=16, b=None, w=None: L.g4_attention_kv4(  # noqa: E731
        q, c, 2, 8, keys, 40, 0, 0, y, b, w)
    refused(call(q=8), "aligned")
    refused(call(y=24), "aligned")
    refused(call(keys=101), "cache of 100")
    refused(call(c=cache(hd=80)), "head_dim")
    refused(call(c=cache(k=24)), "aligned")
    refused(call(c=None), "null cache")
    refused(call(b=16), "before without weights")
    refused(call(b=4096, w=4096 + 196), "overlaps")
    refused(call(b=4096 + 4, w=4096), "overlaps")


def test_attention_weights_operands():
    L = g4hip.lib()
    call = lambda q=16, k=16, hd=256, keys=50, b=None: L.g4_attention_weights(  # noqa: E731
        q, k, 2, 8, hd, keys, 40, 0, 0, b, 4096)
    for hd in (0, 32, 96, 384, 1024, -64):
        refused(call(hd=hd), "head_dim")
    refused(call(q=8), "aligned")
    refused(call(k=20), "aligned")
    refused(call(keys=(1 << 28) + 1), "keylen")
    refused(call(b=4096 - 196), "overlaps")


@pytest.mark.parametrize("stride,sets,n,keep,first,recent", [
    (10, -1, 10, 5, 0, 0), (10, 257, 10, 5, 0, 0), (10, 1, -1, 0, 0, 0), (1 << 25, 1, (1 << 24) + 1, 5, 0, 0),
    (10, 1, 10, -1, 0, 0), (10, 1, 10, 11, 0, 0), (10, 1, 10, 5, -1, 0), (10, 1, 10, 5, 0, -1),
    (10, 1, 10, 5, 6, 0), (10, 1, 10, 5, 0, 6), (10, 1, 10, 5, 3, 3), (10, 1, 10, 5, 0x7fffffff, 0x7fffffff),
    (9, 1, 10, 5, 0, 0), ((1 << 52) + 1, 1, 10, 5, 0, 0), ((1 << 64) - 1, 2, 10, 5, 0, 0)])
def test_evict(stride, sets, n, keep, first, recent):
    refused(g4hip.lib().g4_cache_evict(4096, stride, sets, n, keep, first, recent, 16, None), "g4_cache_evict")


@pytest.mark.parametrize("kept", [4096 + 4, 4096 - 4, 4096 + 4 * 29, 4096 - 4 * 29])
def test_evict_overlap(kept):
    # 2 sets of 10 at a stride of 20: 30 values
    refused(g4hip.lib().g4_cache_evict(4096, 20, 2, 10, 5, 0, 0, 16, kept), "overlaps")


def test_cache_of_other_buffers():
    with pytest.raises(ValueError):
        g4hip.Kv4Cache(8, 64, [16, 16])


@pytest.mark.parametrize("y,w", [(65536, 1 << 20), (65536 + 2 * 8 * 256 * 4 - 16, 1 << 20), (1 << 20, 65536 + 12),
                                 (1 << 20, (1 << 20) + 2 * 8 * 256 * 4 - 4), (1 << 20, (1 << 20) - 196)])
def test_attention_kv4_overlaps(y, w):
    # 2 rows of 8 * 256 at q and y, 50 weights
    refused(g4hip.lib().g4_attention_kv4(65536, cache(), 2, 8, 50, 40, 0, 0, y, None, w), "overlaps")
    refused(g4hip.lib().g4_attention_kv4(65536, cache(), 2, 8, 50, 40, 0, 0, y, y + 16, w), "overlaps")


def test_attention_kv4_overlaps_its_cache():
    # 50 rows of 256: 6400 bytes of codes, 800 of scales
    planes = [1 << 20, 2 << 20, 3 << 20, 4 << 20]
    for p, n in zip(planes, (6400, 6400, 800, 800)):
        for x in (p, p + n - 16):
            for y, w in ((x, 8 << 20), (8 << 20, x)):
                refused(g4hip.lib().g4_attention_kv4(65536, cache(100, 256, *planes), 2, 8, 50, 40, 0, 0, y, None, w),
                        "overlaps")


@pytest.mark.parametrize("w", [65536, 65536 - 196, 65536 + 2 * 8 * 256 * 4 - 4, (1 << 20) - 4, (1 << 20) + 50 * 1024 - 4])
def test_attention_weights_overlaps(w):
    refused(g4hip.lib().g4_attention_weights(65536, 1 << 20, 2, 8, 256, 50, 40, 0, 0, None, w), "overlaps")


@pytest.mark.parametrize("rows,kept", [(4096, None), (4096 + 116, None), (4096 - 36, 1 << 20), ((1 << 20) + 8, 1 << 20)])
def test_evict_rows_overlap(rows, kept):
    # 2 sets of 10 at a stride of 20: 30 weights; 2 * 5 rows
    refused(g4hip.lib().g4_cache_evict(4096, 20, 2, 10, 5, 0, 0, rows, kept), "overlaps")


def test_kv4_rows_overlap_their_cache():
    # rows 3 .. 6 of 256: 512 bytes of codes, 64 of scales
    planes = [1 << 20, 2 << 20, 3 << 20, 4 << 20]
    L = g4hip.lib()
    for p, row in zip(planes, (128, 128, 16, 16)):
        for x in (p + 3 * row, p + 7 * row - 16, p + 3 * row - 4096 + 16):
            for k, v in ((x, 16 << 20), (16 << 20, x)):
                refused(L.g4_kv4_append(cache(100, 256, *planes), k, v, 4, 3), "overlaps")
                refused(L.g4_kv4_read(cache(100, 256, *planes), 3, 4, k, v), "overlaps")
    refused(L.g4_kv4_read(cache(100, 256, *planes), 3, 4, 16 << 20, (16 << 20) + 4080), "overlaps")
