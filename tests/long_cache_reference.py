"""The operators of long caches from their definitions, in 64 bits, for the tests."""
import numpy as np


def bf16(x):
    """FP32 to the nearest BF16 bits, halves to even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def wide(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def pack(x):
    """FP32 rows [n, hd] -> codes uint32 [n, hd / 8], scales BF16 bits [n, hd / 32]."""
    n, hd = x.shape
    g = x.reshape(n, hd // 32, 32)
    finite = np.isfinite(g).all(2)
    safe = np.where(finite[:, :, None], g, 0)
    s = bf16(np.abs(safe).max(2) / np.float32(7))
    s[s == 0] = 0x3f80
    q = np.clip(np.rint(safe.astype(np.float64) / wide(s).astype(np.float64)[:, :, None]), -7, 7)
    s[~finite] = 0x7fc0
    w = (q.astype(np.int64) + 8).astype(np.uint32).reshape(n, hd // 8, 8)
    codes = np.zeros((n, hd // 8), np.uint32)
    for i in range(8):
        codes |= w[:, :, i] << np.uint32(4 * i)
    return codes, s


def unpack(codes, scales):
    n, words = codes.shape
    q = np.stack([(codes >> np.uint32(4 * i)) & 15 for i in range(8)], 2).astype(np.float64) - 8
    s = wide(scales).astype(np.float64)
    return (q.reshape(n, -1, 32) * s[:, :, None]).reshape(n, words * 8)


def weights(q, k, keylen, qpos0, window=0):
    """q [rows, heads, hd], k [>= keylen, hd] -> the softmax weights [rows, heads, keylen]."""
    q, k = q.astype(np.float64), k[:keylen].astype(np.float64)
    out = np.zeros(q.shape[:2] + (keylen,))
    for r in range(len(q)):
        pos = qpos0 + r
        lo = max(0, pos - window + 1) if window else 0
        s = q[r] @ k[lo:pos + 1].T
        p = np.exp(s - s.max(1, keepdims=True))
        out[r, :, lo:pos + 1] = p / p.sum(1, keepdims=True)
    return out


def evict(w, keep, first, recent):
    """(rows that stay, their weights with zeros behind) of one cache."""
    n = len(w)
    mid = np.arange(first, n - recent)
    order = np.where(np.isnan(w[mid]), -np.inf, w[mid].astype(np.float64))
    # NaN behind every number, minus infinity too; then the lowest index
    best = mid[np.lexsort((mid, -order, np.isnan(w[mid])))][:keep - first - recent]
    rows = np.sort(np.concatenate([np.arange(first), best, np.arange(n - recent, n)])).astype(np.int32)
    return rows, np.concatenate([w[rows], np.zeros(n - keep, w.dtype)])
