"""Drafted tokens through one layer from their raw q and k: the norm and RoPE of a tree's nodes, one
call per depth, their rows appended to the caches, and the attention over them; and recordings of
cache rows that overlap their source."""
import math

import numpy as np
import pytest

import draft_reference as ref
import layer_oracle as lo

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,prop,theta,window", [(64, 1.0, 1e4, 24), (256, 1.0, 1e4, 0), (512, 0.25, 1e6, 0)])
def test_norm_and_rope_of_a_tree_by_depth(g4, hd, prop, theta, window):
    heads, prefix, nodes = 8, 61, 40
    rng = np.random.default_rng(hd)
    # nodes in the order of their depth, each below one of the level before
    parents, level, depth = [-1, -1, -1], [0, 1, 2], [0, 0, 0]
    while len(parents) < nodes:
        here = list(range(len(parents), min(nodes, len(parents) + int(rng.integers(2, 9)))))
        parents += [int(rng.choice(level)) for _ in here]
        depth += [depth[level[0]] + 1] * len(here)
        level = here
    x = {n: (2 * rng.standard_normal((prefix + nodes, h, hd))).astype(np.float32) for n, h in (("q", heads), ("k", 1))}
    v = rng.standard_normal((prefix + nodes, hd)).astype(np.float32)
    w = {n: (rng.uniform(0.5, 1.5, hd) / hd ** 0.25).astype(np.float32) for n in "qk"}
    angles = int(math.floor(prop * hd / 2))
    wb = {n: g4.Buffer.from_array(w[n]) for n in "qk"}
    kc, vc = g4.Buffer(x["k"].nbytes), g4.Buffer.from_array(v)
    q = g4.Buffer(nodes * heads * hd * 4)
    raw = {n: g4.Buffer.from_array(x[n]) for n in "qk"}
    # the prefix as a prefill leaves it, then the nodes of a depth as one row
    g4.norm_rope(raw["k"], prefix, 1, hd, 0, wb["k"], angles, theta, kc)
    for d in range(max(depth) + 1):
        at, n = depth.index(d), depth.count(d)
        qrow, krow = heads * hd * 4, hd * 4
        g4.norm_rope(raw["q"].at((prefix + at) * qrow), 1, n * heads, hd, prefix + d, wb["q"], angles, theta,
                     q.at(at * qrow))
        g4.norm_rope(raw["k"].at((prefix + at) * krow), 1, n, hd, prefix + d, wb["k"], angles, theta,
                     kc.at((prefix + at) * krow))
    y, pb = g4.Buffer(q.nbytes), g4.Buffer.from_array(np.array(parents, np.int32))
    g4.attention_tree(q, kc, vc, nodes, heads, hd, prefix, pb, window > 0, window, y)
    got = {"q": q.download(np.float32).reshape(nodes, heads, hd),
           "k": kc.download(np.float32).reshape(prefix + nodes, 1, hd)[prefix:]}
    for n in "qk":
        for i in range(nodes):
            pos = prefix + depth[i]
            want = lo.norm_rope(x[n][prefix + i].reshape(1, -1), 1, x[n].shape[1], hd, pos, w[n], angles, theta)
            # a theta of one ulp more or less (pos * 2^-23), as for a row of its own
            atol = 2e-6 + 2 * (pos + 1) * 1.2e-7 * float(np.abs(want).max())
            np.testing.assert_allclose(got[n][i].reshape(1, -1), want, rtol=1e-5, atol=atol)
    want = ref.attention_tree(got["q"], kc.download(np.float32).reshape(-1, hd), v, prefix, parents, window)
    # |q| |k| <= 1.5^2 sqrt(hd) < 51: a score is off by less than 2^-24 sqrt(512) * 51 < 7e-5, a
    # weight by the same relative amount, the output by no more than twice that of the largest value
    assert np.abs(y.download(np.float32).reshape(want.shape) - want).max() <= 1.4e-4 * np.abs(v).max()


@pytest.mark.parametrize("n,shift", [(5, 4), (64, 260), (100, 256)])
def test_recorded_rows_that_overlap_their_source(g4, n, shift):
    # planes that overlap by part of a row move through scratch whatever their number of rows,
    # so a recording follows one such call
    w, cap, at = 256, 150, 20
    rng = np.random.default_rng([n, shift])
    a = rng.standard_normal(cap * w + shift).astype(np.float32)
    b, idx = g4.Buffer.from_array(a), g4.Buffer.from_array(rng.integers(0, cap, n).astype(np.int32))
    planes = g4.CachePlanes([b.at(4 * shift)], [b], [w])
    planes.rows(idx, n, at, cap)
    with g4.Encoder() as enc:
        planes.rows(idx, n, at, cap)
    for _ in range(3):
        a = rng.standard_normal(cap * w + shift).astype(np.float32)
        rows = rng.integers(0, cap, n).astype(np.int32)
        b.upload(a)
        idx.upload(rows)
        enc.cmdbuf.submit()
        want = a.copy()
        want[shift + at * w:shift + (at + n) * w] = a[:cap * w].reshape(cap, w)[rows].ravel()
        np.testing.assert_array_equal(b.download(np.float32), want)
