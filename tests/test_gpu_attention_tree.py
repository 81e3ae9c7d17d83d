"""g4_attention_tree against its definition in 64 bits.

Tolerance: a score is a sum of at most 512 products of a few units in FP32, so off by
about 2^-24 sqrt(512) * 4 < 6e-6; a weight by the same relative amount (and a few ulps of
its exponential), independently from key to key; the output by no more than that of the
largest value: 2e-5 of max |v|."""
import numpy as np
import pytest

import draft_reference as ref

pytestmark = pytest.mark.gpu


def tree(rng, nodes, kind):
    if kind == "chain":
        return np.arange(-1, nodes - 1, dtype=np.int32)
    if kind == "star":
        return np.full(nodes, -1, np.int32)
    if kind == "binary":
        return np.array([(i - 1) // 2 if i else -1 for i in range(nodes)], np.int32)
    return np.array([rng.integers(max(-1, i - 7), i) if i else -1 for i in range(nodes)], np.int32)


def inputs(rng, nodes, heads, hd, prefix):
    at = 1.5 / hd ** 0.25
    q = (rng.standard_normal((nodes, heads, hd)) * at).astype(np.float32)
    k = (rng.standard_normal((prefix + nodes, hd)) * at).astype(np.float32)
    v = rng.standard_normal((prefix + nodes, hd)).astype(np.float32)
    return q, k, v


def run(g4, q, k, v, prefix, parents, window):
    nodes, heads, hd = q.shape
    b = [g4.Buffer.from_array(a) for a in (q, k, v, np.ascontiguousarray(parents, np.int32))]
    y = g4.Buffer(q.nbytes)
    g4.attention_tree(b[0], b[1], b[2], nodes, heads, hd, prefix, b[3], window > 0, window, y)
    return y.download(np.float32).reshape(q.shape)


def check(g4, rng, nodes, heads, hd, prefix, kind, window):
    print("tree", nodes, heads, hd, prefix, kind, window, flush=True)
    q, k, v = inputs(rng, nodes, heads, hd, prefix)
    parents = tree(rng, nodes, kind)
    got = run(g4, q, k, v, prefix, parents, window)
    want = ref.attention_tree(q, k, v, prefix, parents.tolist(), window)
    assert np.abs(got - want).max() <= 2e-5 * np.abs(v).max()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("nodes,heads,prefix,kind,window", [
    (1, 8, 0, "chain", 0), (1, 1, 1, "chain", 0), (1, 8, 300, "chain", 512),
    (2, 8, 31, "star", 0), (3, 5, 32, "chain", 0), (5, 8, 33, "random", 0),
    (7, 3, 0, "binary", 0), (16, 8, 200, "random", 0), (33, 8, 97, "random", 64),
    (64, 8, 130, "binary", 0), (64, 8, 1000, "random", 512), (65, 2, 63, "random", 3),
    (100, 7, 260, "random", 0), (256, 8, 40, "random", 0), (256, 1, 0, "chain", 100),
    (4, 8, 2500, "random", 512), (12, 6, 3001, "random", 0)])
def test_shapes(g4, hd, nodes, heads, prefix, kind, window):
    check(g4, np.random.default_rng([hd, nodes, heads, prefix]), nodes, heads, hd, prefix, kind,
          window)


@pytest.mark.parametrize("window", [1, 2, 3, 17, 32, 33])
@pytest.mark.parametrize("hd", [256, 512])
def test_windows_that_end_inside_the_tree(g4, hd, window):
    # only the last `window` of a node's own path and prefix
    check(g4, np.random.default_rng([hd, window]), 40, 8, hd, 50, "chain", window)
    check(g4, np.random.default_rng([hd, window]), 40, 8, hd, 50, "random", window)


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_long_prefix(g4, hd):
    check(g4, np.random.default_rng(hd), 9, 8, hd, 20011, "random", 0)


@pytest.mark.parametrize("hd", [256, 512])
def test_unseen_rows_have_no_influence(g4, hd):
    rng = np.random.default_rng(hd + 1)
    nodes, heads, prefix, window = 24, 8, 700, 64
    q, k, v = inputs(rng, nodes, heads, hd, prefix)
    parents = tree(rng, nodes, "random")
    want = run(g4, q, k, v, prefix, parents, window)
    # prefix rows that no node sees (each sees at most window - 1 of them)
    k[:prefix - window + 1], v[:prefix - window + 1] = np.nan, np.inf
    np.testing.assert_array_equal(run(g4, q, k, v, prefix, parents, window), want)
    # and one node's rows: only it and the nodes below see them
    for bad, fill in ((3, np.nan), (3, np.inf), (nodes - 1, np.nan)):
        k2, v2 = k.copy(), v.copy()
        k2[prefix + bad], v2[prefix + bad] = fill, fill
        got = run(g4, q, k2, v2, prefix, parents, window)
        for i in range(nodes):
            if bad not in ref.path_of(parents.tolist(), i):
                np.testing.assert_allclose(got[i], want[i], rtol=0, atol=2e-5 * 5, err_msg=str(i))
                assert np.isfinite(got[i]).all()
            else:
                assert not np.isfinite(got[i]).any()


@pytest.mark.parametrize("hd", [256, 512])
def test_rows_behind_the_last_node_are_not_read(g4, hd):
    rng = np.random.default_rng(hd + 2)
    nodes, heads, prefix = 5, 8, 70
    q, k, v = inputs(rng, nodes, heads, hd, prefix)
    parents = tree(rng, nodes, "random")
    more = np.full((64, hd), np.nan, np.float32)
    a = run(g4, q, k, v, prefix, parents, 0)
    b = run(g4, q, np.concatenate([k, more]), np.concatenate([v, more]), prefix, parents, 0)
    np.testing.assert_array_equal(a, b)


def test_bad_parents_give_nan_rows(g4):
    rng = np.random.default_rng(3)
    q, k, v = inputs(rng, 8, 8, 256, 40)
    parents = np.array([-1, 0, 5, 2, 1, -2, 4, 99], np.int32)  # 2, 5 and 7 are bad; 3 follows 2
    got = run(g4, q, k, v, 40, parents, 0)
    good = np.array([-1, 0, -1, -1, 1, -1, 4, -1])
    want = ref.attention_tree(q, k, v, 40, good.tolist())
    for i in range(8):
        if i in (2, 3, 5, 7):
            assert np.isnan(got[i]).all()
        else:
            assert np.abs(got[i] - want[i]).max() <= 2e-5 * np.abs(v).max()


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("scale", [1e-30, 1e4])
def test_value_ranges(g4, hd, scale):
    # scores in the thousands and values of any size: one key takes all the weight
    rng = np.random.default_rng([hd, 5])
    q, k, v = inputs(rng, 6, 8, hd, 333)
    parents = tree(rng, 6, "random")
    q = (q * 100).astype(np.float32)
    v = (v * np.float32(scale)).astype(np.float32)
    got = run(g4, q, k, v, 333, parents, 0)
    want = ref.attention_tree(q, k, v, 333, parents.tolist())
    # scores of up to about 1000: off by 2^-24 * sqrt(512) * 400 < 6e-4, the weights alike
    assert np.abs(got - want).max() <= 2e-3 * np.abs(v).max()


@pytest.mark.parametrize("hd", [256, 512])
def test_finite_values_beyond_sixteen_bit_ranges(g4, hd):
    # 3.4e38 is finite in FP32 and rounds to infinity in BF16
    rng = np.random.default_rng([hd, 6])
    q, k, v = inputs(rng, 4, 8, hd, 90)
    parents = tree(rng, 4, "chain")
    v[17, 3] = 3.4e38
    k[20, 5] = 3.4e38
    q[:, :, 5] = 1.2e-38
    got = run(g4, q, k, v, 90, parents, 0)
    want = ref.attention_tree(q, k, v, 90, parents.tolist())
    scale = np.abs(want).max(axis=(0, 1))
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= 2e-5 * np.maximum(scale, np.abs(v[np.abs(v) < 1e30]).max())).all()


def test_equal_to_plain_attention_along_a_chain(g4):
    # a chain is causal attention: g4_attention's rows, to FP32 rounding
    rng = np.random.default_rng(11)
    q, k, v = inputs(rng, 6, 8, 256, 80)
    got = run(g4, q, k, v, 80, tree(rng, 6, "chain"), 0)
    b = [g4.Buffer.from_array(a) for a in (q, k, v)]
    y = g4.Buffer(q.nbytes)
    g4.attention(b[0], b[1], b[2], 6, 8, 256, 86, 80, False, 0, y)
    assert np.abs(got - y.download(np.float32).reshape(q.shape)).max() <= 2e-5 * np.abs(v).max()


def test_refuses_short_buffers(g4):
    x = g4.Buffer(4 * 8 * 256 * 4)
    p = g4.Buffer(16)
    kv = g4.Buffer(20 * 256 * 4)
    for args in ((x, kv, kv, 4, 8, 256, 17, p, False, 0, x),     # 21 rows of k
                 (x, kv, kv, 5, 8, 256, 10, p, False, 0, x),     # 5 nodes of q
                 (kv, kv, kv, 2, 8, 256, 10, None, False, 0, x)):
        with pytest.raises(g4.G4Error):
            g4.attention_tree(*args)


@pytest.mark.parametrize("nodes,prefix", [(16, 9000), (7, 16383), (20, 9000)])
def test_key_splits_by_the_row_blocks(g4, nodes, prefix):
    # 8, 4 and 10 blocks of 16 rows, whose key splits are no multiples of 8
    check(g4, np.random.default_rng([nodes, prefix]), nodes, 8, 256, prefix, "random", 0)


@pytest.mark.parametrize("nodes,prefix", [(20, 9000), (13, 8500), (48, 8300)])
def test_key_splits_of_a_cache_past_the_l2s(g4, nodes, prefix):
    check(g4, np.random.default_rng([nodes, prefix, 5]), nodes, 8, 512, prefix, "random", 0)


def test_a_cache_past_32_bits(g4):
    # a window at the end of 4.3 million rows of 512: offsets past 2^31 values
    hd, prefix, nodes, window, near = 512, 4300000, 6, 300, 400
    rng = np.random.default_rng(43)
    q, k, v = inputs(rng, nodes, 4, hd, near)
    parents = tree(rng, nodes, "random")
    kb, vb = (g4.Buffer((prefix + nodes) * hd * 4) for _ in range(2))
    kb.upload(k, (prefix - near) * hd * 4)
    vb.upload(v, (prefix - near) * hd * 4)
    qb, pb, y = g4.Buffer.from_array(q), g4.Buffer.from_array(parents), g4.Buffer(q.nbytes)
    g4.attention_tree(qb, kb, vb, nodes, 4, hd, prefix, pb, True, window, y)
    want = ref.attention_tree(q, k, v, near, parents.tolist(), window)
    assert np.abs(y.download(np.float32).reshape(q.shape) - want).max() <= 2e-5 * np.abs(v).max()
