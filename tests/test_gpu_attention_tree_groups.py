"""g4_attention_tree at head dims 64 and 128, whose blocks share their key tiles among 4 and 2
groups of waves: tile counts that leave groups without a last tile, rows that are not finite
where a row does not see them, windows inside the tree, and the join of the groups.

Tolerances as in test_gpu_attention_tree.py: 2e-5 of the largest value."""
import numpy as np
import pytest

import draft_reference as ref
import test_gpu_attention_tree as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes,heads,prefix,kind,window", [
    (1, 8, 0, "chain", 0), (17, 8, 0, "random", 0), (40, 8, 16, "binary", 0), (3, 8, 15, "chain", 0),
    (16, 8, 64, "random", 5), (33, 7, 80, "random", 0), (256, 8, 5, "random", 0), (256, 8, 300, "chain", 200),
    (200, 8, 1111, "random", 0), (64, 3, 2050, "random", 512)])
def test_tiles_that_the_groups_do_not_share_evenly(g4, hd, nodes, heads, prefix, kind, window):
    base.check(g4, np.random.default_rng([hd, nodes, prefix]), nodes, heads, hd, prefix, kind, window)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 3, 17, 32, 33])
def test_windows_that_end_inside_the_tree(g4, hd, window):
    base.test_windows_that_end_inside_the_tree(g4, hd, window)


@pytest.mark.parametrize("hd", [64, 128])
def test_unseen_rows_have_no_influence(g4, hd):
    base.test_unseen_rows_have_no_influence(g4, hd)


@pytest.mark.parametrize("hd", [64, 128])
def test_rows_behind_the_last_node_are_not_read(g4, hd):
    base.test_rows_behind_the_last_node_are_not_read(g4, hd)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes,prefix,window", [(24, 0, 0), (24, 7, 0), (40, 33, 20), (100, 50, 0), (250, 9, 0)])
def test_every_node_that_is_not_finite(g4, hd, nodes, prefix, window):
    # one node after the other: the nodes that do not see it keep their rows (to rounding: its
    # tile is added key by key)
    rng = np.random.default_rng([hd, nodes, prefix])
    q, k, v = base.inputs(rng, nodes, 8, hd, prefix)
    parents = base.tree(rng, nodes, "random")
    want = ref.attention_tree(q, k, v, prefix, parents.tolist(), window)
    for bad in sorted({0, 1, 15, 16, nodes // 2, nodes - 1}):
        for fill in (np.nan, np.inf, -np.inf):
            k2, v2 = k.copy(), v.copy()
            k2[prefix + bad], v2[prefix + bad] = fill, fill
            got = base.run(g4, q, k2, v2, prefix, parents, window)
            for i in range(nodes):
                path = ref.path_of(parents.tolist(), i)
                sees = bad in path and (not window or path.index(bad) > len(path) - 1 - window)
                if sees:
                    assert not np.isfinite(got[i]).any(), (bad, fill, i)
                else:
                    assert np.abs(got[i] - want[i]).max() <= 2e-5 * np.abs(v).max(), (bad, fill, i)


def test_bad_parents_give_nan_rows(g4):
    for hd in (64, 128, 512):
        rng = np.random.default_rng(hd)
        q, k, v = base.inputs(rng, 40, 8, hd, 90)
        parents = base.tree(rng, 40, "random")
        parents[[4, 17, 39]] = [4, 1 << 30, -(1 << 31)]
        bad = set()
        for i, p in enumerate(parents.tolist()):
            if not -1 <= p < i or p in bad:
                bad.add(i)
        good = np.where([i in bad for i in range(40)], -1, parents)
        got = base.run(g4, q, k, v, 90, parents, 0)
        want = ref.attention_tree(q, k, v, 90, good.tolist())
        for i in range(40):
            if i in bad:
                assert np.isnan(got[i]).all()
            else:
                assert np.abs(got[i] - want[i]).max() <= 2e-5 * np.abs(v).max()
