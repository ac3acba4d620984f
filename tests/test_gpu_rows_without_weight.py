"""Rows without a weight are zeros, whatever the values are: trees of one node that is not there, scores of minus infinity alone."""
import numpy as np
import pytest

from decoding_reference import check
from serving_reference import G, attended, caches, normal, put, read
from test_gpu_tree_attention import _run as run_tree
from test_gpu_window_attention import _run as run_window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("group,length", [(4, 70), (1, 5000), (16, 1), (20, 200)])
def test_a_tree_of_one_node_that_is_not_there(rt, group, length, kind, value):
    lengths = [length, length, 0]
    k, v, table, values = caches(length + group, lengths, 2, 64, 16, kind)
    q = normal(np.random.default_rng(length), (3, 2 * group, 64), kind)
    v[table[0, 0], 0] = value
    parents = np.array([[-2], [-1], [-1]], np.int32)
    for wrong in (-2, 0, 1, 2 ** 31 - 1):
        parents[0] = wrong
        got = run_tree(q, k, v, table, np.array(lengths, np.int32), parents, kind, 0.125)
        assert (got[[0, 2]] == 0).all()
        want, bound = attended(q[1:2], *values[1], np.ones((1, length), bool), 0.125, kind)
        check(got[1:2], want, bound)


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("length", [100, 6000])
def test_scores_of_minus_infinity_beside_any_value(rt, new, length, value):
    k, v, table, _ = caches(1, [length], 1, 64, 16, "bf16")
    q = np.ones((new, 2, 64))
    k[np.isfinite(k)] = -np.inf
    v[table[0, 1], 3] = value
    n = np.array([length], np.int32)
    for window in (0, 80):
        v[table[0, (length - 50) // 16], 3] = value
        assert (run_window(q, k, v, table, n, "bf16", window, 2, 0.125) == 0).all()
    assert (run_tree(q, k, v, table, n, np.arange(new, dtype=np.int32)[None] - 1, "bf16", 0.125) == 0).all()
    g = G.KNGraph()
    try:
        o = g.paged_attention(put(g, q, "bf16"), put(g, k, "bf16"), put(g, v, "bf16"), put(g, table), put(g, n), scale=0.125)
        g.execute_all()
        assert (read(o) == 0).all()
    finally:
        g.close()
