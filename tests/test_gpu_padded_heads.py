"""Heads whose size is no size that kernels are compiled for, over keys with an infinity among their last columns: their scores are what the
formula says, a key whose score is minus infinity has no weight."""
import numpy as np
import pytest

from decoding_reference import check
from serving_reference import attended, caches, normal, tree_seen, window_seen
from test_gpu_tree_attention import _run as run_tree
from test_gpu_window_attention import _run as run_window

pytestmark = pytest.mark.gpu


def _case(seed, new, length, group, head, kind):
    k, v, table, values = caches(seed, [length], 1, head, 16, kind)
    return normal(np.random.default_rng(seed + 1000), (new, group, head), kind), k, v, table, np.array([length], np.int32), values[0]


@pytest.mark.parametrize("value", [np.inf, -np.inf])
@pytest.mark.parametrize("head", [8, 64, 72, 80, 136, 184, 200, 248])
@pytest.mark.parametrize("form,new", [("window", 1), ("window", 40), ("ragged", 1), ("ragged", 40), ("tree", 4), ("tree", 40)])
def test_a_key_with_an_infinity_in_its_last_columns(rt, form, new, head, value):
    kind, length = "fp16" if head % 16 else "bf16", 300
    for column in {head - 1, head - 8}:
        q, k, v, table, n, (keys, values) = _case(head + new, new, length, 3, head, kind)
        parents = np.arange(new, dtype=np.int32)[None] - 1
        seen = tree_seen(length, parents[0]) if form == "tree" else window_seen(length, new, 0, 0)
        j = 250  # every row sees it
        k[table[0, j // 16], j % 16] = 0.0
        k[table[0, j // 16], j % 16, :, column] = value
        got = run_tree(q, k, v, table, n, parents, kind, 0.1) if form == "tree" else \
            run_window(q, k, v, table, n, kind, 0, 0, 0.1, [new] if form == "ragged" else None)
        down = q[:, :, column] * np.sign(value) < 0  # the score is minus infinity
        assert new == 1 or (down.any() and not down.all())
        np.testing.assert_array_equal(np.isnan(got).all(-1), ~down)
        seen[:, j] = False
        want, bound = attended(q, keys[:length], values[:length], seen, 0.1, kind)
        check(got[down], want[down], bound[down])


@pytest.mark.parametrize("head", [8, 72, 80, 136, 200])
@pytest.mark.parametrize("form,new", [("window", 1), ("window", 40), ("ragged", 1), ("ragged", 40), ("tree", 40)])
def test_scores_of_minus_infinity_alone(rt, form, new, head):
    q, k, v, table, n, _ = _case(3, new, 100, 2, head, "fp16")
    q[:] = 1.0
    k[np.isfinite(k).all(-1), -1] = -np.inf
    got = run_tree(q, k, v, table, n, np.arange(new, dtype=np.int32)[None] - 1, "fp16", 0.125) if form == "tree" else \
        run_window(q, k, v, table, n, "fp16", 30, 2, 0.125, [new] if form == "ragged" else None)
    assert (got == 0).all()
