"""Keys whose scores are no numbers, where a row sees no other key of a part that the keys are cut into."""
import numpy as np
import pytest

from decoding_reference import check
from serving_reference import attended, caches, normal, tree_seen, window_seen
from test_gpu_tree_attention import _run as run_tree
from test_gpu_window_attention import _run as run_window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("form", ["window", "ragged", "tree", "trees"])
@pytest.mark.parametrize("length", [256, 1024])  # four parts, and sixteen, which several wavefronts join
def test_a_row_that_sees_no_other_key_of_a_part(rt, kind, form, length):
    """New token 0 sees one key of the last tile, its own."""
    new, count = 64, 2 if form == "trees" else 1
    k, v, table, values = caches(length, [length] * count, 1, 64, 16, kind, width=length // 16)
    q = normal(np.random.default_rng(length), (count * new, 1, 64), kind)
    n, parents = np.full(count, length, np.int32), np.tile(np.arange(new, dtype=np.int32) - 1, (count, 1))
    j = length - new
    k[table[0, j // 16], j % 16] = np.nan
    if form in ("tree", "trees"):
        got = run_tree(q, k, v, table, n, parents, kind, 0.125)
    else:
        got = run_window(q, k, v, table, n, kind, 0, 0, 0.125, [new] if form == "ragged" else None)
    assert np.isnan(got[:new]).all()
    for b in range(1, count):
        want, bound = attended(q[b * new:], *values[b], tree_seen(length, parents[b]), 0.125, kind)
        check(got[b * new:], want, bound)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_the_first_token_alone_in_a_part(rt, kind):
    """The window of the later rows begins behind the part with the first token."""
    new, length, window = 100, 1024, 600
    k, v, table, _ = caches(7, [length], 1, 64, 16, kind, width=length // 16)
    q = normal(np.random.default_rng(7), (new, 1, 64), kind)
    k[table[0, 0], 0] = np.nan
    assert window_seen(length, new, window, 1)[:, 0].all()
    assert np.isnan(run_window(q, k, v, table, np.array([length], np.int32), kind, window, 1, 0.125)).all()
