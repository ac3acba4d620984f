"""Scores of any size that 32 bits hold: keys that are alike have weights that are."""
import numpy as np
import pytest

from decoding_reference import HALF_STEP, check
from serving_reference import G, caches, normal, put, read
from test_gpu_tree_attention import _run as run_tree
from test_gpu_window_attention import _run as run_window

pytestmark = pytest.mark.gpu


def _mean(values, group, kind):
    """Results of equal weights, and how far they may be off.  The weights are the same number; n of them are added up in 32 bits, and n products with
    them, twice over where parts are joined: (n + 16) 2^-23 of the sum of magnitudes each; then a rounding to the type."""
    n, want = len(values), values.mean(0)
    bound = HALF_STEP[kind][0] * np.abs(want) + HALF_STEP[kind][1] + 4 * (n + 16) * 2.0 ** -23 * np.abs(values).mean(0)
    return np.repeat(want, group, 0), np.repeat(bound, group, 0)


def _paged(q, k, v, table, n, kind, scale):
    g = G.KNGraph()
    try:
        o = g.paged_attention(put(g, q, kind), put(g, k, kind), put(g, v, kind), put(g, table), put(g, n), scale=scale)
        g.execute_all()
        return read(o).reshape(q.shape)
    finally:
        g.close()


@pytest.mark.parametrize("kind,size", [(kind, size) for size in (100.0, 999.0, 5001.0, 20011.0, 60013.0, -60013.0) for kind in ("fp16", "bf16")] +
                         [("bf16", 3e9), ("bf16", 3e17)])
@pytest.mark.parametrize("head", [64, 80, 192])
@pytest.mark.parametrize("form,new,length", [("window", 1, 1), ("window", 4, 4), ("window", 40, 500), ("ragged", 1, 77), ("ragged", 600, 700), ("tree", 3, 3),
                                             ("tree", 40, 3000), ("paged", 1, 1), ("paged", 1, 3000), ("paged", 12, 300), ("paged", 40, 300)])
def test_equal_keys(rt, form, new, length, head, kind, size):
    k, v, table, values = caches(length, [length], 1, head, 16, kind)
    k[np.isfinite(k)] = size
    size = float(np.float32(size))
    q = np.full((new, 2, head), abs(size))
    n, scale = np.array([length], np.int32), 0.0883883461356163
    if form == "tree":
        got = run_tree(q, k, v, table, n, np.arange(new, dtype=np.int32)[None] - 1, kind, scale)
    elif form == "paged":
        got = _paged(q, k, v, table, n, kind, scale)
    else:
        got = run_window(q, k, v, table, n, kind, 0, 0, scale, [new] if form == "ragged" else None)
    for t in {0, new // 2, new - 1}:
        want, bound = _mean(values[0][1][:length - (new - 1 - t)], 2, kind)
        check(got[t], want, bound, t)


@pytest.mark.parametrize("form,new", [("window", 1), ("window", 5), ("window", 40), ("tree", 2), ("tree", 40), ("paged", 1), ("paged", 40)])
@pytest.mark.parametrize("largest", [1.0, -1.0])
def test_the_largest_scale(rt, form, new, largest):
    """Scores are zero, or pass 32 bits: those below zero are minus infinity."""
    k, v, table, values = caches(3, [200], 1, 64, 16, "fp16")
    q = np.zeros((new, 1, 64))
    q[-1] = -largest
    k[np.isfinite(k)] = 1.0
    k[table[0, 2], 5] = 0.0
    n, scale = np.array([200], np.int32), largest * float(np.finfo(np.float32).max)
    if form == "tree":
        got = run_tree(q, k, v, table, n, np.arange(new, dtype=np.int32)[None] - 1, "fp16", scale)
    elif form == "paged":
        got = _paged(q, k, v, table, n, "fp16", scale)
    else:
        got = run_window(q, k, v, table, n, "fp16", 0, 0, scale)
    for t in range(new - 1):
        want, bound = _mean(values[0][1][:200 - (new - 1 - t)], 1, "fp16")
        check(got[t], want, bound, t)
    want, bound = _mean(values[0][1][37:38], 1, "fp16")
    check(got[-1], want, bound)
