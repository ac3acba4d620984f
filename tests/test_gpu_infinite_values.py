"""Values that are infinite or NaN among keys that some rows see and others do not: each element of the result is what its own column's say, and none of them
makes a call take many times as long."""
import ctypes

import numpy as np
import pytest

from decoding_reference import check
from serving_reference import G, attended, caches, normal, put, read, tree_seen, window_seen
from test_gpu_tree_attention import _run as run_tree, _tree
from test_gpu_window_attention import _run as run_window

pytestmark = pytest.mark.gpu


def _agree(got, q, keys, values, wild, seen, scale, kind):
    """`wild` [keys, kv_heads, head]: the values in place of `values`, or zero."""
    want, bound = attended(q, keys, values, seen, scale, kind)
    group = q.shape[1] // keys.shape[1]
    some = {}
    for name, its in (("nan", np.isnan(wild)), ("up", wild == np.inf), ("down", wild == -np.inf)):
        some[name] = np.repeat(np.einsum("rk,khd->rhd", seen.astype(np.float64), its.astype(np.float64)) > 0, group, 1)
    nan = some["nan"] | (some["up"] & some["down"])
    up, down = some["up"] & ~nan, some["down"] & ~nan
    clean = ~(nan | up | down)
    assert clean.any() and not clean.all()
    np.testing.assert_array_equal(np.isnan(got), nan)
    assert (got[up] == np.inf).all() and (got[down] == -np.inf).all()
    check(got[clean], want[clean], bound[clean])


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head", [8, 64, 80, 128, 192, 200, 256])
@pytest.mark.parametrize("form,new,length,window", [("window", 4, 200, 90), ("window", 150, 400, 0), ("window", 300, 900, 100), ("ragged", 70, 2500, 0),
                                                    ("ragged", 1, 3000, 0), ("tree", 5, 300, 0), ("tree", 60, 150, 0), ("tree", 100, 3000, 0)])
def test_every_column_by_itself(rt, form, new, length, window, head, kind):
    sinks, kv_heads, group = 5, 2, 3
    seed = head + new
    k, v, table, values = caches(seed, [length], kv_heads, head, 16, kind)
    rng = np.random.default_rng(seed)
    q = normal(rng, (new, kv_heads * group, head), kind)
    keys, its = values[0]
    wild = np.zeros_like(its)
    # among the first and last keys, and those that some rows see only; with a column of both signs
    at = np.unique(np.concatenate([rng.integers(max(0, length - new - 3), length, 12), rng.integers(0, length, 8), [0, length - 1, length - new]]))
    for j in at:
        wild[j, rng.integers(0, kv_heads), rng.integers(0, head)] = rng.choice([np.nan, np.inf, -np.inf])
    wild[length - new, 0, head - 1], wild[length - 1, 0, head - 1] = np.inf, -np.inf
    is_wild = wild != 0
    for j in at:
        page = v[table[0, j // 16], j % 16]
        page[is_wild[j]] = wild[j][is_wild[j]]
    its = np.where(is_wild, 0.0, its)
    n, scale = np.array([length], np.int32), float(np.float32(head ** -0.5))
    if form == "tree":
        parents = _tree(rng, new, "random").astype(np.int32)[None]
        got, seen = run_tree(q, k, v, table, n, parents, kind, scale), tree_seen(length, parents[0])
    else:
        got = run_window(q, k, v, table, n, kind, window, sinks, scale, [new] if form == "ragged" else None)
        seen = window_seen(length, new, window, sinks)
    _agree(got, q, keys, its, wild, seen, scale, kind)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_weights_that_vanish_behind_them(rt, kind):
    """Scores that grow by hundreds behind an infinite value: its column stays what it is, or is NaN, and the others are right."""
    new, length = 100, 700
    k, v, table, values = caches(3, [length], 1, 64, 16, kind)
    q = np.zeros((new, 2, 64))
    q[..., 0] = 8.0
    keys, its = values[0]
    keys[:, 0] = np.round(np.linspace(0.0, 64.0, length) * 4)[:, None] / 4
    for i in range(length):
        k[table[0, i // 16], i % 16] = keys[i]
    v[table[0, 0], 3, 0, 11] = np.inf
    its[3, 0, 11] = 0.0
    got = run_window(q, k, v, table, np.array([length], np.int32), kind, 0, 0, 1.0)
    assert (np.isnan(got[..., 11]) | (got[..., 11] == np.inf)).all()
    want, bound = attended(q, keys, its, window_seen(length, new, 0, 0), 1.0, kind)
    rest = np.arange(64) != 11
    check(got[..., rest], want[..., rest], bound[..., rest])


@pytest.mark.parametrize("form", ["window", "tree"])
def test_a_call_with_one_takes_no_longer_than_ten_without(rt, abi, form):
    """About twice as long; done again row by row it took hundreds of times as long."""
    rng = np.random.default_rng(1)
    new, length, sequences = (1024, 1024, 1) if form == "window" else (64, 3000, 8)
    g = G.KNGraph()
    try:
        pages = -(-length // 16)
        tk, tv = (put(g, normal(rng, (sequences * pages, 16, 4, 128), "bf16"), "bf16") for _ in range(2))
        q = put(g, normal(rng, (sequences * new, 8, 128), "bf16"), "bf16")
        table = put(g, np.arange(sequences * pages, dtype=np.int32).reshape(sequences, pages))
        n = put(g, np.full(sequences, length, np.int32))
        if form == "tree":
            o = g.tree_attention(q, tk, tv, table, n, put(g, np.tile(np.arange(new, dtype=np.int32) - 1, (sequences, 1))))
        else:
            o = g.window_attention(q, tk, tv, table, n, 0)

        def took():
            best = np.inf
            for _ in range(6):
                assert abi.mi355_timer_start() == 0
                for _ in range(5):
                    g.execute_all()
                ms = ctypes.c_float()
                assert abi.mi355_timer_stop(ctypes.byref(ms)) == 0
                best = min(best, ms.value)
            return best

        clean = took()
        v = tv.read_data()
        v[1, 4, 2, 5] = np.inf
        tv.write_data(v)
        wild = took()
        assert (read(o).reshape(sequences * new, 8, 128)[20:new, 4:6, 5] == np.inf).all()
        assert wild <= 10 * clean, (wild, clean)
    finally:
        g.close()
