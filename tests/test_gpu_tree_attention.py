"""tree_attention against its formula in 64 bits: chains, stars, random trees, padded ones and ones out of order; types, heads,
pages, lengths, what lies in places that are not seen, strides."""
import ctypes

import numpy as np
import pytest

from attention_superoptimizer_amd import _native as N
from decoding_reference import check
from serving_reference import G, attended, caches, normal, put, read, tree_seen

pytestmark = pytest.mark.gpu


def _tree(rng, nodes, shape):
    if shape == "chain":
        return np.arange(nodes) - 1
    if shape == "star":
        return np.full(nodes, -1)
    p = np.array([-1 if i == 0 or rng.random() < 0.1 else rng.integers(max(0, i - 9), i) for i in range(nodes)])
    if shape == "padded":
        p[max(1, 2 * nodes // 3):] = -2
    if shape == "wrong":  # itself, later ones, below -1: not there, nor what follows
        for i, wrong in zip(rng.permutation(nodes)[:max(1, nodes // 4)], [0, 1, 2 ** 31 - 1, -2 ** 31, -2, nodes] * nodes):
            p[i] = i + wrong if wrong in (0, 1) else wrong
    return p


def _case(seed, nodes, lengths, kv_heads, group, head, page_size, kind, shape="random", heads_first=False, std=1.0, **more):
    k, v, table, values = caches(seed, lengths, kv_heads, head, page_size, kind, heads_first, **more)
    rng = np.random.default_rng(seed + 1000)
    q = normal(rng, (len(lengths) * nodes, kv_heads * group, head), kind, std)
    parents = np.stack([_tree(rng, nodes, shape) for _ in lengths]).astype(np.int32)
    return q, k, v, table, np.array(lengths, np.int32), parents, values


def _expected(q, values, lengths, parents, scale, kind):
    out, bound, n = np.zeros_like(q), np.zeros_like(q), parents.shape[1]
    for b, ((k, v), length) in enumerate(zip(values, lengths)):
        out[b * n:(b + 1) * n], bound[b * n:(b + 1) * n] = attended(q[b * n:(b + 1) * n], k[:length], v[:length],
                                                                    tree_seen(length, parents[b]), scale, kind)
    return out, bound


def _run(q, k, v, table, lengths, parents, kind, scale, heads_first=False, flat=False):
    g = G.KNGraph()
    try:
        rows = q.reshape(len(q), -1) if flat else q
        o = g.tree_attention(put(g, rows, kind), put(g, k, kind), put(g, v, kind), put(g, table), put(g, lengths), put(g, parents), scale=scale,
                             heads_first=heads_first)
        got = []
        for _ in range(2):
            o.write_data(np.full(o.dims, 7.0))
            g.execute_all()
            got.append(read(o).reshape(q.shape))
        np.testing.assert_array_equal(got[0], got[1])  # the same inputs give the same bits
        return got[0]
    finally:
        g.close()


def _check(seed, nodes, lengths, kv_heads=2, group=4, head=64, page_size=16, kind="fp16", shape="random", heads_first=False, std=1.0,
           scale=None, flat=False):
    *x, values = _case(seed, nodes, lengths, kv_heads, group, head, page_size, kind, shape, heads_first, std)
    scale = float(np.float32(head ** -0.5 if scale is None else scale))
    want, bound = _expected(x[0], values, lengths, x[5], scale, kind)
    check(_run(*x, kind, scale, heads_first, flat), want, bound)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head", [8, 64, 72, 80, 96, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("nodes", [4, 7, 40])
def test_head_sizes(rt, kind, head, nodes):
    _check(head, nodes, [137, 41, 230], head=head, kind=kind)


@pytest.mark.parametrize("shape", ["chain", "star", "random", "padded", "wrong"])
@pytest.mark.parametrize("nodes", [1, 2, 5, 16, 31, 32, 33, 64, 65, 130])
def test_trees(rt, shape, nodes):
    _check(nodes, nodes, [nodes + 50, nodes + 1, nodes, nodes + 203], shape=shape, kind="bf16" if nodes % 2 else "fp16")


@pytest.mark.parametrize("shape", ["chain", "star", "random"])
def test_the_largest_trees(rt, shape):
    _check(1, 1024, [1024, 1500], kv_heads=1, group=1, shape=shape)


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("page_size", [1, 2, 7, 16, 24, 32, 100, 128, 500])
def test_page_sizes(rt, page_size, heads_first):
    _check(page_size, 4, [50, 99, 257, 400], page_size=page_size, heads_first=heads_first, flat=heads_first)
    _check(page_size, 12, [50, 99, 257, 400], page_size=page_size, heads_first=heads_first, flat=heads_first, kind="bf16")
    _check(page_size, 40, [50, 99, 257, 400], page_size=page_size, heads_first=heads_first, flat=heads_first)


@pytest.mark.parametrize("lengths", [[0], [1], [5, 0, 9], [10, 11, 12], [31, 32, 33], [63, 64, 65], [127, 128, 129], [255, 256, 257, 511, 513]])
@pytest.mark.parametrize("nodes", [1, 10, 40])
def test_lengths(rt, lengths, nodes):
    """Among them sequences shorter than their trees: the first nodes are not there."""
    _check(sum(lengths) + nodes, nodes, lengths)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (8, 1), (2, 7), (1, 16), (3, 17), (1, 71), (5, 3)])
@pytest.mark.parametrize("nodes", [3, 20])
def test_heads(rt, kind, kv_heads, group, nodes):
    _check(group * 10 + nodes, nodes, [90, 200, 33], kv_heads=kv_heads, group=group, kind=kind)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head,nodes,group", [(128, 12, 4), (64, 64, 8), (128, 4, 4), (64, 15, 1), (80, 3, 5), (256, 7, 2), (80, 13, 5), (256, 20, 2), (192, 30, 4)])
def test_long_caches(rt, kind, head, nodes, group):
    _check(head, nodes, [5000, 137, 2900], nodes and 2, group, head, kind=kind, std=2.0)
    _check(head, nodes, [9000], 1, group, head, page_size=1, kind=kind)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(rt, scale):
    _check(3, 3, [100, 250], scale=scale)
    _check(3, 12, [100, 250], scale=scale)
    _check(3, 50, [100, 250], scale=scale)


def test_many_sequences(rt):
    _check(4, 6, [6 + (37 * i) % 90 for i in range(150)], kv_heads=1, group=2)
    _check(4, 20, [20 + (137 * i) % 900 for i in range(150)], kv_heads=1, group=2)  # parts dealt to them by their lengths


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("nodes", [5, 9, 40])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_places_that_are_not_seen_hold_anything(rt, value, nodes, kind):
    """A node's key and value that its descendants alone see."""
    *x, values = _case(5, nodes, [nodes + 130], 1, 3, 80, 16, kind)
    q, k, v, table, lengths, parents = x
    want, bound = _expected(q, values, lengths, parents, 0.1, kind)
    seen = tree_seen(nodes + 130, parents[0])
    j = 130 + nodes // 2
    for cache in (k, v):
        cache[table[0, j // 16], j % 16] = value
    got = _run(*x, kind, 0.1)
    clean = ~seen[:, j]
    assert clean.any() and not clean.all()
    check(got[clean], want[clean], bound[clean])
    k[table[0, j // 16], j % 16] = values[0][0][j]  # only the value
    got = _run(*x, kind, 0.1)
    check(got[clean], want[clean], bound[clean])
    assert (np.isnan(got[~clean]) if np.isnan(value) else got[~clean] == value).all()


@pytest.mark.parametrize("value", [np.nan, -np.inf])
@pytest.mark.parametrize("sequences", [1, 2])
def test_such_places_among_keys_that_several_workgroups_read(rt, value, sequences):
    nodes, length = 20, 3000
    *x, values = _case(15, nodes, [length, 700][:sequences], 1, 4, 80, 16, "bf16")
    q, k, v, table, lengths, parents = x
    want, bound = _expected(q, values, lengths, parents, 0.1, "bf16")
    j = length - 8
    v[table[0, j // 16], j % 16] = value
    got = _run(*x, "bf16", 0.1)
    sees = np.concatenate([tree_seen(length, parents[0])[:, j], np.zeros((sequences - 1) * nodes, bool)])
    assert sees.any() and not sees[:nodes].all()
    check(got[~sees], want[~sees], bound[~sees])
    assert (np.isnan(got[sees]) if np.isnan(value) else got[sees] == value).all()


@pytest.mark.parametrize("nodes", [6, 40])
def test_values_at_the_end_of_their_range(rt, nodes):
    """Sums of many of the largest bf16 values pass 32 bits, their mean does not."""
    *x, values = _case(12, nodes, [500], 1, 2, 64, 16, "bf16", std=0.1)
    big = float(np.float32(np.array(0x7f7f0000, np.uint32).view(np.float32)))
    x[2][x[3][0, :32]] = big
    got = _run(*x, "bf16", 0.125)
    assert (np.abs(got / big - 1) <= 2.0 ** -7).all()


def test_lengths_and_pages_out_of_range(rt):
    for nodes in (5, 40):
        *x, values = _case(9, nodes, [96] * 3, 1, 2, 64, 16, "fp16", width=6)
        x[4][:] = [-7, 2 ** 31 - 1, 96]
        x[3][2, 1] = len(x[1])
        want, bound = _expected(x[0], values, [0, 96, 96], x[5], 0.125, "fp16")
        seen = tree_seen(96, x[5][2])
        seen[:, 16:32] = False
        want[2 * nodes:], bound[2 * nodes:] = attended(x[0][2 * nodes:], *values[2], seen, 0.125, "fp16")
        check(_run(*x, "fp16", 0.125), want, bound)


def test_a_chain_is_what_paged_attention_computes(rt):
    """Within what both may be off."""
    for nodes in (4, 30):
        *x, values = _case(6, nodes, [300, 77], 2, 4, 64, 16, "fp16", shape="chain")
        want, bound = _expected(x[0], values, [300, 77], x[5], 0.125, "fp16")
        g = G.KNGraph()
        try:
            o = g.paged_attention(put(g, x[0], "fp16"), put(g, x[1], "fp16"), put(g, x[2], "fp16"), put(g, x[3]), put(g, x[4]), scale=0.125)
            g.execute_all()
            check(_run(*x, "fp16", 0.125), read(o), 2 * bound)
        finally:
            g.close()


def _abi_call(abi, **x):
    return abi.mi355_tree_attention(x["q"], x["q_stride"], x["out"], x["out_stride"], None if x["cache"] is None else ctypes.byref(x["cache"]),
                                    x["table"], x["width"], x["lengths"], x["parents"], x["sequences"], x["nodes"], x["heads"], x["scale"])


@pytest.mark.parametrize("nodes", [3, 6, 33])
def test_strides_and_what_lies_between(rt, abi, nodes):
    g = G.KNGraph()
    try:
        kv_heads, group, head, size = 2, 3, 64, 16
        *x, values = _case(14, nodes, [150, 70], kv_heads, group, head, size, "fp16")
        q, k, v, table, n, parents = x
        wide = normal(np.random.default_rng(1), (2 * nodes, 10, head), "fp16")
        wide[:, 2:8] = q
        apart = [np.full((len(k), 3, size, kv_heads + 1, head + 8), np.nan) for _ in range(2)]
        for a, c in zip(apart, (k, v)):
            a[:, 1, :, 1:, :head] = c
        tq, to = put(g, wide, "fp16"), put(g, np.full((2 * nodes, 9, head), 3.0), "fp16")
        tk, tv = (put(g, a.reshape(len(k), -1), "fp16") for a in apart)
        token = (kv_heads + 1) * (head + 8)
        offset = 2 * (size * token + head + 8)
        cache = N.Mi355PagedCache(tk.device_ptr(False) + offset, tv.device_ptr(False) + offset, len(k), size, kv_heads, head, 3 * size * token,
                                  token, head + 8, 921)
        rc = _abi_call(abi, q=tq.device_ptr(False) + 2 * 2 * head, q_stride=10 * head, out=to.device_ptr(False) + 2 * head, out_stride=9 * head,
                       cache=cache, table=put(g, table).device_ptr(False), width=table.shape[1], lengths=put(g, n).device_ptr(False),
                       parents=put(g, parents).device_ptr(False), sequences=2, nodes=nodes, heads=6, scale=0.125)
        assert rc == 0, N.last_error()
        want, bound = _expected(q, values, [150, 70], parents, 0.125, "fp16")
        got = read(to)
        check(got[:, 1:7], want, bound)
        assert (got[:, :1] == 3.0).all() and (got[:, 7:] == 3.0).all()
    finally:
        g.close()


def test_queues_side_by_side(rt, abi):
    """Keys cut over workgroups, whose sums each queue has in memory of its own."""
    shapes = [(20, [3000, 700, 1500]), (33, [2500]), (40, [900] * 5)]
    cases = [_case(40 + i, nodes, lengths, 2, 4, 64, 16, "bf16") for i, (nodes, lengths) in enumerate(shapes)]
    graphs, outs = [], []
    try:
        for *x, _ in cases:
            g = G.KNGraph()
            graphs.append(g)
            kinds = ("bf16",) * 3 + (None,) * 3
            outs.append(g.tree_attention(*(put(g, a) if kind is None else put(g, a, kind) for a, kind in zip(x, kinds)), scale=0.125))
        for _ in range(10):
            for queue, g in enumerate(graphs):
                assert abi.mi355_queue_select(queue) == 0
                g.execute_all()
        assert abi.mi355_sync() == 0
        for (*x, values), o in zip(cases, outs):
            want, bound = _expected(x[0], values, x[4], x[5], 0.125, "bf16")
            check(read(o).reshape(want.shape), want, bound)
    finally:
        abi.mi355_queue_select(0)
        for g in reversed(graphs):
            g.close()


def test_refusals(rt, abi):
    g = G.KNGraph()
    try:
        at = g.new_input((1 << 15,), G.DT_FLOAT16).device_ptr(False)
        i = put(g, np.zeros(64, np.int32)).device_ptr(False)

        def cache(**change):
            c = N.Mi355PagedCache(at + 16384, at + 24576, 4, 8, 1, 64, 512, 64, 64, 921)
            for name, value in change.items():
                setattr(c, name, value)
            return c

        def call(c=None, **change):
            x = dict(q=at, q_stride=128, out=at + 8192, out_stride=128, cache=cache() if c is None else c, table=i, width=4, lengths=i, parents=i,
                     sequences=2, nodes=3, heads=2, scale=1.0)
            x.update(change)
            return _abi_call(abi, **x)

        assert call() == 0 and call(sequences=0) == 0
        for change in (dict(q=None), dict(out=None), dict(table=None), dict(lengths=None), dict(parents=None), dict(q=at + 2), dict(out=at + 8200),
                       dict(q_stride=132), dict(out_stride=129), dict(width=0), dict(sequences=-1), dict(nodes=0), dict(heads=0), dict(cache=None),
                       dict(scale=float("inf")), dict(q_stride=-128), dict(out_stride=120)):
            assert call(**change) == -3, change
        for change, code in ((dict(kv_heads=3), -3), (dict(k=None), -3), (dict(v=at + 16384), -3), (dict(page_stride=4), -3), (dict(head_dim=60), -4),
                             (dict(head_dim=264), -4), (dict(type=930), -4), (dict(pages=0), -3), (dict(k=at + 8), -3)):
            assert call(cache(**change)) == code, change
        assert call(nodes=1025) == -4 and call(width=1 << 29) == -4 and call(sequences=2 ** 31 - 1, nodes=1024) == -4
    finally:
        g.close()
