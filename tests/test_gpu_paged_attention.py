"""paged_attention against its formula in 64 bits: types, groups, head sizes, page sizes, lengths from nothing to long
ones, several new tokens, windows, both layouts of the cache, pages in any order, and what lies in masked places."""
import ctypes

import numpy as np
import pytest

from attention_superoptimizer_amd import _native as N
from attention_superoptimizer_amd import graph as G
from decoding_reference import TYPES, attention, check, normal, put, read, rounded

pytestmark = pytest.mark.gpu


def _case(seed, lengths, new, kv_heads, group, head, page_size, kind, heads_first=False, spare=3, std=1.0, width=None):
    """q, caches (NaN where no sequence has a key), table (-1 behind a sequence's pages) and lengths."""
    rng = np.random.default_rng(seed)
    need = [-(-max(0, n) // page_size) for n in lengths]
    width = width or max(1, *need) + 1
    pages = sum(need) + spare
    order, at = rng.permutation(pages), 0
    table = np.full((len(lengths), width), -1, np.int32)
    k, v = (np.full((pages, page_size, kv_heads, head), np.nan) for _ in range(2))
    for b, (n, p) in enumerate(zip(lengths, need)):
        table[b, :p] = order[at:at + p]
        at += p
        for j in range(n):
            k[table[b, j // page_size], j % page_size] = normal(rng, (kv_heads, head), kind)
            v[table[b, j // page_size], j % page_size] = normal(rng, (kv_heads, head), kind)
    if heads_first:
        k, v = (np.ascontiguousarray(c.swapaxes(1, 2)) for c in (k, v))
    q = normal(rng, (len(lengths), new, kv_heads * group, head), kind, std)
    return q, k, v, table, np.array(lengths, np.int32)


def _run(q, k, v, table, lengths, kind, scale, window=0, heads_first=False, flat=False, passes=2):
    g = G.KNGraph()
    try:
        rows = q.reshape(-1, q.shape[2] * q.shape[3]) if flat else q.reshape(-1, *q.shape[2:])
        o = g.paged_attention(put(g, rows, kind), put(g, k, kind), put(g, v, kind), put(g, table), put(g, lengths), scale=scale,
                              window=window, heads_first=heads_first)
        got = []
        for _ in range(passes):
            o.write_data(np.full(o.dims, 7.0))
            g.execute_all()
            got.append(read(o).reshape(q.shape))
        for other in got[1:]:  # the same inputs give the same bits
            np.testing.assert_array_equal(got[0], other)
        return got[0]
    finally:
        g.close()


def _check(seed, lengths, new=1, kv_heads=2, group=4, head=64, page_size=16, kind="fp16", window=0, heads_first=False, std=1.0,
           flat=False, scale=None):
    x = _case(seed, lengths, new, kv_heads, group, head, page_size, kind, heads_first, std=std)
    scale = np.float32(head ** -0.5 if scale is None else scale)
    want, bound = attention(*x, float(scale), window, kind, heads_first)
    check(_run(*x, kind, float(scale), window, heads_first, flat), want, bound)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head", [8, 64, 72, 80, 96, 128, 136, 192, 200, 256])
def test_head_sizes(rt, kind, head):
    _check(head, [37, 1, 130], head=head, kind=kind)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("kv_heads,group,new", [(1, 1, 1), (8, 1, 1), (2, 7, 1), (1, 16, 1), (3, 17, 1), (1, 71, 1), (2, 4, 5), (1, 3, 11),
                                                (2, 8, 8), (1, 16, 9), (1, 1, 70)])
def test_rows_of_a_key_value_head(rt, kind, kv_heads, group, new):
    _check(group * 100 + new, [90, 200, max(1, new - 3)], new=new, kv_heads=kv_heads, group=group, kind=kind)


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("page_size", [1, 2, 7, 16, 24, 32, 100, 128, 500])
def test_page_sizes(rt, page_size, heads_first):
    _check(page_size, [1, 99, 100, 257, 400], page_size=page_size, heads_first=heads_first, flat=heads_first, kind="bf16")


@pytest.mark.parametrize("lengths", [[0], [1], [2, 0, 3], [15, 16, 17], [31, 32, 33], [63, 64, 65], [127, 128, 129], [255, 256, 257, 511, 513],
                                     [0, 0, 0, 5]])
@pytest.mark.parametrize("new", [1, 4])
def test_lengths(rt, lengths, new):
    _check(sum(lengths), lengths, new=new, kind="fp16")


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head,new,group", [(128, 1, 4), (64, 3, 8), (256, 1, 2)])
def test_long_cache_split_over_workgroups(rt, kind, head, new, group):
    _check(head, [5000, 37, 2900], new=new, group=group, head=head, kind=kind, std=2.0)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("group,new", [(5, 4), (8, 5), (16, 4), (8, 9), (3, 37)])
def test_many_rows_split_over_workgroups(rt, kind, head, group, new):
    """Rows for two, three, four groups of sixteen and for several blocks of them, a head's keys with several workgroups."""
    _check(head + new, [900, 33], new=new, kv_heads=1, group=group, head=head, kind=kind, std=2.0)


@pytest.mark.parametrize("head,group,new,lengths,kv_heads", [(64, 4, 1, [3000, 100], 2), (96, 1, 1, [1500], 1), (128, 8, 1, [4100, 0, 257], 2),
                                                             (64, 8, 3, [2100, 700], 2), (96, 16, 2, [300, 1300], 1), (128, 9, 3, [2000], 2),
                                                             (64, 12, 4, [2500, 31], 1), (64, 4, 1, list(range(20, 900, 30)), 3)])
@pytest.mark.parametrize("window", [0, 700])
def test_wide_tables(rt, head, group, new, lengths, kv_heads, window):
    """Tables that name room for far more keys than there are: few heads that may have much to read."""
    kind = "bf16" if head == 96 else "fp16"
    x = _case(head + new, lengths, new, kv_heads, group, head, 16, kind, width=4200)
    want, bound = attention(*x, float(np.float32(0.11)), window, kind)
    check(_run(*x, kind, float(np.float32(0.11)), window), want, bound)


def _claimed(abi, x, kind, pages, window=0):
    """The same by the C ABI, of a cache that is said to have `pages` pages (the table names those there are)."""
    q, k, v, table, n = x
    size, kv_heads, head = k.shape[1:]
    q_heads = q.shape[2]
    g = G.KNGraph()
    try:
        tq, tk, tv, tt, tl = put(g, q.reshape(-1, q_heads, head), kind), put(g, k, kind), put(g, v, kind), put(g, table), put(g, n)
        o = put(g, np.full((q.shape[0] * q.shape[1], q_heads, head), 7.0), kind)
        c = N.Mi355PagedCache(tk.device_ptr(False), tv.device_ptr(False), pages, size, kv_heads, head, size * kv_heads * head,
                              kv_heads * head, head, TYPES[kind])
        rc = abi.mi355_paged_attention(tq.device_ptr(False), q_heads * head, o.device_ptr(False), q_heads * head, ctypes.byref(c),
                                       tt.device_ptr(False), table.shape[1], tl.device_ptr(False), q.shape[0], q.shape[1], q_heads, 0.125,
                                       window)
        assert rc == 0, N.last_error()
        want, bound = attention(*x, 0.125, window, kind)
        check(read(o).reshape(q.shape), want, bound)
    finally:
        g.close()


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head,group,new", [(64, 4, 1), (72, 8, 3), (96, 2, 2), (128, 8, 1), (128, 8, 4), (128, 8, 5), (64, 11, 4), (160, 3, 1), (192, 7, 3),
                                            (256, 2, 1), (256, 8, 4)])
def test_caches_larger_than_the_last_level_cache(rt, abi, kind, head, group, new):
    """A cache of which the table could name more than is kept on the chip (and names a few pages)."""
    _claimed(abi, _case(head + new, [1300, 5, 0, 640], new, 2, group, head, 16, kind, width=1 << 15), kind, 1 << 17)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head,group,new,width", [(64, 1, 1, 8), (80, 3, 1, 20), (96, 4, 2, 32), (128, 4, 1, 32), (128, 2, 8, 5), (256, 1, 1, 8)])
@pytest.mark.parametrize("pages", [0, 1 << 15])
def test_many_heads_over_short_tables(rt, abi, kind, head, group, new, width, pages):
    """Thousands of key-value heads of a few hundred keys at most, of caches small and large."""
    rng = np.random.default_rng(head + width)
    lengths = [int(n) for n in rng.integers(0, min(16 * width, 90), 256)] + [16 * width, 0, 1]
    x = _case(head + new, lengths, new, 8, group, head, 16, kind, width=width)
    _claimed(abi, x, kind, max(pages, x[1].shape[0]), window=37 if width == 20 else 0)


@pytest.mark.parametrize("window", [0, 200])
def test_more_heads_than_workgroups(rt, window):
    """Workgroups go on from one head to the next and share the longer ones; the last parts of heads join out of turn."""
    rng = np.random.default_rng(17)
    lengths = [int(n) for n in rng.integers(0, 90, 90)] + [2500, 0, 1] + [int(n) for n in rng.integers(200, 500, 20)]
    _check(18, lengths, new=2, kv_heads=8, group=2, window=window, page_size=32, kind="fp16")


def test_a_page_a_sequence(rt):
    """Pages of more keys than 16 bits count: a cache without paging."""
    _check(19, [70100, 300, 0], kv_heads=1, group=2, page_size=70000, kind="bf16")


def test_many_short_sequences(rt):
    rng = np.random.default_rng(2)
    _check(1, [int(n) for n in rng.integers(0, 60, 300)], kv_heads=4, group=2, kind="bf16")


@pytest.mark.parametrize("window", [1, 2, 16, 33, 100, 1000])
@pytest.mark.parametrize("new", [1, 6])
def test_windows(rt, window, new):
    _check(window, [300, 7, 129, 0], new=new, window=window, page_size=24, kind="bf16")


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(rt, scale):
    """Scores all alike, turned round, and so far apart that all but a few weights vanish."""
    _check(11, [70, 300], scale=scale, kind="fp16", std=2.0)


def test_the_greatest_score_comes_late_and_early(rt):
    """The running maximum grows with every key, or never after the first."""
    q, k, v, table, lengths = _case(3, [400, 400], 1, 1, 2, 64, 16, "fp16")
    q[:] = 1.0
    for b, turn in ((0, 1), (1, -1)):
        for j in range(400):
            k[table[b, j // 16], j % 16] = (j - 200) / 64 * turn
    want, bound = attention(q, k, v, table, lengths, 0.5, 0, "fp16")
    check(_run(q, k, v, table, lengths, "fp16", 0.5), want, bound)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_small_weights_add_up(rt, kind):
    """One key far ahead, thousands whose weights of 2^-15 each matter together only."""
    n, head = 8000, 64
    q, k, v, table, lengths = _case(4, [n], 1, 1, 1, head, 16, kind)
    q[:] = 0.0
    q[..., 0] = 1.0
    flat_k, flat_v = (c.reshape(-1, head) for c in (k, v))
    for j in range(n):
        at = table[0, j // 16] * 16 + j % 16
        flat_k[at] = 0.0
        flat_v[at] = 1.0
    at = table[0, 77 // 16] * 16 + 77 % 16
    flat_k[at, 0] = 10.375  # e^10.375 = 2^14.97
    flat_v[at] = -1.0
    want, bound = attention(q, k, v, table, lengths, 1.0, 0, kind)
    check(_run(q, k, v, table, lengths, kind, 1.0), want, bound)


def test_lengths_out_of_range(rt):
    """Negative lengths are nothing, and one past the table ends with it."""
    q, k, v, table, lengths = _case(6, [40, 40, 40, 48], 3, 2, 2, 64, 16, "fp16", width=3)
    k, v = np.nan_to_num(k), np.nan_to_num(v)
    lengths[:] = [-5, -2147483648, 2147483647, 1000]
    want, bound = attention(q, k, v, table, lengths, 0.125, 0, "fp16")
    assert (want[:2] == 0).all()
    check(_run(q, k, v, table, lengths, "fp16", 0.125), want, bound)


def test_pages_outside_the_cache_hold_no_keys(rt):
    q, k, v, table, lengths = _case(7, [200, 200, 64], 2, 2, 2, 64, 16, "bf16")
    k, v = np.nan_to_num(k), np.nan_to_num(v)
    table[0, 3], table[0, 7], table[1, 12] = -1, k.shape[0], 2147483647
    table[2, :4] = [-2147483648, k.shape[0], -1, 1 << 30]
    want, bound = attention(q, k, v, table, lengths, 0.125, 0, "bf16")
    assert (want[2] == 0).all()
    check(_run(q, k, v, table, lengths, "bf16", 0.125), want, bound)


def test_sequences_share_pages(rt):
    q, k, v, table, lengths = _case(8, [100, 100, 90], 1, 2, 4, 128, 16, "fp16")
    table[1, :5] = table[0, :5]
    table[2] = table[0]
    table[2, 2] = table[2, 1]  # the same page twice
    want, bound = attention(q, k, v, table, lengths, 0.1, 0, "fp16")
    check(_run(q, k, v, table, lengths, "fp16", 0.1), want, bound)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("new,window", [(1, 0), (4, 0), (4, 50), (1, 50), (1, 64)])
def test_masked_places_hold_anything(rt, value, new, window):
    """Behind a sequence's end, before its window and, for all new tokens but the last, at the last token's key: no row
    that does not see the key changes by a bit."""
    lengths = [100, 203, new]
    q, k, v, table, n = _case(9, lengths, new, 2, 3, 64, 16, "bf16")
    k, v = np.nan_to_num(k), np.nan_to_num(v)
    plain = _run(q, k, v, table, n, "bf16", 0.125, window, passes=1)
    for b, length in enumerate(lengths):
        for j in range(-(-length // 16) * 16):
            if j >= length - 1 or (window and j <= length - new - window):
                if new > 1 or j != length - 1:
                    k[table[b, j // 16], j % 16] = v[table[b, j // 16], j % 16] = value
    got = _run(q, k, v, table, n, "bf16", 0.125, window, passes=1)
    rows = slice(0, new - 1) if new > 1 else slice(0, 1)
    np.testing.assert_array_equal(got[:, rows], plain[:, rows])
    if new > 1 and np.isnan(value):
        assert np.isnan(got[:, -1]).all()


def test_values_that_are_seen_and_not_finite(rt):
    """An infinite value makes its column infinite, a NaN key every result of its rows NaN, an infinite score too; scores
    of minus infinity weigh nothing."""
    q, k, v, table, lengths = _case(10, [64, 64, 64, 64], 1, 1, 1, 64, 16, "bf16")
    q[:] = rounded(np.abs(q) + 0.5, "bf16")
    v[table[0, 1], 3, 0, 5] = np.inf
    k[table[1, 2], 9, 0, 7] = np.nan
    k[table[2, 0], 2, 0, 1] = np.inf
    seen = k.copy()
    k[table[3, 0]] = -np.inf
    got = _run(q, k, v, table, lengths, "bf16", 0.125, passes=1)
    assert got[0, 0, 0, 5] == np.inf and np.isfinite(np.delete(got[0, 0, 0], 5)).all()
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all()
    table[3, 0] = -1  # as if those keys were not there
    want, bound = attention(q[3:], seen, v, table[3:], lengths[3:], 0.125, 0, "bf16")
    check(got[3:], want, bound)


def test_strides_and_what_lies_between(rt, abi):
    """Queries within wider rows, results likewise, pages further apart than their keys."""
    kind, head, kv_heads, group, size = "fp16", 64, 2, 2, 8
    q, k, v, table, lengths = _case(12, [50, 9], 2, kv_heads, group, head, size, kind)
    rows, wide, out_wide, page_stride = 4, 4 * 64 + 40, 4 * 64 + 16, size * kv_heads * head + 64
    g = G.KNGraph()
    try:
        big_q, big_o = np.full((rows, wide), np.nan), np.full((rows, out_wide), 3.0)
        big_q[:, 8:8 + 256] = q.reshape(rows, 256)
        apart = [np.full((k.shape[0], page_stride), np.nan) for _ in range(2)]
        for a, c in zip(apart, (k, v)):
            a[:, :size * kv_heads * head] = c.reshape(c.shape[0], -1)
        tq, to, tk, tv = put(g, big_q, kind), put(g, big_o, kind), put(g, apart[0], kind), put(g, apart[1], kind)
        tt, tl = put(g, table), put(g, lengths)
        c = N.Mi355PagedCache(tk.device_ptr(False), tv.device_ptr(False), k.shape[0], size, kv_heads, head, page_stride,
                              kv_heads * head, head, 921)
        rc = abi.mi355_paged_attention(tq.device_ptr(False) + 16, wide, to.device_ptr(False), out_wide, ctypes.byref(c),
                                       tt.device_ptr(False), table.shape[1], tl.device_ptr(False), 2, 2, 4, 0.125, 0)
        assert rc == 0, N.last_error()
        want, bound = attention(q, k, v, table, lengths, 0.125, 0, kind)
        got = read(to)
        check(got[:, :256].reshape(q.shape), want, bound)
        assert (got[:, 256:] == 3.0).all()
    finally:
        g.close()


def test_queues_side_by_side(rt, abi):
    """Two queues run calls of their own at the same time, each split over workgroups and joined."""
    cases = [_case(20 + i, [3000, 700], 1, 2, 4, 128, 16, "fp16") for i in range(2)]
    graphs = []
    try:
        outs = []
        for x in cases:
            g = G.KNGraph()
            graphs.append(g)
            outs.append(g.paged_attention(put(g, x[0].reshape(-1, 8, 128), "fp16"), put(g, x[1], "fp16"), put(g, x[2], "fp16"),
                                          put(g, x[3]), put(g, x[4]), scale=0.09))
        for _ in range(20):
            for queue, g in enumerate(graphs):
                assert abi.mi355_queue_select(queue) == 0
                g.execute_all()
        assert abi.mi355_sync() == 0
        for x, o in zip(cases, outs):
            want, bound = attention(*x, float(np.float32(0.09)), 0, "fp16")
            check(read(o).reshape(want.shape), want, bound)
    finally:
        abi.mi355_queue_select(0)
        for g in reversed(graphs):
            g.close()


def test_a_cache_past_32_bits(rt):
    """Keys more than 2^32 bytes into their cache: pages far apart by their stride, few of them written."""
    import torch
    pages, size, head = 1100, 16, 128
    page_stride = 1 << 21  # elements: 4 MB
    tokens = 40
    q, k, v, table, lengths = _case(13, [tokens], 1, 1, 2, head, size, "fp16", spare=0)
    cache = [torch.zeros(pages * page_stride, dtype=torch.float16, device="cuda") for _ in range(2)]
    far = np.array([[1099, 700, 1050, -1]], np.int32)
    for c, values in zip(cache, (k, v)):
        for p, at in zip(table[0, :3], far[0, :3]):
            rows = torch.from_numpy(np.nan_to_num(values[p, :, 0]).astype(np.float16)).cuda().reshape(-1)
            c[int(at) * page_stride:int(at) * page_stride + rows.numel()] = rows
    torch.cuda.synchronize()
    g = G.KNGraph()
    try:
        tq, tt, tl = put(g, q.reshape(1, 2, head), "fp16"), put(g, far), put(g, lengths)
        o = g.new_input((1, 2, head))
        c = N.Mi355PagedCache(cache[0].data_ptr(), cache[1].data_ptr(), pages, size, 1, head, page_stride, head, head, 921)
        rc = N.backend().mi355_paged_attention(tq.device_ptr(False), 2 * head, o.device_ptr(False), 2 * head, ctypes.byref(c),
                                               tt.device_ptr(False), 4, tl.device_ptr(False), 1, 1, 2, 0.1, 0)
        assert rc == 0, N.last_error()
        want, bound = attention(q, k, v, table, lengths, float(np.float32(0.1)), 0, "fp16")
        check(read(o).reshape(want.shape), want, bound)
    finally:
        g.close()
        del cache
        torch.cuda.empty_cache()


def test_refusals(rt, abi):
    g = G.KNGraph()
    try:
        t = g.new_input((1 << 14,), TYPES["fp16"])
        at = t.device_ptr(False)
        i = put(g, np.zeros(64, np.int32)).device_ptr(False)

        def call(c, **change):
            x = dict(q=at, q_stride=128, out=at + 8192, out_stride=128, table=i, width=4, lengths=i, sequences=2, new=1, heads=2, scale=1.0,
                     window=0)
            x.update(change)
            return abi.mi355_paged_attention(x["q"], x["q_stride"], x["out"], x["out_stride"], None if c is None else ctypes.byref(c),
                                             x["table"], x["width"], x["lengths"], x["sequences"], x["new"], x["heads"], x["scale"],
                                             x["window"])

        def cache(**change):
            c = N.Mi355PagedCache(at + 16384, at + 24576, 4, 8, 1, 64, 512, 64, 64, 921)
            for name, value in change.items():
                setattr(c, name, value)
            return c

        assert call(cache()) == 0
        assert call(cache(), sequences=0) == 0
        for change in (dict(q=None), dict(out=None), dict(table=None), dict(lengths=None), dict(q=at + 2), dict(out=at + 8200),
                       dict(q_stride=132), dict(out_stride=129), dict(width=0), dict(sequences=-1), dict(new=0), dict(heads=0),
                       dict(scale=float("nan")), dict(window=-1), dict(q_stride=-128), dict(out_stride=120)):
            assert call(cache(), **change) == -3, change
        assert call(None) == -3
        for change, code in ((dict(kv_heads=3), -3), (dict(k=None), -3), (dict(v=at + 16384), -3), (dict(page_stride=4), -3),
                             (dict(token_stride=12), -3), (dict(head_dim=60), -4), (dict(head_dim=264), -4), (dict(type=930), -4),
                             (dict(pages=0), -3), (dict(k=at + 8), -3)):
            assert call(cache(**change)) == code, change
        assert call(cache(), width=1 << 29) == -4
        assert call(cache(head_dim=256, token_stride=256, page_stride=2048), heads=1 << 24, q_stride=1 << 32, out_stride=1 << 32) == -4
        assert call(cache(), sequences=1, out_stride=0) == 0  # one row
    finally:
        g.close()
