"""window_attention against its formula in 64 bits: single tokens, chunks and prompts, equal and ragged batches, windows and first
tokens of any size, types, heads, pages, lengths, what lies in places that are not seen, strides, queues."""
import ctypes

import numpy as np
import pytest

from attention_superoptimizer_amd import _native as N
from decoding_reference import check
from serving_reference import G, attended, caches, normal, put, read, window_seen

pytestmark = pytest.mark.gpu


def _case(seed, new, lengths, kv_heads, group, head, page_size, kind, heads_first=False, std=1.0, **more):
    k, v, table, values = caches(seed, lengths, kv_heads, head, page_size, kind, heads_first, **more)
    q = normal(np.random.default_rng(seed + 1000), (sum(new), kv_heads * group, head), kind, std)
    return q, k, v, table, np.array(lengths, np.int32), values


def _expected(q, values, new, lengths, window, sinks, scale, kind):
    out, bound, row = np.zeros_like(q), np.zeros_like(q), 0
    for (k, v), n, length in zip(values, new, lengths):
        length = max(0, length)
        out[row:row + n], bound[row:row + n] = attended(q[row:row + n], k[:length], v[:length], window_seen(length, n, window, sinks), scale, kind)
        row += n
    return out, bound


def _run(q, k, v, table, lengths, kind, window, sinks, scale, new=None, heads_first=False, flat=False, spare_rows=0):
    """new: the ragged form."""
    g = G.KNGraph()
    try:
        rows = np.concatenate([q, np.full((spare_rows, *q.shape[1:]), np.nan)])
        rows = rows.reshape(len(rows), -1) if flat else rows
        starts = None if new is None else put(g, np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        o = g.window_attention(put(g, rows, kind), put(g, k, kind), put(g, v, kind), put(g, table), put(g, lengths), window, sinks, starts,
                               scale=scale, heads_first=heads_first)
        got = []
        for _ in range(2):
            o.write_data(np.full(o.dims, 7.0))
            g.execute_all()
            got.append(read(o).reshape(len(q) + spare_rows, *q.shape[1:]))
        np.testing.assert_array_equal(got[0], got[1])  # the same inputs give the same bits
        assert (got[0][len(q):] == 7.0).all()  # rows behind the last sequence
        return got[0][:len(q)]
    finally:
        g.close()


def _check(seed, new, lengths, window, sinks, kv_heads=2, group=4, head=64, page_size=16, kind="fp16", ragged=False, heads_first=False,
           std=1.0, scale=None, flat=False, spare_rows=0):
    q, k, v, table, n, values = _case(seed, new, lengths, kv_heads, group, head, page_size, kind, heads_first, std)
    scale = float(np.float32(head ** -0.5 if scale is None else scale))
    want, bound = _expected(q, values, new, lengths, window, sinks, scale, kind)
    got = _run(q, k, v, table, n, kind, window, sinks, scale, new if ragged else None, heads_first, flat, spare_rows)
    check(got, want, bound)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head", [8, 64, 72, 80, 96, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("new", [1, 40])
def test_head_sizes(rt, kind, head, new):
    _check(head, [new] * 3, [137, 41, 230], 60, 5, head=head, kind=kind)


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 9), (1, 0), (1, 1), (2, 3), (31, 4), (32, 33), (64, 64), (100, 0), (200, 150), (299, 1), (300, 2),
                                          (1000, 1000), (7, 280), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("new", [1, 3, 70])
def test_windows_and_first_tokens(rt, window, sinks, new):
    _check(window % 1000 + sinks % 1000 + new, [new] * 2, [300, 171], window, sinks, kind="bf16" if new == 3 else "fp16")


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("page_size", [1, 2, 7, 16, 24, 32, 100, 128, 500])
@pytest.mark.parametrize("new", [1, 33])
def test_page_sizes(rt, page_size, heads_first, new):
    _check(page_size, [new] * 4, [50, 99, 257, 400], 90, 10, page_size=page_size, heads_first=heads_first, flat=heads_first, kind="bf16")


@pytest.mark.parametrize("lengths", [[0], [1], [2, 0, 3], [31, 32, 33], [63, 64, 65], [127, 128, 129], [255, 256, 257, 511, 513]])
@pytest.mark.parametrize("new", [1, 4, 50])
@pytest.mark.parametrize("window", [0, 64])
def test_lengths(rt, lengths, new, window):
    """Among them sequences with fewer keys than new tokens: the first of those see nothing."""
    _check(sum(lengths) + new, [new] * len(lengths), lengths, window, 3)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (8, 1), (2, 7), (1, 16), (3, 17), (1, 71), (5, 3), (1, 130)])
@pytest.mark.parametrize("new", [1, 6])
def test_heads(rt, kind, kv_heads, group, new):
    _check(group * 10 + new, [new] * 3, [90, 200, 33], 70, 4, kv_heads=kv_heads, group=group, kind=kind)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("new,past", [([5, 1, 33, 0, 200, 1], [10, 300, 0, 40, 70, 0]), ([0, 0], [5, 9]), ([300], [1]), ([1] * 70, list(range(70))),
                                      ([0] * 66 + [3, 0, 130], [20] * 69), ([129, 1, 127, 128], [64, 63, 500, 0])])
@pytest.mark.parametrize("window", [0, 50])
def test_ragged_batches(rt, kind, new, past, window):
    rows = sum(new)
    _check(rows, new, [n + p for n, p in zip(new, past)], window, 6, kind=kind, ragged=True, kv_heads=3, group=3, spare_rows=0 if rows else 4)
    if rows:
        _check(rows, new, [n + p for n, p in zip(new, past)], window, 6, kind=kind, ragged=True, kv_heads=1, group=2, head=80, spare_rows=9)


@pytest.mark.parametrize("sequences", [64, 65, 1000, 4200])
def test_ragged_batches_of_many_sequences(rt, sequences):
    new = [i * 7 % 4 for i in range(sequences)]
    new[sequences // 3] = 40
    _check(sequences, new, [n + i % 3 for i, n in enumerate(new)], 2, 1, head=8, page_size=8, ragged=True, kv_heads=1, group=7, spare_rows=3)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head", [64, 80, 128, 192, 256])
@pytest.mark.parametrize("window", [0, 2500])
def test_ragged_batches_behind_long_caches(rt, kind, head, window):
    """Few blocks of rows, cut along their keys."""
    _check(head, [3, 0, 50, 1], [4100, 10, 2950, 700], window, 4, head=head, kind=kind, ragged=True, kv_heads=1, group=3, spare_rows=2)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("head,group", [(128, 4), (64, 1), (256, 2)])
def test_prompts(rt, kind, head, group):
    _check(head, [700], [700], 0, 0, head=head, group=group, kind=kind, kv_heads=1)
    _check(head, [700], [900], 300, 4, head=head, group=group, kind=kind, kv_heads=1, std=2.0)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("window", [0, 4096, 1000])
@pytest.mark.parametrize("page_size", [1, 16])
def test_long_caches(rt, kind, window, page_size):
    _check(window, [1, 1], [9000, 3100], window, 4, kind=kind, head=128, page_size=page_size, std=2.0)
    _check(window, [9, 9], [9000, 3100], window, 4, kind=kind, kv_heads=1, page_size=page_size)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("new", [1, 40])
def test_scales(rt, scale, new):
    _check(3, [new] * 2, [100, 250], 80, 4, scale=scale)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("new", [1, 64])
def test_the_greatest_score_comes_late_and_early(rt, kind, new):
    """Scores that grow by hundreds along the keys, and fall by as much: sums are scaled again and again, or weights vanish."""
    for order in (1, -1):
        q, k, v, table, n, values = _case(5, [new], [400], 1, 2, 64, 16, kind)
        ramp = np.linspace(0.0, 4.0, 400)[::order, None, None]
        q[:] = np.where(np.arange(64) < 4, 8.0, q)
        keys = values[0][0]
        keys[:] = np.where(np.arange(64) < 4, np.round(ramp * 16) / 16, keys)
        for i in range(25):
            k[table[0, i]] = keys[16 * i:16 * i + 16]
        want, bound = _expected(q, values, [new], [400], 200, 8, 1.0, kind)
        check(_run(q, k, v, table, n, kind, 200, 8, 1.0), want, bound)


@pytest.mark.parametrize("new,ragged", [(1, False), (9, False), (70, False), (70, True)])
def test_pages_behind_the_window_may_be_anything(rt, new, ragged):
    """Pages that no row sees: their numbers are given back, out of range, or another sequence's."""
    window, sinks, length = 64, 5, 700
    q, k, v, table, n, values = _case(7, [new] * 2, [length] * 2, 2, 4, 64, 16, "fp16")
    want, bound = _expected(q, values, [new] * 2, [length] * 2, window, sinks, 0.125, "fp16")
    last_gone = (length - new + 1 - window) // 16  # pages before this one hold no key of the window
    table[0, 1:last_gone] = -1
    table[1, 1:last_gone] = [2 ** 31 - 1, -2 ** 31, len(k), table[0, -2]] * 20 + [0] * max(0, last_gone - 81) if last_gone > 81 else \
        ([2 ** 31 - 1, -2 ** 31, len(k), table[0, -2]] * 21)[:last_gone - 1]
    check(_run(q, k, v, table, n, "fp16", window, sinks, 0.125, [new] * 2 if ragged else None), want, bound)


def test_pages_outside_the_cache_hold_no_keys(rt):
    for new in (1, 40):
        q, k, v, table, n, values = _case(8, [new], [200], 2, 2, 64, 16, "fp16")
        table[0, 10] = len(k)
        seen = window_seen(200, new, 0, 0)
        seen[:, 160:176] = False
        want, bound = attended(q, *values[0], seen, 0.125, "fp16")
        check(_run(q, k, v, table, n, "fp16", 0, 0, 0.125), want, bound)
        table[:] = -5  # and none at all
        assert (_run(q, k, v, table, n, "fp16", 100, 4, 0.125) == 0).all()


def test_lengths_out_of_range(rt):
    for new in (1, 20):
        q, k, v, table, n, values = _case(9, [new] * 3, [48, 48, 48], 1, 2, 64, 16, "fp16", width=3)
        n[:] = [-7, 2 ** 31 - 1, -2 ** 31]
        want, bound = _expected(q, values, [new] * 3, [0, 48, 0], 30, 2, 0.125, "fp16")
        check(_run(q, k, v, table, n, "fp16", 30, 2, 0.125), want, bound)


def test_starts_out_of_range_stay_in_the_tensors(rt):
    """Rows that starts do not name are left; what is out of order or range is cut to the rows there are."""
    g = G.KNGraph()
    try:
        q, k, v, table, n, values = _case(10, [20, 20], [60, 60], 1, 2, 64, 16, "fp16")
        starts = put(g, np.array([-5, 20, 2 ** 31 - 1], np.int32))
        o = g.window_attention(put(g, q, "fp16"), put(g, k, "fp16"), put(g, v, "fp16"), put(g, table), put(g, n), 30, 2, starts, scale=0.125)
        g.execute_all()
        want, bound = _expected(q, values, [20, 20], [60, 60], 30, 2, 0.125, "fp16")
        check(read(o), want, bound)
        starts.write_data(np.array([20, 0, -9], np.int32))
        o.write_data(np.full(o.dims, 7.0))
        g.execute_all()
        assert (read(o) == 7.0).all()
    finally:
        g.close()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new", [1, 4, 40])
def test_places_that_are_not_seen_hold_anything(rt, value, new):
    """Behind the window, past a row's own key: values and keys that no row sees, or only some do."""
    for kind in ("fp16", "bf16"):
        q, k, v, table, n, values = _case(11, [new], [300], 1, 3, 80, 16, kind)
        want, bound = _expected(q, values, [new], [300], 100, 6, 0.1, kind)
        seen = window_seen(300, new, 100, 6)
        for j in (6, 30, 170, 299, 298):
            for cache in (k, v):
                cache[table[0, j // 16], j % 16] = value
        got = _run(q, k, v, table, n, kind, 100, 6, 0.1)
        clean = ~seen[:, [6, 30, 170, 299, 298]].any(1)
        assert clean.any() == (new > 2)
        check(got[clean], want[clean], bound[clean])
        # only the values: what is seen gives an infinity or NaN in its rows, and nothing to the others
        for j in (170, 299, 298):
            k[table[0, j // 16], j % 16] = values[0][0][j]
        got = _run(q, k, v, table, n, kind, 100, 6, 0.1)
        check(got[clean], want[clean], bound[clean])
        wild = got[seen[:, 299] | seen[:, 298]]
        assert (np.isnan(wild) if np.isnan(value) else wild == value).all()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new,length", [(1, 300), (4, 300), (40, 300), (40, 3000), (600, 900)])
def test_keys_that_are_not_finite(rt, value, new, length):
    """Rows that see such a key, whose score is no number or an infinity of either sign, and rows that do not."""
    q, k, v, table, n, values = _case(18, [new], [length], 1, 3, 80, 16, "bf16")
    want, bound = _expected(q, values, [new], [length], 200, 6, 0.1, "bf16")
    j = length - 1 - new // 2
    k[table[0, j // 16], j % 16] = 0.0
    k[table[0, j // 16], j % 16, :, 5] = value
    got = _run(q, k, v, table, n, "bf16", 200, 6, 0.1)
    sees = window_seen(length, new, 200, 6)[:, j]
    assert sees.any()
    check(got[~sees], want[~sees], bound[~sees])
    wild = np.isnan(got[sees]).all(-1)
    if np.isnan(value):
        assert wild.all()
    else:
        # a score of minus infinity is a key of no weight
        down = (q[sees, :, 5] * np.sign(value)) < 0
        without = window_seen(length, new, 200, 6)
        without[:, j] = False
        other, off = attended(q, values[0][0][:length], values[0][1][:length], without, 0.1, "bf16")
        np.testing.assert_array_equal(wild, ~down)
        assert new == 1 or (down.any() and not down.all())
        check(got[sees][down], other[sees][down], off[sees][down])


@pytest.mark.parametrize("ragged", [False, True])
def test_such_places_among_keys_that_several_workgroups_read(rt, ragged):
    q, k, v, table, n, values = _case(16, [40], [3000], 1, 3, 128, 16, "fp16")
    want, bound = _expected(q, values, [40], [3000], 2000, 6, 0.1, "fp16")
    seen = window_seen(3000, 40, 2000, 6)
    j = 2980
    v[table[0, j // 16], j % 16] = np.inf
    got = _run(q, k, v, table, n, "fp16", 2000, 6, 0.1, [40] if ragged else None)
    check(got[~seen[:, j]], want[~seen[:, j]], bound[~seen[:, j]])
    assert (~seen[:, j]).any() and (got[seen[:, j]] == np.inf).all()


@pytest.mark.parametrize("new", [1, 40])
def test_values_at_the_end_of_their_range(rt, new):
    """Sums of many of the largest bf16 values pass 32 bits, their mean does not."""
    q, k, v, table, n, values = _case(12, [new], [500], 1, 2, 64, 16, "bf16", std=0.1)
    big = float(np.float32(np.array(0x7f7f0000, np.uint32).view(np.float32)))
    values[0][1][:496] = big  # (the last page's four keys keep theirs)
    v[table[0, :31]] = big
    want, bound = _expected(q, values, [new], [500], 300, 4, 0.125, "bf16")
    check(_run(q, k, v, table, n, "bf16", 300, 4, 0.125), want, bound)


def test_scores_that_are_not_finite(rt):
    """Of minus infinity alone: zeros.  Plus infinity or NaN: NaN."""
    for new in (1, 40):
        q, k, v, table, n, _ = _case(13, [new], [100], 1, 2, 64, 16, "fp16")
        q[:] = 1.0
        k[np.isfinite(k)] = -np.inf
        assert (_run(q, k, v, table, n, "fp16", 30, 2, 0.125) == 0).all()
        assert np.isnan(_run(q, k, v, table, n, "fp16", 30, 2, -0.125)).all()


def _abi_call(abi, **x):
    return abi.mi355_window_attention(x["q"], x["q_stride"], x["out"], x["out_stride"], None if x["cache"] is None else ctypes.byref(x["cache"]),
                                      x["table"], x["width"], x["lengths"], x["starts"], x["sequences"], x["tokens"], x["heads"], x["scale"],
                                      x["window"], x["sinks"])


@pytest.mark.parametrize("new", [1, 33])
def test_strides_and_what_lies_between(rt, abi, new):
    """Queries inside a wider projection, results in wider rows, a cache whose heads and tokens lie apart."""
    g = G.KNGraph()
    try:
        kv_heads, group, head, size = 2, 3, 64, 16
        q, k, v, table, n, values = _case(14, [new] * 2, [150, 70], kv_heads, group, head, size, "fp16")
        wide = normal(np.random.default_rng(1), (2 * new, 10, head), "fp16")
        wide[:, 2:8] = q
        apart = [np.full((len(k), 3, size, kv_heads + 1, head + 8), np.nan) for _ in range(2)]
        for a, c in zip(apart, (k, v)):
            a[:, 1, :, 1:, :head] = c
        tq, to = put(g, wide, "fp16"), put(g, np.full((2 * new, 9, head), 3.0), "fp16")
        tk, tv = (put(g, a.reshape(len(k), -1), "fp16") for a in apart)
        token = (kv_heads + 1) * (head + 8)
        offset = 2 * (size * token + head + 8)
        cache = N.Mi355PagedCache(tk.device_ptr(False) + offset, tv.device_ptr(False) + offset, len(k), size, kv_heads, head, 3 * size * token,
                                  token, head + 8, 921)
        rc = _abi_call(abi, q=tq.device_ptr(False) + 2 * 2 * head, q_stride=10 * head, out=to.device_ptr(False) + 2 * head, out_stride=9 * head,
                       cache=cache, table=put(g, table).device_ptr(False), width=table.shape[1], lengths=put(g, n).device_ptr(False), starts=None,
                       sequences=2, tokens=2 * new, heads=6, scale=0.125, window=50, sinks=4)
        assert rc == 0, N.last_error()
        want, bound = _expected(q, values, [new] * 2, [150, 70], 50, 4, 0.125, "fp16")
        got = read(to)
        check(got[:, 1:7], want, bound)
        assert (got[:, :1] == 3.0).all() and (got[:, 7:] == 3.0).all()
    finally:
        g.close()


def test_queues_side_by_side(rt, abi):
    shapes = [([1, 1], [3000, 700], 1000), ([200, 200], [600, 200], 100)]
    cases = [_case(30 + i, new, lengths, 2, 4, 128, 16, "fp16") for i, (new, lengths, _) in enumerate(shapes)]
    graphs = []
    try:
        outs = []
        for x, (_, _, window) in zip(cases, shapes):
            g = G.KNGraph()
            graphs.append(g)
            outs.append(g.window_attention(put(g, x[0], "fp16"), put(g, x[1], "fp16"), put(g, x[2], "fp16"), put(g, x[3]), put(g, x[4]), window, 4,
                                           scale=0.125))
        for _ in range(10):
            for queue, g in enumerate(graphs):
                assert abi.mi355_queue_select(queue) == 0
                g.execute_all()
        assert abi.mi355_sync() == 0
        for x, (new, lengths, window), o in zip(cases, shapes, outs):
            want, bound = _expected(x[0], x[5], new, lengths, window, 4, 0.125, "fp16")
            check(read(o), want, bound)
    finally:
        abi.mi355_queue_select(0)
        for g in reversed(graphs):
            g.close()


@pytest.mark.parametrize("new", [1, 40])
def test_a_cache_past_32_bits(rt, abi, new):
    """Keys more than 2^32 bytes into their cache: pages far apart by their stride, few of them written."""
    import torch
    pages, size, head = 1100, 16, 128
    page_stride = 1 << 21  # elements: 4 MB
    q, k, v, table, n, values = _case(15, [new], [40], 1, 2, head, size, "fp16", spare=0, filler=0.0)
    cache = [torch.zeros(pages * page_stride, dtype=torch.float16, device="cuda") for _ in range(2)]
    far = np.array([[1099, 700, 1050, -1]], np.int32)
    for c, its in zip(cache, (k, v)):
        for p, at in zip(table[0, :3], far[0, :3]):
            rows = torch.from_numpy(its[p, :, 0].astype(np.float16)).cuda().reshape(-1)
            c[int(at) * page_stride:int(at) * page_stride + rows.numel()] = rows
    torch.cuda.synchronize()
    g = G.KNGraph()
    try:
        o = put(g, np.zeros((new, 2, head)), "fp16")
        c = N.Mi355PagedCache(cache[0].data_ptr(), cache[1].data_ptr(), pages, size, 1, head, page_stride, head, head, 921)
        rc = _abi_call(abi, q=put(g, q, "fp16").device_ptr(False), q_stride=2 * head, out=o.device_ptr(False), out_stride=2 * head, cache=c,
                       table=put(g, far).device_ptr(False), width=4, lengths=put(g, n).device_ptr(False), starts=None, sequences=1, tokens=new, heads=2,
                       scale=0.125, window=20, sinks=4)
        assert rc == 0, N.last_error()
        want, bound = _expected(q, values, [new], [40], 20, 4, 0.125, "fp16")
        check(read(o), want, bound)
    finally:
        g.close()
        del cache
        torch.cuda.empty_cache()


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
            x = dict(q=at, q_stride=128, out=at + 8192, out_stride=128, cache=cache() if c is None else c, table=i, width=4, lengths=i, starts=None,
                     sequences=2, tokens=4, heads=2, scale=1.0, window=8, sinks=2)
            x.update(change)
            return _abi_call(abi, **x)

        assert call() == 0 and call(starts=i) == 0 and call(sequences=0, tokens=0) == 0 and call(starts=i, tokens=0) == 0
        assert call(starts=i, sequences=0) == 0
        for change in (dict(q=None), dict(out=None), dict(table=None), dict(lengths=None), dict(q=at + 2), dict(out=at + 8200), dict(q_stride=132),
                       dict(out_stride=129), dict(width=0), dict(sequences=-1), dict(tokens=-1), dict(tokens=5), dict(heads=0), dict(cache=None),
                       dict(scale=float("nan")), dict(window=-1), dict(sinks=-1), dict(q_stride=-128), dict(out_stride=120), dict(sequences=0)):
            assert call(**change) == -3, change
        for change, code in ((dict(kv_heads=3), -3), (dict(k=None), -3), (dict(v=at + 16384), -3), (dict(page_stride=4), -3), (dict(token_stride=12), -3),
                             (dict(head_dim=60), -4), (dict(head_dim=264), -4), (dict(type=930), -4), (dict(pages=0), -3), (dict(k=at + 8), -3)):
            assert call(cache(**change)) == code, change
        assert call(width=1 << 29) == -4
        assert call(heads=1 << 20, tokens=1 << 14, sequences=1, q_stride=1 << 26, out_stride=1 << 26) == -4
        assert call(starts=i, sequences=1 << 24, tokens=4) == -4
    finally:
        g.close()
