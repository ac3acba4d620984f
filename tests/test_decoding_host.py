"""Operators of a decoding step without a device: the tensors they take and refuse, their wire format, the angles of
rotary positions, bf16 values, what fingerprinting says to them, and the C ABI before mi355_init."""
import ctypes
import json
import math

import numpy as np
import pytest

from attention_superoptimizer_amd import _native as N
from attention_superoptimizer_amd import graph as G

F16, BF16, F32, F64, I32 = G.DT_FLOAT16, G.DT_BFLOAT16, G.DT_FLOAT32, G.DT_DOUBLE, G.DT_INT32


@pytest.fixture
def g():
    graph = G.KNGraph()
    yield graph
    graph.close()


def _append_inputs(g, qkv=(5, 12, 64), kind=F16, positions=(5,), angles=(2, 32), slots=(5,), cache=(7, 16, 2, 64), cache_kind=F16,
                   index=I32, angle_kind=F64):
    return [g.new_input(qkv, kind), g.new_input(positions, index), g.new_input(angles, angle_kind), g.new_input(slots, index),
            g.new_input(cache, cache_kind), g.new_input(cache, cache_kind)]


def test_shapes_of_results(g):
    for kind in (F16, BF16):
        x = _append_inputs(g, kind=kind, cache_kind=kind)
        q = g.rotary_append(*x)
        assert q.dims == (5, 8, 64) and q.data_type == kind
        flat = g.rotary_append(g.new_input((5, 12 * 64), kind), *x[1:])
        assert flat.dims == (5, 512)
        y = g.rotary(x[0], x[1], x[2], interleaved=True)
        assert y.dims == (5, 12, 64) and y.data_type == kind
        table, lengths = g.new_input((5, 4), I32), g.new_input((5,), I32)
        assert g.paged_attention(q, x[4], x[5], table, lengths).dims == (5, 8, 64)
        assert g.paged_attention(flat, x[4], x[5], table, lengths).dims == (5, 512)
    first = g.new_input((7, 2, 16, 64)), g.new_input((7, 2, 16, 64))
    assert g.rotary_append(g.new_input((5, 12, 64)), x[1], x[2], x[3], *first, heads_first=True).dims == (5, 8, 64)
    tokens, u = g.new_input((3, 4), I32), g.new_input((3, 5), F32)
    for kind in (F16, BF16, F32):
        for target, draft in (((3, 5, 100), (3, 4, 100)), ((15, 100), (12, 100))):
            n, out = g.verify_drafts(g.new_input(target, kind), g.new_input(draft, kind), tokens, u)
            assert n.dims == (3,) and out.dims == (3, 5) and n.data_type == out.data_type == I32
            assert g.verify_drafts(g.new_input(target, kind), None, tokens, u)[1].dims == (3, 5)


@pytest.mark.parametrize("change", [
    dict(qkv=(5, 4, 64)), dict(qkv=(5, 12, 32)), dict(qkv=(5, 100)), dict(kind=F32), dict(kind=BF16), dict(cache_kind=F32, kind=F32),
    dict(positions=(4,)), dict(positions=(5, 1)), dict(slots=(6,)), dict(index=F32), dict(angles=(1, 32)), dict(angles=(2, 33)),
    dict(angles=(64,)), dict(angle_kind=F32), dict(cache=(7, 16, 128)),
])
def test_rotary_append_refuses(g, change):
    x = _append_inputs(g, **change)
    operators = g.num_operators
    with pytest.raises(G.InfeasibleOperator):
        g.rotary_append(*x)
    assert g.num_operators == operators


def test_rotary_append_refuses_one_tensor_as_both_caches(g):
    x = _append_inputs(g)
    with pytest.raises(G.InfeasibleOperator):
        g.rotary_append(*x[:4], x[4], x[4])
    column = g.new_input((7, 16, 2, 64), layout="DmemColumnMajor")
    with pytest.raises(G.InfeasibleOperator):
        g.rotary_append(*x[:4], x[4], column)


@pytest.mark.parametrize("change", [dict(x=(5, 64)), dict(kind=F32), dict(positions=(6,)), dict(angles=(2, 33)), dict(angles=(3, 8)),
                                    dict(index=F16), dict(x=(5, 1, 4096), angles=(2, 1025))])
def test_rotary_refuses(g, change):
    x = g.new_input(change.get("x", (5, 3, 64)), change.get("kind", F16))
    positions = g.new_input(change.get("positions", (5,)), change.get("index", I32))
    angles = g.new_input(change.get("angles", (2, 32)), F64)
    with pytest.raises(G.InfeasibleOperator):
        g.rotary(x, positions, angles)


@pytest.mark.parametrize("change", [
    dict(q=(7, 8, 64)), dict(q=(6, 9, 64)), dict(q=(6, 8, 72)), dict(q=(6, 65)), dict(kind=BF16), dict(kind=F32, cache_kind=F32),
    dict(cache=(7, 16, 2, 60), q=(6, 8, 60)), dict(cache=(7, 16, 2, 264), q=(6, 8, 264)), dict(cache=(7, 16, 128)),
    dict(table=(3,)), dict(table=(4, 5)), dict(lengths=(2,)), dict(index=F32), dict(scale=math.inf), dict(scale=math.nan),
    dict(window=-1), dict(table=(3, 1 << 27)), dict(table=(3, 1 << 26), q=(6, 512, 64), cache=(7, 16, 256, 64)),
])
def test_paged_attention_refuses(g, change):
    cache = change.get("cache", (7, 16, 2, 64))
    index = change.get("index", I32)
    q = g.new_input(change.get("q", (6, 8, 64)), change.get("kind", F16))
    k, v = (g.new_input(cache, change.get("cache_kind", F16)) for _ in range(2))
    table, lengths = g.new_input(change.get("table", (3, 5)), index), g.new_input(change.get("lengths", (3,)), index)
    with pytest.raises(G.InfeasibleOperator):
        g.paged_attention(q, k, v, table, lengths, scale=change.get("scale", 0.125), window=change.get("window", 0))


@pytest.mark.parametrize("change", [
    dict(target=(3, 4, 100)), dict(target=(14, 100)), dict(target=(3, 5, 99)), dict(draft=(3, 5, 100)), dict(draft_kind=F16),
    dict(kind=F64, draft_kind=F64), dict(tokens=(3, 5)), dict(tokens=(12,)), dict(uniforms=(3, 4)), dict(uniform_kind=F64), dict(index=F32),
])
def test_verify_drafts_refuses(g, change):
    target = g.new_input(change.get("target", (3, 5, 100)), change.get("kind", F32))
    draft = g.new_input(change.get("draft", (3, 4, 100)), change.get("draft_kind", F32))
    tokens = g.new_input(change.get("tokens", (3, 4)), change.get("index", I32))
    uniforms = g.new_input(change.get("uniforms", (3, 5)), change.get("uniform_kind", F32))
    with pytest.raises(G.InfeasibleOperator):
        g.verify_drafts(target, draft, tokens, uniforms)


def test_results_that_do_not_fit_the_arena_are_refused(g):
    left = int(N.runtime().mirage_arena_total() - N.runtime().mirage_arena_offset())
    rows = left // (2 * 64 * 64 * 3) + 1  # the input fits, and the result with its fingerprints does not
    x, positions = g.new_input((rows, 64, 64)), g.new_input((rows,), I32)
    angles = g.new_input((2, 32), F64)
    with pytest.raises(G.InfeasibleOperator):
        g.rotary(x, positions, angles)


def _every_operator(g):
    x = _append_inputs(g)
    q = g.rotary_append(*x, interleaved=True)
    o = g.paged_attention(q, x[4], x[5], g.new_input((5, 4), I32), g.new_input((5,), I32), scale=0.37, window=9)
    g.rotary(o, x[1], x[2])
    first = [g.new_input((7, 2, 16, 64)) for _ in range(2)]
    q = g.rotary_append(*x[:4], *first, heads_first=True)
    g.paged_attention(q, *first, g.new_input((5, 4), I32), g.new_input((5,), I32), heads_first=True)
    target, tokens, u = g.new_input((3, 5, 100), BF16), g.new_input((3, 4), I32), g.new_input((3, 5), F32)
    g.verify_drafts(target, g.new_input((3, 4, 100), BF16), tokens, u)
    n, out = g.verify_drafts(target, None, tokens, u)
    return out


def test_wire_format(g):
    _every_operator(g)
    said = json.loads(g.to_json())
    ops = [o for o in said if o["op_type"] not in ("kn_input_op",)]
    assert [o["op_type"] for o in ops] == ["kn_rotary_append_op", "kn_paged_attention_op", "kn_rotary_op", "kn_rotary_append_op",
                                           "kn_paged_attention_op", "kn_verify_drafts_op", "kn_verify_drafts_op"]
    assert ops[0]["interleaved"] is True and ops[0]["heads_first"] is False and ops[3]["heads_first"] is True
    assert ops[1]["window"] == 9 and np.float32(ops[1]["scale"]) == np.float32(0.37) and ops[4]["heads_first"] is True
    again = G.KNGraph.from_json(said)
    try:
        back = json.loads(again.to_json())
        for o in said + back:
            for t in o["input_tensors"] + o["output_tensors"]:
                del t["guid"]
        assert back == said
    finally:
        again.close()
    ops[1]["window"] = -3
    for o in said:
        for t in o["input_tensors"] + o["output_tensors"]:
            t["guid"] = 0
    with pytest.raises(ValueError):
        G.KNGraph.from_json(said)


def test_graphs_without_a_fingerprint_are_refused(g, capfd):
    _every_operator(g)
    plain = G.KNGraph()
    try:
        plain.exp(plain.new_input((4, 4)))
        for reference, candidates in ((g, [plain]), (plain, [plain, g])):
            with pytest.raises(AssertionError):
                G.verify_batch(candidates, reference)
            with pytest.raises(AssertionError):
                G.verify_batch_begin(candidates, reference)
        with pytest.raises(AssertionError):
            g.fingerprint_seeded(1)
        with pytest.raises(AssertionError):
            g.fingerprint(6)
        assert "kn_rotary_append_op has no fingerprint" in capfd.readouterr().err
    finally:
        plain.close()


def test_popped_operators_leave_the_arena(g):
    x = _append_inputs(g)
    at = N.runtime().mirage_arena_offset()
    g.rotary_append(*x)
    g.pop_operator()
    t = g.new_input((3, 5, 100), F32)
    tokens, u = g.new_input((3, 4), I32), g.new_input((3, 5), F32)
    inner = N.runtime().mirage_arena_offset()
    g.verify_drafts(t, None, tokens, u)
    g.pop_operator()
    assert N.runtime().mirage_arena_offset() == inner
    for _ in range(3):
        g.pop_operator()
    assert N.runtime().mirage_arena_offset() == at


def test_abi_before_init():
    if N.backend().mi355_is_initialised():
        pytest.skip("a device is attached")
    cache = N.Mi355PagedCache()
    assert N.backend().mi355_rotary(None, 0, None, 0, None, None, 1, 1, 2, 1, 0, 921) == -5
    assert N.backend().mi355_rotary_append(None, 0, None, 0, None, 0, None, 0, None, None, None, ctypes.byref(cache), 1, 1, 1, 0) == -5
    assert N.backend().mi355_paged_attention(None, 0, None, 0, ctypes.byref(cache), None, 1, None, 1, 1, 1, 1.0, 0) == -5
    assert N.backend().mi355_verify_drafts(None, None, None, None, None, None, 1, 1, 1, 930) == -5


def test_rotary_angles():
    a = G.rotary_angles(8, base=100.0)
    np.testing.assert_allclose(a[0], [1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75], rtol=1e-15)
    assert (a[1] == 1.0).all() and a.dtype == np.float64
    np.testing.assert_allclose(G.rotary_angles(8, base=100.0, factor=4.0, amplitude=1.2)[0], a[0] / 4, rtol=1e-15)
    # 64 turns and more stay, 2 and fewer are slowed, 33 of them half of each
    w = G.rotary_angles(64)[0]
    s = G.rotary_angles(64, factor=8.0, original_length=4096, fast=64.0, slow=2.0, amplitude=1.1)
    turns = w * 4096 / (2 * np.pi)
    np.testing.assert_allclose(s[0][turns >= 64], w[turns >= 64], rtol=1e-15)
    np.testing.assert_allclose(s[0][turns <= 2], w[turns <= 2] / 8, rtol=1e-15)
    mid = (turns > 2) & (turns < 64)
    assert mid.any()
    share = (turns[mid] - 2) / 62
    np.testing.assert_allclose(s[0][mid], w[mid] * (share + (1 - share) / 8), rtol=1e-14)
    assert (s[1] == 1.1).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, factor=0.0),
                dict(rotary_dim=8, fast=1.0, slow=1.0)):
        with pytest.raises(ValueError):
            G.rotary_angles(**bad)


def test_bf16_values_round_to_the_nearest_even():
    x = np.array([1.0, 1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -8, 1.0 + 2.0 ** -8 + 2.0 ** -20, -0.0, np.inf, -np.inf, 3.3961775e38], np.float32)
    got = (G._bf16_bits(x).astype(np.uint32) << 16).view(np.float32)
    want = np.array([1.0, 1.0, 1.0 + 2.0 ** -6, 1.0 + 2.0 ** -7, -0.0, np.inf, -np.inf, np.inf], np.float32)
    np.testing.assert_array_equal(got.view(np.uint32), want.view(np.uint32))
    nan = G._bf16_bits(np.array([np.nan, np.uint32(0x7f800001).view(np.float32)], np.float32))
    assert ((nan & 0x7f80) == 0x7f80).all() and ((nan & 0x7f) != 0).all()


def test_large_tensors_begin_with_a_cache_line():
    """Wherever the arena stands, and give back what that skipped; small ones follow one another."""
    rt = N.runtime()
    base = rt.mirage_arena_offset()
    for before in (1, 8, 9, 100, 1000):
        g = G.KNGraph()
        g.new_input((before,), G.DT_INT32)
        small = g.new_input((3, 5), G.DT_BFLOAT16)
        large = g.new_input((1 << 19,), G.DT_BFLOAT16)
        assert large.device_ptr(False) % 256 == 0 and 0 <= large.device_ptr(False) - small.device_ptr(False) < 1024
        at = rt.mirage_arena_offset()
        other = g.new_input((1 << 10, 1 << 10), G.DT_FLOAT32)
        assert other.device_ptr(False) % 256 == 0
        g.pop_operator()
        assert rt.mirage_arena_offset() == at
        g.close()
        assert rt.mirage_arena_offset() == base


def test_layout_search_leaves_their_tensors_row_major(g):
    """Whatever a cost says of column-major ones; the tensors of other operators are searched as before."""
    x, y = g.new_input((4, 2, 64)), g.new_input((4, 64))
    g.rotary(g.exp(x), g.new_input((4,), I32), g.new_input((2, 32), F64))
    g.exp(y)
    found = G.optimize_layout(g, lambda op, layouts: 1.0 + sum(1.0 for l in layouts if l == 100))
    layouts = [[t.layout for t in g.outputs(i)] for i in range(g.num_operators)]
    assert layouts == [[101], [101], [100], [100], [100], [100], [101]] and found["assignments"] == 8
