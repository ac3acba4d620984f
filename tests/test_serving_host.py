"""tree_attention, window_attention and log_probabilities without a device: the tensors they take and refuse, their wire format, and the
C ABI before mi355_init."""
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


def _inputs(g, change):
    cache, index, kind = change.get("cache", (7, 16, 2, 64)), change.get("index", I32), change.get("kind", F16)
    q = g.new_input(change.get("q", (6, 8, 64)), kind)
    k, v = (g.new_input(cache, change.get("cache_kind", kind)) for _ in range(2))
    return q, k, v, g.new_input(change.get("table", (3, 5)), index), g.new_input(change.get("lengths", (3,)), index)


def test_shapes_of_results(g):
    for kind in (F16, BF16):
        x = _inputs(g, dict(kind=kind))
        parents, starts = g.new_input((3, 2), I32), g.new_input((4,), I32)
        for y in (g.tree_attention(*x, parents), g.window_attention(*x, 8), g.window_attention(*x, 8, 2, starts), g.window_attention(*x, 0)):
            assert y.dims == (6, 8, 64) and y.data_type == kind
        flat = (g.new_input((6, 512), kind), *x[1:])
        assert g.tree_attention(*flat, parents).dims == g.window_attention(*flat, 8).dims == (6, 512)
        assert g.window_attention(g.new_input((7, 8, 64), kind), *x[1:], 8, starts=starts).dims == (7, 8, 64)
    first = [g.new_input((7, 2, 16, 64)) for _ in range(2)]
    x = _inputs(g, {})
    assert g.window_attention(x[0], *first, *x[3:], 8, heads_first=True).dims == (6, 8, 64)
    for kind in (F16, BF16, F32):
        logits, tokens = g.new_input((6, 100), kind), g.new_input((6,), I32)
        assert [t.dims for t in g.log_probabilities(logits, tokens)] == [(6,), (6,)]
        outs = g.log_probabilities(g.new_input((2, 3, 100), kind), g.new_input((6, 4), I32), top=9, scale=0.5)
        assert [t.dims for t in outs] == [(6, 4), (6,), (6, 9), (6, 9)] and [t.data_type for t in outs] == [F32, F32, F32, I32]


_BAD_CACHES = [
    dict(q=(6, 9, 64)), dict(q=(6, 8, 72)), dict(q=(6, 65)), dict(kind=BF16, cache_kind=F16), dict(kind=F32), dict(cache=(7, 16, 2, 60), q=(6, 8, 60)),
    dict(cache=(7, 16, 2, 264), q=(6, 8, 264)), dict(cache=(7, 16, 128)), dict(table=(3,)), dict(lengths=(2,)), dict(index=F32), dict(scale=math.inf),
    dict(scale=math.nan), dict(table=(3, 1 << 27)),
]


@pytest.mark.parametrize("change", _BAD_CACHES + [dict(q=(7, 8, 64)), dict(table=(4, 5)), dict(parents=(3, 3)), dict(parents=(2, 3)), dict(parents=(6,)),
                                                  dict(parent_kind=F32), dict(parents=(1, 1025), q=(1025, 8, 64), table=(1, 5), lengths=(1,))])
def test_tree_attention_refuses(g, change):
    x = _inputs(g, change)
    parents = g.new_input(change.get("parents", (3, 2)), change.get("parent_kind", I32))
    operators = g.num_operators
    with pytest.raises(G.InfeasibleOperator):
        g.tree_attention(*x, parents, scale=change.get("scale", 0.125))
    assert g.num_operators == operators


@pytest.mark.parametrize("change", _BAD_CACHES + [dict(q=(7, 8, 64)), dict(table=(4, 5), lengths=(4,)), dict(starts=(3,)), dict(starts=(4, 1)),
                                                  dict(starts=(4,), start_kind=F32), dict(window=-1), dict(sinks=-1), dict(window=-2 ** 40)])
def test_window_attention_refuses(g, change):
    x = _inputs(g, change)
    starts = g.new_input(change["starts"], change.get("start_kind", I32)) if "starts" in change else None
    with pytest.raises(G.InfeasibleOperator):
        g.window_attention(*x, change.get("window", 8), change.get("sinks", 1), starts, scale=change.get("scale", 0.125))


def test_windows_that_no_int_holds(g):
    x = _inputs(g, {})
    g.window_attention(*x, 2 ** 40, 2 ** 33)
    said = json.loads(g.to_json())[-1]
    assert said["window"] == said["sinks"] == 2 ** 31 - 1


@pytest.mark.parametrize("change", [dict(logits=(6,)), dict(logits=(5, 100)), dict(logits=(1, 2, 3, 100)), dict(kind=F64), dict(kind=I32), dict(tokens=(5,)),
                                    dict(tokens=(6, 1, 1)), dict(index=F32), dict(top=-1), dict(top=65), dict(top=2 ** 32 + 1), dict(scale=0.0),
                                    dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(layout="DmemColumnMajor")])
def test_log_probabilities_refuses(g, change):
    logits = g.new_input(change.get("logits", (6, 100)), change.get("kind", F32), change.get("layout", "DmemRowMajor"))
    tokens = g.new_input(change.get("tokens", (6,)), change.get("index", I32))
    with pytest.raises(G.InfeasibleOperator):
        g.log_probabilities(logits, tokens, change.get("top", 3), change.get("scale", 1.0))


def test_wire_format(g):
    x = _inputs(g, dict(kind=BF16))
    g.tree_attention(*x, g.new_input((3, 2), I32), scale=0.37)
    y = g.window_attention(*x, 9, 3)
    g.window_attention(y, *x[1:], 0, starts=g.new_input((4,), I32))
    logits, tokens = g.new_input((6, 100), F32), g.new_input((6, 2), I32)
    g.log_probabilities(logits, tokens, 4, 0.7)
    g.log_probabilities(logits, tokens)
    said = json.loads(g.to_json())
    ops = [o for o in said if o["op_type"] != "kn_input_op"]
    assert [o["op_type"] for o in ops] == ["kn_tree_attention_op"] + ["kn_window_attention_op"] * 2 + ["kn_log_probabilities_op"] * 2
    assert np.float32(ops[0]["scale"]) == np.float32(0.37) and (ops[1]["window"], ops[1]["sinks"]) == (9, 3)
    assert len(ops[1]["input_tensors"]) == 5 and len(ops[2]["input_tensors"]) == 6
    assert ops[3]["top"] == 4 and np.float32(ops[3]["scale"]) == np.float32(0.7) and len(ops[3]["output_tensors"]) == 4
    again = G.KNGraph.from_json(said)
    try:
        back = json.loads(again.to_json())
        for o in said + back:
            for t in o["input_tensors"] + o["output_tensors"]:
                del t["guid"]
        assert back == said
    finally:
        again.close()
    for o in said:
        for t in o["input_tensors"] + o["output_tensors"]:
            t["guid"] = 0
    ops[3]["top"] = 99
    with pytest.raises(ValueError):
        G.KNGraph.from_json(said)


def test_no_fingerprints(g, capfd):
    g.log_probabilities(g.new_input((6, 100), F32), g.new_input((6,), I32))
    with pytest.raises(AssertionError):
        g.fingerprint_seeded(1)
    assert "kn_log_probabilities_op has no fingerprint" in capfd.readouterr().err


def test_popped_operators_leave_the_arena(g):
    x = _inputs(g, {})
    at = N.runtime().mirage_arena_offset()
    g.window_attention(*x, 9)
    g.pop_operator()
    assert N.runtime().mirage_arena_offset() == at
    logits, tokens = g.new_input((6, 100), F32), g.new_input((6,), I32)
    inner = N.runtime().mirage_arena_offset()
    g.log_probabilities(logits, tokens, 5)
    g.pop_operator()
    assert N.runtime().mirage_arena_offset() == inner


def test_abi_before_init():
    if N.backend().mi355_is_initialised():
        pytest.skip("a device is attached")
    cache = ctypes.byref(N.Mi355PagedCache())
    assert N.backend().mi355_tree_attention(None, 0, None, 0, cache, None, 1, None, None, 1, 1, 1, 1.0) == -5
    assert N.backend().mi355_window_attention(None, 0, None, 0, cache, None, 1, None, None, 1, 1, 1, 1.0, 0, 0) == -5
    assert N.backend().mi355_log_probabilities(None, 0, None, None, None, None, None, 1, 1, 1, 1, 1.0, 930) == -5
