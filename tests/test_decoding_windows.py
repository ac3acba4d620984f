"""Windows that no int holds: longer than any cache, so no window; never a short one by chance."""
import json

import pytest

from attention_superoptimizer_amd import graph as G


@pytest.fixture
def g():
    graph = G.KNGraph()
    yield graph
    graph.close()


def _tensors(g):
    return [g.new_input((6, 8, 64)), g.new_input((7, 16, 2, 64)), g.new_input((7, 16, 2, 64)), g.new_input((3, 5), G.DT_INT32),
            g.new_input((3,), G.DT_INT32)]


@pytest.mark.parametrize("window,kept", [(0, 0), (7, 7), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 32, 2 ** 31 - 1),
                                         (2 ** 32 + 5, 2 ** 31 - 1), (2 ** 70, 2 ** 31 - 1)])
def test_long_windows(g, window, kept):
    g.paged_attention(*_tensors(g), window=window)
    said = json.loads(g.to_json())
    assert said[-1]["window"] == kept


@pytest.mark.parametrize("window", [-1, -2 ** 31, -2 ** 32, -2 ** 32 + 5])
def test_windows_below_zero_are_refused(g, window):
    with pytest.raises(G.InfeasibleOperator):
        g.paged_attention(*_tensors(g), window=window)


@pytest.mark.parametrize("window,kept", [(2 ** 32 + 5, 2 ** 31 - 1), (-2 ** 32 + 5, None)])
def test_of_the_wire_format(g, window, kept):
    g.paged_attention(*_tensors(g), window=7)
    said = json.loads(g.to_json())
    said[-1]["window"] = window
    if kept is None:
        with pytest.raises(ValueError):
            G.KNGraph.from_json(said)
    else:
        again = G.KNGraph.from_json(said)
        try:
            assert json.loads(again.to_json())[-1]["window"] == kept
        finally:
            again.close()
