"""Matmuls, element-wise operators, reductions and customized operators compute fp16 values: others are built (their fingerprints
know no type), and refused where their values would be computed."""
import pytest

from attention_superoptimizer_amd import graph as G
from attention_superoptimizer_amd import workloads as W

OTHERS = [G.DT_BFLOAT16, G.DT_FLOAT32, G.DT_DOUBLE, G.DT_INT32]


@pytest.fixture
def g():
    graph = G.KNGraph()
    yield graph
    graph.close()


def _operators(g, first, second):
    G.set_smem_budget(1 << 20)
    a, b = g.new_input((64, 64), first), g.new_input((64, 64), second)
    made = [lambda: g.matmul(a, b), lambda: g.add(a, b), lambda: g.mul(b, a), lambda: g.div(a, b)]
    if first == second:
        made += [lambda: g.exp(a), lambda: g.silu(a), lambda: g.reduction(a, 1, 4)]
    spec, _ = W.tiled_matmul(64, 64, 64, (1, 1, 1), 1, (0, -1, -1), (-1, 1, -1), (0, 1, -1))
    made.append(lambda: g.customized([a, b], spec[2]["plan"]))
    return made


@pytest.mark.parametrize("kind", OTHERS)
@pytest.mark.parametrize("mixed", [False, True])
def test_values_of_other_types_are_not_computed(g, capfd, kind, mixed):
    pairs = [(G.DT_FLOAT16, kind), (kind, G.DT_FLOAT16)] if mixed else [(kind, kind)]
    for first, second in pairs:
        for make in _operators(g, first, second):
            make()
            at = g.num_operators - 1
            capfd.readouterr()
            with pytest.raises(AssertionError):
                g.execute(at)
            assert "fp16" in capfd.readouterr().err
            with pytest.raises(AssertionError):
                g.execute_all()
            assert "fp16" in capfd.readouterr().err
            assert g.profile(at) == 1000.0  # milliseconds: what has no kernel
            g.pop_operator()


def test_the_operators_of_a_serving_step_name_what_is_missing(g, capfd):
    """bf16 activations and weights: the projection's product is the first that is refused."""
    x, w = g.new_input((2, 32), G.DT_BFLOAT16), g.new_input((32, 8 * 64), G.DT_BFLOAT16)
    k, v = (g.new_input((4, 16, 2, 64), G.DT_BFLOAT16) for _ in range(2))
    g.rotary_append(g.matmul(x, w), g.new_input((2,), G.DT_INT32), g.new_input((2, 32), G.DT_DOUBLE), g.new_input((2,), G.DT_INT32), k, v)
    with pytest.raises(AssertionError):
        g.execute_all()
    assert "kn_matmul_op" in capfd.readouterr().err


def test_programs_of_other_types_are_not_written(g, capfd, tmp_path):
    a, b = (g.new_input((64, 64), G.DT_BFLOAT16) for _ in range(2))
    spec, _ = W.tiled_matmul(64, 64, 64, (1, 1, 1), 1, (0, -1, -1), (-1, 1, -1), (0, 1, -1))
    g.customized([a, b], spec[2]["plan"])
    with pytest.raises(AssertionError):
        g.generate_hip_program(str(tmp_path / "p.hip"))
    assert "fp16" in capfd.readouterr().err and not (tmp_path / "p.hip").exists()
