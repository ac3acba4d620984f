"""Profiling a graph with operators of a decoding step: its inputs, the caches among them, are what they were."""
import numpy as np
import pytest

from attention_superoptimizer_amd import graph as G
from decoding_reference import normal, put, read

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_a_profile_keeps_the_caches(rt, kind):
    rng = np.random.default_rng(1)
    g = G.KNGraph()
    try:
        k, v = (put(g, normal(rng, (4, 16, 2, 64), kind), kind) for _ in range(2))
        qkv = put(g, normal(rng, (2, 8, 64), kind), kind)
        positions, slots = put(g, np.array([19, 31], np.int32)), put(g, np.array([3, 63], np.int32))
        angles = put(g, G.rotary_angles(64))
        table, lengths = put(g, np.array([[2, 0], [1, 3]], np.int32)), put(g, np.array([20, 32], np.int32))
        q = g.rotary_append(qkv, positions, angles, slots, k, v)
        o = g.paged_attention(q, k, v, table, lengths)
        g.execute_all()
        kept = [qkv, k, v, positions, slots, angles, table, lengths, q, o]
        want = [read(t) for t in kept]
        total, each = g.profile_all()
        assert len(each) == g.num_operators and min(each[-2:]) > 0
        assert abs(total - sum(each[-2:])) <= 2.0 ** -24 * total  # (one addition in 32 bits: off by half a step of its result at most)
        for t, w in zip(kept, want):
            np.testing.assert_array_equal(read(t), w)
        for i in range(g.num_operators):
            assert g.profile(i) >= 0.0
        for t, w in zip(kept, want):
            np.testing.assert_array_equal(read(t), w)
    finally:
        g.close()


def test_a_serving_graph_keeps_its_weights_too(rt):
    """The keys that a profile's passes write come from the activations and the weights."""
    rng = np.random.default_rng(2)
    g = G.KNGraph()
    try:
        x, w = put(g, normal(rng, (2, 32), "fp16"), "fp16"), put(g, normal(rng, (32, 8 * 64), "fp16", 0.2), "fp16")
        k, v = (put(g, normal(rng, (4, 16, 2, 64), "fp16"), "fp16") for _ in range(2))
        positions, slots = put(g, np.array([19, 31], np.int32)), put(g, np.array([3, 63], np.int32))
        g.rotary_append(g.matmul(x, w), positions, put(g, G.rotary_angles(64)), slots, k, v)
        g.execute_all()
        want = [read(t) for t in (x, w, k, v)]
        g.profile_all()
        for t, a in zip((x, w, k, v), want):
            np.testing.assert_array_equal(read(t), a)
    finally:
        g.close()


def test_other_graphs_are_filled_as_before(rt):
    g = G.KNGraph()
    try:
        x = put(g, np.full((4, 64), 7.0), "fp16")
        g.exp(x)
        g.profile_all()
        assert (read(x) != 7.0).any()
    finally:
        g.close()


def test_a_layout_search_keeps_them_too(rt):
    rng = np.random.default_rng(3)
    g = G.KNGraph()
    try:
        x = put(g, normal(rng, (4, 2, 64), "fp16"), "fp16")
        y = g.rotary(x, put(g, np.arange(4, dtype=np.int32)), put(g, G.rotary_angles(64)))
        g.execute_all()
        want = [read(t) for t in (x, y)]
        G.optimize_layout(g)
        for t, a in zip((x, y), want):
            np.testing.assert_array_equal(read(t), a)
    finally:
        g.close()
