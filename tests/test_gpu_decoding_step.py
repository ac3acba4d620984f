"""The operators of a decoding step as a serving loop runs them, in one graph with the matmuls around them: a prompt is
written into the cache page by page, then drafted tokens are decoded and verified, step after step on the same graphs."""
import numpy as np
import pytest

from attention_superoptimizer_amd import graph as G
from decoding_reference import attention, check, normal, put, read, rotary_bound, turned, verified

pytestmark = pytest.mark.gpu
KIND, HIDDEN, Q_HEADS, KV_HEADS, HEAD, PAGE, PAGES, VOCABULARY = "fp16", 192, 6, 2, 64, 16, 24, 700


class _Layer:
    """qkv = x W; q = rotary_append(qkv); o = paged_attention(q); y = o Wo, for `new` tokens of each of `sequences`."""

    def __init__(self, g, sequences, new, k, v, angles, weights, width):
        tokens = sequences * new
        self.sequences, self.new = sequences, new
        self.x = g.new_input((tokens, HIDDEN))
        self.positions, self.slots = (g.new_input((tokens,), G.DT_INT32) for _ in range(2))
        self.table, self.lengths = g.new_input((sequences, width), G.DT_INT32), g.new_input((sequences,), G.DT_INT32)
        self.qkv = g.matmul(self.x, weights[0])
        self.q = g.rotary_append(self.qkv, self.positions, angles, self.slots, k, v)
        self.o = g.paged_attention(self.q, k, v, self.table, self.lengths, window=40)
        self.y = g.matmul(self.o, weights[1])


def test_prompt_then_drafts(rt):
    rng = np.random.default_rng(1)
    sequences, drafts, width = 3, 2, 6
    prompt = [37, 16, 5]
    g = G.KNGraph()
    inner = []
    try:
        k, v = (g.new_input((PAGES, PAGE, KV_HEADS, HEAD)) for _ in range(2))
        for c in (k, v):
            c.write_data(np.full(c.dims, np.nan))
        angles = G.rotary_angles(HEAD, factor=2.0, original_length=4096)
        a = put(g, angles)
        weights = [put(g, normal(rng, dims, KIND, 0.1), KIND) for dims in
                   ((HIDDEN, (Q_HEADS + 2 * KV_HEADS) * HEAD), (Q_HEADS * HEAD, HIDDEN), (HIDDEN, VOCABULARY))]
        table = rng.permutation(PAGES)[:sequences * width].reshape(sequences, width).astype(np.int32)

        def run(graph, layer, x, start):
            """One pass; positions start[b] .. start[b] + new - 1 of every sequence; checked stage by stage."""
            at = np.concatenate([np.arange(s, s + layer.new) for s in start]).astype(np.int32)
            which = np.repeat(np.arange(layer.sequences), layer.new)
            slots = table[which, at // PAGE] * PAGE + at % PAGE
            lengths = np.array(start, np.int32) + layer.new
            before = [read(c) for c in (k, v)]
            for t, data in ((layer.x, x), (layer.positions, at), (layer.slots, slots), (layer.table, table[:layer.sequences]),
                            (layer.lengths, lengths)):
                t.write_data(data)
            graph.execute_all()
            qkv = read(layer.qkv).reshape(len(at), -1, HEAD)
            want, parts = turned(qkv, at, angles, False)
            bound = rotary_bound(want, parts, KIND)
            check(read(layer.q).reshape(len(at), Q_HEADS, HEAD), want[:, :Q_HEADS], bound[:, :Q_HEADS], "q")
            after = [read(c) for c in (k, v)]
            for c, old in zip(after, before):  # other slots are what they were
                kept = np.ones(PAGES * PAGE, bool)
                kept[slots] = False
                np.testing.assert_array_equal(c.reshape(PAGES * PAGE, -1)[kept], old.reshape(PAGES * PAGE, -1)[kept])
            check(after[0].reshape(-1, KV_HEADS, HEAD)[slots], want[:, Q_HEADS:Q_HEADS + KV_HEADS], bound[:, Q_HEADS:Q_HEADS + KV_HEADS], "k")
            np.testing.assert_array_equal(after[1].reshape(-1, KV_HEADS, HEAD)[slots], qkv[:, Q_HEADS + KV_HEADS:])
            q = read(layer.q).reshape(layer.sequences, layer.new, Q_HEADS, HEAD)
            o, bound = attention(q, *after, table[:layer.sequences], lengths, float(np.float32(HEAD ** -0.5)), 40, KIND)
            check(read(layer.o).reshape(o.shape), o, bound, "o")
            assert np.isfinite(read(layer.y)).all()

        # the prompts, a sequence at a time: the whole of one is new
        for b, n in enumerate(prompt):
            p = G.KNGraph()
            inner.append(p)
            layer = _Layer(p, 1, n, k, v, a, weights, width)
            rows = table.copy()
            table[0] = rows[b]
            run(p, layer, normal(rng, (n, HIDDEN), KIND), [0])
            table[:] = rows
            inner.pop().close()

        # steps of all sequences together: a token and its drafts, verified by what the next layer would say of them
        step = G.KNGraph()
        inner.append(step)
        layer = _Layer(step, sequences, drafts + 1, k, v, a, weights, width)
        logits = step.matmul(layer.y, weights[2])
        e = step.exp(logits)
        target = step.div(e, step.reduction(e, 1))
        tokens, uniforms = step.new_input((sequences, drafts), G.DT_INT32), step.new_input((sequences, drafts + 1), G.DT_FLOAT32)
        accepted, out = step.verify_drafts(target, None, tokens, uniforms)
        lengths, outcomes = list(prompt), set()
        for _ in range(6):
            x = normal(rng, (sequences * (drafts + 1), HIDDEN), KIND)
            u = rng.random((sequences, drafts + 1)).astype(np.float32)
            u[:, :drafts] *= 2e-3  # (likelihoods of one token among 700)
            ids = rng.integers(0, VOCABULARY, (sequences, drafts)).astype(np.int32)
            ids[1, 1] = -1  # this sequence has one draft only
            tokens.write_data(ids)
            uniforms.write_data(u)
            run(step, layer, x, lengths)
            p = read(target).reshape(sequences, drafts + 1, VOCABULARY)
            np.testing.assert_allclose(p.sum(-1), 1.0, rtol=0.02)
            want = verified(p, None, ids, u)
            np.testing.assert_array_equal(accepted.read_data(), want[0])
            np.testing.assert_array_equal(out.read_data(), want[1])
            outcomes |= set(want[0].tolist())
            lengths = [n + 1 + int(taken) for n, taken in zip(lengths, want[0])]
        assert len(outcomes) > 1
        once = [t.read_data() for t in (layer.o, accepted, out)]
        for t in (layer.o, accepted, out):
            t.write_data(np.zeros(t.dims))
        for i in range(step.num_operators):  # operator by operator: the same
            step.execute(i)
        for t, w in zip((layer.o, accepted, out), once):
            np.testing.assert_array_equal(t.read_data(), w)
    finally:
        for graph in reversed(inner):
            graph.close()
        g.close()


def test_profile_leaves_tables_alone(rt):
    """The times of a graph's operators: inputs that are no fp16 values keep what was written, results are what a run gives."""
    rng = np.random.default_rng(2)
    g = G.KNGraph()
    try:
        k, v = (put(g, normal(rng, (4, 16, 2, 64), "bf16"), "bf16") for _ in range(2))
        q = put(g, normal(rng, (2, 4, 64), "bf16"), "bf16")
        table, lengths = put(g, np.array([[2, 0], [1, 3]], np.int32)), put(g, np.array([20, 32], np.int32))
        o = g.paged_attention(q, k, v, table, lengths)
        g.execute_all()
        want = read(o)
        total, each = g.profile_all()
        assert len(each) == g.num_operators and each[-1] > 0 and total >= each[-1]
        np.testing.assert_array_equal(table.read_data(), [[2, 0], [1, 3]])
        np.testing.assert_array_equal(read(o), want)
    finally:
        g.close()


def test_layout_search_keeps_rows_in_memory_order(rt):
    """The operators read and write row by row: a search has one choice for their tensors."""
    g = G.KNGraph()
    try:
        x = put(g, normal(np.random.default_rng(3), (4, 2, 64), "fp16"), "fp16")
        positions, angles = put(g, np.arange(4, dtype=np.int32)), put(g, G.rotary_angles(64))
        y = g.rotary(x, positions, angles)
        found = G.optimize_layout(g)
        assert found["assignments"] == 1 and found["unrunnable"] == 0 and {t.layout for t in (x, angles, y)} == {100}
    finally:
        g.close()
