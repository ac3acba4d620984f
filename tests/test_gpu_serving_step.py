"""The operators of serving in a row, as a program runs them: prompts of any lengths appended and attended within a window, steps of
single tokens, and steps of drafted trees, each step's logits with their probabilities.  Every operator against its formula in 64
bits on what the one before it left."""
import numpy as np
import pytest

from decoding_reference import check, normal, rotary_bound, turned
from serving_reference import G, attended, log_probabilities, put, read, tree_seen, window_seen

pytestmark = pytest.mark.gpu

KIND, Q_HEADS, KV_HEADS, HEAD, PAGE, PAGES, HIDDEN, VOCABULARY = "fp16", 6, 2, 64, 16, 40, 96, 701


class _Layer:
    """Projection, rotary positions with the append, attention, logits and their probabilities, of `rows` tokens."""

    def __init__(self, g, rows, k, v, angles, weights, sequences, width, attend, top):
        self.x = g.new_input((rows, HIDDEN))
        qkv = g.matmul(self.x, weights[0])
        self.qkv, self.rows = qkv, rows
        self.positions, self.slots = g.new_input((rows,), G.DT_INT32), g.new_input((rows,), G.DT_INT32)
        self.q = g.rotary_append(qkv, self.positions, angles, self.slots, k, v)
        self.table, self.lengths = g.new_input((sequences, width), G.DT_INT32), g.new_input((sequences,), G.DT_INT32)
        self.o = attend(self.q, k, v, self.table, self.lengths)
        self.logits = g.matmul(self.o, weights[1])
        self.tokens = g.new_input((rows,), G.DT_INT32)
        self.answers = g.log_probabilities(self.logits, self.tokens, top=top, scale=0.8)
        self.k, self.v, self.angles, self.top = k, v, angles, top

    def run(self, g, rng, table, lengths, positions, places, seen_of, rows_of):
        """places: (sequence, place) of every row; seen_of(sequence) -> [its rows, keys]."""
        slots = np.array([table[b, p // PAGE] * PAGE + p % PAGE for b, p in places], np.int32)
        tokens = rng.integers(0, VOCABULARY, self.rows).astype(np.int32)
        for t, a in ((self.x, normal(rng, (self.rows, HIDDEN), KIND)), (self.positions, positions), (self.slots, slots), (self.table, table),
                     (self.lengths, lengths), (self.tokens, tokens)):
            t.write_data(np.asarray(a))
        g.execute_all()
        qkv = read(self.qkv).reshape(self.rows, Q_HEADS + 2 * KV_HEADS, HEAD)
        turned_heads, parts = turned(qkv[:, :Q_HEADS + KV_HEADS], positions, read(self.angles), False)
        bound = rotary_bound(turned_heads, parts, KIND)
        q = read(self.q).reshape(self.rows, Q_HEADS, HEAD)
        check(q, turned_heads[:, :Q_HEADS], bound[:, :Q_HEADS], "q")
        k, v = (read(c).reshape(PAGES * PAGE, KV_HEADS, HEAD) for c in (self.k, self.v))
        check(k[slots], turned_heads[:, Q_HEADS:], bound[:, Q_HEADS:], "k")
        np.testing.assert_array_equal(v[slots], qkv[:, Q_HEADS + KV_HEADS:])
        o = read(self.o).reshape(self.rows, Q_HEADS, HEAD)
        for b in range(len(lengths)):
            at = [table[b, p // PAGE] * PAGE + p % PAGE for p in range(lengths[b])]
            want, off = attended(q[rows_of(b)], k[at], v[at], seen_of(b), float(np.float32(HEAD ** -0.5)), KIND)
            check(o[rows_of(b)], want, off, "o")
        logits = read(self.logits)
        *want, bounds = log_probabilities(logits, tokens[:, None], self.top, float(np.float32(0.8)))
        check(read(self.answers[0]), want[0][:, 0], bounds[0][:, 0], "log probabilities")
        check(read(self.answers[1]), want[1], bounds[1], "entropy")
        check(read(self.answers[2]), want[2], bounds[2], "top")
        np.testing.assert_array_equal(self.answers[3].read_data(), want[3])


def test_prompts_steps_and_trees(rt):
    rng = np.random.default_rng(4)
    window, sinks, width, nodes = 30, 3, 10, 7
    g, inner = G.KNGraph(), []
    try:
        k, v = (put(g, np.zeros((PAGES, PAGE, KV_HEADS, HEAD)), KIND) for _ in range(2))
        angles = put(g, G.rotary_angles(HEAD))
        weights = [put(g, normal(rng, dims, KIND, 0.1), KIND) for dims in ((HIDDEN, (Q_HEADS + 2 * KV_HEADS) * HEAD), (Q_HEADS * HEAD, VOCABULARY))]
        order = rng.permutation(PAGES)
        table = np.stack([order[10 * b:10 * b + 10] for b in range(3)]).astype(np.int32)
        lengths = np.array([45, 1, 80], np.int32)

        # the prompts, all at once, ragged
        p = G.KNGraph()
        inner.append(p)
        begin = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        starts = put(p, begin)
        layer = _Layer(p, int(begin[-1]), k, v, angles, weights, 3, width,
                       lambda q, *c: p.window_attention(q, *c, window, sinks, starts), 5)
        places = [(b, j) for b in range(3) for j in range(lengths[b])]
        layer.run(p, rng, table, lengths, np.array([j for _, j in places], np.int32), places,
                  lambda b: window_seen(lengths[b], lengths[b], window, sinks), lambda b: slice(begin[b], begin[b + 1]))
        inner.pop().close()

        # a token of every sequence
        step = G.KNGraph()
        inner.append(step)
        layer = _Layer(step, 3, k, v, angles, weights, 3, width, lambda q, *c: step.window_attention(q, *c, window, sinks), 20)
        for _ in range(5):
            lengths = lengths + 1
            layer.run(step, rng, table, lengths, lengths - 1, [(b, int(lengths[b]) - 1) for b in range(3)],
                      lambda b: window_seen(lengths[b], 1, window, sinks), lambda b: slice(b, b + 1))
        inner.pop().close()

        # trees of seven drafts, one of them shorter; a path of two is kept, by the rows of its nodes appended again behind the context
        tree = G.KNGraph()
        inner.append(tree)
        parents = np.array([[-1, 0, 0, 1, 3, 2, -1], [-1, -1, 1, 2, -2, -2, -2], [-1, 0, 1, 2, 3, 4, 5]], np.int32)
        tp = put(tree, parents)
        layer = _Layer(tree, 3 * nodes, k, v, angles, weights, 3, width, lambda q, *c: tree.tree_attention(q, *c, tp), 1)
        depth = np.zeros_like(parents)
        for i in range(nodes):
            depth[:, i] = np.where(parents[:, i] >= 0, depth[np.arange(3), np.maximum(parents[:, i], 0)] + 1, 0)
        for _ in range(3):
            drafted = lengths + nodes
            layer.run(tree, rng, table, drafted, (lengths[:, None] + depth).reshape(-1).astype(np.int32),
                      [(b, int(lengths[b]) + i) for b in range(3) for i in range(nodes)],
                      lambda b: tree_seen(int(drafted[b]), parents[b]), lambda b: slice(b * nodes, (b + 1) * nodes))
            lengths = lengths + 2
        # operator by operator: the same
        once = [t.read_data() for t in (layer.o, *layer.answers)]
        for i in range(tree.num_operators):
            tree.execute(i)
        for t, w in zip((layer.o, *layer.answers), once):
            np.testing.assert_array_equal(t.read_data(), w)
        total, each = tree.profile_all()  # inputs of such a graph keep their values
        assert each[-1] > 0 and total >= each[-1]
        np.testing.assert_array_equal(tp.read_data(), parents)
        np.testing.assert_array_equal(layer.o.read_data(), once[0])
    finally:
        for graph in reversed(inner):
            graph.close()
        g.close()
