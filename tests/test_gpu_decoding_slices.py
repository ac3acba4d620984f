"""Batches of the operators of a decoding step that go in more than one launch."""
import numpy as np
import pytest

from attention_superoptimizer_amd import graph as G
from decoding_reference import attention, check, normal, put, read, verified

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,new,window", [("fp16", 1, 0), ("bf16", 3, 100)])
def test_sequences_of_tables_that_fill_a_launch(rt, kind, new, window):
    """A table that names 2^30 keys has 2^23 units a head: 127 sequences go in a launch, and 127, 127 and 6 here.  They
    name one page each, of which they have a few keys."""
    sequences, size, width, head = 260, 65536, 16384, 8
    rng = np.random.default_rng(new)
    lengths = [int(n) for n in rng.integers(0, 300, sequences)]
    q = normal(rng, (sequences, new, 2, head), kind)
    k, v = (np.full((3, size, 1, head), np.nan) for _ in range(2))
    for c in (k, v):
        c[:, :300] = normal(rng, (3, 300, 1, head), kind)
    table = np.full((sequences, width), -1, np.int32)
    table[:, 0] = rng.integers(0, 3, sequences)
    lengths = np.array(lengths, np.int32)
    want, bound = attention(q, k[:, :300], v[:, :300], table[:, :1], lengths, 0.125, window, kind)  # (pages of 300: none is longer)
    g = G.KNGraph()
    try:
        o = g.paged_attention(put(g, q.reshape(-1, 2, head), kind), put(g, k, kind), put(g, v, kind), put(g, table),
                              put(g, lengths), scale=0.125, window=window)
        o.write_data(np.full(o.dims, 7.0))
        g.execute_all()
        check(read(o).reshape(q.shape), want, bound)
    finally:
        g.close()


@pytest.mark.parametrize("kind", ["fp16", "fp32"])
@pytest.mark.parametrize("sequences,drafts,vocabulary", [(4097, 2, 700), (5000, 1, 3001), (65536, 1, 40), (66000, 2, 17)])
@pytest.mark.parametrize("certain", [False, True])
def test_verifications_of_thousands_of_sequences(rt, kind, sequences, drafts, vocabulary, certain):
    """More than 4096 have a workgroup each, and more than 65535 go in several launches."""
    rng = np.random.default_rng(sequences + drafts)
    p = rng.random((sequences, drafts + 1, vocabulary)).astype(np.float32) ** 4
    p /= p.sum(-1, keepdims=True)
    p = p.astype(np.float16 if kind == "fp16" else np.float32)
    q = None
    if not certain:
        q = rng.random((sequences, drafts, vocabulary)).astype(np.float32) ** 4
        q = (q / q.sum(-1, keepdims=True)).astype(p.dtype)
    tokens = rng.integers(-1, vocabulary, (sequences, drafts)).astype(np.int32)
    u = rng.random((sequences, drafts + 1)).astype(np.float32)
    if certain:
        u[:, :drafts] *= 4.0 / vocabulary
    g = G.KNGraph()
    try:
        accepted, out = g.verify_drafts(put(g, p, kind), None if q is None else put(g, q, kind), put(g, tokens), put(g, u))
        for t in (accepted, out):
            t.write_data(np.full(t.dims, -7))
        g.execute_all()
        want = verified(p.astype(np.float64), None if q is None else q.astype(np.float64), tokens, u)
        np.testing.assert_array_equal(accepted.read_data(), want[0])
        np.testing.assert_array_equal(out.read_data(), want[1])
        assert 0 < want[0].sum() < sequences * drafts
    finally:
        g.close()
