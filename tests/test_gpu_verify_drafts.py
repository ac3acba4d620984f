"""verify_drafts against its definition in 64 bits: drafts with and without probabilities, padded ones, borders that are
met exactly, weights that vanish, vocabularies of any size, every type."""
import numpy as np
import pytest

from attention_superoptimizer_amd import _native as N
from attention_superoptimizer_amd import graph as G
from decoding_reference import put, rounded, verified

pytestmark = pytest.mark.gpu


def _run(target, draft, tokens, uniforms, kind, flat=False):
    g = G.KNGraph()
    try:
        v = target.shape[-1]
        shape = (lambda a: a.reshape(-1, v)) if flat else (lambda a: a)
        n, out = g.verify_drafts(put(g, shape(target), kind), None if draft is None else put(g, shape(draft), kind),
                                 put(g, tokens.astype(np.int32)), put(g, uniforms.astype(np.float32)))
        for _ in range(2):
            n.write_data(np.full(n.dims, 99))
            out.write_data(np.full(out.dims, 99))
            g.execute_all()
        return n.read_data(), out.read_data()
    finally:
        g.close()


def _check(target, draft, tokens, uniforms, kind, flat=False):
    uniforms = uniforms.astype(np.float32)
    got, want = _run(target, draft, tokens, uniforms, kind, flat), verified(target, draft, tokens, uniforms)
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)
    return got


def _probabilities(rng, dims, kind, peak=2.0):
    x = np.exp(rng.standard_normal(dims) * peak)
    return rounded(x / x.sum(-1, keepdims=True), kind)


def _case(seed, sequences, drafts, vocabulary, kind, certain=False):
    rng = np.random.default_rng(seed)
    logits = rng.standard_normal((sequences, drafts + 1, vocabulary)) * 2
    target = np.exp(logits) / np.exp(logits).sum(-1, keepdims=True)
    near = np.exp(logits[:, :drafts] + rng.standard_normal((sequences, drafts, vocabulary)) * 0.4)
    draft = near / near.sum(-1, keepdims=True)
    tokens = (draft / rng.exponential(size=draft.shape)).argmax(-1)
    if certain:  # likely enough that some stay
        tokens = np.where(rng.random(tokens.shape) < 0.7, target[:, :drafts].argmax(-1), tokens)
    return rounded(target, kind), None if certain else rounded(draft, kind), tokens.astype(np.int32), rng.random((sequences, drafts + 1))


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("sequences,drafts,vocabulary", [(1, 1, 1), (3, 2, 2), (5, 4, 100), (70, 3, 257), (2, 6, 4096), (4, 3, 5001), (1, 4, 32000),
                                                         (9, 5, 50021), (2, 300, 17)])
def test_verify(rt, kind, certain, sequences, drafts, vocabulary):
    accepted, _ = _check(*_case(sequences + vocabulary, sequences, drafts, vocabulary, kind, certain), kind, flat=certain)
    if sequences >= 5 and not certain:
        assert len(set(accepted.tolist())) > 1  # (the case exercises more than one outcome)


@pytest.mark.parametrize("certain", [False, True])
def test_padded_drafts_end_a_sequence(rt, certain):
    target, draft, tokens, u = _case(3, 12, 4, 500, "fp32", certain)
    tokens = target[:, :4].argmax(-1).astype(np.int32)
    u[:, :4] = 0.0
    for b in range(12):
        tokens[b, b % 5:] = [-1, -2147483648, 500, 2147483647][b % 4]
    accepted, _ = _check(target, draft, tokens, u, "fp32")
    np.testing.assert_array_equal(accepted, np.arange(12) % 5)


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
def test_borders_that_are_met_exactly(rt, kind):
    """Equal weights of 1/64 and uniforms that are multiples of it: the share is passed, not met.  And u q = p refuses."""
    v, rows = 64, 65
    target = np.full((rows, 2, v), 1 / 64)
    draft = np.full((rows, 1, v), 1 / 32)
    tokens = np.arange(rows, dtype=np.int32)[:, None] % v
    u = np.zeros((rows, 2))
    u[:, 0] = 0.5 - 2.0 ** -25
    u[::2, 0] = 0.5
    u[:, 1] = np.minimum(np.arange(rows) / 64, 63 / 64)
    accepted, out = _check(target, draft, tokens, u, kind)
    np.testing.assert_array_equal(accepted, np.arange(rows) % 2)
    taken = accepted == 1
    np.testing.assert_array_equal(out[taken, 1], np.minimum(np.arange(rows), 63)[taken])


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocabulary", [300, 5000, 40000])
def test_weights_that_vanish(rt, kind, vocabulary):
    rng = np.random.default_rng(vocabulary)
    target = np.zeros((8, 2, vocabulary))
    draft = np.zeros((8, 1, vocabulary))
    tokens = np.full((8, 1), 7, np.int32)
    u = np.full((8, 2), 0.5)
    target[0], draft[0] = 0.0, 0.0                                  # nothing at all: -1
    target[1, 0, 11], draft[1, 0] = 0.25, 1.0                       # refused, no difference left: from the target
    target[2, 0, vocabulary - 1], target[2, 0, 7], draft[2, 0, 7] = 0.5, 0.25, 1.0  # the last index
    target[3, 0, 0], draft[3, 0, 7], u[3, 1] = 0.5, 1.0, 0.0        # the first
    target[4, 0, [5, 200]], draft[4, 0, 7], u[4, 1] = 0.5, 1.0, 0.0  # a share of nothing: the first with a weight
    target[5, 0, [5, 200]], draft[5, 0, 7], u[5, 1] = 0.5, 1.0, 1.0  # all of it: the last with a weight
    target[6, 0, 7], draft[6, 0, 7], target[6, 1, 9] = 0.5, 0.5, 1.0  # taken
    target[7, 0], draft[7, 0] = _probabilities(rng, (vocabulary,), kind), 0.0
    target[7, 0, 7] = 0.0                                           # 0 < 0 refuses
    accepted, out = _check(rounded(target, kind), draft, tokens, u, kind)
    assert out[:7, 0].tolist() == [-1, 11, vocabulary - 1, 0, 5, 200, 7] and out[6, 1] == 9
    certain, _ = _check(rounded(target, kind), None, tokens, u, kind)
    assert certain.tolist() == [0, 0, 0, 0, 0, 0, 0, 0]


@pytest.mark.parametrize("kind", ["fp16", "fp32"])
def test_a_certain_draft_that_has_all_the_weight(rt, kind):
    """Refused though nothing else has a weight: drawn again from the target."""
    target = np.zeros((1, 2, 50))
    target[0, 0, 3] = 0.5
    _, out = _check(target, None, np.array([[3]], np.int32), np.array([[0.75, 0.2]]), kind)
    assert out.tolist() == [[3, -1]]


def test_nan_weighs_nothing(rt):
    target, draft, tokens, u = _case(8, 6, 2, 900, "fp32")
    clean = [target.copy(), draft.copy()]
    target[:, :, ::7], clean[0][:, :, ::7] = np.nan, 0.0
    draft[:, :, 3::7], clean[1][:, :, 3::7] = np.nan, 2.0  # (a difference with it is below zero, a share of it above)
    tokens[:] = 3
    want = verified(clean[0], clean[1], tokens, u.astype(np.float32))
    got = _run(target, draft, tokens, u, "fp32")
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("u", [np.nan, -1.0, 1.5, np.inf, -np.inf])
def test_numbers_that_are_no_uniforms(rt, u):
    """Whatever the last number is, the token is one with a weight."""
    target, draft, tokens, uniforms = _case(4, 5, 2, 3001, "fp32")
    target[:, :, :5] = target[:, :, -5:] = 0.0
    uniforms[:, 2] = u
    accepted, out = _run(target, draft, tokens, uniforms, "fp32")
    for b in range(5):
        assert 0 <= out[b, accepted[b]] < 3001 and target[b, accepted[b], out[b, accepted[b]]] > 0


def test_refusals(rt, abi):
    g = G.KNGraph()
    try:
        p, t = put(g, np.zeros(512, np.float32)).device_ptr(False), put(g, np.zeros(64, np.int32)).device_ptr(False)
        o = put(g, np.zeros(64, np.int32)).device_ptr(False)
        good = [p, p, t, p, o, o + 64, 2, 2, 50, 930]
        assert abi.mi355_verify_drafts(*good) == 0
        assert abi.mi355_verify_drafts(p, None, None, p, o, o + 64, 2, 0, 50, 930) == 0  # no drafts: drawn from the target
        assert abi.mi355_verify_drafts(*[0 if n == 6 else x for n, x in enumerate(good)]) == 0
        for place, value, code in ((0, None, -3), (2, None, -3), (3, None, -3), (4, None, -3), (5, None, -3), (6, -1, -3), (7, -1, -3),
                                   (8, 0, -3), (9, 940, -4)):
            assert abi.mi355_verify_drafts(*[value if n == place else x for n, x in enumerate(good)]) == code, (place, N.last_error())
    finally:
        g.close()
