"""log_probabilities against its formula in 64 bits: types, vocabularies of any size, numbers of tokens asked for and of top ones,
scales, equal logits, rows without a probability, values that are not finite, strides."""
import numpy as np
import pytest

from attention_superoptimizer_amd import _native as N
from decoding_reference import check, normal, rounded
from serving_reference import G, log_probabilities, put, read

pytestmark = pytest.mark.gpu


def _run(logits, tokens, top, scale, kind):
    g = G.KNGraph()
    try:
        outs = g.log_probabilities(put(g, logits, kind), put(g, tokens), top, scale)
        got = []
        for _ in range(2):
            for o in outs:
                o.write_data(np.full(o.dims, 77))
            g.execute_all()
            got.append([o.read_data() if i == 3 else read(o) for i, o in enumerate(outs)])
        for a, b in zip(*got):
            np.testing.assert_array_equal(a, b)
        return got[0]
    finally:
        g.close()


def _agree(got, want, bounds, tokens):
    logp, entropy, top_logp, top_tokens = want
    pairs = [(got[0].reshape(tokens.shape), logp, bounds[0]), (got[1], entropy, bounds[1])]
    if len(got) > 2:
        np.testing.assert_array_equal(got[3], top_tokens)
        pairs.append((got[2], top_logp, bounds[2]))
    for a, b, off in pairs:
        np.testing.assert_array_equal(np.isnan(a), np.isnan(b))
        np.testing.assert_array_equal(np.isinf(a), np.isinf(b))
        some = np.isfinite(b)
        np.testing.assert_array_equal(a[np.isinf(b)], b[np.isinf(b)])
        check(a[some], b[some], off[some])


def _check(logits, tokens, top, kind, scale=1.0):
    scale = float(np.float32(scale))
    flat = rounded(logits, kind).reshape(-1, logits.shape[-1])  # what the tensor holds
    two = tokens.reshape(len(flat), -1)
    *want, bounds = log_probabilities(flat, two, top, scale)
    _agree(_run(logits, tokens, top, scale, kind), want, bounds, two)


def _logits(seed, rows, vocabulary, kind, std=3.0):
    rng = np.random.default_rng(seed)
    return normal(rng, (rows, vocabulary), kind, std), rng.integers(0, vocabulary, rows).astype(np.int32)


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,vocabulary", [(1, 1), (3, 2), (2, 63), (2, 64), (2, 65), (5, 1000), (3, 1023), (3, 1025), (2, 4096), (2, 8191), (3, 16411),
                                             (1, 32000), (7, 50021), (2, 131072), (1, 150001)])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_vocabularies(rt, kind, rows, vocabulary, top):
    _check(*_logits(vocabulary + rows, rows, vocabulary, kind), top, kind)


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows", [255, 256, 1023, 1024, 1500])
@pytest.mark.parametrize("top", [0, 7])
def test_many_rows(rt, kind, rows, top):
    """The last one of them begins anywhere in memory."""
    _check(*_logits(rows, rows, 1237, kind), top, kind)


def test_rows_for_several_workgroups_each_and_one(rt):
    for rows in (2, 40, 300, 1100):
        _check(*_logits(rows, rows, 9001, "fp16"), 11, "fp16")


@pytest.mark.parametrize("kind", ["fp16", "fp32"])
@pytest.mark.parametrize("asked", [1, 3, 64, 65, 300])
def test_several_tokens_of_a_row(rt, kind, asked):
    logits, _ = _logits(asked, 4, 3001, kind)
    tokens = np.random.default_rng(asked).integers(-3, 3005, (4, asked)).astype(np.int32)
    tokens[0, 0] = tokens[1, -1] = -1
    tokens[2, 0], tokens[3, 0] = 2 ** 31 - 1, -2 ** 31
    _check(logits, tokens, 3, kind)


def test_rows_in_two_dimensions(rt):
    logits, tokens = _logits(8, 12, 700, "bf16")
    _check(logits.reshape(3, 4, 700), tokens, 4, "bf16")


@pytest.mark.parametrize("scale", [0.01, 0.7, 2.5, 100.0])
@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
def test_scales(rt, scale, kind):
    _check(*_logits(4, 5, 5003, kind), 9, kind, scale)


@pytest.mark.parametrize("rows", [1, 600])
def test_the_largest_and_smallest_scale(rt, rows):
    """All but the most probable six are too improbable for 32 bits; all are alike."""
    logits = np.tile(np.arange(1000) % 7 * -2.0, (rows, 1))
    logits[:, 3::7] = 2.0
    logits[:, 40:] = -20.0  # the greatest: 3, 10, 17, 24, 31, 38
    tokens = np.tile(np.array([10, 11, 999], np.int32), (rows, 1))
    logp, entropy, top_logp, top = _run(logits, tokens, 8, float(np.finfo(np.float32).max), "fp16")
    check(logp[:, 0], np.full(rows, -np.log(6)), 2.0 ** -20)
    check(entropy, np.full(rows, np.log(6)), 2.0 ** -20)
    assert (logp[:, 1:] == -np.inf).all() and (top_logp[:, 6:] == -np.inf).all()
    np.testing.assert_array_equal(top, np.tile([3, 10, 17, 24, 31, 38, 0, 7], (rows, 1)))
    logp, entropy, top_logp, top = _run(logits, tokens, 8, 1e-38, "fp16")
    for x, want in ((logp, -np.log(1000)), (top_logp, -np.log(1000)), (entropy, np.log(1000))):
        check(x, np.full(x.shape, want), 2.0 ** -18)  # of a sum of 1000 ones, exact, the logarithm: within 2^-22 of itself, taken times ln 2
    np.testing.assert_array_equal(top, np.tile([3, 10, 17, 24, 31, 38, 0, 7], (rows, 1)))


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_equal_logits_in_the_order_of_their_tokens(rt, kind, top):
    rng = np.random.default_rng(top)
    flat = np.full((1, 9000), 2.5)
    few = rng.integers(0, 3, (3, 9000)).astype(np.float64)
    signed = np.where(rng.random((2, 9000)) < 0.5, 0.0, -0.0)
    steps = np.floor(np.arange(9000) / 2900.0)[None]
    for logits in (flat, few, signed, steps, -steps):
        _check(logits, np.zeros(len(logits), np.int32), top, kind)


@pytest.mark.parametrize("top", [1, 20, 64])
def test_logits_in_order(rt, top):
    """Every one greater than all before it, and the other way round: bounds that never hold, and at once."""
    rise = np.linspace(-8.0, 8.0, 20000)[None]
    for logits in (rise, -rise, np.abs(rise), -np.abs(rise)):
        x = logits.astype(np.float32).astype(np.float64)
        _check(x, np.array([13], np.int32), top, "fp32")


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
def test_rows_with_few_or_no_probabilities(rt, kind):
    """Logits of minus infinity: a masked vocabulary."""
    rng = np.random.default_rng(3)
    logits = np.full((6, 5000), -np.inf)
    logits[1, 17] = -3.0
    logits[2, [4999, 0, 2500]] = 1.0, 1.0, 60000.0 if kind == "fp16" else 1e30
    logits[3, 100:130] = normal(rng, 30, kind)
    logits[4, ::2] = normal(rng, 2500, kind)
    logits[5, 4999] = -60000.0
    _check(logits, np.array([5, 17, 2500, 99, 2, 4999], np.int32), 6, kind)


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
def test_rows_that_are_not_finite(rt, kind):
    logits, tokens = _logits(5, 6, 40000, kind)
    logits[0, 39999] = np.nan
    logits[2, 3] = np.inf
    logits[3, [7, 30000]] = np.inf, -np.inf
    logits[4, :] = np.nan
    logits[5, 20000] = -np.inf
    _check(logits, tokens, 4, kind)


@pytest.mark.parametrize("kind,largest", [("fp16", 65504.0), ("fp32", 3e38), ("bf16", 3e38)])
def test_logits_at_the_end_of_their_range(rt, kind, largest):
    logits = np.zeros((2, 3000))
    logits[0, 5], logits[0, 6:9] = largest, -largest
    logits[1, :] = -largest
    logits = np.asarray(logits)
    got = _run(logits, np.array([5, 2], np.int32), 2, 1.0, kind)
    assert got[0][0] == 0.0 and got[1][0] == 0.0 and got[3][0, 0] == 5
    np.testing.assert_allclose(got[0][1], -np.log(3000), rtol=1e-6)
    np.testing.assert_allclose(got[1][1], np.log(3000), rtol=1e-6)
    np.testing.assert_array_equal(got[3][1], [0, 1])


def test_a_certain_token(rt):
    """Entropies and log probabilities close to zero, neither below nor far off."""
    logits = np.full((1, 30000), -30.0)
    logits[0, 777] = 5.0
    _check(logits, np.array([777], np.int32), 2, "fp32")
    got = _run(logits, np.array([777], np.int32), 2, 1.0, "fp32")
    assert 0.0 <= got[1][0] < 1e-6 and -1e-6 < got[0][0] <= 0.0


@pytest.mark.parametrize("kind,code", [("fp16", 921), ("fp32", 930)])
def test_strides_and_what_may_be_null(rt, abi, kind, code):
    """Rows inside wider ones that begin between two multiples of 16 bytes; no tokens, no top ones."""
    wide, _ = _logits(6, 5, 4100, kind)
    g = G.KNGraph()
    try:
        size = 4 if kind == "fp32" else 2
        t = put(g, wide, kind)
        n, e, a, b = (put(g, np.full((5, 3), 9.0, np.float32)) for _ in range(4))
        for begin, vocabulary in ((0, 4100), (1, 4099), (3, 2000), (7, 4093)):
            part = wide[:, begin:begin + vocabulary]
            tokens = np.random.default_rng(begin).integers(0, vocabulary, (5, 2)).astype(np.int32)
            logp, entropy, top_logp, top_tokens, bounds = log_probabilities(part, tokens, 3, 1.0)
            top_out = g.new_input((5, 3), G.DT_INT32)
            rc = abi.mi355_log_probabilities(t.device_ptr(False) + begin * size, 4100, put(g, tokens).device_ptr(False), n.device_ptr(False),
                                             e.device_ptr(False), a.device_ptr(False), top_out.device_ptr(False), 5, 2, 3, vocabulary, 1.0, code)
            assert rc == 0, N.last_error()
            assert abi.mi355_sync() == 0
            check(read(n).reshape(-1)[:10].reshape(5, 2), logp, bounds[0])
            check(read(e).reshape(-1)[:5], entropy, bounds[1])
            check(read(a), top_logp, bounds[2])
            np.testing.assert_array_equal(top_out.read_data(), top_tokens)
            rc = abi.mi355_log_probabilities(t.device_ptr(False) + begin * size, 4100, None, None, b.device_ptr(False), None, None, 5, 0, 0,
                                             vocabulary, 1.0, code)
            assert rc == 0
            check(read(b).reshape(-1)[:5], entropy, bounds[1])
    finally:
        g.close()


def test_logits_past_32_bits(rt, abi):
    """Rows more than 2^32 bytes apart."""
    import torch
    stride, vocabulary = (1 << 31) + 5, 5000
    logits, tokens = _logits(9, 2, vocabulary, "fp16")
    far = torch.zeros(stride + vocabulary, dtype=torch.float16, device="cuda")
    for r in range(2):
        far[r * stride:r * stride + vocabulary] = torch.from_numpy(logits[r].astype(np.float16)).cuda()
    torch.cuda.synchronize()
    g = G.KNGraph()
    try:
        n, e = (put(g, np.zeros(2, np.float32)) for _ in range(2))
        assert abi.mi355_log_probabilities(far.data_ptr(), stride, put(g, tokens).device_ptr(False), n.device_ptr(False), e.device_ptr(False), None, None,
                                           2, 1, 0, vocabulary, 1.0, 921) == 0, N.last_error()
        assert abi.mi355_sync() == 0
        *want, bounds = log_probabilities(logits, tokens[:, None], 0, 1.0)
        check(read(n)[:, None], want[0], bounds[0])
        check(read(e), want[1], bounds[1])
    finally:
        g.close()
        del far
        torch.cuda.empty_cache()


def test_queues_side_by_side(rt, abi):
    cases = [_logits(40 + i, 3, 60000, "fp16") for i in range(2)]
    graphs, outs = [], []
    try:
        for logits, tokens in cases:
            g = G.KNGraph()
            graphs.append(g)
            outs.append(g.log_probabilities(put(g, logits, "fp16"), put(g, tokens), 10))
        for _ in range(20):
            for queue, g in enumerate(graphs):
                assert abi.mi355_queue_select(queue) == 0
                g.execute_all()
        assert abi.mi355_sync() == 0
        for (logits, tokens), its in zip(cases, outs):
            *want, bounds = log_probabilities(logits, tokens[:, None], 10, 1.0)
            _agree([o.read_data() if i == 3 else read(o) for i, o in enumerate(its)], want, bounds, tokens[:, None])
    finally:
        abi.mi355_queue_select(0)
        for g in reversed(graphs):
            g.close()


def test_refusals(rt, abi):
    g = G.KNGraph()
    try:
        at = g.new_input((1 << 14,), G.DT_FLOAT32).device_ptr(False)

        def call(**change):
            x = dict(logits=at, stride=100, tokens=at + 8192, log_probs=at + 12288, entropy=at + 16384, top_logp=at + 20480, top_tokens=at + 24576,
                     rows=4, asked=2, top=3, vocabulary=100, scale=1.0, type=930)
            x.update(change)
            return abi.mi355_log_probabilities(*x.values())

        assert call() == 0 and call(rows=0) == 0 and call(rows=1, stride=0) == 0
        for change in (dict(logits=None), dict(tokens=None), dict(log_probs=None), dict(entropy=None), dict(top_logp=None), dict(top_tokens=None),
                       dict(rows=-1), dict(asked=-1), dict(top=-1), dict(vocabulary=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
                       dict(scale=float("nan")), dict(stride=99), dict(logits=at + 2)):
            assert call(**change) == -3, change
        assert call(top=65) == -4 and call(type=950) == -4 and call(vocabulary=(1 << 30) + 1, rows=1) == -4
    finally:
        g.close()
