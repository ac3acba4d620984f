"""log_probabilities of logits far apart: tokens masked by the type's lowest value, and scales that bring the largest and smallest logits close."""
import numpy as np
import pytest

from decoding_reference import check, normal, rounded
from serving_reference import log_probabilities
from test_gpu_log_probabilities import _agree, _run

pytestmark = pytest.mark.gpu

LOWEST = {"fp16": -65504.0, "bf16": -float(np.array([0x7f7f0000], np.uint32).view(np.float32)[0]), "fp32": float(np.finfo(np.float32).min)}


def _check(logits, tokens, top, kind, scale):
    scale = float(np.float32(scale))
    *want, bounds = log_probabilities(rounded(logits, kind), tokens, top, scale)
    for i in (0, 2):  # what no 32 bits hold
        want[i] = np.where(want[i] < LOWEST["fp32"], -np.inf, want[i])
    _agree(_run(logits, tokens, top, scale, kind), want, bounds, tokens)


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("scale", [0.25, 0.69, 1.0, 1.7])
@pytest.mark.parametrize("rows", [1, 3, 600])
def test_tokens_masked_by_the_lowest_value(rt, kind, scale, rows):
    """A masked token has a log probability of its own, and stands behind all others among the top ones."""
    rng = np.random.default_rng(rows)
    logits = np.full((rows, 3001), LOWEST[kind])
    logits[:, [4, 1000, 3000]] = normal(rng, (rows, 3), kind)
    _check(logits, np.tile(np.array([7, 1000, 4, 2999], np.int32), (rows, 1)), 6, kind, scale)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("scale", [1e-38, 3e-38, 0.1])
@pytest.mark.parametrize("rows", [2, 600])
def test_logits_whose_difference_passes_32_bits(rt, kind, scale, rows):
    rng = np.random.default_rng(rows)
    logits = rounded(rng.uniform(-3.3e38, 3.3e38, (rows, 2500)), kind)
    logits[:, 0], logits[:, 2400] = rounded(3.35e38, kind), LOWEST[kind]
    _check(logits, np.tile(np.array([0, 2400, 11], np.int32), (rows, 1)), 5, kind, scale)
