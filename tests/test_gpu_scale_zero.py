"""A scale of zero beside values that are not finite: weights are equal however large queries and keys are."""
import numpy as np
import pytest

from decoding_reference import HALF_STEP, check
from serving_reference import caches
from test_gpu_window_attention import _run as run_window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("length", [100, 3000])
def test_scale_zero_beside_an_infinite_value(rt, new, length):
    k, v, table, values = caches(2, [length], 1, 64, 16, "bf16")
    q = np.full((new, 2, 64), 2.0 ** 70)
    k[np.isfinite(k)] = 2.0 ** 70
    v[table[0, 1], 2, :, 7] = np.inf
    got = run_window(q, k, v, table, np.array([length], np.int32), "bf16", 0, 0, 0.0)
    assert (got[:, :, 7] == np.inf).all()
    rest = np.arange(64) != 7
    for t in range(new):
        its = values[0][1][:length - (new - 1 - t)]
        n, want = len(its), its.mean(0)
        # equal weights, added up and multiplied in 32 bits, and a rounding to the type
        bound = HALF_STEP["bf16"][0] * np.abs(want) + HALF_STEP["bf16"][1] + 4 * (n + 16) * 2.0 ** -23 * np.abs(its).mean(0)
        check(got[t][:, rest], np.repeat(want[:, rest], 2, 0), np.repeat(bound[:, rest], 2, 0))
