"""paged_attention over values as large and as small as bf16 holds: a weighted mean of finite values is finite."""
import numpy as np
import pytest

from decoding_reference import attention, check
from test_gpu_paged_attention import _case, _run

pytestmark = pytest.mark.gpu
LARGEST = (2.0 - 2.0 ** -7) * 2.0 ** 127  # of bf16
SHAPES = [([1, 2, 37], 1, 2, 4, 64, 0), ([300, 7], 5, 1, 4, 128, 0), ([5000, 130], 1, 1, 8, 128, 0), ([900], 6, 2, 3, 96, 0),
          ([2500, 40], 1, 2, 2, 256, 0), ([2000, 300], 3, 1, 2, 64, 700)]


def _both(x, kind, window=0, slack=0.0):
    want, bound = attention(*x, 0.125, window, kind)
    assert np.isfinite(want).all()
    check(_run(*x, kind, 0.125, window), want, bound + slack)


@pytest.mark.parametrize("lengths,new,kv_heads,group,head,window", SHAPES)
def test_values_at_the_end_of_the_range(rt, lengths, new, kv_heads, group, head, window):
    """All of them the largest: so is the mean, which no sum on the way may leave behind."""
    q, k, v, table, n = _case(len(lengths) + head, lengths, new, kv_heads, group, head, 16, "bf16")
    v[np.isfinite(v)] = LARGEST
    v[..., 1::2] *= -1.0
    _both((q, k, v, table, n), "bf16", window)


@pytest.mark.parametrize("lengths,new,kv_heads,group,head,window", SHAPES)
@pytest.mark.parametrize("power", [113, 120, 125])
def test_large_values(rt, lengths, new, kv_heads, group, head, window, power):
    """Of both signs, up to four times the power of two (normal, within 4 of zero)."""
    q, k, v, table, n = _case(power + head, lengths, new, kv_heads, group, head, 16, "bf16")
    seen = np.isfinite(v)
    v[seen] = np.clip(v[seen], -3.984375, 3.984375) * 2.0 ** power  # 3.984375 = 4 - 2^-6, of bf16
    _both((q, k, v, table, n), "bf16", window)


def test_one_value_among_ordinary_ones(rt):
    q, k, v, table, n = _case(5, [200, 200], 1, 1, 4, 64, 16, "bf16")
    v[table[0, 3], 5, 0, 7], v[table[1, 11], 2, 0, 60] = LARGEST, -2.0 ** 115
    _both((q, k, v, table, n), "bf16")


@pytest.mark.parametrize("lengths,new,kv_heads,group,head,window", SHAPES)
@pytest.mark.parametrize("power", [-100, -112])
def test_small_values(rt, lengths, new, kv_heads, group, head, window, power):
    """n weights that add up to less than one are each 2^-log2(4 n) or less: products with values of 2^-112 have 2^-149 as their
    smallest step, which half of is lost n times and divided by that sum, an eighth at least.  Both words of a weight count."""
    q, k, v, table, n = _case(head - power, lengths, new, kv_heads, group, head, 16, "bf16")
    seen = np.isfinite(v)
    v[seen] = v[seen] * 2.0 ** power
    most = max(lengths)
    _both((q, k, v, table, n), "bf16", window, slack=2 * most * 2.0 ** -150 * 4 * most)


def test_values_of_fp16_at_the_end_of_its_range(rt):
    q, k, v, table, n = _case(6, [5000, 3], 1, 2, 4, 64, 16, "fp16")
    v[np.isfinite(v)] = 65504.0
    _both((q, k, v, table, n), "fp16")
