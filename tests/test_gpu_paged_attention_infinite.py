"""Infinite values that a row of paged_attention sees: its column is infinite with their sign, NaN if they have both, and its
other columns are what they are without them."""
import numpy as np
import pytest

from decoding_reference import attention, check
from test_gpu_paged_attention import _case, _run

pytestmark = pytest.mark.gpu


def _compare(x, kind, window=0, scale=0.125):
    with np.errstate(invalid="ignore"):
        want, bound = attention(*x, scale, window, kind)
    got = _run(*x, kind, scale, window)
    finite = np.isfinite(want)
    check(got[finite], want[finite], bound[finite])
    np.testing.assert_array_equal(got[~finite], want[~finite])
    return want


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("lengths,new,kv_heads,group,head,window", [
    ([1, 2, 33], 1, 2, 4, 64, 0), ([300, 7], 5, 1, 4, 128, 0), ([5000, 130], 1, 1, 8, 128, 0), ([900, 5], 6, 2, 3, 96, 0),
    ([2500, 40], 1, 2, 2, 256, 0), ([2000, 300], 3, 1, 20, 64, 700), ([64] * 300, 1, 8, 1, 64, 0), ([700, 5], 5, 1, 16, 128, 0)])
def test_infinite_values(rt, kind, lengths, new, kv_heads, group, head, window):
    """Of either sign at random keys and columns, the first sequence's last key among them; +, - and both meet in column 1."""
    rng = np.random.default_rng(head + new)
    q, k, v, table, n = _case(head + group, lengths, new, kv_heads, group, head, 16, kind)
    marks = 0
    for b, length in enumerate(lengths):
        for _ in range(4):
            j = int(rng.integers(0, length))
            v[table[b, j // 16], j % 16, rng.integers(0, kv_heads), rng.integers(2, head)] = rng.choice([-np.inf, np.inf])
            marks += 1
        if b % 2 == 0:
            v[table[b, (length - 1) // 16], (length - 1) % 16, 0, 1] = np.inf
            v[table[b, 0], 0, 0, 1] = -np.inf
    want = _compare((q, k, v, table, n), kind, window)
    assert np.isinf(want).sum() >= marks // 2


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("new", [1, 4])
def test_weights_of_every_size(rt, kind, new):
    """Column j has its infinite value at the key whose weight is 2^-j of the greatest, exactly: up to 2^-30.  A second word of
    a weight is zero in most of them."""
    head, length = 64, 40
    q, k, v, table, n = _case(1, [length], new, 1, 2, head, 64, kind)
    q[:] = 0.0
    q[..., 0] = 1.0
    at = table[0, 0]
    k[at, :length] = 0.0
    for j in range(31):
        k[at, j, 0, 0] = -j
        v[at, j, 0, j] = np.inf if j % 2 else -np.inf
    want = _compare((q, k, v, table, n), kind, scale=float(np.float32(np.log(2.0))))
    assert np.isinf(want[..., :31]).all() and np.isfinite(want[..., 31:]).all()


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_nan_and_infinite_values_of_one_key(rt, kind):
    q, k, v, table, n = _case(2, [100, 100], 3, 1, 2, 64, 16, kind)
    v[table[0, 2], 3, 0, 5], v[table[0, 2], 3, 0, 6], v[table[0, 2], 3, 0, 7] = np.inf, np.nan, -np.inf
    v[table[0, 4], 1, 0, 6] = np.inf
    want = _compare((q, k, v, table, n), kind)
    assert np.isnan(want[0, ..., 6]).all() and (want[0, ..., 5] == np.inf).all()
