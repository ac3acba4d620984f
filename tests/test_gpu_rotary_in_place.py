"""rotary_append whose queries are turned where they lie, in the projection that they are a part of."""
import ctypes

import numpy as np
import pytest

from attention_superoptimizer_amd import _native as N
from attention_superoptimizer_amd import graph as G
from decoding_reference import check, normal, put, read, rotary_bound, turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,head", [(1, 64), (5, 64), (300, 64), (9, 50)])
def test_queries_in_place(rt, abi, interleaved, tokens, head):
    q_heads, kv_heads, page, pages, half, kind = 3, 2, 16, 24, 20, "fp16"
    rng = np.random.default_rng(tokens + head)
    x = normal(rng, (tokens, q_heads + 2 * kv_heads, head), kind)
    positions, angles = rng.integers(0, 9000, tokens).astype(np.int32), G.rotary_angles(2 * half)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    want, parts = turned(x, positions, angles, interleaved)
    bound = rotary_bound(want, parts, kind)
    g = G.KNGraph()
    try:
        t, p, a, s = put(g, x, kind), put(g, positions), put(g, angles), put(g, slots)
        k, v = (put(g, np.zeros((pages, page, kv_heads, head)), kind) for _ in range(2))
        stride, at = (q_heads + 2 * kv_heads) * head, t.device_ptr(False)
        c = N.Mi355PagedCache(k.device_ptr(False), v.device_ptr(False), pages, page, kv_heads, head, page * kv_heads * head, kv_heads * head,
                              head, 921)

        def call(out, out_stride):
            return abi.mi355_rotary_append(at, stride, at + 2 * q_heads * head, stride, at + 2 * (q_heads + kv_heads) * head, stride, out,
                                           out_stride, p.device_ptr(False), a.device_ptr(False), s.device_ptr(False), ctypes.byref(c),
                                           tokens, q_heads, half, int(interleaved))

        if tokens > 1:  # at another stride a token's results would lie on other tokens' queries
            assert call(at, q_heads * head) == -3 and "in place" in N.last_error()
            assert abi.mi355_rotary(at, stride, at, stride + 8, p.device_ptr(False), a.device_ptr(False), tokens, q_heads, head, half, 0, 921) == -3
            np.testing.assert_array_equal(read(t), x)
        assert call(at, stride) == 0, N.last_error()
        got = read(t)
        check(got[:, :q_heads], want[:, :q_heads], bound[:, :q_heads])
        np.testing.assert_array_equal(got[:, q_heads:], x[:, q_heads:])
        check(read(k).reshape(-1, kv_heads, head)[slots], want[:, q_heads:q_heads + kv_heads], bound[:, q_heads:q_heads + kv_heads])
        np.testing.assert_array_equal(read(v).reshape(-1, kv_heads, head)[slots], x[:, q_heads + kv_heads:])
    finally:
        g.close()
