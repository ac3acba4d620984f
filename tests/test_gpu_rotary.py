"""rotary and rotary_append against their formula in 64 bits: layouts of pairs, part of a head, far positions, both
layouts of the cache, slots that store nothing, sizes and alignments of every kind; through graphs and the C ABI."""
import ctypes

import numpy as np
import pytest

from attention_superoptimizer_amd import _native as N
from attention_superoptimizer_amd import graph as G
from decoding_reference import TYPES, check, normal, put, read, rotary_bound, rounded, turned

pytestmark = pytest.mark.gpu


def _angles(half, far=False):
    return G.rotary_angles(2 * half, factor=4.0, original_length=8192 if not far else None, amplitude=1.25)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,head,half", [(1, 1, 64, 32), (3, 5, 128, 64), (70, 40, 128, 64), (9, 3, 80, 16), (5, 7, 96, 20),
                                                    (4, 2, 10, 3), (2, 3, 7, 2), (6, 1, 256, 128), (300, 4, 64, 4), (1, 2, 640, 320), (1, 128, 64, 32),
                                                    (40, 33, 90, 45)])
def test_rotary(rt, kind, interleaved, tokens, heads, head, half):
    rng = np.random.default_rng(tokens * 1000 + head)
    x = normal(rng, (tokens, heads, head), kind)
    positions = rng.integers(-1000000, 1000000, tokens).astype(np.int32)
    positions[0] = 0
    angles = _angles(half)
    g = G.KNGraph()
    try:
        y = g.rotary(put(g, x, kind), put(g, positions), put(g, angles), interleaved=interleaved)
        y.write_data(np.full(y.dims, 7.0))
        g.execute_all()
        want, parts = turned(x, positions, angles, interleaved)
        check(read(y), want, rotary_bound(want, parts, kind))
        if 2 * half < head:
            np.testing.assert_array_equal(read(y)[..., 2 * half:], x[..., 2 * half:])
    finally:
        g.close()


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_angle_of_far_positions(rt, kind):
    """Frequencies of 1 and 3 radians at the largest positions: 2^31 radians are whole turns and a rest."""
    positions = np.array([2147483647, -2147483648, 123456789], np.int32)
    angles = np.array([[1.0, 3.0], [1.0, 1.0]])
    x = rounded(np.tile([1.0, 0.0, 0.0, 1.0], (3, 1, 1)), kind)
    g = G.KNGraph()
    try:
        y = g.rotary(put(g, x, kind), put(g, positions), put(g, angles))
        g.execute_all()
        # (the product of 2^33 radians is rounded to 2^-20 radians in 64 bits, on either side)
        want, parts = turned(x, positions, angles, False)
        check(read(y), want, rotary_bound(want, parts, kind) + 2.0 ** -19)
    finally:
        g.close()


def test_more_tokens_than_a_launch_has(rt, abi):
    """2^23 + 5 tokens of one pair, a slot each."""
    import torch
    tokens = (1 << 23) + 5
    x = torch.randn(3, tokens, 2, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    out, cache = torch.zeros(tokens, 2, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, tokens, 2, dtype=torch.bfloat16, device="cuda")
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") % 5000
    slots = torch.arange(tokens - 1, -1, -1, dtype=torch.int32, device="cuda")
    angles = torch.tensor([0.5, 1.0], dtype=torch.float64, device="cuda")
    torch.cuda.synchronize()
    c = N.Mi355PagedCache(cache[0].data_ptr(), cache[1].data_ptr(), tokens, 1, 1, 2, 2, 2, 2, 920)
    rc = abi.mi355_rotary_append(x[0].data_ptr(), 2, x[1].data_ptr(), 2, x[2].data_ptr(), 2, out.data_ptr(), 2, positions.data_ptr(),
                                 angles.data_ptr(), slots.data_ptr(), ctypes.byref(c), tokens, 1, 1, 0)
    assert rc == 0, N.last_error()
    assert abi.mi355_sync() == 0
    assert torch.equal(cache[1], x[2].flip(0))
    turn = positions.double() * 0.5
    cos, sin = turn.cos(), turn.sin()
    for got, of in ((out, x[0]), (cache[0].flip(0), x[1])):
        a, b = of.double().unbind(1)
        want = torch.stack([a * cos - b * sin, b * cos + a * sin], 1)
        bound = 2.0 ** -8 * want.abs() + 2.0 ** -20 * (a.abs() + b.abs())[:, None]  # (rotary_bound, rounded up)
        assert ((got.double() - want).abs() <= bound).all()


def _append(rt, kind, tokens, q_heads, kv_heads, head, half, page_size, pages, heads_first, interleaved, flat, slots, seed):
    rng = np.random.default_rng(seed)
    qkv = normal(rng, (tokens, q_heads + 2 * kv_heads, head), kind)
    positions, angles = rng.integers(0, 100000, tokens).astype(np.int32), _angles(half)
    dims = (pages, kv_heads, page_size, head) if heads_first else (pages, page_size, kv_heads, head)
    caches = [normal(rng, dims, kind) for _ in range(2)]
    g = G.KNGraph()
    try:
        k, v = (put(g, c, kind) for c in caches)
        q = g.rotary_append(put(g, qkv.reshape(tokens, -1) if flat else qkv, kind), put(g, positions), put(g, angles), put(g, slots),
                            k, v, interleaved=interleaved, heads_first=heads_first)
        q.write_data(np.full(q.dims, 7.0))
        for _ in range(2):  # (the second pass writes the same)
            g.execute_all()
        want, parts = turned(qkv, positions, angles, interleaved)
        bound = rotary_bound(want, parts, kind)
        check(read(q).reshape(tokens, q_heads, head), want[:, :q_heads], bound[:, :q_heads])
        want_k, want_v = (c.copy() for c in caches)
        bound_k = np.zeros(dims)
        for t, slot in enumerate(slots):
            if 0 <= slot < pages * page_size:
                at = (slot // page_size, slice(None), slot % page_size) if heads_first else (slot // page_size, slot % page_size)
                want_k[at], bound_k[at] = want[t, q_heads:q_heads + kv_heads], bound[t, q_heads:q_heads + kv_heads]
                want_v[at] = qkv[t, q_heads + kv_heads:]
        check(read(k), want_k, bound_k)  # (a bound of 0: slots that nothing is stored in stay as they were)
        np.testing.assert_array_equal(read(v), want_v)
    finally:
        g.close()


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,head,half,page_size,interleaved,flat", [
    (1, 1, 1, 64, 32, 1, False, False), (16, 32, 8, 128, 64, 16, False, True), (33, 6, 2, 80, 16, 7, True, False),
    (130, 8, 1, 128, 64, 32, True, True), (5, 3, 3, 96, 20, 24, False, False), (11, 5, 5, 10, 5, 3, False, True), (257, 4, 2, 256, 128, 64, False, False)])
def test_rotary_append(rt, kind, heads_first, tokens, q_heads, kv_heads, head, half, page_size, interleaved, flat):
    pages = -(-tokens // page_size) + 2
    slots = np.random.default_rng(tokens).permutation(pages * page_size)[:tokens].astype(np.int32)
    _append(rt, kind, tokens, q_heads, kv_heads, head, half, page_size, pages, heads_first, interleaved, flat, slots, tokens)


@pytest.mark.parametrize("heads_first", [False, True])
def test_slots_that_store_nothing(rt, heads_first):
    slots = np.array([-1, 3, 48, 47, -2147483648, 2147483647, 0, 49], np.int32)
    _append(rt, "bf16", 8, 4, 2, 64, 32, 16, 3, heads_first, False, False, slots, 4)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_infinities_and_nan_stay_with_their_pair(rt, kind):
    rng = np.random.default_rng(5)
    x = normal(rng, (4, 2, 64), kind)
    special = x.copy()
    special[1, 1, 5], special[2, 0, 40], special[3, 1, 60] = np.inf, np.nan, -np.inf
    positions, angles = np.arange(4, dtype=np.int32) + 3, _angles(16)  # (elements 32 .. are copied)
    g = G.KNGraph()
    try:
        t = put(g, x, kind)
        y = g.rotary(t, put(g, positions), put(g, angles))
        g.execute_all()
        plain = read(y)
        t.write_data(special)
        g.execute_all()
        got = read(y)
        touched = np.zeros(x.shape, bool)
        touched[1, 1, [5, 21]] = touched[2, 0, 40] = touched[3, 1, 60] = True
        np.testing.assert_array_equal(got[~touched], plain[~touched])
        assert not np.isfinite(got[touched]).any() and np.isnan(got[2, 0, 40]) and got[3, 1, 60] == -np.inf
    finally:
        g.close()


def _block(g, n, kind="fp16"):
    """A tensor of n elements, its device address and element size."""
    t = g.new_input((n,), TYPES[kind])
    return t, t.device_ptr(False)


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("stride_more", [0, 3, 8])
def test_strides_alignment_and_in_place(rt, abi, shift, stride_more):
    """Rows further apart than their heads, beginning anywhere: what lies between them stays; y may be x."""
    tokens, heads, head, half, kind = 7, 3, 64, 32, "fp16"
    stride = heads * head + stride_more
    rng = np.random.default_rng(shift * 10 + stride_more)
    flat = normal(rng, (tokens * stride + 16,), kind)
    x = np.stack([flat[shift + t * stride:][:heads * head].reshape(heads, head) for t in range(tokens)])
    positions, angles = rng.integers(0, 5000, tokens).astype(np.int32), _angles(half)
    want, parts = turned(x, positions, angles, False)
    bound = rotary_bound(want, parts, kind)
    g = G.KNGraph()
    try:
        src, dst = put(g, flat, kind), put(g, flat, kind)
        p, a = put(g, positions), put(g, angles)
        for out in (dst, src):
            rc = abi.mi355_rotary(src.device_ptr(False) + 2 * shift, stride, out.device_ptr(False) + 2 * shift, stride,
                                  p.device_ptr(False), a.device_ptr(False), tokens, heads, head, half, 0, 921)
            assert rc == 0, N.last_error()
            got = read(out)
            rows = np.stack([got[shift + t * stride:][:heads * head].reshape(heads, head) for t in range(tokens)])
            check(rows, want, bound)
            keep = np.ones(flat.shape, bool)
            for t in range(tokens):
                keep[shift + t * stride:][:heads * head] = False
            np.testing.assert_array_equal(got[keep], flat[keep])
    finally:
        g.close()


def test_separate_projections_and_a_strided_cache(rt, abi):
    """q, k and v from tensors of their own with strides of their own, into a cache whose pages lie apart."""
    tokens, q_heads, kv_heads, head, half, size, pages, kind = 6, 4, 2, 64, 24, 4, 3, "bf16"
    rng = np.random.default_rng(9)
    q, k, v = (normal(rng, (tokens, h, head), kind) for h in (q_heads, kv_heads, kv_heads))
    token_stride, head_stride, page_stride = 200, 72, 1000
    cache = normal(rng, (pages * page_stride,), kind)
    positions, angles = rng.integers(0, 5000, tokens).astype(np.int32), _angles(half)
    slots = np.array([0, 5, 11, 3, -1, 7], np.int32)
    g = G.KNGraph()
    try:
        tq, tk, tv = (put(g, x, kind) for x in (q, k, v))
        ck, cv = put(g, cache, kind), put(g, cache, kind)
        out, p, a, s = g.new_input((tokens, q_heads, head), TYPES[kind]), put(g, positions), put(g, angles), put(g, slots)
        c = N.Mi355PagedCache(ck.device_ptr(False), cv.device_ptr(False), pages, size, kv_heads, head, page_stride, token_stride,
                              head_stride, 920)
        at = lambda t: t.device_ptr(False)  # noqa: E731
        rc = abi.mi355_rotary_append(at(tq), q_heads * head, at(tk), kv_heads * head, at(tv), kv_heads * head, at(out), q_heads * head,
                                     at(p), at(a), at(s), ctypes.byref(c), tokens, q_heads, half, 0)
        assert rc == 0, N.last_error()
        want, parts = turned(q, positions, angles, False)
        check(read(out), want, rotary_bound(want, parts, kind))
        want_k, parts = turned(k, positions, angles, False)
        bound = rotary_bound(want_k, parts, kind)
        full, full_bound, full_v = cache.copy(), np.zeros(cache.shape), cache.copy()
        for t, slot in enumerate(slots):
            for h in range(kv_heads) if slot >= 0 else ():
                o = slot // size * page_stride + slot % size * token_stride + h * head_stride
                full[o:o + head], full_bound[o:o + head], full_v[o:o + head] = want_k[t, h], bound[t, h], v[t, h]
        check(read(ck), full, full_bound)
        np.testing.assert_array_equal(read(cv), full_v)
    finally:
        g.close()


def test_refusals(rt, abi):
    g = G.KNGraph()
    try:
        t, at = _block(g, 4096)
        i = put(g, np.zeros(64, np.int32)).device_ptr(False)
        a = put(g, np.zeros(64)).device_ptr(False)
        good = [at, 64, at + 4096, 64, i, a, 4, 1, 64, 32, 0, 921]
        assert abi.mi355_rotary(*good) == 0
        for place, value, code in ((6, -1, -3), (7, 0, -3), (8, 0, -3), (9, 33, -3), (9, 0, -3), (11, 930, -4), (0, None, -3), (1, -64, -3), (3, -64, -3), (3, 56, -3),
                                   (2, None, -3), (4, None, -3), (5, None, -3)):
            assert abi.mi355_rotary(*[value if n == place else x for n, x in enumerate(good)]) == code, (place, value)
        assert abi.mi355_rotary(at, 64, at, 72, i, a, 4, 1, 64, 32, 0, 921) == -3
        assert abi.mi355_rotary(at, 64, at, 64, i, a, 0, 1, 64, 32, 0, 921) == 0  # no tokens
        assert abi.mi355_rotary(at, 4096, at, 4096, i, a, 1, 1, 4096, 2048, 0, 921) == -4
        for change in (dict(k=None), dict(v=at), dict(pages=0), dict(page_size=0), dict(pages=1 << 16, page_size=1 << 15),
                       dict(head_dim=0), dict(kv_heads=0), dict(page_stride=-8), dict(type=930)):
            c = N.Mi355PagedCache(at, at + 4096, 2, 4, 1, 64, 256, 64, 64, 921)
            for name, value in change.items():
                setattr(c, name, value)
            assert abi.mi355_rotary_append(at, 64, at, 64, at, 64, at + 4096, 64, i, a, i, ctypes.byref(c), 1, 1, 32, 0) != 0, change
        assert abi.mi355_rotary_append(at, 64, at, 64, at, 64, at + 4096, 64, i, a, i, None, 1, 1, 32, 0) == -3
    finally:
        g.close()
