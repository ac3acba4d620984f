"""The operators of a decoding step in 64 bits, straight from their formulas, and the bounds their results keep."""
import math

import numpy as np

from attention_superoptimizer_amd import graph as G

TYPES = {"fp16": G.DT_FLOAT16, "bf16": G.DT_BFLOAT16, "fp32": G.DT_FLOAT32}
# half a step, relative to the value, and half of the smallest step
HALF_STEP = {"fp16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134), "fp32": (2.0 ** -24, 2.0 ** -150)}


def rounded(a, kind):
    """`a` to the nearest value of a type, as float64."""
    a = np.asarray(a, np.float64)
    if kind == "bf16":
        return (G._bf16_bits(a.astype(np.float32)).astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(a.shape)
    return a.astype(np.float16 if kind == "fp16" else np.float32).astype(np.float64)


def normal(rng, dims, kind, std=1.0):
    return rounded(rng.standard_normal(dims) * std, kind)


def put(g, a, kind=None):
    """An input tensor of graph `g` that holds `a`."""
    a = np.asarray(a)
    t = g.new_input(a.shape, TYPES[kind] if kind else {np.dtype(np.float64): G.DT_DOUBLE, np.dtype(np.float32): G.DT_FLOAT32,
                                                       np.dtype(np.int32): G.DT_INT32}[a.dtype])
    t.write_data(a)
    return t


def read(t):
    return t.read_data().astype(np.float64)


def turned(x, positions, angles, interleaved):
    """(rotary positions of x [tokens, heads, head], the sum of the magnitudes that each element is made of)."""
    half = angles.shape[1]
    turn = positions.astype(np.float64)[:, None] * angles[0]
    c, s = (angles[1] * f(turn) for f in (np.cos, np.sin))
    c, s = c[:, None], s[:, None]
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y, parts = x.copy(), np.zeros_like(x)
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    parts[..., one] = parts[..., two] = np.abs(angles[1]) * (np.abs(a) + np.abs(b))
    return y, parts


def rotary_bound(y, parts, kind):
    """The fraction of a turn is rounded to 2^-26 turns at most, 2^-23 radians; sine and cosine to two units of 2^-24, the
    amplitude, its product and the two products of the sum to half of one each: within 2^-21 of what they multiply."""
    step, least = HALF_STEP[kind]
    return step * np.abs(y) + least + 2.0 ** -21 * (1 + step) * parts


def attention(q, k_cache, v_cache, table, lengths, scale, window, kind, heads_first=False):
    """(results, bounds) for q [sequences, new, q_heads, head] and caches [pages, page, kv_heads, head]."""
    if heads_first:
        k_cache, v_cache = k_cache.swapaxes(1, 2), v_cache.swapaxes(1, 2)
    sequences, new, q_heads, d = q.shape
    pages, size, kv_heads, _ = k_cache.shape
    step, least = HALF_STEP[kind]
    out, bound = np.zeros_like(q), np.full_like(q, least)
    for b in range(sequences):
        length = max(0, min(int(lengths[b]), table.shape[1] * size))
        for t in range(new):
            end = length - (new - 1 - t)
            begin = max(0, end - window) if window else 0
            keys = [j for j in range(begin, end) if 0 <= table[b, j // size] < pages]
            if not keys:
                continue
            at = [(table[b, j // size], j % size) for j in keys]
            k, v = (np.stack([c[p, i] for p, i in at]) for c in (k_cache, v_cache))
            for h in range(q_heads):
                kk, vv = k[:, h // (q_heads // kv_heads)], v[:, h // (q_heads // kv_heads)]
                with np.errstate(invalid="ignore"):
                    s = scale * (kk @ q[b, t, h])
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[b, t, h] = w @ vv
                    # A score is a sum of d products in 32 bits: within (d + 4) 2^-23 of the sum of their magnitudes (an
                    # addition may truncate).  The exponential's argument, as far from 0 as the scores lie apart, is rounded
                    # twice, its value to 2^-22.  Weights are kept to 2^-16 for the product with the values, whose sums, and
                    # that of the weights, add n numbers in 32 bits, twice over where parts are joined.
                    n = len(keys)
                    score = (d + 4) * 2.0 ** -23 * abs(scale) * (np.abs(kk) @ np.abs(q[b, t, h])).max()
                    spread = min(150.0, s.max() - s.min())
                    weight = 2 * score + 2.0 ** -22 * (spread + 4) + 2.0 ** -16 + 2 * (n + 16) * 2.0 ** -23
                    bound[b, t, h] += step * np.abs(out[b, t, h]) + 2 * weight * (w @ np.abs(vv))
    return out, bound


def verified(target, draft, tokens, uniforms):
    """(accepted, tokens) of verify_drafts."""
    sequences, drafts = tokens.shape
    vocabulary = target.shape[-1]
    accepted, out = np.zeros(sequences, np.int32), np.full((sequences, drafts + 1), -1, np.int32)
    for b in range(sequences):
        n, refused = 0, False
        while n < drafts and 0 <= tokens[b, n] < vocabulary:
            x = tokens[b, n]
            if not float(uniforms[b, n]) * (1.0 if draft is None else draft[b, n, x]) < target[b, n, x]:
                refused = True
                break
            out[b, n] = x
            n += 1
        w = target[b, n].copy()
        if refused:
            if draft is None:
                w[tokens[b, n]] = 0.0
            else:
                w = w - draft[b, n]
        w = np.where(w > 0, w, 0.0)
        if refused and w.sum() == 0:
            w = np.where(target[b, n] > 0, target[b, n], 0.0)
        total = math.fsum(w)
        if total > 0:
            passes = np.flatnonzero((w > 0) & (np.cumsum(w) > float(uniforms[b, drafts]) * total))
            out[b, n] = passes[0] if len(passes) else np.flatnonzero(w > 0)[-1]
        accepted[b] = n
    return accepted, out


def check(got, want, bound, what=""):
    off = np.abs(got - want)
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((off / bound)[bad].max()), np.argwhere(bad)[:4].tolist())
