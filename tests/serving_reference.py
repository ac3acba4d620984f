"""Attention of trees and within windows, and log probabilities, in 64 bits from their formulas, and the bounds that results keep."""
import numpy as np

from attention_superoptimizer_amd import graph as G
from decoding_reference import HALF_STEP, normal, put, read


def caches(seed, lengths, kv_heads, head, page_size, kind, heads_first=False, spare=2, filler=np.nan, width=None):
    """(k, v, table, values): caches that hold `filler` where no sequence has a key, page tables (-1 behind a sequence's pages), and
    the keys and values of every sequence in a row."""
    rng = np.random.default_rng(seed)
    need = [-(-max(0, n) // page_size) for n in lengths]
    width = width or max(1, *need) + 1
    pages = sum(need) + spare
    order, at = rng.permutation(pages), 0
    table = np.full((len(lengths), width), -1, np.int32)
    k, v = (np.full((pages, page_size, kv_heads, head), filler) for _ in range(2))
    values = []
    for b, (n, p) in enumerate(zip(lengths, need)):
        table[b, :p] = order[at:at + p]
        at += p
        its = [normal(rng, (max(0, n), kv_heads, head), kind) for _ in range(2)]
        values.append(its)
        for cache, rows in zip((k, v), its):
            for i in range(p):
                some = rows[i * page_size:(i + 1) * page_size]
                cache[table[b, i], :len(some)] = some
    if heads_first:
        k, v = (np.ascontiguousarray(c.swapaxes(1, 2)) for c in (k, v))
    return k, v, table, values


def window_seen(length, new, window, sinks):
    """[new, length]: which keys a new token sees."""
    end = length - (new - 1 - np.arange(new))[:, None]
    j = np.arange(max(0, length))
    return (j < end) & ((j >= end - window) | (j < sinks) | (window == 0))


def tree_seen(length, parents):
    new = len(parents)
    seen, context = np.zeros((new, max(0, length)), bool), length - new
    for i in range(new):
        chain, at = [], i
        while at >= 0 and context + at >= 0 and -1 <= parents[at] < at:
            chain.append(context + at)
            at = parents[at]
        if at == -1:
            seen[i, :max(0, context)] = True
            seen[i, chain] = True
    return seen


def attended(q, k, v, seen, scale, kind):
    """(results, bounds) of rows q [rows, q_heads, head] over k, v [keys, kv_heads, head] with seen [rows, keys]."""
    rows, q_heads, d = q.shape
    step, least = HALF_STEP[kind]
    out, bound = np.zeros_like(q), np.full_like(q, least)
    if k.shape[0] == 0:
        return out, bound
    some = seen.any(1)
    for h in range(q_heads):
        kk, vv = k[:, h // (q_heads // k.shape[1])], v[:, h // (q_heads // k.shape[1])]
        s = np.where(seen, scale * (q[:, h] @ kk.T), -np.inf)
        top = np.where(some, s.max(1), 0.0)[:, None]
        w = np.exp(s - top)
        total = w.sum(1, keepdims=True)
        w /= np.where(total == 0, 1.0, total)
        y = w @ vv
        # A score is a sum of d products in 32 bits: within (d + 4) 2^-23 of the sum of their magnitudes (an addition may truncate).
        # The exponential's argument, as far from 0 as the scores lie apart, is rounded twice, its value to 2^-22; weights and
        # values add up over n keys in 32 bits, twice over where parts are joined: relative to the weight, and in their sum
        # too.  Each weight is rounded to the values' type once, to half a step of it, and added up as that: the result is off by the sum of
        # what each is off times the distance of its value from the result, half a step of w |v| and of |y| (below 2^-23 of the greatest
        # fp16 weights are cut at 2^-34 of it).  2^-150 and less counts as nothing.
        n = seen.sum(1)
        score = (d + 4) * 2.0 ** -23 * abs(scale) * np.where(seen, np.abs(q[:, h]) @ np.abs(kk).T, 0.0).max(1)
        spread = np.minimum(150.0, np.where(some, (top - np.where(seen, s, np.inf).min(1, keepdims=True))[:, 0], 0.0))
        weight = 2 * score + 2.0 ** -22 * (spread + 4) + 2 * (n + 16) * 2.0 ** -23
        near = np.where(seen, np.abs(vv).T[:, None, :], 0.0).max(-1).T if kind == "fp16" else 0.0
        bound[:, h] += 2 * step * np.abs(y) + (2 * weight + step)[:, None] * (w @ np.abs(vv)) + (2.0 ** -34 * n[:, None] * near if kind == "fp16" else 0.0)
        out[:, h] = y
    return out, bound


def log_probabilities(logits, tokens, top, scale):
    """(log probabilities, entropy, top log probabilities, top tokens, bounds of the first three) of logits [rows, vocabulary] and
    tokens [rows, asked]."""
    rows, vocabulary = logits.shape
    logp, entropy = np.full(tokens.shape, -np.inf), np.zeros(rows)
    top_logp, top_tokens = np.full((rows, top), -np.inf), np.full((rows, top), -1, np.int32)
    bounds = [np.zeros_like(logp), np.zeros_like(entropy), np.zeros_like(top_logp)]
    for r in range(rows):
        x = logits[r]
        if np.isnan(x).any() or (x == np.inf).any():
            logp[r] = entropy[r] = top_logp[r] = np.nan
            continue
        is_one = x > -np.inf
        if not is_one.any():
            continue
        z = np.where(is_one, scale * (np.where(is_one, x, 0.0) - x.max()), -np.inf)
        w = np.exp(z)
        log_z = np.log(w.sum())
        entropy[r] = log_z - (w[is_one] * z[is_one]).sum() / w.sum()
        order = [int(j) for j in np.lexsort((np.arange(vocabulary), -x))[:top] if is_one[j]]
        top_logp[r, :len(order)], top_tokens[r, :len(order)] = z[order] - log_z, order
        for i, t in enumerate(tokens[r]):
            if 0 <= t < vocabulary:
                logp[r, i] = z[t] - log_z
        # In units of log 2: z is a difference and a product with a scale that is rounded itself, three half steps of z.  Two to that
        # power is within 2^-22, its sum of n terms over lanes that add up one in 256 of them and then their joins within (n / 256 + 24)
        # steps; the logarithm within 2^-22 of itself and of 1, and so is what it is taken from.  Terms of z below -126 are nothing.
        own = 2.0 ** -22 * np.abs(z[is_one]) + 2.0 ** -22
        sums = (vocabulary / 256 + 24) * 2.0 ** -24 * 2
        share = w[is_one] / w.sum()
        off_z = (share * own).sum() + sums
        off_log = off_z + 2.0 ** -22 * (abs(log_z) + 1) + 2.0 ** -126
        one = lambda v: np.where(np.isfinite(v), off_log + 2.0 ** -22 * (2 * np.abs(np.where(np.isfinite(v), v, 0.0)) + 1), 0.0)
        bounds[0][r], bounds[2][r] = one(logp[r]), one(top_logp[r])
        mean = (share * np.abs(z[is_one])).sum()
        bounds[1][r] = off_log + (share * np.abs(z[is_one]) * own).sum() + (share * own).sum() + mean * (sums + off_z) + 2.0 ** -22 * (mean + log_z + 1)
    return logp, entropy, top_logp, top_tokens, bounds


__all__ = ["G", "attended", "caches", "log_probabilities", "normal", "put", "read", "tree_seen", "window_seen"]
