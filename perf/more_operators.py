"""Cases of the operators that serving adds where tokens are drafted as trees, caches are kept to a window, and answers come
with their probabilities, through `KNGraph`:

* `tree_attention`: attention of a tree of drafted tokens of every sequence over a paged key-value cache: a token sees the
  sequence before the tree, its ancestors and itself;
* `window_attention`: attention of new tokens (one of every sequence, whole prompts, or a different number of every sequence)
  over the last keys of a paged cache and its first few, which stay visible;
* `log_probabilities`: log probabilities of given tokens, the distribution's entropy and its most probable tokens.

With `own` false `run` computes them in elementary torch operations instead.
"""
import math
import types

import numpy as np
import torch

own = False

TYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # One sequence with a small tree behind a short context: latency.
        {"name": "tree_one", "kind": "tree", "sequences": 1, "nodes": 12, "kv_heads": 8, "group": 4, "head": 128, "page_size": 16,
         "longest": 1000, "heads_first": False, "type": "bf16"},
        # A batch of sequences of any length up to 4096, each with a tree of 24 tokens: 96 rows a key-value head.
        {"name": "tree_batch", "kind": "tree", "sequences": 32, "nodes": 24, "kv_heads": 8, "group": 4, "head": 128, "page_size": 16,
         "longest": 4096, "heads_first": False, "type": "bf16"},
        # A few sequences with large trees and long contexts: 512 rows a key-value head, more work than bytes.
        {"name": "tree_wide", "kind": "tree", "sequences": 4, "nodes": 64, "kv_heads": 4, "group": 8, "head": 64, "page_size": 32,
         "longest": 16384, "heads_first": True, "type": "fp16"},
        # Sizes nobody tuned for.
        {"name": "tree_odd", "kind": "tree", "sequences": 5, "nodes": 13, "kv_heads": 3, "group": 5, "head": 80, "page_size": 24,
         "longest": 3001, "heads_first": False, "type": "fp16"},
        # One new token of one sequence: latency.
        {"name": "window_one", "kind": "window", "sequences": 1, "new": 1, "ragged": False, "kv_heads": 8, "group": 4, "head": 128,
         "page_size": 16, "longest": 20000, "window": 4096, "sinks": 4, "heads_first": False, "type": "bf16"},
        # A decode step of a batch, every sequence far past its window: the bytes that are visible, 537 MB.
        {"name": "window_batch", "kind": "window", "sequences": 64, "new": 1, "ragged": False, "kv_heads": 8, "group": 4, "head": 128,
         "page_size": 16, "longest": 32768, "window": 2048, "sinks": 4, "heads_first": False, "type": "bf16"},
        # A prompt of 8192 tokens: matrix products.
        {"name": "window_prompt", "kind": "window", "sequences": 1, "new": 8192, "ragged": False, "kv_heads": 8, "group": 4,
         "head": 128, "page_size": 16, "longest": 8192, "window": 1024, "sinks": 4, "heads_first": False, "type": "bf16"},
        # What a scheduler puts in one step: chunks of prompts behind what is cached, beside single tokens; odd sizes.
        {"name": "window_chunks", "kind": "window", "sequences": 12, "new": 1500, "ragged": True, "kv_heads": 5, "group": 3,
         "head": 80, "page_size": 24, "longest": 7001, "window": 2000, "sinks": 17, "heads_first": False, "type": "fp16"},
        # The answer's next token with five alternatives: latency.
        {"name": "log_one", "kind": "log", "rows": 1, "asked": 1, "vocabulary": 32000, "top": 5, "scale": 1.0, "type": "fp32"},
        # A decode step of a batch over a large vocabulary, twenty alternatives.
        {"name": "log_batch", "kind": "log", "rows": 64, "asked": 1, "vocabulary": 131072, "top": 20, "scale": 1.0, "type": "bf16"},
        # A prompt is scored: thousands of rows, an odd vocabulary, a temperature.
        {"name": "log_prompt", "kind": "log", "rows": 4096, "asked": 1, "vocabulary": 50021, "top": 1, "scale": 1.25, "type": "fp16"},
        # Answers to choose from, asked for at every row; no alternatives.
        {"name": "log_choices", "kind": "log", "rows": 37, "asked": 6, "vocabulary": 100003, "top": 0, "scale": 1.0, "type": "fp32"},
    ]


def _near(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_heads(rng):
    return {"kv_heads": _near(rng, 1, 16), "group": rng.choice([1, 2, 3, 4, 4, 7, 8, 8, 16]),
            "head": rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256]),
            "page_size": rng.choice([16, 16, 32, 64, 128, rng.randint(1, 100)]), "heads_first": rng.random() < 0.3,
            "type": rng.choice(["fp16", "bf16"])}


def _draw_tree(rng):
    while True:
        nodes = _near(rng, 2, 128)
        c = {"kind": "tree", "sequences": _near(rng, 1, 64), "nodes": nodes, "longest": nodes + _near(rng, 16, 32768), **_draw_heads(rng)}
        padded = 4 * c["sequences"] * _width(c) * c["page_size"] * c["kv_heads"] * c["head"]
        scores = c["sequences"] * nodes * c["group"] * c["kv_heads"] * c["longest"]
        if padded <= 1.1e9 and scores <= 140e6 and work(c)["flops"] <= 5e10:
            return c


def _draw_window(rng):
    while True:
        ragged = rng.random() < 0.4
        new = _near(rng, 2, 2048) if ragged else rng.choice([1, 1, rng.randint(2, 8), _near(rng, 64, 8192)])
        c = {"kind": "window", "sequences": _near(rng, 1, 64), "new": new, "ragged": ragged, "longest": new + _near(rng, 16, 32768),
             "window": _near(rng, 64, 4096), "sinks": rng.choice([0, 1, 4, 4, 4, rng.randint(1, 200)]), **_draw_heads(rng)}
        seen = sum(min(n, c["window"] + t + c["sinks"]) for n, t in zip(_lengths(c), _new(c)))
        if 4 * seen * c["kv_heads"] * c["head"] <= 5.4e8 and work(c)["flops"] <= 1.3e11:
            return c


def _draw_log(rng):
    while True:
        c = {"kind": "log", "rows": _near(rng, 1, 8192), "asked": rng.choice([1, 1, 1, rng.randint(2, 8)]),
             "vocabulary": _near(rng, 1000, 200000), "top": rng.choice([0, 1, 5, 20, rng.randint(2, 50)]),
             "scale": rng.choice([1.0, 1.0, 0.7, 1.6]), "type": rng.choice(["fp32", "fp16", "bf16"])}
        if work(c)["bytes"] <= 4.1e8:
            return c


def draw(rng):
    return rng.choice([_draw_tree, _draw_window, _draw_log])(rng)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _share(i):
    return (i * 0.6180339887498949) % 1.0


def _new(c):
    """New tokens of every sequence.  Ragged: a third of them have one, the others anything up to the most."""
    if c["kind"] == "tree":
        return [c["nodes"]] * c["sequences"]
    if not c["ragged"]:
        return [c["new"]] * c["sequences"]
    return [1 if i % 3 == 2 else max(1, c["new"] - int(c["new"] * _share(i))) for i in range(c["sequences"])]


def _lengths(c):
    """Keys of every sequence, its new tokens among them: spread up to the longest, which the first has.  With a window those of
    a batch of single tokens are all past it, as after a while they are."""
    new, least = _new(c), 0
    if c["kind"] == "window" and not c["ragged"] and c["new"] == 1:
        least = min(c["longest"], c["window"] + c["sinks"])
    out = []
    for i, n in enumerate(new):
        span = c["longest"] - max(n, least)
        out.append(c["longest"] - int(span * _share(i)))
    return out


def _width(c):
    return -(-c["longest"] // c["page_size"])


def _tables(c, host):
    """(table, pages): pages that no new token sees have been given back."""
    size, table, count = c["page_size"], np.full((c["sequences"], _width(c)), -1), 0
    for b, (length, new) in enumerate(zip(_lengths(c), _new(c))):
        for p in range(-(-length // size)):
            gone = c["kind"] == "window" and (p + 1) * size <= length - new + 1 - c["window"] and p * size >= c["sinks"]
            if not gone:
                table[b, p] = count
                count += 1
    pages = count + 3
    order = host.permutation(pages)
    return np.where(table < 0, -1, order[np.maximum(table, 0)]), pages


def _parents(c, host):
    """Of every drafted token the one that it follows (-1: the sequence itself), in the order in which they were drafted; where
    fewer were drafted the rest is marked by -2."""
    out = np.full((c["sequences"], c["nodes"]), -2)
    for b in range(c["sequences"]):
        count = c["nodes"] if b % 4 != 3 else max(1, 3 * c["nodes"] // 4)
        wide = int(host.integers(2, 9))
        for i in range(count):
            out[b, i] = -1 if i < wide // 2 else host.integers(max(0, i - 2 * wide), i)
        out[b, 0] = -1
    return out


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)

    def normal(*dims, std=1.0):
        t = torch.empty(dims, dtype=TYPE[c["type"]], device="cuda")
        flat = t.view(-1)
        for at in range(0, flat.numel(), 1 << 26):  # in pieces: the values are drawn in fp32
            part = flat[at:at + (1 << 26)]
            part.copy_(torch.randn(part.numel(), device="cuda", generator=gen).mul_(std))
        return t

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()

    s = types.SimpleNamespace(case=c, inputs={})
    x = s.inputs
    if c["kind"] == "log":
        n, v = c["rows"], c["vocabulary"]
        x["logits"] = normal(n, v, std=3.0)
        # of 64 tokens at random the likeliest, as what was answered mostly is; the others anything
        tokens = torch.randint(0, v, (n, 63 + c["asked"]), device="cuda", generator=gen)
        best = x["logits"].gather(1, tokens[:, :64]).argmax(1, keepdim=True)
        tokens = torch.cat([tokens.gather(1, best), tokens[:, 64:]], 1)
        x["tokens"] = tokens.to(torch.int32) if c["asked"] > 1 else tokens[:, 0].to(torch.int32)
    else:
        table, pages = _tables(c, host)
        new = _new(c)
        dims = (c["kv_heads"], c["page_size"]) if c["heads_first"] else (c["page_size"], c["kv_heads"])
        x["q"] = normal(sum(new), c["kv_heads"] * c["group"], c["head"], std=2.0)
        x["k_cache"], x["v_cache"] = normal(pages, *dims, c["head"]), normal(pages, *dims, c["head"])
        x["table"], x["lengths"] = ints(table), ints(_lengths(c))
        if c["kind"] == "tree":
            x["parents"] = ints(_parents(c, host))
        elif c["ragged"]:
            x["starts"] = ints(np.concatenate([[0], np.cumsum(new)]))
    if own:
        _keep_in_graph(s)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------
_open = []  # graphs in the order they were built: the device arena they share is a stack


class _Graph:
    """A graph that leaves the arena once nobody holds it or a view of its tensors, and everything built after it has left."""

    def __init__(self):
        from attention_superoptimizer_amd import graph as G
        self.graph = G.KNGraph()
        self.entry = [self.graph, True]
        _open.append(self.entry)

    def __del__(self):
        self.entry[1] = False
        while _open and not _open[-1][1]:
            _open.pop()[0].close()


class _Memory:
    """A device tensor of the framework for torch.as_tensor: no copy."""

    def __init__(self, owner, tensor, kind):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(tensor.dims), "typestr": kind, "data": (tensor.device_ptr(False), False),
                                         "strides": None, "version": 2}


_KIND = {torch.float16: "<f2", torch.bfloat16: "<i2", torch.float32: "<f4", torch.int32: "<i4"}


def _view(owner, tensor, dtype):
    t = torch.as_tensor(_Memory(owner, tensor, _KIND[dtype]), device="cuda")
    return t.view(torch.bfloat16) if dtype == torch.bfloat16 else t


def _keep_in_graph(s):
    """The inputs as tensors of a graph with the one operator."""
    from attention_superoptimizer_amd import graph as G
    kinds = {torch.float16: G.DT_FLOAT16, torch.bfloat16: G.DT_BFLOAT16, torch.float32: G.DT_FLOAT32, torch.int32: G.DT_INT32}
    c, x = s.case, s.inputs
    p = _Graph()
    t = {}
    for name in list(x):
        t[name] = p.graph.new_input(tuple(x[name].shape), kinds[x[name].dtype])
        view = _view(p, t[name], x[name].dtype)
        view.copy_(x[name])
        x[name] = view
    if c["kind"] == "tree":
        y = p.graph.tree_attention(t["q"], t["k_cache"], t["v_cache"], t["table"], t["lengths"], t["parents"], scale=c["head"] ** -0.5,
                                   heads_first=c["heads_first"])
        s.out = [_view(p, y, TYPE[c["type"]])]
    elif c["kind"] == "window":
        y = p.graph.window_attention(t["q"], t["k_cache"], t["v_cache"], t["table"], t["lengths"], window=c["window"],
                                     sinks=c["sinks"], starts=t.get("starts"), scale=c["head"] ** -0.5, heads_first=c["heads_first"])
        s.out = [_view(p, y, TYPE[c["type"]])]
    else:
        outs = p.graph.log_probabilities(t["logits"], t["tokens"], top=c["top"], scale=c["scale"])
        s.out = [_view(p, y, torch.int32 if i == 3 else torch.float32) for i, y in enumerate(outs)]
    s.program = p


# ---------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------
def _weighted(scores, seen, values):
    """Softmax over the seen scores, times the values; zeros where nothing is seen."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    return (weights @ values) / torch.where(total == 0, torch.ones_like(total), total)


def _rows_of(cache, pages, places, heads_first):
    """[..., kv_heads, head] of keys or values at places of pages."""
    return cache[pages, :, places] if heads_first else cache[pages, places]


def _plain_tree(c, x):
    b, t, h, g, d = c["sequences"], c["nodes"], c["kv_heads"], c["group"], c["head"]
    pages = x["table"].long().clamp(min=0)

    def gathered(cache):  # [b, h, keys, d]
        rows = cache[pages]
        rows = rows.permute(0, 2, 1, 3, 4) if c["heads_first"] else rows.permute(0, 3, 1, 2, 4)
        return rows.reshape(b, h, -1, d).float()

    parents, node = x["parents"].long(), torch.arange(t, device="cuda")
    above = (parents[..., None] == node).float() + torch.eye(t, device="cuda")
    for _ in range(max(1, (t - 1).bit_length())):  # one step up, then two, four ..
        above = ((above @ above) > 0).float()
    lost = ((parents < -1) | (parents >= node)).float()
    there = (above @ lost[..., None])[..., 0] == 0
    above = (above > 0) & there[..., None]

    q = x["q"].float().view(b, t, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * g, d)
    scores = (q @ gathered(x["k_cache"]).transpose(2, 3).contiguous()) * d ** -0.5
    key = torch.arange(scores.shape[-1], device="cuda")
    context = x["lengths"].long()[:, None] - t
    at = key - context  # [b, keys]: which node's key
    in_tree = (at >= 0) & (at < t)
    seen = above.gather(2, at.clamp(0, t - 1)[:, None, :].expand(b, t, -1)) & in_tree[:, None]
    seen |= (key < context)[:, None] & there[..., None]
    seen = seen[:, None, :, None, :].expand(b, h, t, g, -1).reshape(scores.shape)
    out = _weighted(scores, seen, gathered(x["v_cache"]))
    return [out.view(b, h, t, g, d).permute(0, 2, 1, 3, 4).reshape(b * t, h * g, d).to(x["q"].dtype)]


def _plain_window_step(c, x):
    """A few new tokens of every sequence: the keys that any of them sees, all sequences together."""
    b, t, h, g, d = c["sequences"], c["new"], c["kv_heads"], c["group"], c["head"]
    lengths = x["lengths"].long()[:, None]
    first = (lengths - (t - 1) - c["window"]).clamp(min=c["sinks"])
    key = torch.cat([torch.arange(c["sinks"], device="cuda").expand(b, -1),
                     first + torch.arange(c["window"] + t - 1, device="cuda")], 1)
    inside = key < lengths
    at = torch.where(inside, key, torch.zeros_like(key))
    pages, places = x["table"].long().gather(1, at // c["page_size"]), at % c["page_size"]
    inside &= pages >= 0
    pages = pages.clamp(min=0)
    k, v = (_rows_of(cache, pages, places, c["heads_first"]).transpose(1, 2).float() for cache in (x["k_cache"], x["v_cache"]))
    limit = lengths[..., None] - (t - 1 - torch.arange(t, device="cuda")[:, None])
    seen = inside[:, None] & (key[:, None] < limit) & ((key[:, None] >= limit - c["window"]) | (key[:, None] < c["sinks"]))
    q = x["q"].float().view(b, t, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * g, d)
    scores = (q @ k.transpose(2, 3).contiguous()) * d ** -0.5
    seen = seen[:, None, :, None, :].expand(b, h, t, g, -1).reshape(scores.shape)
    out = _weighted(scores, seen, v.contiguous())
    return [out.view(b, h, t, g, d).permute(0, 2, 1, 3, 4).reshape(b * t, h * g, d).to(x["q"].dtype)]


def _plain_window(c, x):
    if not c["ragged"] and c["new"] <= 8:
        return _plain_window_step(c, x)
    h, g, d, size = c["kv_heads"], c["group"], c["head"], c["page_size"]
    out, row = torch.empty_like(x["q"]), 0
    for b, (length, new) in enumerate(zip(_lengths(c), _new(c))):
        for t0 in range(0, new, 512):
            t = min(512, new - t0)
            limit = length - new + 1 + t0 + torch.arange(t, device="cuda")[:, None]
            start, end = max(0, length - new + 1 + t0 - c["window"]), length - new + t0 + t
            key = torch.arange(start, end, device="cuda")
            if start > 0 and c["sinks"] > 0:
                key = torch.cat([torch.arange(min(start, c["sinks"]), device="cuda"), key])
            pages = x["table"][b].long()[key // size]
            k, v = (_rows_of(cache, pages, key % size, c["heads_first"]).transpose(0, 1).float() for cache in (x["k_cache"], x["v_cache"]))
            seen = (key < limit) & ((key >= limit - c["window"]) | (key < c["sinks"]))
            q = x["q"][row + t0:row + t0 + t].float().view(t, h, g, d).permute(1, 2, 0, 3).reshape(h, g * t, d)
            scores = (q @ k.transpose(1, 2).contiguous()) * d ** -0.5
            y = _weighted(scores.view(h, g, t, -1), seen, v.contiguous()[:, None])
            out[row + t0:row + t0 + t] = y.permute(2, 0, 1, 3).reshape(t, h * g, d).to(out.dtype)
        row += new
    return [out]


def _plain_log(c, x):
    n, v = c["rows"], c["vocabulary"]
    tokens = x["tokens"].long().view(n, c["asked"])
    logp, entropy = torch.empty(n, c["asked"], device="cuda"), torch.empty(n, device="cuda")
    top_logp = torch.empty(n, c["top"], device="cuda")
    top_tokens = torch.empty(n, c["top"], device="cuda", dtype=torch.int32)
    step = max(1, (1 << 26) // v)
    for i in range(0, n, step):
        z = x["logits"][i:i + step].float()
        raw = z
        z = z * c["scale"]
        top = z.amax(1, keepdim=True)
        z = z - top
        weights = torch.exp(z)
        total = weights.sum(1, keepdim=True)
        log_total = torch.log(total)
        logp[i:i + step] = z.gather(1, tokens[i:i + step]) - log_total
        entropy[i:i + step] = log_total[:, 0] - (weights * torch.where(weights > 0, z, torch.zeros_like(z))).sum(1) / total[:, 0]
        if c["top"] > 0:  # the greatest, of equal ones the lowest index: as whole numbers, the index in the lower half
            bits = (raw + 0.0).view(torch.int32)
            order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * (1 << 32) + (v - 1 - torch.arange(v, device="cuda"))
            best = order.topk(c["top"], 1).values
            at = v - 1 - (best & 0xffffffff)
            top_tokens[i:i + step] = at.to(torch.int32)
            top_logp[i:i + step] = z.gather(1, at) - log_total
    out = [logp if c["asked"] > 1 else logp[:, 0], entropy]
    return out + [top_logp, top_tokens] if c["top"] > 0 else out


def run(s):
    if own:
        s.program.graph.execute_all()
        return s.out
    return {"tree": _plain_tree, "window": _plain_window, "log": _plain_log}[s.case["kind"]](s.case, s.inputs)


# ---------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_rows(c, x, b, length):
    """Keys and values [length, kv_heads, head] of a sequence; of pages that were given back anything."""
    size = c["page_size"]
    pages = x["table"][b, :-(-length // size)].long().clamp(min=0)
    return [(cache[pages].transpose(1, 2) if c["heads_first"] else cache[pages]).reshape(-1, c["kv_heads"], c["head"])[:length]
            for cache in (x["k_cache"], x["v_cache"])]


def _exact_attention(c, x):
    g, d = c["group"], c["head"]
    out, row = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (length, new) in enumerate(zip(_lengths(c), _new(c))):
        k, v = _exact_rows(c, x, b, length)
        past = length - new
        if c["kind"] == "tree":
            seen = np.zeros((new, length), bool)
            parents = x["parents"][b].tolist()
            for i in range(new):
                chain, j = [], i
                while 0 <= j < new and (not chain or j < chain[-1]):
                    chain.append(j)
                    j = parents[j]
                if j == -1:
                    seen[i, :past] = True
                    seen[i, [past + n for n in chain]] = True
            blocks = [(0, new, torch.arange(length, device="cuda"), torch.from_numpy(seen).cuda())]
        else:
            blocks = []
            for t0 in range(0, new, 256):
                t1 = min(new, t0 + 256)
                first = max(0, past + t0 + 1 - c["window"])
                key = torch.cat([torch.arange(min(c["sinks"], first), device="cuda"), torch.arange(first, past + t1, device="cuda")])
                own_place = past + torch.arange(t0, t1, device="cuda")[:, None]
                blocks.append((t0, t1, key, (key <= own_place) & ((own_place - key < c["window"]) | (key < c["sinks"]))))
        for t0, t1, key, seen in blocks:
            kk, vv = k[key].double(), v[key].double()
            empty = ~seen.any(1)
            for h in range(c["kv_heads"]):
                q = x["q"][row + t0:row + t1, h * g:(h + 1) * g].double().transpose(0, 1).reshape(g * (t1 - t0), d)
                s = (q @ kk[:, h].T / math.sqrt(d)).view(g, t1 - t0, -1).masked_fill(~seen, -math.inf)
                w = torch.softmax(s, -1).masked_fill(empty[:, None], 0.0)
                out[row + t0:row + t1, h * g:(h + 1) * g] = (w.view(g * (t1 - t0), -1) @ vv[:, h]).view(g, t1 - t0, d).transpose(0, 1)
        row += new
    return [out]


def _exact_log(c, x):
    outs = [[] for _ in range(4 if c["top"] > 0 else 2)]
    for i in range(0, c["rows"], 64):
        logits = x["logits"][i:i + 64]
        logp = torch.log_softmax(logits.double() * c["scale"], 1)
        outs[0].append(logp.gather(1, x["tokens"][i:i + 64].long().view(len(logp), -1)))
        outs[1].append(-(torch.exp(logp) * logp).sum(1))
        if c["top"] > 0:
            at = torch.sort(logits.double(), dim=1, descending=True, stable=True).indices[:, :c["top"]]
            outs[2].append(logp.gather(1, at))
            outs[3].append(at.to(torch.int32))
    outs = [torch.cat(o) for o in outs]
    return [outs[0] if c["asked"] > 1 else outs[0][:, 0], *outs[1:]]


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        x = prepare(case, seed).inputs
    finally:
        own = kept
    return _exact_log(case, x) if case["kind"] == "log" else _exact_attention(case, x)


# ---------------------------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------------------------
def work(case):
    """Inputs read once, results written once.  Attention reads the keys that some row sees."""
    c = case
    if c["kind"] == "log":
        size = 4 if c["type"] == "fp32" else 2
        return {"bytes": c["rows"] * (c["vocabulary"] * size + 8 * c["asked"] + 4 + 8 * c["top"]), "flops": 6 * c["rows"] * c["vocabulary"]}
    heads = c["kv_heads"] * c["group"]
    bytes_, scores = 4 * sum(_new(c)) * heads * c["head"], 0
    for length, new in zip(_lengths(c), _new(c)):
        past = length - new
        if c["kind"] == "tree":
            keys = length
            scores += new * (past + min(new, 6))  # (a token of these trees has about five ancestors)
            bytes_ += 4 * new
        else:
            first = max(0, past + 1 - c["window"])
            keys = length - first + min(first, c["sinks"])
            # row t sees past + t + 1 keys, of these the window's and the first ones before it
            full = max(0, min(new, c["window"] + c["sinks"] - past - 1))  # rows that see all before them
            scores += full * past + full * (full + 1) // 2 + (new - full) * (c["window"] + c["sinks"])
        bytes_ += 4 * keys * c["kv_heads"] * c["head"] + 4 * (-(-keys // c["page_size"]) + 1)
    return {"bytes": bytes_, "flops": 4 * scores * heads * c["head"]}
