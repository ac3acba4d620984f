"""Cases of the operators that a serving step runs on a paged key-value cache, through `KNGraph`:

* `rotary` / `rotary_append`: rotary positions, and with them the write of new keys and values into their slots of the cache;
* `paged_attention`: attention of one or a few new tokens of every sequence over the cache's pages;
* `verify_drafts`: which of a sequence's drafted tokens the target's probabilities keep, and the token that follows them.

With `own` false `run` computes them in elementary torch operations instead.
"""
import math
import types

import numpy as np
import torch

own = False

HALF = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # A decode step of 16 sequences: their queries and keys are turned, keys and values stored.  The
        # smallest call of the kind, one per layer and token.
        {"name": "append_decode", "kind": "append", "tokens": 16, "q_heads": 32, "kv_heads": 8, "head": 128, "rotary": 128,
         "interleaved": False, "page_size": 16, "heads_first": False, "far": 8192, "type": "bf16"},
        # A prompt of 8192 tokens: bounded by the bytes.
        {"name": "append_prompt", "kind": "append", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "head": 128, "rotary": 128,
         "interleaved": False, "page_size": 16, "heads_first": False, "far": 8192, "type": "fp16"},
        # Positions alone, on part of a head whose size is no power of two, interleaved pairs, far positions.
        {"name": "rotary_part", "kind": "rotary", "tokens": 1001, "q_heads": 20, "head": 80, "rotary": 32, "interleaved": True,
         "far": 1000000, "type": "fp16"},
        # One sequence, one new token, a short cache: latency.
        {"name": "attention_one", "kind": "attention", "sequences": 1, "new": 1, "kv_heads": 8, "group": 4, "head": 128,
         "page_size": 16, "longest": 1000, "window": 0, "heads_first": False, "type": "bf16"},
        # A batch of sequences of any length up to 4096, as a serving loop holds them.
        {"name": "attention_batch", "kind": "attention", "sequences": 64, "new": 1, "kv_heads": 8, "group": 4, "head": 128,
         "page_size": 16, "longest": 4096, "window": 0, "heads_first": False, "type": "bf16"},
        # One sequence with a long cache, 537 MB of keys and values: the cache's bytes.
        {"name": "attention_long", "kind": "attention", "sequences": 1, "new": 1, "kv_heads": 8, "group": 8, "head": 128,
         "page_size": 64, "longest": 131072, "window": 0, "heads_first": False, "type": "fp16"},
        # Verification of four drafted tokens and the one before them: forty rows a key-value head.
        {"name": "attention_drafts", "kind": "attention", "sequences": 16, "new": 5, "kv_heads": 4, "group": 8, "head": 64,
         "page_size": 32, "longest": 4096, "window": 0, "heads_first": True, "type": "fp16"},
        # Sizes nobody tuned for, and a sliding window.
        {"name": "attention_odd", "kind": "attention", "sequences": 7, "new": 2, "kv_heads": 5, "group": 3, "head": 80,
         "page_size": 24, "longest": 3001, "window": 1500, "heads_first": False, "type": "bf16"},
        # One sequence with four drafts: latency.
        {"name": "verify_one", "kind": "verify", "sequences": 1, "drafts": 4, "vocabulary": 32000, "certain": False, "type": "fp32"},
        # A batch over a large vocabulary.
        {"name": "verify_batch", "kind": "verify", "sequences": 64, "drafts": 5, "vocabulary": 131072, "certain": False,
         "type": "fp32"},
        # Drafts without probabilities (found in the prompt), an odd vocabulary, 16-bit probabilities.
        {"name": "verify_certain", "kind": "verify", "sequences": 19, "drafts": 3, "vocabulary": 50021, "certain": True,
         "type": "fp16"},
    ]


def _near(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_rotary(rng):
    while True:
        c = {"kind": rng.choice(["append", "append", "rotary"]), "tokens": _near(rng, 1, 8192), "q_heads": 0, "head": 0, "rotary": 0,
             "interleaved": rng.random() < 0.4, "far": _near(rng, 8192, 1000000), "type": rng.choice(["fp16", "bf16"])}
        c["head"] = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
        c["rotary"] = rng.choice([c["head"], c["head"], c["head"] // 2, 16 * rng.randint(1, c["head"] // 16)])
        if c["kind"] == "append":
            c["kv_heads"] = _near(rng, 1, 16)
            c["q_heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 8])
            c["page_size"] = rng.choice([16, 16, 32, 64, 128, rng.randint(1, 100)])
            c["heads_first"] = rng.random() < 0.3
        else:
            c["q_heads"] = rng.randint(1, 64)
        if work(c)["bytes"] <= 201e6:
            return c


def _draw_attention(rng):
    while True:
        c = {"kind": "attention", "sequences": _near(rng, 1, 128), "new": rng.choice([1, 1, 1, rng.randint(2, 8)]),
             "kv_heads": _near(rng, 1, 32), "group": rng.choice([1, 2, 3, 4, 4, 7, 8, 8, 16]),
             "head": rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256]),
             "page_size": rng.choice([16, 16, 32, 64, 128, rng.randint(1, 100)]), "longest": _near(rng, 16, 131072),
             "window": rng.choice([0, 0, 0, _near(rng, 64, 4096)]), "heads_first": rng.random() < 0.3,
             "type": rng.choice(["fp16", "bf16"])}
        cache = 4 * _pages(c) * c["page_size"] * c["kv_heads"] * c["head"]
        padded = 4 * c["sequences"] * _width(c) * c["page_size"] * c["kv_heads"] * c["head"]
        if cache <= 5.4e8 and padded <= 1.1e9 and c["sequences"] * c["new"] * c["group"] * c["kv_heads"] * c["longest"] <= 64e6:
            return c


def _draw_verify(rng):
    while True:
        c = {"kind": "verify", "sequences": _near(rng, 1, 128), "drafts": rng.randint(1, 8), "vocabulary": _near(rng, 1000, 150000),
             "certain": rng.random() < 0.3, "type": rng.choice(["fp32", "fp32", "fp16", "bf16"])}
        if c["sequences"] * (c["drafts"] + 1) * c["vocabulary"] <= 64 * 6 * 131072:
            return c


def draw(rng):
    return rng.choice([_draw_rotary, _draw_attention, _draw_attention, _draw_verify])(rng)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _lengths(c):
    """Keys of every sequence, its new tokens among them: spread over [new, longest], the first the longest."""
    span = c["longest"] - c["new"]
    return [max(c["new"], c["longest"] - int(span * ((i * 0.6180339887498949) % 1.0))) for i in range(c["sequences"])]


def _width(c):
    return -(-c["longest"] // c["page_size"])


def _pages(c):
    return sum(-(-n // c["page_size"]) for n in _lengths(c)) + 3


def _angles(c):
    """Frequencies and amplitudes of the pairs: the low ones four times slower, those between blended, as a context
    of four times its length is reached."""
    half = c["rotary"] // 2
    w = 10000.0 ** (-np.arange(half, dtype=np.float64) / half)
    blend = np.clip((2.0 * np.pi / w) / 8192.0, 0.0, 1.0)
    return np.stack([w * (1.0 - 0.75 * blend), np.full(half, 1.05)])


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)

    def normal(*dims, std=1.0):
        t = torch.empty(dims, dtype=HALF[c["type"]], device="cuda")
        flat = t.view(-1)
        for at in range(0, flat.numel(), 1 << 26):  # in pieces: the values are drawn in fp32
            part = flat[at:at + (1 << 26)]
            part.copy_(torch.randn(part.numel(), device="cuda", generator=gen).mul_(std))
        return t

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()

    def cache(pages):
        dims = (c["kv_heads"], c["page_size"]) if c["heads_first"] else (c["page_size"], c["kv_heads"])
        return normal(pages, *dims, c["head"])

    s = types.SimpleNamespace(case=c, inputs={})
    x = s.inputs
    if c["kind"] in ("rotary", "append"):
        n = c["tokens"]
        heads = c["q_heads"] + (2 * c["kv_heads"] if c["kind"] == "append" else 0)
        x["x"] = normal(n, heads, c["head"])
        x["positions"] = ints((host.integers(0, c["far"]) + np.arange(n)) % c["far"] if n > 64 else host.integers(0, c["far"], n))
        x["angles"] = torch.from_numpy(_angles(c)).cuda()
        if c["kind"] == "append":
            pages = -(-n // c["page_size"]) + 5
            x["slots"] = ints(host.permutation(pages)[np.arange(n) // c["page_size"]] * c["page_size"] + np.arange(n) % c["page_size"])
            x["k_cache"], x["v_cache"] = cache(pages), cache(pages)
    elif c["kind"] == "attention":
        lengths, pages = _lengths(c), _pages(c)
        free, at = host.permutation(pages), 0
        table = np.full((c["sequences"], _width(c)), -1)
        for b, n in enumerate(lengths):
            k = -(-n // c["page_size"])
            table[b, :k] = free[at:at + k]
            at += k
        x["q"] = normal(c["sequences"] * c["new"], c["kv_heads"] * c["group"], c["head"], std=2.0)
        x["k_cache"], x["v_cache"] = cache(pages), cache(pages)
        x["table"], x["lengths"] = ints(table), ints(lengths)
    else:
        b, t, v = c["sequences"], c["drafts"], c["vocabulary"]
        logits = torch.randn((b, t + 1, v), device="cuda", generator=gen).mul_(3.0)
        x["target"] = torch.softmax(logits, -1).to(HALF[c["type"]])
        draft = torch.softmax(logits[:, :t] + torch.randn((b, t, v), device="cuda", generator=gen).mul_(0.5), -1)
        race = torch.empty((b, t, v), device="cuda").exponential_(generator=gen)  # the largest weight over its wait wins
        x["tokens"] = (draft / race).argmax(-1).to(torch.int32)
        if not c["certain"]:
            x["draft"] = draft.to(HALF[c["type"]])
        x["uniforms"] = torch.rand((b, t + 1), device="cuda", generator=gen)
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


_KIND = {torch.float16: "<f2", torch.bfloat16: "<i2", torch.float32: "<f4", torch.float64: "<f8", torch.int32: "<i4"}


def _view(owner, tensor, dtype):
    t = torch.as_tensor(_Memory(owner, tensor, _KIND[dtype]), device="cuda")
    return t.view(torch.bfloat16) if dtype == torch.bfloat16 else t


def _keep_in_graph(s):
    """The inputs as tensors of a graph with the one operator."""
    from attention_superoptimizer_amd import graph as G
    kinds = {torch.float16: G.DT_FLOAT16, torch.bfloat16: G.DT_BFLOAT16, torch.float32: G.DT_FLOAT32,
             torch.float64: G.DT_DOUBLE, torch.int32: G.DT_INT32}
    c, x = s.case, s.inputs
    p = _Graph()
    t = {}
    for name in list(x):
        t[name] = p.graph.new_input(tuple(x[name].shape), kinds[x[name].dtype])
        view = _view(p, t[name], x[name].dtype)
        view.copy_(x[name])
        x[name] = view
    half = HALF[c["type"]]
    if c["kind"] == "rotary":
        y = p.graph.rotary(t["x"], t["positions"], t["angles"], interleaved=c["interleaved"])
        s.out = [_view(p, y, half)]
    elif c["kind"] == "append":
        y = p.graph.rotary_append(t["x"], t["positions"], t["angles"], t["slots"], t["k_cache"], t["v_cache"],
                                  interleaved=c["interleaved"], heads_first=c["heads_first"])
        s.out = [_view(p, y, half), x["k_cache"], x["v_cache"]]
    elif c["kind"] == "attention":
        y = p.graph.paged_attention(t["q"], t["k_cache"], t["v_cache"], t["table"], t["lengths"], scale=c["head"] ** -0.5,
                                    window=c["window"], heads_first=c["heads_first"])
        s.out = [_view(p, y, half)]
    else:
        n, y = p.graph.verify_drafts(t["target"], t.get("draft"), t["tokens"], t["uniforms"])
        s.out = [_view(p, n, torch.int32), _view(p, y, torch.int32)]
    s.program = p


# ---------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------
def _turned(x, positions, angles, interleaved):
    """Rotary positions of [tokens, heads, head], in 32 bits; angles in 64."""
    half = angles.shape[1]
    turn = positions.double()[:, None] * angles[0]
    cos, sin = ((f(turn) * angles[1]).float()[:, None, :] for f in (torch.cos, torch.sin))
    y = x.float()
    pairs = y[..., :2 * half]
    if interleaved:
        a, b = pairs[..., 0::2], pairs[..., 1::2]
        pairs = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = pairs[..., :half], pairs[..., half:]
        pairs = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([pairs, y[..., 2 * half:]], -1).to(x.dtype)


def _plain_append(c, x):
    q, k, v = x["x"].split([c["q_heads"], c["kv_heads"], c["kv_heads"]], 1)
    slots = x["slots"].long()
    page, at = slots // c["page_size"], slots % c["page_size"]
    k = _turned(k, x["positions"], x["angles"], c["interleaved"])
    for cache, rows in ((x["k_cache"], k), (x["v_cache"], v)):
        if c["heads_first"]:
            cache[page, :, at] = rows
        else:
            cache[page, at] = rows
    return [_turned(q, x["positions"], x["angles"], c["interleaved"]), x["k_cache"], x["v_cache"]]


def _plain_attention(c, x):
    b, t, h, g, d = c["sequences"], c["new"], c["kv_heads"], c["group"], c["head"]
    pages = x["table"].long().clamp(min=0)

    def gathered(cache):  # [b, h, keys, d]
        rows = cache[pages]
        rows = rows.permute(0, 2, 1, 3, 4) if c["heads_first"] else rows.permute(0, 3, 1, 2, 4)
        return rows.reshape(b, h, -1, d).float()

    q = x["q"].float().view(b, t, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * g, d)
    scores = (q @ gathered(x["k_cache"]).transpose(2, 3).contiguous()) * d ** -0.5
    key = torch.arange(scores.shape[-1], device="cuda")
    limit = x["lengths"].long()[:, None] - (t - 1 - torch.arange(t, device="cuda"))
    seen = key < limit[..., None]
    if c["window"]:
        seen &= key >= limit[..., None] - c["window"]
    seen = seen[:, None, :, None, :].expand(b, h, t, g, -1).reshape(scores.shape)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    out = (weights @ gathered(x["v_cache"])) / torch.where(total == 0, torch.ones_like(total), total)
    return [out.view(b, h, t, g, d).permute(0, 2, 1, 3, 4).reshape(b * t, h * g, d).to(x["q"].dtype)]


def _plain_verify(c, x):
    b, t, v = c["sequences"], c["drafts"], c["vocabulary"]
    target, tokens, u = x["target"], x["tokens"].long(), x["uniforms"].double()
    row = torch.arange(b, device="cuda")
    p = target[:, :t].gather(2, tokens[..., None])[..., 0].double()
    q = x["draft"].gather(2, tokens[..., None])[..., 0].double() if not c["certain"] else torch.ones_like(p)
    accepted = (u[:, :t] * q < p).long().cumprod(1).sum(1)
    weights = target[row, accepted].double()
    at = accepted.clamp(max=t - 1)
    if c["certain"]:
        less = weights.scatter(1, tokens[row, at][:, None], 0.0)
    else:
        less = (weights - x["draft"][row, at].double()).clamp(min=0.0)
    less = torch.where((accepted < t)[:, None], less, weights)
    weights = torch.where(less.sum(1, keepdim=True) > 0, less, weights)
    below = weights.cumsum(1)
    token = (below <= (u[:, t] * below[:, -1])[:, None]).sum(1).clamp(max=v - 1)
    place = torch.arange(t + 1, device="cuda")
    out = torch.cat([tokens, torch.full_like(tokens[:, :1], -1)], 1)
    out = torch.where(place < accepted[:, None], out, -1)
    out = torch.where(place == accepted[:, None], token[:, None], out)
    return [accepted.to(torch.int32), out.to(torch.int32)]


def run(s):
    if own:
        s.program.graph.execute_all()
        return s.out
    c, x = s.case, s.inputs
    if c["kind"] == "rotary":
        return [_turned(x["x"], x["positions"], x["angles"], c["interleaved"])]
    return {"append": _plain_append, "attention": _plain_attention, "verify": _plain_verify}[c["kind"]](c, x)


# ---------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_turned(x, positions, angles, interleaved):
    """Every pair as a complex number times e^(i angle)."""
    half = angles.shape[1]
    turn = torch.polar(angles[1].expand(len(positions), half).contiguous(), positions.double()[:, None] * angles[0])[:, None]
    y = x.double().clone()
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        x = prepare(case, seed).inputs
    finally:
        own = kept
    c = case
    if c["kind"] == "rotary":
        return [_exact_turned(x["x"], x["positions"], x["angles"], c["interleaved"])]
    if c["kind"] == "append":
        caches = [x["k_cache"].double(), x["v_cache"].double()]
        q = _exact_turned(x["x"][:, :c["q_heads"]], x["positions"], x["angles"], c["interleaved"])
        k = _exact_turned(x["x"][:, c["q_heads"]:c["q_heads"] + c["kv_heads"]], x["positions"], x["angles"], c["interleaved"])
        for cache, rows in zip(caches, (k, x["x"][:, c["q_heads"] + c["kv_heads"]:].double())):
            for token, slot in enumerate(x["slots"].tolist()):
                page, at = divmod(slot, c["page_size"])
                if c["heads_first"]:
                    cache[page, :, at] = rows[token]
                else:
                    cache[page, at] = rows[token]
        return [q, *caches]
    if c["kind"] == "attention":
        t, g, d = c["new"], c["group"], c["head"]
        out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
        for b, (n, table) in enumerate(zip(x["lengths"].tolist(), x["table"].tolist())):
            pages = table[:-(-n // c["page_size"])]
            k, v = (cache[pages].transpose(1, 2) if c["heads_first"] else cache[pages] for cache in (x["k_cache"], x["v_cache"]))
            k, v = (a.reshape(-1, c["kv_heads"], d)[:n] for a in (k, v))
            for i in range(t):
                end = n - (t - 1 - i)
                start = max(0, end - c["window"]) if c["window"] else 0
                if end <= start:
                    continue
                for h in range(c["kv_heads"]):
                    rows = x["q"][b * t + i, h * g:(h + 1) * g].double()
                    weights = torch.softmax(rows @ k[start:end, h].double().T / math.sqrt(d), -1)
                    out[b * t + i, h * g:(h + 1) * g] = weights @ v[start:end, h].double()
        return [out]
    target, u, tokens = (x[n].cpu().double().numpy() for n in ("target", "uniforms", "tokens"))
    draft = None if c["certain"] else x["draft"].cpu().double().numpy()
    counts, outs = [], []
    for b in range(c["sequences"]):
        n, rejected = 0, False
        while n < c["drafts"] and not rejected:
            j = int(tokens[b, n])
            rejected = not u[b, n] * (1.0 if draft is None else draft[b, n, j]) < target[b, n, j]
            n += not rejected
        w = target[b, n]
        if rejected:
            less = np.where(np.arange(len(w)) == tokens[b, n], 0.0, w) if draft is None else np.maximum(w - draft[b, n], 0.0)
            w = less if less.sum() > 0 else w
        below = np.cumsum(w)
        token = min(int(np.searchsorted(below, u[b, c["drafts"]] * below[-1], side="right")), len(w) - 1)
        counts.append(n)
        outs.append([int(j) for j in tokens[b, :n]] + [token] + [-1] * (c["drafts"] - n))
    return [torch.tensor(counts, dtype=torch.int32), torch.tensor(outs, dtype=torch.int32)]


# ---------------------------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------------------------
def work(case):
    """Inputs read once, results written once.  Attention reads the keys that some row sees; a verification reads the
    drafted tokens' probabilities and the row of the first token that is not taken."""
    c = case
    size = 4 if c["type"] == "fp32" else 2
    if c["kind"] in ("rotary", "append"):
        heads = c["q_heads"] + (2 * c["kv_heads"] if c["kind"] == "append" else 0)
        turned = c["q_heads"] + (c["kv_heads"] if c["kind"] == "append" else 0)
        return {"bytes": 2 * c["tokens"] * (heads * c["head"] * 2 + 4), "flops": 3 * c["tokens"] * turned * c["rotary"]}
    if c["kind"] == "attention":
        rows = c["sequences"] * c["new"] * c["kv_heads"] * c["group"]
        span = [min(n, c["window"] + c["new"] - 1) if c["window"] else n for n in _lengths(c)]
        per_row = [min(n, c["window"]) if c["window"] else n for n in _lengths(c)]
        return {"bytes": sum(span) * c["kv_heads"] * c["head"] * 4 + 4 * rows * c["head"] + 4 * sum(-(-n // c["page_size"]) + 1 for n in span),
                "flops": 4 * sum(per_row) * c["new"] * c["kv_heads"] * c["group"] * c["head"]}
    rows = 1 if c["certain"] else 2
    return {"bytes": c["sequences"] * (rows * (c["vocabulary"] + c["drafts"]) * size + 12 * c["drafts"] + 12),
            "flops": 3 * c["sequences"] * c["vocabulary"]}
