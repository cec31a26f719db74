"""The decoding and cache-eviction operators as they are measured: listed cases, draws of the same ranges, inputs,
the plain form and a 64-bit form of each.

Four operators, used one after another by a program that decodes over the pooled caches:

* ``tree``    attention of drafted tokens (a tree, a chain or one token a request) over a paged K/V cache
* ``weights`` the attention weight that each cached token got from a block of queries
* ``heaviest`` the positions a cache keeps: its first, its last and its heaviest ones
* ``retain``  moving the kept tokens' K/V, per layer and head, to other rows of the pool

Shapes are the text encoder's pool (28 layers, 28 query heads over 4 K/V heads of 128) and generic ones.
"""

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    enc = {"hq": 28, "hkv": 4, "d": 128, "dtype": "bf16"}
    return [
        # one request writes its next token: the smallest call, made once per layer
        {"name": "tree_one_token", "op": "tree", **enc, "page": 64, "batch": 1, "short": 1024, "long": 1024,
         "nodes": 1, "kind": "chain"},
        # a batch of requests of very different ages, one token each
        {"name": "tree_batch_decode", "op": "tree", **enc, "page": 64, "batch": 64, "short": 313, "long": 8191,
         "nodes": 1, "kind": "chain"},
        # a batch with a tree of drafted tokens each
        {"name": "tree_batch_drafts", "op": "tree", **enc, "page": 64, "batch": 8, "short": 701, "long": 6007,
         "nodes": 61, "kind": "tree"},
        # one tree over a cache that fills most of the encoder's 4 GiB pool, token-granular slots
        {"name": "tree_long_cache", "op": "tree", **{**enc, "dtype": "fp16"}, "page": 1, "batch": 1, "short": 65521,
         "long": 65521, "nodes": 24, "kind": "tree"},
        # as many K/V heads as query heads (24 of 128): a chain of guessed tokens over an edit's prefix
        {"name": "tree_own_heads", "op": "tree", "hq": 24, "hkv": 24, "d": 128, "dtype": "bf16", "page": 64,
         "batch": 5, "short": 1500, "long": 4608, "nodes": 4, "kind": "chain"},
        # a decode step that also keeps count of the weights
        {"name": "weights_decode", "op": "weights", **enc, "page": 64, "batch": 32, "short": 257, "long": 8191,
         "nodes": 1, "kind": "chain"},
        # the new tail of a prompt over its cached head
        {"name": "weights_tail", "op": "weights", **enc, "page": 64, "batch": 1, "short": 1024, "long": 1024,
         "nodes": 509, "kind": "chain"},
        # a long prompt's second half over its first
        {"name": "weights_prefill", "op": "weights", **enc, "page": 16, "batch": 1, "short": 16384, "long": 16384,
         "nodes": 16384, "kind": "chain"},
        # one request's cache, every layer and head, cut to a quarter
        {"name": "heaviest_one", "op": "heaviest", "rows": 28 * 4, "short": 4096, "long": 4096, "budget": 1024,
         "sinks": 4, "recent": 128},
        # sixteen long requests of different lengths
        {"name": "heaviest_batch", "op": "heaviest", "rows": 28 * 4 * 16, "short": 3001, "long": 32749,
         "budget": 2048, "sinks": 4, "recent": 511},
        # moving a short cache
        {"name": "retain_small", "op": "retain", "layers": 28, "hkv": 4, "d": 128, "dtype": "bf16", "page": 64,
         "length": 1024, "budget": 251},
        # moving a long one in a token-granular pool
        {"name": "retain_large", "op": "retain", "layers": 28, "hkv": 4, "d": 128, "dtype": "bf16", "page": 1,
         "length": 32768, "budget": 8192},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "weights", "weights", "heaviest", "retain"])
    hkv, group = rng.choice([(4, 7), (4, 4), (2, 8), (8, 4), (24, 1), (1, 12), (3, 5)])
    d, dtype, page = rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "fp16"]), rng.choice([1, 8, 16, 64, 64])
    heads = {"hq": hkv * group, "hkv": hkv, "d": d, "dtype": dtype, "page": page}
    if op in ("tree", "weights"):
        batch = _log(rng, 1, 64)
        # at most about the largest listed batch's cached bytes, and the pool of one long request
        top = min(65521, int(5.5e8 / (batch * hkv * d * 4)))
        long = _log(rng, 16, max(top, 17))
        nodes = 1 if rng.random() < 0.35 else _log(rng, 2, 100)
        kind = rng.choice(["chain", "tree"])
        if op == "weights" and rng.random() < 0.4:
            batch, kind = rng.choice([1, 1, 2]), "chain"
            long, nodes = _log(rng, 64, 8192), _log(rng, 100, 4096)
        return {"op": op, **heads, "batch": batch, "short": rng.randint(0, long), "long": long, "nodes": nodes,
                "kind": kind}
    if op == "heaviest":
        long = _log(rng, 64, 65521)
        rows = _log(rng, 1, max(1, min(2048, int(5e7 / long))))
        budget = _log(rng, 8, long)
        sinks = rng.choice([0, 4, min(7, budget)])
        sinks = min(sinks, budget)
        return {"op": op, "rows": rows, "short": rng.randint(1, long), "long": long, "budget": budget,
                "sinks": sinks, "recent": rng.randint(0, budget - sinks)}
    layers = rng.choice([1, 7, 28])
    length = _log(rng, 2, min(32768, int(28 * 4 * 128 * 32768 / (layers * hkv * d))))
    return {"op": op, "layers": layers, "hkv": hkv, "d": d, "dtype": dtype, "page": page, "length": length,
            "budget": rng.randint(1, max(1, length // 2))}


def _lengths(case):
    """Cached tokens of each request: spread evenly from `short` to `long`, in a mixed order."""
    n = case["batch"] if case["op"] != "heaviest" else case["rows"]
    if n == 1:
        return [case["long"]]
    step = next(s for s in (7, 11, 13, 17, 19) if math.gcd(s, n) == 1)
    return [case["short"] + (case["long"] - case["short"]) * (i * step % n) // (n - 1) for i in range(n)]


def _parents(case):
    """Parent of each drafted node within its request (-1: it follows the cache), the same for every request."""
    n = case["nodes"]
    if case["kind"] == "chain":
        return list(range(-1, n - 1))
    r = random.Random(1000 * n + case["long"])
    return [-1] + [r.randrange(max(0, i - 9), i) if r.random() < 0.95 else -1 for i in range(1, n)]


def _pairs(case):
    """(drafted node, drafted node it sees) pairs of one request."""
    parents = _parents(case)
    if case["kind"] == "chain":
        return len(parents) * (len(parents) + 1) // 2
    depth = []
    for p in parents:
        depth.append(1 if p < 0 else depth[p] + 1)
    return sum(depth)


def work(case):
    if case["op"] in ("tree", "weights"):
        e, d, hq, hkv = 2, case["d"], case["hq"], case["hkv"]
        lens, n = _lengths(case), case["nodes"]
        cached, total = sum(lens), n * case["batch"]
        table = 4 * sum(-(-x // case["page"]) for x in lens)
        pairs = n * cached + case["batch"] * _pairs(case)
        if case["op"] == "tree":
            io = (cached + total) * hkv * d * e * 2 + total * hq * (2 * d * e + 4) + table
            return {"bytes": io, "flops": 4 * pairs * hq * d}
        width = max(lens) + n
        io = (cached + total) * hkv * d * e + total * hq * (d * e + 4) + case["batch"] * hkv * width * 4 + table
        return {"bytes": io, "flops": 2 * pairs * hq * d}
    if case["op"] == "heaviest":
        lens = _lengths(case)
        return {"bytes": 4 * sum(lens) + 8 * case["rows"] * case["budget"], "flops": sum(lens)}
    moved = case["layers"] * 2 * case["hkv"] * case["budget"]
    return {"bytes": 2 * moved * case["d"] * 2 + moved * 2 + 8 * case["budget"], "flops": 0}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _slots(pages, n, page):
    """Pool rows of n tokens that lie in `pages`."""
    t = torch.arange(n, device=DEV)
    return pages[t // page] * page + t % page


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["op"] == "heaviest":
        # accumulated weights: over several powers of ten, with tokens that never got any
        w = torch.empty(case["rows"], case["long"], device=DEV).normal_(generator=g).mul_(2.5).exp_()
        w[torch.rand(w.shape, generator=g, device=DEV) < 0.05] = 0.0
        lens = _lengths(case)
        s["weights"] = w
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        return s
    dt, page, hkv, d = TYPES[case["dtype"]], case["page"], case["hkv"], case["d"]
    lens = [case["length"], case["budget"]] if case["op"] == "retain" else _lengths(case)
    layers = case.get("layers", 2)
    need = [-(-x // page) for x in lens]
    pages = torch.randperm(sum(need) + 3, generator=g, device=DEV) + 1  # a used pool: pages in no order, page 0 is padding
    rows = (sum(need) + 4) * page
    s["kv"] = torch.empty(layers, 2, rows, hkv, d, dtype=dt, device=DEV).normal_(generator=g)
    s["slots"], at = [], 0
    for x, n in zip(lens, need):
        s["slots"].append(_slots(pages[at : at + n], x, page))
        at += n
    if case["op"] == "retain":
        # every layer and head keeps its own positions
        score = torch.rand(layers, hkv, case["length"], generator=g, device=DEV)
        s["keep"] = score.topk(case["budget"]).indices.sort().values.to(torch.int32)
        return s
    s["layer"] = layers - 1
    total = case["batch"] * case["nodes"]
    new = lambda h, x=1.0: torch.empty(total, h, d, dtype=dt, device=DEV).normal_(generator=g).mul_(x)  # noqa: E731
    # scores of a trained model are further apart than those of unit vectors: standard deviation 2
    s["q"], s["k_new"], s["v_new"] = new(case["hq"], 2.0), new(hkv), new(hkv)
    s["lens"] = lens
    s["parents"] = _parents(case)
    s["see"] = _see(case) if case["kind"] == "tree" else None
    s["scale"] = 1.0 / math.sqrt(d)
    if case["op"] == "weights":
        s["lse"] = torch.empty(case["hq"], total, device=DEV)
        for b in range(case["batch"]):
            for kv_head, _, score in _scores(s, b):
                m = score.amax(-1, keepdim=True)
                put = (m + (score - m).exp().sum(-1, keepdim=True).log()).squeeze(-1)
                _head_rows(s, s["lse"], b, kv_head).copy_(put)
    return s


def _see(case):
    """[n, n] truth: node i sees node j (itself and its ancestors)."""
    n = case["nodes"]
    see = torch.zeros(n, n, dtype=torch.bool)
    for i, p in enumerate(_parents(case)):
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
    return see.to(DEV)


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own or case["op"] == "heaviest":
        return s
    from qwenedit_b200.paged import PagedKVPool

    kv = s["kv"]
    layers, _, rows, hkv, d = kv.shape
    page = case["page"]
    budget = (rows - page) * layers * 2 * hkv * d * kv.element_size()
    s["pool"] = PagedKVPool("measured", layers, hkv, d, budget, kv.dtype, DEV, page_size=page, kv=kv)
    if case["op"] == "retain":
        return s
    from qwenedit_b200.drafts import DraftTree, PagedBatch

    s["cache"] = PagedBatch(s["pool"], s["slots"])
    parents = None if case["kind"] == "chain" else s["parents"] * case["batch"]
    s["tree"] = DraftTree([case["nodes"]] * case["batch"], parents, device=DEV)
    return s


# ---- the calls ---------------------------------------------------------------------------------------------------

def run(state):
    s = state
    if s["op"] == "tree":
        if own:
            from qwenedit_b200.drafts import tree_attention

            return tree_attention(s["q"], s["cache"], s["tree"], s["layer"], s["k_new"], s["v_new"],
                                  scale=s["scale"], return_lse=True)
        return _plain_tree(s)
    if s["op"] == "weights":
        if own:
            from qwenedit_b200.evict import attention_weights

            return attention_weights(s["q"], s["lse"], s["cache"], s["tree"], s["layer"], s["k_new"],
                                     scale=s["scale"])
        return _plain_weights(s)
    if s["op"] == "heaviest":
        if own:
            from qwenedit_b200.evict import heaviest

            return heaviest(s["weights"], s["budget"], lengths=s["lengths"], sinks=s["sinks"], recent=s["recent"])
        return _plain_heaviest(s)
    if own:
        s["pool"].retain(s["slots"][0], s["keep"], s["slots"][1])
        return s["kv"]
    return _plain_retain(s)


# ---- plain forms -------------------------------------------------------------------------------------------------

def _head_rows(s, t, b, kv_head):
    """Rows of request b and K/V head kv_head of a [Hq, T] tensor: [G, n]."""
    n, group = s["nodes"], s["hq"] // s["hkv"]
    return t[kv_head * group : (kv_head + 1) * group, b * n : (b + 1) * n]


def _scores(s, b):
    """Per K/V head of request b: (head, V [keys, D] in 32 bits, masked scores [G, n, keys] in 32 bits)."""
    n, group = s["nodes"], s["hq"] // s["hkv"]
    new = slice(b * n, (b + 1) * n)
    own_part = s["see"] if s["see"] is not None else torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
    for kv_head in range(s["hkv"]):
        k = torch.cat([s["kv"][s["layer"], 0, s["slots"][b], kv_head], s["k_new"][new, kv_head]]).float()
        v = torch.cat([s["kv"][s["layer"], 1, s["slots"][b], kv_head], s["v_new"][new, kv_head]]).float()
        q = s["q"][new, kv_head * group : (kv_head + 1) * group].float().transpose(0, 1)
        score = (q @ k.T).mul_(s["scale"])
        score[:, :, s["lens"][b] :].masked_fill_(~own_part, float("-inf"))
        yield kv_head, v, score


def _plain_tree(s):
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["hq"], s["q"].shape[0], device=DEV)
    n, group = s["nodes"], s["hq"] // s["hkv"]
    for b in range(s["batch"]):
        for kv_head, v, score in _scores(s, b):
            m = score.amax(-1, keepdim=True)
            p = (score - m).exp()
            total = p.sum(-1, keepdim=True)
            o = (p @ v) / total
            out[b * n : (b + 1) * n, kv_head * group : (kv_head + 1) * group] = o.transpose(0, 1).to(out.dtype)
            _head_rows(s, lse, b, kv_head).copy_((m + total.log()).squeeze(-1))
    return out, lse


def _plain_weights(s):
    w = torch.zeros(s["batch"], s["hkv"], max(s["lens"]) + s["nodes"], device=DEV)
    for b in range(s["batch"]):
        for kv_head, _, score in _scores(s, b):
            p = (score - _head_rows(s, s["lse"], b, kv_head)[..., None]).exp()
            w[b, kv_head, : p.shape[-1]] = p.sum((0, 1))
    return w


def _plain_heaviest(s):
    w, budget = s["weights"], s["budget"]
    rows, width = w.shape
    at = torch.arange(width, device=DEV)
    length = s["lengths"][:, None].long()
    first, last = at < s["sinks"], (at >= length - s["recent"]) & (at < length)
    rank = torch.where(first | last, float("inf"), w)
    rank = torch.where(at < length, rank, float("-inf"))
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :budget]  # ties: the lowest position first
    order = torch.where(order < length, order, width).sort(dim=1).values
    if order.shape[1] < budget:
        order = torch.cat([order, order.new_full((rows, budget - order.shape[1]), width)], 1)
    there = order < width
    kept = torch.where(there, w.gather(1, order.clamp(max=width - 1)), 0.0)
    return torch.where(there, order, -1).to(torch.int32), kept


def _plain_retain(s):
    kv, (src, dst), keep = s["kv"], s["slots"], s["keep"].long()
    heads = torch.arange(s["hkv"], device=DEV)[:, None]
    for layer in range(s["layers"]):
        rows = src[keep[layer]]  # [Hkv, budget]
        for c in range(2):
            kv[layer, c][dst[None, :], heads] = kv[layer, c][rows, heads]
    return kv


# ---- from the definition, in 64 bits -----------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] not in ("tree", "weights"):
        return None  # positions and moved values: nothing is computed
    s = _inputs(case, seed)
    hq, hkv, n = case["hq"], case["hkv"], case["nodes"]
    total = n * case["batch"]
    out = torch.empty(total, hq, case["d"], dtype=torch.float64, device=DEV)
    lse = torch.empty(hq, total, dtype=torch.float64, device=DEV)
    w = torch.zeros(case["batch"], hkv, max(s["lens"]) + n, dtype=torch.float64, device=DEV)
    # which drafted nodes each node sees, from its walk to the root
    walk = torch.zeros(n, n, dtype=torch.bool)
    if case["kind"] == "chain":
        walk = torch.arange(n)[:, None] >= torch.arange(n)[None, :]
    else:
        for i in range(n):
            j = i
            while j >= 0:
                walk[i, j] = True
                j = s["parents"][j]
    walk = walk.to(DEV)
    for b, length in enumerate(s["lens"]):
        rows = s["slots"][b]
        for h in range(hq):
            kv_head = h // (hq // hkv)
            kc = s["kv"][s["layer"], 0, rows, kv_head].double()
            vc = s["kv"][s["layer"], 1, rows, kv_head].double()
            kn = s["k_new"][b * n : (b + 1) * n, kv_head].double()
            vn = s["v_new"][b * n : (b + 1) * n, kv_head].double()
            for lo in range(0, n, 4096):  # queries in pieces, to bound the memory
                i = slice(b * n + lo, b * n + min(lo + 4096, n))
                q = s["q"][i, h].double()
                a = torch.exp(q @ kc.T * s["scale"])  # scores stay below 100: no maximum is needed in 64 bits
                c = torch.exp(q @ kn.T * s["scale"]) * walk[lo : lo + 4096]
                if case["op"] == "tree":
                    z = a.sum(1) + c.sum(1)
                    out[i, h] = (a @ vc + c @ vn) / z[:, None]
                    lse[h, i] = z.log()
                else:
                    f = torch.exp(-s["lse"][h, i].double())
                    w[b, kv_head, :length] += f @ a
                    w[b, kv_head, length : length + n] += f @ c
    return (out, lse) if case["op"] == "tree" else w
