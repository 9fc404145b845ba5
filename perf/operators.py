"""The operators of a cache that is drafted into and thinned out, as a served model calls them for one layer (attention) or for all
its layers at once (what moves rows of the cache).

A case is a dict of plain values.  ``kind`` says what one pass is:

  tree     attention of the nodes of every request's tree of drafted tokens: all keys that the request holds, and of the drafted
           ones those that the node's mask names
  commit   the drafted tokens that the model's own choices confirm are found, and their keys and values, in all layers, moved behind
           those that the request holds
  mass     causal attention of every request's newest tokens that also adds up, for every key, the weight that it received
  evict    every request and kv head keeps the keys that have received the most weight, beside the first and the latest ones: what
           is kept beyond the budget moves, in all layers, into the places of what is dropped

Caches are paged as the engine lays them out: keys and values [slots, kv heads, head size], slot = page * page size + offset, a block
table a request; the pages of a case come in no order.  Weights of keys and positions are [kv heads, slots].
"""
import math
import random

import torch

own = False          # False: the plain form; True: the framework's kernels

HEADS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128), "tiny-a": (4, 2, 16), "tiny-b": (3, 1, 32), "single": (8, 8, 64)}
LAYERS = {"0.5b": 24, "1.5b": 28, "7b": 28, "tiny-a": 2, "tiny-b": 3, "single": 4}
VOCAB = 151936


def listed():
    return [
        # one user at a terminal whose drafts are short: nothing hides a launch
        {"name": "tree-0.5b-1x8", "kind": "tree", "model": "0.5b", "requests": 1, "context": 2048, "nodes": 8},
        # a server's step: an odd batch at different places, trees of different sizes, heads of 128
        {"name": "tree-1.5b-27-ragged", "kind": "tree", "model": "1.5b", "requests": 27, "context": 4001, "shortest": 65, "nodes": 26, "fewest": 3},
        # wide trees over long contexts of the widest model: the most arithmetic
        {"name": "tree-7b-16x64", "kind": "tree", "model": "7b", "requests": 16, "context": 8000, "nodes": 64},
        # verification in true 32 bits, small pages
        {"name": "tree-0.5b-fp32", "kind": "tree", "model": "0.5b", "dtype": "float32", "requests": 5, "context": 1103, "shortest": 77, "nodes": 21, "fewest": 4, "page": 8},
        # one user's accepted drafts: a few rows in each of 24 layers
        {"name": "commit-0.5b-1x8", "kind": "commit", "model": "0.5b", "requests": 1, "context": 2048, "nodes": 8},
        # the largest batch, odd trees, 28 layers of four kv heads
        {"name": "commit-7b-64-ragged", "kind": "commit", "model": "7b", "requests": 64, "context": 700, "shortest": 33, "nodes": 26, "fewest": 1},
        # one user's decoding step
        {"name": "mass-0.5b-1", "kind": "mass", "model": "0.5b", "requests": 1, "context": 2048},
        # a server's decoding step: an odd batch at different places
        {"name": "mass-1.5b-27-ragged", "kind": "mass", "model": "1.5b", "requests": 27, "context": 4001, "shortest": 65},
        # portions of prompts behind what their requests hold, the widest model
        {"name": "mass-7b-portions", "kind": "mass", "model": "7b", "requests": 4, "context": 1999, "shortest": 301, "rows": 2048, "fewest": 517},
        # a portion in true 32 bits
        {"name": "mass-0.5b-fp32", "kind": "mass", "model": "0.5b", "dtype": "float32", "requests": 2, "context": 131, "rows": 389, "fewest": 57},
        # a decoding step of requests at their budget: one key of every head goes in 24 layers
        {"name": "evict-0.5b-8-one", "kind": "evict", "model": "0.5b", "requests": 8, "context": 1025, "budget": 1024},
        # after their prompts: long requests thinned to a budget, short ones left alone
        {"name": "evict-7b-5-ragged", "kind": "evict", "model": "7b", "requests": 5, "context": 4001, "shortest": 811, "budget": 1024},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "commit", "mass", "mass", "evict"])
    model = rng.choice(["0.5b", "0.5b", "1.5b", "1.5b", "7b", "7b", "tiny-a", "tiny-b", "single"])
    c = {"kind": kind, "model": model, "page": rng.choice([8, 16, 16, 16, 32]), "requests": _log_int(rng, 1, 64)}
    if model.startswith("tiny") or rng.random() < 0.2:
        c["dtype"] = "float32"
    f32 = c.get("dtype") == "float32"
    # keys that the requests hold together, at most
    held = {"tree": 8192 if f32 else 120000, "mass": 8192 if f32 else 120000, "commit": 32768, "evict": 16384 >> f32 >> (model == "7b")}[kind]
    c["context"] = _log_int(rng, 1, min(2048 if f32 else 16384, max(1, held // c["requests"])))
    if c["requests"] > 1 and rng.random() < 0.7:
        c["shortest"] = rng.randint(0 if kind in ("tree", "mass") else 1, c["context"])
    if kind in ("tree", "commit"):
        c["nodes"] = _log_int(rng, 1, 64)
        if kind == "tree" and c["requests"] <= 8 and rng.random() < 0.2:
            c["nodes"], c["context"] = _log_int(rng, 65, 130), min(c["context"], 4096)
            c["shortest"] = min(c.get("shortest", c["context"]), c["context"])
        c["fewest"] = rng.randint(0 if c["requests"] > 1 else 1, c["nodes"])
    if kind == "mass" and rng.random() < 0.5:
        c["rows"] = _log_int(rng, 2, max(2, (512 if f32 else 2048) // c["requests"]))
        c["context"] = min(c["context"], 512 if f32 else 2048)
        c["shortest"] = min(c.get("shortest", c["context"]), c["context"])
        c["fewest"] = rng.randint(1, c["rows"])
    if kind == "evict":
        c["budget"] = _log_int(rng, 1, c["context"] + 1)
    return c


def _spread(low, high, n, salt):
    """``n`` numbers from ``low`` to ``high``, evenly over their logarithm and then moved a little, in no order; ``high`` is among them."""
    r = random.Random(n * 1000003 + high * 31 + salt)
    out = [high] + [max(low, min(high, int((low + 1) * ((high + 1) / (low + 1)) ** (i / max(1, n - 1))) - 1 + (r.randrange(7) if low < high else 0)))
                    for i in range(n - 1)]
    r.shuffle(out)
    return out


def _lengths(case):
    """How many keys each request holds, and how many rows it brings."""
    n = case["requests"]
    held = _spread(case.get("shortest", case["context"]), case["context"], n, 1)
    rows = case.get("nodes") or case.get("rows") or 1
    return held, _spread(case.get("fewest", rows), rows, n, 2)


def _dtype(case):
    return getattr(torch, case.get("dtype", "bfloat16"))


def _tree(r, n):
    """Every node's parent: the root is the newest confirmed token, a drafter adds children near the nodes it made last."""
    return [-1] + [r.randrange(max(0, i - 7), i) for i in range(1, n)]


def _mask_words(parents, words, r):
    """A node sees itself and its ancestors; a node in twenty is filler and sees no drafted token."""
    seen, rows = [], []
    for i, p in enumerate(parents):
        bits = (1 << i) | (seen[p] if p >= 0 else 0)
        seen.append(bits)
        bits = 0 if r.random() < 0.05 else bits
        rows.append([(((bits >> (64 * w)) & (2 ** 64 - 1)) ^ (1 << 63)) - (1 << 63) for w in range(words)])          # as signed numbers
    return rows


def _choices(r, parents, tokens):
    """What the model chooses behind each node: four times in five one of the drafted children."""
    children = [[] for _ in parents]
    for i, p in enumerate(parents[1:], 1):
        children[p].append(i)
    return [tokens[r.choice(c)] if c and r.random() < 0.8 else r.randrange(VOCAB) for c in children]


def prepare(case, seed):
    """Inputs and the index arrays that a step's metadata holds."""
    dev, dt, r = torch.device("cuda"), _dtype(case), random.Random(seed * 7919 + 17)
    g = torch.Generator(device=dev).manual_seed(seed * 1000 + 7)
    hq, hkv, hd = HEADS[case["model"]]
    page, kind = case.get("page", 16), case["kind"]
    held, rows = _lengths(case)
    if kind == "evict":
        rows = [0] * len(held)
    total = [h + n for h, n in zip(held, rows)]
    need = [-(-t // page) for t in total]
    pages = sum(need) + 3
    order = list(range(pages))
    r.shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (max(need) - n))
        at += n
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    slots, T, S = pages * page, sum(rows), len(held)
    s = {"case": case, "scale": hd ** -0.5, "page": page, "heads": (hq, hkv, hd),
         "span_row": i32([sum(rows[:i]) for i in range(S)]), "span_len": i32(rows), "span_pos": i32(held),
         "table": i32(table).reshape(S, -1), "most_rows": max(rows), "most_keys": max(total)}
    # a step's metadata once more: the request and the number of every row, and the request, number and slot of every key
    s["row_of"] = torch.tensor([(i, j) for i in range(S) for j in range(rows[i])], device=dev).reshape(-1, 2)
    j = torch.arange(max(total), device=dev)
    s["slot"] = s["table"].clamp(min=0).long()[:, j // page] * page + j % page                      # [S, keys]
    s["is_key"] = j < torch.tensor(total, device=dev)[:, None]
    s["key_of"] = s["is_key"].nonzero()
    rn = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    if kind in ("tree", "mass"):
        # every head looks the same way in the main, and a request's first key lies there: it draws weight from all queries
        way = rn(hkv, hd)
        way = 2.0 * way / way.norm(dim=-1, keepdim=True)
        s["q"] = (rn(T, hkv, hq // hkv, hd) + way[:, None]).reshape(T, hq * hd).to(dt)
        k = rn(slots, hkv, hd)
        if T:
            k[s["slot"][s["is_key"][:, 0], 0]] += 1.5 * hd ** 0.5 * way / 2.0
        s["k"], s["v"] = k.to(dt), (rn(slots, hkv, hd) + 0.2).to(dt)
        s["out"] = torch.empty_like(s["q"])
    if kind == "tree":
        words = max(1, -(-max(rows) // 64))
        masks = [m for n in rows if n for m in _mask_words(_tree(r, n), words, r)]
        s["mask"] = torch.tensor(masks, dtype=torch.int64, device=dev).reshape(T, words)
    if kind == "mass":
        # (of the size of what a step adds, so that a difference in either shows)
        s["mass"], s["mass_out"] = 0.01 * rn(hkv, slots).square(), torch.zeros((hkv, slots), device=dev)
    if kind in ("commit", "evict"):
        layers = LAYERS[case["model"]]
        shape = (layers, slots, hkv, hd)
        s["k"], s["v"] = (torch.randn(shape, generator=g, device=dev, dtype=dt) for _ in range(2))
    if kind == "commit":
        trees = [_tree(r, n) if n else [] for n in rows]
        tokens = [[r.randrange(VOCAB) for _ in t] for t in trees]
        s["parents"], s["tokens"] = i32([p for t in trees for p in t]), i32([x for t in tokens for x in t])
        s["targets"] = i32([x for t, k in zip(trees, tokens) for x in _choices(r, t, k)])
        s["path"] = torch.empty((S, max(1, max(rows))), dtype=torch.int32, device=dev)
        s["count"], s["next"] = (torch.empty(S, dtype=torch.int32, device=dev) for _ in range(2))
    if kind == "evict":
        # weights as many steps leave them: a few keys have most of it; some never received any that 32 bits show
        mass = torch.exp(2.5 * rn(layers, hkv, slots) - 4.0)
        s["mass"] = torch.where(rn(layers, hkv, slots) > 1.9, 0.0, mass)
        # requests have dropped keys before: a place's position says nothing of its order among the places
        gone = torch.randint(0, 400, (S,), generator=g, device=dev)
        late = torch.argsort(torch.rand((layers, S, hkv, max(total)), generator=g, device=dev).masked_fill(~s["is_key"][None, :, None], 2.0), dim=-1)
        place = torch.argsort(late, dim=-1) + gone[None, :, None, None]
        s["positions"] = torch.zeros((layers, hkv, slots), dtype=torch.int32, device=dev)
        at, key = s["key_of"], s["slot"][s["is_key"]]
        s["positions"][:, :, key] = place[:, at[:, 0], :, at[:, 1]].permute(1, 2, 0).to(torch.int32)
        s["mass_out"], s["positions_out"] = torch.zeros_like(s["mass"]), torch.zeros_like(s["positions"])
        s["ends"] = (s["span_pos"] + gone).to(torch.int32)
        s["keep"] = (min(4, case["budget"] // 2), min(128, case["budget"] // 2))          # how many of the first and of the latest positions stay
    return s


def run(s):
    kind = s["case"]["kind"]
    return (_own if own else _plain)[kind](s)


# ---- the plain forms ------------------------------------------------------------------------------------------------------
def _weights(s, visible):
    """Softmax weights of every row, [S, kv heads, group * rows, keys], 0 in rows that see nothing, and the values, in 32 bits."""
    hq, hkv, hd = s["heads"]
    S, C = s["slot"].shape
    N = s["most_rows"]
    q = torch.zeros((S, N, hq, hd), device=s["q"].device)
    q[s["row_of"][:, 0], s["row_of"][:, 1]] = s["q"].float().reshape(-1, hq, hd)
    k = s["k"][s["slot"]].float().masked_fill(~s["is_key"][..., None, None], 0.0)
    v = s["v"][s["slot"]].float().masked_fill(~s["is_key"][..., None, None], 0.0)
    x = q.reshape(S, N, hkv, hq // hkv, hd).permute(0, 2, 3, 1, 4).reshape(S, hkv, -1, hd) @ k.permute(0, 2, 3, 1) * s["scale"]
    x = x.reshape(S, hkv, hq // hkv, N, C).masked_fill(~visible[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0.0, 1.0)
    return p.reshape(S, hkv, -1, C), v.permute(0, 2, 1, 3)


def _rows_out(s, p, v):
    hq, hkv, hd = s["heads"]
    o = (p @ v).reshape(p.shape[0], hkv, hq // hkv, s["most_rows"], hd).permute(0, 3, 1, 2, 4)
    return o[s["row_of"][:, 0], s["row_of"][:, 1]].reshape(-1, hq * hd).to(s["q"].dtype)


def _plain_tree(s):
    S, C = s["slot"].shape
    N, j = s["most_rows"], torch.arange(C, device=s["q"].device)
    words = torch.zeros((S, N, s["mask"].shape[1]), dtype=torch.int64, device=j.device)
    words[s["row_of"][:, 0], s["row_of"][:, 1]] = s["mask"]
    node = j - s["span_pos"].long()[:, None]                                    # [S, C]: negative for what the request holds
    drafted = (node >= 0) & s["is_key"]
    n = node.clamp(0, words.shape[-1] * 64 - 1)
    bits = (words.gather(2, (n // 64)[:, None].expand(S, N, C)) >> (n % 64)[:, None]) & 1
    visible = (node < 0)[:, None] | (drafted[:, None] & (bits == 1))
    return _rows_out(s, *_weights(s, visible))


def _plain_mass(s):
    S, C = s["slot"].shape
    hkv = s["heads"][1]
    j, i = torch.arange(C, device=s["q"].device), torch.arange(s["most_rows"], device=s["q"].device)
    visible = (j <= s["span_pos"].long()[:, None, None] + i[:, None]) & (i < s["span_len"].long()[:, None])[..., None]
    p, v = _weights(s, visible)
    at, key = s["key_of"], s["slot"][s["key_of"][:, 0], s["key_of"][:, 1]]
    before = s["mass"][:, key] * (at[:, 1] < s["span_pos"].long()[at[:, 0]])
    s["mass_out"][:, key] = before + p.sum(2)[at[:, 0], :, at[:, 1]].reshape(-1, hkv).T
    return {"out": _rows_out(s, p, v), "mass": s["mass_out"]}


def _plain_commit(s):
    S, width = s["path"].shape
    N, n, row = s["most_rows"], s["span_len"].long(), s["span_row"].long()
    i = torch.arange(N, device=n.device)
    rows = (row[:, None] + i).clamp(max=s["tokens"].numel() - 1)
    parent = s["parents"][rows].long()
    up = parent.clamp(min=0)
    fits = (s["tokens"][rows] == s["targets"][rows].gather(1, up)) & (parent >= 0) & (parent < i) & (i < n[:, None])
    # of several children that fit the first one goes on
    earlier = (parent[:, :, None] == parent[:, None]) & fits[:, None] & (i < i[:, None])
    on = (fits & ~earlier.any(-1)) | ((i == 0) & (n > 0)[:, None])
    for _ in range(N.bit_length()):          # confirmed together with all nodes above it: ancestors twice as far each time
        on, up = on & on.gather(1, up), up.gather(1, up)
    count = on.sum(1)
    path = on.byte().sort(dim=1, descending=True, stable=True).indices[:, :width]
    d = torch.arange(path.shape[1], device=n.device)
    path = torch.where(d < count[:, None], path, -1)
    s["path"].copy_(path)
    s["count"].copy_(count)
    last = rows.gather(1, path.amax(1, keepdim=True).clamp(min=0))[:, 0]
    s["next"].copy_(torch.where(count > 0, s["targets"][last], -1))
    # a confirmed node's row moves to its place on the path; what has no place is the root, which stays where it is
    there, here = (torch.where(path >= 0, s["span_pos"].long()[:, None] + x, s["span_pos"].long()[:, None]) for x in (path, d))
    src, dst = (s["slot"].gather(1, x.clamp(max=s["slot"].shape[1] - 1))[n > 0].reshape(-1) for x in (there, here))
    s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
    return {"path": s["path"], "count": s["count"], "next": s["next"], "k": s["k"], "v": s["v"]}


def _plain_evict(s):
    budget, (first, latest) = s["case"]["budget"], s["keep"]
    L, hkv = s["mass"].shape[:2]
    S, C = s["slot"].shape
    h = torch.arange(hkv, device=s["mass"].device)
    mass = s["mass"][:, h[:, None, None], s["slot"]]                                   # [L, kv heads, S, places]
    pos = s["positions"][:, h[:, None, None], s["slot"]]
    stays = (pos < first) | (pos >= s["ends"][:, None] - latest)
    worth = torch.where(stays, math.inf, mass).masked_fill(~s["is_key"], -math.inf)
    rank = worth.sort(dim=-1, descending=True, stable=True).indices.argsort(dim=-1)
    kept = (rank < budget) & s["is_key"]
    place = torch.arange(C, device=h.device)
    hole, filler = ~kept & s["is_key"] & (place < budget), kept & (place >= budget)
    # the i-th hole takes the i-th kept place beyond the budget
    M = max(1, min(C, max(0, C - budget)))
    dst = hole.byte().sort(dim=-1, descending=True, stable=True).indices[..., :M]
    src = filler.byte().sort(dim=-1, descending=True, stable=True).indices[..., :M]
    # (rows of fewer moves repeat their first one; without any, a place that stays is moved onto itself)
    moves = torch.arange(M, device=h.device) < hole.sum(-1, keepdim=True)
    idle = kept.byte().argmax(-1, keepdim=True)
    dst, src = (torch.where(moves, x, torch.where(moves[..., :1], x[..., :1], idle)) for x in (dst, src))
    req = torch.arange(S, device=h.device)[:, None]
    dst, src = s["slot"][req, dst], s["slot"][req, src]
    layer, head = torch.arange(L, device=h.device)[:, None, None, None], h[:, None, None]
    for cache in (s["k"], s["v"]):
        cache[layer, dst, head] = cache[layer, src, head]
    at, key = s["key_of"], s["slot"][s["key_of"][:, 0], s["key_of"][:, 1]]
    key = torch.where(at[:, 1] < budget, key, key[0])          # (the first place is among those that stay in any case)
    for new, old in ((s["mass_out"], s["mass"]), (s["positions_out"], s["positions"])):
        new[:, :, key] = old[:, :, key]
        new[layer, head, dst] = old[layer, head, src]
    return {"k": s["k"], "v": s["v"], "mass": s["mass_out"], "positions": s["positions_out"]}


_plain = {"tree": _plain_tree, "mass": _plain_mass, "commit": _plain_commit, "evict": _plain_evict}


# ---- the framework's calls --------------------------------------------------------------------------------------------------
def _own_tree(s):
    from lightllm_b200.csrc import ops
    ops.tree_attention(s["q"], s["k"], s["v"], s["out"], s["mask"], s["span_row"], s["span_len"], s["span_pos"], s["table"], s["page"],
                       *s["heads"], s["scale"])
    return s["out"]


def _own_mass(s):
    from lightllm_b200.csrc import ops
    ops.paged_attention_mass(s["q"], s["k"], s["v"], s["out"], s["mass_out"], s["span_row"], s["span_len"], s["span_pos"], s["table"],
                             s["page"], *s["heads"], s["scale"], s["most_rows"], mass_in=s["mass"])
    return {"out": s["out"], "mass": s["mass_out"]}


def _own_commit(s):
    from lightllm_b200.csrc import ops
    ops.tree_commit(s["tokens"], s["parents"], s["targets"], s["k"], s["v"], s["span_row"], s["span_len"], s["span_pos"], s["table"],
                    s["page"], s["path"], s["count"], s["next"])
    return {"path": s["path"], "count": s["count"], "next": s["next"], "k": s["k"], "v": s["v"]}


def _own_evict(s):
    from lightllm_b200.csrc import ops
    ops.cache_evict(s["k"], s["v"], s["mass"], s["positions"], s["span_pos"], s["ends"], s["table"], s["page"], s["case"]["budget"],
                    *s["keep"], mass_out=s["mass_out"], positions_out=s["positions_out"])
    return {"k": s["k"], "v": s["v"], "mass": s["mass_out"], "positions": s["positions_out"]}


_own = {"tree": _own_tree, "mass": _own_mass, "commit": _own_commit, "evict": _own_evict}


# ---- work, and the definition in 64 bits --------------------------------------------------------------------------------------
def work(case):
    hq, hkv, hd = HEADS[case["model"]]
    e = 4 if case.get("dtype") == "float32" else 2
    held, rows = _lengths(case)
    kind = case["kind"]
    if kind in ("tree", "mass"):
        keys, T = sum(h + n for h, n in zip(held, rows) if n), sum(rows)
        nbytes = 2 * T * hq * hd * e + 2 * keys * hkv * hd * e
        if kind == "tree":
            # besides what its request holds a node sees itself and its ancestors: about one for every four nodes before it
            pairs = sum(n * (h + 1 + n / 8) for h, n in zip(held, rows))
            nbytes += 8 * T * -(-max(rows) // 64)
        else:
            pairs = sum(n * (h + (n + 1) / 2) for h, n in zip(held, rows))
            nbytes += 8 * keys * hkv
        return {"bytes": nbytes, "flops": 4 * hd * hq * pairs}
    layers = LAYERS[case["model"]]
    if kind == "commit":
        r, moved = random.Random(1), 0
        for n in rows:
            tree = _tree(r, n) if n else []
            tokens = [r.randrange(VOCAB) for _ in tree]
            goes_on, last, d = _choices(r, tree, tokens), 0, 0
            while True:
                last = next((i for i in range(last + 1, n) if tree[i] == last and tokens[i] == goes_on[last]), None)
                if last is None:
                    break
                d += 1
                moved += last != d
        return {"bytes": 12 * sum(rows) + 4 * moved * layers * hkv * hd * e, "flops": 0}
    over = [h for h in held if h > case["budget"]]
    moved = sum(case["budget"] * (h - case["budget"]) / h for h in over)          # of keys in no order so many lie beyond the budget
    kept = sum(min(h, case["budget"]) for h in held)
    return {"bytes": layers * hkv * (8 * sum(held) + 8 * kept + 4 * moved * hd * e), "flops": 0}


def exact(case, seed):
    """Attention request by request in 64 bits; what only moves has no such value."""
    if case["kind"] not in ("tree", "mass"):
        return None
    s = prepare(case, seed)
    hq, hkv, hd = s["heads"]
    held, rows = _lengths(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    mass = torch.zeros((hkv, s["k"].shape[0]), dtype=torch.float64, device=s["q"].device)
    first = 0
    for i, (h, n) in enumerate(zip(held, rows)):
        key = s["slot"][i, :h + n]
        if case["kind"] == "mass":
            mass[:, key[:h]] = s["mass"][:, key[:h]].double()
        if not n:
            continue
        q, k, v = s["q"][first:first + n].double().view(n, hq, hd), s["k"][key].double(), s["v"][key].double()
        sees = torch.ones((n, h + n), dtype=torch.bool, device=key.device)
        if case["kind"] == "tree":
            for a in range(n):
                sees[:, h + a] = (s["mask"][first:first + n, a // 64] >> (a % 64)) & 1 == 1
        else:
            sees[:, h:] = torch.ones((n, n), dtype=torch.bool, device=key.device).tril()
        for head in range(hq):
            x = torch.einsum("nd,kd->nk", q[:, head], k[:, head * hkv // hq]) * s["scale"]
            x = torch.where(sees, x, -math.inf)
            p = torch.where(sees.any(1, keepdim=True), torch.softmax(x, dim=1), 0.0)
            out[first:first + n, head * hd:(head + 1) * hd] = p @ v[:, head * hkv // hq]
            mass[head * hkv // hq, key] += p.sum(0)
        first += n
    return out if case["kind"] == "tree" else {"out": out, "mass": mass}
