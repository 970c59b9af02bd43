"""Operators of a step that checks drafted tokens, as cases that can be timed and checked.

A request brings a tree of drafted tokens to a step: token 0 is the last one it was given, every
other is a guess at what follows its parent.  The step's life, each part an operator here:

* ``attention``: every token of the tree attends to its request's cached keys and to the tokens of
  the tree that a bit mask names (itself and its ancestors), whose keys lie behind the cached ones.
* ``verify``: which guesses stand, by given random numbers, so that the tokens are distributed as
  the target model's own samples; and the next token, from what is left of the distribution.
* ``keep``: the cached rows of the path that stands move together, behind the cached ones.
* ``copy``: whole pages of every layer, for a request that goes on from the middle of a page.

Sizes are those of the repository's own benchmark shapes.  Each kind has a plain form in elementary
tensor operations and the same calls of the package's operators.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
SHAPES = {  # heads, key/value heads, coordinates of a cached row
    "llama-2-7b": (32, 32, 128),
    "llama-2-7b grouped": (32, 8, 128),      # four query heads a key/value head
    "openllama-3b": (32, 32, 112),           # heads of 100, held in rows of 112
    "llama-2-13b": (40, 40, 128),
}
VOCAB = 32000
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------ the cases

def _attention(shape, requests, nodes, low, high, page=16, dtype="bfloat16"):
    return dict(kind="attention", shape=shape, requests=requests, nodes=nodes, low=low, high=high,
                page=page, dtype=dtype)


def _verify(requests, nodes, vocab, draft, replacement=False, greedy=0):
    return dict(kind="verify", requests=requests, nodes=nodes, vocab=vocab, draft=draft,
                replacement=replacement, greedy=greedy)


def _keep(shape, layers, requests, nodes, most, page=16, dtype="bfloat16"):
    return dict(kind="keep", shape=shape, layers=layers, requests=requests, nodes=nodes, most=most,
                page=page, dtype=dtype)


def _copy(shape, layers, pages, page=16, dtype="bfloat16"):
    return dict(kind="copy", shape=shape, layers=layers, pages=pages, page=page, dtype=dtype)


def listed():
    return [
        # one user's chat turn, a short chain of guesses: latency
        dict(name="attention 1x8", **_attention("llama-2-7b", 1, 8, 509, 509)),
        # the batch of the headline decode step, trees of up to 32 guesses
        dict(name="attention 8x32", **_attention("llama-2-7b", 8, 32, 512, 767)),
        # a full serving batch at contexts of all lengths, small trees
        dict(name="attention 64x16", **_attention("llama-2-7b", 64, 16, 128, 2303)),
        # one long document, a wide tree, query heads that share keys, larger pages
        dict(name="attention long 1x64", **_attention("llama-2-7b grouped", 1, 64, 32701, 32701,
                                                      page=32)),
        # the 32-bit path
        dict(name="attention float32 4x24", **_attention("openllama-3b", 4, 24, 200, 1151,
                                                         dtype="float32")),
        # one user, a chain from a small draft model
        dict(name="verify 1x8", **_verify(1, 8, VOCAB, True, replacement=True)),
        # a full serving batch with trees, guesses drawn without putting back
        dict(name="verify 64x32", **_verify(64, 32, VOCAB, True)),
        # guesses looked up in the prompt, no draft model; some requests decode greedily
        dict(name="verify lookup 32x16", **_verify(32, 16, VOCAB, False, greedy=8)),
        # one user's accepted guesses, all layers of the model
        dict(name="keep 1x8", **_keep("llama-2-7b", 32, 1, 16, 4)),
        # a serving batch's
        dict(name="keep 32x32", **_keep("llama-2-7b", 32, 32, 32, 6)),
        # a request is forked in the middle of a page
        dict(name="copy 1", **_copy("llama-2-7b", 32, 1)),
        # many are
        dict(name="copy 64", **_copy("llama-2-7b", 32, 64)),
    ]


def _between(rng, low, high):
    """A whole number, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "verify", "verify", "keep", "copy"])
    shape = rng.choice(sorted(SHAPES))
    dtype = "float32" if rng.random() < 0.25 else "bfloat16"
    page = rng.choice([16, 16, 32, 64])
    heads, kv_heads, dim = SHAPES[shape]
    if kind == "attention":
        requests, nodes = _between(rng, 1, 64), _between(rng, 1, 64)
        # cached tokens a request: no more bytes, and no more products, than the largest listed
        budget = min(64 * 1200 * 32 * 128 // (kv_heads * dim * requests),
                     64 * 32 * 32701 // (heads * requests * nodes))
        if dtype == "float32":
            budget //= 8
        high = _between(rng, 4, max(5, min(32768, budget)))
        low = rng.choice([high, rng.randint(0, high), high // 2])
        return _attention(shape, requests, nodes, low, high, page, dtype)
    if kind == "verify":
        requests, nodes = _between(rng, 1, 64), _between(rng, 1, 48)
        vocab = rng.choice([VOCAB, VOCAB, _between(rng, 300, 130000)])
        if requests * nodes * vocab > 64 * 32 * VOCAB:
            requests = max(1, 64 * 32 * VOCAB // (nodes * vocab))
        return _verify(requests, nodes, vocab, rng.random() < 0.7, rng.random() < 0.4,
                       rng.choice([0, 0, requests // 3]))
    layers = _between(rng, 1, 32)
    if kind == "keep":
        requests = _between(rng, 1, 32)
        if dtype == "float32" or page > 16:
            requests = max(1, requests // 4)
        most = _between(rng, 1, 16)
        return _keep(shape, layers, requests, 2 * most + rng.randint(0, 31), most, page, dtype)
    pages = _between(rng, 1, 64) * 32 * 16 // (kv_heads * page)
    if dtype == "float32":
        pages //= 2
    return _copy(shape, layers, max(1, pages), page, dtype)


# ------------------------------------------------------------- inputs, made from the seed alone

def _rng(case, seed=None):
    """Of a case and a seed; without one, what is the same for every seed (sizes)."""
    words = "|".join(f"{key}={case[key]}" for key in sorted(case) if key != "name")
    return random.Random(f"{words}/{seed}")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _sizes(case):
    """Tokens of every request's tree (the first brings the most), and its cached tokens."""
    rng, nodes = _rng(case), case["nodes"]
    sizes = [nodes] + [rng.randint(max(1, nodes // 2), nodes) for _ in range(case["requests"] - 1)]
    if case["kind"] != "attention":
        return sizes, None
    return sizes, [case["high"]] + [rng.randint(case["low"], case["high"]) for _ in sizes[1:]]


def _parents(count, rng):
    """A tree, parents in front of their children: chains that fork here and there."""
    return [-1] + [j - 1 if rng.random() < 0.5 else rng.randrange(max(0, j - 6), j)
                   for j in range(1, count)]


def _words(trees):
    """Bit j of a token's words: token j of its request is itself or an ancestor."""
    count = -(-max(len(tree) for tree in trees) // 64)
    rows = []
    for tree in trees:
        seen = []
        for j, parent in enumerate(tree):
            seen.append((seen[parent] if parent >= 0 else 0) | (1 << j))
        for bits in seen:
            parts = [(bits >> (64 * w)) & (2 ** 64 - 1) for w in range(count)]
            rows.append([part - 2 ** 64 if part >= 2 ** 63 else part for part in parts])
    return torch.tensor(rows, dtype=torch.int64, device=DEVICE)


def _tables(needed, pool, rng):
    """Block tables of shuffled pages, -1 behind the last."""
    order = list(range(pool))
    rng.shuffle(order)
    width, rows = max(needed), []
    for count in needed:
        rows.append([order.pop() for _ in range(count)] + [-1] * (width - count))
    return _ints(rows)


def _filled(shape, seed, dtype):
    generator = torch.Generator(device=DEVICE)
    generator.manual_seed(seed)
    out = torch.empty(shape, dtype=dtype, device=DEVICE)
    return out.normal_(generator=generator)


def prepare(case, seed):
    rng = _rng(case, seed)
    return {"attention": _prepare_attention, "verify": _prepare_verify, "keep": _prepare_keep,
            "copy": _prepare_copy}[case["kind"]](case, rng)


def _prepare_attention(case, rng):
    heads, kv_heads, dim = SHAPES[case["shape"]]
    dtype, page = DTYPES[case["dtype"]], case["page"]
    sizes, contexts = _sizes(case)
    needed = [-(-(c + n) // page) for c, n in zip(contexts, sizes)]
    pool = sum(needed) + 2
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    tokens = starts[-1]
    shape = (pool, kv_heads, page, dim)
    base = rng.randrange(1 << 30)
    return dict(case=case, requests=len(sizes), most=max(sizes), longest=max(needed) * page,
                q=_filled((tokens, heads * dim), base, dtype), k=_filled(shape, base + 1, dtype),
                v=_filled(shape, base + 2, dtype), visible=_words([_parents(n, rng) for n in sizes]),
                start=_ints(starts), context=_ints(contexts), row=_ints(list(range(len(sizes)))),
                tables=_tables(needed, pool, rng), out=torch.zeros((tokens, heads * dim), dtype=dtype,
                                                                   device=DEVICE),
                status=_ints([0]), scale=1.0 / math.sqrt(100 if dim == 112 else dim))


def _prepare_verify(case, rng):
    sizes, _ = _sizes(case)
    trees = [_parents(n, rng) for n in sizes]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    tokens, vocab = starts[-1], case["vocab"]
    base = rng.randrange(1 << 30)
    # what two language models say: most of the weight on few tokens, much alike
    logits = _filled((tokens, vocab), base, torch.float32) * 3.0
    guess = logits + _filled((tokens, vocab), base + 1, torch.float32)
    greedy = case["greedy"]
    heat = [0.0 if r < greedy else rng.uniform(0.6, 1.1) for r in range(len(sizes))]
    # the children of a token, in order: the draft's samples (a Gumbel number added to a logit
    # makes the largest a sample, the next largest one without putting back); greedy: its best
    generator = torch.Generator(device=DEVICE)
    generator.manual_seed(base + 2)
    keys = torch.empty((tokens, vocab), device=DEVICE).exponential_(generator=generator).log_().neg_()
    of_row = torch.tensor([heat[r] for r, n in enumerate(sizes) for _ in range(n)], device=DEVICE)[:, None]
    keys = torch.where(of_row > 0, guess / of_row.clamp(min=0.1) + keys, guess)
    best = keys.topk(min(vocab, max(1, case["nodes"])), dim=1).indices
    del keys
    born, parents = [0] * tokens, []
    of_parent, rank = [], []
    for r, tree in enumerate(trees):
        for parent in tree:
            parents.append(parent)
            at = starts[r] + max(parent, 0)
            of_parent.append(at)
            rank.append(0 if parent < 0 else born[at])
            if parent >= 0:
                born[at] += 1
    ids = best[torch.tensor(of_parent, device=DEVICE), torch.tensor(rank, device=DEVICE)]
    uniform = torch.rand(tokens, generator=generator, device=DEVICE)
    return dict(case=case, requests=len(sizes), most=max(sizes), logits=logits,
                guess=guess if case["draft"] else None, ids=ids.to(torch.int32), parents=_ints(parents),
                start=_ints(starts), heat=torch.tensor(heat, dtype=torch.float32, device=DEVICE),
                uniform=uniform, path=torch.zeros((len(sizes), max(sizes)), dtype=torch.int32, device=DEVICE),
                kept=_ints([0] * len(sizes)), following=_ints([0] * len(sizes)), status=_ints([0]))


def _prepare_keep(case, rng):
    heads, kv_heads, dim = SHAPES[case["shape"]]
    page, nodes, most = case["page"], case["nodes"], case["most"]
    fixed = _rng(case)
    contexts = [fixed.randint(0, 2 * page) for _ in range(case["requests"])]
    needed = [-(-(c + nodes) // page) for c in contexts]
    # the way down a tree laid out branch by branch: the first branch as far as it stands, then a
    # later one, behind where the kept rows go (so that the same call again changes nothing)
    paths, kept = [], []
    for _ in contexts:
        count = rng.randint(max(1, most // 2), most)
        same = rng.randint(1, count)
        later = sorted(rng.sample(range(count, nodes), count - same))
        paths.append(list(range(same)) + later + [-1] * (most - count))
        kept.append(count)
    shape = (case["layers"], 2, sum(needed) + 1, kv_heads, page, dim)
    return dict(case=case, requests=len(contexts), storage=_filled(shape, rng.randrange(1 << 30),
                                                                   DTYPES[case["dtype"]]),
                tables=_tables(needed, sum(needed) + 1, rng), row=_ints(list(range(len(contexts)))),
                context=_ints(contexts), path=_ints(paths), kept=_ints(kept), status=_ints([0]))


def _prepare_copy(case, rng):
    heads, kv_heads, dim = SHAPES[case["shape"]]
    pages = case["pages"]
    order = list(range(2 * pages + 1))
    rng.shuffle(order)
    shape = (case["layers"], 2, 2 * pages + 1, kv_heads, case["page"], dim)
    return dict(case=case, storage=_filled(shape, rng.randrange(1 << 30), DTYPES[case["dtype"]]),
                source=_ints(order[:pages]), target=_ints(order[pages:2 * pages]), status=_ints([0]))


# ------------------------------------------------------------------------------------- a pass

def run(state):
    return {"attention": _run_attention, "verify": _run_verify, "keep": _run_keep,
            "copy": _run_copy}[state["case"]["kind"]](state)


def _run_attention(s):
    heads, kv_heads, dim = SHAPES[s["case"]["shape"]]
    if own:
        from helix_runtime_b200.ops import library as ops
        if "partial" not in s:      # scratch that a server keeps from step to step
            s["partial"] = torch.empty(
                ops.tree_attention_scratch(s["q"].dtype, heads, kv_heads, dim, s["case"]["page"]),
                dtype=torch.float32, device=s["q"].device)
        ops.tree_attention(s["q"], s["k"], s["v"], s["visible"], s["start"], s["context"], s["row"],
                           s["tables"], s["out"], s["partial"], s["requests"], heads, kv_heads, dim,
                           s["case"]["page"], s["k"].shape[0], s["scale"], s["status"])
        return s["out"]
    # every request padded to the largest tree and the longest context
    requests, most, longest = s["requests"], s["most"], s["longest"]
    start, context = s["start"].long(), s["context"].long()
    sizes = start[1:] - start[:-1]
    node = torch.arange(most, device=DEVICE)
    rows = (start[:-1, None] + node).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(requests, most, kv_heads, heads // kv_heads, dim)
    keys, values = (_unpaged(s[name], s["tables"], s["row"]).float() for name in ("k", "v"))
    place = torch.arange(longest, device=DEVICE) - context[:, None]           # [R, C]; tree: from 0
    words = s["visible"][rows]                                                # [R, T, W]
    bit = place.clamp(min=0, max=64 * words.shape[2] - 1)
    shifted = words.gather(2, (bit // 64)[:, None].expand(-1, most, -1)) >> (bit % 64)[:, None]
    seen = (place < 0)[:, None] | ((shifted & 1 == 1) & (place < sizes[:, None])[:, None])
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(requests, kv_heads, -1, dim),
                          keys.transpose(2, 3)) * s["scale"]
    scores = scores.view(requests, kv_heads, -1, most, longest)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    weights = weights / torch.where(total == 0.0, 1.0, total)
    used = (torch.arange(longest, device=DEVICE) < (context + sizes)[:, None])[:, None, :, None]
    mixed = torch.matmul(weights.view(requests, kv_heads, -1, longest), torch.where(used, values, 0.0))
    mixed = mixed.view(requests, kv_heads, -1, most, dim).permute(0, 3, 1, 2, 4)
    request = torch.searchsorted(start[1:], torch.arange(s["q"].shape[0], device=DEVICE), right=True)
    mine = torch.arange(s["q"].shape[0], device=DEVICE) - start[request]
    return mixed[request, mine].reshape(s["q"].shape).to(s["q"].dtype)


def _unpaged(cache, tables, rows):
    """[requests, kv head, place, coordinate] of the pages that the requests' tables name."""
    pages, kv_heads, page, dim = cache.shape
    piece = 16 // cache.element_size()
    found = cache.view(pages, kv_heads, dim // piece, page, piece)[tables[rows.long()].long().clamp(min=0)]
    found = found.permute(0, 2, 1, 4, 3, 5)          # [R, kv head, page, slot, D / piece, piece]
    return found.reshape(found.shape[0], kv_heads, -1, dim)


def _shares(logits, heat):
    """softmax(logits / heat) in 64 bits."""
    raised = logits.double() / heat[:, None]
    raised = torch.exp(raised - raised.amax(1, keepdim=True))
    return raised / raised.sum(1, keepdim=True)


def _run_verify(s):
    if own:
        from helix_runtime_b200.ops import library as ops
        ops.verify_drafts(s["logits"], s["guess"], s["ids"], s["parents"], s["start"], s["heat"],
                          s["uniform"], s["path"], s["kept"], s["following"], s["requests"],
                          s["status"], replacement=s["case"]["replacement"])
        return dict(path=s["path"], kept=s["kept"], following=s["following"])
    requests, most = s["requests"], s["most"]
    start = s["start"].long()
    sizes = start[1:] - start[:-1]
    begin = start[:-1]
    every = torch.arange(requests, device=DEVICE)
    greedy = s["heat"] <= 0.0
    heat = torch.where(greedy, 1.0, s["heat"]).double()
    uniform = s["uniform"].double()
    ids, parents = s["ids"].long(), s["parents"].long()
    last = s["logits"].shape[0] - 1
    at = torch.zeros(requests, dtype=torch.long, device=DEVICE)          # the token stood on
    path = torch.full((requests, most), -1, dtype=torch.int32, device=DEVICE)
    path[:, 0] = 0
    kept = torch.ones(requests, dtype=torch.long, device=DEVICE)
    # what is left of the distribution: max(p - taken * q, 0) / left; without a draft model p
    # without the tokens that fell, over `left`
    taken = torch.zeros(requests, dtype=torch.float64, device=DEVICE)
    left, gone = torch.ones_like(taken), torch.zeros_like(taken)
    fell = torch.zeros((requests, s["case"]["vocab"]), dtype=torch.bool, device=DEVICE)
    p, q = _shares(s["logits"][begin], heat), None
    best = s["logits"][begin].argmax(1)
    if s["guess"] is not None:
        q = _shares(s["guess"][begin], heat)
    # children have higher numbers than their parent, and siblings are tried in order: one walk
    for node in range(1, most):
        row = (begin + node).clamp(max=last)
        child = (parents[row] == at) & (node < sizes)
        token, u = ids[row], uniform[row]
        p_token = p[every, token]
        if q is None:
            stands = (u * left < p_token) & ~fell[every, token]
        else:
            rest = 1.0 - gone if not s["case"]["replacement"] else torch.ones_like(gone)
            factor = torch.where(rest > 0.0, 1.0 / rest, 0.0)
            q_token = q[every, token]
            stands = (u * q_token * factor * left < p_token - taken * q_token) & (rest > 0.0)
        stands = child & torch.where(greedy, token == best, stands)
        falls = child & ~stands & ~greedy
        if q is None:
            first = falls & ~fell[every, token]
            left = torch.where(first, left - p_token, left)
            fell[every, token] |= falls
        else:
            taken = torch.where(falls, taken + left * factor, taken)
            gone = torch.where(falls, gone + q_token, gone)
            over = (p - taken[:, None] * q).clamp(min=0.0).sum(1)
            left = torch.where(falls, over, left)
        path[every, torch.where(stands, kept, 0)] = torch.where(stands, node, 0).to(torch.int32)
        kept = kept + stands
        at = torch.where(stands, node, at)
        taken = torch.where(stands, 0.0, taken)
        left = torch.where(stands, 1.0, left)
        gone = torch.where(stands, 0.0, gone)
        fell &= ~stands[:, None]
        p = _shares(s["logits"][begin + at], heat)
        best = s["logits"][begin + at].argmax(1)
        if q is not None:
            q = _shares(s["guess"][begin + at], heat)
    weights = p.masked_fill(fell, 0.0) if q is None else (p - taken[:, None] * q).clamp(min=0.0)
    weights = torch.where((weights.sum(1) > 0.0)[:, None], weights, p)
    reached = weights.cumsum(1)
    # the first token whose running sum exceeds the number
    drawn = (reached <= uniform[begin][:, None] * reached[:, -1:]).sum(1)
    following = torch.where(greedy, best, drawn)
    return dict(path=path, kept=kept.to(torch.int32), following=following.to(torch.int32))


def _run_keep(s):
    storage = s["storage"]
    layers, _, pages, kv_heads, page, dim = storage.shape
    if own:
        from helix_runtime_b200.ops import library as ops
        ops.keep_rows(storage, s["tables"], s["row"], s["context"], s["path"], s["kept"], s["requests"],
                      s["status"])
        return storage
    piece = 16 // storage.element_size()
    pieces = storage.view(layers, 2, pages, kv_heads, dim // piece, page, piece)
    order = torch.arange(s["path"].shape[1], device=DEVICE)
    stays = order < s["kept"][:, None]
    # a row that is not kept: the first row moved onto itself
    old = s["context"].long()[:, None] + torch.where(stays, s["path"].long(), s["path"][:, :1].long())
    new = s["context"].long()[:, None] + torch.where(stays, order, s["path"][:, :1].long())
    table = s["tables"][s["row"].long()].long()
    old_page, new_page = (table.gather(1, place // page).reshape(-1) for place in (old, new))
    old_slot, new_slot = ((place % page).reshape(-1) for place in (old, new))
    moved = pieces[:, :, old_page, :, :, old_slot]
    pieces[:, :, new_page, :, :, new_slot] = moved
    return storage


def _run_copy(s):
    storage = s["storage"]
    if own:
        from helix_runtime_b200.ops import library as ops
        ops.copy_pages(storage, s["source"], s["target"], s["status"])
        return storage
    storage[:, :, s["target"].long()] = storage[:, :, s["source"].long()]
    return storage


# ------------------------------------------------------------------------------------- the work

def work(case):
    heads, kv_heads, dim = SHAPES.get(case.get("shape"), (0, 0, 0))
    size = 4 if case.get("dtype") == "float32" else 2
    requests = case.get("requests", 1)
    if case["kind"] == "attention":
        sizes, contexts = _sizes(case)
        pairs = sum(n * (c + n) for n, c in zip(sizes, contexts))
        cached = sum(n + c for n, c in zip(sizes, contexts))
        return dict(bytes=2 * size * dim * (kv_heads * cached + heads * sum(sizes)),
                    flops=4 * heads * dim * pairs)
    if case["kind"] == "verify":
        # the rows of the first token, and the one that the next token is drawn from
        rows = 1 if case["nodes"] == 1 else 3 if case["draft"] else 2
        return dict(bytes=4 * requests * rows * case["vocab"], flops=8 * requests * rows * case["vocab"])
    if case["kind"] == "keep":
        rows = requests * max(1, case["most"] // 2)
        return dict(bytes=2 * 2 * rows * case["layers"] * kv_heads * dim * size, flops=0)
    return dict(bytes=2 * 2 * case["pages"] * case["layers"] * kv_heads * case["page"] * dim * size, flops=0)


# ----------------------------------------------------------------------------- 64 bits, apart

def exact(case, seed):
    if case["kind"] == "attention":
        return _exact_attention(prepare(case, seed))
    if case["kind"] == "verify":
        return _exact_verify(prepare(case, seed))
    return None          # rows that are moved are not computed


def _exact_attention(s):
    heads, kv_heads, dim = SHAPES[s["case"]["shape"]]
    page, start = s["case"]["page"], s["start"].tolist()
    piece = 16 // s["k"].element_size()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for r, context in enumerate(s["context"].tolist()):
        begin, end = start[r], start[r + 1]
        count = end - begin
        pages = s["tables"][r][:-(-(context + count) // page)].long()
        rows = []
        for cache in (s["k"], s["v"]):
            blocks = cache[pages].view(len(pages), kv_heads, dim // piece, page, piece)
            rows.append(blocks.permute(1, 0, 3, 2, 4).reshape(kv_heads, -1, dim)[:, :context + count].double())
        bits = np.array(s["visible"][begin:end].cpu().numpy(), dtype="<i8").view(np.uint8).reshape(count, -1)
        tree = np.unpackbits(bits, axis=1, bitorder="little")[:, :count].astype(bool)
        seen = torch.ones((count, context + count), dtype=torch.bool, device=DEVICE)
        seen[:, context:] = torch.from_numpy(tree).to(DEVICE)
        q = s["q"][begin:end].double().view(count, kv_heads, heads // kv_heads, dim)
        for h in range(heads // kv_heads):
            scores = torch.einsum("thd,hcd->htc", q[:, :, h], rows[0]) * s["scale"]
            shares = torch.softmax(scores.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
            mixed = torch.einsum("htc,hcd->thd", shares, rows[1])
            out[begin:end].view(count, kv_heads, heads // kv_heads, dim)[:, :, h] = mixed
    return out


def _exact_verify(s):
    vocab = s["case"]["vocab"]
    start, parents, ids = s["start"].tolist(), s["parents"].tolist(), s["ids"].tolist()
    uniform, heat = s["uniform"].double().tolist(), s["heat"].double().tolist()
    path = torch.full((s["requests"], s["most"]), -1, dtype=torch.int32)
    kept, following = [], []
    for r in range(s["requests"]):
        begin, tree = start[r], parents[start[r]:start[r + 1]]
        here, way = 0, [0]
        while True:
            row = s["logits"][begin + here].cpu().numpy().astype(np.float64)
            if heat[r] <= 0.0:
                best = int(np.argmax(row))
                found = [j for j, parent in enumerate(tree) if parent == here and ids[begin + j] == best]
                if found:
                    here = found[0]
                    way.append(here)
                    continue
                following.append(best)
                break
            rest = np.exp((row - row.max()) / heat[r])
            rest /= rest.sum()
            draft = None
            if s["guess"] is not None:
                draft = s["guess"][begin + here].cpu().numpy().astype(np.float64)
                draft = np.exp((draft - draft.max()) / heat[r])
                draft /= draft.sum()
            found = None
            for j, parent in enumerate(tree):
                if parent != here:
                    continue
                token = ids[begin + j]
                guess = np.zeros(vocab) if draft is None else draft
                if draft is None:
                    guess[token] = 1.0
                if uniform[begin + j] * guess[token] < rest[token]:
                    found = j
                    break
                rest = np.maximum(rest - guess, 0.0)
                rest /= rest.sum()
                if draft is not None and not s["case"]["replacement"]:
                    draft = draft.copy()
                    draft[token] = 0.0
                    draft /= draft.sum()
            if found is None:
                sums = np.cumsum(rest)
                following.append(int(np.searchsorted(sums, uniform[begin] * sums[-1], side="right")))
                break
            here = found
            way.append(here)
        path[r, :len(way)] = torch.tensor(way, dtype=torch.int32)
        kept.append(len(way))
    return dict(path=path, kept=torch.tensor(kept, dtype=torch.int32),
                following=torch.tensor(following, dtype=torch.int32))
