"""Attention of drafted tokens over the paged cache, against the plain form in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helix_runtime_b200.ops import library as ops
from plain_tree import Batch, ancestors, from_cache, random_parents, to_cache

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("contexts,nodes,heads,kv_heads,head_dim,page", [
    ([5], [1], 1, 1, 64, 16),                                  # one token of one head
    ([0], [1], 2, 2, 128, 16),                                 # no cached key
    ([63, 64, 65, 127, 128], [1, 1, 1, 1, 1], 4, 4, 128, 16),  # keys end at and around a tile's border
    ([100, 3], [5, 9], 4, 4, 128, 16),
    ([700, 0, 65], [20, 1, 64], 4, 1, 128, 16),                # heads that share keys; 64 and 256 rows
    ([700, 0, 65], [20, 1, 64], 4, 2, 112, 32),
    ([300, 31], [40, 7], 2, 2, 64, 64),
    ([300, 31], [140, 70], 4, 2, 96, 16),                      # more than two words of a mask
    ([33, 10], [129, 2], 2, 2, 80, 16),                        # a second tile of one row
    ([40], [9], 12, 4, 64, 32),                                # groups of three
    ([50], [3], 96, 1, 64, 16),                                # one token a tile
    ([50], [3], 260, 2, 64, 16),                               # a token's heads take two tiles
    ([50, 7], [6, 3], 2, 1, 160, 16),                          # heads of other kernels
    ([50, 7], [40, 3], 2, 1, 256, 32),
    ([50, 700], [6, 33], 4, 2, 64, 8),
    ([50, 70], [6, 33], 4, 2, 64, 24),                         # pages no tensor-core kernel takes
    ([50, 70], [6, 3], 4, 2, 100, 7),
    ([50, 70], [6, 3], 4, 2, 300, 8),
    ([50, 70], [6, 3], 4, 4, 6, 1),
    ([5000], [64], 8, 2, 128, 32),                             # one request over all CTAs
])
def test_sizes(dtype, contexts, nodes, heads, kv_heads, head_dim, page):
    for stale in (float("nan"), 0.5):      # what lies in the pages behind the last key
        batch = Batch(1, contexts, nodes, heads, kv_heads, head_dim, page, dtype, row_pad=8, stale=stale)
        batch.run(ops)
        batch.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 64])
def test_many_items_a_run(dtype, page):
    """CTAs whose runs end items, hold whole ones and begin others."""
    rng = np.random.default_rng(5)
    contexts = [int(c) for c in rng.integers(0, 900, 20)]
    nodes = [int(n) for n in rng.integers(1, 20, 20)]
    nodes[7] = 0                       # a request without tokens
    for stale in (float("nan"), 0.5):
        batch = Batch(2, contexts, nodes, 32, 32, 64, page, dtype, stale=stale)
        for most in (1, 64):               # of a kernel's choice: the streaming one, or the tensor cores'
            batch.out.fill_(7.0)
            batch.run(ops, max_nodes=most)
            batch.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_short_items_many_a_run(dtype):
    batch = Batch(3, [3] * 70, [1 + i % 5 for i in range(70)], 32, 32, 64, 16, dtype)
    batch.run(ops)
    batch.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("head_dim,page", [(64, 16), (64, 8), (6, 4)])
def test_masks(dtype, head_dim, page):
    """Tokens that see nothing, all, later tokens, none of the drafted ones, only the last."""
    rng = np.random.default_rng(7)
    count = 70
    seen = [np.zeros((count, count), dtype=bool), rng.random((count, count)) < 0.3]
    seen[0][3] = True
    seen[0][5, count - 1] = True
    seen[1][0] = False
    for contexts in ([0, 0], [130, 0], [0, 61]):
        batch = Batch(4, contexts, [count, count], 4, 4, head_dim, page, dtype, seen=seen)
        batch.run(ops)
        batch.check()
        if contexts[0] == 0:
            assert bool((batch.out[0, :4 * head_dim] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_words(dtype):
    """More words than the tokens need (bits behind the last token name nothing), and fewer."""
    for words in (1, 3):
        seen = [np.ones((90, 90), dtype=bool), np.ones((20, 20), dtype=bool)]
        batch = Batch(5, [40, 7], [90, 20], 2, 2, 64, 16, dtype, seen=seen, words=words)
        if words == 3:
            batch.visible[:] = -1
        batch.run(ops)
        batch.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("head_dim,page", [(128, 16), (128, 8), (6, 4)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_reach_who_sees_them(dtype, head_dim, page, bad):
    """A drafted key and value that are not finite change nothing for tokens that do not see them;
    a value reaches, coordinate by coordinate, those that do."""
    nodes, context = 12, 100
    seen = [ancestors([-1, 0, 0, 1, 1, 2, 2, 3, 3, 5, 5, 6])]
    clean = Batch(6, [context], [nodes], 2, 2, head_dim, page, dtype, seen=seen)
    clean.run(ops)
    batch = Batch(6, [context], [nodes], 2, 2, head_dim, page, dtype, seen=seen)
    place = context + 2                     # token 2: its branch is 2, 5, 6, 9, 10, 11
    page_id = int(batch.tables[batch.row[0], place // page])
    rows = torch.zeros((2, page, head_dim), dtype=dtype)
    rows[:, place % page, 1] = bad
    from plain_tree import to_cache
    hit = to_cache(rows, dtype).ne(0).to(batch.v.device)
    batch.v[page_id][hit] = bad
    batch.run(ops)
    branch = [2, 5, 6, 9, 10, 11]
    others = [n for n in range(nodes) if n not in branch]
    got, want = batch.out[:nodes, :2 * head_dim], clean.out[:nodes, :2 * head_dim]
    assert torch.equal(got[others], want[others])
    columns = [1, head_dim + 1]
    kept = [c for c in range(2 * head_dim) if c not in columns]
    assert torch.equal(got[branch][:, kept], want[branch][:, kept])
    reached = got[branch][:, columns]
    assert bool((reached.isnan() if bad != bad else reached == bad).all())
    batch.v.copy_(clean.v)
    batch.k[page_id][hit] = bad
    batch.run(ops)
    assert torch.equal(batch.out[:nodes][others], clean.out[:nodes][others])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("head_dim,page,nodes", [(128, 16, 12), (128, 16, 90), (128, 64, 12), (128, 24, 12), (6, 4, 12)])
def test_cached_values_that_are_not_finite_reach_every_token(dtype, head_dim, page, nodes):
    """Also where they share a tile of keys with drafted ones, and wherever the work is cut."""
    for context, place in ((100, 99), (100, 3), (40, 33)):
        batch = Batch(19, [context], [nodes], 2, 2, head_dim, page, dtype)
        clean = Batch(19, [context], [nodes], 2, 2, head_dim, page, dtype)
        clean.run(ops)
        from plain_tree import to_cache
        rows = torch.zeros((2, page, head_dim), dtype=dtype)
        rows[0, place % page, 2] = float("inf")
        rows[1, place % page, 4] = float("nan")
        laid = to_cache(rows, dtype).to(batch.v.device)
        page_id = int(batch.tables[batch.row[0], place // page])
        batch.v[page_id] = torch.where(laid.ne(0), laid, batch.v[page_id])
        batch.run(ops)
        got, want = batch.out[:nodes, :2 * head_dim], clean.out[:nodes, :2 * head_dim]
        # (a bfloat16 kernel's weight is a sum of two terms, hi + lo, of which lo may be zero or negative:
        # hi * inf + lo * inf is then not a number.  So what reaches a token is not finite, and no more)
        reached = ~got[:, 2].isfinite() if dtype == torch.bfloat16 else got[:, 2] == float("inf")
        assert bool(reached.all()) and bool(got[:, head_dim + 4].isnan().all())
        kept = [c for c in range(2 * head_dim) if c not in (2, head_dim + 4)]
        assert torch.equal(got[:, kept], want[:, kept])


@pytest.mark.parametrize("dtype", DTYPES)
def test_scratch_needs_nothing_and_is_reused(dtype):
    floats = ops.tree_attention_scratch(dtype, 4, 4, 128, 16)
    partial = torch.full((floats + 1,), float("nan"), device="cuda:0")
    for seed, contexts, nodes in ((8, [700, 20], [30, 4]), (9, [64], [1]), (10, [5000, 90, 3], [7, 60, 1])):
        batch = Batch(seed, contexts, nodes, 4, 4, 128, 16, dtype)
        batch.run(ops, partial[:floats])
        batch.check()
    assert bool(partial[floats:].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_outside_the_pool_are_reported(dtype):
    for index, wrong in ((0, -1), (3, 10 ** 6)):
        batch = Batch(11, [50, 50], [4, 4], 2, 2, 64, 16, dtype, stale=0.0)
        batch.tables[batch.row[0], index] = wrong
        batch.run(ops)
        assert int(batch.status.item()) == ops.FLAG_BAD_PAGE
        expected, weighed, largest = batch.expected()
        off = (batch.out[4:8, :128].double().cpu() - expected[4:]).abs()
        assert bool((off <= batch.tolerance(expected, weighed, largest)[4:]).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_to_do(dtype):
    batch = Batch(12, [9], [0], 2, 2, 64, 16, dtype)
    batch.run(ops)
    assert bool((batch.out == 7.0).all())
    batch.requests = 0
    batch.run(ops)
    assert bool((batch.out == 7.0).all()) and int(batch.status.item()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_graph_is_replayed_over_other_trees(dtype):
    """A recorded call reads lengths, masks and tables when it is replayed."""
    args = ([400, 90], [17, 30], 4, 4, 128, 16, dtype)
    batch = Batch(13, *args)
    partial = torch.empty(ops.tree_attention_scratch(dtype, 4, 4, 128, 16), device="cuda:0")
    batch.run(ops, partial)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.run(ops, partial)
    other = Batch(14, [33, 401], [30, 16], *args[2:])
    for name in ("q", "out", "visible", "start", "context", "row", "status"):
        mine, theirs = getattr(batch, name), getattr(other, name)
        mine[:theirs.shape[0]].copy_(theirs)
    batch.out.fill_(7.0)
    pages = min(batch.num_pages, other.num_pages)
    assert other.num_pages <= batch.num_pages and other.tables.shape[1] <= batch.tables.shape[1]
    batch.k[:pages].copy_(other.k[:pages])
    batch.v[:pages].copy_(other.v[:pages])
    batch.tables.fill_(-1)
    batch.tables[:, :other.tables.shape[1]].copy_(other.tables)
    graph.replay()
    torch.cuda.synchronize()
    other.check(batch.out[:other.out.shape[0]])


@pytest.mark.parametrize("dtype", DTYPES)
def test_other_stream(dtype):
    batch = Batch(15, [400, 90], [17, 30], 4, 4, 128, 16, dtype)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        batch.run(ops)
    stream.synchronize()
    batch.check()


def test_offsets_beyond_32_bits():
    """Pages behind the first 2^31 elements of a layer's keys and values."""
    small = Batch(16, [200, 30], [9, 20], 32, 32, 128, 64, torch.bfloat16, stale=0.0)
    pages = (1 << 31) // (32 * 64 * 128) + small.num_pages + 1
    shift = pages - small.num_pages
    for name in ("k", "v"):
        wide = torch.empty((pages, *getattr(small, name).shape[1:]), dtype=torch.bfloat16, device="cuda:0")
        wide[shift:] = getattr(small, name)
        setattr(small, name, wide)
    small.tables = torch.where(small.tables >= 0, small.tables + shift, small.tables)
    small.num_pages = pages
    small.run(ops)
    small.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_chain_is_what_causal_attention_computes(dtype):
    """Drafts in a row: the causal kernel over the same pages."""
    contexts, nodes = [77, 300], [6, 9]
    seen = [np.tril(np.ones((n, n), dtype=bool)) for n in nodes]
    batch = Batch(17, contexts, nodes, 4, 2, 128, 16, dtype, seen=seen, stale=0.0)
    batch.run(ops)
    tokens = sum(nodes)
    positions = torch.tensor([c + j for c, n in zip(contexts, nodes) for j in range(n)], dtype=torch.int32,
                             device="cuda:0")
    request = torch.tensor([r for r, n in enumerate(nodes) for _ in range(n)], dtype=torch.int32, device="cuda:0")
    causal = torch.zeros((tokens, 4 * 128), dtype=dtype, device="cuda:0")
    ops.paged_attention(batch.q, batch.k, batch.v, positions, request, batch.row, batch.tables, causal, None,
                        tokens, 4, 2, 128, 16, batch.num_pages, 0, batch.scale, 256, 2, batch.status)
    expected, weighed, largest = batch.expected()
    allowed = 2 * batch.tolerance(expected, weighed, largest)
    assert bool(((batch.out[:tokens, :512] - causal).double().cpu().abs() <= allowed).all())
    batch.check()


def test_refusals():
    batch = Batch(18, [50], [4], 2, 2, 64, 16, torch.bfloat16)
    base = dict(vars(batch))

    def refused(**changes):
        for name, value in {**base, **changes}.items():
            setattr(batch, name, value)
        with pytest.raises(ops.KernelError):
            batch.run(ops)
        assert bool((base["out"] == 7.0).all())

    refused(head_dim=63)
    refused(head_dim=1026)
    refused(kv_heads=3)
    refused(page_size=0)
    refused(num_pages=0)
    refused(scale=0.0)
    refused(scale=-1.0)
    refused(heads=0)
    refused(visible=batch.visible.to(torch.int32))
    refused(visible=batch.visible[:2])
    refused(start=batch.start[:1])
    refused(k=batch.k.float())
    refused(k=batch.k[:1].expand(batch.k.shape))      # one page held, many named
    refused(context=batch.context[:1, None].expand(4, 1))
    refused(tables=batch.tables[0])
    refused(scale=float("inf"))
    refused(q=batch.q.double())
    refused(q=torch.zeros((7, 130), dtype=torch.bfloat16, device="cuda:0")[:, 1:129])      # not aligned


@pytest.mark.parametrize("head_dim,page,rows", [(128, 16, 16), (128, 16, 32), (64, 8, 32), (64, 32, 32), (128, 16, 128),
                                                (128, 32, 128), (112, 64, 128), (64, 8, 128)])
def test_weights_keep_sixteen_bits(head_dim, page, rows):
    """A weight enters the products as two bfloat16 terms whichever kernel takes the step, as it does in the
    kernels of prompts and single tokens: what follows its parent is scored alike however many others are drafted.

    The tolerance.  With d = 2^-8 the first term leaves at most d of a weight and the second at most d of that: a
    weight is off by 2^-16 of itself.  The sum of the weights takes them as they are.  The tensor cores' sums
    may cut where float32 rounds, u = 2^-23 a step: head_dim products of a score (and three
    roundings of its scale and reference) in numerator and denominator, two terms of a key in the numerator and
    one in the denominator; exponentials, correction of the reference and joined parts 64 u.  Last the output's rounding,
    2^-8 of it.  Of many outputs some are nearly zero beside what was weighed, and there one term alone (2^-8 of each
    weight) is off by a multiple of this."""
    batch = Batch(20, [40, 9, 300], [12, 30, 3], 4, 2, head_dim, page, torch.bfloat16)
    batch.q_host = batch.q_host * 0.25
    batch.q *= 0.25
    batch.run(ops, max_nodes=rows // 2)
    expected, weighed, largest = batch.expected()
    u, keys = 2.0 ** -23, 303
    near = weighed * (2.0 ** -16 + 2 * (head_dim + 3) * u * largest + (4 * keys + 64) * u)
    allowed = near + 2.0 ** -8 * (expected.abs() + near)
    off = (batch.out[:batch.tokens, :4 * head_dim].double().cpu() - expected).abs()
    assert bool((off <= allowed).all()), f"{int((off > allowed).sum())} of {off.numel()} outputs are further off"
    assert int(batch.status.item()) == 0


def put(batch, cache, token, coordinate, number):
    """``number`` into one coordinate of the drafted token ``token`` of every request, in every key/value head."""
    page, dtype = batch.page_size, cache.dtype
    for r, context in enumerate(batch.contexts):
        place = context + token
        page_id = int(batch.tables[batch.row[r], place // page])
        held = from_cache(cache[page_id]).clone()
        held[:, place % page, coordinate] = number
        cache[page_id] = to_cache(held, dtype)


@pytest.mark.parametrize("head_dim,page", [(128, 16), (64, 32), (112, 64), (80, 8)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("contexts,heads,extra", [
    ([1 + 7 * (i % 8) for i in range(48)], 32, 0),       # short requests: a CTA has many items of one tile
    ([1 + 7 * (i % 8) for i in range(48)], 32, 33),      # ... of one or two, half of the warps with rows
    ([0, 700, 20], 4, 0),                                # items cut over CTAs
    ([700, 64, 1], 4, 90),
])
def test_tensor_memory_values_that_are_not_finite_in_every_item(head_dim, page, bad, contexts, heads, extra):
    """A drafted token whose values overflowed in all heads: every item of a CTA has such a value, and each
    reaches, coordinate by coordinate, the tokens that see it and no other."""
    nodes = 12 + extra
    parents = [-1, 0, 0, 1, 1, 2, 2, 3, 3, 5, 5, 6] + [4] * extra
    seen = [ancestors(parents)] * len(contexts)
    args = (23, contexts, [nodes] * len(contexts), heads, heads, head_dim, page, torch.bfloat16)
    clean = Batch(*args, seen=seen)
    clean.run(ops, max_nodes=128)
    batch = Batch(*args, seen=seen)
    put(batch, batch.v, 2, 1, bad)
    hit = torch.zeros((len(contexts), nodes, heads, head_dim), dtype=torch.bool, device=batch.out.device)
    hit[:, [2, 5, 6, 9, 10, 11], :, 1] = True
    hit = hit.view(batch.tokens, heads * head_dim)
    want = clean.out[:batch.tokens]
    assert bool(want.isfinite().all())
    for _ in range(5):
        batch.out.fill_(7.0)
        batch.run(ops, max_nodes=128)
        got = batch.out[:batch.tokens]
        assert bool((got[hit].isnan() if bad != bad else got[hit] == bad).all())
        assert torch.equal(got[~hit], want[~hit])
    assert int(batch.status.item()) == 0


# A call of each kernel: its type, heads and pages, and the rows (tokens times query heads of a key/value
# head) that the call is told a request has at most.
KERNELS = [
    ("streaming, one warp", torch.bfloat16, 128, 16, 1),
    ("streaming, two warps", torch.bfloat16, 128, 16, 32),
    ("streaming, two warps", torch.bfloat16, 64, 8, 32),
    ("tensor memory", torch.bfloat16, 128, 16, 128),
    ("tensor memory", torch.bfloat16, 64, 32, 128),
    ("tensor memory", torch.bfloat16, 112, 64, 128),
    ("tensor memory", torch.bfloat16, 80, 8, 128),
    ("tiles", torch.bfloat16, 64, 24, 1),
    ("tiles", torch.float32, 128, 16, 1),
    ("tiles", torch.float32, 256, 16, 1),
    ("rows", torch.bfloat16, 300, 8, 1),
    ("rows", torch.float32, 6, 4, 1),
]


@pytest.mark.parametrize("kernel,dtype,head_dim,page,rows", KERNELS)
@pytest.mark.parametrize("contexts", [[0, 0], [20, 20], [300, 300], [320, 320], [1500, 40]])
def test_a_query_that_is_no_number_says_so(kernel, dtype, head_dim, page, rows, contexts):
    """Whatever the length, so whether or not its keys are cut over CTAs; no other row is touched."""
    nodes, heads = [9, 5], 4
    clean = Batch(21, contexts, nodes, heads, 2, head_dim, page, dtype)
    clean.run(ops, max_nodes=max(1, rows // 2))
    batch = Batch(21, contexts, nodes, heads, 2, head_dim, page, dtype)
    bad = torch.zeros(batch.out.shape, dtype=torch.bool, device=batch.out.device)
    for token, head in ((0, 0), (4, 3), (8, 1), (13, 2)):
        batch.q[token, head * head_dim + 1] = float("nan")
        bad[token, head * head_dim:(head + 1) * head_dim] = True
    batch.run(ops, max_nodes=max(1, rows // 2))
    assert bool(batch.out[bad].isnan().all())
    assert torch.equal(batch.out[~bad], clean.out[~bad])


@pytest.mark.parametrize("kernel,dtype,head_dim,page,rows", KERNELS)
@pytest.mark.parametrize("contexts", [[0, 0], [20, 40], [320, 700]])
def test_a_drafted_key_that_is_no_number_reaches_who_sees_it(kernel, dtype, head_dim, page, rows, contexts):
    heads, nodes = 4, 12
    seen = [ancestors([-1, 0, 0, 1, 1, 2, 2, 3, 3, 5, 5, 6])] * 2
    args = (24, contexts, [nodes] * 2, heads, heads, head_dim, page, dtype)
    clean = Batch(*args, seen=seen)
    clean.run(ops, max_nodes=rows)
    batch = Batch(*args, seen=seen)
    put(batch, batch.k, 2, 0, float("nan"))
    batch.run(ops, max_nodes=rows)
    branch = [r * nodes + n for r in range(2) for n in (2, 5, 6, 9, 10, 11)]
    others = [n for n in range(2 * nodes) if n not in branch]
    width = heads * head_dim
    assert bool(batch.out[branch, :width].isnan().all())
    assert torch.equal(batch.out[others, :width], clean.out[others, :width])


@pytest.mark.parametrize("kernel,dtype,head_dim,page,rows",
                         [case for case in KERNELS if case[0] != "tensor memory"])
@pytest.mark.parametrize("context,place", [(0, 2), (60, 62), (64, 66), (100, 102), (100, 99), (100, 3), (40, 33),
                                           (64, 63)])
def test_a_weight_of_zero_does_not_hide_a_value(kernel, dtype, head_dim, page, rows, context, place):
    """A key that a token sees with a score so low that its weight is zero in 32 bits, and a value that is not finite:
    the output is not finite, wherever a tile of keys begins.  Who does not see it gets what it got."""
    nodes, heads = 12, 2
    parents = [-1, 0, 0, 1, 1, 2, 2, 3, 3, 5, 5, 6]
    seen = [ancestors(parents)]
    outs = []
    for value in (0.0, float("inf")):
        batch = Batch(22, [context], [nodes], heads, heads, head_dim, page, dtype, seen=seen)
        batch.q.copy_(batch.q.abs())
        page_id = int(batch.tables[batch.row[0], place // page])
        for cache, number in ((batch.k, -1e4), (batch.v, value)):
            held = from_cache(cache[page_id]).clone()
            held[:, place % page] = number
            cache[page_id] = to_cache(held, dtype)
        batch.run(ops, max_nodes=rows)
        assert int(batch.status.item()) == 0
        outs.append(batch.out[:nodes, :heads * head_dim].clone())
    sees = [n for n in range(nodes) if place < context or seen[0][n, place - context]]
    others = [n for n in range(nodes) if n not in sees]
    assert bool(outs[0].isfinite().all())
    assert not bool(outs[1][sees].isfinite().any())
    assert torch.equal(outs[1][others], outs[0][others])
