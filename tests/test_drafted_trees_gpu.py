"""Trees of drafted tokens through a whole model: a step scores them, verification picks a branch,
the cache keeps its rows, and the requests go on, drafted again or token by token."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import random_tokens
from engine_harness import Harness, assert_close, tolerance
from helix_runtime_b200.engine.graphs import DecodeGraphs
from helix_runtime_b200.engine.step import StepEntry, StepError
from helix_runtime_b200.ops import library as ops
from helix_runtime_b200.sampling.sampler import Sampler
from plain_tree import random_parents
from tiny_configs import PAGE_SIZE, tiny_config

pytestmark = pytest.mark.gpu

CASES = [("A", "float32"), ("B", "float32"), ("A", "bfloat16"), ("B", "bfloat16"), ("C", "bfloat16")]


def harness_of(name, dtype, folders, **options):
    return Harness(folders(name, dtype), dtype, PAGE_SIZE[name], num_pages=64, **options)


def drafts(rng, plain, given, count, vocab):
    """A tree behind ``given``: the plain implementation's own continuation as a branch, the other
    tokens drawn, some below the branch."""
    parents = random_parents(rng, count)
    tokens = [given[-1]] + [int(t) for t in rng.integers(0, vocab, count - 1)]
    node, text = 0, list(given)
    while node < count:
        below = [child for child in range(node + 1, count) if parents[child] == node]
        if not below or rng.random() < 0.1:
            break
        node = below[int(rng.integers(0, len(below)))]
        tokens[node] = int(np.argmax(plain.logits(text)[-1]))
        text.append(tokens[node])
    return tokens, parents


def branch_of(parents, node):
    path = []
    while node >= 0:
        path.append(node)
        node = parents[node]
    return path[::-1]


def walk_greedily(tokens, parents, logits):
    """The branch that the logits' own arg-maxima follow, and the token behind it."""
    path = [0]
    while True:
        best = int(np.argmax(logits[path[-1]]))
        child = next((c for c in range(path[-1] + 1, len(tokens))
                      if parents[c] == path[-1] and tokens[c] == best), None)
        if child is None:
            return path, best
        path.append(child)


@pytest.mark.parametrize("name,dtype", CASES)
@pytest.mark.parametrize("counts", [(1, 6, 13), (21, 34, 70)])
def test_trees_scored_verified_and_kept(name, dtype, counts, folders, plain_models):
    plain, vocab = plain_models(name, dtype), tiny_config(name).vocab_size
    rng = np.random.default_rng(len(name) + sum(counts))
    harness = harness_of(name, dtype, folders)
    sampler = Sampler(torch.device("cuda:0"), 512)
    given = {f"r{i}": random_tokens(vocab, length, seed=50 + i) for i, length in enumerate((2, 19, 33))}
    harness.run([(request, tokens[:-1], ()) for request, tokens in given.items()])
    stood = 0
    for turn in range(3):
        entries = []
        for (request, tokens), count in zip(given.items(), counts if turn < 2 else counts[::-1]):
            room = tiny_config(name).max_position_embeddings - len(tokens)
            drafted, parents = drafts(rng, plain, tokens, min(count, room), vocab)
            entries.append(StepEntry(request, drafted, range(len(drafted)), parents))
        logits = harness.step.run(entries)
        rows = logits.float().cpu().numpy().copy()
        ctx = harness.step.last_context
        cursor, paths = 0, []
        for entry in entries:
            own = rows[cursor:cursor + len(entry.tokens)]
            cursor += len(entry.tokens)
            before = given[entry.request][:-1]
            for node in {0, len(entry.tokens) - 1, *rng.integers(0, len(entry.tokens), 4).tolist()}:
                text = before + [entry.tokens[n] for n in branch_of(entry.parents, node)]
                assert_close(own[node:node + 1], plain.logits(text)[-1:],
                             f"{entry.request} turn {turn} token {node}", **tolerance(dtype, name))
            paths.append(walk_greedily(entry.tokens, entry.parents, own))
        path, kept, following = sampler.verify(ctx, logits, [0.0] * len(entries),
                                               [0.5] * ctx.n_tokens)
        assert following.tolist() == [token for _, token in paths]
        with pytest.raises(StepError, match="wait for"):
            harness.step.run([StepEntry("r0", [1])])
        assert harness.step.keep(path, kept) == [len(p) for p, _ in paths]
        for entry, row, (p, token) in zip(entries, path.tolist(), paths):
            assert row[:len(p)] == p and set(row[len(p):]) <= {-1}
            given[entry.request] += [entry.tokens[n] for n in p[1:]] + [token]
            assert harness.cache.length(entry.request) == len(given[entry.request]) - 1
            stood += len(p) - 1
        harness.cache.check()
    assert stood > 0
    # and on without drafts, on the rows that were kept
    for turn in range(2):
        out = harness.run([(request, tokens[-1:], [0]) for request, tokens in given.items()])
        want = np.stack([plain.logits(tokens)[-1] for tokens in given.values()])
        assert_close(out, want, f"token {turn} behind the drafts", **tolerance(dtype, name))
        for tokens, row in zip(given.values(), out):
            tokens.append(int(np.argmax(row)))


def test_a_chain_of_drafts_is_a_prompt(folders):
    """A tree without forks is the request's next tokens: the same rows end up in the cache."""
    tokens = random_tokens(tiny_config("A").vocab_size, 30, seed=9)
    outs, caches = [], []
    for drafted in (False, True):
        harness = harness_of("A", "float32", folders)
        harness.run([("r", tokens[:11], ())])
        parents = list(range(-1, 18)) if drafted else None
        out = harness.step.run([StepEntry("r", tokens[11:], range(19), parents)])
        outs.append(out.float().cpu().numpy().copy())
        if drafted:
            path = torch.arange(19, dtype=torch.int32, device="cuda:0")[None]
            assert harness.step.keep(path, torch.full((1,), 19, dtype=torch.int32, device="cuda:0")) == [19]
        assert harness.cache.length("r") == 30
        keys, values = harness.cache.layer_storage(0)       # [page, kv head, ...], pages of 8
        table = torch.tensor(harness.cache._requests["r"].tables[0][:3], device="cuda:0")
        caches.append((keys[table].cpu(), values[table].cpu()))
    assert_close(outs[1], outs[0], "chain", **tolerance("float32"))
    for ours, theirs in zip(caches[1], caches[0]):
        assert torch.equal(ours, theirs)        # the first layer's rows do not depend on attention


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("C", "bfloat16")])
@pytest.mark.parametrize("at", [1, 7, 16, 21, 24])
def test_branches_go_their_own_ways(name, dtype, at, folders, plain_models):
    plain, vocab = plain_models(name, dtype), tiny_config(name).vocab_size
    harness = harness_of(name, dtype, folders)
    tokens = random_tokens(vocab, 24, seed=3)
    harness.run([("trunk", tokens, ())])
    harness.cache.branch("trunk", "left", at)
    harness.cache.branch("left", "right", at)
    harness.cache.check()
    texts = {"trunk": tokens, "left": tokens[:at], "right": tokens[:at]}
    for turn in range(2):
        more = {request: random_tokens(vocab, 3, seed=10 * turn + i) for i, request in enumerate(texts)}
        texts = {request: text + more[request] for request, text in texts.items()}
        out = harness.run([(request, more[request], [2]) for request in texts])
        want = np.stack([plain.logits(text)[-1] for text in texts.values()])
        assert_close(out, want, f"branches at {at}", **tolerance(dtype, name))
    for request in ("trunk", "left", "right"):
        harness.end(request)
    harness.cache.check()
    assert harness.cache.free_pages() == [64]


def test_requests_that_end_before_their_trees_are_settled(folders):
    """The pages of a request that ended are another's when the rest is kept."""
    harness = harness_of("A", "float32", folders)
    tokens = random_tokens(256, 24, seed=5)
    harness.run([("a", tokens[:5], ()), ("b", tokens[5:14], ())])
    parents = [-1, 0, 0, 1, 2]
    harness.step.run([StepEntry("a", tokens[:5], (), parents), StepEntry("b", tokens[5:10], (), parents)])
    storage = harness.cache.groups[0].storage
    path = torch.tensor([[0, 2, 4, -1, -1]] * 2, dtype=torch.int32, device="cuda:0")
    kept = torch.full((2,), 3, dtype=torch.int32, device="cuda:0")
    with pytest.raises(ValueError, match="not recorded"):
        DecodeGraphs(harness.step, None).run(harness.step.last_context, None, 0, True)
    with pytest.raises(StepError, match="6 tokens kept"):
        harness.step.keep(path, kept + 3)
    harness.end("a")
    before = storage.clone()
    assert harness.step.keep(path, kept) == [0, 3]
    assert harness.cache.length("b") == 12 and harness.cache.reserved("b") == 12
    pages = harness.cache._requests["b"].tables[0]
    others = [page for page in range(64) if page not in pages]
    assert torch.equal(storage[:, :, others].view(torch.int32), before[:, :, others].view(torch.int32))
    harness.cache.check()
    with pytest.raises(StepError, match="no drafted trees"):
        harness.step.keep(path, kept)


def test_a_path_that_is_none_publishes_nothing(folders):
    harness = harness_of("A", "float32", folders)
    harness.run([("a", [1, 2, 3], ())])
    harness.step.run([StepEntry("a", [4, 5, 6, 7], (), [-1, 0, 0, 1])])
    path = torch.tensor([[0, 3, 1, -1]], dtype=torch.int32, device="cuda:0")
    before = harness.cache.groups[0].storage.clone()
    kept = torch.full((1,), 3, dtype=torch.int32, device="cuda:0")
    for wrong in ([0, 3, 1, -1], [0, 2, 3, -1], [0, 1, 4, -1], [1, 3, -1, -1], [0, 1, -1, -1], [0, 1, 2, 3]):
        with pytest.raises(StepError, match="no branch"):
            harness.step.keep(torch.tensor([wrong], dtype=torch.int32, device="cuda:0"), kept)
    with pytest.raises(StepError, match="3 tokens kept"):
        harness.step.keep(path[:, :2].contiguous(), kept)
    assert torch.equal(harness.cache.groups[0].storage.view(torch.int32), before.view(torch.int32))
    assert harness.cache.length("a") == 3 and harness.cache.reserved("a") == 7
    path = torch.tensor([[0, 1, 3, -1]], dtype=torch.int32, device="cuda:0")
    assert harness.step.keep(path, kept) == [3]
    assert harness.cache.length("a") == 6 and harness.cache.reserved("a") == 6
    harness.cache.check()
    assert harness.run([("a", [4], [0])]) is not None


def test_verification_wants_the_step_s_rows(folders):
    harness = harness_of("A", "float32", folders)
    sampler = Sampler(torch.device("cuda:0"), 8)
    harness.run([("a", [1, 2, 3], ())])
    logits = harness.step.run([StepEntry("a", [4, 5], [0, 1])])
    with pytest.raises(ValueError, match="trees"):
        sampler.verify(harness.step.last_context, logits, [0.0], [0.0, 0.0])
    logits = harness.step.run([StepEntry("a", [4, 5, 6], [0, 2], [-1, 0, 1])])
    with pytest.raises(ValueError, match="trees"):
        sampler.verify(harness.step.last_context, logits, [0.0], [0.0] * 3)
    harness.step.fail([StepEntry("a", [])])
    logits = harness.step.run([StepEntry("a", [4, 5, 6], range(3), [-1, 0, 1])])
    for temperatures, uniforms in (([0.0, 0.0], [0.0] * 3), ([0.0], [0.0] * 2)):
        with pytest.raises(ValueError, match="uniform"):
            sampler.verify(harness.step.last_context, logits, temperatures, uniforms)
    # sampled, with the drafts' own distribution: token 0 stands and something follows
    path, kept, following = sampler.verify(harness.step.last_context, logits, [0.8], [0.1, 0.9, 0.4],
                                           draft_logits=logits.clone())
    assert kept.item() == 3 and 0 <= following.item() < 256     # p = q: every draft stands
    assert harness.step.keep(path, kept) == [3]
    assert ops.sm_count() > 0 and harness.cache.length("a") == 8
