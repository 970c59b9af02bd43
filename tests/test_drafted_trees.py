"""Steps of drafted trees and branches of a request on the host: what a step describes, what it
refuses, and the cache manager's books."""
from __future__ import annotations

import types

import numpy as np
import pytest
import torch

from helix_runtime_b200.cache import CacheManager, KvNeed, OutOfPages, StateNeed
from helix_runtime_b200.config import architecture_for
from helix_runtime_b200.engine import step as steps
from helix_runtime_b200.engine.step import StepEntry, StepError, StepFunction
from helix_runtime_b200.models import DecoderModel
from plain_tree import ancestors, random_parents, words_of
from rekasun_configs import CONFIGS
from tiny_configs import tiny_config

CPU = torch.device("cpu")


def manager(num_pages=60, window=None, states=None, max_requests=4, max_positions=200):
    needs = {0: KvNeed(2, 8), 1: KvNeed(2, 8, window=window)}
    return CacheManager(needs, states or {}, 4, num_pages, max_requests, max_positions, torch.float32, CPU,
                        poison=True)


def function(cache, takes_trees=True, max_tokens=140):
    model = types.SimpleNamespace(device=CPU, dtype=torch.float32, vocab_size=50, max_positions=200,
                                  takes_trees=takes_trees)
    return StepFunction(model, cache, max_tokens=max_tokens, max_requests=4)


def published(cache, request, tokens):
    cache.admit(request)
    cache.extend(request, tokens)
    cache.commit(request, tokens)


@pytest.mark.parametrize("counts", [(1,), (5, 1), (64, 2), (3, 70, 20), (1, 129)])
def test_what_a_step_describes(counts):
    rng = np.random.default_rng(sum(counts))
    cache = manager()
    step = function(cache)
    entries = []
    for index, count in enumerate(counts):
        published(cache, index, 3 * index + 1)
        entries.append(StepEntry(index, [7] * count, (), random_parents(rng, count)))
    ctx, _, _, lengths = step.prepare(entries)
    words, cursor = -(-max(counts) // 64), 0
    for index, entry in enumerate(entries):
        count, before = len(entry.tokens), 3 * index + 1
        seen, mine = ancestors(entry.parents), slice(cursor, cursor + count)
        assert np.array_equal(ctx.trees.visible[mine].numpy(), words_of(seen, words))
        assert ctx.trees.places[mine].tolist() == list(range(before, before + count))
        assert ctx.trees.parents[mine].tolist() == list(entry.parents)
        assert ctx.positions[mine].tolist() == (before + seen.sum(axis=1) - 1).tolist()
        assert lengths[index] == cache.reserved(index) == before + count
        assert cache.length(index) == before
        cursor += count
    assert ctx.trees.visible.shape == (cursor, words)
    # the same step function prepares plain steps, and wider trees, as before
    step.fail(entries)
    ctx, _, _, _ = step.prepare([StepEntry(0, [1, 2, 3])])
    assert ctx.trees is None and ctx.positions[:3].tolist() == [1, 2, 3]
    cache.check()


def test_steps_that_are_refused_reserve_nothing():
    cache = manager()
    step = function(cache)
    published(cache, "a", 3)
    published(cache, "b", 4)
    for entries in ([StepEntry("a", [1, 2], (), [-1, 0]), StepEntry("b", [1])],
                    [StepEntry("a", [1, 2], (), [-1])], [StepEntry("a", [1, 2], (), [-1, 1])],
                    [StepEntry("a", [1, 2], (), [0, 0])], [StepEntry("a", [1, 2], (), [])],
                    [StepEntry("a", [1] * 141, (), list(range(-1, 140)))]):
        with pytest.raises(StepError):
            step.prepare(entries)
    with pytest.raises(StepError, match="none"):
        step.prepare([StepEntry("a", [1], (), [-1])], feed_rows=[0])
    with pytest.raises(StepError, match="takes no drafted trees"):
        function(cache, takes_trees=False).prepare([StepEntry("a", [1], (), [-1])])
    with pytest.raises(StepError, match="no drafted trees"):
        step.keep(torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    assert cache.reserved("a") == 3 and cache.reserved("b") == 4
    cache.check()


def test_what_is_kept_is_published_and_the_rest_given_back(monkeypatch):
    moved = []
    monkeypatch.setattr(steps.ops, "keep_rows",
                        lambda storage, tables, rows, context, path, kept, requests, status:
                        moved.append((kept[:requests].tolist(), requests)))
    cache = manager()
    step = function(cache)
    published(cache, "a", 3)
    published(cache, "b", 8)
    parents = [-1, 0, 0, 1, 3, 4] + [5] * 15
    entries = [StepEntry("a", [1] * 21, (), parents), StepEntry("b", [1] * 6, (), parents[:6])]
    free = cache.free_pages()
    ctx, _, _, lengths = step.prepare(entries)
    step.finish(entries, lengths, ctx)
    assert (cache.length("a"), cache.reserved("a")) == (3, 24)
    path = torch.tensor([[0, 1, 3, 4, 5, 6], [0, 1, 3, 4, 5, -1]], dtype=torch.int32)
    with pytest.raises(StepError, match="wait for"):
        step.prepare([StepEntry("a", [1])])
    with pytest.raises(StepError, match="22 tokens kept"):
        step.keep(path, torch.tensor([22, 1], dtype=torch.int32))
    with pytest.raises(StepError, match="no branch"):
        step.keep(path.flip(1), torch.tensor([3, 1], dtype=torch.int32))
    assert not moved
    assert step.keep(path, torch.tensor([3, 5], dtype=torch.int32)) == [3, 5]
    assert moved == [([3, 5], 2)]
    assert (cache.length("a"), cache.reserved("a")) == (6, 6)
    assert (cache.length("b"), cache.reserved("b")) == (13, 13)
    assert cache.free_pages() == [free[0] - 1 - 2]      # 6 tokens in two pages, 13 in four
    cache.check()
    # a request that ended in between keeps nothing, the others do
    ctx, _, _, lengths = step.prepare(entries)
    step.finish(entries, lengths, ctx)
    cache.release("a")
    published(cache, "a", 1)
    assert step.keep(path, torch.tensor([3, 5], dtype=torch.int32)) == [0, 5]
    assert moved[-1] == ([0, 5], 2) and cache.length("a") == 1 and cache.length("b") == 18
    # flagged moves publish nothing
    ctx, _, _, lengths = step.prepare(entries)
    step.finish(entries, lengths, ctx)
    step.status.fill_(steps.ops.FLAG_BAD_MOVE)
    with pytest.raises(StepError, match="move in the cache"):
        step.keep(path, torch.tensor([3, 5], dtype=torch.int32))
    assert cache.length("b") == cache.reserved("b") == 18 and cache.length("a") == 1
    cache.check()
    step.prepare([StepEntry("a", [1])])


def test_models_that_take_trees():
    def model(document):
        entry = architecture_for(document)
        return DecoderModel(entry.build_spec(entry.config_from_dict(document)))

    assert model(tiny_config("A").to_dict()).takes_trees
    for config in CONFIGS.values():
        document = config if isinstance(config, dict) else config.to_dict()
        assert not model(document).takes_trees      # windows and filters over time


def test_branches_share_whole_pages_and_copy_the_last():
    cache = manager(num_pages=8)
    published(cache, "a", 10)
    group = cache.groups[0]
    rng = torch.Generator().manual_seed(1)
    for page in cache._requests["a"].tables[0]:
        group.storage[:, :, page] = torch.randn(group.storage[:, :, page].shape, generator=rng)
    for tokens, name in ((10, "b"), (8, "c"), (1, "d")):
        cache.branch("a", name, tokens)
        mine, theirs = cache._requests[name].tables[0], cache._requests["a"].tables[0]
        whole = tokens // 4
        assert mine[:whole] == theirs[:whole] and len(mine) == -(-tokens // 4)
        assert cache.length(name) == cache.reserved(name) == tokens
        if tokens % 4:
            assert mine[-1] != theirs[whole]
            assert torch.equal(group.storage[:, :, mine[-1]], group.storage[:, :, theirs[whole]])
        cache.check()
    for name in ("d", "a", "b", "c"):
        cache.release(name)
    cache.check()
    assert cache.free_pages() == [8]


def test_branches_that_are_refused_change_nothing():
    cache = manager(num_pages=3, max_requests=2)
    published(cache, "a", 10)
    for tokens in (0, -1, 11):
        with pytest.raises(ValueError):
            cache.branch("a", "b", tokens)
    with pytest.raises(OutOfPages):
        cache.branch("a", "b", 9)
    with pytest.raises(KeyError):
        cache.branch("a", "a", 8)
    with pytest.raises(KeyError):
        cache.branch("nobody", "b", 8)
    cache.check()
    cache.branch("a", "b", 8)
    with pytest.raises(OutOfPages):
        cache.branch("a", "c", 8)       # no slot
    cache.check()
    windowed = manager(window=5)
    published(windowed, "a", 30)
    with pytest.raises(ValueError, match="given back"):
        windowed.branch("a", "b", 9)
    windowed.branch("a", "b", 29)
    windowed.check()
    stateful = manager(states={0: StateNeed((4,))})
    published(stateful, "a", 10)
    with pytest.raises(ValueError, match="no state"):
        stateful.branch("a", "b", 9)
    stateful.state(0)[stateful.slot("a")] = 7.0
    stateful.keep_state("a", 10, stateful.snapshot_state("a"))
    stateful.branch("a", "b", 10)
    assert stateful.state(0)[stateful.slot("b")].tolist() == [7.0] * 4
    stateful.check()


def recorder(monkeypatch):
    """Calls of the operator that moves rows, in place of it: context and kept rows of each request."""
    moved = []
    monkeypatch.setattr(steps.ops, "keep_rows",
                        lambda storage, tables, rows, context, path, kept, requests, status:
                        moved.append((context[:requests].tolist(), kept[:requests].tolist())))
    return moved


def test_a_tree_that_is_given_up_is_forgotten(monkeypatch):
    """Plain tokens of its request, queued ahead, are not taken for it, and it can no longer be kept."""
    moved = recorder(monkeypatch)
    path, one = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for count in (1, 3):
        cache = manager()
        step = function(cache)
        published(cache, "a", 3)
        tree = [StepEntry("a", [1] * count, (), list(range(-1, count - 1)))]
        ctx, _, _, lengths = step.prepare(tree)
        step.finish(tree, lengths, ctx)
        step.fail(tree)
        with pytest.raises(StepError, match="no drafted trees"):
            step.keep(path, one)
        plain = [StepEntry("a", [2] * count)]
        first = step.prepare(plain)
        with pytest.raises(StepError, match="no drafted trees"):
            step.keep(path, one)
        step.prepare([StepEntry("a", [0])], feed_rows=[0])      # queued behind it
        with pytest.raises(StepError, match="no drafted trees"):
            step.keep(path, one)
        step.finish(plain, first[3], first[0])
        assert cache.length("a") == 3 + count and cache.reserved("a") == 4 + count
        cache.check()
    assert not moved


def test_a_request_of_the_same_name_has_no_tree(monkeypatch):
    """What another request of that name has reserved is not the tree's of the one that ended."""
    moved = recorder(monkeypatch)
    cache = manager()
    step = function(cache)
    published(cache, "a", 3)
    published(cache, "b", 3)
    tree = [StepEntry("a", [1] * 4, (), [-1, 0, 0, 0]), StepEntry("b", [1] * 4, (), [-1, 0, 0, 0])]
    ctx, _, _, lengths = step.prepare(tree)
    step.finish(tree, lengths, ctx)
    cache.release("a")
    published(cache, "a", 3)
    cache.extend("a", 7)
    path = torch.tensor([[0, 2], [0, 2]], dtype=torch.int32)
    assert step.keep(path, torch.tensor([2, 2], dtype=torch.int32)) == [0, 2]
    assert moved == [([3, 3], [0, 2])]
    assert (cache.length("a"), cache.reserved("a")) == (3, 7) and cache.length("b") == 5
    cache.check()


def test_no_step_is_prepared_over_a_tree_that_waits(monkeypatch):
    """From its preparation on: a step queued behind it would overwrite what its rows are moved by."""
    moved = recorder(monkeypatch)
    cache = manager(num_pages=20)
    step = function(cache)
    published(cache, "a", 3)
    published(cache, "b", 9)
    tree = [StepEntry("a", [1] * 4, (), [-1, 0, 0, 0])]
    ctx, _, _, lengths = step.prepare(tree)
    path, two = torch.tensor([[0, 2]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    with pytest.raises(StepError, match="wait for"):
        step.prepare([StepEntry("b", [1])])
    with pytest.raises(StepError, match="not run"):
        step.keep(path, two)
    assert cache.reserved("b") == 9 and ctx.request_context[0] == 3
    step.finish(tree, lengths, ctx)
    assert step.keep(path, two) == [2]
    assert moved == [([3], [2])] and cache.length("a") == 5
    # a preparation that fails, and a tree given up before it has run, leave the way free
    with pytest.raises(OutOfPages):
        step.prepare([StepEntry("b", [1] * 100, (), list(range(-1, 99)))])
    tree = [StepEntry("a", [1] * 4, (), [-1, 0, 0, 0])]
    step.prepare(tree)
    step.fail(tree)
    step.prepare([StepEntry("b", [1])])
    cache.check()


def test_a_tree_waits_for_the_steps_in_front_of_it(monkeypatch):
    """Its rows lie behind tokens that an earlier step has reserved and not yet published."""
    moved = recorder(monkeypatch)
    cache = manager()
    step = function(cache)
    published(cache, "a", 3)
    plain, tree = [StepEntry("a", [1, 2])], [StepEntry("a", [1] * 4, (), [-1, 0, 0, 0])]
    earlier = step.prepare(plain)
    ctx, _, _, lengths = step.prepare(tree)
    step.finish(tree, lengths, ctx)
    path, two = torch.tensor([[0, 2]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    with pytest.raises(StepError, match="earlier step"):
        step.keep(path, two)
    assert not moved and cache.length("a") == 3
    step.finish(plain, earlier[3], earlier[0])
    assert step.keep(path, two) == [2]
    assert cache.length("a") == cache.reserved("a") == 7
    cache.check()
