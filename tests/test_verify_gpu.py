"""Verification of drafted tokens against a walk in 64 bits that holds every distribution whole."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helix_runtime_b200.ops import library as ops
from plain_tree import random_parents, walk

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


class Drafts:
    def __init__(self, seed, nodes, vocab, draft=True, replacement=False, heat=0.8, noise=0.7, width=None,
                 parents=None, pad=0):
        rng = np.random.default_rng(seed)
        self.nodes, self.vocab, self.replacement = nodes, vocab, replacement
        self.trees = parents or [random_parents(rng, n) for n in nodes]
        tokens = sum(nodes)
        self.logits = (3.0 * rng.normal(size=(tokens, vocab))).astype(np.float32)
        self.draft = (self.logits + noise * rng.normal(size=(tokens, vocab))).astype(np.float32)
        self.heat = np.full(len(nodes), heat, dtype=np.float32) if np.isscalar(heat) else \
            np.asarray(heat, dtype=np.float32)
        self.uniform = (rng.integers(0, 1 << 24, tokens) / float(1 << 24)).astype(np.float32)
        self.ids = np.zeros(tokens, dtype=np.int32)
        at = 0
        for r, tree in enumerate(self.trees):
            for node in range(nodes[r]):
                children = [j for j in range(nodes[r]) if tree[j] == node]
                if not children:
                    continue
                scaled = self.draft[at + node].astype(np.float64) / max(float(self.heat[r]), 1e-3)
                if self.heat[r] > 0 and replacement:
                    share = np.exp(scaled - scaled.max())
                    picked = rng.choice(vocab, size=len(children), p=share / share.sum())
                else:
                    keys = scaled + (rng.gumbel(size=vocab) if self.heat[r] > 0 else 0.0)
                    picked = np.argsort(-keys)[:len(children)]
                    picked = np.resize(picked, len(children))
                self.ids[[at + j for j in children]] = picked
            at += nodes[r]
        self.has_draft = draft
        self.width = width or max(1, max(nodes))
        self.pad = pad

    def run(self):
        count, tokens = len(self.nodes), sum(self.nodes)

        def tensor(array, dtype):
            return torch.as_tensor(array, device=DEVICE).to(dtype)

        def matrix(array):
            wide = torch.full((tokens, self.vocab + self.pad), float("nan"), device=DEVICE)
            wide[:, :self.vocab] = tensor(array, torch.float32)
            return wide[:, :self.vocab]

        self.status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        self.path = torch.full((count + 1, self.width + 2), -7, dtype=torch.int32, device=DEVICE)
        self.kept, self.next = (torch.full((count + 1,), -7, dtype=torch.int32, device=DEVICE) for _ in range(2))
        parents = np.concatenate([np.asarray(t[:n], dtype=np.int32) for t, n in zip(self.trees, self.nodes)] +
                                 [np.zeros(0, dtype=np.int32)])
        self.arguments = (matrix(self.logits), matrix(self.draft) if self.has_draft else None,
                          tensor(self.ids, torch.int32), tensor(parents, torch.int32),
                          tensor(np.concatenate([[0], np.cumsum(self.nodes)]), torch.int32),
                          tensor(self.heat, torch.float32), tensor(self.uniform, torch.float32),
                          self.path[:, :self.width], self.kept, self.next, count, self.status)
        ops.verify_drafts(*self.arguments, replacement=self.replacement)
        return self

    def check(self, status=0):
        path, kept, following = self.path.cpu().numpy(), self.kept.cpu().numpy(), self.next.cpu().numpy()
        at = 0
        for r, n in enumerate(self.nodes):
            here = slice(at, at + n)
            if n == 0:
                want, token = [], -1
            else:
                want, token = walk(self.logits[here], self.draft[here] if self.has_draft else None, self.ids[here],
                                   self.trees[r], float(self.heat[r]), self.uniform[here].astype(np.float64),
                                   self.replacement, self.width)
            assert list(path[r, :self.width]) == want + [-1] * (self.width - len(want)), f"request {r}"
            assert kept[r] == len(want) and following[r] == token, f"request {r}"
            at += n
        assert (path[:, self.width:] == -7).all() and (path[-1] == -7).all()
        assert kept[-1] == -7 and following[-1] == -7
        assert int(self.status.item()) == status


@pytest.mark.parametrize("mode", ["without", "with", "lookup"])
@pytest.mark.parametrize("nodes,vocab", [
    ([1], 1), ([2], 2), ([1, 1, 1], 40), ([9, 4, 16], 33), ([20, 1, 7, 30], 300), ([12, 12], 2049),
    ([8], 32000), ([30, 11, 5, 17, 24, 9], 5000), ([6, 9], 70001)])
def test_walks(mode, nodes, vocab):
    for seed in range(4):
        Drafts(seed, nodes, vocab, draft=mode != "lookup", replacement=mode == "with", pad=seed % 2 * 3).run().check()


@pytest.mark.parametrize("mode", ["without", "with", "lookup"])
@pytest.mark.parametrize("requests", [40, 100, 200, 400])      # clusters of fewer CTAs
def test_many_requests(mode, requests):
    rng = np.random.default_rng(requests)
    nodes = [int(n) for n in rng.integers(0, 9, requests)]
    heat = rng.choice([0.0, 0.3, 0.8, 1.0, 2.5], requests)
    Drafts(requests, nodes, 700, draft=mode != "lookup", replacement=mode == "with", heat=heat).run().check()


@pytest.mark.parametrize("mode", ["without", "with", "lookup"])
def test_wide_trees(mode):
    """Seventy children of one token, hardly any of which stands; a token drafted more than once."""
    for noise in (0.5, 6.0):
        drafts = Drafts(3, [71, 71], 200, draft=mode != "lookup", replacement=mode == "with", noise=noise,
                        parents=[[-1] + [0] * 70] * 2)
        drafts.uniform[1:71] = 1.0 - 2.0 ** -24
        drafts.uniform[72:] = 0.97
        if mode == "lookup":
            drafts.ids[10:20] = drafts.ids[5]
        drafts.run().check()


def test_long_chains_and_paths_that_are_full():
    chain = [list(range(-1, 99))]
    drafts = Drafts(4, [100], 50, noise=0.0, parents=chain)          # the draft is the target: all stand
    drafts.run().check()
    assert int(drafts.kept[0]) == 100
    for width in (1, 5):
        drafts = Drafts(4, [100], 50, noise=0.0, parents=chain, width=width)
        drafts.run().check()
        assert int(drafts.kept[0]) == width


def test_greedy_takes_the_lowest_id_among_the_maxima():
    drafts = Drafts(5, [8, 8], 640, heat=0.0)
    drafts.logits[:, 100] = drafts.logits[:, 500] = 50.0
    drafts.ids[:] = 500
    drafts.ids[[3, 11]] = 100
    drafts.run().check()
    assert int(drafts.next[0]) == 100


def test_numbers_at_their_ends():
    """Numbers of zero and just below one, for tokens that a draft is sure of."""
    for value in (0.0, 1.0 - 2.0 ** -24):
        for mode in ("without", "with", "lookup"):
            drafts = Drafts(6, [9, 5], 100, draft=mode != "lookup", replacement=mode == "with")
            drafts.uniform[:] = value
            drafts.run().check()


def test_drafts_may_leave_tokens_out():
    drafts = Drafts(7, [10, 10], 400)
    out = np.ones(400, dtype=bool)
    out[np.unique(drafts.ids)] = False
    drafts.draft[:, out] = -np.inf
    drafts.draft[:, 128:256] = -np.inf          # whole stretches
    drafts.run().check()


@pytest.mark.parametrize("where,value", [("logits", np.nan), ("logits", np.inf), ("logits", -np.inf),
                                         ("draft", np.nan), ("draft", np.inf)])
def test_logits_that_are_not_finite(where, value):
    """The request that walks over them is told so; the others, and rows off the way, are not."""
    drafts = Drafts(8, [5, 5, 5], 900)
    getattr(drafts, where)[5, 777] = value            # the second request's first token
    drafts.run().check(status=ops.FLAG_NONFINITE)
    assert int(drafts.next[1]) == -1
    drafts = Drafts(8, [5, 5], 900, parents=[[-1, 0, 1, 2, 3]] * 2)
    drafts.uniform[1] = 1.0 - 2.0 ** -24
    drafts.logits[0, drafts.ids[1]] = -40.0           # the first draft falls: token 4 is never reached
    getattr(drafts, where)[4, 3] = value
    drafts.run().check()
    drafts = Drafts(8, [3], 900)
    drafts.draft[0] = -np.inf
    drafts.run()
    assert int(drafts.next[0]) == -1 and int(drafts.status.item()) == ops.FLAG_NONFINITE


def test_tokens_outside_the_vocabulary_are_passed_over():
    for mode in ("without", "lookup"):
        drafts = Drafts(9, [6, 6], 50, draft=mode != "lookup", parents=[[-1, 0, 0, 0, 0, 0]] * 2)
        drafts.ids[1], drafts.ids[2] = -1, 50
        drafts.run().check(status=ops.FLAG_BAD_TOKEN)


def test_tokens_are_distributed_as_the_target_says():
    """The first token after the root, over many requests of the same tree: its frequencies are the
    target's within five standard deviations of a count (four hundred counts of other trees would stay
    within them but for one in 4,000)."""
    vocab, requests, heat = 7, 40000, 0.9
    rng = np.random.default_rng(11)
    target = rng.normal(size=vocab).astype(np.float32)
    guess = rng.normal(size=vocab).astype(np.float32)
    p, q = (np.exp(v.astype(np.float64) / heat) for v in (target, guess))
    p, q = p / p.sum(), q / q.sum()
    nodes = 4
    for mode in ("without", "with", "lookup"):
        logits = torch.as_tensor(np.tile(target, (requests * nodes, 1)), device=DEVICE)
        draft = torch.as_tensor(np.tile(guess, (requests * nodes, 1)), device=DEVICE)
        if mode == "lookup":
            picked = np.tile([2, 5, 2], (requests, 1))
        elif mode == "with":
            picked = rng.choice(vocab, size=(requests, 3), p=q)
        else:
            picked = np.argsort(-(np.log(q) + rng.gumbel(size=(requests, vocab))), axis=1)[:, :3]
        ids = torch.as_tensor(np.concatenate([np.zeros((requests, 1), dtype=np.int64), picked], axis=1).reshape(-1),
                              device=DEVICE).to(torch.int32)
        parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device=DEVICE).repeat(requests)
        start = torch.arange(0, requests * nodes + 1, nodes, dtype=torch.int32, device=DEVICE)
        uniform = torch.as_tensor(rng.random(requests * nodes).astype(np.float32) * np.float32(1 - 2 ** -23),
                                  device=DEVICE)
        path = torch.zeros((requests, 2), dtype=torch.int32, device=DEVICE)
        kept, following, status = (torch.zeros(n, dtype=torch.int32, device=DEVICE) for n in (requests, requests, 1))
        ops.verify_drafts(logits, None if mode == "lookup" else draft, ids, parents, start,
                          torch.full((requests,), heat, device=DEVICE), uniform, path, kept, following, requests,
                          status, replacement=mode == "with")
        first = torch.where(kept == 2, ids.view(requests, nodes).gather(1, path[:, 1:].clamp(min=0).long())[:, 0],
                            following)
        counts = torch.bincount(first.long(), minlength=vocab).cpu().numpy()
        spread = np.sqrt(requests * p * (1 - p))
        assert (np.abs(counts - requests * p) <= 5 * spread).all(), (mode, counts / requests, p)


def test_recorded_and_replayed():
    drafts = Drafts(12, [9, 6], 3000).run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.verify_drafts(*drafts.arguments)
    other = Drafts(13, [9, 6], 3000)
    other.trees, parents = drafts.trees, None
    drafts.arguments[0].copy_(torch.as_tensor(other.logits, device=DEVICE))
    drafts.arguments[1].copy_(torch.as_tensor(other.draft, device=DEVICE))
    drafts.arguments[2].copy_(torch.as_tensor(other.ids, device=DEVICE))
    drafts.arguments[6].copy_(torch.as_tensor(other.uniform, device=DEVICE))
    graph.replay()
    torch.cuda.synchronize()
    drafts.logits, drafts.draft, drafts.ids, drafts.uniform = other.logits, other.draft, other.ids, other.uniform
    drafts.check()


def test_nothing_to_do():
    drafts = Drafts(14, [0, 3, 0], 30).run()
    drafts.check()


def test_refusals():
    drafts = Drafts(15, [4, 4], 64).run()
    names = ("logits", "draft_logits", "token_ids", "parents", "request_start", "temperature", "uniform", "path",
             "kept", "next_tokens", "requests", "status")
    good = dict(zip(names, drafts.arguments))

    def refused(**changes):
        with pytest.raises(ops.KernelError):
            ops.verify_drafts(**{**good, **changes})

    refused(logits=good["logits"].double())
    refused(logits=good["logits"].cpu())
    refused(draft_logits=good["draft_logits"][:, :63])
    refused(draft_logits=good["draft_logits"][:7])
    refused(token_ids=good["token_ids"].long())
    refused(token_ids=good["token_ids"][:7])
    refused(parents=good["parents"][:7])
    refused(uniform=good["uniform"][:7])
    refused(request_start=good["request_start"][:2])
    refused(temperature=good["temperature"].double())
    refused(temperature=good["temperature"][:1].expand(2))
    refused(path=good["path"][:1])
    refused(path=good["path"].reshape(-1)[:2])
    refused(path=good["path"][:, :0])
    refused(kept=good["kept"][:1])
    refused(requests=-1)


@pytest.mark.parametrize("replacement", [False, True])
@pytest.mark.parametrize("vocab", [300, 5000, 130000])
@pytest.mark.parametrize("fallen", [1, 2, 3, 4, 5, 8])
def test_nothing_is_left_of_the_distribution(fallen, vocab, replacement):
    """Target and draft agree on a few tokens, and the children are others, which weigh nothing in either: each
    falls, the first takes all of the target with it, and the next token is the target's own sample."""
    heavy = [vocab - 90, vocab - 60, vocab - 7]
    drafts = Drafts(16, [fallen + 1] * 3, vocab, replacement=replacement, heat=0.01,
                    parents=[[-1] + [0] * fallen] * 3)
    drafts.logits[:] = -1000.0
    drafts.logits[:, heavy] = [0.5, 0.5, 0.5]
    drafts.draft[:] = drafts.logits
    drafts.ids[:] = np.arange(drafts.ids.size)
    for request, number in enumerate((0.1, 0.5, 0.9)):
        drafts.uniform[request * (fallen + 1)] = number
    drafts.run()
    assert drafts.next[:3].tolist() == heavy
    assert drafts.kept[:3].tolist() == [1, 1, 1] and int(drafts.status.item()) == 0


@pytest.mark.parametrize("vocab", [12, 300])
def test_a_token_drafted_twice_without_putting_back(vocab):
    """It cannot have been drawn a second time: nothing of the draft is left of it, and nothing more goes."""
    for seed in range(40, 52):
        drafts = Drafts(seed, [9, 9], vocab, noise=2.0, parents=[[-1] + [0] * 8] * 2)
        drafts.ids[3] = drafts.ids[2] = drafts.ids[1]
        drafts.ids[[12, 16]] = drafts.ids[10]
        drafts.uniform[1:9] = 1.0 - 2.0 ** -24
        drafts.uniform[[10, 11, 12, 13]] = 1.0 - 2.0 ** -24
        drafts.run().check()


@pytest.mark.parametrize("mode", ["without", "with", "lookup"])
@pytest.mark.parametrize("nodes,vocab", [([257], 90), ([300, 40, 256], 70), ([701, 1], 500)])
def test_trees_past_the_shared_tables(mode, nodes, vocab):
    """Trees of which shared memory holds no copy, walked over their whole depth."""
    for seed, noise in ((30, 0.7), (31, 0.0)):
        parents = [[-1] + [j - 1 if j % 3 else max(0, j - 4) for j in range(1, n)] for n in nodes]
        drafts = Drafts(seed, nodes, vocab, draft=mode != "lookup", replacement=mode == "with", noise=noise,
                        parents=parents)
        drafts.run().check()
    if mode != "lookup":      # (the last drafts are the target's: every first child stands, half of the tokens are on the way)
        assert int(drafts.kept[0]) >= nodes[0] // 2


@pytest.mark.parametrize("mode", ["without", "with", "lookup"])
@pytest.mark.parametrize("vocab", [102400, 102401, 130000, 262147])
def test_vocabularies_whose_exponentials_are_computed_again(mode, vocab):
    for seed in (32, 33):
        Drafts(seed, [6, 9, 4], vocab, draft=mode != "lookup", replacement=mode == "with", heat=[0.8, 1.1, 0.0],
               pad=seed % 2 * 3).run().check()


@pytest.mark.parametrize("heat", [1.0, 0.8])
def test_the_exponential_is_as_exact_as_64_bits(heat):
    """Two tokens, and numbers next to the first one's share: as near as a few roundings in 64 bits allow.

    With logits x <= 0 and 0 the first token follows when u is below e / (1 + e), e = exp(x / T).  In units of
    2^-53 the factor 64 / (T ln 2) and its product with x are off by 1.5 + 1.5, so e by 3 |x| / T; table, polynomial
    and their product add 4, the sums, the share and the product with u 8.  Among many x those are taken whose share lies
    beyond that, and up to 30 times as far, from a float32 u; which side it lies on is told in 80 bits."""
    if np.finfo(np.longdouble).eps > 1e-18:
        pytest.skip("no 80-bit numbers here")
    rng = np.random.default_rng(17)
    low, high, found = 2.0 ** -53, 30 * 2.0 ** -53, []
    wide_heat = np.longdouble(np.float32(heat))
    for _ in range(20):
        x = (-2.0 * rng.random(1 << 20)).astype(np.float32)
        scaled = x.astype(np.longdouble) / wide_heat
        share = np.exp(scaled) / (1 + np.exp(scaled))
        u = share.astype(np.float32)
        away = np.abs((u.astype(np.longdouble) - share) / share) / (3 * np.abs(scaled) + 12)
        near = (away > low) & (away < high)
        found += list(zip(x[near], u[near], (u.astype(np.longdouble) >= share)[near]))
    assert len(found) > 20
    x, u, wanted = (np.array(column) for column in zip(*found))
    requests = len(found)
    drafts = Drafts(18, [1] * requests, 2, draft=False, heat=heat)
    drafts.logits[:] = 0.0
    drafts.logits[:, 0] = x
    drafts.uniform = u.astype(np.float32)
    drafts.run()
    assert np.array_equal(drafts.next[:requests].cpu().numpy(), wanted.astype(np.int32))
    assert int(drafts.status.item()) == 0
