"""Plain forms, in 64 bits, of what a step with drafted tokens computes, and inputs for them."""
from __future__ import annotations

import math

import numpy as np
import torch


def chunk_elements(dtype, head_dim):
    widest = 8 if dtype == torch.bfloat16 else 4
    if head_dim % widest == 0:
        return widest
    return 4 if widest > 4 and head_dim % 4 == 0 else 2


def to_cache(rows, dtype):
    """[..., page, kv head, slot, coordinate] to the cache's order of the last two axes."""
    *lead, slots, dim = rows.shape
    c = chunk_elements(dtype, dim)
    return rows.reshape(*lead, slots, dim // c, c).transpose(-3, -2).contiguous().reshape(*lead, slots, dim)


def from_cache(cache, dtype=None):
    *lead, slots, dim = cache.shape
    c = chunk_elements(dtype or cache.dtype, dim)
    return cache.reshape(*lead, dim // c, slots, c).transpose(-3, -2).reshape(*lead, slots, dim)


def ancestors(parents):
    """Boolean [nodes, nodes]: row i names i and its ancestors."""
    count = len(parents)
    seen = np.zeros((count, count), dtype=bool)
    for i, parent in enumerate(parents):
        if parent >= 0:
            seen[i] = seen[parent]
        seen[i, i] = True
    return seen


def words_of(seen, words):
    """Boolean [nodes, nodes] to int64 [nodes, words]."""
    out = np.zeros((seen.shape[0], words), dtype=np.uint64)
    for i in range(seen.shape[0]):
        for j in np.flatnonzero(seen[i]):
            if j < 64 * words:
                out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def random_parents(rng, count):
    return ([-1] + [int(rng.integers(max(0, j - 5), j)) for j in range(1, count)])[:count]


class Batch:
    """Drafted tokens of several requests over a shuffled paged cache."""

    def __init__(self, seed, contexts, nodes, heads, kv_heads, head_dim, page_size, dtype,
                 device="cuda:0", seen=None, words=None, row_pad=0, stale=float("nan")):
        rng = np.random.default_rng(seed)
        self.contexts, self.nodes = list(contexts), list(nodes)
        self.heads, self.kv_heads, self.head_dim, self.page_size = heads, kv_heads, head_dim, page_size
        self.dtype, self.requests = dtype, len(contexts)
        needed = [-(-(c + n) // page_size) for c, n in zip(contexts, nodes)]
        self.num_pages = sum(needed) + 2
        order = rng.permutation(self.num_pages)
        width = max(1, max(needed))
        tables = np.full((self.requests + 1, width), -1, dtype=np.int32)
        rows = rng.permutation(self.requests + 1)[:self.requests]
        generator = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
        tokens = sum(nodes)
        self.tokens = tokens
        shape = (self.num_pages, kv_heads, page_size, head_dim)
        k_rows, v_rows = (torch.full(shape, stale) for _ in range(2))
        self.keys, self.values, self.seen = [], [], []
        cursor = 0
        for r, (context, count) in enumerate(zip(contexts, nodes)):
            total = context + count
            k, v = (torch.randn((total, kv_heads, head_dim), generator=generator).to(dtype) for _ in range(2))
            self.keys.append(k.double())
            self.values.append(v.double())
            for p in range(needed[r]):
                page = int(order[cursor])
                cursor += 1
                tables[rows[r], p] = page
                here = slice(p * page_size, min((p + 1) * page_size, total))
                length = here.stop - here.start
                k_rows[page, :, :length] = k[here].transpose(0, 1).float()
                v_rows[page, :, :length] = v[here].transpose(0, 1).float()
            self.seen.append(ancestors(random_parents(rng, count)) if seen is None else seen[r])
        words = words or max(1, -(-max(nodes) // 64))
        self.words = words
        packed = np.concatenate([words_of(s[:, :64 * words], words) for s in self.seen if len(s)] or
                                [np.zeros((0, words), dtype=np.int64)])
        wide = heads * head_dim + row_pad

        def tensor(array, kind):
            return torch.as_tensor(np.asarray(array)).to(device=device, dtype=kind)

        self.q_host = torch.randn((tokens, heads * head_dim), generator=generator).to(dtype)
        self.q = torch.full((tokens + 3, wide), float("nan"), dtype=dtype, device=device)
        self.q[:tokens, :heads * head_dim] = self.q_host.to(device)
        self.out = torch.full((tokens + 3, wide), 7.0, dtype=dtype, device=device)
        self.k = to_cache(k_rows, dtype).to(device=device, dtype=dtype)
        self.v = to_cache(v_rows, dtype).to(device=device, dtype=dtype)
        self.visible = tensor(np.concatenate([packed, np.full((3, words), -1, dtype=np.int64)]), torch.int64)
        self.start = tensor(np.concatenate([[0], np.cumsum(nodes)]), torch.int32)
        self.context = tensor(contexts, torch.int32)
        self.row = tensor(rows, torch.int32)
        self.tables = tensor(tables, torch.int32)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.scale = 1.0 / math.sqrt(head_dim)

    def run(self, ops, partial=None, out=None, max_nodes=0):
        ops.tree_attention(self.q, self.k, self.v, self.visible, self.start, self.context, self.row,
                           self.tables, self.out if out is None else out, partial, self.requests,
                           self.heads, self.kv_heads, self.head_dim, self.page_size, self.num_pages,
                           self.scale, self.status, max_nodes)
        return self.out if out is None else out

    def expected(self):
        """In 64 bits, from the values that the tensors hold: the output ``[tokens, heads * head_dim]``,
        the weighted sum of the values' magnitudes beside it, and the largest sum of magnitudes of a
        score's products (what rounding errors are measured by)."""
        result, weighed = (torch.zeros((self.tokens, self.heads, self.head_dim), dtype=torch.float64)
                           for _ in range(2))
        at, largest = 0, 0.0
        group = self.heads // self.kv_heads
        for r, count in enumerate(self.nodes):
            q = self.q_host[at:at + count].double().view(count, self.heads, self.head_dim)
            context = self.contexts[r]
            for n in range(count):
                named = [j for j in range(min(count, 64 * self.words)) if self.seen[r][n, j]]
                index = list(range(context)) + [context + j for j in named]
                if not index:
                    continue
                k, v = self.keys[r][index], self.values[r][index]      # [keys, kv heads, dim]
                mine = q[n].view(self.kv_heads, group, self.head_dim)
                scores = torch.einsum("gad,cgd->gac", mine, k) * self.scale
                largest = max(largest, float((torch.einsum("gad,cgd->gac", mine.abs(), k.abs())
                                              * self.scale).max()))
                share = torch.softmax(scores, -1)
                result[at + n] = torch.einsum("gac,cgd->gad", share, v).reshape(self.heads, -1)
                weighed[at + n] = torch.einsum("gac,cgd->gad", share, v.abs()).reshape(self.heads, -1)
            at += count
        return result.view(self.tokens, -1), weighed.view(self.tokens, -1), largest

    def tolerance(self, expected, weighed, largest):
        """How far an output may be off.  With u = 2^-24: a score is a sum of head_dim products in
        float32, off by at most (head_dim + 3) u times their magnitudes (the scale, the base-2
        factor and the difference to the maximum are one rounding each), and an exponent's
        error is a weight's relative error, in numerator and denominator: twice that.  Exponential
        2^-21, sums of n terms n u each, joined parts a few more: (2 n + 64) u.  In bfloat16 a weight is
        rounded once, by at most d = 2^-8 of itself, and divided by the sum of the rounded ones: sum w (1 + d_j)
        v / sum w (1 + d_j) is off by at most d (sum w |v| + |output|) / (1 - d).  Last the output's own
        rounding, again 2^-8 of it."""
        u = 2.0 ** -24
        keys = max(c + n for c, n in zip(self.contexts, self.nodes))
        share = 2 * (self.head_dim + 3) * u * largest + (2 * keys + 64) * u
        if self.dtype == torch.bfloat16:
            d = 2.0 ** -8
            near = d / (1 - d) * (weighed + expected.abs()) + share * weighed
            return near + d * (expected.abs() + near)
        return u * expected.abs() + share * weighed

    def check(self, out=None):
        """Every output within its tolerance, nothing else written, no complaint."""
        out = self.out if out is None else out
        width = self.heads * self.head_dim
        got = out[:self.tokens, :width].double().cpu()
        expected, weighed, largest = self.expected()
        off = (got - expected).abs()
        allowed = self.tolerance(expected, weighed, largest)
        assert bool(torch.isfinite(got).all())
        assert bool((off <= allowed).all()), f"off by {float((off - allowed).max())} more than allowed"
        assert bool((out[self.tokens:] == 7.0).all()) and bool((out[:, width:] == 7.0).all())
        assert int(self.status.item()) == 0


def walk(logits, draft, ids, parents, heat, uniform, replacement, width):
    """One request's verification in 64 bits, with distributions held whole: (path, next token)."""
    count, vocab = logits.shape
    here, path = 0, [0]
    while True:
        row = logits[here].astype(np.float64)
        if not np.isfinite(row).all():
            return path, -1
        children = [j for j in range(here + 1, count) if parents[j] == here] if len(path) < width else []
        if heat <= 0.0:
            best = int(np.argmax(row))
            children = [j for j in children if ids[j] == best]
            if not children:
                return path, best
            here = children[0]
            path.append(here)
            continue
        left = np.exp((row - row.max()) / heat)
        left /= left.sum()
        guess = None
        if draft is not None and children:
            guess = draft[here].astype(np.float64)
            if np.isnan(guess).any() or guess.max() in (np.inf, -np.inf):
                return path, -1
            guess = np.exp((guess - guess.max()) / heat)
            guess /= guess.sum()
        stands = None
        for j in children:
            token = int(ids[j])
            if not 0 <= token < vocab:
                continue
            q = np.zeros(vocab)
            if guess is None:
                q[token] = 1.0
            else:
                q = guess
            if q.sum() <= 0.0:
                continue
            if uniform[j] * q[token] < left[token]:
                stands = j
                break
            left = np.maximum(left - q, 0.0)
            left /= left.sum()
            if guess is not None and not replacement:
                guess = guess.copy()
                guess[token] = 0.0
                if guess.sum() > 0.0:
                    guess /= guess.sum()
        if stands is None:
            sums = np.cumsum(left)
            return path, int(np.searchsorted(sums, uniform[0] * sums[-1], side="right"))
        here = stands
        path.append(here)
