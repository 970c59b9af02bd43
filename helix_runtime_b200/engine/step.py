"""The step function: one batch of (request, its next tokens) through the model.

A step holds, for every request in it, the next tokens of that request: a portion of
a prompt (cut anywhere) or a single decoded token.  All of them run as ONE flattened
batch against the cache that earlier steps left, and the logits at the wanted
positions come back.  The reference has no such function; its engine runs the work
items of an iteration one after the other (src/runtime/cpu_engine.cpp:344-361).

Transaction: pages are reserved before the launch and lengths are published after
it; if anything raises, reserved pages go back and no length moves
(src/runtime/cpu_engine.cpp:191, 207, 235).
"""
from __future__ import annotations

import dataclasses
from typing import Hashable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..cache.manager import CacheManager
from ..models.decoder import DecoderModel
from ..ops import library as ops
from ..parts.base import DraftedTrees, StepContext, Workspace


def ancestor_words(parents: Sequence[int], words: int = 0) -> np.ndarray:
    """The masks of a tree of drafted tokens (``parents``: each one's number, smaller than its
    child's; -1 for token 0), int64 ``[tokens, words]`` as
    :func:`helix_runtime_b200.ops.library.tree_attention` reads them: bit ``j`` of word ``w`` of a
    token's row is set where token ``64 w + j`` is itself or an ancestor.  ``words`` 0: as many as
    the tokens need."""
    count = len(parents)
    words = words or max(1, -(-count // 64))
    if count > 64 * words:
        raise ValueError(f"{count} tokens need {-(-count // 64)} words of 64 bits")
    masks = np.zeros((count, words), dtype=np.uint64)
    for token, parent in enumerate(parents):
        if not (parent == -1 if token == 0 else 0 <= parent < token):
            raise ValueError(f"token {token} of a tree has the parent {parent}: token 0 has -1, every "
                             "other one that comes before it")
        if token:
            masks[token] = masks[parent]
        masks[token, token // 64] |= np.uint64(1) << np.uint64(token % 64)
    return masks.view(np.int64)


@dataclasses.dataclass
class StepEntry:
    request: Hashable
    tokens: Sequence[int]
    want: Sequence[int] = ()          # places among ``tokens`` whose logits are asked for
    # Drafted tokens: ``tokens`` are a tree, token 0 its root and the rest drafts of what follows
    # their parents (each one's number among ``tokens``, smaller than its own; -1 for token 0).
    # A token sees the cached ones and its ancestors, and its position is its depth behind them.
    # Nothing of a tree is published before :meth:`StepFunction.keep` says what stays.
    parents: Optional[Sequence[int]] = None


@dataclasses.dataclass
class OpenTrees:
    """A step of drafted trees whose requests wait for :meth:`StepFunction.keep`, from its
    preparation on: what they are moved by lies where the next step's description would."""
    entries: List[StepEntry]
    ctx: StepContext
    admissions: List[object]          # each entry's request as admitted, see CacheManager.admission
    lengths: List[int]                # up to where each has reserved
    run: bool = False


class StepError(RuntimeError):
    """The batch is not runnable (bad token, too long, unknown request) or a kernel failed."""


class StepFunction:
    def __init__(self, model: DecoderModel, cache: CacheManager, max_tokens: int,
                 max_requests: int, attention_split_keys: int = 256,
                 ordered_sums: bool = False) -> None:
        if model.device is None:
            raise StepError("the model has no weights bound")
        self.model = model
        self.cache = cache
        self.device = model.device
        self.dtype = model.dtype
        self.max_tokens = int(max_tokens)
        self.max_requests = int(max_requests)
        self.attention_split_keys = int(attention_split_keys)
        self.ordered_sums = bool(ordered_sums)
        self.workspace = Workspace(self.device)
        cap, req = self.max_tokens, self.max_requests
        # one packed int32 block: a single host-to-device copy per step
        self._layout = {}
        cursor = 0
        for name, size in (("token_ids", cap), ("positions", cap), ("token_request", cap),
                           ("want_rows", cap), ("request_slot", req), ("request_start", req + 1),
                           ("request_context", req), ("feed_rows", req)):
            self._layout[name] = (cursor, cursor + size)
            cursor += size
        pin = self.device.type == "cuda"
        self._host = torch.zeros(cursor, dtype=torch.int32, pin_memory=pin)
        self._host_np = self._host.numpy()
        self._device = torch.zeros(cursor, dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._uploaded = torch.cuda.Event() if pin else None
        self._tree_host: Optional[torch.Tensor] = None      # made at the first step of trees
        self._tree_device: Optional[torch.Tensor] = None
        self._trees: Optional[OpenTrees] = None
        self.last_context: Optional[StepContext] = None
        self.steps_run = 0
        self.tokens_run = 0

    def _view(self, name: str, device: bool):
        begin, end = self._layout[name]
        return (self._device if device else self._host_np)[begin:end]

    # --------------------------------------------------------------------- run

    @property
    def upload_bytes(self) -> int:
        """Bytes of the packed batch description that every step copies to the device."""
        return self._host.numel() * self._host.element_size()

    @property
    def feed_rows(self) -> torch.Tensor:
        """Device view of the rows named by ``prepare(..., feed_rows=...)``."""
        return self._view("feed_rows", True)

    def prepare(self, entries: Sequence[StepEntry], context_hint: int = 0,
                feed_rows: Optional[Sequence[int]] = None):
        """Validate, reserve pages, fill and upload the batch description.
        Returns ``(context, want_rows_device, n_want, new_lengths)``.  ``context_hint`` raises
        the context length that launches are sized for (a caller that will replay the step
        while the requests grow passes the length they will reach).  ``feed_rows``: the step
        is prepared before the host knows its tokens; every entry brings one placeholder token
        and names the row of the previous step's sampled tokens that the device puts in its
        place (:func:`helix_runtime_b200.ops.library.feed_tokens`)."""
        if not entries:
            raise StepError("a step needs at least one entry")
        if len(entries) > self.max_requests:
            raise StepError(f"{len(entries)} requests in one step, at most {self.max_requests}")
        total = sum(len(entry.tokens) for entry in entries)
        if feed_rows is not None and (len(feed_rows) != len(entries) or total != len(entries)):
            raise StepError("a step fed on the device has one token and one row per request")
        if self._trees is not None:
            if any(self._open_trees()):
                raise StepError("the last step's drafted trees wait for what is kept of them")
            self._trees = None
        masks = self._tree_masks(entries, feed_rows) \
            if any(entry.parents is not None for entry in entries) else None
        if total > self.max_tokens:
            raise StepError(f"{total} tokens in one step, at most {self.max_tokens}")
        seen = set()
        vocab = self.model.vocab_size
        for entry in entries:
            if entry.request in seen:
                raise StepError(f"request {entry.request!r} appears twice in one step")
            seen.add(entry.request)
            if not self.cache.has(entry.request):
                raise StepError(f"request {entry.request!r} is not admitted to the cache")
            if len(entry.tokens) == 0:
                raise StepError(f"request {entry.request!r} brings no tokens")
            ids = np.asarray(entry.tokens, dtype=np.int64)
            if ids.ndim != 1 or int(ids.min()) < 0 or int(ids.max()) >= vocab:
                bad = [int(t) for t in ids.reshape(-1) if not 0 <= int(t) < vocab][:1]
                raise StepError(f"token id {bad[0] if bad else '?'} of request {entry.request!r} "
                                f"is outside the vocabulary of {vocab}")
            for place in entry.want:
                if not 0 <= int(place) < len(entry.tokens):
                    raise StepError(f"wanted place {place} of request {entry.request!r} is "
                                    f"outside its {len(entry.tokens)} tokens")
            if self.cache.reserved(entry.request) + len(entry.tokens) > self.model.max_positions:
                raise StepError(f"request {entry.request!r} would exceed the model's "
                                f"{self.model.max_positions} positions")

        if self._uploaded is not None:
            self._uploaded.synchronize()    # the last upload has left the pinned block
        token_ids = self._view("token_ids", False)
        positions = self._view("positions", False)
        token_request = self._view("token_request", False)
        want_rows = self._view("want_rows", False)
        request_slot = self._view("request_slot", False)
        request_start = self._view("request_start", False)
        request_context = self._view("request_context", False)

        new_lengths: List[int] = []
        reserved: List[Tuple[Hashable, int]] = []
        cursor = 0
        n_want = 0
        max_query = 0
        min_query = 1 << 30
        max_context = 0
        try:
            for index, entry in enumerate(entries):
                count = len(entry.tokens)
                # a step still in flight has reserved its positions already: go on from there
                before = self.cache.reserved(entry.request)
                self.cache.extend(entry.request, before + count)
                reserved.append((entry.request, before))
                token_ids[cursor:cursor + count] = np.asarray(entry.tokens, dtype=np.int32)
                if masks is None:
                    positions[cursor:cursor + count] = np.arange(before, before + count, dtype=np.int32)
                else:
                    self._fill_tree(entry, before, cursor, positions, masks[index])
                token_request[cursor:cursor + count] = index
                request_slot[index] = self.cache.slot(entry.request)
                request_start[index] = cursor
                request_context[index] = before
                for place in entry.want:
                    want_rows[n_want] = cursor + int(place)
                    n_want += 1
                cursor += count
                new_lengths.append(before + count)
                max_query = max(max_query, count)
                min_query = min(min_query, count)
                max_context = max(max_context, before + count)
            request_start[len(entries)] = cursor
            if feed_rows is not None:
                self._view("feed_rows", False)[:len(entries)] = np.asarray(feed_rows, dtype=np.int32)
        except Exception:
            for request, before in reserved:
                self.cache.rollback(request, keep_length=before)
            raise

        self._device.copy_(self._host, non_blocking=True)
        trees = None if masks is None else self._upload_trees(cursor, masks)
        if self._uploaded is not None:
            self._uploaded.record()
        self.cache.sync_tables()
        ctx = StepContext(
            dtype=self.dtype, device=self.device, workspace=self.workspace,
            capacity=self.max_tokens, n_tokens=cursor, n_requests=len(entries),
            token_ids=self._view("token_ids", True), positions=self._view("positions", True),
            token_request=self._view("token_request", True),
            request_slot=self._view("request_slot", True),
            request_start=self._view("request_start", True),
            request_context=self._view("request_context", True),
            status=self.status, max_query_len=max_query, min_query_len=min_query,
            max_context_len=max(max_context, context_hint),
            attention_split_keys=self.attention_split_keys, ordered_sums=self.ordered_sums,
            host_request_slots=[int(v) for v in request_slot[:len(entries)]],
            host_request_starts=[int(v) for v in request_start[:len(entries) + 1]],
            host_request_contexts=[int(v) for v in request_context[:len(entries)]],
            host_query_lengths=[len(entry.tokens) for entry in entries], trees=trees,
        )
        if trees is not None:
            self._trees = OpenTrees(list(entries), ctx,
                                    [self.cache.admission(entry.request) for entry in entries],
                                    list(new_lengths))
        return ctx, self._view("want_rows", True), n_want, new_lengths

    # ----------------------------------------------------------- drafted trees

    def _tree_masks(self, entries: Sequence[StepEntry], feed_rows) -> List[np.ndarray]:
        """The entries' masks, all as wide as the largest tree's."""
        if feed_rows is not None or any(entry.parents is None for entry in entries):
            raise StepError("a step brings drafted trees for all of its requests or for none")
        if not self.model.takes_trees:
            raise StepError("the model has a part that takes no drafted trees")
        words = max(1, -(-max(len(entry.tokens) for entry in entries) // 64))
        masks = []
        for entry in entries:
            if len(entry.parents) != len(entry.tokens):
                raise StepError(f"request {entry.request!r} brings {len(entry.tokens)} tokens and "
                                f"{len(entry.parents)} parents")
            try:
                masks.append(ancestor_words(entry.parents, words))
            except ValueError as error:
                raise StepError(f"request {entry.request!r}: {error}") from None
        size = self.max_tokens * (1 + words)
        if self._tree_host is None or self._tree_host.numel() < size:
            # places and parents (two int32 an element), then the masks
            self._tree_host = torch.zeros(size, dtype=torch.int64, pin_memory=self._uploaded is not None)
            self._tree_device = torch.zeros(size, dtype=torch.int64, device=self.device)
        return masks

    def _fill_tree(self, entry: StepEntry, before: int, cursor: int, positions: np.ndarray,
                   mask: np.ndarray) -> None:
        count, words = mask.shape
        depth = np.zeros(count, dtype=np.int32)
        for token in range(1, count):
            depth[token] = depth[entry.parents[token]] + 1
        positions[cursor:cursor + count] = before + depth
        block, cap = self._tree_host.numpy(), self.max_tokens
        places, parents = block[:cap].view(np.int32).reshape(2, cap)
        places[cursor:cursor + count] = np.arange(before, before + count, dtype=np.int32)
        parents[cursor:cursor + count] = np.asarray(entry.parents, dtype=np.int32)
        block[cap + cursor * words:cap + (cursor + count) * words] = mask.reshape(-1)

    def _upload_trees(self, tokens: int, masks: List[np.ndarray]) -> DraftedTrees:
        cap, words = self.max_tokens, masks[0].shape[1]
        used = cap + tokens * words
        self._tree_device[:used].copy_(self._tree_host[:used], non_blocking=True)
        places, parents = self._tree_device[:cap].view(torch.int32).view(2, cap)
        return DraftedTrees(self._tree_device[cap:used].view(tokens, words), places, parents)

    def _open_trees(self) -> List[bool]:
        """Which requests of the last step of trees still hold what it reserved for them (one that
        has ended, though another of its name may be there, or whose step was given up does not)."""
        open_trees = self._trees
        return [admission is not None and self.cache.admission(entry.request) is admission
                and self.cache.reserved(entry.request) == length
                for entry, admission, length in zip(open_trees.entries, open_trees.admissions,
                                                    open_trees.lengths)]

    def keep(self, path: torch.Tensor, kept: torch.Tensor) -> List[int]:
        """Settle the last step's drafted trees: of request ``r`` (in the order of the entries) the
        ``kept[r]`` tokens ``path[r]`` stay, a branch from the root down, as
        :meth:`helix_runtime_b200.sampling.sampler.Sampler.verify` names them.  Their keys and
        values move together, the request's length is published and the other tokens' pages are
        given back.  Returns the tokens kept of each (waits for the device).  What is no branch of its
        tree is refused and changes nothing."""
        if self._trees is None:
            raise StepError("the last step brought no drafted trees")
        if not self._trees.run:
            raise StepError("the step of the drafted trees has not run")
        entries, ctx = self._trees.entries, self._trees.ctx
        live = self._open_trees()
        for entry, there, context in zip(entries, live, ctx.host_request_contexts):
            if there and self.cache.length(entry.request) != context:
                raise StepError(f"an earlier step of request {entry.request!r} has not been published")
        if not all(live):
            # what a request that has ended held may be another's by now
            kept = kept[:len(entries)] * torch.tensor(live, dtype=kept.dtype, device=kept.device)
        counts = kept[:len(entries)].tolist()
        for entry, count, row in zip(entries, counts, path[:len(entries)].tolist()):
            if not 0 <= count <= min(len(entry.tokens), len(row)):
                raise StepError(f"{count} tokens kept of the {len(entry.tokens)} of request "
                                f"{entry.request!r}")
            for token, parent in zip(row[:count], [-1] + row):
                if not 0 <= token < len(entry.tokens) or entry.parents[token] != parent:
                    raise StepError(f"what is kept of request {entry.request!r} is no branch of its "
                                    "tree from the root down")
        for group in self.cache.groups:
            ops.keep_rows(group.storage, group.device_tables, ctx.request_slot, ctx.request_context,
                          path, kept, len(entries), self.status)
        self._trees = None
        try:
            self.raise_on_status()
        except Exception:
            self.fail(entries)
            raise
        for entry, count, there in zip(entries, counts, live):
            if there:
                self.cache.commit(entry.request, self.cache.length(entry.request) + count)
                self.cache.rollback(entry.request)
        return counts

    def run(self, entries: Sequence[StepEntry], check_status: bool = True) -> Optional[torch.Tensor]:
        """Run one step.  Returns float32 logits ``[wanted, vocab]`` in the order of the entries
        and of their ``want`` lists (a view that the next step overwrites), or None."""
        ctx, want_rows, n_want, new_lengths = self.prepare(entries)
        try:
            logits = self.model.forward(ctx, self.cache, want_rows, n_want)
            if check_status:
                self.raise_on_status()
        except Exception:
            self.fail(entries)
            raise
        self.finish(entries, new_lengths, ctx)
        return logits

    def finish(self, entries: Sequence[StepEntry], new_lengths: Sequence[int],
               ctx: StepContext) -> None:
        """The step succeeded: publish the new lengths (drafted trees wait for :meth:`keep`)."""
        if ctx.trees is not None:
            if self._trees is not None and self._trees.ctx is ctx:
                self._trees.run = True
        else:
            for entry, length in zip(entries, new_lengths):
                if self.cache.has(entry.request):    # a request may have ended while in flight
                    self.cache.commit(entry.request, length)
        self.last_context = ctx
        self.steps_run += 1
        self.tokens_run += ctx.n_tokens

    def fail(self, entries: Sequence[StepEntry],
             keep_lengths: Optional[Sequence[int]] = None, after: Optional[int] = None) -> None:
        """The step failed: give back what was reserved for it; no length moves.
        ``keep_lengths``: what an earlier step that is still in flight has reserved for each
        entry, which stays.  ``after``: a later step, already queued on the device, that may
        still write the pages given back (they are parked until it completes)."""
        self.workspace.clear_accumulators()
        for index, entry in enumerate(entries):
            if self.cache.has(entry.request):
                self.cache.rollback(entry.request,
                                    None if keep_lengths is None else keep_lengths[index],
                                    after=after)
        if self._trees is not None and not any(self._open_trees()):
            self._trees = None

    @staticmethod
    def describe_status(flags: int) -> str:
        names = [name for bit, name in ((ops.FLAG_BAD_TOKEN, "token id outside the vocabulary"),
                                        (ops.FLAG_BAD_PAGE, "block table entry outside the pool"),
                                        (ops.FLAG_WAIT_TIMEOUT, "a bounded kernel wait ran out"),
                                        (ops.FLAG_NONFINITE, "non-finite logits"),
                                        (ops.FLAG_BAD_POSITION,
                                         "a position outside the position table"),
                                        (ops.FLAG_BAD_MOVE,
                                         "a move in the cache over what another needs"))
                 if flags & bit]
        return "the step's kernels reported: " + "; ".join(names)

    def raise_on_status(self) -> None:
        """Read the device status word (synchronises) and raise if a kernel flagged a fault."""
        flags = int(self.status.item())
        if flags:
            self.status.zero_()
            raise StepError(self.describe_status(flags))
