"""Moving kept rows and whole pages of the paged cache, against indexing on the host."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helix_runtime_b200.ops import library as ops
from plain_tree import from_cache, to_cache

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


class Rows:
    """Requests with `width` rows behind their cached ones, in shuffled pages."""

    def __init__(self, seed, contexts, paths, layers=2, kv_heads=2, head_dim=64, page=16, dtype=torch.bfloat16,
                 width=None):
        rng = np.random.default_rng(seed)
        self.contexts, self.paths, self.page, self.dtype = contexts, paths, page, dtype
        reach = [c + max([*p, 0]) + 1 for c, p in zip(contexts, paths)]
        needed = [-(-n // page) for n in reach]
        self.num_pages = sum(needed) + 3
        order = rng.permutation(self.num_pages)
        self.table_rows = rng.permutation(len(contexts) + 2)[:len(contexts)]
        self.tables = np.full((len(contexts) + 2, max(needed)), -1, dtype=np.int32)
        cursor = 0
        for r, count in enumerate(needed):
            self.tables[self.table_rows[r], :count] = order[cursor:cursor + count]
            cursor += count
        shape = (layers, 2, self.num_pages, kv_heads, page, head_dim)
        self.rows = torch.as_tensor(rng.integers(-10 ** 6, 10 ** 6, shape)).to(dtype)
        self.storage = to_cache(self.rows, dtype).to(DEVICE)
        self.width = width or max(1, max(len(p) for p in paths))
        self.path = np.full((len(paths), self.width), -1, dtype=np.int32)
        for r, p in enumerate(paths):
            self.path[r, :min(len(p), self.width)] = p[:self.width]
        self.kept = [len(p) for p in paths]

    def tensor(self, array):
        return torch.as_tensor(np.asarray(array, dtype=np.int32), device=DEVICE)

    def run(self, requests=None):
        self.status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        self.arguments = (self.tensor(self.tables), self.tensor(self.table_rows), self.tensor(self.contexts),
                          self.tensor(self.path), self.tensor(self.kept),
                          len(self.contexts) if requests is None else requests, self.status)
        ops.keep_rows(self.storage, *self.arguments)
        return self

    def place(self, r, place):
        return int(self.tables[self.table_rows[r], place // self.page]), place % self.page

    def check(self, left=(), status=0):
        want = self.rows.clone()
        for r, p in enumerate(self.paths):
            if r in left:
                continue
            for k, j in enumerate(p):
                page, slot = self.place(r, self.contexts[r] + j)
                to_page, to_slot = self.place(r, self.contexts[r] + k)
                want[:, :, to_page, :, to_slot] = self.rows[:, :, page, :, slot]
        got = from_cache(self.storage).cpu()
        assert torch.equal(got, want)
        assert int(self.status.item()) == status


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("head_dim,kv_heads,page", [(128, 4, 16), (112, 3, 32), (64, 2, 64), (12, 1, 5), (6, 2, 1),
                                                    (2, 1, 16)])
def test_paths(dtype, head_dim, kv_heads, page):
    rng = np.random.default_rng(head_dim)
    contexts = [0, 15, 16, 100, 3, 64]
    paths = [[0], [0, 3, 4], [0, 1, 2, 3], [0, 2, 3, 4, 5, 6, 7], [], sorted(rng.choice(70, 40, replace=False))]
    Rows(1, contexts, paths, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype).run().check()


def test_paths_longer_than_a_warp_and_a_block():
    """Rows that move by one over others that move: every old row is read before it is written."""
    for count in (31, 32, 33, 64, 65, 300, 700):
        Rows(2, [7, 9], [[0] + list(range(2, count + 1)), list(range(5, count + 5))], layers=1, page=16).run().check()


def test_requests_are_apart():
    rng = np.random.default_rng(3)
    contexts = [int(c) for c in rng.integers(0, 50, 40)]
    paths = [[0] + sorted(int(j) for j in rng.choice(np.arange(1, 30), rng.integers(0, 9), replace=False))
             for _ in contexts]
    Rows(3, contexts, paths, layers=3).run().check()
    Rows(3, contexts, paths, layers=1).run(requests=11).check(left=range(11, 40))


def test_paths_that_are_none_are_left():
    """A path that does not ascend, is longer than its row, or leads outside the request's pages."""
    good = [0, 2, 5]
    for bad in ([0, 5, 5], [0, 7, 3], [-1, 2, 3]):
        Rows(4, [20, 20], [good, bad]).run().check(left=[1], status=ops.FLAG_BAD_MOVE)
    rows = Rows(5, [20, 20], [good, [0, 2, 3, 8]], width=3)
    rows.run().check(left=[1], status=ops.FLAG_BAD_MOVE)
    rows = Rows(6, [20, 20], [good, [0, 4, 30]])
    rows.tables[rows.table_rows[1], 3] = -1
    rows.run().check(left=[1], status=ops.FLAG_BAD_PAGE)
    rows = Rows(6, [20, 20], [good, [0, 4, 30]])
    rows.tables[rows.table_rows[1], 3] = rows.num_pages
    rows.run().check(left=[1], status=ops.FLAG_BAD_PAGE)
    rows = Rows(6, [20, 20], [good, [0, 4, 30]])
    rows.path[1, 2] = 2 ** 31 - 5
    rows.run().check(left=[1], status=ops.FLAG_BAD_MOVE)
    rows = Rows(6, [20, 20], [good, [0, 4, 30]])
    rows.path[1, 2] = 10 ** 6
    rows.run().check(left=[1], status=ops.FLAG_BAD_PAGE)


def test_keep_recorded_and_replayed():
    rows = Rows(7, [20, 33], [[0, 2, 5], [0, 1, 4]]).run()
    rows.check()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.keep_rows(rows.storage, *rows.arguments)
    rows.storage.copy_(to_cache(rows.rows, rows.dtype))
    rows.paths = [[0, 3], [0, 2, 4]]
    rows.arguments[3].copy_(rows.tensor([[0, 3, -1], [0, 2, 4]]))
    rows.arguments[4].copy_(rows.tensor([2, 3]))
    graph.replay()
    torch.cuda.synchronize()
    rows.check()


def pages_of(shape, dtype, seed=0):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    return torch.randn(shape, generator=generator, device=DEVICE).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(2, 2, 9, 4, 16, 128), (1, 2, 9, 3, 5, 6), (3, 2, 9, 1, 1, 2), (1, 2, 9, 2, 32, 112),
                                   (2, 2, 9, 8, 64, 256)])
def test_copied_pages(dtype, shape):
    storage = pages_of(shape, dtype)
    before = storage.clone()
    source, target = [3, 0, 3, 8], [1, 7, 2, 4]
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    ops.copy_pages(storage, torch.tensor(source, dtype=torch.int32, device=DEVICE),
                   torch.tensor(target, dtype=torch.int32, device=DEVICE), status)
    before[:, :, target] = before[:, :, source]
    assert torch.equal(storage, before) and int(status.item()) == 0


@pytest.mark.parametrize("source,target,copied,flag", [
    ([0, 1], [2, 9], [0], "FLAG_BAD_PAGE"),            # outside the pool
    ([0, -1], [2, 3], [0], "FLAG_BAD_PAGE"),
    ([0, 1], [2, 2], [], "FLAG_BAD_MOVE"),             # two pairs write one page
    ([0, 2], [2, 3], [1], "FLAG_BAD_MOVE"),            # a page that another pair reads
    ([0, 1], [1, 0], [], "FLAG_BAD_MOVE"),
    ([4, 1], [4, 3], [1], None),                       # a page onto itself
])
def test_pairs_that_cannot_be_copied(source, target, copied, flag):
    storage = pages_of((2, 2, 9, 2, 16, 64), torch.bfloat16)
    want = storage.clone()
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    ops.copy_pages(storage, torch.tensor(source, dtype=torch.int32, device=DEVICE),
                   torch.tensor(target, dtype=torch.int32, device=DEVICE), status)
    for i in copied:
        want[:, :, target[i]] = want[:, :, source[i]]
    assert torch.equal(storage, want)
    assert int(status.item()) == (getattr(ops, flag) if flag else 0)


def test_more_pairs_than_a_block_has_threads():
    storage = pages_of((1, 2, 1300, 1, 4, 8), torch.float32)
    want = storage.clone()
    order = torch.randperm(1300, generator=torch.Generator().manual_seed(3)).to(device=DEVICE, dtype=torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    ops.copy_pages(storage, order[:650], order[650:], status)
    want[:, :, order[650:].long()] = want[:, :, order[:650].long()]
    assert torch.equal(storage, want) and int(status.item()) == 0
    ops.copy_pages(storage, order[:0], order[:0], status)
    assert torch.equal(storage, want)


def test_storage_beyond_32_bits():
    """Planes that begin behind the first 2^32 bytes: a page's copy, and kept rows."""
    shape = (6, 2, 900, 32, 16, 64)                     # 708 MB of keys a layer
    storage = torch.zeros(shape, dtype=torch.float32, device=DEVICE)
    storage[:, :, 3] = pages_of((6, 2, 32, 16, 64), torch.float32)
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    ops.copy_pages(storage, torch.tensor([3], dtype=torch.int32, device=DEVICE),
                   torch.tensor([899], dtype=torch.int32, device=DEVICE), status)
    assert torch.equal(storage[:, :, 899], storage[:, :, 3])
    one = torch.tensor([0], dtype=torch.int32, device=DEVICE)
    ops.keep_rows(storage, torch.tensor([[899]], dtype=torch.int32, device=DEVICE), one, one + 2,
                  torch.tensor([[0, 4]], dtype=torch.int32, device=DEVICE), one + 2, 1, status)
    kept, old = from_cache(storage[:, :, 899]), from_cache(storage[:, :, 3])
    assert torch.equal(kept[..., 3, :], old[..., 6, :]) and torch.equal(kept[..., 4:, :], old[..., 4:, :])
    assert int(status.item()) == 0 and not bool(storage[:, :, 4:899].any())


def test_refusals():
    rows = Rows(8, [20], [[0, 2, 5]]).run()
    tables, table_rows, contexts, path, kept, requests, status = rows.arguments
    with pytest.raises(ops.KernelError):
        ops.keep_rows(rows.storage[:, :, :4], *rows.arguments)          # not contiguous
    with pytest.raises(ops.KernelError):
        ops.keep_rows(rows.storage[0], *rows.arguments)
    with pytest.raises(ops.KernelError):
        ops.keep_rows(rows.storage.double(), *rows.arguments)
    with pytest.raises(ops.KernelError):
        ops.keep_rows(rows.storage, tables.long(), *rows.arguments[1:])
    with pytest.raises(ops.KernelError):
        ops.keep_rows(rows.storage, tables, table_rows, contexts, path[:, ::2], kept, requests, status)
    with pytest.raises(ops.KernelError):
        ops.keep_rows(rows.storage, tables, table_rows, contexts, path, kept, 2, status)
    pages = path[0, :2].contiguous()
    with pytest.raises(ops.KernelError):
        ops.copy_pages(rows.storage, pages, pages[:1], status)
    with pytest.raises(ops.KernelError):
        ops.copy_pages(rows.storage, pages.long(), pages.long(), status)
    with pytest.raises(ops.KernelError):
        ops.copy_pages(rows.storage.cpu(), pages, pages, status)
