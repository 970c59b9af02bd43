"""Trees of drafted tokens on the host: masks, and what the operators refuse before any launch."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from helix_runtime_b200.engine.step import ancestor_words
from helix_runtime_b200.ops import library as ops
from plain_tree import ancestors, random_parents, words_of


@pytest.mark.parametrize("count", [1, 2, 63, 64, 65, 130])
def test_masks_name_ancestors(count):
    parents = random_parents(np.random.default_rng(count), count)
    words = -(-count // 64)
    assert np.array_equal(ancestor_words(parents), words_of(ancestors(parents), words))
    assert np.array_equal(ancestor_words(parents, words + 2)[:, :words], ancestor_words(parents))
    assert not ancestor_words(parents, words + 2)[:, words:].any()


def test_trees_that_are_none():
    for parents in ([0], [-1, 1], [-1, 0, 3], [-1, -1], [-1, 0, -2], [1, 0]):
        with pytest.raises(ValueError):
            ancestor_words(parents)
    with pytest.raises(ValueError):
        ancestor_words([-1] + list(range(64)), words=1)
    assert ancestor_words([]).shape == (0, 1)


def test_entry_points_refuse_sizes_on_the_host():
    """Refused by the library itself, with a message, and nothing launched."""
    library, launches = ops.lib(), ops.launch_count()
    word = (ctypes.c_int * 4)()
    some = ctypes.addressof(word) & ~15

    def attention(dtype=1, words=1, ld=1, heads=4, kv_heads=2, dim=64, page=16, pages=8, stride=4, scale=1.0,
                  partial=some, status=some, requests=1, k=some):
        return library.hx_tree_attention(some, 256, k, some, dtype, some, ld, words, some, some, some, some, stride,
                                         some, 256, partial, requests, heads, kv_heads, dim, page, pages, scale, 0,
                                         status, None)

    for changes in (dict(dtype=2), dict(words=0), dict(ld=0), dict(heads=3), dict(heads=0), dict(kv_heads=0),
                    dict(dim=0), dict(dim=7), dict(dim=1026), dict(page=0), dict(pages=0), dict(stride=0),
                    dict(scale=0.0), dict(scale=float("nan")), dict(partial=None), dict(status=None),
                    dict(requests=-1), dict(k=some + 2), dict(pages=2 ** 31 - 1)):
        assert attention(**changes) == -1, changes
        assert b"hx_tree_attention" in library.hx_last_error()
    assert attention(requests=0) == 0

    def verify(ld=64, draft=None, ld_draft=0, vocab=64, ld_path=4, width=4, requests=1, uniform=some, status=some):
        return library.hx_verify_drafts(some, ld, draft, ld_draft, vocab, some, some, some, some, uniform, some,
                                        ld_path, width, some, some, requests, 0, status, None)

    for changes in (dict(ld=63), dict(draft=some, ld_draft=63), dict(vocab=0), dict(width=0), dict(ld_path=3),
                    dict(requests=-1), dict(uniform=None), dict(status=None)):
        assert verify(**changes) == -1, changes
    assert verify(requests=0) == 0

    def keep(dtype=1, planes=4, pages=8, kv_heads=2, page=16, dim=64, stride=4, ld_path=4, width=4, requests=1,
             status=some, storage=some):
        return library.hx_keep_rows(storage, dtype, planes, pages, kv_heads, page, dim, some, stride, some, some, some,
                                    ld_path, width, some, requests, status, None)

    for changes in (dict(dtype=3), dict(planes=0), dict(planes=2 ** 30), dict(pages=0), dict(kv_heads=0), dict(page=0),
                    dict(dim=0), dict(dim=9), dict(stride=0), dict(ld_path=3), dict(width=0), dict(requests=-1),
                    dict(requests=65536), dict(status=None), dict(storage=some + 8)):
        assert keep(**changes) == -1, changes
    assert keep(requests=0) == 0

    def copy(planes=4, pages=8, size=64, pairs=1, status=some, storage=some):
        return library.hx_copy_pages(storage, planes, pages, size, some, some, pairs, status, None)

    for changes in (dict(planes=0), dict(planes=65536), dict(pages=0), dict(size=0), dict(size=6), dict(pairs=-1),
                    dict(pairs=65536), dict(status=None), dict(storage=some + 2)):
        assert copy(**changes) == -1, changes
    assert copy(pairs=0) == 0
    assert library.hx_tree_attention_scratch_floats(1, 4, 3, 64, 16) == -1
    assert ops.launch_count() == launches


def test_operators_refuse_tensors_of_the_host():
    storage = torch.zeros((1, 2, 4, 1, 16, 8))
    pages = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ops.KernelError):
        ops.copy_pages(storage, pages, pages, pages)
    with pytest.raises(ops.KernelError):
        ops.keep_rows(storage, pages[None], pages, pages, pages[None], pages, 1, pages)
    with pytest.raises(ops.KernelError):
        ops.verify_drafts(torch.zeros((1, 4)), None, pages, pages, pages, storage, storage, pages[None], pages, pages, 1,
                          pages)
    with pytest.raises(ops.KernelError):
        ops.tree_attention(torch.zeros((1, 8)), storage, storage, torch.zeros((1, 1), dtype=torch.int64), pages, pages,
                           pages, pages[None], torch.zeros((1, 8)), None, 1, 1, 1, 8, 16, 4, 1.0, pages)
