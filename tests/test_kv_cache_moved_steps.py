"""Steps and trees that a compaction moved: they count only while the pages that they wrote are still their sequences'.
Without a GPU: page moves are torch's."""

from __future__ import annotations

import pytest
import torch

from flextensor_amd import kv_cache as kvc

PAGE = 32


@pytest.fixture
def pool(monkeypatch):
    def copy(codes, scales, src, dst):
        codes.view(torch.uint8)[:, dst] = codes.view(torch.uint8)[:, src]
        scales[:, dst] = scales[:, src]

    monkeypatch.setattr(kvc, "copy_pages", copy)
    monkeypatch.setattr(kvc, "keep", lambda *args: None)
    return kvc.PagedKVCache(1, 1, 64, 16, page_tokens=PAGE, dtype=torch.int8, device="cpu")


def _moved(pool, reserve):
    """A sequence of 30 tokens with reserved pages, all of which a compaction moves."""
    first, a = pool.open(), pool.open()
    pool.commit(pool.begin([first, a], [100, 30]))
    held = reserve(a)
    pool.close(first)
    assert pool.compact()
    return a, held


def test_a_moved_step_whose_pages_were_given_back_does_not_count(pool):
    a, step = _moved(pool, lambda a: pool.begin([a], 40))
    pool.truncate(a, 30)  # the reserved pages are free again
    with pytest.raises(ValueError, match="changed"):
        pool.commit(step)
    assert pool.length(a) == 30


def test_a_moved_tree_whose_pages_were_given_back_is_not_accepted(pool):
    a, tree = _moved(pool, lambda a: pool.draft([a], [-1, 0, 0, 2]))
    pool.truncate(a, 30)
    with pytest.raises(ValueError, match="changed"):
        pool.accept(tree, [[0, 2, 3]])
    assert pool.length(a) == 30


def test_a_moved_step_and_a_moved_tree_that_nothing_touched_count(pool):
    a, step = _moved(pool, lambda a: pool.begin([a], 40))
    pool.commit(step)
    assert pool.length(a) == 70
    b, tree = _moved(pool, lambda a: pool.draft([a], [-1, 0, 0, 2]))
    pool.accept(tree, [[0, 2, 3]])
    assert pool.length(b) == 33
