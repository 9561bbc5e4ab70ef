"""Rows of a paged cache by the numbers of its sequences; CPU only."""

from __future__ import annotations

import pytest
import torch

from local_kimi_amd.paged import PagedCache


def _cache():
    return PagedCache(8, 3, 48, layers=1, kv_heads=1, d_qk=8, d_v=8, page_rows=16, dtype=torch.float16, device="cpu")


@pytest.mark.parametrize("sequences,named", [([3], 3), ([0, -1], -1), ([0, 1, 2, 99], 99), ([2 ** 40], 2 ** 40)])
def test_rows_of_sequences_that_there_are_not(sequences, named):
    with pytest.raises(ValueError, match=f"there is no sequence {named} of 3"):
        _cache().rows_of(sequences)


def test_rows_of_sequences_in_any_order():
    cache = _cache()
    a, b = cache.add(), cache.add()
    cache.extend([a, b], [20, 3])
    for order in ([b, a], (b, a), torch.tensor([b, a])):
        table, lengths = cache.rows_of(order)
        assert table.tolist() == [[2, -1, -1], [0, 1, -1]] and lengths.tolist() == [3, 20]
    table, lengths = cache.rows_of([2, a, a])  # not in use; one twice
    assert table.tolist() == [[-1, -1, -1], [0, 1, -1], [0, 1, -1]] and lengths.tolist() == [0, 20, 20]
    table, lengths = cache.rows_of([])
    assert table.shape == (0, 3) and lengths.shape == (0,)


@pytest.mark.parametrize("of", [list, tuple, torch.tensor, lambda x: torch.tensor(x).numpy()])
def test_numbers_of_any_kind(of):
    """A sequence named twice is refused however it is named, and changes nothing; the book keeps
    plain numbers."""
    cache = _cache()
    a, b = cache.add(), cache.add()
    with pytest.raises(ValueError, match="each sequence once"):
        cache.extend(of([a, a]), of([1, 1]))
    assert cache.book.lengths == [0, 0, 0] and cache.book.free_pages == 8
    cache.extend(of([a, b]), of([17, 2]))
    cache.extend(of([b, a]), of([0, 1]))
    assert cache.lengths.tolist() == [18, 2, 0] and cache.step_lengths.tolist() == [18, 0, 0]
    assert all(type(n) is int for n in cache.book.lengths)
    for s in of([a]):
        cache.free(s)
    assert cache.lengths.tolist() == [0, 2, 0] and cache.fork(b) == a
    assert cache.lengths.tolist() == [2, 2, 0] and cache.step_lengths.tolist() == [0, 0, 0]
