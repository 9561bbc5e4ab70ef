"""The book of pages against a model that stores every sequence's tokens, and its
refusals; CPU only."""

from __future__ import annotations

import random

import pytest
import torch

from local_kimi_amd.paged import PageBook, PagedCache


def _same(book, store, model):
    """What the pages hold is what each sequence has; users are counted."""
    users = [0] * len(book.users)
    for s, tokens in model.items():
        held = book.pages[s]
        assert book.lengths[s] == len(tokens) and len(held) == -(-len(tokens) // book.page_rows)
        assert [store[p][i] for p in held for i in range(book.page_rows)][:len(tokens)] == tokens
        for p in held:
            users[p] += 1
    assert users == book.users
    assert sorted(book._free) == [p for p, n in enumerate(users) if not n]


@pytest.mark.parametrize("seed", range(6))
def test_sequences_keep_their_tokens(seed):
    rng = random.Random(seed)
    rows, pages = rng.choice([1, 4, 16]), rng.randint(4, 30)
    book = PageBook(pages, rows, 6, 9)
    store = [[None] * rows for _ in range(pages)]
    model, token, refused = {}, 0, 0
    for _ in range(400):
        what = rng.choice(["add", "fork", "free", "extend", "extend", "extend", "compact"])
        before = ([list(p) if p is not None else None for p in book.pages], list(book.users), list(book.lengths))
        try:
            if what == "add":
                model[book.add()] = []
            elif what == "fork" and model:
                s = rng.choice(list(model))
                model[book.fork(s)] = list(model[s])
            elif what == "free" and model:
                s = rng.choice(list(model))
                book.free(s)
                del model[s]
            elif what == "compact":
                src, dst = book.compact()
                assert not set(src) & set(dst) and len(set(dst)) == len(dst) == len(src)
                for a, b in zip(src, dst):
                    store[b] = list(store[a])
                used = [p for p, n in enumerate(book.users) if n]
                assert used == list(range(len(used)))
            elif what == "extend" and model:
                seqs = rng.sample(list(model), rng.randint(1, len(model)))
                counts = [rng.choice([0, 1, 1, rng.randint(0, 3 * rows)]) for _ in seqs]
                src, dst = book.extend(seqs, counts)
                assert not set(src) & set(dst) and len(set(dst)) == len(dst)
                for a, b in zip(src, dst):
                    store[b] = list(store[a])
                for s, n in zip(seqs, counts):
                    for _ in range(n):
                        at = len(model[s])
                        page = book.pages[s][at // rows]
                        assert book.users[page] == 1  # nobody else reads what is written
                        store[page][at % rows] = token
                        model[s].append(token)
                        token += 1
        except (RuntimeError, ValueError):
            refused += 1
            assert before == ([list(p) if p is not None else None for p in book.pages], book.users, book.lengths)
        _same(book, store, model)
    assert refused and token > 50


def test_refusals():
    book = PageBook(3, 16, 2, 2)
    with pytest.raises(ValueError, match="no sequence 0"):
        book.extend([0], [1])
    a = book.add()
    for seqs, counts in (([a, a], [1, 1]), ([a], [1, 2]), ([a], [-1])):
        with pytest.raises(ValueError):
            book.extend(seqs, counts)
    with pytest.raises(ValueError, match="at most 2"):
        book.extend([a], [33])
    b = book.add()
    with pytest.raises(RuntimeError, match="in use"):
        book.fork(a)
    book.extend([a], [32])
    with pytest.raises(RuntimeError, match="2 pages are needed, 1 are free"):
        book.extend([b], [17])
    book.free(b)
    with pytest.raises(ValueError, match="no sequence"):
        book.free(b)
    with pytest.raises(ValueError, match="no sequence"):
        book.fork(-1)
    for bad in ((-1, 16, 1, 1), (1, 0, 1, 1), (1, 16, 0, 1), (1, 16, 1, 0)):
        with pytest.raises(ValueError):
            PageBook(*bad)
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedCache(4, 2, 64, layers=1, kv_heads=1, d_qk=8, d_v=8, page_rows=24, device="cpu")


def test_two_that_share_a_page_and_both_grow_need_one_copy():
    book = PageBook(2, 16, 3, 4)
    a = book.add()
    book.extend([a], [5])
    b = book.fork(a)
    src, dst = book.extend([a, b], [1, 1])
    assert (src, dst) == ([0], [1]) and book.pages[a] == [1] and book.pages[b] == [0]
    full = PageBook(3, 16, 3, 4)
    a = full.add()
    full.extend([a], [16])
    b = full.fork(a)
    assert full.extend([a, b], [1, 1]) == ([], []) and full.pages[a] == [0, 1] and full.pages[b] == [0, 2]


def test_a_cache_mirrors_its_book():
    cache = PagedCache(6, 3, 40, layers=2, kv_heads=1, d_qk=8, d_v=16, page_rows=16, dtype=torch.float16,
                       device="cpu")
    assert len(cache.k_pages) == 2 and cache.v_pages[1].shape == (6, 16, 1, 16)
    a, b = cache.add(), cache.add()
    cache.extend([a, b], [20, 3])
    assert cache.page_table.tolist() == [[0, 1, -1], [2, -1, -1], [-1, -1, -1]]
    assert cache.lengths.tolist() == [20, 3, 0]
    table, lengths = cache.rows_of([b, a])
    assert table.tolist() == [[2, -1, -1], [0, 1, -1]] and lengths.tolist() == [3, 20]
    c = cache.fork(a)
    assert c == 2 and cache.page_table[2].tolist() == [0, 1, -1] and cache.lengths.tolist() == [20, 3, 20]
    cache.extend([b], [13])  # to the end of its page: the table stays
    assert cache.page_table[1].tolist() == [2, -1, -1] and cache.lengths.tolist() == [20, 16, 20]
    cache.extend([b], [1])
    assert cache.page_table[1].tolist() == [2, 3, -1]
    cache.free(c)
    cache.free(b)
    assert cache.lengths.tolist() == [20, 0, 0] and cache.page_table[1].tolist() == [-1, -1, -1]
    assert cache.compact() == 0
