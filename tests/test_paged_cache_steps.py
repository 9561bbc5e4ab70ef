"""Steps over all sequences of a paged cache of which some sit out."""

from __future__ import annotations

import pytest
import torch

from local_kimi_amd.paged import PagedCache


def test_step_lengths_count_those_that_grew():
    cache = PagedCache(12, 4, 48, layers=1, kv_heads=1, d_qk=8, d_v=8, page_rows=16, dtype=torch.float16,
                       device="cpu")
    at = cache.lengths.data_ptr(), cache.step_lengths.data_ptr()

    def seen():
        assert at == (cache.lengths.data_ptr(), cache.step_lengths.data_ptr())
        assert cache.lengths.is_contiguous() and cache.step_lengths.is_contiguous()
        return cache.lengths.tolist(), cache.step_lengths.tolist()

    assert seen() == ([0] * 4, [0] * 4)
    a, b = cache.add(), cache.add()
    cache.extend([a, b], [16, 3])
    assert seen() == ([16, 3, 0, 0], [16, 3, 0, 0])
    cache.extend([b], [1])
    assert seen() == ([16, 4, 0, 0], [0, 4, 0, 0])
    c = cache.fork(a)  # has its parent's tokens, and none of its own yet
    assert seen() == ([16, 4, 16, 0], [0, 4, 0, 0])
    cache.extend((c, b), (1, 0))
    assert seen() == ([16, 4, 17, 0], [0, 0, 17, 0])
    with pytest.raises(ValueError):
        cache.extend([a, b], [1, 60])  # changes nothing
    cache.compact()
    assert seen() == ([16, 4, 17, 0], [0, 0, 17, 0])
    cache.free(c)
    assert seen() == ([16, 4, 0, 0], [0] * 4)
    assert cache.add() == c
    cache.extend([], [])
    assert seen() == ([16, 4, 0, 0], [0] * 4)


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_a_sequence_that_sits_out_keeps_its_tokens(captured):
    """A fork's parent, its page shared, while the fork and another sequence take steps over the whole
    cache; then the parent's turn, and the fork sits out. Every token stays bit for bit, and each
    result is that of the sequence alone."""
    from local_kimi_amd.kernels import attention_paged, paged_append

    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    g = torch.Generator(device="cuda").manual_seed(4)
    hk, d, steps = 2, 64, 14
    cache = PagedCache(30, 5, 96, layers=1, kv_heads=hk, d_qk=d, d_v=d, page_rows=16)
    k, v = cache.k_pages[0], cache.v_pages[0]
    tokens = {}  # sequence -> its keys, [n, hk, d]; values are their double

    def filled(s, n):
        table, lengths = cache.rows_of([s])
        x = torch.randn((1, n, hk, d), generator=g, device="cuda").bfloat16()
        paged_append(x, 2 * x, k, v, table, lengths)
        tokens[s] = x[0]

    parent, other, idle = cache.add(), cache.add(), cache.add()
    for s, n in ((parent, 21), (other, 40), (idle, 5)):
        cache.extend([s], [n])
        filled(s, n)
    fork = cache.fork(parent)
    tokens[fork] = tokens[parent]
    x = torch.zeros((5, 1, hk, d), device="cuda").bfloat16()

    def step():
        paged_append(x, 2 * x, k, v, cache.page_table, cache.step_lengths)
        return attention_paged(x, k, v, cache.page_table, cache.step_lengths)

    if captured:
        cache.extend([], [])  # nobody grows: the first call writes nowhere
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
    for i in range(steps):
        grow = [fork, other] if i < 9 else [parent]
        cache.extend(grow, [1] * len(grow))
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        if captured:
            graph.replay()
        else:
            out = step()
        for s in grow:
            tokens[s] = torch.cat((tokens[s], x[s]))
        for s in (parent, other, idle, fork):
            table, lengths = cache.rows_of([s])
            n = int(lengths[0])
            pages = table[0, :-(-n // 16)].long()
            assert n == len(tokens[s])
            assert torch.equal(k[pages].flatten(0, 1)[:n], tokens[s]), (i, s)
            assert torch.equal(v[pages].flatten(0, 1)[:n], 2 * tokens[s]), (i, s)
            if s in grow:
                assert torch.equal(out[s], attention_paged(x[s:s + 1], k, v, table, lengths)[0]), (i, s)
            else:
                assert not out[s].any(), (i, s)
        assert not out[4].any()


@pytest.mark.gpu
def test_a_capture_refuses_what_uploads():
    """Before anything changes, in the book or on the device; the capture goes on."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    cache = PagedCache(30, 4, 96, layers=1, kv_heads=1, d_qk=8, d_v=8, page_rows=16)
    a = cache.add()
    cache.extend([a], [20])
    b = cache.fork(a)
    before = [list(x) for x in (cache.book.lengths, cache.book.users, cache.book.pages[a], cache.book.pages[b])]
    graph, x = torch.cuda.CUDAGraph(), torch.ones(8, device="cuda")
    with torch.cuda.graph(graph):
        y = x + 1
        for call in (lambda: cache.extend([a], [1]), lambda: cache.fork(a), lambda: cache.free(b), cache.compact,
                     lambda: cache.rows_of([a])):
            with pytest.raises(RuntimeError, match="outside the captured graph"):
                call()
        z = cache.step_lengths + 1
    assert before == [list(x) for x in (cache.book.lengths, cache.book.users, cache.book.pages[a], cache.book.pages[b])]
    cache.extend([b], [2])
    for _ in range(3):
        x += 1
        graph.replay()
        assert torch.equal(y, x + 1) and z.tolist() == [1, 23, 1, 1]
