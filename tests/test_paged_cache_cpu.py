"""The paged cache's host side: pages handed out, grown and taken back, the page
table's rows, and prompts copied into scattered pages."""
from __future__ import annotations

import pytest
import torch

import aicas_b200 as ab


def _cache(num_pages=6, page_size=8, layers=2, hkv=2, d=64):
    return ab.PagedKVCache(layers, num_pages, page_size, hkv, d, dtype=torch.bfloat16, device="cpu")


def test_requests_come_grow_and_go():
    c = _cache()
    a, b = c.add(9), c.add(0)
    assert a != b and len(c.pages(a)) == 2 and c.pages(b) == [] and c.free_pages == 4
    c.grow(a, 16)  # still fits its pages
    assert len(c.pages(a)) == 2
    first = c.pages(a)
    c.grow(a, 17)
    assert c.pages(a)[:2] == first and c.free_pages == 3
    c.grow(a, 1)  # never takes any away
    assert len(c.pages(a)) == 3
    c.grow(b, 24)
    assert c.free_pages == 0 and not set(c.pages(a)) & set(c.pages(b))
    c.release(a)
    assert c.free_pages == 3
    d = c.add(24)
    assert d not in (a, b) and not set(c.pages(d)) & set(c.pages(b))
    for call in (lambda: c.pages(a), lambda: c.release(a), lambda: c.grow(a, 1)):
        with pytest.raises(ValueError, match="holds no pages"):
            call()


def test_a_full_pool_refuses_and_takes_nothing():
    c = _cache()
    a = c.add(40)
    with pytest.raises(ValueError, match="full"):
        c.add(16)
    with pytest.raises(ValueError, match="full"):
        c.grow(a, 57)
    with pytest.raises(ValueError, match="negative"):
        c.add(-1)
    assert c.free_pages == 1 and len(c.pages(a)) == 5
    assert len(c.pages(c.add(8))) == 1


def test_page_table_rows():
    c = _cache()
    a, b = c.add(17), c.add(8)
    t = c.page_table([b, a])
    assert t.dtype is torch.int32 and t.tolist() == [c.pages(b) + [-1, -1], c.pages(a)]
    assert c.page_table([a], max_pages=4).tolist() == [c.pages(a) + [-1]]
    assert c.page_table([c.add(0)]).tolist() == [[-1]]  # at least one column
    assert c.page_table([]).shape == (0, 1)
    with pytest.raises(ValueError, match="max_pages"):
        c.page_table([a], max_pages=2)


@pytest.mark.parametrize("tokens", [1, 7, 8, 9, 24, 27])
def test_store_puts_tokens_where_the_table_says(tokens):
    c = _cache()
    c.release(c.add(8))
    hole = c.add(8)
    a = c.add(27)
    c.release(hole)
    k, v = (torch.randn(2, tokens, 64).to(torch.bfloat16) for _ in range(2))
    c.store(1, a, k, v)
    row = c.page_table([a])[0].tolist()
    for t in range(tokens):
        assert torch.equal(c.keys[1][row[t // 8], :, t % 8], k[:, t])
        assert torch.equal(c.values[1][row[t // 8], :, t % 8], v[:, t])
    assert not c.keys[0].any()  # the other layer's pool
    assert int((c.keys[1] != 0).any(-1).any(1).sum()) == tokens  # and no other row


def test_refusals():
    for args in ((0, 6, 8, 2, 64), (2, 0, 8, 2, 64), (2, 6, 12, 2, 64), (2, 6, 0, 2, 64), (2, 6, 8, 0, 64),
                 (2, 6, 8, 2, 65)):
        with pytest.raises(ValueError):
            ab.PagedKVCache(*args, dtype=torch.bfloat16, device="cpu")
    with pytest.raises(ValueError):
        ab.PagedKVCache(2, 6, 8, 2, 64, dtype=torch.float64, device="cpu")
    c = _cache()
    a = c.add(8)
    k = torch.zeros(2, 9, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="do not fit"):
        c.store(0, a, k, k)
    with pytest.raises(ValueError, match="must be"):
        c.store(0, a, k[:, :8].float(), k[:, :8].float())
    with pytest.raises(ValueError, match="must be"):
        c.store(0, a, k[:, :8], k[:1, :8])
