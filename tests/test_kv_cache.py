"""CPU tests of the paged cache's book-keeping (naylis_b200/attention.PagedKVCache)."""
import pytest
import torch

from naylis_b200.attention import PagedKVCache


def test_extend_tables_and_free():
    c = PagedKVCache(2, 6, 8, 3, 64, device="cpu")
    assert c.k.shape == (2, 6, 3, 8, 64) and c.free_pages == 6
    a, b = c.add(), c.add()
    pos, slots = c.extend([a, b], [10, 3])
    assert pos.tolist() == list(range(10)) + [0, 1, 2] and c.free_pages == 3
    table, lens, longest = c.tables([b, a])
    assert lens.tolist() == [3, 10] and longest == 10 and table.shape == (2, 2) and table.dtype == torch.int32
    owned = table[1].tolist()
    assert slots[:10].tolist() == [owned[t // 8] * 8 + t % 8 for t in range(10)]
    assert slots[10:].tolist() == [int(table[0, 0]) * 8 + t for t in range(3)]
    pos, slots = c.extend([b, a], [1, 0])
    assert pos.tolist() == [3] and slots.tolist() == [int(table[0, 0]) * 8 + 3]
    c.free(a)
    assert c.free_pages == 5 and c.length(b) == 4
    d = c.add()
    pos, slots = c.extend([d], [40])
    assert c.free_pages == 0 and len(set(slots.tolist())) == 40
    assert not set((slots // 8).tolist()) & {int(table[0, 0])}


def test_running_out_changes_nothing():
    c = PagedKVCache(1, 2, 16, 1, 128, device="cpu")
    a, b = c.add(), c.add()
    c.extend([a], [16])
    with pytest.raises(RuntimeError, match="pages needed"):
        c.extend([a, b], [1, 1])
    assert c.length(a) == 16 and c.length(b) == 0 and c.free_pages == 1
    assert [t.numel() for t in c.extend([], [])] == [0, 0]
    assert c.tables([])[2] == 0
    for args in (([a, a], [1, 1]), ([a], [1, 2]), ([a], [-1])):
        with pytest.raises(RuntimeError):
            c.extend(*args)
    for bad in ((0, 1, 16, 1, 64), (1, -1, 16, 1, 64), (1, 1, 12, 1, 64), (1, 1, 16, 1, 80)):
        with pytest.raises(RuntimeError):
            PagedKVCache(*bad, device="cpu")
