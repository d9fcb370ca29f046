"""Host bookkeeping of the paged cache, without a GPU."""
import random

import pytest
import torch

from lvar_b200.paged import PagedKVCache, PageTable


def test_pages_are_owned_once_and_come_back():
    t = PageTable(4, 100, page_size=16, num_pages=20, device="cpu")
    assert t.per_sequence == 7 and (t.table == -1).all()
    r = random.Random(0)
    have = [0] * 4
    for _ in range(200):
        s = r.randrange(4)
        if r.random() < 0.3:
            t.release(s)
            have[s] = 0
        else:
            n = r.randint(0, 100)
            before = [t.pages_of(i) for i in range(4)]
            try:
                t.reserve(s, n)
                have[s] = max(have[s], -(-n // 16))
            except RuntimeError as e:
                assert "out of pages" in str(e)
                assert before == [t.pages_of(i) for i in range(4)]
        owned = [t.pages_of(i) for i in range(4)]
        flat = sum(owned, [])
        assert [len(o) for o in owned] == have
        assert len(set(flat)) == len(flat) and len(flat) + t.free_pages == 20
        for i in range(4):
            assert t.table[i, :have[i]].tolist() == owned[i] and (t.table[i, have[i]:] == -1).all()


def test_table_keeps_its_address_and_earlier_pages():
    t = PageTable(2, 64, page_size=16, device="cpu")
    at = t.table.data_ptr()
    t.reserve(0, 17)
    first = t.pages_of(0)
    t.reserve_all({0: 40, 1: 64})
    assert t.pages_of(0)[:2] == first and t.table.data_ptr() == at and t.free_pages == 1
    t.reserve(0, 1)  # fewer than it has: nothing changes
    assert len(t.pages_of(0)) == 3


def test_refusals():
    with pytest.raises(ValueError):
        PageTable(1, 10, page_size=24, device="cpu")
    with pytest.raises(ValueError):
        PageTable(0, 10, device="cpu")
    t = PageTable(1, 32, page_size=16, device="cpu")
    with pytest.raises(RuntimeError, match="exceed"):
        t.reserve(0, 33)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 96, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 64, dtype=torch.float16, device="cpu")


def test_cache_shapes_and_bytes():
    a = PagedKVCache(3, 2, 64, 32, device="cpu")
    b = PagedKVCache(3, 2, 64, 32, dtype=torch.float8_e4m3fn, device="cpu")
    assert a.k.shape == (3, 2, 32, 64) and a.scales is None and a.nbytes == 2 * 3 * 2 * 32 * 64 * 2
    assert b.scales.shape == (3, 2, 32, 2) and b.nbytes == 3 * 2 * 32 * (2 * 64 + 2)


def test_sequences_are_named_once():
    """A negative number is no second name for a sequence, and a number that is none changes nothing."""
    t = PageTable(3, 64, page_size=16, num_pages=12, device="cpu")
    t.reserve(1, 20)
    before = (t.table.clone(), [t.pages_of(i) for i in range(3)], t.free_pages)
    for call in (lambda: t.reserve_all({2: 64, -1: 64}), lambda: t.reserve(-1, 16), lambda: t.reserve(3, 16),
                 lambda: t.reserve_all({0: 16, 3: 16}), lambda: t.release(-2), lambda: t.release(3), lambda: t.pages_of(-2)):
        with pytest.raises(IndexError):
            call()
        assert torch.equal(t.table, before[0]) and [t.pages_of(i) for i in range(3)] == before[1] and t.free_pages == before[2]
