"""CPU tests of lia_page_cache_detach: a sequence whose keys are cut leaves its prefix pages as they are, and gets pages that
no key names and nobody else uses."""
import ctypes as C

import numpy as np
import pytest

NS = b"\x11" * 32
P = 4


class World:
    """A cache over a dict of payloads; a page of a sealed prefix holds its tokens."""

    def __init__(self, lia, pages, store=True):
        self.lia, self.store, self.pool = lia, {} if store else None, {p: b"\xee" * 16 for p in range(pages)}
        self.cache = lia.PageCache(NS, pages, P, store=self.store, pool=self.pool, page_bytes=16)

    def start(self, tokens, seal=True):
        seq, cached = self.cache.attach(tokens)
        for pos in range(cached, len(tokens)):
            assert self.cache.ensure_position(seq, pos)
            block = tokens[pos // P * P:pos // P * P + P]
            self.pool[seq.pages[pos // P]] = np.array(block + [0] * (P - len(block)), np.uint32).tobytes()
        if seal:
            self.cache.seal(seq, tokens, len(tokens))
        return seq, cached

    def holds(self, seq, tokens):
        return [self.pool[p] for p in seq.pages[:len(tokens) // P]] == [
            np.array(tokens[i:i + P], np.uint32).tobytes() for i in range(0, len(tokens) // P * P, P)]


def test_the_prefix_stays_for_others(lia):
    w = World(lia, 20)
    tokens = list(range(100, 122))  # five full pages and two tokens
    a, _ = w.start(tokens)
    b, cached = w.start(tokens[:13])
    assert cached == 12 and b.pages[:3] == a.pages[:3]
    before, free = a.pages, w.cache.available_pages()
    assert w.cache.detach([a], [10])
    assert len(a.pages) == 3 and not set(a.pages) & set(before) and w.holds(b, tokens[:12])
    for p in a.pages:  # the moved keys
        w.pool[p] = b"\xaa" * 16
    # three pages went to the sequence; its last three, which b does not share, came back
    assert w.cache.available_pages() == free
    w.cache.seal(a, tokens, 10)  # its rows are no longer these tokens
    w.cache.seal(a, tokens, 22)
    w.cache.release(a)
    w.cache.release(b)
    c, cached = w.cache.attach(tokens)
    assert cached == 20 and c.pages == before[:5] and w.holds(c, tokens[:20])


def test_pages_without_a_key_stay(lia):
    w = World(lia, 10)
    tokens = list(range(30))
    a, _ = w.start(tokens, seal=False)
    before = a.pages
    assert w.cache.detach([a], [9]) and a.pages == before[:3]
    w.cache.seal(a, tokens, 12)
    w.cache.release(a)
    assert w.cache.attach(tokens)[1] == 0 and w.cache.available_pages() == 10


@pytest.mark.parametrize("store", [True, False])
def test_a_full_pool(lia, store):
    """No idle page: the sequence's own pages lose their keys, to the store where there is one."""
    w = World(lia, 6, store)
    tokens = list(range(50, 73))
    a, _ = w.start(tokens)
    before = a.pages
    assert w.cache.available_pages() == 0
    assert w.cache.detach([a], [8]) and a.pages == before[:2]
    for p in a.pages:
        w.pool[p] = b"\xaa" * 16
    assert w.cache.available_pages() == 4
    b, cached = w.cache.attach(tokens)
    # of the four, three hold the prefix's later blocks: one block can be restored before the pool is full
    assert cached == (4 if store else 0) and w.holds(b, tokens[:cached]) and not set(b.pages) & set(a.pages)
    w.cache.release(a)
    w.cache.release(b)
    b, cached = w.cache.attach(tokens)
    assert cached == (20 if store else 0) and w.holds(b, tokens[:cached])


def test_an_occupied_pool_changes_nothing(lia):
    w = World(lia, 6)
    tokens = list(range(23))
    a, _ = w.start(tokens)
    b, cached = w.cache.attach(tokens[:9])
    assert cached == 8 and w.cache.available_pages() == 0
    before = a.pages
    assert not w.cache.detach([a], [12])  # its first two pages are b's too
    assert a.pages == before and b.pages == before[:2]
    w.cache.release(b)
    assert w.cache.detach([a], [12])


def test_sequences_of_one_call_get_pages_of_their_own(lia):
    """No page of the call's sequences before it is one of theirs after it at another place."""
    w = World(lia, 40)
    one, two = list(range(40)), list(range(20)) + list(range(90, 110))
    a, _ = w.start(one)
    b, _ = w.start(two)
    before = a.pages, b.pages
    assert before[0][:5] == before[1][:5]
    assert w.cache.detach([a, b], [17, 12])
    assert len(a.pages) == 5 and len(b.pages) == 3 and not set(a.pages) & set(b.pages)
    assert not (set(a.pages) | set(b.pages)) & (set(before[0]) | set(before[1]))
    c, cached = w.cache.attach(one)
    assert cached == 36 and w.holds(c, one[:36])
    c, cached = w.cache.attach(two)
    assert cached == 36 and w.holds(c, two[:36])


def test_refusals(lia):
    w = World(lia, 10)
    a, _ = w.start(list(range(9)))
    before = a.pages
    for sequences, keys, status in (([a, a], [4, 4], -20), ([a], [13], -15)):
        with pytest.raises(lia.LiaError) as e:
            w.cache.detach(sequences, keys)
        assert e.value.status == status and a.pages == before
    with pytest.raises(lia.LiaError):
        w.cache.detach([a], [])
    assert w.cache.detach([], [])
    L = lia.lib()
    assert L.lia_page_cache_detach(None, 0, None, None) == -20
    assert L.lia_page_cache_detach(w.cache.handle, 1, None, None) == -20
    assert L.lia_page_cache_detach(w.cache.handle, 1, (C.c_void_p * 1)(None), (C.c_size_t * 1)(0)) == -20


def test_a_failing_store_gives_the_taken_pages_back(lia):
    class Broken(dict):
        def __setitem__(self, key, value):
            raise OSError

    w = World(lia, 8)
    tokens = list(range(23))
    a, _ = w.start(tokens)               # six pages, five of them keyed
    x, _ = w.start([7, 7, 7, 7, 7])
    w.cache.release(x)                   # two idle ones, one of them keyed
    w.cache.store = Broken()
    before = a.pages
    with pytest.raises(lia.LiaError) as e:
        w.cache.detach([a], [20])
    assert e.value.status == -24 and a.pages == before and w.cache.available_pages() == 2
    w.cache.store = w.store
    assert w.cache.detach([a], [20]) and len(a.pages) == 5
