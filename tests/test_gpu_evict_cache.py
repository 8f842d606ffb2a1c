"""Eviction of a page cache's sequences: the pages that prefix keys name keep their rows."""
import numpy as np
import pytest
import torch

from fp4_data import BF16, FP4
from oracle import mxfp4 as M

pytestmark = pytest.mark.gpu
PAGE, LAYERS = 16, 2


def _engine(lia, kv, pool_pages):
    e = lia.Engine(8, 2, 64, pool_tokens=PAGE * pool_pages, layers=LAYERS, page_size=PAGE, kv_dtype=kv, prefill_batch=512,
                   q_dtype=BF16, track_weights=True)
    e.configure_paging(4, 512)
    return e


def _transfer(lia, e):
    scaled = e.kv_dtype == FP4
    return lia.KVTransfer(lia.KVLayout(e.hkv, e.d, PAGE, e.pool_pages, e.kv_dtype), e.k, e.v,
                          e.k_scales if scaled else None, e.v_scales if scaled else None)


def _rows(e, sequence, first, n, seed):
    """Appends and attends rows first .. first + n - 1 of one sequence in every layer."""
    rng = np.random.default_rng(seed)
    e.stage([(1, first + i, 0) for i in range(n)], [sequence.pages])
    for layer in range(LAYERS):
        q = torch.from_numpy(rng.standard_normal((n, 8, 64)).astype(np.float32)).to(torch.bfloat16).cuda()
        k, v = (torch.from_numpy(rng.standard_normal((n, 128)).astype(np.float32)).cuda() for _ in range(2))
        e.attention(layer, q, k, v)


def _start(cache, e, tokens, seed):
    seq, cached = cache.attach(tokens)
    for pos in range(cached, len(tokens)):
        assert cache.ensure_position(seq, pos)
    _rows(e, seq, cached, len(tokens) - cached, seed)
    return seq, cached


@pytest.mark.parametrize("kv", [BF16, FP4])
@pytest.mark.parametrize("transfer", [True, False])
def test_page_lists_of_a_cache_are_refused(lia, kv, transfer):
    e = _engine(lia, kv, 32)
    t = _transfer(lia, e)
    cache = lia.PageCache(bytes(32), 32, PAGE, store={} if transfer else None, transfer=t if transfer else None)
    tokens = list(range(200))
    seq, _ = _start(cache, e, tokens, 1)
    cache.seal(seq, tokens, 200)
    before = t.read_kv_pages(seq.pages[:12])
    print(f"[case] a cache's page lists kv={kv}", flush=True)
    for tables in [[seq.pages], [list(seq.pages)]][:1 + transfer]:
        with pytest.raises(lia.LiaError) as err:
            e.evict(tables, [200], 64, 16)
        assert err.value.status == -16
    assert t.read_kv_pages(seq.pages[:12]) == before


@pytest.mark.parametrize("kv", [BF16, FP4])
@pytest.mark.parametrize("pool_pages", [64, 26])  # idle pages for the moved keys, or none
def test_the_prefix_is_found_after_an_eviction(lia, kv, pool_pages):
    e = _engine(lia, kv, pool_pages)
    t, store = _transfer(lia, e), {}
    cache = lia.PageCache(bytes(32), pool_pages, PAGE, store=store, transfer=t)
    tokens, other = list(range(200)), list(range(96)) + list(range(900, 1010))
    a, _ = _start(cache, e, tokens, 1)
    cache.seal(a, tokens, 200)
    b, cached = _start(cache, e, other, 2)
    cache.seal(b, other, 206)
    assert cached == 96 and b.pages[:6] == a.pages[:6]
    prefix = t.read_kv_pages(a.pages[:12])
    was = [(x[i].clone(), w) for x in (e.k, e.v) for i, w in enumerate(e.weights)]
    old, mass = a.pages, [w.clone() for w in e.weights]
    rest = t.read_kv_pages(b.pages[:13])
    print(f"[case] eviction beside a cache kv={kv} pool={pool_pages}", flush=True)
    counts, freed = e.evict([a, b], [200, 206], 204, 30, cache=cache)  # b alone loses keys
    assert counts == [200, 204] and freed == [[], []] and a.pages == old
    assert t.read_kv_pages(a.pages[:12]) == prefix
    counts, freed = e.evict([a], [200], 70, 30, cache=cache)
    assert counts == [70] and freed == [[]] and len(a.pages) == 5
    # the kept keys, by the weights of the sequence's rows
    for layer in range(LAYERS):
        flat = mass[layer].cpu().numpy()
        w = np.concatenate([flat[p] for p in old], 1)[:, :200]
        got = e.weights[layer].cpu().numpy()
        got = np.concatenate([got[p] for p in a.pages], 1)[:, :70]
        for h in range(2):
            assert np.array_equal(got[h], w[h][M.select(w[h], 70, 30)])
        if kv == BF16:
            for i, plane in ((layer, e.k), (LAYERS + layer, e.v)):
                src = was[i][0].view(torch.int16).reshape(-1, PAGE, 2, 64).cpu().numpy()
                dst = plane[layer].view(torch.int16).reshape(-1, PAGE, 2, 64).cpu().numpy()
                src = np.concatenate([src[p] for p in old])[:200]
                dst = np.concatenate([dst[p] for p in a.pages])[:70]
                for h in range(2):
                    assert np.array_equal(dst[:, h], src[M.select(w[h], 70, 30), h])
    cache.seal(a, tokens, 70)  # says nothing of the moved keys
    for pos in range(70, 90):
        assert cache.ensure_position(a, pos)
    _rows(e, a, 70, 20, 3)
    cache.release(a)
    c, cached = cache.attach(tokens)
    assert cached == 192 and t.read_kv_pages(c.pages) == prefix
    cache.release(b)
    d, cached = cache.attach(other)
    assert cached == 192 and t.read_kv_pages(d.pages) == rest[:12]


def test_pages_a_cache_restores_begin_without_weights(lia):
    """A page of another sequence's is taken for a restored prefix: what its former keys received is not the prefix's."""
    e = _engine(lia, BF16, 8)
    store = {}
    cache = lia.PageCache(bytes(32), 8, PAGE, store=store, transfer=e.kv_transfer())
    tokens = list(range(50))
    a, _ = _start(cache, e, tokens, 4)
    cache.seal(a, tokens, 50)
    cache.release(a)
    b, _ = _start(cache, e, list(range(500, 620)), 5)  # takes every page: the prefix goes to the store
    assert len(b.pages) == 8 and len(store) == 3
    cache.release(b)
    assert all((w > 0).any() for w in e.weights)
    print("[case] restored by a cache", flush=True)
    c, cached = cache.attach(tokens)
    assert cached == 48
    for w in e.weights:
        assert (w[c.pages[:3]] == 0).all() and (w[[p for p in range(8) if p not in c.pages]] > 0).any()


def test_written_pages_are_ready_for_every_stream(lia):
    """A page transfer ends with its stream synchronised; so do the weights it clears, which the next step may read on
    another stream."""
    e = lia.Engine(8, 2, 64, pool_tokens=PAGE * 16, layers=64, page_size=PAGE, kv_dtype=BF16, q_dtype=BF16,
                   track_weights=True)
    e.configure_paging(2, 64)
    payload = bytes(e.kv_transfer().page_bytes)
    print("[case] writes and streams", flush=True)
    e.write_kv_page(0, payload)
    for i in range(5):
        for w in e.weights:
            w.fill_(3.0)
        e.write_kv_pages([(p, payload) for p in range(1, 9)])
        assert torch.cuda.current_stream().query()
        for w in e.weights:
            assert (w[1:9] == 0).all() and (w[9:] == 3).all()
