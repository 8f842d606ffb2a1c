"""Eviction on the GPU: the selection and the move against the oracle, and the operators together as a server of long
contexts uses them."""
import numpy as np
import pytest
import torch

import gpu_data as G
from fp4_data import BF16, F16, F32, FP4, FP8, bf16_round
from oracle import mxfp4 as M

pytestmark = pytest.mark.gpu

FILLS = {
    "spread": lambda r, n: r.random(n).astype(np.float32) ** 8,
    "ties": lambda r, n: r.integers(0, 4, n).astype(np.float32),
    "zeros": lambda r, n: np.where(r.random(n) < 0.97, 0.0, r.random(n)).astype(np.float32),
    "odd": lambda r, n: r.choice(np.array([0.0, -0.0, -1.0, 1e-45, -1e-45, 3e38, np.inf, -np.inf, np.nan, 1.0], np.float32), n),
    "equal": lambda r, n: np.full(n, 0.25, np.float32),
}


class Pool:
    """Tables of scattered pages and a weight plane."""

    def __init__(self, lengths, page, hkv, fill, seed, spare=0):
        rng = np.random.default_rng(seed)
        self.lengths, self.page, self.hkv = np.asarray(lengths), page, hkv
        need = -(-self.lengths // page)
        self.stride = int(max(need.max(), 1)) + 2
        self.pages = int(need.sum()) + spare + 3
        perm = rng.permutation(self.pages).astype(np.uint32)
        self.table = np.full((len(lengths) + 2, self.stride), M.NONE, np.uint32)
        at = 0
        self.rows = rng.permutation(len(lengths) + 2)[:len(lengths)]
        for r, n in zip(self.rows, need):
            self.table[r, :n] = perm[at:at + n]
            at += n
        self.spare = perm[at:at + spare]
        self.mass = FILLS[fill](rng, self.pages * hkv * page).reshape(self.pages, hkv, page)

    def of(self, i, h):
        n, row = int(self.lengths[i]), self.table[self.rows[i]]
        key = np.arange(n)
        page = row[key // self.page].astype(np.int64)
        ok = page < self.pages
        return np.where(ok, self.mass[np.where(ok, page, 0), h, key % self.page], np.float32(0))

    def select(self, lia, budget, recent):
        n = len(self.lengths)
        kept = torch.full((n, self.hkv, budget), 77, dtype=torch.int32, device="cuda")
        counts = torch.full((n + 1,), 77, dtype=torch.int32, device="cuda")
        layout = lia.KVLayout(self.hkv, 128, self.page, self.pages, BF16)
        lia.kv_select(layout, G.u32_dev(self.rows), G.u32_dev(self.lengths), G.u32_dev(self.table.reshape(-1)), self.stride,
                      budget, recent, torch.from_numpy(self.mass).cuda(), kept, counts)
        assert int(counts[n]) == 77
        return kept.cpu().numpy().view(np.uint32), counts[:n].cpu().numpy()

    def check(self, lia, budget, recent):
        kept, counts = self.select(lia, budget, recent)
        assert np.array_equal(counts, np.minimum(self.lengths, budget))
        for i in range(len(self.lengths)):
            for h in range(self.hkv):
                want = M.select(self.of(i, h), budget, recent)
                assert np.array_equal(kept[i, h, :len(want)], want), (i, h, budget, recent)
                assert (kept[i, h, len(want):] == M.NONE).all()
        return kept, counts


@pytest.mark.parametrize("fill", list(FILLS))
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (100, 0), (100, 33), (100, 100), (100, 500), (2000, 7)])
def test_select(lia, fill, budget, recent):
    lengths = [1, 99, 100, 101, 102, 1023, 1024, 1025, 2001, 5000, 9000, 0]
    print(f"[case] select {fill} budget={budget} recent={recent}", flush=True)
    Pool(lengths, 16, 2, fill, seed=1).check(lia, budget, recent)


@pytest.mark.parametrize("n,page,hkv,budget,recent,fill", [
    (8192 - 16, 16, 3, 1, 0, "ties"), (40000, 64, 1, 777, 0, "spread"), (131072, 32, 2, 8192, 1000, "zeros"),
    (33000, 16, 1, 32999, 5, "odd"), (70000, 128, 1, 5000, 4999, "ties"),
])
def test_select_of_long_sequences(lia, n, page, hkv, budget, recent, fill):
    """Keys in registers, and the ones past them read again."""
    print(f"[case] select long n={n} {fill}", flush=True)
    Pool([n, n - 12345 if n > 20000 else 5], page, hkv, fill, seed=2).check(lia, budget, recent)


def test_select_with_pages_outside_the_pool(lia):
    pool = Pool([500, 300], 16, 2, "spread", seed=3)
    pool.table[pool.rows[0], 4], pool.table[pool.rows[1], 0] = pool.pages, M.NONE
    print("[case] select, pages outside", flush=True)
    pool.check(lia, 100, 20)


def _planes(rng, pool, d, kv):
    """K or V in the pool's layout as [page][token][head] rows of bytes, and the scales' rows."""
    shape = (pool.pages, pool.hkv, pool.page)
    if kv == FP4:
        return [rng.integers(0, 256, (*shape, w), dtype=np.uint8) for w in (d // 2, d // 32)]
    return [rng.integers(0, 1 << 16, (pool.pages, pool.page, pool.hkv, d), dtype=np.uint16).astype(np.uint16), None]


@pytest.mark.parametrize("kv,d", [(FP4, 128), (FP4, 64), (BF16, 128), (F16, 64)])
@pytest.mark.parametrize("where", ["in place", "other pages", "some pages"])
@pytest.mark.parametrize("lengths,budget,recent", [([300, 40, 2000, 1], 64, 20), ([9000, 3000], 2500, 300)])
def test_compact(lia, kv, d, where, lengths, budget, recent):
    page, hkv = 16, 2
    need = -(-budget // page) * len(lengths)
    pool = Pool(lengths, page, hkv, "spread", seed=4, spare=need)
    rng = np.random.default_rng(5)
    kept, counts = pool.check(lia, budget, recent)
    to = pool.table.copy()
    if where != "in place":  # destinations of their own: all of them, or every second one
        at = 0
        for r, c in zip(pool.rows, counts):
            for i in range(0, -(-int(c) // page), 1 if where == "other pages" else 2):
                to[r, i] = pool.spare[at]
                at += 1
    (k, ks), (v, vs) = _planes(rng, pool, d, kv), _planes(rng, pool, d, kv)
    mass = pool.mass.copy()
    dev = [None if x is None else G.to_dev(x.view(np.int16) if x.dtype == np.uint16 else x) for x in (k, v, ks, vs, mass)]
    print(f"[case] compact kv={kv} d={d} {where} {lengths}", flush=True)
    layout = lia.KVLayout(hkv, d, page, pool.pages, kv)
    lia.kv_compact(layout, G.u32_dev(pool.rows), G.u32_dev(pool.table.reshape(-1)), G.u32_dev(to.reshape(-1)), pool.stride,
                   G.to_dev(kept.view(np.int32)), G.u32_dev(counts), dev[0], dev[1], mass=dev[4], k_scales=dev[2], v_scales=dev[3])
    for x, got in zip((k, v, ks, vs, mass), dev):
        if x is None:
            continue
        headmajor = x.ndim == 3 or kv == FP4
        want = x.copy()
        rows = want if headmajor else want.transpose(0, 2, 1, 3)
        old = (x if headmajor else x.transpose(0, 2, 1, 3)).copy()
        for i, r in enumerate(pool.rows):
            c = int(counts[i])
            dst = np.arange(c)
            for h in range(hkv):
                src = kept[i, h, :c]
                rows[to[r, dst // page].astype(int), h, dst % page] = old[pool.table[r, src // page].astype(int), h, src % page]
        assert np.array_equal(got.cpu().numpy().view(want.dtype), want), x.shape


def test_compact_without_weights_and_with_bad_entries(lia):
    """mass NULL; kept keys and destinations outside the table or the pool move nothing."""
    pool = Pool([200, 100], 16, 2, "spread", seed=6)
    rng = np.random.default_rng(7)
    kept, counts = pool.check(lia, 50, 10)
    kept = kept.copy()
    kept[0, 0, 49] = pool.stride * 16 + 5
    kept[1, 1, 3] = M.NONE
    to = pool.table.copy()
    to[pool.rows[1], 1] = pool.pages + 7
    (k, ks), (v, vs) = _planes(rng, pool, 128, FP4), _planes(rng, pool, 128, FP4)
    dev = [G.to_dev(x) for x in (k, v, ks, vs)]
    print("[case] compact with bad entries", flush=True)
    lia.kv_compact(lia.KVLayout(2, 128, 16, pool.pages, FP4), G.u32_dev(pool.rows), G.u32_dev(pool.table.reshape(-1)),
                   G.u32_dev(to.reshape(-1)), pool.stride, G.to_dev(kept.view(np.int32)), G.u32_dev(counts), dev[0], dev[1],
                   k_scales=dev[2], v_scales=dev[3])
    for x, got in zip((k, v, ks, vs), dev):
        want, old = x.copy(), x
        for i, r in enumerate(pool.rows):
            for h in range(2):
                for j in range(int(counts[i])):
                    s = int(kept[i, h, j])
                    if s >= pool.stride * 16 or to[r, j // 16] >= pool.pages:
                        continue
                    want[to[r, j // 16], h, j % 16] = old[pool.table[r, s // 16], h, s % 16]
        assert np.array_equal(got.cpu().numpy(), want)


def test_captured_eviction(lia):
    """Select and compact captured once; replays on new weights (other pages as destination) against eager calls."""
    pool = Pool([700, 90, 4000], 16, 2, "spread", seed=8, spare=3 * 16)
    rng = np.random.default_rng(9)
    to = pool.table.copy()
    for i, r in enumerate(pool.rows):
        to[r, :16] = pool.spare[16 * i:16 * i + 16]
    (k, ks), (v, vs) = _planes(rng, pool, 128, FP4), _planes(rng, pool, 128, FP4)
    layout = lia.KVLayout(2, 128, 16, pool.pages, FP4)
    rows, lengths, table, dest = (G.u32_dev(x) for x in (pool.rows, pool.lengths, pool.table.reshape(-1), to.reshape(-1)))
    mass = torch.from_numpy(pool.mass).cuda()
    sets = []
    for _ in range(2):
        sets.append(dict(p=[G.to_dev(x) for x in (k, v, ks, vs)], kept=torch.zeros((3, 2, 250), dtype=torch.int32, device="cuda"),
                         counts=torch.zeros(3, dtype=torch.int32, device="cuda")))
    print("[case] captured eviction", flush=True)

    def step(s):
        lia.kv_select(layout, rows, lengths, table, pool.stride, 250, 60, mass, s["kept"], s["counts"])
        lia.kv_compact(layout, rows, table, dest, pool.stride, s["kept"], s["counts"], s["p"][0], s["p"][1],
                       k_scales=s["p"][2], v_scales=s["p"][3])
    step(sets[0])
    step(sets[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(sets[0])
    for i in range(3):
        mass.uniform_(generator=torch.Generator(device="cuda").manual_seed(i))
        graph.replay()
        torch.cuda.synchronize()
        step(sets[1])
        torch.cuda.synchronize()
        for a, b in zip([*sets[0]["p"], sets[0]["kept"], sets[0]["counts"]], [*sets[1]["p"], sets[1]["kept"], sets[1]["counts"]]):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("kv", [FP4, BF16, F16])
def test_serving_with_eviction(lia, kv):
    """Append, attention, weights, selection and move together through the engine: two chats, prompts, decode steps,
    an eviction in the middle, decode steps after it, against a 64-bit replay of what the pool holds."""
    rng = np.random.default_rng(10)
    hq, hkv, d, page, layers, budget, recent = 8, 2, 64, 16, 2, 96, 24
    e = lia.Engine(hq, hkv, d, pool_tokens=page * 64, layers=layers, page_size=page, kv_dtype=kv, prefill_batch=512,
                   q_dtype=BF16, track_weights=True)
    e.configure_paging(4, 512)
    for w in e.weights:
        w.fill_(7.0)  # what former owners of the pages left
    perm = rng.permutation(64)
    tables = [[int(x) for x in perm[:20]], [int(x) for x in perm[20:40]]]
    lengths = [0, 0]
    mass = [[np.zeros((hkv, 0)) for _ in range(2)] for _ in range(layers)]  # the replay's, by layer and sequence

    def values(plane, scales):
        if kv == FP4:
            return M.dequantise(plane.cpu().numpy(), scales.cpu().numpy())
        t = plane.view(torch.int16).view(torch.bfloat16 if kv == BF16 else torch.float16)
        return t.double().cpu().numpy().reshape(64, page, hkv, d).transpose(0, 2, 1, 3)

    def step(rows):
        nonlocal lengths
        e.stage([(1, lengths[s] + i, s) for s in range(2) for i in range(rows[s])], tables)
        total = sum(rows)
        for layer in range(layers):
            q = torch.from_numpy(rng.standard_normal((total, hq, d)).astype(np.float32)).to(torch.bfloat16).cuda()
            k, v = (torch.from_numpy(rng.standard_normal((total, hkv * d)).astype(np.float32)).cuda() for _ in range(2))
            out = e.attention(layer, q, k, v).cpu().numpy()
            kk, vv = values(e.k[layer], e.k_scales[layer]), values(e.v[layer], e.v_scales[layer])
            at = 0
            for s in range(2):
                m, n = rows[s], lengths[s] + rows[s]
                if m == 0:
                    continue
                ks, vs = M.keys_of(kk, tables[s], n, page), M.keys_of(vv, tables[s], n, page)
                qs = q[at:at + m].float().cpu().numpy()
                ref = M.attention(qs, ks, vs, lengths[s], e.scale)
                bound = M.attention(qs, ks, np.abs(vs), lengths[s], e.scale) * 2.5 * 2.0 ** -8  # (fp4_data.py's)
                assert (np.abs(out[at:at + m] - ref) <= bound + 1e-30).all()
                w = M.softmax_weights(qs, ks, lengths[s], e.scale).sum((1, 2))
                old = np.pad(mass[layer][s], ((0, 0), (0, m)))
                mass[layer][s] = old + w
                got = np.concatenate([e.weights[layer].cpu().numpy()[p] for p in tables[s][:-(-n // page)]], 1)[:, :n]
                assert np.allclose(got, mass[layer][s], rtol=1e-3, atol=0)  # (test_gpu_weights.py bounds a step's)
                mass[layer][s] = got.astype(np.float64)
                at += m
        lengths = [n + m for n, m in zip(lengths, rows)]

    print(f"[case] serving with eviction kv={kv}", flush=True)
    step([200, 60])
    step([1, 1])
    step([3, 1])
    before = [(values(e.k[i], e.k_scales[i]), values(e.v[i], e.v_scales[i])) for i in range(layers)]
    counts, freed = e.evict(tables, lengths, budget, recent)
    assert counts == [96, 62] and freed == [tables[0][6:], tables[1][4:]]
    for layer in range(layers):
        for s in range(2):
            w = mass[layer][s].astype(np.float32)
            keep = [M.select(w[h], budget, recent) for h in range(hkv)]
            for old, plane, scales in zip(before[layer], (e.k, e.v), (e.k_scales, e.v_scales)):
                was = M.keys_of(old, tables[s], lengths[s], page)
                now = M.keys_of(values(plane[layer], scales[layer]), tables[s], counts[s], page)
                for h in range(hkv):
                    assert np.array_equal(now[h], was[h][keep[h]])
            mass[layer][s] = np.stack([mass[layer][s][h][keep[h]] for h in range(hkv)])
    lengths, tables = counts, [t[:len(t) - len(f)] + f[:2] for t, f in zip(tables, freed)]
    step([1, 1])
    step([2, 20])
    step([1, 0])


def test_engine_refuses(lia):
    e = lia.Engine(8, 2, 64, pool_tokens=256, page_size=16, kv_dtype=FP4, track_weights=True)
    with pytest.raises(lia.LiaError):
        e.evict([[0]], [1], 1, 0)
    e.configure_paging(4, 128)
    for args in (([[0, 1]], [33], 8, 0), ([[0, 1], [1, 2]], [20, 20], 8, 0), ([[0, 99]], [20], 8, 0), ([[0]], [5, 6], 8, 0),
                 ([[0]], [5], 0, 0), ([[0, 0]], [32], 8, 0)):
        with pytest.raises(lia.LiaError):
            e.evict(*args)
    with pytest.raises(lia.LiaError):  # a page of two sequences, with weights tracked
        e.stage([(1, 0, 0), (1, 17, 1)], [[3], [3, 4]])
    plain = lia.Engine(8, 2, 64, pool_tokens=256, page_size=16, kv_dtype=FP4)
    plain.configure_paging(4, 128)
    with pytest.raises(lia.LiaError):
        plain.evict([[0]], [1], 1, 0)
