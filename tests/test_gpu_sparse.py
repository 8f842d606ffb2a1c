"""Page summaries and page selection equal to the oracle; attention over selected pages against 64 bits, bounds counted in half
steps of the weights' and the output's types."""
import numpy as np
import pytest
import torch

import gpu_data as G
import sparse_data as D
from sparse_data import BF16, F16, F32, FP4, FP8, NONE

pytestmark = pytest.mark.gpu


def _summaries(lia, pool, slots, stream=None):
    codes = torch.full((pool.pages, pool.hkv, 2, pool.d), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((pool.pages, pool.hkv), -3.0, device="cuda")
    lia.page_summaries(pool.layout(lia), G.u32_dev(slots), pool.kc, codes, scales, k_scales=pool.ks, stream=stream)
    return codes.cpu().numpy(), scales.cpu().numpy()


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("page,hkv,d", [(16, 2, 128), (16, 3, 64), (32, 8, 128), (64, 1, 64), (128, 2, 128)])
def test_summaries(lia, kv, page, hkv, d):
    print(f"[case] summaries kv={kv} page={page} hkv={hkv} d={d}", flush=True)
    rng = np.random.default_rng(page + hkv)
    pool = D.Pool(rng, 9, page, hkv, d, kv, key_size=10.0 ** rng.integers(-3, 3))
    pages = [7, 0, 3, 8]
    slots = [page * 2 + page - 2, *(p * page + page - 1 for p in pages), 9 * page + page - 1, NONE, page * 5]
    codes, scales = _summaries(lia, pool, slots)
    c, s = pool.summaries()
    assert np.array_equal(codes[pages], c[pages]) and np.array_equal(scales[pages], s[pages])
    rest = [p for p in range(9) if p not in pages]  # pages that no slot ends
    assert (codes[rest] == 99).all() and (scales[rest] == -3.0).all()


def test_summaries_of_edges(lia):
    """Zeros, the smallest and the largest values, infinities and NaNs; one head's do not reach the other's."""
    pool = D.Pool(np.random.default_rng(1), 6, 16, 2, 64, BF16)
    kc = pool.kc
    kc[0, :, 0] = 0.0
    kc[1, :, 0] = -1e-40
    kc[2, 3, 1, 5] = float("inf")
    kc[3, 15, 0, 63] = float("nan")
    kc[4, 7, 1, 0] = 3.3e38
    kc[5] = kc[5].abs()  # every lower bound above 0
    pool.k = kc.double().cpu().numpy()
    codes, scales = _summaries(lia, pool, np.arange(6) * 16 + 15)
    c, s = pool.summaries()
    assert np.array_equal(codes, c) and np.array_equal(scales, s)
    assert np.isinf(scales).tolist() == [[False, False], [False, False], [False, True], [True, False], [False] * 2, [False] * 2]


def _select_case(lia, b, hq, hkv, d, budget, first, recent, q_type=BF16, seed=0, label="", change=None, extra=0, rows=None,
                 **more):
    rng = np.random.default_rng(seed)
    pool = D.Pool(rng, b.pool_pages, b.page, hkv, d, BF16)
    codes, scales = pool.summaries()
    q, qv = D.queries(rng, b.rows, hq, d, q_type)
    if change:
        change(codes, scales, q, qv)
        qv = q.float().cpu().numpy()
    cfg = b.config(lia, hq, hkv, d, BF16, q_type, max_rows=b.rows + 3, **more)
    print(f"[case] select {label} hq={hq} hkv={hkv} d={d} page={b.page} budget={budget}", flush=True)
    got, counts = D.select(lia, b, cfg, b.device(), q, G.to_dev(codes), G.to_dev(scales), budget, first, recent, extra)
    out_codes = np.concatenate([codes, np.zeros_like(codes[:1])])
    out_scales = np.concatenate([scales, np.zeros_like(scales[:1])])
    ref, n = D.expected(b, qv, hq // hkv, out_codes, out_scales, budget, first, recent, rows)
    at = np.arange(b.rows) if rows is None else rows
    assert np.array_equal(counts[at], n[at])
    assert np.array_equal(got[at], ref[at])
    assert (got[b.rows:] == 12345).all() and (counts[b.rows:] == 54321).all()
    return got


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 64), (4, 2, 128), (3, 1, 64), (8, 2, 128), (5, 1, 128), (16, 2, 64), (9, 1, 128),
                                      (16, 1, 128), (20, 1, 64), (64, 2, 128)])
@pytest.mark.parametrize("q_type", [BF16, F32])
def test_select_groups(lia, hq, hkv, d, q_type):
    """Decode and verify rows and prompt rows, of every size of a group."""
    b = D.Batch([1, 3, 1, 2], [1000, 333, 5, 700], 16, seed=hq)
    _select_case(lia, b, hq, hkv, d, 12, 1, 2, q_type, seed=hq, label="few rows")
    b = D.Batch([70, 41], [300, 1201], 16, seed=hq + 1)
    _select_case(lia, b, hq, hkv, d, 9, 2, 3, q_type, seed=hq + 1, label="chunks")


@pytest.mark.parametrize("page", [16, 32, 64, 256])
def test_select_pages(lia, page):
    b = D.Batch([1, 2, 1, 30], [40 * page, 17 * page - 1, page - 1, 9 * page + 3], page, seed=page)
    _select_case(lia, b, 8, 2, 64, 6, 1, 1, seed=page, label="page sizes")


@pytest.mark.parametrize("budget,first,recent", [(1, 0, 1), (2, 1, 1), (7, 3, 4), (5, 0, 5), (62, 0, 1), (63, 1, 1), (64, 1, 1),
                                                 (65, 0, 1), (200, 2, 2), (8, 0, 1)])
def test_select_budgets(lia, budget, first, recent):
    """Budgets that the first and the recent pages fill, one below a row's pages, all of them, more than a table holds."""
    b = D.Batch([1, 1, 1, 1], [63 * 16, 62 * 16, 0, 127 * 16 + 15], 16, seed=budget)
    _select_case(lia, b, 8, 2, 64, budget, first, recent, seed=budget, label=f"first={first} recent={recent}")


@pytest.mark.parametrize("page_of_all", [False, True])
def test_select_equal_scores(lia, page_of_all):
    """Equal scores go by the lower page: summaries and queries of zeros, and pages all alike."""
    def change(codes, scales, q, qv):
        if page_of_all:
            codes[:], scales[:] = codes[0], scales[0]
        else:
            q.zero_()
    b = D.Batch([1, 2, 1], [3000, 900, 16 * 300], 16, seed=5)
    got = _select_case(lia, b, 8, 2, 64, 90, 1, 2, seed=5, label="equal scores", change=change)
    assert got[0, 0, :88].tolist() == list(range(88))


def test_select_few_values(lia):
    """Runs of equal scores across the border: whole bins of more than 64 of them."""
    def change(codes, scales, q, qv):
        codes[:] = codes[np.random.default_rng(3).integers(0, 3, len(codes))]
        scales[:] = scales[0]
    b = D.Batch([1, 1], [16 * 1900, 16 * 700], 16, seed=6)
    for budget in (30, 400, 1000):
        _select_case(lia, b, 8, 2, 64, budget, 1, 2, seed=6, label="three values", change=change)


def test_select_infinite_pages_and_missing_ones(lia):
    b = D.Batch([1, 1, 40], [1000, 999, 500], 16, seed=7)
    b.table[b.row_of[1], 5:30] = NONE
    b.table[b.row_of[1], 30] = b.pool_pages

    def change(codes, scales, q, qv):
        for p in (3, 9, 17, 40):
            scales[p], codes[p] = np.inf, 0
    _select_case(lia, b, 8, 2, 128, 10, 1, 2, seed=7, label="infinite and missing pages", change=change)


@pytest.mark.parametrize("pages,budget", [(2047, 64), (2048, 300), (2049, 64), (8300, 1000), (20000, 70)])
def test_select_long(lia, pages, budget):
    """Tables past what a workgroup of either size holds in registers."""
    rng = np.random.default_rng(pages)
    b = D.Batch([1], [pages * 16 - 1], 16, seed=pages)
    hq, hkv, d = 2, 1, 64
    codes = rng.integers(-127, 128, (b.pool_pages, 1, 2, d)).astype(np.int8)
    scales = (2.0 ** rng.integers(-7, -4, (b.pool_pages, 1))).astype(np.float32)
    q, qv = D.queries(rng, 1, hq, d, BF16)
    cfg = b.config(lia, hq, hkv, d, BF16)
    print(f"[case] select {pages} pages", flush=True)
    got, counts = D.select(lia, b, cfg, b.device(), q, G.to_dev(codes), G.to_dev(scales), budget, 2, 5)
    ref, n = D.expected(b, qv, 2, codes, scales, budget, 2, 5)
    assert np.array_equal(got, ref) and np.array_equal(counts, n)


@pytest.mark.parametrize("pages", [2500, 12288, 12289])
def test_select_many_rows_of_long_tables(lia, pages):
    """Workgroups enough that scores and picks are one launch with the scores of a long table in LDS, up to what it holds."""
    rng = np.random.default_rng(pages)
    cached = rng.integers(0, 60 * 16, 128)
    cached[[3, 77]] = pages * 16 - 1
    b = D.Batch([1] * 128, cached, 16, seed=pages)
    codes = rng.integers(-127, 128, (b.pool_pages, 1, 2, 64)).astype(np.int8)
    scales = (2.0 ** rng.integers(-7, -4, (b.pool_pages, 1))).astype(np.float32)
    q, qv = D.queries(rng, 128, 8, 64, BF16)
    cfg = b.config(lia, 8, 1, 64, BF16)
    print(f"[case] select 128 rows of up to {pages} pages", flush=True)
    got, counts = D.select(lia, b, cfg, b.device(), q, G.to_dev(codes), G.to_dev(scales), 40, 1, 2)
    ref, n = D.expected(b, qv, 8, codes, scales, 40, 1, 2)
    assert np.array_equal(got, ref) and np.array_equal(counts, n)


@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 64), (8, 2, 128), (5, 1, 128), (16, 2, 128), (32, 2, 64), (34, 2, 64), (32, 1, 128)])
def test_select_large_chunks(lia, hq, hkv, d):
    """Chunks of a table long enough that four tiles of columns share the pages' codes."""
    rng = np.random.default_rng(hq)
    b = D.Batch([70, 41, 17], [300, 1201, 16 * 14000 + 5], 16, seed=hq)
    codes = rng.integers(-127, 128, (b.pool_pages, hkv, 2, d)).astype(np.int8)
    scales = (2.0 ** rng.integers(-7, -4, (b.pool_pages, hkv))).astype(np.float32)
    q, qv = D.queries(rng, b.rows, hq, d, BF16)
    cfg = b.config(lia, hq, hkv, d, BF16)
    print(f"[case] select large chunks, {hq} heads over {hkv} of {d}", flush=True)
    got, counts = D.select(lia, b, cfg, b.device(), q, G.to_dev(codes), G.to_dev(scales), 20, 1, 2)
    ref, n = D.expected(b, qv, hq // hkv, codes, scales, 20, 1, 2)
    assert np.array_equal(got, ref) and np.array_equal(counts, n)


def test_select_sequence_in_several_groups(lia):
    """Rows of one sequence that the batch names twice, one behind the other and apart."""
    b = D.Batch([6, 5], [700, 300], 16, seed=31)
    order = [0, 1, 2, 3, 6, 7, 8, 4, 5, 9, 10]
    b.sequences, b.positions = b.sequences[order], b.positions[order]
    b.cu, b.n = np.array([0, 2, 4, 7, 9, 11], np.uint32), 5
    _select_case(lia, b, 8, 2, 64, 9, 1, 2, seed=31, label="a sequence in several groups")
    _attend_case(lia, b, 8, 2, 64, BF16, 9, seed=31, label="a sequence in several groups")


def test_select_queries_that_are_not_finite(lia):
    """Their pages are unspecified, but some of the row's, and the other rows' are as ever."""
    def change(codes, scales, q, qv):
        q[1, 3, 7], q[1, 12, 0], q[2, 0] = float("nan"), float("inf"), float("-inf")
    b = D.Batch([1, 1, 1, 1], [900, 800, 700, 600], 16, seed=32)
    got = _select_case(lia, b, 16, 2, 128, 7, 1, 2, seed=32, label="queries of NaNs", change=change, rows=[0, 3])
    for r, n in ((1, 51), (2, 44)):
        assert (np.diff(got[r].astype(np.int64), axis=-1) > 0).all() and (got[r] < n).all()
        assert (got[r, :, 0] == 0).all() and (got[r, :, -2:] == [n - 2, n - 1]).all()


def test_select_rows_behind_the_last_sequence(lia):
    """Padding rows are left as they were, and of a rejected step (no sequence has rows) all are."""
    b = D.Batch([1, 2], [400, 700], 16, seed=8)
    _select_case(lia, b, 8, 2, 64, 6, 1, 1, seed=8, label="padding", extra=2)
    rng = np.random.default_rng(8)
    pool = D.Pool(rng, b.pool_pages, 16, 2, 64, BF16)
    codes, scales = pool.summaries()
    q, _ = D.queries(rng, 3, 8, 64, BF16)
    q5 = torch.cat([q, q[:2]])
    cfg = b.config(lia, 8, 2, 64, BF16, max_rows=5)
    dev = b.device()
    for cu, live in ((b.cu, 3), (np.zeros(3, np.uint32), 0)):
        dev["cu"] = G.u32_dev(cu)
        dev["positions"] = G.u32_dev(np.concatenate([b.positions, [0x7FFFFFFF, 3]]))
        dev["sequences"] = G.u32_dev(np.concatenate([b.sequences, [0x7FFFFFFF, 0xFFFFFFFF]]))
        selected = torch.full((5, 2, 6), 77, dtype=torch.int32, device="cuda")
        counts = torch.full((5,), 78, dtype=torch.int32, device="cuda")
        ws = torch.empty(lia.page_select_workspace_bytes(cfg), dtype=torch.uint8, device="cuda")
        print(f"[case] rows behind the last sequence, {live} live", flush=True)
        lia.page_select(cfg, 2, dev["cu"], dev["positions"], dev["sequences"], dev["pages"], q5, G.to_dev(codes),
                        G.to_dev(scales), 1, 1, selected, counts, ws)
        assert (selected[live:] == 77).all() and (counts[live:] == 78).all()
        assert live == 0 or (counts[:live] == 6).all()
        out = torch.full((5, 8, 64), 5.0, dtype=torch.bfloat16, device="cuda")
        ws = torch.empty(lia.selected_attention_workspace_bytes(cfg, 6), dtype=torch.uint8, device="cuda")
        lia.selected_attention(cfg, 2, dev["cu"], dev["positions"], dev["sequences"], dev["pages"], q5, pool.kc, pool.vc,
                               selected, counts, out, ws)
        assert (out[live:] == 5.0).all() and not (out[:live] == 5.0).all(-1).any()


def _pages(rng, b, hkv, budget, order=False):
    """Distinct pages of every row and head, some rows with few or none."""
    selected = np.full((b.rows, hkv, budget), NONE, np.uint32)
    counts = np.zeros(b.rows, np.uint32)
    for r in range(b.rows):
        n = int(b.positions[r]) // b.page + 1
        counts[r] = min(n, budget) if r % 5 != 3 else rng.integers(0, min(n, budget) + 1)
        for h in range(hkv):
            pick = rng.permutation(n)[:counts[r]]
            selected[r, h, :counts[r]] = pick if order else np.sort(pick)
    return selected, counts


def _attend_case(lia, b, hq, hkv, d, kv, budget, q_type=BF16, out_type=BF16, seed=0, label="", order=False, change=None):
    rng = np.random.default_rng(seed)
    pool = D.Pool(rng, b.pool_pages, b.page, hkv, d, kv)
    q, qv = D.queries(rng, b.rows, hq, d, q_type)
    selected, counts = _pages(rng, b, hkv, budget, order)
    if change:
        change(pool, selected, counts)
    cfg = b.config(lia, hq, hkv, d, kv, q_type, out_type)
    label = f"attend {label} kv={kv} hq={hq} hkv={hkv} d={d} page={b.page} budget={budget} rows={b.rows}"
    print("[case]", label, flush=True)
    got = D.attend(lia, b, cfg, b.device(), q, pool, selected, counts, out_type, extra=1)
    assert torch.isnan(got[b.rows:]).all()
    out, bound = D.reference(b, pool, qv, hq // hkv, selected, counts, cfg.scale, out_type)
    D.check(got[:b.rows], out, bound, label)
    return got


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (16, 2, 128), (3, 3, 128), (20, 1, 64), (64, 2, 128)])
@pytest.mark.parametrize("q_type,out_type", [(BF16, BF16), (F32, F32)])
def test_attend_types(lia, kv, hq, hkv, d, q_type, out_type):
    """Decode and verify rows over parts that are joined, and rows of few pages."""
    b = D.Batch([1, 3, 1, 2], [1000, 333, 5, 0], 16, seed=hq)
    _attend_case(lia, b, hq, hkv, d, kv, 12, q_type, out_type, seed=hq + d)


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("page,budget", [(16, 1), (16, 3), (16, 70), (16, 129), (32, 5), (64, 7), (128, 3), (1024, 2)])
def test_attend_pages(lia, kv, page, budget):
    """Lists of one page, odd ones, past 64 entries; pages of many tiles; the last page partly filled."""
    b = D.Batch([1, 2, 1, 1], [150 * 16 + 7, 900, 17, 4095], page, seed=page + budget)
    _attend_case(lia, b, 8, 2, 64, kv, budget, seed=budget, order=True)


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_chunks(lia, kv, d):
    """Enough rows that a workgroup takes a row and head whole."""
    b = D.Batch([200, 77], [300, 0], 16, seed=d)
    _attend_case(lia, b, 8, 2, d, kv, 9, F32 if d == 64 else BF16, seed=d, label="chunks")


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
def test_attend_one_key(lia, kv):
    b = D.Batch([1], [0], 16)
    _attend_case(lia, b, 8, 2, 128, kv, 4, F32, F32, label="one key")


def test_attend_rows_without_keys(lia):
    """No pages, entries outside the table or behind the row: zeros.  A count past the budget stands for the budget."""
    b = D.Batch([1, 1, 1, 1, 1], [100, 200, 300, 10, 400], 16, seed=3)

    def change(pool, selected, counts):
        counts[0] = 0
        selected[1], counts[1] = NONE, 3
        selected[2], counts[2] = [b.stride, 0x7FFFFFFF, 0x10000000, NONE], 4
        selected[3], counts[3] = [1, 2, 3, 5], 4          # behind position 10
        selected[4], counts[4] = [3, 1, 7, 25], 1000
    got = _attend_case(lia, b, 8, 2, 64, BF16, 4, label="rows without keys", change=change)
    assert (got[:4] == 0).all() and (got[4] != 0).any()


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
def test_attend_pages_outside_the_pool(lia, kv):
    """Table entries outside the pool hold keys of zeros."""
    b = D.Batch([1, 2], [300, 200], 16, seed=4)
    b.table[b.row_of[0], 2] = NONE
    b.table[b.row_of[0], 18] = b.pool_pages
    b.table[b.row_of[1], 12] = 1 << 30
    _attend_case(lia, b, 8, 2, 64, kv, 30, label="pages outside the pool", change=lambda p, s, c: (
        s.__setitem__((slice(None), slice(None), slice(0, 19)), np.arange(19)), c.__setitem__(slice(None), [19, 13, 13])))


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
def test_attend_slots_without_keys_hold_anything(lia, kv):
    """Rows behind a row's position - other rows' keys, a former owner's - are NaNs and infinities there."""
    b = D.Batch([1, 3], [37, 70], 16, seed=5)

    def change(pool, selected, counts):
        dead = []
        for s, last in ((0, 37), (1, 72)):
            page = int(b.table[b.row_of[s], last // 16])
            dead += [(page, o) for o in range(last % 16 + 1, 16)]
        for page, o in dead:
            for plane, scales in ((pool.kc, pool.ks), (pool.vc, pool.vs)):
                if kv == FP4:
                    plane[page, :, o], scales[page, :, o] = 0x77, 255 if o % 2 else 254
                elif kv == FP8:
                    plane[page, o] = 0x7F
                else:
                    plane[page, o] = float("nan") if o % 2 else float("inf")
    got = _attend_case(lia, b, 8, 2, 128, kv, 8, label="dead slots", change=change)
    assert torch.isfinite(got[:b.rows]).all()


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("hq,hkv,d,page", [(3, 3, 64, 64), (20, 1, 64, 32), (40, 2, 128, 64), (1, 1, 128, 128)])
def test_attend_dead_tiles_of_longer_pages(lia, kv, hq, hkv, d, page):
    """The same where whole tiles of a page, and parts of one, lie behind the row; and of pages outside the pool."""
    new, cached = [1, 3, 1, 1], [37, 2 * page + 5, 3 * page - 1, 5 * page + 20]
    b = D.Batch(new, cached, page, seed=page + d)
    b.table[b.row_of[3], 1:3] = [NONE, b.pool_pages]

    def change(pool, selected, counts):
        for s in range(4):
            last = cached[s] + new[s] - 1
            at = int(b.table[b.row_of[s], last // page]), slice(last % page + 1, page)
            for plane, scales in ((pool.kc, pool.ks), (pool.vc, pool.vs)):
                if kv == FP4:
                    plane[at[0], :, at[1]], scales[at[0], :, at[1]] = 0x77, 255
                elif kv == FP8:
                    plane[at] = 0x7F
                else:
                    plane[at] = float("nan")
    got = _attend_case(lia, b, hq, hkv, d, kv, 6, label="dead tiles", change=change, seed=page)
    assert torch.isfinite(got[:b.rows]).all()


@pytest.mark.parametrize("kv", [F16, BF16])
def test_attend_infinities_reach_their_rows(lia, kv):
    """V's of a key that later rows of the step attend, not the earlier ones; K's make their rows NaN."""
    b = D.Batch([4], [60], 16, seed=6)  # positions 60 .. 63, page 3

    def change(pool, selected, counts):
        selected[:], counts[:] = np.arange(8), 4
        pool.vc[int(b.table[b.row_of[0], 3]), 14, 1, 5] = float("inf")
        pool.v[int(b.table[b.row_of[0], 3]), 14, 1, 5] = np.inf
    rng = np.random.default_rng(6)
    pool = D.Pool(rng, b.pool_pages, 16, 2, 64, kv)
    q, _ = D.queries(rng, 4, 8, 64, BF16)
    selected, counts = np.tile(np.arange(8, dtype=np.uint32), (4, 2, 1)), np.full(4, 4, np.uint32)
    change(pool, selected, counts)
    cfg, dev = b.config(lia, 8, 2, 64, kv), b.device()
    print(f"[case] infinities of V kv={kv}", flush=True)
    got = D.attend(lia, b, cfg, dev, q, pool, selected, counts)
    odd = (~torch.isfinite(got)).nonzero().cpu().numpy()
    assert (odd[:, 0] >= 2).all() and (odd[:, 1] >= 4).all() and (odd[:, 2] == 5).all() and len(odd) == 2 * 4
    pool.kc[int(b.table[b.row_of[0], 3]), 13, 0, 9] = float("nan")
    got = D.attend(lia, b, cfg, dev, q, pool, selected, counts)
    nan = torch.isnan(got).all(-1).cpu().numpy()
    assert nan[1:, :4].all() and not nan[0].any() and not nan[:, 4:].any()


def test_attend_low_and_high_scores(lia):
    """First keys whose scores lie far below the later ones', and all far below 0."""
    b = D.Batch([1, 1], [16 * 40, 16 * 33], 16, seed=9)
    rng = np.random.default_rng(9)
    pool = D.Pool(rng, b.pool_pages, 16, 2, 64, BF16)
    q, qv = D.queries(rng, 2, 8, 64, F32)
    q.fill_(1.0), qv.fill(1.0)
    for i in range(41):
        pool.kc[int(b.table[b.row_of[0], i])] = -30.0 + i * 0.7
    for i in range(34):
        pool.kc[int(b.table[b.row_of[1], i])] = -40.0 - i * 0.3
    pool.k = pool.kc.double().cpu().numpy()
    selected, counts = np.tile(np.arange(41, dtype=np.uint32), (2, 2, 1)), np.array([41, 34], np.uint32)
    cfg = b.config(lia, 8, 2, 64, BF16, F32, F32)
    got = D.attend(lia, b, cfg, b.device(), q, pool, selected, counts, F32)
    out, bound = D.reference(b, pool, qv, 4, selected, counts, cfg.scale, F32)
    D.check(got[:2], out, bound * 4, "scores far below 0")  # (scores of up to 350 in the log2 domain, not 60)


@pytest.mark.parametrize("kv", [BF16, FP8, FP4])
def test_all_pages_selected_is_the_dense_attention(lia, kv):
    """With a budget of every page the rows' outputs are paged_attention's, within both calls' bounds."""
    b = D.Batch([1, 4, 30], [600, 77, 10], 16, seed=11)
    rng = np.random.default_rng(11)
    pool = D.Pool(rng, b.pool_pages, 16, 2, 128, kv)
    q, qv = D.queries(rng, b.rows, 16, 128, BF16)
    cfg, dev = b.config(lia, 16, 2, 128, kv), b.device()
    codes, scales = _summaries(lia, pool, np.arange(b.pool_pages) * 16 + 15)
    selected, counts = D.select(lia, b, cfg, dev, q, G.to_dev(codes), G.to_dev(scales), b.stride, 1, 1)
    got = D.attend(lia, b, cfg, dev, q, pool, selected, counts)
    out, bound = D.reference(b, pool, qv, 8, selected, counts, cfg.scale)
    D.check(got[:b.rows], out, bound, f"every page kv={kv}")
    dense = torch.empty((b.rows, 16, 128), dtype=torch.bfloat16, device="cuda")
    lia.paged_attention(cfg, b.n, dev["cu"], dev["positions"], dev["sequences"], dev["pages"], q, pool.kc, pool.vc, dense,
                        G.dirty_workspace(lia, cfg), pool.ks, pool.vs)
    assert (np.abs(dense.double().cpu().numpy() - got.double().cpu().numpy()) <= 2 * bound + (2e-2 if kv == FP8 else 0)).all()


def test_pages_past_four_gib(lia):
    """Pages whose elements, summaries and slots lie past 2^32 bytes and 2^31 elements into their planes."""
    page, hkv, d = 64, 8, 128
    pages = (5 << 30) // (page * hkv * d * 2) + 7
    kc, vc = (torch.zeros((pages, page, hkv, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    n = 40
    codes = torch.zeros((pages, hkv, 2, d), dtype=torch.int8, device="cuda")
    scales = torch.zeros((pages, hkv), device="cuda")
    rng = np.random.default_rng(12)
    b = D.Batch([2], [n * page - 2], page, slack=0)
    held = np.concatenate([np.arange(pages - 30, pages), rng.permutation(pages - 40)[:n - 30]])
    b.table[b.row_of[0], :n] = rng.permutation(held)
    b.pool_pages = pages
    small = D.Pool(rng, n, page, hkv, d, BF16)
    at = torch.from_numpy(b.table[b.row_of[0], :n].astype(np.int64)).cuda()
    kc[at], vc[at] = small.kc, small.vc
    print("[case] planes past 4 GiB", flush=True)
    slots = (b.table[b.row_of[0], :n].astype(np.int64) * page + page - 1).astype(np.uint32)
    lia.page_summaries(lia.KVLayout(hkv, d, page, pages, BF16), G.u32_dev(slots), kc, codes, scales)
    c, s = small.summaries()
    assert np.array_equal(codes[at].cpu().numpy(), c) and np.array_equal(scales[at].cpu().numpy(), s)
    q, qv = D.queries(rng, 2, 16, d, BF16)
    cfg, dev = b.config(lia, 16, hkv, d, BF16), b.device()
    selected, counts = D.select(lia, b, cfg, dev, q, codes, scales, 10, 1, 2)
    few = D.Batch([2], [n * page - 2], page, slack=0)  # the same sequence on a pool of its pages alone
    few.table[few.row_of[0], :n] = np.arange(n)
    few.sequences = np.full(2, few.row_of[0], np.uint32)
    ref, m = D.expected(few, qv, 2, c, s, 10, 1, 2)
    assert np.array_equal(selected, ref) and np.array_equal(counts, m)
    pool = type("P", (), dict(kc=kc, vc=vc, ks=None, vs=None))
    got = D.attend(lia, b, cfg, dev, q, pool, selected, counts)
    out, bound = D.reference(few, small, qv, 2, selected, counts, cfg.scale)
    D.check(got, out, bound, "planes past 4 GiB")


def _step(lia, pool, b, cfg, dev, q, new, table, query, codes, scales, selected, counts, out, ws, budget):
    """A layer of a decode step as it is used: rotation and append, summaries, selection, attention."""
    slots = dev["slots"]
    lia.qk_norm_rope_kv_append(pool.layout(lia), cfg.num_q_heads, table, new, query, pool.kc, pool.vc, slot_mapping=slots,
                               q_weight=dev["wq"], k_weight=dev["wk"], k_scales=pool.ks, v_scales=pool.vs)
    lia.page_summaries(pool.layout(lia), slots, pool.kc, codes, scales, k_scales=pool.ks)
    lia.page_select(cfg, b.n, dev["cu"], dev["positions"], dev["sequences"], dev["pages"], query, codes, scales, 1, 2, selected,
                    counts, ws[0])
    lia.selected_attention(cfg, b.n, dev["cu"], dev["positions"], dev["sequences"], dev["pages"], query, pool.kc, pool.vc,
                           selected, counts, out, ws[1], pool.ks, pool.vs)


class Layer:
    """A layer's step with its tensors; run() issues it."""

    def __init__(self, lia, kv, seed, new=(1, 3, 1, 20), cached=(1000, 445, 15, 300), budget=8):
        rng = np.random.default_rng(seed)
        self.lia, self.budget = lia, budget
        self.b = b = D.Batch(list(new), list(cached), 16, seed=seed)
        self.hq, self.hkv, self.d = 8, 2, 128
        self.pool = D.Pool(rng, b.pool_pages, 16, 2, 128, kv)
        self.cfg = b.config(lia, 8, 2, 128, kv)
        self.dev = b.device()
        entry = b.table[b.sequences, b.positions // 16]
        self.slots = (entry * 16 + b.positions % 16).astype(np.uint32)
        self.dev.update(slots=G.u32_dev(self.slots), wq=torch.rand(128, device="cuda") + 0.5,
                        wk=torch.rand(128, device="cuda") + 0.5)
        codes, scales = self.pool.summaries()
        self.codes, self.scales = G.to_dev(codes), G.to_dev(scales)
        self.new = torch.randn((b.rows, 12 * 128), device="cuda").bfloat16()
        f = torch.from_numpy(lia.rope_frequencies(64, 1e4)).cuda()
        self.f, self.table = f, torch.empty((b.rows, 32, 2), device="cuda")
        self.query = torch.empty((b.rows, 8, 128), dtype=torch.bfloat16, device="cuda")
        self.selected = torch.zeros((b.rows, 2, budget), dtype=torch.int32, device="cuda")
        self.counts = torch.zeros(b.rows, dtype=torch.int32, device="cuda")
        self.out = torch.zeros((b.rows, 8, 128), dtype=torch.bfloat16, device="cuda")
        self.ws = [torch.full((n,), 0x7E, dtype=torch.uint8, device="cuda")
                   for n in (lia.page_select_workspace_bytes(self.cfg),
                             lia.selected_attention_workspace_bytes(self.cfg, budget))]

    def run(self):
        self.lia.rope_table(self.dev["positions"], self.f, self.table)
        _step(self.lia, self.pool, self.b, self.cfg, self.dev, None, self.new, self.table, self.query, self.codes, self.scales,
              self.selected, self.counts, self.out, self.ws, self.budget)

    def results(self):
        return [t.clone() for t in (self.query, self.selected, self.counts, self.codes, self.scales, self.out)]


@pytest.mark.parametrize("kv", [BF16, FP8, FP4])
def test_step_together(lia, kv):
    """The chain as it is used, against the oracle on what the append left in the pool."""
    s = Layer(lia, kv, 21)
    print(f"[case] step kv={kv}", flush=True)
    s.run()
    b, pool = s.b, s.pool
    ko, vo = (torch.empty((b.pool_pages * 16, 2, 128), device="cuda") for _ in range(2))
    lia.kv_gather(pool.layout(lia), torch.arange(b.pool_pages * 16, dtype=torch.int32, device="cuda"), pool.kc, pool.vc, ko, vo,
                  k_scales=pool.ks, v_scales=pool.vs)
    pool.k, pool.v = (x.double().cpu().numpy().reshape(b.pool_pages, 16, 2, 128) for x in (ko, vo))
    codes, scales = pool.summaries()
    done = s.slots[s.slots % 16 == 15] // 16
    assert len(done) and np.array_equal(s.codes.cpu().numpy()[done], codes[done])
    codes, scales = s.codes.cpu().numpy(), s.scales.cpu().numpy()  # (others as they were: the row's own are not read)
    qv = s.query.float().cpu().numpy()
    ref, n = D.expected(b, qv, 4, codes, scales, s.budget, 1, 2)
    assert np.array_equal(s.selected.cpu().numpy().view(np.uint32), ref) and np.array_equal(s.counts.cpu().numpy(), n)
    out, bound = D.reference(b, pool, qv, 4, ref, n, s.cfg.scale)
    D.check(s.out, out, bound, f"step kv={kv}")


@pytest.mark.parametrize("kv", [BF16, FP8])
def test_captured_step_replays(lia, kv):
    """A captured step, replayed with other rows written and eager work between, equals the eager step bit for bit."""
    s = Layer(lia, kv, 22)
    s.run()
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    state = [t for t in (s.pool.kc, s.pool.vc, s.pool.ks, s.pool.vs, s.codes, s.scales) if t is not None]
    before = [t.clone() for t in state]
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        s.run()
    for i in range(4):
        print(f"[case] replay {i} kv={kv}", flush=True)
        s.new.copy_(torch.randn_like(s.new, dtype=torch.float32))
        for t, x in zip(state, before):
            t.copy_(x)
        s.run()
        torch.cuda.synchronize()
        expect = s.results()
        for t, x in zip(state, before):
            t.copy_(x)
        for t in (s.query, s.selected, s.counts, s.out):
            t.zero_()
        for w in s.ws:
            w.fill_(0x7E)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(s.results(), expect)), i


def test_two_streams_at_once(lia):
    layers = [Layer(lia, BF16, 23), Layer(lia, FP4, 24, (1,) * 9, (2000,) * 9), Layer(lia, F16, 25, (40,), (900,))]
    expect = []
    for s in layers:
        s.run()
        torch.cuda.synchronize()
        expect.append(s.results())
    streams = [torch.cuda.Stream() for _ in layers]
    for rep in range(3):
        print(f"[case] streams round {rep}", flush=True)
        for s in layers:
            s.out.zero_()
        torch.cuda.synchronize()
        for _ in range(2):
            for s, st in zip(layers, streams):
                with torch.cuda.stream(st):
                    s.run()
        torch.cuda.synchronize()
        for s, e in zip(layers, expect):
            assert all(torch.equal(x, y) for x, y in zip(s.results(), e))


# ------------------------------------------------------------------ the engine

def _engine(lia, kv, **more):
    e = lia.Engine(8, 2, 64, pool_tokens=16 * 128, layers=2, page_size=16, kv_dtype=kv, q_dtype=BF16, out_dtype=BF16,
                   prefill_batch=256, page_summaries=True, **more)
    e.configure_paging(4, 1024)
    return e


def _feed(e, rows, tables, seed, how="attention", layers=2, **more):
    g = torch.Generator(device="cuda").manual_seed(seed)
    e.stage(rows, tables)
    outs = []
    for layer in range(layers):
        q, k, v = (torch.randn((len(rows), h, 64), generator=g, device="cuda").bfloat16() for h in (8, 2, 2))
        outs.append(getattr(e, how)(layer, q, k, v, **more))
    return outs


def _full_pages_summarised(lia, e, pages):
    ends = G.u32_dev([p * 16 + 15 for p in pages])
    layout = lia.KVLayout(2, 64, 16, 128, e.kv_dtype)
    for layer in range(2):
        codes, scales = (torch.zeros_like(t) for t in e.summaries[layer])
        lia.page_summaries(layout, ends, e.k[layer], codes, scales, k_scales=e.k_scales[layer])
        at = torch.tensor(pages).cuda()
        assert torch.equal(codes[at], e.summaries[layer][0][at]) and torch.equal(scales[at], e.summaries[layer][1][at])
        assert (scales[at] > 0).all()


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
def test_engine_steps(lia, kv):
    """Prompts through the dense path, decode steps over selected pages: with a budget of all pages as the dense path, and the
    summaries those of the pool's pages."""
    e, f = _engine(lia, kv), _engine(lia, kv)
    tables = [list(range(40)), [100, 90, 80, 70, 60, 50]]
    prompt = [(1, i, 0) for i in range(200)] + [(1, i, 1) for i in range(50)]
    for x in (e, f):
        _feed(x, prompt, tables, 1)
    _full_pages_summarised(lia, e, list(range(12)) + [100, 90, 80])
    for step in range(20):
        rows = [(1, 200 + step, 0), (1, 50 + step, 1)]
        print(f"[case] engine step {step} kv={kv}", flush=True)
        a = _feed(e, rows, tables, 10 + step, "selected_attention", budget=64)
        d = _feed(f, rows, tables, 10 + step)
        for x, y in zip(a, d):
            assert (x.float() - y.float()).abs().max() < 4e-2
    assert torch.equal(e.k[1], f.k[1]) and torch.equal(e.v[0], f.v[0])
    _full_pages_summarised(lia, e, list(range(13)) + [100, 90, 80, 70])
    _feed(e, [(1, 220, 0), (1, 70, 1)], tables, 99, "selected_attention", budget=3)


def test_engine_captured_layer(lia):
    """A captured layer's replays append, summarise, select and attend what is staged then."""
    e, f = _engine(lia, BF16), _engine(lia, BF16)
    tables = [list(range(40)), [100, 90, 80, 70, 60, 50]]
    for x in (e, f):
        _feed(x, [(1, i, 0) for i in range(157)] + [(1, i, 1) for i in range(77)], tables, 1)
    q, k, v = (torch.zeros((2, h, 64), dtype=torch.bfloat16, device="cuda") for h in (8, 2, 2))
    e.stage([(1, 157, 0), (1, 77, 1)], tables)
    e.selected_attention(0, q, k, v, 5)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        out = e.selected_attention(0, q, k, v, 5)
    for i in range(6):
        rows = [(1, 157 + i, 0), (1, 77 + i, 1)]
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda"))
        f.stage(rows, tables)
        expect = f.selected_attention(0, q, k, v, 5)
        e.stage(rows, tables)
        print(f"[case] engine replay {i}", flush=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expect) and torch.equal(e.k[0], f.k[0])
        assert torch.equal(e.summaries[0][0], f.summaries[0][0]) and torch.equal(e.summaries[0][1], f.summaries[0][1])


def test_engine_eviction_and_restored_pages(lia):
    e = _engine(lia, BF16, track_weights=True)
    table = list(range(20, 40))
    _feed(e, [(1, i, 0) for i in range(200)], [table], 1)
    print("[case] engine eviction", flush=True)
    counts, _ = e.evict([table], [200], 90, 20)
    assert counts == [90]
    _full_pages_summarised(lia, e, table[:5])
    _feed(e, [(1, 90, 0), (1, 91, 0)], [table], 2, "selected_attention", budget=4)
    assert all((w[table[5], :, 10:12] == 0).all() for w in e.weights)
    pages = e.kv_transfer().read_kv_pages(table[:5])
    e.write_kv_pages(list(zip([3, 1, 4, 5, 9], pages)))
    _full_pages_summarised(lia, e, [3, 1, 4, 5, 9])
    for codes, scales in e.summaries:
        assert torch.equal(codes[[3, 1, 4, 5, 9]], codes[table[:5]])
