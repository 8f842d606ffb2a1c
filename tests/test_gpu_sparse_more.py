"""Steps over selected pages as programs make them: captured ones that keep attention weights, rows that lie in a projection,
budgets past every table, the longest tables of the one-launch selection."""
import numpy as np
import pytest
import torch

import gpu_data as G
import sparse_data as D

pytestmark = pytest.mark.gpu

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4
TABLES = [list(range(40)), [100, 90, 80, 70, 60, 50]]


def _engine(lia, kv=BF16, **more):
    e = lia.Engine(8, 2, 64, pool_tokens=16 * 128, layers=2, page_size=16, kv_dtype=kv, q_dtype=BF16, out_dtype=BF16,
                   prefill_batch=256, page_summaries=True, **more)
    e.configure_paging(4, 1024)
    return e


def _prompt(e, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = [(1, i, 0) for i in range(157)] + [(1, i, 1) for i in range(77)]
    e.stage(rows, TABLES)
    for layer in range(2):
        e.attention(layer, *(torch.randn((len(rows), h, 64), generator=g, device="cuda").bfloat16() for h in (8, 2, 2)))


@pytest.mark.parametrize("track", [False, True])
def test_captured_steps_of_projections(lia, track):
    """Two layers in one graph, q, k and v as slices of one projection; replays with eager work of the same engine between."""
    e, f = _engine(lia, track_weights=track), _engine(lia, track_weights=track)
    for x in (e, f):
        _prompt(x)
    x = torch.zeros((2, 12 * 64), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((2, 8, 64), dtype=torch.bfloat16, device="cuda")
    k, v = x[:, 8 * 64:10 * 64], x[:, 10 * 64:]
    # (the warm-up's and the capture's own step is replayed, so it writes the same slots again)
    e.stage([(1, 157, 0), (1, 77, 1)], TABLES)
    for layer in range(2):
        e.selected_attention(layer, q, k, v, 5)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        outs = [e.selected_attention(layer, q, k, v, 5) for layer in range(2)]
    for i in range(6):
        rows = [(1, 157 + i, 0), (1, 77 + i, 1)]
        x.copy_(torch.randn(x.shape, device="cuda"))
        q.copy_(x[:, :8 * 64].view(2, 8, 64))
        for y in (e, f):
            y.stage(rows, TABLES)
            if track:
                for w in y.weights:  # what the slots' former keys left
                    w[TABLES[0][(157 + i) // 16], :, (157 + i) % 16] = 3.0
        expect = [f.selected_attention(layer, q, k.contiguous(), v.contiguous(), 5) for layer in range(2)]
        print(f"[case] replay {i} track={track}", flush=True)
        graph.replay()
        torch.cuda.synchronize()
        for layer in range(2):
            assert torch.equal(outs[layer], expect[layer])
            assert torch.equal(e.k[layer], f.k[layer]) and torch.equal(e.v[layer], f.v[layer])
            assert all(torch.equal(a, b) for a, b in zip(e.summaries[layer], f.summaries[layer]))
            if track:
                assert (e.weights[layer][TABLES[0][(157 + i) // 16], :, (157 + i) % 16] == 0).all()
                assert torch.equal(e.weights[layer], f.weights[layer])


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("how", ["attention", "selected_attention"])
def test_rows_of_a_projection(lia, kv, how):
    e, f = _engine(lia, kv), _engine(lia, kv)
    more = dict(budget=5) if how == "selected_attention" else {}
    for y in (e, f):
        _prompt(y)
        y.stage([(1, 157, 0), (1, 158, 0), (1, 77, 1)], TABLES)
    x = torch.randn((3, 12 * 64), device="cuda").to(torch.float16 if kv == F16 else torch.bfloat16)
    q = torch.randn((3, 8, 64), device="cuda").bfloat16()
    k, v = x[:, 8 * 64:10 * 64], x[:, 10 * 64:].unflatten(1, (2, 64))
    print(f"[case] rows of a projection {how} kv={kv}", flush=True)
    a = getattr(e, how)(0, q, k, v, **more)
    b = getattr(f, how)(0, q, k.contiguous(), v.contiguous(), **more)
    assert torch.equal(a, b) and torch.equal(e.k[0], f.k[0]) and torch.equal(e.v[0], f.v[0])


def test_budget_past_every_table(lia):
    e, f = _engine(lia), _engine(lia)
    for y in (e, f):
        _prompt(y)
        y.stage([(1, 157, 0), (1, 77, 1)], TABLES)
    q, k, v = (torch.randn((2, h, 64), device="cuda").bfloat16() for h in (8, 2, 2))
    print("[case] budgets past the table", flush=True)
    a, b = e.selected_attention(0, q, k, v, 1 << 40), f.selected_attention(0, q, k, v, 64)
    assert torch.equal(a, b)


@pytest.mark.parametrize("pages", [12288, 12289])
def test_longest_tables_of_one_launch(lia, pages):
    """128 single rows over one table, on either side of the length up to which one launch keeps its scores."""
    b = D.Batch([1], [pages * 16 - 1], 16, seed=pages, stride=pages)
    b.n = b.rows = 128
    b.sequences = np.repeat(b.sequences, 128)
    b.cu = np.arange(129, dtype=np.uint32)
    b.positions = (pages * 16 - 1 - 16 * 37 * np.arange(128)).astype(np.uint32)
    rng = np.random.default_rng(pages)
    codes = rng.integers(-127, 128, (b.pool_pages, 1, 2, 64)).astype(np.int8)
    scales = (2.0 ** rng.integers(-6, 0, (b.pool_pages, 1))).astype(np.float32)
    q, qv = D.queries(rng, 128, 2, 64, BF16)
    cfg = b.config(lia, 2, 1, 64, BF16)
    print(f"[case] select over {pages} pages", flush=True)
    got, counts = D.select(lia, b, cfg, b.device(), q, G.to_dev(codes), G.to_dev(scales), 40, 1, 3)
    rows = [0, 1, 63, 127]
    ref, n = D.expected(b, qv, 2, codes, scales, 40, 1, 3, rows)
    assert np.array_equal(counts[rows], n[rows]) and np.array_equal(got[rows], ref[rows])
    assert (np.diff(got.astype(np.int64), axis=-1) > 0).all() and (counts == 40).all()
