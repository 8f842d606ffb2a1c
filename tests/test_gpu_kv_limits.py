"""MXFP4 pools, attention weights and eviction at their limits: pages past 32-bit offsets, calls at once on two streams,
chunks of odd groups and many sequences, keys restored into a page."""
import numpy as np
import pytest
import torch

import gpu_data as G
import test_gpu_weights as W
from fp4_data import BF16, F16, F32, FP4, FP8, bf16_round
from oracle import mxfp4 as M

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d,kv,q", [(3, 1, 128, FP4, F32), (5, 1, 64, BF16, F32), (20, 1, 128, F16, BF16),
                                           (32, 1, 64, FP4, BF16), (5, 5, 128, FP8, F32), (7, 7, 64, FP8, BF16),
                                           (24, 2, 128, BF16, BF16)])
def test_chunks_of_odd_groups(lia, wl, hq, hkv, d, kv, q):
    """Prompt chunks whose blocks of columns end inside rows, from one key to blocks' edges."""
    b = wl.custom([600, 77, 1000, 33, 1, 513], [300, 77, 40, 1, 1, 129], geom=wl.Geometry(hq, hkv, d, 32), seed=21)
    W.Case(b, kv, q, seed=22).check(lia, f"chunk group {hq}/{hkv}x{d} kv={kv} q={q}")


@pytest.mark.parametrize("ctx,rows", [(17, 17), (16, 16), (4096, 16), (4097, 600), (700, 700)])
def test_one_chunk(lia, wl, ctx, rows):
    """Fewer units than workgroups, and a block that many share."""
    b = wl.custom([ctx], [rows], geom=wl.Geometry(8, 2, 128, 16), seed=23)
    W.Case(b, BF16, seed=24).check(lia, f"one chunk {ctx}/{rows}")


def test_chunks_of_many_sequences(lia, wl):
    """More chunks than one scan holds, some sequences without rows."""
    rng = np.random.default_rng(25)
    q_len = rng.integers(16, 24, 300)
    q_len[::37] = 0
    b = wl.custom(q_len + rng.integers(1, 90, 300), q_len, geom=wl.Geometry(4, 2, 64, 16), seed=26)
    assert b.n_rows >= 16 * b.n_seqs
    W.Case(b, FP4, seed=27).check(lia, "300 chunks")


def test_scores_that_rise(lia, wl):
    """Keys whose scores rise by thousands: the running reference has to follow."""
    b = wl.custom([900, 900], [1, 300], geom=wl.Geometry(4, 2, 64, 16), seed=28)
    for batch in (b, wl.custom([900, 40], [1, 1], geom=wl.Geometry(4, 2, 64, 16), seed=29)):
        case = W.Case(batch, F16, seed=30)
        for s in range(batch.n_seqs):
            n = int(batch.ctx[s])
            for j in range(n):
                page = int(case.flat[s * batch.stride + j // 16])
                case.store[page, j % 16] *= (j + 1) / n * 40
        case.k = case.store.double().numpy().transpose(0, 2, 1, 3)
        case.check(lia, "rising scores")


def test_fresh_keys(lia, wl):
    """`fresh`: the step's own keys begin at 0, whatever a page's former owner left; the others keep theirs."""
    for ctx, rows in (([40, 300, 17], [1, 3, 17]), ([500, 64], [200, 64]), ([40, 300], [1, 1])):
        b = wl.custom(ctx, rows, geom=wl.Geometry(8, 2, 64, 16), seed=31)
        case = W.Case(b, BF16, seed=32)
        clean = case.mass.copy()
        for s in range(b.n_seqs):
            for j in range(int(b.cached[s]), int(b.ctx[s])):
                page = int(case.flat[s * b.stride + j // 16])
                case.mass[page, :, j % 16] = np.nan
                clean[page, :, j % 16] = 0
        cfg = case.config(lia)
        q = torch.from_numpy(case.q).to(torch.bfloat16).cuda()
        out = []
        for mass, fresh in ((case.mass, True), (clean, False)):
            plane = torch.from_numpy(mass).cuda()
            ws = torch.empty(lia.attention_weights_workspace_bytes(cfg), dtype=torch.uint8, device="cuda")
            lia.attention_weights(cfg, b.n_seqs, G.u32_dev(b.cu_seqlens()), G.u32_dev(b.positions()),
                                  G.u32_dev(b.sequences()), G.u32_dev(case.flat), q, case.store.cuda(), plane, ws,
                                  fresh=fresh)
            out.append(plane.cpu().numpy())
        assert not np.isnan(out[0]).any()
        assert np.array_equal(out[0].view(np.uint32), out[1].view(np.uint32))


def test_two_streams_at_once(lia, wl):
    """Calls with workspaces of their own on two streams: each has the bits it has alone."""
    cases = [W.Case(wl.custom([3000, 900], [1, 1], geom=wl.Geometry(16, 2, 128, 16), seed=33), FP4, seed=34),
             W.Case(wl.custom([2000, 700], [300, 400], geom=wl.Geometry(8, 2, 128, 16), seed=35), BF16, seed=36)]
    alone = [c.run(lia) for c in cases]
    jobs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for c in cases:
        cfg, b = c.config(lia), c.b
        jobs.append((cfg, b, [G.u32_dev(x) for x in (b.cu_seqlens(), b.positions(), b.sequences(), c.flat)],
                     torch.from_numpy(c.q).to(torch.bfloat16).cuda(), c.store.cuda(),
                     None if c.scales is None else torch.from_numpy(c.scales).cuda(),
                     [torch.from_numpy(c.mass).cuda() for _ in range(5)],
                     torch.empty(lia.attention_weights_workspace_bytes(cfg), dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()
    for i in range(5):
        for s, (cfg, b, meta, q, kc, ks, masses, ws) in zip(streams, jobs):
            with torch.cuda.stream(s):
                lia.attention_weights(cfg, b.n_seqs, *meta, q, kc, masses[i], ws, k_scales=ks)
    torch.cuda.synchronize()
    for ref, job in zip(alone, jobs):
        for plane in job[6]:
            assert np.array_equal(plane.cpu().numpy().view(np.uint32), ref.view(np.uint32))


def test_pages_past_four_gigabytes(lia, O):
    """Append, gather, attention, weights, selection and compaction on the last pages of planes of more than 2^32 bytes
    (MXFP4 codes), elements and weights apart by as much: the bits of a small pool's same pages."""
    hq, hkv, d, P, n = 8, 4, 128, 64, 300
    far, near = (1 << 32) // (hkv * P * d // 2) + 9, 9
    rng = np.random.default_rng(37)
    rows = [torch.from_numpy(rng.standard_normal((n, hkv, d)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(2)]
    q = torch.from_numpy(rng.standard_normal((1, hq, d)).astype(np.float32)).to(torch.bfloat16).cuda()
    results = []
    for pages in (near, far):
        layout = lia.KVLayout(hkv, d, P, pages, FP4)
        kc, vc = (torch.empty((pages, hkv, P, d // 2), dtype=torch.uint8, device="cuda") for _ in range(2))
        ks, vs = (torch.empty((pages, hkv, P, d // 32), dtype=torch.uint8, device="cuda") for _ in range(2))
        mass = torch.empty((pages, hkv, P), dtype=torch.float32, device="cuda")
        ids = np.array([pages - 1 - i for i in (3, 0, 5, 1, 2)], np.uint32)  # 300 keys in the last pages
        for plane in (kc, vc, ks, vs, mass):
            plane[pages - near:] = 0
        slots = ids[np.arange(n) // P] * np.uint32(P) + np.arange(n, dtype=np.uint32) % P
        lia.kv_append(layout, *rows, kc, vc, slot_mapping=G.u32_dev(slots), k_scales=ks, v_scales=vs)
        ko, vo = (torch.empty((n, hkv, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        lia.kv_gather(layout, G.u32_dev(slots), kc, vc, ko, vo, k_scales=ks, v_scales=vs)
        stride = len(ids)
        cfg = lia.AttentionConfig(hq, hkv, d, P, pages, stride, BF16, FP4, F32, d ** -0.5, 1, 1, n)
        meta = [G.u32_dev(np.array(x, np.uint32)) for x in ([0, 1], [n - 1], [0])]
        table, out = G.u32_dev(ids), torch.empty((1, hq, d), dtype=torch.float32, device="cuda")
        lia.paged_attention(cfg, 1, *meta, table, q, kc, vc, out,
                            torch.empty(lia.workspace_bytes(cfg), dtype=torch.uint8, device="cuda"), ks, vs)
        lia.attention_weights(cfg, 1, *meta, table, q, kc, mass,
                              torch.empty(lia.attention_weights_workspace_bytes(cfg), dtype=torch.uint8, device="cuda"),
                              k_scales=ks)
        weights = mass[pages - near:].cpu().numpy()
        kept = torch.empty((1, hkv, 100), dtype=torch.int32, device="cuda")
        counts = torch.empty(1, dtype=torch.int32, device="cuda")
        one, length = G.u32_dev(np.zeros(1, np.uint32)), G.u32_dev(np.array([n], np.uint32))
        lia.kv_select(layout, one, length, table, stride, 100, 10, mass, kept, counts)
        lia.kv_compact(layout, one, table, table, stride, kept, counts, kc, vc, mass, ks, vs)
        torch.cuda.synchronize()
        results.append([x.float().cpu().numpy() for x in (ko, vo, out)] + [weights, kept.cpu().numpy(), counts.cpu().numpy()] +
                       [x[pages - near:].cpu().numpy() for x in (kc, vc, ks, vs, mass)])
        del kc, vc, ks, vs, mass
    assert (results[0][0] != 0).any() and (results[0][3] != 0).any()
    for a, b in zip(*results):
        assert np.array_equal(a, b)
    # and the gathered rows are the format's values
    codes, scales = M.quantise(rows[0].float().cpu().numpy())
    assert np.array_equal(results[0][0], bf16_round(M.dequantise(codes, scales)))


def test_restored_pages_begin_without_weights(lia):
    """A page written from a saved payload holds other keys: the weight its former keys received is not theirs."""
    e = lia.Engine(num_q_heads=4, num_kv_heads=2, head_dim=64, pool_tokens=256, layers=2, page_size=16, kv_dtype=BF16,
                   q_dtype=F32, out_dtype=F32, prefill_batch=64, track_weights=True)
    e.configure_paging(2, 64)
    g = torch.Generator(device="cuda").manual_seed(5)
    e.stage([(1, i, 0) for i in range(40)], [[3, 4, 5]])
    for layer in range(2):
        q = torch.randn((40, 4, 64), generator=g, device="cuda")
        k, v = (torch.randn((40, 2, 64), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        e.attention(layer, q, k, v)
    before = [w.clone() for w in e.weights]
    assert all((w[[3, 4]] > 0).all() for w in before)
    payload = e.read_kv_page(3)
    e.write_kv_page(4, payload)
    for w, old in zip(e.weights, before):
        assert (w[4] == 0).all() and torch.equal(w[[3, 5]], old[[3, 5]])
    e.write_kv_pages([(3, payload), (5, payload)])
    for w in e.weights:
        assert (w[[3, 4, 5]] == 0).all()


def test_selection_on_another_stream(lia):
    """Long tables with a workspace of the caller's, in any state, on a stream of its own: the bits of the default call's."""
    rng = np.random.default_rng(51)
    hkv, page, lengths, budget, recent = 2, 64, [20000, 700, 9000], 900, 100
    stride = -(-max(lengths) // page)
    pages = stride * len(lengths)
    layout = lia.KVLayout(hkv, 128, page, pages, BF16)
    table = G.u32_dev(rng.permutation(pages).astype(np.uint32))
    rows, held = G.u32_dev(np.arange(3, dtype=np.uint32)), G.u32_dev(np.array(lengths, np.uint32))
    mass = torch.from_numpy(rng.random((pages, hkv, page)).astype(np.float32)).cuda()
    size = lia.kv_select_workspace_bytes(layout, 3, stride)
    assert size > 0
    out = []
    s = torch.cuda.Stream()
    for workspace, stream in ((None, None), (torch.full((size,), 0x7E, dtype=torch.uint8, device="cuda"), s)):
        kept = torch.full((3, hkv, budget), 5, dtype=torch.int32, device="cuda")
        counts = torch.full((3,), 5, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        lia.kv_select(layout, rows, held, table, stride, budget, recent, mass, kept, counts, workspace,
                      stream=stream)
        torch.cuda.synchronize()
        out.append((kept.cpu().numpy().view(np.uint32), counts.cpu().numpy()))
    assert np.array_equal(out[0][0], out[1][0]) and np.array_equal(out[0][1], out[1][1])
    flat, weights = table.cpu().numpy().reshape(3, stride), mass.cpu().numpy()
    for i, n in enumerate(lengths):
        for h in range(hkv):
            key = np.arange(n)
            m = weights[flat[i][key // page], h, key % page]
            assert np.array_equal(out[1][0][i, h, :min(n, budget)], M.select(m, budget, recent))
