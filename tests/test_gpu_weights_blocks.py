"""Attention weights of prompt chunks at the edges of their second pass's blocks of 512 keys (the search for a block takes
64, 64 * 64 and 64 * 64 * 64 of them a step), and of selections at the edges of their segments of 8,192 keys."""
import numpy as np
import pytest
import torch

import gpu_data as G
import test_gpu_weights as W
from fp4_data import BF16, FP4, bf16_round
from oracle import mxfp4 as M
from test_gpu_evict import Pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("blocks", [1, 64])
@pytest.mark.parametrize("more", [-1, 0, 1, 16])
def test_chunks_at_block_edges(lia, wl, blocks, more):
    n = 512 * blocks + more
    for rows in (16, 100):
        b = wl.custom([n], [rows], geom=wl.Geometry(4, 2, 64, 16), seed=61)
        W.Case(b, BF16, seed=62).check(lia, f"chunk of {rows} over {n} keys")


@pytest.mark.parametrize("keys", [(1 << 21) + 5, (1 << 27) + 5, (1 << 28) - 4080])  # past 64^2 and 64^3 blocks, and most
def test_more_blocks_than_a_step_of_the_search_covers(lia, keys):
    """A table whose pages lie outside the pool but for its first, one past the 2^27th key and its last: keys outside weigh
    as zeros do, and the three pages' weights have closed forms."""
    hq, hkv, d, P, rows = 8, 1, 64, 65536, 16
    stride = -(-keys // P)
    names = sorted({0, min(stride - 1, (1 << 27) // P), stride - 1})
    pool = len(names)
    rng = np.random.default_rng(63)
    codes, scales = M.quantise((0.25 * rng.standard_normal((pool, hkv, P, d))).astype(np.float32))
    q = bf16_round(rng.standard_normal((rows, hq, d)).astype(np.float32))
    table = np.full(stride, 0xFFFFFFFF, np.uint32)
    table[names] = np.arange(pool)
    cfg = lia.AttentionConfig(hq, hkv, d, P, pool, stride, BF16, FP4, BF16, d ** -0.5, 1, rows, keys)
    size = lia.attention_weights_workspace_bytes(cfg)
    assert size > 0
    mass = torch.zeros((pool, hkv, P), dtype=torch.float32, device="cuda")
    print(f"[case] weights over {keys} keys", flush=True)
    lia.attention_weights(cfg, 1, G.u32_dev([0, rows]), G.u32_dev(np.arange(keys - rows, keys)), G.u32_dev(np.zeros(rows)),
                          G.u32_dev(table), torch.from_numpy(q).to(torch.bfloat16).cuda(), G.to_dev(codes), mass,
                          torch.empty(size, dtype=torch.uint8, device="cuda"), k_scales=G.to_dev(scales))
    got = mass.cpu().numpy()[:, 0]
    k = M.dequantise(codes, scales)[:, 0]
    s = np.einsum("rad,pkd->rapk", q.astype(np.float64), k) * d ** -0.5
    key = np.array(names)[:, None] * P + np.arange(P)
    live = key[None] <= (keys - rows + np.arange(rows))[:, None, None]
    e = np.where(live[:, None], np.exp(s), 0.0)
    outside = (keys - rows + 1 + np.arange(rows)) - live.sum((1, 2))
    total = e.sum((2, 3)) + outside[:, None]
    want = (e / total[:, :, None, None]).sum((0, 1))
    assert (want[-1, :(keys - 1) % P + 1] > 0).all()
    # test_gpu_weights.py's bound, |q||k| scale below 16, but for the lse's sum: a lane takes a quarter of its share's keys,
    # four at a time, so that its mass is a sum of keys / 16 / shares terms, each addition off by 2^-24 of it
    shares = 2 * lia.lib().lia_device_cus()
    rel = 2 * d * 2.0 ** -24 * 16 + 2.0 ** -17 + 2.0 ** -12 + (keys / 16 / shares) * 2.0 ** -24
    assert np.abs(s).max() < 16
    assert (np.abs(got - want) <= rel * want).all()


@pytest.mark.parametrize("candidates", [8191, 8192, 8193, 16385, 65536, 65537])
@pytest.mark.parametrize("recent", [0, 33])
@pytest.mark.parametrize("fill", ["spread", "ties", "odd"])
def test_selection_at_segment_edges(lia, candidates, recent, fill):
    print(f"[case] select {candidates} of them, recent {recent}, {fill}", flush=True)
    Pool([candidates + recent, 700], 16, 2, fill, seed=64).check(lia, 500, recent)


def test_sequences_past_the_steps_rows(lia, wl):
    """cu_seqlens past n_rows: the sequences behind it are none of the step's, and their keys' weights stay."""
    b = wl.custom([400, 90, 200], [1, 3, 40], geom=wl.Geometry(16, 2, 128, 16), seed=65)
    case = W.Case(b, FP4, seed=66)
    for cut in (1, 2):  # decode and verify rows alone
        cfg = case.config(lia)
        rows = int(b.cu_seqlens()[cut])
        mass = torch.from_numpy(case.mass).cuda()
        print(f"[case] weights, {rows} rows of {b.n_rows}", flush=True)
        lia.attention_weights(cfg, 3, G.u32_dev(b.cu_seqlens()), G.u32_dev(b.positions()), G.u32_dev(b.sequences()),
                              G.u32_dev(case.flat), torch.from_numpy(case.q[:rows]).to(torch.bfloat16).cuda(),
                              case.store.cuda(), mass,
                              torch.empty(lia.attention_weights_workspace_bytes(cfg), dtype=torch.uint8, device="cuda"),
                              k_scales=torch.from_numpy(case.scales).cuda())
        got = mass.cpu().numpy()
        for s in range(3):
            changed = got[b.tables[s]] != case.mass[b.tables[s]]
            assert changed.any() == (s < cut)
