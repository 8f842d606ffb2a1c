"""Attention over selected pages where a list is shared by several workgroups and joined: long lists of 16-bit pools between
64 and 128 rows and heads too.  A joined call writes its parts' records into the workspace, one that is not leaves it."""
import numpy as np
import pytest
import torch

import gpu_data as G
import sparse_data as D

pytestmark = pytest.mark.gpu

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4


def _lists(b, hkv, budget, seed):
    """Each row's first and last page and random others of its own, ascending."""
    rng = np.random.default_rng(seed)
    selected, counts = np.full((b.rows, hkv, budget), D.NONE, np.uint32), np.zeros(b.rows, np.uint32)
    for r in range(b.rows):
        n = int(b.positions[r]) // b.page + 1
        counts[r] = min(n, budget)
        for h in range(hkv):
            inner = 1 + rng.permutation(n - 2)[:max(int(counts[r]) - 2, 0)]
            selected[r, h, :counts[r]] = np.sort(np.concatenate([[0], inner, [n - 1]]))[:counts[r]]
    return selected, counts


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [33, 48, 64])
@pytest.mark.parametrize("keys,shared", [(768, None), (4096, True)])
def test_long_lists_of_more_than_64_rows_and_heads(lia, kv, d, rows, keys, shared):
    print(f"[case] parts kv={kv} d={d} rows={rows} keys={keys}", flush=True)
    hq, hkv, page, budget = 6, 2, 16, keys // 16
    b = D.Batch([rows], [keys + 700], page, seed=rows)
    rng = np.random.default_rng(keys + d)
    pool = D.Pool(rng, b.pool_pages, page, hkv, d, kv)
    cfg, dev = b.config(lia, hq, hkv, d, kv, q=BF16, out=F32), b.device()
    q, values = D.queries(rng, rows, hq, d, BF16)
    selected, counts = _lists(b, hkv, budget, rows)
    out = torch.full((rows, hq, d), float("nan"), device="cuda")
    ws = torch.full((lia.selected_attention_workspace_bytes(cfg, budget),), 0x7E, dtype=torch.uint8, device="cuda")
    lia.selected_attention(cfg, b.n, dev["cu"], dev["positions"], dev["sequences"], dev["pages"], q, pool.kc, pool.vc,
                           G.u32_dev(selected), G.u32_dev(counts), out, ws, pool.ks, pool.vs)
    if shared is None:  # FP8 lists are shared from here on
        shared = kv == FP8
    assert bool((ws != 0x7E).any()) == shared
    ref, bound = D.reference(b, pool, values, hq // hkv, selected, counts, cfg.scale, F32)
    D.check(out, ref, bound, f"kv={kv} rows={rows} keys={keys}")
