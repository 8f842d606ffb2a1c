"""Appends through the block table: a row whose position lies past its table row is not written, whoever owns the page
that the next row of the table begins with."""
import numpy as np
import pytest
import torch

import gpu_data as G

pytestmark = pytest.mark.gpu

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4
ENTRIES = ["kv_append", "rope_kv_append", "qk_norm_rope_kv_append"]


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("d", [64, 128])
def test_positions_past_the_table_row(lia, entry, kv, d):
    """Two sequences of two pages each (stride 2): positions 32 to 35 of the first would be the second's first slots, those of
    the second lie past the table."""
    print(f"[case] {entry} kv={kv} d={d}", flush=True)
    hq, hkv, page, pages = 2, 2, 16, 5
    table = np.array([4, 1, 3, 0], np.uint32)
    sequences = np.array([0, 0, 0, 0, 1, 1, 1, 0], np.uint32)
    positions = np.array([31, 32, 35, 0xFFFFFFFF, 5, 32, 40, 2], np.uint32)
    live = positions // page < 2
    rows = len(positions)
    layout = lia.KVLayout(hkv, d, page, pages, kv)
    if kv == FP4:
        shape, scales, kind = (pages, hkv, page, d // 2), (pages, hkv, page, d // 32), torch.uint8
        ks, vs = (torch.full(scales, 127, dtype=torch.uint8, device="cuda") for _ in range(2))
    else:
        shape, kind = (pages, page, hkv, d), {F16: torch.float16, BF16: torch.bfloat16, FP8: torch.uint8}[kv]
        ks, vs = (torch.ones((pages, hkv), device="cuda") if kv == FP8 else None for _ in range(2))
    x = torch.from_numpy(np.random.default_rng(d).standard_normal((rows, (hq + 2 * hkv) * d)).astype(np.float32)).cuda()
    angle = np.random.default_rng(1).uniform(0, 6.3, (rows, d // 2))
    coefficients = G.to_dev(np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32))

    def run(**how):
        kc, vc = (torch.full(shape, 1, dtype=kind, device="cuda") for _ in range(2))
        query = torch.full((rows, hq, d), float("nan"), device="cuda")
        more = dict(k_scales=None if ks is None else ks.clone(), v_scales=None if vs is None else vs.clone(), **how)
        if entry == "kv_append":
            lia.kv_append(layout, x[:, hq * d:(hq + hkv) * d].contiguous(), x[:, (hq + hkv) * d:].contiguous(), kc, vc, **more)
        elif entry == "rope_kv_append":
            lia.rope_kv_append(layout, hq, coefficients, x, query, kc, vc, **more)
        else:
            lia.qk_norm_rope_kv_append(layout, hq, coefficients, x, query, kc, vc, **more)
        return [t.cpu().view(torch.uint8) for t in (kc, vc, more["k_scales"], more["v_scales"]) if t is not None], query

    entries = table.reshape(2, 2)[sequences, np.where(live, positions // page, 0)]
    slots = np.where(live, entries * page + positions % page, 0xFFFFFFFF).astype(np.uint32)
    by_slot, q_slot = run(slot_mapping=G.u32_dev(slots))
    by_table, q_table = run(positions=G.u32_dev(positions), sequences=G.u32_dev(sequences), pages=G.u32_dev(table), stride=2)
    assert all(torch.equal(a, b) for a, b in zip(by_table, by_slot))
    if entry != "kv_append":  # every row gives its queries
        assert torch.equal(q_table, q_slot) and not torch.isnan(q_table).any()
    plane = by_table[0].reshape(pages, -1)
    start = torch.full(shape, 1, dtype=kind).view(torch.uint8).reshape(pages, -1)
    touched = [p for p in range(pages) if not torch.equal(plane[p], start[p])]
    assert touched == [1, 3, 4]  # page 3 by the second sequence's own row 5
