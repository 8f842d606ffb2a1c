"""Attention weights of keys that hold an infinity: one whose scores are -infinity in every column has a weight of 0, and the
columns that only fill up a tile have no say in it."""
import numpy as np
import pytest
import torch

import test_gpu_weights as W
from fp4_data import BF16, F16, FP4
from oracle import mxfp4 as M

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [BF16, F16, FP4])
@pytest.mark.parametrize("hq,hkv", [(16, 2), (3, 1), (32, 2)])
@pytest.mark.parametrize("ctx,q_len", [([300, 40, 1000], [1, 1, 1]), ([300, 40, 1000], [3, 2, 5]), ([300, 600], [40, 33])])
def test_keys_of_minus_infinity(lia, wl, kv, hq, hkv, ctx, q_len):
    b = wl.custom(ctx, q_len, geom=wl.Geometry(hq, hkv, 64, 16), seed=51)
    case = W.Case(b, kv, seed=52)
    case.q[..., 5] = np.abs(case.q[..., 5]) + 0.5
    marked = np.zeros(case.mass.shape, bool)
    for s, n in enumerate(ctx):
        for key in (0, 17, n // 2):
            page, off = int(b.tables[s][key // 16]), key % 16
            if kv == FP4:  # -6 x 2^126 in dim 5, the block's other elements 0
                case.codes[page, :, off, :16] = 0
                case.codes[page, :, off, 2] = 0xF0
                case.scales[page, :, off, 0] = 253
            else:
                case.store[page, off, :, 5] = -torch.inf
            marked[page, :, off] = True
    if kv == FP4:
        case.store = torch.from_numpy(case.codes)
        k = M.dequantise(case.codes, case.scales)
        case.k = np.where(np.abs(k) >= 2.0 ** 128, -np.inf, k)
    else:
        case.k = case.store.double().numpy().transpose(0, 2, 1, 3)
    print(f"[case] weights of -infinity kv={kv} {hq}/{hkv} rows {q_len}", flush=True)
    got = case.run(lia)
    case.k = np.where(np.isinf(case.k), -1e30, case.k)  # (the same weights, of finite scores)
    ref, added, _ = case.reference()
    assert (added[marked] == 0).all()
    assert np.array_equal(got[marked], case.mass[marked])
    # test_gpu_weights.py's bound with the scores of the other keys: below 64 |q| |k| scale = 64 x 7 x 6 x 0.125 = 336
    rel = 2 * 64 * 2.0 ** -24 * 336 + 2.0 ** -17 + 2.0 ** -12
    assert (np.abs(got - ref) <= rel * added + 2.0 ** -23 * np.abs(ref) + 1e-30).all()
