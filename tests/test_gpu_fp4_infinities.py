"""Infinities of V on an MXFP4 pool (large codes under the scales 253 and 254): those in slots that hold no key change
nothing, and those of a key reach the rows that attend it and no earlier one."""
import numpy as np
import pytest
import torch

import gpu_data as G
from fp4_data import BF16, F32, FP4, Fp4Case
from oracle import mxfp4 as M

pytestmark = pytest.mark.gpu

STEPS = [([900, 77, 33], [1, 1, 1]), ([900, 77, 40], [3, 2, 8]), ([400, 90], [100, 50]), ([1], [1]), ([33], [33]),
         ([2500, 1100], [130, 70])]


def _batch(wl, ctx, q_len, d, out=BF16):
    """Tables that do not name page 0."""
    b = wl.custom(ctx, q_len, geom=wl.Geometry(16, 2, d, 16, FP4, BF16, out), seed=41)
    b.pool_pages += 3
    b.tables = [np.asarray(t) + 2 for t in b.tables]
    return b


def _live(b, page=16):
    live = np.zeros((b.pool_pages, page), bool)
    for t, n in zip(b.tables, b.ctx):
        key = np.arange(int(n))
        live[t[key // page], key % page] = True
    return live


@pytest.mark.parametrize("ctx,q_len", STEPS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("fill", [253, 254, 255, "random"])
def test_slots_without_a_key_hold_anything(lia, wl, ctx, q_len, d, fill):
    b = _batch(wl, ctx, q_len, d)
    case, rng, dead = Fp4Case(b, seed=42), np.random.default_rng(43), ~_live(b)
    assert dead[0].all() and dead.any()
    want = Fp4Case(b, seed=42).run(lia)
    for codes, scales in ((case.kc, case.ks), (case.vc, case.vs)):
        c, s = codes.transpose(0, 2, 1, 3), scales.transpose(0, 2, 1, 3)
        c[dead] = rng.integers(0, 256, c[dead].shape) if fill == "random" else 0x77
        s[dead] = rng.integers(0, 256, s[dead].shape) if fill == "random" else fill
    if fill == "random":  # (one of every kind at least)
        case.vs[0, 0, :4, 0] = 252, 253, 254, 255
    case.check(lia, f"dead slots {fill} d={d} rows {b.n_rows}")
    got = case.run(lia)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("ctx,q_len", STEPS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("out", [BF16, F32])
def test_infinities_reach_the_rows_that_attend_them(lia, wl, ctx, q_len, d, out):
    """Whole numbers of the last keys' blocks: infinities of one sign and, in a dim of two keys, of both."""
    b = _batch(wl, ctx, q_len, d, out)
    case, rng = Fp4Case(b, seed=44), np.random.default_rng(45)
    for t, n in zip(b.tables, b.ctx):
        for back, h, blk, s in ((1, 0, 0, 253), (2, 1, d // 32 - 1, 254), (3, 0, 0, 254), (4, 1, 0, 255), (20, 0, 1, 253),
                               (int(n) // 2 + 1, 1, 0, 254)):
            key = int(n) - back
            if key < 0:
                continue
            at = (t[key // 16], h, key % 16)
            case.vs[(*at, blk)] = s
            # codes 0 and +-6 (0x7, 0xF): 6 x 2^126 is past 2^128
            case.vc[at][16 * blk:16 * blk + 16] = rng.choice(np.array([0x00, 0x07, 0x70, 0x0F, 0xF0, 0x08], np.uint8), 16)
    g, v = case.g, M.dequantise(case.vc, case.vs)
    far = np.abs(v) >= 2.0 ** 128
    plain = case.vc.copy(), case.vs.copy()
    want = []
    for s in range(b.n_seqs):
        n, first, lo, hi = int(b.ctx[s]), int(b.cached[s]), int(case.cu[s]), int(case.cu[s + 1])
        table = case.flat[s * b.stride:(s + 1) * b.stride]
        k = M.keys_of(M.dequantise(case.kc, case.ks), table, n, 16)
        finite = M.keys_of(np.where(far, 0.0, v), table, n, 16)
        o = M.attention(case.q[lo:hi], k, finite, first, g.scale)
        live = (np.arange(n)[None, :] <= first + np.arange(hi - lo)[:, None]).astype(np.float64)
        for sign in (1, -1):
            x = M.keys_of((far & (np.sign(v) == sign)).astype(np.float64), table, n, 16)
            hit = np.einsum("rk,hkd->rhd", live, x) > 0
            with np.errstate(invalid="ignore"):
                o += np.where(np.repeat(hit, g.hq // g.hkv, 1), sign * np.inf, 0.0)
        a = M.attention(case.q[lo:hi], k, np.abs(finite), first, g.scale)
        want.append((o, a * (2.5 + (out == BF16)) * 2.0 ** -8 + 1e-30))  # (the bound of fp4_data.py)
    ref, bound = (np.concatenate(x) for x in zip(*want))
    assert np.isinf(ref).any() and np.isnan(ref).any() == (max(ctx) > 3) and (np.isfinite(ref).any() or b.n_rows == 1)
    print(f"[case] infinities d={d} rows {b.n_rows} out={out}", flush=True)
    got = case.run(lia).float().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(np.where(np.isinf(got), got, 0.0), np.where(np.isinf(ref), ref, 0.0))
    ok = np.isfinite(ref)
    assert (np.abs(got[ok] - ref[ok]) <= bound[ok]).all()
    assert np.array_equal(plain[0], case.vc) and np.array_equal(plain[1], case.vs)


def test_gathered_values_of_every_scale(lia):
    """Every code under every scale, as f32, bf16 and f16: past the type's range an infinity, 255 a NaN."""
    page, pool = 16, 16
    codes = np.tile(np.arange(16, dtype=np.uint8), 2)
    kc = np.broadcast_to(codes[0::2] | codes[1::2] << 4, (pool, 1, page, 16)).copy()
    ks = np.arange(256, dtype=np.uint8).reshape(pool, 1, page, 1)
    slots = G.u32_dev(np.arange(256, dtype=np.uint32))
    layout = lia.KVLayout(1, 32, page, pool, FP4)
    print("[case] gather, every scale", flush=True)
    ref = M.dequantise(kc, ks).reshape(256, 1, 32)
    for t in (torch.float32, torch.bfloat16, torch.float16):
        ko, vo = (torch.empty((256, 1, 32), dtype=t, device="cuda") for _ in range(2))
        lia.kv_gather(layout, slots, G.to_dev(kc), G.to_dev(kc), ko, vo, k_scales=G.to_dev(ks), v_scales=G.to_dev(ks))
        want = torch.from_numpy(ref).to(torch.float32).to(t)
        assert torch.equal(torch.nan_to_num(ko.cpu(), nan=-7.0, posinf=8e4, neginf=-8e4),
                           torch.nan_to_num(want, nan=-7.0, posinf=8e4, neginf=-8e4)), t
        assert torch.equal(ko.view(torch.uint8), vo.view(torch.uint8))
