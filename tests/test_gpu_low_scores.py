"""Rows whose first keys' scores lie far below zero (below -128 in the log2 domain): the running softmax has no mass to
scale when it takes its first reference there."""
import numpy as np
import pytest

import gpu_data as G
from fp4_data import BF16, F16, F32, FP4, FP8, Fp4Case, bf16_round
from oracle import mxfp4 as M

pytestmark = pytest.mark.gpu

STEPS = {"decode": ([900, 260, 4000], [1, 1, 1]), "verify": ([900, 700], [3, 3]), "prefill": ([600, 300], [100, 60])}


@pytest.mark.parametrize("kind", list(STEPS))
@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (4, 4, 64)])
def test_low_scores_first(lia, wl, O, kind, kv, hq, hkv, d):
    ctx, q_len = STEPS[kind]
    b = wl.custom(ctx, q_len, geom=wl.Geometry(hq, hkv, d, 16, q_dtype=BF16, kv_dtype=F16 if kv == FP4 else kv, out_dtype=F32),
                  seed=40)
    rng = np.random.default_rng(41)
    flat, P = b.flat_table(), 16
    k = rng.standard_normal((b.pool_pages, hkv, P, d)).astype(np.float32)
    v = rng.standard_normal((b.pool_pages, hkv, P, d)).astype(np.float32)
    for s in range(b.n_seqs):  # whole pages, so that an FP8 page's scale fits its rows
        for page in flat[s * b.stride:][:200 // P]:
            k[page] = -5 + 0.3 * k[page]
    q = bf16_round(4 + rng.standard_normal((b.n_rows, hq, d)).astype(np.float32))
    case = (Fp4Case if kv == FP4 else G.Case)(b, seed=42)
    if kv == FP4:
        (case.kc, case.ks), (case.vc, case.vs) = M.quantise(k), M.quantise(v)
        case.q = q
        k64, v64 = case.values()
    else:
        rows = [np.ascontiguousarray(x.transpose(0, 2, 1, 3)).reshape(-1, hkv, d) for x in (k, v)]
        if kv == FP8:
            O.kv_quantize_pages(O.KVLayout(hkv, d, P, b.pool_pages, FP8), np.arange(b.pool_pages), *rows, case.kc,
                                case.vc, case.k_scales, case.v_scales)
        else:
            case.kc, case.vc = (O.from_f32(x, kv).reshape(-1) for x in rows)
        case.q_store = O.from_f32(q, BF16)

        def values(store, scales):
            x = O.to_f32(store, kv).astype(np.float64).reshape(b.pool_pages, P, hkv, d).transpose(0, 2, 1, 3)
            return x if scales is None else x * scales.astype(np.float64).reshape(b.pool_pages, hkv, 1, 1)
        k64, v64 = values(case.kc, case.k_scales), values(case.vc, case.v_scales)
    got = case.run(lia)
    got = got if isinstance(got, np.ndarray) else got.float().cpu().numpy()
    cu = b.cu_seqlens()
    for s in range(b.n_seqs):
        n, first, lo, hi = int(b.ctx[s]), int(b.cached[s]), int(cu[s]), int(cu[s + 1])
        table = flat[s * b.stride:(s + 1) * b.stride]
        ks, vs = M.keys_of(k64, table, n, P), M.keys_of(v64, table, n, P)
        low = (q[lo:hi].reshape(hi - lo, hkv, -1, d).transpose(1, 0, 2, 3).reshape(hkv, -1, d).astype(np.float64)
               @ ks[:, :176].transpose(0, 2, 1)).max() * b.geom.scale
        assert low < -128 * np.log(2), low
        ref = M.attention(q[lo:hi], ks, vs, first, b.geom.scale)
        a = M.attention(q[lo:hi], ks, np.abs(vs), first, b.geom.scale)
        # As in Fp4Case.reference: the weights' rounding (bf16 at the coarsest) above and below the fraction line, 2^-8
        # each of a, and half a step for f32 sums and exponentials; a score is a sum of d products, |q||k| <= d 6 5.5,
        # each addition off by 2^-24 of it, in the exponent: 2 d d 33 2^-24 scale.
        rel = 2.5 * 2.0 ** -8 + 2 * d * d * 33 * 2.0 ** -24 * b.geom.scale
        assert np.isfinite(got[lo:hi]).all()
        far = np.abs(got[lo:hi] - ref) / (rel * a + 1e-30)
        print(f"[case] low scores {kind} kv={kv}: {far.max():.3f} of the bound", flush=True)
        assert far.max() <= 1.0
