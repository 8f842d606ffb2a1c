"""A ragged batch on an MXFP4 pool for the GPU tests: seeded codes and scales, the device tensors, and the
f64 reference with its error bound."""
import numpy as np
import torch

import gpu_data as G
from oracle import mxfp4 as M

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4


def bf16_round(x):
    """f32 to the nearest bf16, as f32."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000
    return u.astype(np.uint32).view(np.float32)


class Fp4Case:
    """K and V are quantised N(0, 1) rows times `spread`-wide powers of two per block, by default sharp enough
    that some keys of a thousand carry most of a row."""

    def __init__(self, batch, seed=0, spread=1, q_scale=1.5):
        g, self.batch = batch.geom, batch
        self.g = g
        rng = np.random.default_rng(seed + 500)
        shape = (batch.pool_pages, g.hkv, g.page_size, g.d)

        def plane():
            x = rng.standard_normal(shape, dtype=np.float32).reshape(*shape[:3], -1, 32)
            x *= (2.0 ** rng.integers(-spread, spread + 1, (*x.shape[:-1], 1))).astype(np.float32)
            return M.quantise(x.reshape(shape))
        (self.kc, self.ks), (self.vc, self.vs) = plane(), plane()
        q = (q_scale * rng.standard_normal((batch.n_rows, g.hq, g.d))).astype(np.float32)
        self.q = bf16_round(q) if g.q_dtype == BF16 else q
        self.positions, self.sequences = batch.positions(), batch.sequences()
        self.cu, self.flat = batch.cu_seqlens(), batch.flat_table()

    def values(self):
        return M.dequantise(self.kc, self.ks), M.dequantise(self.vc, self.vs)

    def reference(self):
        """(softmax(q K^T) V, a bound of the kernels' error) in f64, from the queries as bf16."""
        g, b = self.g, self.batch
        k, v = self.values()
        q = bf16_round(self.q)
        out, bound = [], []
        for s in range(b.n_seqs):
            n, first = int(b.ctx[s]), int(b.cached[s])
            lo, hi = int(self.cu[s]), int(self.cu[s + 1])
            table = self.flat[s * b.stride:(s + 1) * b.stride]
            ks, vs = M.keys_of(k, table, n, g.page_size), M.keys_of(v, table, n, g.page_size)
            o = M.attention(q[lo:hi], ks, vs, first, g.scale)
            a = M.attention(q[lo:hi], ks, np.abs(vs), first, g.scale)
            # Each weight is rounded to bf16 (2^-8 of it) above the fraction line and below it, where the sum
            # cancels all but |o| 2^-8 <= a 2^-8; the output is rounded to bf16 (2^-8 of |o| <= a).  f32 sums of
            # n terms (n 2^-24 of a), the exponentials' own error (an ulp or two, 2^-22) and the scores' (d products
            # below |q||k|: d 2^-24 of a score of up to about 60 in the log2 domain) stay below 2^-9 of a.
            steps = 2 + (g.out_dtype == BF16) + 0.5
            out.append(o)
            bound.append(a * steps * 2.0 ** -8 + 1e-30)
        return np.concatenate(out), np.concatenate(bound)

    def device(self):
        g = self.g
        q = torch.from_numpy(self.q)
        return dict(kc=G.to_dev(self.kc), vc=G.to_dev(self.vc), ks=G.to_dev(self.ks), vs=G.to_dev(self.vs),
                    q=(q.to(torch.bfloat16) if g.q_dtype == BF16 else q).cuda(), positions=G.u32_dev(self.positions),
                    sequences=G.u32_dev(self.sequences), cu=G.u32_dev(self.cu), pages=G.u32_dev(self.flat))

    def config(self, lia, **more):
        g, b = self.g, self.batch
        a = dict(max_seqs=b.n_seqs, max_rows=max(b.n_rows, 1))
        a.update(more)
        return lia.AttentionConfig(g.hq, g.hkv, g.d, g.page_size, b.pool_pages, b.stride, g.q_dtype, FP4, g.out_dtype,
                                   g.scale, a["max_seqs"], a["max_rows"], int(b.ctx.max()))

    def run(self, lia, dev=None, **more):
        dev = dev or self.device()
        cfg = self.config(lia, **more)
        out = torch.full((self.batch.n_rows, self.g.hq, self.g.d), float("nan"), device="cuda",
                         dtype=torch.float32 if self.g.out_dtype == F32 else torch.bfloat16)
        lia.paged_attention(cfg, self.batch.n_seqs, dev["cu"], dev["positions"], dev["sequences"], dev["pages"],
                            dev["q"], dev["kc"], dev["vc"], out, G.dirty_workspace(lia, cfg), dev["ks"], dev["vs"])
        return out

    def check(self, lia, label, dev=None, **more):
        print(f"[case] fp4 {label}", flush=True)
        got = self.run(lia, dev, **more).float().cpu().numpy()
        ref, bound = self.reference()
        assert np.array_equal(np.isnan(got), np.isnan(ref)), label
        far = np.nan_to_num(np.abs(got - ref) / bound)
        print(f"[case] fp4 {label}: {far.max():.3f} of the bound", flush=True)
        assert far.max() <= 1.0, (label, float(far.max()))
