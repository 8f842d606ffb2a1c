"""lia_attention_weights on the GPU against 64 bits: every pool type, decode, verify and prompt rows, long and many
sequences, decays, hidden NaNs, dead pages."""
import numpy as np
import pytest
import torch

import gpu_data as G
from fp4_data import BF16, F16, F32, FP4, FP8, bf16_round
from oracle import mxfp4 as M

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, batch, kv, q_dtype=BF16, seed=0):
        g, self.b, self.kv, self.q_dtype = batch.geom, batch, kv, q_dtype
        self.g = g
        rng = np.random.default_rng(seed + 900)
        x = rng.standard_normal((batch.pool_pages, g.hkv, g.page_size, g.d), dtype=np.float32)
        self.scales = None
        if kv == FP4:
            self.codes, self.scales = M.quantise(x)
            self.k = M.dequantise(self.codes, self.scales)
            self.store = torch.from_numpy(self.codes)
        else:
            t = torch.from_numpy(x.transpose(0, 2, 1, 3).copy())
            if kv == FP8:
                self.scales = rng.uniform(0.005, 0.012, (batch.pool_pages, g.hkv)).astype(np.float32)
                t = (t * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
                self.store = t.view(torch.uint8)
                self.k = t.double().numpy().transpose(0, 2, 1, 3) * self.scales.astype(np.float64)[:, :, None, None]
            else:
                self.store = t.to(torch.bfloat16 if kv == BF16 else torch.float16)
                self.k = self.store.double().numpy().transpose(0, 2, 1, 3)
        q = (1.5 * rng.standard_normal((batch.n_rows, g.hq, g.d))).astype(np.float32)
        self.q = bf16_round(q) if q_dtype == BF16 else q
        self.mass = rng.uniform(0, 1e-2, (batch.pool_pages, g.hkv, g.page_size)).astype(np.float32)
        self.flat = batch.flat_table()

    def config(self, lia, **more):
        g, b = self.g, self.b
        a = dict(max_seqs=b.n_seqs, max_rows=b.n_rows)
        a.update(more)
        return lia.AttentionConfig(g.hq, g.hkv, g.d, g.page_size, b.pool_pages, b.stride, self.q_dtype, self.kv, BF16,
                                   g.scale, a["max_seqs"], a["max_rows"], int(b.ctx.max()))

    def run(self, lia, decay=1.0, mass=None, **more):
        b = self.b
        cfg = self.config(lia, **more)
        ws = torch.full((lia.attention_weights_workspace_bytes(cfg),), 0x7E, dtype=torch.uint8, device="cuda")
        mass = torch.from_numpy(self.mass if mass is None else mass).cuda()
        q = torch.from_numpy(self.q)
        q = (q.to(torch.bfloat16) if self.q_dtype == BF16 else q).cuda()
        lia.attention_weights(cfg, b.n_seqs, G.u32_dev(b.cu_seqlens()), G.u32_dev(b.positions()),
                              G.u32_dev(b.sequences()), G.u32_dev(self.flat), q, self.store.cuda(), mass, ws,
                              k_scales=None if self.scales is None else torch.from_numpy(self.scales).cuda(), decay=decay)
        return mass.cpu().numpy()

    def reference(self, decay=1.0):
        """The weight plane and a bound of the kernels' relative error of what they add."""
        g, b = self.g, self.b
        q = bf16_round(self.q) if self.kv in (BF16, FP4) else self.q.astype(np.float16).astype(np.float32)
        cu = b.cu_seqlens()
        mass = self.mass.astype(np.float64)
        added, worst = np.zeros_like(mass), 0.0
        for s in range(b.n_seqs):
            n, first, lo, hi = int(b.ctx[s]), int(b.cached[s]), int(cu[s]), int(cu[s + 1])
            if hi == lo:
                continue
            table = self.flat[s * b.stride:(s + 1) * b.stride]
            k = M.keys_of(self.k, table, n, g.page_size)
            w = M.softmax_weights(q[lo:hi], k, first, g.scale).sum((1, 2))
            worst = max(worst, float(np.nanmax(np.abs(q[lo:hi])) * np.nansum(np.abs(k), -1).max()))
            for i in range(-(-n // g.page_size)):
                e, part = int(table[i]), w[:, i * g.page_size:(i + 1) * g.page_size]
                if e < b.pool_pages:
                    m = part.shape[1]
                    added[e, :, :m] += part
                    mass[e, :, :m] = part + (decay * mass[e, :, :m] if decay else 0)
        # The products are exact; a score is a sum of d of them, each addition off by 2^-24 of at most sum |q||k|
        # (<= worst), and so is the lse: 2 d 2^-24 worst scale, in the exponent (natural).  The exponent's own
        # rounding (values below 128: 2^-18) and the exponentials' and logarithms' (2^-21), and the sums of n weights in
        # tiles of 4 lanes x 4 and then of the rows (below 2^12 additions in a row: 2^-12 at most, in truth far less).
        rel = 2 * g.d * 2.0 ** -24 * worst * g.scale + 2.0 ** -17 + 2.0 ** -12
        return mass, added, rel

    def check(self, lia, label, decay=1.0, **more):
        print(f"[case] weights {label}", flush=True)
        got = self.run(lia, decay, **more)
        ref, added, rel = self.reference(decay)
        assert np.array_equal(np.isnan(got), np.isnan(ref)), label
        bound = rel * added + 2.0 ** -23 * np.abs(ref) + 1e-30
        far = np.nan_to_num(np.abs(got - ref) / bound)
        typical = np.nan_to_num(np.linalg.norm(np.nan_to_num(got - ref)) / np.linalg.norm(np.nan_to_num(added)))
        print(f"[case] weights {label}: {far.max():.3f} of the bound, error {typical:.2e}", flush=True)
        assert far.max() <= 1.0, label
        live = added != 0
        return got, live


STEPS = {
    "decode": ([1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 511, 513, 2049, 5000], [1] * 15),
    "verify": ([40, 1200, 17, 3000, 300], [3, 1, 2, 4, 8]),
    "prompt": ([300, 1077, 2040], [300, 77, 1000]),
    "mixed": ([700, 33, 1500, 64, 9], [130, 1, 1, 64, 9]),
}


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("kind", list(STEPS))
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 2, 128, 16), (8, 2, 64, 64)])
def test_weights(lia, wl, kv, kind, hq, hkv, d, page):
    ctx, q_len = STEPS[kind]
    b = wl.custom(ctx, q_len, geom=wl.Geometry(hq, hkv, d, page), seed=1)
    case = Case(b, kv, seed=2)
    got, _ = case.check(lia, f"{kind} kv={kv} {hq}/{hkv}x{d} page {page}")
    again = case.run(lia)
    assert np.array_equal(got.view(np.uint32), again.view(np.uint32))  # a fixed order


@pytest.mark.parametrize("hq,hkv,kv,q", [(3, 1, FP4, F32), (20, 1, BF16, F32), (32, 1, FP4, BF16), (5, 5, F16, F32),
                                         (24, 2, FP8, F32), (7, 7, FP4, BF16)])
def test_groups_and_query_types(lia, wl, hq, hkv, kv, q):
    b = wl.custom([600, 33, 90], [40, 1, 3], geom=wl.Geometry(hq, hkv, 128, 32), seed=3)
    Case(b, kv, q, seed=4).check(lia, f"group {hq}/{hkv} kv={kv} q={q}")


def test_a_long_context(lia, wl):
    """More than 64 splits of 512 keys."""
    b = wl.custom([70001, 40000], [1, 2], geom=wl.Geometry(8, 1, 128, 16), seed=5)
    Case(b, FP4, seed=6).check(lia, "long")


def test_a_long_prompt(lia, wl):
    """More than 32 splits of 1,024 keys."""
    b = wl.custom([34000], [40], geom=wl.Geometry(4, 2, 64, 64), seed=7)
    Case(b, FP4, seed=8).check(lia, "long prompt")


@pytest.mark.parametrize("n", [300, 1100])
def test_many_sequences(lia, wl, n):
    """More sequences than a workgroup's threads, and than one scan holds; some without rows."""
    rng = np.random.default_rng(n)
    q_len = (rng.random(n) < 0.8).astype(int)
    q_len[0] = 1
    q_len[n // 2] = 20
    ctx = np.maximum(rng.integers(1, 40, n), q_len)
    b = wl.custom(ctx, q_len, geom=wl.Geometry(4, 2, 64, 16), seed=9)
    Case(b, BF16, seed=10).check(lia, f"{n} sequences")


@pytest.mark.parametrize("decay", [0.0, 0.5, 1.0, 2.0])
def test_decay(lia, wl, decay):
    b = wl.custom([400, 90, 70], [1, 3, 65], geom=wl.Geometry(16, 2, 128, 16), seed=11)
    case = Case(b, FP4, seed=12)
    got, live = case.check(lia, f"decay {decay}", decay)
    rest = np.ones_like(live)
    for t, n in zip(b.tables, b.ctx):
        key = np.arange(int(n))
        rest[np.asarray(t)[key // 16], :, key % 16] = False
    assert np.array_equal(got[rest], case.mass[rest])  # keys of no sequence stay as they were
    if decay == 0.0:  # nothing of the old values, NaNs among them
        nan = case.run(lia, 0.0, mass=np.full_like(case.mass, np.nan))
        assert np.array_equal(nan[~rest], got[~rest]) and np.isnan(nan[rest]).all()


def test_nans_stay_with_their_rows(lia, wl):
    """A NaN key makes the weights of the rows that attend it NaN and leaves earlier rows' alone."""
    b = wl.custom([90, 200, 150], [4, 1, 100], geom=wl.Geometry(16, 2, 128, 16), seed=13)
    case = Case(b, FP4, seed=14)
    for s, key, h in ((0, 87, 0), (1, 3, 1), (2, 120, 0)):
        case.scales[b.tables[s][key // 16], h, key % 16, 2] = 255
    case.k = M.dequantise(case.codes, case.scales)
    ref, _, _ = case.reference()
    assert np.isnan(ref).any()
    case.check(lia, "NaN keys")
    case = Case(b, FP8, seed=14)
    for s, key, h in ((0, 87, 0), (1, 3, 1), (2, 120, 0)):
        at = (b.tables[s][key // 16], key % 16, h, 77)
        case.store[at] = 0xFF
        case.k[at[0], h, at[1], 77] = np.nan
    case.check(lia, "NaN keys, FP8")


def test_pages_outside_the_pool(lia, wl):
    b = wl.custom([200, 100], [1, 70], geom=wl.Geometry(16, 2, 128, 16), seed=15)
    case = Case(b, BF16, seed=16)
    case.flat = case.flat.copy()
    case.flat[3], case.flat[b.stride + 1] = b.pool_pages, 0xFFFFFFFF
    case.check(lia, "pages outside")


def test_capacity_and_stream(lia, wl):
    """A larger configuration, on a stream of its own; and a step over its configuration's room does nothing."""
    b = wl.custom([400, 90], [1, 3], geom=wl.Geometry(16, 2, 128, 16), seed=17)
    case = Case(b, FP4, seed=18)
    want = case.run(lia)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    print("[case] weights on a stream", flush=True)
    with torch.cuda.stream(s):
        got = case.run(lia, max_seqs=50, max_rows=4096)
    assert np.array_equal(got, want)


def test_captured(lia, wl):
    """Captured once and replayed with other queries: each replay against the eager call."""
    b = wl.custom([900, 90], [1, 40], geom=wl.Geometry(16, 2, 128, 16), seed=19)
    case = Case(b, FP4, seed=20)
    cfg = case.config(lia)
    ws = [torch.zeros(lia.attention_weights_workspace_bytes(cfg), dtype=torch.uint8, device="cuda") for _ in range(2)]
    mass = [torch.from_numpy(case.mass).cuda() for _ in range(2)]
    q = torch.from_numpy(case.q).to(torch.bfloat16).cuda()
    kc, ks = case.store.cuda(), torch.from_numpy(case.scales).cuda()
    meta = [G.u32_dev(x) for x in (b.cu_seqlens(), b.positions(), b.sequences(), case.flat)]
    print("[case] weights captured", flush=True)

    def step(i):
        lia.attention_weights(cfg, 2, *meta, q, kc, mass[i], ws[i], k_scales=ks, decay=0.9)
    step(0)
    step(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(0)
    for i in range(3):
        q.normal_(generator=torch.Generator(device="cuda").manual_seed(i))
        graph.replay()
        torch.cuda.synchronize()
        step(1)
        torch.cuda.synchronize()
        assert torch.equal(mass[0].view(torch.int32), mass[1].view(torch.int32)), i
