"""MXFP4 pools on the GPU: the append and the gather bit for bit against the oracle, attention of every kind
against 64 bits within a bound derived beside it (fp4_data.py), page transfers and the engine."""
import numpy as np
import pytest
import torch

import gpu_data as G
from fp4_data import BF16, F16, F32, FP4, FP8, Fp4Case, bf16_round
from oracle import mxfp4 as M

pytestmark = pytest.mark.gpu

SRC = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}


def _rows(rng, rows, hkv, d, src):
    """Rows with blocks of every kind: ordinary, ties, zero, tiny, huge, NaN and infinite."""
    x = rng.standard_normal((rows, hkv, d)).astype(np.float32)
    b = x.reshape(-1, 32)
    for i in range(len(b)):
        kind = i % 11
        if kind == 1:
            b[i] = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, -0.25, -5.0], 32)
        elif kind == 2:
            b[i] = 0.0
        elif kind == 3:
            b[i] *= 2.0 ** -140 if src == F32 else 2.0 ** -22
        elif kind == 4:
            b[i] *= 1e37 if src != F16 else 1e4
        elif kind == 5 and i % 2:
            b[i, i % 32] = [np.nan, np.inf, -np.inf][i % 3]
        elif kind == 6:
            b[i] *= rng.choice([1.0, 2.0 ** -10], 32)
        elif kind == 7:
            b[i] = -0.0
    t = torch.from_numpy(x).to(SRC[src])
    return t, t.float().numpy()


@pytest.mark.parametrize("rows,hkv,d,page,src", [
    (1, 2, 128, 16, BF16), (3, 1, 64, 16, F32), (17, 2, 128, 32, F16), (64, 8, 128, 16, BF16), (257, 3, 64, 64, BF16),
    (130, 8, 128, 32, F32), (33, 2, 96, 16, F32), (65, 5, 32, 16, F16),
])
@pytest.mark.parametrize("by", ["slots", "tables"])
def test_append_and_gather_bit_exact(lia, rows, hkv, d, page, src, by):
    rng = np.random.default_rng(rows + d + src)
    pool_pages = -(-rows // page) + 4
    stride = pool_pages
    table = rng.permutation(pool_pages).astype(np.uint32)
    positions = np.sort(rng.choice(pool_pages * page, rows, replace=False)).astype(np.uint32)
    slots = table[positions // page] * page + positions % page
    lost = np.zeros(rows, bool)
    if by == "slots" and rows > 2:  # a row without a slot, and one outside the pool
        slots = slots.astype(np.uint32)
        slots[1], slots[rows // 2] = 0xFFFFFFFF, pool_pages * page + 3
        lost[[1, rows // 2]] = True
    print(f"[case] fp4 append rows={rows} hkv={hkv} d={d} page={page} src={src} by={by}", flush=True)
    (k, kf), (v, vf) = _rows(rng, rows, hkv, d, src), _rows(rng, rows, hkv, d, src)
    shape = (pool_pages, hkv, page)
    planes = [rng.integers(0, 256, (*shape, w), dtype=np.uint8) for w in (d // 2, d // 2, d // 32, d // 32)]
    want = [x.copy() for x in planes]
    for c, s, x in ((0, 2, kf), (1, 3, vf)):
        codes, scales = M.quantise(x)
        for r in np.flatnonzero(~lost):
            at = (slots[r] // page, slice(None), slots[r] % page)
            want[c][at], want[s][at] = codes[r], scales[r]
    kc, vc, ks, vs = (torch.from_numpy(x).cuda() for x in planes)
    layout = lia.KVLayout(hkv, d, page, pool_pages, FP4)
    how = dict(slot_mapping=G.u32_dev(slots)) if by == "slots" else dict(
        positions=G.u32_dev(positions), sequences=G.u32_dev(np.zeros(rows)), pages=G.u32_dev(table), stride=stride)
    lia.kv_append(layout, k.cuda().reshape(rows, -1), v.cuda().reshape(rows, -1), kc, vc, k_scales=ks, v_scales=vs, **how)
    for got, ref, name in zip((kc, vc, ks, vs), want, ("k", "v", "k scales", "v scales")):
        got = got.cpu().numpy()
        bad = np.argwhere(got != ref)
        assert not len(bad), (name, bad[:4], got[tuple(bad[0])], ref[tuple(bad[0])])
    # and back: every type, the lost rows zeros
    for dt, t in SRC.items():
        ko, vo = (torch.full((rows + 1, hkv, d), 7.0, dtype=t, device="cuda") for _ in range(2))
        lia.kv_gather(layout, G.u32_dev(slots), kc, vc, ko, vo, k_scales=ks, v_scales=vs)
        for out, c, s in ((ko, 0, 2), (vo, 1, 3)):
            ref = np.zeros((rows, hkv, d))
            ok = ~lost
            ref[ok] = M.dequantise(want[c], want[s])[slots[ok] // page, :, slots[ok] % page]
            ref = torch.from_numpy(ref.astype(np.float32)).to(t)
            assert torch.equal(torch.nan_to_num(out[:rows].cpu(), nan=-7.0), torch.nan_to_num(ref, nan=-7.0)), (dt, c)
            assert (out[rows] == 7.0).all()


@pytest.mark.parametrize("kv", [F16, BF16, FP8])
@pytest.mark.parametrize("dst", [F32, F16, BF16])
def test_gather_of_the_other_pools(lia, O, kv, dst):
    rng = np.random.default_rng(kv * 10 + dst)
    hkv, d, page, pool_pages, rows = 3, 64, 16, 6, 41
    layout = lia.KVLayout(hkv, d, page, pool_pages, kv)
    x = rng.standard_normal((2, pool_pages * page, hkv, d)).astype(np.float32)
    scales = rng.uniform(0.5, 2, (2, pool_pages, hkv)).astype(np.float32)
    slots = rng.integers(0, pool_pages * page + 9, rows)
    print(f"[case] gather kv={kv} dst={dst}", flush=True)
    if kv == FP8:
        codes = torch.from_numpy(x * 20).to(torch.float8_e4m3fn)
        vals = codes.float() * torch.from_numpy(scales).repeat_interleave(page, 1)[..., None]
        planes = codes.view(torch.uint8)
    else:
        planes = torch.from_numpy(x).to(SRC[kv])
        vals = planes.float()
    ko, vo = (torch.full((rows, hkv, d), 7.0, dtype=SRC[dst], device="cuda") for _ in range(2))
    pc = planes.cuda()
    sc = torch.from_numpy(scales).cuda()
    lia.kv_gather(layout, G.u32_dev(slots), pc[0], pc[1], ko, vo, k_scales=sc[0] if kv == FP8 else None,
                  v_scales=sc[1] if kv == FP8 else None)
    inside = slots < pool_pages * page
    for got, i in ((ko, 0), (vo, 1)):
        want = torch.zeros((rows, hkv, d))
        want[torch.from_numpy(inside)] = vals[i][torch.from_numpy(slots[inside])]
        assert torch.equal(got.cpu(), want.to(SRC[dst]))


@pytest.mark.parametrize("hq,hkv,d,qdt", [(16, 2, 128, F32), (8, 2, 64, BF16), (4, 4, 128, BF16)])
def test_rope_append(lia, O, hq, hkv, d, qdt):
    """The rotated rows that the f32 path gives, quantised by the oracle."""
    rng = np.random.default_rng(hq + d)
    rows, page, pool_pages = 21, 16, 4
    positions = np.sort(rng.choice(5000, rows, replace=False)).astype(np.uint32)
    slots = rng.permutation(pool_pages * page)[:rows].astype(np.uint32)
    slots[5] = 0xFFFFFFFF
    combined = rng.uniform(-4, 4, (rows, (hq + 2 * hkv) * d)).astype(np.float32)
    combined[3, hq * d + 7] = np.nan       # a block of row 3's first key
    combined[4, (hq + hkv) * d + 40] = np.inf
    coeffs = O.rope_coefficients(positions, d)
    print(f"[case] fp4 rope append hq={hq} d={d} q={qdt}", flush=True)
    # the rotation in f64: one rounding of the product, one of the sum (as the kernel's fma)
    x = combined.reshape(rows, hq + 2 * hkv, d)
    cs = coeffs.reshape(rows, 1, d // 2, 2)
    a, b = x[..., :d // 2].astype(np.float64), x[..., d // 2:].astype(np.float64)
    c, s = cs[..., 0].astype(np.float64), cs[..., 1].astype(np.float64)
    with np.errstate(invalid="ignore"):
        lo = (a * c - (b * s).astype(np.float32)).astype(np.float32)
        hi = (b * c + (a * s).astype(np.float32)).astype(np.float32)
    rot = np.concatenate([lo, hi], -1)
    shape = (pool_pages, hkv, page)
    kc, vc = (torch.zeros((*shape, d // 2), dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((*shape, d // 32), 9, dtype=torch.uint8, device="cuda") for _ in range(2))
    query = torch.empty((rows, hq, d), dtype=torch.float32 if qdt == F32 else torch.bfloat16, device="cuda")
    layout = lia.KVLayout(hkv, d, page, pool_pages, FP4)
    lia.rope_kv_append(layout, hq, torch.from_numpy(coeffs.reshape(-1)).cuda(), torch.from_numpy(combined).cuda(),
                       query, kc, vc, slot_mapping=G.u32_dev(slots), k_scales=ks, v_scales=vs)
    for got, sc, heads in ((kc, ks, rot[:, hq:hq + hkv]), (vc, vs, x[:, hq + hkv:])):
        codes, scales = M.quantise(heads)
        wc, wsc = np.zeros(got.shape, np.uint8), np.full(sc.shape, 9, np.uint8)
        for r in range(rows):
            if slots[r] != 0xFFFFFFFF:
                wc[slots[r] // page, :, slots[r] % page] = codes[r]
                wsc[slots[r] // page, :, slots[r] % page] = scales[r]
        assert np.array_equal(sc.cpu().numpy(), wsc) and np.array_equal(got.cpu().numpy(), wc)
    want = torch.from_numpy(rot[:, :hq].copy()).to(query.dtype)
    assert torch.equal(query.cpu(), want)


DECODE = {
    "lengths": [1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 511, 1000, 1025, 2049, 4100],
    "one": [1], "short": [23], "long": [70001], "pair": [9000, 3],
}


@pytest.mark.parametrize("kind", list(DECODE))
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 2, 128, 16), (8, 2, 64, 32), (8, 8, 128, 64), (5, 1, 64, 16)])
def test_decode(lia, wl, kind, hq, hkv, d, page):
    ctx = DECODE[kind] if hkv < 8 else [min(c, 9000) for c in DECODE[kind]]
    g = wl.Geometry(hq, hkv, d, page, FP4, BF16, F32 if d == 64 else BF16)
    b = wl.custom(ctx, [1] * len(ctx), geom=g, seed=1)
    Fp4Case(b, seed=2).check(lia, f"decode {kind} {hq}/{hkv}x{d} page {page}")


@pytest.mark.parametrize("ctx,q_len,hq,hkv,d,page,q,out", [
    ([40, 1200, 17, 5000, 300], [3, 1, 2, 4, 1], 16, 2, 128, 16, BF16, BF16),
    ([40, 1200, 17, 2500, 300], [3, 15, 2, 4, 1], 32, 8, 128, 16, BF16, F32),
    ([700, 33], [2, 5], 20, 1, 64, 32, F32, F32),           # a group of 20: two column tiles
    ([700, 4], [1, 1], 32, 1, 128, 16, BF16, BF16),         # a group of 32
    ([9, 5], [9, 5], 12, 4, 64, 16, F32, BF16),             # a group of 3, rows over their own keys
    ([100] * 30, [4] * 30, 16, 2, 128, 16, BF16, BF16),
])
def test_verify(lia, wl, ctx, q_len, hq, hkv, d, page, q, out):
    g = wl.Geometry(hq, hkv, d, page, FP4, q, out)
    b = wl.custom(ctx, q_len, geom=g, seed=3)
    Fp4Case(b, seed=4).check(lia, f"verify {hq}/{hkv}x{d} rows {b.n_rows}")


@pytest.mark.parametrize("ctx,q_len,hq,hkv,d,page,q,out", [
    ([300, 1077, 2040], [300, 77, 40], 16, 2, 128, 16, BF16, BF16),
    ([16, 33, 100], [16, 33, 100], 16, 2, 128, 16, BF16, F32),
    ([700, 1300], [65, 130], 32, 8, 128, 32, BF16, BF16),
    ([64, 3000, 129], [64, 200, 1], 8, 2, 64, 64, F32, F32),
    ([150, 40, 2000], [150, 40, 1], 32, 1, 64, 16, BF16, BF16),
    ([500, 1500], [500, 17], 6, 2, 64, 16, BF16, F32),
])
def test_prefill(lia, wl, ctx, q_len, hq, hkv, d, page, q, out):
    g = wl.Geometry(hq, hkv, d, page, FP4, q, out)
    b = wl.custom(ctx, q_len, geom=g, seed=5)
    Fp4Case(b, seed=6).check(lia, f"prefill {hq}/{hkv}x{d} rows {b.n_rows}")


def test_wide_scales(lia, wl):
    """Blocks up to 2^24 apart, one of the keys far ahead of the others."""
    g = wl.Geometry(16, 2, 128, 16, FP4, BF16, F32)
    for ctx, q_len in (([900, 77], [1, 1]), ([900, 77], [3, 2]), ([400, 200], [100, 50])):
        case = Fp4Case(wl.custom(ctx, q_len, geom=g, seed=7), seed=8, spread=1)
        rng = np.random.default_rng(9)
        case.vs[...] = (case.vs.astype(int) + rng.integers(-12, 13, case.vs.shape)).astype(np.uint8)
        case.check(lia, f"wide scales rows {case.batch.n_rows}")


@pytest.mark.parametrize("ctx,q_len", [([900, 77, 33], [1, 1, 1]), ([900, 77, 40], [3, 2, 8]), ([400, 90], [100, 50])])
@pytest.mark.parametrize("d", [64, 128])
def test_nans_reach_the_rows_that_attend_them(lia, wl, ctx, q_len, d):
    """NaN blocks of V (and of K) at keys that some rows attend and earlier rows do not, at dead slots and in pages
    that no table names."""
    g = wl.Geometry(16, 2, d, 16, FP4, BF16, BF16)
    b = wl.custom(ctx, q_len, geom=g, seed=11)
    for where in ("v", "k", "dead"):
        case = Fp4Case(b, seed=12)
        live = np.zeros((b.pool_pages, g.page_size), bool)
        for t, n in zip(b.tables, b.ctx):
            key = np.arange(int(n))
            live[np.asarray(t)[key // 16], key % 16] = True
        if where == "dead":
            for plane in (case.ks, case.vs):
                plane.transpose(0, 2, 1, 3)[~live] = 255
        else:
            # of each sequence: the last key's first block in head 0, and the third last's last block in head 1
            plane = case.vs if where == "v" else case.ks
            for t, n in zip(b.tables, b.ctx):
                for key, h, blk in ((int(n) - 1, 0, 0), (int(n) - 3, 1, d // 32 - 1)):
                    plane[t[key // 16], h, key % 16, blk] = 255
        ref, _ = case.reference()
        assert np.isnan(ref).any() == (where != "dead")
        assert not np.isnan(ref).all() or (where == "k" and b.n_rows == 3)  # (a key's NaN is its rows' whole answer)
        case.check(lia, f"NaN {where} d={d} rows {b.n_rows}")


def test_pages_outside_the_pool_read_as_zeros(lia, wl):
    g = wl.Geometry(16, 2, 128, 16, FP4, BF16, BF16)
    for ctx, q_len in (([200, 100], [1, 1]), ([200, 100], [3, 2]), ([200, 100], [64, 32])):
        b = wl.custom(ctx, q_len, geom=g, seed=13)
        case = Fp4Case(b, seed=14)
        case.flat = case.flat.copy()
        case.flat[3], case.flat[b.stride + 1] = b.pool_pages, 0xFFFFFFFE
        case.check(lia, f"pages outside rows {b.n_rows}")


def test_rows_behind_the_batch_are_left(lia, wl):
    """A configuration for more rows and sequences than the step has; the output's other rows are untouched."""
    g = wl.Geometry(16, 2, 128, 16, FP4, BF16, BF16)
    b = wl.custom([300, 50, 1200], [1, 1, 1], geom=g, seed=15)
    case, dev = Fp4Case(b, seed=16), None
    dev = case.device()
    cfg = case.config(lia, max_rows=256, max_seqs=40)
    out = torch.full((b.n_rows + 4, g.hq, g.d), 7.0, dtype=torch.bfloat16, device="cuda")
    print("[case] fp4 rows behind the batch", flush=True)
    lia.paged_attention(cfg, 3, dev["cu"], dev["positions"], dev["sequences"], dev["pages"], dev["q"], dev["kc"],
                        dev["vc"], out, G.dirty_workspace(lia, cfg), dev["ks"], dev["vs"])
    assert (out[3:] == 7.0).all()
    ref, bound = case.reference()
    assert (np.abs(out[:3].float().cpu().numpy() - ref) <= bound).all()


def test_stages_and_streams(lia, wl):
    """Plan once, then partial and merge of two layers on another stream; bit for bit the one call's output."""
    g = wl.Geometry(16, 2, 128, 16, FP4, BF16, BF16)
    b = wl.custom([900, 4100, 30], [1, 1, 1], geom=g, seed=17)
    cases = [Fp4Case(b, seed=s) for s in (18, 19)]
    devs = [c.device() for c in cases]
    want = [c.run(lia, d) for c, d in zip(cases, devs)]
    cfg = cases[0].config(lia)
    ws = G.dirty_workspace(lia, cfg)
    print("[case] fp4 stages on another stream", flush=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = [torch.full_like(w, 7.0) for w in want]
    with torch.cuda.stream(s):
        d = devs[0]
        lia.attention_plan(cfg, 3, 3, d["cu"], d["positions"], d["sequences"], ws, d["pages"])
        for d, out in zip(devs, outs):
            lia.attention_partial(cfg, 3, d["pages"], d["q"], d["kc"], d["vc"], out, ws, d["ks"], d["vs"])
            lia.attention_merge(cfg, 3, 3, out, ws)
    s.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o.view(torch.int16), w.view(torch.int16))


def test_captured_step(lia, wl):
    """Append and attention captured once, replayed over a growing context, each replay against the eager call."""
    g = wl.Geometry(16, 2, 128, 16, FP4, BF16, BF16)
    b = wl.custom([700, 90], [1, 1], geom=g, seed=20)
    case = Fp4Case(b, seed=21)
    d = case.device()
    layout = lia.KVLayout(g.hkv, g.d, 16, b.pool_pages, FP4)
    cfg = case.config(lia)
    ws = G.dirty_workspace(lia, cfg)
    out = torch.zeros((2, g.hq, g.d), dtype=torch.bfloat16, device="cuda")
    nk, nv = (torch.zeros((2, g.hkv * g.d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = G.u32_dev(np.zeros(2))
    print("[case] fp4 captured step", flush=True)

    def step(o, w):
        lia.kv_append(layout, nk, nv, d["kc"], d["vc"], slot_mapping=slots, k_scales=d["ks"], v_scales=d["vs"])
        lia.paged_attention(cfg, 2, d["cu"], d["positions"], d["sequences"], d["pages"], d["q"], d["kc"], d["vc"], o, w,
                            d["ks"], d["vs"])
    slots.copy_(G.u32_dev(b.slot_mapping()))
    step(out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, ws)
    rng = torch.Generator(device="cuda").manual_seed(3)
    for i in range(4):
        back = 3 - i  # shorter contexts of the same tables first
        pos = case.positions.astype(np.int64) - back
        d["positions"].copy_(G.u32_dev(pos))
        page = case.flat.reshape(2, -1)[np.arange(2), pos // 16].astype(np.int64)
        slots.copy_(G.u32_dev(page * 16 + pos % 16))
        nk.copy_(torch.randn(nk.shape, generator=rng, device="cuda"))
        nv.copy_(torch.randn(nv.shape, generator=rng, device="cuda"))
        d["q"].copy_(torch.randn(d["q"].shape, generator=rng, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = torch.zeros_like(out)
        step(eager, G.dirty_workspace(lia, cfg))
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), eager.view(torch.int16)), i


def test_pages_travel(lia):
    """Download, upload to other pages and back: codes and scales byte for byte."""
    rng = np.random.default_rng(22)
    hkv, d, page, pool, layers = 2, 128, 32, 9, 3
    mk = lambda w: [torch.from_numpy(rng.integers(0, 256, (pool, hkv, page, w), dtype=np.uint8)).cuda() for _ in range(layers)]  # noqa: E731
    k, v, ks, vs = mk(d // 2), mk(d // 2), mk(d // 32), mk(d // 32)
    t = lia.KVTransfer(lia.KVLayout(hkv, d, page, pool, FP4), k, v, ks, vs)
    print("[case] fp4 page transfer", flush=True)
    before = [[x.clone() for x in planes] for planes in (k, v, ks, vs)]
    got = t.read_kv_pages([4, 1, 7])
    want = b"".join(x[i][4].cpu().numpy().tobytes() for i in range(layers) for x in (k, v))
    want += b"".join(x[i][4].cpu().numpy().tobytes() for i in range(layers) for x in (ks, vs))
    assert bytes(got[0]) == want
    t.write_kv_pages([(0, got[0]), (8, got[1])])
    for planes, old in zip((k, v, ks, vs), before):
        for x, o in zip(planes, old):
            o[0], o[8] = o[4], o[1]
            assert torch.equal(x, o)


def test_engine(lia):
    """The engine on an MXFP4 pool: a prompt, then decode steps, against 64 bits on what its pool holds."""
    rng = np.random.default_rng(23)
    hq, hkv, d, page = 16, 2, 128, 32
    e = lia.Engine(hq, hkv, d, pool_tokens=page * 40, layers=2, page_size=page, kv_dtype=FP4, prefill_batch=256)
    e.configure_paging(4, 1024)
    table, done = [7, 3, 30, 12, 9], 0
    print("[case] fp4 engine", flush=True)
    for rows in (100, 1, 1, 3, 1):
        e.stage([(1, done + i, 0) for i in range(rows)], [table], [rows - 1])
        for layer in range(2):
            q = torch.from_numpy(rng.standard_normal((rows, hq, d)).astype(np.float32)).cuda()
            k, v = (torch.from_numpy(rng.standard_normal((rows, hkv * d)).astype(np.float32)).cuda() for _ in range(2))
            out = e.attention(layer, q, k, v).cpu().numpy()
            codes, scales = M.quantise(k.cpu().numpy().reshape(rows, hkv, d))
            for i in range(rows):
                at = (table[(done + i) // page], slice(None), (done + i) % page)
                assert np.array_equal(e.k[layer].cpu().numpy()[at], codes[i])
                assert np.array_equal(e.k_scales[layer].cpu().numpy()[at], scales[i])
            n = done + rows
            kk, vv = (M.keys_of(M.dequantise(x.cpu().numpy(), s.cpu().numpy()), table, n, page)
                      for x, s in ((e.k[layer], e.k_scales[layer]), (e.v[layer], e.v_scales[layer])))
            q16 = bf16_round(q.cpu().numpy())
            ref = M.attention(q16, kk, vv, done, e.scale)
            bound = M.attention(q16, kk, np.abs(vv), done, e.scale) * 2.5 * 2.0 ** -8  # (fp4_data.py's, f32 outputs)
            assert (np.abs(out - ref) <= bound).all()
        done += rows
    payload = e.read_kv_page(3)
    e.write_kv_page(5, bytes(payload))
    assert torch.equal(e.k[1][5], e.k[1][3]) and torch.equal(e.v_scales[0][5], e.v_scales[0][3])
