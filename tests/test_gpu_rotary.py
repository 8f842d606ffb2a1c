"""Rotation tables from given frequencies, and rows normalised, rotated and appended, against 64 bits; bit for bit against
the calls whose work they share."""
import numpy as np
import pytest
import torch

import gpu_data as G
from oracle import sparse as S

pytestmark = pytest.mark.gpu

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # half a step, relative


@pytest.mark.parametrize("rows,n", [(1, 4), (1, 128), (7, 64), (63, 80), (1000, 96), (4097, 128)])
@pytest.mark.parametrize("attention", [1.0, 1.2079])
def test_table(lia, rows, n, attention):
    print(f"[case] table rows={rows} n={n}", flush=True)
    rng = np.random.default_rng(rows)
    f = lia.rope_frequencies(n, 1e6, "turns", factor=8.0, context=4096)
    f[0] = 1.0
    positions = rng.integers(0, 1 << 20, rows).astype(np.uint32)
    positions[:4] = [0, 131071, 1, 0xFFFFFFFF][:min(rows, 4)]
    out = torch.full((rows + 1, n // 2, 2), 7.0, device="cuda")
    lia.rope_table(G.u32_dev(positions), torch.from_numpy(f).cuda(), out, attention=attention)
    got = out.cpu().numpy()
    angle = positions.astype(np.float64)[:, None] * f
    ref = np.stack([np.cos(angle), np.sin(angle)], -1) * attention
    # the reduced angle and its series are good to 2^-24 and less than an ulp of 1 in the sums behind (2 . 2^-24), the factor
    # and the product are rounded (2 . 2^-24); an angle of 2^32 is itself a product rounded to 2^-53 of it, 2^-21
    far = positions.astype(np.float64)[:, None, None] * 2.0 ** -53
    assert (np.abs(got[:rows] - ref) <= attention * (5 * 2.0 ** -24 + far)).all()
    assert (got[rows:] == 7.0).all()


def test_table_of_quadrants(lia):
    """Angles next to multiples of pi / 4, where the reduction changes sides."""
    at = np.arange(0, 64)
    f = np.array([np.pi / 4, np.nextafter(np.pi / 4, 0), np.nextafter(np.pi / 4, 1), np.pi / 2])
    out = torch.empty((64, 4, 2), device="cuda")
    lia.rope_table(G.u32_dev(at), torch.from_numpy(f).cuda(), out)
    angle = at[:, None] * f
    assert np.abs(out.cpu().numpy() - np.stack([np.cos(angle), np.sin(angle)], -1)).max() <= 5 * 2.0 ** -24


class Rows:
    """A step's projections on a pool of scattered pages, every row with a slot but some."""

    def __init__(self, lia, rows, hq, hkv, d, page, kv, src, n, pad=0, seed=0, scale=1.0):
        rng = np.random.default_rng(seed + rows)
        self.rows, self.hq, self.hkv, self.d, self.page, self.kv = rows, hq, hkv, d, page, kv
        self.pool_pages = -(-rows // page) + 3
        self.layout = lia.KVLayout(hkv, d, page, self.pool_pages, kv)
        slots = rng.permutation(self.pool_pages * page)[:rows].astype(np.uint32)
        self.slots = slots
        width = (hq + 2 * hkv) * d
        wide = np.exp(rng.standard_normal(width))
        x = (scale * wide * rng.standard_normal((rows, width))).astype(np.float32)
        self.buffer = torch.full((rows, width + pad), 3.0e4, device="cuda", dtype=TORCH[src])
        self.x = self.buffer[:, :width]
        self.x.copy_(torch.from_numpy(x))
        angle = rng.uniform(0, 6.3, (rows, n // 2))
        self.table = (1.1 * np.stack([np.cos(angle), np.sin(angle)], -1)).astype(np.float32)
        self.wq, self.wk = (torch.from_numpy((1 + 0.3 * rng.standard_normal(d)).astype(np.float32)).cuda() for _ in range(2))
        if kv == FP4:
            shape, sshape, fill = (self.pool_pages, hkv, page, d // 2), (self.pool_pages, hkv, page, d // 32), torch.uint8
            self.ks, self.vs = (torch.full(sshape, 127, dtype=fill, device="cuda") for _ in range(2))
        else:
            shape, fill = (self.pool_pages, page, hkv, d), torch.uint8 if kv == FP8 else TORCH[kv]
            self.ks = self.vs = None
            if kv == FP8:
                s = rng.uniform(0.005, 0.05, (2, self.pool_pages, hkv)).astype(np.float32)
                s[:, rng.random(self.pool_pages) < 0.3] = 0.0  # pages never quantised
                self.ks, self.vs = torch.from_numpy(s[0]).cuda(), torch.from_numpy(s[1]).cuda()
        self.kc, self.vc = (torch.full(shape, 1, dtype=fill, device="cuda") for _ in range(2))

    def run(self, lia, q=BF16, interleaved=False, wq=None, wk=None, eps=1e-6, n=None, **more):
        query = torch.full((self.rows, self.hq, self.d), float("nan"), dtype=TORCH[q], device="cuda")
        table = G.to_dev(self.table) if self.table.shape[1] else None
        a = dict(slot_mapping=G.u32_dev(self.slots))
        a.update(more)
        lia.qk_norm_rope_kv_append(self.layout, self.hq, table, self.x, query, self.kc, self.vc, q_weight=wq, k_weight=wk,
                                   eps=eps, interleaved=interleaved, k_scales=self.ks, v_scales=self.vs, **a)
        return query

    def exact(self, interleaved, wq, wk, eps):
        """(value, bound of the f32 steps' error) of queries, keys and values."""
        x = self.x.double().cpu().numpy().reshape(self.rows, -1, self.d)
        parts = x[:, :self.hq], x[:, self.hq:self.hq + self.hkv]
        out = []
        for y, w in zip(parts, (wq, wk)):
            # the mean of d squares (d 2^-24 of it, half of that in its root), root, quotient and two products: below
            # (d / 2 + 6) 2^-24 of each normalised element, then a rotation of two roundings more
            steps = 3
            if w is not None:
                y = S.normalised(y, w.double().cpu().numpy(), eps)
                steps += self.d / 2 + 6
            value, size = S.rotated(y, self.table, interleaved)
            out.append((value, size * steps * 2.0 ** -24))
        return (*out, (x[:, self.hq + self.hkv:], 0.0))

    def gathered(self, lia):
        ko, vo = (torch.empty((self.rows, self.hkv, self.d), device="cuda") for _ in range(2))
        lia.kv_gather(self.layout, G.u32_dev(self.slots), self.kc, self.vc, ko, vo, k_scales=self.ks, v_scales=self.vs)
        return ko.double().cpu().numpy(), vo.double().cpu().numpy()

    def pool_error(self, value, scales):
        """Half a step of the pool's type at each value."""
        size = np.abs(value)
        if self.kv in (F16, BF16):
            return size * HALF[self.kv] + 2.0 ** -25  # (f16's subnormals)
        if self.kv == FP8:
            s = scales.cpu().numpy()[self.slots // self.page]
            s = np.where(s == 0, 1.0, s)[..., None]
            return np.where(size > 448 * s, size - 448 * s, 0) + size * 2.0 ** -4 + s * 2.0 ** -10
        # E2M1 values are a quarter of a value apart to either side from 2 on, half a unit below, and 6 stands for up to 8: a
        # quarter of the value or of the block's unit, whose largest magnitude rounded up may double it
        b = size.reshape(*size.shape[:-1], -1, 32)
        unit = 2.0 ** (np.floor(np.log2(b.max(-1, keepdims=True) * (1 + 2.0 ** -16) + 1e-300)) - 2)
        return np.maximum(b, unit).reshape(size.shape) / 4

    def check(self, lia, label, q=BF16, interleaved=False, wq=None, wk=None, eps=1e-6):
        print(f"[case] rotate {label}", flush=True)
        query = self.run(lia, q, interleaved, wq, wk, eps).double().cpu().numpy()
        (qr, qe), (kr, ke), (vr, ve) = self.exact(interleaved, wq, wk, eps)
        assert (np.abs(query - qr) <= (qe + np.abs(qr) * HALF[q]) * (1 + 2.0 ** -7) + 1e-38).all()
        k, v = self.gathered(lia)
        assert (np.abs(k - kr) <= (ke + self.pool_error(kr, self.ks)) * (1 + 2.0 ** -3 * (self.kv == FP8) + 2.0 ** -7)).all()
        assert (np.abs(v - vr) <= self.pool_error(vr, self.vs) * (1 + 2.0 ** -7) + ve).all()
        # other slots as they were
        taken = np.zeros(self.pool_pages * self.page, bool)
        taken[self.slots] = True
        for plane in (self.kc, self.vc):
            x = plane.float().cpu().numpy()
            if self.kv == FP4:
                x = x.transpose(0, 2, 1, 3)
            assert (x.reshape(len(taken), -1)[~taken] == 1).all()


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("src", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types(lia, kv, src, interleaved):
    for rows, d, n, pad in ((1, 64, 64, 0), (37, 128, 128, 8), (90, 64, 16, 0), (5, 128, 48, 1024)):
        r = Rows(lia, rows, 6, 2, d, 16, kv, src, n, pad, scale=0.5)
        r.check(lia, f"kv={kv} src={src} rows={rows} d={d} n={n}", F32 if rows == 37 else BF16, interleaved, r.wq, r.wk)


@pytest.mark.parametrize("rows,hq,hkv,d,page,n", [(1, 1, 1, 64, 16, 32), (3, 5, 5, 128, 64, 96), (513, 32, 8, 128, 32, 64),
                                                  (2, 64, 1, 64, 16, 48), (300, 24, 2, 128, 128, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_shapes(lia, rows, hq, hkv, d, page, n, interleaved):
    r = Rows(lia, rows, hq, hkv, d, page, BF16, BF16, n, seed=3)
    r.check(lia, f"rows={rows} hq={hq} hkv={hkv} d={d} n={n}", F32, interleaved, r.wq, r.wk)
    r = Rows(lia, rows, hq, hkv, d, page, BF16, BF16, n, seed=4)
    r.check(lia, f"keys' norm alone rows={rows}", BF16, interleaved, None, r.wk)
    r = Rows(lia, rows, hq, hkv, d, page, BF16, BF16, n, seed=5)
    r.check(lia, f"queries' norm alone rows={rows}", BF16, interleaved, r.wq, None, eps=0.25)


@pytest.mark.parametrize("wt", [F32, F16, BF16])
def test_weight_types_and_zeros(lia, wt):
    r = Rows(lia, 9, 4, 2, 128, 16, BF16, F32, 64, seed=6)
    r.x[2] = 0.0   # a head of zeros stays zeros
    r.x[3] *= 1e-18
    r.wq, r.wk = r.wq.to(TORCH[wt]), r.wk.to(TORCH[wt])
    r.check(lia, f"weights of type {wt}", F32, False, r.wq, r.wk)


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("src", [F32, F16, BF16])
def test_rows_that_pass_are_appended_as_ever(lia, kv, src):
    """No norm, no rotation: the pool and the queries are kv_append's and the input's."""
    r = Rows(lia, 77, 4, 2, 64, 16, kv, src, 0, seed=7)
    k, v = (t.clone() for t in (r.kc, r.vc))
    ks, vs = (None if t is None else t.clone() for t in (r.ks, r.vs))
    query = r.run(lia, F32)
    assert torch.equal(query, r.x[:, :4 * 64].float().reshape(query.shape))
    new = r.x.reshape(77, -1, 64)
    lia.kv_append(r.layout, new[:, 4:6].contiguous(), new[:, 6:].contiguous(), k, v, slot_mapping=G.u32_dev(r.slots),
                  k_scales=ks, v_scales=vs)
    assert torch.equal(r.kc.view(torch.uint8), k.view(torch.uint8)) and torch.equal(r.vc.view(torch.uint8), v.view(torch.uint8))
    if ks is not None:
        assert torch.equal(r.ks, ks) and torch.equal(r.vs, vs)


@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
@pytest.mark.parametrize("d", [64, 128])
def test_whole_heads_by_halves_are_rope_kv_appends(lia, kv, d):
    r = Rows(lia, 50, 8, 2, d, 32, kv, F32, d, seed=8)
    k, v = (t.clone() for t in (r.kc, r.vc))
    ks, vs = (None if t is None else t.clone() for t in (r.ks, r.vs))
    query, ref = r.run(lia, BF16), torch.empty((50, 8, d), dtype=torch.bfloat16, device="cuda")
    lia.rope_kv_append(r.layout, 8, G.to_dev(r.table), r.x, ref, k, v, slot_mapping=G.u32_dev(r.slots), k_scales=ks, v_scales=vs)
    assert torch.equal(query, ref)
    assert torch.equal(r.kc.view(torch.uint8), k.view(torch.uint8)) and torch.equal(r.vc.view(torch.uint8), v.view(torch.uint8))


def test_slots_from_tables_and_rows_without_one(lia):
    """Positions and tables in the place of slots; pages outside the pool and no slot leave the pool alone."""
    r = Rows(lia, 40, 4, 2, 64, 16, BF16, BF16, 32, seed=9)
    table = np.full((3, 4), 0xFFFFFFFF, np.uint32)
    table[0, :2], table[2, :2] = [3, 1], [0, 99]
    sequences = np.repeat([0, 2], 20).astype(np.uint32)
    positions = np.tile(np.arange(5, 25), 2).astype(np.uint32)
    entry = table[sequences, positions // 16]
    held = entry < r.pool_pages
    r.slots = np.where(held, entry * 16 + positions % 16, 0xFFFFFFFF).astype(np.uint32)
    one = r.run(lia)
    k, v = r.kc.clone(), r.vc.clone()
    r.kc.fill_(1), r.vc.fill_(1)
    two = r.run(lia, slot_mapping=None, positions=G.u32_dev(positions), sequences=G.u32_dev(sequences),
                pages=G.u32_dev(table.reshape(-1)), stride=4)
    assert torch.equal(one, two) and torch.equal(r.kc, k) and torch.equal(r.vc, v)
    assert not torch.isnan(one).any()
    taken = np.unique(r.slots[held])
    rest = np.setdiff1d(np.arange(r.pool_pages * 16), taken)
    assert (k.view(-1, 2 * 64)[torch.from_numpy(rest).cuda()] == 1).all() and 0 < held.sum() < 40


def test_nan_and_infinity_stay_in_their_head(lia):
    r = Rows(lia, 4, 4, 2, 64, 16, BF16, F32, 64, seed=10)
    r.x[1, 2 * 64 + 5] = float("nan")     # query head 2
    r.x[2, 4 * 64 + 7] = float("inf")     # key head 0
    query = r.run(lia, BF16, False, r.wq, r.wk)
    bad = torch.isnan(query).any(-1).nonzero().tolist()
    assert bad == [[1, 2]] and torch.isnan(query[1, 2]).all()
    k, v = r.gathered(lia)
    assert np.argwhere(np.isnan(k)).tolist() == [[2, 0, 7], [2, 0, 39]] and np.isfinite(v).all()
    rest = np.delete(k[2, 0], [7, 39])
    assert (rest == 0).all()


def test_planes_past_four_gib(lia):
    """Slots whose elements lie past 2^32 bytes into the planes, rows that lie past it in the input."""
    d, hkv, page = 128, 8, 32
    pages = (5 << 30) // (page * hkv * d * 2)
    layout = lia.KVLayout(hkv, d, page, pages, BF16)
    kc, vc = (torch.empty((pages * page, hkv, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    rows, stride = 3, 3 << 28
    width = (1 + 2 * hkv) * d
    buffer = torch.empty((rows - 1) * stride + width, dtype=torch.bfloat16, device="cuda")
    x = buffer.as_strided((rows, width), (stride, 1))
    x.copy_(torch.randn(rows, width, device="cuda"))
    slots = np.array([0, pages * page - 1, (pages - 2) * page + 5], np.uint32)
    query = torch.empty((rows, 1, d), dtype=torch.bfloat16, device="cuda")
    print("[case] planes past 4 GiB", flush=True)
    lia.qk_norm_rope_kv_append(layout, 1, None, x, query, kc, vc, slot_mapping=G.u32_dev(slots))
    at = torch.from_numpy(slots.astype(np.int64)).cuda()
    assert torch.equal(kc[at].reshape(rows, -1), x[:, d:(1 + hkv) * d]) and torch.equal(query[:, 0], x[:, :d])
    assert torch.equal(vc[at].reshape(rows, -1), x[:, (1 + hkv) * d:])
