"""A ragged batch over a pool of any type for the GPU tests of page summaries, selection and attention over selected pages:
seeded values, the device tensors, and the oracle's results in 64 bits."""
import numpy as np
import torch

import gpu_data as G
from fp4_data import bf16_round
from oracle import mxfp4 as M
from oracle import sparse as S

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4
NONE = 0xFFFFFFFF


class Pool:
    """K and V planes on the device and their values [page][page_size][kv head][d] in 64 bits."""

    def __init__(self, rng, pages, page, hkv, d, kv, key_size=1.0):
        self.pages, self.page, self.hkv, self.d, self.kv = pages, page, hkv, d, kv
        self.kc, self.ks, self.k = self._plane(rng, key_size)
        self.vc, self.vs, self.v = self._plane(rng, 1.0)

    def _plane(self, rng, size):
        wide = size * np.exp(0.5 * rng.standard_normal((self.hkv, self.d)))
        x = (rng.standard_normal((self.pages, self.page, self.hkv, self.d)) * wide).astype(np.float32)
        if self.kv == FP4:
            codes, scales = M.quantise(x.transpose(0, 2, 1, 3))
            return G.to_dev(codes), G.to_dev(scales), M.dequantise(codes, scales).transpose(0, 2, 1, 3)
        if self.kv == FP8:
            s = (np.abs(x).max((1, 3)) / 448).astype(np.float32)
            t = torch.from_numpy(x / s[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
            return t.view(torch.uint8).cuda(), G.to_dev(s), t.double().numpy() * s[:, None, :, None].astype(np.float64)
        t = torch.from_numpy(x).to(torch.float16 if self.kv == F16 else torch.bfloat16)
        return t.cuda(), None, t.double().numpy()

    def layout(self, lia):
        return lia.KVLayout(self.hkv, self.d, self.page, self.pages, self.kv)

    def summaries(self):
        """Oracle summaries of every page."""
        got = [S.summary(np.asarray(self.k[p], np.float32).transpose(1, 0, 2)) for p in range(self.pages)]
        return np.stack([c for c, _ in got]), np.stack([s for _, s in got])


class Batch:
    """new and cached rows of sequences; table rows are permuted, so that a sequence's is not its number."""

    def __init__(self, new, cached, page, seed=0, slack=3, stride=None):
        rng = np.random.default_rng(seed)
        new, cached = np.asarray(new), np.asarray(cached)
        self.n, self.rows, self.page = len(new), int(new.sum()), page
        ctx = new + cached
        need = -(-ctx // page)
        self.pool_pages, self.max_context = int(need.sum()) + slack, int(ctx.max())
        perm = rng.permutation(self.pool_pages).astype(np.uint32)
        self.stride = stride or int(need.max()) + 1
        self.table = np.full((self.n + 1, self.stride), NONE, np.uint32)
        at, self.row_of = 0, rng.permutation(self.n + 1)[:self.n]
        for s in range(self.n):
            self.table[self.row_of[s], :need[s]] = perm[at:at + need[s]]
            at += need[s]
        self.spare = perm[at:]
        self.sequences = np.repeat(self.row_of, new).astype(np.uint32)
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        self.positions = (np.arange(self.rows) - np.repeat(self.cu[:-1].astype(np.int64) - cached, new)).astype(np.uint32)

    def config(self, lia, hq, hkv, d, kv, q=BF16, out=BF16, scale=None, **more):
        a = dict(max_seqs=self.n, max_rows=max(self.rows, 1), max_context=self.max_context, pool_pages=self.pool_pages)
        a.update(more)
        return lia.AttentionConfig(hq, hkv, d, self.page, a["pool_pages"], self.stride, q, kv, out,
                                   scale or float(1 / np.sqrt(d)), a["max_seqs"], a["max_rows"], a["max_context"])

    def device(self):
        return dict(cu=G.u32_dev(self.cu), positions=G.u32_dev(self.positions), sequences=G.u32_dev(self.sequences),
                    pages=G.u32_dev(self.table.reshape(-1)))


def queries(rng, rows, hq, d, kind, size=1.5):
    """(device tensor, its values as f32)."""
    q = (size * rng.standard_normal((rows, hq, d))).astype(np.float32)
    if kind == BF16:
        q = bf16_round(q)
        return torch.from_numpy(q).to(torch.bfloat16).cuda(), q
    return torch.from_numpy(q).cuda(), q


def select(lia, b, cfg, dev, q, codes, scales, budget, first, recent, extra=0):
    """The call's selected pages and counts, with `extra` rows behind that have to stay as they were."""
    selected = torch.full((b.rows + extra, cfg.num_kv_heads, budget), 12345, dtype=torch.int32, device="cuda")
    counts = torch.full((b.rows + extra,), 54321, dtype=torch.int32, device="cuda")
    ws = torch.full((lia.page_select_workspace_bytes(cfg),), 0x7E, dtype=torch.uint8, device="cuda")
    lia.page_select(cfg, b.n, dev["cu"], dev["positions"], dev["sequences"], dev["pages"], q, codes, scales, first, recent,
                    selected, counts, ws)
    return selected.cpu().numpy().view(np.uint32), counts.cpu().numpy().view(np.uint32)


def expected(b, q, group, codes, scales, budget, first, recent, rows=None):
    """The oracle's selected pages and counts; codes and scales with an entry for pages outside the pool."""
    hkv = codes.shape[1]
    selected = np.full((b.rows, hkv, budget), NONE, np.uint32)
    counts = np.zeros(b.rows, np.uint32)
    for r in range(b.rows) if rows is None else rows:
        n = int(b.positions[r]) // b.page + 1
        entry = np.minimum(b.table[b.sequences[r], :n].astype(np.int64), len(codes) - 1)
        for h in range(hkv):
            score = S.scores(q[r, h * group:(h + 1) * group], codes[entry, h], scales[entry, h])
            keep = S.select(score, n, budget, first, recent)
            selected[r, h, :len(keep)] = keep
            counts[r] = len(keep)
    return selected, counts


def attend(lia, b, cfg, dev, q, pool, selected, counts, out_type=BF16, extra=0):
    out = torch.full((b.rows + extra, cfg.num_q_heads, cfg.head_dim), float("nan"), device="cuda",
                     dtype=torch.float32 if out_type == F32 else torch.bfloat16)
    ws = torch.full((lia.selected_attention_workspace_bytes(cfg, selected.shape[2]),), 0x7E, dtype=torch.uint8, device="cuda")
    lia.selected_attention(cfg, b.n, dev["cu"], dev["positions"], dev["sequences"], dev["pages"], q, pool.kc, pool.vc,
                           G.u32_dev(selected), G.u32_dev(counts), out, ws, pool.ks, pool.vs)
    return out


def reference(b, pool, q, group, selected, counts, scale, out_type=BF16):
    """(output, a bound of the kernel's error) in 64 bits."""
    rounded = torch.from_numpy(q).to(torch.float16 if pool.kv == F16 else torch.bfloat16).double().numpy()
    zeros = np.zeros((1, *pool.k.shape[1:]))
    k, v = np.concatenate([pool.k, zeros]), np.concatenate([pool.v, zeros])
    rows, hkv, budget = selected.shape
    out, size = np.zeros((rows, hkv * group, pool.d)), np.zeros((rows, hkv * group, pool.d))
    for r in range(rows):
        table = b.table[b.sequences[r]]
        for h in range(hkv):
            pages = [(int(p), min(int(table[p]), pool.pages)) for p in selected[r, h, :min(int(counts[r]), budget)]
                     if p < b.stride]
            heads = slice(h * group, (h + 1) * group)
            out[r, heads], size[r, heads] = S.attention(rounded[r, heads], k[:, :, h], v[:, :, h], pages, len(pages),
                                                        int(b.positions[r]), b.page, scale)
    # Each weight is rounded to the products' type above the fraction line and below it (FP8: times its page's scale above
    # it), half a step each; the output is rounded.  f32 sums of n terms, the exponentials' own error and the scores' (d
    # products: d 2^-24 of a score of up to about 60 in the log2 domain) stay below 2^-9 of the sum of magnitudes.  f16
    # weights below 2^-14 are subnormal: 2^-25 of each of up to 4,096 keys' largest value.
    step = 2.0 ** (-11 if pool.kv == F16 else -8)
    bound = size * (2 * step + (2.0 ** -8 if out_type == BF16 else 0) + 2.0 ** -9) + 1e-30
    if pool.kv == F16:
        bound += 2.0 ** -25 * 4096 * 2.0 ** -8 * np.abs(pool.v).max()
    return out, bound


def check(got, out, bound, label):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(out)), label
    far = np.nan_to_num(np.abs(got - out) / bound)
    print(f"[case] {label}: {far.max():.3f} of the bound", flush=True)
    assert far.max() <= 1.0, (label, float(far.max()))
