"""Operators of a long-context attention step, each in its plain form and as the framework's calls.

    table   the rotation's table of a step: cosines and sines of far positions, from given frequencies
    rotate  queries and keys normalised for each head, rotated (half or interleaved pairs, whole heads or
            part), and appended to the paged KV pool with the values
    select  summaries of the pages that a step completes (the largest and smallest value of each channel,
            as 8-bit codes), and for each row and KV head the pages whose summaries promise it most
    attend  causal attention of each row over its selected pages alone

Codes are whole numbers times a power of two, and so are the queries' in the scores: the scores are exact, and
a row's pages have one answer whatever the order of the sums.

16-bit and FP8 planes hold [page][token][kv head][head_dim], 4-bit planes (MXFP4) codes [page][kv head][token]
[head_dim / 2] and scales [page][kv head][token][head_dim / 32]; summaries [page][kv head][largest, smallest]
[head_dim].  Pages are scattered by a seeded permutation.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
CODE = {"f32": 0, "f16": 1, "bf16": 2, "fp8": 3, "fp4": 4}
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GEOMETRY = [(16, 2, 128), (16, 2, 128), (32, 8, 128), (8, 2, 64)]  # query heads, KV heads, head_dim
EPS = 1e-6


def package():
    """The package of the working folder's tree (its folder name is no Python identifier)."""
    if "lia_rs_amd" not in sys.modules:
        folder = os.path.join(os.getcwd(), "lia.rs_amd")
        spec = importlib.util.spec_from_file_location(
            "lia_rs_amd", os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        sys.modules["lia_rs_amd"] = module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    return sys.modules["lia_rs_amd"]


# ------------------------------------------------------------------ the cases

def _text(values):
    return ",".join(str(int(v)) for v in values)


def _ints(text):
    return np.array([int(v) for v in text.split(",")], dtype=np.int64)


def _case(name, kind, **more):
    case = dict(kind=kind)
    if kind != "table":
        case.update(hq=16, hkv=2, d=128, page=16)
    case.update(more)
    return dict(name=name, **case) if name else case


def listed():
    r = np.random.default_rng(0)
    ctx8 = r.integers(1024, 32768, size=8, endpoint=True)
    r = np.random.default_rng(0)
    new32 = 1 + r.integers(1, 3, size=32, endpoint=True)
    ctx32 = r.integers(512, 16384, size=32, endpoint=True)
    r = np.random.default_rng(1)
    ctx64 = r.integers(16384, 32768, size=64, endpoint=True)
    ones8, ones64 = _text(ctx8 * 0 + 1), _text(ctx64 * 0 + 1)
    return [
        # the rows of a decode step of eight chats, half of a head rotated
        _case("table_decode", "table", rows=8, n=64, first=30000),
        # the largest packed prompt of a long document, past 100k positions
        _case("table_prompt", "table", rows=4096, n=128, first=100001),
        # the projections of a decode step of eight chats
        _case("rotate_decode", "rotate", rows=8, n=128, pairs="half", norm=True, src="bf16", kv="bf16", q="bf16"),
        # a packed prompt of the largest batch, many KV heads, interleaved pairs of half the head
        _case("rotate_prompt", "rotate", rows=4096, hq=32, hkv=8, page=32, n=64, pairs="interleaved", norm=True,
              src="bf16", kv="bf16", q="bf16"),
        # the ordinary decode step: eight ragged contexts, 64 pages each
        _case("select_b8", "select", new=ones8, cached=_text(ctx8 - 1), kv="bf16", budget=64, first=1, recent=4),
        # a full server of long contexts: 64 sequences of 16k to 32k keys, 128 pages each
        _case("select_b64", "select", new=ones64, cached=_text(ctx64 - 1), kv="bf16", budget=128, first=1, recent=8),
        # two prompt chunks over long prefixes: their own pages are summarised in the pass
        _case("select_chunk", "select", new="512,300", cached="16384,9001", kv="bf16", budget=64, first=1, recent=4),
        # one short chat of a small model, an f16 pool: latency
        _case("attend_chat", "attend", new="1", cached="699", hq=8, d=64, kv="f16", budget=32),
        # the ordinary decode step, 1,024 keys of each context
        _case("attend_b8", "attend", new=ones8, cached=_text(ctx8 - 1), kv="bf16", budget=64),
        # speculative decoding on a 4-bit pool: 32 sequences verify two to four rows each
        _case("attend_verify", "attend", new=_text(new32), cached=_text(ctx32 - new32), kv="fp4", budget=64),
        # a full server, 2,048 keys of each context on an FP8 pool
        _case("attend_b64", "attend", new=ones64, cached=_text(ctx64 - 1), kv="fp8", budget=128),
        # two prompt chunks, each row over pages of its own
        _case("attend_chunk", "attend", new="512,300", cached="16384,9001", kv="bf16", budget=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["table", "rotate", "rotate", "select", "select", "select", "attend", "attend", "attend"])
    if kind == "table":
        return _case(None, "table", rows=_log(rng, 1, 4096), n=rng.choice([16, 32, 64, 80, 96, 128]),
                     first=_log(rng, 1, 130000))
    more = dict(zip(("hq", "hkv", "d"), rng.choice(GEOMETRY)), page=rng.choice([16, 16, 32, 64]))
    if kind == "rotate":
        return _case(None, "rotate", rows=_log(rng, 1, 4096), n=rng.choice([more["d"], 16, 32, more["d"] // 2]),
                     pairs=rng.choice(["half", "interleaved"]), norm=rng.random() < 0.8,
                     src=rng.choice(["bf16", "bf16", "f16", "f32"]), kv=rng.choice(["bf16", "bf16", "f16"]),
                     q=rng.choice(["bf16", "f32"]), **more)
    if rng.random() < 0.25:  # prompt chunks
        n = rng.randint(1, 3)
        new, cached = [_log(rng, 17, 500) for _ in range(n)], [rng.choice([0, _log(rng, 1, 16384)]) for _ in range(n)]
    else:                    # decode and verify rows
        n, top, verify = _log(rng, 1, 64), _log(rng, 64, 32768), rng.random() < 0.3
        new = [rng.randint(2, 4) if verify else 1 for _ in range(n)]
        cached = [_log(rng, max(1, top // 32), top) for _ in range(n)]
    case = _case(None, kind, new=_text(new), cached=_text(cached), kv=rng.choice(["bf16", "bf16", "f16", "fp8", "fp4"]),
                 budget=_log(rng, 8, 2048 // more["page"]), **more)
    if kind == "select":
        case.update(first=rng.randint(0, 2), recent=rng.randint(1, 5))
    while _cost(case) > (6.9e7 if kind == "select" else 2.0e8):
        new, cached = [max(1, c * 3 // 4) for c in new], [c * 3 // 4 for c in cached]
        case.update(new=_text(new), cached=_text(cached))
        if max(new) <= 4:
            case.update(budget=max(8, case["budget"] * 3 // 4))
    return case


def _cost(case):
    """Elements that the plain form gathers: of the selected keys, or of the sequences' summaries and scores."""
    new, ctx = _ints(case["new"]), _ints(case["new"]) + _ints(case["cached"])
    if case["kind"] == "attend":
        return int(new.sum()) * case["hkv"] * case["budget"] * case["page"] * case["d"]
    pages = len(new) * int(ctx.max()) // case["page"]
    return pages * case["hkv"] * (2 * case["d"] + int(new.max()) * case["hq"] // case["hkv"])


# ------------------------------------------------------------------ inputs (plain torch)

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _i32(values):
    return torch.from_numpy(np.asarray(values, np.uint32).view(np.int32).copy()).to(DEV)


class _Batch:
    """A ragged batch on a pool of scattered pages: per-sequence counts and the block table."""

    def __init__(self, new, cached, page, seed, slack=5):
        self.new, self.cached, self.page = np.asarray(new), np.asarray(cached), page
        self.ctx = self.new + self.cached
        self.n, self.rows = len(self.new), int(self.new.sum())
        need = -(-self.ctx // page)
        used = int(need.sum())
        self.pool_pages = used + slack
        perm = np.random.default_rng(seed).permutation(self.pool_pages).astype(np.uint32)
        self.stride = int(need.max()) + 1
        self.table = np.full((self.n, self.stride), 0xFFFFFFFF, np.uint32)
        self.table[np.arange(self.stride)[None, :] < need[:, None]] = perm[:used]
        self.sequences = np.repeat(np.arange(self.n), self.new)
        self.cu = np.concatenate([[0], np.cumsum(self.new)])
        self.positions = np.arange(self.rows) - np.repeat(self.cu[:-1] - self.cached, self.new)
        self.slots = (self.table[self.sequences, self.positions // page].astype(np.int64) * page
                      + self.positions % page)


def _frequencies(n):
    """Frequencies stretched eightfold for a long context: those that turn less than once over 4,096
    positions by all of it, those that turn over 32 times not at all, and a ramp between."""
    f = 1e6 ** (-np.arange(0, n, 2) / n)
    turns = 4096 * f / (2 * math.pi)
    keep = np.clip((turns - 1) / (32 - 1), 0, 1)
    return f * keep + f / 8 * (1 - keep), 0.1 * math.log(8) + 1


def _pack(x):
    """[..., d] f32 as 4-bit codes [..., d / 2] and scales [..., d / 32] (uint8)."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    s = ((top.view(torch.int32) >> 23) - 2).clamp_(0, 254)
    y = b.abs() * torch.ldexp(torch.ones_like(top), 127 - s)
    code = torch.bucketize(y, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)).to(torch.uint8)
    code |= (b < 0).to(torch.uint8) << 3
    code = code.reshape(*x.shape[:-1], -1, 2)
    return code[..., 0] | code[..., 1] << 4, s[..., 0].to(torch.uint8)


_LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _unpack(codes, scales):
    levels = torch.tensor(_LEVELS, device=codes.device)
    x = torch.stack([levels[(codes & 15).int()], levels[(codes >> 4).int()]], -1).flatten(-2)
    scale = (scales.int() << 23).view(torch.float32)
    return (x.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _plane(g, case, pages):
    """One plane of N(0, 1) keys or values, some channels larger than others, in the case's type:
    {"x": ..., "s": scales or None}."""
    hkv, d, page, kv = case["hkv"], case["d"], case["page"], case["kv"]
    wide = torch.exp(0.5 * _randn(g, hkv, d))
    wide /= wide.square().mean(-1, keepdim=True).sqrt()
    if kv == "fp4":
        x, s = _pack(_randn(g, pages, hkv, page, d) * wide[:, None, :])
        return dict(x=x, s=s)
    x = _randn(g, pages, page, hkv, d) * wide
    if kv == "fp8":
        s = x.abs().amax((1, 3)) / 448.0
        return dict(x=(x / s[:, None, :, None]).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), s=s)
    return dict(x=x.to(TORCH[kv]), s=None)


def _values(plane, kv, pages):
    """The values of a plane's pages (any index), f32 [..., kv head, token, d]."""
    x = plane["x"][pages]
    if kv == "fp4":
        return _unpack(x, plane["s"][pages])
    if kv == "fp8":
        return x.view(torch.float8_e4m3fn).float().transpose(-2, -3) * plane["s"][pages][..., None, None]
    return x.transpose(-2, -3).float()


def _step(case, seed):
    """A step's batch and its metadata on the device."""
    b = _Batch(_ints(case["new"]), _ints(case["cached"]), case["page"], seed)
    held = torch.from_numpy(np.where(b.table == 0xFFFFFFFF, 0, b.table).astype(np.int64)).to(DEV)
    at = torch.from_numpy(b.sequences * int(b.new.max()) + np.arange(b.rows) - b.cu[b.sequences]).to(DEV)
    return b, dict(case=case, b=b, held=held, at=at, cu=_i32(b.cu), positions=_i32(b.positions),
                   sequences=_i32(b.sequences), flat=_i32(b.table.reshape(-1)), slots=_i32(b.slots))


def _config(s):
    """What a program of the framework keeps for its steps: the geometry."""
    case, b = s["case"], s["b"]
    return package().AttentionConfig(case["hq"], case["hkv"], case["d"], case["page"], b.pool_pages, b.stride,
                                     CODE["bf16"], CODE[case["kv"]], CODE["bf16"], 1.0 / math.sqrt(case["d"]), b.n,
                                     b.rows, int(b.ctx.max()))


def _queries(g, case, rows):
    """Queries as sharp as a model's: the scores' standard deviation is about 2."""
    return (2.0 * _randn(g, rows, case["hq"], case["d"])).to(torch.bfloat16)


# ------------------------------------------------------------------ prepare and run

def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def run(state):
    return state["own" if own else "plain"](state)


# ---- table

def _prepare_table(case, seed):
    f, attention = _frequencies(case["n"])
    start = case["first"] + int(np.random.default_rng(seed).integers(0, 1000))
    positions = start + np.arange(case["rows"]) * (1 if case["rows"] > 64 else 997)
    return dict(plain=_table_plain, own=_table_own, positions=_i32(positions), f=torch.from_numpy(f).to(DEV),
                attention=attention, out=torch.empty((case["rows"], case["n"] // 2, 2), device=DEV))


def _table_plain(s):
    angle = s["positions"].double()[:, None] * s["f"]
    return (torch.stack([angle.cos(), angle.sin()], -1) * s["attention"]).float()


def _table_own(s):
    package().rope_table(s["positions"], s["f"], s["out"], attention=s["attention"])
    return s["out"]


# ---- rotate

def _prepare_rotate(case, seed):
    rows, hq, hkv, d, page = case["rows"], case["hq"], case["hkv"], case["d"], case["page"]
    if rows <= 64:  # a decode step: a row of each of `rows` sequences
        b = _Batch(np.ones(rows, np.int64), 40 + np.arange(rows) % 7, page, seed)
    else:           # a prompt
        b = _Batch([rows], [0], page, seed)
    g = _gen(seed)
    f, attention = _frequencies(case["n"])
    angle = (_i32(b.positions).double() + 30000)[:, None] * torch.from_numpy(f).to(DEV)
    pool = lambda: torch.zeros((b.pool_pages, page, hkv, d), dtype=TORCH[case["kv"]], device=DEV)  # noqa: E731
    weight = lambda: (1 + 0.2 * _randn(g, d)).to(torch.bfloat16) if case["norm"] else None  # noqa: E731
    # projections: N(0, 1) times a size of each channel's own
    wide = torch.exp(0.5 * _randn(g, (hq + 2 * hkv) * d))
    return dict(plain=_rotate_plain, own=_rotate_own, case=case, pages=b.pool_pages, slots=_i32(b.slots),
                x=(_randn(g, rows, (hq + 2 * hkv) * d) * wide).to(TORCH[case["src"]]), wq=weight(), wk=weight(),
                table=(torch.stack([angle.cos(), angle.sin()], -1) * attention).float(), kc=pool(), vc=pool(),
                query=torch.empty((rows, hq, d), dtype=TORCH[case["q"]], device=DEV))


def _rotated(x, w, table, case, eps=EPS):
    """Heads [rows, heads, d] normalised and rotated, in x's type."""
    n = case["n"]
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.to(x.dtype)
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    if case["pairs"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., n:]], -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., n:]], -1)


def _rotate_plain(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    x = s["x"].float().view(-1, hq + 2 * hkv, d)
    s["query"].copy_(_rotated(x[:, :hq], s["wq"], s["table"], case))
    at = s["slots"].long()
    s["kc"].view(-1, hkv, d)[at] = _rotated(x[:, hq:hq + hkv], s["wk"], s["table"], case).to(s["kc"].dtype)
    s["vc"].view(-1, hkv, d)[at] = x[:, hq + hkv:].to(s["vc"].dtype)
    return dict(query=s["query"], k=s["kc"], v=s["vc"])


def _rotate_own(s):
    case, lia = s["case"], package()
    layout = lia.KVLayout(case["hkv"], case["d"], case["page"], s["pages"], CODE[case["kv"]])
    lia.qk_norm_rope_kv_append(layout, case["hq"], s["table"], s["x"], s["query"], s["kc"], s["vc"], slot_mapping=s["slots"],
                               q_weight=s["wq"], k_weight=s["wk"], eps=EPS, interleaved=case["pairs"] == "interleaved")
    return dict(query=s["query"], k=s["kc"], v=s["vc"])


# ---- select

def _codes(x):
    """Whole numbers (f32, within +-127) and a power of two for each last axis: x is about their product."""
    top = x.abs().amax(-1, keepdim=True)
    unit = ((top.view(torch.int32) >> 23).clamp_min(7) - 6 << 23).view(torch.float32)
    return (x / unit).round_().clamp_(-127, 127), unit


def _summaries(k):
    """Codes [..., kv head, 2, d] and units [..., kv head] of pages' keys [..., kv head, token, d]."""
    codes, unit = _codes(torch.stack([k.amax(-2), k.amin(-2)], -2).flatten(-2))
    return codes.unflatten(-1, (2, -1)).to(torch.int8), unit[..., 0]


def _prepare_select(case, seed):
    b, s = _step(case, seed)
    g = _gen(seed)
    hkv, d, budget = case["hkv"], case["d"], case["budget"]
    k = _plane(g, case, b.pool_pages)
    codes = torch.zeros((b.pool_pages, hkv, 2, d), dtype=torch.int8, device=DEV)
    scales = torch.zeros((b.pool_pages, hkv), device=DEV)
    done = torch.from_numpy(b.slots[b.slots % b.page == b.page - 1] // b.page).to(DEV)  # pages this step completes
    old = np.unique(b.table[np.arange(b.stride)[None, :] < (b.cached // b.page)[:, None]].astype(np.int64))
    if len(old):  # earlier pages were summarised when they were full
        old = torch.from_numpy(old).to(DEV)
        codes[old], scales[old] = _summaries(_values(k, case["kv"], old))
    s.update(plain=_select_plain, own=_select_own, q=_queries(g, case, b.rows), k=k, codes=codes, scales=scales, done=done,
             pages=torch.from_numpy(b.positions // b.page + 1).to(DEV),
             selected=torch.full((b.rows, hkv, budget), -1, dtype=torch.int32, device=DEV),
             counts=torch.zeros(b.rows, dtype=torch.int32, device=DEV))
    if own:
        s["config"] = _config(s)
        s["ws"] = torch.empty(package().page_select_workspace_bytes(s["config"]), dtype=torch.uint8, device=DEV)
    return s


def _select_plain(s):
    case, b, held = s["case"], s["b"], s["held"]
    hq, hkv, d, budget, most, group = case["hq"], case["hkv"], case["d"], case["budget"], int(b.new.max()), case["hq"] // case["hkv"]
    s["codes"][s["done"]], s["scales"][s["done"]] = _summaries(_values(s["k"], case["kv"], s["done"]))
    c, unit = _codes(s["q"].float())
    both = torch.cat([c.clamp_min(0), c.clamp_max(0)], -1)  # against the largest, against the smallest
    pad = lambda x: torch.zeros((b.n * most, *x.shape[1:]), device=DEV).index_copy_(0, s["at"], x)  # noqa: E731
    both = pad(both).view(b.n, most, hkv, group, 2 * d).transpose(1, 2).reshape(b.n, hkv, most * group, 2 * d)
    unit = pad(unit).view(b.n, most, hkv, group).transpose(1, 2).reshape(b.n, hkv, most * group, 1)
    sums = s["codes"][held].float().flatten(-2).permute(0, 2, 3, 1).contiguous()  # [n, kv head, 2 d, page]
    score = torch.matmul(both, sums)  # whole numbers below 2^22: exact
    score *= unit
    of = s["scales"][held].transpose(1, 2)[:, :, None, :]
    score = torch.where(of < math.inf, score * of, math.inf)
    score = score.view(b.n, hkv, most, group, -1).amax(3).transpose(1, 2).reshape(b.n * most, hkv, -1)[s["at"]] + 0.0
    n, page = s["pages"][:, None, None], torch.arange(b.stride, device=DEV)
    bits = score.view(torch.int32).long()
    order = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits) * (1 << 24) - page
    order = torch.where((page < case["first"]) | (page >= n - case["recent"]), (1 << 60) - page, order)
    order = torch.where(page < n, order, -(1 << 62) - page)
    top = order.topk(min(budget, b.stride), -1).indices
    place = torch.arange(top.shape[-1], device=DEV)
    live = place < n.clamp(max=budget)
    top = torch.where(live, top, 1 << 40).sort(-1).values
    s["selected"][..., :top.shape[-1]] = torch.where(live, top, -1).int()
    s["counts"].copy_(s["pages"].clamp(max=budget))
    return dict(selected=s["selected"], counts=s["counts"], codes=s["codes"], scales=s["scales"])


def _select_own(s):
    case, b, lia = s["case"], s["b"], package()
    layout = lia.KVLayout(case["hkv"], case["d"], case["page"], b.pool_pages, CODE[case["kv"]])
    lia.page_summaries(layout, s["slots"], s["k"]["x"], s["codes"], s["scales"], k_scales=s["k"]["s"])
    lia.page_select(s["config"], b.n, s["cu"], s["positions"], s["sequences"], s["flat"], s["q"], s["codes"], s["scales"],
                    case["first"], case["recent"], s["selected"], s["counts"], s["ws"])
    return dict(selected=s["selected"], counts=s["counts"], codes=s["codes"], scales=s["scales"])


# ---- attend

def _prepare_attend(case, seed):
    b, s = _step(case, seed)
    g = _gen(seed)
    hkv, budget = case["hkv"], case["budget"]
    n = torch.from_numpy(b.positions // b.page + 1).to(DEV)[:, None, None]
    page = torch.arange(b.stride, device=DEV)
    key = torch.rand((b.rows, hkv, b.stride), generator=g, device=DEV)
    key = torch.where((page == 0) | (page == n - 1), 2.0, key)  # the first page and the row's own are always there
    key = torch.where(page < n, key, -1.0)
    top = key.topk(min(budget, b.stride), -1)
    selected = torch.full((b.rows, hkv, budget), 1 << 40, dtype=torch.int64, device=DEV)
    selected[..., :top.indices.shape[-1]] = torch.where(top.values >= 0, top.indices, 1 << 40)
    selected = selected.sort(-1).values
    s.update(plain=_attend_plain, own=_attend_own, q=_queries(g, case, b.rows), k=_plane(g, case, b.pool_pages),
             v=_plane(g, case, b.pool_pages), selected=torch.where(selected < 1 << 40, selected, -1).int(),
             counts=n.flatten().clamp(max=budget).int(),
             out=torch.empty((b.rows, case["hq"], case["d"]), dtype=torch.bfloat16, device=DEV))
    if own:
        s["config"] = _config(s)
        s["ws"] = torch.empty(package().selected_attention_workspace_bytes(s["config"], budget), dtype=torch.uint8,
                              device=DEV)
    return s


def _gathered(s, plane, f64=False):
    """The selected keys or values [rows, kv head, budget * token, d]."""
    case = s["case"]
    heads = torch.arange(case["hkv"], device=DEV)[None, :, None]
    pages = s["held"][s["sequences"].long()[:, None, None], s["selected"].long().clamp_min(0)]
    if case["kv"] == "fp4":
        x = _unpack(plane["x"][pages, heads], plane["s"][pages, heads])
    else:
        x = plane["x"].transpose(1, 2)[pages, heads]
        x = (x.view(torch.float8_e4m3fn).double() if f64 else x.view(torch.float8_e4m3fn).float()) * (
            plane["s"][pages, heads][..., None, None]) if case["kv"] == "fp8" else x
    x = x.flatten(2, 3)
    return x.double() if f64 else x.float()


def _hidden(s):
    """[rows, kv head, budget * token]: keys that the row does not attend."""
    at = s["selected"].long()[..., None] * s["case"]["page"] + torch.arange(s["case"]["page"], device=DEV)
    return ((at < 0) | (at > s["positions"].long()[:, None, None, None])).flatten(2)


def _attend_plain(s):
    case = s["case"]
    q = s["q"].float().view(-1, case["hkv"], case["hq"] // case["hkv"], case["d"])
    score = torch.matmul(q, _gathered(s, s["k"]).transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(case["d"]))
    score.masked_fill_(_hidden(s)[:, :, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp_min(-1e30)
    score.exp_()
    score /= score.sum(-1, keepdim=True).clamp_min(1e-30)
    s["out"].copy_(torch.matmul(score, _gathered(s, s["v"])).reshape(s["out"].shape))
    return s["out"]


def _attend_own(s):
    b = s["b"]
    package().selected_attention(s["config"], b.n, s["cu"], s["positions"], s["sequences"], s["flat"], s["q"], s["k"]["x"],
                                 s["v"]["x"], s["selected"], s["counts"], s["out"], s["ws"], k_scales=s["k"]["s"],
                                 v_scales=s["v"]["s"])
    return s["out"]


# ------------------------------------------------------------------ work

def _row_bytes(kv, d):
    """Bytes of one key or value of one head."""
    return {"fp4": d // 2 + d // 32, "fp8": d, "f16": 2 * d, "bf16": 2 * d}[kv]


def work(case):
    if case["kind"] == "table":
        n = case["rows"] * case["n"] // 2
        return dict(bytes=4 * case["rows"] + 4 * case["n"] + 8 * n, flops=20 * n)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["kind"] == "rotate":
        rows = case["rows"]
        # the projections read, the queries and the pool's rows written, the table
        return dict(bytes=rows * d * ((hq + 2 * hkv) * size[case["src"]] + hq * size[case["q"]] + 2 * hkv * size[case["kv"]])
                    + rows * (4 * case["n"] + 4), flops=8 * rows * (hq + hkv) * d)
    new, cached = _ints(case["new"]), _ints(case["cached"])
    ctx = new + cached
    rows, own_pages = int(new.sum()), -(-ctx // page)
    io = rows * hq * d * 2 + 4 * int(own_pages.sum())
    if case["kind"] == "select":
        done = int((ctx // page - cached // page).sum()) * hkv  # pages summarised, read whole
        pairs = int((new * own_pages).sum()) * hq
        return dict(bytes=io + done * (page * _row_bytes(case["kv"], d) + 2 * d + 4) + int(own_pages.sum()) * hkv * (2 * d + 4)
                    + rows * (hkv * case["budget"] + 1) * 4, flops=4 * d * pairs)
    picked = np.minimum(own_pages, case["budget"])
    # a sequence's pages are read at most once, whatever number of rows selects them
    read = int(np.minimum(new * picked, own_pages).sum()) * hkv * page
    return dict(bytes=2 * io + 2 * read * _row_bytes(case["kv"], d) + int((new * picked).sum()) * hkv * 4,
                flops=4 * d * hq * page * int((new * picked).sum()))


# ------------------------------------------------------------------ the same in 64 bits, from the definitions

def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))


def _exact_table(case, s):
    turn = torch.exp(1j * (s["positions"].double().unsqueeze(1) * s["f"].unsqueeze(0)).to(torch.complex128))
    return torch.view_as_real(turn * s["attention"])


def _exact_rotate(case, s):
    hq, hkv, d, n = case["hq"], case["hkv"], case["d"], case["n"]
    x = s["x"].double().unflatten(-1, (hq + 2 * hkv, d))
    turn = torch.view_as_complex(s["table"].double())[:, None]

    def rotated(y, w):
        if w is not None:
            y = y / ((y * y).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        part = y[..., :n]
        z = (torch.complex(part[..., :n // 2].contiguous(), part[..., n // 2:].contiguous()) if case["pairs"] == "half"
             else torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous())) * turn
        z = torch.cat([z.real, z.imag], -1) if case["pairs"] == "half" else torch.view_as_real(z).flatten(-2)
        return torch.cat([z, y[..., n:]], -1)
    k, v = (torch.zeros(s["kc"].shape, dtype=torch.float64, device=DEV) for _ in range(2))
    page, off = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
    k[page, off] = rotated(x[:, hq:hq + hkv], s["wk"])
    v[page, off] = x[:, hq + hkv:]
    return dict(query=rotated(x[:, :hq], s["wq"]), k=k, v=v)


def _exact_select(case, s):
    """The units of the summaries; everything else is whole numbers, compared as they are."""
    scales = s["scales"].double()
    k = _values(s["k"], case["kv"], s["done"]).double()
    if len(k):
        scales[s["done"]] = torch.pow(2.0, torch.frexp(k.abs().amax((-1, -2))).exponent.double() - 7)
    return dict(selected=None, counts=None, codes=None, scales=scales)


def _exact_attend(case, s):
    q = s["q"].double().unflatten(1, (case["hkv"], -1))
    score = torch.einsum("rhgd,rhkd->rhgk", q, _gathered(s, s["k"], True)) / math.sqrt(case["d"])
    p = torch.softmax(torch.where(_hidden(s)[:, :, None], -math.inf, score), -1)
    return torch.einsum("rhgk,rhkd->rhgd", p, _gathered(s, s["v"], True)).flatten(1, 2)
