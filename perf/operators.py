"""Operators of a long-context KV cache, each in its plain form and as the framework's calls.

    append     rows quantised into a 4-bit pool (MXFP4: E2M1 codes, one power-of-two scale for 32
               elements) and read back as the values they stand for
    attention  paged causal attention over a 4-bit pool: decode, verify rows, prompt chunks
    weights    the attention weight that every cached key received in a step, added up per KV head
    evict      the keys of a sequence that are kept (the most recent and the heaviest), moved together

A 4-bit plane holds codes [page][kv head][token][head_dim / 2] (element 2i in the low nibble) and
scales [page][kv head][token][head_dim / 32]; 16-bit and FP8 planes hold [page][token][kv head][head_dim].
The weight plane is f32 [page][kv head][token].  Pages are scattered by a seeded permutation.
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
    case = dict(kind=kind, hq=16, hkv=2, d=128, page=16)
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
    r = np.random.default_rng(2)
    len16 = r.integers(2048, 8192, size=16, endpoint=True)
    return [
        # the rows of a decode step of eight chats
        _case("append_decode", "append", rows=8, first=3000, src="bf16"),
        # a packed prompt of the largest batch, many KV heads
        _case("append_prompt", "append", rows=4096, first=1000, hq=32, hkv=8, page=32, src="bf16"),
        # one short chat of a small model: latency
        _case("decode_chat", "attention", new="1", cached="699", hq=8, d=64, layers=2),
        # the ordinary decode step: eight ragged contexts, four layers on one plan
        _case("decode_b8", "attention", new=_text(ctx8 * 0 + 1), cached=_text(ctx8 - 1), layers=4),
        # speculative decoding: 32 sequences verify two to four rows each
        _case("verify_b32", "attention", new=_text(new32), cached=_text(ctx32 - new32), layers=2),
        # a full server of long contexts: 64 sequences of 16k to 32k keys
        _case("decode_b64", "attention", new=_text(ctx64 * 0 + 1), cached=_text(ctx64 - 1), layers=1),
        # four odd prompt chunks, three of them over cached prefixes, many KV heads
        _case("prefill", "attention", new="777,1024,300,1500", cached="0,3001,6000,513", hq=32, hkv=8, page=32,
              layers=1),
        # the weights that a decode step gives the keys of eight contexts on a 4-bit pool
        _case("weights_b8", "weights", new=_text(ctx8 * 0 + 1), cached=_text(ctx8 - 1), kv="fp4", decay=1.0),
        # the weights of two prompt chunks over their prefixes on a bf16 pool
        _case("weights_chunk", "weights", new="512,300", cached="4096,1701", kv="bf16", decay=1.0),
        # the weights of a full server's decode step, fading
        _case("weights_b64", "weights", new=_text(ctx64 * 0 + 1), cached=_text(ctx64 - 1), kv="fp4", decay=0.75),
        # sixteen chats cut to 1,024 keys
        _case("evict_b16", "evict", lengths=_text(len16), budget=1024, recent=256, kv="fp4"),
        # two documents of 128k keys cut to 8,192, many KV heads, a 16-bit pool
        _case("evict_long", "evict", lengths="131072,100001", budget=8192, recent=1000, hq=32, hkv=8, page=32,
              kv="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "verify", "prefill", "weights", "weights", "evict", "evict"])
    more = dict(zip(("hq", "hkv", "d"), rng.choice(GEOMETRY)), page=rng.choice([16, 16, 32, 64]))
    if kind == "append":
        return _case(None, "append", rows=_log(rng, 1, 4096), first=_log(rng, 1, 60000),
                     src=rng.choice(["bf16", "bf16", "f16", "f32"]), **more)
    if kind == "evict":
        n, top = _log(rng, 1, 32), _log(rng, 64, 65536)
        lengths = [_log(rng, 1, top) for _ in range(n)]
        while sum(lengths) * more["hkv"] > 1.5e6:
            lengths = [max(1, c // 2) for c in lengths]
        budget = _log(rng, 1, max(2, top // 2))
        return _case(None, "evict", lengths=_text(lengths), budget=budget, recent=rng.randint(0, budget),
                     kv=rng.choice(["fp4", "fp4", "bf16", "f16"]), **more)
    prompt = kind == "prefill" or (kind == "weights" and rng.random() < 0.5)
    if prompt:
        n = rng.randint(1, 5)
        new = [_log(rng, 17, 1500) for _ in range(n)]
        cached = [rng.choice([0, _log(rng, 1, 8000)]) for _ in range(n)]
    else:
        n, top = _log(rng, 1, 64), _log(rng, 64, 32768)
        new = [rng.randint(2, 4) if kind == "verify" else 1 for _ in range(n)]
        cached = [_log(rng, max(1, top // 32), top) for _ in range(n)]
    case = _case(None, "weights" if kind == "weights" else "attention", new=_text(new), cached=_text(cached), **more)
    if kind == "weights":
        case.update(kv=rng.choice(["fp4", "fp4", "bf16", "f16", "fp8"]), decay=rng.choice([1.0, 1.0, 0.0, 0.9]))
    else:
        case.update(layers=1 if prompt else rng.randint(1, 3))
    while work(case)["bytes"] > 2.0e8 or work(case)["flops"] > 1.0e11:
        cached = [c // 2 for c in cached]
        new = [max(1, c * 3 // 4) for c in new] if prompt else new
        case.update(new=_text(new), cached=_text(cached))
    return case


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
        self.used = int(need.sum())
        self.pool_pages = self.used + slack
        perm = np.random.default_rng(seed).permutation(self.pool_pages).astype(np.uint32)
        self.stride = int(need.max()) + 1
        self.table = np.full((self.n, self.stride), 0xFFFFFFFF, np.uint32)
        held = np.arange(self.stride)[None, :] < need[:, None]
        self.table[held] = perm[:self.used]
        self.spare = perm[self.used:]
        self.sequences = np.repeat(np.arange(self.n), self.new)
        self.cu = np.concatenate([[0], np.cumsum(self.new)])
        self.positions = np.arange(self.rows) - np.repeat(self.cu[:-1] - self.cached, self.new)
        self.slots = _slots(self.table, self.sequences, self.positions, page)


def _slots(table, sequences, positions, page):
    return table[sequences, positions // page].astype(np.int64) * page + positions % page


def _pack(x):
    """[..., d] f32 as 4-bit codes [..., d / 2] and scales [..., d / 32] (uint8)."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    s = ((top.view(torch.int32) >> 23) - 2).clamp_(0, 254)
    y = b.abs() * torch.ldexp(torch.ones_like(top), 127 - s)  # a power of two: exact
    code = (y > 0.25).to(torch.uint8)
    code += y >= 0.75
    code += y > 1.25
    code += y >= 1.75
    code += y > 2.5
    code += y >= 3.5
    code += y > 5.0
    code |= (b < 0).to(torch.uint8) << 3
    code = code.reshape(*x.shape[:-1], -1, 2)
    return code[..., 0] | code[..., 1] << 4, s[..., 0].to(torch.uint8)


_LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _unpack(codes, scales):
    """The values of 4-bit codes [..., d / 2] and scales [..., d / 32], f32 [..., d]."""
    levels = torch.tensor(_LEVELS, device=codes.device)
    x = torch.stack([levels[(codes & 15).int()], levels[(codes >> 4).int()]], -1).flatten(-2)
    scale = (scales.int() << 23).view(torch.float32)  # 2^(s - 127); a scale of 0 is only ever beside codes of 0
    return (x.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _plane(g, case, pages):
    """One plane of N(0, 1) keys or values in the case's type: {"x": ..., "s": scales or None}."""
    hkv, d, page, kv = case["hkv"], case["d"], case["page"], case.get("kv", "fp4")
    if kv == "fp4":
        parts = [_pack(_randn(g, n, hkv, page, d)) for n in _parts(pages, max(1, (1 << 27) // (hkv * page * d)))]
        return dict(x=torch.cat([p[0] for p in parts]), s=torch.cat([p[1] for p in parts]))
    x = _randn(g, pages, page, hkv, d)
    if kv == "fp8":
        s = (1.0 + 0.25 * torch.rand(pages, hkv, generator=g, device=DEV)) / 125.0
        return dict(x=(x * 125.0).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), s=s)
    return dict(x=x.to(TORCH[kv]), s=None)


def _parts(n, most):
    return [min(most, n - i) for i in range(0, n, most)]


def _values(plane, kv, pages):
    """The values of a plane's pages (any index), f32 [..., kv head, token, d]."""
    x = plane["x"][pages]
    if kv == "fp4":
        return _unpack(x, plane["s"][pages])
    if kv == "fp8":
        return x.view(torch.float8_e4m3fn).float().transpose(-2, -3) * plane["s"][pages][..., None, None]
    return x.transpose(-2, -3).float()


def _queries(g, case, rows):
    """Queries as sharp as a model's: the scores' standard deviation is about 2."""
    return (2.0 * _randn(g, rows, case["hq"], case["d"])).to(torch.bfloat16)


# ------------------------------------------------------------------ prepare and run

def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def run(state):
    return state["own" if own else "plain"](state)


def _layout(case, pages):
    return package().KVLayout(case["hkv"], case["d"], case["page"], pages, CODE[case.get("kv", "fp4")])


def _prepare_append(case, seed):
    rows, page, hkv, d = case["rows"], case["page"], case["hkv"], case["d"]
    if rows <= 64:  # a decode step: a row of each of `rows` sequences
        b = _Batch(np.ones(rows, np.int64), case["first"] + np.arange(rows) % 7, page, seed)
    else:           # a prompt
        b = _Batch([rows], [case["first"]], page, seed)
    g = _gen(seed)
    k, v = (_randn(g, rows, hkv, d).to(TORCH[case["src"]]) for _ in range(2))
    z = lambda w: torch.zeros((b.pool_pages, hkv, page, w), dtype=torch.uint8, device=DEV)  # noqa: E731
    return dict(plain=_append_plain, own=_append_own, case=case, k=k, v=v, pages=b.pool_pages, slots=_i32(b.slots),
                kc=dict(x=z(d // 2), s=z(d // 32)), vc=dict(x=z(d // 2), s=z(d // 32)),
                ko=torch.empty((rows, hkv, d), dtype=torch.bfloat16, device=DEV),
                vo=torch.empty((rows, hkv, d), dtype=torch.bfloat16, device=DEV))


def _append_plain(s):
    at = s["slots"].long()
    page, off = at // s["case"]["page"], at % s["case"]["page"]
    for c, x in (("kc", s["k"]), ("vc", s["v"])):
        codes, scales = _pack(x.float())
        s[c]["x"][page, :, off] = codes
        s[c]["s"][page, :, off] = scales
    return dict(k=_unpack(s["kc"]["x"][page, :, off], s["kc"]["s"][page, :, off]).to(torch.bfloat16),
                v=_unpack(s["vc"]["x"][page, :, off], s["vc"]["s"][page, :, off]).to(torch.bfloat16))


def _append_own(s):
    lia, layout, kc, vc = package(), _layout(s["case"], s["pages"]), s["kc"], s["vc"]
    lia.kv_append(layout, s["k"], s["v"], kc["x"], vc["x"], slot_mapping=s["slots"], k_scales=kc["s"], v_scales=vc["s"])
    lia.kv_gather(layout, s["slots"], kc["x"], vc["x"], s["ko"], s["vo"], k_scales=kc["s"], v_scales=vc["s"])
    return dict(k=s["ko"], v=s["vo"])


def _step(case, seed):
    """What attention and weights have in common: the batch and its metadata on the device."""
    b = _Batch(_ints(case["new"]), _ints(case["cached"]), case["page"], seed)
    held = torch.from_numpy(np.where(b.table == 0xFFFFFFFF, 0, b.table).astype(np.int64)).to(DEV)
    rows = torch.from_numpy(b.sequences * int(b.new.max()) + np.arange(b.rows) - b.cu[b.sequences]).to(DEV)
    return b, dict(case=case, b=b, held=held, at=rows, cu=_i32(b.cu), positions=_i32(b.positions),
                   sequences=_i32(b.sequences), flat=_i32(b.table.reshape(-1)))


def _handle(s, workspace):
    """What a program of the framework keeps for its steps: the geometry and a workspace."""
    case, b, lia = s["case"], s["b"], package()
    cfg = lia.AttentionConfig(case["hq"], case["hkv"], case["d"], case["page"], b.pool_pages, b.stride, CODE["bf16"],
                              CODE[case.get("kv", "fp4")], CODE["bf16"], 1.0 / math.sqrt(case["d"]), b.n, b.rows,
                              int(b.ctx.max()))
    return dict(config=cfg, ws=torch.zeros(getattr(lia, workspace)(cfg), dtype=torch.uint8, device=DEV))


def _prepare_attention(case, seed):
    b, s = _step(case, seed)
    g = _gen(seed)
    s.update(plain=_attention_plain, own=_attention_own, layers=[
        dict(q=_queries(g, case, b.rows), k=_plane(g, case, b.pool_pages), v=_plane(g, case, b.pool_pages),
             o=torch.empty((b.rows, case["hq"], case["d"]), dtype=torch.bfloat16, device=DEV))
        for _ in range(case["layers"])])
    if own:
        s.update(_handle(s, "workspace_bytes"))
    return s


def _probabilities(s, q, k):
    """softmax weights [n, kv head, row * group, key] of the padded batch; 0 where a key is not attended."""
    case, b = s["case"], s["b"]
    n, hkv, group, most, d = b.n, case["hkv"], case["hq"] // case["hkv"], int(b.new.max()), case["d"]
    padded = torch.zeros((n * most, case["hq"], d), device=DEV)
    padded[s["at"]] = q.float()
    last = torch.full((n * most,), -1, dtype=torch.int64, device=DEV)
    last[s["at"]] = s["positions"].long()
    padded = padded.view(n, most, hkv, group, d).transpose(1, 2).reshape(n, hkv, most * group, d)
    scores = torch.matmul(padded, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(d))
    keys = torch.arange(k.shape[-2], device=DEV)
    live = keys <= last.view(n, 1, most, 1, 1).expand(n, 1, most, group, 1).reshape(n, 1, most * group, 1)
    scores.masked_fill_(~live, -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp_min_(-1e30)
    scores.exp_()
    scores /= scores.sum(-1, keepdim=True).clamp_min_(1e-30)
    return scores


def _attend(s, t):
    case, b = s["case"], s["b"]
    n, hkv, group, most, d = b.n, case["hkv"], case["hq"] // case["hkv"], int(b.new.max()), case["d"]
    k = _values(t["k"], "fp4", s["held"]).transpose(1, 2).reshape(n, hkv, -1, d)
    p = _probabilities(s, t["q"], k)
    del k
    v = _values(t["v"], "fp4", s["held"]).transpose(1, 2).reshape(n, hkv, -1, d)
    o = torch.matmul(p, v).view(n, hkv, most, group, d).transpose(1, 2).reshape(n * most, case["hq"], d)
    return o[s["at"]].to(torch.bfloat16)


def _attention_plain(s):
    return [_attend(s, t) for t in s["layers"]]


def _attention_own(s):
    """One plan of the step for all layers, then each layer's attention and its combine."""
    lia, b, cfg, ws = package(), s["b"], s["config"], s["ws"]
    lia.attention_plan(cfg, b.n, b.rows, s["cu"], s["positions"], s["sequences"], ws, s["flat"])
    for t in s["layers"]:
        lia.attention_partial(cfg, b.n, s["flat"], t["q"], t["k"]["x"], t["v"]["x"], t["o"], ws, t["k"]["s"], t["v"]["s"])
        lia.attention_merge(cfg, b.n, b.rows, t["o"], ws)
    return [t["o"] for t in s["layers"]]


def _prepare_weights(case, seed):
    b, s = _step(case, seed)
    g = _gen(seed)
    s.update(plain=_weights_plain, own=_weights_own, q=_queries(g, case, b.rows),
             k=_plane(g, case, b.pool_pages),
             # what earlier steps gave the keys: as much as this one gives a key of a few thousand
             mass=torch.rand((b.pool_pages, case["hkv"], case["page"]), generator=g, device=DEV).mul_(1e-3))
    if own:
        s.update(_handle(s, "attention_weights_workspace_bytes"))
    s["live"] = torch.arange(b.stride * case["page"], device=DEV) < torch.from_numpy(b.ctx).to(DEV)[:, None]
    return s


def _weights_plain(s):
    case, b = s["case"], s["b"]
    n, hkv, page, d = b.n, case["hkv"], case["page"], case["d"]
    k = _values(s["k"], case["kv"], s["held"]).transpose(1, 2).reshape(n, hkv, -1, d)
    w = _probabilities(s, s["q"], k).sum(2)  # [n, kv head, key]
    seq, key = s["live"].nonzero(as_tuple=True)
    at, off = s["held"][seq, key // page], key % page
    s["mass"][at, :, off] = s["mass"][at, :, off] * case["decay"] + w[seq, :, key]
    return s["mass"]


def _weights_own(s):
    package().attention_weights(s["config"], s["b"].n, s["cu"], s["positions"], s["sequences"], s["flat"], s["q"],
                                s["k"]["x"], s["mass"], s["ws"], k_scales=s["k"]["s"], decay=s["case"]["decay"])
    return s["mass"]


def _prepare_evict(case, seed):
    lengths, page, hkv, d, budget = _ints(case["lengths"]), case["page"], case["hkv"], case["d"], case["budget"]
    counts = np.minimum(lengths, budget)
    fresh = -(-counts // page)  # the pages that the kept keys move to
    b = _Batch(lengths, 0 * lengths, page, seed, slack=int(fresh.sum()) + 5)
    g = _gen(seed)
    to = np.full_like(b.table, 0xFFFFFFFF)
    held = np.arange(b.stride)[None, :] < fresh[:, None]
    to[held] = b.spare[:int(fresh.sum())]
    sequences = np.repeat(np.arange(b.n), counts)
    positions = np.arange(int(counts.sum())) - np.repeat(np.cumsum(counts) - counts, counts)
    # the weights of keys that a few heads look at: most light, some heavy, and many of the lightest equal
    mass = torch.rand((b.pool_pages, hkv, page), generator=g, device=DEV).pow_(8).mul_(40.0)
    mass = torch.where(mass < 1e-6, torch.zeros_like(mass), mass)
    kv = "bf16" if case["kv"] == "fp4" else case["kv"]
    out = lambda: torch.empty((int(counts.sum()), hkv, d), dtype=TORCH[kv], device=DEV)  # noqa: E731
    return dict(plain=_evict_plain, own=_evict_own, case=case, b=b, k=_plane(g, case, b.pool_pages),
                v=_plane(g, case, b.pool_pages), mass=mass, rows=_i32(np.arange(b.n)), lengths=_i32(lengths),
                flat=_i32(b.table.reshape(-1)), to=_i32(to.reshape(-1)), slots=_i32(_slots(to, sequences, positions, page)),
                sequences=torch.from_numpy(sequences).to(DEV), positions=torch.from_numpy(positions).to(DEV),
                kept=torch.full((b.n, hkv, budget), -1, dtype=torch.int32, device=DEV),
                counts=torch.zeros(b.n, dtype=torch.int32, device=DEV), ko=out(), vo=out(),
                table=torch.from_numpy(np.where(b.table == 0xFFFFFFFF, 0, b.table).astype(np.int64)).to(DEV))


def _evict_plain(s):
    case, b, mass, table = s["case"], s["b"], s["mass"], s["table"]
    hkv, page, budget, n = case["hkv"], case["page"], case["budget"], s["lengths"].long()
    key = torch.arange(b.stride * page, device=DEV)
    m = mass[table].transpose(1, 2).reshape(b.n, hkv, -1)  # [n, kv head, key]
    bits = m.view(torch.int32).long()
    order = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits)  # the total order of floats, as whole numbers
    order = order * (1 << 24) - key
    recent = key >= (n[:, None, None] - case["recent"])
    order = torch.where(recent, (1 << 60) - key, order)
    order = torch.where(key < n[:, None, None], order, -(1 << 62) - key)
    top = order.topk(min(budget, order.shape[-1]), -1).indices
    count = n.clamp(max=budget)
    place = torch.arange(top.shape[-1], device=DEV)
    top = torch.where(place < count[:, None, None], top, 1 << 40).sort(-1).values
    live = place < count[:, None, None]
    s["kept"].fill_(-1)
    s["kept"][..., :top.shape[-1]] = torch.where(live, top, -1).int()
    s["counts"].copy_(count)
    seq, i = s["sequences"], s["positions"]
    src = top[seq, :, i]                                   # [rows, kv head]: the key that moves to row's place
    heads = torch.arange(hkv, device=DEV)
    sp, so = table[seq[:, None], src // page], src % page
    at = s["slots"].long()
    dp, do = (at // page)[:, None], (at % page)[:, None]
    fp4 = case["kv"] == "fp4"
    got = []
    for t in (s["k"], s["v"]):
        if fp4:
            t["x"][dp, heads, do] = t["x"][sp, heads, so]
            t["s"][dp, heads, do] = t["s"][sp, heads, so]
            got.append(_unpack(t["x"][dp, heads, do], t["s"][dp, heads, do]).to(torch.bfloat16))
        else:
            t["x"][dp, do, heads] = t["x"][sp, so, heads]
            got.append(t["x"][dp, do, heads])
    mass[dp, heads, do] = mass[sp, heads, so]
    return dict(kept=s["kept"], counts=s["counts"], k=got[0], v=got[1], mass=mass)


def _evict_own(s):
    lia, case, k, v = package(), s["case"], s["k"], s["v"]
    layout, stride = _layout(case, s["b"].pool_pages), s["b"].stride
    lia.kv_select(layout, s["rows"], s["lengths"], s["flat"], stride, case["budget"], case["recent"], s["mass"],
                  s["kept"], s["counts"])
    lia.kv_compact(layout, s["rows"], s["flat"], s["to"], stride, s["kept"], s["counts"], k["x"], v["x"],
                   mass=s["mass"], k_scales=k["s"], v_scales=v["s"])
    lia.kv_gather(layout, s["slots"], k["x"], v["x"], s["ko"], s["vo"], k_scales=k["s"], v_scales=v["s"])
    return dict(kept=s["kept"], counts=s["counts"], k=s["ko"], v=s["vo"], mass=s["mass"])


# ------------------------------------------------------------------ work

def _row_bytes(kv, d):
    """Bytes of one key or value of one head."""
    return {"fp4": d // 2 + d // 32, "fp8": d, "f16": 2 * d, "bf16": 2 * d}[kv]


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "append":
        n = case["rows"] * hkv * d
        size = {"f32": 4, "f16": 2, "bf16": 2}[case["src"]]
        # the rows, their codes and scales written and read back, and the values
        return dict(bytes=2 * (n * size + 2 * case["rows"] * hkv * _row_bytes("fp4", d) + 2 * n) + 8 * case["rows"],
                    flops=2 * n)
    if case["kind"] == "evict":
        lengths, kv = _ints(case["lengths"]), case["kv"]
        kept = int(np.minimum(lengths, case["budget"]).sum()) * hkv
        row, value = _row_bytes(kv, d), 2 * d
        # the weights read, the kept indices; each kept row read, written, and read back as values
        return dict(bytes=int(lengths.sum()) * hkv * 4 + 8 * kept + kept * (2 * (3 * row + value) + 8),
                    flops=int(lengths.sum()) * hkv)
    new, cached, kv = _ints(case["new"]), _ints(case["cached"]), case.get("kv", "fp4")
    keys = int((new + cached).sum()) * hkv
    pairs = int((new * cached + new * (new + 1) // 2).sum()) * hq
    rows = int(new.sum()) * hq * d * 2
    if case["kind"] == "weights":
        return dict(bytes=keys * (_row_bytes(kv, d) + (8 if case["decay"] else 4)) + rows, flops=2 * d * pairs)
    return dict(bytes=case["layers"] * (2 * keys * _row_bytes(kv, d) + 2 * rows), flops=4 * d * pairs * case["layers"])


# ------------------------------------------------------------------ the same in 64 bits, from the definitions

def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))


def _exact_quantised(x):
    """The MXFP4 values nearest to x (f64): every level's distance, ties to the even code."""
    b = x.double().unflatten(-1, (-1, 32))
    exponent = torch.frexp(b.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -125)).exponent - 1 - 2
    scale = torch.pow(2.0, exponent.double())
    y = b / scale
    levels = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device=DEV)  # even codes first
    near = (y.abs()[..., None] - levels).abs().argmin(-1)
    return (torch.copysign(levels[near], y) * scale).flatten(-2)


def _exact_append(case, s):
    return dict(k=_exact_quantised(s["k"]), v=_exact_quantised(s["v"]))


def _exact_keys(case, s, plane, b):
    """[kv head, key, d] of sequence b in f64, page by page."""
    n, page, kv = int(s["b"].ctx[b]), case["page"], case.get("kv", "fp4")
    pages = torch.from_numpy(s["b"].table[b, :-(-n // page)].astype(np.int64)).to(DEV)
    x = plane["x"][pages]
    if kv == "fp4":
        lo, hi = (x % 16).double(), (x // 16).double()
        c = torch.stack([lo, hi], -1).flatten(-2)
        sign, m = torch.where(c >= 8, -1.0, 1.0), c % 8
        value = torch.where(m < 2, m * 0.5, (1.0 + (m % 2) * 0.5) * torch.pow(2.0, m.div(2, rounding_mode="floor") - 1))
        scale = torch.pow(2.0, plane["s"][pages].double() - 127.0).repeat_interleave(32, -1)
        return (sign * value * scale).transpose(0, 1).flatten(1, 2)[:, :n]
    x = (x.view(torch.float8_e4m3fn) if kv == "fp8" else x).double().permute(2, 0, 1, 3)
    if kv == "fp8":
        x = x * plane["s"][pages].double().t()[:, :, None, None]
    return x.flatten(1, 2)[:, :n]


def _exact_softmax(case, s, q, k, b):
    """Softmax weights [kv head, row, group, key] of sequence b."""
    lo, hi, first = int(s["b"].cu[b]), int(s["b"].cu[b + 1]), int(s["b"].cached[b])
    hkv, group, d = case["hkv"], case["hq"] // case["hkv"], case["d"]
    x = q[lo:hi].double().view(hi - lo, hkv, group, d).permute(1, 0, 2, 3).reshape(hkv, -1, d)
    score = torch.matmul(x, k.transpose(1, 2).contiguous()) / math.sqrt(d)
    score = score.view(hkv, hi - lo, group, -1)
    hidden = torch.arange(score.shape[-1], device=DEV)[None, :] > first + torch.arange(hi - lo, device=DEV)[:, None]
    score = score.masked_fill(hidden[None, :, None, :], -math.inf)
    return torch.softmax(score, -1)


def _exact_attention(case, s):
    outs = []
    for t in s["layers"]:
        rows = []
        for b in range(s["b"].n):
            p = _exact_softmax(case, s, t["q"], _exact_keys(case, s, t["k"], b), b)
            hkv, m, group, n = p.shape
            o = torch.matmul(p.view(hkv, m * group, n), _exact_keys(case, s, t["v"], b))
            rows.append(o.view(hkv, m, group, -1).transpose(0, 1).reshape(m, case["hq"], -1))
        outs.append(torch.cat(rows))
    return outs


def _exact_weights(case, s):
    mass, page = s["mass"].double(), case["page"]
    for b in range(s["b"].n):
        w = _exact_softmax(case, s, s["q"], _exact_keys(case, s, s["k"], b), b).sum((1, 2))
        n = w.shape[1]
        for i in range(-(-n // page)):
            part = w[:, i * page:(i + 1) * page]
            row = mass[int(s["b"].table[b, i])]
            row[:, :part.shape[1]] = row[:, :part.shape[1]] * case["decay"] + part
    return mass


def _exact_evict(case, s):
    """The kept values and weights; the whole numbers (kept, counts) are compared as they are."""
    page, hkv, table = case["page"], case["hkv"], s["b"].table
    to = s["to"].cpu().numpy().reshape(table.shape)
    mass = s["mass"].double()
    ks, vs = [], []
    for b in range(s["b"].n):
        n = int(s["b"].ctx[b])
        count, r = min(n, case["budget"]), min(case["recent"], n)
        pages = torch.from_numpy(table[b, :-(-n // page)].astype(np.int64)).to(DEV)
        m = s["mass"][pages].transpose(0, 1).flatten(1, 2)[:, :n]
        order = m[:, :n - r].sort(dim=-1, descending=True, stable=True).indices[:, :max(0, count - r)]
        last = torch.arange(n - min(r, count), n, device=DEV).expand(hkv, -1)
        keep = torch.cat([order, last], 1).sort(-1).values
        for out, plane in ((ks, s["k"]), (vs, s["v"])):
            x = _exact_keys(case, s, plane, b)
            out.append(torch.gather(x, 1, keep[..., None].expand(-1, -1, x.shape[-1])).transpose(0, 1))
        moved = torch.gather(m, 1, keep)
        for i in range(-(-count // page)):
            part = moved[:, i * page:(i + 1) * page]
            mass[int(to[b, i])][:, :part.shape[1]] = part.double()
    return dict(kept=None, counts=None, k=torch.cat(ks), v=torch.cat(vs), mass=mass)
