"""CPU tests of the oracle of page summaries and selection, and of what the entry points over selected pages refuse: every case
breaks one thing of a call that passes, and none reaches a launch (the addresses are placeholders)."""
import contextlib
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import sparse as S

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4
E_ARG, E_ALIGN, E_WORKSPACE, E_UNSUPPORTED = -20, -21, -22, -23
A = 0x100000


def test_scores_bound_the_products():
    """A page's score is no less than any product of a query with its keys, less the codes' rounding: half a unit of each
    of the d channels' bounds, times the query, and half a unit of the query's times the bounds."""
    rng = np.random.default_rng(0)
    for seed in range(50):
        q = rng.standard_normal((4, 64)) * np.exp(rng.standard_normal((4, 1)))
        keys = rng.standard_normal((1, 16, 64)) * np.exp(rng.standard_normal(64))
        c, s = S.summary(keys)
        score = S.scores(q, c, s)
        _, unit = S.codes(q)
        slack = (0.5 * s[0] * np.abs(q).sum(1) + 0.5 * unit * (np.abs(keys[0]).max(0) + s[0]).sum()).max()
        assert score[0] >= (q @ keys[0].T).max() - slack * 1.001
        assert score[0] <= (np.abs(q) @ np.abs(keys[0]).max(0)).max() + slack * 1.001


def test_codes_of_edges():
    c, u = S.codes(np.array([[0.0, 0.0], [1.0, -1.0], [2.0 - 2 ** -20, 1.0], [1e-44, 0.0], [3e38, -1e38]]))
    assert u.tolist() == [2.0 ** -126, 2.0 ** -6, 2.0 ** -6, 2.0 ** -126, 2.0 ** 121]
    assert c.tolist() == [[0, 0], [64, -64], [127, 64], [0, 0], [113, -38]]
    assert np.isinf(S.summary(np.full((1, 16, 64), np.inf))[1][0]) and np.isinf(S.summary(np.full((1, 16, 64), np.nan))[1][0])


SUMMARY = dict(rows=4, slots=A, kc=A, ks=None, codes=A, scales=A, stream=None)
LAYOUT = dict(hkv=2, d=128, page=16, pool=64, dtype=BF16)


def _summaries(lia, **bad):
    layout, a = dict(LAYOUT), dict(SUMMARY)
    for k, v in bad.items():
        (layout if k in layout else a)[k] = v
    return lia.lib().lia_page_summaries(C.byref(lia.KVLayout(*layout.values())), *a.values())


@pytest.mark.parametrize("bad,status", [
    (dict(slots=None), E_ARG), (dict(kc=None), E_ARG), (dict(codes=None), E_ARG), (dict(scales=None), E_ARG),
    (dict(hkv=0), E_ARG), (dict(page=8), E_UNSUPPORTED), (dict(page=24), E_UNSUPPORTED), (dict(d=96), E_UNSUPPORTED),
    (dict(dtype=F32), E_UNSUPPORTED), (dict(dtype=FP8), E_ARG), (dict(dtype=FP4), E_ARG), (dict(kc=A + 8), E_ALIGN),
    (dict(codes=A + 8), E_ALIGN), (dict(scales=A + 2), E_ALIGN), (dict(slots=A + 1), E_ALIGN), (dict(rows=1 << 25), E_ARG)])
def test_summaries_refused(lia, bad, status):
    assert _summaries(lia, **bad) == status
    assert _summaries(lia, rows=0) == 0


CONFIG = dict(num_q_heads=16, num_kv_heads=2, head_dim=128, page_size=16, pool_pages=64, stride=8, q_dtype=BF16,
              kv_dtype=BF16, out_dtype=BF16, scale=0.088, max_seqs=4, max_rows=8, max_context=128)
SELECT = dict(n_seqs=2, n_rows=2, cu=A, positions=A, sequences=A, pages=A, q=A, codes=A, scales=A, budget=4, first=1, recent=2,
              selected=A, counts=A, ws=A, bytes=8 * 2 * 8 * 4, stream=None)
ATTEND = dict(n_seqs=2, n_rows=2, cu=A, positions=A, sequences=A, pages=A, q=A, kc=A, vc=A, ks=None, vs=None, budget=4,
              selected=A, counts=A, ws=A, bytes=1 << 30, out=A, stream=None)

GEOMETRY = [(dict(num_kv_heads=0), E_ARG), (dict(num_q_heads=0), E_ARG), (dict(num_q_heads=15), E_ARG),
            (dict(num_q_heads=66), E_UNSUPPORTED), (dict(head_dim=96), E_UNSUPPORTED), (dict(page_size=8), E_UNSUPPORTED),
            (dict(page_size=48), E_UNSUPPORTED), (dict(q_dtype=F16), E_UNSUPPORTED), (dict(stride=0), E_ARG),
            (dict(max_seqs=0), E_ARG), (dict(max_rows=0), E_ARG), (dict(max_context=0), E_ARG), (dict(pool_pages=0), E_ARG),
            (dict(max_rows=1 << 22), E_UNSUPPORTED), (dict(max_rows=1 << 21, num_q_heads=64), E_UNSUPPORTED),
            (dict(num_q_heads=65536, num_kv_heads=65536), E_UNSUPPORTED),
            (dict(pool_pages=1 << 31), E_UNSUPPORTED)]  # 2^32 heads of pages


def _call(lia, name, base, **bad):
    config, a = dict(CONFIG), dict(base)
    for k, v in bad.items():
        (config if k in config else a)[k] = v
    return getattr(lia.lib(), name)(C.byref(lia.AttentionConfig(*config.values())), *a.values())


@pytest.mark.parametrize("bad,status", GEOMETRY + [
    (dict(n_seqs=0), E_ARG), (dict(n_seqs=5), E_ARG), (dict(n_rows=0), E_ARG), (dict(n_rows=9), E_ARG),
    *((dict([(k, None)]), E_ARG) for k in ("cu", "positions", "sequences", "pages", "q", "codes", "scales", "selected",
                                           "counts", "ws")),
    (dict(recent=0), E_ARG), (dict(first=3), E_ARG), (dict(recent=4), E_ARG), (dict(budget=2), E_ARG), (dict(budget=0), E_ARG),
    (dict(first=0xFFFFFFFF), E_ARG), (dict(q=A + 8), E_ALIGN), (dict(codes=A + 8), E_ALIGN), (dict(ws=A + 8), E_ALIGN),
    (dict(scales=A + 2), E_ALIGN), (dict(selected=A + 2), E_ALIGN), (dict(counts=A + 2), E_ALIGN),
    (dict(bytes=8 * 2 * 8 * 4 - 1), E_WORKSPACE),
    (dict(stride=0xFFFFFFFF, max_context=0xFFFFFFFF), E_UNSUPPORTED)])
def test_select_refused(lia, bad, status):
    assert _call(lia, "lia_page_select", SELECT, **bad) == status


@pytest.mark.parametrize("bad,status", GEOMETRY + [
    (dict(n_seqs=0), E_ARG), (dict(n_seqs=5), E_ARG), (dict(n_rows=0), E_ARG), (dict(n_rows=9), E_ARG),
    *((dict([(k, None)]), E_ARG) for k in ("cu", "positions", "sequences", "pages", "q", "kc", "vc", "selected", "counts",
                                           "ws", "out")),
    (dict(budget=0), E_ARG), (dict(budget=1 << 27), E_ARG), (dict(kv_dtype=F32), E_UNSUPPORTED),
    (dict(page_size=1 << 22), E_UNSUPPORTED),  # a page of 2^31 bytes
    (dict(out_dtype=F16), E_UNSUPPORTED), (dict(kv_dtype=FP8), E_ARG), (dict(kv_dtype=FP4, ks=A), E_ARG),
    (dict(scale=0.0), E_ARG), (dict(scale=math.inf), E_ARG), (dict(scale=math.nan), E_ARG), (dict(q=A + 8), E_ALIGN),
    (dict(kc=A + 8), E_ALIGN), (dict(vc=A + 8), E_ALIGN), (dict(ws=A + 8), E_ALIGN), (dict(out=A + 8), E_ALIGN),
    (dict(selected=A + 2), E_ALIGN), (dict(counts=A + 2), E_ALIGN), (dict(bytes=1024), E_WORKSPACE)])
def test_attend_refused(lia, bad, status):
    assert _call(lia, "lia_selected_attention", ATTEND, **bad) == status


@pytest.mark.parametrize("bad,status", GEOMETRY)
def test_workspaces_of_refused_geometries(lia, bad, status):
    cfg = lia.AttentionConfig(*dict(CONFIG, **bad).values())
    assert lia.page_select_workspace_bytes(cfg) == 0 and lia.selected_attention_workspace_bytes(cfg, 4) == 0
    cfg = lia.AttentionConfig(*CONFIG.values())
    assert lia.page_select_workspace_bytes(cfg) == 8 * 2 * 8 * 4 and lia.selected_attention_workspace_bytes(cfg, 4) > 0


def test_wrappers_refuse(lia, monkeypatch):
    """What the entry points cannot see: lengths, strides and types of the tensors."""
    monkeypatch.setattr(lia, "_stream", lambda s=None: None)
    cfg, layout = lia.AttentionConfig(*CONFIG.values()), lia.KVLayout(2, 128, 16, 64, BF16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    codes, scales = torch.zeros(64, 2, 2, 128, dtype=torch.int8), torch.zeros(64, 2)
    q = torch.zeros(2, 16, 128, dtype=torch.bfloat16)
    for c, s in ((codes.float(), scales), (codes, scales.half()), (codes[:63], scales), (codes, scales[1:]),
                 (codes.transpose(2, 3), scales), (codes, scales.t())):
        with pytest.raises(lia.LiaError):
            lia.page_summaries(layout, i32(3), q, c, s)
        with pytest.raises(lia.LiaError):
            lia.page_select(cfg, 2, i32(3), i32(2), i32(2), i32(16), q, c, s, 1, 1, i32(2, 2, 4), i32(2), torch.zeros(4096))
    for sel, counts, first, recent in ((i32(2, 2, 8)[..., ::2], i32(2), 1, 1), (i32(2, 4), i32(2), 1, 1),
                                       (i32(1, 2, 4), i32(2), 1, 1), (i32(2, 1, 4), i32(2), 1, 1), (i32(2, 2, 4), i32(1), 1, 1),
                                       (i32(2, 2, 4).long(), i32(2), 1, 1), (i32(2, 2, 4), i32(2), -1, 1),
                                       (i32(2, 2, 4), i32(2), 1, -1), (i32(2, 2, 4), i32(2), 1 << 40, 1),
                                       (i32(2, 2, 4), i32(2), 0, 1 << 40)):
        with pytest.raises(lia.LiaError):
            lia.page_select(cfg, 2, i32(3), i32(2), i32(2), i32(16), q, codes, scales, first, recent, sel, counts,
                            torch.zeros(4096))
        if first == recent == 1:
            with pytest.raises(lia.LiaError):
                lia.selected_attention(cfg, 2, i32(3), i32(2), i32(2), i32(16), q, q, q, sel, counts, q, torch.zeros(1 << 22))


def test_wrappers_refuse_rows(lia, monkeypatch):
    """Queries, outputs and positions of other sizes, types and strides than the configuration's."""
    monkeypatch.setattr(lia, "_stream", lambda s=None: None)
    cfg, layout = lia.AttentionConfig(*CONFIG.values()), lia.KVLayout(2, 128, 16, 64, BF16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    codes, scales = torch.zeros(64, 2, 2, 128, dtype=torch.int8), torch.zeros(64, 2)
    q = torch.zeros(2, 16, 128, dtype=torch.bfloat16)
    good = dict(cu=i32(3), positions=i32(2), sequences=i32(2), pages=i32(4, 8), q=q, out=q.clone())
    for bad in (dict(q=q.float()), dict(q=q.half()), dict(q=torch.cat([q, q], -1)[..., ::2]), dict(q=q[:, :15].contiguous()),
                dict(q=q.transpose(1, 2)), dict(positions=i32(1)), dict(positions=i32(2).long()), dict(out=q.float()),
                dict(out=q[:1]), dict(out=torch.cat([q, q], -1)[..., ::2])):
        a = dict(good, **bad)
        step = cfg, 2, a["cu"], a["positions"], a["sequences"], a["pages"], a["q"]
        if "out" not in bad:
            with pytest.raises(lia.LiaError) as e:
                lia.page_select(*step, codes, scales, 1, 1, i32(2, 2, 4), i32(2), torch.zeros(4096))
            assert e.value.status == E_ARG and "page_select" in str(e.value)
        with pytest.raises(lia.LiaError) as e:
            lia.selected_attention(*step, q, q, i32(2, 2, 4), i32(2), a["out"], torch.zeros(1 << 22))
        assert e.value.status == E_ARG and "selected_attention" in str(e.value)
    for slots in (i32(3).long(), i32(6)[::2]):
        with pytest.raises(lia.LiaError):
            lia.page_summaries(layout, slots, q, codes, scales)


@pytest.fixture
def engine(lia, monkeypatch):
    """An engine on host memory; .calls: (name, arguments) of its launches."""
    calls = []
    for name in ("kv_append", "attention_plan", "attention_partial", "attention_partial_append", "attention_merge",
                 "attention_weights", "page_summaries", "page_select", "selected_attention", "kv_select", "kv_compact"):
        monkeypatch.setattr(lia, name, lambda *a, _name=name, **k: calls.append((_name, a)))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), dict(synchronize=lambda s: None))())
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, pin_memory=False, **k: zeros(*a, **k))

    def make(**more):
        e = lia.Engine(8, 2, 64, pool_tokens=512, page_size=16, kv_dtype=BF16, q_dtype=BF16, out_dtype=BF16, device="cpu",
                       **more)
        e.configure_paging(4, 256)
        e.calls = calls
        return e
    return make


def _names(e):
    got = [c[0] for c in e.calls]
    del e.calls[:]
    return got


def test_engine_summarises_completed_pages(engine, lia):
    e = engine(page_summaries=True)
    kv = lambda n: torch.zeros((n, 2, 64), dtype=torch.bfloat16)  # noqa: E731
    for first, completes in ((0, False), (14, False), (15, True), (16, False)):
        e.stage([(1, first, 0)], [list(range(8))])
        del e.calls[:]
        e.attention(0, torch.zeros(1, 8, 64), kv(1), kv(1))
        assert ("page_summaries" in _names(e)) == completes
        e.selected_attention(0, torch.zeros(1, 8, 64), kv(1), kv(1), 4)
        assert _names(e) == ["kv_append"] + ["page_summaries"] * completes + ["page_select", "selected_attention"]
    e.stage([(1, i, 0) for i in range(40)], [list(range(8))])
    del e.calls[:]
    e.selected_attention(0, torch.zeros(40, 8, 64), kv(40), kv(40), 4, first=2, recent=2)
    (_, a), = [c for c in e.calls if c[0] == "page_summaries"]
    assert a[1].tolist() == list(range(40)) and a[3] is e.summaries[0][0]


def test_engine_refuses(engine, lia):
    e = engine()
    kv = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    e.stage([(1, 0, 0)], [[0]])
    with pytest.raises(lia.LiaError, match="without page_summaries"):
        e.selected_attention(0, torch.zeros(1, 8, 64), kv, kv, 4)
    e = engine(page_summaries=True)
    e.stage([(1, 0, 0)], [[0]])
    for budget, first, recent in ((4, -1, 1), (4, 0, 0), (4, 3, 2), (0, 0, 1)):
        with pytest.raises(lia.LiaError):
            e.selected_attention(0, torch.zeros(1, 8, 64), kv, kv, budget, first, recent)
    with pytest.raises(lia.LiaError):
        e.selected_attention(0, torch.zeros(2, 8, 64), kv, kv, 4)


def test_engine_eviction_summarises_moved_pages(engine, lia):
    e = engine(page_summaries=True, track_weights=True)
    e.evict([[3, 1, 4, 5, 9, 2, 6, 8], [10, 11]], [115, 20], 60, 7)
    (_, a), = [c for c in e.calls if c[0] == "page_summaries"]
    assert a[1].tolist() == [3 * 16 + 15, 31, 4 * 16 + 15, 10 * 16 + 15]  # 60 keys: three full pages; 20: one
    assert [c[0] for c in e.calls] == ["kv_select", "kv_compact", "page_summaries"]
    weights = e.weights[0].fill_(1.0)
    e.stage([(1, 60, 0), (1, 61, 0)], [[3, 1, 4, 5]])
    kv = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    e.selected_attention(0, torch.zeros(2, 8, 64), kv, kv, 3)
    assert (weights == 0).nonzero().tolist() == [[5, h, o] for h in range(2) for o in (12, 13)]
