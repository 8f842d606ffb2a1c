"""MXFP4 pools on the CPU: the oracle's format against its definition, and what the entry points refuse
(no case reaches a launch: the addresses are placeholders)."""
import ctypes as C

import numpy as np
import pytest

from oracle import mxfp4 as M

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4
OK, E_ARG, E_ALIGN, E_WORKSPACE, E_UNSUPPORTED = 0, -20, -21, -22, -23
A, ODD = 0x100000, 0x100008


def p(x):
    return None if x is None else C.c_void_p(x)


def test_codes_are_the_nearest_values():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal((200, 64)), rng.uniform(-8, 8, (200, 64)) * 2.0 ** rng.integers(-40, 40, (200, 1))])
    x = x.astype(np.float32)
    codes, scales = M.quantise(x)
    got = M.dequantise(codes, scales)
    b = x.reshape(-1, 32).astype(np.float64)
    unit = 2.0 ** (np.floor(np.log2(np.abs(b).max(1))) - 2)
    assert np.array_equal(scales.reshape(-1), np.log2(unit) + 127)
    levels = np.concatenate([M.LEVELS, -M.LEVELS])
    best = np.abs(b[..., None] / unit[:, None, None] - levels).min(-1) * unit[:, None]
    assert np.array_equal(np.abs(got.reshape(-1, 32) - b), best)


def test_ties_go_to_even_codes_and_large_values_saturate():
    x = np.zeros((1, 32), np.float32)
    x[0, :10] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.75]  # 7.9 sets the scale to 1
    codes, scales = M.quantise(x)
    assert scales[0, 0] == 127
    assert M.dequantise(codes, scales)[0, :10].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -1.0]


def test_special_blocks():
    x = np.zeros((5, 32), np.float32)
    x[1, 3] = np.inf
    x[2, 4] = np.nan
    x[3, 5] = 1e-45
    x[4, 6] = 3e38
    codes, scales = M.quantise(x)
    assert scales[:, 0].tolist() == [0, 255, 255, 0, 252]
    assert not codes[:3].any()
    v = M.dequantise(codes, scales)
    assert np.isnan(v[1:3]).all() and not v[0].any() and np.isfinite(v[3:]).all()


def test_selection_keeps_the_recent_and_the_heaviest():
    m = np.array([1, 5, 5, 0, -0.0, 5, 2, 9, 0, 0], np.float32)
    assert M.select(m, 10, 3).tolist() == list(range(10))
    assert M.select(m, 4, 2).tolist() == [1, 7, 8, 9]
    assert M.select(m, 3, 1).tolist() == [1, 7, 9]
    assert M.select(m, 3, 3).tolist() == [7, 8, 9]
    assert M.select(m, 3, 9).tolist() == [7, 8, 9]
    assert M.select(m, 0, 0).tolist() == []
    assert M.select(m, 9, 0).tolist() == [0, 1, 2, 3, 5, 6, 7, 8, 9]  # -0 is below 0


def _append(lia, layout, **kw):
    a = dict(rows=4, slots=A, positions=None, src=BF16, k=A, v=A, kc=A, vc=A, ks=A, vs=A)
    a.update(kw)
    return lia.lib().lia_kv_append(C.byref(layout), a["rows"], p(a["positions"]), None, None, 0, p(a["slots"]),
                                   a["src"], p(a["k"]), p(a["v"]), p(a["kc"]), p(a["vc"]), p(a["ks"]), p(a["vs"]), None)


def _gather(lia, layout, **kw):
    a = dict(rows=4, slots=A, dst=BF16, ko=A, vo=A, kc=A, vc=A, ks=A, vs=A)
    a.update(kw)
    return lia.lib().lia_kv_gather(C.byref(layout), a["rows"], p(a["slots"]), p(a["kc"]), p(a["vc"]), p(a["ks"]),
                                   p(a["vs"]), a["dst"], p(a["ko"]), p(a["vo"]), None)


def _layout(lia, **kw):
    a = dict(num_kv_heads=2, head_dim=128, page_size=16, pool_pages=8, dtype=FP4)
    a.update(kw)
    return lia.KVLayout(*a.values())


@pytest.mark.parametrize("change,expect", [
    (dict(ks=None), E_ARG), (dict(vs=None), E_ARG), (dict(k=None), E_ARG), (dict(vc=None), E_ARG),
    (dict(slots=None), E_ARG), (dict(src=FP8), E_UNSUPPORTED), (dict(src=FP4), E_UNSUPPORTED),
    (dict(k=ODD), E_ALIGN), (dict(v=ODD), E_ALIGN), (dict(kc=ODD), E_ALIGN), (dict(vc=ODD), E_ALIGN),
    (dict(rows=0), OK), (dict(rows=1 << 28), E_ARG),
])
def test_append_refusals(lia, change, expect):
    assert _append(lia, _layout(lia), **change) == expect


@pytest.mark.parametrize("change,expect", [
    (dict(head_dim=48), E_UNSUPPORTED), (dict(head_dim=0), E_ARG), (dict(num_kv_heads=0), E_ARG),
    (dict(page_size=24), E_ARG), (dict(dtype=5), E_UNSUPPORTED),
])
def test_append_and_gather_refuse_layouts(lia, change, expect):
    assert _append(lia, _layout(lia, **change)) == expect
    assert _gather(lia, _layout(lia, **change)) == expect


@pytest.mark.parametrize("change,expect", [
    (dict(ks=None), E_ARG), (dict(vs=None), E_ARG), (dict(ko=None), E_ARG), (dict(slots=None), E_ARG),
    (dict(dst=FP8), E_UNSUPPORTED), (dict(dst=FP4), E_UNSUPPORTED), (dict(vo=ODD), E_ALIGN), (dict(kc=ODD), E_ALIGN),
    (dict(rows=0), OK), (dict(rows=1 << 28), E_ARG),
])
def test_gather_refusals(lia, change, expect):
    assert _gather(lia, _layout(lia), **change) == expect


def test_rope_append_refusals(lia):
    def call(layout, ks=A, kc=A, vc=A):
        return lia.lib().lia_rope_kv_append(C.byref(layout), 16, 4, None, None, None, 0, p(A), p(A), p(A), p(A), BF16,
                                            p(kc), p(vc), p(ks), p(A), None)
    assert call(_layout(lia), ks=None) == E_ARG
    assert call(_layout(lia), kc=ODD) == E_ALIGN and call(_layout(lia), vc=ODD) == E_ALIGN
    assert call(_layout(lia, head_dim=96)) == E_UNSUPPORTED


def _config(lia, **kw):
    a = dict(num_q_heads=16, num_kv_heads=2, head_dim=128, page_size=16, pool_pages=64, stride=8, q_dtype=BF16,
             kv_dtype=FP4, out_dtype=BF16, scale=0.088, max_seqs=4, max_rows=64, max_context=128)
    a.update(kw)
    return lia.AttentionConfig(*a.values())


def test_attention_refusals(lia):
    L, cfg = lia.lib(), _config(lia)
    size = lia.workspace_bytes(cfg)
    assert size > 0

    def paged(ks=A, vs=A, kc=A, ws_bytes=size, c=cfg, out=A):
        return L.lia_paged_attention(C.byref(c), 2, 2, p(A), p(A), p(A), p(A), p(A), p(kc), p(A), p(ks), p(vs), p(A),
                                     ws_bytes, p(out), None)
    assert paged(ks=None) == E_ARG and paged(vs=None) == E_ARG
    assert paged(kc=ODD) == E_ALIGN and paged(out=ODD) == E_ALIGN
    assert paged(ws_bytes=size - 1) == E_WORKSPACE
    assert paged(c=_config(lia, head_dim=96)) == E_UNSUPPORTED
    # the fused appends and the read measurement are of the other pool types
    assert L.lia_attention_partial_append(C.byref(cfg), 2, 2, p(A), p(A), p(A), p(A), p(A), p(A), p(A), p(A), size,
                                          p(A), None) == E_UNSUPPORTED
    assert L.lia_attention_partial_append_fp8(C.byref(cfg), 2, 2, p(A), p(A), p(A), p(A), p(A), p(A), p(A), p(A), p(A),
                                              p(A), size, p(A), None) == E_UNSUPPORTED
    assert L.lia_paged_read(C.byref(cfg), 2, 2, p(A), p(A), p(A), p(A), p(A), p(A), p(A), size, p(A), 1 << 20,
                            None) == E_UNSUPPORTED


def test_attention_weights_refusals(lia):
    L, cfg = lia.lib(), _config(lia)
    size = lia.attention_weights_workspace_bytes(cfg)
    assert size > 0

    def call(c=cfg, seqs=2, rows=2, cu=A, q=A, kc=A, ks=A, decay=1.0, mass=A, ws=A, ws_bytes=size):
        return L.lia_attention_weights(None if c is None else C.byref(c), seqs, rows, p(cu), p(A), p(A), p(A), p(q), p(kc),
                                       p(ks), decay, 0, p(mass), p(ws), ws_bytes, None)
    assert call(c=None) == E_ARG
    for change in (dict(seqs=0), dict(seqs=5), dict(rows=0), dict(rows=65), dict(cu=None), dict(q=None), dict(kc=None),
                   dict(ks=None), dict(mass=None), dict(ws=None), dict(decay=-1.0), dict(decay=float("nan")),
                   dict(decay=float("inf"))):
        assert call(**change) == E_ARG, change
    for change in (dict(q=ODD), dict(kc=ODD), dict(ws=ODD), dict(mass=A + 2)):
        assert call(**change) == E_ALIGN, change
    assert call(ws_bytes=size - 1) == E_WORKSPACE
    for change, expect in ((dict(num_q_heads=15), E_ARG), (dict(num_q_heads=66), E_UNSUPPORTED), (dict(head_dim=96), E_UNSUPPORTED),
                           (dict(page_size=8), E_UNSUPPORTED), (dict(q_dtype=F16), E_UNSUPPORTED), (dict(kv_dtype=F32), E_UNSUPPORTED),
                           (dict(kv_dtype=5), E_UNSUPPORTED), (dict(stride=0), E_ARG), (dict(max_context=0), E_ARG),
                           (dict(scale=0.0), E_ARG), (dict(max_rows=1 << 20), E_UNSUPPORTED)):
        bad = _config(lia, **change)
        assert call(c=bad) == expect and lia.attention_weights_workspace_bytes(bad) == 0, change


def test_attention_weights_refuse_what_32_bits_do_not_count(lia):
    """Units of work and a key's columns: contexts whose counts would wrap (a table that holds less bounds them)."""
    far = dict(max_context=0xFFFFFFFF, page_size=64)
    assert lia.attention_weights_workspace_bytes(_config(lia, **far)) > 0  # a short table
    for change in (dict(far, stride=1 << 26), dict(far, stride=1 << 24, num_q_heads=64, num_kv_heads=64, max_rows=4096)):
        assert lia.attention_weights_workspace_bytes(_config(lia, **change)) == 0, change


def test_selection_refusals(lia):
    def call(layout, seqs=2, rows=A, lengths=A, pages=A, stride=8, budget=4, recent=1, mass=A, kept=A, counts=A, ws=None,
             ws_bytes=0):
        return lia.lib().lia_kv_select(C.byref(layout), seqs, p(rows), p(lengths), p(pages), stride, budget, recent,
                                       p(mass), p(kept), p(counts), p(ws), ws_bytes, None)
    ok = _layout(lia)
    for change in (dict(rows=None), dict(lengths=None), dict(pages=None), dict(mass=None), dict(kept=None),
                   dict(counts=None), dict(stride=0), dict(budget=0), dict(seqs=1 << 30)):
        assert call(ok, **change) == E_ARG, change
    for change in (dict(mass=A + 2), dict(kept=A + 1), dict(counts=A + 2)):
        assert call(ok, **change) == E_ALIGN, change
    assert call(ok, seqs=0) == OK
    assert call(_layout(lia, num_kv_heads=0)) == E_ARG and call(_layout(lia, page_size=24)) == E_ARG
    size = lia.kv_select_workspace_bytes(ok, 2, 513)  # 8,208 keys
    assert lia.kv_select_workspace_bytes(ok, 2, 512) == 0 and size == 2 * 2 * 3 * (2 * 4096 + 8)
    assert call(ok, stride=513) == E_WORKSPACE and call(ok, stride=513, ws=A, ws_bytes=size - 1) == E_WORKSPACE
    assert call(ok, stride=513, ws=ODD, ws_bytes=size) == E_ALIGN


def test_compaction_refusals(lia):
    def call(layout, seqs=2, rows=A, pages=A, to=A, stride=8, budget=4, kept=A, counts=A, kc=A, vc=A, ks=A, vs=A, mass=A):
        return lia.lib().lia_kv_compact(C.byref(layout), seqs, p(rows), p(pages), p(to), stride, budget, p(kept),
                                        p(counts), p(kc), p(vc), p(ks), p(vs), p(mass), None)
    ok = _layout(lia)
    for change in (dict(rows=None), dict(pages=None), dict(to=None), dict(kept=None), dict(counts=None), dict(kc=None),
                   dict(vc=None), dict(ks=None), dict(vs=None), dict(stride=0), dict(budget=0), dict(budget=1 << 27)):
        assert call(ok, **change) == E_ARG, change
    for change in (dict(kc=ODD), dict(vc=ODD), dict(ks=A + 2), dict(vs=A + 1), dict(mass=A + 2)):
        assert call(ok, **change) == E_ALIGN, change
    assert call(ok, seqs=0) == OK and call(ok, seqs=0, mass=None) == OK
    assert call(_layout(lia, dtype=FP8)) == E_UNSUPPORTED and call(_layout(lia, dtype=F32)) == E_UNSUPPORTED
    assert call(_layout(lia, head_dim=96)) == E_UNSUPPORTED
    assert call(_layout(lia, dtype=BF16), seqs=0, ks=None, vs=None) == OK


def test_page_payloads(lia):
    # codes and scales of every layer and plane
    layout = _layout(lia, page_size=32)
    assert lia.lib().lia_kv_page_bytes(C.byref(layout), 3) == 3 * 2 * 32 * 2 * (64 + 4)
    assert lia.lib().lia_kv_page_bytes(C.byref(_layout(lia, head_dim=48)), 3) == 0
