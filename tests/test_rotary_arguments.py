"""CPU tests of the rotation frequencies and of what the rotation's entry points refuse: every case breaks one thing of a call
that passes, and none reaches a launch (the addresses are placeholders)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import sparse as S

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4
E_ARG, E_ALIGN, E_UNSUPPORTED = -20, -21, -23
A = 0x100000


@pytest.mark.parametrize("n", [2, 4, 16, 32, 64, 80, 96, 128])
@pytest.mark.parametrize("base", [1.5, 1e4, 5e6])
@pytest.mark.parametrize("how", [{}, dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
                                 dict(scaling="turns", factor=8.0, context=8192, low=1.0, high=4.0),
                                 dict(scaling="index", factor=40.0, context=4096),
                                 dict(scaling="index", factor=1.0, context=3, low=1e-3, high=1e3)])
def test_frequencies(lia, n, base, how):
    if n == 2 and how.get("scaling") == "base":
        with pytest.raises(lia.LiaError):
            lia.rope_frequencies(n, base, **how)
        return
    got, ref = lia.rope_frequencies(n, base, **how), S.frequencies(n, base, **how)
    # powers and logarithms are within a few units of 2^-53; exponents of up to 23 bits and the ramps' quotients magnify it
    assert got.shape == (n // 2,) and got.dtype == np.float64
    assert np.abs(got / ref - 1).max() < 1e-11


def test_ramps_end_at_the_plain_and_the_stretched(lia):
    """The fastest pair of a long rotation keeps its frequency, the slowest is stretched by the whole factor."""
    plain = lia.rope_frequencies(128, 1e4)
    for scaling in ("turns", "index"):
        f = lia.rope_frequencies(128, 1e4, scaling, factor=16.0, context=4096)
        assert f[0] == plain[0] and math.isclose(f[-1], plain[-1] / 16, rel_tol=1e-12)
        assert (np.diff(f) < 0).all()


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=3), dict(base=1.0), dict(base=math.nan), dict(base=math.inf),
                                 dict(scaling=1, factor=0.5), dict(scaling=1, factor=math.nan),
                                 dict(scaling=2, factor=math.inf), dict(scaling=2, factor=1e300, base=1e300),
                                 dict(scaling=3, context=0.0), dict(scaling=3, low=0.0),
                                 dict(scaling=4, low=2.0, high=2.0), dict(scaling=4, high=math.inf), dict(out=None)])
def test_frequencies_refused(lia, bad):
    out = np.zeros(64)
    a = dict(n=64, base=1e4, scaling=0, factor=2.0, context=4096.0, low=1.0, high=32.0, out=out.ctypes.data)
    a.update(bad)
    assert lia.lib().lia_rope_frequencies(*a.values()) == E_ARG
    assert lia.lib().lia_rope_frequencies(64, 1e4, 5, 2.0, 4096.0, 1.0, 32.0, out.ctypes.data) == E_UNSUPPORTED
    with pytest.raises(lia.LiaError):
        lia.rope_frequencies(64, scaling="other")
    for n in (0, -1, -4, 1 << 32, (1 << 32) + 4):
        with pytest.raises(lia.LiaError):
            lia.rope_frequencies(n)


@pytest.mark.parametrize("bad,status", [(dict(positions=None), E_ARG), (dict(f=None), E_ARG), (dict(out=None), E_ARG),
                                        (dict(n=0), E_UNSUPPORTED), (dict(n=66), E_UNSUPPORTED),
                                        (dict(out=A + 8), E_ALIGN), (dict(f=A + 4), E_ALIGN),
                                        (dict(rows=1 << 31), E_ARG)])
def test_table_refused(lia, bad, status):
    a = dict(rows=4, n=64, positions=A, f=A, attention=1.0, out=A, stream=None)
    a.update(bad)
    assert lia.lib().lia_rope_table(*a.values()) == status


def test_table_of_no_rows(lia):
    assert lia.lib().lia_rope_table(0, 64, A, A, 1.0, A, None) == 0


ROTATE = dict(hq=16, rows=4, positions=None, sequences=None, pages=None, stride=0, slots=A, n=64, interleaved=0, table=A,
              wq=A, wk=A, wt=BF16, eps=1e-6, x=A, xt=BF16, xs=20 * 128, q=A, qt=BF16, kc=A, vc=A, ks=None, vs=None,
              stream=None)
LAYOUT = dict(hkv=2, d=128, page=16, pool=64, dtype=BF16)


def _rotate(lia, **bad):
    layout, a = dict(LAYOUT), dict(ROTATE)
    for k, v in bad.items():
        (layout if k in layout else a)[k] = v
    return lia.lib().lia_qk_norm_rope_kv_append(C.byref(lia.KVLayout(*layout.values())), *a.values())


@pytest.mark.parametrize("bad,status", [
    (dict(hq=0), E_ARG), (dict(hkv=0), E_ARG), (dict(page=0), E_ARG), (dict(page=24), E_ARG), (dict(d=96), E_UNSUPPORTED),
    (dict(d=256), E_UNSUPPORTED), (dict(dtype=F32), E_UNSUPPORTED), (dict(dtype=9), E_UNSUPPORTED), (dict(n=8), E_UNSUPPORTED),
    (dict(n=136), E_UNSUPPORTED), (dict(n=144), E_UNSUPPORTED), (dict(qt=F16), E_UNSUPPORTED), (dict(xt=FP8), E_UNSUPPORTED),
    (dict(wt=FP8), E_UNSUPPORTED), (dict(table=None), E_ARG), (dict(eps=-1.0), E_ARG), (dict(eps=math.nan), E_ARG),
    (dict(slots=None), E_ARG), (dict(slots=None, positions=A, sequences=A, pages=A), E_ARG), (dict(x=None), E_ARG),
    (dict(q=None), E_ARG), (dict(kc=None), E_ARG), (dict(vc=None), E_ARG), (dict(dtype=FP8), E_ARG),
    (dict(dtype=FP4, ks=A), E_ARG), (dict(x=A + 8), E_ALIGN), (dict(q=A + 8), E_ALIGN), (dict(kc=A + 8), E_ALIGN),
    (dict(vc=A + 4), E_ALIGN), (dict(table=A + 8), E_ALIGN), (dict(wq=A + 2), E_ALIGN), (dict(wk=A + 2), E_ALIGN),
    (dict(xs=20 * 128 - 8), E_ARG), (dict(xs=20 * 128 + 4), E_ALIGN), (dict(rows=1 << 30), E_ARG),
    (dict(rows=1 << 22, xs=1 << 40), E_ARG), (dict(hq=1 << 25, xs=1 << 33), E_ARG)])
def test_rotate_refused(lia, bad, status):
    assert _rotate(lia, **bad) == status


@pytest.mark.parametrize("fine", [dict(), dict(wq=None, wk=None, wt=77, eps=-1.0), dict(n=0, table=None), dict(n=128),
                                  dict(dtype=FP8, ks=A, vs=A), dict(dtype=FP4, ks=A, vs=A), dict(xs=1 << 20),
                                  dict(slots=None, positions=A, sequences=A, pages=A, stride=4), dict(d=64, n=64)])
def test_rotate_of_no_rows(lia, fine):
    assert _rotate(lia, rows=0, **fine) == 0


def test_wrapper_refuses(lia, monkeypatch):
    """What the entry point cannot see: lengths, strides and types of the tensors."""
    monkeypatch.setattr(lia, "_stream", lambda s=None: None)
    layout = lia.KVLayout(2, 64, 16, 4, BF16)
    good = dict(table=torch.zeros(3, 16, 2), combined=torch.zeros(3, 8 * 64), query=torch.zeros(3, 4, 64),
                kc=torch.zeros(4), vc=torch.zeros(4), q_weight=torch.ones(64), k_weight=torch.ones(64))
    for bad in (dict(combined=torch.zeros(3, 7 * 64)), dict(combined=torch.zeros(8 * 64, 3).t()),
                dict(query=torch.zeros(2, 4, 64)), dict(query=torch.zeros(3, 4, 128)[..., ::2]),
                dict(table=torch.zeros(2, 16, 2)), dict(table=torch.zeros(3, 16, 2, dtype=torch.float64)),
                dict(table=torch.zeros(3, 32)), dict(q_weight=torch.ones(32)), dict(k_weight=torch.ones(64).bfloat16()),
                dict(k_weight=torch.ones(128)[::2])):
        a = dict(good, **bad)
        with pytest.raises(lia.LiaError) as e:
            lia.qk_norm_rope_kv_append(layout, 4, a.pop("table"), a.pop("combined"), a.pop("query"), a.pop("kc"),
                                       a.pop("vc"), slot_mapping=torch.zeros(3, dtype=torch.int32), **a)
        assert e.value.status == E_ARG
    f = torch.zeros(16, dtype=torch.float64)
    for args in ((f.float(), torch.zeros(3, 16, 2)), (f, torch.zeros(3, 15, 2)), (f[::2], torch.zeros(3, 8, 2)),
                 (f, torch.zeros(3, 16, 2, dtype=torch.float64))):
        with pytest.raises(lia.LiaError):
            lia.rope_table(torch.zeros(3, dtype=torch.int32), *args)
    for positions in (torch.zeros(3, dtype=torch.int64), torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(lia.LiaError):
            lia.rope_table(positions, f, torch.zeros(3, 16, 2))
    a = dict(good, stride=4, pages=torch.zeros(16, dtype=torch.int32))
    args = [layout, 4] + [a.pop(k) for k in ("table", "combined", "query", "kc", "vc")]
    i32 = torch.zeros(3, dtype=torch.int32)
    for slots in (dict(slot_mapping=i32[:2]), dict(slot_mapping=i32.long()), dict(positions=i32, sequences=i32[:2]),
                  dict(positions=i32.long(), sequences=i32), dict(positions=i32, sequences=i32.repeat(2)[::2])):
        with pytest.raises(lia.LiaError):
            lia.qk_norm_rope_kv_append(*args, **a, **slots)
