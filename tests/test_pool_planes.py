"""CPU tests of the planes and scales that the rotated append, the page summaries and the attention over selected pages refuse:
others than the layout's in type, size or stride, which the kernels would read or write all the same."""
import pytest
import torch

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4
E_ARG = -20
PAGES, PAGE, HKV, D = 6, 16, 2, 64


@pytest.fixture
def calls(lia, monkeypatch):
    """The names of the entry points reached; none launches."""
    got = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: got.append(name) or 0
    monkeypatch.setattr(lia, "lib", lambda: Library())
    monkeypatch.setattr(lia, "_stream", lambda s=None: None)
    return got


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _rotate(lia, kv, kc, vc, ks, vs):
    lia.qk_norm_rope_kv_append(lia.KVLayout(HKV, D, PAGE, PAGES, kv), 4, None, torch.zeros(3, 8 * D), torch.zeros(3, 4, D), kc,
                               vc, slot_mapping=i32(3), k_scales=ks, v_scales=vs)


def _summaries(lia, kv, kc, vc, ks, vs):
    lia.page_summaries(lia.KVLayout(HKV, D, PAGE, PAGES, kv), i32(3), kc, torch.zeros(PAGES, HKV, 2, D, dtype=torch.int8),
                       torch.zeros(PAGES, HKV), k_scales=ks)


def _attend(lia, kv, kc, vc, ks, vs):
    cfg = lia.AttentionConfig(4, HKV, D, PAGE, PAGES, 4, F32, kv, F32, 0.1, 2, 2, 64)
    q = torch.zeros(2, 4, D)
    lia.selected_attention(cfg, 2, i32(3), i32(2), i32(2), i32(2, 4), q, kc, vc, i32(2, HKV, 3), i32(2), q.clone(),
                           torch.zeros(1 << 20), k_scales=ks, v_scales=vs)


def _good(kv):
    if kv == FP4:
        plane, scales = torch.zeros(PAGES, HKV, PAGE, D // 2, dtype=torch.uint8), torch.zeros(PAGES, HKV, PAGE, D // 32, dtype=torch.uint8)
    elif kv == FP8:
        plane, scales = torch.zeros(PAGES, PAGE, HKV, D, dtype=torch.uint8), torch.zeros(PAGES, HKV)
    else:
        plane, scales = torch.zeros(PAGES, PAGE, HKV, D, dtype=torch.float16 if kv == F16 else torch.bfloat16), None
    return dict(kc=plane, vc=plane.clone(), ks=scales, vs=None if scales is None else scales.clone())


@pytest.mark.parametrize("call", [_rotate, _summaries, _attend])
@pytest.mark.parametrize("kv", [F16, BF16, FP8, FP4])
def test_planes(lia, calls, call, kv):
    good = _good(kv)
    plane, scales = good["kc"], good["ks"]
    bits = torch.uint8 if kv in (FP8, FP4) else torch.uint16
    larger = {k: None if x is None else torch.cat([x, x]) for k, x in good.items()}
    fine = [good, larger, {k: None if x is None else x.flatten() for k, x in good.items()},
            dict(good, kc=plane.view(bits), vc=plane.view(bits))]
    for a in fine:
        call(lia, kv, **a)
    assert len(calls) == len(fine)
    both = call is not _summaries
    other = {F16: torch.bfloat16, BF16: torch.float16}.get(kv, torch.int16)
    wrong = [plane[:-1], plane.float(), plane.to(other), torch.cat([plane, plane], -1)[..., ::2], plane.transpose(1, 2)]
    for name in ("kc", "vc") if both else ("kc",):
        for bad in wrong:
            with pytest.raises(lia.LiaError) as e:
                call(lia, kv, **dict(good, **{name: bad}))
            assert e.value.status == E_ARG, (name, bad.shape, bad.dtype)
    for name in () if scales is None else ("ks", "vs") if both else ("ks",):
        for bad in (scales[:-1], scales.half(), torch.cat([scales, scales], -1)[..., ::2]):
            with pytest.raises(lia.LiaError) as e:
                call(lia, kv, **dict(good, **{name: bad}))
            assert e.value.status == E_ARG, (name, bad.shape, bad.dtype)
    assert len(calls) == len(fine)
