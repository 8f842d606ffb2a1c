"""CPU tests of what the calls over selected pages and the rotated append refuse of a step's metadata: the kernels read it as
32-bit words one behind the other, without a length."""
import pytest
import torch

F32, F16, BF16, FP8, FP4 = 0, 1, 2, 3, 4
E_ARG = -20


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


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


CONFIG = dict(num_q_heads=16, num_kv_heads=2, head_dim=128, page_size=16, pool_pages=64, stride=8, q_dtype=BF16,
              kv_dtype=BF16, out_dtype=BF16, scale=0.088, max_seqs=4, max_rows=8, max_context=128)
WRONG = [dict(positions=i32(1)), dict(positions=i32(4)[::2]), dict(positions=torch.zeros(2)), dict(positions=i32(2).long()),
         dict(positions=i32(4).short()), dict(sequences=i32(1)), dict(sequences=i32(2).long()), dict(sequences=i32(4)[::2]),
         dict(sequences=torch.zeros(2)), dict(cu=i32(2)), dict(cu=i32(3).long()), dict(cu=i32(6)[::2]), dict(cu=torch.zeros(3)),
         dict(pages=i32(7)), dict(pages=i32(12)), dict(pages=i32(0)), dict(pages=i32(4, 16)[:, ::2]), dict(pages=i32(8, 4).t()),
         dict(pages=i32(4, 8).long()), dict(pages=torch.zeros(4, 8))]


def _step(lia, **more):
    a = dict(cu=i32(3), positions=i32(2), sequences=i32(2), pages=i32(4, 8))
    a.update(more)
    return lia.AttentionConfig(*CONFIG.values()), 2, a["cu"], a["positions"], a["sequences"], a["pages"]


def _select(lia, selected=None, counts=None, **more):
    codes, scales = torch.zeros(64, 2, 2, 128, dtype=torch.int8), torch.zeros(64, 2)
    lia.page_select(*_step(lia, **more), torch.zeros(2, 16, 128, dtype=torch.bfloat16), codes, scales, 1, 1,
                    i32(2, 2, 4) if selected is None else selected, i32(2) if counts is None else counts, torch.zeros(4096))


def _attend(lia, selected=None, counts=None, **more):
    q, plane = torch.zeros(2, 16, 128, dtype=torch.bfloat16), torch.zeros(64, 16, 2, 128, dtype=torch.bfloat16)
    lia.selected_attention(*_step(lia, **more), q, plane, plane.clone(), i32(2, 2, 4) if selected is None else selected,
                           i32(2) if counts is None else counts, q.clone(), torch.zeros(1 << 22))


@pytest.mark.parametrize("call,entry", [(_select, "lia_page_select"), (_attend, "lia_selected_attention")])
def test_step(lia, calls, call, entry):
    for fine in (dict(), dict(pages=i32(32)), dict(pages=i32(1, 8)), dict(cu=i32(9), positions=i32(7), sequences=i32(7)),
                 dict(positions=i32(2).view(torch.uint32))):
        call(lia, **fine)
        assert calls.pop() == entry
    for bad in WRONG + [dict(selected=torch.zeros(2, 2, 4)), dict(counts=torch.zeros(2)), dict(counts=i32(4)[::2])]:
        with pytest.raises(lia.LiaError) as e:
            call(lia, **bad)
        assert e.value.status == E_ARG and entry[4:] in str(e.value) and not calls, bad


def test_slots_of_summaries(lia, calls):
    layout = lia.KVLayout(2, 128, 16, 64, BF16)
    kc, codes, scales = torch.zeros(64, 16, 2, 128, dtype=torch.bfloat16), torch.zeros(64, 2, 2, 128, dtype=torch.int8), torch.zeros(64, 2)
    lia.page_summaries(layout, i32(3), kc, codes, scales)
    lia.page_summaries(layout, i32(0), kc, codes, scales)
    assert calls == ["lia_page_summaries"] * 2
    for slots in (torch.zeros(3), i32(6)[::2], i32(3).long()):
        with pytest.raises(lia.LiaError) as e:
            lia.page_summaries(layout, slots, kc, codes, scales)
        assert e.value.status == E_ARG
    assert len(calls) == 2


def test_rotated_append(lia, calls):
    layout = lia.KVLayout(2, 64, 16, 4, BF16)
    planes = [torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16) for _ in range(2)]
    args = [layout, 4, torch.zeros(3, 16, 2), torch.zeros(3, 8 * 64), torch.zeros(3, 4, 64), *planes]
    table = dict(positions=i32(3), sequences=i32(3), pages=i32(4, 4), stride=4)
    lia.qk_norm_rope_kv_append(*args, **table)
    lia.qk_norm_rope_kv_append(*args, slot_mapping=i32(3))
    lia.rope_table(i32(3), torch.zeros(16, dtype=torch.float64), torch.zeros(3, 16, 2))
    assert calls == ["lia_qk_norm_rope_kv_append"] * 2 + ["lia_rope_table"]
    del calls[:]
    for bad in (dict(positions=torch.zeros(3)), dict(sequences=torch.zeros(3)), dict(pages=i32(15)), dict(pages=i32(3)),
                dict(pages=i32(4, 4).t()), dict(pages=i32(16).long()), dict(pages=torch.zeros(16)), dict(pages=i32(0)),
                dict(slot_mapping=torch.zeros(3))):
        with pytest.raises(lia.LiaError) as e:
            lia.qk_norm_rope_kv_append(*args, **dict(table, **bad))
        assert e.value.status == E_ARG, bad
    with pytest.raises(lia.LiaError):
        lia.rope_table(torch.zeros(3), torch.zeros(16, dtype=torch.float64), torch.zeros(3, 16, 2))
    assert not calls
