"""CPU tests of the keys and values that an engine's step takes: rows of one type and of all KV heads; slices of wider rows are
appended as the values they hold."""
import contextlib

import pytest
import torch

F16, BF16 = 1, 2
E_ARG = -20


@pytest.fixture
def engine(lia, monkeypatch):
    """An engine on host memory; .calls: (name, arguments) of its launches."""
    calls = []
    for name in ("attention_plan", "attention_partial", "attention_partial_append", "attention_merge", "page_summaries",
                 "page_select", "selected_attention", "paged_attention"):
        monkeypatch.setattr(lia, name, lambda *a, _name=name, **k: calls.append((_name, a)))

    class Library:
        def __init__(self, library):
            self.library = library

        def __getattr__(self, name):
            if name == "lia_kv_append":
                return lambda *a: calls.append(("kv_append", a)) or 0
            return getattr(self.library, name)
    library = Library(lia.lib())
    monkeypatch.setattr(lia, "lib", lambda: library)
    monkeypatch.setattr(lia, "_stream", lambda s=None: None)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), dict(synchronize=lambda s: None))())
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, pin_memory=False, **k: zeros(*a, **k))
    e = lia.Engine(8, 2, 64, pool_tokens=512, page_size=16, kv_dtype=BF16, q_dtype=BF16, out_dtype=BF16, device="cpu",
                   page_summaries=True)
    e.configure_paging(4, 256)
    e.stage([(1, 5, 0), (1, 6, 0), (1, 7, 1)], [[0], [1]])
    del calls[:]
    e.calls = calls
    return e


def _attention(e, k, v):
    e.attention(0, torch.zeros(3, 8, 64, dtype=torch.bfloat16), k, v)


def _selected(e, k, v):
    e.selected_attention(0, torch.zeros(3, 8, 64, dtype=torch.bfloat16), k, v, 4)


@pytest.mark.parametrize("call", [_attention, _selected])
@pytest.mark.parametrize("k,v", [
    (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)])
def test_types_that_differ(lia, engine, call, k, v):
    """The append reads both in one type: the values, or past the shorter one's end."""
    with pytest.raises(lia.LiaError) as e:
        call(engine, torch.zeros(3, 2, 64, dtype=k), torch.zeros(3, 2, 64, dtype=v))
    assert e.value.status == E_ARG and not engine.calls


@pytest.mark.parametrize("call", [_attention, _selected])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_fewer_heads(lia, engine, call, dtype):
    good = torch.zeros(3, 2, 64, dtype=dtype)
    for bad in (good[:, :1], good[:2], torch.zeros(3, 32, dtype=dtype)):
        for k, v in ((bad, good), (good, bad), (bad, bad)):
            with pytest.raises(lia.LiaError) as e:
                call(engine, k, v)
            assert e.value.status == E_ARG and not engine.calls


@pytest.mark.parametrize("call", [_attention, _selected])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_slices_of_wider_rows(lia, engine, call, dtype, monkeypatch):
    """k and v as they lie in a projection's rows."""
    x = torch.arange(3 * 12 * 64).reshape(3, 12 * 64).to(dtype)
    seen = []
    append = lia.kv_append
    monkeypatch.setattr(lia, "kv_append", lambda layout, k, v, *a, **m: seen.append((k, v)) or append(layout, k, v, *a, **m))
    monkeypatch.setattr(lia, "attention_partial_append", lambda c, n, p, s, q, k, v, *a, **m: seen.append((k, v)))
    call(engine, x[:, 8 * 64:10 * 64], x[:, 10 * 64:].unflatten(1, (2, 64)))
    (k, v), = seen
    assert k.is_contiguous() and v.is_contiguous() and k.shape == v.shape == (3, 128)
    assert torch.equal(k, x[:, 8 * 64:10 * 64]) and torch.equal(v, x[:, 10 * 64:])


def test_append_itself(lia, engine):
    layout = lia.KVLayout(2, 64, 16, 32, BF16)
    k = torch.zeros(3, 128)
    planes = [torch.zeros(512, 2, 64, dtype=torch.bfloat16) for _ in range(2)]
    slots = torch.zeros(3, dtype=torch.int32)
    for a, b in ((k, k), (k.view(3, 2, 64), k), (torch.zeros(3, 256), torch.zeros(3, 256)), (k[:0], k[:0])):
        lia.kv_append(layout, a, b, *planes, slot_mapping=slots)
    assert len(engine.calls) == 4
    for a, b in ((k, k.half()), (k.bfloat16(), k), (k, k[:2]), (k[:, :64].contiguous(), k), (torch.zeros(128, 3).t(), k),
                 (k, torch.zeros(3, 256)[:, ::2])):
        with pytest.raises(lia.LiaError) as e:
            lia.kv_append(layout, a, b, *planes, slot_mapping=slots)
        assert e.value.status == E_ARG
    assert len(engine.calls) == 4
