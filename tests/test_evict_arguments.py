"""CPU tests of what Engine.evict and the selection and compaction calls make of their arguments, with the launches recorded
instead of issued."""
import contextlib

import numpy as np
import pytest
import torch


@pytest.fixture
def engine(lia, monkeypatch):
    """An engine on host memory; .calls: (name, arguments) of its launches."""
    calls = []
    for name in ("kv_select", "kv_compact"):
        monkeypatch.setattr(lia, name, lambda *a, _name=name, **k: calls.append((_name, a)))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, pin_memory=False, **k: zeros(*a, **k))
    e = lia.Engine(8, 2, 64, pool_tokens=512, page_size=16, kv_dtype=2, device="cpu", track_weights=True)
    e.configure_paging(4, 256)
    e.calls = calls
    return e


@pytest.mark.parametrize("kind", [int, np.int64, np.int32, np.uint32, np.uint64, np.uint8])
def test_numbers_of_every_kind(engine, kind):
    tables = [list(range(8)), list(range(8, 14))]
    counts, freed = engine.evict(tables, [kind(115), kind(40)], kind(60), kind(7))
    assert counts == [60, 40] and freed == [[4, 5, 6, 7], [11, 12, 13]]
    (_, select), (_, compact) = engine.calls
    assert select[2].tolist() == [115, 40] and (select[5], select[6]) == (60, 7)
    del engine.calls[:]
    array = np.array(tables[0], np.uint32)
    assert engine.evict([array], np.array([115], np.dtype(kind)), 60, 7) == ([60], [[4, 5, 6, 7]])
    assert len(engine.calls) == 2


@pytest.fixture
def selection(lia, monkeypatch):
    """kv_select and kv_compact with the library's entry points recorded: their arguments."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, a)) or 0

    monkeypatch.setattr(lia, "lib", lambda: Lib())
    monkeypatch.setattr(lia, "_stream", lambda s=None: None)
    return calls


def test_more_recent_keys_than_32_bits_count(lia, selection):
    """The entry point takes 32 bits: 2^32 of them are all of the budget, not none."""
    one, mass = torch.zeros(1, dtype=torch.int32), torch.zeros(4)
    layout = lia.KVLayout(1, 64, 16, 4, 2)
    for recent, expect in ((0, 0), (3, 3), (8, 8), (9, 8), (1 << 32, 8), ((1 << 40) + 1, 8)):
        del selection[:]
        lia.kv_select(layout, one, one, one, 4, 8, recent, mass, torch.zeros((1, 1, 8), dtype=torch.int32), one,
                      workspace=mass)
        (name, args), = selection
        assert name == "lia_kv_select" and (args[6], args[7]) == (8, expect)
    with pytest.raises(lia.LiaError) as e:
        lia.kv_select(layout, one, one, one, 4, 8, -1, mass, torch.zeros((1, 1, 8), dtype=torch.int32), one, workspace=mass)
    assert e.value.status == -20


def test_views_with_gaps_are_refused(lia, selection):
    """A kept list or an output that is a slice of a wider tensor: its rows are not where the call writes or reads them."""
    one, mass = torch.zeros(2, dtype=torch.int32), torch.zeros(4)
    layout = lia.KVLayout(2, 64, 16, 4, 2)
    wide, rows = torch.zeros((2, 2, 16), dtype=torch.int32), torch.zeros((2, 2, 128), dtype=torch.float32)
    calls = [lambda kept: lia.kv_select(layout, one, one, one, 4, 8, 2, mass, kept, one, workspace=mass),
             lambda kept: lia.kv_compact(layout, one, one, one, 4, kept, one, mass, mass)]
    for call in calls:
        call(wide[:, :, :8].contiguous())
        with pytest.raises(lia.LiaError) as e:
            call(wide[:, :, :8])
        assert e.value.status == -20
    lia.kv_gather(layout, one, mass, mass, rows[..., :64].contiguous(), rows[..., :64].contiguous())
    for pair in ((rows[..., :64], rows), (rows, rows[..., :64])):
        with pytest.raises(lia.LiaError):
            lia.kv_gather(layout, one, mass, mass, *pair)
    assert len(selection) == 3


def test_an_engine_whose_weights_are_refused_is_not_configured(lia, monkeypatch):
    """The weights' kernels take heads of 64 and 128: the refusal leaves paging as it was."""
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, pin_memory=False, **k: zeros(*a, **k))
    e = lia.Engine(8, 2, 96, pool_tokens=512, page_size=16, kv_dtype=2, device="cpu", track_weights=True)
    for _ in range(2):
        with pytest.raises(lia.LiaError) as err:
            e.configure_paging(4, 256)
        assert err.value.status == -23 and e.paging is None
