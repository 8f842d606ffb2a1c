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
