"""An engine step over selected pages with budgets past its tables: every row keeps all its pages, and the lists are no longer
than a table (CPU)."""
import contextlib

import pytest
import torch

BF16 = 2


@pytest.mark.parametrize("budget,first,recent,expect", [
    (3, 1, 2, (3, 1, 2)), (16, 1, 2, (16, 1, 2)), (16, 8, 8, (16, 8, 8)), (17, 1, 2, (16, 0, 1)), (1 << 20, 0, 1, (16, 0, 1)),
    (1 << 40, 1 << 39, 1 << 39, (16, 0, 1))])
def test_budgets(lia, monkeypatch, budget, first, recent, expect):
    calls = {}
    for name in ("attention_plan", "kv_append", "page_summaries", "page_select", "selected_attention"):
        monkeypatch.setattr(lia, name, lambda *a, _name=name, **k: calls.update({_name: a}))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), dict(synchronize=lambda s: None))())
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, pin_memory=False, **k: zeros(*a, **k))
    e = lia.Engine(8, 2, 64, pool_tokens=512, page_size=16, kv_dtype=BF16, q_dtype=BF16, out_dtype=BF16, device="cpu",
                   page_summaries=True)
    e.configure_paging(4, 256)  # tables of 16 pages
    e.stage([(1, 250, 0), (1, 3, 1)], [list(range(16)), [20]])
    kv = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    e.selected_attention(0, torch.zeros(2, 8, 64, dtype=torch.bfloat16), kv, kv, budget, first, recent)
    a = calls["page_select"]
    assert tuple(a[11].shape) == tuple(calls["selected_attention"][9].shape) == (2, 2, expect[0])
    assert (a[9], a[10]) == expect[1:]
