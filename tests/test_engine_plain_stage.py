"""An engine without page summaries stages and attends without the work that they take (CPU)."""
import contextlib

import pytest
import torch

BF16 = 2


@pytest.mark.parametrize("summaries", [False, True])
def test_completed_pages_are_looked_for_where_summaries_are_kept(lia, monkeypatch, summaries):
    asked = []
    for name in ("attention_plan", "attention_partial", "attention_partial_append", "attention_merge", "kv_append",
                 "page_summaries"):
        monkeypatch.setattr(lia, name, lambda *a, **k: None)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), dict(synchronize=lambda s: None))())
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: asked.append(1) and False)
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, pin_memory=False, **k: zeros(*a, **k))
    e = lia.Engine(8, 2, 64, pool_tokens=512, page_size=16, kv_dtype=BF16, q_dtype=BF16, out_dtype=BF16, device="cpu",
                   page_summaries=summaries)
    e.configure_paging(4, 256)
    rows = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    for position, completes in ((14, False), (15, summaries)):
        e.stage([(1, position, 0)], [[3]])
        assert e.paging["completes"] is completes
        del asked[:]
        e.attention(0, torch.zeros(1, 8, 64), rows, rows)
        assert len(asked) == 1 + (summaries and not completes)  # attention()'s own, and that of the summaries
