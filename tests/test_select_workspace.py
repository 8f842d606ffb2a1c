"""kv_select without a workspace allocates one that belongs to the stream it runs on: memory of the current stream's pool may
still be in use by work queued there."""
import contextlib
import ctypes as C
import types

import numpy as np
import pytest
import torch


def test_the_workspace_is_the_streams_own(lia, monkeypatch):
    """On host memory, the launch recorded: the allocation happens inside the stream's context."""
    inside, made, calls = [], [], []

    @contextlib.contextmanager
    def on(stream):
        inside.append(stream)
        yield
        inside.pop()

    empty = torch.empty
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: (made.append(inside[-1] if inside else "current"), empty(*a, **k))[1])
    real = lia.lib()
    select = lambda *a: calls.append((a[-3], a[-2], a[-1])) or 0  # noqa: E731
    monkeypatch.setattr(lia, "lib", lambda: types.SimpleNamespace(
        lia_kv_select=select, lia_kv_select_workspace_bytes=real.lia_kv_select_workspace_bytes))
    layout = lia.KVLayout(2, 128, 16, 4096, 2)
    one = torch.zeros(1, dtype=torch.int32)
    kept, mass = torch.zeros((1, 2, 8), dtype=torch.int32), torch.zeros(4)
    stream = types.SimpleNamespace(cuda_stream=77)
    for stride, expect in ((513, [stream]), (512, [])):
        del made[:]
        lia.kv_select(layout, one, one, one, stride, 8, 0, mass, kept, one, stream=stream)
        assert made == expect
    assert calls[0][1] == real.lia_kv_select_workspace_bytes(C.byref(layout), 1, 513) and calls[0][0] and calls[0][2] == 77
    assert calls[1][1] == 0 and calls[1][0] is None


@pytest.mark.gpu
def test_selection_while_the_current_stream_works(lia):
    """The current stream gives back a block of the workspace's size with writes to it still queued; the selection on
    another stream has the bits of the default call's."""
    rng = np.random.default_rng(3)
    hkv, page, n, budget = 2, 64, 60000, 900
    stride = -(-n // page)
    layout = lia.KVLayout(hkv, 128, page, stride, 2)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.uint32).view(np.int32)).cuda()  # noqa: E731
    table, rows, held = dev(rng.permutation(stride)), dev([0]), dev([n])
    mass = torch.from_numpy(rng.random((stride, hkv, page)).astype(np.float32)).cuda()
    size = lia.kv_select_workspace_bytes(layout, 1, stride)
    outs = [(torch.zeros((1, hkv, budget), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
            for _ in range(2)]
    s = torch.cuda.Stream()
    lia.kv_select(layout, rows, held, table, stride, budget, 100, mass, *outs[0])
    torch.cuda.synchronize()
    print("[case] selection beside queued work", flush=True)
    block = torch.empty(size, dtype=torch.uint8, device="cuda")
    for i in range(200):
        block.fill_(i)
    del block
    lia.kv_select(layout, rows, held, table, stride, budget, 100, mass, *outs[1], stream=s)
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a, b)
