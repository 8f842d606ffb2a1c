"""MXFP4 pools the attention refuses (on the CPU: no case reaches a launch, the addresses are placeholders)."""
import ctypes as C

import pytest

E_ARG, FP4, BF16 = -20, 4, 2
A = C.c_void_p(0x100000)


@pytest.mark.parametrize("rows,seqs", [(2, 2), (4, 2), (64, 2)])  # decode, verify and prompt rows
def test_a_pool_without_pages(lia, rows, seqs):
    """The decode kernel reads page 0 in the place of pages outside the pool: there has to be one."""
    cfg = lia.AttentionConfig(16, 2, 128, 16, 0, 8, BF16, FP4, BF16, 0.088, 4, 64, 128)
    size = 1 << 30
    L = lia.lib()
    assert L.lia_paged_attention(C.byref(cfg), seqs, rows, A, A, A, A, A, A, A, A, A, A, size, A, None) == E_ARG
    assert L.lia_attention_plan(C.byref(cfg), seqs, rows, A, A, A, A, A, size, None) == E_ARG
    assert L.lia_attention_partial(C.byref(cfg), seqs, rows, A, A, A, A, A, A, A, size, A, None) == E_ARG
