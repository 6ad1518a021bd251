"""More of what the operators around the decode refuse on the host, before anything is launched
(CPU only: the pointers are never followed)."""
import ctypes

import pytest

from mx_flash_attn_kernel_opt__b200 import _lib

A = 0x10000  # an aligned address that is never read


def evict(seq_lens, new_lens, B):
    a = _lib.PgqaEvictArgs(struct_size=ctypes.sizeof(_lib.PgqaEvictArgs), k_cache=A, v_cache=A, weights=A,
                           seq_lens=seq_lens, block_table=A, kept=A, new_lens=new_lens, batch_size=B, num_heads_k=2,
                           headdim=128, page_size=16, num_pages=9, bt_stride=4, keep=20, sinks=2, recent=4)
    return _lib.lib().pgqa_evict(ctypes.byref(a), None)


@pytest.mark.parametrize("B,off,refused", [(1, 0, True), (1, 4, False), (1, -4, False), (8, 4, True), (8, 28, True),
                                           (8, 32, False), (8, -28, True), (8, -32, False)])
def test_new_lengths_over_the_lengths_that_are_read(B, off, refused):
    """The clusters of one sequence read its length while those of another write theirs."""
    assert (evict(A, A + off, B) == 2) == refused
