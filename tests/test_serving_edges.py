"""More of what the operators around the decode refuse on the host, before anything is launched
(CPU only: the pointers are never followed)."""
import ctypes

import pytest

from mx_flash_attn_kernel_opt__b200 import _lib

A = 0x10000  # an aligned address that is never read


def evict(seq_lens, new_lens, B, k_cache=A, v_cache=A + (1 << 20), kv_format=0):
    a = _lib.PgqaEvictArgs(struct_size=ctypes.sizeof(_lib.PgqaEvictArgs), k_cache=k_cache, v_cache=v_cache,
                           weights=A, kv_format=kv_format, seq_lens=seq_lens, block_table=A, kept=A, new_lens=new_lens, batch_size=B, num_heads_k=2,
                           headdim=128, page_size=16, num_pages=9, bt_stride=4, keep=20, sinks=2, recent=4)
    return _lib.lib().pgqa_evict(ctypes.byref(a), None)


@pytest.mark.parametrize("B,off,refused", [(1, 0, True), (1, 4, False), (1, -4, False), (8, 4, True), (8, 28, True),
                                           (8, 32, False), (8, -28, True), (8, -32, False)])
def test_new_lengths_over_the_lengths_that_are_read(B, off, refused):
    """The clusters of one sequence read its length while those of another write theirs."""
    assert (evict(A, A + off, B) == 2) == refused


@pytest.mark.parametrize("off,refused", [(0, True), (16, True), (9 * 16 * 2 * 128 - 16, True), (9 * 16 * 2 * 128, False)])
@pytest.mark.parametrize("kv_format", [0, 1])
def test_k_and_v_in_one_pool(off, refused, kv_format):
    """Their rows move in place independently of each other."""
    off *= 1 if kv_format else 2
    for k, v in ((A, A + off), (A + off, A)):
        assert (evict(A, A + 64, 2, k, v, kv_format) == 2) == refused
