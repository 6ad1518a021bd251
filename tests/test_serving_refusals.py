"""What the operators around the decode refuse, on the host, before anything is launched
(CPU only: the pointers are never followed)."""
import ctypes

import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from mx_flash_attn_kernel_opt__b200 import _lib

A = 0x10000  # an aligned address that is never read


def rope(**kw):
    a = _lib.PgqaRopeArgs(struct_size=ctypes.sizeof(_lib.PgqaRopeArgs), q=A, k_new=A, v_new=A, q_out=A,
                          k_cache=A, v_cache=A, seq_lens=A, block_table=A, cos=A, sin=A, positions=A,
                          batch_size=2, seqlen=3, tokens=6, num_heads=8, num_heads_k=2, headdim=128,
                          page_size=16, num_pages=9, bt_stride=4, q_strides=(2048, 1024, 128),
                          k_strides=(768, 256, 128), v_strides=(768, 256, 128), table_rows=100,
                          rotary_dim=128, num_axes=1)
    for n, v in kw.items():
        setattr(a, n, v)
    return _lib.lib().pgqa_rope_append(ctypes.byref(a), None)


@pytest.mark.parametrize("status,kw", [
    (2, dict(struct_size=8)), (1, dict(q=None, k_new=None, v_new=None)), (1, dict(q_out=None)),
    (1, dict(v_new=None)), (1, dict(cos=None)), (1, dict(seq_lens=None)), (1, dict(block_table=None)),
    (1, dict(k_cache=None)), (2, dict(batch_size=0)), (2, dict(tokens=7)), (2, dict(tokens=-6, seqlen=-3)),
    (3, dict(headdim=64)), (3, dict(page_size=24)), (2, dict(page_size=0)), (2, dict(num_pages=0)),
    (2, dict(bt_stride=0)), (3, dict(num_pages=1 << 27)), (2, dict(rotary_dim=0)), (2, dict(rotary_dim=256)),
    (3, dict(rotary_dim=40)), (2, dict(num_axes=0)), (2, dict(num_axes=65)), (2, dict(table_rows=0)),
    (1, dict(num_axes=2, positions=None)), (2, dict(pair_axis=(ctypes.c_uint8 * 64)(*[1] * 64))),
    (3, dict(kv_format=2)), (3, dict(table_format=2)), (2, dict(k_scale=A)),
    (4, dict(q_strides=(ctypes.c_int64 * 3)(2048, 1020, 128))), (4, dict(v_strides=(ctypes.c_int64 * 3)(0, -256, 128))),
    (4, dict(q=A + 8)), (4, dict(k_cache=A + 4)), (4, dict(positions=A + 2)), (4, dict(cos=A + 4)),
    (2, dict(num_heads=0)), (2, dict(num_heads=70000)),
    (2, dict(k_new=None, v_new=None, weights=A)),
])
def test_rope_append(status, kw):
    assert rope(**kw) == status
    assert _lib.lib().pgqa_last_status() == status


def test_packed_structs_match_the_mirrors():
    from mx_flash_attn_kernel_opt__b200 import serving
    for packed, mirror in ((serving._ROPE, _lib.PgqaRopeArgs), (serving._WEIGHTS, _lib.PgqaWeightsArgs),
                           (serving._EVICT, _lib.PgqaEvictArgs), (serving._CROSS, _lib.PgqaCrossArgs)):
        assert packed.size == ctypes.sizeof(mirror)


def test_rope_append_null_struct():
    assert _lib.lib().pgqa_rope_append(None, None) == 1


def weights(**kw):
    a = _lib.PgqaWeightsArgs(struct_size=ctypes.sizeof(_lib.PgqaWeightsArgs), q=A, k_cache=A, softmax_lse=A,
                             weights=A, seq_lens=A, block_table=A, batch_size=2, seqlen_q=1, num_heads=8,
                             num_heads_k=2, headdim=128, page_size=16, num_pages=9, bt_stride=4, scale=0.1)
    for n, v in kw.items():
        setattr(a, n, v)
    return _lib.lib().pgqa_accumulate_weights(ctypes.byref(a), None)


@pytest.mark.parametrize("status,kw", [
    (2, dict(struct_size=8)), (1, dict(q=None)), (1, dict(softmax_lse=None)), (1, dict(weights=None)),
    (2, dict(num_heads=9)), (2, dict(num_heads=0)), (2, dict(seqlen_q=0)), (3, dict(seqlen_q=5000)),
    (2, dict(causal=2)), (2, dict(scale=0.0)), (2, dict(scale=float("nan"))), (2, dict(scale=float("inf"))),
    (3, dict(kv_format=3)), (2, dict(k_scale=A)), (4, dict(q=A + 2)), (4, dict(weights=A + 2)),
    (3, dict(headdim=256)), (3, dict(page_size=20)), (2, dict(batch_size=-1)), (3, dict(bt_stride=1 << 27)),
])
def test_accumulate_weights(status, kw):
    assert weights(**kw) == status


def evict(**kw):
    a = _lib.PgqaEvictArgs(struct_size=ctypes.sizeof(_lib.PgqaEvictArgs), k_cache=A, v_cache=A, weights=A,
                           seq_lens=A, block_table=A, kept=A, new_lens=A + 64, batch_size=2, num_heads_k=2,
                           headdim=128, page_size=16, num_pages=9, bt_stride=4, keep=20, sinks=2, recent=4)
    for n, v in kw.items():
        setattr(a, n, v)
    return _lib.lib().pgqa_evict(ctypes.byref(a), None)


@pytest.mark.parametrize("status,kw", [
    (2, dict(struct_size=8)), (1, dict(k_cache=None)), (1, dict(weights=None)), (1, dict(kept=None)),
    (1, dict(new_lens=None)), (2, dict(keep=0)), (2, dict(keep=1 << 31)), (2, dict(sinks=-1)),
    (2, dict(recent=-1)), (2, dict(sinks=21)), (2, dict(sinks=10, recent=11)), (3, dict(kv_format=2)),
    (4, dict(v_cache=A + 8)), (4, dict(kept=A + 2)), (4, dict(weights=A + 8)), (4, dict(weights_out=A + 4)), (2, dict(new_lens=A)), (3, dict(headdim=64)),
    (3, dict(batch_size=1 << 20, num_heads_k=1 << 9)),
])
def test_evict(status, kw):
    assert evict(**kw) == status


def test_python_entry_points_refuse_cpu_tensors():
    z = torch.zeros
    k = z(4, 16, 2, 128, dtype=torch.bfloat16)
    bt, lens = z(2, 2, dtype=torch.int32), z(2, dtype=torch.int32)
    q, kn = z(2, 8, 128, dtype=torch.bfloat16), z(2, 2, 128, dtype=torch.bfloat16)
    t = z(8, 64)
    with pytest.raises(ValueError, match="CUDA"):
        pgqa.rope_append_kv(q, kn, kn, k, k, bt, lens, t, t)
    with pytest.raises(ValueError, match="required"):
        pgqa.rope_append_kv(q, None, None, k, k, bt, lens, t, t)
    with pytest.raises(ValueError, match="CUDA"):
        pgqa.accumulate_weights(q, k, bt, lens, z(2, 8, 1), z(4, 2, 16))
    with pytest.raises(ValueError, match="CUDA"):
        pgqa.evict_kv(k, k, z(4, 2, 16), bt, lens, 4)


@pytest.mark.gpu
def test_python_entry_points_refuse_bad_tensors(cuda_device):
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=cuda_device)  # noqa: E731
    bf, i32 = torch.bfloat16, torch.int32
    k = z(4, 16, 2, 128, dtype=bf)
    bt, lens, w = z(2, 2, dtype=i32), z(2, dtype=i32), z(4, 2, 16)
    q, kn, t, pos = z(2, 8, 128, dtype=bf), z(2, 2, 128, dtype=bf), z(8, 64), z(3, 2, dtype=i32)
    lse = z(2, 8, 1)

    def rope(**kw):
        a = dict(q=q, k_new=kn, v_new=kn, k_cache=k, v_cache=k, block_table=bt, seq_lens=lens, cos=t, sin=t)
        a.update(kw)
        return pgqa.rope_append_kv(**a)

    for error, kw in (
            (TypeError, dict(q=q.float())), (TypeError, dict(k_new=kn.half())),
            (TypeError, dict(seq_lens=lens.long())), (TypeError, dict(cos=t.half(), sin=t.half())),
            (TypeError, dict(positions=pos[0].long())), (ValueError, dict(positions=pos)),
            (ValueError, dict(k_scale=1.0)), (ValueError, dict(sin=t.cpu())),
            (ValueError, dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))),
            (pgqa.PgqaError, dict(q=q[:1])), (pgqa.PgqaError, dict(k_new=q)),
            (pgqa.PgqaError, dict(positions=pos, axes=[0, 1, 2])),
            (pgqa.PgqaError, dict(positions=pos, axes=[3] * 64)),
            (pgqa.PgqaError, dict(positions=z(3, 5, dtype=i32), axes=[0] * 64)),
            (pgqa.PgqaError, dict(cos=z(8, 60), sin=z(8, 60))), (pgqa.PgqaError, dict(sin=z(7, 64))),
            (pgqa.PgqaError, dict(weights=z(4, 16, 2))), (pgqa.PgqaError, dict(q_out=z(2, 4, 128, dtype=bf))),
            (pgqa.PgqaError, dict(cu_seqlens=z(2, dtype=i32)))):
        with pytest.raises(error):
            rope(**kw)
    for error, args in (
            (TypeError, (q.float(), k, bt, lens, lse, w)), (TypeError, (q, k, bt, lens, lse.half(), w)),
            (pgqa.PgqaError, (q, k, bt, lens, z(2, 1, 8), w)), (pgqa.PgqaError, (q, k, bt, lens[:1], lse, w)),
            (pgqa.PgqaError, (q[:, :7].contiguous(), k, bt, lens, z(2, 7, 1), w)),
            (pgqa.PgqaError, (q, k, bt, lens, lse, z(4, 16, 2)))):
        with pytest.raises(error):
            pgqa.accumulate_weights(*args)
    for kw in (dict(keep=0), dict(keep=4, sinks=5), dict(keep=4, recent=-1), dict(keep=4, weights_out=z(4, 16, 2))):
        with pytest.raises(pgqa.PgqaError):
            pgqa.evict_kv(k, k.clone(), w, bt, lens, **kw)
    with pytest.raises(pgqa.PgqaError):
        pgqa.evict_kv(k, z(5, 16, 2, 128, dtype=bf), w, bt, lens, 4)
    torch.cuda.synchronize()


def cross(**kw):
    a = _lib.PgqaCrossArgs(struct_size=ctypes.sizeof(_lib.PgqaCrossArgs), q=A, k_cache=A, v_cache=A, out=A,
                           seq_lens=A, block_table=A, cu_seqlens=A, batch_size=2, tokens=10, q_stride=1024,
                           num_heads=8, num_heads_k=2, headdim=128, page_size=16, num_pages=9, bt_stride=4,
                           scale=0.1)
    for n, v in kw.items():
        setattr(a, n, v)
    return _lib.lib().pgqa_cross_attention(ctypes.byref(a), None)


@pytest.mark.parametrize("status,kw", [
    (2, dict(struct_size=8)), (1, dict(q=None)), (1, dict(out=None)), (1, dict(block_table=None)),
    (2, dict(tokens=-1)), (2, dict(num_heads=9)), (3, dict(num_heads=258)), (3, dict(headdim=64)),
    (3, dict(page_size=8)), (2, dict(num_pages=0)), (3, dict(num_pages=1 << 27)), (2, dict(cu_seqlens=None)),
    (2, dict(scale=-1.0)), (2, dict(scale=float("nan"))), (2, dict(q_stride=1016)), (4, dict(q_stride=1028)),
    (4, dict(q=A + 8)), (4, dict(out=A + 8)), (4, dict(workspace=A + 128)), (4, dict(softmax_lse=A + 2)),
    (3, dict(q_stride=1 << 39)), (2, dict(batch_size=0)),
    (3, dict(kv_format=2)), (2, dict(k_scale=A)), (4, dict(kv_format=1, v_scale=A + 2)),
])
def test_cross_attention(status, kw):
    assert cross(**kw) == status


def test_cross_attention_python_refusals():
    z = torch.zeros
    k = z(4, 16, 2, 128, dtype=torch.bfloat16)
    bt, lens = z(2, 2, dtype=torch.int32), z(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        pgqa.cross_attention(z(2, 3, 8, 128, dtype=torch.bfloat16), k, k, bt, lens)


@pytest.mark.gpu
def test_cross_attention_refuses_bad_tensors(cuda_device):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=cuda_device)  # noqa: E731
    i32 = torch.int32
    k, bt, lens, q = z(4, 16, 2, 128), z(2, 2, dtype=i32), z(2, dtype=i32), z(2, 3, 8, 128)
    for error, args, kw in (
            (ValueError, (q, k, k), dict(v_scale=1.0)), (TypeError, (q, k.to(torch.float8_e4m3fn), k), {}),
            (TypeError, (q.float(), k, k), {}),
            (ValueError, (q.cpu(), k, k), {}), (ValueError, (z(2, 4, 8, 128)[:, :3], k, k), {}),
            (ValueError, (z(2, 3, 128, 8).transpose(2, 3), k, k), {}),
            (ValueError, (z(2, 3, 16, 128)[:, :, ::2], k, k), {}),
            (pgqa.PgqaError, (z(3, 3, 8, 128), k, k), {}), (pgqa.PgqaError, (z(6, 8, 128), k, k), {}),
            (pgqa.PgqaError, (z(6, 8, 128), k, k), dict(cu_seqlens_q=z(2, dtype=i32))),
            (TypeError, (z(6, 8, 128), k, k), dict(cu_seqlens_q=z(3, dtype=torch.int64))),
            (pgqa.PgqaError, (z(2, 3, 7, 128), k, k), {}), (pgqa.PgqaError, (q, k, k), dict(out=z(6, 8, 128))),
            (pgqa.PgqaError, (q, k, z(5, 16, 2, 128)), {}), (pgqa.PgqaError, (q, k, k), dict(scale=0.0))):
        with pytest.raises(error):
            pgqa.cross_attention(*args, bt, lens, **kw)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_batches_past_the_shared_memory_table_are_refused(cuda_device):
    """accumulate_weights keeps the chunk counts of all sequences in shared memory."""
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=cuda_device)  # noqa: E731
    k, w = z(1, 16, 1, 128, dtype=torch.bfloat16), z(1, 1, 16)
    for B, Sq, ok in ((20000, 1, True), (40000, 1, False), (40000, 9, False), (20000, 17, False), (9000, 17, True)):
        call = lambda: pgqa.accumulate_weights(  # noqa: E731
            z(B, Sq, 1, 128, dtype=torch.bfloat16), k, z(B, 1, dtype=torch.int32), z(B, dtype=torch.int32),
            z(B, 1, Sq), w)
        if ok:
            call()
        else:
            with pytest.raises(pgqa.PgqaError) as e:
                call()
            assert e.value.status == 3
    pgqa.check_device_error()
    assert (w == 0).all()
