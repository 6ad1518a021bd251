"""Operators around the paged decode, for serving: rotary positions with the append of new
tokens, the attention weight each cached token receives, eviction by that weight, and the
attention of prompt tokens over an encoder's states.

    q = rope_append_kv(q, k, v, k_cache, v_cache, block_table, seq_lens, cos, sin, ...)
    out, lse = decode(q, k_cache, v_cache, block_table, seq_lens + 1, return_lse=True)
    accumulate_weights(q, k_cache, block_table, seq_lens + 1, lse, weights)
    kept, seq_lens = evict_kv(k_cache, v_cache, weights, block_table, seq_lens + 1, keep)
    out = cross_attention(q, enc_k, enc_v, enc_table, enc_lens, cu_seqlens_q=cu)

`weights` is a float32 pool [num_pages, Hkv, P] beside the K and V pools.  Every call runs
on torch's current stream of the tensors' device, allocates nothing but its outputs and can
be captured into a CUDA graph after one eager call.  Errors that only the device sees (a
page id, length or position out of range) are read with `check_device_error()`.
"""
import ctypes
import math

import torch

from . import _lib
from ._lib import PgqaError, check, lib
from .ops import FP8, _scale_array

_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16


def _check(what, device, *named):
    """named: (name, tensor, dtype); every tensor contiguous and on `device`."""
    for name, t, dt in named:
        if t.dtype != dt:
            raise TypeError(f"{what}: {name} must be {dt}, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{what}: {name} must be on {device}, got {t.device}")
        if not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous")


def _pools(what, k_cache, v_cache, block_table, seq_lens):
    """Checks pools, table and lengths; returns (device, e4m3, num_pages, P, Hkv, D, B)."""
    if not k_cache.is_cuda:
        raise ValueError(f"{what}: k_cache must be a CUDA tensor")
    dt = FP8 if k_cache.dtype == FP8 else _BF16
    dev = k_cache.device
    _check(what, dev, ("k_cache", k_cache, dt), ("block_table", block_table, _I32),
           ("seq_lens", seq_lens, _I32))
    if k_cache.dim() != 4 or block_table.dim() != 2:
        raise PgqaError(2, f"{what}: pools must be [num_pages, P, Hkv, D], block_table [B, width]")
    if v_cache is not None:
        _check(what, dev, ("v_cache", v_cache, dt))
        if v_cache.shape != k_cache.shape:
            raise PgqaError(2, f"{what}: K and V pools must have one shape")
    B = block_table.shape[0]
    if seq_lens.dim() != 1 or seq_lens.shape[0] != B:
        raise PgqaError(2, f"{what}: seq_lens must be [B]")
    return (dev, dt is FP8, *k_cache.shape, B)


def _weight_pool(what, weights, name, dev, num_pages, Hkv, P):
    _check(what, dev, (name, weights, _F32))
    if tuple(weights.shape) != (num_pages, Hkv, P):
        raise PgqaError(2, f"{what}: {name} must be [num_pages, Hkv, P] = {(num_pages, Hkv, P)}")


def _launch(fn, args, device, what):
    stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
    if device.index == torch.cuda.current_device():
        st = fn(ctypes.byref(args), stream)
    else:
        with torch.cuda.device(device):
            st = fn(ctypes.byref(args), stream)
    check(st, what)


def _rows(what, name, x, lead, D, device):
    """Checks q / k_new / v_new [*lead, heads, D] (heads contiguous inside, any strides that
    are multiples of 16 bytes); returns (heads, element strides of sequence, token, head)."""
    if x.dtype != _BF16:
        raise TypeError(f"{what}: {name} must be {_BF16}, got {x.dtype}")
    if x.device != device:
        raise ValueError(f"{what}: {name} must be on {device}, got {x.device}")
    if x.dim() != len(lead) + 2 or tuple(x.shape[:-2]) != lead or x.shape[-1] != D:
        raise PgqaError(2, f"{what}: {name} must be [{', '.join(map(str, lead))}, heads, {D}]")
    if x.stride(-1) != 1:
        raise ValueError(f"{what}: the elements of a head of {name} must be contiguous")
    s = x.stride()
    return x.shape[-2], ((s[0], s[1], s[2]) if len(lead) == 2 else (0, s[0], s[1]))


def _turn(what, q, k_new, v_new, k_cache, v_cache, block_table, seq_lens, cos, sin, positions,
          axes, interleaved, cu_seqlens, weights, k_scale, v_scale, q_out):
    """One pgqa_rope_append call.  q, or k_new and v_new, may be None (nothing to turn or to
    append); with k_new None the pools and the table are not used."""
    first = q if q is not None else k_new
    if first is None:
        raise ValueError(f"{what}: give q, or k_new and v_new")
    if (k_new is None) != (v_new is None):
        raise ValueError(f"{what}: k_new and v_new go together")
    if not first.is_cuda:
        raise ValueError(f"{what}: q / k_new must be CUDA tensors")
    dev = first.device
    a = _lib.PgqaRopeArgs(struct_size=ctypes.sizeof(_lib.PgqaRopeArgs))
    D = first.shape[-1]
    if k_new is not None:
        _, fp8, num_pages, P, Hkv, D, B = _pools(what, k_cache, v_cache, block_table, seq_lens)
        if k_cache.device != dev:
            raise ValueError(f"{what}: all tensors must be on one device")
        if not fp8 and (k_scale is not None or v_scale is not None):
            raise ValueError("k_scale / v_scale apply to float8_e4m3fn pools only")
        a.k_cache, a.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
        a.block_table, a.bt_stride = block_table.data_ptr(), block_table.shape[1]
        a.num_pages, a.page_size, a.num_heads_k, a.kv_format = num_pages, P, Hkv, int(fp8)
    else:
        if weights is not None:
            raise ValueError(f"{what}: weights goes with k_new and v_new")
        B = seq_lens.shape[0] if seq_lens is not None else (
            cu_seqlens.shape[0] - 1 if cu_seqlens is not None else first.shape[0])
    if seq_lens is not None:
        _check(what, dev, ("seq_lens", seq_lens, _I32))
        a.seq_lens = seq_lens.data_ptr()
    if cu_seqlens is not None:
        _check(what, dev, ("cu_seqlens", cu_seqlens, _I32))
        if tuple(cu_seqlens.shape) != (B + 1,) or first.dim() != 3:
            raise PgqaError(2, f"{what}: with cu_seqlens [B + 1], q / k_new are [tokens, heads, D]")
        lead = (first.shape[0],)
        a.cu_seqlens = cu_seqlens.data_ptr()
    else:
        if first.dim() not in (3, 4) or first.shape[0] != B:
            raise PgqaError(2, f"{what}: q / k_new must be [B, heads, D] or [B, S, heads, D]")
        lead = tuple(first.shape[:-2])
        a.seqlen = lead[1] if len(lead) == 2 else 1
    a.tokens = math.prod(lead)
    a.batch_size, a.headdim = B, D

    def strides(x):
        heads, s = _rows(what, x[0], x[1], lead, D, dev)
        # [B, heads, D]: one token per sequence, so the first stride is the sequence's
        return heads, (ctypes.c_int64 * 3)(s[1], 0, s[2]) if cu_seqlens is None and len(lead) == 1 \
            else (ctypes.c_int64 * 3)(*s)

    if k_new is not None:
        hk, a.k_strides = strides(("k_new", k_new))
        hv, a.v_strides = strides(("v_new", v_new))
        if hk != Hkv or hv != Hkv:
            raise PgqaError(2, f"{what}: k_new / v_new must have the pools' {Hkv} heads")
        a.k_new, a.v_new = k_new.data_ptr(), v_new.data_ptr()
    if q is not None:
        a.num_heads, a.q_strides = strides(("q", q))
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=_BF16, device=dev)
        else:
            _check(what, dev, ("q_out", q_out, _BF16))
            if q_out.shape != q.shape:
                raise PgqaError(2, f"{what}: q_out must have q's shape")
        a.q, a.q_out = q.data_ptr(), q_out.data_ptr()

    dt = _BF16 if cos.dtype == _BF16 else _F32
    _check(what, dev, ("cos", cos, dt), ("sin", sin, dt))
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise PgqaError(2, f"{what}: cos and sin must be [rows, rotary_dim / 2]")
    pairs = cos.shape[1]
    a.cos, a.sin, a.table_rows, a.rotary_dim = cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * pairs
    a.table_format, a.interleaved = int(dt is _BF16), int(bool(interleaved))
    a.num_axes = 1
    if positions is not None:
        _check(what, dev, ("positions", positions, _I32))
        if tuple(positions.shape) != lead:
            if tuple(positions.shape[1:]) != lead or positions.dim() != len(lead) + 1:
                raise PgqaError(2, f"{what}: positions must be [axes, {', '.join(map(str, lead))}], "
                                   "or without the first dimension for one axis")
            a.num_axes = positions.shape[0]
        a.positions = positions.data_ptr()
    if axes is not None:
        if len(axes) != pairs or pairs > 64 or not all(0 <= int(x) < a.num_axes for x in axes):
            raise PgqaError(2, f"{what}: axes must name one of the {a.num_axes} axes for each of "
                               f"the {pairs} pairs")
        a.pair_axis[:pairs] = [int(x) for x in axes]
    elif a.num_axes > 1:
        raise ValueError(f"{what}: positions on several axes need axes, the axis of each pair")
    if weights is not None:
        _weight_pool(what, weights, "weights", dev, num_pages, Hkv, P)
        a.weights = weights.data_ptr()
    ks = vs = None
    if k_new is not None and fp8:
        ks, vs = _scale_array(k_scale, Hkv, dev), _scale_array(v_scale, Hkv, dev)
        a.k_scale = ks.data_ptr() if ks is not None else None
        a.v_scale = vs.data_ptr() if vs is not None else None
    if a.tokens:  # torch gives empty tensors no address
        _launch(lib().pgqa_rope_append, a, dev, "pgqa_rope_append")
    return q_out


def rope_append_kv(q, k_new, v_new, k_cache, v_cache, block_table, seq_lens, cos, sin, *,
                   positions=None, axes=None, interleaved=False, cu_seqlens=None, weights=None,
                   k_scale=None, v_scale=None, q_out=None):
    """Turn q and k_new by their positions and append k_new / v_new to the paged cache, in
    one launch.  Returns the turned q (contiguous bf16, or `q_out`).

    q [B, S, Hq, 128], k_new / v_new [B, S, Hkv, 128] bf16 (or [B, heads, 128] for one token
    per sequence; or packed [tokens, heads, 128] with `cu_seqlens` [B + 1] int32, ascending
    from 0).  They may be slices of one projection's output: any strides that are multiples
    of 8 elements, with a head's 128 elements contiguous.  q None only appends.

    cos / sin [rows, R / 2] fp32 or bf16, R a multiple of 16 up to 128: pair i of a head --
    elements (i, i + R/2), or (2i, 2i + 1) if `interleaved` -- turns by row p of the tables,
    elements from R on are copied.  p = positions[axes[i], token] for `positions` int32
    [axes, B, S] (or [axes, tokens]); one axis may leave out the first dimension and
    `axes`.  Without `positions` p is the token's place in its sequence, L_b + s.

    Token s of sequence b goes to position L_b + s (L_b = seq_lens[b], not modified) of its
    pages, bf16 or e4m3: float8_e4m3fn pools hold value / k_scale[h] (v_scale for V),
    rounded once and saturated at +-448.  `weights` [num_pages, Hkv, P] fp32 (optional): the
    new tokens' entries become 0.

    A token with a position outside the tables, a place past the block table or a bad page
    id is not written; `check_device_error()` reports it."""
    if k_new is None or v_new is None:
        raise ValueError("rope_append_kv: k_new and v_new are required")
    return _turn("rope_append_kv", q, k_new, v_new, k_cache, v_cache, block_table, seq_lens, cos,
                 sin, positions, axes, interleaved, cu_seqlens, weights, k_scale, v_scale, q_out)


def accumulate_weights(q, k_cache, block_table, seq_lens, lse, weights, *, scale=None,
                       causal=False, k_scale=None):
    """Add to `weights` [num_pages, Hkv, P] fp32 the attention weight that every cached token
    received from a decode: for token t of sequence b and KV head kv, the sum over the query
    rows of kv that see t of exp(scale * q.k_t - lse).  Returns `weights`.

    q, k_cache, block_table, seq_lens (the lengths attended over), scale, causal and k_scale
    are the decode's, lse [B, Hq, Sq] fp32 is what it returned with `return_lse`.  A row that
    sees no token (lse -inf) adds nothing, and entries past a sequence's length are left as
    they are.  Unless sequences share pages, the result does not depend on any order."""
    what = "accumulate_weights"
    dev, fp8, num_pages, P, Hkv, D, B = _pools(what, k_cache, None, block_table, seq_lens)
    _check(what, dev, ("q", q, _BF16), ("lse", lse, _F32))
    if q.dim() not in (3, 4) or q.shape[0] != B or q.shape[-1] != D:
        raise PgqaError(2, f"{what}: q must be [B, Hq, D] or [B, Sq, Hq, D]")
    Sq = q.shape[1] if q.dim() == 4 else 1
    Hq = q.shape[-2]
    if tuple(lse.shape) != (B, Hq, Sq):
        raise PgqaError(2, f"{what}: lse must be [B, Hq, Sq] = {(B, Hq, Sq)}")
    _weight_pool(what, weights, "weights", dev, num_pages, Hkv, P)
    if not fp8 and k_scale is not None:
        raise ValueError("k_scale applies to float8_e4m3fn pools only")
    ks = _scale_array(k_scale, Hkv, dev) if fp8 else None
    a = _lib.PgqaWeightsArgs(
        ctypes.sizeof(_lib.PgqaWeightsArgs), q.data_ptr(), k_cache.data_ptr(), lse.data_ptr(),
        weights.data_ptr(), seq_lens.data_ptr(), block_table.data_ptr(),
        ks.data_ptr() if ks is not None else None, B, Sq, Hq, Hkv, D, P, num_pages,
        block_table.shape[1], int(bool(causal)),
        float(scale) if scale is not None else 1.0 / math.sqrt(D), int(fp8))
    _launch(lib().pgqa_accumulate_weights, a, dev, "pgqa_accumulate_weights")
    return weights


def evict_kv(k_cache, v_cache, weights, block_table, seq_lens, keep, *, sinks=0, recent=0,
             weights_out=None):
    """Cut every sequence of more than `keep` tokens to `keep`, for each KV head on its own,
    in place.  Returns (kept [B, Hkv, keep] int32, new_lens [B] int32).

    Kept are the first `sinks` tokens, the last `recent` and, of those between, the
    keep - sinks - recent with the highest `weights` [num_pages, Hkv, P] fp32 (equal weights:
    the lowest index first; NaN counts as the highest), in their order, in slots [0, keep) of
    the sequence's own pages.  kept lists their former indices; a sequence of L <= keep
    tokens is left as it is and gets 0 .. L-1, then -1.  new_lens = min(seq_lens, keep).

    The weights move along, in place or into `weights_out` (the entries of every sequence's
    first new_lens slots; the others are left as they are).  Pages from ceil(keep / P) on
    are the caller's to free.  Sequences that share pages cannot be cut."""
    what = "evict_kv"
    dev, fp8, num_pages, P, Hkv, D, B = _pools(what, k_cache, v_cache, block_table, seq_lens)
    _weight_pool(what, weights, "weights", dev, num_pages, Hkv, P)
    if weights_out is not None:
        _weight_pool(what, weights_out, "weights_out", dev, num_pages, Hkv, P)
    keep = int(keep)
    if keep < 1:
        raise PgqaError(2, f"{what}: keep must be at least 1")
    kept = torch.empty(B, Hkv, keep, dtype=_I32, device=dev)
    new_lens = torch.empty(B, dtype=_I32, device=dev)
    a = _lib.PgqaEvictArgs(
        ctypes.sizeof(_lib.PgqaEvictArgs), k_cache.data_ptr(), v_cache.data_ptr(),
        weights.data_ptr(), weights_out.data_ptr() if weights_out is not None else None,
        seq_lens.data_ptr(), block_table.data_ptr(), kept.data_ptr(), new_lens.data_ptr(), B,
        Hkv, D, P, num_pages, block_table.shape[1], keep, int(sinks), int(recent), int(fp8))
    _launch(lib().pgqa_evict, a, dev, "pgqa_evict")
    return kept, new_lens


def cross_attention(q, k_cache, v_cache, block_table, seq_lens, *, cu_seqlens_q=None, scale=None,
                    out=None, return_lse=False):
    """Attention of query tokens over each sequence's encoder states, held in pages:
    softmax(scale * q K^T) V over the first seq_lens[b] tokens of sequence b, no causal mask.

    q [B, Sq, Hq, 128] bf16, or packed [tokens, Hq, 128] with `cu_seqlens_q` [B + 1] int32,
    ascending from 0; its token stride may be any multiple of 8 elements (a slice of a
    projection), heads contiguous.  k_cache / v_cache [num_pages, P, Hkv, 128] bf16,
    block_table [B, width] int32, seq_lens [B] int32 (0: the sequence's rows are zeros).

    Returns out (contiguous, q's shape) or (out, lse) with `return_lse`: fp32 [Hq, tokens]
    for packed q, else [B, Hq, Sq]; -inf where a row sees no key.  Rows of packed tokens
    behind the last sequence are left as they are in `out`."""
    what = "cross_attention"
    dev, fp8, num_pages, P, Hkv, D, B = _pools(what, k_cache, v_cache, block_table, seq_lens)
    if fp8:
        raise NotImplementedError(f"{what}: float8_e4m3fn pools are not implemented here")
    if q.dtype != _BF16:
        raise TypeError(f"{what}: q must be {_BF16}, got {q.dtype}")
    if q.device != dev:
        raise ValueError(f"{what}: q must be on {dev}, got {q.device}")
    if cu_seqlens_q is not None:
        _check(what, dev, ("cu_seqlens_q", cu_seqlens_q, _I32))
        if q.dim() != 3 or tuple(cu_seqlens_q.shape) != (B + 1,):
            raise PgqaError(2, f"{what}: with cu_seqlens_q [B + 1], q is [tokens, Hq, D]")
        tokens, Sq, stride = q.shape[0], 0, q.stride(0)
    else:
        if q.dim() != 4 or q.shape[0] != B:
            raise PgqaError(2, f"{what}: q must be [B, Sq, Hq, D], or packed with cu_seqlens_q")
        Sq, stride = q.shape[1], q.stride(1)
        tokens = B * Sq
        if B > 1 and Sq > 1 and q.stride(0) != Sq * stride:
            raise ValueError(f"{what}: the sequences of q must follow each other without a gap")
        if Sq == 1:
            stride = q.stride(0)
    Hq = q.shape[-2]
    if q.shape[-1] != D:
        raise PgqaError(2, f"{what}: q and the pools must have one head dimension")
    if q.stride(-1) != 1 or (Hq > 1 and q.stride(-2) != D):
        raise ValueError(f"{what}: the heads of a token of q must be contiguous")
    if tokens <= 1:
        stride = Hq * D
    if out is None:
        out = torch.empty(q.shape, dtype=_BF16, device=dev)
    else:
        _check(what, dev, ("out", out, _BF16))
        if out.shape != q.shape:
            raise PgqaError(2, f"{what}: out must have q's shape")
    lse = None
    if return_lse:
        lse = torch.empty((Hq, tokens) if cu_seqlens_q is not None else (B, Hq, Sq), dtype=_F32, device=dev)
    if tokens:
        L = lib()
        with torch.cuda.device(dev):
            need = L.pgqa_cross_workspace_size(tokens, B, Hq, Hkv, D, P, block_table.shape[1])
        # a buffer of this call's own: calls on two streams or in two graphs share none
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        a = _lib.PgqaCrossArgs(
            ctypes.sizeof(_lib.PgqaCrossArgs), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            out.data_ptr(), lse.data_ptr() if lse is not None else None, seq_lens.data_ptr(),
            block_table.data_ptr(), cu_seqlens_q.data_ptr() if cu_seqlens_q is not None else None, B,
            Sq, tokens, stride, Hq, Hkv, D, P, num_pages, block_table.shape[1],
            float(scale) if scale is not None else 1.0 / math.sqrt(D), 0,
            ws.data_ptr() if ws is not None else None, need)
        _launch(L.pgqa_cross_attention, a, dev, "pgqa_cross_attention")
    return (out, lse) if return_lse else out
