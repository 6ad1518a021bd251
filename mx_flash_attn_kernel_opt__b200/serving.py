"""Operators around the paged decode, for serving: rotary positions with the append of new
tokens, the attention weight each cached token receives, eviction by that weight, and the
attention of prompt tokens over an encoder's states.

    q = rope_append_kv(q, k, v, k_cache, v_cache, block_table, seq_lens, cos, sin, ...)
    out, lse = decode(q, k_cache, v_cache, block_table, seq_lens + 1, return_lse=True)
    accumulate_weights(q, k_cache, block_table, seq_lens + 1, lse, weights)
    kept, seq_lens = evict_kv(k_cache, v_cache, weights, block_table, seq_lens + 1, keep)
    out = cross_attention(q, enc_k, enc_v, enc_table, enc_lens, cu_seqlens_q=cu)

`weights` is a float32 pool [num_pages, Hkv, P] beside the K and V pools.  Every call runs
on torch's current stream of the tensors' device, allocates its outputs (cross_attention: and
a workspace) by torch and can be captured into a CUDA graph after one eager call.  Errors that only the device sees (a
page id, length or position out of range) are read with `check_device_error()`.
"""
import functools
import math
import struct

import torch

from ._lib import PgqaError, check, lib
from .ops import FP8, _scale_array

_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16
_AXES = bytes(range(64))

# include/pgqa.h's argument structs, field by field
_ROPE = struct.Struct("N15P21q4i64s")
_WEIGHTS = struct.Struct("N7P9qfi")
_EVICT = struct.Struct("N8P9q2i")
_CROSS = struct.Struct("N8P10qfi3PN")


# The handle of torch's current stream (a Stream object takes twenty times as long to make).
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _ptr(what, name, t, dtype, dev):
    """Address of a contiguous tensor of `dtype` on CUDA device number `dev`."""
    if t.dtype is dtype and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype:
        raise TypeError(f"{what}: {name} must be {dtype}, got {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{what}: {name} must be on cuda:{dev}, got {t.device}")
    raise ValueError(f"{what}: {name} must be contiguous")


def _cache(what, k_cache, block_table, seq_lens):
    """Checks a pool, its table and lengths.  Returns (device number, e4m3, pool shape,
    B, table width, address of the pool, of the table, of the lengths)."""
    if not k_cache.is_cuda:
        raise ValueError(f"{what}: k_cache must be a CUDA tensor")
    dev, fp8 = k_cache.get_device(), k_cache.dtype is FP8
    pool = _ptr(what, "k_cache", k_cache, FP8 if fp8 else _BF16, dev)
    table = _ptr(what, "block_table", block_table, _I32, dev)
    lens = _ptr(what, "seq_lens", seq_lens, _I32, dev)
    shape, bt = k_cache.shape, block_table.shape
    if len(shape) != 4 or len(bt) != 2:
        raise PgqaError(2, f"{what}: pools must be [num_pages, P, Hkv, D], block_table [B, width]")
    if seq_lens.shape != bt[:1]:
        raise PgqaError(2, f"{what}: seq_lens must be [B]")
    return dev, fp8, shape, bt[0], bt[1], pool, table, lens


def _v_pool(what, v_cache, k_cache, dev):
    p = _ptr(what, "v_cache", v_cache, k_cache.dtype, dev)
    if v_cache.shape != k_cache.shape:
        raise PgqaError(2, f"{what}: K and V pools must have one shape")
    return p


def _weight_pool(what, name, weights, dev, shape):
    p = _ptr(what, name, weights, _F32, dev)
    if weights.shape != (shape[0], shape[2], shape[1]):
        raise PgqaError(2, f"{what}: {name} must be [num_pages, Hkv, P] = {(shape[0], shape[2], shape[1])}")
    return p


def _scales(x, Hkv, dev):
    """Per-head factors as a float32 tensor of the device (None stays None)."""
    if torch.is_tensor(x) and x.dtype is _F32 and x.get_device() == dev and x.shape == (Hkv,) \
            and x.is_contiguous():
        return x
    at = torch.device("cuda", dev)
    if x is not None and not torch.is_tensor(x):  # filled on the device: a copy from the host cannot be captured
        return torch.full((Hkv,), float(x), dtype=_F32, device=at)
    return _scale_array(x, Hkv, at)


def _call(fn, args, dev, what):
    """Launches on torch's current stream of the device, with that device current."""
    if dev == torch.cuda.current_device():
        st = fn(args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(args, _stream(dev))
    check(st, what)


def _rows(what, name, x, want, dev, step):
    """Checks q / k_new / v_new of shape `want` [..., heads, D] (a head's elements contiguous,
    any other strides); returns (address, element strides of sequence, token, head).  step:
    the one leading dimension counts sequences rather than tokens."""
    if x.dtype is not _BF16:
        raise TypeError(f"{what}: {name} must be {_BF16}, got {x.dtype}")
    if x.get_device() != dev:
        raise ValueError(f"{what}: {name} must be on cuda:{dev}, got {x.device}")
    if x.shape != want:
        raise PgqaError(2, f"{what}: {name} must be {list(want)}, got {list(x.shape)}")
    s = x.stride()
    if s[-1] != 1:
        raise ValueError(f"{what}: the elements of a head of {name} must be contiguous")
    return x.data_ptr(), s[:3] if len(s) == 4 else ((s[0], 0, s[1]) if step else (0, s[0], s[1]))


def _like(x):
    """An uninitialised contiguous tensor of x's shape and type."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


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
    dev, full = first.get_device(), first.shape
    D = full[-1]
    Hkv = P = num_pages = width = fp8 = 0
    kp = vp = tp = lp = wp = cup = posp = qp = qo = knp = vnp = ksp = vsp = 0
    if k_new is not None:
        at, fp8, shape, B, width, kp, tp, lp = _cache(what, k_cache, block_table, seq_lens)
        if at != dev:
            raise ValueError(f"{what}: all tensors must be on one device")
        vp = _v_pool(what, v_cache, k_cache, dev)
        num_pages, P, Hkv, D = shape
        if weights is not None:
            wp = _weight_pool(what, "weights", weights, dev, shape)
        if fp8:
            ks, vs = _scales(k_scale, Hkv, dev), _scales(v_scale, Hkv, dev)
            ksp = 0 if ks is None else ks.data_ptr()
            vsp = 0 if vs is None else vs.data_ptr()
        elif k_scale is not None or v_scale is not None:
            raise ValueError("k_scale / v_scale apply to float8_e4m3fn pools only")
    else:
        if weights is not None:
            raise ValueError(f"{what}: weights goes with k_new and v_new")
        B = seq_lens.shape[0] if seq_lens is not None else (
            cu_seqlens.shape[0] - 1 if cu_seqlens is not None else full[0])
        if seq_lens is not None:
            lp = _ptr(what, "seq_lens", seq_lens, _I32, dev)
    seqlen, step = 0, False
    if cu_seqlens is not None:
        cup = _ptr(what, "cu_seqlens", cu_seqlens, _I32, dev)
        if cu_seqlens.shape != (B + 1,) or len(full) != 3:
            raise PgqaError(2, f"{what}: with cu_seqlens [B + 1], q / k_new are [tokens, heads, D]")
        lead = full[:1]
        tokens = full[0]
    else:
        if len(full) not in (3, 4) or full[0] != B:
            raise PgqaError(2, f"{what}: q / k_new must be [B, heads, D] or [B, S, heads, D]")
        step = len(full) == 3
        lead = full[:-2]
        seqlen = 1 if step else full[1]
        tokens = B * seqlen
    none = (0, 0, 0)
    qs = kst = vst = none
    Hq = 0
    if k_new is not None:
        want = (*lead, Hkv, D)
        knp, kst = _rows(what, "k_new", k_new, want, dev, step)
        vnp, vst = _rows(what, "v_new", v_new, want, dev, step)
    if q is not None:
        Hq = full[-2]
        qp, qs = _rows(what, "q", q, (*lead, Hq, D), dev, step)
        if q_out is None:
            q_out = _like(q)
            qo = q_out.data_ptr()
        else:
            qo = _ptr(what, "q_out", q_out, _BF16, dev)
            if q_out.shape != full:
                raise PgqaError(2, f"{what}: q_out must have q's shape")
    tdt = _BF16 if cos.dtype is _BF16 else _F32
    cp, sp = _ptr(what, "cos", cos, tdt, dev), _ptr(what, "sin", sin, tdt, dev)
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise PgqaError(2, f"{what}: cos and sin must be [rows, rotary_dim / 2]")
    rows, pairs = cos.shape
    num_axes = 1
    if positions is not None:
        posp = _ptr(what, "positions", positions, _I32, dev)
        ps = positions.shape
        if ps != lead:
            if ps[1:] != lead or len(ps) != len(lead) + 1:
                raise PgqaError(2, f"{what}: positions must be [axes, {', '.join(map(str, lead))}], "
                                   "or without the first dimension for one axis")
            num_axes = ps[0]
    if axes is not None:
        try:
            axes = bytes(axes)
        except ValueError:  # an entry below 0 or above 255
            axes = b""
        if len(axes) != pairs or axes.translate(None, _AXES[:num_axes]):
            raise PgqaError(2, f"{what}: axes must name one of the {num_axes} axes for each of "
                               f"the {pairs} pairs")
    elif num_axes > 1:
        raise ValueError(f"{what}: positions on several axes need axes, the axis of each pair")
    if tokens:  # torch gives empty tensors no address
        _call(lib().pgqa_rope_append, _ROPE.pack(
            _ROPE.size, qp, knp, vnp, qo, kp, vp, lp, tp, cp, sp, posp, cup, wp, ksp, vsp, B, seqlen,
            tokens, Hq, Hkv, D, P, num_pages, width, *qs, *kst, *vst, rows, 2 * pairs, num_axes,
            1 if interleaved else 0, 1 if fp8 else 0, 1 if tdt is _BF16 else 0, 0, axes or b""),
            dev, "pgqa_rope_append")
    return q_out


def rope_append_kv(q, k_new, v_new, k_cache, v_cache, block_table, seq_lens, cos, sin, *,
                   positions=None, axes=None, interleaved=False, cu_seqlens=None, weights=None,
                   k_scale=None, v_scale=None, q_out=None):
    """Turn q and k_new by their positions and append k_new / v_new to the paged cache, in
    one launch.  Returns the turned q (contiguous bf16, or `q_out`; rows of packed tokens behind
    the last sequence are not written).

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
    they are.  The sums are fp32, one addition to an entry per 32 query rows of its KV head;
    unless sequences share pages, the result does not depend on any order."""
    what = "accumulate_weights"
    dev, fp8, shape, B, width, kp, tp, lp = _cache(what, k_cache, block_table, seq_lens)
    num_pages, P, Hkv, D = shape
    qp, lsep = _ptr(what, "q", q, _BF16, dev), _ptr(what, "lse", lse, _F32, dev)
    qs = q.shape
    if len(qs) not in (3, 4) or qs[0] != B or qs[-1] != D:
        raise PgqaError(2, f"{what}: q must be [B, Hq, D] or [B, Sq, Hq, D]")
    Sq, Hq = qs[1] if len(qs) == 4 else 1, qs[-2]
    if lse.shape != (B, Hq, Sq):
        raise PgqaError(2, f"{what}: lse must be [B, Hq, Sq] = {(B, Hq, Sq)}")
    wp = _weight_pool(what, "weights", weights, dev, shape)
    ks = None
    if fp8:
        ks = _scales(k_scale, Hkv, dev)
    elif k_scale is not None:
        raise ValueError("k_scale applies to float8_e4m3fn pools only")
    if B:  # torch gives empty tensors no address
        _call(lib().pgqa_accumulate_weights, _WEIGHTS.pack(
            _WEIGHTS.size, qp, kp, lsep, wp, lp, tp, 0 if ks is None else ks.data_ptr(), B, Sq, Hq, Hkv, D,
            P, num_pages, width, 1 if causal else 0, 1.0 / math.sqrt(D) if scale is None else scale,
            1 if fp8 else 0), dev, "pgqa_accumulate_weights")
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
    are the caller's to free.  Sequences that share pages cannot be cut, nor one pool that
    holds both K and V."""
    what = "evict_kv"
    dev, fp8, shape, B, width, kp, tp, lp = _cache(what, k_cache, block_table, seq_lens)
    num_pages, P, Hkv, D = shape
    vp = _v_pool(what, v_cache, k_cache, dev)
    wp = _weight_pool(what, "weights", weights, dev, shape)
    op = 0 if weights_out is None else _weight_pool(what, "weights_out", weights_out, dev, shape)
    if keep < 1:
        raise PgqaError(2, f"{what}: keep must be at least 1")
    kept, new_lens = seq_lens.new_empty((B, Hkv, keep)), seq_lens.new_empty((B,))
    if B:
        _call(lib().pgqa_evict, _EVICT.pack(
            _EVICT.size, kp, vp, wp, op, lp, tp, kept.data_ptr(), new_lens.data_ptr(), B, Hkv, D, P,
            num_pages, width, keep, sinks, recent, 1 if fp8 else 0, 0), dev, "pgqa_evict")
    return kept, new_lens


@functools.lru_cache(maxsize=4096)
def _cross_workspace(dev, *shape):
    with torch.cuda.device(dev):
        return lib().pgqa_cross_workspace_size(*shape)


def cross_attention(q, k_cache, v_cache, block_table, seq_lens, *, cu_seqlens_q=None, scale=None,
                    k_scale=None, v_scale=None, out=None, return_lse=False):
    """Attention of query tokens over each sequence's encoder states, held in pages:
    softmax(scale * q K^T) V over the first seq_lens[b] tokens of sequence b, no causal mask.

    q [B, Sq, Hq, 128] bf16, or packed [tokens, Hq, 128] with `cu_seqlens_q` [B + 1] int32,
    ascending from 0; its token stride may be any multiple of 8 elements (a slice of a
    projection), heads contiguous, sequences one after the other.  k_cache / v_cache
    [num_pages, P, Hkv, 128] bf16 or float8_e4m3fn (an element of KV head h is worth
    e4m3 * k_scale[h], v_scale for V), block_table [B, width] int32, seq_lens [B] int32 (0:
    the sequence's rows are zeros).

    Returns out (contiguous, q's shape; 16-byte aligned, as every tensor of 16-bit or 8-bit
    elements here) or (out, lse) with `return_lse`: fp32 [Hq, tokens] for packed q, else
    [B, Hq, Sq]; -inf where a row sees no key.  Scores, sums and accumulators are fp32, the
    weights that multiply V are rounded to bf16.  Rows of packed tokens behind the last
    sequence are left as they are in `out` (without `out`, and in lse, they hold anything)."""
    what = "cross_attention"
    dev, fp8, shape, B, width, kp, tp, lp = _cache(what, k_cache, block_table, seq_lens)
    num_pages, P, Hkv, D = shape
    vp = _v_pool(what, v_cache, k_cache, dev)
    ks = vs = None
    if fp8:
        ks, vs = _scales(k_scale, Hkv, dev), _scales(v_scale, Hkv, dev)
    elif k_scale is not None or v_scale is not None:
        raise ValueError("k_scale / v_scale apply to float8_e4m3fn pools only")
    if q.dtype is not _BF16:
        raise TypeError(f"{what}: q must be {_BF16}, got {q.dtype}")
    if q.get_device() != dev:
        raise ValueError(f"{what}: q must be on cuda:{dev}, got {q.device}")
    qs, st = q.shape, q.stride()
    cup = 0
    if cu_seqlens_q is not None:
        cup = _ptr(what, "cu_seqlens_q", cu_seqlens_q, _I32, dev)
        if len(qs) != 3 or cu_seqlens_q.shape != (B + 1,):
            raise PgqaError(2, f"{what}: with cu_seqlens_q [B + 1], q is [tokens, Hq, D]")
        tokens, Sq, stride = qs[0], 0, st[0]
    else:
        if len(qs) != 4 or qs[0] != B:
            raise PgqaError(2, f"{what}: q must be [B, Sq, Hq, D], or packed with cu_seqlens_q")
        Sq, stride = qs[1], st[1]
        tokens = B * Sq
        if B > 1 and Sq > 1 and st[0] != Sq * stride:
            raise ValueError(f"{what}: the sequences of q must follow each other without a gap")
        if Sq == 1:
            stride = st[0]
    Hq = qs[-2]
    if qs[-1] != D:
        raise PgqaError(2, f"{what}: q and the pools must have one head dimension")
    if st[-1] != 1 or (Hq > 1 and st[-2] != D):
        raise ValueError(f"{what}: the heads of a token of q must be contiguous")
    if tokens <= 1:
        stride = Hq * D
    if out is None:
        out = _like(q)
        op = out.data_ptr()
    else:
        op = _ptr(what, "out", out, _BF16, dev)
        if out.shape != qs:
            raise PgqaError(2, f"{what}: out must have q's shape")
    lse = None
    if return_lse:
        lse = seq_lens.new_empty((Hq, tokens) if cup else (B, Hq, Sq), dtype=_F32)
    if tokens:
        need = _cross_workspace(dev, tokens, B, Hq, Hkv, D, P, width)
        # a buffer of this call's own: calls on two streams or in two graphs share none
        ws = seq_lens.new_empty((need,), dtype=torch.uint8) if need else None
        _call(lib().pgqa_cross_attention, _CROSS.pack(
            _CROSS.size, q.data_ptr(), kp, vp, op, 0 if lse is None else lse.data_ptr(), lp, tp, cup, B,
            Sq, tokens, stride, Hq, Hkv, D, P, num_pages, width,
            1.0 / math.sqrt(D) if scale is None else scale, 1 if fp8 else 0, 0 if ks is None else ks.data_ptr(),
            0 if vs is None else vs.data_ptr(), 0 if ws is None else ws.data_ptr(), need), dev, "pgqa_cross_attention")
    return (out, lse) if return_lse else out
