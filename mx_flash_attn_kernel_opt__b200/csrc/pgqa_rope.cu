/*
 * pgqa_rope.cu - rotary positions on one or several axes, fused with the append to the
 * paged cache.
 *
 * For token x of sequence b and pair i < R/2 of a head, with p = positions[axis(i)][x]
 * (or L_b + s, the token's place in the sequence, when no positions are given):
 *     (x_i, y_i) -> (x_i c - y_i s, y_i c + x_i s),   c = cos[p][i], s = sin[p][i]
 * The pairs of a head are (i, i + R/2) or, interleaved, (2i, 2i + 1); elements R and up
 * are copied.  q goes to q_out in bf16; k (turned) and v go to slot (L_b + s) % P of page
 * block_table[b][(L_b + s) / P], in bf16 or as e4m3(value / scale[head]).  The products
 * and the division are in fp32 and the result is rounded once.  The slot's entries of the
 * attention-weight pool are set to zero, so that a page used again starts empty.
 *
 * Bound by HBM traffic (a few operations per byte): a warp carries one token and up to 12
 * of its Hq + 2 Hkv rows, 8 lanes per row with two 16-byte pieces each.  A lane's 8 pairs are
 * the same in every row it visits, so cosines and sines are read once per warp into
 * registers.  What a warp waits for is a chain of small loads (sequence, length, page), so
 * the loads that depend on the token's number alone, rows and positions, go first, a warp is a
 * CTA (it leaves its place to the next as soon as it is done), and 72 registers a thread let
 * 26 of them wait on an SM at once.  Prompts of 18,000 tokens with 28 + 8 heads: 56.3 us (5.4
 * TB/s, 0.83 of a copy's rate); with four warps per CTA 62.2 us, with 8 rows per warp 86.7 us.
 */
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pgqa_host.h"
#include "pgqa_ptx.cuh"

namespace pgqa {
namespace rope {

constexpr int kThreads = 32;
constexpr int kRowsPerLane = 3;  // rows a lane visits: 12 rows of a token per warp

struct Params {
    const __nv_bfloat16 *q, *k, *v;
    __nv_bfloat16* q_out;
    void *k_cache, *v_cache;
    const int32_t *seq_lens, *block_table, *positions, *cu;
    const void *cos, *sin;
    float* weights;
    const float *k_scale, *v_scale;
    int32_t* err;
    int64_t qs[3], ks[3], vs[3];  // strides in elements: sequence, token, head
    int64_t T, bt_stride, cap_tokens, table_rows;
    int32_t B, S, Hq, Hk, P, page_shift, num_pages;  // Hk = 0: no append
    int32_t blocks, rows_per_block;                  // row blocks per token, rows in each (multiple of 4)
    int32_t R, interleaved, table_bf16, runs8;
    uint8_t axis[64];
};

/* Largest b in [0, B) with cu[b] <= x (cu ascending), 32 probes at a time. */
__device__ __forceinline__ int32_t find_sequence(const int32_t* cu, int32_t B, int64_t x, int lane) {
    int32_t lo = 0, hi = B;
    while (hi - lo > 1) {
        const int32_t step = (hi - lo + 31) / 32;
        const int32_t at = lo + (lane + 1) * step;
        const bool le = at < hi && (int64_t)ptx::ld(cu + at) <= x;
        const int32_t n = __popc(__ballot_sync(0xffffffffu, le));
        lo += n * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

__device__ __forceinline__ void unpack8(uint4 u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ uint4 pack8_bf16(const float (&f)[8]) {
    return make_uint4(ptx::pack_bf16x2(f[0], f[1]), ptx::pack_bf16x2(f[2], f[3]),
                      ptx::pack_bf16x2(f[4], f[5]), ptx::pack_bf16x2(f[6], f[7]));
}

/* e4m3 of f / scale: a true division, so that the result is the rounding of one quotient */
__device__ __forceinline__ uint2 pack8_e4m3(const float (&f)[8], float scale) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = ptx::f32x2_to_e4m3x2(__fdiv_rn(f[2 * i], scale), __fdiv_rn(f[2 * i + 1], scale));
    return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

template <bool KV8>
__global__ void __launch_bounds__(kThreads, 26) rope_append_kernel(const Params p) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int64_t x = unit / p.blocks;
    if (x >= p.T) return;
    const int32_t block = (int32_t)(unit - x * p.blocks);
    const int t = lane & 7, sub = lane >> 3;
    // a lane's two 16-byte pieces of a row
    const int turned = p.R >> 4;  // lanes that hold pairs
    int c0, c1;
    if (p.interleaved) {
        c0 = 2 * t;
        c1 = c0 + 1;
    } else if (t < turned) {
        c0 = t;
        c1 = t + turned;
    } else {
        c0 = 2 * t;  // past the pairs: 2 * turned + 2 * (t - turned)
        c1 = c0 + 1;
    }
    // what depends on the token's number alone: its rows and positions
    const int32_t b_pad = p.cu ? 0 : (int32_t)(x / p.S);
    const int64_t sx = x - (int64_t)b_pad * p.S;
    uint4 a[kRowsPerLane], e[kRowsPerLane];
    const int row0 = block * p.rows_per_block + sub;
    const int row_end = min(p.Hq + 2 * p.Hk, (block + 1) * p.rows_per_block);
#pragma unroll
    for (int i = 0; i < kRowsPerLane; ++i) {
        const int r = row0 + 4 * i;
        if (r < row_end) {
            const __nv_bfloat16* src;
            if (r < p.Hq) src = p.q + b_pad * p.qs[0] + sx * p.qs[1] + r * p.qs[2];
            else if (r < p.Hq + p.Hk) src = p.k + b_pad * p.ks[0] + sx * p.ks[1] + (r - p.Hq) * p.ks[2];
            else src = p.v + b_pad * p.vs[0] + sx * p.vs[1] + (r - p.Hq - p.Hk) * p.vs[2];
            const uint4* s4 = reinterpret_cast<const uint4*>(src);
            a[i] = ptx::ld(s4 + c0);
            e[i] = ptx::ld(s4 + c1);
        }
    }
    // positions of this lane's pairs [8 t, 8 t + 8): one, or one per pair
    int32_t pos[8];
    if (t < turned && p.positions != nullptr) {
        pos[0] = ptx::ld(p.positions + (int64_t)p.axis[8 * t] * p.T + x);
        if (!p.runs8) {
#pragma unroll
            for (int j = 1; j < 8; ++j) pos[j] = ptx::ld(p.positions + (int64_t)p.axis[8 * t + j] * p.T + x);
        }
    }
    int32_t b = b_pad;
    int64_t s = sx;
    if (p.cu != nullptr) {
        b = find_sequence(p.cu, p.B, x, lane);
        s = x - ptx::ld(p.cu + b);
        // in front of the first sequence or behind the last: left as it was
        if (s < 0 || x >= ptx::ld(p.cu + b + 1)) return;
    }
    const int64_t tok = (p.seq_lens != nullptr ? (int64_t)ptx::ld(p.seq_lens + b) : 0) + s;
    // cosines and sines
    float c[8], n[8];
    bool bad = false;
    if (t < turned) {
        auto row_of = [&](int64_t q) -> int64_t {
            if (q < 0 || q >= p.table_rows) {
                bad = true;
                return 0;
            }
            return q * (p.R >> 1);
        };
        if (p.runs8 || p.positions == nullptr) {  // the eight pairs turn about one axis
            const int64_t at = row_of(p.positions ? (int64_t)pos[0] : tok) + 8 * t;
            if (p.table_bf16) {
                unpack8(ptx::ld(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.cos) + at)), c);
                unpack8(ptx::ld(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.sin) + at)), n);
            } else {
                const float4* cp = reinterpret_cast<const float4*>(static_cast<const float*>(p.cos) + at);
                const float4* np = reinterpret_cast<const float4*>(static_cast<const float*>(p.sin) + at);
                const float4 u0 = ptx::ld(cp), u1 = ptx::ld(cp + 1), w0 = ptx::ld(np), w1 = ptx::ld(np + 1);
                c[0] = u0.x; c[1] = u0.y; c[2] = u0.z; c[3] = u0.w; c[4] = u1.x; c[5] = u1.y; c[6] = u1.z; c[7] = u1.w;
                n[0] = w0.x; n[1] = w0.y; n[2] = w0.z; n[3] = w0.w; n[4] = w1.x; n[5] = w1.y; n[6] = w1.z; n[7] = w1.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t at = row_of(pos[j]) + 8 * t + j;
                if (p.table_bf16) {
                    c[j] = __bfloat162float(ptx::ld(static_cast<const __nv_bfloat16*>(p.cos) + at));
                    n[j] = __bfloat162float(ptx::ld(static_cast<const __nv_bfloat16*>(p.sin) + at));
                } else {
                    c[j] = ptx::ld(static_cast<const float*>(p.cos) + at);
                    n[j] = ptx::ld(static_cast<const float*>(p.sin) + at);
                }
            }
        }
    }
    // the token's place in the cache
    int32_t pid = -1, slot = 0;
    if (p.Hk > 0) {
        if (tok < s || tok >= p.cap_tokens) {  // a negative length, or past the table
            if (lane == 0) atomicOr(p.err, kDevErrBadSeqlen);
            return;
        }
        const int32_t page = p.page_shift >= 0 ? (int32_t)(tok >> p.page_shift) : (int32_t)(tok / p.P);
        slot = (int32_t)(tok - (int64_t)page * p.P);
        pid = ptx::ld(p.block_table + (int64_t)b * p.bt_stride + page);
        if ((uint32_t)pid >= (uint32_t)p.num_pages) {
            if (lane == 0) atomicOr(p.err, kDevErrBadPage);
            return;
        }
    }
    if (__any_sync(0xffffffffu, bad)) {  // nothing of this token is written
        if (lane == 0) atomicOr(p.err, kDevErrBadPosition);
        return;
    }
#pragma unroll
    for (int i = 0; i < kRowsPerLane; ++i) {
        const int r = row0 + 4 * i;
        if (r >= row_end) continue;
        const bool is_v = r >= p.Hq + p.Hk;
        float f[8], g[8];
        if (!is_v && t < turned) {
            unpack8(a[i], f);
            unpack8(e[i], g);
            float y0[8], y1[8];
            if (p.interleaved) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y0[2 * j] = f[2 * j] * c[j] - f[2 * j + 1] * n[j];
                    y0[2 * j + 1] = f[2 * j + 1] * c[j] + f[2 * j] * n[j];
                    y1[2 * j] = g[2 * j] * c[4 + j] - g[2 * j + 1] * n[4 + j];
                    y1[2 * j + 1] = g[2 * j + 1] * c[4 + j] + g[2 * j] * n[4 + j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    y0[j] = f[j] * c[j] - g[j] * n[j];
                    y1[j] = g[j] * c[j] + f[j] * n[j];
                }
            }
            if (r < p.Hq || !KV8) {
                a[i] = pack8_bf16(y0);
                e[i] = pack8_bf16(y1);
            } else {
                const float sc = p.k_scale ? ptx::ld(p.k_scale + (r - p.Hq)) : 1.f;
                const uint2 u0 = pack8_e4m3(y0, sc), u1 = pack8_e4m3(y1, sc);
                a[i].x = u0.x; a[i].y = u0.y;
                e[i].x = u1.x; e[i].y = u1.y;
            }
        } else if (KV8 && r >= p.Hq) {
            unpack8(a[i], f);
            unpack8(e[i], g);
            const float* scale = is_v ? p.v_scale : p.k_scale;
            const float sc = scale ? ptx::ld(scale + (r - p.Hq - (is_v ? p.Hk : 0))) : 1.f;
            const uint2 u0 = pack8_e4m3(f, sc), u1 = pack8_e4m3(g, sc);
            a[i].x = u0.x; a[i].y = u0.y;
            e[i].x = u1.x; e[i].y = u1.y;
        }
        if (r < p.Hq) {
            uint4* d = reinterpret_cast<uint4*>(p.q_out + (x * p.Hq + r) * 128);
            d[c0] = a[i];
            d[c1] = e[i];
        } else {
            const int h = r - p.Hq - (is_v ? p.Hk : 0);
            const int64_t row = ((int64_t)pid * p.P + slot) * p.Hk + h;
            void* pool = is_v ? p.v_cache : p.k_cache;
            if (KV8) {
                uint2* d = static_cast<uint2*>(pool) + row * 16;
                d[c0] = make_uint2(a[i].x, a[i].y);
                d[c1] = make_uint2(e[i].x, e[i].y);
            } else {
                uint4* d = static_cast<uint4*>(pool) + row * 16;
                d[c0] = a[i];
                d[c1] = e[i];
            }
            if (!is_v && t == 0 && p.weights != nullptr)
                p.weights[((int64_t)pid * p.Hk + h) * p.P + slot] = 0.f;
        }
    }
}

bool strides_ok(const int64_t (&s)[3]) {
    // 16-byte pieces: every stride a multiple of 8 elements, none negative
    for (int i = 0; i < 3; ++i)
        if (s[i] < 0 || s[i] % 8 != 0) return false;
    return true;
}

int entry(const pgqa_rope_args* a, cudaStream_t stream) {
    if (a == nullptr) return PGQA_ERR_NULL_POINTER;
    if (a->struct_size != sizeof(pgqa_rope_args)) return PGQA_ERR_BAD_SHAPE;
    const bool append = a->k_new != nullptr || a->v_new != nullptr;
    if (!a->cos || !a->sin || (!append && !a->q) || (a->q && !a->q_out)) return PGQA_ERR_NULL_POINTER;
    if (append && (!a->k_new || !a->v_new || !a->k_cache || !a->v_cache || !a->seq_lens || !a->block_table))
        return PGQA_ERR_NULL_POINTER;
    if (!a->positions && !a->seq_lens) return PGQA_ERR_NULL_POINTER;
    const bool kv8 = a->kv_format == 1;
    if ((a->kv_format != 0 && !kv8) || (a->table_format != 0 && a->table_format != 1)) return PGQA_ERR_UNSUPPORTED;
    if (!kv8 && (a->k_scale || a->v_scale)) return PGQA_ERR_BAD_SHAPE;
    int st = PGQA_OK;
    if (append) {
        st = host_check_pages(a->batch_size, a->num_heads_k, a->headdim, a->page_size, a->num_pages, a->bt_stride);
    } else {
        if (a->weights || a->batch_size <= 0 || a->batch_size > INT32_MAX) return PGQA_ERR_BAD_SHAPE;
        if (a->headdim != 128) st = a->headdim <= 0 ? PGQA_ERR_BAD_SHAPE : PGQA_ERR_UNSUPPORTED;
    }
    if (st != PGQA_OK) return st;
    const int64_t Hq = a->q ? a->num_heads : 0, Hk = append ? a->num_heads_k : 0;
    if (Hq < 0 || (a->q && Hq == 0) || Hq > 65536 || Hk > 65536) return PGQA_ERR_BAD_SHAPE;
    if (a->tokens < 0 || a->table_rows <= 0 || a->num_axes < 1 || a->num_axes > 64) return PGQA_ERR_BAD_SHAPE;
    if (a->cu_seqlens == nullptr &&
        (a->seqlen < 0 || a->seqlen > INT32_MAX || a->tokens != a->batch_size * a->seqlen))
        return PGQA_ERR_BAD_SHAPE;
    if (a->tokens > INT32_MAX) return PGQA_ERR_UNSUPPORTED;
    if (a->rotary_dim <= 0 || a->rotary_dim > 128) return PGQA_ERR_BAD_SHAPE;
    if (a->rotary_dim % 16 != 0) return PGQA_ERR_UNSUPPORTED;
    if (a->num_axes > 1 && !a->positions) return PGQA_ERR_NULL_POINTER;
    for (int i = 0; i < a->rotary_dim / 2; ++i)
        if (a->pair_axis[i] >= a->num_axes) return PGQA_ERR_BAD_SHAPE;
    Params p = {};
    // a dimension of one entry may come with any stride: no address depends on it
    const bool used[3] = {!a->cu_seqlens && a->batch_size > 1, (a->cu_seqlens ? a->tokens : a->seqlen) > 1, true};
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = used[i] && (i < 2 || Hq > 1) ? a->q_strides[i] : 0;
        p.ks[i] = used[i] && (i < 2 || Hk > 1) ? a->k_strides[i] : 0;
        p.vs[i] = used[i] && (i < 2 || Hk > 1) ? a->v_strides[i] : 0;
    }
    if ((a->q && !strides_ok(p.qs)) || (append && (!strides_ok(p.ks) || !strides_ok(p.vs)))) return PGQA_ERR_MISALIGNED;
    if (!host_aligned(a->q, 16) || !host_aligned(a->k_new, 16) || !host_aligned(a->v_new, 16) ||
        !host_aligned(a->q_out, 16) || !host_aligned(a->k_cache, 16) || !host_aligned(a->v_cache, 16) ||
        !host_aligned(a->cos, 16) || !host_aligned(a->sin, 16) || !host_aligned(a->seq_lens, 4) ||
        !host_aligned(a->block_table, 4) || !host_aligned(a->positions, 4) || !host_aligned(a->cu_seqlens, 4) ||
        !host_aligned(a->weights, 4) || !host_aligned(a->k_scale, 4) || !host_aligned(a->v_scale, 4))
        return PGQA_ERR_MISALIGNED;
    int dev, sms, optin;
    if ((st = host_device(&dev, &sms, &optin)) != PGQA_OK) return st;
    if ((st = host_error_word(dev, &p.err)) != PGQA_OK) return st;
    if (a->tokens == 0) return PGQA_OK;
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.k = static_cast<const __nv_bfloat16*>(a->k_new);
    p.v = static_cast<const __nv_bfloat16*>(a->v_new);
    p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.seq_lens = a->seq_lens;
    p.block_table = a->block_table;
    p.positions = a->positions;
    p.cu = a->cu_seqlens;
    p.cos = a->cos;
    p.sin = a->sin;
    p.weights = a->weights;
    p.k_scale = a->k_scale;
    p.v_scale = a->v_scale;
    p.T = a->tokens;
    p.bt_stride = a->bt_stride;
    p.cap_tokens = a->bt_stride * a->page_size;
    p.table_rows = a->table_rows;
    p.B = (int32_t)a->batch_size;
    p.S = (int32_t)a->seqlen;
    p.Hq = (int32_t)Hq;
    p.Hk = (int32_t)Hk;
    p.P = (int32_t)a->page_size;
    p.page_shift = host_shift(a->page_size);
    p.num_pages = (int32_t)a->num_pages;
    const int64_t rows = Hq + 2 * Hk;
    p.blocks = (int32_t)((rows + 4 * kRowsPerLane - 1) / (4 * kRowsPerLane));
    p.rows_per_block = (int32_t)(((rows + p.blocks - 1) / p.blocks + 3) / 4 * 4);
    p.R = (int32_t)a->rotary_dim;
    p.interleaved = a->interleaved != 0;
    p.table_bf16 = a->table_format == 1;
    p.runs8 = 1;
    for (int i = 0; i < 64; ++i) {
        p.axis[i] = i < p.R / 2 ? a->pair_axis[i] : 0;
        if (i < p.R / 2 && p.axis[i] != p.axis[i & ~7]) p.runs8 = 0;
    }
    const int64_t warps = p.T * p.blocks;
    const int64_t ctas = (warps + kThreads / 32 - 1) / (kThreads / 32);
    if (ctas > INT32_MAX) return PGQA_ERR_UNSUPPORTED;
    auto kern = kv8 ? rope_append_kernel<true> : rope_append_kernel<false>;
    return host_launch(kern, dim3((unsigned)ctas), kThreads, 0, stream, 1, p);
}

}  // namespace rope
}  // namespace pgqa

extern "C" int pgqa_rope_append(const pgqa_rope_args* args, void* stream) {
    return pgqa::host_set_status(pgqa::rope::entry(args, static_cast<cudaStream_t>(stream)));
}
