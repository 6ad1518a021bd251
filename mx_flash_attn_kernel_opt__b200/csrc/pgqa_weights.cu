/*
 * pgqa_weights.cu - the attention weight that each cached token receives, added to its
 * entry of the weight pool [num_pages, Hkv, P]:
 *
 *     w[b, kv, t] += sum over rows r of KV head kv that see t of exp(scale q_r . k_t - lse_r)
 *
 * with the rows (query head, query token) and the masks of the decode, and lse_r the
 * log-sum-exp that the decode returned for the row.  Scores, exponents and sums are fp32.
 *
 * Bound by the one pass over K (256 or 128 bytes per token and KV head against 8 bytes of
 * weights).  Each warp owns an equal contiguous slice of 16-token chunks over the actual
 * lengths (the same cut as the decode's, in units of warps) and works alone: no shared
 * memory rings and no barriers in the stream.  K goes from global memory straight into
 * mma.sync A fragments: the order of the 128 dimensions inside the dot product is free as
 * long as q uses the same one, so lane (g, t) takes 16-byte pieces t, t + 4, ... of token
 * rows g and g + 8, whole 64-byte runs per row, and q rows are loaded by the same
 * addresses as B fragments.  Two or three chunks
 * are held, one at work and the others in flight.  The four lanes
 * that share a token add their partial sums by shuffles, and the token's weight gets one
 * red.add for every 32 query rows, all from the same lane: no other warp of the call adds to it
 * (unless sequences share a page), so the result does not depend on any order.
 *
 * e4m3 keys become f16 in registers, exactly (4 significant bits), and q is turned into f16
 * once per unit: each row times the power of two that brings its largest element to [2^14,
 * 2^15), undone in fp32.  8 significant bits fit f16's 11; elements more than 2^31 times smaller
 * than their row's largest are rounded to a multiple of 2^-24, which is off by 2^-39 of the
 * largest at most.  Rows whose largest is below 2^-112 are only brought up by 2^126.
 *
 * Measured: 290,000 tokens in 256 sequences, 8 KV heads, 4 rows each, bf16 101 us (6.1 TB/s,
 * 0.93 of a copy's rate).  2 sequences of 32,768 tokens, 8 KV heads, rows per KV head:
 *               1      8     16     32     64    256   (us; start and end of the call, about 8)
 *   bf16       27     27     28     36     66    240   K takes 21 us to read
 *   e4m3       20     20     24     31     54    190   11 us
 * From 32 rows on the products and exponentials of a chunk take longer than its load, and every
 * 32 rows are a pass over K of their own.  Rows that are no multiple of 16 or 32 cost as much as
 * the next one, and lose the path without comparisons (28 rows over 4 KV heads, half the
 * keys: 24 us bf16, 22 us e4m3, where half of the 32 rows' are 18 and 16).
 */
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pgqa_host.h"
#include "pgqa_partition.h"
#include "pgqa_ptx.cuh"

namespace pgqa {
namespace weights {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct Params {
    const __nv_bfloat16* q;  // [B, Sq, Hq, 128]
    const void* k_cache;
    const float* lse;        // [B, Hq, Sq]
    float* weights;          // [num_pages, Hkv, P]
    const int32_t *seq_lens, *block_table;
    const float* k_scale;
    int32_t* err;
    int64_t bt_stride, cap_tokens;
    int32_t B, Sq, Hq, Hkv, g, rows, P, page_shift, num_pages, causal;
    float scale_log2;
};

/* One 16-token chunk of one KV head in A-fragment order: per lane, pieces of rows g and g + 8. */
template <bool KV8>
struct Chunk {
    static constexpr int kPieces = KV8 ? 2 : 4;
    uint4 lo[kPieces], hi[kPieces];
};

/* q fragments of one group of 8 rows, in the dimension order of the chunk's pieces. */
struct QFrag {
    uint4 v[4];
};

__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t v, float up) {
    return ptx::pack_f16x2(__uint_as_float(v << 16) * up, __uint_as_float(v & 0xffff0000u) * up);
}

/* Row r of the unit (b, kvh): query head r / Sq of the group, query token r % Sq. */
__device__ __forceinline__ void row_of(const Params& p, int32_t b, int32_t kvh, int r, int64_t& qoff, int64_t& loff,
                                       int32_t& tok) {
    const int h = r / p.Sq;
    tok = r - h * p.Sq;
    const int head = kvh * p.g + h;
    qoff = (((int64_t)b * p.Sq + tok) * p.Hq + head) * 128;
    loff = ((int64_t)b * p.Hq + head) * p.Sq + tok;
}

/* Per lane: the q pieces of row 8 j + g, and for rows 8 j + 2 t, 8 j + 2 t + 1 (its two
 * columns of the score tile) the score's factor in log2 units, the negated log2-sum-exp and
 * the number of tokens seen. */
template <bool KV8>
__device__ __forceinline__ void load_group(const Params& p, int32_t b, int32_t kvh, int32_t L, float mul, int j,
                                           int lane, QFrag& f, float (&ml)[2], float (&nl)[2], int32_t (&lim)[2]) {
    const int g = lane >> 2, t = lane & 3;
    int64_t qo, lo;
    int32_t tok;
    const int r = 8 * j + g;
    if (r < p.rows) {
        row_of(p, b, kvh, r, qo, lo, tok);
        const uint4* src = reinterpret_cast<const uint4*>(p.q + qo);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            // e4m3: a 16-byte piece of K covers two consecutive pieces of q
            f.v[i] = ptx::ld(src + (KV8 ? 8 * (i >> 1) + 2 * t + (i & 1) : 4 * i + t));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f.v[i] = make_uint4(0, 0, 0, 0);
    }
    float down = 1.f;
    if (KV8) {
        uint32_t mx = 0;  // largest magnitude of the row, as its bits
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w[4] = {f.v[i].x, f.v[i].y, f.v[i].z, f.v[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = max(mx, max(w[e] << 16 & 0x7fffffffu, w[e] & 0x7fff0000u));
        }
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // every finite maximum down to 2^-112; 2^e and 2^-e are both normal numbers
        const int e = max(-113, min(126, 14 - ((int)(mx >> 23) - 127)));
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            f.v[i] = make_uint4(bf16x2_to_f16x2(f.v[i].x, up), bf16x2_to_f16x2(f.v[i].y, up),
                                bf16x2_to_f16x2(f.v[i].z, up), bf16x2_to_f16x2(f.v[i].w, up));
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int c = 8 * j + 2 * t + e;
        ml[e] = mul;
        if (KV8) ml[e] *= __shfl_sync(0xffffffffu, down, 4 * (2 * t + e));
        nl[e] = 0.f;
        lim[e] = 0;
        if (c < p.rows) {
            row_of(p, b, kvh, c, qo, lo, tok);
            const float l = ptx::ld(p.lse + lo);
            // a row that saw nothing (-inf) has no weight to give
            if (l != -INFINITY) {
                nl[e] = -l * 1.4426950408889634f;
                lim[e] = p.causal ? L - p.Sq + 1 + tok : L;
            }
        }
    }
}

template <bool KV8>
__device__ __forceinline__ void load_chunk(const Params& p, int32_t pid, int32_t slot, int32_t kvh, int lane,
                                           Chunk<KV8>& c) {
    const int g = lane >> 2, t = lane & 3;
    constexpr int kRow = KV8 ? 8 : 16;  // 16-byte pieces per token row
    const int64_t row = ((int64_t)pid * p.P + slot + g) * p.Hkv + kvh;
    const uint4* a = static_cast<const uint4*>(p.k_cache) + row * kRow + t;
    const uint4* d = a + (int64_t)8 * p.Hkv * kRow;
#pragma unroll
    for (int i = 0; i < Chunk<KV8>::kPieces; ++i) {
        c.lo[i] = __ldcg(a + 4 * i);  // read once: no line in L1
        c.hi[i] = __ldcg(d + 4 * i);
    }
}

/* A chunk's A fragments of the eight 16-dimension steps. */
struct AFrag {
    uint32_t a[8][4];
};

/* e4m3 is converted once per chunk, not per group of rows: the conversions are what the SM
 * does fewest of per clock here. */
template <bool KV8>
__device__ __forceinline__ void fragments(const Chunk<KV8>& c, AFrag& f) {
#pragma unroll
    for (int i = 0; i < Chunk<KV8>::kPieces; ++i) {
        const uint32_t lo[4] = {c.lo[i].x, c.lo[i].y, c.lo[i].z, c.lo[i].w};
        const uint32_t hi[4] = {c.hi[i].x, c.hi[i].y, c.hi[i].z, c.hi[i].w};
        if (!KV8) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint32_t(&a)[4] = f.a[(2 * i + s) & 7];
                a[0] = lo[2 * s];
                a[1] = hi[2 * s];
                a[2] = lo[2 * s + 1];
                a[3] = hi[2 * s + 1];
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                uint32_t(&a)[4] = f.a[(4 * i + s) & 7];
                ptx::e4m3x4_to_f16(lo[s], a[0], a[2]);
                ptx::e4m3x4_to_f16(hi[s], a[1], a[3]);
            }
        }
    }
}

/* Scores of the chunk's 16 tokens against 8 rows: two chains of four products each. */
template <bool KV8>
__device__ __forceinline__ void scores(const AFrag& f, const QFrag& q, float (&s)[4]) {
    float u[4] = {0.f, 0.f, 0.f, 0.f};
    s[0] = s[1] = s[2] = s[3] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint4 v = q.v[i >> 1];
        const uint32_t b0 = (i & 1) ? v.z : v.x, b1 = (i & 1) ? v.w : v.y;
        float(&d)[4] = (i & 1) ? u : s;
        if (KV8) ptx::mma_f16_16816(d, f.a[i][0], f.a[i][1], f.a[i][2], f.a[i][3], b0, b1);
        else ptx::mma_bf16_16816(d, f.a[i][0], f.a[i][1], f.a[i][2], f.a[i][3], b0, b1);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += u[e];
}

/* Chunks held by a warp: the one at work and those in flight. */
__host__ __device__ constexpr int depth(bool KV8, int NT) { return KV8 && NT == 1 ? 3 : 2; }
/* Shared memory of a warp for the q fragments of NT >= 2 groups, which would leave the
 * registers no room for the chunks in flight, and for their columns' factors and bounds. */
struct Cols {
    float ml[2], nl[2];
    int32_t lim[2];
    int32_t pad[2];
};
__host__ __device__ constexpr int warp_smem(int NT) { return NT >= 2 ? NT * (4 * 32 * 16 + 4 * (int)sizeof(Cols)) : 0; }

/* NT groups of 8 rows at a time, their q fragments held over a unit: in registers for one, in
 * the warp's shared memory for two or four.  More than 32 rows take several turns over the
 * warp's chunks; a token's additions then come from the same lane, in the turns' order. */
template <bool KV8, int NT>
__global__ void __launch_bounds__(kThreads, 2) weights_kernel(const Params p) {
    extern __shared__ uint4 smem[];  // the warps' q fragments, then pre
    uint32_t* pre = reinterpret_cast<uint32_t*>(smem) + kWarps * warp_smem(NT) / 4;  // chunks of the sequences before b, [B + 1]
    __shared__ uint32_t wsum[kWarps];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    {
        const int per = (p.B + kThreads - 1) / kThreads;
        const int s0 = min(p.B, tid * per), s1 = min(p.B, s0 + per);
        uint32_t local = 0;
        bool bad = false;
        for (int b = s0; b < s1; ++b) {
            const int32_t L = ptx::ld(p.seq_lens + b);
            bad = bad || L < 0 || L > p.cap_tokens;
            local += (uint32_t)seq_chunks(L, p.cap_tokens);
        }
        if (bad && blockIdx.x == 0) atomicOr(p.err, kDevErrBadSeqlen);
        uint32_t incl = local;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) wsum[warp] = incl;
        __syncthreads();
        uint32_t run = incl - local;
        for (int w = 0; w < warp; ++w) run += wsum[w];
        for (int b = s0; b < s1; ++b) {
            pre[b] = run;
            run += (uint32_t)seq_chunks(ptx::ld(p.seq_lens + b), p.cap_tokens);
        }
        if (s1 == p.B) pre[p.B] = run;  // every thread past the last sequence writes the same total
        __syncthreads();
    }
    const int64_t total = (int64_t)pre[p.B] * p.Hkv;
    const int64_t nw = (int64_t)gridDim.x * kWarps;
    const int64_t w = (int64_t)warp * gridDim.x + blockIdx.x;  // few chunks: spread over the SMs first
    int64_t cur = slice_begin(w, nw, total);
    const int64_t end = slice_begin(w + 1, nw, total);
    if (cur >= end) return;
    int32_t lo = 0, hi = p.B;
    while (hi - lo > 1) {
        const int32_t mid = (lo + hi) >> 1;
        if ((int64_t)pre[mid] * p.Hkv <= cur) lo = mid; else hi = mid;
    }
    int32_t b = lo;
    int32_t n = (int32_t)(pre[b + 1] - pre[b]);
    const int64_t in = cur - (int64_t)pre[b] * p.Hkv;
    int32_t kvh = (int32_t)(in / n), c = (int32_t)(in - (int64_t)kvh * n);
    const int t = lane & 3, g = lane >> 2;
    uint4* const my_q = smem + warp * (warp_smem(NT) / 16) + lane;
    Cols* const my_cols = reinterpret_cast<Cols*>(smem + warp * (warp_smem(NT) / 16) + NT * 128) + t;
    constexpr int D = depth(KV8, NT);
    const int groups = (p.rows + 7) / 8;

    while (cur < end) {
        // the slice's part of the unit (b, kvh): chunks [c, ce)
        const int32_t ce = (int32_t)((end - cur < n - c) ? c + (end - cur) : n);
        const int64_t L64 = ptx::ld(p.seq_lens + b);
        const int32_t L = (int32_t)(L64 > p.cap_tokens ? p.cap_tokens : L64);
        const float ks = (KV8 && p.k_scale) ? ptx::ld(p.k_scale + kvh) : 1.f;
        const float mul = p.scale_log2 * ks;
        const int32_t* bt = p.block_table + (int64_t)b * p.bt_stride;
        auto page_of = [&](int32_t chunk, int32_t& pid, int32_t& slot) {
            const int32_t tok = chunk * kChunkTokens;
            const int32_t page = p.page_shift >= 0 ? tok >> p.page_shift : tok / p.P;
            slot = tok - page * p.P;
            pid = ptx::ld(bt + page);
        };
        auto check = [&](int32_t& pid) -> bool {
            if ((uint32_t)pid < (uint32_t)p.num_pages) return true;
            if (lane == 0) atomicOr(p.err, kDevErrBadPage);
            pid = 0;  // read, not added to
            return false;
        };
        const int32_t c_first = c;
#pragma unroll 1
        for (int j0 = 0; j0 < groups; j0 += NT) {
            c = c_first;
            QFrag qf;
            Cols cl;
            int32_t all_see = INT32_MAX;  // every row of the turn sees the tokens before this one
            if (NT == 1) {
                load_group<KV8>(p, b, kvh, L, mul, 0, lane, qf, cl.ml, cl.nl, cl.lim);
            } else {
                __syncwarp();  // the last rows' are no longer read
#pragma unroll 1
                for (int j = 0; j < NT; ++j) {
                    load_group<KV8>(p, b, kvh, L, mul, j0 + j, lane, qf, cl.ml, cl.nl, cl.lim);
#pragma unroll
                    for (int i = 0; i < 4; ++i) my_q[(4 * j + i) * 32] = qf.v[i];
                    if (g == 0) my_cols[4 * j] = cl;
                    all_see = min(all_see, min(cl.lim[0], cl.lim[1]));
                }
                all_see = __reduce_min_sync(0xffffffffu, all_see);
                __syncwarp();
            }
            Chunk<KV8> ring[D];
            int32_t pid[D], slot[D];
            bool ok[D];
#pragma unroll
            for (int u = 0; u < D; ++u) {
                if (c + u < ce) {
                    page_of(c + u, pid[u], slot[u]);
                    ok[u] = check(pid[u]);
                    load_chunk<KV8>(p, pid[u], slot[u], kvh, lane, ring[u]);
                }
            }
            int32_t npid = 0, nslot = 0;  // of the chunk to be loaded next
            if (c + D < ce) page_of(c + D, npid, nslot);
            auto work = [&](const Chunk<KV8>& k, int32_t pid, int32_t slot, bool ok, int32_t c) {
                const int32_t tok = c * kChunkTokens + g;
                AFrag fr;
                fragments<KV8>(k, fr);
                float w0 = 0.f, w1 = 0.f;  // weights of tokens g and g + 8 over this lane's rows
                auto add = [&](const QFrag& f, const Cols& c) {
                    float s[4];
                    scores<KV8>(fr, f, s);
                    // selected, never multiplied: a masked score may be infinite or NaN
                    w0 += tok < c.lim[0] ? ptx::ex2(fmaf(s[0], c.ml[0], c.nl[0])) : 0.f;
                    w0 += tok < c.lim[1] ? ptx::ex2(fmaf(s[1], c.ml[1], c.nl[1])) : 0.f;
                    w1 += tok + 8 < c.lim[0] ? ptx::ex2(fmaf(s[2], c.ml[0], c.nl[0])) : 0.f;
                    w1 += tok + 8 < c.lim[1] ? ptx::ex2(fmaf(s[3], c.ml[1], c.nl[1])) : 0.f;
                };
                auto add_all = [&](const QFrag& f, const Cols& c) {  // no row masks a token of the chunk
                    float s[4];
                    scores<KV8>(fr, f, s);
                    w0 += ptx::ex2(fmaf(s[0], c.ml[0], c.nl[0]));
                    w0 += ptx::ex2(fmaf(s[1], c.ml[1], c.nl[1]));
                    w1 += ptx::ex2(fmaf(s[2], c.ml[0], c.nl[0]));
                    w1 += ptx::ex2(fmaf(s[3], c.ml[1], c.nl[1]));
                };
                if (NT == 1) {
                    add(qf, cl);
                } else if ((c + 1) * kChunkTokens <= all_see) {
                    // nearly every chunk of a long sequence, in turns without a padding row or a row
                    // that saw nothing (their bounds are 0): no comparisons and no selects (2
                    // sequences of 32,768 tokens, 32 rows: 33.7 -> 30.9 us e4m3, 40.2 -> 36.2 us bf16)
#pragma unroll 4
                    for (int j = 0; j < NT; ++j) {
                        QFrag f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) f.v[i] = my_q[(4 * j + i) * 32];
                        add_all(f, my_cols[4 * j]);
                    }
                } else {
#pragma unroll 1
                    for (int j = 0; j < NT; ++j) {
                        QFrag f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) f.v[i] = my_q[(4 * j + i) * 32];
                        add(f, my_cols[4 * j]);
                    }
                }
                w0 += __shfl_xor_sync(0xffffffffu, w0, 1);
                w1 += __shfl_xor_sync(0xffffffffu, w1, 1);
                w0 += __shfl_xor_sync(0xffffffffu, w0, 2);
                w1 += __shfl_xor_sync(0xffffffffu, w1, 2);
                if (ok && t < 2) {
                    const int i = g + 8 * t;
                    if (c * kChunkTokens + i < L)
                        atomicAdd(p.weights + ((int64_t)pid * p.Hkv + kvh) * p.P + slot + i, t == 0 ? w0 : w1);
                }
            };
            for (; c < ce; c += D) {
#pragma unroll
                for (int u = 0; u < D; ++u) {
                    if (c + u >= ce) break;
                    work(ring[u], pid[u], slot[u], ok[u], c + u);
                    if (c + u + D < ce) {
                        pid[u] = npid;
                        slot[u] = nslot;
                        ok[u] = check(pid[u]);
                        load_chunk<KV8>(p, pid[u], slot[u], kvh, lane, ring[u]);
                        if (c + u + D + 1 < ce) page_of(c + u + D + 1, npid, nslot);
                    }
                }
            }
        }
        cur = (int64_t)pre[b] * p.Hkv + (int64_t)kvh * n + ce;
        c = 0;
        if (cur < end && ++kvh == p.Hkv) {
            kvh = 0;
            do { ++b; } while (pre[b + 1] == pre[b]);
            n = (int32_t)(pre[b + 1] - pre[b]);
        }
    }
}

template <bool KV8, int NT>
int launch(const Params& p, int dev, int sms, int optin, cudaStream_t stream) {
    const int smem = kWarps * warp_smem(NT) + (p.B + 1) * 4;
    // the chunk counts before each sequence live in shared memory; two CTAs per SM (the static
    // bytes and the system's fit into the 1024)
    const int most = optin / 2 - 1024;
    if (smem > most) return PGQA_ERR_UNSUPPORTED;
    static HostSmemDone done;
    auto kern = weights_kernel<KV8, NT>;
    const int st = host_smem_limit(kern, dev, most, done);
    if (st != PGQA_OK) return st;
    return host_launch(kern, dim3((unsigned)(2 * sms)), kThreads, (size_t)smem, stream, 1, p);
}

template <bool KV8>
int launch_nt(const Params& p, int dev, int sms, int optin, cudaStream_t stream) {
    if (p.rows <= 8) return launch<KV8, 1>(p, dev, sms, optin, stream);
    if (p.rows <= 16) return launch<KV8, 2>(p, dev, sms, optin, stream);
    return launch<KV8, 4>(p, dev, sms, optin, stream);
}

int entry(const pgqa_weights_args* a, cudaStream_t stream) {
    if (a == nullptr) return PGQA_ERR_NULL_POINTER;
    if (a->struct_size != sizeof(pgqa_weights_args)) return PGQA_ERR_BAD_SHAPE;
    if (!a->q || !a->k_cache || !a->softmax_lse || !a->weights || !a->seq_lens || !a->block_table)
        return PGQA_ERR_NULL_POINTER;
    int st = host_check_pages(a->batch_size, a->num_heads_k, a->headdim, a->page_size, a->num_pages, a->bt_stride);
    if (st != PGQA_OK) return st;
    if (a->num_heads <= 0 || a->num_heads % a->num_heads_k != 0 || a->num_heads > 65536) return PGQA_ERR_BAD_SHAPE;
    if (a->seqlen_q <= 0) return PGQA_ERR_BAD_SHAPE;
    if (a->seqlen_q > 4096) return PGQA_ERR_UNSUPPORTED;
    if (a->causal != 0 && a->causal != 1) return PGQA_ERR_BAD_SHAPE;
    if (!(a->scale > 0.f) || !isfinite(a->scale)) return PGQA_ERR_BAD_SHAPE;
    if (a->kv_format != 0 && a->kv_format != 1) return PGQA_ERR_UNSUPPORTED;
    if (a->kv_format == 0 && a->k_scale) return PGQA_ERR_BAD_SHAPE;
    if (!host_aligned(a->q, 16) || !host_aligned(a->k_cache, 16) || !host_aligned(a->softmax_lse, 4) ||
        !host_aligned(a->weights, 4) || !host_aligned(a->seq_lens, 4) || !host_aligned(a->block_table, 4) ||
        !host_aligned(a->k_scale, 4))
        return PGQA_ERR_MISALIGNED;
    int dev, sms, optin;
    if ((st = host_device(&dev, &sms, &optin)) != PGQA_OK) return st;
    if (a->batch_size > optin / 8) return PGQA_ERR_UNSUPPORTED;  // (see launch)
    Params p = {};
    if ((st = host_error_word(dev, &p.err)) != PGQA_OK) return st;
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.k_cache = a->k_cache;
    p.lse = a->softmax_lse;
    p.weights = a->weights;
    p.seq_lens = a->seq_lens;
    p.block_table = a->block_table;
    p.k_scale = a->k_scale;
    p.bt_stride = a->bt_stride;
    p.cap_tokens = a->bt_stride * a->page_size;
    p.B = (int32_t)a->batch_size;
    p.Sq = (int32_t)a->seqlen_q;
    p.Hq = (int32_t)a->num_heads;
    p.Hkv = (int32_t)a->num_heads_k;
    p.g = p.Hq / p.Hkv;
    p.rows = p.g * p.Sq;
    p.P = (int32_t)a->page_size;
    p.page_shift = host_shift(a->page_size);
    p.num_pages = (int32_t)a->num_pages;
    p.causal = (int32_t)a->causal;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    return a->kv_format == 1 ? launch_nt<true>(p, dev, sms, optin, stream)
                             : launch_nt<false>(p, dev, sms, optin, stream);
}

}  // namespace weights
}  // namespace pgqa

extern "C" int pgqa_accumulate_weights(const pgqa_weights_args* args, void* stream) {
    return pgqa::host_set_status(pgqa::weights::entry(args, static_cast<cudaStream_t>(stream)));
}
