/*
 * pgqa_evict.cu - eviction from the paged cache by accumulated attention weight.
 *
 * A sequence of L > keep tokens is cut to `keep` of them, for each KV head on its own: its
 * first `sinks`, its last `recent`, and between them the keep - sinks - recent tokens of
 * the highest weight (equal weights: the lowest index first; a NaN counts as the highest).
 * The kept tokens keep their order and move to slots [0, keep) of the sequence's own pages;
 * their indices go to kept[b, kv, :].  A sequence of L <= keep stays as it is (kept: 0 .. L-1,
 * then -1).
 *
 * Two launches:
 *
 * select_kernel, one CTA per (sequence, KV head).  The middle tokens' weights become
 * sortable 32-bit keys in shared memory (or are re-read from L2 when they do not fit); a
 * radix select over digits of 11, 11 and 10 bits finds the key of the last token kept and
 * how many of its equals stay, and one ordered pass with a block scan writes the indices.
 * 4 bytes per token are read from HBM once.
 *
 * move_kernel, in place.  Row j of the result comes from row kept[j] >= j, and kept is
 * ascending, so a CTA that goes through j in ascending batches may overwrite [j0, j0 + n)
 * as soon as its own loads of that batch are done: every later source lies at j0 + n or
 * above.  One barrier per batch orders the two, and the next batch's loads are in flight
 * across it.  Different byte columns of the rows never meet, so (K or V) x column ranges
 * x (sequence, KV head) are independent CTAs: the rule below takes as few columns as fill
 * the SMs.  Rows before the first evicted one are not touched.  Bound by reading and
 * writing the moved rows.
 */
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pgqa_host.h"
#include "pgqa_ptx.cuh"

namespace pgqa {
namespace evict {

constexpr int kSelThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kMoveDepth = 8;          // 16-byte pieces a thread holds per batch
constexpr int kBins = 2048;
constexpr int kMaxKeys = 48 * 1024;    // keys held in shared memory (192 KB)

struct Params {
    void *k_cache, *v_cache;
    const float* weights;
    float* weights_out;
    const int32_t *seq_lens, *block_table;
    int32_t *kept, *new_lens;
    int32_t* err;
    int64_t bt_stride, cap_tokens;
    int32_t Hkv, P, page_shift, num_pages, keep, sinks, recent;
    int32_t smem_keys;               // keys that fit in the launch's shared memory
    int32_t row_pieces, col_pieces;  // 16-byte pieces in a row, and in one CTA's columns
    int32_t cols;                    // column ranges per row
};

__device__ __forceinline__ int32_t page_of(const Params& p, int32_t tok) {
    return p.page_shift >= 0 ? tok >> p.page_shift : tok / p.P;
}

__device__ __forceinline__ int32_t length_of(const Params& p, int32_t b) {
    const int32_t L = __ldg(p.seq_lens + b);
    return L < 0 ? 0 : (L > p.cap_tokens ? (int32_t)p.cap_tokens : L);
}

/* Order-preserving key of a weight: larger weight, larger key; -0 equals +0, NaN is highest. */
__device__ __forceinline__ uint32_t key_of(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(kSelThreads) select_kernel(const Params p) {
    extern __shared__ uint32_t keys[];
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t wsum[32];
    __shared__ uint32_t found[2];  // the digit of the last kept key, and how many above it
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t b = blockIdx.x / p.Hkv, h = blockIdx.x - b * p.Hkv;
    const int32_t L0 = __ldg(p.seq_lens + b);
    const int32_t L = length_of(p, b);
    if (h == 0 && tid == 0) {
        if (L != L0) atomicOr(p.err, kDevErrBadSeqlen);
        p.new_lens[b] = min(L, p.keep);
    }
    int32_t* kept = p.kept + (int64_t)blockIdx.x * p.keep;
    if (L <= p.keep) {
        for (int j = tid; j < p.keep; j += kSelThreads) kept[j] = j < L ? j : -1;
        return;
    }
    const int32_t M = L - p.sinks - p.recent;            // candidates
    const int32_t m = p.keep - p.sinks - p.recent;       // of which m < M stay
    for (int j = tid; j < p.sinks; j += kSelThreads) kept[j] = j;
    for (int j = tid; j < p.recent; j += kSelThreads) kept[p.sinks + m + j] = L - p.recent + j;
    if (m == 0) return;
    const int32_t* bt = p.block_table + (int64_t)b * p.bt_stride;
    const bool held = M <= p.smem_keys;
    bool bad = false;
    auto load_key = [&](int32_t i) -> uint32_t {
        const int32_t tok = p.sinks + i;
        const int32_t page = page_of(p, tok);
        const int32_t pid = __ldg(bt + page);
        if ((uint32_t)pid >= (uint32_t)p.num_pages) {
            bad = true;
            return 0;
        }
        return key_of(__ldg(p.weights + ((int64_t)pid * p.Hkv + h) * p.P + (tok - page * p.P)));
    };
    if (held) {
        // four loads in flight per thread
        for (int32_t i0 = tid; i0 < M; i0 += 4 * kSelThreads) {
            uint32_t k[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) k[u] = i0 + u * kSelThreads < M ? load_key(i0 + u * kSelThreads) : 0;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i0 + u * kSelThreads < M) keys[i0 + u * kSelThreads] = k[u];
        }
        __syncthreads();
    }
    auto key_at = [&](int32_t i) -> uint32_t { return held ? keys[i] : load_key(i); };

    uint32_t prefix = 0, mask = 0;  // digits fixed so far
    uint32_t need = (uint32_t)m;    // tokens still to take among those that match them
    bool all = false;               // every match of `prefix` stays
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
        const int bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int32_t i = tid; i < M; i += kSelThreads) {
            const uint32_t k = key_at(i);
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // counts from the top: thread t owns bins 2047 - 2 t and 2046 - 2 t
        const uint32_t h0 = hist[kBins - 1 - 2 * tid], h1 = hist[kBins - 2 - 2 * tid];
        uint32_t incl = h0 + h1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) wsum[warp] = incl;
        __syncthreads();
        uint32_t above = incl - h0 - h1;
        for (int w = 0; w < warp; ++w) above += wsum[w];
        if (above < need && need <= above + h0) {
            found[0] = (uint32_t)(kBins - 1 - 2 * tid);
            found[1] = above;
        } else if (above + h0 < need && need <= above + h0 + h1) {
            found[0] = (uint32_t)(kBins - 2 - 2 * tid);
            found[1] = above + h0;
        }
        __syncthreads();
        const uint32_t digit = found[0];
        need -= found[1];
        prefix |= digit << shift;
        mask |= ((1u << bits) - 1) << shift;
        all = hist[digit] == need;
        if (all) break;
        __syncthreads();
    }
    // kept: keys above the prefix (under its mask), and the first `need` that match it
    int32_t base = p.sinks;
    uint32_t eq_before = 0;
    for (int32_t i0 = 0; i0 < M; i0 += 4 * kSelThreads) {
        uint32_t cnt = 0, flags = 0;  // (above | equal << 16) of this thread's four tokens
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int32_t i = i0 + 4 * tid + u;
            if (i < M) {
                const uint32_t k = key_at(i) & mask;
                if (k > prefix) {
                    cnt += 1;
                    flags |= 1u << u;
                } else if (k == prefix) {
                    cnt += 0x10000u;
                    flags |= 16u << u;
                }
            }
        }
        uint32_t incl = cnt;  // at most 4096 of each kind: no carry between the halves
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        __syncthreads();
        if (lane == 31) wsum[warp] = incl;
        __syncthreads();
        uint32_t before = incl - cnt, total = 0;
        for (int w = 0; w < 32; ++w) {
            const uint32_t v = wsum[w];
            if (w < warp) before += v;
            total += v;
        }
        uint32_t gt = before & 0xffffu, eq = eq_before + (before >> 16);
        const uint32_t eq0 = eq_before < need ? eq_before : need;  // equals already taken in `base`
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int32_t tok = p.sinks + i0 + 4 * tid + u;
            const uint32_t taken = (eq < need ? eq : need) - eq0;
            if (flags & (1u << u)) {
                kept[base + gt + taken] = tok;
                ++gt;
            } else if (flags & (16u << u)) {
                if (eq < need) kept[base + gt + taken] = tok;
                ++eq;
            }
        }
        eq_before += total >> 16;
        base += (int32_t)((total & 0xffffu) + (eq_before < need ? eq_before : need) - eq0);
    }
    if (bad) atomicOr(p.err, kDevErrBadPage);
}

/* Slot of token `tok` in the pool's token order, or -1 for a bad page. */
__device__ __forceinline__ int32_t slot_of(const Params& p, const int32_t* bt, int32_t tok, int32_t& pid) {
    const int32_t page = page_of(p, tok);
    pid = __ldg(bt + page);
    if ((uint32_t)pid >= (uint32_t)p.num_pages) {
        atomicOr(p.err, kDevErrBadPage);
        return -1;
    }
    return tok - page * p.P;
}

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const Params p) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int tid = threadIdx.x;
    const int32_t b = blockIdx.x / p.Hkv, h = blockIdx.x - b * p.Hkv;
    const int32_t L = length_of(p, b);
    const int32_t* kept = p.kept + (int64_t)blockIdx.x * p.keep;
    const int32_t* bt = p.block_table + (int64_t)b * p.bt_stride;
    const int part = blockIdx.y;
    if (part == 2 * p.cols) {
        // the weights: one 4-byte element per token
        const bool in_place = p.weights_out == p.weights;
        const int32_t n = min(L, p.keep);
        if (in_place && L <= p.keep) return;
        constexpr int kU = 4;
        for (int32_t j0 = 0; j0 < n; j0 += kU * kMoveThreads) {
            float v[kU];
            int64_t dst[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int32_t j = j0 + u * kMoveThreads + tid;
                dst[u] = -1;
                if (j < n) {
                    const int32_t src = __ldg(kept + j);
                    int32_t sp, dp;
                    const int32_t ss = slot_of(p, bt, src, sp), ds = slot_of(p, bt, j, dp);
                    if (ss >= 0 && ds >= 0 && !(in_place && src == j)) {
                        // not __ldg: in place this array is written by the same kernel
                        v[u] = __ldcg(p.weights + ((int64_t)sp * p.Hkv + h) * p.P + ss);
                        dst[u] = ((int64_t)dp * p.Hkv + h) * p.P + ds;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (dst[u] >= 0) p.weights_out[dst[u]] = v[u];
        }
        return;
    }
    if (L <= p.keep) return;
    uint4* pool = static_cast<uint4*>(part < p.cols ? p.k_cache : p.v_cache);
    const int col = (part < p.cols ? part : part - p.cols) * p.col_pieces;
    const int piece = col + tid % p.col_pieces, r0 = tid / p.col_pieces;
    const int rows = kMoveThreads / p.col_pieces;  // rows that the CTA covers at a time
    const int32_t n = p.keep, batch = rows * kMoveDepth;
    // rows that stay where they are form a prefix; skip whole strides of it
    const int32_t stride = (n + kMoveThreads - 1) / kMoveThreads;
    const bool still = tid * stride < n && __ldg(kept + tid * stride) == tid * stride;
    const int32_t fixed = __syncthreads_count(still);
    int32_t j0 = fixed > 0 ? (fixed - 1) * stride : 0;
    uint4 v[kMoveDepth];
    int64_t dst[kMoveDepth];
    auto load = [&](int32_t at, uint4 (&w)[kMoveDepth], int64_t (&d)[kMoveDepth]) {
        int64_t s[kMoveDepth];
#pragma unroll
        for (int u = 0; u < kMoveDepth; ++u) {
            const int32_t j = at + u * rows + r0;
            d[u] = -1;
            s[u] = -1;
            if (j < n) {
                const int32_t src = __ldg(kept + j);
                if (src != j) {
                    int32_t sp, dp;
                    const int32_t ss = slot_of(p, bt, src, sp), ds = slot_of(p, bt, j, dp);
                    if (ss >= 0 && ds >= 0) {
                        s[u] = (((int64_t)sp * p.P + ss) * p.Hkv + h) * p.row_pieces + piece;
                        d[u] = (((int64_t)dp * p.P + ds) * p.Hkv + h) * p.row_pieces + piece;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kMoveDepth; ++u)
            if (s[u] >= 0) w[u] = __ldcg(pool + s[u]);
    };
    load(j0, v, dst);
    for (; j0 < n; j0 += batch) {
        uint4 vn[kMoveDepth];
        int64_t dn[kMoveDepth];
        // every load of this batch is back before any of its rows is overwritten
        load(j0 + batch, vn, dn);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveDepth; ++u)
            if (dst[u] >= 0) pool[dst[u]] = v[u];
#pragma unroll
        for (int u = 0; u < kMoveDepth; ++u) {
            v[u] = vn[u];
            dst[u] = dn[u];
        }
    }
}

int entry(const pgqa_evict_args* a, cudaStream_t stream) {
    if (a == nullptr) return PGQA_ERR_NULL_POINTER;
    if (a->struct_size != sizeof(pgqa_evict_args)) return PGQA_ERR_BAD_SHAPE;
    if (!a->k_cache || !a->v_cache || !a->weights || !a->seq_lens || !a->block_table || !a->kept || !a->new_lens)
        return PGQA_ERR_NULL_POINTER;
    int st = host_check_pages(a->batch_size, a->num_heads_k, a->headdim, a->page_size, a->num_pages, a->bt_stride);
    if (st != PGQA_OK) return st;
    if (a->kv_format != 0 && a->kv_format != 1) return PGQA_ERR_UNSUPPORTED;
    if (a->keep <= 0 || a->keep > INT32_MAX || a->sinks < 0 || a->recent < 0 || a->sinks > a->keep ||
        a->recent > a->keep - a->sinks)
        return PGQA_ERR_BAD_SHAPE;
    if (a->new_lens == a->seq_lens) return PGQA_ERR_BAD_SHAPE;
    if (a->batch_size * a->num_heads_k > INT32_MAX) return PGQA_ERR_UNSUPPORTED;
    if (!host_aligned(a->k_cache, 16) || !host_aligned(a->v_cache, 16) || !host_aligned(a->weights, 4) ||
        !host_aligned(a->weights_out, 4) || !host_aligned(a->seq_lens, 4) || !host_aligned(a->block_table, 4) ||
        !host_aligned(a->kept, 4) || !host_aligned(a->new_lens, 4))
        return PGQA_ERR_MISALIGNED;
    int dev, sms, optin;
    if ((st = host_device(&dev, &sms, &optin)) != PGQA_OK) return st;
    Params p = {};
    if ((st = host_error_word(dev, &p.err)) != PGQA_OK) return st;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.weights = a->weights;
    p.weights_out = a->weights_out ? a->weights_out : a->weights;
    p.seq_lens = a->seq_lens;
    p.block_table = a->block_table;
    p.kept = a->kept;
    p.new_lens = a->new_lens;
    p.bt_stride = a->bt_stride;
    p.cap_tokens = a->bt_stride * a->page_size;
    p.Hkv = (int32_t)a->num_heads_k;
    p.P = (int32_t)a->page_size;
    p.page_shift = host_shift(a->page_size);
    p.num_pages = (int32_t)a->num_pages;
    p.keep = (int32_t)a->keep;
    p.sinks = (int32_t)a->sinks;
    p.recent = (int32_t)a->recent;
    p.row_pieces = a->kv_format == 1 ? 8 : 16;
    const int64_t items = a->batch_size * a->num_heads_k;
    int64_t hold = p.cap_tokens - p.sinks - p.recent;
    if (hold > kMaxKeys) hold = kMaxKeys;
    if (hold < 0) hold = 0;
    if (hold * 4 > optin - 12 * 1024) hold = (optin - 12 * 1024) / 4;
    p.smem_keys = (int32_t)hold;
    static int done[kHostMaxDevices] = {0};
    const int smem = (int)hold * 4;
    if (smem > 32 * 1024 && (st = host_smem_limit(select_kernel, dev, smem, done)) != PGQA_OK) return st;
    st = host_launch(select_kernel, dim3((unsigned)items), kSelThreads, (size_t)smem, stream, p);
    if (st != PGQA_OK) return st;
    // column ranges of at least 64 bytes: as few as give every SM two CTAs
    p.cols = 1;
    while (items * 2 * p.cols < 2 * sms && p.row_pieces / (2 * p.cols) >= 4) p.cols *= 2;
    p.col_pieces = p.row_pieces / p.cols;
    return host_launch(move_kernel, dim3((unsigned)items, (unsigned)(2 * p.cols + 1)), kMoveThreads, 0, stream, p);
}

}  // namespace evict
}  // namespace pgqa

extern "C" int pgqa_evict(const pgqa_evict_args* args, void* stream) {
    return pgqa::host_set_status(pgqa::evict::entry(args, static_cast<cudaStream_t>(stream)));
}
