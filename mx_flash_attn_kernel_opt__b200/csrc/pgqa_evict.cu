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
 * One launch, a cluster of 2, 4 or 8 CTAs per (sequence, KV head), in two phases.
 *
 * Select: each CTA takes a contiguous range of the middle tokens.  Their weights become
 * sortable 32-bit keys in shared memory (or are re-read from L2 when they do not fit); a
 * radix select over digits of 11, 11 and 10 bits, the CTAs' histograms added over
 * distributed shared memory, finds the key of the last token kept and how many of its equals
 * stay, and one ordered pass with a block scan writes the indices.  4 bytes per token are
 * read from HBM once; what bounds this phase is the latency of its dozen dependent steps,
 * which the move of another pair on the same SM covers.
 *
 * Move, in place.  Row j of the result comes from row kept[j] >= j, and kept is ascending,
 * so whoever goes through j in ascending batches may overwrite [j0, j0 + n) as soon as the
 * loads of that batch are done: every later source lies at j0 + n or above.  So loads run
 * ahead through a ring of asynchronous copies to shared memory (80 KB in flight per CTA) and
 * one barrier per batch orders its stores behind its loads.  Half of the cluster's CTAs move
 * K, half V; the rows of a batch are dealt out among them, whole rows each, and the barrier
 * is then the cluster's.  The rows' places are looked up 2048 at a time, so no load waits
 * for an index.  Rows before the first evicted one are not touched.  Bound by reading and
 * writing the moved rows.
 *
 * Measured: 16 sequences of 1025 tokens cut to 1024, 8 heads, bf16 14.5 us (0.9 of a copy's
 * rate over the rows that move); 64 sequences of up to 8192 tokens cut to 2048, 4 heads 92 us
 * (4.2 TB/s over all of the call, of which the first selects take 12 us); 2 of 32,000 cut to
 * 8192, 8 heads, e4m3 37 us, of which the select 14.
 */
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pgqa_host.h"
#include "pgqa_ptx.cuh"

namespace pgqa {
namespace evict {

constexpr int kThreads = 512;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kPieces = 2;             // 16-byte pieces of a thread per batch
constexpr int kStages = 5;             // batches in the ring
constexpr int kStagePieces = kThreads * kPieces;
constexpr int kRows = 2048;            // rows looked up at a time by a CTA
constexpr int kRingBytes = kStages * kStagePieces * 16;
constexpr int kSmem = kRingBytes + 2 * kRows * 4;  // so many that kCtasPerSm fit
constexpr int kCtasPerSm = 1024 / kThreads;
constexpr int kHistBytes = kBins * 4;
constexpr int kMaxGroups = (kRingBytes - kHistBytes) / 16;  // groups of four keys held in the ring before the move
static_assert(2 * kRows >= 2 * kBins, "two of the select's histograms lie in the rows' places, one in the ring");

struct Params {
    void *k_cache, *v_cache;
    const float* weights;
    float* weights_out;
    const int32_t *seq_lens, *block_table;
    int32_t *kept, *new_lens;
    int32_t* err;
    int64_t bt_stride, cap_tokens;
    int32_t Hkv, P, page_shift, num_pages, keep, sinks, recent;
    int32_t row_pieces;              // 16-byte pieces in a row
    int32_t cluster;                 // CTAs per (sequence, KV head)
};

__device__ __forceinline__ int32_t page_of(const Params& p, int32_t tok) {
    return p.page_shift >= 0 ? tok >> p.page_shift : tok / p.P;
}

__device__ __forceinline__ int32_t length_of(const Params& p, int32_t b) {
    const int32_t L = ptx::ld(p.seq_lens + b);
    return L < 0 ? 0 : (L > p.cap_tokens ? (int32_t)p.cap_tokens : L);
}

/* Order-preserving key of a weight: larger weight, larger key; -0 equals +0, NaN is highest. */
__device__ __forceinline__ uint32_t key_of(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

/* Cluster barrier and a load from another CTA's shared memory. */
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
/* Arrival that orders no memory: for a barrier that only says that loads have returned.  A
 * releasing arrival waits for the thread's stores to reach L2 as well (2 sequences of 32,000
 * tokens cut to 8192, 8 heads, e4m3: 55.4 us instead of 45.7). */
__device__ __forceinline__ void cluster_arrive_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr, uint32_t rank) {
    uint32_t v;
    asm volatile(
        "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}"
        : "=r"(v)
        : "r"(addr), "r"(rank)
        : "memory");
    return v;
}
/* Sum of v over the threads before this one, and over all, of a block; two
 * 16-bit counts packed in a word pass through as long as neither total reaches 2^16. */
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* wsum, int lane, int warp, uint32_t& total) {
    uint32_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    __syncthreads();  // the last use of wsum is over
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    uint32_t ws = lane < kThreads / 32 ? wsum[lane] : 0;
    const uint32_t own = ws;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, ws, o);
        if (lane >= o) ws += u;
    }
    total = __shfl_sync(0xffffffffu, ws, 31);
    return incl - v + __shfl_sync(0xffffffffu, ws - own, warp);
}

/* Place of token `tok` in the pool's token order, given its page's id, or -1 for a bad one
 * (`bad` is then set).  The ids are loaded apart, many at a time. */
__device__ __forceinline__ int32_t place_of(const Params& p, int32_t tok, int32_t pid, bool& bad) {
    if ((uint32_t)pid >= (uint32_t)p.num_pages) {
        bad = true;
        return -1;
    }
    return pid * p.P + (tok - page_of(p, tok) * p.P);
}
/* Entry of the weight pool at a place. */
__device__ __forceinline__ int64_t weight_at(const Params& p, int32_t place, int32_t h) {
    const int32_t pid = page_of(p, place);
    return ((int64_t)pid * p.Hkv + h) * p.P + (place - pid * p.P);
}

/* Writes kept[0, keep) of a sequence of L > keep tokens: C CTAs of a cluster together, each
 * with the keys of its range in `keys`, or (C = 1) one CTA alone, which leaves the first kRows
 * of them in `places` too.  The three passes have a histogram each (at `places` and at the
 * end of the ring), so one cluster barrier per pass will do; and nothing is stored to global
 * memory before the last pass, since a releasing barrier waits for such stores. */
__device__ void select_kept(const Params& p, const int32_t* bt, int32_t L, int32_t h, int32_t* kept, int C, int rank,
                            uint4* keys, uint32_t* places) {
    __shared__ uint32_t wsum[32];
    __shared__ uint32_t found[2];   // the digit of the last kept key, and how many lie above it
    __shared__ uint32_t counts[2];  // the CTAs before: tokens above the digit, and with it
    __shared__ uint32_t coarse[3][kBins / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int t_all = rank * kThreads + tid, n_all = C * kThreads;
    const int32_t lo = p.sinks, hi = L - p.recent;       // candidates [lo, hi)
    const int32_t m = p.keep - p.sinks - p.recent;       // of which m < hi - lo stay
    // this CTA's groups of four tokens (a group never crosses a page): [g0, g1)
    const int32_t ga = lo >> 2, gn = ((hi + 3) >> 2) - ga, per = (gn + C - 1) / C;
    const int32_t g0 = ga + min(gn, rank * per), g1 = ga + min(gn, (rank + 1) * per);
    const bool held = per <= kMaxGroups;
    bool bad = false;
    auto load_group = [&](int32_t g) -> uint4 {
        const int32_t tok = 4 * g, page = page_of(p, tok);
        const int32_t pid = ptx::ld(bt + page);
        if ((uint32_t)pid >= (uint32_t)p.num_pages) {
            bad = true;
            return make_uint4(0, 0, 0, 0);
        }
        const float4 w = ptx::ld(reinterpret_cast<const float4*>(p.weights + ((int64_t)pid * p.Hkv + h) * p.P +
                                                               (tok - page * p.P)));
        return make_uint4(key_of(w.x), key_of(w.y), key_of(w.z), key_of(w.w));
    };
    auto group_at = [&](int32_t g) -> uint4 { return held ? keys[g - g0] : load_group(g); };
    // f(key, token) for the candidates of a group
    auto each = [&](int32_t g, const uint4& k, auto&& f) {
        const uint32_t v[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (4 * g + u >= lo && 4 * g + u < hi) f(v[u], u);
    };

    uint32_t prefix = 0, mask = 0;  // digits fixed so far
    uint32_t need = (uint32_t)m;    // tokens still to take among those that match them
    uint32_t gt_before = 0, eq_before = 0;  // kept for sure, and equal to the last, in the CTAs before
    uint32_t* const third = reinterpret_cast<uint32_t*>(keys + kMaxGroups);
    for (int i = tid; i < 2 * kBins; i += kThreads) places[i] = 0;
    for (int i = tid; i < kBins; i += kThreads) third[i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int pass = 0; pass < 3 && m > 0; ++pass) {
        uint32_t* const hist = pass < 2 ? places + pass * kBins : third;
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
        const uint32_t digits = pass == 2 ? 1023u : 2047u;
        auto count = [&](int32_t g, const uint4& k) {
            each(g, k, [&](uint32_t key, int) {
                if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & digits], 1u);
            });
        };
        if (pass == 0 && held) {
            // the keys come in, four groups in flight per thread, and are counted on the way
            for (int32_t gb = g0 + tid; gb < g1; gb += 4 * kThreads) {
                uint4 k[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (gb + u * kThreads < g1) k[u] = load_group(gb + u * kThreads);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (gb + u * kThreads < g1) {
                        keys[gb + u * kThreads - g0] = k[u];
                        count(gb + u * kThreads, k[u]);
                    }
                }
            }
        } else {
            for (int32_t g = g0 + tid; g < g1; g += kThreads) count(g, group_at(g));
        }
        __syncthreads();
        if (C == 1) {
            // alone: all bins at once, from the top; thread t owns those from `top` down.  The
            // warp whose bins hold the `need`-th key of those left, then the thread and the bin
            // (three levels by one warp, as below: 16.4 us instead of 13.9 for 16 sequences of 1025
            // tokens cut to 1024, 8 heads)
            constexpr int kOwn = kBins / kThreads;
            const int top = kBins - 1 - kOwn * tid;
            uint32_t c[kOwn], sum = 0;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                c[i] = hist[top - i];
                sum += c[i];
            }
            const uint32_t mine = __reduce_add_sync(0xffffffffu, sum);
            if (lane == 0) wsum[warp] = mine;
            __syncthreads();
            uint32_t above = __reduce_add_sync(0xffffffffu, lane < warp ? wsum[lane] : 0);
            if (above < need && need <= above + mine) {
                uint32_t incl = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                above += incl - sum;
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    if (above < need && need <= above + c[i]) {
                        found[0] = (uint32_t)(top - i);
                        found[1] = above | (c[i] == need - above ? 0x80000000u : 0u);
                    }
                    above += c[i];
                }
            }
            if (tid < 2) counts[tid] = 0;
        } else {
            // together: sums of 32 bins each, so that the others read these and one group of
            // 32 of this CTA's histogram instead of all of it (37 us instead of 44 for 2 sequences
            // of 32,000 tokens cut to 8192, 8 heads, e4m3)
            for (int i = warp; i < kBins / 32; i += kThreads / 32) {
                const uint32_t v = __reduce_add_sync(0xffffffffu, hist[32 * i + lane]);
                if (lane == 0) coarse[pass][i] = v;
            }
            cluster_sync();
        }
        if (C > 1 && warp == 0) {
            // the group of bins, then the bin, that hold the `need`-th key from the top (of those
            // left); and how many keys above it, and in it, the CTAs before this one have
            uint32_t whole = 0;         // keys in the bin found
            uint32_t over = 0, gt = 0;  // keys above so far, of all CTAs and of those before
            const uint32_t at_coarse = ptx::smem_u32(&coarse[pass][0]);
            int group = 0;
            auto search = [&](uint32_t at, int top, uint32_t& eq) -> int {  // 32 words down from `top`
                uint32_t sum = 0, low = 0, v[kMaxCluster];
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) v[r] = r < C ? ld_cluster(at + 4u * (top - lane), (uint32_t)r) : 0;
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) {
                    sum += v[r];
                    if (r < rank) low += v[r];
                }
                uint32_t incl = sum, lincl = low;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t a = __shfl_up_sync(0xffffffffu, incl, o), b = __shfl_up_sync(0xffffffffu, lincl, o);
                    if (lane >= o) {
                        incl += a;
                        lincl += b;
                    }
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, over + incl >= need);
                const int f = hit ? __ffs(hit) - 1 : 32;  // lanes before f lie above
                const int prev = f > 0 ? f - 1 : 0;
                const uint32_t a = __shfl_sync(0xffffffffu, incl, prev), b = __shfl_sync(0xffffffffu, lincl, prev);
                if (f > 0) {
                    over += a;
                    gt += b;
                }
                eq = f < 32 ? __shfl_sync(0xffffffffu, low, f) : 0;
                whole = f < 32 ? __shfl_sync(0xffffffffu, sum, f) : 0;
                return f;
            };
            uint32_t eq = 0;
            int f = search(at_coarse, kBins / 32 - 1, eq);
            group = kBins / 32 - 1 - f;
            if (f == 32) {
                f = search(at_coarse, kBins / 32 - 33, eq);
                group = kBins / 32 - 33 - f;
            }
            f = search(ptx::smem_u32(hist), 32 * group + 31, eq);
            if (lane == 0) {
                found[0] = (uint32_t)(32 * group + 31 - f);
                found[1] = over | (whole == need - over ? 0x80000000u : 0u);
                counts[0] = gt;
                counts[1] = eq;
            }
        }
        __syncthreads();
        gt_before += counts[0];
        eq_before = counts[1];
        const uint32_t digit = found[0], over = found[1];
        need -= over & 0x7fffffffu;
        prefix |= digit << shift;
        mask |= digits << shift;
        if (over >> 31) break;  // every token that matches the prefix stays
    }
    // kept: keys above the prefix (under its mask), and the first `need` that match it; none
    // of the middle (m = 0) is above an all-ones prefix
    if (m == 0) {
        prefix = mask = 0xffffffffu;
        need = 0;
    }
    auto put = [&](int32_t at, int32_t tok) {
        kept[at] = tok;
        if (C == 1 && at < kRows) places[at] = (uint32_t)tok;
    };
    for (int32_t gb = g0; gb < g1; gb += kThreads) {
        const int32_t g = gb + tid;
        uint32_t cnt = 0, flags = 0;  // (above | equal << 16) of this thread's four tokens
        if (g < g1)
            each(g, group_at(g), [&](uint32_t key, int u) {
                const uint32_t k = key & mask;
                if (k > prefix) {
                    cnt += 1;
                    flags |= 1u << u;
                } else if (k == prefix) {
                    cnt += 0x10000u;
                    flags |= 16u << u;
                }
            });
        uint32_t total;
        const uint32_t before = block_scan(cnt, wsum, lane, warp, total);  // at most 4096 of each
        uint32_t gt = gt_before + (before & 0xffffu), eq = eq_before + (before >> 16);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t at = (uint32_t)p.sinks + gt + (eq < need ? eq : need);
            const bool above = (flags & (1u << u)) != 0, equal = (flags & (16u << u)) != 0;
            if (above || (equal && eq < need)) put((int32_t)at, 4 * g + u);
            gt += above;
            eq += equal;
        }
        gt_before += total & 0xffffu;
        eq_before += total >> 16;
    }
    for (int j = t_all; j < p.sinks; j += n_all) put(j, j);
    for (int j = t_all; j < p.recent; j += n_all) put(p.sinks + m + j, L - p.recent + j);
    if (bad) atomicOr(p.err, kDevErrBadPage);
}

__global__ void __launch_bounds__(kThreads, kCtasPerSm) evict_kernel(const Params p) {
    extern __shared__ uint4 ring[];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int tid = threadIdx.x;
    const int32_t C = p.cluster, item = blockIdx.x / C, rank = blockIdx.x - item * C;
    const int32_t b = item / p.Hkv, h = item - b * p.Hkv;
    const int32_t L0 = ptx::ld(p.seq_lens + b);
    const int32_t L = length_of(p, b);
    const int32_t n = min(L, p.keep);
    if (h == 0 && tid == 0 && rank == 0) {
        if (L != L0) atomicOr(p.err, kDevErrBadSeqlen);
        p.new_lens[b] = n;
    }
    int32_t* kept = p.kept + (int64_t)item * p.keep;
    const int32_t* bt = p.block_table + (int64_t)b * p.bt_stride;
    const bool cut = L > p.keep;  // the same in all of the cluster, as is every count of a loop with a barrier
    int32_t* src_slot = reinterpret_cast<int32_t*>(ring + kRingBytes / 16);
    int32_t* dst_slot = src_slot + kRows;
    const bool solo = C == 2;
    if (cut) {
        // a pair of CTAs: each selects for itself (and writes the same indices), which costs
        // less than meeting at every step; more of them divide the tokens
        select_kept(p, bt, L, h, kept, solo ? 1 : C, solo ? 0 : rank, ring, reinterpret_cast<uint32_t*>(src_slot));
        // kept is complete; every weight has been read, and nobody reads another's shared
        // memory (a pair shares none, and meets before it overwrites a weight)
        if (solo) __syncthreads();
        else cluster_sync();
    } else {
        for (int j = rank * kThreads + tid; j < p.keep; j += C * kThreads) kept[j] = j < L ? j : -1;
    }
    // the j-th kept token; a CTA that selected alone has the first ones at hand until the first
    // rows' places are looked up
    bool at_hand = solo;
    auto kept_at = [&](int32_t j) { return at_hand && j < kRows ? src_slot[j] : __ldcg(kept + j); };

    // the weights, one 4-byte element per token
    const bool in_place = p.weights_out == p.weights;
    auto move_weights = [&]() {
        bool bad = false;
        constexpr int kU = 4;
#pragma unroll 1
        for (int32_t j0 = 0; j0 < n; j0 += kU * C * kThreads) {
            float v[kU];
            int32_t from[kU], to[kU], sp[kU], dp[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                to[u] = j0 + (u * C + rank) * kThreads + tid;
                from[u] = to[u] < n ? (cut ? __ldcg(kept + to[u]) : to[u]) : -1;
                if (in_place && from[u] == to[u]) from[u] = -1;
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                sp[u] = dp[u] = 0;
                if (from[u] >= 0) {
                    sp[u] = ptx::ld(bt + page_of(p, from[u]));
                    dp[u] = ptx::ld(bt + page_of(p, to[u]));
                }
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (from[u] < 0) continue;
                from[u] = place_of(p, from[u], sp[u], bad);
                to[u] = place_of(p, to[u], dp[u], bad);
                if (to[u] < 0) from[u] = -1;
                if (from[u] >= 0) v[u] = __ldcg(p.weights + weight_at(p, from[u], h));
            }
            if (in_place) cluster_sync();
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (from[u] >= 0) p.weights_out[weight_at(p, to[u], h)] = v[u];
        }
        if (bad) atomicOr(p.err, kDevErrBadPage);
    };
    if (!cut) {
        if (!in_place) move_weights();
        return;
    }
    const int32_t S = C / 2, part = rank >> 1;  // CTAs that share the rows of K, or of V
    uint4* pool = static_cast<uint4*>((rank & 1) == 0 ? p.k_cache : p.v_cache);
    const int r0 = tid / p.row_pieces;
    const int rows = kThreads / p.row_pieces;        // rows that the CTA covers at a time
    const int32_t batch = rows * kPieces;            // and in a batch: a power of two
    const int lb = __ffs(batch) - 1;
    pool += (int64_t)h * p.row_pieces + tid % p.row_pieces;
    const int64_t pitch = (int64_t)p.Hkv * p.row_pieces;
    // rows that stay where they are form a prefix; skip whole strides of it
    const int32_t stride = (n + kThreads - 1) / kThreads;
    const bool still = tid * stride < n && kept_at(tid * stride) == tid * stride;
    const int32_t fixed = __syncthreads_count(still);
    bool weights_done = false;
    for (int32_t j0 = fixed > 0 ? (fixed - 1) * stride : 0; j0 < n; j0 += kRows * S) {
        const int32_t here = min(kRows * S, n - j0);
        // this CTA's i-th row is row (i / batch * S + part) * batch + i % batch of them
        auto row_of = [&](int32_t i) { return ((i >> lb) * S + part) * batch + (i & (batch - 1)); };
        __syncthreads();
        int32_t from[kRows / kThreads];
#pragma unroll
        for (int u = 0; u < kRows / kThreads; ++u) {
            const int32_t r = row_of(u * kThreads + tid);
            from[u] = r < here ? kept_at(j0 + r) : -1;
        }
        if (at_hand) __syncthreads();  // they are overwritten now
        at_hand = false;
        bool bad = false;
        int32_t sp[kRows / kThreads], dp[kRows / kThreads];
#pragma unroll
        for (int u = 0; u < kRows / kThreads; ++u) {
            const int32_t to = j0 + row_of(u * kThreads + tid);
            if (from[u] == to) from[u] = -1;
            sp[u] = dp[u] = 0;
            if (from[u] >= 0) {
                sp[u] = ptx::ld(bt + page_of(p, from[u]));
                dp[u] = ptx::ld(bt + page_of(p, to));
            }
        }
#pragma unroll
        for (int u = 0; u < kRows / kThreads; ++u) {
            const int32_t i = u * kThreads + tid;
            int32_t s = -1, d = -1;
            if (from[u] >= 0) {
                s = place_of(p, from[u], sp[u], bad);
                d = place_of(p, j0 + row_of(i), dp[u], bad);
                if (d < 0) s = -1;
            }
            src_slot[i] = s;
            dst_slot[i] = d;
        }
        if (bad) atomicOr(p.err, kDevErrBadPage);
        __syncthreads();
        const int32_t batches = (here + batch * S - 1) / (batch * S);  // at most kRows / batch
        auto fetch = [&](int32_t k) {
            if (k < batches) {
                uint4* to = ring + (k % kStages) * kStagePieces + tid;
#pragma unroll
                for (int u = 0; u < kPieces; ++u) {
                    const int32_t s = src_slot[k * batch + u * rows + r0];
                    if (s >= 0)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(to + u * kThreads)),
                                     "l"(pool + s * pitch)
                                     : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int k = 0; k < kStages; ++k) fetch(k);
        if (!weights_done) {  // while the first rows are on their way
            move_weights();
            weights_done = true;
        }
        // Every load of a batch, by all who share the rows, is back before any of its rows is
        // overwritten; a thread stores what it loaded itself.  The stores come one batch
        // later, so the wait for the others has a batch's time to pass.
        for (int32_t k = 0; k <= batches; ++k) {
            if (k < batches) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
                if (S > 1) cluster_arrive_relaxed();
            }
            if (k > 0) {
                const uint4* at = ring + ((k - 1) % kStages) * kStagePieces + tid;
#pragma unroll
                for (int u = 0; u < kPieces; ++u) {
                    const int32_t i = (k - 1) * batch + u * rows + r0;
                    if (src_slot[i] >= 0) pool[dst_slot[i] * pitch] = at[u * kThreads];
                }
                fetch(k - 1 + kStages);
            }
            if (k < batches) {
                if (S > 1) cluster_wait();
                else __syncthreads();
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
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
    if (a->batch_size * a->num_heads_k > INT32_MAX / kMaxCluster) return PGQA_ERR_UNSUPPORTED;
    {  // the clusters of a sequence's heads read its length when another's may have been written
        const uintptr_t r = reinterpret_cast<uintptr_t>(a->seq_lens), w = reinterpret_cast<uintptr_t>(a->new_lens);
        const uintptr_t bytes = 4 * (uintptr_t)a->batch_size;
        if (r < w + bytes && w < r + bytes) return PGQA_ERR_BAD_SHAPE;
    }
    if (!host_aligned(a->k_cache, 16) || !host_aligned(a->v_cache, 16) || !host_aligned(a->weights, 16) ||
        !host_aligned(a->weights_out, 16) || !host_aligned(a->seq_lens, 4) || !host_aligned(a->block_table, 4) ||
        !host_aligned(a->kept, 4) || !host_aligned(a->new_lens, 4))
        return PGQA_ERR_MISALIGNED;
    {  // K and V rows move independently of each other, in place
        const uintptr_t k = reinterpret_cast<uintptr_t>(a->k_cache), v = reinterpret_cast<uintptr_t>(a->v_cache);
        const uintptr_t bytes = (uintptr_t)a->num_pages * a->page_size * a->num_heads_k * (a->kv_format == 1 ? 128 : 256);
        if (k < v + bytes && v < k + bytes) return PGQA_ERR_BAD_SHAPE;
    }
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
    // CTAs per pair: two (K and V), or as many more as still run at once (kCtasPerSm), as
    // long as each has 1024 tokens or more by the capacity
    p.cluster = 2;
    while (p.cluster < kMaxCluster && items * 2 * p.cluster <= kCtasPerSm * sms && p.cap_tokens / (2 * p.cluster) >= 1024)
        p.cluster *= 2;
    static HostSmemDone done;
    if ((st = host_smem_limit(evict_kernel, dev, kSmem, done)) != PGQA_OK) return st;
    return host_launch(evict_kernel, dim3((unsigned)(items * p.cluster)), kThreads, kSmem, stream, p.cluster, p);
}

}  // namespace evict
}  // namespace pgqa

extern "C" int pgqa_evict(const pgqa_evict_args* args, void* stream) {
    return pgqa::host_set_status(pgqa::evict::entry(args, static_cast<cudaStream_t>(stream)));
}
