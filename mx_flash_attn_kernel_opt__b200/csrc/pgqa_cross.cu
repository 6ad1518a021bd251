/*
 * pgqa_cross.cu - attention of packed prompt tokens over each sequence's encoder states,
 * held in pages (cross attention: no causal mask, two unrelated lengths):
 *
 *     out[x, h] = softmax(scale * q[x, h] . K[kv]^T) . V[kv],   kv = h / g, g = Hq / Hkv
 *
 * over the first seq_lens[b] tokens of sequence b's pages for every prompt token x of
 * sequence b, x in [cu[b], cu[b + 1]).
 *
 * Tensor-core bound: 4 * 128 flop per (query row, key) against 512 bytes of K and V per key
 * that all rows of a KV head share.  The g query heads of a KV head are rows of one tile
 * (row = token * g + head), so a 128-row tile holds 128 / g tokens and K and V are read
 * once per 256 rows.  A work item is (sequence, KV head, two such tiles).  The items' key
 * tiles, one after the other, each item's with kItemCost more for its Q tiles and its output,
 * are cut into equal slices, one per persistent CTA (one CTA per SM); a cut that would fall
 * within 1/24 of a slice of an item's end is moved there.  An item that is cut all the same
 * leaves its parts' normalised O (fp32) and log-sum-exps in the workspace, and a second
 * launch joins them.  Every role of a CTA walks the same items:
 *
 *   warps 0-3, 4-7  softmax and output of tile 0 and tile 1: thread = row = TMEM lane, a
 *                   step of 64 keys at a time.  The running maximum is moved only when a
 *                   score exceeds it by 2^8 (O is then rescaled in TMEM), so the O
 *                   accumulator is touched once per item in the usual case; sums and
 *                   statistics are fp32, P is rounded to bf16 (2^-8 relative at most, of
 *                   weights that are summed in fp32) and goes back to TMEM over the scores it
 *                   came from.
 *   warp 8          TMA: Q tiles, and 128-key tiles of K and V by page boxes through one
 *                   ring of five 32 KB slots; it zeroes V rows behind the last key, so that
 *                   a weight of 0 never meets a NaN left in a page.
 *   warps 12-15     (e4m3 pages) turn the tiles that TMA brings as they are into bf16, exactly,
 *                   in the ring that the MMAs read (four slots then); the scales go into the
 *                   score's factor and the normaliser.  Two such warpgroups leave 96
 *                   registers a thread, and the spills cost more (long prompts 9% slower).
 *   warps 9, 10     issue the MMAs of tile 0 and of tile 1: S = Q K^T (both from shared
 *                   memory), O += P V (P from TMEM).
 * TMEM: two score buffers of 64 columns for each tile (from columns 0 and 128), O at 256 and
 * 384.  The scores of step i + 2 are issued right behind the PV of step i, which frees their
 * buffer, so while a warpgroup works on step i + 1 its next scores are computed and neither
 * waits for the other.  The price is QK^T with N = 64, which re-reads Q from shared memory
 * twice as often: 48 clocks an MMA instead of 32.  With one buffer of 128 columns per tile, where
 * the softmax waits for PV and QK^T of every step, long prompts took 15% more.
 *
 * Measured, 40 calls after a pause / a loop of 0.6 s, in which the 1000 W cap holds the clock
 * down (us):                                                    bf16 pages    e4m3 pages
 *   2 x 4096 tokens, 32 + 8 heads, over 8192 keys              916 / 1045    1029 / 1116
 *   8 prompts of 17 to 1024 tokens, 28 + 4 heads, 197 to 4097   166 / 180     190 / 193
 *   16 x 3 tokens, 32 + 8 heads, over 16,000 keys               200 / 234     250 / 250
 * The first is 1200 / 1052 TFLOP/s, the second 897 / 826; K and V of the third take 161 us (e4m3
 * 81 us) to read once.
 *
 * Every wait is bounded: one that expires sets the device error word and the CTA's abort
 * flag, every role leaves its loop, loads and MMAs in flight are drained and TMEM is freed.
 */
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdlib.h>

#include "pgqa_host.h"
#include "pgqa_partition.h"
#include "pgqa_ptx.cuh"

namespace pgqa {
namespace cross {

constexpr int kThreads = 352;              // bf16 pages; e4m3 pages: and a warpgroup that converts
constexpr int kTile = 128;                 // rows of a tile, and keys of a K / V tile
constexpr int kHalf = kTile * 128;         // one 64-dimension half of a tile, bf16
constexpr int kSlot = 2 * kHalf;
constexpr int kStep = 64;                  // keys of a softmax step
constexpr int kQOff = 0, kRingOff = 2 * kSlot;
/* Shared memory: Q tiles, the ring of bf16 K and V tiles, for e4m3 pages a ring of tiles as
 * they come, barriers, then 16 bytes. */
template <bool KV8>
struct Geo {
    static constexpr int kThreads = KV8 ? 512 : cross::kThreads;
    static constexpr int kSlots = KV8 ? 4 : 5;
    static constexpr int kRaw = KV8 ? 2 : 0;  // tiles of kHalf bytes
    static constexpr int kRawOff = kRingOff + kSlots * kSlot;
    static constexpr int kBarOff = kRawOff + kRaw * kHalf;
    static constexpr int kBars = 2 * kSlots + 16 + 2 * kRaw;
    static constexpr int kSmem = 1024 + kBarOff + kBars * 8 + 16;
};
constexpr int kRows = 2 * kTile;           // rows of a work item
// What an item costs beside its key tiles, in key tiles (1 to 4 measured in one session: 175, 159,
// 167, 166 us for ragged prompts of 17 to 1024 tokens over 197 to 4097 keys; calls of one build
// spread by as much as 2 from 3 and 4, so only 1 is ruled out), and the least length of a slice
// (1, 2 and 3: 17.7, 14.0, 16.7 us for 10 + 13 tokens over 1024 keys, 32 + 8 heads, in a graph).
constexpr int kItemCost = 2, kMinSlice = 2;
constexpr int kSnap = 24;
constexpr float kLazyLog2 = 8.f;
constexpr uint64_t kWaitLimitNs = 1000000000ull;

struct Params {
    __nv_bfloat16* out;      // [T, Hq, 128]
    float* lse;              // optional: [Hq, T] packed, [B, Hq, S] padded
    float *rec_o, *rec_lse;  // parts of cut items: [2 * grid][256 rows][128], [2 * grid][256] (log2 units)
    const int32_t *seq_lens, *block_table, *cu;
    const float *k_scale, *v_scale;  // e4m3 pools: factor per KV head (null = 1)
    struct Cut* cuts;        // [grid]
    int32_t* err;
    int64_t bt_stride, cap_tokens;
    int32_t B, S, T, Hq, Hkv, g, P, page_shift, num_pages;
    int32_t tile_tokens;     // prompt tokens per tile: 128 / g
    int32_t box;             // tokens of one TMA box of a pool: a power of two that divides P
    int32_t grid;            // CTAs of the first launch
    float scale_log2;
    uint64_t wait_limit_ns;
    // Test hooks, PGQA_DEBUG_STUCK_BARRIER = n or -n, read per call:
    int32_t debug_stuck;     // > 0 makes every CTA's first load expect 16 bytes too many
    int32_t debug_long;      // key tiles that the last slice believes to have too many
    int32_t out_32;          // out is 32-byte aligned (torch gives a view any multiple of its element)
};

__device__ __forceinline__ uint64_t sdesc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
/* fp32 accumulator, bf16 A and B, M = 128; B major: 0 = K, 1 = N */
__host__ __device__ constexpr uint32_t idesc(uint32_t b_mn, uint32_t n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
/* Steps of an item's key tiles [t0, t1): the last one may have a single one. */
__device__ __forceinline__ int steps_of(int32_t L, int32_t t0, int32_t t1) {
    return t1 == t0 ? 0 : 2 * (t1 - t0) - (L - (t1 - 1) * kTile <= kStep ? 1 : 0);
}

/* A sequence's prompt tokens [tok0, tok1), keys L, key tiles n (at least 1), items (all tile
 * pairs of a KV head, then of the next). */
struct Seq {
    int32_t tok0, tok1, L, n, pairs, items;
    __device__ int32_t len() const { return n + kItemCost; }  // of an item
    __device__ int64_t size() const { return (int64_t)items * len(); }
};

__device__ __forceinline__ Seq load_seq(const Params& p, int32_t b, bool report) {
    Seq q;
    q.tok0 = q.tok1 = q.L = q.pairs = q.items = 0;
    q.n = 1;
    if (b >= p.B) return q;
    q.tok0 = p.cu ? ptx::ld(p.cu + b) : b * p.S;
    q.tok1 = p.cu ? ptx::ld(p.cu + b + 1) : q.tok0 + p.S;
    int64_t L = ptx::ld(p.seq_lens + b);
    if (q.tok0 < 0 || q.tok1 < q.tok0 || q.tok1 > p.T || L < 0 || L > p.cap_tokens) {
        if (report) atomicOr(p.err, kDevErrBadSeqlen);
        q.tok0 = max(0, min(q.tok0, p.T));
        q.tok1 = max(q.tok0, min(q.tok1, p.T));
        L = L < 0 ? 0 : (L > p.cap_tokens ? p.cap_tokens : L);
    }
    q.L = (int32_t)L;
    q.n = max(1, (q.L + kTile - 1) / kTile);
    q.pairs = (q.tok1 - q.tok0 + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
    q.items = q.pairs * p.Hkv;
    return q;
}

/* Slice [lo, hi) of CTA c of the n active ones, and the item at its start. */
struct Slice {
    int64_t lo, hi;
    int64_t base;               // start of sequence b, which holds lo
    int64_t item_lo, item_len;  // the item that holds lo: its start, its length
    int64_t n, total;           // active CTAs, length of all slices
    int32_t b;
};

/* A cut at most 1/kSnap of a slice away from an item's end is moved there, as is one before
 * the item's first key tile. */
__device__ __forceinline__ int64_t snap_range(int64_t n, int64_t total) { return total / n / kSnap; }
__device__ __forceinline__ int64_t snapped(int64_t off, int64_t len, int64_t tol) {
    return off <= max(tol, (int64_t)kItemCost) ? 0 : (len - off <= tol ? len : off);
}

/* By all threads of a block (a multiple of 32, at most 1024); the result in shared memory. */
template <int kThreads>
__device__ void find_slice(const Params& p, int32_t c, Slice& out) {
    __shared__ int64_t wsum[kThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    int64_t local = 0;
    for (int b = b0; b < b1; ++b) local += load_seq(p, b, blockIdx.x == 0).size();
    int64_t incl = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) wsum[warp] = incl;
    if (tid == kThreads - 1) {  // an empty slice, should no sequence below be found to hold its start
        out.lo = INT64_MAX;
        out.hi = out.base = out.item_lo = 0;
        out.item_len = 1;
        out.b = 0;
    }
    __syncthreads();
    int64_t run = incl - local, total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) run += wsum[w];
        total += wsum[w];
    }
    int64_t n = total / kMinSlice;
    n = n < 1 ? 1 : (n > p.grid ? p.grid : n);
    if (tid == 0) {
        out.n = n;
        out.total = total;
    }
    if (c >= n || total == 0) {
        if (tid == 0) out.lo = out.hi = total;
    } else {
        const int64_t x0 = slice_begin(c, n, total), x1 = slice_begin(c + 1, n, total), tol = snap_range(n, total);
        if (tid == 0 && c + 1 == n) out.hi = total;
        for (int b = b0; b < b1; ++b) {
            const Seq q = load_seq(p, b, false);
            const int64_t end = run + q.size();
            auto snap = [&](int64_t x) {
                const int64_t off = (x - run) % q.len();
                return x - off + snapped(off, q.len(), tol);
            };
            if (run <= x0 && x0 < end) {
                const int64_t lo = snap(x0);
                out.lo = lo;
                out.base = run;
                out.b = b;
                out.item_lo = lo - (lo - run) % q.len();
                out.item_len = q.len();
            }
            if (c + 1 < n && run <= x1 && x1 < end) out.hi = snap(x1);
            run = end;
        }
    }
    __syncthreads();
}

struct Item {
    int32_t b, kvh, tok0, tok_end, L, t0, t1;  // prompt tokens from tok0, key tiles [t0, t1)
    bool cut;                                  // other CTAs have tiles of it too
};

/* Walks a slice's items; called by whole warps, every role with a copy of its own.  Lengths are
 * read again on the way: should they have changed since the slice was cut (or the slice be
 * longer than what there is), the walk ends with the error word set.  It never passes the
 * last sequence, and every item it gives lies within the tensors. */
struct Walker {
    int64_t left;             // of the slice
    int32_t b, kvh, pair, off;  // the next item, and where in it the slice goes on
    Seq mine, cur;            // this lane's of the 32 sequences from b - cur_lane, and the one at work
    int cur_lane;
    __device__ void pick() {
        cur.tok0 = __shfl_sync(0xffffffffu, mine.tok0, cur_lane);
        cur.tok1 = __shfl_sync(0xffffffffu, mine.tok1, cur_lane);
        cur.L = __shfl_sync(0xffffffffu, mine.L, cur_lane);
        cur.n = __shfl_sync(0xffffffffu, mine.n, cur_lane);
        cur.pairs = __shfl_sync(0xffffffffu, mine.pairs, cur_lane);
        cur.items = __shfl_sync(0xffffffffu, mine.items, cur_lane);
    }
    __device__ void stop(const Params& p, int lane) {
        left = 0;
        if (lane == 0) atomicOr(p.err, kDevErrBadSeqlen);
    }
    __device__ void init(const Params& p, const Slice& s, int lane) {
        left = s.hi - s.lo;
        if (left > 0 && s.hi == s.total) left += p.debug_long;
        b = s.b;
        cur_lane = 0;
        kvh = pair = off = 0;
        if (left > 0) {
            mine = load_seq(p, b + lane, false);
            pick();
            const int64_t in = s.lo - s.base;  // a cut moved to the sequence's end: kvh = Hkv
            if (cur.items == 0 || in > cur.size()) {
                stop(p, lane);
                return;
            }
            const int32_t unit = (int32_t)(in / cur.len());
            off = (int32_t)(in - (int64_t)unit * cur.len());
            kvh = unit / cur.pairs;
            pair = unit - kvh * cur.pairs;
        }
    }
    __device__ bool next(const Params& p, int lane, Item& it) {
        if (left <= 0) return false;
        if (pair == cur.pairs) {
            pair = 0;
            ++kvh;
        }
        if (kvh == p.Hkv) {
            kvh = 0;
            // the next sequence with items; some is left, so there is one
            int32_t from = cur_lane + 1;
            uint32_t some = __ballot_sync(0xffffffffu, mine.items > 0 && lane >= from);
            b += 1;
            while (some == 0) {
                b += 32 - from;
                from = 0;
                if (b >= p.B) {
                    stop(p, lane);
                    return false;
                }
                mine = load_seq(p, b + lane, false);
                some = __ballot_sync(0xffffffffu, mine.items > 0);
            }
            cur_lane = __ffs(some) - 1;
            b += cur_lane - from;
            pick();
        }
        it.b = b;
        it.kvh = kvh;
        it.tok0 = cur.tok0 + pair * 2 * p.tile_tokens;
        it.tok_end = cur.tok1;
        it.L = cur.L;
        it.t0 = max(0, off - kItemCost);
        const bool ends = left >= cur.len() - off;
        it.t1 = ends ? cur.n : max(it.t0, off + (int32_t)left - kItemCost);
        it.cut = off > 0 || !ends;
        left -= ends ? cur.len() - off : (int32_t)left;
        off = 0;
        ++pair;
        if (it.L == 0) it.t1 = it.t0;  // a sequence without keys: nothing to read
        return true;
    }
};

/* What the second launch needs to know of the item that slice c cuts first (is not set where
 * the slice begins with a whole item, or where an earlier cut is the item's first). */
struct Cut {
    int32_t is, last, b, kvh, tok0, tok_end, pad[2];  // its parts are of CTAs c - 1 .. last
};
__device__ Cut cut_of(const Params& p, int32_t c, const Slice& s) {
    Cut k = {};
    if (s.lo >= s.hi || s.item_lo == s.lo) return k;
    const int64_t tol = snap_range(s.n, s.total);
    const int64_t before = slice_begin(c - 1, s.n, s.total) - s.item_lo;
    if (before > 0 && snapped(before, s.item_len, tol) != 0) return k;
    // the slice that holds the item's last tile, unless its start was moved behind that
    int32_t last = (int32_t)slice_owner(s.item_lo + s.item_len - 1, s.n, s.total);
    const int64_t off = slice_begin(last, s.n, s.total) - s.item_lo;
    if (off > 0 && snapped(off, s.item_len, tol) == s.item_len) --last;
    const Seq q = load_seq(p, s.b, false);
    const int32_t unit = (int32_t)((s.item_lo - s.base) / s.item_len);
    if (unit >= q.items) return k;  // the lengths have changed; the walk reports it
    k.is = 1;
    k.last = last;
    k.b = s.b;
    k.kvh = unit / q.pairs;
    k.tok0 = q.tok0 + (unit - k.kvh * q.pairs) * 2 * p.tile_tokens;
    k.tok_end = q.tok1;
    return k;
}

/* Four e4m3 numbers as bf16 pairs, NaN excepted (comes out as 480): the exponent and mantissa
 * bits stand in the low bits of bf16's, which is the value times 2^(7 - 127), subnormals
 * too, and the product with 2^120 is exact.  Shifts by multiplication, so that the integer
 * and the FMA pipes share the work; the four converting warps are what bounds short prompts
 * (16 x 3 tokens, 32 + 8 heads, over 16,000 keys, in one session: 262 us with conversion
 * instructions, which leave at a fraction of the rate, 245 us with shifts and masks, 224 to 232
 * us so; in later sessions 250 us). */
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t b, uint32_t& lo, uint32_t& hi) {
    // 16-bit lanes 0000 s eeee mmm 0000; the sign goes from bit 11 to bit 15: + 15 * 2^11
    const uint32_t x = __byte_perm(b, 0, 0x4140) * 16u, y = __byte_perm(b, 0, 0x4342) * 16u;
    const uint32_t mx = (x & 0x08000800u) * 15u + x, my = (y & 0x08000800u) * 15u + y;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(mx), "r"(0x7b807b80u));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(my), "r"(0x7b807b80u));
}

/* 32 bytes to global memory in one instruction; the address must be a multiple of 32. */
__device__ __forceinline__ void st_global_32(void* p, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
/* The same in two instructions, for a multiple of 16. */
__device__ __forceinline__ void st_global_16x2(void* p, const uint32_t (&v)[8]) {
    uint4* d = static_cast<uint4*>(p);
    d[0] = make_uint4(v[0], v[1], v[2], v[3]);
    d[1] = make_uint4(v[4], v[5], v[6], v[7]);
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y,
                                         int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
            "r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

template <bool KV8>
__global__ void __launch_bounds__(Geo<KV8>::kThreads, 1)
cross_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
             const __grid_constant__ CUtensorMap vmap, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sb = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (sb - ptx::smem_u32(smem_raw));
    constexpr int kSlots = Geo<KV8>::kSlots, kRaw = Geo<KV8>::kRaw, kBarOff = Geo<KV8>::kBarOff;
    const uint32_t bars = sb + kBarOff;
    auto FULL = [&](int s) { return bars + 8u * s; };
    auto EMPTY = [&](int s) { return bars + 8u * (kSlots + s); };
    // score buffer u of tile w
    auto SFULL = [&](int w, int u) { return bars + 8u * (2 * kSlots + 2 * w + u); };
    auto PFULL = [&](int w, int u) { return bars + 8u * (2 * kSlots + 4 + 2 * w + u); };
    // one per buffer: when the scores in a buffer are there, the PV before the last is done,
    // so a wait for the last one cannot take an earlier phase for it
    auto PVDONE = [&](int w, int u) { return bars + 8u * (2 * kSlots + 8 + 2 * w + u); };
    const uint32_t QFULL = bars + 8u * (2 * kSlots + 12), QEMPTY = bars + 8u * (2 * kSlots + 13);
    const uint32_t TAIL = bars + 8u * (2 * kSlots + 14), MMADONE = bars + 8u * (2 * kSlots + 15);
    // e4m3 pages: a tile as it came is there, and has been converted
    auto RFULL = [&](int s) { return bars + 8u * (2 * kSlots + 16 + s); };
    auto REMPTY = [&](int s) { return bars + 8u * (2 * kSlots + 16 + kRaw + s); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kBarOff + Geo<KV8>::kBars * 8);
    volatile int32_t* abort_flag = reinterpret_cast<volatile int32_t*>(tmem_slot + 1);

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform for the compiler too
    if (tid == 0) {
        ptx::prefetch_tensormap(&qmap);
        ptx::prefetch_tensormap(&kmap);
        ptx::prefetch_tensormap(&vmap);
        for (int s = 0; s < kSlots; ++s) {
            ptx::mbar_init(FULL(s), KV8 ? 4 : 1);  // e4m3: one arrival per converting warp
            ptx::mbar_init(EMPTY(s), 2);  // both tiles are done with it
        }
        for (int w = 0; w < 2; ++w) {
            for (int u = 0; u < 2; ++u) {
                ptx::mbar_init(SFULL(w, u), 1);
                ptx::mbar_init(PFULL(w, u), 4);  // one arrival per warp
                ptx::mbar_init(PVDONE(w, u), 1);
            }
        }
        ptx::mbar_init(QFULL, 1);
        ptx::mbar_init(QEMPTY, 2);
        for (int s = 0; s < kRaw; ++s) {
            ptx::mbar_init(RFULL(s), 1);
            ptx::mbar_init(REMPTY(s), 4);
        }
        ptx::mbar_init(TAIL, 1);
        ptx::mbar_init(MMADONE, 2);
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 9) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    // all 512 columns: the allocation starts at column 0, so every TMEM address is a constant
    constexpr uint32_t tmem = 0;
    if (tid == 0 && *tmem_slot != tmem) {
        *abort_flag = 1;
        atomicOr(p.err, kDevErrTimeout);
    }
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();

    // Bounded wait on phase `parity`; gives up at once when another thread has aborted.
    auto wait_bar = [&](uint32_t bar, uint32_t parity) -> bool {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        const uint64_t t0 = ptx::globaltimer_ns();
        for (uint32_t it = 1;; ++it) {
            if (ptx::mbar_try_wait(bar, parity)) return true;
            if ((it & 63u) == 0u) {
                if (*abort_flag) return false;
                if (ptx::globaltimer_ns() - t0 > p.wait_limit_ns) {
                    *abort_flag = 1;
                    atomicOr(p.err, kDevErrTimeout);
                    return false;
                }
            }
        }
    };
    auto drain_bar = [&](uint32_t bar, uint32_t parity) {
        const uint64_t t0 = ptx::globaltimer_ns();
        while (!ptx::mbar_try_wait(bar, parity)) {
            if (ptx::globaltimer_ns() - t0 > p.wait_limit_ns) {
                atomicOr(p.err, kDevErrTimeout);
                return;
            }
        }
    };
    auto wait_all = [&](uint32_t bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait_bar(bar, parity));
    };

    __shared__ Slice slice;
    find_slice<Geo<KV8>::kThreads>(p, blockIdx.x, slice);
    if (tid == 0) p.cuts[blockIdx.x] = cut_of(p, blockIdx.x, slice);
    Walker wk;
    wk.init(p, slice, lane);
    Item it;

    if (warp == 8) {
        /* ================= TMA producer ================= */
        int n_kv = 0, n_q = 0, n_tail = 0;
        bool ok = true;
        const int P = p.P, box = p.box;
        while (ok && wk.next(p, lane, it)) {
            if (it.t0 == it.t1) continue;
            const int32_t* bt = p.block_table + (int64_t)it.b * p.bt_stride;
            // this lane's box of a tile (box >= 16: at most 8), its page looked up a tile ahead
            auto page_id = [&](int32_t tile) -> int32_t {
                const int32_t tok = tile * kTile + lane * box;
                if (lane * box >= kTile || tok >= it.L || tile >= it.t1) return 0;
                return ptx::ld(bt + (p.page_shift >= 0 ? tok >> p.page_shift : tok / P));
            };
            int32_t pid = page_id(it.t0);
            for (int32_t tile = it.t0; ok && tile < it.t1; ++tile) {
                const int32_t next_pid = page_id(tile + 1);
                const int32_t tok = tile * kTile + lane * box;
                const bool mine = lane * box < kTile && tok < it.L;
                if (mine && (uint32_t)pid >= (uint32_t)p.num_pages) {
                    atomicOr(p.err, kDevErrBadPage);
                    pid = 0;
                }
                const int32_t z = pid * P + (p.page_shift >= 0 ? tok & (P - 1) : tok % P);
                const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
                const int32_t nvalid = min(kTile, it.L - tile * kTile);
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    constexpr int kRing = KV8 ? kRaw : kSlots;
                    const int slot = n_kv % kRing;
                    if (n_kv >= kRing && !wait_all(KV8 ? REMPTY(slot) : EMPTY(slot), ((n_kv / kRing) - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = KV8 ? sb + Geo<KV8>::kRawOff + (uint32_t)slot * kHalf
                                             : sb + kRingOff + (uint32_t)slot * kSlot;
                    // a bf16 V tile that ends inside a 16-key step is finished here before its release
                    const bool tail = !KV8 && kv == 1 && (nvalid & 15) != 0;
                    const uint32_t bar = KV8 ? RFULL(slot) : (tail ? TAIL : FULL(slot));
                    if (lane == 0) {
                        const bool stuck = p.debug_stuck > 0 && n_kv == 0;
                        ptx::mbar_arrive_expect_tx(bar, (uint32_t)(boxes * box * (KV8 ? 128 : 256)) + (stuck ? 16u : 0u));
                    }
                    __syncwarp();
                    if (mine) {
                        const CUtensorMap* map = kv ? &vmap : &kmap;
                        // K and V tiles are read again by the other q tiles of the sequence: no
                        // eviction hint
                        tma_load(dst + (uint32_t)(lane * box) * 128u, map, bar, 0, it.kvh, z);
                        if (!KV8) tma_load(dst + kHalf + (uint32_t)(lane * box) * 128u, map, bar, 64, it.kvh, z);
                    }
                    ++n_kv;
                    if (tail) {
                        if (!wait_all(TAIL, n_tail & 1)) {
                            drain_bar(TAIL, n_tail & 1);
                            ok = false;
                            // the slot's phase never completes: nothing of it is in flight
                            --n_kv;
                            break;
                        }
                        ++n_tail;
                        const int r1 = (nvalid + 15) & ~15;
                        for (int x = lane; x < (r1 - nvalid) * 16; x += 32) {
                            const uint32_t a = dst + (uint32_t)(nvalid + (x >> 4)) * 128u + (uint32_t)(x & 7) * 16u +
                                               ((x & 8) ? (uint32_t)kHalf : 0u);
                            ptx::sts_u4(a, make_uint4(0, 0, 0, 0));
                        }
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive(FULL(slot));
                    }
                    if (kv == 0 && tile == it.t0) {
                        // the item's Q tiles, once the last item's scores are done with theirs
                        if (n_q > 0 && !wait_all(QEMPTY, (n_q - 1) & 1)) {
                            ok = false;
                            break;
                        }
                        if (lane == 0) {
                            const bool two = it.tok0 + p.tile_tokens < it.tok_end;
                            const uint32_t bytes = (uint32_t)(p.tile_tokens * p.g) * 256u;
                            ptx::mbar_arrive_expect_tx(QFULL, two ? 2 * bytes : bytes);
                            for (int w = 0; w < (two ? 2 : 1); ++w)
                                for (int hf = 0; hf < 2; ++hf)
                                    tma_load(sb + kQOff + (uint32_t)(w * kSlot + hf * kHalf), &qmap, QFULL, hf * 64,
                                             it.kvh * p.g, it.tok0 + w * p.tile_tokens);
                        }
                        __syncwarp();
                        ++n_q;
                    }
                }
                pid = next_pid;
            }
        }
        // loads of the last slots may still be in flight (after an abort)
        if (lane == 0) {
            constexpr int kRing = KV8 ? kRaw : kSlots;
            for (int k = n_kv > kRing ? n_kv - kRing : 0; k < n_kv; ++k)
                drain_bar(KV8 ? RFULL(k % kRing) : FULL(k % kRing), (k / kRing) & 1);
            if (n_q > 0) drain_bar(QFULL, (n_q - 1) & 1);
        }
        __syncwarp();
    } else if (warp == 9 || warp == 10) {
        /* ================= MMA issuers: warp 9 tile 0, warp 10 tile 1 ================= */
        const int w = warp - 9;
        const uint32_t tS = tmem + (uint32_t)w * 128u, tO = tmem + 256u + (uint32_t)w * 128u;
        const uint64_t qd = sdesc(sb + kQOff + (uint32_t)w * kSlot, 16, 1024);
        const uint64_t kd = sdesc(sb + kRingOff, 16, 1024), vd = sdesc(sb + kRingOff, kHalf, 1024);
        // ring places of the next K and V tile (loads alternate: K, V, K, V ...), their phases
        int ks = 0, vs = 1, n_q = 0, n = 0;  // Q loads, steps so far
        uint32_t kph = 0, vph = 0;
        bool ok = true;
        auto advance = [&](int& slot, uint32_t& phase) {
            slot += 2;
            if (slot >= kSlots) {
                slot -= kSlots;
                phase ^= 1u;
            }
        };
        while (ok && wk.next(p, lane, it)) {
            const int m = __shfl_sync(0xffffffffu, steps_of(it.L, it.t0, it.t1), 0);
            if (m == 0) continue;
            const bool active = __shfl_sync(0xffffffffu, it.tok0 + w * p.tile_tokens < it.tok_end ? 1 : 0, 0) != 0;
            const int keys = __shfl_sync(0xffffffffu, it.L - it.t0 * kTile, 0);
            ok = wait_all(QFULL, n_q & 1);
            ++n_q;
            if (!active) {  // nothing but the releases
                for (int i = 0; i < m && ok; i += 2) {
                    ok = wait_all(FULL(ks), kph);
                    if (ok && lane == 0) ptx::mbar_arrive(EMPTY(ks));
                    ok = ok && wait_all(FULL(vs), vph);
                    if (ok && lane == 0) ptx::mbar_arrive(EMPTY(vs));
                    advance(ks, kph);
                    advance(vs, vph);
                }
                if (ok && lane == 0) ptx::mbar_arrive(QEMPTY);
                continue;
            }
            // step i of the item: scores of keys [64 i, 64 i + 64) into buffer (n + i) & 1
            auto qk = [&](int i) -> bool {
                const int h = i & 1, u = (n + i) & 1;
                if (h == 0 && !wait_all(FULL(ks), kph)) return false;
                ptx::tc_fence_after();
                const uint64_t k = kd + (uint64_t)((ks * kSlot + h * (kStep * 128)) >> 4);
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const uint64_t o = (uint64_t)((x >> 2) * kHalf + (x & 3) * 32) >> 4;
                    ptx::tc_mma_f16_elect(tS + (uint32_t)(u * kStep), qd + o, k + o, idesc(0, kStep), x > 0 ? 1u : 0u);
                }
                ptx::tc_commit_elect(SFULL(w, u));
                if (h == 1 || i + 1 == m) {
                    ptx::tc_commit_elect(EMPTY(ks));
                    advance(ks, kph);
                    if (i + 1 == m) ptx::tc_commit_elect(QEMPTY);
                }
                return true;
            };
            ok = ok && qk(0);
            if (m > 1) ok = ok && qk(1);
#pragma unroll 1
            for (int i = 0; i < m && ok; ++i) {
                const int h = i & 1, u = (n + i) & 1;
                ok = (h == 1 || wait_all(FULL(vs), vph)) && wait_all(PFULL(w, u), ((n + i) >> 1) & 1);
                if (!ok) break;
                ptx::tc_fence_after();
                const uint64_t v = vd + (uint64_t)((vs * kSlot + h * (kStep * 128)) >> 4);
                const int left = keys - i * kStep, k16 = left >= kStep ? kStep / 16 : (left + 15) >> 4;
#pragma unroll
                for (int x = 0; x < kStep / 16; ++x)
                    if (x < k16)
                        ptx::tc_mma_f16_ts_elect(tO, tS + (uint32_t)(u * kStep + x * 8), v + (uint64_t)(x * 128),
                                                 idesc(1, 128), (i == 0 && x == 0) ? 0u : 1u);
                ptx::tc_commit_elect(PVDONE(w, u));
                if (h == 1 || i + 1 == m) {
                    ptx::tc_commit_elect(EMPTY(vs));
                    advance(vs, vph);
                }
                if (i + 2 < m) ok = qk(i + 2);
            }
            n += m;
        }
        // every MMA issued is complete before TMEM is freed
        ptx::tc_commit_elect(MMADONE);
        if (lane == 0) drain_bar(MMADONE, 0);
        __syncwarp();
    } else if (warp >= 12) {
        /* ================= e4m3 tiles to bf16 (KV8) ================= */
        // thread = key: its 128 bytes become two 128-byte halves in the swizzle the MMAs read;
        // V rows behind the last key, up to the end of their 16-key step, become zeros
        const int row = tid - 384;
        const uint32_t sw = (uint32_t)(row & 7);
        int n = 0;
        bool ok = KV8;
        while (ok && wk.next(p, lane, it)) {
            for (int32_t tile = it.t0; ok && tile < it.t1; ++tile) {
                const int32_t nvalid = it.L - tile * kTile;
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv, ++n) {
                    constexpr int kRing = KV8 ? kRaw : 1;
                    const int raw = n % kRing, slot = n % kSlots;
                    // both at once where neither is waited for
                    const bool r = ptx::mbar_try_wait(RFULL(raw), (n / kRing) & 1);
                    const bool e = n < kSlots || ptx::mbar_try_wait(EMPTY(slot), ((n / kSlots) - 1) & 1);
                    if (!__all_sync(0xffffffffu, r && e)) {
                        ok = wait_all(RFULL(raw), (n / kRing) & 1) &&
                             (n < kSlots || wait_all(EMPTY(slot), ((n / kSlots) - 1) & 1));
                        if (!ok) break;
                    }
                    const uint32_t src = sb + Geo<KV8>::kRawOff + (uint32_t)(raw * kHalf + row * 128);
                    const uint32_t dst = sb + kRingOff + (uint32_t)(slot * kSlot + row * 128);
                    if (row >= nvalid) {
                        if (row < ((nvalid + 15) & ~15))
                            for (uint32_t x = 0; x < 16; ++x)
                                ptx::sts_u4(dst + (x >> 3) * kHalf + ((x & 7u) << 4), make_uint4(0, 0, 0, 0));
                    } else {
                        uint32_t nan = 0;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {  // 16 dimensions each
                            const uint4 v = ptx::lds_u4(src + (((uint32_t)c ^ sw) << 4));
                            const uint32_t b[4] = {v.x, v.y, v.z, v.w};
                            uint32_t h[8];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                e4m3x4_to_bf16(b[e], h[2 * e], h[2 * e + 1]);
                                nan |= (b[e] & 0x7f7f7f7fu) + 0x01010101u;
                            }
                            const uint32_t half = dst + (uint32_t)((c >> 2) * kHalf), cc = (uint32_t)(2 * (c & 3));
                            ptx::sts_u4(half + ((cc ^ sw) << 4), make_uint4(h[0], h[1], h[2], h[3]));
                            ptx::sts_u4(half + (((cc + 1) ^ sw) << 4), make_uint4(h[4], h[5], h[6], h[7]));
                        }
                        if (nan & 0x80808080u) {  // some element is NaN: its bytes read again
#pragma unroll 1
                            for (uint32_t x = 0; x < 128; ++x) {
                                const uint32_t at = ((x >> 4) ^ sw) * 16u + (x & 15u);
                                const uint32_t to = (x >> 6) * kHalf + ((((x >> 3) & 7u) ^ sw) << 4) + (x & 7u) * 2u;
                                if ((smem[src - sb + at] & 0x7fu) == 0x7fu)
                                    *reinterpret_cast<uint16_t*>(smem + (dst - sb) + to) = 0x7fffu;
                            }
                        }
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::mbar_arrive(FULL(slot));
                        ptx::mbar_arrive(REMPTY(raw));
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp < 8) {
        /* ================= softmax and output ================= */
        const int w = warp >> 2;
        const int row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = (tmem + (uint32_t)w * 128u) | lanes, tO = (tmem + 256u + (uint32_t)w * 128u) | lanes;
        const int my_tok = row / p.g, my_head = row - my_tok * p.g;
        int n_s = 0;  // steps of this tile so far
        bool ok = true;
        while (ok && wk.next(p, lane, it)) {
            const int32_t first = it.tok0 + w * p.tile_tokens;
            if (first >= it.tok_end) continue;
            const int32_t tok = first + my_tok;
            const bool valid = row < p.tile_tokens * p.g && tok < it.tok_end;
            const int head = it.kvh * p.g + my_head;
            float m_ref = -INFINITY, l = 0.f;
            float mul = p.scale_log2, sign = 1.f;
            if (KV8 && p.k_scale) {
                // the factor has to be positive for the masked -inf and the maximum: a scale of
                // zero (a head quantised from zeros) or below goes into the scores instead
                mul *= ptx::ld(p.k_scale + it.kvh);
                if (mul <= 0.f) {
                    sign = mul < 0.f ? -1.f : 0.f;
                    mul = mul < 0.f ? -mul : 1.f;
                }
            }
            const int m = steps_of(it.L, it.t0, it.t1);
#pragma unroll 1
            for (int i = 0; i < m; ++i, ++n_s) {
                const uint32_t tB = tS + (uint32_t)((n_s & 1) * kStep);
                if (!wait_all(SFULL(w, n_s & 1), (n_s >> 1) & 1)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after();
                float s[kStep];
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    ptx::tc_ld32(tB + 32u * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
                ptx::tc_wait_ld();
                if (KV8 && sign != 1.f) {
#pragma unroll
                    for (int k = 0; k < kStep; ++k) s[k] *= sign;
                }
                const int32_t nvalid = it.L - (it.t0 * kTile + i * kStep);
                if (nvalid < kStep) {
#pragma unroll
                    for (int k = 0; k < kStep; ++k) s[k] = k < nvalid ? s[k] : -INFINITY;
                }
                // eight chains of three-operand maxima
                float m8[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) m8[e] = fmaxf(fmaxf(s[e], s[8 + e]), s[16 + e]);
#pragma unroll
                for (int k = 24; k < 56; k += 16)
#pragma unroll
                    for (int e = 0; e < 8; ++e) m8[e] = fmaxf(fmaxf(m8[e], s[k + e]), s[k + 8 + e]);
#pragma unroll
                for (int e = 0; e < 8; ++e) m8[e] = fmaxf(m8[e], s[56 + e]);
                const float mx = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])),
                                       fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7]))) * mul;
                const bool raise = mx > m_ref + kLazyLog2;
                if (__any_sync(0xffffffffu, raise)) {
                    const float m_new = raise ? mx : m_ref;
                    const float alpha = raise ? ptx::ex2(m_ref - m_new) : 1.f;
                    m_ref = m_new;
                    l *= alpha;
                    if (i > 0) {  // the products so far
                        if (!wait_all(PVDONE(w, (n_s - 1) & 1), ((n_s - 1) >> 1) & 1)) {
                            ok = false;
                            break;
                        }
                        ptx::tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < 8; ++c) {
                            float o[16];
                            ptx::tc_ld16(tO + 16u * c, o);
                            ptx::tc_wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] *= alpha;
                            ptx::tc_st16(tO + 16u * c, o);
                        }
                    }
                }
                const float base = m_ref == -INFINITY ? 0.f : m_ref;
                const float2 mul2 = make_float2(mul, mul), sub2 = make_float2(-base, -base);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint32_t pk[kStep / 2];
#pragma unroll
                for (int k = 0; k < kStep / 2; ++k) {
                    float2 x = ptx::fma2(make_float2(s[2 * k], s[2 * k + 1]), mul2, sub2);
                    x.x = ptx::ex2(x.x);
                    x.y = ptx::ex2(x.y);
                    sum[k & 1] = ptx::add2(sum[k & 1], x);
                    pk[k] = ptx::pack_bf16x2(x.x, x.y);
                }
                ptx::tc_st32(tB, pk);
                sum[0] = ptx::add2(sum[0], sum[1]);
                l += sum[0].x + sum[0].y;
                ptx::tc_wait_st();
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(PFULL(w, n_s & 1));
            }
            if (!ok) break;
            const bool none = !(it.t1 > it.t0);
            if (!none) {
                if (!wait_all(PVDONE(w, (n_s - 1) & 1), ((n_s - 1) >> 1) & 1)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after();
            }
            // a row whose scores are all -inf has no weight to normalise by
            const float inv = l == 0.f ? 0.f : (KV8 && p.v_scale ? ptx::ld(p.v_scale + it.kvh) : 1.f) / l;
            const int64_t at = (int64_t)tok * p.Hq + head;
            // part of a cut item: the slice's first one if it begins before the slice, else its last
            const int64_t rec = (int64_t)(2 * blockIdx.x + (it.t0 > 0 ? 0 : 1)) * kRows + w * kTile + row;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                if (!none) {
                    ptx::tc_ld32(tO + 32u * c, o);
                    ptx::tc_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                if (!valid) continue;
                if (!it.cut) {
                    __nv_bfloat16* dst = p.out + at * 128 + 32 * c;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t h[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            h[e] = l == 0.f ? 0u : ptx::pack_bf16x2(__uint_as_float(o[16 * i + 2 * e]) * inv,
                                                                    __uint_as_float(o[16 * i + 2 * e + 1]) * inv);
                        if (p.out_32) st_global_32(dst + 16 * i, h);
                        else st_global_16x2(dst + 16 * i, h);
                    }
                } else if (l != 0.f) {
                    float* dst = p.rec_o + rec * 128 + 32 * c;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t h[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) h[e] = __float_as_uint(__uint_as_float(o[8 * i + e]) * inv);
                        st_global_32(dst + 8 * i, h);
                    }
                }
            }
            ptx::tc_fence_before();
            if (valid) {
                const float l2 = l == 0.f ? -INFINITY : m_ref + log2f(l);
                if (it.cut) p.rec_lse[rec] = l2;
                else if (p.lse != nullptr)
                    p.lse[p.cu ? (int64_t)head * p.T + tok : ((int64_t)it.b * p.Hq + head) * p.S + (tok - it.b * p.S)] =
                        l2 * 0.6931471805599453f;
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(*tmem_slot, 512);
    }
}

/* Joins the parts of cut items: out = sum_s 2^(l_s - l) O_s with 2^l = sum_s 2^(l_s); a
 * part without weight has l_s = -inf and no O.  Block (j, y): 32 rows of the item that slice
 * j + 1 cuts first, each thread 16 dimensions of one, with the maximum moved as the parts come. */
constexpr int kJoinThreads = 256, kParts = 2;
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Params p) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int32_t j = blockIdx.x;
    const int4* k4 = reinterpret_cast<const int4*>(p.cuts + j + 1);
    const int4 k0 = __ldcg(k4);
    const int4 k1 = __ldcg(k4 + 1);
    if (k0.x == 0) return;
    const int32_t last = k0.y, b = k0.z, kvh = k0.w, tok0 = k1.x, tok_end = k1.y;
    const int32_t r = blockIdx.y * 32 + (threadIdx.x >> 3), d = (threadIdx.x & 7) * 16;
    const int32_t w = r >> 7, row = r & (kTile - 1), t = row / p.g;
    const int32_t tok = tok0 + w * p.tile_tokens + t, head = kvh * p.g + (row - t * p.g);
    if (t >= p.tile_tokens || tok >= tok_end) return;
    auto rec_of = [&](int32_t c) { return (int64_t)(2 * c + (c == j ? 1 : 0)) * kRows + r; };
    float m = -INFINITY, sum = 0.f, acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    // kParts parts in flight, with their log-sum-exps: one token over 8000 keys, 8 + 1 heads,
    // 27 -> 19 us; with four in flight the registers cost more where whole tiles are joined (ragged
    // prompts: 169 instead of 163 us in one session)
#pragma unroll 1
    for (int32_t c0 = j; c0 <= last; c0 += kParts) {
        float l2[kParts], top = m;
        float4 o[kParts][4];
#pragma unroll
        for (int u = 0; u < kParts; ++u) {
            const int64_t rec = rec_of(min(c0 + u, last));
            l2[u] = __ldcg(p.rec_lse + rec);
            const float4* src = reinterpret_cast<const float4*>(p.rec_o + rec * 128 + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[u][i] = __ldcg(src + i);
        }
#pragma unroll
        for (int u = 0; u < kParts; ++u) {
            if (c0 + u > last) l2[u] = -INFINITY;
            top = fmaxf(top, l2[u]);
        }
        const float base = top == -INFINITY ? 0.f : top, alpha = exp2f(m - base);
        m = top;
        sum *= alpha;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] *= alpha;
#pragma unroll
        for (int u = 0; u < kParts; ++u) {
            if (l2[u] == -INFINITY) continue;        // whose O was not written
            const float wgt = exp2f(l2[u] - base);   // NaN parts reach the result through their weight
            sum += wgt;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[4 * i] = fmaf(wgt, o[u][i].x, acc[4 * i]);
                acc[4 * i + 1] = fmaf(wgt, o[u][i].y, acc[4 * i + 1]);
                acc[4 * i + 2] = fmaf(wgt, o[u][i].z, acc[4 * i + 2]);
                acc[4 * i + 3] = fmaf(wgt, o[u][i].w, acc[4 * i + 3]);
            }
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint4* dst = reinterpret_cast<uint4*>(p.out + ((int64_t)tok * p.Hq + head) * 128 + d);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        dst[i] = make_uint4(ptx::pack_bf16x2(acc[8 * i] * inv, acc[8 * i + 1] * inv),
                            ptx::pack_bf16x2(acc[8 * i + 2] * inv, acc[8 * i + 3] * inv),
                            ptx::pack_bf16x2(acc[8 * i + 4] * inv, acc[8 * i + 5] * inv),
                            ptx::pack_bf16x2(acc[8 * i + 6] * inv, acc[8 * i + 7] * inv));
    if (d == 0 && p.lse != nullptr) {
        const float l2 = sum == 0.f ? -INFINITY : m + log2f(sum);
        p.lse[p.cu ? (int64_t)head * p.T + tok : ((int64_t)b * p.Hq + head) * p.S + (tok - b * p.S)] =
            l2 * 0.6931471805599453f;
    }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

/* (128 dims, heads, tokens) with boxes of 128 bytes of a row (64 bf16, 128 e4m3), 128-byte
 * swizzle; boxes past the end read zeros. */
int encode(CUtensorMap* map, const void* base, int64_t heads, int64_t tokens, int64_t token_stride_bytes,
           int64_t box_heads, int64_t box_tokens, bool e4m3 = false) {
    EncodeFn fn = reinterpret_cast<EncodeFn>(host_encode_tiled());
    if (fn == nullptr) return PGQA_ERR_CUDA;
    cuuint64_t dims[3] = {128, (cuuint64_t)heads, (cuuint64_t)tokens};
    cuuint64_t strides[2] = {e4m3 ? 128u : 256u, (cuuint64_t)token_stride_bytes};
    cuuint32_t box[3] = {e4m3 ? 128u : 64u, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
    cuuint32_t step[3] = {1, 1, 1};
    return fn(map, e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
              const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              e4m3 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? PGQA_OK
               : PGQA_ERR_CUDA;
}

/* CTAs of the first launch: one per SM, or fewer where the key tiles are fewer (by the
 * table's capacity). */
int grid_for(int64_t T, int64_t B, int64_t Hkv, int64_t g, int64_t cap_tokens, int sms) {
    const int64_t items = (T / (2 * (kTile / g)) + B) * Hkv;  // at least as many as there are
    const int64_t tiles = (cap_tokens + kTile - 1) / kTile;
    if (items >= sms || tiles >= sms) return sms;
    const int64_t n = items * (tiles + kItemCost) / kMinSlice;
    return (int)(n < 1 ? 1 : (n < sms ? n : sms));
}

int shape_ok(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t P, int64_t bt_stride) {
    const int st = host_check_pages(B, Hkv, D, P, 1, bt_stride);
    if (st != PGQA_OK) return st;
    if (T < 0 || Hq <= 0 || Hq % Hkv != 0) return PGQA_ERR_BAD_SHAPE;
    if (T > INT32_MAX || Hq / Hkv > kTile || Hq > 65536) return PGQA_ERR_UNSUPPORTED;
    return PGQA_OK;
}

size_t workspace_bytes(int grid) { return (size_t)grid * (2 * kRows * (128 + 1) * 4 + sizeof(Cut)); }

template <bool KV8>
int launch(const Params& p, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, int dev,
           cudaStream_t stream) {
    static HostSmemDone done;
    using G = Geo<KV8>;
    const int st = host_smem_limit(cross_kernel<KV8>, dev, G::kSmem, done);
    if (st != PGQA_OK) return st;
    return host_launch(cross_kernel<KV8>, dim3((unsigned)p.grid), G::kThreads, G::kSmem, stream, 1, qm, km, vm, p);
}

int entry(const pgqa_cross_args* a, cudaStream_t stream) {
    if (a == nullptr) return PGQA_ERR_NULL_POINTER;
    if (a->struct_size != sizeof(pgqa_cross_args)) return PGQA_ERR_BAD_SHAPE;
    if (!a->q || !a->k_cache || !a->v_cache || !a->out || !a->seq_lens || !a->block_table)
        return PGQA_ERR_NULL_POINTER;
    int st = shape_ok(a->tokens, a->batch_size, a->num_heads, a->num_heads_k, a->headdim, a->page_size, a->bt_stride);
    if (st != PGQA_OK) return st;
    if (a->kv_format != 0 && a->kv_format != 1) return PGQA_ERR_UNSUPPORTED;
    const bool kv8 = a->kv_format == 1;
    if (!kv8 && (a->k_scale || a->v_scale)) return PGQA_ERR_BAD_SHAPE;
    if (a->num_pages <= 0) return PGQA_ERR_BAD_SHAPE;
    if (a->num_pages >= ((int64_t)1 << 31) / a->page_size) return PGQA_ERR_UNSUPPORTED;
    if (!a->cu_seqlens && (a->seqlen_q < 0 || a->tokens != a->batch_size * a->seqlen_q)) return PGQA_ERR_BAD_SHAPE;
    if (!(a->scale > 0.f) || !isfinite(a->scale)) return PGQA_ERR_BAD_SHAPE;
    if (a->q_stride < a->num_heads * 128) return PGQA_ERR_BAD_SHAPE;
    if (a->q_stride % 8 != 0 || !host_aligned(a->q, 16) || !host_aligned(a->k_cache, 16) ||
        !host_aligned(a->v_cache, 16) || !host_aligned(a->out, 16) || !host_aligned(a->softmax_lse, 4) ||
        !host_aligned(a->seq_lens, 4) || !host_aligned(a->block_table, 4) || !host_aligned(a->cu_seqlens, 4) ||
        !host_aligned(a->workspace, 256) || !host_aligned(a->k_scale, 4) || !host_aligned(a->v_scale, 4))
        return PGQA_ERR_MISALIGNED;
    if (a->q_stride >= ((int64_t)1 << 39)) return PGQA_ERR_UNSUPPORTED;  // a tensor map's stride is 40 bits
    int dev, sms, optin;
    if ((st = host_device(&dev, &sms, &optin)) != PGQA_OK) return st;
    Params p = {};
    if ((st = host_error_word(dev, &p.err)) != PGQA_OK) return st;
    if (a->tokens == 0) return PGQA_OK;
    // items are counted in 32 bits
    if ((a->tokens / (kTile / (a->num_heads / a->num_heads_k)) + a->batch_size) * a->num_heads_k > INT32_MAX)
        return PGQA_ERR_UNSUPPORTED;
    p.g = (int32_t)(a->num_heads / a->num_heads_k);
    p.cap_tokens = a->bt_stride * a->page_size;
    p.grid = grid_for(a->tokens, a->batch_size, a->num_heads_k, p.g, p.cap_tokens, sms);
    if (a->workspace == nullptr || a->workspace_bytes < workspace_bytes(p.grid)) return PGQA_ERR_WORKSPACE;
    p.rec_o = static_cast<float*>(a->workspace);
    p.rec_lse = p.rec_o + (size_t)2 * p.grid * kRows * 128;
    p.cuts = reinterpret_cast<Cut*>(p.rec_lse + (size_t)2 * p.grid * kRows);
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.out_32 = host_aligned(a->out, 32);
    p.lse = a->softmax_lse;
    p.seq_lens = a->seq_lens;
    p.block_table = a->block_table;
    p.cu = a->cu_seqlens;
    p.k_scale = a->k_scale;
    p.v_scale = a->v_scale;
    p.bt_stride = a->bt_stride;
    p.B = (int32_t)a->batch_size;
    p.S = (int32_t)a->seqlen_q;
    p.T = (int32_t)a->tokens;
    p.Hq = (int32_t)a->num_heads;
    p.Hkv = (int32_t)a->num_heads_k;
    p.P = (int32_t)a->page_size;
    p.page_shift = host_shift(a->page_size);
    p.num_pages = (int32_t)a->num_pages;
    p.tile_tokens = kTile / p.g;
    p.box = 16;
    while (p.box < kTile && a->page_size % (2 * p.box) == 0) p.box *= 2;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    const char* lim = getenv("PGQA_WAIT_LIMIT_NS");
    p.wait_limit_ns = (lim && *lim) ? strtoull(lim, nullptr, 10) : kWaitLimitNs;
    if (p.wait_limit_ns == 0 || p.wait_limit_ns > 10 * kWaitLimitNs) p.wait_limit_ns = kWaitLimitNs;
    const char* stuck = getenv("PGQA_DEBUG_STUCK_BARRIER");
    const int hook = (stuck && *stuck) ? atoi(stuck) : 0;
    p.debug_stuck = hook > 0 ? hook : 0;
    p.debug_long = hook < 0 ? -hook : 0;
    CUtensorMap qm, km, vm;
    const int64_t slots = a->num_pages * a->page_size;
    const int64_t row = kv8 ? 128 : 256;
    if ((st = encode(&qm, a->q, a->num_heads, a->tokens, a->q_stride * 2, p.g, p.tile_tokens)) != PGQA_OK ||
        (st = encode(&km, a->k_cache, a->num_heads_k, slots, a->num_heads_k * row, 1, p.box, kv8)) != PGQA_OK ||
        (st = encode(&vm, a->v_cache, a->num_heads_k, slots, a->num_heads_k * row, 1, p.box, kv8)) != PGQA_OK)
        return st;
    st = kv8 ? launch<true>(p, qm, km, vm, dev, stream) : launch<false>(p, qm, km, vm, dev, stream);
    if (st != PGQA_OK || p.grid == 1) return st;
    return host_launch(join_kernel, dim3((unsigned)(p.grid - 1), kRows / 32), kJoinThreads, 0, stream, 1, p);
}

}  // namespace cross
}  // namespace pgqa

extern "C" size_t pgqa_cross_workspace_size(int64_t tokens, int64_t batch_size, int64_t num_heads,
                                            int64_t num_heads_k, int64_t headdim, int64_t page_size,
                                            int64_t bt_stride) {
    using namespace pgqa;
    int st = cross::shape_ok(tokens, batch_size, num_heads, num_heads_k, headdim, page_size, bt_stride);
    int dev, sms = 0, optin;
    if (st == PGQA_OK) st = host_device(&dev, &sms, &optin);
    if (host_set_status(st) != PGQA_OK || tokens == 0) return 0;
    return cross::workspace_bytes(cross::grid_for(tokens, batch_size, num_heads_k, num_heads / num_heads_k,
                                                  bt_stride * page_size, sms));
}

extern "C" int pgqa_cross_attention(const pgqa_cross_args* args, void* stream) {
    return pgqa::host_set_status(pgqa::cross::entry(args, static_cast<cudaStream_t>(stream)));
}
