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
 * once per 256 rows.  A work item is (sequence, KV head, two such tiles, a range of keys);
 * one persistent CTA per SM walks the items in the same order in all of its roles:
 *
 *   warps 0-3, 4-7  softmax and output of tile 0 and tile 1: thread = row = TMEM lane.  The
 *                   running maximum is moved only when a score exceeds it by 2^8 (O is then
 *                   rescaled in TMEM), so the O accumulator is touched once per item in the
 *                   usual case; sums and statistics are fp32, P is rounded to bf16 (half a
 *                   step, 2^-9 relative to its power of two, of weights that are summed in
 *                   fp32) and goes back to TMEM over the scores it came from.
 *   warp 8          TMA: Q tiles, and 128-key tiles of K and V by page boxes through one
 *                   ring of five 32 KB slots; it zeroes V rows behind the last key, so that
 *                   a weight of 0 never meets a NaN left in a page.
 *   warp 9          issues the MMAs (one thread): S_w = Q_w K^T (both from shared memory),
 *                   O_w += P_w V (P from TMEM).  The score tile of the next keys is issued
 *                   right behind the PV of the present ones, and the two tiles alternate,
 *                   so the tensor core works for one while the other's softmax runs.
 * TMEM: S and P of the tiles at columns 0 and 128, O at 256 and 384.
 *
 * With fewer items than SMs the keys are cut into ranges as well: each range writes its
 * normalised O (fp32) and log-sum-exp, and a second launch joins them.
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
#include "pgqa_ptx.cuh"

namespace pgqa {
namespace cross {

constexpr int kThreads = 320;
constexpr int kTile = 128;                 // rows of a tile, and keys of a K / V tile
constexpr int kHalf = kTile * 128;         // one 64-dimension half of a tile, bf16
constexpr int kSlot = 2 * kHalf;
constexpr int kSlots = 5;
constexpr int kQOff = 0, kRingOff = 2 * kSlot, kBarOff = kRingOff + kSlots * kSlot;
constexpr int kBars = 2 * kSlots + 10;
constexpr int kSmem = 1024 + kBarOff + kBars * 8 + 16;
constexpr float kLazyLog2 = 8.f;
constexpr uint64_t kWaitLimitNs = 1000000000ull;
constexpr int kMaxSplits = 32;

struct Params {
    __nv_bfloat16* out;      // [T, Hq, 128]
    float* lse;              // optional: [Hq, T] packed, [B, Hq, S] padded
    float *part_o, *part_lse;  // key ranges: [splits][T][Hq][128] and [splits][T][Hq] (log2 units)
    const int32_t *seq_lens, *block_table, *cu;
    int32_t* err;
    int64_t bt_stride, cap_tokens;
    int32_t B, S, T, Hq, Hkv, g, P, page_shift, num_pages;
    int32_t tile_tokens;     // prompt tokens per tile: 128 / g
    int32_t box;             // tokens of one TMA box of a pool: a power of two that divides P
    int32_t splits;
    float scale_log2;
    uint64_t wait_limit_ns;
};

__device__ __forceinline__ uint64_t sdesc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
/* fp32 accumulator, bf16 A and B, M = N = 128; B major: 0 = K, 1 = N */
__host__ __device__ constexpr uint32_t idesc(uint32_t b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
}

struct Item {
    int32_t b, kvh, tok0, tok_end, L, t0, t1, split;  // prompt tokens from tok0, key tiles [t0, t1)
};

/* Walks this CTA's items; called by whole warps, every role with a copy of its own. */
struct Walker {
    int64_t at, base;        // next item, items before sequence b0
    int32_t b0, total;       // block of 32 sequences, and its items
    int32_t cnt, incl, tok0, tok1;  // this lane's sequence: items, running sum, prompt tokens
    __device__ void load(const Params& p, int lane) {
        const int32_t b = b0 + lane;
        cnt = 0;
        tok0 = tok1 = 0;
        if (b < p.B) {
            tok0 = p.cu ? __ldg(p.cu + b) : b * p.S;
            tok1 = p.cu ? __ldg(p.cu + b + 1) : tok0 + p.S;
            if (tok0 < 0 || tok1 < tok0 || tok1 > p.T) {
                atomicOr(p.err, kDevErrBadSeqlen);
                tok0 = max(0, min(tok0, p.T));
                tok1 = max(tok0, min(tok1, p.T));
            }
            cnt = (tok1 - tok0 + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens) * p.Hkv * p.splits;
        }
        incl = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        total = __shfl_sync(0xffffffffu, incl, 31);
    }
    __device__ void init(const Params& p, int lane) {
        at = blockIdx.x;
        base = 0;
        b0 = 0;
        load(p, lane);
    }
    __device__ bool next(const Params& p, int lane, Item& it) {
        while (at >= base + total) {
            base += total;
            b0 += 32;
            if (b0 >= p.B) return false;
            load(p, lane);
        }
        const int32_t r0 = (int32_t)(at - base);
        const int f = __ffs(__ballot_sync(0xffffffffu, incl > r0)) - 1;
        const int32_t r = r0 - __shfl_sync(0xffffffffu, incl - cnt, f);
        const int32_t t_lo = __shfl_sync(0xffffffffu, tok0, f);
        it.tok_end = __shfl_sync(0xffffffffu, tok1, f);
        it.b = b0 + f;
        const int32_t pairs = (it.tok_end - t_lo + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
        const int32_t unit = r / p.splits;
        it.split = r - unit * p.splits;
        it.kvh = unit / pairs;
        it.tok0 = t_lo + (unit - it.kvh * pairs) * 2 * p.tile_tokens;
        int64_t L = __ldg(p.seq_lens + it.b);
        if (L < 0 || L > p.cap_tokens) {
            if (lane == 0) atomicOr(p.err, kDevErrBadSeqlen);
            L = L < 0 ? 0 : p.cap_tokens;
        }
        it.L = (int32_t)L;
        const int32_t n = (it.L + kTile - 1) / kTile, per = (n + p.splits - 1) / p.splits;
        it.t0 = min(n, it.split * per);
        it.t1 = min(n, it.t0 + per);
        at += gridDim.x;
        return true;
    }
};

__global__ void __launch_bounds__(kThreads, 1)
cross_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
             const __grid_constant__ CUtensorMap vmap, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sb = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (sb - ptx::smem_u32(smem_raw));
    const uint32_t bars = sb + kBarOff;
    auto FULL = [&](int s) { return bars + 8u * s; };
    auto EMPTY = [&](int s) { return bars + 8u * (kSlots + s); };
    auto SFULL = [&](int w) { return bars + 8u * (2 * kSlots + w); };
    auto PFULL = [&](int w) { return bars + 8u * (2 * kSlots + 2 + w); };
    auto PVDONE = [&](int w) { return bars + 8u * (2 * kSlots + 4 + w); };
    const uint32_t QFULL = bars + 8u * (2 * kSlots + 6), QEMPTY = bars + 8u * (2 * kSlots + 7);
    const uint32_t TAIL = bars + 8u * (2 * kSlots + 8), MMADONE = bars + 8u * (2 * kSlots + 9);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kBarOff + kBars * 8);
    volatile int32_t* abort_flag = reinterpret_cast<volatile int32_t*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        ptx::prefetch_tensormap(&qmap);
        ptx::prefetch_tensormap(&kmap);
        ptx::prefetch_tensormap(&vmap);
        for (int s = 0; s < kSlots; ++s) {
            ptx::mbar_init(FULL(s), 1);
            ptx::mbar_init(EMPTY(s), 1);
        }
        for (int w = 0; w < 2; ++w) {
            ptx::mbar_init(SFULL(w), 1);
            ptx::mbar_init(PFULL(w), 4);  // one arrival per warp
            ptx::mbar_init(PVDONE(w), 1);
        }
        ptx::mbar_init(QFULL, 1);
        ptx::mbar_init(QEMPTY, 1);
        ptx::mbar_init(TAIL, 1);
        ptx::mbar_init(MMADONE, 1);
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
    const uint32_t tmem = *tmem_slot;
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

    Walker wk;
    wk.init(p, lane);
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
                return __ldg(bt + (p.page_shift >= 0 ? tok >> p.page_shift : tok / P));
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
                    const int slot = n_kv % kSlots;
                    if (n_kv >= kSlots && !wait_all(EMPTY(slot), ((n_kv / kSlots) - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = sb + kRingOff + (uint32_t)slot * kSlot;
                    // a V tile that ends inside a 16-key step is finished here before its release
                    const bool tail = kv == 1 && (nvalid & 15) != 0;
                    const uint32_t bar = tail ? TAIL : FULL(slot);
                    if (lane == 0) ptx::mbar_arrive_expect_tx(bar, (uint32_t)(boxes * box * 256));
                    __syncwarp();
                    if (mine) {
                        const CUtensorMap* map = kv ? &vmap : &kmap;
                        // K and V tiles are read again by the other q tiles of the sequence
                        asm volatile(
                            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                            " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst + (uint32_t)(lane * box) * 128u),
                            "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(it.kvh), "r"(z)
                            : "memory");
                        asm volatile(
                            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                            " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst + kHalf + (uint32_t)(lane * box) * 128u),
                            "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(64), "r"(it.kvh), "r"(z)
                            : "memory");
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
                                    asm volatile(
                                        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx"
                                        "::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                                            sb + kQOff + (uint32_t)(w * kSlot + hf * kHalf)),
                                        "l"(reinterpret_cast<uint64_t>(&qmap)), "r"(QFULL), "r"(hf * 64),
                                        "r"(it.kvh * p.g), "r"(it.tok0 + w * p.tile_tokens)
                                        : "memory");
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
            for (int k = n_kv > kSlots ? n_kv - kSlots : 0; k < n_kv; ++k) drain_bar(FULL(k % kSlots), (k / kSlots) & 1);
            if (n_q > 0) drain_bar(QFULL, (n_q - 1) & 1);
        }
        __syncwarp();
    } else if (warp == 9) {
        /* ================= MMA issuer ================= */
        int n_kv = 0, n_q = 0, n_s[2] = {0, 0};
        bool ok = true;
        auto qk = [&](int w, int slot) {
            const uint32_t qb = sb + kQOff + (uint32_t)w * kSlot, kb = sb + kRingOff + (uint32_t)slot * kSlot;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const uint32_t o = (uint32_t)((ks >> 2) * kHalf + (ks & 3) * 32);
                ptx::tc_mma_f16(tmem + (uint32_t)w * 128u, sdesc(qb + o, 16, 1024), sdesc(kb + o, 16, 1024), idesc(0),
                                ks > 0 ? 1u : 0u);
            }
        };
        auto pv = [&](int w, int slot, int steps, bool first) {
            const uint32_t vb = sb + kRingOff + (uint32_t)slot * kSlot;
            for (int ks = 0; ks < steps; ++ks)
                ptx::tc_mma_f16_ts(tmem + 256u + (uint32_t)w * 128u, tmem + (uint32_t)(w * 128 + ks * 8),
                                   sdesc(vb + (uint32_t)ks * 2048u, kHalf, 1024), idesc(1), (first && ks == 0) ? 0u : 1u);
        };
        while (ok && wk.next(p, lane, it)) {
            const int n = it.t1 - it.t0;
            if (n == 0) continue;
            if (lane == 0) {
                const int last = it.tok0 + p.tile_tokens < it.tok_end ? 1 : 0;  // last active tile
                do {
                    ok = wait_bar(QFULL, n_q & 1) && wait_bar(FULL(n_kv % kSlots), (n_kv / kSlots) & 1);
                    if (!ok) break;
                    ptx::tc_fence_after();
                    for (int w = 0; w <= last; ++w) {
                        qk(w, n_kv % kSlots);
                        ptx::tc_commit(SFULL(w));
                    }
                    ptx::tc_commit(EMPTY(n_kv % kSlots));
                    if (n == 1) ptx::tc_commit(QEMPTY);
                    for (int j = 0; j < n && ok; ++j) {
                        const int kv_v = n_kv + 2 * j + 1, kv_k = kv_v + 1;
                        const int nvalid = min(kTile, it.L - (it.t0 + j) * kTile);
                        for (int w = 0; w <= last; ++w) {
                            ok = wait_bar(PFULL(w), n_s[w] & 1) &&
                                 (w > 0 || wait_bar(FULL(kv_v % kSlots), (kv_v / kSlots) & 1));
                            if (!ok) break;
                            ++n_s[w];
                            ptx::tc_fence_after();
                            pv(w, kv_v % kSlots, (nvalid + 15) >> 4, j == 0);
                            ptx::tc_commit(PVDONE(w));
                            if (w == last) ptx::tc_commit(EMPTY(kv_v % kSlots));
                            if (j + 1 < n) {
                                ok = w > 0 || wait_bar(FULL(kv_k % kSlots), (kv_k / kSlots) & 1);
                                if (!ok) break;
                                ptx::tc_fence_after();
                                qk(w, kv_k % kSlots);
                                ptx::tc_commit(SFULL(w));
                                if (w == last) {
                                    ptx::tc_commit(EMPTY(kv_k % kSlots));
                                    if (j + 2 == n) ptx::tc_commit(QEMPTY);
                                }
                            }
                        }
                    }
                } while (false);
            }
            n_kv += 2 * n;
            ++n_q;
            ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        }
        if (lane == 0) {  // every MMA issued is complete before TMEM is freed
            ptx::tc_commit(MMADONE);
            drain_bar(MMADONE, 0);
        }
        __syncwarp();
    } else {
        /* ================= softmax and output ================= */
        const int w = warp >> 2;
        const int row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = (tmem + (uint32_t)w * 128u) | lanes, tO = (tmem + 256u + (uint32_t)w * 128u) | lanes;
        const int my_tok = row / p.g, my_head = row - my_tok * p.g;
        int n_s = 0;  // key tiles seen by this tile so far
        bool ok = true;
        while (ok && wk.next(p, lane, it)) {
            const int32_t first = it.tok0 + w * p.tile_tokens;
            if (first >= it.tok_end) continue;
            const int32_t tok = first + my_tok;
            const bool valid = row < p.tile_tokens * p.g && tok < it.tok_end;
            const int head = it.kvh * p.g + my_head;
            float m_ref = -INFINITY, l = 0.f;
            for (int32_t tile = it.t0; tile < it.t1; ++tile, ++n_s) {
                if (!wait_all(SFULL(w), n_s & 1)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after();
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) ptx::tc_ld32(tS + 32u * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
                ptx::tc_wait_ld();
                const int32_t nvalid = it.L - tile * kTile;
                if (nvalid < kTile) {
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = i < nvalid ? s[i] : -INFINITY;
                }
                float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < 128; ++i) m4[i & 3] = fmaxf(m4[i & 3], s[i]);
                const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scale_log2;
                const bool raise = mx > m_ref + kLazyLog2;
                if (__any_sync(0xffffffffu, raise)) {
                    const float m_new = raise ? mx : m_ref;
                    const float alpha = raise ? ptx::ex2(m_ref - m_new) : 1.f;
                    m_ref = m_new;
                    l *= alpha;
                    if (tile > it.t0) {
                        if (!wait_all(PVDONE(w), (n_s - 1) & 1)) {
                            ok = false;
                            break;
                        }
                        ptx::tc_fence_after();
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            float o[16];
                            ptx::tc_ld16(tO + 16u * c, o);
                            ptx::tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] *= alpha;
                            ptx::tc_st16(tO + 16u * c, o);
                        }
                    }
                }
                const float base = m_ref == -INFINITY ? 0.f : m_ref;
                float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float a = ptx::ex2(fmaf(s[64 * c + 2 * i], p.scale_log2, -base));
                        const float b = ptx::ex2(fmaf(s[64 * c + 2 * i + 1], p.scale_log2, -base));
                        l4[(2 * i) & 3] += a;
                        l4[(2 * i + 1) & 3] += b;
                        pk[i] = ptx::pack_bf16x2(a, b);
                    }
                    ptx::tc_st32(tS + 32u * c, pk);
                }
                l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                ptx::tc_wait_st();
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(PFULL(w));
            }
            if (!ok) break;
            const bool none = !(it.t1 > it.t0);
            if (!none) {
                if (!wait_all(PVDONE(w), (n_s - 1) & 1)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after();
            }
            // a row whose scores are all -inf has no weight to normalise by
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int64_t at = (int64_t)tok * p.Hq + head;
            const int64_t part = (int64_t)it.split * p.T * p.Hq + at;
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
                if (p.splits == 1) {
                    uint4* dst = reinterpret_cast<uint4*>(p.out + at * 128 + 32 * c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t h[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            h[e] = l == 0.f ? 0u : ptx::pack_bf16x2(__uint_as_float(o[8 * i + 2 * e]) * inv,
                                                                    __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
                        dst[i] = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                } else if (l != 0.f) {
                    float4* dst = reinterpret_cast<float4*>(p.part_o + part * 128 + 32 * c);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        dst[i] = make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv,
                                             __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
                }
            }
            ptx::tc_fence_before();
            if (valid) {
                const float l2 = l == 0.f ? -INFINITY : m_ref + log2f(l);
                if (p.splits > 1) p.part_lse[part] = l2;
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
        ptx::tmem_dealloc(tmem, 512);
    }
}

/* Joins the key ranges of one (token, head) per warp: out = sum_s 2^(l_s - l) O_s with
 * 2^l = sum_s 2^(l_s).  A range without keys has l_s = -inf and no O. */
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t rows = (int64_t)p.T * p.Hq;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int32_t tok = (int32_t)(row / p.Hq), head = (int32_t)(row - (int64_t)tok * p.Hq);
    if (p.cu != nullptr && (tok < __ldg(p.cu) || tok >= __ldg(p.cu + p.B))) return;  // no sequence's
    const float mine = lane < p.splits ? __ldcg(p.part_lse + lane * rows + row) : -INFINITY;
    float m = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // NaN ranges reach the sum through their own weight
    const float base = m == -INFINITY ? 0.f : m;
    const float wgt = mine == -INFINITY ? 0.f : exp2f(mine - base);
    float sum = wgt;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.splits; ++s) {
        const float ws = __shfl_sync(0xffffffffu, wgt, s);
        if (__shfl_sync(0xffffffffu, mine, s) == -INFINITY) continue;
        const float4 o = __ldcg(reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * 128) + lane);
        acc.x = fmaf(ws, o.x, acc.x);
        acc.y = fmaf(ws, o.y, acc.y);
        acc.z = fmaf(ws, o.z, acc.z);
        acc.w = fmaf(ws, o.w, acc.w);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    reinterpret_cast<uint2*>(p.out + row * 128)[lane] =
        make_uint2(ptx::pack_bf16x2(acc.x * inv, acc.y * inv), ptx::pack_bf16x2(acc.z * inv, acc.w * inv));
    if (lane == 0 && p.lse != nullptr) {
        const float l2 = sum == 0.f ? -INFINITY : m + log2f(sum);
        const int32_t b = p.cu ? 0 : tok / p.S;
        p.lse[p.cu ? (int64_t)head * p.T + tok : ((int64_t)b * p.Hq + head) * p.S + (tok - b * p.S)] =
            l2 * 0.6931471805599453f;
    }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

/* (128 dims, heads, tokens) with 64-dimension boxes, 128-byte swizzle; boxes past the end read zeros. */
int encode(CUtensorMap* map, const void* base, int64_t heads, int64_t tokens, int64_t token_stride_bytes,
           int64_t box_heads, int64_t box_tokens) {
    EncodeFn fn = reinterpret_cast<EncodeFn>(host_encode_tiled());
    if (fn == nullptr) return PGQA_ERR_CUDA;
    cuuint64_t dims[3] = {128, (cuuint64_t)heads, (cuuint64_t)tokens};
    cuuint64_t strides[2] = {256, (cuuint64_t)token_stride_bytes};
    cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
    cuuint32_t step[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? PGQA_OK
               : PGQA_ERR_CUDA;
}

/* Key ranges per (sequence, KV head, tile pair).  One as soon as the pairs fill the SMs;
 * else enough to fill them, of at least four key tiles (512 keys) each by the table's
 * capacity, so that an item's fixed cost (its Q tiles, its output) stays below its stream. */
int splits_for(int64_t T, int64_t B, int64_t Hkv, int64_t g, int64_t cap_tokens, int sms) {
    const int64_t per = 2 * (kTile / g);
    int64_t pairs = (T + per - 1) / per;
    if (pairs < B) pairs = B < T ? B : T;  // each sequence with a token has one
    const int64_t items = pairs * Hkv;
    if (items <= 0 || items * 2 > sms) return 1;
    int64_t s = sms / items;
    const int64_t most = cap_tokens / (4 * kTile);
    if (s > most) s = most;
    if (s > kMaxSplits) s = kMaxSplits;
    return s < 1 ? 1 : (int)s;
}

int shape_ok(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t P, int64_t bt_stride) {
    const int st = host_check_pages(B, Hkv, D, P, 1, bt_stride);
    if (st != PGQA_OK) return st;
    if (T < 0 || Hq <= 0 || Hq % Hkv != 0) return PGQA_ERR_BAD_SHAPE;
    if (T > INT32_MAX || Hq / Hkv > kTile || Hq > 65536) return PGQA_ERR_UNSUPPORTED;
    return PGQA_OK;
}

size_t workspace_bytes(int64_t T, int64_t Hq, int splits) {
    return splits > 1 ? (size_t)splits * (size_t)T * (size_t)Hq * (128 + 1) * 4 : 0;
}

int entry(const pgqa_cross_args* a, cudaStream_t stream) {
    if (a == nullptr) return PGQA_ERR_NULL_POINTER;
    if (a->struct_size != sizeof(pgqa_cross_args)) return PGQA_ERR_BAD_SHAPE;
    if (!a->q || !a->k_cache || !a->v_cache || !a->out || !a->seq_lens || !a->block_table)
        return PGQA_ERR_NULL_POINTER;
    int st = shape_ok(a->tokens, a->batch_size, a->num_heads, a->num_heads_k, a->headdim, a->page_size, a->bt_stride);
    if (st != PGQA_OK) return st;
    if (a->num_pages <= 0) return PGQA_ERR_BAD_SHAPE;
    if (a->num_pages >= ((int64_t)1 << 31) / a->page_size) return PGQA_ERR_UNSUPPORTED;
    if (!a->cu_seqlens && (a->seqlen_q < 0 || a->tokens != a->batch_size * a->seqlen_q)) return PGQA_ERR_BAD_SHAPE;
    if (!(a->scale > 0.f) || !isfinite(a->scale)) return PGQA_ERR_BAD_SHAPE;
    if (a->q_stride < a->num_heads * 128) return PGQA_ERR_BAD_SHAPE;
    if (a->q_stride % 8 != 0 || !host_aligned(a->q, 16) || !host_aligned(a->k_cache, 16) ||
        !host_aligned(a->v_cache, 16) || !host_aligned(a->out, 16) || !host_aligned(a->softmax_lse, 4) ||
        !host_aligned(a->seq_lens, 4) || !host_aligned(a->block_table, 4) || !host_aligned(a->cu_seqlens, 4) ||
        !host_aligned(a->workspace, 256))
        return PGQA_ERR_MISALIGNED;
    if (a->q_stride >= ((int64_t)1 << 39)) return PGQA_ERR_UNSUPPORTED;  // a tensor map's stride is 40 bits
    int dev, sms, optin;
    if ((st = host_device(&dev, &sms, &optin)) != PGQA_OK) return st;
    Params p = {};
    if ((st = host_error_word(dev, &p.err)) != PGQA_OK) return st;
    if (a->tokens == 0) return PGQA_OK;
    // items are counted in 32 bits
    if ((a->tokens / (kTile / (a->num_heads / a->num_heads_k)) + a->batch_size) * a->num_heads_k * kMaxSplits > INT32_MAX)
        return PGQA_ERR_UNSUPPORTED;
    p.g = (int32_t)(a->num_heads / a->num_heads_k);
    p.cap_tokens = a->bt_stride * a->page_size;
    p.splits = splits_for(a->tokens, a->batch_size, a->num_heads_k, p.g, p.cap_tokens, sms);
    if (p.splits > 1) {
        const size_t need = workspace_bytes(a->tokens, a->num_heads, p.splits);
        if (a->workspace == nullptr || a->workspace_bytes < need) return PGQA_ERR_WORKSPACE;
        p.part_o = static_cast<float*>(a->workspace);
        p.part_lse = p.part_o + (size_t)p.splits * a->tokens * a->num_heads * 128;
    }
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.lse = a->softmax_lse;
    p.seq_lens = a->seq_lens;
    p.block_table = a->block_table;
    p.cu = a->cu_seqlens;
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
    CUtensorMap qm, km, vm;
    const int64_t slots = a->num_pages * a->page_size;
    if ((st = encode(&qm, a->q, a->num_heads, a->tokens, a->q_stride * 2, p.g, p.tile_tokens)) != PGQA_OK ||
        (st = encode(&km, a->k_cache, a->num_heads_k, slots, a->num_heads_k * 256, 1, p.box)) != PGQA_OK ||
        (st = encode(&vm, a->v_cache, a->num_heads_k, slots, a->num_heads_k * 256, 1, p.box)) != PGQA_OK)
        return st;
    static int done[kHostMaxDevices] = {0};
    if ((st = host_smem_limit(cross_kernel, dev, kSmem, done)) != PGQA_OK) return st;
    const int64_t per = 2 * p.tile_tokens;
    int64_t ctas = (a->tokens / per + a->batch_size) * a->num_heads_k * p.splits;  // at least the items
    if (ctas > sms) ctas = sms;
    st = host_launch(cross_kernel, dim3((unsigned)ctas), kThreads, kSmem, stream, 1, qm, km, vm, p);
    if (st != PGQA_OK || p.splits == 1) return st;
    return host_launch(join_kernel, dim3((unsigned)((a->tokens * a->num_heads + 7) / 8)), 256, 0, stream, 1, p);
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
    return cross::workspace_bytes(tokens, num_heads,
                                  cross::splits_for(tokens, batch_size, num_heads_k, num_heads / num_heads_k,
                                                    bt_stride * page_size, sms));
}

extern "C" int pgqa_cross_attention(const pgqa_cross_args* args, void* stream) {
    return pgqa::host_set_status(pgqa::cross::entry(args, static_cast<cudaStream_t>(stream)));
}
