// Causal attention over whole prompts: any length, grouped heads, packed sequences.
//
// Query-tile stationary like tile_fwd.cu, whose schedule it shares (two softmax groups on alternating key blocks, separate issue of
// S = Q K^T and O += P V, P in tensor memory over S, three S buffers), with the tile laid out for what prompts look like: its 128 rows are
// all heads of one KV head times 128 / group consecutive tokens (one TMA box), so that K and V are fetched once for the whole group, a
// tile of a short prompt is full from 128 / group tokens on, and tiles, like key blocks, begin at their sequence's first token wherever
// that lies.  A first kernel lists the tiles, those that visit most key blocks first, from boundaries in device memory; persistent CTAs
// draw (tile, KV head) from it.
//
// Values that no row of a tile sees - later tokens, the next sequence, whatever lies behind the last one - must not reach it, not as
// 0 * NaN either.  A tile is first done as if there were none that is not finite.  Where a result is not finite the tile is done once more,
// carefully: where the causal edge crosses a block, the group that turns its scores into probabilities first clears V's rows behind the
// tile's last token in shared memory, sets values that are not finite to zero in the others, and they are added, after the last block, to
// the rows that do see them.  (Every tile done carefully: B=1 S=8100 Hq=20 Hkv=4 as eleven sequences 72 us, first like this 65.)
//
// Two groups of softmax warps pass an item's key blocks to one another; four more warps write its rows while the groups are at the next item
// (one of the groups did before: 56 us for those eleven sequences, 53.3 now, 660 TFLOP/s).  S=8192 Hq=32 Hkv=8: 440 us alone, 1.25 PFLOP/s, 504 back to
// back at 1.57 GHz (power); 333 tokens as five sequences 9.4 us, one launch.  Bound by exponentials and issue beside them (a block of
// 128 keys takes a group about 2900 cycles: 400 for the maximum, 400 to 500 for the hand-over, 1600 to 2250 for exponentials and stores), and, with
// few key blocks to an item, by the first block of the next item.
#include "host_common.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace fmsa {
namespace {

struct PromptParams {
    const int32_t* cu;          // [n_seqs + 1], or [B][n_seqs + 1], or null
    const float* sinks;         // [Hq] or null
    const __nv_bfloat16* v;     // (B,Hkv,S,128)
    int64_t vs[3];
    __nv_bfloat16* out;         // [B][S][Hq*128]
    int32_t* counter;           // next item; behind it the number of tiles
    int4* tiles;                // [cap]: batch element, first token, tokens, first token of the sequence
    int32_t* status;
    int32_t B, S, Hq, Hkv, group, tokens, n_seqs, per_batch, cap, shift;   // tokens: of a full tile
    int32_t direct;             // CTA u does item u: there is no list
    float scale_log2e;
};

constexpr int kPlanThreads = 1024, kPlanBins = 2048;

__device__ __forceinline__ void sequence_of(const PromptParams& P, int b, int i, int& lo, int& hi) {
    lo = 0;
    hi = P.S;
    if (P.cu) {
        const int32_t* cu = P.cu + (P.per_batch ? static_cast<int64_t>(b) * (P.n_seqs + 1) : 0);
        lo = min(max(cu[i], 0), P.S);
        hi = min(max(cu[i + 1], lo), P.S);
    }
}

// Whether boundaries rise (where they do not, rows can be nobody's or two sequences'): thread `at` of `threads`.
__device__ __forceinline__ void check_boundaries(const PromptParams& P, int at, int threads) {
    for (int b = 0; b < (P.per_batch ? P.B : 1); ++b)
        for (int i = at; i < P.n_seqs; i += threads)
            if (bad_boundaries(P.cu + static_cast<int64_t>(b) * (P.n_seqs + 1), i, P.S)) atomicMax(P.status, kStatusBadIndex);
}

// Sets the rows behind the last sequences to zero: thread `at` of `threads`.
__device__ __forceinline__ void clear_tails(const PromptParams& P, int64_t at, int64_t threads) {
    for (int b = 0; b < P.B; ++b) {
        int lo, hi;
        sequence_of(P, b, P.n_seqs - 1, lo, hi);
        const int64_t row = static_cast<int64_t>(P.Hq) * 16;   // 16-byte pieces
        uint4* to = reinterpret_cast<uint4*>(P.out) + (static_cast<int64_t>(b) * P.S + hi) * row;
        for (int64_t i = at; i < (P.S - hi) * row; i += threads) to[i] = make_uint4(0, 0, 0, 0);
    }
}

// Block 0 lists the tiles, by a counting sort on the key blocks they visit; the others set the rows behind the last sequences to zero.
__global__ void __launch_bounds__(kPlanThreads) prompt_plan_kernel(const PromptParams P) {
    __shared__ uint32_t bins[kPlanBins], sums[32];
    wait_for_previous_kernel();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (blockIdx.x > 0) {
        const int at = (blockIdx.x - 1) * kPlanThreads + tid, threads = (gridDim.x - 1) * kPlanThreads;
        clear_tails(P, at, threads);
        check_boundaries(P, at, threads);
        return;
    }
    for (int i = tid; i < kPlanBins; i += kPlanThreads) bins[i] = 0;
    __syncthreads();
    const int pairs = P.B * P.n_seqs;
    auto each = [&](auto&& what) {   // what(batch element, first token, tokens, the sequence's first token, bin)
        for (int p = warp; p < pairs; p += kPlanThreads / 32) {
            const int b = p / P.n_seqs;
            int lo, hi;
            sequence_of(P, b, p - b * P.n_seqs, lo, hi);
            for (int at = lo + lane * P.tokens; at < hi; at += 32 * P.tokens) {
                const int n = min(P.tokens, hi - at);
                what(b, at, n, lo, (at + n - lo + kBlock - 1) / kBlock >> P.shift);
            }
        }
    };
    each([&](int, int, int, int, int bin) { atomicAdd(&bins[bin], 1u); });
    __syncthreads();
    // where each bin begins: thread i has the two bins from the top
    const uint32_t b0 = bins[kPlanBins - 1 - 2 * tid], b1 = bins[kPlanBins - 2 - 2 * tid];
    uint32_t sum = b0 + b1;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    uint32_t before = sum - b0 - b1;
    for (int w = 0; w < warp; ++w) before += sums[w];
    bins[kPlanBins - 1 - 2 * tid] = before;
    bins[kPlanBins - 2 - 2 * tid] = before + b0;
    if (tid == kPlanThreads - 1) {
        const uint32_t all = before + b0 + b1;
        // (more than `cap` where boundaries fall, which the other blocks report)
        P.counter[0] = 0;
        P.counter[1] = static_cast<int32_t>(min(all, static_cast<uint32_t>(P.cap)));
    }
    __syncthreads();
    each([&](int b, int at, int n, int lo, int bin) {
        const uint32_t to = atomicAdd(&bins[bin], 1u);
        if (to < static_cast<uint32_t>(P.cap)) P.tiles[to] = make_int4(b, at, n, lo);
    });
}

struct PromptItem {
    int32_t b, head, row0, count;   // batch element, KV head, first token, tokens
    int32_t lo;                     // first token of the sequence
    int32_t steps;                  // visited key blocks; < 0: no more work
    int32_t careful;
    // 32-key pieces of the first visited block (the last of the sequence) that the tile sees
    __device__ __forceinline__ int pieces() const { return (row0 + count - lo - (steps - 1) * kBlock + 31) >> 5; }
};

constexpr int kPrKvStages = 5, kPrBuffers = 3, kPrRing = 4;
constexpr int kPrThreads = 4 * 128;
// Registers per thread after the warpgroups re-divide the register file: 512 threads are launched with 128.
constexpr int kPrRegsLaunch = 128, kPrRegsSoftmax = 176, kPrRegsRows = 104, kPrRegsMisc = 56;
static_assert(2 * kPrRegsSoftmax + kPrRegsRows + kPrRegsMisc <= 4 * kPrRegsLaunch, "register re-division must balance");
static_assert(kPrRegsLaunch == (65536 / kPrThreads) / 8 * 8, "registers per thread at launch");

struct PromptCtrl {
    uint64_t q_full, q_empty, kv_full[kPrKvStages], kv_empty[kPrKvStages];
    uint64_t s_full[kPrBuffers], p_full[kPrBuffers][2], pv_done[kPrBuffers];   // p_full: [half of the keys]
    uint64_t chain[2][4];                        // [group][quarter]
    uint64_t sum_full[kPrRing], o_free;
    uint64_t item_full[kPrRing], item_empty[kPrRing];
    PromptItem items[kPrRing];
    uint32_t odd[kPrRing][2][4];                 // careful: keys of the item's first two blocks that hold a value that is not finite
    uint32_t again[kPrRing];                     // a result of the item is not finite
    float top[128];                              // running maximum of every row (log2 domain)
    float2 part[kPrRing][2][128];                // [group] (max, sum) at the end of an item
    uint32_t tmem_slot;
};
constexpr size_t kPrTileBytes = static_cast<size_t>(1 + kPrKvStages) * kTileBytes;
constexpr int kPrStaging = 32 * 64;              // of a warp: 32 columns of its rows on their way out
constexpr size_t kPrSmemBytes = kPrTileBytes + 4 * kPrStaging + 1024 + sizeof(PromptCtrl);
static_assert(kPrSmemBytes <= 232448, "shared memory budget of one CTA");

// As in tile_fwd.cu: rows whose maximum grows by less than this (log2) keep the old one; fp16 P are 2^7 times larger.
constexpr float kPrLazyRescale = 8.f;
template <bool FP16>
constexpr float kPrLiftP = FP16 ? 7.f : 0.f;

template <bool FP16>
__device__ __forceinline__ uint32_t times_zero(uint32_t w, uint32_t acc) {   // acc (+0 or NaN pairs) + w * 0: NaN where w is not finite
    if (FP16) {
        const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0)), *reinterpret_cast<const __half2*>(&acc));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w), __bfloat162bfloat162(__ushort_as_bfloat16(0)),
                                     *reinterpret_cast<const __nv_bfloat162*>(&acc));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <bool FP16>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {   // halves that are not finite become zero
    constexpr uint32_t e = FP16 ? 0x7c00u : 0x7f80u;
    if ((w & e) == e) w &= 0xffff0000u;
    if ((w & e << 16) == e << 16) w &= 0xffffu;
    return w;
}

// K and V tiles pass through one ring in the order K_0 K_1 K_2 V_0 K_3 V_1 ..
template <bool FP16>
__global__ void __launch_bounds__(kPrThreads, 1) prompt_fwd_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                                                                   const __grid_constant__ CUtensorMap tmap_v, const PromptParams P) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t tile_q = tiles, tile_kv = tiles + kTileBytes;
    PromptCtrl* sm = reinterpret_cast<PromptCtrl*>(smem_raw + (tiles - smem_u32(smem_raw)) + kPrTileBytes + 4 * kPrStaging);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    auto BAR = [&](uint64_t& b) { return smem_u32(&b); };

    if (tid == 0) {
        mbar_init(BAR(sm->q_full), 1);
        mbar_init(BAR(sm->q_empty), 1);
        mbar_init(BAR(sm->o_free), 4);
        for (int i = 0; i < 8; ++i) mbar_init(BAR(sm->chain[i >> 2][i & 3]), 1);
        for (int i = 0; i < kPrBuffers; ++i) {
            mbar_init(BAR(sm->s_full[i]), 1);
            mbar_init(BAR(sm->p_full[i][0]), 4);
            mbar_init(BAR(sm->p_full[i][1]), 4);
            mbar_init(BAR(sm->pv_done[i]), 1);
        }
        for (int i = 0; i < kPrKvStages; ++i) {
            mbar_init(BAR(sm->kv_full[i]), 1);
            mbar_init(BAR(sm->kv_empty[i]), 1);
        }
        for (int i = 0; i < kPrRing; ++i) {
            mbar_init(BAR(sm->item_full[i]), 1);
            mbar_init(BAR(sm->item_empty[i]), 15);   // loads, issue (2), eight softmax warps, four that write rows
            mbar_init(BAR(sm->sum_full[i]), 8);
        }
        fence_mbar_init();
        prefetch_tmap(&tmap_q);
        prefetch_tmap(&tmap_k);
        prefetch_tmap(&tmap_v);
    }
    // (rows of the query tile that no token has - 128 is not always a multiple of the group - are zero for good)
    for (int i = tid; i < kTileBytes / 16; i += kPrThreads) st_shared_v4(tile_q + 16 * i, 0, 0, 0, 0);
    fence_async_smem();
    if (warp == 0) {
        tmem_alloc(smem_u32(&sm->tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    constexpr uint32_t tmem = 0, tmem_o = 128 * kPrBuffers;   // all 512 columns: the allocation starts at column 0
    if (sm->tmem_slot != tmem) {
        wait_for_previous_kernel();
        if (tid == 0) atomicMax(P.status, kStatusBadSmem);
        __syncthreads();
        if (warp == 0) tmem_dealloc(sm->tmem_slot, 512);
        return;
    }
    wait_for_previous_kernel();

    bool bad = false;   // a bounded wait gave up (here or in another role): the thread stops taking work
    auto wait = [&](uint32_t bar, uint32_t parity) {   // every lane of the warp calls it; the result is warp-uniform
        if (!bad) bad = __any_sync(0xffffffffu, !mbar_wait_role(bar, parity));
    };
    auto wait1 = [&](uint32_t bar, uint32_t parity) {   // the same in a role that a single thread runs
        if (!bad) bad = !mbar_wait_role(bar, parity);
    };
    auto warp_arrive = [&](uint32_t bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    if (warp >= 12) {
        reg_dec<kPrRegsMisc>();
        if (warp == 14) {
            // =========================== items ===========================
            uint32_t n_items = 0, draw = 0;
            int4 tile = make_int4(0, 0, 0, 0);   // direct: this CTA's
            if (!P.direct) {
                n_items = static_cast<uint32_t>(P.counter[1]) * P.Hkv;
            } else {
                const int wanted = blockIdx.x / P.Hkv, pairs = P.B * P.n_seqs;
                for (int p0 = 0, before = 0; p0 < pairs && before <= wanted; p0 += 32) {
                    const int p = p0 + lane, b = p / P.n_seqs;
                    int lo = 0, hi = 0;
                    if (p < pairs) sequence_of(P, b, p - b * P.n_seqs, lo, hi);
                    const int n = (hi - lo + P.tokens - 1) / P.tokens;
                    int upto = n;
                    for (int o = 1; o < 32; o <<= 1) {
                        const int v = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += v;
                    }
                    const int mine = wanted - (before + upto - n);
                    const uint32_t who = __ballot_sync(0xffffffffu, mine >= 0 && mine < n);
                    if (who) {
                        const int at = lo + mine * P.tokens, from = __ffs(who) - 1;
                        tile = make_int4(__shfl_sync(0xffffffffu, b, from), __shfl_sync(0xffffffffu, at, from),
                                         __shfl_sync(0xffffffffu, min(P.tokens, hi - at), from), __shfl_sync(0xffffffffu, lo, from));
                        n_items = 1;
                        break;
                    }
                    before += __shfl_sync(0xffffffffu, upto, 31);
                }
            }
            auto publish = [&](const PromptItem& it) {   // (lane 0 has it)
                const uint32_t slot = draw++ % kPrRing;
                if (lane == 0) {
                    sm->items[slot] = it;
                    sm->again[slot] = 0;
                    for (int i = 0; i < 8; ++i) sm->odd[slot][i >> 2][i & 3] = 0;
                }
                warp_arrive(BAR(sm->item_full[slot]));
            };
            auto finished = [&](uint32_t d) { wait(BAR(sm->item_empty[d % kPrRing]), (d / kPrRing) & 1); };
            for (bool more = true; more;) {
                if (draw >= kPrRing) finished(draw - kPrRing);
                if (bad) break;
                PromptItem it = {};
                if (lane == 0) {
                    it = sm->items[draw % kPrRing];
                    if (draw >= kPrRing && sm->again[draw % kPrRing]) {
                        it.careful = 1;
                    } else {
                        it = {};
                        it.steps = -1;
                        const uint32_t u = P.direct ? draw : static_cast<uint32_t>(atomicAdd(P.counter, 1));
                        if (u < n_items) {
                            const int4 t = P.direct ? tile : P.tiles[u / P.Hkv];
                            it.b = t.x;
                            it.head = static_cast<int>(P.direct ? blockIdx.x % P.Hkv : u % P.Hkv);
                            it.row0 = t.y;
                            it.count = t.z;
                            it.lo = t.w;
                            it.steps = (t.y + t.z - t.w + kBlock - 1) / kBlock;
                        }
                    }
                }
                more = __shfl_sync(0xffffffffu, it.steps, 0) >= 0;
                if (more) publish(it);
                if (more && draw == 1 && P.direct && P.cu) clear_tails(P, blockIdx.x * 32 + lane, static_cast<int64_t>(gridDim.x) * 32);
            }
            if (draw == 0 && P.direct && P.cu) clear_tails(P, blockIdx.x * 32 + lane, static_cast<int64_t>(gridDim.x) * 32);
            // the items still worked on (in the other slots), those of them that are done again, and the end
            PromptItem last[kPrRing - 1] = {};
            const uint32_t drawn = draw;
#pragma unroll
            for (uint32_t i = 1; i < kPrRing; ++i) {
                if (drawn < i || bad) continue;
                finished(drawn - i);
                const uint32_t slot = (drawn - i) % kPrRing;
                if (!bad && sm->again[slot]) last[i - 1] = sm->items[slot];
            }
            __syncwarp();
#pragma unroll
            for (uint32_t i = 1; i < kPrRing; ++i) {
                last[i - 1].careful = 1;
                if (last[i - 1].steps > 0 && !bad) publish(last[i - 1]);
            }
            PromptItem none = {};
            none.steps = -1;
            if (!bad) publish(none);
            if (P.direct && P.cu) check_boundaries(P, blockIdx.x * 32 + lane, gridDim.x * 32);
        } else if (warp == 12 && elect_one()) {
            // =========================== tile loads ===========================
            uint32_t st = 0, ph = 1, items = 0;   // stage of the ring, phase bit of its kv_empty, items so far
            for (uint32_t draw = 0;; ++draw, ++items) {
                const uint32_t slot = draw % kPrRing;
                wait1(BAR(sm->item_full[slot]), (draw / kPrRing) & 1);
                if (bad) break;
                const PromptItem it = sm->items[slot];
                if (it.steps < 0) break;
                for (int t = -kPrBuffers; t < it.steps && !bad; ++t) {
#pragma unroll 1
                    for (int v = 1; v >= 0; --v) {   // V of step t, K of step t + 3
                        const int k = v ? t : t + kPrBuffers;
                        if (k < 0 || k >= it.steps) continue;
                        wait1(BAR(sm->kv_empty[st]), ph);   // (the first round finds every stage free)
                        if (bad) break;
                        mbar_arrive_expect_tx(BAR(sm->kv_full[st]), kTileBytes);
                        tma_load_tile(tile_kv + st * kTileBytes, v ? &tmap_v : &tmap_k, it.lo + (it.steps - 1 - k) * kBlock, it.head, it.b, BAR(sm->kv_full[st]));
                        if (++st == kPrKvStages) {
                            st = 0;
                            ph ^= 1;
                        }
                    }
                    if (t == -kPrBuffers) {
                        if (items > 0) wait1(BAR(sm->q_empty), (items - 1) & 1);
                        if (bad) break;
                        mbar_arrive_expect_tx(BAR(sm->q_full), 256u * P.group * P.tokens);
                        for (int p = 0; p < 2; ++p)
                            tma_load_4d(tile_q + p * kPanelBytes, &tmap_q, 64 * p, it.head * P.group, it.row0, it.b, BAR(sm->q_full));
                    }
                }
                mbar_arrive(BAR(sm->item_empty[slot]));
            }
        } else if ((warp == 13 || warp == 15) && elect_one()) {
            // =========================== S (warp 13) and P V (warp 15) ===========================
            const bool pv = warp == 15;
            uint32_t st0 = 0, ph0 = 0;       // ring position (stage, phase bit) of the item's first tile
            uint32_t buf = 0, bph = 0;       // S buffer and its phase bit
            for (uint32_t draw = 0;; ++draw) {
                const uint32_t slot = draw % kPrRing;
                wait1(BAR(sm->item_full[slot]), (draw / kPrRing) & 1);
                if (bad) break;
                const int steps = sm->items[slot].steps, pieces = sm->items[slot].pieces();
                if (steps < 0) break;
                if (!pv) wait1(BAR(sm->q_full), draw & 1);
                // position of K_t: t, and one for every V before it (V_u comes before K_{u + 3}); of V_t: the K up to t + 2 and the V before it
                uint32_t st = st0, ph = ph0;
                auto skip = [&](uint32_t n) {   // n <= kPrKvStages
                    st += n;
                    if (st >= kPrKvStages) {
                        st -= kPrKvStages;
                        ph ^= 1;
                    }
                };
                if (pv) skip(min(steps, kPrBuffers));
#pragma unroll 1
                for (int t = 0; t < steps && !bad; ++t) {
                    const uint32_t at = tile_kv + st * kTileBytes, sbuf = tmem + 128 * buf;
                    if (!pv) {
                        wait1(BAR(sm->kv_full[st]), ph);
                        wait1(BAR(sm->pv_done[buf]), bph ^ 1);   // (the first round finds every buffer free)
                        if (bad) break;
                        tc_fence_after_sync();
                        umma_tile_128<false, false, FP16>(sbuf, tile_q, at, false);   // S = Q K_j^T
                        umma_commit(BAR(sm->s_full[buf]));
                        umma_commit(BAR(sm->kv_empty[st]));
                        skip(t + 1 < kPrBuffers ? 1 : 2);
                    } else {
                        wait1(BAR(sm->p_full[buf][0]), bph);
                        wait1(BAR(sm->kv_full[st]), ph);
                        // the first product of an item overwrites O: the rows of the item before must have been read
                        if (t == 0 && draw > 0) wait1(BAR(sm->o_free), (draw - 1) & 1);
                        if (bad) break;
                        tc_fence_after_sync();
                        // O += P V_j, of the first block the keys that are seen
                        const bool part = t == 0 && pieces < 4;
                        if (part && pieces == 1) umma_ts<2, 8, FP16>(tmem_o, sbuf, at, false);
                        else umma_ts<4, 8, FP16>(tmem_o, sbuf, at, t > 0);
                        wait1(BAR(sm->p_full[buf][1]), bph);
                        if (bad) break;
                        tc_fence_after_sync();
                        if (!part) umma_ts<4, 8, FP16>(tmem_o, sbuf + 32, at + 64 * 128, true);
                        else if (pieces == 3) umma_ts<2, 8, FP16>(tmem_o, sbuf + 32, at + 64 * 128, true);
                        umma_commit(BAR(sm->pv_done[buf]));
                        umma_commit(BAR(sm->kv_empty[st]));
                        skip(t + kPrBuffers < steps ? 2 : 1);
                    }
                    if (++buf == kPrBuffers) {
                        buf = 0;
                        bph ^= 1;
                    }
                }
                if (bad) break;
                if (!pv) umma_commit(BAR(sm->q_empty));
                st0 += 2 * steps;
                ph0 ^= st0 / kPrKvStages & 1;
                st0 %= kPrKvStages;
                mbar_arrive(BAR(sm->item_empty[slot]));
            }
        }
    } else if (warp >= 8) {
        reg_dec<kPrRegsRows>();
        // =========================== rows on their way out ===========================
        const int tok = row / P.group, hh = row - tok * P.group;   // (rows behind the last whole token: tok >= P.tokens)
        uint32_t done = 0;               // steps so far
        for (uint32_t draw = 0;; ++draw) {
            const uint32_t slot = draw % kPrRing;
            wait(BAR(sm->item_full[slot]), (draw / kPrRing) & 1);
            if (bad) break;
            const PromptItem it = sm->items[slot];
            if (it.steps < 0) break;
            done += it.steps;
            const int ahead = it.row0 - it.lo;
            const bool careful = it.careful;
            wait(BAR(sm->sum_full[slot]), (draw / kPrRing) & 1);
            if (bad) break;
            const float2 a = sm->part[slot][0][row], b = sm->part[slot][1][row];
            const float m = fmaxf(a.x, b.x);   // (maxima only rise: the one of the group that had the last step)
            float l = (a.x == -INFINITY ? 0.f : a.y * fast_exp2(a.x - m)) + (b.x == -INFINITY ? 0.f : b.y * fast_exp2(b.x - m));
            const int head = it.head * P.group + hh;
            const bool real = tok < it.count && tok < P.tokens;
            if (P.sinks && real) l += fast_exp2(P.sinks[head] * kLog2e + (m == -INFINITY ? 0.f : kPrLiftP<FP16> - m));
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const float2 inv2 = make_float2(inv, inv);
            wait(BAR(sm->pv_done[(done - 1) % kPrBuffers]), (done - 1) / kPrBuffers & 1);
            if (bad) break;
            tc_fence_after_sync();
            __nv_bfloat16* to = P.out + (static_cast<int64_t>(it.b) * P.S + it.row0 + tok) * (static_cast<int64_t>(P.Hq) * kHeadDim) +
                                static_cast<int64_t>(head) * kHeadDim;
            // Rows leave through shared memory, 32 columns at a time, so that four lanes write 64 bytes of a row: a lane with a row of its
            // own wrote 16 bytes here and there and took 4000 cycles a tile, 2600 this way.
            const uint32_t staged = tiles + kPrTileBytes + quarter * kPrStaging;
            int64_t out_of[4];               // where this lane's pieces of rows 8 i + lane / 4 go, or -1
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t at = real ? to - P.out : -1;
                out_of[i] = __shfl_sync(0xffffffffu, at, 8 * i + (lane >> 2));
            }
            uint32_t finite = 0;             // 0 or NaN
            uint32_t o[2][32];
            tmem_ld32(tmem_addr(tmem_o, quarter, 0), o[0]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {    // (the columns after these are on their way meanwhile)
                tmem_ld_wait();
                if (c < 3) {
                    tmem_ld32(tmem_addr(tmem_o, quarter, 32 * c + 32), o[(c + 1) & 1]);
                } else {
                    tc_fence_before_sync();
                    warp_arrive(BAR(sm->o_free));
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    uint32_t pk[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float2 r = f2_mul(f2_from_bits(o[c & 1][8 * y + 2 * z], o[c & 1][8 * y + 2 * z + 1]), inv2);
                        pk[z] = pack_act<FP16>(r.x, r.y);
                        finite = times_zero<FP16>(pk[z], finite);
                    }
                    st_shared_v4(staged + lane * 64 + ((y ^ (lane >> 1 & 3)) << 4), pk[0], pk[1], pk[2], pk[3]);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 8 * i + (lane >> 2);
                    const uint4 x = ld_shared_v4(staged + r * 64 + (((lane & 3) ^ (r >> 1 & 3)) << 4));
                    if (out_of[i] >= 0) *reinterpret_cast<uint4*>(P.out + out_of[i] + 32 * c + 8 * (lane & 3)) = x;
                }
                __syncwarp();
            }
            if (!careful && __any_sync(0xffffffffu, real && (finite & 0x7fff7fffu)) && lane == 0) sm->again[slot] = 1;
            // values that are not finite, for the rows that see them (what they were multiplied with does not matter)
#pragma unroll 1
            for (int t = 0; careful && t < 2; ++t) {
#pragma unroll 1
                for (int w = 0; w < 4; ++w) {
#pragma unroll 1
                    for (uint32_t odd = sm->odd[slot][t][w]; odd; odd &= odd - 1) {
                        const int key = (it.steps - 1 - t) * kBlock + 32 * w + __ffs(odd) - 1;
                        if (!real || key > ahead + tok) continue;
                        const __nv_bfloat16* from = P.v + it.b * P.vs[0] + it.head * P.vs[1] + (it.lo + key) * P.vs[2];
#pragma unroll 1
                        for (int c = 0; c < 128; c += 2) {
                            const uint32_t x = *reinterpret_cast<const uint32_t*>(from + c), y = *reinterpret_cast<const uint32_t*>(to + c);
                            const float x0 = act_lo<FP16>(x), x1 = act_hi<FP16>(x);
                            const float y0 = act_lo<FP16>(y) + (isfinite(x0) ? 0.f : x0), y1 = act_hi<FP16>(y) + (isfinite(x1) ? 0.f : x1);
                            *reinterpret_cast<uint32_t*>(to + c) = pack_act<FP16>(y0, y1);
                        }
                    }
                }
            }
            warp_arrive(BAR(sm->item_empty[slot]));
        }
    } else {
        reg_inc<kPrRegsSoftmax>();
        // =========================== softmax ===========================
        // Thread = row.  The running maximum of a row is handed from group to group, step by step; either group sums the P of its own
        // steps.  At the end of an item both leave their sums to the warps that write its rows.
        const int g = warp >> 2;
        const uint32_t chain_in = BAR(sm->chain[g ^ 1][quarter]), chain_out = BAR(sm->chain[g][quarter]);
        const float2 sc2 = make_float2(P.scale_log2e, P.scale_log2e);
        const int tok = row / P.group;   // (rows behind the last whole token: tok >= P.tokens)
        uint32_t step = 0;               // steps so far
        uint32_t buf = 0, bph = 0;       // S buffer and its phase bit
        uint32_t last = 0, last_ph = 0;  // S buffer of the step before, its phase bit
        uint32_t ring = 0;               // ring position (stage + 5 * phase bit) of the item's first tile
        for (uint32_t draw = 0;; ++draw) {
            const uint32_t slot = draw % kPrRing;
            wait(BAR(sm->item_full[slot]), (draw / kPrRing) & 1);
            if (bad) break;
            const int steps = sm->items[slot].steps;
            if (steps < 0) break;
            const int ahead = sm->items[slot].row0 - sm->items[slot].lo, count = sm->items[slot].count;   // tokens before the tile; its own
            const bool careful = sm->items[slot].careful;
            float m = -INFINITY, l = 0.f;   // running maximum (log2 domain), and this group's sum relative to it
            const uint32_t prev = last, prev_ph = last_ph;   // of the last step of the item before
#pragma unroll 1
            for (int t = 0; t < steps; ++t, ++step) {
                if ((step & 1) == static_cast<uint32_t>(g)) {
                    const uint32_t ts = tmem + 128 * buf;
                    const int first = (steps - 1 - t) * kBlock;        // the block's first key in the sequence
                    const bool edge = first + kBlock > ahead + 1;      // (the tile's first row does not see all of it)
                    wait(BAR(sm->s_full[buf]), bph);
                    if (edge && careful) {
                        // V before it is multiplied: rows behind the tile's last token become zero, values that are not finite too.  (A stage
                        // is waited for when what it held before has come: this item's first K with S, the V of the item before with its
                        // last product.  Before that the barrier's phase bit would still mean the use before.)
                        if (draw > 0) wait(BAR(sm->pv_done[prev]), prev_ph);
                        const uint32_t at = (ring + t + min(steps, t + kPrBuffers)) % (2 * kPrKvStages);
                        wait(BAR(sm->kv_full[at % kPrKvStages]), at / kPrKvStages);
                        if (bad) break;
                        const uint32_t vrow = tile_kv + (at % kPrKvStages) * kTileBytes + row * 128;
                        if (first + row >= ahead + count) {
#pragma unroll 4
                            for (int i = 0; i < 16; ++i) st_shared_v4(vrow + (i >> 3) * kPanelBytes + ((i + row & 7) << 4), 0, 0, 0, 0);
                        } else {
                            uint32_t acc = 0;
#pragma unroll 4
                            for (int i = 0; i < 16; ++i) {
                                const uint4 x = ld_shared_v4(vrow + (i >> 3) * kPanelBytes + ((i + row & 7) << 4));
                                acc = times_zero<FP16>(x.w, times_zero<FP16>(x.z, times_zero<FP16>(x.y, times_zero<FP16>(x.x, acc))));
                            }
                            if (acc & 0x7fff7fffu) {
#pragma unroll 1
                                for (int i = 0; i < 16; ++i) {
                                    const uint32_t p = vrow + (i >> 3) * kPanelBytes + ((i + row & 7) << 4);
                                    const uint4 x = ld_shared_v4(p);
                                    st_shared_v4(p, finite_only<FP16>(x.x), finite_only<FP16>(x.y), finite_only<FP16>(x.z), finite_only<FP16>(x.w));
                                }
                                atomicOr(&sm->odd[slot][t][quarter], 1u << lane);
                            }
                        }
                        fence_async_smem();
                    }
                    if (bad) break;
                    tc_fence_after_sync();
                    const int seen = t == 0 ? (ahead + count - first + 31) >> 5 : 4;   // pieces of 32 keys that the tile sees
                    if (edge) {   // logits that one row sees and another does not become -inf where they are hidden
                        const int limit = ahead + tok - first;
#pragma unroll 1
                        for (int c = max(ahead - first + 1, 0) & ~15; c < 32 * seen; c += 16) {
                            uint32_t v[16];
                            tmem_ld16(tmem_addr(ts, quarter, c), v);
                            tmem_ld_wait();
#pragma unroll
                            for (int y = 0; y < 16; ++y)
                                if (c + y > limit) v[y] = 0xff800000u;
                            tmem_st16(tmem_addr(ts, quarter, c), v);
                        }
                        tmem_st_wait();
                    }
                    uint32_t s[4][32];
                    float mx0 = -INFINITY, mx1 = -INFINITY;
                    tmem_ld32(tmem_addr(ts, quarter, 0), s[0]);
                    tmem_ld32(tmem_addr(ts, quarter, 32), s[1]);
                    tmem_ld_wait();
                    tmem_ld32(tmem_addr(ts, quarter, 64), s[2]);
                    tmem_ld32(tmem_addr(ts, quarter, 96), s[3]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (c == 2) tmem_ld_wait();
                        if (c >= seen) continue;
#pragma unroll
                        for (int y = 0; y < 32; y += 4) {
                            mx0 = fmax3(mx0, __uint_as_float(s[c][y]), __uint_as_float(s[c][y + 1]));
                            mx1 = fmax3(mx1, __uint_as_float(s[c][y + 2]), __uint_as_float(s[c][y + 3]));
                        }
                    }
                    const float mt = fmaxf(mx0, mx1) * P.scale_log2e;   // raw logits: scale > 0, so the maximum commutes with it
                    if (step) wait(chain_in, g ? (step >> 1) & 1 : ((step >> 1) - 1) & 1);
                    if (bad) break;
                    const float top = t > 0 ? sm->top[row] : -INFINITY;   // the row's maximum so far
                    const bool any_raise = __any_sync(0xffffffffu, mt > top + kPrLazyRescale);
                    const float mn = any_raise ? fmaxf(top, mt) : top;
                    if (any_raise || t == 0) sm->top[row] = mn;
                    warp_arrive(chain_out);
                    if (mn != m) {   // (raised here or by the other group)
                        l *= m == -INFINITY ? 0.f : fast_exp2(m - mn);
                        m = mn;
                    }
                    if (any_raise && t > 0) {
                        // the product of the step before may still be adding to O
                        wait(BAR(sm->pv_done[last]), last_ph);
                        if (bad) break;
                        tc_fence_after_sync();
                        const float alpha = top == -INFINITY ? 0.f : fast_exp2(top - mn);
                        const float2 a2 = make_float2(alpha, alpha);
#pragma unroll 1
                        for (int c = 0; c < 128; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(tmem_addr(tmem_o, quarter, c), o);
                            tmem_ld_wait();
#pragma unroll
                            for (int y = 0; y < 16; y += 2) {
                                const float2 r = f2_mul(f2_from_bits(o[y], o[y + 1]), a2);
                                o[y] = __float_as_uint(r.x);
                                o[y + 1] = __float_as_uint(r.y);
                            }
                            tmem_st16(tmem_addr(tmem_o, quarter, c), o);
                        }
                    }
                    const float nm = m == -INFINITY ? 0.f : kPrLiftP<FP16> - m;   // (a row that has not seen anything yet)
                    const float2 nm2 = make_float2(nm, nm);
                    float2 l2a = make_float2(0.f, 0.f), l2b = make_float2(0.f, 0.f);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t pk[16];
                        if (c < seen) {
#pragma unroll
                        for (int y = 0; y < 32; y += 4) {
                            const float2 a = f2_fma(f2_from_bits(s[c][y], s[c][y + 1]), sc2, nm2);
                            const float2 b = f2_fma(f2_from_bits(s[c][y + 2], s[c][y + 3]), sc2, nm2);
                            const float2 pa = make_float2(fast_exp2(a.x), fast_exp2(a.y)), pb = make_float2(fast_exp2(b.x), fast_exp2(b.y));
                            l2a = f2_add(l2a, pa);
                            l2b = f2_add(l2b, pb);
                            pk[y >> 1] = pack_act<FP16>(pa.x, pa.y);
                            pk[(y >> 1) + 1] = pack_act<FP16>(pb.x, pb.y);
                        }
                        tmem_st16(tmem_addr(ts, quarter, 16 * c), pk);
                        }
                        if (c & 1) {
                            tmem_st_wait();
                            tc_fence_before_sync();
                            warp_arrive(BAR(sm->p_full[buf][c >> 1]));
                        }
                    }
                    l += (l2a.x + l2a.y) + (l2b.x + l2b.y);
                }
                last = buf;
                last_ph = bph;
                if (++buf == kPrBuffers) {
                    buf = 0;
                    bph ^= 1;
                }
            }
            if (bad) break;
            ring = (ring + 2 * steps) % (2 * kPrKvStages);
            sm->part[slot][g][row] = make_float2(m, l);
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(BAR(sm->sum_full[slot]));
                mbar_arrive(BAR(sm->item_empty[slot]));
            }
        }
    }
    if (bad) {
        atomicMax(P.status, kStatusWaitTimeout);
        // Give loads and products that are still in flight time to finish before shared memory and TMEM are released.
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000) __nanosleep(1000);
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
}

struct PromptSpace {
    int32_t group, tokens;
    int64_t cap, bytes;
};
bool prompt_space(int B, int S, int Hq, int Hkv, int n_seqs, PromptSpace* w) {
    if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 128 || n_seqs <= 0) return false;
    w->group = Hq / Hkv;
    w->tokens = 128 / w->group;
    w->cap = static_cast<int64_t>(B) * (static_cast<int64_t>(S) / w->tokens + n_seqs);   // (a sequence has at most one tile that is not full)
    w->bytes = 256 + 16 * w->cap;
    return true;
}

// As many CTAs as there can be tiles: each finds its own, and nothing is listed.  (Searching the sequences takes a few loads per 32 of them.)
bool prompt_direct(const PromptSpace& w, int B, int Hkv, int n_seqs, int sms) {
    return w.cap * Hkv <= sms && static_cast<int64_t>(B) * n_seqs <= 256;
}

}  // namespace
}  // namespace fmsa

extern "C" int32_t fmsa_prompt_launches(int32_t B, int32_t S, int32_t Hq, int32_t Hkv, int32_t n_seqs) {
    fmsa::PromptSpace w;
    if (!fmsa::prompt_space(B, S, Hq, Hkv, n_seqs, &w)) return -1;
    return fmsa::prompt_direct(w, B, Hkv, n_seqs, fmsa::device_sm_count()) ? 1 : 2;
}

extern "C" int64_t fmsa_prompt_workspace_bytes(int32_t B, int32_t S, int32_t Hq, int32_t Hkv, int32_t n_seqs) {
    fmsa::PromptSpace w;
    if (!fmsa::prompt_space(B, S, Hq, Hkv, n_seqs, &w)) return -1;
    return fmsa::prompt_direct(w, B, Hkv, n_seqs, fmsa::device_sm_count()) ? 0 : w.bytes;
}

extern "C" int fmsa_prompt_fwd(const fmsa_prompt_args* args, void* stream) {
    using namespace fmsa;
    FMSA_REQUIRE(args);
    const fmsa_tensor *q = &args->q, *k = &args->k, *v = &args->v;
    const int32_t B = args->B, S = args->S, Hq = args->Hq, Hkv = args->Hkv, dtype = args->dtype, *cu_seqlens = args->cu_seqlens;
    int32_t n_seqs = args->n_seqs;
    const float scale = args->scale;
    void *out = args->out, *workspace = args->workspace;
    int32_t* status = args->status;
    if (!cu_seqlens) n_seqs = 1;
    PromptSpace w;
    FMSA_REQUIRE(q->ptr && k->ptr && v->ptr && out && status && aligned16(out));
    FMSA_REQUIRE(B > 0 && S > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && n_seqs > 0 && scale > 0.f);
    FMSA_REQUIRE(dtype == FMSA_DTYPE_BF16 || dtype == FMSA_DTYPE_FP16);
    if (!prompt_space(B, S, Hq, Hkv, n_seqs, &w)) return FMSA_ERR_UNSUPPORTED;
    if (S > (1 << 30) || w.cap * Hkv >= 0x7f000000LL || static_cast<int64_t>(B) * n_seqs >= 0x7f000000LL) return FMSA_ERR_UNSUPPORTED;
    const int sms = device_sm_count();
    const bool direct = prompt_direct(w, B, Hkv, n_seqs, sms);
    if (!direct) {
        FMSA_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0);
        if (args->workspace_bytes < w.bytes) return FMSA_ERR_WORKSPACE;
    }
    for (const fmsa_tensor* t : {q, k, v}) FMSA_REQUIRE(tma_compatible(t->ptr, t->stride_b, t->stride_h, t->stride_s));
    CUtensorMap tq, tk, tv;
    if (!make_tmap_heads(&tq, q->ptr, B, Hq, S, q->stride_b, q->stride_h, q->stride_s, w.group, w.tokens) ||
        !make_tmap_bhsd(&tk, k->ptr, B, Hkv, S, k->stride_b, k->stride_h, k->stride_s, 128) ||
        !make_tmap_bhsd(&tv, v->ptr, B, Hkv, S, v->stride_b, v->stride_h, v->stride_s, 128))
        return FMSA_ERR_CUDA;
    PromptParams P = {};
    P.cu = cu_seqlens;
    P.sinks = args->sinks;
    P.v = static_cast<const __nv_bfloat16*>(v->ptr);
    P.vs[0] = v->stride_b; P.vs[1] = v->stride_h; P.vs[2] = v->stride_s;
    P.out = static_cast<__nv_bfloat16*>(out);
    if (!direct) {
        P.counter = static_cast<int32_t*>(workspace);
        P.tiles = reinterpret_cast<int4*>(static_cast<char*>(workspace) + 256);
    }
    P.status = status;
    P.B = B; P.S = S; P.Hq = Hq; P.Hkv = Hkv; P.group = w.group; P.tokens = w.tokens;
    P.n_seqs = n_seqs; P.per_batch = args->per_batch ? 1 : 0; P.cap = static_cast<int32_t>(w.cap);
    while (((S + kBlock - 1) / kBlock >> P.shift) >= kPlanBins) ++P.shift;
    P.scale_log2e = scale * kLog2e;
    auto kernel = dtype == FMSA_DTYPE_FP16 ? prompt_fwd_kernel<true> : prompt_fwd_kernel<false>;
    if (sms <= 0 || !ensure_smem_attr(reinterpret_cast<const void*>(kernel), kPrSmemBytes)) return FMSA_ERR_CUDA;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t items = w.cap * Hkv;
    P.direct = direct;
    if (!direct) launch_chained(prompt_plan_kernel, cu_seqlens ? 33 : 1, kPlanThreads, 0, st, P);
    launch_chained(kernel, static_cast<unsigned>(items < sms ? items : sms), kPrThreads, kPrSmemBytes, st, tq, tk, tv, P);
    return check_launch();
}
