// Attention over the cache held in 4 bits where many query rows share a KV head (17 and more, or 9 and more over few pages or with weights:
// form_of() in cache_attend.cu, which has the others).
//
// There the instructions per row, not those per nibble, are what counts: scaling sums and probabilities of 16 tokens x 8 rows in registers for
// mma.sync takes 140 of them, and blocks of 16 rows unpack the cache again and again.  Here a page is unpacked once, with its scales, into
// fp16 tiles in shared memory, and tcgen05 has both operands from there:
//   S^T = K Q^T     M: the page's 128 tokens, N: the rows (a multiple of 16, up to 64 a block), so that a thread has one token, and what
//                   belongs to a token - the power of two that its scales were divided by - is one factor of the thread's;
//   O^T += V^T P^T  M: the channels, N: the rows; P goes through shared memory, [token][row] as the threads have it.
// A code times a scale has at most 3 + 8 significant bits: fp16 holds it exactly while a group's scale is not below 2^-27 of the token's largest.
// (A nibble moved under the exponent of 16 is 16 + q, and (16 + q) s - 24 s one fma; 24 s has ten bits.)
// The reference of a row (the maximum of logit + log2 of the token's V factor, less kLift) is raised when a token exceeds it by more than
// kSlack; probabilities times V's factor are rounded to fp16 relative to it, sums are of the unrounded ones.
//
// A CTA has a range of the line of pages (of all pairs of sequence and KV head, and blocks of rows); what is cut goes to the workspace as in
// cache_attend.cu.  One warp loads halves of records, four unpack K, four V, eight have a token and half of the rows a thread, one issues the
// products, two prepare queries.  WEIGHTS: the probabilities of every token summed over the rows, relative to the log-sum-exps that the
// first kernel left (K alone; two groups of four warps have every other page).
//
// B=16 Hq=48 Hkv=4 n=4 (48 rows), lengths to 6001 (41 MB): 30.4 us, 3.8 for what was cut, and 17.0 for the weights; in blocks of 16 rows
// through registers 46 + 4 + 24.  Bound by latency: a page takes 2600 cycles in the warps that have tokens (500 for S out of tensor memory, 550
// for the common decision on the reference, 780 for probabilities, the rest barriers and fences) and 2200 in those that unpack (950 for
// the codes), at a third of the issue rate; 8000 cycles go by before the first page is multiplied and 3000 at the end.
#include "cache_attend.cuh"
#include "host_common.h"
#include "sm100.cuh"

namespace fmsa {
namespace {

constexpr int kRowsThreads = 640;
constexpr int kRegsTokens = 120, kRegsUnpack = 80, kRegsRest = 80;   // 96 each at launch
static_assert(2 * kRegsTokens + 2 * kRegsUnpack + kRegsRest <= 5 * 96, "register re-division must balance");
constexpr int kOddSlots = 4;
constexpr uint32_t kIdleNs = 200;
// Halves of a record on their way, K or V, codes and scales.  (Each part is always the same warps': a barrier's parity tells two phases apart, not
// four, so everyone who waits for a part has to see each of its phases.)
constexpr int kRawParts = 4, kRawBytes = kRecordBytes / 2;
static_assert(kKScales == 8192 && kVCodes == kRawBytes && kVScales == kRawBytes + 8192, "the halves look alike");

template <int N>
struct RowsCtrl {
    uint64_t raw_full[kRawParts], raw_empty[kRawParts], k_full[2], v_full[2], v_empty[2], s_full[2], s_empty[2];
    uint64_t p_full[2], pv_done[2], q_full[2], q_empty[2], o_free[2];
    float4 scale[2][N / 2];          // [slot of queries][two rows]: product -> logit of either row, -reference (WEIGHTS: -log-sum-exp) of either
    float2 alpha[N / 2], delta[N / 2];   // of a raise: the factor for what there is, and by how much
    float part[4][N];                // [warp]: maxima or sums
    float inv[N];
    float k_factor[4][kPage], v_factor[4][kPage];   // [page, modulo 4][token]: read before S of the page after the next one is made
    int32_t limit[2][N];             // tokens the row sees, less the sequence's length
    // A page that does not exist: nothing was loaded.  Its tokens' K factors are zero, which no other token's is, and nobody sees them.
    uint32_t gone[kRawParts];
    uint32_t odd[kOddSlots];         // a piece has V that is not finite in tokens that some rows do not see
    int32_t first, rest, length;     // sequence in which the range begins, units of it before, its length
    int32_t sums[kRowsThreads / 32];
    uint32_t tmem_slot;
};
constexpr int kTileStages = 2;
template <bool WEIGHTS> constexpr size_t kRowsTiles = static_cast<size_t>(WEIGHTS ? kTileStages + 1 : 2 * kTileStages + 1) * kTileBytes + (WEIGHTS ? 0 : kPanelBytes);   // K, Q, (V, P)
template <int N, bool WEIGHTS> constexpr size_t kRowsSmem = kRowsTiles<WEIGHTS> + kRawParts * kRawBytes + sizeof(RowsCtrl<N>) + 1024;
static_assert(kRowsSmem<64, false> <= 232448, "shared memory budget of one CTA");

// A range of the line of pages: page `page` of KV head `head` and block of rows `block` of sequence `seq`, `left` pages with this one.
struct Walk {
    int seq, length, pages, head, block, page, left;
    bool begin;   // of a piece
    __device__ __forceinline__ bool last() const { return page == pages - 1 || left == 1; }
    __device__ __forceinline__ void advance(const AttendParams& P) {
        begin = ++page == pages;
        --left;
        if (!begin) return;
        page = 0;
        if (left <= 0 || ++block < P.blocks) return;
        block = 0;
        if (++head < P.cache.heads) return;
        head = 0;
        do length = P.cache.length(++seq); while (length == 0);
        pages = (length + kPage - 1) / kPage;
    }
};

// Sums (or maxima) of v[0] .. v[N - 1] over the lanes: each of a few lanes then has some of them, v[0 .. the result's second) of columns from the
// first on.
template <int N, class F>
__device__ __forceinline__ int2 over_lanes(float (&v)[N], int lane, F&& join) {
    int first = 0, n = N;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const bool upper = lane & o, halve = n % 2 == 0;
        if (halve) {
            n /= 2;
            first += upper ? n : 0;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) {
                const float mine = halve && upper ? v[i + n < N ? i + n : 0] : v[i], other = halve && !upper ? v[i + n < N ? i + n : 0] : v[i];
                v[i] = join(mine, __shfl_xor_sync(0xffffffffu, other, o));
            }
    }
    return make_int2(first, n);
}
__device__ __forceinline__ bool any_of_half(int half, bool mine) {   // over the 128 threads of one half of the rows
    uint32_t r;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.u32 p, %1, 0;\n"
        "bar.red.or.pred q, %2, 128, p;\n"
        "selp.u32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(mine)), "r"(3 + half)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ uint32_t half2_word(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }

// Eight codes as four pairs of fp16 (q - 8) * s, bits 0..3 and 16..19 first; back: -24 s.  A nibble at bits 6..9 under the exponent of 16 is 16 + q.
__device__ __forceinline__ uint4 unpack8(uint32_t w, __half2 s, __half2 back, uint32_t sixteen) {
    constexpr uint32_t at = 0x03c003c0u;
    return make_uint4(half2_word(__hfma2(as_half2(masked_or(w << 6, at, sixteen)), s, back)), half2_word(__hfma2(as_half2(masked_or(w << 2, at, sixteen)), s, back)),
                      half2_word(__hfma2(as_half2(masked_or(w >> 2, at, sixteen)), s, back)), half2_word(__hfma2(as_half2(masked_or(w >> 6, at, sixteen)), s, back)));
}
__device__ __forceinline__ void st_piece(uint32_t at, uint4 x) { st_shared_v4(at, x.x, x.y, x.z, x.w); }
__device__ __forceinline__ uint2 ld_shared_v2(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
// Scales of a token, times the power of two that takes the largest to [2^10, 2^11) (24 times that is fp16 still); returns its reciprocal.
__device__ __forceinline__ float token_scales(uint2 w, float (&s)[4]) {
    s[0] = __uint_as_float(w.x << 16);
    s[1] = __uint_as_float(w.x & 0xffff0000u);
    s[2] = __uint_as_float(w.y << 16);
    s[3] = __uint_as_float(w.y & 0xffff0000u);
    const float top = fmaxf(fmax3(s[0], s[1], s[2]), s[3]);   // (a NaN beside others is passed over)
    const uint32_t e = min(max(__float_as_uint(top) >> 23, 44u), 224u);   // exponent; 2^-83 is the smallest scale there is
    const float mul = __uint_as_float((264u - e) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] *= mul;
    return __uint_as_float((e - 10u) << 23);
}

template <bool V> struct IsV { static constexpr bool value = V; };

template <int N, bool WEIGHTS>
__global__ void __launch_bounds__(kRowsThreads, 1) cache_rows_kernel(const AttendParams P) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* tiles_at = smem_raw + (tiles - smem_u32(smem_raw));
    // queries: block of slot s at + s * 8 KB (64 rows of either panel of one tile); P: one panel
    const uint32_t tile_k = tiles, tile_q = tile_k + kTileStages * kTileBytes, tile_v = tile_q + kTileBytes, tile_p = tile_v + kTileStages * kTileBytes;
    uint8_t* raw_at = tiles_at + kRowsTiles<WEIGHTS>;
    RowsCtrl<N>* sm = reinterpret_cast<RowsCtrl<N>*>(raw_at + kRawParts * kRawBytes);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, cta = blockIdx.x;
    auto BAR = [&](uint64_t& b) { return smem_u32(&b); };

    constexpr int kReaders = WEIGHTS ? 4 : 8;   // warps that read one page's S
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(BAR(sm->k_full[i]), 4);
            mbar_init(BAR(sm->v_full[i]), 4);
            mbar_init(BAR(sm->v_empty[i]), 1);
            mbar_init(BAR(sm->s_full[i]), 1 + (WEIGHTS ? 4 : 8));   // the product, the warps that have written the factors
            mbar_init(BAR(sm->s_empty[i]), kReaders);
            mbar_init(BAR(sm->p_full[i]), 8);
            mbar_init(BAR(sm->pv_done[i]), 1);
            mbar_init(BAR(sm->q_full[i]), 8);
            mbar_init(BAR(sm->q_empty[i]), 1 + 8);
            mbar_init(BAR(sm->o_free[i]), 8);
        }
        for (int i = 0; i < kRawParts; ++i) {
            mbar_init(BAR(sm->raw_full[i]), 1);
            mbar_init(BAR(sm->raw_empty[i]), 4);
        }
        for (int i = 0; i < kOddSlots; ++i) sm->odd[i] = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(&sm->tmem_slot), 256);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sm->tmem_slot;   // S of even and odd pages, O of even and odd pieces: 64 columns each
    wait_for_previous_kernel();

    // ---- the line of pages, and this CTA's range of it
    const int per = P.cache.heads * P.blocks, seqs = P.cache.seqs;
    auto scan = [&](int c0, int before, auto&& what) {
        const int b = c0 + tid, length = b < seqs ? P.cache.length(b) : 0, p = (length + kPage - 1) / kPage;
        int sum = p;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) sm->sums[warp] = sum;
        __syncthreads();
        const int w = lane < kRowsThreads / 32 ? sm->sums[lane] : 0;
        const int ahead = __reduce_add_sync(0xffffffffu, lane < warp ? w : 0), all = __reduce_add_sync(0xffffffffu, w);
        what(b, before + ahead + sum - p, length, before + all);
        __syncthreads();
        return before + all;
    };
    Ranges R;
    auto claim = [&](int b, int at, int length) {
        if (!WEIGHTS && b < seqs && cta == 0) P.prefix[b] = at;
        const int p = (length + kPage - 1) / kPage, u = R.begin(cta);
        if (at * per <= u && u < (at + p) * per) {
            sm->first = b;
            sm->rest = u - at * per;
            sm->length = length;
        }
    };
    int pages_all = 0;
    if (seqs <= kRowsThreads) {
        pages_all = scan(0, 0, [&](int b, int at, int length, int all) {
            R = Ranges(all * per, P.grid);
            claim(b, at, length);
        });
    } else {
        for (int c0 = 0; c0 < seqs; c0 += kRowsThreads) pages_all = scan(c0, pages_all, [](int, int, int, int) {});
        R = Ranges(pages_all * per, P.grid);
        int before = 0;
        for (int c0 = 0; c0 < seqs; c0 += kRowsThreads) before = scan(c0, before, [&](int b, int at, int length, int) { claim(b, at, length); });
    }
    if (!WEIGHTS && cta == 0 && tid == 0) P.prefix[seqs] = pages_all;
    Walk at = {};
    at.left = R.begin(cta + 1) - R.begin(cta);
    if (at.left > 0) {
        at.seq = sm->first;
        at.length = sm->length;
        at.pages = (at.length + kPage - 1) / kPage;
        const int item = sm->rest / at.pages;
        at.page = sm->rest - item * at.pages;
        at.head = item / P.blocks;
        at.block = item - at.head * P.blocks;
        at.begin = true;
    }
    bool bad = false;
    auto wait = [&](uint32_t bar, uint32_t parity) {   // every lane of the warp calls it; after one that ran out nothing is waited for
        for (uint32_t n = 0; !bad && !__all_sync(0xffffffffu, mbar_try_wait_parked(bar, parity, kRoleParkNs)); ++n) bad = n > kRoleWaitTries;
    };
    auto wait1 = [&](uint32_t bar, uint32_t parity) {   // the same in a role that a single thread runs
        if (!bad) bad = !mbar_wait_role(bar, parity);
    };
    // For those that are ahead: looks again after about `ns`.  (Warps that look all the time took half of the issue slots.)
    auto wait_idle = [&](uint32_t bar, uint32_t parity, uint32_t ns) {
        for (uint32_t n = 0; !bad && !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); ++n) {
            bad = n > 1000000;   // (a try and a sleep take a microsecond or two)
            __nanosleep(ns);
        }
    };
    auto warp_arrive = [&](uint32_t bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };

    // Eight rows of the queries, number e8 of the block, as an operand, and what belongs to them; by a warp.
    auto prepare = [&](const RawQueries& raw, int e8, uint32_t slot, int head, int block) {
        const int row = 8 * e8 + (lane >> 2), t = lane & 3;
        float f[4][8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w[4] = {raw.x[i].x, raw.x[i].y, raw.x[i].z, raw.x[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[i][2 * e] = P.fp16 ? act_lo<true>(w[e]) : act_lo<false>(w[e]);
                f[i][2 * e + 1] = P.fp16 ? act_hi<true>(w[e]) : act_hi<false>(w[e]);
                top = max(top, max(__float_as_uint(f[i][2 * e]) & 0x7fffffffu, __float_as_uint(f[i][2 * e + 1]) & 0x7fffffffu));
            }
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // largest magnitude to [2^13, 2^14)
        const int up = min(max(13 + 127 - static_cast<int>(top >> 23), -90), 126);
        const float mul = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // channels 32 i + 8 t .., in the order in which unpack8() has K's
#pragma unroll
            for (int e = 0; e < 8; ++e) f[i][e] *= mul;
            st_shared_v4(tile_q + slot * (kPanelBytes / 2) + swz_offset(row, 4 * i + t), pack_act<true>(f[i][0], f[i][4]), pack_act<true>(f[i][1], f[i][5]),
                         pack_act<true>(f[i][2], f[i][6]), pack_act<true>(f[i][3], f[i][7]));
        }
        if (t == 0) {
            const bool real = block * N + row < P.rows;
            float* sc = reinterpret_cast<float*>(&sm->scale[slot][row >> 1]) + (row & 1);
            sc[0] = real ? __uint_as_float(static_cast<uint32_t>(127 - up) << 23) * P.scale_log2e : 0.f;
            float ref = 0.f;
            if (WEIGHTS) ref = real ? P.lse[(static_cast<int64_t>(at.seq) * P.cache.heads + head) * P.lse_rows + block * N + row] : INFINITY;
            sc[2] = -ref;
            sm->limit[slot][row] = raw.limit;
        }
    };
    // (the first piece's by the warps that will have tokens, one eight each, while the first page is on its way)
    if (warp < 8 && at.left > 0) {
        if (warp < N / 8) {
            RawQueries raw;
            raw.load(P, at.seq, at.head, at.block * N + 8 * warp, lane);
            prepare(raw, warp, 0, at.head, at.block);
        }
        fence_async_smem();
        warp_arrive(BAR(sm->q_full[0]));
    }

    if (warp < 8) {
        // =========================== a token and half of the rows a thread (WEIGHTS: all rows, of even or of odd pages) ===========================
        reg_inc<kRegsTokens>();
        constexpr int H = WEIGHTS ? N : N / 2;
        const int half = warp >> 2, quarter = warp & 3, token = tid & 127, low = WEIGHTS ? 0 : H * half;   // first row of this half
        float2 l[H / 2];
        uint32_t pieces = 0;
        int begun = 0;            // first page of the piece
        bool fresh = true;        // no page of the piece so far
        int ids = -1, from = 0;   // pages from `from` on, a lane each
        for (uint32_t it = 0; at.left > 0; ++it, at.advance(P)) {
            const uint32_t st = it & 1, ph = it >> 1 & 1, slot = pieces & 1;
            const int head = at.head, block = at.block, place = at.page * kPage + token - at.length;
            const bool edge = (at.page + 1) * kPage > at.length - P.n + 1;   // (some tokens are not seen by some row, or are not there)
            if (at.begin) {
                begun = at.page;
                fresh = true;
                wait(BAR(sm->q_full[slot]), pieces >> 1 & 1);
                if (!WEIGHTS && at.page == 0 && tid == 0) {   // (the part that begins a pair says where its parts are)
                    const int behind = R.begin(cta + 1) - at.left + at.pages;   // the unit behind the pair's last
                    P.parts[static_cast<int64_t>(at.seq) * per + head * P.blocks + block] =
                        make_int2(2 * cta + (pieces ? 1 : 0), at.left >= at.pages ? 0 : R.owner(behind - 1) - cta + 1);
                }
            }
            if constexpr (WEIGHTS) {
                if (at.begin || at.page - from == 32) {
                    from = at.page;
                    ids = at.page + lane < at.pages ? P.cache.page(at.seq, at.page + lane) : -1;
                }
                if (st == static_cast<uint32_t>(half)) {
                    const int page = __shfl_sync(0xffffffffu, ids, at.page - from);
                    float* weight = P.weights + (static_cast<int64_t>(max(page, 0)) * P.cache.heads + head) * kPage + token;
                    const bool there = page >= 0 && place < 0;
                    const float old = there && P.accumulate ? *weight : 0.f;
                    wait(BAR(sm->s_full[st]), ph);
                    const float factor = sm->k_factor[it & 3][token];
                    tc_fence_after_sync();
                    uint32_t s[N / 8][8];
#pragma unroll
                    for (int i = 0; i < N / 8; ++i) tmem_ld8(tmem_addr(tmem + 64 * st, quarter, 8 * i), s[i]);
                    tmem_ld_wait();
                    tc_fence_before_sync();
                    warp_arrive(BAR(sm->s_empty[st]));
                    const float2 f2 = make_float2(factor, factor);
                    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                    for (int c = 0; c < N / 2; ++c) {
                        const float4 sc = sm->scale[slot][c];
                        float2 y = f2_fma(f2_mul(f2_from_bits(s[c >> 2][2 * (c & 3)], s[c >> 2][2 * (c & 3) + 1]), f2), make_float2(sc.x, sc.y), make_float2(sc.z, sc.w));
                        if (edge) {
                            const int2 lim = *reinterpret_cast<const int2*>(&sm->limit[slot][2 * c]);
                            if (place >= lim.x) y.x = -INFINITY;
                            if (place >= lim.y) y.y = -INFINITY;
                        }
                        sum = f2_add(sum, make_float2(fast_exp2(y.x), fast_exp2(y.y)));
                    }
                    if (there) *weight = old + (sum.x + sum.y);
                }
                if (at.last()) {
                    warp_arrive(BAR(sm->q_empty[slot]));
                    ++pieces;
                }
            } else {
                wait(BAR(sm->s_full[st]), ph);
                const float factor_k = sm->k_factor[it & 3][token], factor_v = sm->v_factor[it & 3][token];
                tc_fence_after_sync();
                float2 y[H / 2];   // logits less the reference, log2 domain
                {
                    uint32_t s[H / 8][8];
#pragma unroll
                    for (int i = 0; i < H / 8; ++i) tmem_ld8(tmem_addr(tmem + 64 * st, quarter, low + 8 * i), s[i]);
                    tmem_ld_wait();
                    tc_fence_before_sync();
                    warp_arrive(BAR(sm->s_empty[st]));
                    const float2 f2 = make_float2(factor_k, factor_k);
#pragma unroll
                    for (int c = 0; c < H / 2; ++c) {
                        const float4 sc = sm->scale[slot][low / 2 + c];
                        y[c] = f2_fma(f2_mul(f2_from_bits(s[c >> 2][2 * (c & 3)], s[c >> 2][2 * (c & 3) + 1]), f2), make_float2(sc.x, sc.y), make_float2(sc.z, sc.w));
                    }
                }
                const bool gone = factor_k == 0.f;   // (of all 128 tokens or of none)
                if (edge || gone) {
#pragma unroll
                    for (int c = 0; c < H / 2; ++c) {
                        const int2 lim = *reinterpret_cast<const int2*>(&sm->limit[slot][low + 2 * c]);
                        if (gone || place >= lim.x) y[c].x = -INFINITY;
                        if (gone || place >= lim.y) y[c].y = -INFINITY;
                    }
                }
                const float lg = static_cast<float>(static_cast<int>(__float_as_uint(factor_v) >> 23) - 127);
                float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                for (int c = 0; c < H / 2; c += 2) {
                    m0 = fmax3(m0, y[c].x, y[c].y);
                    m1 = fmax3(m1, y[c + 1].x, y[c + 1].y);
                }
                if (fresh || any_of_half(half, fmaxf(m0, m1) + lg > kLift + kSlack)) {
                    // the references: set by a piece's first page, else raised, for every row by what it needs
                    float v[H];
#pragma unroll
                    for (int c = 0; c < H; ++c) v[c] = (c & 1 ? y[c >> 1].y : y[c >> 1].x) + lg;
                    const int2 mine = over_lanes<H>(v, lane, [](float a, float b) { return fmaxf(a, b); });
#pragma unroll
                    for (int i = 0; i < H; ++i)
                        if (i < mine.y) sm->part[quarter][low + mine.x + i] = v[i];
                    named_barrier_sync(1 + half, 128);
                    if (token < H) {
                        const int c = low + token;
                        const float top = fmaxf(fmaxf(sm->part[0][c], sm->part[1][c]), fmaxf(sm->part[2][c], sm->part[3][c])) - kLift;
                        const float by = top < INFINITY && (fresh ? top > -INFINITY : top > 0.f) ? top : 0.f;
                        reinterpret_cast<float*>(sm->delta)[c] = by;
                        reinterpret_cast<float*>(sm->alpha)[c] = fast_exp2(-by);
                        reinterpret_cast<float*>(&sm->scale[slot][c >> 1])[2 + (c & 1)] -= by;
                    }
                    named_barrier_sync(1 + half, 128);
#pragma unroll
                    for (int c = 0; c < H / 2; ++c) {
                        const float2 by = sm->delta[low / 2 + c];
                        y[c] = f2_add(y[c], make_float2(-by.x, -by.y));
                    }
                    if (fresh) {             // (O is not there yet, or zero)
#pragma unroll
                        for (int c = 0; c < H / 2; ++c) l[c] = make_float2(0.f, 0.f);
                    } else {
#pragma unroll
                        for (int c = 0; c < H / 2; ++c) l[c] = f2_mul(l[c], sm->alpha[low / 2 + c]);
                        wait(BAR(sm->pv_done[st ^ 1]), (it - 1) >> 1 & 1);   // the product of the page before may still be adding to O
                        tc_fence_after_sync();
                        const uint32_t o_at = tmem + 128 + 64 * slot;
#pragma unroll 1
                        for (int i = low; i < low + H; i += 8) {
                            uint32_t o[8];
                            tmem_ld8(tmem_addr(o_at, quarter, i), o);
                            tmem_ld_wait();
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const float2 r = f2_mul(f2_from_bits(o[2 * c], o[2 * c + 1]), sm->alpha[i / 2 + c]);
                                o[2 * c] = __float_as_uint(r.x);
                                o[2 * c + 1] = __float_as_uint(r.y);
                            }
                            tmem_st8(tmem_addr(o_at, quarter, i), o);
                        }
                        tmem_st_wait();
                    }
                    named_barrier_sync(1 + half, 128);   // (part, alpha and delta may be written again)
                    fresh &= gone;
                }
                if (it >= 1) wait(BAR(sm->pv_done[st ^ 1]), (it - 1) >> 1 & 1);   // (P of the page before has been read)
                const uint32_t p_at = tile_p + token * 128;
                const float2 fv = make_float2(factor_v, factor_v);
#pragma unroll
                for (int c = 0; c < H / 2; c += 4) {
                    uint32_t pk[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 p = make_float2(fast_exp2(y[c + i].x), fast_exp2(y[c + i].y));
                        l[c + i] = f2_add(l[c + i], p);
                        const float2 w = f2_mul(p, fv);
                        pk[i] = pack_act<true>(w.x, w.y);
                    }
                    st_shared_v4(p_at + (((low >> 3) + (c >> 2) ^ token & 7) << 4), pk[0], pk[1], pk[2], pk[3]);
                }
                fence_async_smem();
                tc_fence_before_sync();
                warp_arrive(BAR(sm->p_full[st]));
                if (at.last()) {
                    // ---- the end of a piece
                    const bool whole = begun == 0 && at.page == at.pages - 1;
                    const int64_t part_slot = 2LL * cta + (pieces ? 1 : 0);
                    {
                        float v[H];
#pragma unroll
                        for (int c = 0; c < H; ++c) v[c] = c & 1 ? l[c >> 1].y : l[c >> 1].x;
                        const int2 mine = over_lanes<H>(v, lane, [](float a, float b) { return a + b; });
#pragma unroll
                        for (int i = 0; i < H; ++i)
                            if (i < mine.y) sm->part[quarter][low + mine.x + i] = v[i];
                    }
                    named_barrier_sync(1 + half, 128);
                    const int rows = min(N, P.rows - block * N);   // of this block
                    if (token < H) {
                        const int c = low + token, row = block * N + c;
                        float sum = (sm->part[0][c] + sm->part[1][c]) + (sm->part[2][c] + sm->part[3][c]);
                        const float ref = -reinterpret_cast<const float*>(&sm->scale[slot][c >> 1])[2 + (c & 1)];
                        if (whole) {
                            if (P.sinks && c < rows) sum += fast_exp2(P.sinks[head * P.group + row / P.n] * kLog2e - ref);
                            sm->inv[c] = sum == 0.f ? 0.f : 1.f / sum;
                            if (c < rows) P.lse[(static_cast<int64_t>(at.seq) * P.cache.heads + head) * P.lse_rows + row] = ref + fast_log2(sum);
                        } else {
                            if (c < rows) P.ml_part[part_slot * N + c] = make_float2(sum == 0.f ? -INFINITY : ref, sum);
                        }
                    }
                    // position of this thread in O -> channel
                    const int channel = 32 * (2 * (token >> 3 & 1) + (token & 1)) + 4 * (token >> 4) + (token >> 1 & 3);
                    // V that is not finite where not every row sees it (it was left out of the product)
                    uint32_t poison = 0;
                    if (sm->odd[pieces % kOddSlots])
#pragma unroll 1
                        for (int t = max(at.length - P.n + 1, begun * kPage); t < min(at.length, (at.page + 1) * kPage); ++t) {
                            const int page = P.cache.page(at.seq, t / kPage);
                            if (page < 0) continue;
                            const uint32_t s = *reinterpret_cast<const uint16_t*>(P.cache.record(page, head) + kVScales + t % kPage * 8 + channel / 32 * 2);
                            if (s < 0x7f80u) continue;
#pragma unroll 1
                            for (int c = 0; c < H; ++c)
                                if (t - at.length < sm->limit[slot][low + c]) poison |= 1u << c;
                        }
                    wait(BAR(sm->pv_done[st]), ph);
                    tc_fence_after_sync();
                    named_barrier_sync(1 + half, 128);
                    uint8_t* staging = tiles_at + (tile_p - tiles);   // (P of this page has been read)
#pragma unroll 1
                    for (int i = low; i < low + H; i += 8) {
                        uint32_t o[8];
                        tmem_ld8(tmem_addr(tmem + 128 + 64 * slot, quarter, i), o);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            if (poison >> (i - low + c) & 1) o[c] = 0x7fffffffu;
                        if (whole) {
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                const float x = __uint_as_float(o[c]) * sm->inv[i + c];
                                *reinterpret_cast<uint16_t*>(staging + (i + c) * 256 + 2 * channel) =
                                    static_cast<uint16_t>(P.fp16 ? pack_act<true>(x, x) : pack_act<false>(x, x));
                            }
                        } else {
                            float* to = P.o_part + (part_slot * N + i) * kHeadDim + channel;
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                if (i + c < rows) to[c * kHeadDim] = __uint_as_float(o[c]);
                        }
                    }
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(BAR(sm->o_free[slot]));
                        mbar_arrive(BAR(sm->q_empty[slot]));
                    }
                    named_barrier_sync(1 + half, 128);
                    if (whole) {
                        for (int r = low + (token >> 4); r < min(rows, low + H); r += 8) {
                            const int row = block * N + r, hh = row / P.n, j = row - hh * P.n, h = head * P.group + hh;
                            *reinterpret_cast<uint4*>(P.out + ((static_cast<int64_t>(at.seq) * P.n + j) * P.Hq + h) * kHeadDim + 8 * (token & 15)) =
                                *reinterpret_cast<const uint4*>(staging + r * 256 + 16 * (token & 15));
                        }
                    }
                    named_barrier_sync(5, 256);   // (P may be written again)
                    if (tid == 0) sm->odd[pieces % kOddSlots] = 0;
                    ++pieces;
                }
            }
        }
    } else if (warp < 16) {
        // =========================== K, V: codes and scales -> fp16 ===========================
        reg_dec<kRegsUnpack>();
        // A lane has a token.  The order in which it takes the 16-byte pieces of its row, and the tiles' own order, let eight neighbouring lanes
        // read and write all places of 128 bytes.
        const int group = (warp >> 2) - 2, row = tid & 127, turn = row >> 1 & 3;
        const uint32_t tile_row = row * 128, sixteen = P.magic - 0x18001800u;   // 16, 16 in fp16 (not a constant: see P.magic)
        auto unpack = [&](auto which) {
            constexpr bool is_v = decltype(which)::value;
            uint32_t pieces = 0, n = is_v || (WEIGHTS && group) ? 1 : 0;   // n: parts so far, of either kind
            if (WEIGHTS && group && at.left > 0) at.advance(P);   // (K of even pages, and of odd ones)
            for (uint32_t it = WEIGHTS ? group : 0; at.left > 0; it += WEIGHTS ? 2 : 1, n += 2) {
                const uint32_t st = it & 1, ph = it >> 1 & 1, part = n % kRawParts;
                wait(BAR(sm->raw_full[part]), n / kRawParts & 1);
                if (bad) break;
                const uint32_t raw = smem_u32(raw_at) + part * kRawBytes;
                uint2 w = ld_shared_v2(raw + 8192 + row * 8);
                const bool gone = sm->gone[part];
                if (is_v) {
                    const int place = at.page * kPage + row - at.length;
                    if (place >= 0 || gone) {
                        w = make_uint2(0, 0);     // not there
                    } else if (place > -P.n) {    // not seen by all rows: 0 * NaN must not reach the others
                        const uint2 old = w;
                        if ((w.x & 0x7f80u) == 0x7f80u) w.x &= 0xffff0000u;
                        if ((w.x & 0x7f800000u) == 0x7f800000u) w.x &= 0xffffu;
                        if ((w.y & 0x7f80u) == 0x7f80u) w.y &= 0xffff0000u;
                        if ((w.y & 0x7f800000u) == 0x7f800000u) w.y &= 0xffffu;
                        if (w.x != old.x || w.y != old.y) sm->odd[pieces % kOddSlots] = 1;
                    }
                }
                float s[4];
                const float factor = token_scales(w, s);
                const __half2 s01 = __floats2half2_rn(s[0], s[1]), s23 = __floats2half2_rn(s[2], s[3]);
                const __half2 b01 = __hmul2(s01, __float2half2_rn(-24.f)), b23 = __hmul2(s23, __float2half2_rn(-24.f));
                // (K goes when S of the page two before is complete, factors and all: nobody arrives there twice.  The first round finds both free)
                wait_idle(BAR((is_v ? sm->v_empty : sm->s_full)[st]), ph ^ 1, kIdleNs);
                if (bad) break;
                (is_v ? sm->v_factor : sm->k_factor)[it & 3][row] = !is_v && gone ? 0.f : factor;
                const uint32_t tile = (is_v ? tile_v : tile_k) + st * kTileBytes + tile_row;
#pragma unroll 2
                for (int k = 0; k < 4; ++k) {
                    const uint32_t u = k ^ turn;
                    const uint4 x = ld_shared_v4(raw + row * 64 + u * 16);
                    if (is_v) {
                        // places 2 u and 2 u + 1, chunks c = place ^ (row & 4) of the channels: pieces 2 c, 2 c + 1
                        const uint32_t to = tile + ((u >> 1 ^ (row >> 2 & 1)) * kPanelBytes) + ((4 * (u & 1) ^ (row & 7)) << 4);
                        st_piece(to, unpack8(x.x, s01, b01, sixteen));
                        st_piece(to ^ 16, unpack8(x.y, s23, b23, sixteen));
                        st_piece(to ^ 32, unpack8(x.z, s01, b01, sixteen));
                        st_piece(to ^ 48, unpack8(x.w, s23, b23, sixteen));
                    } else {
                        // words 0..3: pieces u, 4 + u, 8 + u, 12 + u, a scale each
                        const uint32_t to = tile + ((u ^ (row & 7)) << 4);
                        st_piece(to, unpack8(x.x, __low2half2(s01), __low2half2(b01), sixteen));
                        st_piece(to ^ 64, unpack8(x.y, __high2half2(s01), __high2half2(b01), sixteen));
                        st_piece(to + kPanelBytes, unpack8(x.z, __low2half2(s23), __low2half2(b23), sixteen));
                        st_piece((to ^ 64) + kPanelBytes, unpack8(x.w, __high2half2(s23), __high2half2(b23), sixteen));
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(BAR((is_v ? sm->v_full : sm->k_full)[st]));
                    mbar_arrive(BAR(sm->s_full[st]));
                    mbar_arrive(BAR(sm->raw_empty[part]));
                }
                if (is_v) pieces += at.last();
                at.advance(P);
                if (WEIGHTS && at.left > 0) at.advance(P);
            }
        };
        if (!WEIGHTS && group) unpack(IsV<true>());
        else unpack(IsV<false>());
    } else {
        reg_dec<kRegsRest>();
        if (warp == 16) {
            // =========================== products ===========================
            if (elect_one()) {
                uint32_t pieces = 0;
                // the page before: its place in the rings
                auto product = [&](uint32_t it, uint32_t piece, bool first) {   // O^T += V^T P^T of page `it`
                    const uint32_t st = it & 1, ph = it >> 1 & 1;
                    wait1(BAR(sm->v_full[st]), ph);
                    if (first) wait1(BAR(sm->o_free[piece & 1]), (piece >> 1 & 1) ^ 1);
                    wait1(BAR(sm->p_full[st]), ph);
                    if (bad) return;
                    tc_fence_after_sync();
                    umma_ss<N, 8, true, true, true>(tmem + 128 + 64 * (piece & 1), tile_v + st * kTileBytes, tile_p, !first);
                    umma_commit(BAR(sm->v_empty[st]));
                    umma_commit(BAR(sm->pv_done[st]));
                };
                uint32_t it = 0, before_piece = 0;
                bool before_first = false;
                for (; at.left > 0 && !bad; ++it) {
                    const uint32_t st = it & 1, ph = it >> 1 & 1, slot = pieces & 1;
                    if (at.begin) wait1(BAR(sm->q_full[slot]), pieces >> 1 & 1);
                    wait1(BAR(sm->k_full[st]), ph);
                    wait1(BAR(sm->s_empty[st]), ph ^ 1);   // (the first round finds both free)
                    if (bad) break;
                    tc_fence_after_sync();
                    umma_ss<N, 8, false, false, true>(tmem + 64 * st, tile_k + st * kTileBytes, tile_q + slot * (kPanelBytes / 2), false);   // S^T = K Q^T
                    umma_commit(BAR(sm->s_full[st]));
                    const bool first = at.begin, last = at.last();
                    if (last) umma_commit(BAR(sm->q_empty[slot]));
                    if (!WEIGHTS) {
                        if (it > 0) product(it - 1, before_piece, before_first);
                        before_piece = pieces;
                        before_first = first;
                    }
                    if (last) ++pieces;
                    at.advance(P);
                }
                if (!WEIGHTS && it > 0 && !bad) product(it - 1, before_piece, before_first);
            }
        } else if (warp == 17) {
            // =========================== pages ===========================
            int ids = -1, from = 0;          // pages from `from` on, a lane each
            for (uint32_t n = 0; at.left > 0; at.advance(P)) {
                if (at.begin || at.page - from == 32) {
                    from = at.page;
                    ids = at.page + lane < at.pages ? P.cache.page(at.seq, at.page + lane) : -1;
                }
                const int page = __shfl_sync(0xffffffffu, ids, at.page - from);
                const uint32_t tokens = min(kPage, (at.length - at.page * kPage + 15) & ~15);   // of the last page what is in use
                for (int v = 0; v < (WEIGHTS ? 1 : 2); ++v, ++n) {
                    const uint32_t part = n % kRawParts, bar = BAR(sm->raw_full[part]), to = smem_u32(raw_at) + part * kRawBytes;
                    wait_idle(BAR(sm->raw_empty[part]), (n / kRawParts & 1) ^ 1, kIdleNs);   // (the first round finds all parts free)
                    if (bad || lane) continue;
                    sm->gone[part] = page < 0;
                    if (page < 0) {
                        mbar_arrive(bar);
                        continue;
                    }
                    const uint8_t* rec = P.cache.record(page, at.head) + v * kRawBytes;
                    mbar_arrive_expect_tx(bar, tokens * 72);
                    if (tokens == kPage) {
                        bulk_load(to, rec, kRawBytes, bar);
                    } else {
                        bulk_load(to, rec, tokens * 64, bar);
                        bulk_load(to + 8192, rec + 8192, tokens * 8, bar);
                    }
                }
                __syncwarp();
                if (bad) break;
            }
        } else {
            // =========================== queries ===========================
            for (uint32_t pieces = 0; at.left > 0 && !bad; ++pieces) {
                if (pieces > 0) {
                    const uint32_t slot = pieces & 1;
                    RawQueries raw;
                    raw.load(P, at.seq, at.head, at.block * N + 8 * (warp - 18), lane);
                    wait_idle(BAR(sm->q_empty[slot]), (pieces >> 1 & 1) ^ 1, 4 * kIdleNs);
                    if (bad) break;
#pragma unroll 1
                    for (int e8 = warp - 18; e8 < N / 8; e8 += 2) {
                        if (e8 >= 2) raw.load(P, at.seq, at.head, at.block * N + 8 * e8, lane);
                        prepare(raw, e8, slot, at.head, at.block);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane < 4) mbar_arrive(BAR(sm->q_full[slot]));   // (eight in all, as from the eight warps of the first piece)
                }
                const int take = min(at.left, at.pages - at.page);   // to the next piece
                at.page += take - 1;
                at.left -= take - 1;
                at.advance(P);
            }
        }
    }
    if (bad) {
        atomicMax(P.cache.status, kStatusWaitTimeout);
        const uint64_t t0 = global_timer_ns();   // products in flight end before shared memory and tensor memory are released
        while (global_timer_ns() - t0 < 200000) __nanosleep(1000);
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 256);
}

template <int N, bool WEIGHTS>
bool launch(const AttendParams& P, cudaStream_t st) {
    const auto kernel = cache_rows_kernel<N, WEIGHTS>;
    if (!ensure_smem_attr(reinterpret_cast<const void*>(kernel), kRowsSmem<N, WEIGHTS>)) return false;
    launch_chained(kernel, P.grid, kRowsThreads, kRowsSmem<N, WEIGHTS>, st, P);
    return true;
}
template <bool WEIGHTS>
bool launch(const AttendParams& P, cudaStream_t st) {
    switch (rows_of_block(P.rows)) {
        case 16: return launch<16, WEIGHTS>(P, st);
        case 32: return launch<32, WEIGHTS>(P, st);
        case 48: return launch<48, WEIGHTS>(P, st);
        default: return launch<64, WEIGHTS>(P, st);
    }
}

}  // namespace

bool launch_attend_rows(const AttendParams& P, cudaStream_t st) { return launch<false>(P, st); }
bool launch_weights_rows(const AttendParams& P, cudaStream_t st) { return launch<true>(P, st); }

}  // namespace fmsa
