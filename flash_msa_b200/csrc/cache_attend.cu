// Attention over the cache held in 4 bits: the last few tokens of every sequence, their heads sharing KV heads.  Here up to 16 query rows to a
// KV head, and the merging of what is cut; cache_rows.cu has the others (form_of() chooses).
//
// 144 bytes per token and KV head are read once, whatever the number of query rows (heads of the group x new tokens); beside HBM it is
// bound by the instructions per nibble.  So:
//   * the pages of all (sequence, KV head) pairs stand in one line that is cut into equal ranges, four per SM: a long sequence is split, short
//     ones share an SM, and nothing depends on lengths that the host would have to know.  At most two pieces of a range are parts of a cut
//     pair; they go to the workspace and a second kernel merges them.  (Few pairs with few pages: a cluster of CTAs per pair, one launch.)
//   * a range belongs to a team: one warp keeps two records in flight and prepares queries, four others take 32 tokens of a page each;
//   * products on mma.sync m16n8k16 with the cache as the 16-row operand and 8 query rows beside it.  (tcgen05 wants its cache operand
//     from shared memory: the 16-bit copy of every nibble would be written and read there, four times the bytes that come in.)  A word of
//     eight nibbles gives four operand registers:
//       K   S^T = K Q^T: the nibbles are masked out as fp16 numbers as they stand (kLow, kHigh), the odd ones 16 times larger, which queries
//           divided by 16 make up for.  The 8 of (code = q - 8): sum over the groups of scale * -8 sum(Q), a product of its own of the
//           scales as they stand and sum(Q) in three bf16 parts, where the sum of the groups' products begins.
//       V   O^T = V^T P^T sums over the whole sequence, where such an offset would cost accuracy (and carry a NaN of one group into the
//           others): q - 8 by one more fma per pair.
//   * scales are per token and group, so they are applied to sums (K) and to probabilities (V), not to values.
// Queries are scaled by a power of two per row to [2^13, 2^14), so that fp16 holds bf16 ones exactly.  Probabilities times V scales are
// rounded to fp16, relative to the running maximum of (logit + log2 scale): neither large nor tiny values of V leave fp16's range. That
// rounding (2^-11) is an eighth of a bf16 result's own and as large as an fp16 result's.  (A group of channels 2^-r below its token's largest has its
// products at 2^(6-r): normal numbers down to r = 20.)
//
// B=32 Hq=32 Hkv=8, lengths to 8192 (158 MB): 38.4 us and 4.5 us for what was cut, 3.7 TB/s; without its products the first kernel takes
// 32 us (6 us of them before the first page and behind the last), whatever the depth of the ring.  A tile of 16 tokens takes 300
// instructions; at first, with one ring for 16 warps and the products' offsets as start values in registers, 505, and 66 + 10 us.
#include "cache_attend.cuh"
#include "host_common.h"
#include "sm100.cuh"

namespace fmsa {
namespace {

template <bool V> struct Bool { static constexpr bool value = V; };

// Teams of four warps, each with a range of pages, a ring of records and a fifth warp that loads pages and prepares queries; a warp takes 32
// tokens of a page.  (One range and one ring for all warps of an SM, which then wait for one another at the end of every pair, B=32 Hq=32
// Hkv=8, lengths to 8192: 46.7 us against 41.3.)
template <int NT> constexpr int kTeams = NT == 1 ? 4 : 3;
constexpr int kParts = 4;           // halves of a record (K or V: codes and scales) of a team; K's goes back as soon as the logits are known
constexpr int kPartBytes = kRecordBytes / 2, kPartScales = 8192;   // scales behind the codes
static_assert(kKScales == kPartScales && kVCodes == kPartBytes && kVScales == kPartBytes + kPartScales, "the halves look alike");
template <int NT> constexpr int kAttendThreads = (kTeams<NT> + 1) * 128;
// Registers per thread after the warpgroups re-divide the register file.
template <int NT> constexpr int kRegsLaunch = NT == 1 ? 96 : 128;
template <int NT> constexpr int kRegsMath = NT == 1 ? 104 : 152;
template <int NT> constexpr int kRegsLoad = NT == 1 ? 64 : 56;
template <int NT> constexpr bool kRegsBalance = kTeams<NT> * kRegsMath<NT> + kRegsLoad<NT> <= kAttendThreads<NT> / 128 * kRegsLaunch<NT>;
static_assert(kRegsBalance<1> && kRegsBalance<2>, "register re-division must balance");

// Query rows of one block as the second operand of the products, and what belongs to the columns of a product (a lane's: rows
// 8 nt + 2 (lane % 4), + 1).  Every warp's lanes hold the same, so one warp prepares it and the others read it.
template <int NT>
struct Queries {
    uint4 b[NT][4][32];      // [group of 32 channels][lane]: registers of two steps
    uint2 corr[NT][32];      // -8 units * sum of a group's queries in three bf16 parts, the operand beside K's scales
    float2 factor[NT][32];   // product -> logit in the log2 domain
    int2 limit[NT][32];      // tokens the row sees, less the sequence's length
};

constexpr int kNowhere = 0x7fffff80;   // behind every length

template <int NT>
struct AttendTeam {
    Queries<NT> q[2];
    float4 part[4][3][NT][2][32];    // [channels of a group, warp number][other warp][][row 2t, 2t + 1][lane]: what they have of these channels
    float2 ml[4][8 * NT];            // [warp][row]: (reference, sum)
    float2 total[8 * NT];            // [row]: the team's (in a cluster)
    uint64_t full[kParts], empty[kParts], q_full[2], q_empty[2];
    int32_t from[kParts / 2];        // first token of the page whose halves are parts 2 i and 2 i + 1; kNowhere if it does not exist: nothing was loaded
    int32_t first, rest, length;     // sequence in which the range begins, units of it before, its length
};
template <int NT>
struct AttendCtrl {
    AttendTeam<NT> team[kTeams<NT>];
    int32_t sums[32];
};
template <int NT> constexpr size_t kAttendSmem = static_cast<size_t>(kParts) * kTeams<NT> * kPartBytes + sizeof(AttendCtrl<NT>) + 128;
static_assert(kAttendSmem<1> <= 232448 && kAttendSmem<2> <= 232448, "shared memory budget of one CTA");

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0,
                                         float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma16816_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ void scales_of(uint2 w, float (&s)[4]) {   // four bf16
    s[0] = __uint_as_float(w.x << 16);
    s[1] = __uint_as_float(w.x & 0xffff0000u);
    s[2] = __uint_as_float(w.y << 16);
    s[3] = __uint_as_float(w.y & 0xffff0000u);
}
// The token of row r (0..7) of an 8-row block: neighbours of opposite parity everywhere, which the shared-memory reads of K and V both
// need to be free of bank conflicts.
__device__ __forceinline__ int token_of_row(int r) { return r ^ ((r >> 1) & 1); }

template <int NT>
__device__ __forceinline__ void prepare_queries(Queries<NT>& to, const AttendParams& P, const RawQueries& raw, int nt, int lane) {
    const int t = lane & 3;
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
    float part[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] *= e & 1 ? mul * 0.0625f : mul;
        const __half2 a0 = __floats2half2_rn(f[i][0], f[i][4]), a1 = __floats2half2_rn(f[i][2], f[i][6]);
        const __half2 a2 = __floats2half2_rn(f[i][1], f[i][5]), a3 = __floats2half2_rn(f[i][3], f[i][7]);
        to.b[nt][i][lane] = make_uint4(half2_bits(a0), half2_bits(a1), half2_bits(a2), half2_bits(a3));
        const float lo = (__low2float(a0) + __high2float(a0)) + (__low2float(a1) + __high2float(a1));
        const float hi = (__low2float(a2) + __high2float(a2)) + (__low2float(a3) + __high2float(a3));
        float sum = lo + 16.f * hi;
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        part[i] = sum * (-8.f * kUnitLow);
    }
    // as an operand: steps 2t, 2t + 1 of row g are groups 2 (t % 2), + 1; first parts (t < 2) and second ones, then third ones and nothing
    const float c0 = t & 1 ? part[2] : part[0], c1 = t & 1 ? part[3] : part[1];
    const float h0 = __bfloat162float(__float2bfloat16_rn(c0)), h1 = __bfloat162float(__float2bfloat16_rn(c1));
    const float m0 = __bfloat162float(__float2bfloat16_rn(c0 - h0)), m1 = __bfloat162float(__float2bfloat16_rn(c1 - h1));
    to.corr[nt][lane] = make_uint2(t < 2 ? pack_bf16(h0, h1) : pack_bf16(m0, m1), t < 2 ? pack_bf16(c0 - h0 - m0, c1 - h1 - m1) : 0u);
    const float fac = __uint_as_float(static_cast<uint32_t>(127 + 21 - up) << 23) * P.scale_log2e;
    const int lim = raw.limit;
    to.factor[nt][lane] = make_float2(__shfl_sync(0xffffffffu, fac, 8 * t), __shfl_sync(0xffffffffu, fac, 8 * t + 4));
    to.limit[nt][lane] = make_int2(__shfl_sync(0xffffffffu, lim, 8 * t), __shfl_sync(0xffffffffu, lim, 8 * t + 4));
}

// s[j][nt] = {token A x row 2t, A x 2t + 1, B x 2t, B x 2t + 1} in units of 1 / factor, for the tokens of J tiles whose codes (k[j][0], [1])
// and scales (w[j][0], [1]) are given; words: the scales' word t % 2.
template <int NT, int J>
__device__ __forceinline__ void logits(float (&s)[J][NT][4], const uint4 (&k)[J][2], const uint2 (&w)[J][2], const Queries<NT>& Q, int lane) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const uint32_t a = lane & 1 ? w[j][0].y : w[j][0].x, b = lane & 1 ? w[j][1].y : w[j][1].x;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint2 c = Q.corr[nt][lane];
            mma16816_bf16(s[j][nt], a, b, a, b, c.x, c.y);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint4 q = Q.b[nt][i][lane];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const uint32_t a = i == 0 ? k[j][0].x : i == 1 ? k[j][0].y : i == 2 ? k[j][0].z : k[j][0].w;
                const uint32_t c = i == 0 ? k[j][1].x : i == 1 ? k[j][1].y : i == 2 ? k[j][1].z : k[j][1].w;
                const uint32_t a0 = a << 3, c0 = c << 3, a1 = a >> 5, c1 = c >> 5;
                const uint32_t wa = i < 2 ? w[j][0].x : w[j][0].y, wb = i < 2 ? w[j][1].x : w[j][1].y;
                const float fa = __uint_as_float(i & 1 ? wa & 0xffff0000u : wa << 16), fb = __uint_as_float(i & 1 ? wb & 0xffff0000u : wb << 16);
                float d[4];
                mma16816(d, a0 & kLow, c0 & kLow, a1 & kLow, c1 & kLow, q.x, q.y, 0.f, 0.f, 0.f, 0.f);
                mma16816(d, a0 & kHigh, c0 & kHigh, a1 & kHigh, c1 & kHigh, q.z, q.w, d[0], d[1], d[2], d[3]);
                s[j][nt][0] = fmaf(fa, d[0], s[j][nt][0]);
                s[j][nt][1] = fmaf(fa, d[1], s[j][nt][1]);
                s[j][nt][2] = fmaf(fb, d[2], s[j][nt][2]);
                s[j][nt][3] = fmaf(fb, d[3], s[j][nt][3]);
            }
        }
    }
}

// Code q - 8 of nibbles 0 and 4 (bits 0..3 of each half) as fp16, and of nibbles 1 and 5 (bits 4..7): 1024 + q and 1024 + 16 q are what the
// nibble gives under the exponent bits of `magic` (0x64006400: not a constant here, so that it stays in a register and both logical
// operations are one instruction).
__device__ __forceinline__ uint32_t less_eight(uint32_t x, uint32_t magic) {
    const uint32_t y = masked_or(x, 0x000f000fu, magic);
    return half2_bits(__hadd2(*reinterpret_cast<const __half2*>(&y), __float2half2_rn(-1032.f)));
}
__device__ __forceinline__ uint32_t less_eight_high(uint32_t x, uint32_t magic) {
    const uint32_t y = masked_or(x, 0x00f000f0u, magic);
    return half2_bits(__hfma2(*reinterpret_cast<const __half2*>(&y), __float2half2_rn(0.0625f), __float2half2_rn(-72.f)));
}

// Cluster barrier, by every thread of every CTA of the cluster.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
// Address in CTA `rank` of the cluster of what this CTA has at `addr`, and reads there.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// CLUSTER: for few pairs of sequence and KV head and not too many pages: `spread` CTAs, a cluster, share a pair's pages, and its parts meet
// in their shared memory: one launch, and nothing but the result is written.
template <int NT, bool CLUSTER>
__global__ void __launch_bounds__(kAttendThreads<NT>, 1) cache_attend_kernel(const AttendParams P) {
    extern __shared__ uint8_t smem_raw[];
    constexpr int kRows = 8 * NT, kT = kTeams<NT>, kThreads = kAttendThreads<NT>;
    const uint32_t base = (smem_u32(smem_raw) + 127u) & ~127u;
    AttendCtrl<NT>* sm = reinterpret_cast<AttendCtrl<NT>*>(smem_raw + (base - smem_u32(smem_raw)) + kParts * kT * kPartBytes);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    auto BAR = [&](uint64_t& b) { return smem_u32(&b); };

    if (tid < kT) {
        for (int i = 0; i < kParts; ++i) {
            mbar_init(BAR(sm->team[tid].full[i]), 1);
            mbar_init(BAR(sm->team[tid].empty[i]), 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(BAR(sm->team[tid].q_full[i]), 1);
            mbar_init(BAR(sm->team[tid].q_empty[i]), 4);
        }
        fence_mbar_init();
    }
    wait_for_previous_kernel();

    const bool loads = warp >= 4 * kT;
    const int team = loads ? warp - 4 * kT : warp >> 2;
    AttendTeam<NT>* tm = &sm->team[min(team, kT - 1)];
    const uint32_t ring = base + team * kParts * kPartBytes;
    const int per = P.cache.heads * P.blocks, cta = blockIdx.x;
    int units = 0, range = 0, left = 0;
    int seq = 0, length = 0, pages = 1, item = 0, page = 0;   // item: KV head * blocks + block of rows
    Ranges R = {};
    if constexpr (CLUSTER) {
        __syncthreads();   // (the barriers are there)
        const int pair = cta / P.spread;
        seq = pair / per;
        item = pair - seq * per;
        length = P.cache.length(seq);
        pages = (length + kPage - 1) / kPage;
        R = Ranges(pages, P.spread * kT);
        range = team * P.spread + cta % P.spread;
        page = R.begin(range);
        left = team < kT ? R.begin(range + 1) - page : 0;
    } else {
        // ---- the line of pages, and the teams' ranges of it (a unit is a page of a (sequence, KV head, block of rows)); ranges are numbered
        // team by team, so that few units go to as many SMs
        const int seqs = P.cache.seqs;
        // Pages of up to kThreads sequences, from c0 on: what(sequence, its first page, its length, sum so far) for the thread's own; returns the sum.
        auto scan = [&](int c0, int before, auto&& what) {
            const int b = c0 + tid, length = b < seqs ? P.cache.length(b) : 0, p = (length + kPage - 1) / kPage;
            int sum = p;
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            if (lane == 31) sm->sums[warp] = sum;
            __syncthreads();
            const int w = lane < kThreads / 32 ? sm->sums[lane] : 0;
            const int ahead = __reduce_add_sync(0xffffffffu, lane < warp ? w : 0), all = __reduce_add_sync(0xffffffffu, w);
            what(b, before + ahead + sum - p, length, before + all);
            __syncthreads();
            return before + all;
        };
        auto divide = [&](int pages) {
            units = pages * per;
            R = Ranges(units, P.grid * kT);
        };
        auto claim = [&](int b, int at, int length) {
            const int p = (length + kPage - 1) / kPage;
            if (b < seqs && cta == 0) P.prefix[b] = at;
#pragma unroll
            for (int i = 0; i < kT; ++i) {
                const int u = R.begin(i * P.grid + cta);
                if (at * per <= u && u < (at + p) * per) {
                    sm->team[i].first = b;
                    sm->team[i].rest = u - at * per;
                    sm->team[i].length = length;
                }
            }
        };
        int pages_all = 0;
        if (seqs <= kThreads) {
            pages_all = scan(0, 0, [&](int b, int at, int length, int all) { divide(all); claim(b, at, length); });
        } else {
            for (int c0 = 0; c0 < seqs; c0 += kThreads) pages_all = scan(c0, pages_all, [](int, int, int, int) {});
            divide(pages_all);
            int before = 0;
            for (int c0 = 0; c0 < seqs; c0 += kThreads) before = scan(c0, before, [&](int b, int at, int length, int) { claim(b, at, length); });
        }
        if (cta == 0 && tid == 0) P.prefix[seqs] = pages_all;
        if (R.begin(cta) == units) return;   // (nothing for any team)
        range = team * P.grid + cta;
        left = team < kT ? R.begin(range + 1) - R.begin(range) : 0;
        if (left > 0) {
            seq = tm->first;
            length = tm->length;
            pages = (length + kPage - 1) / kPage;
            item = tm->rest / pages;
            page = tm->rest - item * pages;
        }
    }
    uint32_t part = 0, phase = 0, pieces = 0;    // ring position of the next page's K (V's is one further); pieces so far
    bool bad = false;
    auto next = [&](int took) {
        left -= took;
        page = 0;
        ++pieces;
        if (left > 0 && ++item == per) {
            item = 0;
            do length = P.cache.length(++seq); while (length == 0);
            pages = (length + kPage - 1) / kPage;
        }
    };
    auto step = [&]() {
        part ^= 2;
        phase ^= part == 0;
    };
    auto wait = [&](uint32_t bar, uint32_t parity) {   // every lane of the warp calls it; after one that ran out nothing is waited for
        if (!bad) bad = __any_sync(0xffffffffu, !mbar_wait_role(bar, parity));
    };

    if (loads) {
        // =========================== pages and queries ===========================
        reg_dec<kRegsLoad<NT>>();
        while (left > 0) {
            const int take = min(left, pages - page), head = item / P.blocks;
            RawQueries raw;   // (the first eight rows, on their way while the pages are found; the others of a block when they are needed)
            raw.load(P, seq, head, (item - head * P.blocks) * kRows, lane);
            int id = -1;
            for (int i = 0; i < take; ++i) {
                if ((i & 31) == 0) id = i + lane < take ? P.cache.page(seq, page + i + lane) : -1;
                const int pg = __shfl_sync(0xffffffffu, id, i & 31);
                const uint32_t tokens = min(kPage, (length - (page + i) * kPage + 15) & ~15);   // of the last page what is in use
                for (int v = 0; v < 2; ++v) {
                    const uint32_t bar = BAR(tm->full[part + v]), to = ring + (part + v) * kPartBytes;
                    wait(BAR(tm->empty[part + v]), phase ^ 1);   // (the first round finds all parts free)
                    if (!bad && lane == 0) {                     // (after a wait that ran out nothing is asked for; the others give up too)
                        if (v == 0) tm->from[part >> 1] = pg < 0 ? kNowhere : (page + i) * kPage;
                        if (pg < 0) {
                            mbar_arrive(bar);
                        } else {
                            const uint8_t* from = P.cache.record(pg, head) + v * kPartBytes;
                            mbar_arrive_expect_tx(bar, tokens * 72);
                            if (tokens == kPage) {
                                bulk_load(to, from, kPartBytes, bar);
                            } else {
                                bulk_load(to, from, tokens * 64, bar);
                                bulk_load(to + kPartScales, from + kPartScales, tokens * 8, bar);
                            }
                        }
                    }
                }
                __syncwarp();
                step();
                if (i == min(take, kParts / 2) - 1) {
                    const uint32_t slot = pieces & 1;
                    if (pieces >= 2) wait(BAR(tm->q_empty[slot]), (pieces / 2 - 1) & 1);
#pragma unroll 1
                    for (int nt = 0; nt < NT; ++nt) {
                        if (nt) raw.load(P, seq, head, (item - head * P.blocks) * kRows + 8 * nt, lane);
                        prepare_queries<NT>(tm->q[slot], P, raw, nt, lane);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(BAR(tm->q_full[slot]));
                }
            }
            next(take);
        }
        if (CLUSTER) {
            cluster_sync();
            cluster_sync();
        }
    } else {
        // =========================== products ===========================
        reg_inc<kRegsMath<NT>>();
        if (CLUSTER && left == 0 && (warp & 3) == 0 && lane < kRows) tm->total[lane] = make_float2(-INFINITY, 0.f);
        const int g = lane >> 2, t = lane & 3, mine = warp & 3, tile = mine * 32;
        const int tok_a = tile + token_of_row(g), tok_v0 = tile + token_of_row(2 * t), tok_v1 = tile + token_of_row(2 * t + 1);
        const uint32_t k_at = tok_a * 64 + t * 16, s_at = kPartScales + tok_a * 8;
        const uint32_t v0_at = kPartBytes + tok_v0 * 64 + (g ^ (tok_v0 & 4)) * 8, v1_at = kPartBytes + tok_v1 * 64 + (g ^ (tok_v1 & 4)) * 8;
        while (left > 0) {
            const int take = min(left, pages - page);
            const int head = item / P.blocks, block = item - head * P.blocks;
            const Queries<NT>& Q = tm->q[pieces & 1];
            wait(BAR(tm->q_full[pieces & 1]), (pieces / 2) & 1);
            float ref[NT][2], sum[NT][2], o[NT][8][4];
            float2 factor[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                factor[nt] = Q.factor[nt][lane];
                ref[nt][0] = ref[nt][1] = -INFINITY;
                sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
                for (int m = 0; m < 8; ++m)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[nt][m][c] = 0.f;
            }
            // Two tiles of 16 tokens.  EDGE: some of them are not seen by some row, or are not there (their bytes may be anything).
            auto two_tiles = [&](auto edge, const uint8_t* at, int first) {
                constexpr bool EDGE = decltype(edge)::value;
                float s[2][NT][4];
                {
                    uint4 kc[2][2];
                    uint2 ks[2][2];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            kc[j][y] = *reinterpret_cast<const uint4*>(at + k_at + (2 * j + y) * 512);
                            ks[j][y] = *reinterpret_cast<const uint2*>(at + s_at + (2 * j + y) * 64);
                        }
                    logits<NT, 2>(s, kc, ks, Q, lane);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(BAR(tm->empty[part]));
                wait(BAR(tm->full[part + 1]), phase);
                uint32_t pb[2][NT][4][2];   // p * scale of the four groups, as the second operand
                uint2 vs[2][2];
                float x[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = -INFINITY;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        vs[j][y] = *reinterpret_cast<const uint2*>(at + kPartBytes + s_at + (2 * j + y) * 64);
                        const int place = first + tok_a + 16 * j + 8 * y - length;
                        if (EDGE && place >= 0) vs[j][y] = make_uint2(0, 0);
                        // log2 of the largest scale (a word as it stands is its upper half and less than one of its steps)
                        const float lg = fast_log2(fmaxf(fmax3(__uint_as_float(vs[j][y].x), __uint_as_float(vs[j][y].x << 16), __uint_as_float(vs[j][y].y)),
                                                         fmaxf(__uint_as_float(vs[j][y].y << 16), 8.27e-25f)));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            s[j][nt][2 * y] *= factor[nt].x;
                            s[j][nt][2 * y + 1] *= factor[nt].y;
                            if (EDGE) {
                                const int2 lim = Q.limit[nt][lane];
                                if (place >= lim.x) s[j][nt][2 * y] = -INFINITY;
                                if (place >= lim.y) s[j][nt][2 * y + 1] = -INFINITY;
                            }
                            x[nt][0] = fmaxf(x[nt][0], s[j][nt][2 * y] + lg);
                            x[nt][1] = fmaxf(x[nt][1], s[j][nt][2 * y + 1] + lg);
                        }
                    }
                // the reference: raised, for every row by what it needs, when one is exceeded by more than the slack
                bool raise = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) raise |= x[nt][0] > ref[nt][0] + (kLift + kSlack) || x[nt][1] > ref[nt][1] + (kLift + kSlack);
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float top = x[nt][c];
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                            top = fmaxf(top - kLift, ref[nt][c]);
                            const float by = ref[nt][c] == -INFINITY ? 0.f : fast_exp2(ref[nt][c] - top);
                            ref[nt][c] = top;
                            sum[nt][c] *= by;
#pragma unroll
                            for (int m = 0; m < 8; ++m) {
                                o[nt][m][c] *= by;
                                o[nt][m][c + 2] *= by;
                            }
                        }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        float v[4];
                        scales_of(vs[j][y], v);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float r0 = EDGE && ref[nt][0] == -INFINITY ? 0.f : ref[nt][0], r1 = EDGE && ref[nt][1] == -INFINITY ? 0.f : ref[nt][1];
                            const float p0 = fast_exp2(s[j][nt][2 * y] - r0), p1 = fast_exp2(s[j][nt][2 * y + 1] - r1);
                            sum[nt][0] += p0;
                            sum[nt][1] += p1;
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t w = half2_bits(__floats2half2_rn(p0 * v[c], p1 * v[c]));
                                // (0 * NaN: a token that is not finite is nothing to rows that do not see it)
                                if (EDGE) w &= (p0 == 0.f ? 0u : 0xffffu) | (p1 == 0.f ? 0u : 0xffff0000u);
                                pb[j][nt][c][y] = transpose8x8(w);
                            }
                        }
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint2 v0 = *reinterpret_cast<const uint2*>(at + v0_at + j * 1024), v1 = *reinterpret_cast<const uint2*>(at + v1_at + j * 1024);
                    const uint2 v2 = *reinterpret_cast<const uint2*>(at + v0_at + j * 1024 + 512), v3 = *reinterpret_cast<const uint2*>(at + v1_at + j * 1024 + 512);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t sel = i & 1 ? 0x7632u : 0x5410u;
                        const uint32_t xx = __byte_perm(i < 2 ? v0.x : v0.y, i < 2 ? v1.x : v1.y, sel);   // four channels of tokens 2t, 2t + 1
                        const uint32_t yy = __byte_perm(i < 2 ? v2.x : v2.y, i < 2 ? v3.x : v3.y, sel);   // ... and of the two 8 further
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t x1 = h ? xx >> 8 : xx, y1 = h ? yy >> 8 : yy;
                            const uint32_t a0 = less_eight(x1, P.magic), a1 = less_eight_high(x1, P.magic);
                            const uint32_t a2 = less_eight(y1, P.magic), a3 = less_eight_high(y1, P.magic);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float(&d)[4] = o[nt][2 * i + h];
                                mma16816(d, a0, a1, a2, a3, pb[j][nt][i][0], pb[j][nt][i][1], d[0], d[1], d[2], d[3]);
                            }
                        }
                    }
                }
            };
#pragma unroll 1
            for (int i = 0; i < take; ++i) {
                wait(BAR(tm->full[part]), phase);
                const int first = tm->from[part >> 1];   // first token of the page
                if (!bad && first + tile < length) {
                    const uint8_t* at = smem_raw + (ring - smem_u32(smem_raw)) + part * kPartBytes;
                    if (first + kPage > length - P.n + 1) two_tiles(Bool<true>(), at, first);
                    else two_tiles(Bool<false>(), at, first);
                } else {
                    wait(BAR(tm->full[part + 1]), phase);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(BAR(tm->empty[part]));
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(BAR(tm->empty[part + 1]));
                step();
            }
            if (lane == 0) mbar_arrive(BAR(tm->q_empty[pieces & 1]));
            // ---- the end of a piece: warp w takes the channels of group w from the other three
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float l = sum[nt][c];
                    l += __shfl_xor_sync(0xffffffffu, l, 4);
                    l += __shfl_xor_sync(0xffffffffu, l, 8);
                    l += __shfl_xor_sync(0xffffffffu, l, 16);
                    if (g == 0) tm->ml[mine][nt * 8 + 2 * t + c] = make_float2(ref[nt][c], l);
                }
            float4 own[NT][2] = {};   // channels 32 w + 4 g ..: rows g and g + 8 of two operand tiles
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float4 x = make_float4(o[nt][2 * i][c], o[nt][2 * i][c + 2], o[nt][2 * i + 1][c], o[nt][2 * i + 1][c + 2]);
                        if (i == mine) own[nt][c] = x;
                        else tm->part[i][(mine - i + 3) & 3][nt][c][lane] = x;   // (warp i + 1 + y, modulo 4, is number y)
                    }
            named_barrier_sync(1 + team, 128);
            const bool whole = !CLUSTER && page == 0 && take == pages;
            if (!CLUSTER && page == 0 && mine == 0 && lane == 0) {   // (the part that begins a pair says where its parts are)
                const int behind = R.begin(range + 1) - left + pages;   // the unit behind the pair's last
                P.parts[static_cast<int64_t>(seq) * per + item] = make_int2(2 * range + (pieces ? 1 : 0), whole ? 0 : R.owner(behind - 1) - range + 1);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int r = nt * 8 + 2 * t + c, row = block * kRows + r;
                    const float2 ml[4] = {tm->ml[0][r], tm->ml[1][r], tm->ml[2][r], tm->ml[3][r]};
                    const float top = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), m = top == -INFINITY ? 0.f : top;
                    float l = 0.f;
#pragma unroll
                    for (int y = 0; y < 4; ++y) l = fmaf(ml[y].y, fast_exp2(ml[y].x - m), l);
                    float by = fast_exp2(ref[nt][c] - m);
                    float4 acc = make_float4(own[nt][c].x * by, own[nt][c].y * by, own[nt][c].z * by, own[nt][c].w * by);
#pragma unroll
                    for (int y = 0; y < 3; ++y) {
                        const float4 x = tm->part[mine][y][nt][c][lane];
                        by = fast_exp2(tm->ml[(mine + 1 + y) & 3][r].x - m);
                        acc = make_float4(fmaf(x.x, by, acc.x), fmaf(x.y, by, acc.y), fmaf(x.z, by, acc.z), fmaf(x.w, by, acc.w));
                    }
                    if (row >= P.rows) continue;
                    const int ch = 32 * mine + 4 * g;
                    if (CLUSTER) {   // (where the team's pages were: all of them have been read)
                        *reinterpret_cast<float4*>(smem_raw + (ring - smem_u32(smem_raw)) + (r * kHeadDim + ch) * 4) = acc;
                        if (ch == 0) tm->total[r] = make_float2(top, l);
                    } else if (whole) {
                        const int hh = row / P.n, j = row - hh * P.n, h = head * P.group + hh;
                        if (P.sinks) l += fast_exp2(P.sinks[h] * kLog2e - m);
                        const float inv = l == 0.f ? 0.f : 1.f / l;
                        uint2 y;
                        y.x = P.fp16 ? pack_act<true>(acc.x * inv, acc.y * inv) : pack_act<false>(acc.x * inv, acc.y * inv);
                        y.y = P.fp16 ? pack_act<true>(acc.z * inv, acc.w * inv) : pack_act<false>(acc.z * inv, acc.w * inv);
                        *reinterpret_cast<uint2*>(P.out + ((static_cast<int64_t>(seq) * P.n + j) * P.Hq + h) * kHeadDim + ch) = y;
                        if (ch == 0) P.lse[(static_cast<int64_t>(seq) * P.cache.heads + head) * P.lse_rows + row] = m + fast_log2(l);
                    } else {
                        const int64_t slot = 2LL * range + (pieces ? 1 : 0);
                        *reinterpret_cast<float4*>(P.o_part + (slot * kRows + r) * kHeadDim + ch) = acc;
                        if (ch == 0) P.ml_part[slot * kRows + r] = make_float2(top, l);
                    }
                }
            named_barrier_sync(1 + team, 128);
            next(take);
        }
        if (CLUSTER) {
            cluster_sync();
            const int head = item / P.blocks, block = item - head * P.blocks, parts = P.spread * kT;   // at most 32; team p / spread of CTA p % spread
            const int shift = __ffs(P.spread) - 1, low = P.spread - 1;
            const uint32_t all_rings = base, totals = smem_u32(sm->team[0].total);
            for (int r = (cta & low) + (warp << shift); r < kRows; r += (4 * kT) << shift) {
                const int row = block * kRows + r;
                if (row >= P.rows) break;
                float2 ml = make_float2(-INFINITY, 0.f);
                if (lane < parts) ml = ld_cluster_v2(in_cta(totals + (lane >> shift) * static_cast<int>(sizeof(AttendTeam<NT>)) + r * 8, lane & low));
                float top = ml.x;
                for (int o2 = 16; o2; o2 >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o2));
                const float m = top == -INFINITY ? 0.f : top, by = fast_exp2(ml.x - m);
                float l = ml.y * by;
                for (int o2 = 16; o2; o2 >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o2);
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                for (uint32_t live = __ballot_sync(0xffffffffu, by != 0.f); live;) {   // the parts that have something, eight reads at once
                    float f[8];
                    float4 x[8];
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        const int p = live ? __ffs(live) - 1 : 0;
                        f[y] = __shfl_sync(0xffffffffu, by, p);
                        x[y] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (live) x[y] = ld_cluster_v4(in_cta(all_rings + (p >> shift) * (kParts * kPartBytes) + (r * kHeadDim + 4 * lane) * 4, p & low));
                        else f[y] = 0.f;
                        live &= live - 1;
                    }
#pragma unroll
                    for (int y = 0; y < 8; ++y) acc = make_float4(fmaf(x[y].x, f[y], acc.x), fmaf(x[y].y, f[y], acc.y), fmaf(x[y].z, f[y], acc.z), fmaf(x[y].w, f[y], acc.w));
                }
                const int hh = row / P.n, j = row - hh * P.n, h = head * P.group + hh;
                if (P.sinks) l += fast_exp2(P.sinks[h] * kLog2e - m);
                const float inv = l == 0.f ? 0.f : 1.f / l;
                uint2 y;
                y.x = P.fp16 ? pack_act<true>(acc.x * inv, acc.y * inv) : pack_act<false>(acc.x * inv, acc.y * inv);
                y.y = P.fp16 ? pack_act<true>(acc.z * inv, acc.w * inv) : pack_act<false>(acc.z * inv, acc.w * inv);
                *reinterpret_cast<uint2*>(P.out + ((static_cast<int64_t>(seq) * P.n + j) * P.Hq + h) * kHeadDim + 4 * lane) = y;
            }
            cluster_sync();   // (no CTA leaves while another one reads from it)
        }
    }
    if (bad) {
        atomicMax(P.cache.status, kStatusWaitTimeout);
        const uint64_t t0 = global_timer_ns();   // copies in flight land before shared memory is given back
        while (global_timer_ns() - t0 < 200000) __nanosleep(1000);
    }
}

// Merges what ranges cut.  A pair's parts are the slot its first range names, then slot 2 r of the ranges r behind it.  A warp has a row,
// four channels a lane; WARPS: 1, or 16 that share the parts of one row where few pairs are cut into many.  Sequences without a token get
// their zeros here.
template <int NT, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : 32 * WARPS) cache_combine_kernel(const AttendParams P) {
    constexpr int kRows = 8 * NT;
    __shared__ float4 acc_of[WARPS][32];
    __shared__ float2 ml_of[WARPS];
    wait_for_previous_kernel();
    const int per = P.cache.heads * P.blocks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = WARPS == 1 ? blockIdx.y * 4 + warp : blockIdx.y, seq = blockIdx.x / per, item = blockIdx.x % per;
    const int head = item / P.blocks, row = (item % P.blocks) * kRows + r;
    if (r >= kRows || row >= P.rows) return;
    const int2 parts = P.parts[blockIdx.x];
    const bool none = P.cache.length(seq) == 0;
    if (!none && parts.y == 0) return;
    const int hh = row / P.n, j = row - hh * P.n, h = head * P.group + hh;
    const float sink = P.sinks ? P.sinks[h] * kLog2e : -INFINITY;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    if (!none) {
        constexpr int kAtOnce = WARPS == 1 ? 4 : 8;
        for (int i0 = WARPS == 1 ? 0 : warp; i0 < parts.y; i0 += kAtOnce * WARPS) {
            float2 ml[kAtOnce];
            float4 x[kAtOnce];
#pragma unroll
            for (int y = 0; y < kAtOnce; ++y) {
                const int i = i0 + y * WARPS;
                const int64_t at = static_cast<int64_t>(i == 0 ? parts.x : 2 * (parts.x / 2 + i)) * kRows + r;
                ml[y] = i < parts.y ? P.ml_part[at] : make_float2(-INFINITY, 0.f);
                x[y] = i < parts.y ? *reinterpret_cast<const float4*>(P.o_part + at * kHeadDim + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            float top = m;
#pragma unroll
            for (int y = 0; y < kAtOnce; ++y) top = fmaxf(top, ml[y].x);
            const float ref = top == -INFINITY ? 0.f : top;
            const float old = fast_exp2(m - ref);
            acc = make_float4(acc.x * old, acc.y * old, acc.z * old, acc.w * old);
            l *= old;
            m = top;
#pragma unroll
            for (int y = 0; y < kAtOnce; ++y) {
                const float by = fast_exp2(ml[y].x - ref);
                l = fmaf(ml[y].y, by, l);
                acc = make_float4(fmaf(x[y].x, by, acc.x), fmaf(x[y].y, by, acc.y), fmaf(x[y].z, by, acc.z), fmaf(x[y].w, by, acc.w));
            }
        }
        if (WARPS > 1) {
            acc_of[warp][lane] = acc;
            if (lane == 0) ml_of[warp] = make_float2(m, l);
            __syncthreads();
            if (warp > 0) return;
            float top = m;
            for (int w = 1; w < WARPS; ++w) top = fmaxf(top, ml_of[w].x);
            const float ref = top == -INFINITY ? 0.f : top;
            const float old = fast_exp2(m - ref);
            acc = make_float4(acc.x * old, acc.y * old, acc.z * old, acc.w * old);
            l *= old;
            m = top;
#pragma unroll
            for (int w = 1; w < WARPS; ++w) {
                const float by = fast_exp2(ml_of[w].x - ref);
                const float4 x = acc_of[w][lane];
                l = fmaf(ml_of[w].y, by, l);
                acc = make_float4(fmaf(x.x, by, acc.x), fmaf(x.y, by, acc.y), fmaf(x.z, by, acc.z), fmaf(x.w, by, acc.w));
            }
        }
    }
    if (WARPS > 1 && warp > 0) return;
    m = m == -INFINITY ? 0.f : m;
    l += fast_exp2(sink - m);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint2 y;
    y.x = P.fp16 ? pack_act<true>(acc.x * inv, acc.y * inv) : pack_act<false>(acc.x * inv, acc.y * inv);
    y.y = P.fp16 ? pack_act<true>(acc.z * inv, acc.w * inv) : pack_act<false>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(P.out + ((static_cast<int64_t>(seq) * P.n + j) * P.Hq + h) * kHeadDim + 4 * lane) = y;
    if (lane == 0) P.lse[(static_cast<int64_t>(seq) * P.cache.heads + head) * P.lse_rows + row] = m + fast_log2(l);
}

// The probabilities of every token, summed over the query rows of its KV head: the logits once more (half of the cache's bytes, most of
// them still in L2), relative to the log-sum-exps that are known now.  (Keeping the logits of the first kernel instead would move 4 bytes
// per row and token twice, as much as K's 72 bytes from nine rows on, and needs a buffer for the longest lengths.)  A block takes a range
// of the pages of all (sequence, KV head) pairs, a warp tiles of 16 tokens; all rows' queries lie in shared memory.
constexpr int kWeightWarps = 8;
template <int NT>
struct WeightRows {
    Queries<NT> q;
    float2 lse[NT][32];
};
template <int NT>
__global__ void __launch_bounds__(kWeightWarps * 32, 2) cache_weights_kernel(const AttendParams P, int held) {
    extern __shared__ uint8_t smem_raw[];
    WeightRows<NT>* rows = reinterpret_cast<WeightRows<NT>*>(smem_raw);   // [held]: blocks of rows
    wait_for_previous_kernel();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, heads = P.cache.heads;
    const long long units = static_cast<long long>(P.prefix[P.cache.seqs]) * heads;
    const long long u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
    if (u0 == u1) return;
    __shared__ int begins;   // the sequence in whose pages the range begins
    for (int b = threadIdx.x; b < P.cache.seqs; b += kWeightWarps * 32)
        if (static_cast<long long>(P.prefix[b]) * heads <= u0 && u0 < static_cast<long long>(P.prefix[b + 1]) * heads) begins = b;
    __syncthreads();
    const int tok = token_of_row(g);
    long long u = u0;
    for (int seq = begins; u < u1; ++seq) {
        const long long begin = static_cast<long long>(P.prefix[seq]) * heads;
        const int pages = P.prefix[seq + 1] - P.prefix[seq], length = P.cache.length(seq);
        while (u < u1 && u < begin + static_cast<long long>(pages) * heads) {
            const int head = static_cast<int>((u - begin) / pages), page = static_cast<int>((u - begin) % pages);
            const int take = static_cast<int>(min(u1 - u, static_cast<long long>(pages - page)));
            for (int lot = 0; lot < P.blocks; lot += held) {   // (more rows than shared memory holds go lot by lot)
                const int n = min(held, P.blocks - lot);
                __syncthreads();
                for (int i = warp; i < n * NT; i += kWeightWarps) {
                    RawQueries raw;
                    raw.load(P, seq, head, (lot * NT + i) * 8, lane);
                    prepare_queries<NT>(rows[i / NT].q, P, raw, i % NT, lane);
                    const int row = (lot * NT + i) * 8 + 2 * t;
                    const float* lse = P.lse + (static_cast<int64_t>(seq) * heads + head) * P.lse_rows + row;
                    rows[i / NT].lse[i % NT][lane] = make_float2(row < P.rows ? lse[0] : 0.f, row + 1 < P.rows ? lse[1] : 0.f);
                }
                __syncthreads();
                // Warp w has tile w of every page.
                uint4 kc[1][2], kn[2] = {};
                uint2 ks[1][2], kt[2] = {};
                int ids = -1, pn = -1;
                auto fetch = [&](int i) {   // codes and scales of page i's tokens
                    if ((i & 31) == 0) ids = i + lane < take ? P.cache.page(seq, page + i + lane) : -1;
                    pn = __shfl_sync(0xffffffffu, ids, i & 31);
                    if (i >= take || pn < 0) return;
                    const uint8_t* from = P.cache.record(pn, head);
                    const int at = warp * 16 + tok;
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        kn[y] = *reinterpret_cast<const uint4*>(from + kKCodes + (at + 8 * y) * 64 + t * 16);
                        kt[y] = *reinterpret_cast<const uint2*>(from + kKScales + (at + 8 * y) * 8);
                    }
                };
                fetch(0);
                for (int i0 = 0; i0 < take; ++i0) {
                    const int pg = pn, pa = (page + i0) * kPage + warp * 16 + tok - length, pb = pa + 8;
                    if (pa - tok >= 0) break;   // (no token of the tile is there)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        kc[0][y] = kn[y];
                        ks[0][y] = kt[y];
                    }
                    fetch(i0 + 1);
                    if (pg < 0) continue;
                    float wa = 0.f, wb = 0.f;
#pragma unroll 1
                    for (int i = 0; i < n; ++i) {
                        const Queries<NT>& Q = rows[i].q;
                        float s[1][NT][4];
                        logits<NT, 1>(s, kc, ks, Q, lane);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float2 f = Q.factor[nt][lane], lse = rows[i].lse[nt][lane];
                            const int2 lim = Q.limit[nt][lane];
                            wa += pa < lim.x ? fast_exp2(fmaf(s[0][nt][0], f.x, -lse.x)) : 0.f;
                            wa += pa < lim.y ? fast_exp2(fmaf(s[0][nt][1], f.y, -lse.y)) : 0.f;
                            wb += pb < lim.x ? fast_exp2(fmaf(s[0][nt][2], f.x, -lse.x)) : 0.f;
                            wb += pb < lim.y ? fast_exp2(fmaf(s[0][nt][3], f.y, -lse.y)) : 0.f;
                        }
                    }
                    wa += __shfl_xor_sync(0xffffffffu, wa, 1);
                    wb += __shfl_xor_sync(0xffffffffu, wb, 1);
                    wa += __shfl_xor_sync(0xffffffffu, wa, 2);
                    wb += __shfl_xor_sync(0xffffffffu, wb, 2);
                    if (t < 2 && (t ? pb : pa) < 0) {
                        float* to = P.weights + (static_cast<int64_t>(pg) * heads + head) * kPage + warp * 16 + tok + 8 * t;
                        const float w = t ? wb : wa;
                        *to = lot || P.accumulate ? *to + w : w;
                    }
                }
            }
            u += take;
        }
    }
}

struct AttendSpace {
    int64_t prefix, parts, o_part, ml_part, lse, bytes;
};
// How a call is done: eights of rows of a block; whether a page is unpacked into shared memory (cache_rows.cu); ranges of a CTA; CTAs of a
// cluster that shares a pair of sequence and KV head (0: none).
struct Form {
    int nt, by_rows, teams, spread;
};
Form form_of(const fmsa_cache4& c, int64_t rows, bool weights, int sms);
AttendSpace carve_attend(const Form& form, int seqs, int heads, int64_t rows, int grid) {
    const int64_t block = 8 * form.nt;
    AttendSpace w;
    int64_t off = 0;
    auto take = [&](int64_t bytes) {
        const int64_t at = off;
        off += round_up(bytes, 256);
        return at;
    };
    w.prefix = take(4LL * (seqs + 1));
    w.parts = take(8LL * seqs * heads * (round_up(rows, block) / block));
    const int64_t ranges = static_cast<int64_t>(grid) * form.teams;
    w.o_part = take(2 * ranges * block * kHeadDim * 4);
    w.ml_part = take(2 * ranges * block * 8);
    w.lse = take(4LL * seqs * heads * round_up(rows, block));
    w.bytes = off;
    return w;
}

constexpr int kWeightBlocks = 7;   // blocks of rows whose queries the weights kernel holds at once: 44 KB
static_assert(kWeightBlocks * sizeof(WeightRows<2>) <= 48 * 1024, "more needs an attribute");
Form form_of(const fmsa_cache4& c, int64_t rows, bool weights, int sms) {
    const int64_t pairs = static_cast<int64_t>(c.seqs) * c.heads, pages = pairs * c.width;   // (at the longest lengths that the table can hold)
    // Nine to sixteen rows: unpacking into shared memory costs less where a CTA has few pages, and with weights, whose second pass it shortens;
    // over many pages a tile's shorter way through registers counts.  (Through registers -> this way, 16 rows, 2 heads: one sequence of 4K
    // 13.0 -> 9.5 us, 32 of 8K 32.8 -> 36.3, with weights 59.0 -> 58.1; 12 rows, 1 head: one of 64K (6.9 pages an SM) 18.1 -> 16.7, 32 of 8K
    // (13.8) 21.7 -> 24.0, with weights 39.9 -> 36.9.  20 rows, 4 heads, 32 of 8K: 92.5 -> 71.2, with weights 153 -> 111.)
    if (rows > 16 || (rows > 8 && (weights || pages <= 8LL * sms))) return {rows_of_block(rows) / 8, 1, 1, 0};
    // Clusters: a power of two up to 8 that fits the GPU, where a team's pages are at most one more than with all SMs' teams on all pages.
    // (The weights need what the other form leaves in the workspace.)
    Form f = {rows > 8 ? 2 : 1, 0, rows > 8 ? kTeams<2> : kTeams<1>, 0};
    if (weights || pairs * 2 > sms) return f;
    int spread = 2;
    while (spread < 8 && pairs * spread * 2 <= sms) spread *= 2;
    auto rounds = [](int64_t pages, int64_t by) { return (pages + by - 1) / by; };
    if (rounds(c.width, spread * f.teams) <= rounds(pages, static_cast<int64_t>(sms) * f.teams) + 1) f.spread = spread;
    return f;
}

template <int NT>
bool launch_attend(const AttendParams& P, cudaStream_t st) {
    if (P.spread) {
        const auto kernel = cache_attend_kernel<NT, true>;
        if (!ensure_smem_attr(reinterpret_cast<const void*>(kernel), kAttendSmem<NT>)) return false;
        launch_clusters(kernel, P.cache.seqs * P.cache.heads * P.spread, P.spread, kAttendThreads<NT>, kAttendSmem<NT>, st, P);
        return true;
    }
    const auto kernel = cache_attend_kernel<NT, false>;
    if (!ensure_smem_attr(reinterpret_cast<const void*>(kernel), kAttendSmem<NT>)) return false;
    launch_chained(kernel, P.grid, kAttendThreads<NT>, kAttendSmem<NT>, st, P);
    return true;
}
// Everything behind the first kernel.
template <int NT>
void launch_combine(const AttendParams& P, int teams, cudaStream_t st) {
    // A pair is cut into about ranges / pairs parts (+ 1): 16 warps a row where that is many.
    const int64_t pairs = static_cast<int64_t>(P.cache.seqs) * P.cache.heads * P.blocks;
    const int rows = P.rows < 8 * NT ? P.rows : 8 * NT;
    if (pairs * 16 < P.grid * teams) launch_chained(cache_combine_kernel<NT, 16>, dim3(static_cast<unsigned>(pairs), rows), 512, 0, st, P);
    else launch_chained(cache_combine_kernel<NT, 1>, dim3(static_cast<unsigned>(pairs), (rows + 3) / 4), 128, 0, st, P);
}
template <int NT>
void launch_weights(const AttendParams& P, cudaStream_t st) {
    const int held = P.blocks < kWeightBlocks ? P.blocks : kWeightBlocks;
    launch_chained(cache_weights_kernel<NT>, device_sm_count() * 2, kWeightWarps * 32, held * sizeof(WeightRows<NT>), st, P, held);
}
int launch_all(const AttendParams& P, const Form& form, cudaStream_t st) {
    if (!(form.by_rows ? launch_attend_rows(P, st) : form.nt == 1 ? launch_attend<1>(P, st) : launch_attend<2>(P, st))) return FMSA_ERR_CUDA;
    if (!P.spread) {
        switch (form.nt) {
            case 1: launch_combine<1>(P, form.teams, st); break;
            case 2: launch_combine<2>(P, form.teams, st); break;
            case 4: launch_combine<4>(P, form.teams, st); break;
            case 6: launch_combine<6>(P, form.teams, st); break;
            default: launch_combine<8>(P, form.teams, st);
        }
    }
    if (P.weights) {
        if (!form.by_rows) {
            launch_weights<1>(P, st);
        } else if (P.blocks == 1) {
            if (!launch_weights_rows(P, st)) return FMSA_ERR_CUDA;
        } else {   // (a token's rows in several blocks: one kernel has to have them all)
            AttendParams W = P;
            W.blocks = (P.rows + 15) / 16;
            launch_weights<2>(W, st);
        }
    }
    return check_launch();
}

}  // namespace
}  // namespace fmsa

extern "C" int32_t fmsa_cache_attend_launches(int32_t seqs, int32_t Hq, int32_t heads, int32_t n, int32_t width, int32_t weights) {
    using namespace fmsa;
    const int sms = device_sm_count();
    if (seqs <= 0 || heads <= 0 || Hq <= 0 || Hq % heads || n <= 0 || width <= 0 || sms <= 0) return -1;
    fmsa_cache4 c = {};
    c.seqs = seqs; c.heads = heads; c.width = width;
    return weights ? 3 : form_of(c, static_cast<int64_t>(Hq / heads) * n, false, sms).spread ? 1 : 2;
}

extern "C" int64_t fmsa_cache_attend_workspace_bytes(int32_t seqs, int32_t Hq, int32_t heads, int32_t n, int32_t width, int32_t weights) {
    using namespace fmsa;
    const int sms = device_sm_count();
    if (seqs <= 0 || heads <= 0 || Hq <= 0 || Hq % heads || n <= 0 || width <= 0 || sms <= 0) return -1;
    fmsa_cache4 c = {};
    c.seqs = seqs; c.heads = heads; c.width = width;
    const int64_t rows = static_cast<int64_t>(Hq / heads) * n;
    const Form form = form_of(c, rows, weights != 0, sms);
    return form.spread ? 0 : carve_attend(form, seqs, heads, rows, sms).bytes;
}

extern "C" int fmsa_cache_attend(const fmsa_cache_attend_args* args, void* stream) {
    using namespace fmsa;
    FMSA_REQUIRE(args);
    const fmsa_cache4* cache = &args->cache;
    const fmsa_tensor* q = &args->q;
    const int32_t Hq = args->Hq, n = args->n, dtype = args->dtype;
    int32_t* status = args->status;
    void *out = args->out, *workspace = args->workspace;
    FMSA_REQUIRE(cache4_ok(cache) && q->ptr && out && status && Hq > 0 && n > 0 && Hq % cache->heads == 0);
    FMSA_REQUIRE(dtype == FMSA_DTYPE_BF16 || dtype == FMSA_DTYPE_FP16);
    FMSA_REQUIRE(aligned16(q->ptr) && q->stride_b % 8 == 0 && q->stride_h % 8 == 0 && q->stride_s % 8 == 0);
    const int64_t rows = static_cast<int64_t>(Hq / cache->heads) * n;
    const int sms = device_sm_count();
    const Form form = form_of(*cache, rows, args->weights != nullptr, sms);
    const int64_t block = 8 * form.nt, blocks = (rows + block - 1) / block, items = blocks * cache->heads * cache->seqs;
    if (items > 0x7fffffffLL || items * cache->width > 0x7fffffffLL) return FMSA_ERR_UNSUPPORTED;   // (units are counted in 32 bits)
    AttendParams P = {};
    P.grid = sms;
    P.spread = form.spread;
    AttendSpace w = {};
    if (!P.spread) {
        FMSA_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0);
        w = carve_attend(form, cache->seqs, cache->heads, rows, sms);
        if (args->workspace_bytes < w.bytes) return FMSA_ERR_WORKSPACE;
    }
    if (sms <= 0) return FMSA_ERR_CUDA;
    char* ws = static_cast<char*>(workspace);
    P.cache = device_cache(cache, status);
    P.q = static_cast<const uint16_t*>(q->ptr);
    P.qs[0] = q->stride_b; P.qs[1] = q->stride_h; P.qs[2] = q->stride_s;
    P.sinks = args->sinks;
    P.out = static_cast<uint16_t*>(out);
    P.weights = args->weights;
    P.prefix = reinterpret_cast<int32_t*>(ws + w.prefix);
    P.parts = reinterpret_cast<int2*>(ws + w.parts);
    P.o_part = reinterpret_cast<float*>(ws + w.o_part);
    P.ml_part = reinterpret_cast<float2*>(ws + w.ml_part);
    P.lse = reinterpret_cast<float*>(ws + w.lse);
    P.Hq = Hq; P.n = n; P.group = Hq / cache->heads; P.rows = static_cast<int32_t>(rows); P.blocks = static_cast<int32_t>(blocks);
    P.lse_rows = static_cast<int32_t>(blocks * block);
    P.fp16 = dtype == FMSA_DTYPE_FP16; P.accumulate = args->accumulate ? 1 : 0;
    P.scale_log2e = args->scale * kLog2e;
    P.magic = 0x64006400u;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return launch_all(P, form, st);
}
