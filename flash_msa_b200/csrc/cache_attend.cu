// Attention over the cache held in 4 bits: the last few tokens of every sequence, their heads sharing KV heads.
//
// Bound by HBM: 144 bytes per token and KV head are read once, whatever the number of query rows (heads of the group x new tokens).  So the
// kernel is built around a pipe that never empties and around few instructions per nibble:
//   * the pages of all (sequence, KV head) pairs stand in one line that is cut into equal ranges, one per SM: a long sequence is split, short
//     ones share an SM, and nothing depends on lengths the host would have to know.  At most two pieces of a range are parts of a cut
//     pair; they go to the workspace and a second kernel merges them.
//   * one warp keeps kStages records in flight (one bulk copy of 18 KB each), the others take 16 tokens of a page each;
//   * products on mma.sync m16n8k16 with the cache as the 16-row operand and 8 query rows beside it.  (tcgen05 wants its cache operand
//     from shared memory: the 16-bit copy of every nibble would be written and read there, four times the bytes that come in.)  A word of
//     eight nibbles gives four operand registers with a mask each:
//       K   S^T = K Q^T: nibbles 0, 2, 4, 6 (0x000f000f) are fp16 denormals q * 2^-24 as they stand, nibbles 1, 3, 5, 7 (0x00f000f0)
//           q * 2^-20, which queries divided by 16 make up for; the 8 of (q - 8) is a start value of the sum, -8 * sum(Q) per group.  So a
//           K nibble costs 5/8 instruction.  The start value costs no accuracy: a group's sum has two steps.
//       V   O^T = V^T P^T sums over the whole sequence, where such a start value would cost accuracy: the nibbles become q - 8 (fp16) by
//           one more fma per pair (1024 + q and 1024 + 16 q are what a mask with 0x6400 gives).
//   * scales are per token and group, so they are applied to sums (K) and to probabilities (V), not to values.
// Queries are scaled by a power of two per row to [2^13, 2^14), so that fp16 holds bf16 ones exactly.  Probabilities times V scales are
// fp16 relative to the running maximum of (logit + log2 scale): neither large nor tiny values of V leave fp16's range.
#include "cache4.cuh"
#include "host_common.h"
#include "sm100.cuh"

namespace fmsa {
namespace {

struct AttendParams {
    Cache4 cache;
    const uint16_t* q;          // (seqs,Hq,n,128)
    int64_t qs[3];
    const float* sinks;         // [Hq] or null
    uint16_t* out;              // [seqs][n][Hq*128]
    float* weights;             // [pages][heads][128] or null
    int32_t* prefix;            // [seqs + 1]: pages of the sequences before
    float* o_part;              // [2 * grid][rows of a block][128]
    float2* ml_part;            // [2 * grid][rows of a block]: (reference, sum), log2 domain
    float* lse;                 // [seqs][heads][blocks * rows of a block], log2 domain
    int32_t Hq, n, group, rows, blocks, fp16, accumulate, grid;   // group: heads per KV head; rows = group * n; blocks of 8 * NT rows
    float scale_log2e;
};

constexpr int kStages = 8;
constexpr int kMergeStride = 132;   // floats of a row in the merge area: rows 2t of four lanes start 8 banks apart
template <int NT> constexpr int kWarps = NT == 1 ? 16 : 8;       // consumer warps; 16 of them take pages in turn, eight each
template <int NT> constexpr int kAttendThreads = (kWarps<NT> + 4) * 32;   // and a warpgroup of which one warp loads
// Registers per thread after the warpgroups re-divide the register file.
template <int NT> constexpr int kRegsLaunch = (65536 / kAttendThreads<NT>) / 8 * 8;
template <int NT> constexpr int kRegsMath = NT == 1 ? 112 : 216;
template <int NT> constexpr int kRegsLoad = NT == 1 ? 32 : 72;
static_assert(4 * kRegsMath<1> + kRegsLoad<1> <= 5 * kRegsLaunch<1> && 2 * kRegsMath<2> + kRegsLoad<2> <= 3 * kRegsLaunch<2>,
              "register re-division must balance");

struct AttendCtrl {
    uint64_t full[kStages], empty[kStages];
    unsigned long long total;
    long long rest;
    int32_t first, sums[32];
    float2 ml[16][16];          // [warp][row]
};
template <int NT> constexpr size_t kMergeBytes = static_cast<size_t>(kWarps<NT>) * 8 * NT * kMergeStride * 4;
template <int NT> constexpr size_t kAttendSmem = static_cast<size_t>(kStages) * kRecordBytes + kMergeBytes<NT> + sizeof(AttendCtrl) + 128;
static_assert(kAttendSmem<1> <= 232448 && kAttendSmem<2> <= 232448, "shared memory budget of one CTA");

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0,
                                         float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint2 ld_shared_v2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 half2_from(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
__device__ __forceinline__ void scales_of(uint2 w, float (&s)[4]) {   // four bf16
    s[0] = __uint_as_float(w.x << 16);
    s[1] = __uint_as_float(w.x & 0xffff0000u);
    s[2] = __uint_as_float(w.y << 16);
    s[3] = __uint_as_float(w.y & 0xffff0000u);
}
// The token of row r (0..7) of an 8-row block: neighbours of opposite parity everywhere, which the shared-memory reads of K and V both
// need to be free of bank conflicts.
__device__ __forceinline__ int token_of_row(int r) { return r ^ ((r >> 1) & 1); }

// Query rows of one block as the second operand, and what belongs to the columns of a product (this thread's: rows 8 nt + 2t, + 1).
template <int NT>
struct Queries {
    uint32_t b[NT][4][4];   // [group of 32 channels][registers of two steps]
    float corr[NT][4][2];   // -8 * 2^-24 * sum of the group's queries
    float factor[NT][2];    // product -> logit in the log2 domain
    int limit[NT][2];       // tokens the row sees, less the sequence's length

    __device__ __forceinline__ void load(const AttendParams& P, int seq, int kv, int block, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = (block * NT + nt) * 8 + g;
            float f[4][8];
            uint32_t top = 0;
            const bool real = row < P.rows;
            const int hh = real ? row / P.n : 0, j = real ? row - hh * P.n : 0;
            const uint16_t* from = P.q + seq * P.qs[0] + (static_cast<int64_t>(kv) * P.group + hh) * P.qs[1] + j * P.qs[2] + 8 * t;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 x = real ? __ldg(reinterpret_cast<const uint4*>(from + 32 * i)) : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
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
            float sum[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[i][e] *= e & 1 ? mul * 0.0625f : mul;
                const __half2 a0 = __floats2half2_rn(f[i][0], f[i][4]), a1 = __floats2half2_rn(f[i][2], f[i][6]);
                const __half2 a2 = __floats2half2_rn(f[i][1], f[i][5]), a3 = __floats2half2_rn(f[i][3], f[i][7]);
                b[nt][i][0] = half2_bits(a0);
                b[nt][i][1] = half2_bits(a1);
                b[nt][i][2] = half2_bits(a2);
                b[nt][i][3] = half2_bits(a3);
                const float lo = (__low2float(a0) + __high2float(a0)) + (__low2float(a1) + __high2float(a1));
                const float hi = (__low2float(a2) + __high2float(a2)) + (__low2float(a3) + __high2float(a3));
                sum[i] = lo + 16.f * hi;
                sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
                sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
            }
            const float fac = __uint_as_float(static_cast<uint32_t>(127 + 24 - up) << 23) * P.scale_log2e;
            const int lim = real ? 1 - P.n + j : -0x40000000;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int from_lane = (2 * t + c) * 4;
                factor[nt][c] = __shfl_sync(0xffffffffu, fac, from_lane);
                limit[nt][c] = __shfl_sync(0xffffffffu, lim, from_lane);
#pragma unroll
                for (int i = 0; i < 4; ++i) corr[nt][i][c] = __shfl_sync(0xffffffffu, sum[i], from_lane) * (-8.f / 16777216.f);
            }
        }
    }
    // s[nt] = {token A x row 2t, A x 2t + 1, B x 2t, B x 2t + 1} in units of 1 / factor, for the tokens whose codes and scales are given.
    __device__ __forceinline__ void logits(float (&s)[NT][4], uint4 ka, uint4 kb, uint2 sa, uint2 sb) const {
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
        float fa[4], fb[4];
        scales_of(sa, fa);
        scales_of(sb, fb);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a = wa[i], c = wb[i], a8 = a >> 8, c8 = c >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float d[4];
                mma16816(d, a & 0x000f000fu, c & 0x000f000fu, a8 & 0x000f000fu, c8 & 0x000f000fu, b[nt][i][0], b[nt][i][1], corr[nt][i][0],
                         corr[nt][i][1], corr[nt][i][0], corr[nt][i][1]);
                mma16816(d, a & 0x00f000f0u, c & 0x00f000f0u, a8 & 0x00f000f0u, c8 & 0x00f000f0u, b[nt][i][2], b[nt][i][3], d[0], d[1], d[2], d[3]);
                if (i == 0) {
                    s[nt][0] = fa[0] * d[0];
                    s[nt][1] = fa[0] * d[1];
                    s[nt][2] = fb[0] * d[2];
                    s[nt][3] = fb[0] * d[3];
                } else {
                    s[nt][0] = fmaf(fa[i], d[0], s[nt][0]);
                    s[nt][1] = fmaf(fa[i], d[1], s[nt][1]);
                    s[nt][2] = fmaf(fb[i], d[2], s[nt][2]);
                    s[nt][3] = fmaf(fb[i], d[3], s[nt][3]);
                }
            }
        }
    }
};

__device__ __forceinline__ int pages_of(const Cache4& c, int seq) { return (c.length(seq) + kPage - 1) / kPage; }

// Logits (log2 domain) that a tile keeps below 2^kSlack times the reference before the reference is raised, and how far below the largest
// (logit + log2 scale) the reference is set: fp16 holds p * s up to 2^(kSlack + kLift) and, at full precision, down to 2^-14.
constexpr float kSlack = 8.f, kLift = 6.f;

template <int NT>
__global__ void __launch_bounds__(kAttendThreads<NT>, 1) cache_attend_kernel(const AttendParams P) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 127u) & ~127u;
    uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
    float* merge = reinterpret_cast<float*>(smem + kStages * kRecordBytes);
    AttendCtrl* sm = reinterpret_cast<AttendCtrl*>(smem + kStages * kRecordBytes + kMergeBytes<NT>);
    constexpr int kRows = 8 * NT, kNW = kWarps<NT>, kThreads = kAttendThreads<NT>, kTeams = kNW / 8;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto BAR = [&](uint64_t& b) { return smem_u32(&b); };

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(BAR(sm->full[i]), 1);
            mbar_init(BAR(sm->empty[i]), 8);
        }
        sm->total = 0;
        fence_mbar_init();
    }
    __syncthreads();
    wait_for_previous_kernel();

    // ---- the line of pages, and this CTA's range of it (a unit is a page of a (sequence, KV head, block of rows))
    const int seqs = P.cache.seqs, per = P.cache.heads * P.blocks;
    {
        unsigned long long mine = 0;
        for (int b = tid; b < seqs; b += kThreads) mine += pages_of(P.cache, b);
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0 && mine) atomicAdd(&sm->total, mine);
    }
    __syncthreads();
    const long long units = static_cast<long long>(sm->total) * per;
    const long long grid = min(static_cast<long long>(P.grid), units);
    const int cta = blockIdx.x;
    if (cta > 0 && cta >= grid) return;
    const long long u0 = grid ? units * cta / grid : 0, u1 = grid ? units * (cta + 1) / grid : 0;
    long long before = 0;
    for (int c0 = 0; c0 < seqs; c0 += kThreads) {
        const int b = c0 + tid, p = b < seqs ? pages_of(P.cache, b) : 0;
        int sum = p;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) sm->sums[warp] = sum;
        __syncthreads();
        long long at = before + sum - p;
        int chunk = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
            const int v = sm->sums[w];
            if (w < warp) at += v;
            chunk += v;
        }
        if (b < seqs && cta == 0) P.prefix[b] = static_cast<int32_t>(at);
        if (p && at * per <= u0 && u0 < (at + p) * per) {
            sm->first = b;
            sm->rest = u0 - at * per;
        }
        before += chunk;
        __syncthreads();
    }
    if (cta == 0 && tid == 0) P.prefix[seqs] = static_cast<int32_t>(before);
    if (u0 == u1) return;

    int seq = sm->first, pages = pages_of(P.cache, seq);
    int item = static_cast<int>(sm->rest / pages), page = static_cast<int>(sm->rest % pages);   // item: KV head * blocks + block of rows
    long long left = u1 - u0;
    uint32_t k = 0;   // pages so far
    bool bad = false;
    auto next = [&](int took) {
        left -= took;
        page = 0;
        if (left > 0 && ++item == per) {
            item = 0;
            do ++seq; while ((pages = pages_of(P.cache, seq)) == 0);
        }
    };

    if (warp >= kNW) {
        // =========================== loads ===========================
        reg_dec<kRegsLoad<NT>>();
        while (warp == kNW && left > 0) {
            const int take = static_cast<int>(min(left, static_cast<long long>(pages - page))), head = item / P.blocks, length = P.cache.length(seq);
            int id = -1;
            for (int i = 0; i < take; ++i, ++k) {
                if ((i & 31) == 0 && i + lane < take) id = P.cache.page(seq, page + i + lane);
                const int pg = __shfl_sync(0xffffffffu, id, i & 31);
                const uint32_t stage = k % kStages, bar = BAR(sm->full[stage]);
                if (k >= kStages && !bad) bad = __any_sync(0xffffffffu, !mbar_wait_role(BAR(sm->empty[stage]), (k / kStages - 1) & 1));
                if (bad) continue;   // (nothing is asked for any more; the others give up in the same way)
                if (lane == 0) {
                    const uint32_t to = base + stage * kRecordBytes;
                    const uint32_t tokens = min(kPage, (length - (page + i) * kPage + 15) & ~15);
                    if (pg < 0) {
                        mbar_arrive(bar);
                    } else if (tokens == kPage) {
                        mbar_arrive_expect_tx(bar, kRecordBytes);
                        bulk_load(to, P.cache.record(pg, head), kRecordBytes, bar);
                    } else {   // the last page: what of it is in use
                        const uint8_t* from = P.cache.record(pg, head);
                        mbar_arrive_expect_tx(bar, tokens * 144);
                        bulk_load(to + kKCodes, from + kKCodes, tokens * 64, bar);
                        bulk_load(to + kKScales, from + kKScales, tokens * 8, bar);
                        bulk_load(to + kVCodes, from + kVCodes, tokens * 64, bar);
                        bulk_load(to + kVScales, from + kVScales, tokens * 8, bar);
                    }
                }
                __syncwarp();
            }
            next(take);
        }
    } else {
        // =========================== products ===========================
        reg_inc<kRegsMath<NT>>();
        const int g = lane >> 2, t = lane & 3, team = warp >> 3, tile = (warp & 7) * 16;
        const int tok_a = tile + token_of_row(g), tok_v0 = tile + token_of_row(2 * t), tok_v1 = tile + token_of_row(2 * t + 1);
        const uint32_t k_at = kKCodes + tok_a * 64 + t * 16, ks_at = kKScales + tok_a * 8, vs_at = kVScales + tok_a * 8;
        const uint32_t v0_at = kVCodes + tok_v0 * 64 + (g ^ (tok_v0 & 4)) * 8, v1_at = kVCodes + tok_v1 * 64 + (g ^ (tok_v1 & 4)) * 8;
        bool first_piece = true;
        while (left > 0) {
            const int take = static_cast<int>(min(left, static_cast<long long>(pages - page)));
            const int head = item / P.blocks, block = item % P.blocks, length = P.cache.length(seq);
            Queries<NT> Q;
            Q.load(P, seq, head, block, lane);
            float ref[NT][2], sum[NT][2], o[NT][8][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                ref[nt][0] = ref[nt][1] = -INFINITY;
                sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
                for (int m = 0; m < 8; ++m)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[nt][m][c] = 0.f;
            }
#pragma unroll 1
            for (int i = 0; i < take; ++i, ++k) {
                if (kTeams > 1 && static_cast<int>(k % kTeams) != team) continue;
                const uint32_t stage = k % kStages;
                if (!bad) bad = __any_sync(0xffffffffu, !mbar_wait_role(BAR(sm->full[stage]), (k / kStages) & 1));
                const int first = (page + i) * kPage;   // first token of the page
                if (!bad && first + tile < length) {
                    const uint32_t at = base + stage * kRecordBytes;
                    const uint4 ka = ld_shared_v4(at + k_at), kb = ld_shared_v4(at + k_at + 8 * 64);
                    float s[NT][4];
                    Q.logits(s, ka, kb, ld_shared_v2(at + ks_at), ld_shared_v2(at + ks_at + 64));
                    float va[4], vb[4];
                    scales_of(ld_shared_v2(at + vs_at), va);
                    scales_of(ld_shared_v2(at + vs_at + 64), vb);
                    const bool edge = first + kPage > length - P.n + 1;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[nt][c] *= Q.factor[nt][c & 1];
                    if (edge) {   // tokens that a row does not see, and those that are not there (whose bytes may be anything)
                        const int pa = first + tok_a - length, pb = pa + 8;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if ((c < 2 ? pa : pb) >= Q.limit[nt][c & 1]) s[nt][c] = -INFINITY;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            if (pa >= 0) va[c] = 0.f;
                            if (pb >= 0) vb[c] = 0.f;
                        }
                    }
                    // the reference: raised, for every row by what it needs, when one is exceeded by more than the slack
                    const float ea = fast_log2(fmaxf(fmaxf(fmaxf(va[0], va[1]), fmaxf(va[2], va[3])), 8.27e-25f));
                    const float eb = fast_log2(fmaxf(fmaxf(fmaxf(vb[0], vb[1]), fmaxf(vb[2], vb[3])), 8.27e-25f));
                    float x[NT][2];
                    bool raise = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            x[nt][c] = fmaxf(s[nt][c] + ea, s[nt][c + 2] + eb) - kLift;
                            raise |= x[nt][c] > ref[nt][c] + kSlack;
                        }
                    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                float top = x[nt][c];
                                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                                top = fmaxf(top, ref[nt][c]);
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
                    uint32_t pb0[NT][4], pb1[NT][4];   // p * scale of the four groups, as the second operand
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float r0 = ref[nt][0] == -INFINITY ? 0.f : ref[nt][0], r1 = ref[nt][1] == -INFINITY ? 0.f : ref[nt][1];
                        const float p0 = fast_exp2(s[nt][0] - r0), p1 = fast_exp2(s[nt][1] - r1);
                        const float p2 = fast_exp2(s[nt][2] - r0), p3 = fast_exp2(s[nt][3] - r1);
                        sum[nt][0] += p0 + p2;
                        sum[nt][1] += p1 + p3;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            pb0[nt][c] = half2_bits(__floats2half2_rn(p0 * va[c], p1 * va[c]));
                            pb1[nt][c] = half2_bits(__floats2half2_rn(p2 * vb[c], p3 * vb[c]));
                        }
                        if (edge) {   // (0 * NaN: a token that is not finite is nothing to rows that do not see it)
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                pb0[nt][c] &= (p0 == 0.f ? 0u : 0xffffu) | (p1 == 0.f ? 0u : 0xffff0000u);
                                pb1[nt][c] &= (p2 == 0.f ? 0u : 0xffffu) | (p3 == 0.f ? 0u : 0xffff0000u);
                            }
                        }
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            pb0[nt][c] = transpose8x8(pb0[nt][c]);
                            pb1[nt][c] = transpose8x8(pb1[nt][c]);
                        }
                    }
                    const uint2 v0 = ld_shared_v2(at + v0_at), v1 = ld_shared_v2(at + v1_at);
                    const uint2 v2 = ld_shared_v2(at + v0_at + 8 * 64), v3 = ld_shared_v2(at + v1_at + 8 * 64);
                    const __half2 off = __float2half2_rn(-1032.f), off16 = __float2half2_rn(-72.f), sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
                    for (int i2 = 0; i2 < 4; ++i2) {
                        const uint32_t sel = i2 & 1 ? 0x7632u : 0x5410u;
                        uint32_t xx = __byte_perm(i2 < 2 ? v0.x : v0.y, i2 < 2 ? v1.x : v1.y, sel);   // four channels of tokens 2t, 2t + 1
                        uint32_t yy = __byte_perm(i2 < 2 ? v2.x : v2.y, i2 < 2 ? v3.x : v3.y, sel);   // ... and of the two 8 further
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t a0 = half2_bits(__hadd2(half2_from((xx & 0x000f000fu) | 0x64006400u), off));
                            const uint32_t a1 = half2_bits(__hfma2(half2_from((xx & 0x00f000f0u) | 0x64006400u), sixteenth, off16));
                            const uint32_t a2 = half2_bits(__hadd2(half2_from((yy & 0x000f000fu) | 0x64006400u), off));
                            const uint32_t a3 = half2_bits(__hfma2(half2_from((yy & 0x00f000f0u) | 0x64006400u), sixteenth, off16));
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float(&d)[4] = o[nt][2 * i2 + h];
                                mma16816(d, a0, a1, a2, a3, pb0[nt][i2], pb1[nt][i2], d[0], d[1], d[2], d[3]);
                            }
                            xx >>= 8;
                            yy >>= 8;
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(BAR(sm->empty[stage]));
            }
            // ---- the end of a piece: the warps' parts become one
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float l = sum[nt][c];
                    l += __shfl_xor_sync(0xffffffffu, l, 4);
                    l += __shfl_xor_sync(0xffffffffu, l, 8);
                    l += __shfl_xor_sync(0xffffffffu, l, 16);
                    const int r = nt * 8 + 2 * t + c;
                    if (g == 0) sm->ml[warp][r] = make_float2(ref[nt][c], l);
                    float* to = merge + (warp * kRows + r) * kMergeStride + 4 * g;
#pragma unroll
                    for (int i = 0; i < 4; ++i)   // channels 32 i + 4 g ..: rows g and g + 8 of two operand tiles
                        *reinterpret_cast<float4*>(to + 32 * i) = make_float4(o[nt][2 * i][c], o[nt][2 * i][c + 2], o[nt][2 * i + 1][c], o[nt][2 * i + 1][c + 2]);
                }
            }
            named_barrier_sync(1, kNW * 32);
            const bool whole = page == 0 && take == pages;
            const int ch = tid & 127;
            for (int r = tid >> 7; r < kRows; r += kNW / 4) {
                const int row = block * kRows + r;
                if (row >= P.rows) break;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kNW; ++w) top = fmaxf(top, sm->ml[w][r].x);
                const float m = top == -INFINITY ? 0.f : top;
                float l = 0.f, acc = 0.f;
#pragma unroll
                for (int w = 0; w < kNW; ++w) {
                    const float2 ml = sm->ml[w][r];
                    const float by = fast_exp2(ml.x - m);
                    l = fmaf(ml.y, by, l);
                    acc = fmaf(merge[(w * kRows + r) * kMergeStride + ch], by, acc);
                }
                if (whole) {
                    const int hh = row / P.n, j = row - hh * P.n, h = head * P.group + hh;
                    if (P.sinks) l += fast_exp2(P.sinks[h] * kLog2e - m);
                    const float y = l == 0.f ? 0.f : acc / l;
                    P.out[((static_cast<int64_t>(seq) * P.n + j) * P.Hq + h) * kHeadDim + ch] =
                        static_cast<uint16_t>(P.fp16 ? pack_act<true>(y, 0.f) : pack_act<false>(y, 0.f));
                    if (ch == 0) P.lse[(static_cast<int64_t>(seq) * P.cache.heads + head) * (P.blocks * kRows) + row] = m + fast_log2(l);
                } else {
                    const int64_t slot = 2LL * cta + (first_piece ? 0 : 1);
                    P.o_part[(slot * kRows + r) * kHeadDim + ch] = acc;
                    if (ch == 0) P.ml_part[slot * kRows + r] = make_float2(top, l);
                }
            }
            named_barrier_sync(1, kNW * 32);
            first_piece = false;
            next(take);
        }
    }
    if (bad) {
        atomicMax(P.cache.status, kStatusWaitTimeout);
        const uint64_t t0 = global_timer_ns();   // copies in flight land before shared memory is given back
        while (global_timer_ns() - t0 < 200000) __nanosleep(1000);
    }
}

// Merges what ranges cut: a block per (sequence, KV head, block of rows) and row.  Pairs that lay in one range are done; sequences without
// a token get their zeros here.
template <int NT>
__global__ void __launch_bounds__(512) cache_combine_kernel(const AttendParams P) {
    constexpr int kRows = 8 * NT;
    __shared__ float factor[512], part[3][128], red[2][16];
    wait_for_previous_kernel();
    const int per = P.cache.heads * P.blocks, r = blockIdx.y, tid = threadIdx.x, ch = tid & 127, lane = tid & 31;
    const int seq = blockIdx.x / per, item = blockIdx.x % per, head = item / P.blocks, row = (item % P.blocks) * kRows + r;
    if (row >= P.rows) return;
    const long long total = P.prefix[P.cache.seqs], units = total * per, grid = min(static_cast<long long>(P.grid), units);
    const long long at = P.prefix[seq], pages = P.prefix[seq + 1] - at, first = at * per + item * pages;
    const int hh = row / P.n, j = row - hh * P.n, h = head * P.group + hh;
    uint16_t* out = P.out + ((static_cast<int64_t>(seq) * P.n + j) * P.Hq + h) * kHeadDim;
    float* lse = P.lse + (static_cast<int64_t>(seq) * P.cache.heads + head) * (P.blocks * kRows) + row;
    if (pages == 0) {
        if (tid < 128) out[tid] = 0;
        if (tid == 0) *lse = P.sinks ? P.sinks[h] * kLog2e : -INFINITY;
        return;
    }
    const int c0 = static_cast<int>(((first + 1) * grid - 1) / units), c1 = static_cast<int>(((first + pages) * grid - 1) / units);
    if (c0 == c1) return;
    const int n = c1 - c0 + 1;   // <= grid <= 512
    const bool second = units * c0 / grid < first;   // in its range c0 had another piece before this one
    auto slot = [&](int i) { return 2LL * (c0 + i) + (i == 0 && second ? 1 : 0); };
    const float2 ml = tid < n ? P.ml_part[slot(tid) * kRows + r] : make_float2(-INFINITY, 0.f);
    float top = ml.x;
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) red[0][tid >> 5] = top;
    __syncthreads();
    for (int w = 0; w < 16; ++w) top = fmaxf(top, red[0][w]);
    const float m = top == -INFINITY ? 0.f : top, by = fast_exp2(ml.x - m);
    factor[tid] = by;
    float l = ml.y * by;
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) red[1][tid >> 5] = l;
    __syncthreads();
    l = 0.f;
    for (int w = 0; w < 16; ++w) l += red[1][w];
    float acc = 0.f;
#pragma unroll 4
    for (int i = tid >> 7; i < n; i += 4) acc = fmaf(P.o_part[(slot(i) * kRows + r) * kHeadDim + ch], factor[i], acc);
    if (tid >= 128) part[(tid >> 7) - 1][ch] = acc;
    __syncthreads();
    if (tid < 128) {
        acc += part[0][ch] + part[1][ch] + part[2][ch];
        if (P.sinks) l += fast_exp2(P.sinks[h] * kLog2e - m);
        const float y = l == 0.f ? 0.f : acc / l;
        out[ch] = static_cast<uint16_t>(P.fp16 ? pack_act<true>(y, 0.f) : pack_act<false>(y, 0.f));
        if (tid == 0) *lse = m + fast_log2(l);
    }
}

// The probabilities of every token, summed over the query rows of its KV head: the logits once more (half of the cache's bytes, most of
// them still in L2), relative to the log-sum-exps that are known now.  (Keeping the logits of the first kernel instead would move 4 bytes
// per row and token twice, as much as K's 72 bytes from nine rows on, and needs a buffer for the longest lengths.)
constexpr int kWeightWarps = 8;
template <int NT>
__global__ void __launch_bounds__(kWeightWarps * 32) cache_weights_kernel(const AttendParams P) {
    constexpr int kRows = 8 * NT;
    wait_for_previous_kernel();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, heads = P.cache.heads;
    const long long units = static_cast<long long>(P.prefix[P.cache.seqs]) * heads;
    const long long u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
    if (u0 == u1) return;
    int lo = 0, hi = P.cache.seqs;   // the sequence whose pages begin at or before u0
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (static_cast<long long>(P.prefix[mid]) * heads <= u0) lo = mid; else hi = mid;
    }
    const int tok_a = warp * 16 + token_of_row(g);
    long long u = u0;
    for (int seq = lo; u < u1; ++seq) {
        const long long begin = static_cast<long long>(P.prefix[seq]) * heads;
        const int pages = P.prefix[seq + 1] - P.prefix[seq], length = P.cache.length(seq);
        while (u < u1 && u < begin + static_cast<long long>(pages) * heads) {
            const int head = static_cast<int>((u - begin) / pages), page = static_cast<int>((u - begin) % pages);
            const int take = static_cast<int>(min(u1 - u, static_cast<long long>(pages - page)));
            for (int block = 0; block < P.blocks; ++block) {
                Queries<NT> Q;
                Q.load(P, seq, head, block, lane);
                float lse[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        lse[nt][c] = P.lse[(static_cast<int64_t>(seq) * heads + head) * (P.blocks * kRows) + min(block * kRows + nt * 8 + 2 * t + c, P.rows - 1)];
                for (int i = 0; i < take; ++i) {
                    const int first = (page + i) * kPage;
                    if (first + warp * 16 >= length) break;
                    const int pg = P.cache.page(seq, page + i);
                    if (pg < 0) continue;
                    const uint8_t* from = P.cache.record(pg, head);
                    const uint4 ka = *reinterpret_cast<const uint4*>(from + kKCodes + tok_a * 64 + t * 16);
                    const uint4 kb = *reinterpret_cast<const uint4*>(from + kKCodes + (tok_a + 8) * 64 + t * 16);
                    const uint2 sa = *reinterpret_cast<const uint2*>(from + kKScales + tok_a * 8);
                    const uint2 sb = *reinterpret_cast<const uint2*>(from + kKScales + (tok_a + 8) * 8);
                    float s[NT][4];
                    Q.logits(s, ka, kb, sa, sb);
                    const int pa = first + tok_a - length, pb = pa + 8;
                    float wa = 0.f, wb = 0.f;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            if (pa < Q.limit[nt][c]) wa += fast_exp2(fmaf(s[nt][c], Q.factor[nt][c], -lse[nt][c]));
                            if (pb < Q.limit[nt][c]) wb += fast_exp2(fmaf(s[nt][c + 2], Q.factor[nt][c], -lse[nt][c]));
                        }
                    wa += __shfl_xor_sync(0xffffffffu, wa, 1);
                    wb += __shfl_xor_sync(0xffffffffu, wb, 1);
                    wa += __shfl_xor_sync(0xffffffffu, wa, 2);
                    wb += __shfl_xor_sync(0xffffffffu, wb, 2);
                    if (t < 2 && (t ? pb : pa) < 0) {
                        float* to = P.weights + (static_cast<int64_t>(pg) * heads + head) * kPage + tok_a + 8 * t;
                        const float w = t ? wb : wa;
                        *to = block || P.accumulate ? *to + w : w;
                    }
                }
            }
            u += take;
        }
    }
}

struct AttendSpace {
    int64_t prefix, o_part, ml_part, lse, bytes;
};
int tiles_for(int64_t rows) { return rows <= 8 ? 1 : 2; }
AttendSpace carve_attend(int seqs, int Hq, int heads, int n, int grid) {
    const int64_t rows = static_cast<int64_t>(Hq / heads) * n, block = 8 * tiles_for(rows);
    AttendSpace w;
    int64_t off = 0;
    auto take = [&](int64_t bytes) {
        const int64_t at = off;
        off += round_up(bytes, 256);
        return at;
    };
    w.prefix = take(4LL * (seqs + 1));
    w.o_part = take(2LL * grid * block * kHeadDim * 4);
    w.ml_part = take(2LL * grid * block * 8);
    w.lse = take(4LL * seqs * heads * round_up(rows, block));
    w.bytes = off;
    return w;
}

template <int NT>
int launch_attend(const AttendParams& P, int weights, cudaStream_t st) {
    const int sms = device_sm_count();
    if (!ensure_smem_attr(reinterpret_cast<const void*>(cache_attend_kernel<NT>), kAttendSmem<NT>)) return FMSA_ERR_CUDA;
    launch_chained(cache_attend_kernel<NT>, P.grid, kAttendThreads<NT>, kAttendSmem<NT>, st, P);
    launch_chained(cache_combine_kernel<NT>, dim3(static_cast<unsigned>(P.cache.seqs * P.cache.heads * P.blocks), 8 * NT), 512, 0, st, P);
    if (weights) launch_chained(cache_weights_kernel<NT>, sms * 4, kWeightWarps * 32, 0, st, P);
    return check_launch();
}

constexpr int kMaxGrid = 512;   // ranges that the combine holds the factors of

}  // namespace
}  // namespace fmsa

extern "C" int64_t fmsa_cache_attend_workspace_bytes(int32_t seqs, int32_t Hq, int32_t heads, int32_t n) {
    using namespace fmsa;
    const int sms = device_sm_count();
    if (seqs <= 0 || heads <= 0 || Hq <= 0 || Hq % heads || n <= 0 || sms <= 0) return -1;
    return carve_attend(seqs, Hq, heads, n, sms < kMaxGrid ? sms : kMaxGrid).bytes;
}

extern "C" int fmsa_cache_attend(const fmsa_cache4* cache, const fmsa_tensor* q, int32_t Hq, int32_t n, float scale, int32_t dtype,
                                 const float* sinks, float* weights, int32_t accumulate, void* out, void* workspace, int64_t workspace_bytes,
                                 int32_t* status, void* stream) {
    using namespace fmsa;
    FMSA_REQUIRE(cache4_ok(cache) && q && q->ptr && out && workspace && status && Hq > 0 && n > 0 && Hq % cache->heads == 0);
    FMSA_REQUIRE(dtype == FMSA_DTYPE_BF16 || dtype == FMSA_DTYPE_FP16);
    FMSA_REQUIRE(aligned16(q->ptr) && q->stride_b % 8 == 0 && q->stride_h % 8 == 0 && q->stride_s % 8 == 0);
    const int64_t rows = static_cast<int64_t>(Hq / cache->heads) * n;
    const int nt = tiles_for(rows);
    const int64_t blocks = (rows + 8 * nt - 1) / (8 * nt), items = blocks * cache->heads * cache->seqs;
    if (items > 0x7fffffffLL || static_cast<int64_t>(cache->seqs) * cache->width > 0x7fffffffLL) return FMSA_ERR_UNSUPPORTED;
    const int sms = device_sm_count();
    if (sms <= 0) return FMSA_ERR_CUDA;
    AttendParams P = {};
    P.grid = sms < kMaxGrid ? sms : kMaxGrid;
    const AttendSpace w = carve_attend(cache->seqs, Hq, cache->heads, n, P.grid);
    if (workspace_bytes < w.bytes) return FMSA_ERR_WORKSPACE;
    FMSA_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0);
    char* ws = static_cast<char*>(workspace);
    P.cache = device_cache(cache, status);
    P.q = static_cast<const uint16_t*>(q->ptr);
    P.qs[0] = q->stride_b; P.qs[1] = q->stride_h; P.qs[2] = q->stride_s;
    P.sinks = sinks;
    P.out = static_cast<uint16_t*>(out);
    P.weights = weights;
    P.prefix = reinterpret_cast<int32_t*>(ws + w.prefix);
    P.o_part = reinterpret_cast<float*>(ws + w.o_part);
    P.ml_part = reinterpret_cast<float2*>(ws + w.ml_part);
    P.lse = reinterpret_cast<float*>(ws + w.lse);
    P.Hq = Hq; P.n = n; P.group = Hq / cache->heads; P.rows = static_cast<int32_t>(rows); P.blocks = static_cast<int32_t>(blocks);
    P.fp16 = dtype == FMSA_DTYPE_FP16; P.accumulate = accumulate ? 1 : 0;
    P.scale_log2e = scale * kLog2e;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return nt == 1 ? launch_attend<1>(P, weights != nullptr, st) : launch_attend<2>(P, weights != nullptr, st);
}
