// What the kernels of attention over the cache share (cache_attend.cu, cache_rows.cu).
#pragma once

#include "cache4.cuh"
#include "host_common.h"
#include "sm100.cuh"

namespace fmsa {

struct AttendParams {
    Cache4 cache;
    const uint16_t* q;          // (seqs,Hq,n,128)
    int64_t qs[3];
    const float* sinks;         // [Hq] or null
    uint16_t* out;              // [seqs][n][Hq*128]
    float* weights;             // [pages][heads][128] or null
    int32_t* prefix;            // [seqs + 1]: pages of the sequences before
    int2* parts;                // [seqs][heads][blocks]: first slot of a pair that is cut and the number of its parts; 0 parts: not cut
    float* o_part;              // [2 * ranges][rows of a block][128]
    float2* ml_part;            // [2 * ranges][rows of a block]: (reference, sum), log2 domain
    float* lse;                 // [seqs][heads][blocks * rows of a block], log2 domain
    int32_t Hq, n, group, rows, blocks, fp16, accumulate, grid;   // group: heads per KV head; rows = group * n, in blocks
    int32_t lse_rows;           // blocks * rows of a block
    float scale_log2e;
    uint32_t magic;             // 1024, 1024 in fp16
    int32_t spread;             // CTAs of a cluster, a power of two
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// Nibbles as fp16: bits 3..6 of a half are q * 2^-21 (a denormal), bits 7..10 q * 2^-17 (from 8 on a normal number, which goes on where
// the denormals end).  Not lower in the half: the tensor core aligns its sums by the operands' exponent fields, so every leading zero of a
// denormal costs a bit of the sum.  (With K and V at bits 0..3 and 4..7 a row over 900 tokens was 1.7 times further from 64 bits' than the
// other roundings allow for.)
constexpr uint32_t kLow = 0x00780078u, kHigh = 0x07800780u;
constexpr float kUnitLow = 1.f / (1 << 21);

// (x & mask) | or_with as one instruction, if one of them is in a register.
__device__ __forceinline__ uint32_t masked_or(uint32_t x, uint32_t mask, uint32_t or_with) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(or_with));
    return y;
}

// What a kernel's preparation of queries works on: 8 query rows (number nt of a block), loaded by all lanes of a warp, which may do something else meanwhile.
struct RawQueries {
    uint4 x[4];
    int limit;
    __device__ __forceinline__ void load(const AttendParams& P, int seq, int kv, int row, int lane) {   // row: the eight's first
        row += lane >> 2;
        const bool real = row < P.rows;
        const int hh = real ? row / P.n : 0, j = real ? row - hh * P.n : 0;
        const uint16_t* from = P.q + seq * P.qs[0] + (static_cast<int64_t>(kv) * P.group + hh) * P.qs[1] + j * P.qs[2] + 8 * (lane & 3);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = real ? __ldg(reinterpret_cast<const uint4*>(from + 32 * i)) : make_uint4(0, 0, 0, 0);
        limit = real ? 1 - P.n + j : -0x40000000;
    }
};
// `units` pages in at most `most` ranges, the first ones one page longer: unit begin(r) is the first of range r (or `units` behind the last).
struct Ranges {
    int units, size, longer, n;
    __device__ Ranges() {}
    __device__ __forceinline__ Ranges(int all, int most) : units(all), n(min(all, most)) {
        size = n ? all / n : 0;
        longer = all - size * n;
    }
    __device__ __forceinline__ int begin(int r) const { return r < n ? size * r + min(r, longer) : units; }
    __device__ __forceinline__ int owner(int u) const {
        const int split = longer * (size + 1);
        return u < split ? u / (size + 1) : longer + (u - split) / size;
    }
};

// Logits (log2 domain) that a tile keeps below 2^kSlack times the reference before the reference is raised, and how far below the largest
// (logit + log2 scale) the reference is set: fp16 holds p * s up to 2^(kSlack + kLift) and, at full precision, down to 2^-14.
constexpr float kSlack = 8.f, kLift = 6.f;

// cache_rows.cu: pairs of sequence and KV head with many query rows.
constexpr int kRowsMost = 64;                  // rows of a block
inline int rows_of_block(int64_t rows) {       // blocks of equal size, whole sixteens
    const int64_t blocks = (rows + kRowsMost - 1) / kRowsMost;
    return static_cast<int>(((rows + blocks - 1) / blocks + 15) / 16 * 16);
}
bool launch_attend_rows(const AttendParams& P, cudaStream_t st);    // everything but the merging
bool launch_weights_rows(const AttendParams& P, cudaStream_t st);   // one block of rows

}  // namespace fmsa
