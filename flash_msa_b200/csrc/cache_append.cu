// New keys and values into the cache held in 4 bits.
//
// Per token, KV head and group of 32 channels: scale s = bf16(max |x| / 7), code = x / s rounded to the nearest whole number, halves away
// from zero (so -7..7), stored as code + 8.  A group below 2^-80 is stored as zeros (its scale would near the end of bf16's range), one with
// a value that is not finite gets the scale NaN: it stays visible instead of spoiling its neighbours' codes only.
// The rounding is exact although it multiplies by a reciprocal: with x of at most 11 significant bits and s of 8, x / s is either a half
// (k + 1/2) itself or at least 2^-13 away from one, while the product with r = (1 / s) * (1 + 2^-21) is above |x| / s by no more than 4e-6
// and never below it - so a half is always above k + 1/2 when it is rounded, and nothing else crosses it.
//
// Bound by HBM: 512 bytes in and 144 out per token and head (656 / 1168 with the stored values).  A warp takes four rows; 16 lanes hold a
// row of K, 16 the row of V, 8 channels a lane: a lane's K codes are one word of the record as it stands, two lanes exchange a halfword for V.
#include "cache4.cuh"
#include "host_common.h"
#include "sm100.cuh"

namespace fmsa {
namespace {

struct AppendParams {
    Cache4 cache;
    const uint16_t *k, *v;                     // (B,H,n,128)
    int64_t ks[3], vs[3];                      // element strides
    uint16_t *k_out, *v_out;                   // the stored values, or null; strides below
    int64_t kos[3], vos[3];
    float* weights;                            // [pages][heads][128] or null
    const int32_t* cu;                         // [seqs + 1] or null: sequence i is batch row i
    uint32_t rows, n;
};

constexpr int kAppendRows = 4, kAppendWarps = 8;

template <bool FP16>
__global__ void __launch_bounds__(kAppendWarps * 32) cache_append_kernel(const AppendParams P) {
    wait_for_previous_kernel();
    const int lane = threadIdx.x & 31;
    const uint32_t row0 = (blockIdx.x * kAppendWarps + (threadIdx.x >> 5)) * kAppendRows;
    if (row0 >= P.rows) return;
    const bool is_v = lane >= 16;
    const int l = lane & 15, group = l >> 2, t = l & 3;

    // lanes 0..3: where rows 0..3 of the warp go (-1: nowhere)
    int64_t src = 0, dst_out = 0, record = -1;
    int slot = 0;
    const uint16_t* from = is_v ? P.v : P.k;
    uint4 x[kAppendRows];
    {
        const uint32_t r = row0 + (lane & 3);
        if (r < P.rows) {
            const uint32_t bh = r / P.n, j = r - bh * P.n, b = bh / P.cache.heads, h = bh - b * P.cache.heads;
            src = is_v ? b * P.vs[0] + h * P.vs[1] + j * P.vs[2] : b * P.ks[0] + h * P.ks[1] + j * P.ks[2];
            dst_out = is_v ? b * P.vos[0] + h * P.vos[1] + j * P.vos[2] : b * P.kos[0] + h * P.kos[1] + j * P.kos[2];
            if (lane < kAppendRows) {
                int seq = static_cast<int>(b), behind = static_cast<int>(P.n - j);   // rows from this one to its sequence's end
                if (P.cu) {
                    int lo = 0, hi = P.cache.seqs;   // the sequence with cu[seq] <= j < cu[seq + 1]
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) >> 1;
                        if (P.cu[mid] <= static_cast<int>(j)) lo = mid; else hi = mid;
                    }
                    seq = lo;
                    // (an empty sequence has its neighbour's boundary: the search ends at the last that begins here)
                    const int end = P.cu[seq + 1];
                    behind = static_cast<int>(j) >= P.cu[seq] && static_cast<int>(j) < end ? end - static_cast<int>(j) : 0;
                }
                const int64_t length = P.cache.lengths[seq], at = length - behind;
                if (behind > 0 && at >= 0) {
                    if (at < static_cast<int64_t>(P.cache.width) * kPage) {
                        const int page = P.cache.page(seq, static_cast<int>(at / kPage));
                        slot = static_cast<int>(at % kPage);
                        if (page >= 0) record = static_cast<int64_t>(page) * P.cache.heads + h;
                    } else {
                        atomicMax(P.cache.status, kStatusBadIndex);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kAppendRows; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, src, (lane & 16) + i);
        x[i] = make_uint4(0, 0, 0, 0);
        if (row0 + i < P.rows) x[i] = __ldg(reinterpret_cast<const uint4*>(from + at + 8 * l));
    }
#pragma unroll
    for (int i = 0; i < kAppendRows; ++i) {
        const int64_t rec = __shfl_sync(0xffffffffu, record, i);
        const int sl = __shfl_sync(0xffffffffu, slot, i);
        const int64_t out_at = __shfl_sync(0xffffffffu, dst_out, (lane & 16) + i);
        if (row0 + i >= P.rows) break;   // (uniform)
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        float f[8];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[2 * e] = act_lo<FP16>(w[e]);
            f[2 * e + 1] = act_hi<FP16>(w[e]);
            // (as whole numbers the magnitudes compare like the values, infinity and NaN above all)
            top = max(top, max(__float_as_uint(f[2 * e]) & 0x7fffffffu, __float_as_uint(f[2 * e + 1]) & 0x7fffffffu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        __nv_bfloat16 scale = __float2bfloat16_rn(__fdiv_rn(__uint_as_float(top), 7.f));
        float r = __frcp_rn(__bfloat162float(scale)) * (1.f + 4.76837158203125e-7f);
        if (top < 0x17800000u) {                        // 2^-80
            scale = __float2bfloat16_rn(0.f);
            r = 0.f;
        }
        const bool odd = top >= 0x7f800000u;
        if (odd) {
            scale = __ushort_as_bfloat16(0x7fffu);
            r = 0.f;
        }
        uint32_t code = 0;
        float q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // 1.5 * 2^23 + 8: the sum's last bits are the code; one rounding, of the exact product
            const float m = __fmaf_rn(odd ? 0.f : f[e], r, 12582920.f);
            code |= (__float_as_uint(m) & 15u) << (4 * e);
            q[e] = m - 12582920.f;
        }
        if (rec >= 0) {
            uint8_t* to = P.cache.records + rec * kRecordBytes;
            if (!is_v) {
                *reinterpret_cast<uint32_t*>(to + kKCodes + sl * 64 + t * 16 + group * 4) = code;
                if (t == 0) *reinterpret_cast<__nv_bfloat16*>(to + kKScales + sl * 8 + group * 2) = scale;
            }
            // V: this lane's 8 channels are halfword `group` of chunks 2t and 2t + 1; with the lane of group ^ 1 it makes whole words
            const uint32_t got = __shfl_xor_sync(0xffffffffu, group & 1 ? code & 0xffffu : code >> 16, 4);
            if (is_v) {
                const uint32_t word = group & 1 ? got | (code & 0xffff0000u) : (code & 0xffffu) | got << 16;
                const int chunk = 2 * t + (group & 1);
                *reinterpret_cast<uint32_t*>(to + kVCodes + sl * 64 + (chunk ^ (sl & 4)) * 8 + (group & 2) * 2) = word;
                if (t == 0) *reinterpret_cast<__nv_bfloat16*>(to + kVScales + sl * 8 + group * 2) = scale;
            }
            if (P.weights && lane == 0) P.weights[rec * kPage + sl] = 0.f;
        }
        uint16_t* out = is_v ? P.v_out : P.k_out;
        if (out) {
            const float s = rec >= 0 ? __bfloat162float(scale) : 0.f;
            uint32_t pk[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) pk[e] = rec >= 0 ? pack_act<FP16>(q[2 * e] * s, q[2 * e + 1] * s) : 0u;
            *reinterpret_cast<uint4*>(out + out_at + 8 * l) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
    }
}

}  // namespace
}  // namespace fmsa

extern "C" int fmsa_cache_append(const fmsa_cache4* cache, const fmsa_tensor* k, const fmsa_tensor* v, int32_t B, int32_t n, int32_t dtype,
                                 const int32_t* cu_seqlens, float* weights, const fmsa_tensor* k_values, const fmsa_tensor* v_values,
                                 int32_t* status, void* stream) {
    using namespace fmsa;
    FMSA_REQUIRE(cache4_ok(cache) && k && v && k->ptr && v->ptr && status && B > 0 && n > 0);
    FMSA_REQUIRE(dtype == FMSA_DTYPE_BF16 || dtype == FMSA_DTYPE_FP16);
    FMSA_REQUIRE(cu_seqlens ? B == 1 : B == cache->seqs);
    FMSA_REQUIRE((k_values == nullptr) == (v_values == nullptr));
    for (const fmsa_tensor* t : {k, v, k_values, v_values})
        if (t) FMSA_REQUIRE(t->ptr && aligned16(t->ptr) && t->stride_b % 8 == 0 && t->stride_h % 8 == 0 && t->stride_s % 8 == 0);
    const int64_t rows = static_cast<int64_t>(B) * cache->heads * n;
    if (rows > 0x7fffff00LL) return FMSA_ERR_UNSUPPORTED;
    AppendParams P = {};
    P.cache = device_cache(cache, status);
    P.k = static_cast<const uint16_t*>(k->ptr);
    P.v = static_cast<const uint16_t*>(v->ptr);
    auto strides = [](int64_t (&to)[3], const fmsa_tensor* t) { to[0] = t->stride_b; to[1] = t->stride_h; to[2] = t->stride_s; };
    strides(P.ks, k);
    strides(P.vs, v);
    if (k_values) {
        P.k_out = static_cast<uint16_t*>(const_cast<void*>(k_values->ptr));
        P.v_out = static_cast<uint16_t*>(const_cast<void*>(v_values->ptr));
        strides(P.kos, k_values);
        strides(P.vos, v_values);
    }
    P.weights = weights;
    P.cu = cu_seqlens;
    P.rows = static_cast<uint32_t>(rows);
    P.n = static_cast<uint32_t>(n);
    const unsigned grid = static_cast<unsigned>((rows + kAppendRows * kAppendWarps - 1) / (kAppendRows * kAppendWarps));
    launch_chained(dtype == FMSA_DTYPE_FP16 ? cache_append_kernel<true> : cache_append_kernel<false>, grid, kAppendWarps * 32, 0,
                   static_cast<cudaStream_t>(stream), P);
    return check_launch();
}
