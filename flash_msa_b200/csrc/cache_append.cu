// New keys and values into the cache held in 4 bits.
//
// Per token, KV head and group of 32 channels: scale s = bf16(max |x| / 7), code = x / s rounded to the nearest whole number, halves away
// from zero (so -7..7), stored as code + 8.  A group below 2^-80 is stored as zeros (its scale would near the end of bf16's range), one with
// a value that is not finite gets the scale NaN: it stays visible instead of spoiling its neighbours' codes only.
// The rounding is exact although it multiplies by a reciprocal: with x of at most 11 significant bits and s of 8, x / s is either a half
// (k + 1/2) itself or at least 2^-13 away from one, while the product with r = (1 / s) * (1 + 2^-21) is above |x| / s by no more than 4e-6
// and never below it - so a half is always above k + 1/2 when it is rounded, and nothing else crosses it.
//
// 512 bytes come in and 144 leave per token and head (656 with the stored values); at first bound by instructions, so few are
// spent: the maximum is taken on 16-bit pairs, the codes are the last bits of one fma each and join by multiply-adds.  16 lanes hold a row of
// K, 16 the row of V, 8 channels a lane: a lane's K codes are one word of the record as it stands, two lanes exchange a halfword for V.
// 32768 tokens of 8 heads with the stored values (307 MB): 61.5 us, 5.0 TB/s; with a division and logical operations 103 us.
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
    uint32_t rows, n, blocks;                  // blocks: that have rows
};

constexpr int kAppendWarps = 8;

// Largest magnitude of eight packed values as fp32; NaN if one is NaN.
template <bool FP16>
__device__ __forceinline__ float largest(const uint32_t (&w)[4]) {
    if (FP16) {
        const __half2* h = reinterpret_cast<const __half2*>(w);
        const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
        return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
    }
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}
__device__ __forceinline__ float reciprocal(float x) {   // to 2^-23
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ROWS rows (of the B * heads * n) a warp.
template <bool FP16, int ROWS>
__global__ void __launch_bounds__(kAppendWarps * 32) cache_append_kernel(const AppendParams P) {
    wait_for_previous_kernel();
    if (P.cu && blockIdx.x == P.blocks) {   // with boundaries there is a block behind the rows, which looks whether they rise
        for (int i = threadIdx.x; i < P.cache.seqs; i += kAppendWarps * 32)
            if (bad_boundaries(P.cu, i, static_cast<int>(P.n))) atomicMax(P.cache.status, kStatusBadIndex);
        return;
    }
    const int lane = threadIdx.x & 31;
    const uint32_t row0 = (blockIdx.x * kAppendWarps + (threadIdx.x >> 5)) * ROWS;
    if (row0 >= P.rows) return;
    const bool is_v = lane >= 16;
    const int l = lane & 15, group = l >> 2, t = l & 3;

    // lanes i and 16 + i, i < ROWS: where row i of K and of V is and goes
    int64_t src = 0, dst_out = 0;
    int place = -1;                  // record * 128 + slot, or -1: nowhere  (16 million records are more than a GPU holds)
    if (l < ROWS && row0 + l < P.rows) {
        const uint32_t r = row0 + l, bh = r / P.n, j = r - bh * P.n, b = bh / P.cache.heads, h = bh - b * P.cache.heads;
        src = is_v ? b * P.vs[0] + h * P.vs[1] + j * P.vs[2] : b * P.ks[0] + h * P.ks[1] + j * P.ks[2];
        dst_out = is_v ? b * P.vos[0] + h * P.vos[1] + j * P.vos[2] : b * P.kos[0] + h * P.kos[1] + j * P.kos[2];
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
        const int at = P.cache.length(seq) - behind;
        if (behind > 0 && at >= 0) {
            const int page = P.cache.page(seq, at / kPage);
            if (page >= 0) place = (page * P.cache.heads + static_cast<int>(h)) * kPage + at % kPage;
        }
    }
    const uint16_t* from = (is_v ? P.v : P.k) + 8 * l;
    uint16_t* out = is_v ? P.v_out : P.k_out;
    uint4 x[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, src, (lane & 16) + i);
        x[i] = make_uint4(0, 0, 0, 0);
        if (row0 + i < P.rows) x[i] = __ldg(reinterpret_cast<const uint4*>(from + at));
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (row0 + i >= P.rows) break;   // (uniform)
        const int to = __shfl_sync(0xffffffffu, place, i);
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        float top = largest<FP16>(w);
        // (as whole numbers magnitudes compare like the values, infinity and NaN above all)
        uint32_t bits = __float_as_uint(top);
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
        top = __uint_as_float(bits);
        // top / 7, correctly rounded: one correction of the product with the rounded reciprocal (Markstein 1990); then to bf16
        constexpr float kSeventh = 1.f / 7.f;
        const float guess = top * kSeventh;
        __nv_bfloat16 scale = __float2bfloat16_rn(fmaf(fmaf(-7.f, guess, top), kSeventh, guess));
        float r = reciprocal(__bfloat162float(scale)) * (1.f + 4.76837158203125e-7f);
        if (bits < 0x17800000u) {        // 2^-80
            scale = __ushort_as_bfloat16(0);
            r = 0.f;
        }
        const bool odd = bits >= 0x7f800000u;
        if (odd) scale = __ushort_as_bfloat16(0x7fffu);
        // 1.5 * 2^23 + 8: the sum's last bits are the code; one rounding, of the exact product
        float m[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m[2 * e] = __fmaf_rn(act_lo<FP16>(w[e]), r, 12582920.f);
            m[2 * e + 1] = __fmaf_rn(act_hi<FP16>(w[e]), r, 12582920.f);
        }
        uint32_t code = __float_as_uint(m[7]);
#pragma unroll
        for (int e = 6; e >= 0; --e) code = code * 16 + __float_as_uint(m[e]);
        code -= 0x4b400000u * 0x11111111u;   // (what the sums' upper bits came to, modulo 2^32)
        if (odd) code = 0x88888888u;
        // V: this lane's 8 channels are halfword `group` of chunks 2t and 2t + 1; with the lane of group ^ 1 it makes whole words
        const uint32_t got = __shfl_xor_sync(0xffffffffu, group & 1 ? code : code >> 16, 4);
        if (to >= 0) {
            const int slot = to & (kPage - 1);
            uint8_t* rec = P.cache.records + static_cast<int64_t>(to / kPage) * kRecordBytes;
            const uint32_t word = !is_v ? code : group & 1 ? __byte_perm(got, code, 0x7610) : __byte_perm(code, got, 0x5410);
            const int chunk = 2 * t + (group & 1);
            *reinterpret_cast<uint32_t*>(rec + slot * 64 + (is_v ? kVCodes + (chunk ^ (slot & 4)) * 8 + (group & 2) * 2 : kKCodes + t * 16 + group * 4)) = word;
            if (t == 0) *reinterpret_cast<__nv_bfloat16*>(rec + (is_v ? kVScales : kKScales) + slot * 8 + group * 2) = scale;
            if (P.weights && lane == 0) P.weights[to] = 0.f;
        }
        if (out) {
            const int64_t out_at = __shfl_sync(0xffffffffu, dst_out, (lane & 16) + i);
            const float s = __bfloat162float(scale);
            uint32_t pk[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 q = f2_mul(f2_add(make_float2(m[2 * e], m[2 * e + 1]), make_float2(-12582920.f, -12582920.f)), make_float2(s, s));
                pk[e] = to >= 0 ? pack_act<FP16>(q.x, q.y) : 0u;
            }
            *reinterpret_cast<uint4*>(out + out_at + 8 * l) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
    }
}

}  // namespace
}  // namespace fmsa

extern "C" int fmsa_cache_append(const fmsa_cache_append_args* args, void* stream) {
    using namespace fmsa;
    FMSA_REQUIRE(args);
    const fmsa_cache4* cache = &args->cache;
    const fmsa_tensor *k = &args->k, *v = &args->v, *k_values = args->k_values.ptr ? &args->k_values : nullptr,
                      *v_values = args->v_values.ptr ? &args->v_values : nullptr;
    const int32_t B = args->B, n = args->n, dtype = args->dtype, *cu_seqlens = args->cu_seqlens;
    float* weights = args->weights;
    int32_t* status = args->status;
    FMSA_REQUIRE(cache4_ok(cache) && k->ptr && v->ptr && status && B > 0 && n > 0);
    FMSA_REQUIRE(dtype == FMSA_DTYPE_BF16 || dtype == FMSA_DTYPE_FP16);
    FMSA_REQUIRE(cu_seqlens ? B == 1 : B == cache->seqs);
    FMSA_REQUIRE((k_values == nullptr) == (v_values == nullptr));
    for (const fmsa_tensor* t : {k, v, k_values, v_values})
        if (t) FMSA_REQUIRE(t->ptr && aligned16(t->ptr) && t->stride_b % 8 == 0 && t->stride_h % 8 == 0 && t->stride_s % 8 == 0);
    const int64_t rows = static_cast<int64_t>(B) * cache->heads * n;
    if (rows > 0x7fffff00LL || static_cast<int64_t>(cache->pages) * cache->heads >= (1 << 24)) return FMSA_ERR_UNSUPPORTED;   // (places are 32 bits)
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
    // Four rows a warp once they fill the GPU (64 warps an SM; of 32768 tokens two rows took 74 us, four 61.5, eight 63.6, sixteen 74), one where
    // latency is what counts.
    const int sms = device_sm_count();
    if (sms <= 0) return FMSA_ERR_CUDA;
    const bool many = rows >= static_cast<int64_t>(sms) * 64 * 4, fp16 = dtype == FMSA_DTYPE_FP16;
    const int64_t per_block = kAppendWarps * (many ? 4 : 1);
    P.blocks = static_cast<uint32_t>((rows + per_block - 1) / per_block);
    launch_chained(fp16 ? (many ? cache_append_kernel<true, 4> : cache_append_kernel<true, 1>) : (many ? cache_append_kernel<false, 4> : cache_append_kernel<false, 1>),
                   P.blocks + (cu_seqlens ? 1 : 0), kAppendWarps * 32, 0, static_cast<cudaStream_t>(stream), P);
    return check_launch();
}
