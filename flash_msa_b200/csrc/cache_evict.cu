// Eviction from the cache by accumulated attention weight, per sequence and KV head: the last `recent` tokens stay, and of the others the
// keep - recent with the largest weight; their bytes are copied, in their order, to pages of their own.  (Into other pages, so that every
// copy is independent of every other one, pages that sequences share stay what they are, and order is kept: `recent` means the same the
// next time.)
//
// First kernel, a block per (sequence, KV head): the weight of rank keep - recent by three passes of a radix selection over the weights as
// ordered whole numbers (11 + 11 + 10 bits, one histogram in shared memory), then the list of kept tokens: every warp owns a run of
// tokens, counts, and writes behind what the warps before it count.  The weights are read from memory once (up to kKeysHeld of them are
// held in shared memory; of longer sequences they come from L2 again).  Second kernel, a block per page that is written: 144 + 4 bytes per
// token, bound by HBM.
#include "cache4.cuh"
#include "host_common.h"
#include "sm100.cuh"

namespace fmsa {
namespace {

struct EvictParams {
    Cache4 cache;
    float* weights;             // [pages][heads][128]
    const int32_t* to;          // [seqs][to_stride]
    int32_t* new_lengths;       // [seqs]
    int32_t* kept;              // [seqs][heads][keep]
    int32_t to_stride, to_width, keep, recent, held;
};

constexpr int kSelectThreads = 1024, kBins = 2048, kKeysHeld = 24576;

// Larger weight, larger number; NaN above everything, the two zeros alike.
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) cache_select_kernel(const EvictParams P) {
    extern __shared__ uint32_t keys[];   // [held]
    __shared__ uint32_t bins[kBins], sums[32];
    __shared__ uint32_t found, above;    // digit of the wanted rank, numbers above that digit
    wait_for_previous_kernel();
    const int seq = blockIdx.x / P.cache.heads, head = blockIdx.x % P.cache.heads, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int length = P.cache.length(seq), left = min(length, P.keep);
    int32_t* kept = P.kept + static_cast<int64_t>(blockIdx.x) * P.keep;
    if (head == 0 && tid == 0) P.new_lengths[seq] = left;
    for (int i = left + tid; i < P.keep; i += kSelectThreads) kept[i] = -1;
    if (length <= P.keep) {
        for (int i = tid; i < left; i += kSelectThreads) kept[i] = i;
        return;
    }
    const int others = length - P.recent;    // (recent <= keep < length)
    uint32_t need = P.keep - P.recent;       // of these
    auto weight = [&](int i) {
        const int p = P.cache.page(seq, i / kPage);
        return p < 0 ? 0u : ordered(P.weights[(static_cast<int64_t>(p) * P.cache.heads + head) * kPage + i % kPage]);
    };
    const bool held = others <= P.held;
    if (held)
        for (int i = tid; i < others; i += kSelectThreads) keys[i] = weight(i);
    auto key = [&](int i) { return held ? keys[i] : weight(i); };

    uint32_t prefix = 0, mask = 0;           // digits found so far
    if (need > 0) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0;
            __syncthreads();
            for (int i = tid; i < others; i += kSelectThreads) {
                const uint32_t v = key(i);
                if ((v & mask) == prefix) atomicAdd(&bins[(v >> shift) & ((1u << bits) - 1)], 1u);
            }
            __syncthreads();
            // from the largest digit down: thread i has the two bins from the top
            const uint32_t b0 = bins[kBins - 1 - 2 * tid], b1 = bins[kBins - 2 - 2 * tid];
            uint32_t sum = b0 + b1;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            if (lane == 31) sums[warp] = sum;
            __syncthreads();
            uint32_t before = sum - b0 - b1;
            for (int w = 0; w < warp; ++w) before += sums[w];
            if (before < need && need <= before + b0) {
                found = kBins - 1 - 2 * tid;
                above = before;
            } else if (before + b0 < need && need <= before + b0 + b1) {
                found = kBins - 2 - 2 * tid;
                above = before + b0;
            }
            __syncthreads();
            prefix |= found << shift;
            mask |= ((1u << bits) - 1) << shift;
            need -= above;
            __syncthreads();
        }
    }
    // Kept: numbers above `prefix`, the first `need` equal to it, and the last tokens.  (need = 0: none of the others.)
    const bool none = P.keep == P.recent;
    const int run = ((length + 31) / 32 + 31) / 32 * 32, lo = min(warp * run, length), hi = min(lo + run, length);
    auto classify = [&](int i, bool& more, bool& equal) {
        const bool last = i >= others;
        const uint32_t v = last || i >= hi || none ? 0u : key(i);
        more = i < hi && (last || (!none && v > prefix));
        equal = i < hi && !last && !none && v == prefix;
    };
    uint32_t n_more = 0, n_equal = 0;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        bool more, equal;
        classify(i0 + lane, more, equal);
        n_more += __popc(__ballot_sync(0xffffffffu, more));
        n_equal += __popc(__ballot_sync(0xffffffffu, equal));
    }
    if (lane == 0) {
        sums[warp] = n_more;
        bins[warp] = n_equal;
    }
    __syncthreads();
    uint32_t c_more = 0, c_equal = 0;
    for (int w = 0; w < warp; ++w) {
        c_more += sums[w];
        c_equal += bins[w];
    }
    const uint32_t before_lane = (1u << lane) - 1;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        bool more, equal;
        classify(i0 + lane, more, equal);
        const uint32_t m = __ballot_sync(0xffffffffu, more), e = __ballot_sync(0xffffffffu, equal);
        const uint32_t my_more = c_more + __popc(m & before_lane), my_equal = c_equal + __popc(e & before_lane);
        if (more || (equal && my_equal < need)) kept[my_more + min(my_equal, need)] = i0 + lane;
        c_more += __popc(m);
        c_equal += __popc(e);
    }
}

__global__ void __launch_bounds__(256) cache_move_kernel(const EvictParams P) {
    __shared__ int64_t from[kPage];      // record index * 128 + slot, or -1
    wait_for_previous_kernel();
    const int tid = threadIdx.x, head = blockIdx.y, seq = blockIdx.z, first = blockIdx.x * kPage;
    const int left = P.new_lengths[seq], tokens = min(left - first, kPage);
    if (tokens <= 0) return;
    const int page = P.to[static_cast<int64_t>(seq) * P.to_stride + blockIdx.x];
    if (page < 0 || page >= P.cache.pages) {
        if (tid == 0) atomicMax(P.cache.status, kStatusBadIndex);
        return;
    }
    if (tid < kPage) {
        int64_t f = -1;
        if (tid < tokens) {
            const int at = P.kept[(static_cast<int64_t>(seq) * P.cache.heads + head) * P.keep + first + tid];
            const int p = at >= 0 ? P.cache.page(seq, at / kPage) : -1;
            if (p >= 0) f = (static_cast<int64_t>(p) * P.cache.heads + head) * kPage + at % kPage;
        }
        from[tid] = f;
    }
    __syncthreads();
    uint8_t* to = P.cache.record(page, head);
    const int part = tid & 7;            // 16 bytes of a row: four of K, four of V
    uint4 x[4];
    uint2 sc = make_uint2(0, 0);
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t f = from[(tid >> 3) + 32 * i];
        const int token = (tid >> 3) + 32 * i;
        if (f >= 0) {
            // (a V row's halves stand exchanged where bit 2 of the slot is set)
            const int at = part < 4 ? kKCodes + part * 16 : kVCodes + (part & 3 ^ (((static_cast<int>(f) ^ token) & 4) >> 1)) * 16;
            x[i] = *reinterpret_cast<const uint4*>(P.cache.records + (f / kPage) * kRecordBytes + (f % kPage) * 64 + at);
        }
    }
    const int64_t fs = from[tid & 127];
    if (fs >= 0) {
        sc = *reinterpret_cast<const uint2*>(P.cache.records + (fs / kPage) * kRecordBytes + (tid < kPage ? kKScales : kVScales) + (fs % kPage) * 8);
        if (tid < kPage) w = P.weights[fs];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int token = (tid >> 3) + 32 * i;
        if (from[token] >= 0) *reinterpret_cast<uint4*>(to + token * 64 + (part < 4 ? kKCodes + part * 16 : kVCodes + (part & 3) * 16)) = x[i];
    }
    if (fs >= 0) {
        *reinterpret_cast<uint2*>(to + (tid < kPage ? kKScales : kVScales) + (tid & 127) * 8) = sc;
        if (tid < kPage) P.weights[(static_cast<int64_t>(page) * P.cache.heads + head) * kPage + tid] = w;
    }
}

}  // namespace
}  // namespace fmsa

extern "C" int fmsa_cache_evict(const fmsa_cache_evict_args* args, void* stream) {
    using namespace fmsa;
    FMSA_REQUIRE(args);
    const fmsa_cache4* cache = &args->cache;
    const int32_t new_width = args->new_width, keep = args->keep, recent = args->recent, *new_table = args->new_table;
    const int64_t new_table_stride = args->new_table_stride;
    float* weights = args->weights;
    int32_t *new_lengths = args->new_lengths, *kept = args->kept, *status = args->status;
    FMSA_REQUIRE(cache4_ok(cache) && weights && new_table && new_lengths && kept && status);
    FMSA_REQUIRE(keep > 0 && recent >= 0 && recent <= keep && new_width > 0 && static_cast<int64_t>(new_width) * kPage >= keep);
    FMSA_REQUIRE(new_table_stride >= 0 && new_table_stride < (1LL << 31));
    if (static_cast<int64_t>(cache->seqs) * cache->heads > 0x7fffffffLL || cache->heads > 65535 || cache->seqs > 65535) return FMSA_ERR_UNSUPPORTED;
    EvictParams P = {};
    P.cache = device_cache(cache, status);
    P.weights = weights;
    P.to = new_table;
    P.to_stride = static_cast<int32_t>(new_table_stride);
    P.to_width = new_width;
    P.new_lengths = new_lengths;
    P.kept = kept;
    P.keep = keep;
    P.recent = recent;
    const int64_t longest = static_cast<int64_t>(cache->width) * kPage;
    P.held = static_cast<int32_t>(longest < kKeysHeld ? longest : kKeysHeld);
    const size_t smem = static_cast<size_t>(P.held) * 4;
    if (!ensure_smem_attr(reinterpret_cast<const void*>(cache_select_kernel), static_cast<size_t>(kKeysHeld) * 4)) return FMSA_ERR_CUDA;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    launch_chained(cache_select_kernel, static_cast<unsigned>(cache->seqs * cache->heads), kSelectThreads, smem, st, P);
    const unsigned pages = static_cast<unsigned>((keep + kPage - 1) / kPage);
    launch_chained(cache_move_kernel, dim3(pages, static_cast<unsigned>(cache->heads), static_cast<unsigned>(cache->seqs)), 256, 0, st, P);
    return check_launch();
}
