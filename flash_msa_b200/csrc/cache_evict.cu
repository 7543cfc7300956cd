// Eviction from the cache by accumulated attention weight, per sequence and KV head: the last `recent` tokens stay, and of the others the
// keep - recent with the largest weight; their bytes are copied, in their order, to pages of their own.  (Into other pages, so that every
// copy is independent of every other one, pages that sequences share stay what they are, and order is kept: `recent` means the same the
// next time.)
//
// First kernel, a block per (sequence, KV head): the weight of rank keep - recent among the weights as ordered whole numbers by up to three
// histograms of 2048 bins in shared memory, then the list of kept tokens in order.  Up to kHeld * 512 tokens the numbers stay in registers, bins
// divide the range that is still open, the search ends with the bin whose keys are just those still needed, and the list comes from one
// scan of (larger, equal) counts.  (32 sequences of up to 8192 tokens, 8 heads: 13.8 us, most of it waiting: lengths, table, weights, and the
// block's barriers; bins of the keys' upper bits 14.9, bit by bit with one count over the block each 22.7.)  Of longer sequences kKeysHeld numbers
// are held in shared memory and more come from L2 again, by radix selection (11 + 11 + 10 bits); every warp counts and writes a run of tokens.
// Second kernel, a block per page that is written: 144 + 4 bytes per token, 45 us there: at the memory rate (6.2 TB/s of what passes HBM).
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
    int32_t to_stride, keep, recent, held;
};

constexpr int kSelectThreads = 1024, kBins = 2048, kKeysHeld = 24576, kHeldThreads = 512, kHeld = 64;

// Larger weight, larger number; NaN above everything, the two zeros alike.
__device__ __forceinline__ uint32_t ordered(float w) {
    const uint32_t u = __float_as_uint(w + 0.f);
    const uint32_t v = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
    return w != w ? 0xffffffffu : v;
}

// Weights of the first `others` tokens of a sequence, as ordered numbers (all of them above 0; tokens of pages that do not exist below all others).
__device__ __forceinline__ uint32_t weight_of(const EvictParams& P, int seq, int head, int i) {
    const int p = P.cache.page(seq, i / kPage);
    return p < 0 ? 1u : ordered(P.weights[(static_cast<int64_t>(p) * P.cache.heads + head) * kPage + i % kPage]);
}
// What both forms begin with: new lengths, the end of the list, sequences that are short enough.  True if there is nothing left to do.
__device__ __forceinline__ bool short_enough(const EvictParams& P, int seq, int head, int length, int32_t* kept) {
    const int left = min(length, P.keep), tid = threadIdx.x;
    if (head == 0 && tid == 0) P.new_lengths[seq] = left;
    for (int i = left + tid; i < P.keep; i += blockDim.x) kept[i] = -1;
    if (length > P.keep) return false;
    for (int i = tid; i < left; i += blockDim.x) kept[i] = i;
    return true;
}

// Sequences of up to HELD * kHeldThreads tokens.
template <int HELD>
__global__ void __launch_bounds__(kHeldThreads, HELD <= 16 ? 2 : 1) cache_select_held_kernel(const EvictParams P) {
    constexpr int kWarps = kHeldThreads / 32;
    __shared__ uint32_t bins[kBins], sums[kWarps], counts[HELD * kWarps];
    __shared__ uint3 digit;   // the wanted bin, keys of larger ones, its own keys
    wait_for_previous_kernel();
    const int seq = blockIdx.x / P.cache.heads, head = blockIdx.x % P.cache.heads, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int length = P.cache.length(seq);
    int32_t* kept = P.kept + static_cast<int64_t>(blockIdx.x) * P.keep;
    if (short_enough(P, seq, head, length, kept)) return;
    const int others = length - P.recent;    // (recent <= keep < length)
    const uint32_t need = P.keep - P.recent; // of these
    uint32_t key[HELD];                      // of token kHeldThreads * j + tid; 0 behind the last
    // (all pages, then all weights, then what they are: with a branch between two loads each would wait for the one before, 16000 cycles
    // instead of 2000 for 8192 tokens.  A page that does not exist is page 0 until then.)
    const int32_t* table = P.cache.table + static_cast<int64_t>(seq) * P.cache.table_stride;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < HELD; ++j) key[j] = static_cast<uint32_t>(table[min(j * kHeldThreads + tid, others - 1) / kPage]);
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const bool fine = key[j] < static_cast<uint32_t>(P.cache.pages);
        bad |= !fine;
        const int64_t page = fine ? key[j] : 0u;
        key[j] = __float_as_uint(P.weights[(page * P.cache.heads + head) * kPage + (j * kHeldThreads + tid) % kPage]);
    }
#pragma unroll
    for (int j = 0; j < HELD; ++j) key[j] = j * kHeldThreads + tid < others ? ordered(__uint_as_float(key[j])) : 0u;
    if (bad) {   // (here, out of the way of the loads)
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const int i = j * kHeldThreads + tid;
            if (i < others && P.cache.page(seq, i / kPage) < 0) key[j] = 1u;
        }
    }
    // the largest number that `need` keys reach.  Bins divide the range of the keys that are there (weights lie in a few octaves: under the
    // keys' upper 11 bits most atomics of a warp would meet in the same bins), then the range of one bin, until that holds just the keys that
    // are still needed, or one number.
    uint32_t rank = 0xffffffffu, rest = need, lo = 0xffffffffu, width = 0;   // of keys from lo to lo + width - 1
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        lo = min(lo, key[j] - 1);    // (0 is none, and goes round)
        width = max(width, key[j]);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    width = __reduce_max_sync(0xffffffffu, width);
    if (lane == 0) {
        sums[warp] = lo;
        counts[warp] = width;
    }
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, sums[lane % kWarps]) + 1;
    width = __reduce_max_sync(0xffffffffu, counts[lane % kWarps]) - lo + 1;
    while (rest) {                   // at most three times: 11 bits of the range each
        const int shift = max(21 - __clz(width - 1), 0);
        for (int i = tid; i < kBins; i += kHeldThreads) bins[i] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < HELD; ++j)
            if (key[j] - lo < width) atomicAdd(&bins[(key[j] - lo) >> shift], 1u);
        __syncthreads();
        // from the largest bin down: a thread has kRun
        constexpr int kRun = kBins / kHeldThreads;
        uint32_t n[kRun], sum = 0;
#pragma unroll
        for (int y = 0; y < kRun; ++y) sum += n[y] = bins[kBins - 1 - kRun * tid - y];
        uint32_t at = sum;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += v;
        }
        if (lane == 31) sums[warp] = at;
        __syncthreads();
        const uint32_t w = lane < kWarps ? sums[lane] : 0;
        at += __reduce_add_sync(0xffffffffu, lane < warp ? w : 0) - sum;   // keys of larger bins
#pragma unroll
        for (int y = 0; y < kRun; ++y) {
            if (at < rest && rest <= at + n[y]) digit = make_uint3(kBins - 1 - kRun * tid - y, at, n[y]);
            at += n[y];
        }
        __syncthreads();
        const uint3 d = digit;
        lo += d.x << shift;
        rank = lo;
        rest -= d.y;
        if (rest == d.z) {
            --rank;       // (all keys from here on: none is equal to the number below, but for some that there is no room for)
            break;
        }
        if (shift == 0) break;
        width = min(1u << shift, 0u - lo);   // (not past the largest number, which is NaN's: the 0 of threads without a token would be in it)
    }
    // Kept: keys above `rank`, the first ones equal to it as far as there is room, and the last tokens.  Counts of both in one word.
    uint32_t mine[HELD];       // before this token, in its row of 32
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const int i = j * kHeldThreads + tid;
        const uint32_t more = __ballot_sync(0xffffffffu, i < length && (i >= others || key[j] > rank));
        const uint32_t equal = __ballot_sync(0xffffffffu, i < others && key[j] == rank);
        const uint32_t before = (1u << lane) - 1;
        mine[j] = __popc(more & before) | __popc(equal & before) << 16;
        if (lane == 0) counts[j * kWarps + warp] = __popc(more) | __popc(equal) << 16;
    }
    __syncthreads();
    // exclusive sums of the counts, of which a lane of the first warp has a run (at most 32K tokens: the halves do not run over)
    if (warp == 0) {
        constexpr int kRun = HELD * kWarps / 32;
        uint32_t c[kRun], sum = 0;
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
            c[j] = counts[lane * kRun + j];
            sum += c[j];
        }
        uint32_t at = sum;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += v;
        }
        if (lane == 31) sums[0] = at;
        at -= sum;
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
            counts[lane * kRun + j] = at;
            at += c[j];
        }
    }
    __syncthreads();
    const uint32_t room = P.keep - (sums[0] & 0xffffu);
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const int i = j * kHeldThreads + tid;
        const bool more = i < length && (i >= others || key[j] > rank), equal = i < others && key[j] == rank;
        const uint32_t at = counts[j * kWarps + warp] + mine[j], equals = at >> 16;
        if (more || (equal && equals < room)) kept[(at & 0xffffu) + min(equals, room)] = i;
    }
}

__global__ void __launch_bounds__(kSelectThreads) cache_select_kernel(const EvictParams P) {
    extern __shared__ uint32_t keys[];   // [held]
    __shared__ uint32_t bins[kBins], sums[32];
    __shared__ uint32_t found, above;    // digit of the wanted rank, numbers above that digit
    wait_for_previous_kernel();
    const int seq = blockIdx.x / P.cache.heads, head = blockIdx.x % P.cache.heads, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int length = P.cache.length(seq);
    int32_t* kept = P.kept + static_cast<int64_t>(blockIdx.x) * P.keep;
    if (short_enough(P, seq, head, length, kept)) return;
    const int others = length - P.recent;    // (recent <= keep < length)
    uint32_t need = P.keep - P.recent;       // of these
    auto weight = [&](int i) { return weight_of(P, seq, head, i); };
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
        const uint32_t to = my_more + min(my_equal, need);   // (below keep, unless the weights change meanwhile)
        if ((more || (equal && my_equal < need)) && to < static_cast<uint32_t>(P.keep)) kept[to] = i0 + lane;
        c_more += __popc(m);
        c_equal += __popc(e);
    }
}

__global__ void __launch_bounds__(256) cache_move_kernel(const EvictParams P) {
    __shared__ int64_t from[kPage];      // record index * 128 + slot; -1 behind the last token, -2 (zeros) if its page does not exist
    wait_for_previous_kernel();
    const int tid = threadIdx.x, head = blockIdx.y, seq = blockIdx.z, first = blockIdx.x * kPage;
    const int page = P.to[static_cast<int64_t>(seq) * P.to_stride + blockIdx.x];
    bool some = false;
    if (tid < kPage) {
        int64_t f = -1;
        const int at = first + tid < P.keep ? P.kept[(static_cast<int64_t>(seq) * P.cache.heads + head) * P.keep + first + tid] : -1;
        const int p = at >= 0 ? P.cache.page(seq, at / kPage) : -1;
        if (at >= 0) f = p < 0 ? -2 : (static_cast<int64_t>(p) * P.cache.heads + head) * kPage + at % kPage;
        from[tid] = f;
        some = f != -1;
    }
    if (!__syncthreads_or(some)) return;
    if (page < 0 || page >= P.cache.pages) {
        if (tid == 0) atomicMax(P.cache.status, kStatusBadIndex);
        return;
    }
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
    uint8_t* half = to + (tid < kPage ? kKCodes : kVCodes);
    if (fs == -2) {
#pragma unroll
        for (int c = 0; c < 4; ++c) reinterpret_cast<uint4*>(half + (tid & 127) * 64)[c] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
    }
    if (fs != -1) {
        *reinterpret_cast<uint2*>(half + kKScales + (tid & 127) * 8) = sc;
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
    P.new_lengths = new_lengths;
    P.kept = kept;
    P.keep = keep;
    P.recent = recent;
    const int64_t longest = static_cast<int64_t>(cache->width) * kPage;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned blocks = static_cast<unsigned>(cache->seqs * cache->heads);
    // (by the longest sequence that the table can hold, which is what the host knows)
    if (longest <= 4 * kHeldThreads) {
        launch_chained(cache_select_held_kernel<4>, blocks, kHeldThreads, 0, st, P);
    } else if (longest <= 16 * kHeldThreads) {
        launch_chained(cache_select_held_kernel<16>, blocks, kHeldThreads, 0, st, P);
    } else if (longest <= kHeld * kHeldThreads) {
        launch_chained(cache_select_held_kernel<kHeld>, blocks, kHeldThreads, 0, st, P);
    } else {
        P.held = kKeysHeld;
        const size_t smem = static_cast<size_t>(P.held) * 4;
        if (!ensure_smem_attr(reinterpret_cast<const void*>(cache_select_kernel), smem)) return FMSA_ERR_CUDA;
        launch_chained(cache_select_kernel, blocks, kSelectThreads, smem, st, P);
    }
    const unsigned pages = static_cast<unsigned>((keep + kPage - 1) / kPage);
    launch_chained(cache_move_kernel, dim3(pages, static_cast<unsigned>(cache->heads), static_cast<unsigned>(cache->seqs)), 256, 0, st, P);
    return check_launch();
}
