// The key/value cache held in 4 bits: layout of a record and what its kernels share.
//
// A record holds 128 tokens of one KV head: K codes [128][64 bytes], K scales bf16 [128][4], V codes [128][64 bytes], V scales bf16
// [128][4].  A value is (nibble - 8) * the scale of its token and group of 32 channels; nibbles are 1..15 (0 never written: the code is
// symmetric).  Every token's bytes are its own, so that one token can be written or moved alone; inside a row the order of the channels is
// the one in which the tensor core wants them from a thread (cache_attend.cu):
//   K: 16-byte chunk t (0..3), word i (0..3), nibble j (0..7): channel 32 i + 8 t + j
//   V: 8-byte chunk c (0..7) at place c ^ (token & 4), halfword i (0..3), nibble j (0..3): channel 32 i + 4 c + j
// (the exchanged halves of a V row let 16 lanes read 8 bytes of four rows from shared memory without a bank conflict).
#pragma once

#include <stdint.h>

#include "host_common.h"
#include "sm100.cuh"

namespace fmsa {

constexpr int kPage = 128;
constexpr int kKCodes = 0, kKScales = 8192, kVCodes = 9216, kVScales = 17408, kRecordBytes = 18432;
constexpr int kGroup = 32;   // channels that share a scale

// The cache as its kernels see it.  A sequence whose length is beyond what its row of the block table can hold counts as empty (and the status
// word says so): where its last tokens are is not known, so nothing of it is read or written.
struct Cache4 {
    uint8_t* records;         // [pages][heads][kRecordBytes]
    const int32_t* table;     // [seqs][table_stride]
    const int32_t* lengths;   // [seqs]
    int32_t* status;
    int32_t pages, heads, seqs, width, table_stride;

    __device__ __forceinline__ int length(int seq) const {
        const int n = lengths[seq];
        if (n > width * kPage) {
            atomicMax(status, kStatusBadIndex);
            return 0;
        }
        return max(n, 0);
    }
    // Page of a place of a sequence, or -1 (and the status word) where the table does not name one.  0 <= place < width * kPage.
    __device__ __forceinline__ int page(int seq, int at) const {
        const int p = table[static_cast<int64_t>(seq) * table_stride + at];
        if (p >= 0 && p < pages) return p;
        atomicMax(status, kStatusBadIndex);
        return -1;
    }
    __device__ __forceinline__ uint8_t* record(int page, int head) const {
        return records + (static_cast<int64_t>(page) * heads + head) * kRecordBytes;
    }
};

inline bool cache4_ok(const fmsa_cache4* c) {
    return c && c->records && c->block_table && c->lengths && aligned16(c->records) && c->pages > 0 && c->heads > 0 && c->seqs > 0 &&
           c->width > 0 && c->width < (1 << 24) && c->table_stride >= 0 && c->table_stride < (1LL << 31);
}
inline Cache4 device_cache(const fmsa_cache4* c, int32_t* status) {
    Cache4 d;
    d.records = static_cast<uint8_t*>(c->records);
    d.table = c->block_table;
    d.lengths = c->lengths;
    d.status = status;
    d.pages = c->pages; d.heads = c->heads; d.seqs = c->seqs; d.width = c->width;
    d.table_stride = static_cast<int32_t>(c->table_stride);
    return d;
}

}  // namespace fmsa
