// The 8-bit K/V cache: its record and what its kernels are launched with.
//
// One record per (page, layer, K/V head), hdp = the head size rounded up to 16:
//   K codes   int8 [4][hdp/16][4][16]: token 4a + r, dimension 16c + i at
//             ((a * hdp/16 + c) * 4 + r) * 16 + i
//   V codes   int8 [hdp][16]: dimension d, token t at d * 16 + t
//   K scales, V scales   fp32 [16] each, one per token
// Both orders are those of the integer matrix instructions' operands: a lane's
// 16 bytes are 16 dimensions of one K row, or the page's 16 tokens of one V
// column, so attention loads operands straight from the cache.  A scale covers
// one token of one head: pages fill a token at a time (and a batch may write
// several tokens of a page at once), and a scale over more tokens would have to
// be raised, and older codes rounded again, as they arrive.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace nitro {

constexpr int kv_q8_padded(int head_dim) { return (head_dim + 15) / 16 * 16; }
constexpr int kv_q8_record_bytes(int head_dim) { return 32 * kv_q8_padded(head_dim) + 128; }

// A layer of an 8-bit cache.
struct KvQ8 {
    uint8_t* cache;
    int64_t page_stride, layer_off;  // bytes, multiples of 128; pages * page_stride < 2^39
    int32_t kv_heads, head_dim, hdp, record, num_pages;
    int32_t* bad_pages;
};

// New rows of a step: row r lies at position pos[r] in slot slots[r] (page * 16
// + position % 16).  together: they are mostly chunks, consecutive rows of one
// sequence, and taken by whole pages (any rows would come out the same).
struct KvQ8Rows {
    const int32_t* slots;
    const int32_t* pos;
    int32_t rows;
    bool together;
};

struct PrefillSeq;

// Appends k, v [rows][kv_heads * head_dim].  With freq_real, q [rows][n_heads *
// head_dim] and k are first rotated in place.
hipError_t launch_kv_q8_append(const KvQ8& c, const KvQ8Rows& r, float* q, float* k,
                               const float* v, const float* freq_real, const float* freq_imag, int n_heads,
                               hipStream_t stream);
// k, v = the values that those slots hold.
hipError_t launch_kv_q8_read(const KvQ8& c, const KvQ8Rows& r, float* k, float* v,
                             hipStream_t stream);

// Keys that a wave takes at a time: four pages.
constexpr int KV_Q8_TILE = 64;
// Query heads of one K/V head that a decode workgroup serves at most (the
// columns of its matrix instructions).
constexpr int KV_Q8_COLUMNS = 16;

// Sequences of a decode launch that are taken in an order of their own at most.
constexpr int KV_Q8_ORDERED = 128;

struct KvQ8Decode {
    KvQ8 c;
    const float* q;
    float* out;
    const int32_t* tables;
    const int32_t* positions;
    float* partials;    // per (b, split, head): acc[head_dim], m, l; pstride floats
    int32_t* counters;  // per (b, K/V head, group of its query heads), zero between launches
    int32_t batch, n_heads, max_pages, ctx_limit;
    int32_t tiles_per_split, num_splits, waves, pstride;
    int32_t stream_kv;  // no record is read twice: loads that stay out of the caches
    float qscale;  // log2(e) / sqrt(head_dim)
    // Not 0 (the number of CUs): unsplit sequences are taken in this order, every
    // second round of CUs backwards.  Any order of them is right.
    int32_t ordered;
    uint8_t order[KV_Q8_ORDERED];
};
// Waves per SIMD of the decode kernel.
constexpr int kv_q8_decode_occupancy(int hdp) { return hdp <= 64 ? 4 : hdp <= 128 ? 2 : 1; }
// Floats of a partial: acc[head_dim], m, l, on 16 bytes.
inline int kv_q8_partial_floats(int head_dim) { return (head_dim + 2 + 3) / 4 * 4; }
constexpr size_t KV_Q8_LDS = 65536 - 64;  // of a decode workgroup at most
// Bytes of LDS of a decode workgroup: its waves' parts, later a join's factors.
inline size_t kv_q8_decode_lds(int n_heads, int kv_heads, int pstride, int waves, int num_splits) {
    const int kv_mul = n_heads / kv_heads, cols = kv_mul < KV_Q8_COLUMNS ? kv_mul : KV_Q8_COLUMNS;
    const size_t parts = (size_t)waves * cols * pstride, join = (size_t)cols * (num_splits + 1);
    return sizeof(float) * (parts > join ? parts : join);
}
hipError_t launch_kv_q8_decode(const KvQ8Decode& a, hipStream_t stream);

struct KvQ8Prefill {
    KvQ8 c;
    const float* q;
    float* out;
    const int32_t* tables;
    const PrefillSeq* seqs;
    const int32_t* work;  // pairs (seq, first query row of the chunk)
    int32_t work_items, item_rows, n_heads, max_pages, num_cus;
    float qscale;
};
hipError_t launch_kv_q8_prefill(const KvQ8Prefill& a, hipStream_t stream);

}  // namespace nitro
