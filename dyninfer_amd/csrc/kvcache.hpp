// The quantized paged cache as kernels see it, and the launches of the cache,
// rotary, attention and verification kernels (kvcache.hip, attention*.hip,
// verify.hip).  The byte layout is stated in include/dyninfer_mi355x.h.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.hpp"

namespace dmx {

enum { KV_Q8 = 1, KV_Q4 = 2 };  // DYNINFER_KV_*

struct KvView {
    uint8_t* k;
    uint8_t* v;
    uint64_t k_scales, v_scales;  // byte offsets of the scales in k and v
    uint64_t pages;
    uint32_t heads, dim;
    uint32_t page_shift;  // log2(page_size)
    uint32_t k_bits, v_bits;
};

struct KvBatch {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* starts;
    uint32_t seqs, table_pages, tokens, max_new;
};

struct KvRows {
    void* p;
    int64_t ts, hs;  // strides in elements
    uint32_t bf16;
    uint32_t vec;  // 1: every row of a head starts at a 16-byte boundary
};

struct RopeView {
    const float* table;
    const int32_t* positions;
    uint32_t table_positions, rot, half;  // half: layout (i, i + rot / 2), else interleaved
};

// A sequence's rows in the call and its committed length.
struct SeqRange {
    uint32_t row0, n;
    uint32_t len;
};

__device__ __forceinline__ SeqRange seq_range(const KvBatch& b, uint32_t s) {
    const int32_t a = b.starts[s], e = b.starts[s + 1];
    const uint32_t row0 = a < 0 ? 0u : min((uint32_t)a, b.tokens);
    const uint32_t end = e < 0 ? 0u : min((uint32_t)e, b.tokens);
    const int32_t l = b.lengths[s];
    return {row0, end > row0 ? min(end - row0, b.max_new) : 0u, l < 0 ? 0u : (uint32_t)l};
}

// The page of chunk c (positions 16c..16c+15) of sequence s, or -1 where absent.
__device__ __forceinline__ int64_t chunk_page(const KvView& kv, const KvBatch& b, uint32_t s, uint32_t c) {
    const uint32_t i = c >> (kv.page_shift - 4u);
    if (i >= b.table_pages) return -1;
    const int32_t p = b.table[(size_t)s * b.table_pages + i];
    return p >= 0 && (uint64_t)p < kv.pages ? (int64_t)p : -1;
}

// First token slot (in tokens of one head) of chunk c of head h on page p: the
// index of its scales' row, and times a token's bytes the place of its codes.
__device__ __forceinline__ uint64_t chunk_slot(const KvView& kv, int64_t p, uint32_t h, uint32_t c) {
    const uint32_t in_page = c & ((1u << (kv.page_shift - 4u)) - 1u);
    return (((uint64_t)p * kv.heads + h) << kv.page_shift) + 16u * in_page;
}

// A launch's threads are counted in 32 bits.  The launches below return kTooManyThreads, and
// enqueue nothing, for calls that would need more.
constexpr hipError_t kTooManyThreads = hipErrorInvalidConfiguration;
inline bool launchable(uint64_t blocks, uint32_t threads) { return blocks <= 0xFFFFFFFFull / threads; }

hipError_t rope_table_launch(uint32_t rot, uint32_t scaling, double theta, double factor, double original, double lo,
                             double hi, double attn, uint32_t positions, float* out, hipStream_t st);
hipError_t rope_launch(const KvRows& x, const KvRows& y, uint32_t tokens, uint32_t heads, uint32_t dim,
                       const RopeView& rope, hipStream_t st);
// rope.table NULL: no rotation; q_heads 0: no queries.
hipError_t kv_append_launch(const KvView& kv, const KvBatch& b, const KvRows& k, const KvRows& v, const RopeView& rope,
                            const KvRows& q, const KvRows& q_out, uint32_t q_heads, hipStream_t st);
// k.p / v.p NULL: not read.
hipError_t kv_read_launch(const KvView& kv, const KvBatch& b, const KvRows& k, const KvRows& v, hipStream_t st);
hipError_t kv_commit_launch(const KvView& kv, const KvBatch& b, const int32_t* path, uint32_t path_stride,
                            const int32_t* counts, hipStream_t st);

// Attention: how a call is cut (host), its workspace and its launch.
struct AttnPlan {
    uint32_t tiles;      // 16-row tiles a workgroup holds: 1 or 2 by every wave, 4, 8 or 16 one or two a wave
    uint32_t row_tiles;  // of the sequence with the most rows
    uint32_t shares;     // equal pieces of all units' steps, a workgroup each; 0: a unit each
    uint32_t parts;      // of a unit, about
    uint64_t grid;
    uint64_t bytes, stats, where;  // workspace, and where its parts begin
};
AttnPlan attn_plan(const KvView& kv, const KvBatch& b, uint64_t max_length, uint32_t q_heads, bool bf16, bool chain);
struct AttnArgs {
    KvView kv;
    KvBatch b;
    KvRows q, out;
    const int64_t* mask;
    float* lse;
    float* parts;     // [share + unit][row of the tile][dim], not yet over their sums
    float* stats;     // [share + unit][row of the tile][2]: what exponents are from, sum
    uint32_t* where;  // [sequence][kv head][row tile][2]: its first and its last part
    uint32_t mask_words, group, row_tiles, shares;
    float scale;
};
hipError_t attn_launch(AttnArgs a, const AttnPlan& plan, uint8_t* work, hipStream_t st);

struct VerifyArgs {
    const void* logits;
    const void* probs;
    int64_t logits_stride, probs_stride, noise_stride;
    uint32_t logits_bf16, probs_bf16;
    const int64_t* tokens_in;
    const int32_t* parents;
    const int32_t* starts;
    const float* temperature;
    const float* uniform;
    const float* noise;
    uint32_t vocab, seqs, tokens, max_new;
    int32_t* path;
    int32_t* counts;
    int64_t* next;
};
uint64_t verify_workspace_bytes(uint32_t seqs, uint32_t tokens, uint32_t vocab);
hipError_t verify_launch(const VerifyArgs& a, uint8_t* work, hipStream_t st);

}  // namespace dmx
