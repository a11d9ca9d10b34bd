// What the attention of prompts and the launch that joins its parts share (prompt_impl.hpp, prompt.hip).
#pragma once
#include "kvcache.hpp"

namespace dmx {

namespace {

constexpr uint32_t kPromptRows = 128;  // of a row tile: four waves (of 256 dims four pairs) of 32

// A number that is the same in every lane, as a scalar.
__device__ __forceinline__ uint32_t scalar(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ __forceinline__ uint64_t scalar64(uint64_t x) {
    return (uint64_t)scalar((uint32_t)(x >> 32)) << 32 | scalar((uint32_t)x);
}

// A sequence's rows and keys in the call.
struct PromptRange {
    uint32_t row0, n;   // rows that the call takes
    uint32_t key0, nk;
    int64_t off;        // row i sees keys j <= i + off
};

__device__ __forceinline__ PromptRange prompt_range(const PromptArgs& a, uint32_t s) {
    auto clip = [](int32_t x, uint32_t top) { return x < 0 ? 0u : min((uint32_t)x, top); };
    const uint32_t r0 = clip(a.q_starts[s], a.tokens), r1 = clip(a.q_starts[s + 1], a.tokens);
    const uint32_t k0 = clip(a.k_starts[s], a.keys), k1 = clip(a.k_starts[s + 1], a.keys);
    PromptRange r;
    r.row0 = r0;
    r.key0 = k0;
    const uint32_t n = r1 > r0 ? r1 - r0 : 0u;
    r.nk = k1 > k0 ? k1 - k0 : 0u;
    r.n = min(n, a.max_new);
    r.off = (int64_t)r.nk - n;
    return r;
}

// Keys, from the first on, that token i of the sequence sees: below 2^31, as rows of one kv head are too.
__device__ __forceinline__ uint32_t prompt_keys(const PromptRange& r, uint32_t token) {
    const int64_t n = (int64_t)token + r.off + 1;
    return n <= 0 ? 0u : (uint32_t)n;
}

// How the keys of a row tile are cut: parts of `each` steps of 64 keys.
struct PromptCut {
    uint32_t parts, each;
};
__device__ __forceinline__ PromptCut prompt_cut(const PromptArgs& a, uint32_t keys) {
    const uint32_t steps = (uint32_t)(((uint64_t)keys + 63) / 64);
    const uint32_t n = steps > a.each ? min((steps + a.each - 1) / a.each, a.parts) : 1u;  // more keys than the plan was told of: larger parts
    return {n, (steps + n - 1) / n};
}

}  // namespace

}  // namespace dmx
