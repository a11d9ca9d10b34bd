// Attention of prompts: how a call is cut into workgroups, and the second launch that joins the
// parts of rows whose keys were split (prompt_impl.hpp holds the kernel itself).
#include "kvcache.hpp"

#include <algorithm>
#include <type_traits>

namespace dmx {

namespace {

// A wave per (row, query head): its parts brought to the common maximum.
template <int D>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs a, uint32_t rows_of_tile) {
    constexpr int W = D <= 128 ? 2 : 4;  // dims of a lane
    typedef float vec __attribute__((ext_vector_type(W)));
    const uint32_t lane = threadIdx.x & 63u, q_heads = a.heads * a.group;
    const uint64_t id = (uint64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t per = (uint64_t)a.max_new * q_heads;
    if (id >= per * a.seqs) return;
    const uint32_t seq = (uint32_t)(id / per), i = (uint32_t)(id % per / q_heads), h = (uint32_t)(id % q_heads);
    auto clip = [&](int32_t x) { return x < 0 ? 0u : min((uint32_t)x, a.tokens); };
    const uint32_t r0 = clip(a.q_starts[seq]), r1 = clip(a.q_starts[seq + 1]);
    if (r1 <= r0 || i >= r1 - r0) return;
    const uint32_t head = h / a.group;
    const uint64_t row = (uint64_t)i * a.group + (h - head * a.group);
    const uint64_t unit = (row / rows_of_tile * a.seqs + seq) * a.heads + head;
    const uint64_t at = unit * a.parts * rows_of_tile + row % rows_of_tile;  // of part 0; parts are rows_of_tile apart
    const uint32_t d0 = W * lane, from = d0 < D ? d0 : 0;
    float top = -__builtin_inff();
    for (uint32_t p = 0; p < a.parts; p++) top = fmaxf(top, gptr<float>(a.stats)[2 * (at + (uint64_t)p * rows_of_tile)]);
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    vec o = {};
    for (uint32_t p = 0; p < a.parts; p++) {
        const uint64_t slot = at + (uint64_t)p * rows_of_tile;
        const float pm = gptr<float>(a.stats)[2 * slot];
        if (pm == -__builtin_inff()) continue;  // saw nothing
        const float f = __builtin_amdgcn_exp2f(pm - ref);
        sum += gptr<float>(a.stats)[2 * slot + 1] * f;
        o += *gptr<vec>(a.part_o + slot * D + from) * f;
    }
    const bool none = top == -__builtin_inff();
    if (a.lse && lane == 0)
        gptr_mut<float>(a.lse)[(r0 + (uint64_t)i) * q_heads + h] = none ? top : (top + log2f(sum)) * 0.69314718055994531f;
    if (d0 >= D) return;
    const float inv = none ? 0.0f : 1.0f / sum;
    const int64_t e = (int64_t)(r0 + (uint64_t)i) * a.out.ts + (int64_t)h * a.out.hs + d0;
#pragma unroll
    for (int j = 0; j < W; j++) {
        if (a.out.bf16)
            gptr_mut<uint16_t>(a.out.p)[e + j] = f32_to_bf16_bits(o[j] * inv);
        else
            gptr_mut<float>(a.out.p)[e + j] = o[j] * inv;
    }
}

}  // namespace

PromptPlan prompt_plan(uint32_t seqs, uint32_t max_new, uint32_t max_keys, uint32_t heads, uint32_t group, uint32_t dim,
                       bool f32) {
    PromptPlan p = {};
    const uint64_t rows = (uint64_t)max_new * group;
    p.waves = rows <= 32 ? 1 : 4;
    const uint32_t tile = 32 * p.waves;
    p.row_tiles = (uint32_t)((rows + tile - 1) / tile);
    const uint64_t units = (uint64_t)seqs * heads * p.row_tiles;
    const uint64_t full = p.waves == 1 ? 1024 : 512, least = 256;  // workgroups at a time, keys of a part
    p.parts = 1;
    if (units && units < full) p.parts = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(full / units, max_keys / least));
    p.grid = units * p.parts;
    if (p.parts > 1) {
        p.stats = p.grid * tile * dim * 4;
        p.bytes = (p.stats + p.grid * tile * 8 + 255) / 256 * 256;
    }
    return p;
}

template <bool F32>
hipError_t prompt_launch_typed(const PromptArgs&, const PromptPlan&, hipStream_t);
extern template hipError_t prompt_launch_typed<false>(const PromptArgs&, const PromptPlan&, hipStream_t);
extern template hipError_t prompt_launch_typed<true>(const PromptArgs&, const PromptPlan&, hipStream_t);

hipError_t prompt_launch(PromptArgs a, const PromptPlan& plan, uint8_t* work, hipStream_t st) {
    if (plan.grid == 0) return hipSuccess;
    if (!launchable(plan.grid, 64 * plan.waves)) return kTooManyThreads;
    a.row_tiles = plan.row_tiles;
    a.parts = plan.parts;
    a.part_o = reinterpret_cast<float*>(work);
    a.stats = reinterpret_cast<float*>(work + plan.stats);
    const hipError_t e = a.q.bf16 ? prompt_launch_typed<false>(a, plan, st) : prompt_launch_typed<true>(a, plan, st);
    if (e != hipSuccess || plan.parts == 1) return e;
    const uint64_t waves = (uint64_t)a.seqs * a.max_new * a.heads * a.group;
    auto join = [&](auto d) {
        prompt_join_kernel<decltype(d)::value><<<(uint32_t)((waves + 3) / 4), 256, 0, st>>>(a, 32 * plan.waves);
        return hipGetLastError();
    };
    switch (a.dim) {
    case 64: return join(std::integral_constant<int, 64>());
    case 96: return join(std::integral_constant<int, 96>());
    case 128: return join(std::integral_constant<int, 128>());
    case 256: return join(std::integral_constant<int, 256>());
    }
    return hipErrorInvalidValue;
}

}  // namespace dmx
