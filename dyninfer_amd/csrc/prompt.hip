// Attention of prompts: how a call is cut into workgroups, and the second launch that joins the
// parts of rows whose keys were split (prompt_impl.hpp holds the kernel itself).
#include "prompt_common.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace dmx {

namespace {

// Lanes of a row: four dims each, a power of two of them.
template <int D>
constexpr uint32_t kJoinLanes = D <= 64 ? 16 : D <= 128 ? 32 : 64;

// A row (token, query head) by kJoinLanes<D> * groups threads: each group brings every groups-th
// part to its own maximum, then the groups are joined in LDS.  A part that has no maximum has a sum of 0 (no
// keys for the row, or scores of -inf alone) or of NaN (scores of NaN), which times 0 stays that.  What it reads is small (a float a dim and part);
// bound by latency where rows are few: one token of 32 heads after 16000, 62 parts, by one group took
// 34 us, by groups of about four parts each 5.
template <int D>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs a, uint32_t groups) {
    constexpr uint32_t L = kJoinLanes<D>;
    typedef float vec __attribute__((ext_vector_type(4)));
    __shared__ vec sm_o[256];
    __shared__ float sm_m[256 / L], sm_l[256 / L];
    const uint32_t q_heads = a.heads * a.group, lane = threadIdx.x % L, group = threadIdx.x / L % groups;
    const uint32_t id = blockIdx.x * (256 / L / groups) + threadIdx.x / L / groups;  // rows of split calls are below 2^17
    const uint32_t per = a.max_new * q_heads;
    const uint32_t seq = min(id / per, a.seqs - 1), i = id % per / q_heads, h = id % q_heads;
    const PromptRange r = prompt_range(a, seq);
    const uint32_t r0 = r.row0, head = h / a.group;
    const uint32_t row = i * a.group + (h - head * a.group), tile = row / kPromptRows;
    const uint32_t last_row = min((tile + 1) * kPromptRows, r.n * a.group) - 1;
    const uint32_t parts = i < r.n ? prompt_cut(a, prompt_keys(r, last_row / a.group)).parts : 1u;
    const bool live = id < per * a.seqs && parts > 1;  // the others are written
    const uint32_t d0 = 4 * lane, from = d0 < D ? d0 : 0;
    float m = -__builtin_inff(), l = 0.0f;
    vec o = {};
    if (live) {
        const uint64_t unit = (uint64_t)(tile * a.seqs + seq) * a.heads + head;
        const uint64_t at = unit * a.parts * a.tile_rows + row % kPromptRows;  // of part 0
        for (uint32_t p0 = group; p0 < parts; p0 += 4 * groups) {  // four loads in flight
            float pm[4], pl[4];
            vec po[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                const uint32_t p = p0 + k * groups;
                const uint64_t slot = at + (uint64_t)min(p, parts - 1) * a.tile_rows;
                pm[k] = p < parts ? gptr<float>(a.stats)[2 * slot] : -__builtin_inff();
                pl[k] = p < parts ? gptr<float>(a.stats)[2 * slot + 1] : 0.0f;
                po[k] = *gptr<vec>(a.part_o + slot * D + from);
            }
            const float now = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), m);
            const float ref = now == -__builtin_inff() ? 0.0f : now, f = __builtin_amdgcn_exp2f(m - ref);
            l *= f;
            o *= f;
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                const float g = __builtin_amdgcn_exp2f(pm[k] - ref);
                l += pl[k] * g;
                if (pm[k] != -__builtin_inff()) o += po[k] * g;
            }
            m = now;
        }
    }
    if (groups > 1) {
        sm_o[threadIdx.x] = o;
        if (lane == 0) sm_m[threadIdx.x / L] = m, sm_l[threadIdx.x / L] = l;
        __syncthreads();
        if (group != 0) return;
        const uint32_t t0 = threadIdx.x / L;
        float top = m, sum = 0.0f;
        for (uint32_t g = 1; g < groups; g++) top = fmaxf(top, sm_m[t0 + g]);
        o = vec{};
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        for (uint32_t g = 0; g < groups; g++) {
            const float f = __builtin_amdgcn_exp2f(sm_m[t0 + g] - ref);
            sum += sm_l[t0 + g] * f;
            o += sm_o[threadIdx.x + g * L] * f;
        }
        m = top;
        l = sum;
    }
    if (!live) return;
    const bool none = prompt_keys(r, i) == 0;
    if (a.lse && lane == 0)
        gptr_mut<float>(a.lse)[(r0 + (uint64_t)i) * q_heads + h] = none ? -__builtin_inff() : (m + log2f(l)) * 0.69314718055994531f;
    if (d0 >= D) return;
    const float inv = 1.0f / l;
    const int64_t e = (int64_t)(r0 + (uint64_t)i) * a.out.ts + (int64_t)h * a.out.hs + d0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float y = none ? 0.0f : o[j] * inv;
        if (a.out.bf16)
            gptr_mut<uint16_t>(a.out.p)[e + j] = f32_to_bf16_bits(y);
        else
            gptr_mut<float>(a.out.p)[e + j] = y;
    }
}

}  // namespace

// Tiles of 128 rows, also where there are fewer: waves without rows still copy.  (32 rows by one wave: one token
// of 32/8 heads of 128 dims after 16000 24 us, with four 21; 8 x 8 tokens after 4000 40 and 31, in f32 107
// and 74.)
//
// Whether and into how many parts keys are cut is the least of these times in us, e steps of 64 keys a part:
//   whole   the longest row tile, or all tiles' steps over the places for workgroups
//   parts   a part, or all of them over the places, and the second launch with what it reads and was written for it
// where a workgroup costs some 5 us to begin and end (f32 8), a step what `step` says, as measured on one
// workgroup a compute unit, and where two share one 1.3 times that (f32 1.75); 256 dims fill a unit's LDS.  Of
// 64 dims more than two fit a unit, which the model leaves out: the places are 512 there too.
//   one token after 1000, f32 of 32/8 heads of 128 dims: whole 107 us, parts of 4, 2, 1 (taken) steps 35, 22, 16
//   512 tokens of the same: whole 57 us, parts of 4, 2, 1 steps 44, 42, 57 (taken 46); in bf16 whole (taken) 17, of 4 23,
//   of 2 24, of 1 37
//   2 x 700 tokens of 8/2 heads of 256 dims in f32: whole 124 us, parts of 4, 2 steps 66, 83 (taken 89)
//   2 x 96 tokens of 12/4 heads of 64 dims after 24000 in bf16: whole 349 us, parts of 36, 18, 9, 6 steps 52, 36, 36, 43 (taken 35)
//   3 x 1500 of 8/2 heads of 256 dims in f32, all of one length: whole 253 us, parts of 13, 6, 4 steps 258, 306, 287 (taken 250)
// Above 1024 units the model takes no parts (asked for 1025 to 8192 units of many shapes), so it is not asked there, and the
// join's rows stay below 2^17.
PromptPlan prompt_plan(uint32_t seqs, uint32_t max_new, uint32_t max_keys, uint32_t heads, uint32_t group, uint32_t dim,
                       bool f32) {
    PromptPlan p = {};
    const uint64_t rows = (uint64_t)max_new * group;
    p.row_tiles = (uint32_t)((rows + kPromptRows - 1) / kPromptRows);
    p.tile_rows = (uint32_t)std::min(rows, (uint64_t)kPromptRows);
    const uint64_t units = (uint64_t)seqs * heads * p.row_tiles;
    const uint32_t steps = (uint32_t)(((uint64_t)max_keys + 63) / 64);
    p.parts = 1;
    p.each = 0xFFFFFFFFu;
    if (units && units <= 1024 && steps > 1) {
        const double places = dim > 128 ? 256 : 512;
        const double step = f32 ? (dim == 64 ? 3.5 : dim == 96 ? 4.9 : dim == 128 ? 6.1 : 10)
                                : (dim == 64 ? 1 : dim == 96 ? 1.2 : dim == 128 ? 1.35 : 3);
        const double shared = dim > 128 ? 1 : f32 ? 1.75 : 1.3, ends = f32 ? 8 : 5;
        const double span = std::min(max_new, max_keys) / 64.0, mean = steps - span / 2;  // steps of a row tile, on average
        // n workgroups, of `each` steps the longest and `typical` on average
        auto time = [&](double n, double each, double typical) {
            const double s = step * (n > 256 ? shared : 1);
            return std::max(ends + step * each, n > places ? (n / places + 0.5) * (ends + s * typical) : ends + s * typical);
        };
        double best = time(units, steps, mean);
        const double load = units * mean / places;
        for (uint32_t e = std::max(1u, (uint32_t)(load / 2)); e < steps && e < 8 * load + 64; e += std::max(1u, e / 4)) {
            const double most = (steps + e - 1) / e, least = std::ceil(std::max(steps - span, 1.0) / e), parts = (most + least) / 2;
            const double join = 4.5 + 2.0 * seqs * heads * rows * parts * dim * 4 / 3.8e6;  // one write, one read
            const double t = time(units * parts, e, std::min((double)e, mean / parts)) + join;
            if (t < best) {
                best = t;
                p.each = e;
                p.parts = (uint32_t)most;
            }
        }
    }
    p.grid = units * p.parts;
    if (p.parts > 1) {
        const uint64_t slots = p.grid * p.tile_rows;
        p.stats = slots * dim * 4;
        p.bytes = (p.stats + slots * 8 + 255) / 256 * 256;
    }
    return p;
}

template <bool F32>
hipError_t prompt_launch_typed(const PromptArgs&, const PromptPlan&, hipStream_t);
extern template hipError_t prompt_launch_typed<false>(const PromptArgs&, const PromptPlan&, hipStream_t);
extern template hipError_t prompt_launch_typed<true>(const PromptArgs&, const PromptPlan&, hipStream_t);

hipError_t prompt_launch(PromptArgs a, const PromptPlan& plan, uint8_t* work, hipStream_t st) {
    if (plan.grid == 0) return hipSuccess;
    if (!launchable(plan.grid, a.dim > 128 ? 512 : 256)) return kTooManyThreads;
    a.row_tiles = plan.row_tiles;
    a.tile_rows = plan.tile_rows;
    a.parts = plan.parts;
    a.each = plan.each;
    a.part_o = reinterpret_cast<float*>(work);
    a.stats = reinterpret_cast<float*>(work + plan.stats);
    const hipError_t e = a.q.bf16 ? prompt_launch_typed<false>(a, plan, st) : prompt_launch_typed<true>(a, plan, st);
    if (e != hipSuccess || plan.parts == 1) return e;
    const uint64_t rows = (uint64_t)a.seqs * a.max_new * a.heads * a.group;
    auto join = [&](auto d) {
        constexpr int D = decltype(d)::value;
        uint32_t groups = 1;  // about four parts each
        while (groups < 256 / kJoinLanes<D> && 4 * groups < plan.parts) groups *= 2;
        const uint64_t per = 256 / kJoinLanes<D> / groups, grid = (rows + per - 1) / per;  // split: below 2^17 rows in all
        prompt_join_kernel<D><<<(uint32_t)grid, 256, 0, st>>>(a, groups);
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
