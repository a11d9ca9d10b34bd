// Attention over the quantized cache: how a call is cut into workgroups, and the
// second launch that joins the parts of a row whose positions were split
// (attention_impl.hpp holds the kernel itself).
#include "attention_impl.hpp"

namespace dmx {

template <> hipError_t attend_launch<8, 8>(const AttnArgs&, uint32_t, uint64_t, hipStream_t);
template <> hipError_t attend_launch<8, 4>(const AttnArgs&, uint32_t, uint64_t, hipStream_t);
template <> hipError_t attend_launch<4, 8>(const AttnArgs&, uint32_t, uint64_t, hipStream_t);
template <> hipError_t attend_launch<4, 4>(const AttnArgs&, uint32_t, uint64_t, hipStream_t);

namespace {

// One wave per (row, query head): the parts' maxima and sums, then the parts'
// outputs, each brought to the common maximum.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
    constexpr int W = D <= 128 ? 2 : 4;  // dims of a lane
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t q_heads = (uint64_t)a.kv.heads * a.group;
    const uint64_t id = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t h = (uint32_t)(id % q_heads);
    const uint64_t rest = id / q_heads;
    const uint32_t i = (uint32_t)(rest % a.b.max_new);
    if (rest / a.b.max_new >= a.b.seqs) return;
    const SeqRange r = seq_range(a.b, (uint32_t)(rest / a.b.max_new));
    if (i >= r.n) return;
    const uint64_t token = r.row0 + i, total = (uint64_t)r.len + r.n;
    const uint32_t parts = (uint32_t)min((uint64_t)a.splits, (total + a.span - 1) / a.span);
    const uint64_t at = (token * q_heads + h) * a.splits;
    const float* po = a.work + at * D;
    const float* ml = a.work + (uint64_t)a.b.tokens * q_heads * a.splits * D + 2 * at;

    float top = -__builtin_inff();
    for (uint32_t s = lane; s < parts; s += 64) top = fmaxf(top, gptr<float>(ml)[2 * s]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    for (uint32_t s = lane; s < parts; s += 64) sum += gptr<float>(ml)[2 * s + 1] * exp2f(gptr<float>(ml)[2 * s] - ref);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);

    const uint32_t d0 = W * lane;
    if (a.lse && lane == 0)
        gptr_mut<float>(a.lse)[token * q_heads + h] = (top + log2f(sum)) * 0.69314718055994531f;
    if (d0 >= D) return;
    float o[W] = {};
    for (uint32_t s = 0; s < parts; s++) {
        const float f = exp2f(gptr<float>(ml)[2 * s] - ref);
#pragma unroll
        for (int j = 0; j < W; j++) o[j] += f * gptr<float>(po + (uint64_t)s * D)[d0 + j];
    }
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : __builtin_nanf(""));
    const int64_t e = (int64_t)token * a.out.ts + (int64_t)h * a.out.hs + d0;
#pragma unroll
    for (int j = 0; j < W; j++) {
        if (a.out.bf16)
            gptr_mut<uint16_t>(a.out.p)[e + j] = f32_to_bf16_bits(o[j] * inv);
        else
            gptr_mut<float>(a.out.p)[e + j] = o[j] * inv;
    }
}

}  // namespace

// Rows beyond 16 share a pass in twos of tiles where the registers hold them.
// Positions are split until some 768 workgroups are there, or one step of a
// workgroup (256 positions) each is left.
AttnPlan attn_plan(const KvView& kv, const KvBatch& b, uint64_t max_length, uint32_t q_heads, bool bf16) {
    AttnPlan p = {};
    const uint64_t rows = (uint64_t)b.max_new * (q_heads / kv.heads);
    p.tiles = rows <= 16 || (kv.dim > 128 && !bf16) ? 1 : rows <= 32 || kv.dim > 128 || !bf16 ? 2 : 4;
    p.row_tiles = (uint32_t)((rows + 16 * p.tiles - 1) / (16 * p.tiles));
    const uint64_t step = kTile * kWaves;
    const uint64_t steps = max_length > step ? (max_length + step - 1) / step : 1;
    const uint64_t units = (uint64_t)b.seqs * kv.heads * p.row_tiles;
    uint64_t want = units ? (768 + units - 1) / units : 1;
    if (want > steps) want = steps;
    const uint64_t each = (steps + want - 1) / want;
    uint64_t span = each * step;
    if (span > 0x40000000u) span = 0x40000000u;
    p.span = (uint32_t)span;
    p.splits = (uint32_t)((steps * step + span - 1) / span);
    if (p.splits < 1) p.splits = 1;
    if (p.splits > 1) p.bytes = (uint64_t)b.tokens * q_heads * p.splits * (kv.dim + 2) * 4;
    return p;
}

// Units of one part of one head of one sequence, to a multiple of the XCDs, times the row tiles.
uint64_t attn_blocks(const AttnPlan& plan, uint32_t heads, uint32_t seqs) {
    return ((uint64_t)heads * plan.splits * seqs + 7) / 8 * 8 * plan.row_tiles;
}

hipError_t attn_launch(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
    const uint64_t grid = attn_blocks(plan, a.kv.heads, a.b.seqs);
    if (grid == 0) return hipSuccess;
    hipError_t e;
    if (a.kv.k_bits == 8)
        e = a.kv.v_bits == 8 ? attend_launch<8, 8>(a, plan.tiles, grid, st) : attend_launch<8, 4>(a, plan.tiles, grid, st);
    else
        e = a.kv.v_bits == 8 ? attend_launch<4, 8>(a, plan.tiles, grid, st) : attend_launch<4, 4>(a, plan.tiles, grid, st);
    if (e != hipSuccess || plan.splits == 1) return e;
    const uint64_t waves = (uint64_t)a.b.seqs * a.b.max_new * a.kv.heads * a.group;
    const uint32_t blocks = (uint32_t)((waves + 3) / 4);
    switch (a.kv.dim) {
    case 64: join_kernel<64><<<blocks, 256, 0, st>>>(a); break;
    case 96: join_kernel<96><<<blocks, 256, 0, st>>>(a); break;
    case 128: join_kernel<128><<<blocks, 256, 0, st>>>(a); break;
    case 256: join_kernel<256><<<blocks, 256, 0, st>>>(a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace dmx
