// Attention over the quantized cache: how a call is cut into workgroups, and the
// second launch that joins the parts of a unit whose steps were split
// (attention_impl.hpp holds the kernel itself).
#include "attention_impl.hpp"

namespace dmx {

template <> hipError_t attend_launch<8, 8>(const AttnArgs&, uint32_t, uint64_t, hipStream_t);
template <> hipError_t attend_launch<8, 4>(const AttnArgs&, uint32_t, uint64_t, hipStream_t);
template <> hipError_t attend_launch<4, 8>(const AttnArgs&, uint32_t, uint64_t, hipStream_t);
template <> hipError_t attend_launch<4, 4>(const AttnArgs&, uint32_t, uint64_t, hipStream_t);

namespace {

// SPLIT waves per (row, query head) whose unit was split: the parts' maxima and
// sums, then the parts' outputs, each brought to the common maximum; of SPLIT waves
// every one takes four parts of each 4 SPLIT.  Bound by latency:
// 5.3 us for 8192 rows of two or three parts (7.9 when every wave found its parts by
// itself, with some 260 scalar instructions).
template <int D, int SPLIT>
__global__ __launch_bounds__(SPLIT == 1 ? 256 : 64 * SPLIT) void join_kernel(AttnArgs a, uint32_t tile_shift) {
    constexpr int W = D <= 128 ? 2 : 4;  // dims of a lane
    const uint32_t lane = threadIdx.x & 63u, wave = scalar(threadIdx.x >> 6), p0 = SPLIT == 1 ? 0 : 4 * wave;
    const uint32_t q_heads = a.kv.heads * a.group, seq = blockIdx.y, id = SPLIT == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    const uint32_t i = id / q_heads, h = id - i * q_heads;
    if (i >= a.b.max_new) return;
    const uint32_t kv_head = h / a.group, row = i * a.group + (h - kv_head * a.group);
    const uint32_t* const noted = a.where + 2 * ((seq * a.kv.heads + kv_head) * a.row_tiles + (row >> tile_shift));
    const SeqRange r = seq_range(a.b, seq);
    if (i >= r.n) return;
    const uint32_t parts = noted[1] - noted[0] + 1;
    if (parts == 1) return;  // written by the first launch
    const uint32_t rows_of_tile = 1u << tile_shift;
    const uint64_t at = (uint64_t)noted[0] * rows_of_tile + (row & (rows_of_tile - 1));
    const float* po = a.parts + at * D;
    const float* ml = a.stats + 2 * at;
    const uint64_t pitch = rows_of_tile;  // rows from one part to the next

    const uint32_t d0 = W * lane;
    typedef float vec __attribute__((ext_vector_type(W)));
    vec v[4];
    float f[4];
    auto fetch = [&](uint32_t p) {  // four loads in flight, the first of them before the statistics
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const uint64_t part = min(p + k, parts - 1);
            v[k] = *gptr<vec>(po + part * pitch * D + (d0 < D ? d0 : 0));
            f[k] = gptr<float>(ml)[2 * pitch * part];
        }
    };
    fetch(p0);

    float top = -__builtin_inff();
    for (uint32_t p = lane; p < parts; p += 64) top = fmaxf(top, gptr<float>(ml)[2 * pitch * p]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    for (uint32_t p = lane; p < parts; p += 64)
        sum += gptr<float>(ml)[2 * pitch * p + 1] * exp2f(gptr<float>(ml)[2 * pitch * p] - ref);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);

    if (a.lse && threadIdx.x % (64 * SPLIT) == 0)
        gptr_mut<float>(a.lse)[(r.row0 + (uint64_t)i) * q_heads + h] = (top + log2f(sum)) * 0.69314718055994531f;
    vec o = {};
    for (uint32_t p = p0; p < parts; p += 4 * SPLIT) {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
            if (p + k < parts) o += v[k] * exp2f(f[k] - ref);
        if (p + 4 * SPLIT < parts) fetch(p + 4 * SPLIT);
    }
    if constexpr (SPLIT > 1) {
        __shared__ vec sm[SPLIT][64];
        sm[wave][lane] = o;
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int w = 1; w < SPLIT; w++) o += sm[w][lane];
    }
    if (d0 >= D) return;
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : __builtin_nanf(""));
    const int64_t e = (r.row0 + (int64_t)i) * a.out.ts + (int64_t)h * a.out.hs + d0;
#pragma unroll
    for (int j = 0; j < W; j++) {
        if (a.out.bf16)
            gptr_mut<uint16_t>(a.out.p)[e + j] = f32_to_bf16_bits(o[j] * inv);
        else
            gptr_mut<float>(a.out.p)[e + j] = o[j] * inv;
    }
}

// Eight waves a row for few rows of many parts (whole calls, one wave and eight: one
// row of 8 heads after 16000, 64 parts, 26.5 and 20.0 us, of one head after 100000, 512 parts,
// 87.8 and 35.5; 2016 rows after 2000, 42 parts, 22.9 and 29.2).
template <int D>
void join_launch(const AttnArgs& a, uint32_t shift, uint32_t parts, hipStream_t st) {
    const uint64_t rows = (uint64_t)a.b.max_new * a.kv.heads * a.group;
    // with shares there are fewer sequences than the grid's second axis allows
    if (parts >= 8 && rows * a.b.seqs <= 1024) join_kernel<D, 8><<<dim3((uint32_t)rows, a.b.seqs), 512, 0, st>>>(a, shift);
    else join_kernel<D, 1><<<dim3((uint32_t)((rows + 3) / 4), a.b.seqs), 256, 0, st>>>(a, shift);
}

}  // namespace

// Row tiles: one or two of 16 rows held by every wave, or four, eight or sixteen held
// one or two a wave (four waves, eight of sixteen).  Larger ones decode a position for
// more rows, smaller ones make more workgroups and leave out more of a prompt.  Times (us, ten
// calls in a graph) of 32 query over 8 kv heads, 8 bits, 128 dims [64 dims], with 2, 4, 8 and 16
// tiles, by `work`, the steps of all units of eight tiles:
//   1 x 63 tokens after 500 (80): 18.0 15.2 18.6 23.3 [14.1 13.2 15.7 18.2]; after 4000 (504):
//   30.4 32.3 37.2 38.5 [22.4 24.7 27.8 29.1]; 32 x 63 after 4000 (16128): 409 385 274 263
//   [268 284 204 200]; 1 x 16 after 4000 (128): 24.4 19.4 21.4 27.2 [18.0 15.1 16.7 21.6], after
//   64000 (2004): 65 63 77 103 [45 47 60 87]; 32 x 16 after 1000 (1024): 36 43 55 53 [25 34 44 45]
//   prompts: 1 x 512 (512): 18.6 23.6 31.2 38.3 [13.0 18.9 24.9 30.0]; 1 x 1024 (2048): 44.2 43.6
//   55.1 66.2 [30.8 33.2 43.1 52.5]; 4 x 2048 (32768): 429 391 291 307 [294 208 186 225]; 1 x 512
//   after 8000 (8576): 189 211 154 151 [131 157 116 116]
// f32, whose queries' second terms are in LDS where a wave holds two tiles, with 1, 2, 4 and 16:
//   1 x 8 after 500: 12.0 15.7 14.1 20.1 [10.4 12.9 12.6 16.0], after 60000 (940): 54 49 61 136
//   [37 35 48 92]; 32 x 8 after 4000 (2048): 102 87 115 271 [66 57 88 179]; 32 x 16 after 4000: 189
//   134 130 280 [118 88 94 183]; 8 x 63 after 2000 (2142): 97 73 79 79 [68 52 61 55]; 32 x 63 after
//   1000 (4536): 195 149 121 109 [129 99 72 70]; 4 x 1024 as a prompt: 233 185 131 177 [154 123 82 112]
// 256 dims, with 1 and 4: 1 x 63 after 4000 63 53, 32 x 16 after 1000 121 71, 1 x 16 after 4000 29 36,
// f32 32 x 8 after 4000 248 280.  96 dims and 4 bits order themselves alike, most times within a tenth.
// The rule misses the best by more than a tenth in three places: f32 from 33 rows over contexts that are
// not long (two tiles: 52 for 61 and 88 for 94 above, at 64 dims), f32 prompts of 512 (22.6 for 26.1),
// 256 dims of 64 rows over a short context (29 for 36).
// The steps of all units go in equal shares to as many workgroups as the CUs
// hold at once (two each; one of 256 dims), or one step each if they are fewer:
// sequences differ in length, and a share may end in the middle of a unit.
// Writing and joining parts costs as much as some steps, so units of few steps, and
// units so many that they fill the CUs several times over, are a workgroup each.  In shares and
// whole: one row over 380 positions 11.3 10.5 [10.2 8.7], over 760 11.8 15.7 [10.8 12.5]; 32 ragged
// sequences with 8 rows of up to 500 26.4 18.7 [20.2 13.1], 1000 30.9 27.5 [24.5 19.8], 2000 38.4
// 44.1 [30.9 31.3]; 100 of up to 1500 76.3 76.3 [52.6 50.1], of up to 8000 242 294 [160 207].  256 dims
// 14.0 15.8, 14.5 24.0, 41 37, 53 54, 83 98, 190 226 (taken whole, the rule's loss there), 736 848.
// Rows of a chain see only what lies before them, so a prompt's row tiles differ in
// length, which only whole units make use of: taken where what is left out is worth
// a unit a CU.
AttnPlan attn_plan(const KvView& kv, const KvBatch& b, uint64_t max_length, uint32_t q_heads, bool bf16, bool chain) {
    AttnPlan p = {};
    const uint64_t rows = (uint64_t)b.max_new * (q_heads / kv.heads);
    const bool two = kv.dim <= 128;  // registers hold two tiles of at most 128 dims
    const uint64_t steps = max_length > kStep ? (max_length + kStep - 1) / kStep : 1;
    const double heads = (double)b.seqs * kv.heads, eights = heads * (double)rows / 128, work = eights * (double)steps;
    const bool fresh = chain && 2ull * b.max_new > max_length;  // mostly a prompt
    if (rows <= 16) p.tiles = 1;
    else if (!two) p.tiles = rows <= 32 ? 1 : 4;
    else if (!bf16 && rows <= 32) p.tiles = work <= 900 ? 1 : 2;
    else if (!bf16) p.tiles = rows <= 128 || fresh || work <= 3000 ? 4 : 16;
    else if (rows <= 32) p.tiles = 2;
    else if (work <= 200) p.tiles = 4;
    else if (work <= 1024 || rows <= 64) p.tiles = 2;
    else if (fresh && eights <= 512 && steps <= 16) p.tiles = 4;
    else p.tiles = rows <= 128 || fresh ? 8 : 16;
    const uint32_t tile = 16 * p.tiles;
    p.row_tiles = (uint32_t)((rows + tile - 1) / tile);
    const uint64_t units = (uint64_t)b.seqs * kv.heads * p.row_tiles;
    const uint64_t full = kv.dim > 128 || p.tiles == 16 ? 256 : 512;
    const uint64_t few = (p.tiles <= 2 ? 3 : 1) + units / 32;
    const bool prompt = chain && units * (double)b.max_new >= 2.0 * full * max_length;
    if (steps <= (few < 12 ? few : 12) || units >= 8 * full || prompt) {
        p.grid = units;
        return p;
    }
    const uint64_t places = units * (steps + kUnitCost);
    p.shares = (uint32_t)(places < full ? places : full);
    p.grid = p.shares;
    p.parts = (uint32_t)(p.shares / units);
    const uint64_t slots = (units + p.shares) * tile;
    p.stats = slots * kv.dim * 4;
    p.where = p.stats + slots * 8;
    p.bytes = p.where + 8 * units;
    return p;
}

hipError_t attn_launch(AttnArgs a, const AttnPlan& plan, uint8_t* work, hipStream_t st) {
    if (plan.grid == 0) return hipSuccess;
    // sixteen tiles: eight waves.  A call in shares has few rows, its second launch always fits
    if (!launchable(plan.grid, plan.tiles == 16 ? 512 : 256)) return kTooManyThreads;
    a.row_tiles = plan.row_tiles;
    a.shares = plan.shares;
    a.parts = reinterpret_cast<float*>(work);
    a.stats = reinterpret_cast<float*>(work + plan.stats);
    a.where = reinterpret_cast<uint32_t*>(work + plan.where);
    hipError_t e;
    if (a.kv.k_bits == 8)
        e = a.kv.v_bits == 8 ? attend_launch<8, 8>(a, plan.tiles, plan.grid, st) : attend_launch<8, 4>(a, plan.tiles, plan.grid, st);
    else
        e = a.kv.v_bits == 8 ? attend_launch<4, 8>(a, plan.tiles, plan.grid, st) : attend_launch<4, 4>(a, plan.tiles, plan.grid, st);
    if (e != hipSuccess || plan.shares == 0) return e;
    const uint32_t shift = (uint32_t)__builtin_ctz(16 * plan.tiles);
    switch (a.kv.dim) {
    case 64: join_launch<64>(a, shift, plan.parts, st); break;
    case 96: join_launch<96>(a, shift, plan.parts, st); break;
    case 128: join_launch<128>(a, shift, plan.parts, st); break;
    case 256: join_launch<256>(a, shift, plan.parts, st); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace dmx
