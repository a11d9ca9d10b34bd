// Causal attention of whole prompts over their own keys and values, sequences of different
// lengths packed together; instantiated per type in prompt_bf16.hip and prompt_f32.hip.
//
//   S = scale Q K^T,  out = softmax(S) V  over keys j <= i + (keys - rows) for row i of a sequence
//
// Rows of one kv head are its tokens times the query heads that share it, r = token * group +
// head, so that a tile of rows reads each key once for all of them.  A wave holds 32
// rows; the waves of a workgroup take the same keys, KT at a time, copied into LDS a tile ahead.
//
// The products are 32x32 MFMAs with the keys (and the values, turned) as the first operand: a row of
// the output belongs to lanes l and l ^ 32, whose statistics are their own, and the
// exponentials are the second operand of the product with V as they come out of S:
//   S: lane l holds keys 8 a + 4 (l / 32) + b of 32, register 4 a + b
//   P, as operand of 16 keys: lane l holds registers 8 s .. 8 s + 7 of that order
// The sum over keys may take them in any order if V's operand agrees.
//
// What bounds it: 32 rows by 64 keys of 128 dims are 32 MFMAs of 32 cycles, 1024, and some 160 vector
// instructions, 32 exponentials among them, about as many cycles again; the two waves of a SIMD
// overlap them in part (1830 cycles for the two kinds, the matrix units busy for 56 %).  16384 tokens of 32/8
// heads of 128 dims in bf16 take 2.02 to 2.11 ms by card (1041 to 1091 TFLOP/s; a product of two 8192 x
// 8192 matrices reaches 1400), 8192 tokens of 64 dims 299 to 309 us (890 to 920), of 16/4 heads of 96 234 to 242 (two
// waves a SIMD, whose products and exponentials hardly overlap); 4096 tokens of 32/8 heads in f32 724 to 746 us (184 to
// 190, of six products each).  Prompts of some hundred tokens are bound by their
// rows' bytes and the latencies of a tile's beginning and end: 24 x 700 tokens of 16/8 heads 84 to 86 us.
// Tried without gain: tiles of 32 keys (2319 us instead of 2068), three waves on a SIMD (registers
// spill, 2948), two tiles ahead at 64 dims (316 instead of 284), wave priorities.
#pragma once
#include <algorithm>
#include <type_traits>

#include "prompt_common.hpp"

namespace dmx {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kNone = -__builtin_inff();

// 16 bytes a lane from base + off (base wave-uniform) to LDS offset `to` + 16 lane.  In assembly, because
// the compiler, which cannot tell one stage of the tiles from the other, puts a wait for
// all copies in flight before every read of LDS behind the builtin; ring_barrier waits for these.
// No register is loaded, and the compiler's own counts of what is in flight only become stricter.
// Five wait states lie between a vector instruction that writes the address's scalars (v_readfirstlane)
// and the copy, one between m0 and the copy.
__device__ __forceinline__ void copy16(uint64_t base, uint32_t off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(scalar(to)), "v"(off), "s"(scalar64(base))
                 : "memory");
}
__device__ __forceinline__ void copy16(const uint8_t* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(scalar(to)), "v"(from) : "memory");
}

// 0 times two bf16: NaN where one is not finite.
__device__ __forceinline__ uint32_t times_0(uint32_t x) {
    return ((x & 0x7F80u) == 0x7F80u ? 0x7FC0u : 0u) | ((x & 0x7F800000u) == 0x7F800000u ? 0x7FC00000u : 0u);
}

// The kernel's arguments read again where they are needed: held in scalar registers through the
// loop over the keys they would push out what the loop itself uses.
__device__ __forceinline__ PromptArgs late_args() {
    typedef const __attribute__((address_space(4))) uint32_t word;
    word* p = (word*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    struct Words {
        uint32_t w[sizeof(PromptArgs) / 4];
    } x;
#pragma unroll
    for (uint32_t i = 0; i < sizeof(PromptArgs) / 4; i++) x.w[i] = p[i];
    return __builtin_bit_cast(PromptArgs, x);
}

// f32 in three bf16 terms, x = hi + mid + lo to 2^-24: hi cut off (so that no finite number
// becomes infinite), the others rounded.  Products of terms below 2^-23 of the whole are left out: six
// matrix instructions take the place of eight f32 ones of twice the cycles each (4096 tokens 1230 us with those).
// Split in the kernel, tile by tile: split beforehand into a workspace they took 654 to 730 us, no
// faster, and 104 instead of 56 where 16 rows follow 4000.
struct Terms {
    bf16x8 t[3];
};
__device__ __forceinline__ Terms split8(const float (&x)[8]) {
    u32x4 w[3];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float r[2], m[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float v = x[2 * j + i];
            r[i] = v - __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
            if (fabsf(v) == __builtin_inff()) r[i] = 0.0f;
        }
        w[0][j] = __builtin_amdgcn_perm(__float_as_uint(x[2 * j + 1]), __float_as_uint(x[2 * j]), 0x07060302u);
        w[1][j] = f32x2_to_bf16x2_bits(r[0], r[1]);
        m[0] = r[0] - __uint_as_float(w[1][j] << 16);
        m[1] = r[1] - __uint_as_float(w[1][j] & 0xFFFF0000u);
        w[2][j] = f32x2_to_bf16x2_bits(m[0], m[1]);
    }
    return {{__builtin_bit_cast(bf16x8, w[0]), __builtin_bit_cast(bf16x8, w[1]), __builtin_bit_cast(bf16x8, w[2])}};
}
// a b added to c, small products first.
__device__ __forceinline__ f32x16 mfma_terms(const Terms& a, const Terms& b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[2], b.t[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[0], b.t[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[1], b.t[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[1], b.t[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[0], b.t[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[0], b.t[0], c, 0, 0, 0);
}

// How a tile of KT keys (or values) lies in LDS: rows of RS units of 16 bytes (a power of two),
// unit c of row k at c ^ mix(k); in f32 three planes of them, one for each term.  LDS has 64 banks, 256
// bytes: sixteen lanes that read one unit of consecutive keys, and the rows that one read of the
// values takes together (64 bytes of four keys), are on different ones.
template <int D, bool F32>
struct TileShape {
    static constexpr uint32_t CH = D / 8;  // units of a row
    static constexpr uint32_t RS = CH <= 8 ? 8 : CH <= 16 ? 16 : 32;
    static constexpr uint32_t RSB = RS * 16;
    static constexpr uint32_t KT = RS <= 16 && !F32 ? 64 : 32;
    static constexpr uint32_t PLANE = KT * RSB, BYTES = PLANE * (F32 ? 3 : 1);  // of a term, of K or of V
    // Linear in the bits of k: mix(a ^ b) = mix(a) ^ mix(b).
    static constexpr __device__ uint32_t mix(uint32_t k) {
        return RS == 8 ? (k >> 1 & 1u) << 2 | (k >> 2 & 3u) : (k & 3u) << 2 | (k >> 2 & 3u);
    }
};

// What a wave holds of its 32 rows: all dims, or (HALVES 2) half of them.
template <int D, bool F32, int HALVES>
struct PromptWave {
    using T = TileShape<D, F32>;
    static constexpr int SUB = T::KT / 32, DT = D / 32 / HALVES, QN = D / 16 / HALVES;
    using Frag = std::conditional_t<F32, Terms, bf16x8>;

    Frag q[QN];
    f32x16 o[DT];
    float m, l;        // what exponents are from (in powers of two; kNone: nothing seen yet), sum of this lane's
    float c;           // scale in powers of two
    uint32_t sees;     // keys that this lane's row sees
    static constexpr uint32_t KA = T::RS == 8 ? 4 : 8, VA = T::RS == 8 ? 2 : 4;
    static constexpr uint32_t HALF = D * 2 / HALVES;  // bytes of a half in a row
    static_assert(HALVES == 1 || HALF % 256 == 0, "the second half's units do not mix with the first's");
    uint32_t k_at[KA], v_at[2][VA];  // this lane's places in a tile

    __device__ __forceinline__ void places(uint32_t lane, uint32_t half_of_dims) {
        const uint32_t col = lane & 31u, g = lane >> 5, h0 = half_of_dims * HALF;
#pragma unroll
        for (uint32_t t = 0; t < KA; t++) k_at[t] = h0 + col * T::RSB + (((2 * t + g) ^ T::mix(col)) << 4);
        const uint32_t i = lane & 15u, half = (lane >> 4) & 1u;
#pragma unroll
        for (uint32_t e = 0; e < 2; e++)
#pragma unroll
            for (uint32_t p = 0; p < VA; p++) {
                const uint32_t row = 8 * e + 4 * g + i / 4;
                v_at[e][p] = h0 + row * T::RSB + (((4 * p + 2 * half + (i & 3u) / 2) ^ T::mix(row)) << 4) + 8 * (i & 1u);
            }
    }

    // Of keys k0 + 32 sub + 4 (lane / 32) and on: how many this lane's row sees, up to 32.
    __device__ __forceinline__ uint32_t seen_of(uint32_t k0, uint32_t sub, uint32_t lane) const {
        const uint32_t from = k0 + 32 * sub + 4 * (lane >> 5);
        return sees > from ? min(sees - from, 32u) : 0u;
    }

    // scores of 32 keys
    __device__ __forceinline__ f32x16 scores(const uint8_t* kt, uint32_t sub) const {
        f32x16 s = {};
#pragma unroll
        for (uint32_t t = 0; t < QN; t++) {
            const uint8_t* const at = kt + k_at[t % KA] + (sub * 32 * T::RSB + t / KA * KA * 32);
            if constexpr (F32) {
                Terms k;
#pragma unroll
                for (uint32_t i = 0; i < 3; i++) k.t[i] = *reinterpret_cast<const bf16x8*>(at + i * T::PLANE);
                s = mfma_terms(k, q[t], s);
            } else {
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(at), q[t], s, 0, 0, 0);
            }
        }
        return s;
    }

    // The operand of 32 dims of the values of 16 keys in the order of P.
    __device__ __forceinline__ bf16x8 values(const uint8_t* vt, uint32_t s, uint32_t dt) const {
        typedef __attribute__((address_space(3))) i16x4 lds4;
        i16x4 x[2];
#pragma unroll
        for (uint32_t e = 0; e < 2; e++)
            x[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds4*)(vt + v_at[e][dt % VA] + (16 * s * T::RSB + dt / VA * VA * 64)));
        const u32x2 a = __builtin_bit_cast(u32x2, x[0]), b = __builtin_bit_cast(u32x2, x[1]);
        return __builtin_bit_cast(bf16x8, u32x4{a.x, a.y, b.x, b.y});
    }

    // P V added to the output.  bf16: the exponentials are rounded to 8 bits of mantissa, an error of the
    // size of the output's own rounding.
    __device__ __forceinline__ void add(const f32x16 (&p)[SUB], const uint8_t* vt) {
#pragma unroll
        for (uint32_t s = 0; s < 2 * SUB; s++) {
            float x[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) x[j] = p[s / 2][8 * (s & 1u) + j];
            if constexpr (F32) {
                const Terms pt = split8(x);
#pragma unroll
                for (uint32_t dt = 0; dt < DT; dt++) {
                    Terms v;
#pragma unroll
                    for (uint32_t i = 0; i < 3; i++) v.t[i] = values(vt + i * T::PLANE, s, dt);
                    o[dt] = mfma_terms(v, pt, o[dt]);
                }
            } else {
                u32x4 w;
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) w[j] = f32x2_to_bf16x2_bits(x[2 * j], x[2 * j + 1]);
#pragma unroll
                for (uint32_t dt = 0; dt < DT; dt++)
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(values(vt, s, dt), __builtin_bit_cast(bf16x8, w), o[dt], 0, 0, 0);
            }
        }
    }

    // A tile of keys from k0 on, from the scores on.  masked: some row does not see all of them.
    __device__ __forceinline__ void finish(f32x16 (&p)[SUB], const uint8_t* vt, uint32_t k0, uint32_t lane, bool masked) {
        float top = kNone;
        if (masked) {
            asm volatile("");  // a branch, not a selection in every step
#pragma unroll
            for (uint32_t sub = 0; sub < SUB; sub++) {
                const uint32_t some = seen_of(k0, sub, lane);
#pragma unroll
                for (uint32_t i = 0; i < 16; i++)
                    if (8 * (i >> 2) + (i & 3u) >= some) p[sub][i] = kNone;
            }
        }
#pragma unroll
        for (uint32_t sub = 0; sub < SUB; sub++)
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) top = fmaxf(top, p[sub][i]);
        top *= c;
        // the reference moves only when the largest is 2^8 above it
        if (__any(top > m + 8.0f)) {
            const float now = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
            const float f = now == kNone ? 1.0f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= f;
#pragma unroll
            for (uint32_t dt = 0; dt < DT; dt++) o[dt] *= f;
        }
        const float from = m == kNone ? 0.0f : m;
#pragma unroll
        for (uint32_t sub = 0; sub < SUB; sub++)
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) {
                p[sub][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[sub][i], c, -from));
                l += p[sub][i];
            }
        add(p, vt);
    }
};

template <bool F32>
__device__ __forceinline__ float prompt_element(const KvRows& x, int64_t at) {
    return F32 ? gptr<float>(x.p)[at] : bf16_bits_to_f32(gptr<uint16_t>(x.p)[at]);
}

// Dims d0 .. d0 + DO - 1 of one row by a wave, key after key, each that the row sees and no other: for rows
// beside which infinite or NaN values are masked, where 0 times the value is not 0, and in f32 for rows that
// see an infinity.  A wave takes some 0.17 us a row and key (f32 0.05): one infinite value that all rows see makes
// 4096 tokens of 32/8 heads in f32 35 ms instead of 0.87, one late in them 27, in bf16 24 instead of 0.17.
template <int D, int DO, bool F32>
__device__ __forceinline__ void prompt_row_by_itself(const PromptArgs& a, uint32_t d0, uint64_t q_row, uint32_t q_head, uint64_t key0, uint32_t head,
                                                  int64_t from, int64_t to, bool parts, uint64_t slot) {
    constexpr int N = (DO + 63) / 64;
    const uint32_t lane = threadIdx.x & 63u;
    const float c = a.scale * 1.4426950408889634f;
    const int64_t qa = (int64_t)q_row * a.q.ts + (int64_t)q_head * a.q.hs;
    const int64_t ka = (int64_t)key0 * a.k.ts + (int64_t)head * a.k.hs, va = (int64_t)key0 * a.v.ts + (int64_t)head * a.v.hs;
    float m = kNone, l = 0.0f, o[N] = {};
    for (int64_t j0 = from; j0 < to; j0 += 64) {
        const bool in = j0 + lane < to;
        const int64_t kj = ka + (in ? j0 + (int64_t)lane : j0) * a.k.ts;
        float s = 0.0f;
#pragma unroll 4
        for (int d = 0; d < D; d++) s = __builtin_fmaf(prompt_element<F32>(a.q, qa + d), prompt_element<F32>(a.k, kj + d), s);
        s = in ? s * c : kNone;
        float top = s;
        for (int x = 32; x; x /= 2) top = fmaxf(top, __shfl_xor(top, x));
        const float now = fmaxf(m, top), f = m == kNone ? 0.0f : __builtin_amdgcn_exp2f(m - now), ref = now == kNone ? 0.0f : now;
        const float p = in ? __builtin_amdgcn_exp2f(s - ref) : 0.0f;
        float sum = p;
        for (int x = 32; x; x /= 2) sum += __shfl_xor(sum, x);
        l = l * f + sum;
        if (m != kNone)
            for (int i = 0; i < N; i++) o[i] *= f;
        m = now;
        const int32_t n = (int32_t)min(to - j0, (int64_t)64);
#pragma unroll 1
        for (int32_t j = 0; j < n; j++) {
            const float pj = __shfl(p, j);
            for (int i = 0; i < N; i++)
                if (lane + 64 * i < DO) o[i] = __builtin_fmaf(pj, prompt_element<F32>(a.v, va + (j0 + j) * a.v.ts + d0 + lane + 64 * i), o[i]);
        }
    }
    const bool none = from >= to;
    if (parts) {
        if (lane == 0 && d0 == 0) gptr_mut<float>(a.stats)[2 * slot] = m, gptr_mut<float>(a.stats)[2 * slot + 1] = l;
        for (int i = 0; i < N; i++)
            if (lane + 64 * i < DO) gptr_mut<float>(a.part_o)[slot * D + d0 + lane + 64 * i] = o[i];
        return;
    }
    if (a.lse && lane == 0 && d0 == 0)
        gptr_mut<float>(a.lse)[q_row * (a.heads * a.group) + q_head] = none ? kNone : (m + log2f(l)) * 0.69314718055994531f;
    for (int i = 0; i < N; i++) {
        if (lane + 64 * i >= DO) continue;
        const float y = none ? 0.0f : o[i] / l;
        const int64_t at = (int64_t)q_row * a.out.ts + (int64_t)q_head * a.out.hs + d0 + lane + 64 * i;
        if (F32)
            gptr_mut<float>(a.out.p)[at] = y;
        else
            gptr_mut<uint16_t>(a.out.p)[at] = f32_to_bf16_bits(y);
    }
}

// Workgroup (row tile, sequence, kv head, part of the keys), the last row tiles, which see most
// keys, first.  Four groups of 32 rows; of 256 dims, whose registers would leave one wave to a SIMD, two
// waves share a group: each takes the scores of its half of the dims, the halves are added through LDS,
// and each keeps its half of the output (8192 tokens of 8/2 heads 362 us, by one wave each 540).  VEC: keys and values lie on 16-byte boundaries, less than 64 MB apart.
template <int D>
constexpr int kPromptHalves = D > 128 ? 2 : 1;

template <int D, bool F32, bool VEC>
__global__ __launch_bounds__(2 * kPromptRows * kPromptHalves<D>, 2) void prompt_kernel(PromptArgs a) {
    constexpr int HALVES = kPromptHalves<D>, ALL = kPromptRows / 32 * HALVES;
    using T = TileShape<D, F32>;
    using W = PromptWave<D, F32, HALVES>;
    constexpr uint32_t ROWS = kPromptRows, STAGE = 2 * T::BYTES, STAGES = F32 ? 1 : 2;
    __shared__ __align__(16) uint8_t lds[STAGES * STAGE];
    constexpr uint32_t TURNS = HALVES == 2 && !F32 ? 2 : 1;
    __shared__ f32x4 other[HALVES == 2 ? TURNS * ALL * W::SUB * 4 * 64 : 1];  // scores of the other half
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t group = wave / HALVES, half = wave % HALVES;
    const uint32_t g = lane >> 5, col = lane & 31u;

    uint32_t id = blockIdx.x;
    const uint32_t part = id % a.parts;  // a.parts: the most of any tile
    id /= a.parts;
    const uint32_t head = id % a.heads;
    id /= a.heads;
    const uint32_t seq = id % a.seqs, tile = a.row_tiles - 1 - id / a.seqs;
    PromptRange r = prompt_range(a, seq);
    r = {scalar(r.row0), scalar(r.n), scalar(r.key0), scalar(r.nk), (int64_t)scalar64((uint64_t)r.off)};
    const uint32_t rows = r.n * a.group, tile_row = tile * ROWS;  // below 2^31
    if (tile_row >= rows) return;
    const uint32_t last_row = min(tile_row + ROWS, rows) - 1;
    // keys that some row of the tile sees, and of them this part's
    const uint32_t keys = prompt_keys(r, last_row / a.group);
    const PromptCut cut = prompt_cut(a, keys);
    if (part >= cut.parts) return;
    constexpr uint32_t PER_STEP = 64 / T::KT;
    const uint32_t all = (uint32_t)(((uint64_t)keys + T::KT - 1) / T::KT);
    const uint32_t t0 = min(part * cut.each * PER_STEP, all), t1 = min(t0 + cut.each * PER_STEP, all);

    W w;
    w.places(lane, half);
    const uint32_t wave_row = tile_row + 32 * group, row = wave_row + col;
    const uint32_t token = min(row, last_row) / a.group;
    const uint32_t q_head = head * a.group + (min(row, last_row) - token * a.group);
    w.sees = row <= last_row ? prompt_keys(r, token) : 0u;
    // all keys up to `open` are seen by every row of this wave, none from `shut` on by any
    const bool whole = wave_row + 31 <= last_row;
    const uint32_t open = whole ? prompt_keys(r, wave_row / a.group) : 0u;
    const uint32_t shut = wave_row > last_row ? 0u : prompt_keys(r, min(wave_row + 31, last_row) / a.group);

    // this wave's rows; a negative scale turns their signs, a scale of 0 makes them 0 (what is not finite NaN)
    const float scale = fabsf(a.scale);
    w.c = scale == 0.0f ? 1.0f : scale * 1.4426950408889634f;
    // bf16 rows and outputs on 16-byte boundaries pass through the stage of the tiles that is not in use (256 dims: rows through the place
    // of the halves' scores), whole rows at a time: read and written in pieces of 16 or 32 bytes, as the products hold them, a row's lines move eight
    // times (192 x 128 tokens of 16/8 heads of 128 dims 93 us instead of 78, 768 x 64 of 64 dims 74 instead of 59, 192 x
    // 256 of 256 dims 498 instead of 404; 8192 tokens of 64 dims on the other hand 307 instead of 313).
    uint8_t* const held = HALVES == 1 ? lds + STAGE : reinterpret_cast<uint8_t*>(other);  // rows, before the first tile
    static_assert(F32 || ROWS * T::RSB <= (HALVES == 1 ? STAGE : sizeof(other)), "room for the rows");
    auto load_rows = [&] {  // behind the first tile's copies: one latency for both
        const int64_t at = (int64_t)((uint64_t)r.row0 + token) * a.q.ts + (int64_t)q_head * a.q.hs + half * (D / HALVES);
        const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;
#pragma unroll
        for (uint32_t t = 0; t < W::QN; t++) {
            if constexpr (!F32) {
                u32x4 x;
                if (a.q.vec) {
                    x = *reinterpret_cast<const u32x4*>(held + 32 * group * T::RSB + w.k_at[t % W::KA] + t / W::KA * W::KA * 32);
                } else {
                    const uint16_t* p = static_cast<const uint16_t*>(a.q.p) + at + 16 * t + 8 * g;
#pragma unroll
                    for (int j = 0; j < 4; j++) x[j] = gptr<uint16_t>(p)[2 * j] | (uint32_t)gptr<uint16_t>(p)[2 * j + 1] << 16;
                }
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = a.scale == 0.0f ? times_0(x[j]) : x[j] ^ (a.scale < 0.0f ? 0x80008000u : 0u);
                w.q[t] = __builtin_bit_cast(bf16x8, x);
            } else {
                const float* p = static_cast<const float*>(a.q.p) + at + 16 * t + 8 * g;
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    if (a.q.vec) {
                        const f32x4 y = *gptr<f32x4>(p + j);
#pragma unroll
                        for (int i = 0; i < 4; i++) x[j + i] = y[i] * sign;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) x[j + i] = gptr<float>(p)[j + i] * sign;
                    }
                }
                w.q[t] = split8(x);
            }
        }
    };
    w.m = kNone;
    w.l = 0.0f;
#pragma unroll
    for (uint32_t dt = 0; dt < W::DT; dt++) w.o[dt] = f32x16{};

    // Tile t: its scores, from its keys at LDS offset `at`, and the rest, from its values.
    typedef f32x16 Scores[W::SUB];
    auto live = [&](uint32_t t) { return t * T::KT < shut; };
    auto scores = [&](uint32_t t, uint32_t at, Scores& p) {
        if (!live(t)) return;
#pragma unroll
        for (uint32_t sub = 0; sub < W::SUB; sub++) p[sub] = w.scores(lds + at, sub);
    };
    auto finish = [&](uint32_t t, uint32_t at, Scores& p) {
        if (live(t)) w.finish(p, lds + at, t * T::KT, lane, (t + 1) * T::KT > open);
    };
    // (HALVES 2) The scores of this half of the dims to the other wave, and its own added.
    auto place = [&](uint32_t of, uint32_t i) { return other + (of * W::SUB * 4 + i) * 64 + lane; };
    auto give = [&](uint32_t t, const Scores& p, uint32_t turn) {
        if (!live(t)) return;
#pragma unroll
        for (uint32_t i = 0; i < 4 * W::SUB; i++)
            *place(turn * ALL + wave, i) = f32x4{p[i / 4][4 * (i & 3u)], p[i / 4][4 * (i & 3u) + 1], p[i / 4][4 * (i & 3u) + 2], p[i / 4][4 * (i & 3u) + 3]};
    };
    auto take = [&](uint32_t t, Scores& p, uint32_t turn) {
        if (!live(t)) return;
#pragma unroll
        for (uint32_t i = 0; i < 4 * W::SUB; i++) {
            const f32x4 x = *place(turn * ALL + (wave ^ 1u), i);
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) p[i / 4][4 * (i & 3u) + j] += x[j];
        }
    };

    // Where this head's keys and values begin, and bytes from one to the next.
    auto first = [&](const KvRows& x) {
        return scalar64((uint64_t)(uintptr_t)x.p + (uint64_t)((int64_t)r.key0 * x.ts + (int64_t)head * x.hs) * (F32 ? 4 : 2));
    };
    const uint64_t from[2] = {first(a.k), first(a.v)};
    const uint64_t stride[2] = {scalar64((uint64_t)a.k.ts * (F32 ? 4 : 2)), scalar64((uint64_t)a.v.ts * (F32 ? 4 : 2))};

    if constexpr (F32) {
        // A tile goes through registers, where it is split into its terms: thread i takes units i + 64 ALL j,
        // eight dims each.  The next tile's loads are in flight while this one is worked on.
        constexpr uint32_t UNITS = T::KT * T::CH, N = (UNITS + 64 * ALL - 1) / (64 * ALL);
        f32x4 raw[N][2][2];
        auto load = [&](uint32_t t) {
            const uint32_t left = min(r.nk - t * T::KT, T::KT);  // keys behind the end are the last one
#pragma unroll
            for (uint32_t j = 0; j < N; j++) {
                const uint32_t u = min(threadIdx.x + 64 * ALL * j, UNITS - 1), key = min(u / T::CH, left - 1);
#pragma unroll
                for (uint32_t i = 0; i < 2; i++) {
                    const char* const base = reinterpret_cast<const char*>(from[i] + t * (stride[i] * T::KT));
                    if constexpr (VEC) {
                        const uint32_t at = key * (uint32_t)stride[i] + 32 * (u % T::CH);
#pragma unroll
                        for (uint32_t e = 0; e < 2; e++) raw[j][i][e] = *gptr<f32x4>(base + at + 16 * e);
                    } else {
                        const char* const p = base + key * stride[i] + 32 * (u % T::CH);
#pragma unroll
                        for (uint32_t e = 0; e < 8; e++) raw[j][i][e / 4][e % 4] = gptr<float>(p)[e];
                    }
                }
            }
        };
        if (t0 < t1) load(t0);
        load_rows();
        for (uint32_t t = t0; t < t1; t++) {
            ring_barrier<63>();  // the tile before has been read
#pragma unroll
            for (uint32_t j = 0; j < N; j++) {
                const uint32_t u = threadIdx.x + 64 * ALL * j, key = u / T::CH;
                if (UNITS % (64 * ALL) && u >= UNITS) break;
                uint8_t* const to = lds + key * T::RSB + ((u % T::CH ^ T::mix(key)) << 4);
#pragma unroll
                for (uint32_t i = 0; i < 2; i++) {
                    float x[8];
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) x[e] = raw[j][i][e / 4][e % 4];
                    const Terms y = split8(x);
#pragma unroll
                    for (uint32_t e = 0; e < 3; e++) *reinterpret_cast<bf16x8*>(to + i * T::BYTES + e * T::PLANE) = y.t[e];
                }
            }
            if (t + 1 < t1) load(t + 1);
            ring_barrier<63>();
            Scores p;
            scores(t, 0, p);
            if constexpr (HALVES == 2) {
                give(t, p, 0);
                ring_barrier<63>();
                take(t, p, 0);
            }
            finish(t, T::BYTES, p);
        }
    } else {
        // Copies of a tile: unit blk * 64 + lane of K and of V, blk = wave + ALL j, its key key0 + STEP j,
        // where key0 < STEP, a power of two.  Addresses are a uniform one and 32 bits of the lane's; keys
        // behind the end are the last one.
        constexpr uint32_t COPIES = T::KT * T::RS / 64 / ALL;   // of a wave for K, and for V
        constexpr uint32_t PER = 64 / T::RS, STEP = ALL * PER;  // keys of a copy, of all waves'
        static_assert(COPIES * 64 * ALL == T::KT * T::RS, "whole copies");
        const uint32_t key0 = wave * PER + lane / T::RS, chunk0 = (lane % T::RS) ^ T::mix(key0);
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
        auto fetch = [&](uint32_t t, uint32_t first, uint32_t count) {  // keys (0), values (1)
            const uint32_t at = ((t - t0) & 1u) * STAGE + wave * 1024;
            const uint32_t left = min(r.nk - t * T::KT, T::KT);  // keys that there are
#pragma unroll
            for (uint32_t i = first; i < first + count; i++) {
                uint64_t base = from[i] + t * (stride[i] * T::KT);
                const uint32_t to = at + i * T::BYTES;
                if constexpr (!VEC) {
#pragma unroll 1
                    for (uint32_t j = 0; j < COPIES; j++) {
                        const uint32_t chunk = chunk0 ^ T::mix(STEP * j);
                        if (T::CH < T::RS && chunk >= T::CH) continue;
                        const uint8_t* const p = reinterpret_cast<const uint8_t*>(base + min(key0 + STEP * j, left - 1) * stride[i] + 16 * chunk);
                        u32x4 x;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            x[e] = gptr<uint16_t>(p)[2 * e] | (uint32_t)gptr<uint16_t>(p)[2 * e + 1] << 16;
                        *reinterpret_cast<u32x4*>(lds + to + ALL * j * 1024 + 16 * lane) = x;
                    }
                } else if (left == T::KT) {
                    const uint32_t mine = key0 * (uint32_t)stride[i];
#pragma unroll
                    for (uint32_t j = 0; j < COPIES; j++, base += stride[i] * STEP) {
                        const uint32_t chunk = chunk0 ^ T::mix(STEP * j);
                        if (T::CH < T::RS && chunk >= T::CH) continue;
                        copy16(base, mine + 16 * chunk, lds0 + to + ALL * j * 1024);
                    }
                } else {
#pragma unroll 1
                    for (uint32_t j = 0; j < COPIES; j++) {
                        const uint32_t chunk = chunk0 ^ T::mix(STEP * j);
                        if (T::CH < T::RS && chunk >= T::CH) continue;
                        copy16(base, min(key0 + STEP * j, left - 1) * (uint32_t)stride[i] + 16 * chunk, lds0 + to + ALL * j * 1024);
                    }
                }
            }
        };
        if (t0 < t1) fetch(t0, 0, 2);
        if (a.q.vec) {
            constexpr uint32_t N = ROWS * T::RS / 64 / ALL;
            const uint32_t held0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)held;
#pragma unroll 1
            for (uint32_t j = 0; j < N; j++) {
                const uint32_t at = key0 + STEP * j, chunk = (lane % T::RS) ^ T::mix(at), of = min(tile_row + at, last_row);
                if (T::CH < T::RS && chunk >= T::CH) continue;
                const uint32_t i = of / a.group, h = head * a.group + (of - i * a.group);
                copy16(static_cast<const uint8_t*>(a.q.p) + 2 * ((int64_t)((uint64_t)r.row0 + i) * a.q.ts + (int64_t)h * a.q.hs + 8 * chunk),
                       held0 + wave * 1024 + ALL * j * 1024);
            }
            ring_barrier<0>();
        }
        load_rows();
        if constexpr (HALVES == 1) {
            auto next_tile = [&](uint32_t t) {
                ring_barrier<0>();  // tile t has landed, and the other stage has been read
                if (t + 1 < t1) fetch(t + 1, 0, 2);
            };
            // tiles that some row of this wave sees, then those that others see: one loop for both would have the
            // compiler move an output's registers with every tile
            const uint32_t mine = max(min((shut + T::KT - 1) / T::KT, t1), t0);
            for (uint32_t t = t0; t < mine; t++) {
                next_tile(t);
                const uint32_t at = ((t - t0) & 1u) * STAGE;
                Scores p;
#pragma unroll
                for (uint32_t sub = 0; sub < W::SUB; sub++) p[sub] = w.scores(lds + at, sub);
                w.finish(p, lds + at + T::BYTES, t * T::KT, lane, (t + 1) * T::KT > open);
            }
            for (uint32_t t = mine; t < t1; t++) next_tile(t);
        } else if (t0 < t1) {
            // The scores of a tile ahead of the rest of the one before: one barrier a tile, and products beside
            // exponentials (362 us instead of 397; in f32, whose registers are full, no gain).
            Scores p, next;
            if (t0 + 1 < t1) fetch(t0 + 1, 0, 1);
            ring_barrier<0>();
            scores(t0, 0, next);
            give(t0, next, 0);
            for (uint32_t t = t0; t < t1; t++) {
                ring_barrier<0>();  // values of t and keys of t + 1 have landed, the stages of those before have been read
                const uint32_t turn = (t - t0) & 1u;
                if (t + 1 < t1) fetch(t + 1, 1, 1);
                if (t + 2 < t1) fetch(t + 2, 0, 1);
#pragma unroll
                for (int i = 0; i < W::SUB; i++) p[i] = next[i];
                take(t, p, turn);
                if (t + 1 < t1) {
                    scores(t + 1, (turn ^ 1u) * STAGE, next);
                    give(t + 1, next, turn ^ 1u);
                }
                finish(t, turn * STAGE + T::BYTES, p);
            }
        }
    }

    const PromptArgs b = late_args();
    const uint64_t slot0 = ((((uint64_t)tile * b.seqs + seq) * b.heads + head) * b.parts + part) * b.tile_rows + 32 * group;
    // An infinity or a NaN in the output: of what the row sees, or of values that are masked for it.  In f32 also of
    // an infinity that it sees: a product of terms is NaN (inf 0, or inf - inf) where that of the numbers is infinite.
    // A row whose query holds a NaN is what it should be: no search of all keys for its sake.
    float zeros[4] = {};  // NaN as soon as one is not finite
#pragma unroll
    for (uint32_t dt = 0; dt < W::DT; dt++)
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) zeros[i & 3u] = __builtin_fmaf(w.o[dt][i], 0.0f, zeros[i & 3u]);
    const bool odd = !(zeros[0] + zeros[1] + zeros[2] + zeros[3] == 0.0f);
    const int64_t key_end = min((int64_t)t1 * T::KT, (int64_t)r.nk), key_begin = (int64_t)t0 * T::KT;
    bool bad = false, alone = false;  // alone: rows one by one
    const uint64_t odd_lanes = __ballot(odd);
    uint32_t odd_rows = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);
    if constexpr (F32) {
        for (uint32_t left = odd_rows; left; left &= left - 1) {
            const uint32_t i = (uint32_t)__builtin_ctz(left), rr = min(wave_row + i, last_row), tok = rr / b.group;
            const int64_t at = (int64_t)((uint64_t)r.row0 + tok) * b.q.ts + (int64_t)(head * b.group + (rr - tok * b.group)) * b.q.hs;
            bool nan = false, inf = false;
            for (uint32_t d = lane; d < D; d += 64) {
                const float x = prompt_element<F32>(b.q, at + d);
                nan |= x != x;
                inf |= fabsf(x) == __builtin_inff();
            }
            if (__any(nan))
                odd_rows &= ~(1u << i);
            else
                bad |= inf;
        }
    }
    if (odd_rows) {
        const int64_t first = max((int64_t)prompt_keys(r, min(wave_row, last_row) / b.group), key_begin);
        const int64_t masked = max(min(first, key_end - 1), (int64_t)0);  // the last one stands for keys behind the end as well
#pragma unroll 2
        for (int64_t j = F32 ? key_begin : masked; j < key_end; j++)
            for (uint32_t d = lane; d < D; d += 64) {
                const float v = fabsf(prompt_element<F32>(b.v, (int64_t)(r.key0 + j) * b.v.ts + (int64_t)head * b.v.hs + d));
                bad |= v == __builtin_inff() || (j >= masked && v != v);
                if (F32) bad |= fabsf(prompt_element<F32>(b.k, (int64_t)(r.key0 + j) * b.k.ts + (int64_t)head * b.k.hs + d)) == __builtin_inff();
            }
        alone = __any(bad);
    }
    if constexpr (HALVES == 2) {  // both halves or neither: they share the sum and what exponents are from
        __shared__ bool flag[ALL];
        if (lane == 0) flag[wave] = alone;
        ring_barrier<63>();
        alone = flag[wave] || flag[wave ^ 1u];
    }
    if (alone) {
#pragma unroll 1
        for (uint32_t i = 0; i < 32 && wave_row + i <= last_row; i++) {
            const uint32_t rr = wave_row + i, tok = rr / b.group;
            const int64_t end = min((int64_t)prompt_keys(r, tok), key_end);
            prompt_row_by_itself<D, D / HALVES, F32>(b, half * (D / HALVES), (uint64_t)r.row0 + tok, head * b.group + (rr - tok * b.group),
                                                     r.key0, head, key_begin, end, cut.parts > 1, slot0 + i);
        }
        return;
    }

    w.l += __shfl_xor(w.l, 32);
    const bool live_row = row <= last_row;
    if (cut.parts > 1) {
        if (!live_row) return;
        const uint64_t slot = slot0 + col;
        if (g == 0 && half == 0) {
            gptr_mut<float>(b.stats)[2 * slot] = w.m;
            gptr_mut<float>(b.stats)[2 * slot + 1] = w.l;
        }
#pragma unroll
        for (uint32_t dt = 0; dt < W::DT; dt++)
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                *gptr_mut<f32x4>(b.part_o + slot * D + half * (D / HALVES) + 32 * dt + 8 * i + 4 * g) =
                    f32x4{w.o[dt][4 * i], w.o[dt][4 * i + 1], w.o[dt][4 * i + 2], w.o[dt][4 * i + 3]};
        return;
    }
    const uint32_t i0 = row / b.group, h0 = head * b.group + (row - i0 * b.group);  // computed again, not held
    const uint64_t to_row = (uint64_t)r.row0 + i0;
    // What sees nothing is told by its keys, not by its statistics: scores of NaN, which the maximum passes
    // over, leave a sum of NaN, scores of -inf alone one of 0, and the quotients are NaN.
    const bool none = prompt_keys(r, i0) == 0;
    const float inv = 1.0f / w.l;
    if (b.lse && g == 0 && half == 0 && live_row)
        gptr_mut<float>(b.lse)[to_row * (b.heads * b.group) + h0] = none ? kNone : (w.m + log2f(w.l)) * 0.69314718055994531f;
    const int64_t to = (int64_t)to_row * b.out.ts + (int64_t)h0 * b.out.hs + half * (D / HALVES);
    if (!F32 && b.out.vec) {
        // the stage of the last tile but one, which all waves have left; of 256 dims, behind a barrier, both
        constexpr uint32_t CO = D / HALVES / 8, RO = CO <= 8 ? 128 : 256;  // units of a row (of a half), bytes from one to the next
        uint8_t* const mine = HALVES == 1 ? lds + ((t1 - t0) % 2 ? STAGE : 0) + 32 * group * RO : lds + 32 * wave * RO;
        if (live_row) {
#pragma unroll
            for (uint32_t dt = 0; dt < W::DT; dt++)
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    float y[4];
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) y[j] = none ? 0.0f : w.o[dt][4 * i + j] * inv;
                    *reinterpret_cast<u32x2*>(mine + col * RO + (((4 * dt + i) ^ T::mix(col)) << 4) + 8 * g) =
                        u32x2{f32x2_to_bf16x2_bits(y[0], y[1]), f32x2_to_bf16x2_bits(y[2], y[3])};
                }
        }
        ring_wait<63>();
        const uint32_t count = wave_row > last_row ? 0u : min(last_row - wave_row + 1, 32u);
#pragma unroll
        for (uint32_t j = 0; j < CO / 2; j++) {
            const uint32_t u = 64 * j + lane, of = u / CO, chunk = u % CO;
            const int64_t at = (int64_t)((uint64_t)(uint32_t)__shfl((int)(uint32_t)((uint64_t)to >> 32), (int)of) << 32 |
                                         (uint32_t)__shfl((int)(uint32_t)(uint64_t)to, (int)of));
            if (of < count)
                *gptr_mut<u32x4>(static_cast<uint16_t*>(b.out.p) + at + 8 * chunk) =
                    *reinterpret_cast<const u32x4*>(mine + of * RO + ((chunk ^ T::mix(of)) << 4));
        }
        return;
    }
    if (!live_row) return;
#pragma unroll
    for (uint32_t dt = 0; dt < W::DT; dt++)
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            float y[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) y[j] = none ? 0.0f : w.o[dt][4 * i + j] * inv;
            const int64_t d = to + 32 * dt + 8 * i + 4 * g;
            if constexpr (F32) {
                float* p = static_cast<float*>(b.out.p) + d;
                if (b.out.vec) {
                    *gptr_mut<f32x4>(p) = f32x4{y[0], y[1], y[2], y[3]};
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) gptr_mut<float>(p)[j] = y[j];
                }
            } else {
                uint16_t* p = static_cast<uint16_t*>(b.out.p) + d;
                const u32x2 x = {f32x2_to_bf16x2_bits(y[0], y[1]), f32x2_to_bf16x2_bits(y[2], y[3])};
#pragma unroll
                for (int j = 0; j < 4; j++) gptr_mut<uint16_t>(p)[j] = (uint16_t)(x[j / 2] >> (16 * (j & 1)));
            }
        }
}

}  // namespace

template <bool F32>
hipError_t prompt_launch_typed(const PromptArgs& a, const PromptPlan& plan, hipStream_t st) {
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        constexpr int E = F32 ? 4 : 2;
        const bool vec = a.k.vec && a.v.vec && std::max(a.k.ts, a.v.ts) * E < (1 << 26);
        auto run = [&](auto v) {
            constexpr bool VEC = decltype(v)::value;
            prompt_kernel<D, F32, VEC><<<(uint32_t)plan.grid, 2 * kPromptRows * kPromptHalves<D>, 0, st>>>(a);
        };
        if (vec)
            run(std::true_type());
        else
            run(std::false_type());
        return hipGetLastError();
    };
    switch (a.dim) {
    case 64: return go(std::integral_constant<int, 64>());
    case 96: return go(std::integral_constant<int, 96>());
    case 128: return go(std::integral_constant<int, 128>());
    case 256: return go(std::integral_constant<int, 256>());
    }
    return hipErrorInvalidValue;
}

}  // namespace dmx
