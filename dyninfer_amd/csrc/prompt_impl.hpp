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
#pragma once
#include <type_traits>

#include "kvcache.hpp"

namespace dmx {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kNone = -__builtin_inff();

// A number that is the same in every lane, as a scalar.
__device__ __forceinline__ uint32_t scalar(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ __forceinline__ uint64_t scalar64(uint64_t x) {
    return (uint64_t)scalar((uint32_t)(x >> 32)) << 32 | scalar((uint32_t)x);
}

// 16 bytes a lane from base + off (base wave-uniform) to LDS offset `to` + 16 lane.  In assembly, because
// the compiler, which cannot tell one stage of the tiles from the other, puts a wait for
// all copies in flight before every read of LDS behind the builtin; ring_barrier waits for these.
// No register is loaded, and the compiler's own counts of what is in flight only become stricter.
// Five wait states lie between a vector instruction that writes the address's scalars (v_readfirstlane)
// and the copy, one between m0 and the copy.
__device__ __forceinline__ void copy16(uint64_t base, uint32_t off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base)
                 : "memory");
}
__device__ __forceinline__ void copy16(const uint8_t* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}

// A sequence's rows and keys in the call.
struct PromptRange {
    uint32_t row0, n;   // rows that the call takes
    uint32_t key0, nk;
    int64_t off;        // row i sees keys j <= i + off
};

__device__ __forceinline__ PromptRange prompt_range(const PromptArgs& a, uint32_t s) {
    auto clip = [](int32_t x, uint32_t top) { return scalar(x < 0 ? 0u : min((uint32_t)x, top)); };
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

// How a tile of KT keys (or values) lies in LDS: rows of RS units of 16 bytes (a power of two),
// unit c of row k at c ^ mix(k).  LDS has 64 banks, 256 bytes: sixteen lanes that read one unit of
// consecutive keys, and the rows that one read of the values takes together (bf16: 64 bytes of four
// keys; f32: 128 bytes of two, four keys apart), are on different ones.
template <int D, bool F32>
struct TileShape {
    static constexpr uint32_t E = F32 ? 4 : 2, CH = D * E / 16;  // bytes of an element, units of a row
    static constexpr uint32_t RS = CH <= 8 ? 8 : CH <= 16 ? 16 : CH <= 32 ? 32 : 64;
    static constexpr uint32_t RSB = RS * 16;
    static constexpr uint32_t KT = RS <= 16 ? 64 : 32;
    static constexpr uint32_t BYTES = KT * RSB;  // of K or of V
    // Linear in the bits of k: mix(a ^ b) = mix(a) ^ mix(b).
    static constexpr __device__ uint32_t mix(uint32_t k) {
        if (F32) return (k >> 2 & 1u) << 3 | (k >> 3 & 1u) << 2 | (k & 3u);
        return RS == 8 ? (k >> 1 & 1u) << 2 | (k >> 2 & 3u) : (k & 3u) << 2 | (k >> 2 & 3u);
    }
};

template <int D, bool F32, int WAVES>
struct PromptWave {
    using T = TileShape<D, F32>;
    static constexpr int SUB = T::KT / 32, DT = D / 32, QN = F32 ? D / 8 : D / 16;
    using Frag = std::conditional_t<F32, f32x4, bf16x8>;

    Frag q[QN];
    f32x16 o[DT];
    float m, l;        // what exponents are from (in powers of two; kNone: nothing seen yet), sum of this lane's
    float c;           // scale in powers of two
    int64_t pos;       // the last key that this lane's row sees, -1: none
    static constexpr uint32_t KA = T::RS == 8 ? 4 : 8, VA = F32 ? 4 : T::RS == 8 ? 2 : 4;
    uint32_t k_at[KA], v_at[F32 ? 1 : 2][VA];  // this lane's places in a tile

    __device__ __forceinline__ void places(uint32_t lane) {
        const uint32_t col = lane & 31u, g = lane >> 5;
#pragma unroll
        for (uint32_t t = 0; t < KA; t++) k_at[t] = col * T::RSB + (((2 * t + g) ^ T::mix(col)) << 4);
        if constexpr (F32) {
#pragma unroll
            for (uint32_t b = 0; b < 4; b++) v_at[0][b] = (4 * g + b) * T::RSB + (((col / 4) ^ T::mix(4 * g + b)) << 4) + 4 * (col & 3u);
        } else {
            const uint32_t i = lane & 15u, half = (lane >> 4) & 1u;
#pragma unroll
            for (uint32_t e = 0; e < 2; e++)
#pragma unroll
                for (uint32_t p = 0; p < VA; p++) {
                    const uint32_t row = 8 * e + 4 * g + i / 4;
                    v_at[e][p] = row * T::RSB + (((4 * p + 2 * half + (i & 3u) / 2) ^ T::mix(row)) << 4) + 8 * (i & 1u);
                }
        }
    }

    // Of keys k0 + 32 sub + 4 (lane / 32) and on: how many this lane's row sees, up to 32.
    __device__ __forceinline__ int32_t seen_of(uint64_t k0, uint32_t sub, uint32_t lane) const {
        return (int32_t)max(min(pos + 1 - (int64_t)(k0 + 32 * sub + 4 * (lane >> 5)), (int64_t)32), (int64_t)0);
    }

    // scores of 32 keys
    __device__ __forceinline__ f32x16 scores(const uint8_t* kt, uint32_t sub) const {
        f32x16 s = {};
#pragma unroll
        for (uint32_t t = 0; t < QN; t++) {
            const Frag k = *reinterpret_cast<const Frag*>(kt + k_at[t % KA] + (sub * 32 * T::RSB + t / KA * KA * 32));
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < 4; j++) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k[j], q[t][j], s, 0, 0, 0);
            } else {
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[t], s, 0, 0, 0);
            }
        }
        return s;
    }

    // The operand of 32 dims of the values of 16 keys (bf16) in the order of P.
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
    // (f32): one dim of the value of key number i of 32.
    __device__ __forceinline__ float value(const uint8_t* vt, uint32_t sub, uint32_t i, uint32_t dt) const {
        const uint32_t at = v_at[0][i & 3u] ^ ((i >> 2 & 1u) << 6 | (dt & 1u) << 7);  // mix of key 8 (i / 4), and an odd dt
        return *reinterpret_cast<const float*>(vt + at + ((32 * sub + 8 * (i >> 2)) * T::RSB + (dt >> 1) * 256));
    }

    // P V added to the output.  bf16: the exponentials are rounded to 8 bits of mantissa, an error of the
    // size of the output's own rounding.
    template <class VF>
    __device__ __forceinline__ void add(const f32x16 (&p)[SUB], VF&& v) {
        if constexpr (F32) {
#pragma unroll
            for (uint32_t sub = 0; sub < SUB; sub++)
#pragma unroll
                for (uint32_t i = 0; i < 16; i++)
#pragma unroll
                    for (uint32_t dt = 0; dt < DT; dt++)
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v(sub, i, dt), p[sub][i], o[dt], 0, 0, 0);
        } else {
#pragma unroll
            for (uint32_t s = 0; s < 2 * SUB; s++) {
                u32x4 w;
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) w[j] = f32x2_to_bf16x2_bits(p[s / 2][8 * (s & 1u) + 2 * j], p[s / 2][8 * (s & 1u) + 2 * j + 1]);
                const bf16x8 pf = __builtin_bit_cast(bf16x8, w);
#pragma unroll
                for (uint32_t dt = 0; dt < DT; dt++)
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v(s, 0u, dt), pf, o[dt], 0, 0, 0);
            }
        }
    }

    // A tile of keys from k0 on.  masked: some row does not see all of them.
    __device__ __forceinline__ void step(const uint8_t* kt, const uint8_t* vt, uint64_t k0, uint32_t lane, bool masked) {
        f32x16 p[SUB];
        float top = kNone;
#pragma unroll
        for (uint32_t sub = 0; sub < SUB; sub++) p[sub] = scores(kt, sub);
        if (masked) {
            asm volatile("");  // a branch, not a selection in every step
#pragma unroll
            for (uint32_t sub = 0; sub < SUB; sub++) {
                const int32_t sees = seen_of(k0, sub, lane);
#pragma unroll
                for (int32_t i = 0; i < 16; i++)
                    if (8 * (i >> 2) + (i & 3) >= sees) p[sub][i] = kNone;
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
        if constexpr (F32) {
            add(p, [&](uint32_t sub, uint32_t i, uint32_t dt) { return value(vt, sub, i, dt); });
        } else {
            add(p, [&](uint32_t s, uint32_t, uint32_t dt) { return values(vt, s, dt); });
        }
    }
};

template <bool F32>
__device__ __forceinline__ float prompt_element(const KvRows& x, int64_t at) {
    return F32 ? gptr<float>(x.p)[at] : bf16_bits_to_f32(gptr<uint16_t>(x.p)[at]);
}

// One row by a wave, key after key, each that the row sees and no other: for rows
// beside which infinite or NaN values are masked, where 0 times the value is not 0.  Takes
// some forty times as long as the tiles do.
template <int D, bool F32>
__device__ __forceinline__ void prompt_row_by_itself(const PromptArgs& a, uint64_t q_row, uint32_t q_head, uint64_t key0, uint32_t head,
                                                  int64_t from, int64_t to, uint64_t slot) {
    constexpr int N = (D + 63) / 64;
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
                if (lane + 64 * i < D) o[i] = __builtin_fmaf(pj, prompt_element<F32>(a.v, va + (j0 + j) * a.v.ts + lane + 64 * i), o[i]);
        }
    }
    const bool none = from >= to;
    const float ref = none ? kNone : m == kNone ? 0.0f : m;  // scores without a number: the sum is NaN
    if (a.parts > 1) {
        if (lane == 0) gptr_mut<float>(a.stats)[2 * slot] = ref, gptr_mut<float>(a.stats)[2 * slot + 1] = l;
        for (int i = 0; i < N; i++)
            if (lane + 64 * i < D) gptr_mut<float>(a.part_o)[slot * D + lane + 64 * i] = o[i];
        return;
    }
    if (a.lse && lane == 0)
        gptr_mut<float>(a.lse)[q_row * (a.heads * a.group) + q_head] = none ? kNone : (ref + log2f(l)) * 0.69314718055994531f;
    for (int i = 0; i < N; i++) {
        if (lane + 64 * i >= D) continue;
        const float y = none ? 0.0f : o[i] / l;
        const int64_t at = (int64_t)q_row * a.out.ts + (int64_t)q_head * a.out.hs + lane + 64 * i;
        if (F32)
            gptr_mut<float>(a.out.p)[at] = y;
        else
            gptr_mut<uint16_t>(a.out.p)[at] = f32_to_bf16_bits(y);
    }
}

// Workgroup (row tile, sequence, kv head, part of the keys), the last row tiles, which see most
// keys, first.
template <int D, bool F32, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (TileShape<D, F32>::RS <= 16 ? 2 : 1)) void prompt_kernel(PromptArgs a) {
    using T = TileShape<D, F32>;
    using W = PromptWave<D, F32, WAVES>;
    constexpr uint32_t ROWS = 32 * WAVES, STAGE = 2 * T::BYTES;
    constexpr uint32_t COPIES = T::KT * T::RS / 64 / WAVES;  // of a wave for K, and for V
    constexpr uint32_t PER = 64 / T::RS;                     // keys of a copy
    __shared__ __align__(16) uint8_t lds[2 * STAGE];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 5, col = lane & 31u;

    uint32_t id = blockIdx.x;
    const uint32_t part = id % a.parts;
    id /= a.parts;
    const uint32_t head = id % a.heads;
    id /= a.heads;
    const uint32_t seq = id % a.seqs, tile = a.row_tiles - 1 - id / a.seqs;
    const PromptRange r = prompt_range(a, seq);
    const uint64_t rows = (uint64_t)r.n * a.group, tile_row = (uint64_t)tile * ROWS;
    if (tile_row >= rows) return;
    const uint64_t last_row = min(tile_row + ROWS, rows) - 1;
    // keys that some row of the tile sees, those of this part
    const int64_t some = (int64_t)(last_row / a.group) + r.off + 1;
    const uint32_t all = some <= 0 ? 0u : (uint32_t)(((uint64_t)some + T::KT - 1) / T::KT);
    const uint32_t each = (all + a.parts - 1) / a.parts;
    const uint32_t t0 = min(part * each, all), t1 = min(t0 + each, all);

    W w;
    w.places(lane);
    const uint64_t wave_row = tile_row + 32 * wave, row = wave_row + col;
    const uint64_t token = min(row, last_row) / a.group;
    const uint32_t q_head = head * a.group + (uint32_t)(min(row, last_row) - token * a.group);
    w.pos = row <= last_row ? (int64_t)token + r.off : -1;
    // all keys up to `open` are seen by every row of this wave, none from `shut` on by any
    const bool whole = wave_row + 31 <= last_row;
    const int64_t open = whole ? (int64_t)(wave_row / a.group) + r.off + 1 : 0;
    const int64_t shut = wave_row > last_row ? 0 : (int64_t)(min(wave_row + 31, last_row) / a.group) + r.off + 1;

    // this wave's rows; a negative scale turns their signs, a scale of 0 makes them 0
    const float scale = fabsf(a.scale);
    w.c = scale == 0.0f ? 1.0f : scale * 1.4426950408889634f;
    {
        const int64_t at = (int64_t)(r.row0 + token) * a.q.ts + (int64_t)q_head * a.q.hs;
        const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;
#pragma unroll
        for (uint32_t t = 0; t < W::QN; t++) {
            if constexpr (F32) {
                const float* p = static_cast<const float*>(a.q.p) + at + 8 * t + 4 * g;
                f32x4 x;
                if (a.q.vec) {
                    x = *gptr<f32x4>(p);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) x[j] = gptr<float>(p)[j];
                }
                w.q[t] = x * sign;
            } else {
                const uint16_t* p = static_cast<const uint16_t*>(a.q.p) + at + 16 * t + 8 * g;
                u32x4 x;
                if (a.q.vec) {
                    x = *gptr<u32x4>(p);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) x[j] = gptr<uint16_t>(p)[2 * j] | (uint32_t)gptr<uint16_t>(p)[2 * j + 1] << 16;
                }
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = a.scale == 0.0f ? 0u : x[j] ^ (a.scale < 0.0f ? 0x80008000u : 0u);
                w.q[t] = __builtin_bit_cast(bf16x8, x);
            }
        }
    }

    // Copies tile t into a stage: unit blk * 64 + lane of K and of V, blk = wave + WAVES j, its key
    // key0 + STEP j, where key0 < STEP, a power of two.  Whole tiles go
    // straight from memory, addresses a uniform one and 32 bits of the lane's; keys behind the end are the last one.
    constexpr uint32_t STEP = WAVES * PER;
    const uint8_t* const kb = static_cast<const uint8_t*>(a.k.p) + ((int64_t)r.key0 * a.k.ts + (int64_t)head * a.k.hs) * T::E;
    const uint8_t* const vb = static_cast<const uint8_t*>(a.v.p) + ((int64_t)r.key0 * a.v.ts + (int64_t)head * a.v.hs) * T::E;
    const uint32_t key0 = wave * PER + lane / T::RS, chunk0 = (lane % T::RS) ^ T::mix(key0);
    const bool vec = a.k.vec && a.v.vec, near = vec && max(a.k.ts, a.v.ts) * (int64_t)T::E < (1 << 26);
    const uint32_t k_row = key0 * (uint32_t)a.k.ts * T::E, v_row = key0 * (uint32_t)a.v.ts * T::E;  // if near
    uint64_t k_step = (uint32_t)a.k.ts * T::E * STEP, v_step = (uint32_t)a.v.ts * T::E * STEP;
    uint64_t k_base = scalar64((uint64_t)(uintptr_t)kb), v_base = scalar64((uint64_t)(uintptr_t)vb);
    asm volatile("" : "+s"(k_step), "+s"(v_step), "+s"(k_base), "+s"(v_base));  // kept as scalars
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    auto copy = [&](uint32_t t, uint32_t stage) {
        const uint32_t to = lds0 + stage * STAGE + wave * 1024;
        const uint32_t k0 = t * T::KT;
        if (near && (uint64_t)k0 + T::KT <= r.nk) {
            uint64_t ks = k_base + t * (k_step * COPIES), vs = v_base + t * (v_step * COPIES);
#pragma unroll
            for (uint32_t j = 0; j < COPIES; j++, ks += k_step, vs += v_step) {
                const uint32_t chunk = chunk0 ^ T::mix(STEP * j);
                if (T::CH < T::RS && chunk >= T::CH) continue;
                copy16(ks, k_row + 16 * chunk, to + WAVES * j * 1024);
                copy16(vs, v_row + 16 * chunk, to + T::BYTES + WAVES * j * 1024);
            }
            return;
        }
#pragma unroll 1
        for (uint32_t j = 0; j < COPIES; j++) {
            const uint32_t chunk = chunk0 ^ T::mix(STEP * j);
            const int64_t at = (int64_t)min((uint64_t)k0 + key0 + STEP * j, (uint64_t)r.nk - 1);
            const uint8_t* const from[2] = {kb + at * a.k.ts * T::E + 16 * chunk, vb + at * a.v.ts * T::E + 16 * chunk};
            if (T::CH < T::RS && chunk >= T::CH) continue;
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) {
                if (vec) {
                    copy16(from[i], to + i * T::BYTES + WAVES * j * 1024);
                    continue;
                }
                u32x4 x;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (F32)
                        x[e] = gptr<uint32_t>(from[i])[e];
                    else
                        x[e] = gptr<uint16_t>(from[i])[2 * e] | (uint32_t)gptr<uint16_t>(from[i])[2 * e + 1] << 16;
                }
                *reinterpret_cast<u32x4*>(lds + stage * STAGE + i * T::BYTES + (wave + WAVES * j) * 1024 + 16 * lane) = x;
            }
        }
    };

    w.m = kNone;
    w.l = 0.0f;
#pragma unroll
    for (uint32_t dt = 0; dt < W::DT; dt++) w.o[dt] = f32x16{};
    if (t0 < t1) copy(t0, 0);
    for (uint32_t t = t0; t < t1; t++) {
        ring_barrier<0>();  // tile t has landed, and the other stage has been read
        if (t + 1 < t1) copy(t + 1, (t + 1 - t0) & 1u);
        const uint8_t* const kt = lds + ((t - t0) & 1u) * STAGE;
        const uint64_t k0 = (uint64_t)t * T::KT;
        if ((int64_t)k0 >= shut) continue;
        w.step(kt, kt + T::BYTES, k0, lane, (int64_t)(k0 + T::KT) > open);
    }

    const uint64_t slot0 = ((((uint64_t)tile * a.seqs + seq) * a.heads + head) * a.parts + part) * ROWS + 32 * wave;
    // An infinity or a NaN in the output: of what the row sees, or of values that are masked for it
    bool odd = false;
#pragma unroll
    for (uint32_t dt = 0; dt < W::DT; dt++)
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) odd |= !(fabsf(w.o[dt][i]) < __builtin_inff());
    if (__any(odd)) {
        bool masked = false;
        const int64_t key_end = min((int64_t)t1 * T::KT, (int64_t)r.nk), key_begin = (int64_t)t0 * T::KT;
        const int64_t first = max((int64_t)(min(wave_row, last_row) / a.group) + r.off + 1, key_begin);
        for (int64_t j = max(min(first, key_end - 1), (int64_t)0); j < key_end; j++)  // the last one stands for keys behind the end as well
            for (uint32_t d = lane; d < D; d += 64)
                masked |= !(fabsf(prompt_element<F32>(a.v, (int64_t)(r.key0 + j) * a.v.ts + (int64_t)head * a.v.hs + d)) < __builtin_inff());
        if (__any(masked)) {
#pragma unroll 1
            for (uint32_t i = 0; i < 32 && wave_row + i <= last_row; i++) {
                const uint64_t rr = wave_row + i, tok = rr / a.group;
                const int64_t end = min((int64_t)tok + r.off + 1, key_end);
                prompt_row_by_itself<D, F32>(a, r.row0 + tok, head * a.group + (uint32_t)(rr - tok * a.group), r.key0, head, key_begin,
                                             end, slot0 + i);
            }
            return;
        }
    }

    w.l += __shfl_xor(w.l, 32);
    if (row > last_row) return;
    if (a.parts > 1) {
        const uint64_t slot = slot0 + col;
        if (g == 0) {
            gptr_mut<float>(a.stats)[2 * slot] = w.m;
            gptr_mut<float>(a.stats)[2 * slot + 1] = w.l;
        }
#pragma unroll
        for (uint32_t dt = 0; dt < W::DT; dt++)
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                *gptr_mut<f32x4>(a.part_o + slot * D + 32 * dt + 8 * i + 4 * g) =
                    f32x4{w.o[dt][4 * i], w.o[dt][4 * i + 1], w.o[dt][4 * i + 2], w.o[dt][4 * i + 3]};
        return;
    }
    const float inv = w.m == kNone ? 0.0f : 1.0f / w.l;
    if (a.lse && g == 0)
        gptr_mut<float>(a.lse)[(r.row0 + token) * (uint64_t)(a.heads * a.group) + q_head] =
            w.m == kNone ? kNone : (w.m + log2f(w.l)) * 0.69314718055994531f;
    const int64_t to = (int64_t)(r.row0 + token) * a.out.ts + (int64_t)q_head * a.out.hs;
#pragma unroll
    for (uint32_t dt = 0; dt < W::DT; dt++)
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            float y[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) y[j] = w.m == kNone ? 0.0f : w.o[dt][4 * i + j] * inv;
            const int64_t d = to + 32 * dt + 8 * i + 4 * g;
            if constexpr (F32) {
                float* p = static_cast<float*>(a.out.p) + d;
                if (a.out.vec) {
                    *gptr_mut<f32x4>(p) = f32x4{y[0], y[1], y[2], y[3]};
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) gptr_mut<float>(p)[j] = y[j];
                }
            } else {
                uint16_t* p = static_cast<uint16_t*>(a.out.p) + d;
                const u32x2 x = {f32x2_to_bf16x2_bits(y[0], y[1]), f32x2_to_bf16x2_bits(y[2], y[3])};
                if (a.out.vec) {
                    *gptr_mut<u32x2>(p) = x;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) gptr_mut<uint16_t>(p)[j] = (uint16_t)(x[j / 2] >> (16 * (j & 1)));
                }
            }
        }
}

}  // namespace

template <bool F32>
hipError_t prompt_launch_typed(const PromptArgs& a, const PromptPlan& plan, hipStream_t st) {
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (plan.waves == 1)
            prompt_kernel<D, F32, 1><<<(uint32_t)plan.grid, 64, 0, st>>>(a);
        else
            prompt_kernel<D, F32, 4><<<(uint32_t)plan.grid, 256, 0, st>>>(a);
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
