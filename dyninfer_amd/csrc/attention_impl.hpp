// Attention of a few new tokens a sequence (a chain or a tree of drafts) over
// the quantized paged cache: the kernel, instantiated per pair of encodings in
// attention_k<bits>v<bits>.hip.
//
//   S[p, r] = scale q_r . k_p,  out_r = sum_p exp(S - max) v_p / sum_p exp(S - max)
//
// over the positions p that row r sees.  Rows of one kv head are the new tokens
// times the query heads that share it, r = token * group + head: up to 256 of
// them share one pass over the cache.
//
// One pass, online: a step takes 32 positions; the running maximum and sum of
// every row and the unnormalised output stay in registers.  In tiles of up to 32 rows every
// wave of a workgroup holds all of them and takes its own positions, and the
// four join in LDS at the end; beyond, every wave holds its own rows, all take
// the same positions and share their decoding.  Where positions are split over
// workgroups, the parts are joined through the workspace by a second small launch.
// Few rows over a long context are bound by the cache's bytes; from about 64 rows
// the vector instructions around the products are.
//
// The products are 16x16x32 MFMAs with the cache as the first operand, so that
// a row of the output (a column of the second operand) belongs to lanes l with
// l % 16 = r: its statistics are in the lane, and the exponentials that come
// out of S are, unmoved, the second operand of the product with V:
//   S (16 positions x 16 rows): lane l holds positions 4(l / 16) + i, i < 4
//   P (32 positions x 16 rows): lane l holds positions 8(l / 16) + j, j < 8
// The sum over positions may take them in any order if both operands agree, so
// lane group g's eight positions of a step, 4s + i of them being row 4g + i of
// the s-th S, are eight in a row: for one dim of V eight codes in a row.
//
// Numerics: K codes are exact in f16 (0x6400 | byte is 1024 + byte; the offset
// is taken off exactly), queries are scaled to a power of two that puts the
// row's largest in [2^14, 2^15) and are exact in f16 down to 2^-29 of it (f32
// queries: a second f16 holds what the first leaves), each block's sum is
// multiplied by its f32 scale.  V codes are exact in bf16; p times the value's
// scale, of unknown range, is split into bf16 terms: two (16 bits) for bf16
// outputs, three (24 bits) for f32 ones.  A third term for bf16 took 295 us instead of 261 for
// 64 tokens over 131071 positions and 4.26 ms instead of 3.72 for a prompt of 16384; of the first's outputs
// 0.25% are not the 64-bit value rounded to bf16 with two terms and 0.07% with three, 0.28% where
// the same is computed in f32 throughout.
#pragma once
#include <type_traits>

#include "kvcache.hpp"

namespace dmx {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kTile = 32;   // positions of a wave's step
constexpr uint32_t kWaves = 4;   // waves of a workgroup, each on its own tiles

// Four codes of a dword of bytes 128 + code (or 16 (8 + code)) as exact f16.
__device__ __forceinline__ void k_bytes_f16(uint32_t w, f16x2& a, f16x2& b) {
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
    b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
}

// Eight codes (two dwords of bytes) as an MFMA operand.
__device__ __forceinline__ f16x8 k_frag(uint32_t w0, uint32_t w1) {
    f16x2 a, b, c, d;
    k_bytes_f16(w0, a, b);
    k_bytes_f16(w1, c, d);
    return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Four signed bytes as bf16 pairs (exact: the high halves of their f32).
__device__ __forceinline__ u32x2 v_bytes_bf16(uint32_t w) {
    const uint32_t a = __float_as_uint((float)(int8_t)w), b = __float_as_uint((float)(int8_t)(w >> 8));
    const uint32_t c = __float_as_uint((float)(int8_t)(w >> 16)), d = __float_as_uint((float)((int32_t)w >> 24));
    return u32x2{__builtin_amdgcn_perm(b, a, 0x07060302u), __builtin_amdgcn_perm(d, c, 0x07060302u)};
}

__device__ __forceinline__ bf16x8 v_frag(uint32_t w0, uint32_t w1) {
    const u32x2 a = v_bytes_bf16(w0), b = v_bytes_bf16(w1);
    return __builtin_bit_cast(bf16x8, u32x4{a.x, a.y, b.x, b.y});
}

// Largest / sum over the four lanes that share a row (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float rows_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float rows_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// A row's sum at the end.  Exponents are exact differences from m, which is the largest score
// rounded to 24 bits; beyond 2^31 that alone may lie outside the exponential's range, the sum be 0 or
// infinite: NaN, so that the row is not taken for one that sees nothing.
__device__ __forceinline__ float row_sum(float l, float m) {
    l = rows_sum(l);
    return m == -__builtin_inff() || (l > 0.0f && l < __builtin_inff()) ? l : __builtin_nanf("");
}

// How a tile of the cache (two chunks of 16 positions) lies in a wave's LDS, in
// 16-byte units, each copied by one lane straight from memory.  The order is the
// one in which lanes read it back, so that a wave's reads are consecutive.
//   K, 8 bits: per S and pair of blocks, unit [part][row]: 16 bytes of one lane;
//      a last odd block: per S, units [row][2], 8 bytes of one lane
//   K, 4 bits: per S and pair, units [row][2], 8 bytes of one lane; a last odd
//      block: per S, unit [row], 4 bytes of one lane
//   V, 8 bits: per 16 dims, unit [chunk][dim]; 4 bits: [chunk][dim / 2]
//   scales as they lie in the cache, chunk after chunk, K's then V's
template <int D, int KB, int VB>
struct TileLds {
    static constexpr uint32_t NB = D / 32, PAIRS = D / 64, ODD = NB % 2;
    static constexpr uint32_t KMAIN = 2 * PAIRS * (KB == 8 ? 64 : 32);  // units of all pairs
    static constexpr uint32_t KODD = ODD ? 2 * (KB == 8 ? 32 : 16) : 0;
    static constexpr uint32_t V = 2 * D * VB / 8;                       // of the V codes
    static constexpr uint32_t KS = 4 * NB, VS = 4;                      // of the scales
    static constexpr uint32_t DMA = KMAIN / 64 + (ODD ? 1 : 0) + (V + 63) / 64 + 1;  // copies of a tile
    static constexpr uint32_t V0 = (KMAIN + KODD) * 16, KS0 = V0 + V * 16, VS0 = KS0 + KS * 16;
    static constexpr uint32_t BYTES = VS0 + VS * 16;
    static_assert(KMAIN % 64 == 0 && V % 32 == 0 && KS + VS <= 64, "whole copies");
    // Tiles a wave holds: one is worked on while the others are on their way.  Two
    // of 8-bit codes and 128 dims make some 70 KB a workgroup, two of them a CU.
    static constexpr uint32_t STAGES = BYTES > 6656 ? 2 : BYTES > 4608 ? 3 : 4;
};

// 16 bytes a lane from src + OFF to dst + 16 lane.  OFF is the instruction's own
// offset, which it adds to both addresses: one register pair serves all the
// copies of a tile.  dst lies at least OFF behind the start of the wave's LDS.
template <uint32_t OFF>
__device__ __forceinline__ void dma16_at(const uint8_t* src, uint8_t* dst) {
    static_assert(OFF < 4096, "the offset's 13 signed bits");
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)(dst - OFF), 16, (int)OFF, 0);
}

// f(0), f(1), .. f(N - 1) with the numbers as types.
template <uint32_t N, class F, uint32_t I = 0>
__device__ __forceinline__ void each(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<uint32_t, I>());
        each<N, F, I + 1>(static_cast<F&&>(f));
    }
}

// Copies a tile: slot[c] is the first slot of its chunk c.  Row m of S number s is
// position 8 (m / 4) + 4 s + m % 4 of the tile.
template <int D, int KB, int VB>
__device__ __forceinline__ void copy_tile(const KvView& kv, uint64_t slot0, uint64_t slot1, uint32_t lane, uint8_t* lds) {
    using T = TileLds<D, KB, VB>;
    constexpr uint32_t RB = D * KB / 8;
    auto row = [&](uint32_t m) { return kv.k + ((m & 8u ? slot1 : slot0) + 2 * (m & 4u) + (m & 3u)) * RB; };
    if constexpr (KB == 8) {
        const uint8_t* p = row(lane & 15u) + 16 * (lane >> 4);
        each<2 * T::PAIRS>([&](auto i) {
            constexpr uint32_t s = decltype(i)::value / T::PAIRS, j = decltype(i)::value % T::PAIRS;
            dma16_at<4 * s * RB + 64 * j>(p, lds + (s * T::PAIRS + j) * 1024);
        });
        if constexpr (T::ODD)  // lanes 0..31 the first S, 32..63 the second
            dma16_at<0>(row(lane >> 1 & 15u) + 4 * (lane >> 5) * RB + 64 * T::PAIRS + 16 * (lane & 1u), lds + T::KMAIN * 16);
    } else {
        const uint8_t* p = row(lane >> 1 & 15u) + 16 * (lane & 1u);
        if constexpr (T::PAIRS == 1) {  // both S in one copy
            dma16_at<0>(p + 4 * (lane >> 5) * RB, lds);
        } else {  // two pairs in one copy
            each<T::PAIRS>([&](auto i) {
                constexpr uint32_t s = decltype(i)::value / (T::PAIRS / 2), j = decltype(i)::value % (T::PAIRS / 2);
                dma16_at<4 * s * RB + 64 * j>(p + 32 * (lane >> 5), lds + (s * T::PAIRS / 2 + j) * 1024);
            });
        }
        if constexpr (T::ODD)
            if (lane < 32) dma16_at<0>(row(lane & 15u) + 4 * (lane >> 4) * RB + 32 * T::PAIRS, lds + T::KMAIN * 16);
    }
    if constexpr (VB == 8) {
        const uint8_t* p = kv.v + (lane & 16u ? slot1 : slot0) * D + 256 * (lane >> 5) + 16 * (lane & 15u);
        each<D / 32>([&](auto d) { dma16_at<512 * decltype(d)::value>(p, lds + T::V0 + 1024 * decltype(d)::value); });
    } else {
        const uint8_t* p = kv.v + (lane & 8u ? slot1 : slot0) * (D / 2) + 128 * (lane >> 4) + 16 * (lane & 7u);
        each<D / 64>([&](auto d) { dma16_at<512 * decltype(d)::value>(p, lds + T::V0 + 1024 * decltype(d)::value); });
        if constexpr (D % 64) {
            if (lane < 32) dma16_at<512 * (D / 64)>(p, lds + T::V0 + 1024 * (D / 64));
        }
    }
    if (lane < T::KS + T::VS) {
        constexpr uint32_t U = 2 * T::NB;  // units of a chunk's K scales
        const bool v = lane >= T::KS;
        const uint32_t i = v ? lane - T::KS : lane % U;
        const uint64_t slot = (v ? i >= 2 : lane >= U) ? slot1 : slot0;
        const uint8_t* p = v ? kv.v + kv.v_scales + slot * 2 + 16 * (i & 1u) : kv.k + kv.k_scales + slot * (2 * T::NB) + 16 * i;
        dma16_at<0>(p, lds + T::KS0);
    }
}

// Words of this lane's row of S number s, from LDS.
template <int D, int KB, int VB>
__device__ __forceinline__ void read_k(const uint8_t* lds, uint32_t s, uint32_t col, uint32_t g,
                                       uint32_t (&w)[D / 16 * KB / 8]) {
    using T = TileLds<D, KB, VB>;
#pragma unroll
    for (uint32_t j = 0; j < T::PAIRS; j++) {
        if constexpr (KB == 8) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(lds + (s * T::PAIRS + j) * 1024 + (16 * g + col) * 16);
#pragma unroll
            for (int i = 0; i < 4; i++) w[4 * j + i] = x[i];
        } else {
            const u32x2 x = *reinterpret_cast<const u32x2*>(lds + (s * T::PAIRS + j) * 512 + col * 32 + g * 8);
            w[2 * j] = x.x;
            w[2 * j + 1] = x.y;
        }
    }
    if constexpr (T::ODD) {
        if constexpr (KB == 8) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(lds + T::KMAIN * 16 + s * 512 + col * 32 + g * 8);
            w[4 * T::PAIRS] = x.x;
            w[4 * T::PAIRS + 1] = x.y;
        } else {
            w[2 * T::PAIRS] = *reinterpret_cast<const uint32_t*>(lds + T::KMAIN * 16 + s * 256 + col * 16 + g * 4);
        }
    }
}

// Block b's operand from those words.
template <int D, int KB>
__device__ __forceinline__ f16x8 k_block(const uint32_t (&w)[D / 16 * KB / 8], int b) {
    if constexpr (KB == 8) {
        return k_frag(w[2 * b], w[2 * b + 1]);
    } else {  // nibbles as the high half of a byte: 16 (8 + code)
        return k_frag((w[b] << 4) & 0xF0F0F0F0u, w[b] & 0xF0F0F0F0u);
    }
}

// Which of positions 8g..8g+7 of a tile (the lane group's) row i of the
// sequence sees, one bit each.  j0: the first of them, from the first new token.
__device__ __forceinline__ uint32_t sees(const int64_t* mask, uint32_t words, uint64_t row, uint32_t i, uint32_t n,
                                         int64_t j0) {
    if (j0 <= -8) return 0xFFu;
    if (j0 >= (int64_t)n) return 0u;
    if (!mask) {  // rows j <= i
        const int64_t c = (int64_t)i + 1 - j0;
        return c <= 0 ? 0u : c >= 8 ? 0xFFu : (1u << c) - 1u;
    }
    const uint32_t lead = j0 < 0 ? (uint32_t)-j0 : 0u;  // committed positions among the eight
    const uint32_t j = (uint32_t)(j0 + lead);
    const int64_t* m = mask + row * words;
    const uint32_t w = j >> 6, sh = j & 63u;
    uint64_t v = (uint64_t)m[w] >> sh;
    if (sh && w + 1 < words) v |= (uint64_t)m[w + 1] << (64 - sh);
    const uint32_t left = n - j;
    if (left < 8) v &= (1ull << left) - 1ull;
    return ((uint32_t)(v << lead) | ((1u << lead) - 1u)) & 0xFFu;
}

// ring_wait<k N>() for a wave-uniform k in 0..K: the copies of all but the last
// k tiles of N copies each have landed.
template <uint32_t N, uint32_t K>
__device__ __forceinline__ void tiles_wait(uint32_t k) {
    if constexpr (K == 0) {
        ring_wait<0>();
    } else {
        if (k >= K)
            ring_wait<K * N>();
        else
            tiles_wait<N, K - 1>(k);
    }
}

// Half of a dword of bf16 pairs as f32.
__device__ __forceinline__ float bf16_of(uint32_t w, int i) { return __uint_as_float(i ? w & 0xFFFF0000u : w << 16); }

constexpr uint32_t kStep = kTile * kWaves;  // positions a workgroup takes at a time

// What beginning and ending a unit costs, in steps: 32 ragged sequences of up to
// 4096 positions, a new one among them (units of one step), took 95.7 us with 0,
// 67.4 with 2, 70.4 with 4.
constexpr uint32_t kUnitCost = 2;

// The work of a call as a line: sequence after sequence, of each its units (head
// after head, row tile after row tile), of each kUnitCost places and then its
// steps along the positions.  A share is one of a.shares equal pieces of that line.
struct Share {
    uint64_t unit0;       // units before this sequence's
    uint32_t share;       // which piece
    uint32_t seq;
    uint32_t unit;        // in the sequence
    uint32_t row_tiles, units, unit_steps;  // of the sequence
    uint32_t place;       // first place in the unit
    uint32_t places;      // left in the share

    __device__ __forceinline__ void load(const AttnArgs& a, uint32_t rows_of_tile) {
        const SeqRange r = seq_range(a.b, seq);
        row_tiles = (r.n * a.group + rows_of_tile - 1) / rows_of_tile;
        units = row_tiles * a.kv.heads;
        unit_steps = r.n ? (uint32_t)(((uint64_t)r.len + r.n + kStep - 1) / kStep) : 0;
    }

    // The share's steps of this unit: first one, and the one after the last.
    __device__ __forceinline__ uint32_t first_step() const { return place > kUnitCost ? place - kUnitCost : 0; }
    __device__ __forceinline__ uint32_t end_step() const {
        const uint32_t e = min(place + places, unit_steps + kUnitCost);
        return e > kUnitCost ? e - kUnitCost : 0;
    }

    // On to the next unit.
    __device__ __forceinline__ void next(const AttnArgs& a, uint32_t rows_of_tile) {
        places -= min(places, unit_steps + kUnitCost - place);
        place = 0;
        if (places == 0 || ++unit < units) return;
        do {
            unit0 += units;
            unit = 0;
            if (++seq >= a.b.seqs) {
                places = 0;
                return;
            }
            load(a, rows_of_tile);
        } while (units == 0);
    }
};

// Workgroups go round the eight XCDs; this numbering gives each XCD a run of
// consecutive numbers, so that row tiles that read the same part of the cache
// at the same time find it in one L2.
__device__ __forceinline__ uint32_t by_xcd(uint32_t id, uint32_t n) {
    const uint32_t each = n / 8, more = n % 8, x = id % 8;
    return x * each + min(x, more) + id / 8;
}

// Shares in use: no share is empty.
__device__ __forceinline__ uint32_t shares_of(const AttnArgs& a, uint64_t all) {
    return (uint32_t)min((uint64_t)a.shares, all);
}

// Positions that some of the rows first..end-1 of a unit's may see are below this: in a
// chain those up to the last of their tokens, otherwise all.
__device__ __forceinline__ uint64_t seen_by_some(const AttnArgs& a, const SeqRange& r, uint32_t end) {
    return (uint64_t)r.len + (a.mask ? r.n : (end - 1) / a.group + 1);
}

// Tiles of TILE positions below this are seen whole by all rows from first on.
template <uint32_t TILE>
__device__ __forceinline__ uint32_t open_tiles(const AttnArgs& a, const SeqRange& r, uint32_t first) {
    return (uint32_t)(((uint64_t)r.len + (a.mask ? 0u : first / a.group + 1)) / TILE);
}

// Notes which parts a unit has, for the second launch: the share that has its first step
// writes the first, the one that has its last step the last.
__device__ __forceinline__ void note_parts(const AttnArgs& a, const Share& sh, uint32_t head, uint32_t now0, uint32_t now1) {
    if (a.shares == 0 || threadIdx.x != 0) return;
    uint32_t* const to = a.where + 2 * ((sh.seq * a.kv.heads + head) * a.row_tiles + (sh.unit - head * sh.row_tiles));
    const uint32_t part = sh.share + (uint32_t)sh.unit0 + sh.unit;
    if (now0 == 0) to[0] = part;
    if (now1 == sh.unit_steps) to[1] = part;
}

// Without shares: workgroup (sequence, head, row tile), all of its steps; the last
// row tile first, which has the most positions where rows form a chain.
__device__ __forceinline__ Share whole_unit(const AttnArgs& a, uint32_t rows_of_tile) {
    Share s = {};
    uint32_t id = by_xcd(blockIdx.x, gridDim.x);
    const uint32_t rt = a.row_tiles - 1 - id % a.row_tiles;
    id /= a.row_tiles;
    s.seq = id / a.kv.heads;
    s.load(a, rows_of_tile);
    s.unit = id % a.kv.heads * s.row_tiles + rt;
    s.places = rt < s.row_tiles ? s.unit_steps + kUnitCost : 0;
    return s;
}

// Places and units of sequence s.
__device__ __forceinline__ void seq_work(const AttnArgs& a, uint32_t rows_of_tile, uint32_t s, uint64_t& places, uint64_t& units) {
    places = units = 0;
    if (s >= a.b.seqs) return;
    Share x = {};
    x.seq = s;
    x.load(a, rows_of_tile);
    units = x.units;
    places = x.units * (uint64_t)(x.unit_steps + kUnitCost);
}

// A number that is the same in every lane, as a scalar.
__device__ __forceinline__ uint32_t scalar(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t scalar64(uint64_t x) {
    return (uint64_t)scalar((uint32_t)(x >> 32)) << 32 | scalar((uint32_t)x);
}

// x / y, mostly of numbers below 2^32 (a division of 64 bits takes some hundred
// instructions).
__device__ __forceinline__ uint64_t divide(uint64_t x, uint64_t y) {
    return (x | y) >> 32 ? x / y : (uint64_t)((uint32_t)x / (uint32_t)y);
}

// This workgroup's share.  Every wave finds it by itself, 64 sequences at a time, so
// that no barrier stands before its first copies.
__device__ __forceinline__ Share share_of(const AttnArgs& a, uint32_t rows_of_tile) {
    const uint32_t lane = threadIdx.x & 63u;
    uint64_t places = 0, units = 0, at = 0, to = 0, all = 0;
    uint32_t share = 0;
    if (a.b.seqs > 64) {  // how many places there are
        for (uint32_t s = lane; s < a.b.seqs; s += 64) {
            seq_work(a, rows_of_tile, s, places, units);
            all += places;
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) all += __shfl_xor((unsigned long long)all, d);
        all = scalar64(all);
    }
    Share f = {};
    uint64_t before = 0, units_before = 0;
    for (uint32_t s0 = 0; s0 < a.b.seqs; s0 += 64) {
        seq_work(a, rows_of_tile, s0 + lane, places, units);
        uint64_t x = places, y = units;  // sums over the lanes up to this one
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t u = __shfl_up((unsigned long long)x, d), v = __shfl_up((unsigned long long)y, d);
            if (lane >= (uint32_t)d) x += u, y += v;
        }
        if (a.b.seqs <= 64) all = scalar64(__shfl((unsigned long long)x, 63));
        if (s0 == 0) {
            const uint32_t n = shares_of(a, all);
            share = n < a.shares ? blockIdx.x : by_xcd(blockIdx.x, n);
            if (share < n) {
                at = divide(share * all, n);
                to = divide((share + 1ull) * all, n);
            }
        }
        const uint64_t first = before + x - places, unit0 = units_before + y - units;
        const unsigned long long who = __ballot(at < to && first <= at && at < first + places);
        if (who) {  // the sequence of the share's first place
            const int w = __builtin_ctzll(who);
            const uint64_t in = scalar64(at - __shfl((unsigned long long)first, w));
            f.share = share;
            f.seq = s0 + (uint32_t)w;
            f.load(a, rows_of_tile);
            f.unit0 = __shfl((unsigned long long)unit0, w);
            f.unit = (uint32_t)divide(in, f.unit_steps + kUnitCost);
            f.place = (uint32_t)(in - (uint64_t)f.unit * (f.unit_steps + kUnitCost));
            f.places = (uint32_t)(to - at);
            break;
        }
        before += __shfl((unsigned long long)x, 63);
        units_before += __shfl((unsigned long long)y, 63);
    }
    f.seq = scalar(f.seq);
    f.unit = scalar(f.unit);
    f.row_tiles = scalar(f.row_tiles);
    f.units = scalar(f.units);
    f.unit_steps = scalar(f.unit_steps);
    f.place = scalar(f.place);
    f.places = scalar(f.places);
    f.unit0 = scalar64(f.unit0);
    return f;
}

// x, opaque: what is computed from it stays in its branch.  (The tests of the mask's bits
// were done in every step, a tenth of its vector instructions.)
__device__ __forceinline__ uint32_t here(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A wave's rows: NQ tiles of 16, their queries as operands, running statistics
// and unnormalised outputs.  The two kernels differ in how the cache's codes come
// to hold as operands; a step takes 32 positions, of which lane group g holds
// eight in a row.
template <int D, int KB, int VB, int NQ, bool F32>
struct WaveRows {
    static constexpr int NB = D / 32;          // blocks of a key
    static constexpr int DT = D / 16;          // 16-dim tiles of the output
    static constexpr int TERMS = F32 ? 3 : 2;  // bf16 terms of a probability
    // second terms of f32 queries: in registers, with two tiles in LDS, a lane's NQ NB apart
    static constexpr bool LOWS = F32 && NQ == 2;
    f16x8 qf[NQ][NB], ql[F32 && !LOWS ? NQ : 1][F32 && !LOWS ? NB : 1];
    f16x8* lows;
    float factor[NQ], m[NQ], l[NQ];  // m: what exponents are taken from, about the largest so far (log2)
    uint32_t tok[NQ];
    f32x4 o[NQ][DT];

    // The queries as they lie in memory, loaded before the first tile is asked for:
    // loads come back in order.
    struct Raw {
        u32x4 w[NQ][NB][F32 ? 2 : 1];
    };

    // Rows first_row + 16 t + lane % 16 of the unit's.
    __device__ __forceinline__ void load(const AttnArgs& a, const SeqRange& r, uint32_t head, uint32_t first_row,
                                         uint32_t rows, uint32_t lane, Raw& raw) {
        const uint32_t g = lane >> 4, col = lane & 15u;
#pragma unroll
        for (int t = 0; t < NQ; t++) {
            const uint32_t row = first_row + 16u * t + col;
            const bool live = row < rows;
            tok[t] = live ? row / a.group : 0u;
            const uint32_t h = head * a.group + (live ? row - tok[t] * a.group : 0u);
            const int64_t at = (int64_t)(r.row0 + tok[t]) * a.q.ts + (int64_t)h * a.q.hs + 8 * g;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if constexpr (F32) {
                    const float* p = static_cast<const float*>(a.q.p) + at + 32 * b;
                    if (a.q.vec) {
                        raw.w[t][b][0] = *gptr<u32x4>(p);
                        raw.w[t][b][1] = *gptr<u32x4>(p + 4);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) raw.w[t][b][i / 4][i % 4] = gptr<uint32_t>(p)[i];
                    }
                } else {
                    const uint16_t* p = static_cast<const uint16_t*>(a.q.p) + at + 32 * b;
                    if (a.q.vec) {
                        raw.w[t][b][0] = *gptr<u32x4>(p);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            raw.w[t][b][0][i] = gptr<uint16_t>(p)[2 * i] | (uint32_t)gptr<uint16_t>(p)[2 * i + 1] << 16;
                    }
                }
            }
        }
    }

    // The operands and the rows' factors; statistics and outputs begin.
    __device__ __forceinline__ void begin(const AttnArgs& a, const Raw& raw, uint32_t first_row, uint32_t rows, uint32_t lane) {
        const float sign = a.scale < 0.0f ? -1.0f : 1.0f;  // so that the largest score is that of the largest sum
#pragma unroll
        for (int t = 0; t < NQ; t++) {
            const bool live = first_row + 16u * t + (lane & 15u) < rows;
            float x[NB][8], big = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if constexpr (F32) x[b][i] = __uint_as_float(raw.w[t][b][i / 4][i % 4]);
                    else x[b][i] = bf16_of(raw.w[t][b][0][i / 2], i & 1);
                    big = fmaxf(big, fabsf(x[b][i]));
                }
            big = rows_max(big);
            // exponent e of the row's largest: 2^(14 - e) scales it into [2^14, 2^15)
            int e = (int)((__float_as_uint(big) >> 23) & 255u) - 127;
            e = max(e, -100);
            const float up = sign * __uint_as_float((uint32_t)(14 - e + 127) << 23);
            factor[t] = sign * a.scale * 1.44269504088896341f * (KB == 4 ? 0.0625f : 1.0f);
            factor[t] *= __uint_as_float((uint32_t)(e - 14 + 127) << 23);
            factor[t] = fmaxf(factor[t], 1.2e-38f);  // a masked score is -inf also at scale 0
#pragma unroll
            for (int b = 0; b < NB; b++) {
                f16x8 low;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float s = live ? x[b][i] * up : 0.0f;
                    qf[t][b][i] = (_Float16)s;
                    if constexpr (F32) low[i] = (_Float16)(s - (float)qf[t][b][i]);
                }
                if constexpr (LOWS) lows[(t * NB + b) * 64] = low;
                else if constexpr (F32) ql[t][b] = low;
            }
            m[t] = -__builtin_inff();
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[t][d] = f32x4{0, 0, 0, 0};
        }
    }

    // 32 positions.  In src, of the lane group's eight positions: key(s, f): f[b] =
    // operand of block b of S number s (positions 4s..4s+3 of the eight);
    // key_scales(s, w): w[position][block] of those four; value_scales(w): of the
    // eight; raw(d): what value(x) makes the operand of dims 16d..16d+15 of.
    // masked: vis[t] has a bit for each of the eight that row t sees; otherwise all
    // are seen.  LDS reads are issued well before their use: two waves a SIMD do not
    // hide them.
    template <class Src>
    __device__ __forceinline__ void step(const Src& src, bool masked, const uint32_t (&vis)[NQ]) {
        constexpr int AHEAD = 2;  // operands of V read before they are needed
        f32x4 sc[NQ][2];
        f16x8 kf[NB];
        float kw[4 * NB], vs[8];
        typename Src::Raw vr[DT];
        src.key(0, kf);
        src.key_scales(0, kw);
#pragma unroll
        for (int s = 0; s < 2; s++) {
            // all products first: a sum is read well after it was begun
            f32x4 x[NB][NQ];
#pragma unroll
            for (int b = 0; b < NB; b++) {
#pragma unroll
                for (int t = 0; t < NQ; t++) {
                    x[b][t] = f32x4{0, 0, 0, 0};
                    if constexpr (F32)
                        x[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[b], LOWS ? lows[(t * NB + b) * 64] : ql[LOWS ? 0 : t][LOWS ? 0 : b],
                                                                         x[b][t], 0, 0, 0);
                    x[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[b], qf[t][b], x[b][t], 0, 0, 0);
                }
            }
            float w[4 * NB];
#pragma unroll
            for (int i = 0; i < 4 * NB; i++) w[i] = kw[i];
            if (s == 0) {
                src.key(1, kf);
                src.key_scales(1, kw);
            } else {
                src.value_scales(vs);
#pragma unroll
                for (int d = 0; d < AHEAD; d++) vr[d] = src.raw(d);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int t = 0; t < NQ; t++)
                        sc[t][s][i] = b == 0 ? x[b][t][i] * w[i * NB + b] : sc[t][s][i] + x[b][t][i] * w[i * NB + b];
        }
        if (masked) {
#pragma unroll
            for (int t = 0; t < NQ; t++) {
                const uint32_t see = here(vis[t]);
#pragma unroll
                for (int i = 0; i < 8; i++) sc[t][i / 4][i % 4] = see >> i & 1u ? sc[t][i / 4][i % 4] : -__builtin_inff();
            }
        }

        // Exponentials, from a reference that follows the row's largest score only when
        // one is 2^8 above it: the sums are f32 either way, and most steps then need
        // neither the maximum over lanes nor a rescaling.
        bf16x8 pf[NQ][TERMS];
#pragma unroll
        for (int t = 0; t < NQ; t++) {
            float top = sc[t][0][0];
#pragma unroll
            for (int i = 1; i < 8; i++) top = fmaxf(top, sc[t][i / 4][i % 4]);
            top *= factor[t];
            if (__any(top > m[t] + 8.0f)) {
                top = fmaxf(m[t], rows_max(top));
                const float back = m[t] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m[t] - top);
                l[t] *= back;
#pragma unroll
                for (int d = 0; d < DT; d++) o[t][d] *= back;
                m[t] = top;
            }
            const float ref = m[t] == -__builtin_inff() ? 0.0f : m[t];
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i / 4][i % 4], factor[t], -ref));
                l[t] += e;
                p[i] = e * vs[i];
            }
            if (masked) {  // a masked value's scale may be anything
                const uint32_t see = here(vis[t]);
#pragma unroll
                for (int i = 0; i < 8; i++) p[i] = see >> i & 1u ? p[i] : 0.0f;
            }
#pragma unroll
            for (int n = 0; n < TERMS; n++) {
                u32x4 w;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    w[j] = f32x2_to_bf16x2_bits(p[2 * j], p[2 * j + 1]);
                    if (n + 1 < TERMS) {
                        p[2 * j] -= bf16_of(w[j], 0);
                        p[2 * j + 1] -= bf16_of(w[j], 1);
                    }
                }
                pf[t][n] = __builtin_bit_cast(bf16x8, w);
            }
        }

        // the product with V
#pragma unroll
        for (int d = 0; d < DT; d++) {
            if (d + AHEAD < DT) vr[d + AHEAD] = src.raw(d + AHEAD);
            const bf16x8 vf = src.value(vr[d]);
#pragma unroll
            for (int n = TERMS - 1; n >= 0; n--)
#pragma unroll
                for (int t = 0; t < NQ; t++)
                    o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[t][n], o[t][d], 0, 0, 0);
        }
    }

    // Writes the rows: the outputs where the unit is one workgroup's alone, the
    // parts for the second launch otherwise.  m: log2 of what l is to be multiplied
    // with; o still times 16 where V has 4 bits.
    __device__ __forceinline__ void store(const AttnArgs& a, const Share& sh, const SeqRange& r, uint32_t head, uint32_t tile_row,
                                          uint32_t first_row, uint32_t rows, uint32_t rows_of_tile, bool alone, uint32_t lane) {
        const uint32_t g = lane >> 4, col = lane & 15u;
#pragma unroll
        for (int t = 0; t < NQ; t++) {
            const uint32_t row = first_row + 16u * t + col;
            if (row >= rows) continue;
            const uint32_t h = head * a.group + row % a.group;
            const uint64_t token = r.row0 + row / a.group, q_heads = (uint64_t)a.kv.heads * a.group;
            if (!alone) {
                // parts of a unit are handed to the second launch; (share, unit) pairs climb a
                // staircase, so share + unit numbers them without gaps
                const uint64_t at = (sh.share + sh.unit0 + sh.unit) * rows_of_tile + (row - tile_row);
                float* po = a.parts + at * D;
#pragma unroll
                for (int d = 0; d < DT; d++) *gptr_mut<f32x4>(po + 16 * d + 4 * g) = o[t][d] * (VB == 4 ? 0.0625f : 1.0f);
                if (g == 0) {
                    gptr_mut<float>(a.stats)[2 * at] = m[t];
                    gptr_mut<float>(a.stats)[2 * at + 1] = l[t];
                }
            } else {
                float inv = l[t] > 0.0f ? 1.0f / l[t] : (l[t] == 0.0f ? 0.0f : __builtin_nanf(""));
                if (VB == 4) inv *= 0.0625f;
                const int64_t at = (int64_t)token * a.out.ts + (int64_t)h * a.out.hs;
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const f32x4 x = o[t][d] * inv;
                    const int64_t e = at + 16 * d + 4 * g;
                    if constexpr (F32) {
                        if (a.out.vec) {
                            *gptr_mut<f32x4>(static_cast<float*>(a.out.p) + e) = x;
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; i++) gptr_mut<float>(a.out.p)[e + i] = x[i];
                        }
                    } else {
                        const u32x2 w = {f32x2_to_bf16x2_bits(x[0], x[1]), f32x2_to_bf16x2_bits(x[2], x[3])};
                        if (a.out.vec) {
                            *gptr_mut<u32x2>(static_cast<uint16_t*>(a.out.p) + e) = w;
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                gptr_mut<uint16_t>(a.out.p)[e + i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
                        }
                    }
                }
                if (a.lse && g == 0) gptr_mut<float>(a.lse)[token * q_heads + h] = (m[t] + log2f(l[t])) * 0.69314718055994531f;
            }
        }
    }
};

// Page ids, all lanes alike (scalar loads).
struct Pages {
    uint64_t table;
    uint32_t count, shift;
    __device__ __forceinline__ Pages(const AttnArgs& a, uint32_t seq)
        : table((uint64_t)(a.b.table + (size_t)seq * a.b.table_pages)), count(a.b.table_pages), shift(a.kv.page_shift - 4u) {}
    __device__ __forceinline__ int32_t operator()(uint32_t chunk) const {
        const uint32_t i = chunk >> shift;
        return i < count ? *(const __attribute__((address_space(4))) int32_t*)(table + 4ull * i) : -1;
    }
};

// bf16 scales as f32.
template <int N>
__device__ __forceinline__ void read_bf16(const uint8_t* p, float (&w)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p + 2 * i);
        w[i] = bf16_of(x.x, 0), w[i + 1] = bf16_of(x.x, 1), w[i + 2] = bf16_of(x.y, 0), w[i + 3] = bf16_of(x.y, 1);
    }
}

// A tile in LDS as it was copied: codes, decoded as they are read.
template <int D, int KB, int VB>
struct CodeTile {
    using T = TileLds<D, KB, VB>;
    using Raw = u32x2;
    static constexpr int NB = D / 32;
    const uint8_t* tile;
    uint32_t g, col;
    __device__ __forceinline__ void key(int s, f16x8 (&f)[NB]) const {
        uint32_t w[D / 16 * KB / 8];
        read_k<D, KB, VB>(tile, s, col, g, w);
#pragma unroll
        for (int b = 0; b < NB; b++) f[b] = k_block<D, KB>(w, b);
    }
    __device__ __forceinline__ void key_scales(int s, float (&w)[4 * NB]) const {
        read_bf16(tile + T::KS0 + (8 * g + 4 * s) * (2 * NB), w);
    }
    __device__ __forceinline__ void value_scales(float (&w)[8]) const { read_bf16(tile + T::VS0 + 16 * g, w); }
    __device__ __forceinline__ Raw raw(int d) const {
        if constexpr (VB == 8)
            return *reinterpret_cast<const u32x2*>(tile + T::V0 + 512 * d + 256 * (g >> 1) + 16 * col + 8 * (g & 1u));
        else
            return u32x2{*reinterpret_cast<const uint32_t*>(tile + T::V0 + 256 * d + 128 * (g >> 1) + 8 * col + 4 * (g & 1u)), 0};
    }
    __device__ __forceinline__ bf16x8 value(Raw x) const {
        if constexpr (VB == 8) return v_frag(x.x, x.y);
        return v_frag((x.x << 4) & 0xF0F0F0F0u, x.x & 0xF0F0F0F0u);  // nibbles as the high half of a byte: 16 code
    }
};

// Half of a tile in LDS that other waves have decoded: operands, scales in f32.
template <int D>
struct OperandTile {
    using Raw = bf16x8;
    static constexpr int NB = D / 32;
    const f16x8* kf;
    const bf16x8* vf;
    const float* ks;
    const float* vs;
    __device__ __forceinline__ void key(int s, f16x8 (&f)[NB]) const {
#pragma unroll
        for (int b = 0; b < NB; b++) f[b] = kf[(s * NB + b) * 64];
    }
    __device__ __forceinline__ void key_scales(int s, float (&w)[4 * NB]) const {
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const f32x4 x = reinterpret_cast<const f32x4*>(ks + 4 * s * NB)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) w[4 * i + j] = x[j];
        }
    }
    __device__ __forceinline__ void value_scales(float (&w)[8]) const {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const f32x4 x = reinterpret_cast<const f32x4*>(vs)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) w[4 * i + j] = x[j];
        }
    }
    __device__ __forceinline__ Raw raw(int d) const { return vf[d * 64]; }
    __device__ __forceinline__ bf16x8 value(Raw x) const { return x; }
};

// Workgroups of four waves that a CU is to hold at once (the registers allow it).
constexpr int resident(int d, int nq) { return d * nq <= 256 && d < 256 ? 2 : 1; }

// Few rows (up to 16 NQ): every wave holds all of them and takes every fourth
// tile of positions, copied straight into LDS and decoded as it is read.  32 ragged
// sequences of up to 4096 positions, 8 tokens of 32 / 8 heads of 128 dims: 53 us, 188 MB
// at 3.5 TB/s, a wave issuing in 41% of its cycles and waiting in 34%; one token
// over 700 positions 8.8 us, latency.
template <int D, int KB, int VB, int NQ, bool F32>
__global__ __launch_bounds__(256, resident(D, NQ)) void attend_kernel(AttnArgs a) {
    using T = TileLds<D, KB, VB>;
    constexpr int DT = D / 16;
    constexpr uint32_t ROWS = 16u * NQ, LOWS = WaveRows<D, KB, VB, NQ, F32>::LOWS ? NQ * (D / 32) * 64 : 0;
    // a stage less where the queries' second terms would leave one workgroup a CU
    constexpr uint32_t R = T::STAGES - (LOWS != 0 && kWaves * T::STAGES * T::BYTES + LOWS * 16 + 2048 > 80 * 1024 ? 1 : 0);
    constexpr uint32_t JOIN = NQ * DT * 1024;  // bytes of a wave's output
    constexpr uint32_t LDS = kWaves * R * T::BYTES > 2 * JOIN ? kWaves * R * T::BYTES : 2 * JOIN;
    __shared__ __align__(16) uint8_t lds[LDS];
    __shared__ float sm_m[kWaves][ROWS], sm_l[kWaves][ROWS];
    __shared__ f16x8 sm_low[LOWS ? LOWS : 1];  // every wave writes the same
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    Share sh = a.shares == 0 ? whole_unit(a, ROWS) : share_of(a, ROWS);
    for (; sh.places != 0; sh.next(a, ROWS)) {
        const uint32_t now0 = sh.first_step(), now1 = sh.end_step();  // steps of this unit
        if (now0 >= now1) continue;
        const uint32_t seq = sh.seq, head = sh.unit / sh.row_tiles, tile_row = sh.unit % sh.row_tiles * ROWS;
        const SeqRange r = seq_range(a.b, seq);
        const uint32_t rows = r.n * a.group;
        const uint64_t total = seen_by_some(a, r, min(tile_row + ROWS, rows));
        const uint32_t open = open_tiles<kTile>(a, r, tile_row);
        const bool alone = now0 == 0 && now1 == sh.unit_steps;
        const uint64_t begin = (uint64_t)now0 * kStep;
        // a multiple of the tile, but for the end of what the rows see, where sees() ends
        const uint64_t end = min(total, (uint64_t)now1 * kStep);

        // This wave's tiles: every fourth from the wave-th.
        uint8_t* const mine = lds + wave * (R * T::BYTES);
        const uint32_t tile0 = (uint32_t)(begin / kTile) + wave;
        const uint32_t ends = (uint32_t)((end + kTile - 1) / kTile);
        const uint32_t count = tile0 < ends ? (ends - tile0 + kWaves - 1) / kWaves : 0;
        const Pages page_of(a, seq);
        int32_t id0 = -1, id1 = -1;  // of the next tile to fetch
        auto look_up = [&](uint32_t k) {
            const uint32_t c = 2 * (tile0 + kWaves * k);
            id0 = page_of(c);
            id1 = page_of(c + 1);
        };
        // Copies tile k, whose page ids are at hand, into its stage.  An absent chunk
        // is copied from slot 0 and masked: two bits of `absent` for each tile held.
        uint32_t absent = 0;
        auto fetch = [&](uint32_t k, uint32_t place) {
            const uint32_t c = 2 * (tile0 + kWaves * k);
            const bool ok0 = id0 >= 0 && (uint64_t)(uint32_t)id0 < a.kv.pages, ok1 = id1 >= 0 && (uint64_t)(uint32_t)id1 < a.kv.pages;
            absent |= ((ok0 ? 0u : 1u) | (ok1 ? 0u : 2u)) << (2 * place);
            uint32_t ln = lane;
            asm volatile("" : "+v"(ln));  // addresses are made here, not held in registers
            copy_tile<D, KB, VB>(a.kv, ok0 ? chunk_slot(a.kv, id0, head, c) : 0, ok1 ? chunk_slot(a.kv, id1, head, c + 1) : 0, ln,
                                 mine + k % R * T::BYTES);
        };
        using Rows = WaveRows<D, KB, VB, NQ, F32>;
        Rows w;
        w.lows = sm_low + lane;
        typename Rows::Raw raw;
        w.load(a, r, head, tile_row, rows, lane, raw);
        for (uint32_t k = 0; k < R && k < count; k++) {
            look_up(k);
            fetch(k, k);
        }
        if (R < count) look_up(R);
        w.begin(a, raw, tile_row, rows, lane);

        for (uint32_t k = 0; k < count; k++) {
            const uint32_t p0 = (tile0 + kWaves * k) * kTile;
            const uint8_t* const tile = mine + k % R * T::BYTES;
            const uint32_t gone = absent & 3u;
            absent >>= 2;
            tiles_wait<T::DMA, R - 1>(count - 1 - k);
            uint32_t ln = lane;
            asm volatile("" : "+v"(ln));
            const uint32_t g = ln >> 4, col = ln & 15u;
            const bool masked = gone != 0 || tile0 + kWaves * k >= open;
            uint32_t vis[NQ] = {};
            if (masked) {
#pragma unroll
                for (int t = 0; t < NQ; t++)
                    vis[t] = gone >> (g >> 1) & 1u ? 0u
                                                   : sees(a.mask, a.mask_words, r.row0 + w.tok[t], w.tok[t], r.n,
                                                          (int64_t)p0 + 8 * g - (int64_t)r.len);
            }
            w.step(CodeTile<D, KB, VB>{tile, g, col}, masked, vis);
            ring_wait<63>();  // the tile has been read: its stage is free
            if (k + R < count) {
                fetch(k + R, R - 1);
                if (k + R + 1 < count) look_up(k + R + 1);
            }
        }

        // join the four waves: every wave brings its rows to the common maximum, then
        // 2 and 3 hand theirs to 0 and 1, and 1 to 0
        const uint32_t g = lane >> 4, col = lane & 15u;
#pragma unroll
        for (int t = 0; t < NQ; t++) {
            w.l[t] = row_sum(w.l[t], w.m[t]);
            if (g == 0) {
                sm_m[wave][16 * t + col] = w.m[t];
                sm_l[wave][16 * t + col] = w.l[t];
            }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NQ; t++) {
            float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
            for (uint32_t v = 0; v < kWaves; v++) top = fmaxf(top, sm_m[v][16 * t + col]);
            // a wave that has seen no number yet has nothing to bring (or a NaN: times 1)
            auto back = [&](float mw) { return mw == -__builtin_inff() ? 1.0f : exp2f(mw - top); };
#pragma unroll
            for (uint32_t v = 0; v < kWaves; v++) sum += sm_l[v][16 * t + col] * back(sm_m[v][16 * t + col]);
            const float own = back(w.m[t]);
            w.m[t] = sum == 0.0f ? -__builtin_inff() : top == -__builtin_inff() ? 0.0f : top;
            w.l[t] = sum;
#pragma unroll
            for (int d = 0; d < DT; d++) w.o[t][d] *= own;
        }
        f32x4* const sm_o = reinterpret_cast<f32x4*>(lds);
#pragma unroll
        for (uint32_t half = 2; half >= 1; half /= 2) {
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int t = 0; t < NQ; t++)
#pragma unroll
                    for (int d = 0; d < DT; d++) sm_o[((wave - half) * NQ * DT + t * DT + d) * 64 + lane] = w.o[t][d];
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int t = 0; t < NQ; t++)
#pragma unroll
                    for (int d = 0; d < DT; d++) w.o[t][d] += sm_o[(wave * NQ * DT + t * DT + d) * 64 + lane];
            }
            __syncthreads();
        }
        if (wave == 0) w.store(a, sh, r, head, tile_row, tile_row, rows, ROWS, alone, lane);
        note_parts(a, sh, head, now0, now1);
        __syncthreads();  // the LDS is the next unit's
    }
}

// Many rows (16 NQ WAVES): every wave holds its own and all take the same
// positions, 64 at a time.  The waves decode a part of the tile each and leave the
// operands in LDS for all, one tile ahead; the codes of the tile after that are on
// their way into registers.  A step of few rows spends two fifths of its vector
// instructions on decoding; here that is shared by four or eight waves.  64 tokens over
// 131071 positions of 8 heads, 256 rows each: 252 us, 137 GFLOP at 545 TFLOP/s (and half
// as many products again for the probabilities' second terms), bound by the issue of the vector
// instructions around the products: 34% of the SIMDs' cycles are MFMAs.
constexpr uint32_t kWideTile = 64;

template <int D, int KB, int VB, int NQ, bool F32, int WAVES>
__global__ __launch_bounds__(64 * WAVES, D < 256 ? 2 : 1) void attend_wide_kernel(AttnArgs a) {
    constexpr int NB = D / 32, DT = D / 16, PAIRS = D / 64, ODD = NB % 2;
    constexpr uint32_t ROWS = 16u * NQ * WAVES;
    constexpr uint32_t RB = D * KB / 8;                  // bytes of a key
    constexpr uint32_t KF = 0, VF = 4 * NB * 1024;       // operands: [S][block][lane], [half][dims][lane]
    constexpr uint32_t KS = VF + 2 * DT * 1024, VS = KS + 64 * NB * 4, BUF = VS + 256;  // scales in f32
    constexpr int KU = (4 * PAIRS + WAVES - 1) / WAVES, VU = (DT + WAVES - 1) / WAVES;  // units of a wave: (S, pair), 16 dims
    constexpr uint32_t LOWS = WaveRows<D, KB, VB, NQ, F32>::LOWS ? NQ * NB * 64 : 0;
    __shared__ __align__(16) uint8_t lds[2 * BUF];
    __shared__ f16x8 sm_low[LOWS ? WAVES * LOWS : 1];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    Share sh = a.shares == 0 ? whole_unit(a, ROWS) : share_of(a, ROWS);
    for (; sh.places != 0; sh.next(a, ROWS)) {
        const uint32_t now0 = sh.first_step(), now1 = sh.end_step();
        if (now0 >= now1) continue;
        const uint32_t seq = sh.seq, head = sh.unit / sh.row_tiles, tile_row = sh.unit % sh.row_tiles * ROWS;
        const uint32_t first_row = tile_row + wave * (16u * NQ);
        const SeqRange r = seq_range(a.b, seq);
        const uint32_t rows = r.n * a.group;
        const uint64_t total = seen_by_some(a, r, min(tile_row + ROWS, rows));
        const uint32_t open = scalar(open_tiles<kWideTile>(a, r, first_row));
        const bool alone = now0 == 0 && now1 == sh.unit_steps;
        const uint32_t tile0 = now0 * (kStep / kWideTile);
        const uint32_t ends = (uint32_t)((min(total, (uint64_t)now1 * kStep) + kWideTile - 1) / kWideTile);
        const uint32_t count = tile0 < ends ? ends - tile0 : 0;
        const Pages page_of(a, seq);

        int32_t ids[4];  // of the next tile to load
        auto look_up = [&](uint32_t k) {
#pragma unroll
            for (uint32_t c = 0; c < 4; c++) ids[c] = page_of(4 * (tile0 + k) + c);
        };
        // A tile's codes, this wave's part: keys of an S and a pair of blocks (row m of S
        // number s is position 16 (m / 4) + 4 s + m % 4), values of 16 dims and all positions
        // (lane group g holds 16g..16g+15), wave 0 the keys' scales, wave 1 the values'.
        // Unit u of the keys: S u % 4, pair u / 4.
        u32x4 kr[KU], vr[VU], sr;
        u32x2 ko;
        uint32_t absent_raw = 0;  // four bits: chunks of the tile in registers that are not there
        auto load = [&](uint32_t k) {
            uint32_t ln = lane;
            asm volatile("" : "+v"(ln));
            const uint32_t g = ln >> 4, col = ln & 15u;
            uint64_t slot[4];
            absent_raw = 0;
#pragma unroll
            for (uint32_t c = 0; c < 4; c++) {
                const bool ok = ids[c] >= 0 && (uint64_t)(uint32_t)ids[c] < a.kv.pages;
                slot[c] = ok ? chunk_slot(a.kv, ids[c], head, 4 * (tile0 + k) + c) : 0;
                absent_raw |= ok ? 0u : 1u << c;
            }
            auto pick = [&](uint32_t i) {
                const uint64_t x = i & 1u ? slot[1] : slot[0], y = i & 1u ? slot[3] : slot[2];
                return i & 2u ? y : x;
            };
            const uint8_t* p = a.kv.k + (pick(col >> 2) + 4 * (wave % 4) + (col & 3u)) * RB;
#pragma unroll
            for (int j = 0; j < KU; j++) {
                const uint32_t pair = (wave + WAVES * j) / 4;
                if ((4 * PAIRS) % WAVES == 0 || pair < (uint32_t)PAIRS) {
                    if constexpr (KB == 8) {
                        kr[j] = *gptr<u32x4>(p + 64 * pair + 16 * g);
                    } else {
                        const u32x2 x = *gptr<u32x2>(p + 32 * pair + 8 * g);
                        kr[j].x = x.x, kr[j].y = x.y;
                    }
                }
            }
            if constexpr (ODD) {
                if (wave < 4) {
                    if constexpr (KB == 8) ko = *gptr<u32x2>(p + 64 * PAIRS + 8 * g);
                    else ko.x = *gptr<uint32_t>(p + 32 * PAIRS + 4 * g);
                }
            }
            const uint8_t* q = a.kv.v + pick(g) * (D * VB / 8) + col * (2 * VB);
#pragma unroll
            for (int j = 0; j < VU; j++) {
                const uint32_t d = wave + WAVES * j;
                if (DT % WAVES == 0 || d < (uint32_t)DT) {
                    if constexpr (VB == 8) {
                        vr[j] = *gptr<u32x4>(q + 256 * d);
                    } else {
                        const u32x2 x = *gptr<u32x2>(q + 128 * d);
                        vr[j].x = x.x, vr[j].y = x.y;
                    }
                }
            }
            if (wave == 0) {
                if (ln < 8u * NB)
                    sr = *gptr<u32x4>(a.kv.k + a.kv.k_scales + pick(ln / (2 * NB)) * (2 * NB) + ln % (2 * NB) * 16);
            } else if (wave == 1) {
                if (ln < 8) sr = *gptr<u32x4>(a.kv.v + a.kv.v_scales + pick(ln >> 1) * 2 + 16 * (ln & 1u));
            }
        };
        // those codes as operands into a buffer
        auto decode = [&](uint8_t* buf) {
            uint32_t ln = lane;
            asm volatile("" : "+v"(ln));
            f16x8* const kf = reinterpret_cast<f16x8*>(buf + KF + wave % 4 * (NB * 1024)) + ln;
#pragma unroll
            for (int j = 0; j < KU; j++) {
                const uint32_t pair = (wave + WAVES * j) / 4;
                if ((4 * PAIRS) % WAVES == 0 || pair < (uint32_t)PAIRS) {
                    if constexpr (KB == 8) {
                        kf[128 * pair] = k_frag(kr[j].x, kr[j].y);
                        kf[128 * pair + 64] = k_frag(kr[j].z, kr[j].w);
                    } else {
                        kf[128 * pair] = k_frag((kr[j].x << 4) & 0xF0F0F0F0u, kr[j].x & 0xF0F0F0F0u);
                        kf[128 * pair + 64] = k_frag((kr[j].y << 4) & 0xF0F0F0F0u, kr[j].y & 0xF0F0F0F0u);
                    }
                }
            }
            if constexpr (ODD) {
                if (wave < 4) {
                    if constexpr (KB == 8) kf[64 * (NB - 1)] = k_frag(ko.x, ko.y);
                    else kf[64 * (NB - 1)] = k_frag((ko.x << 4) & 0xF0F0F0F0u, ko.x & 0xF0F0F0F0u);
                }
            }
            bf16x8* const vf = reinterpret_cast<bf16x8*>(buf + VF) + ln;
#pragma unroll
            for (int j = 0; j < VU; j++) {
                const uint32_t d = wave + WAVES * j;
                if (DT % WAVES == 0 || d < (uint32_t)DT) {
                    if constexpr (VB == 8) {
                        vf[64 * d] = v_frag(vr[j].x, vr[j].y);
                        vf[64 * (DT + d)] = v_frag(vr[j].z, vr[j].w);
                    } else {
                        vf[64 * d] = v_frag((vr[j].x << 4) & 0xF0F0F0F0u, vr[j].x & 0xF0F0F0F0u);
                        vf[64 * (DT + d)] = v_frag((vr[j].y << 4) & 0xF0F0F0F0u, vr[j].y & 0xF0F0F0F0u);
                    }
                }
            }
            if (ln < (wave == 0 ? 8u * NB : wave == 1 ? 8u : 0u)) {
                f32x4* const to = reinterpret_cast<f32x4*>(buf + (wave == 0 ? KS : VS) + 32 * ln);
                to[0] = f32x4{bf16_of(sr.x, 0), bf16_of(sr.x, 1), bf16_of(sr.y, 0), bf16_of(sr.y, 1)};
                to[1] = f32x4{bf16_of(sr.z, 0), bf16_of(sr.z, 1), bf16_of(sr.w, 0), bf16_of(sr.w, 1)};
            }
        };

        using Rows = WaveRows<D, KB, VB, NQ, F32>;
        Rows w;
        w.lows = sm_low + wave * LOWS + lane;
        typename Rows::Raw raw;
        w.load(a, r, head, first_row, rows, lane, raw);
        look_up(0);
        load(0);
        if (1 < count) look_up(1);
        w.begin(a, raw, first_row, rows, lane);
        decode(lds);
        uint32_t absent = absent_raw;  // of the tile being worked on
        if (1 < count) {
            load(1);
            if (2 < count) look_up(2);
        }
        __syncthreads();
        for (uint32_t k = 0; k < count; k++) {
            const uint32_t p0 = (tile0 + k) * kWideTile;
            const uint8_t* const buf = lds + (k & 1u) * BUF;
            const uint32_t gone = absent;
            if (k + 1 < count) {
                decode(lds + ((k + 1) & 1u) * BUF);
                absent = absent_raw;
                if (k + 2 < count) {
                    load(k + 2);
                    if (k + 3 < count) look_up(k + 3);
                }
            }
            if (first_row < rows) {
#pragma unroll 1
                for (uint32_t c = 0; c < 2; c++) {
                    uint32_t ln = lane;
                    asm volatile("" : "+v"(ln));
                    const uint32_t g = ln >> 4;
                    const bool masked = gone != 0 || tile0 + k >= open;
                    uint32_t vis[NQ] = {};
                    if (masked) {
#pragma unroll
                        for (int t = 0; t < NQ; t++)
                            vis[t] = gone >> g & 1u ? 0u
                                                    : sees(a.mask, a.mask_words, r.row0 + w.tok[t], w.tok[t], r.n,
                                                           (int64_t)p0 + 16 * g + 8 * c - (int64_t)r.len);
                    }
                    w.step(OperandTile<D>{reinterpret_cast<const f16x8*>(buf + KF) + 2 * c * NB * 64 + ln,
                                          reinterpret_cast<const bf16x8*>(buf + VF) + c * DT * 64 + ln,
                                          reinterpret_cast<const float*>(buf + KS) + (16 * g + 8 * c) * NB,
                                          reinterpret_cast<const float*>(buf + VS) + 16 * g + 8 * c},
                           masked, vis);
                }
            }
            __syncthreads();
        }
        if (first_row < rows) {
#pragma unroll
            for (int t = 0; t < NQ; t++) {
                w.l[t] = row_sum(w.l[t], w.m[t]);
                w.m[t] = w.l[t] == 0.0f ? -__builtin_inff() : w.m[t] == -__builtin_inff() ? 0.0f : w.m[t];
            }
            uint32_t ln = lane;
            asm volatile("" : "+v"(ln));  // the places are made here, not held through the loop
            w.store(a, sh, r, head, tile_row, first_row, rows, ROWS, alone, ln);
        }
        note_parts(a, sh, head, now0, now1);
    }
}

// Launches the instantiation of (head_dim, tiles, dtype) for one pair of encodings.
template <int KB, int VB>
hipError_t attend_launch(const AttnArgs& a, uint32_t tiles, uint64_t grid, hipStream_t st);

template <int D, int KB, int VB>
hipError_t attend_launch_dim(const AttnArgs& a, uint32_t tiles, uint64_t grid, hipStream_t st) {
    const dim3 gd((uint32_t)grid), bd(64 * kWaves);
    if (tiles >= 4) {  // 64, 128 or 256 rows
        if (tiles == 4) {
            if (a.q.bf16) attend_wide_kernel<D, KB, VB, 1, false, 4><<<gd, bd, 0, st>>>(a);
            else attend_wide_kernel<D, KB, VB, 1, true, 4><<<gd, bd, 0, st>>>(a);
        } else {
            if constexpr (D <= 128) {
                if (!a.q.bf16) attend_wide_kernel<D, KB, VB, 2, true, 8><<<gd, dim3(512), 0, st>>>(a);
                else if (tiles == 8) attend_wide_kernel<D, KB, VB, 2, false, 4><<<gd, bd, 0, st>>>(a);
                else attend_wide_kernel<D, KB, VB, 2, false, 8><<<gd, dim3(512), 0, st>>>(a);
            } else {
                return hipErrorInvalidValue;
            }
        }
    } else if (tiles == 1) {
        if (a.q.bf16) attend_kernel<D, KB, VB, 1, false><<<gd, bd, 0, st>>>(a);
        else attend_kernel<D, KB, VB, 1, true><<<gd, bd, 0, st>>>(a);
    } else {
        if constexpr (D <= 128) {
            if (a.q.bf16) attend_kernel<D, KB, VB, 2, false><<<gd, bd, 0, st>>>(a);
            else attend_kernel<D, KB, VB, 2, true><<<gd, bd, 0, st>>>(a);
        } else {
            return hipErrorInvalidValue;
        }
    }
    return hipGetLastError();
}

#define DMX_ATTEND_INSTANCE(KB, VB)                                                                             \
    namespace dmx {                                                                                             \
    template <>                                                                                                 \
    hipError_t attend_launch<KB, VB>(const AttnArgs& a, uint32_t tiles, uint64_t grid, hipStream_t st) {        \
        switch (a.kv.dim) {                                                                                     \
        case 64: return attend_launch_dim<64, KB, VB>(a, tiles, grid, st);                                      \
        case 96: return attend_launch_dim<96, KB, VB>(a, tiles, grid, st);                                      \
        case 128: return attend_launch_dim<128, KB, VB>(a, tiles, grid, st);                                    \
        case 256: return attend_launch_dim<256, KB, VB>(a, tiles, grid, st);                                    \
        }                                                                                                       \
        return hipErrorInvalidValue;                                                                            \
    }                                                                                                           \
    }

}  // namespace dmx
