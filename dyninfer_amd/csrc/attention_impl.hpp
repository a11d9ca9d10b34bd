// Attention of a few new tokens a sequence (a chain or a tree of drafts) over
// the quantized paged cache: the kernel, instantiated per pair of encodings in
// attention_k<bits>v<bits>.hip.
//
//   S[p, r] = scale q_r . k_p,  out_r = sum_p exp(S - max) v_p / sum_p exp(S - max)
//
// over the positions p that row r sees.  Rows of one kv head are the new tokens
// times the query heads that share it, r = token * group + head: up to 32 of
// them share one pass over the cache.
//
// One pass, online: a wave takes 64 positions at a time, keeps the running
// maximum and sum of every row and the unnormalised output in registers, and
// joins its state with the other three waves' in LDS at the end, and, when the
// positions are split over workgroups, through the workspace and a second
// small launch.  Few rows over a long context are bound by the cache's bytes;
// from about 64 rows the vector instructions around the products are.
//
// The products are 16x16x32 MFMAs with the cache as the first operand, so that
// a row of the output (a column of the second operand) belongs to lanes l with
// l % 16 = r: its statistics are in the lane, and the exponentials that come
// out of S are, unmoved, the second operand of the product with V:
//   S (16 positions x 16 rows): lane l holds positions 4(l / 16) + i, i < 4
//   P (32 positions x 16 rows): lane l holds positions 8(l / 16) + j, j < 8
// The sum over positions may take them in any order if both operands agree, so
// position 16g + 4s + i of a tile is row 4g + i of the s-th S: lane group g then
// holds positions 16g..16g+15, which for one dim of V are 16 codes in a row.
//
// Numerics: K codes are exact in f16 (0x6400 | byte is 1024 + byte; the offset
// is taken off exactly), queries are scaled to a power of two that puts the
// row's largest in [2^14, 2^15) and are exact in f16 down to 2^-29 of it (f32
// queries: a second f16 holds what the first leaves), each block's sum is
// multiplied by its f32 scale.  V codes are exact in bf16; p times the value's
// scale, of unknown range, is split into bf16 terms: two (16 bits) for bf16
// outputs, three (24 bits) for f32 ones.
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
    static constexpr uint32_t STAGES = BYTES > 9216 ? 2 : BYTES > 6656 ? 2 : BYTES > 4608 ? 3 : 4;
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

// Workgroups of four waves that a CU is to hold at once (the registers allow it).
constexpr int resident(int d, int nq) { return d * nq <= 256 && d < 256 ? 2 : 1; }

template <int D, int KB, int VB, int NQ, bool F32>
__global__ __launch_bounds__(256, resident(D, NQ)) void attend_kernel(AttnArgs a) {
    using T = TileLds<D, KB, VB>;
    constexpr int NB = D / 32;            // blocks of a key
    constexpr int DT = D / 16;            // 16-dim tiles of the output
    constexpr int TERMS = F32 ? 3 : 2;    // bf16 terms of a probability
    constexpr uint32_t R = T::STAGES;
    constexpr uint32_t JOIN = NQ * DT * 1024;  // bytes of a wave's output
    constexpr uint32_t LDS = kWaves * R * T::BYTES > 2 * JOIN ? kWaves * R * T::BYTES : 2 * JOIN;
    __shared__ __align__(16) uint8_t lds[LDS];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15u;

    // Workgroups go round the eight XCDs; those that share a piece of the cache
    // (row tiles of one part of one head) are eight apart, on one XCD and its L2.
    const uint32_t rt = blockIdx.x / 8 % a.row_tiles;
    uint32_t id = blockIdx.x / 8 / a.row_tiles * 8 + blockIdx.x % 8;
    const uint32_t head = id % a.kv.heads;
    id /= a.kv.heads;
    const uint32_t split = id % a.splits, seq = id / a.splits;
    if (seq >= a.b.seqs) return;
    const SeqRange r = seq_range(a.b, seq);
    const uint32_t rows = r.n * a.group;
    if (rt * (16u * NQ) >= rows) return;
    const uint64_t total = (uint64_t)r.len + r.n;
    const uint64_t begin = (uint64_t)split * a.span;
    if (begin >= total) return;
    // a multiple of the tile, but for the sequence's own end, where sees() ends
    const uint64_t end = split + 1 == a.splits ? total : min(total, begin + a.span);

    // This wave's tiles: every fourth from the wave-th.
    uint8_t* const mine = lds + wave * (R * T::BYTES);
    const uint32_t tile0 = (uint32_t)(begin / kTile) + wave;
    const uint32_t ends = (uint32_t)((end + kTile - 1) / kTile);
    const uint32_t count = tile0 < ends ? (ends - tile0 + kWaves - 1) / kWaves : 0;
    // Page ids of a tile's two chunks, all lanes alike (scalar loads).
    const uint64_t table = (uint64_t)(a.b.table + (size_t)seq * a.b.table_pages);
    auto page_of = [&](uint32_t chunk) -> int32_t {
        const uint32_t i = chunk >> (a.kv.page_shift - 4u);
        return i < a.b.table_pages ? *(const __attribute__((address_space(4))) int32_t*)(table + 4ull * i) : -1;
    };
    int32_t id0 = -1, id1 = -1;
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
    for (uint32_t k = 0; k < R - 1 && k < count; k++) {
        look_up(k);
        fetch(k, k);
    }
    if (R - 1 < count) look_up(R - 1);

    // this lane's rows (columns of the products), their queries as operands
    f16x8 qf[NQ][NB], ql[F32 ? NQ : 1][F32 ? NB : 1];
    float factor[NQ], m[NQ], l[NQ];  // m: what exponents are taken from, about the largest so far (log2)
    uint32_t tok[NQ];
    const float sign = a.scale < 0.0f ? -1.0f : 1.0f;  // so that the largest score is that of the largest sum
#pragma unroll
    for (int t = 0; t < NQ; t++) {
        const uint32_t row = rt * (16u * NQ) + 16u * t + col;
        const bool live = row < rows;
        tok[t] = live ? row / a.group : 0u;
        const uint32_t h = head * a.group + (live ? row % a.group : 0u);
        const int64_t at = (int64_t)(r.row0 + tok[t]) * a.q.ts + (int64_t)h * a.q.hs;
        float x[NB][8], big = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int64_t e = at + 32 * b + 8 * g;
            if (a.q.vec && !F32) {
                const u32x4 w = *gptr<u32x4>(static_cast<const uint16_t*>(a.q.p) + e);
#pragma unroll
                for (int i = 0; i < 8; i++) x[b][i] = bf16_of(w[i / 2], i & 1);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    x[b][i] = F32 ? gptr<float>(a.q.p)[e + i] : bf16_bits_to_f32(gptr<uint16_t>(a.q.p)[e + i]);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[b][i]));
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
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float s = live ? x[b][i] * up : 0.0f;
                qf[t][b][i] = (_Float16)s;
                if constexpr (F32) ql[t][b][i] = (_Float16)(s - (float)qf[t][b][i]);
            }
        }
        m[t] = -__builtin_inff();
        l[t] = 0.0f;
    }

    f32x4 o[NQ][DT];
#pragma unroll
    for (int t = 0; t < NQ; t++)
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] = f32x4{0, 0, 0, 0};

    for (uint32_t k = 0; k < count; k++) {
        const uint32_t p0 = (tile0 + kWaves * k) * kTile;
        const uint8_t* const tile = mine + k % R * T::BYTES;
        // the stage of tile k - 1 is free: its last reads have been waited for
        if (k + R - 1 < count) {
            fetch(k + R - 1, R - 1);
            if (k + R < count) look_up(k + R);
        }
        const uint32_t gone = absent & 3u;
        absent >>= 2;
        tiles_wait<T::DMA, R - 1>(count - 1 - k);
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));
        const uint32_t g = ln >> 4, col = ln & 15u;

        // S: 16 positions x 16 rows at a time
        f32x4 sc[NQ][2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            uint32_t kw[D / 16 * KB / 8], ks[2 * NB];  // bf16 scales of four positions
            read_k<D, KB, VB>(tile, s, col, g, kw);
#pragma unroll
            for (int i = 0; i < 2 * NB; i += 2) {
                const u32x2 x = *reinterpret_cast<const u32x2*>(tile + T::KS0 + (8 * g + 4 * s) * (2 * NB) + 4 * i);
                ks[i] = x.x, ks[i + 1] = x.y;
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const f16x8 kf = k_block<D, KB>(kw, b);
#pragma unroll
                for (int t = 0; t < NQ; t++) {
                    f32x4 x = {0, 0, 0, 0};
                    if constexpr (F32) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[t][b], x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[t][b], x, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int at = i * NB + b;
                        const float w = bf16_of(ks[at / 2], at & 1);
                        sc[t][s][i] = b == 0 ? x[i] * w : sc[t][s][i] + x[i] * w;
                    }
                }
            }
        }

        const bool edge = gone != 0 || (uint64_t)p0 + kTile > r.len;
        uint32_t vis[NQ];
        if (edge) {
#pragma unroll
            for (int t = 0; t < NQ; t++) {
                vis[t] = gone >> (g >> 1) & 1u ? 0u
                                               : sees(a.mask, a.mask_words, r.row0 + tok[t], tok[t], r.n,
                                                      (int64_t)p0 + 8 * g - (int64_t)r.len);
#pragma unroll
                for (int i = 0; i < 8; i++) sc[t][i / 4][i % 4] = vis[t] >> i & 1u ? sc[t][i / 4][i % 4] : -__builtin_inff();
            }
        }

        // Exponentials, from a reference that follows the row's largest score only when
        // one is 2^8 above it: the sums are f32 either way, and most tiles then need
        // neither the maximum over lanes nor a rescaling.
        const u32x4 vs = *reinterpret_cast<const u32x4*>(tile + T::VS0 + 16 * g);
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
                p[i] = e * bf16_of(vs[i / 2], i & 1);
            }
            if (edge) {  // a masked value's scale may be anything
#pragma unroll
                for (int i = 0; i < 8; i++) p[i] = vis[t] >> i & 1u ? p[i] : 0.0f;
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
            bf16x8 vf;
            if constexpr (VB == 8) {
                const u32x2 x = *reinterpret_cast<const u32x2*>(tile + T::V0 + 512 * d + 256 * (g >> 1) + 16 * col + 8 * (g & 1u));
                vf = v_frag(x.x, x.y);
            } else {  // nibbles as the high half of a byte: 16 code
                const uint32_t x = *reinterpret_cast<const uint32_t*>(tile + T::V0 + 256 * d + 128 * (g >> 1) + 8 * col + 4 * (g & 1u));
                vf = v_frag((x << 4) & 0xF0F0F0F0u, x & 0xF0F0F0F0u);
            }
#pragma unroll
            for (int n = TERMS - 1; n >= 0; n--)
#pragma unroll
                for (int t = 0; t < NQ; t++)
                    o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[t][n], o[t][d], 0, 0, 0);
        }
        ring_wait<63>();  // the tile has been read
    }

    // join the four waves: every wave brings its rows to the common maximum, then
    // 2 and 3 hand theirs to 0 and 1, and 1 to 0
    __shared__ float sm_m[kWaves][16 * NQ], sm_l[kWaves][16 * NQ];
#pragma unroll
    for (int t = 0; t < NQ; t++) {
        l[t] = rows_sum(l[t]);
        if (g == 0) {
            sm_m[wave][16 * t + col] = m[t];
            sm_l[wave][16 * t + col] = l[t];
        }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NQ; t++) {
        float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; w++) top = fmaxf(top, sm_m[w][16 * t + col]);
        // a wave that has seen no number yet has nothing to bring (or a NaN: times 1)
        auto back = [&](float mw) { return mw == -__builtin_inff() ? 1.0f : exp2f(mw - top); };
#pragma unroll
        for (uint32_t w = 0; w < kWaves; w++) sum += sm_l[w][16 * t + col] * back(sm_m[w][16 * t + col]);
        const float own = back(m[t]) * (VB == 4 ? 0.0625f : 1.0f);
        m[t] = sum == 0.0f ? -__builtin_inff() : top == -__builtin_inff() ? 0.0f : top;
        l[t] = sum;
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] *= own;
    }
    f32x4* const sm_o = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (uint32_t half = 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int t = 0; t < NQ; t++)
#pragma unroll
                for (int d = 0; d < DT; d++) sm_o[((wave - half) * NQ * DT + t * DT + d) * 64 + lane] = o[t][d];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int t = 0; t < NQ; t++)
#pragma unroll
                for (int d = 0; d < DT; d++) o[t][d] += sm_o[(wave * NQ * DT + t * DT + d) * 64 + lane];
        }
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int t = 0; t < NQ; t++) {
        const uint32_t row = rt * (16u * NQ) + 16u * t + col;
        if (row >= rows) continue;
        const uint32_t h = head * a.group + row % a.group;
        const uint64_t token = r.row0 + row / a.group, q_heads = (uint64_t)a.kv.heads * a.group;
        if (a.splits > 1) {
            const uint64_t at = (token * q_heads + h) * a.splits + split;
            float* po = a.work + at * D;
#pragma unroll
            for (int d = 0; d < DT; d++) *gptr_mut<f32x4>(po + 16 * d + 4 * g) = o[t][d];
            if (g == 0) {
                float* ml = a.work + (uint64_t)a.b.tokens * q_heads * a.splits * D + 2 * at;
                gptr_mut<float>(ml)[0] = m[t];
                gptr_mut<float>(ml)[1] = l[t];
            }
        } else {
            const float inv = l[t] > 0.0f ? 1.0f / l[t] : (l[t] == 0.0f ? 0.0f : __builtin_nanf(""));
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

// Launches the instantiation of (head_dim, tiles, dtype) for one pair of encodings.
template <int KB, int VB>
hipError_t attend_launch(const AttnArgs& a, uint32_t tiles, uint64_t grid, hipStream_t st);

template <int D, int KB, int VB>
hipError_t attend_launch_dim(const AttnArgs& a, uint32_t tiles, uint64_t grid, hipStream_t st) {
    const dim3 gd((uint32_t)grid), bd(64 * kWaves);
    if (!a.q.bf16) {
        if (tiles == 1) {
            attend_kernel<D, KB, VB, 1, true><<<gd, bd, 0, st>>>(a);
        } else {
            if constexpr (D <= 128) attend_kernel<D, KB, VB, 2, true><<<gd, bd, 0, st>>>(a);
            else return hipErrorInvalidValue;
        }
    } else if (tiles == 1) {
        attend_kernel<D, KB, VB, 1, false><<<gd, bd, 0, st>>>(a);
    } else if (tiles == 2) {
        attend_kernel<D, KB, VB, 2, false><<<gd, bd, 0, st>>>(a);
    } else {
        if constexpr (D <= 128) attend_kernel<D, KB, VB, 4, false><<<gd, bd, 0, st>>>(a);
        else return hipErrorInvalidValue;
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
