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
#include "kvcache.hpp"

namespace dmx {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kTile = 64;   // positions of a wave's step
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

// Dwords a lane loads for one token's K codes (its part of every block), and
// for one dim's 16 V codes.
template <int D, int KB>
constexpr int kKWords = D / 16 * KB / 8;

// K codes of this lane's part of a token's row: per pair of blocks one load.
template <int D, int KB>
__device__ __forceinline__ void load_k(const uint8_t* row, uint32_t part, uint32_t (&w)[kKWords<D, KB>]) {
#pragma unroll
    for (int p = 0; p < D / 64; p++) {
        if constexpr (KB == 8) {
            const u32x4 x = *gptr<u32x4>(row + 64 * p + 16 * part);
#pragma unroll
            for (int i = 0; i < 4; i++) w[4 * p + i] = x[i];
        } else {
            const u32x2 x = *gptr<u32x2>(row + 32 * p + 8 * part);
            w[2 * p] = x.x;
            w[2 * p + 1] = x.y;
        }
    }
    if constexpr (D % 64) {
        constexpr int P = D / 64;
        if constexpr (KB == 8) {
            const u32x2 x = *gptr<u32x2>(row + 64 * P + 8 * part);
            w[4 * P] = x.x;
            w[4 * P + 1] = x.y;
        } else {
            w[2 * P] = *gptr<uint32_t>(row + 32 * P + 4 * part);
        }
    }
}

// Block b's operand from those words.
template <int D, int KB>
__device__ __forceinline__ f16x8 k_block(const uint32_t (&w)[kKWords<D, KB>], int b) {
    if constexpr (KB == 8) {
        return k_frag(w[2 * b], w[2 * b + 1]);
    } else {  // nibbles as the high half of a byte: 16 (8 + code)
        return k_frag((w[b] << 4) & 0xF0F0F0F0u, w[b] & 0xF0F0F0F0u);
    }
}

// Which of positions 16g..16g+15 of a tile (the lane group's) row `row` of the
// sequence sees, one bit each.  j0: the first of them, from the first new token.
__device__ __forceinline__ uint32_t sees(const int64_t* mask, uint32_t words, uint64_t row, uint32_t i, uint32_t n,
                                         int64_t j0) {
    if (j0 <= -16) return 0xFFFFu;
    if (j0 >= (int64_t)n) return 0u;
    if (!mask) {  // rows j <= i
        const int64_t c = (int64_t)i + 1 - j0;
        return c <= 0 ? 0u : c >= 16 ? 0xFFFFu : (1u << c) - 1u;
    }
    const uint32_t lead = j0 < 0 ? (uint32_t)-j0 : 0u;  // committed positions among the sixteen
    const uint32_t j = (uint32_t)(j0 + lead);
    const int64_t* m = mask + row * words;
    const uint32_t w = j >> 6, sh = j & 63u;
    uint64_t v = (uint64_t)m[w] >> sh;
    if (sh && w + 1 < words) v |= (uint64_t)m[w + 1] << (64 - sh);
    const uint32_t left = n - j;
    if (left < 16) v &= (1ull << left) - 1ull;
    return ((uint32_t)(v << lead) | ((1u << lead) - 1u)) & 0xFFFFu;
}

template <int D, int KB, int VB, int NQ, bool F32>
__global__ __launch_bounds__(256) void attend_kernel(AttnArgs a) {
    constexpr int NB = D / 32;            // blocks of a key
    constexpr int DT = D / 16;            // 16-dim tiles of the output
    constexpr int TERMS = F32 ? 3 : 2;    // bf16 terms of a probability
    constexpr int KW = kKWords<D, KB>, VW = VB / 2;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t g = lane >> 4, col = lane & 15u;

    uint32_t id = blockIdx.x;
    const uint32_t rt = id % a.row_tiles;
    id /= a.row_tiles;
    const uint32_t head = id % a.kv.heads;
    id /= a.kv.heads;
    const uint32_t split = id % a.splits, seq = id / a.splits;
    const SeqRange r = seq_range(a.b, seq);
    const uint32_t rows = r.n * a.group;
    if (rt * (16u * NQ) >= rows) return;
    const uint64_t total = (uint64_t)r.len + r.n;
    const uint64_t begin = (uint64_t)split * a.span;
    if (begin >= total) return;
    // a multiple of the tile, but for the sequence's own end, where sees() ends
    const uint64_t end = split + 1 == a.splits ? total : min(total, begin + a.span);

    // this lane's rows (columns of the products), their queries as operands
    f16x8 qf[NQ][NB], ql[F32 ? NQ : 1][F32 ? NB : 1];
    float factor[NQ], m[NQ], l[NQ];
    uint32_t tok[NQ];
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
                for (int i = 0; i < 4; i++) {
                    x[b][2 * i] = bf16_bits_to_f32(w[i] & 0xFFFFu);
                    x[b][2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                }
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
        const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
        factor[t] = a.scale * 1.44269504088896341f * (KB == 4 ? 0.0625f : 1.0f);
        factor[t] *= __uint_as_float((uint32_t)(e - 14 + 127) << 23);
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

    const uint16_t* ksc = reinterpret_cast<const uint16_t*>(a.kv.k + a.kv.k_scales);
    const uint16_t* vsc = reinterpret_cast<const uint16_t*>(a.kv.v + a.kv.v_scales);

    for (uint64_t p0 = begin + kTile * wave; p0 < end; p0 += kTile * kWaves) {
        // chunk addresses: the one whose keys this lane loads, the one whose values and scales
        const uint32_t c0 = (uint32_t)(p0 / 16);
        const int64_t pk = chunk_page(a.kv, a.b, seq, c0 + col / 4);
        const int64_t pv = chunk_page(a.kv, a.b, seq, c0 + g);
        const uint64_t sk = pk < 0 ? 0 : chunk_slot(a.kv, pk, head, c0 + col / 4);
        const uint64_t sv = pv < 0 ? 0 : chunk_slot(a.kv, pv, head, c0 + g);
        const bool edge = __any(p0 + kTile > r.len || pv < 0);

        uint32_t kw[4][KW], vw[DT][VW];
#pragma unroll
        for (int s = 0; s < 4; s++)
            load_k<D, KB>(a.kv.k + (sk + 4 * s + col % 4) * (D * KB / 8), g, kw[s]);
        uint32_t ks[4][4 * NB / 2];  // bf16 scales of this lane's four positions of each S
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(ksc + (sv + 4 * s) * NB);
#pragma unroll
            for (int i = 0; i < 2 * NB; i += 4) {
                if constexpr (NB % 2 == 0) {
                    const u32x4 x = *gptr<u32x4>(p + i);
#pragma unroll
                    for (int j = 0; j < 4; j++) ks[s][i + j] = x[j];
                } else {
                    const u32x2 x = *gptr<u32x2>(p + i);
                    ks[s][i] = x.x, ks[s][i + 1] = x.y;
                    if (i + 2 < 2 * NB) {
                        const u32x2 y = *gptr<u32x2>(p + i + 2);
                        ks[s][i + 2] = y.x, ks[s][i + 3] = y.y;
                    }
                }
            }
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const uint8_t* p = a.kv.v + sv * (D * VB / 8) + (16 * d + col) * (2 * VB);
            if constexpr (VB == 8) {
                const u32x4 x = *gptr<u32x4>(p);
#pragma unroll
                for (int i = 0; i < 4; i++) vw[d][i] = x[i];
            } else {
                const u32x2 x = *gptr<u32x2>(p);
                vw[d][0] = x.x, vw[d][1] = x.y;
            }
        }
        uint32_t vs[8];
        {
            const u32x4 x = *gptr<u32x4>(vsc + sv), y = *gptr<u32x4>(vsc + sv + 8);
#pragma unroll
            for (int i = 0; i < 4; i++) vs[i] = x[i], vs[4 + i] = y[i];
        }

        // S: 16 positions x 16 rows at a time
        f32x4 sc[NQ][4];
#pragma unroll
        for (int s = 0; s < 4; s++) {
            f16x8 kf[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) kf[b] = k_block<D, KB>(kw[s], b);
#pragma unroll
            for (int t = 0; t < NQ; t++) {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    f32x4 x = {0, 0, 0, 0};
                    if constexpr (F32) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[b], ql[t][b], x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[b], qf[t][b], x, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int at = i * NB + b;  // bf16 number in ks[s]
                        const float w = __uint_as_float(at & 1 ? ks[s][at / 2] & 0xFFFF0000u : ks[s][at / 2] << 16);
                        sc[t][s][i] = b == 0 ? x[i] * w : sc[t][s][i] + x[i] * w;
                    }
                }
            }
        }

        // running maximum, exponentials
#pragma unroll
        for (int t = 0; t < NQ; t++) {
            uint32_t vis = 0xFFFFu;
            if (edge) {
                vis = pv < 0 ? 0u
                             : sees(a.mask, a.mask_words, r.row0 + tok[t], tok[t], r.n,
                                    (int64_t)(p0 + 16 * g) - (int64_t)r.len);
            }
            float top = m[t];
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x = sc[t][s][i] * factor[t];
                    if (edge) x = (vis >> (4 * s + i)) & 1u ? x : -__builtin_inff();
                    sc[t][s][i] = x;
                    top = fmaxf(top, x);
                }
            top = rows_max(top);
            const float ref = top == -__builtin_inff() ? 0.0f : top;
            if (__any(top > m[t])) {
                const float back = exp2f(m[t] - ref);
                l[t] *= back;
#pragma unroll
                for (int d = 0; d < DT; d++) o[t][d] *= back;
            }
            m[t] = top;
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = __builtin_amdgcn_exp2f(sc[t][s][i] - ref);
                    l[t] += e;
                    const int at = 4 * s + i;
                    const float w = __uint_as_float(at & 1 ? vs[at / 2] & 0xFFFF0000u : vs[at / 2] << 16);
                    float p = e * w;
                    if (edge) p = (vis >> at) & 1u ? p : 0.0f;  // a masked value's scale may be anything
                    sc[t][s][i] = p;
                }
        }

        // the product with V, 32 positions at a time
#pragma unroll
        for (int c = 0; c < 2; c++) {
            bf16x8 pf[NQ][TERMS];
#pragma unroll
            for (int t = 0; t < NQ; t++) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] = sc[t][2 * c + j / 4][j % 4];
#pragma unroll
                for (int k = 0; k < TERMS; k++) {
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        w[j] = f32x2_to_bf16x2_bits(p[2 * j], p[2 * j + 1]);
                        if (k + 1 < TERMS) {
                            p[2 * j] -= __uint_as_float(w[j] << 16);
                            p[2 * j + 1] -= __uint_as_float(w[j] & 0xFFFF0000u);
                        }
                    }
                    pf[t][k] = __builtin_bit_cast(bf16x8, w);
                }
            }
#pragma unroll
            for (int d = 0; d < DT; d++) {
                bf16x8 vf;
                if constexpr (VB == 8)
                    vf = v_frag(vw[d][2 * c], vw[d][2 * c + 1]);
                else  // nibbles as the high half of a byte: 16 code
                    vf = v_frag((vw[d][c] << 4) & 0xF0F0F0F0u, vw[d][c] & 0xF0F0F0F0u);
#pragma unroll
                for (int t = 0; t < NQ; t++)
#pragma unroll
                    for (int k = TERMS - 1; k >= 0; k--)
                        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[t][k], o[t][d], 0, 0, 0);
            }
        }
    }

    // join the four waves: every wave brings its rows to the common maximum, then
    // 2 and 3 hand theirs to 0 and 1, and 1 to 0
    __shared__ float sm_m[kWaves][16 * NQ], sm_l[kWaves][16 * NQ];
    __shared__ f32x4 sm_o[2][NQ * DT][64];
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
        const float ref = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; w++) sum += sm_l[w][16 * t + col] * exp2f(sm_m[w][16 * t + col] - ref);
        const float back = exp2f(m[t] - ref) * (VB == 4 ? 0.0625f : 1.0f);
        m[t] = top;
        l[t] = sum;
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] *= back;
    }
#pragma unroll
    for (uint32_t half = 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int t = 0; t < NQ; t++)
#pragma unroll
                for (int d = 0; d < DT; d++) sm_o[wave - half][t * DT + d][lane] = o[t][d];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int t = 0; t < NQ; t++)
#pragma unroll
                for (int d = 0; d < DT; d++) o[t][d] += sm_o[wave][t * DT + d][lane];
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
#define DMX_ATTEND(NQ)                                                           \
    if (a.q.bf16)                                                                \
        attend_kernel<D, KB, VB, NQ, false><<<gd, bd, 0, st>>>(a);               \
    else                                                                         \
        attend_kernel<D, KB, VB, NQ, true><<<gd, bd, 0, st>>>(a);
    if (tiles == 1) {
        DMX_ATTEND(1)
    } else if constexpr (D <= 128) {
        DMX_ATTEND(2)
    } else {
        return hipErrorInvalidValue;
    }
#undef DMX_ATTEND
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
