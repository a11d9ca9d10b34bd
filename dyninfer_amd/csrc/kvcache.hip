// Norms of heads, rotary positions and the quantized paged cache: writing, reading back, and
// keeping an accepted path.  All are bound by memory (large calls) or by the
// latency of one launch (small ones); the arithmetic is small beside either.
//
// Rows: a lane holds 8 consecutive dims of one head (16 bytes of bf16), a head
// takes D / 8 lanes of one wave (rounded up to a power of two), so a block of
// 32 dims is 4 lanes and its extremes take two shuffles, and the dims of a
// rotary pair are in the lane itself (interleaved) or one more load away.
//
// Results are bit-identical to the plain sequence of f32 operations: products,
// sums and quotients are rounded one by one (no contraction), the division by
// a scale is the correctly rounded one.
#include "kvcache.hpp"

#include <type_traits>

#pragma clang fp contract(off)

namespace dmx {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Lanes that hold one head of D dims.
template <int D>
constexpr int kLanes = D <= 64 ? 8 : D <= 128 ? 16 : 32;

__device__ __forceinline__ float load1(const KvRows& r, int64_t at) {
    return r.bf16 ? bf16_bits_to_f32(gptr<uint16_t>(r.p)[at]) : gptr<float>(r.p)[at];
}

// Eight elements from element offset `at` (of a row of 16-byte boundaries if r.vec).
__device__ __forceinline__ void load8(const KvRows& r, int64_t at, float (&x)[8]) {
    if (r.vec && r.bf16) {
        const u32x4 w = *gptr<u32x4>(static_cast<const uint16_t*>(r.p) + at);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = bf16_bits_to_f32(w[i] & 0xFFFFu);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else if (r.vec) {
        const f32x4 a = *gptr<f32x4>(static_cast<const float*>(r.p) + at);
        const f32x4 b = *gptr<f32x4>(static_cast<const float*>(r.p) + at + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = load1(r, at + i);
    }
}

__device__ __forceinline__ void store8(const KvRows& r, int64_t at, const float (&x)[8]) {
    if (r.bf16) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = f32x2_to_bf16x2_bits(x[2 * i], x[2 * i + 1]);
        uint16_t* p = static_cast<uint16_t*>(r.p) + at;
        if (r.vec) {
            *gptr_mut<u32x4>(p) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) gptr_mut<uint16_t>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    } else {
        float* p = static_cast<float*>(r.p) + at;
        if (r.vec) {
            *gptr_mut<f32x4>(p) = f32x4{x[0], x[1], x[2], x[3]};
            *gptr_mut<f32x4>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) gptr_mut<float>(p)[i] = x[i];
        }
    }
}

// What a row's values are multiplied by before they are rotated: nothing, or ..
struct NoNorm {
    __device__ __forceinline__ void apply(uint32_t, float (&)[8]) const {}
    __device__ __forceinline__ void apply(uint32_t, float (&)[4]) const {}
    __device__ __forceinline__ float one(uint32_t, float x) const { return x; }
};

// .. its root mean square's inverse and the weight of the dim: (x f) r (w + offset), where f is
// 1, or 2^-72 for a row whose squares would leave f32.
struct HeadNorm {
    const NormView& n;
    float f, r;

    __device__ __forceinline__ float one(uint32_t d, float x) const {
        x = x * f * r;
        if (!n.weight) return x * (1.0f + n.offset);
        return x * ((n.bf16 ? bf16_bits_to_f32(gptr<uint16_t>(n.weight)[d]) : gptr<float>(n.weight)[d]) + n.offset);
    }
    template <int N>
    __device__ __forceinline__ void apply(uint32_t d0, float (&x)[N]) const {
        float w[N];
        if (!n.weight) {
#pragma unroll
            for (int i = 0; i < N; i++) w[i] = 1.0f;
        } else if (n.vec && n.bf16) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const u32x2 a = *gptr<u32x2>(static_cast<const uint16_t*>(n.weight) + d0 + i);
#pragma unroll
                for (int j = 0; j < 4; j++) w[i + j] = __uint_as_float(j & 1 ? a[j / 2] & 0xFFFF0000u : a[j / 2] << 16);
            }
        } else if (n.vec) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const f32x4 a = *gptr<f32x4>(static_cast<const float*>(n.weight) + d0 + i);
#pragma unroll
                for (int j = 0; j < 4; j++) w[i + j] = a[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
                w[i] = n.bf16 ? bf16_bits_to_f32(gptr<uint16_t>(n.weight)[d0 + i]) : gptr<float>(n.weight)[d0 + i];
        }
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = x[i] * f * r * (w[i] + n.offset);
    }
};

// Sum over the N lanes around this one (N a power of two, 8 to 32, aligned), the same in all of them.
template <int N>
__device__ __forceinline__ float lanes_sum(float x) {
    auto moved = [](float v, auto ctrl) {
        return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    x += moved(x, std::integral_constant<int, 0xB1>());   // lane ^ 1
    x += moved(x, std::integral_constant<int, 0x4E>());   // lane ^ 2
    x += moved(x, std::integral_constant<int, 0x141>());  // mirrored in 8
    if constexpr (N > 8) x += moved(x, std::integral_constant<int, 0x140>());  // mirrored in 16
    if constexpr (N > 16) x += __shfl_xor(x, 16);
    return x;
}

// The norm of the head whose D dims the kLanes<D> lanes around this one hold, eight in each
// (zeros in lanes without dims; the lanes of a head come here together).  v_rsq_f32 is off by
// one ulp at most, beside the two roundings of the product.  Rows of 1e19 and more, whose squares
// overflow, are summed again at 2^-72 of their size; eps is then far below the mean.  A NaN
// makes the head NaN, an infinity its own dim (the others become 0).
template <int D>
__device__ __forceinline__ HeadNorm head_norm(const NormView& n, const float (&x)[8]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) s += x[i] * x[i];
    s = lanes_sum<kLanes<D>>(s);
    float f = 1.0f, e = n.eps;
    if (!(s <= 3.0e38f)) {
        f = 0x1p-72f;
        e = n.eps * 0x1p-72f * 0x1p-72f;
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) s += x[i] * f * (x[i] * f);
        s = lanes_sum<kLanes<D>>(s);
    }
    return {n, f, __builtin_amdgcn_rsqf(s * (1.0f / D) + e)};
}

// x: dims d0..d0+7 of the row at element offset `row`, after `norm`; rotated in place.  The
// wide forms need the pairs of the eight dims to be eight dims or eight pairs
// of floats in a row: rot / 2 (half) a multiple of 8, rot (interleaved) too.
template <class N>
__device__ __forceinline__ void rotate8(const KvRows& r, int64_t row, uint32_t token, uint32_t d0, const RopeView& rp,
                                        const N& norm, float (&x)[8]) {
    if (d0 >= rp.rot) return;
    const uint32_t h = rp.rot / 2;
    const int32_t pos = gptr<int32_t>(rp.positions)[token];
    if (pos < 0 || (uint32_t)pos >= rp.table_positions) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (d0 + i < rp.rot) x[i] = __builtin_nanf("");
        return;
    }
    const float* t = rp.table + (size_t)pos * rp.rot;
    if (rp.half && h % 8 == 0) {
        const bool first = d0 < h;
        float y[8];
        load8(r, row + (first ? d0 + h : d0 - h), y);
        norm.apply(first ? d0 + h : d0 - h, y);
        const f32x4* cs = reinterpret_cast<const f32x4*>(t + 2 * (first ? d0 : d0 - h));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f32x4 w = *gptr<f32x4>(cs + i);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int e = 2 * i + j;
                const float c = w[2 * j], s = w[2 * j + 1];
                // first half: a c - b s with b the partner; second: a s + b c with a the partner
                x[e] = first ? x[e] * c - y[e] * s : y[e] * s + x[e] * c;
            }
        }
    } else if (!rp.half && rp.rot % 8 == 0) {
        const f32x4* cs = reinterpret_cast<const f32x4*>(t + d0);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const f32x4 w = *gptr<f32x4>(cs + i);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int e = 4 * i + 2 * j;
                const float a = x[e], b = x[e + 1], c = w[2 * j], s = w[2 * j + 1];
                x[e] = a * c - b * s;
                x[e + 1] = a * s + b * c;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t d = d0 + i;
            if (d >= rp.rot) continue;
            const uint32_t f = rp.half ? (d < h ? d : d - h) : d / 2;
            const bool first = rp.half ? d < h : d % 2 == 0;
            const uint32_t e = rp.half ? (first ? d + h : d - h) : (d ^ 1u);
            const float y = norm.one(e, load1(r, row + e));
            const float c = gptr<float>(t)[2 * f], s = gptr<float>(t)[2 * f + 1], a = x[i];
            x[i] = first ? a * c - y * s : y * s + a * c;
        }
    }
}

// Four elements from element offset `at`, a multiple of four.
__device__ __forceinline__ void load4(const KvRows& r, int64_t at, float (&x)[4]) {
    if (r.bf16 && r.vec) {
        const u32x2 w = *gptr<u32x2>(static_cast<const uint16_t*>(r.p) + at);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    } else if (r.vec) {
        const f32x4 w = *gptr<f32x4>(static_cast<const float*>(r.p) + at);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = load1(r, at + i);
    }
}
__device__ __forceinline__ void store4(const KvRows& r, int64_t at, const float (&x)[4]) {
    if (r.bf16) {
        const u32x2 w = {f32x2_to_bf16x2_bits(x[0], x[1]), f32x2_to_bf16x2_bits(x[2], x[3])};
        uint16_t* p = static_cast<uint16_t*>(r.p) + at;
        if (r.vec) {
            *gptr_mut<u32x2>(p) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) gptr_mut<uint16_t>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    } else {
        float* p = static_cast<float*>(r.p) + at;
        if (r.vec) {
            *gptr_mut<f32x4>(p) = f32x4{x[0], x[1], x[2], x[3]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) gptr_mut<float>(p)[i] = x[i];
        }
    }
}

// One head of one token: loads, rotates, stores.  Halves of whole fours: a lane takes four
// pairs (with eight dims of one half it loads their partners as well and twice the cosines:
// append over 4 x 2048 tokens 36.0 us instead of 30.7, one token 2.2 instead of 1.8).  Otherwise
// in place is safe as well: a head's lanes are one wave's, which has loaded all of it before its
// first store.
template <int D>
__device__ __forceinline__ void rope_row(const KvRows& x, const KvRows& y, uint32_t token, uint32_t head, uint32_t lane,
                                         const RopeView& rp) {
    const uint32_t d0 = 8 * lane;
    const int64_t row = (int64_t)token * x.ts + (int64_t)head * x.hs;
    if (rp.half && rp.rot % 8 == 0 && d0 < rp.rot) {
        const int64_t to = (int64_t)token * y.ts + (int64_t)head * y.hs;
        const uint32_t i0 = 4 * lane, i1 = i0 + rp.rot / 2;
        const int32_t pos = gptr<int32_t>(rp.positions)[token];
        float a[4], b[4], p[4], q[4];
        load4(x, row + i0, a);
        load4(x, row + i1, b);
        const bool in = pos >= 0 && (uint32_t)pos < rp.table_positions;
        f32x4 cs[2] = {};
        if (in) {
            const float* t = rp.table + (size_t)pos * rp.rot + 2 * i0;
            cs[0] = *gptr<f32x4>(t);
            cs[1] = *gptr<f32x4>(t + 4);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const f32x4 w = cs[i];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int e = 2 * i + j;
                const float c = w[2 * j], s = w[2 * j + 1];
                p[e] = in ? a[e] * c - b[e] * s : __builtin_nanf("");
                q[e] = in ? a[e] * s + b[e] * c : __builtin_nanf("");
            }
        }
        store4(y, to + i0, p);
        store4(y, to + i1, q);
        return;
    }
    float v[8];
    if (d0 < D) {
        load8(x, row + d0, v);
        rotate8(x, row, token, d0, rp, NoNorm(), v);
    }
    __builtin_amdgcn_wave_barrier();
    if (d0 < D) store8(y, (int64_t)token * y.ts + (int64_t)head * y.hs + d0, v);
}

// The same with the head's norm before the rotation.  A function of its own: sharing one, the rotation alone loaded
// its cosines behind the rows instead of beside them (append over 4 x 2048 tokens and reading back 53.5 us
// instead of 50.5).
template <int D>
__device__ __forceinline__ void norm_rope_row(const KvRows& x, const KvRows& y, uint32_t token, uint32_t head, uint32_t lane,
                                              const RopeView& rp, const NormView& nv) {
    const uint32_t d0 = 8 * lane;
    const int64_t row = (int64_t)token * x.ts + (int64_t)head * x.hs;
    const int64_t to = (int64_t)token * y.ts + (int64_t)head * y.hs;
    const bool pairs = rp.half && rp.rot % 8 == 0 && d0 < rp.rot;
    const uint32_t i0 = 4 * lane, i1 = i0 + rp.rot / 2;
    float v[8] = {};  // eight dims, or four pairs: first all of the one side
    if (pairs) {
        float a[4], b[4];
        load4(x, row + i0, a);
        load4(x, row + i1, b);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = a[i], v[4 + i] = b[i];
    } else if (d0 < D) {
        load8(x, row + d0, v);
    }
    const HeadNorm norm = head_norm<D>(nv, v);
    if (pairs) {
        const int32_t pos = gptr<int32_t>(rp.positions)[token];
        float a[4], b[4], p[4], q[4];
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = v[i], b[i] = v[4 + i];
        const bool in = pos >= 0 && (uint32_t)pos < rp.table_positions;
        f32x4 cs[2] = {};
        if (in) {
            const float* t = rp.table + (size_t)pos * rp.rot + 2 * i0;
            cs[0] = *gptr<f32x4>(t);
            cs[1] = *gptr<f32x4>(t + 4);
        }
        norm.apply(i0, a);
        norm.apply(i1, b);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const f32x4 w = cs[i];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int e = 2 * i + j;
                const float c = w[2 * j], s = w[2 * j + 1];
                p[e] = in ? a[e] * c - b[e] * s : __builtin_nanf("");
                q[e] = in ? a[e] * s + b[e] * c : __builtin_nanf("");
            }
        }
        store4(y, to + i0, p);
        store4(y, to + i1, q);
        return;
    }
    if (d0 < D) {
        norm.apply(d0, v);
        rotate8(x, row, token, d0, rp, norm, v);
    }
    __builtin_amdgcn_wave_barrier();
    if (d0 < D) store8(y, to + d0, v);
}

// 4099 tokens of 40 heads of 128 dims in f32: 28.9 us, 6.0 TB/s; one token 1.8 us.  (Four
// heads of a token by a thread, which share its cosines: 29.4 and 3.7.)
template <int D>
__global__ __launch_bounds__(256) void rope_kernel(KvRows x, KvRows y, uint32_t tokens, uint32_t heads, RopeView rp) {
    constexpr uint32_t L = kLanes<D>;
    const uint64_t i = (uint64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (i >= (uint64_t)tokens * heads) return;
    rope_row<D>(x, y, (uint32_t)(i / heads), (uint32_t)(i % heads), threadIdx.x % L, rp);
}

// Queries in the first q_blocks workgroups, then keys.  A head is read once: its squares are
// summed over its lanes, and the rotation takes the products from registers.
template <int D>
__global__ __launch_bounds__(256) void norm_rope_kernel(KvRows q, KvRows q_out, uint32_t q_heads, NormView q_norm, KvRows k,
                                                        KvRows k_out, uint32_t k_heads, NormView k_norm, uint32_t tokens,
                                                        uint32_t q_blocks, RopeView rp) {
    constexpr uint32_t L = kLanes<D>;
    const bool keys = blockIdx.x >= q_blocks;
    const uint32_t heads = keys ? k_heads : q_heads;
    const uint64_t i = (uint64_t)(blockIdx.x - (keys ? q_blocks : 0u)) * (256 / L) + threadIdx.x / L;
    if (i >= (uint64_t)tokens * heads) return;
    const uint32_t token = (uint32_t)(i / heads), head = (uint32_t)(i % heads), lane = threadIdx.x % L;
    const KvRows x = keys ? k : q, y = keys ? k_out : q_out;
    const NormView n = keys ? k_norm : q_norm;
    if (n.on)
        norm_rope_row<D>(x, y, token, head, lane, rp, n);
    else
        rope_row<D>(x, y, token, head, lane, rp);
}

// The same where every row and weight begins at 16 bytes and rot is whole eights (or none): a lane takes two
// groups of four dims, four pairs of halves or eight in a row, and the eight floats of the table that
// belong to them are at 8 lane in both layouts.  Bound by memory: two bytes of traffic for each byte of a row
// and about forty operations for eight elements.  All loads are issued before the first is used, and the
// types are the kernel's: 8191 tokens of 40 heads of 128 dims take in bf16 40 us (172 MB, 4.3 TB/s; 33 where two calls
// take turns and the last cache holds a part of their rows), in f32 61 (340 MB, 5.6); through the general form, whose loads
// wait for each other's branches (the rows' for their layout, the cosines' for the sum), 64 and 70.
template <int D, bool BF16, bool WBF16>
__global__ __launch_bounds__(256) void norm_rope_wide_kernel(KvRows q, KvRows q_out, uint32_t q_heads, NormView q_norm, KvRows k,
                                                             KvRows k_out, uint32_t k_heads, NormView k_norm, uint32_t tokens,
                                                             uint32_t q_blocks, RopeView rp) {
    constexpr uint32_t L = kLanes<D>;
    const bool keys = blockIdx.x >= q_blocks;
    const uint32_t heads = keys ? k_heads : q_heads, lane = threadIdx.x % L, d0 = 8 * lane;
    const uint32_t i = (blockIdx.x - (keys ? q_blocks : 0u)) * (256 / L) + threadIdx.x / L;  // below 2^32: of a launch's threads
    const uint32_t token = i / heads, head = i - token * heads;
    if (token >= tokens) return;
    const KvRows x = keys ? k : q, y = keys ? k_out : q_out;
    const NormView n = keys ? k_norm : q_norm;
    const int32_t pos = rp.rot ? gptr<int32_t>(rp.positions)[token] : 0;
    const bool turned = d0 < rp.rot, pairs = turned && rp.half;
    const uint32_t i0 = pairs ? 4 * lane : d0 < D ? d0 : 0u, i1 = pairs ? 4 * lane + rp.rot / 2 : i0 + 4;
    const int64_t from = (int64_t)token * x.ts + (int64_t)head * x.hs, to = (int64_t)token * y.ts + (int64_t)head * y.hs;
    typedef std::conditional_t<BF16, u32x2, f32x4> X;
    typedef std::conditional_t<WBF16, u32x2, f32x4> WT;
    constexpr uint32_t E = BF16 ? 2 : 4, WE = WBF16 ? 2 : 4;
    const X xa = *gptr<X>(static_cast<const char*>(x.p) + (from + i0) * E), xb = *gptr<X>(static_cast<const char*>(x.p) + (from + i1) * E);
    const WT wa = *gptr<WT>(static_cast<const char*>(n.weight) + i0 * WE), wb = *gptr<WT>(static_cast<const char*>(n.weight) + i1 * WE);
    const bool in = pos >= 0 && (uint32_t)pos < rp.table_positions;
    f32x4 c0 = {}, c1 = {};
    if (turned && in) {
        const float* t = rp.table + (size_t)pos * rp.rot + 8 * lane;
        c0 = *gptr<f32x4>(t);
        c1 = *gptr<f32x4>(t + 4);
    }
    auto four = [](auto v, float (&f)[4]) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (sizeof(v) == 8)
                f[j] = __uint_as_float(j & 1 ? v[j / 2] & 0xFFFF0000u : v[j / 2] << 16);
            else
                f[j] = v[j];
        }
    };
    float a[4], b[4], u[4], v[4];
    four(xa, a), four(xb, b), four(wa, u), four(wb, v);
    float all[8];
#pragma unroll
    for (int j = 0; j < 4; j++) all[j] = d0 < D ? a[j] : 0.0f, all[4 + j] = d0 < D ? b[j] : 0.0f;
    const HeadNorm norm = head_norm<D>(n, all);
#pragma unroll
    for (int j = 0; j < 4; j++) a[j] = a[j] * norm.f * norm.r * (u[j] + n.offset), b[j] = b[j] * norm.f * norm.r * (v[j] + n.offset);
    if (turned) {
        float p[4], r[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            // halves: pair j is (a[j], b[j]); otherwise pairs 0, 1 are a's and 2, 3 b's
            const float c = j < 2 ? c0[2 * j] : c1[2 * j - 4], s = j < 2 ? c0[2 * j + 1] : c1[2 * j - 3];
            const float g = rp.half ? a[j] : j < 2 ? a[2 * j] : b[2 * j - 4], h = rp.half ? b[j] : j < 2 ? a[2 * j + 1] : b[2 * j - 3];
            p[j] = in ? g * c - h * s : __builtin_nanf("");
            r[j] = in ? g * s + h * c : __builtin_nanf("");
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            a[j] = rp.half ? p[j] : j & 1 ? r[j / 2] : p[j / 2];
            b[j] = rp.half ? r[j] : j & 1 ? r[2 + j / 2] : p[2 + j / 2];
        }
    }
    if (d0 >= D) return;
    auto store = [&](uint32_t at, const float (&f)[4]) {
        X z;
        if constexpr (BF16)
            z = u32x2{f32x2_to_bf16x2_bits(f[0], f[1]), f32x2_to_bf16x2_bits(f[2], f[3])};
        else
            z = f32x4{f[0], f[1], f[2], f[3]};
        *gptr_mut<X>(static_cast<char*>(y.p) + (to + at) * E) = z;
    };
    store(i0, a);
    store(i1, b);
}

// Largest of the N lanes around this one (N a power of two, aligned), by moves
// within rows of 16 lanes.
template <int N>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, true));   // lane ^ 1
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, true));   // lane ^ 2
    if (N > 4) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, true));  // mirrored in 8
    if (N > 8) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xF, 0xF, true));  // mirrored in 16
    if (N > 16) x = max(x, (uint32_t)__shfl_xor((int)x, 16));
    return x;
}

// A block's scale and this lane's eight codes of it.  N lanes hold the block;
// a lane without dims passes zeros.  Magnitudes are compared as the whole numbers
// their bits are, which puts infinities and NaN on top.
template <int BITS, int N>
__device__ __forceinline__ uint16_t quantize(const float (&x)[8], int32_t (&c)[8]) {
    uint32_t top = 0, low = 0;  // of the positive and of the negative values (8 bits: of all)
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t u = __float_as_uint(x[i]);
        if (BITS == 8) {
            top = max(top, u & 0x7FFFFFFFu);
        } else {
            top = max(top, u >> 31 ? 0u : u);
            low = max(low, u >> 31 ? u & 0x7FFFFFFFu : 0u);
        }
    }
    top = lanes_max<N>(top);
    if (BITS == 4) low = lanes_max<N>(low);
    if (max(top, low) >= 0x7F800000u) {  // an infinity or a NaN: the block reads back as NaN
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = 0;
        return 0x7FC0u;
    }
    const float d = BITS == 8 ? __uint_as_float(top) / 127.0f
                              : (top > low ? __uint_as_float(top) : -__uint_as_float(low)) / -8.0f;
    const uint16_t bits = f32_to_bf16_bits(d);
    const float s = bf16_bits_to_f32(bits);
    // x / s, correctly rounded: with r the correctly rounded reciprocal, one step from
    // x r is (Markstein), as long as nothing leaves the range of normal numbers
    const bool plain = fabsf(s) >= 0x1p-100f && fabsf(s) <= 0x1p100f;
    const float r = 1.0f / (plain ? s : 1.0f);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float q = x[i] * r;
        q = __builtin_fmaf(__builtin_fmaf(-q, s, x[i]), r, q);
        if (!plain) q = s == 0.0f ? 0.0f : x[i] / s;
        // the rounded scale may be a little small: the largest code is clamped
        c[i] = (int32_t)fminf(fmaxf(rintf(q), BITS == 8 ? -127.0f : -8.0f), BITS == 8 ? 127.0f : 7.0f);
    }
    return bits;
}

// Place of block b, part t of a K row, in codes.
template <int D>
__device__ __forceinline__ uint32_t k_place(uint32_t b, uint32_t t) {
    return (b / 2) * 64 + ((b | 1u) * 32 < D ? t * 16 + (b & 1) * 8 : t * 8);
}

// A workgroup of the append and read kernels takes a chunk of 16 positions of
// some heads; a thread has 8 dims of 4 of its tokens, whose loads are in flight
// together.  For values, which lie [dim][token], that is one dword a dim (8 bits),
// turned in registers: through LDS, byte by byte, 8 x 16k tokens of 8 heads took
// 192 us to read, with 4 heads a workgroup 282, this way 133 (a copy of their bytes: 140).
template <int D>
constexpr uint32_t kHeads = 64 / kLanes<D>;
template <int D>
constexpr uint32_t kKeyHeads = kLanes<D> == 8 ? 2 : 1;  // of the append's keys

struct Chunk {
    SeqRange r;
    uint64_t pos0;      // of its token 0
    int64_t page;       // -1: absent
    uint64_t slot;      // of this thread's head and token 0
    uint32_t c, h;      // chunk, head
    uint32_t lo, hi;    // tokens lo..hi-1 are the call's
    bool live;          // the head exists

    __device__ __forceinline__ uint32_t row(uint32_t t) const { return r.row0 + (uint32_t)(pos0 + t - r.len); }
    __device__ __forceinline__ bool has(uint32_t t) const { return live && t >= lo && t < hi; }
    // a token of the call near t, for loads that need not be switched off
    __device__ __forceinline__ uint32_t near(uint32_t t) const { return min(max(t, lo), hi - 1); }
};

// Workgroup blk of (sequence, chunk, HEADS heads), its head number `which`; false:
// nothing of the call is there.
template <uint32_t HEADS>
__device__ __forceinline__ bool find_chunk(const KvView& kv, const KvBatch& b, uint32_t blk, uint32_t chunks, uint32_t which,
                                           Chunk& c) {
    const uint32_t groups = (kv.heads + HEADS - 1) / HEADS;
    c.h = blk % groups * HEADS + which;
    c.live = c.h < kv.heads;
    const uint32_t rest = blk / groups, seq = rest / chunks;
    c.r = seq_range(b, seq);
    c.c = c.r.len / 16 + rest % chunks;
    c.pos0 = 16ull * c.c;
    if (c.r.n == 0 || c.pos0 >= (uint64_t)c.r.len + c.r.n) return false;
    c.lo = c.r.len > c.pos0 ? (uint32_t)(c.r.len - c.pos0) : 0u;
    c.hi = (uint32_t)min((uint64_t)16, (uint64_t)c.r.len + c.r.n - c.pos0);
    c.page = chunk_page(kv, b, seq, c.c);
    c.slot = c.page < 0 ? 0 : chunk_slot(kv, c.page, c.live ? c.h : 0, c.c);
    return true;
}

// Bytes i of four dwords as one dword each: x[j] byte i -> x[i] byte j.
__device__ __forceinline__ void turn4(uint32_t (&x)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
    x[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    x[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    x[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    x[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Grid: `k_blocks` workgroups for the keys, one per (sequence, chunk, 256 / lanes
// of a row / 16 heads), a thread 8 dims of one token; `v_blocks` for the values,
// one per (sequence, chunk, kHeads heads); then the queries' rows.  A chunk of a
// head's values is one wave's alone, so values of 4 bits, two tokens to a byte, are
// merged without atomics.  (Keys by four tokens a thread: 220 registers, the whole
// launch over 4 x 2048 tokens, 146 MB in 30.7 us, 4.8 TB/s now, 86 us instead of 37 then.)
// NORM: keys and queries by their norms first.
template <int D, int KB, int VB, bool NORM>
__global__ __launch_bounds__(256) void append_kernel(KvView kv, KvBatch b, KvRows k, NormView k_norm, KvRows v, RopeView rp,
                                                     KvRows q, NormView q_norm, KvRows q_out, uint32_t q_heads,
                                                     uint32_t chunks, uint32_t k_blocks, uint32_t v_blocks) {
    constexpr uint32_t L = kLanes<D>, ROWS = 256 / L;
    const uint32_t lane = threadIdx.x % L, d0 = 8 * lane;
    uint32_t blk = blockIdx.x;
    if (blk >= k_blocks + v_blocks) {
        const uint64_t i = (uint64_t)(blk - k_blocks - v_blocks) * ROWS + threadIdx.x / L;
        if (i >= (uint64_t)b.tokens * q_heads) return;
        const uint32_t token = (uint32_t)(i / q_heads), head = (uint32_t)(i % q_heads);
        if (NORM && q_norm.on)
            norm_rope_row<D>(q, q_out, token, head, lane, rp, q_norm);
        else
            rope_row<D>(q, q_out, token, head, lane, rp);
        return;
    }
    Chunk c;
    if (blk < k_blocks) {
        constexpr uint32_t HEADS = kKeyHeads<D>;
        if (!find_chunk<HEADS>(kv, b, blk, chunks, threadIdx.x / L / 16, c) || c.page < 0) return;
        for (uint32_t t = threadIdx.x / L % 16; t < 16; t += ROWS) {
            if (!c.has(t)) continue;  // whole rows leave together: the shuffles stay within a row
            const uint32_t token = c.row(t);
            const int64_t row = (int64_t)token * k.ts + (int64_t)c.h * k.hs;
            float x[8] = {};
            if (NORM && k_norm.on) {
                if (d0 < D) load8(k, row + d0, x);
                const HeadNorm norm = head_norm<D>(k_norm, x);
                if (d0 < D) {
                    norm.apply(d0, x);
                    if (rp.table) rotate8(k, row, token, d0, rp, norm, x);
                }
            } else if (d0 < D) {
                load8(k, row + d0, x);
                if (rp.table) rotate8(k, row, token, d0, rp, NoNorm(), x);
            }
            int32_t code[8];
            const uint16_t sc = quantize<KB, 4>(x, code);
            if (d0 >= D) continue;
            const uint32_t blk32 = lane / 4, part = lane % 4, in_row = k_place<D>(blk32, part);
            const uint64_t at = c.slot + t;
            if constexpr (KB == 8) {
                u32x2 w = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; j++) w[j / 4] |= (uint32_t)(code[j] + 128) << (8 * (j % 4));
                *gptr_mut<u32x2>(kv.k + at * D + in_row) = w;
            } else {
                uint32_t w = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) w |= (uint32_t)(code[j] + 8) << (8 * (j % 4) + 4 * (j / 4));
                *gptr_mut<uint32_t>(kv.k + at * (D / 2) + in_row / 2) = w;
            }
            if (part == 0) gptr_mut<uint16_t>(kv.k + kv.k_scales)[at * (D / 32) + blk32] = sc;
        }
        return;
    }
    const uint32_t which = threadIdx.x / L, quad = which % 4, t0 = 4 * quad;
    if (!find_chunk<kHeads<D>>(kv, b, blk - k_blocks, chunks, which / 4, c) || c.page < 0) return;
    float x[4][8] = {};
    if (d0 < D) {
#pragma unroll
        for (uint32_t t = 0; t < 4; t++)
            load8(v, (int64_t)c.row(c.near(t0 + t)) * v.ts + (int64_t)(c.live ? c.h : 0) * v.hs + d0, x[t]);
    }
    int32_t code[4][8];
    uint16_t sc[4];
    uint32_t mask = 0;  // bytes of the tokens that are the call's
#pragma unroll
    for (uint32_t t = 0; t < 4; t++) {
        sc[t] = quantize<VB, (int)L>(x[t], code[t]);
        if (!c.has(t0 + t)) continue;
        mask |= 255u << (8 * t);
        if (lane == 0) gptr_mut<uint16_t>(kv.v + kv.v_scales)[c.slot + t0 + t] = sc[t];
    }
    if constexpr (VB == 8) {
        if (d0 >= D) return;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t w = (code[0][j] & 255u) | (code[1][j] & 255u) << 8 | (code[2][j] & 255u) << 16 | (uint32_t)code[3][j] << 24;
            uint8_t* dst = kv.v + c.slot * D + (d0 + j) * 16 + t0;
            if (mask == ~0u) {
                *gptr_mut<uint32_t>(dst) = w;
            } else {
#pragma unroll
                for (uint32_t t = 0; t < 4; t++)
                    if (mask >> (8 * t) & 1u) gptr_mut<uint8_t>(dst)[t] = (uint8_t)(w >> (8 * t));
            }
        }
    } else {
        // even quads take the low nibbles of a dword, odd ones, L lanes on, the high
        // ones; the even quad's lane writes both
        const uint32_t other = __shfl_xor((int)mask, (int)L);
        const uint32_t all = (mask & 0x0F0F0F0Fu) | (other & 0xF0F0F0F0u);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t w = (code[0][j] & 15u) | (code[1][j] & 15u) << 8 | (code[2][j] & 15u) << 16 | (code[3][j] & 15u) << 24;
            const uint32_t hi = __shfl_xor((int)w, (int)L);
            if (d0 >= D || quad % 2 || all == 0) continue;
            uint32_t* dst = reinterpret_cast<uint32_t*>(kv.v + c.slot * (D / 2) + (d0 + j) * 8 + t0 / 2);
            uint32_t y = w | hi << 4;
            if (all != ~0u) y = (y & all) | (*gptr<uint32_t>(dst) & ~all);
            *gptr_mut<uint32_t>(dst) = y;
        }
    }
}

// One workgroup per (sequence, chunk, kHeads heads), keys then values.  8 x 16k tokens of
// 8 heads of 128 dims, 8 bits to bf16: 133 us, 5.2 TB/s, two thirds of it writes.
template <int D, int KB, int VB>
__global__ __launch_bounds__(256) void read_kernel(KvView kv, KvBatch b, KvRows k, KvRows v, uint32_t chunks,
                                                   uint32_t kv_blocks) {
    constexpr uint32_t L = kLanes<D>;
    const uint32_t lane = threadIdx.x % L, d0 = 8 * lane;
    uint32_t blk = blockIdx.x;
    const bool keys = k.p != nullptr && blk < kv_blocks;
    if (k.p != nullptr && !keys) blk -= kv_blocks;
    const uint32_t which = threadIdx.x / L, quad = which % 4, t0 = 4 * quad;
    Chunk c;
    if (!find_chunk<kHeads<D>>(kv, b, blk, chunks, which / 4, c) || d0 >= D || !c.live) return;
    float x[4][8], s[4];
    if (c.page < 0) {
#pragma unroll
        for (uint32_t t = 0; t < 4; t++)
#pragma unroll
            for (int j = 0; j < 8; j++) x[t][j] = __builtin_nanf("");
    } else if (keys) {
        const uint32_t at = k_place<D>(lane / 4, lane % 4);
        uint32_t w[4][KB / 4];
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) {
            const uint64_t row = c.slot + t0 + t;
            s[t] = bf16_bits_to_f32(gptr<uint16_t>(kv.k + kv.k_scales)[row * (D / 32) + lane / 4]);
            if constexpr (KB == 8) {
                const u32x2 y = *gptr<u32x2>(kv.k + row * D + at);
                w[t][0] = y.x, w[t][1] = y.y;
            } else {
                w[t][0] = *gptr<uint32_t>(kv.k + row * (D / 2) + at / 2);
            }
        }
#pragma unroll
        for (uint32_t t = 0; t < 4; t++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int32_t code = KB == 8 ? (int32_t)((w[t][j / 4 % (KB / 4)] >> (8 * (j % 4))) & 255u) - 128
                                             : (int32_t)((w[t][0] >> (8 * (j % 4) + 4 * (j / 4))) & 15u) - 8;
                x[t][j] = (float)code * s[t];
            }
    } else {
        uint32_t w[2][4];  // [half of the dims][dim]: four tokens each
#pragma unroll
        for (int j = 0; j < 8; j++)
            w[j / 4][j % 4] = VB == 8 ? *gptr<uint32_t>(kv.v + c.slot * D + (d0 + j) * 16 + t0)
                                      : *gptr<uint32_t>(kv.v + c.slot * (D / 2) + (d0 + j) * 8 + 4 * (quad / 2));
        const u32x2 sw = *gptr<u32x2>(kv.v + kv.v_scales + 2 * (c.slot + t0));
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) s[t] = bf16_bits_to_f32(sw[t / 2] >> (16 * (t % 2)) & 0xFFFFu);
        if constexpr (VB == 4) {
#pragma unroll
            for (int j = 0; j < 8; j++) {  // nibble n (signed) as a byte: bit 3 set, bits 4..7 too
                const uint32_t n = (w[j / 4][j % 4] >> (4 * (quad % 2))) & 0x0F0F0F0Fu;
                w[j / 4][j % 4] = n | ((n & 0x08080808u) * 30u);
            }
        }
        turn4(w[0]);
        turn4(w[1]);
#pragma unroll
        for (uint32_t t = 0; t < 4; t++)
#pragma unroll
            for (int j = 0; j < 8; j++) x[t][j] = (float)(int8_t)(w[j / 4][t] >> (8 * (j % 4))) * s[t];
    }
    const KvRows& o = keys ? k : v;
#pragma unroll
    for (uint32_t t = 0; t < 4; t++)
        if (c.has(t0 + t)) store8(o, (int64_t)c.row(t0 + t) * o.ts + (int64_t)c.h * o.hs + d0, x[t]);
}

// One workgroup per (sequence, head, keys or values).  A thread owns the same
// bytes of every row (a dword of a key, a dim of a value), so its moves are in
// order by themselves: a row's source lies at or after every row written so far.
// Latency, some four dependent loads a move, one move after another: 7.6 us for 16 paths out of trees of 24,
// 9.0 for 16 paths of ten, 43 for 16 of 64.
template <int D, int KB, int VB>
__global__ __launch_bounds__(256) void commit_kernel(KvView kv, KvBatch b, const int32_t* path, uint32_t path_stride,
                                                     const int32_t* counts) {
    const uint32_t head = blockIdx.x % kv.heads, seq = blockIdx.x / kv.heads % b.seqs;
    const bool keys = blockIdx.x < kv.heads * b.seqs;
    const SeqRange r = seq_range(b, seq);
    const int32_t cn = counts[seq];
    const uint32_t n = cn < 0 ? 0u : min((uint32_t)cn, min(r.n, path_stride));
    const uint32_t i = threadIdx.x;
    for (uint32_t j = 0; j < n; j++) {
        const int32_t from = path[(size_t)seq * path_stride + j];
        if (from <= (int32_t)j || (uint32_t)from >= r.n) continue;
        const uint64_t ps = (uint64_t)r.len + (uint32_t)from, pd = (uint64_t)r.len + j;
        const uint32_t cs = (uint32_t)(ps / 16), cd = (uint32_t)(pd / 16);
        const int64_t gs = chunk_page(kv, b, seq, cs), gd = chunk_page(kv, b, seq, cd);
        if (gs < 0 || gd < 0) continue;
        const uint64_t ss = chunk_slot(kv, gs, head, cs), sd = chunk_slot(kv, gd, head, cd);
        const uint32_t ts = ps % 16, td = pd % 16;
        if (keys) {
            constexpr uint32_t RB = D * KB / 8, NS = D / 32;
            if (i < RB / 4)
                *gptr_mut<uint32_t>(kv.k + (sd + td) * RB + 4 * i) = *gptr<uint32_t>(kv.k + (ss + ts) * RB + 4 * i);
            else if (i >= 128 && i < 128 + NS) {
                uint16_t* sc = reinterpret_cast<uint16_t*>(kv.k + kv.k_scales);
                gptr_mut<uint16_t>(sc)[(sd + td) * NS + i - 128] = gptr<uint16_t>(sc)[(ss + ts) * NS + i - 128];
            }
        } else {
            if (i < D) {
                if constexpr (VB == 8) {
                    gptr_mut<uint8_t>(kv.v)[sd * D + i * 16 + td] = gptr<uint8_t>(kv.v)[ss * D + i * 16 + ts];
                } else {
                    const uint32_t from_b = gptr<uint8_t>(kv.v)[ss * (D / 2) + i * 8 + ts / 8 * 4 + ts % 4];
                    const uint64_t at = sd * (D / 2) + i * 8 + td / 8 * 4 + td % 4;
                    const uint32_t sh = td % 8 / 4 * 4, nib = (from_b >> (ts % 8 / 4 * 4)) & 15u;
                    const uint32_t old = gptr<uint8_t>(kv.v)[at];
                    gptr_mut<uint8_t>(kv.v)[at] = (uint8_t)((old & ~(15u << sh)) | (nib << sh));
                }
            }
            if (i == 0) {
                uint16_t* sc = reinterpret_cast<uint16_t*>(kv.v + kv.v_scales);
                gptr_mut<uint16_t>(sc)[sd + td] = gptr<uint16_t>(sc)[ss + ts];
            }
        }
    }
}

// Angles in 64 bits: the frequency of a pair, times the position, and one
// rounding of the cosine and sine.
__global__ __launch_bounds__(256) void rope_table_kernel(uint32_t rot, uint32_t scaling, double theta, double factor,
                                                         double original, double lo, double hi, double attn,
                                                         uint32_t positions, float* out) {
    const uint32_t h = rot / 2;
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (uint64_t)positions * h) return;
    const uint32_t f = (uint32_t)(i % h);
    double w = pow(theta, -2.0 * f / rot);
    if (scaling == 1) {
        w /= factor;
    } else if (scaling == 2) {  // lo, hi: the pairs between which the scaling sets in
        const double ramp = fmin(fmax((f - lo) / fmax(hi - lo, 0.001), 0.0), 1.0);
        w = w / factor * ramp + w * (1.0 - ramp);
    } else if (scaling == 3) {  // lo, hi: turns over the original length
        const double turns = original * w / 6.283185307179586476925;
        const double s = fmin(fmax((turns - lo) / (hi - lo), 0.0), 1.0);
        w = (1.0 - s) * w / factor + s * w;
    }
    const double a = w * (double)(i / h);
    out[2 * i] = (float)(cos(a) * attn);
    out[2 * i + 1] = (float)(sin(a) * attn);
}

uint32_t chunk_bound(uint32_t max_new) { return max_new ? (max_new + 14u) / 16u + 1u : 0u; }

template <class F>
hipError_t by_dim(uint32_t dim, F f) {
    switch (dim) {
    case 64: return f(std::integral_constant<int, 64>());
    case 96: return f(std::integral_constant<int, 96>());
    case 128: return f(std::integral_constant<int, 128>());
    case 256: return f(std::integral_constant<int, 256>());
    }
    return hipErrorInvalidValue;
}

template <class F>
hipError_t by_cache(const KvView& kv, F f) {
    return by_dim(kv.dim, [&](auto d) {
        using A = std::integral_constant<int, 8>;
        using B = std::integral_constant<int, 4>;
        if (kv.k_bits == 8) return kv.v_bits == 8 ? f(d, A(), A()) : f(d, A(), B());
        return kv.v_bits == 8 ? f(d, B(), A()) : f(d, B(), B());
    });
}

}  // namespace

hipError_t rope_table_launch(uint32_t rot, uint32_t scaling, double theta, double factor, double original, double lo,
                             double hi, double attn, uint32_t positions, float* out, hipStream_t st) {
    const uint64_t n = (uint64_t)positions * (rot / 2);
    if (n == 0) return hipSuccess;
    if (!launchable((n + 255) / 256, 256)) return kTooManyThreads;
    rope_table_kernel<<<(uint32_t)((n + 255) / 256), 256, 0, st>>>(rot, scaling, theta, factor, original, lo, hi, attn,
                                                                   positions, out);
    return hipGetLastError();
}

hipError_t rope_launch(const KvRows& x, const KvRows& y, uint32_t tokens, uint32_t heads, uint32_t dim,
                       const RopeView& rope, hipStream_t st) {
    if (tokens == 0) return hipSuccess;
    return by_dim(dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        constexpr uint64_t rows = 256 / kLanes<D>;
        const uint64_t grid = ((uint64_t)tokens * heads + rows - 1) / rows;
        if (!launchable(grid, 256)) return kTooManyThreads;
        rope_kernel<D><<<(uint32_t)grid, 256, 0, st>>>(x, y, tokens, heads, rope);
        return hipGetLastError();
    });
}

hipError_t qk_norm_rope_launch(const KvRows& q, const KvRows& q_out, uint32_t q_heads, const NormView& q_norm,
                               const KvRows& k, const KvRows& k_out, uint32_t k_heads, const NormView& k_norm,
                               uint32_t tokens, uint32_t dim, const RopeView& rope, hipStream_t st) {
    if (tokens == 0) return hipSuccess;
    return by_dim(dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        constexpr uint64_t rows = 256 / kLanes<D>;
        const uint64_t q_blocks = ((uint64_t)tokens * q_heads + rows - 1) / rows;
        const uint64_t grid = q_blocks + ((uint64_t)tokens * k_heads + rows - 1) / rows;
        if (!launchable(grid, 256)) return kTooManyThreads;
        const bool both = k_heads != 0;
        const bool wide = q.vec && q_out.vec && q_norm.on && q_norm.weight && q_norm.vec && rope.rot % 8 == 0 &&
                          (!both || (k.vec && k_out.vec && k_norm.on && k_norm.weight && k_norm.vec && k.bf16 == q.bf16 &&
                                     k_norm.bf16 == q_norm.bf16));
        if (wide) {
            auto go = [&](auto io, auto wt) {
                norm_rope_wide_kernel<D, decltype(io)::value, decltype(wt)::value><<<(uint32_t)grid, 256, 0, st>>>(
                    q, q_out, q_heads, q_norm, k, k_out, k_heads, k_norm, tokens, (uint32_t)q_blocks, rope);
                return hipGetLastError();
            };
            using Y = std::true_type;
            using N = std::false_type;
            if (q.bf16) return q_norm.bf16 ? go(Y(), Y()) : go(Y(), N());
            return q_norm.bf16 ? go(N(), Y()) : go(N(), N());
        }
        norm_rope_kernel<D><<<(uint32_t)grid, 256, 0, st>>>(q, q_out, q_heads, q_norm, k, k_out, k_heads, k_norm, tokens,
                                                            (uint32_t)q_blocks, rope);
        return hipGetLastError();
    });
}

hipError_t kv_append_launch(const KvView& kv, const KvBatch& b, const KvRows& k, const NormView& k_norm, const KvRows& v,
                            const RopeView& rope, const KvRows& q, const NormView& q_norm, const KvRows& q_out,
                            uint32_t q_heads, hipStream_t st) {
    return by_cache(kv, [&](auto d, auto kb, auto vb) {
        constexpr int D = decltype(d)::value;
        constexpr uint64_t rows = 256 / kLanes<D>;
        const uint32_t chunks = chunk_bound(b.max_new);
        // below 2^64: at most 2^24 sequences, 2^27 + 1 chunks, 2^12 heads (values: half of them)
        const uint64_t k_blocks = (uint64_t)b.seqs * chunks * ((kv.heads + kKeyHeads<D> - 1) / kKeyHeads<D>);
        const uint64_t v_blocks = (uint64_t)b.seqs * chunks * ((kv.heads + kHeads<D> - 1) / kHeads<D>);
        const uint64_t grid = k_blocks + v_blocks + ((uint64_t)b.tokens * q_heads + rows - 1) / rows;
        if (grid == 0) return hipSuccess;
        if (!launchable(grid, 256)) return kTooManyThreads;
        auto go = [&](auto norm) {
            append_kernel<D, decltype(kb)::value, decltype(vb)::value, decltype(norm)::value><<<(uint32_t)grid, 256, 0, st>>>(
                kv, b, k, k_norm, v, rope, q, q_norm, q_out, q_heads, chunks, (uint32_t)k_blocks, (uint32_t)v_blocks);
            return hipGetLastError();
        };
        return k_norm.on || q_norm.on ? go(std::true_type()) : go(std::false_type());
    });
}

hipError_t kv_read_launch(const KvView& kv, const KvBatch& b, const KvRows& k, const KvRows& v, hipStream_t st) {
    return by_cache(kv, [&](auto d, auto kb, auto vb) {
        constexpr int D = decltype(d)::value;
        const uint32_t chunks = chunk_bound(b.max_new);
        const uint64_t kv_blocks = (uint64_t)b.seqs * chunks * ((kv.heads + kHeads<D> - 1) / kHeads<D>);
        const uint64_t grid = kv_blocks * ((k.p != nullptr) + (v.p != nullptr));
        if (grid == 0) return hipSuccess;
        if (!launchable(grid, 256)) return kTooManyThreads;
        read_kernel<D, decltype(kb)::value, decltype(vb)::value>
            <<<(uint32_t)grid, 256, 0, st>>>(kv, b, k, v, chunks, (uint32_t)kv_blocks);
        return hipGetLastError();
    });
}

hipError_t kv_commit_launch(const KvView& kv, const KvBatch& b, const int32_t* path, uint32_t path_stride,
                            const int32_t* counts, hipStream_t st) {
    return by_cache(kv, [&](auto d, auto kb, auto vb) {
        constexpr int D = decltype(d)::value;
        const uint64_t grid = 2ull * b.seqs * kv.heads;
        if (grid == 0) return hipSuccess;
        if (!launchable(grid, 256)) return kTooManyThreads;
        commit_kernel<D, decltype(kb)::value, decltype(vb)::value>
            <<<(uint32_t)grid, 256, 0, st>>>(kv, b, path, path_stride, counts);
        return hipGetLastError();
    });
}

}  // namespace dmx
