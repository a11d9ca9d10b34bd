// Log probabilities of given tokens, their ranks, the entropy and the likeliest
// alternatives of logits [rows, vocab].
//
//   t_i = (x_i - m) / T with m = max x,  S = sum e^t_i,  U = sum e^t_i t_i
//   log p_i = t_i - ln S,  entropy = ln S - U / S
//
// One pass: a workgroup holds a piece of a row in registers, so its maximum is
// known before the exponentials and every logit is read once; a second small
// launch joins a row's pieces.  Bound by the logits' bytes where rows are many
// (some eleven vector instructions a logit, the exponential counted as four,
// fill four fifths of the time the bytes take), by two launches where they are few.
//
// The order is that of (logit, lower token first), held as one 64-bit key: the
// float's bits as a whole number of the same order, and the token's complement.
// A piece's largest `top`: of its threads' largest logits a bound is found
// that `top` of them reach; what reaches it (few more than `top`, unless many
// logits tie) is gathered in LDS and each key finds its place by counting the larger ones.
#include "kvcache.hpp"

#include <type_traits>

namespace dmx {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / 64;
constexpr uint32_t kHeld = 32;                    // logits a thread holds
constexpr uint32_t kPiece = kThreads * kHeld;     // 8192
constexpr uint32_t kGathered = 512;               // keys that LDS has room for
constexpr float kInf = __builtin_inff();
constexpr float kMost = 3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Stats {
    float m, s, u;   // largest logit, S and U from it, exponents in powers of two
    uint32_t above;  // logits before the given token in the order
};

// A NaN counts as -inf, +inf as the largest f32, -0 as 0.
__device__ __forceinline__ float plain(float x) { return x == x ? fminf(x, kMost) + 0.0f : -kInf; }

// The next smaller f32 (of -inf itself).
__device__ __forceinline__ float next_below(float x) {
    const uint32_t u = __float_as_uint(x);
    return x == -kInf ? x : x == 0.0f ? -1.401298464e-45f : __uint_as_float(u >> 31 ? u + 1u : u - 1u);
}

__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return __uint_as_float(o >> 31 ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ u64 key_of(float x, uint32_t token) { return (u64)ordered(x) << 32 | (uint32_t)~token; }
constexpr uint32_t kNothing = 0x007FFFFFu;  // ordered(-inf): what is not above it is no alternative

// Of the temperature: the factor of logits in powers of two.  1 / T beyond what f32 exponents
// resolve counts as the nearest such factor.
__device__ __forceinline__ float factor(const float* temperature, uint32_t row) {
    if (!temperature) return kLog2e;
    const float t = temperature[row];
    if (t <= 0.0f) return -1.0f;  // all of the distribution at the largest logit
    const float c = kLog2e / t;
    return c != c ? c : fminf(fmaxf(c, 1e-36f), 1e36f);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// (x - m) c, not below what a product with 0 survives; also for x = m = -inf.
__device__ __forceinline__ float exponent(float x, float m, float c) { return fmaxf((x - m) * c, -1e38f); }

template <class F>
__device__ __forceinline__ float wave_all(float x, F f) {
#pragma unroll
    for (int d = 32; d; d /= 2) x = f(x, __shfl_xor(x, d));
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
    return wave_all(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
    return wave_all(x, [](float a, float b) { return a + b; });
}

struct TopLds {
    uint32_t most[kThreads];
    u64 keys[kGathered];
    u64 best[kWaves];
    uint32_t count;
};

// The `top` largest keys in out[0..top-1], descending, 0 where there are fewer.  `largest`: the
// largest of this thread's keys' high halves; each(f) calls f(key) for its keys, in the
// same order in all threads of a wave.  Keys are different and above kNothing's.
template <class E>
__device__ __forceinline__ void select_top(TopLds& l, uint32_t top, uint32_t largest, const E& each, u64* out) {
    const uint32_t lane = threadIdx.x & 63u;
    l.most[threadIdx.x] = largest;
    if (threadIdx.x == 0) l.count = 0;
    __syncthreads();
    // a bound that at least `top` threads reach, and at most twice as many if there is one
    uint32_t v[kWaves], hi = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; i++) v[i] = l.most[lane + 64 * i], hi = max(hi, v[i]);
#pragma unroll
    for (int d = 32; d; d /= 2) hi = max(hi, (uint32_t)__shfl_xor((int)hi, d));
    hi = __builtin_amdgcn_readfirstlane(hi);
    uint32_t lo = kNothing + 1;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        uint32_t n = 0;
#pragma unroll
        for (uint32_t i = 0; i < kWaves; i++) n += (uint32_t)__popcll(__ballot(v[i] >= mid));
        if (n >= top) {
            lo = mid;
            if (n <= 2 * top) break;
        } else {
            hi = mid - 1;
        }
    }
    each([&](u64 key) {
        const bool in = (uint32_t)(key >> 32) >= lo;
        const u64 mask = __ballot(in);
        if (!mask) return;
        uint32_t at = 0;
        if (lane == (uint32_t)__ffsll(mask) - 1u) at = atomicAdd(&l.count, (uint32_t)__popcll(mask));
        at = (uint32_t)__shfl((int)at, __ffsll(mask) - 1) + (uint32_t)__popcll(mask & ((1ull << lane) - 1ull));
        if (in && at < kGathered) l.keys[at] = key;
    });
    __syncthreads();
    const uint32_t n = l.count;
    if (n <= kGathered) {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const u64 key = l.keys[i];
            uint32_t place = 0;
            for (uint32_t j = 0; j < n; j++) place += l.keys[j] > key;
            if (place < top) out[place] = key;
        }
        for (uint32_t i = n + threadIdx.x; i < top; i += kThreads) out[i] = 0;
        return;
    }
    // too many (ties): one after another, each the largest below the one before
    u64 last = ~0ull;
    for (uint32_t i = 0; i < top; i++) {
        u64 best = 0;
        each([&](u64 key) {
            if ((uint32_t)(key >> 32) > kNothing && key < last && key > best) best = key;
        });
#pragma unroll
        for (int d = 32; d; d /= 2) {
            const u64 o = __shfl_xor(best, d);
            best = o > best ? o : best;
        }
        if (lane == 0) l.best[threadIdx.x / 64] = best;
        __syncthreads();
        best = l.best[0];
#pragma unroll
        for (uint32_t w = 1; w < kWaves; w++) best = l.best[w] > best ? l.best[w] : best;
        __syncthreads();
        if (threadIdx.x == 0) out[i] = best;
        last = best;  // 0: nothing is below it
    }
}

// Workgroup (row, piece).  Pieces are whole 16-byte units of memory: a row that does not begin
// at one has its first piece begin before the row, and the last may end behind it (units without
// a logit of the row are not read; what lies beside it in one is not looked at).
template <bool BF16, bool TOP>
__global__ __launch_bounds__(kThreads) void piece_kernel(LogprobArgs a, uint32_t pieces) {
    constexpr uint32_t U = BF16 ? 8 : 4, LOADS = kHeld / U;  // logits of a load
    __shared__ float part[3][kWaves];
    __shared__ uint32_t counts[kWaves];
    __shared__ std::conditional_t<TOP, TopLds, char> top;
    const uint32_t row = blockIdx.x / pieces, piece = blockIdx.x % pieces;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64;
    const uintptr_t base = reinterpret_cast<uintptr_t>(a.logits) + (uint64_t)((int64_t)row * a.stride) * (BF16 ? 2 : 4);
    const uint32_t shift = (uint32_t)(base & 15u) / (BF16 ? 2 : 4);
    const char* const src = reinterpret_cast<const char*>(base & ~(uintptr_t)15);
    // this thread's load j holds logits first + j * kThreads * U ..
    const int64_t first = (int64_t)piece * kPiece + threadIdx.x * U - shift;
    float x[kHeld];
    u32x4 w[LOADS];
#pragma unroll
    for (uint32_t j = 0; j < LOADS; j++) {
        const int64_t i = first + j * kThreads * U;
        const bool some = i < (int64_t)a.vocab;
        w[j] = some ? *gptr<u32x4>(src + 16 * ((uint64_t)piece * (kPiece / U) + j * kThreads + threadIdx.x)) : u32x4{};
    }
    const int64_t tok = a.tokens ? a.tokens[row] : -1;
    const bool given = tok >= 0 && tok < (int64_t)a.vocab;
    float xt = kInf;
    if (given) {
        const char* p = reinterpret_cast<const char*>(base) + tok * (BF16 ? 2 : 4);
        xt = plain(BF16 ? bf16_bits_to_f32(*gptr<uint16_t>(p)) : *gptr<float>(p));
    }
    const float c = factor(a.temperature, row);
    float most = -kInf;
#pragma unroll
    for (uint32_t j = 0; j < LOADS; j++) {
        const int64_t i = first + j * kThreads * U;
#pragma unroll
        for (uint32_t e = 0; e < U; e++)
            x[j * U + e] = BF16 ? __uint_as_float(e & 1u ? w[j][e / 2] & 0xFFFF0000u : w[j][e / 2] << 16) : __uint_as_float(w[j][e]);
        if (i < 0 || i + U > (int64_t)a.vocab) {  // the row's edges
#pragma unroll
            for (uint32_t e = 0; e < U; e++)
                if (i + (int64_t)e < 0 || i + (int64_t)e >= (int64_t)a.vocab) x[j * U + e] = -kInf;
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kHeld; i++) most = fmaxf(most, x[i]);  // of a NaN and a number the number
    float m = wave_max(most);
    if (lane == 0) part[0][wave] = m;
    __syncthreads();
    m = part[0][0];
#pragma unroll
    for (uint32_t i = 1; i < kWaves; i++) m = fmaxf(m, part[0][i]);
    if (m == kInf) {  // an infinity among them
#pragma unroll
        for (uint32_t i = 0; i < kHeld; i++) x[i] = plain(x[i]);
        most = plain(most);
        m = kMost;
    }
    float s = 0.0f, u = 0.0f;
    // one product a logit where nothing leaves f32: x c - M with M = m c rounded, which then
    // is taken off by what it was rounded by
    const float M = m * c, off = __builtin_fmaf(m, c, -M);
    if (c > 0.0f && fabsf(M) < 1e30f) {
#pragma unroll
        for (uint32_t i = 0; i < kHeld; i++) {
            const float t = fmaxf(__builtin_fmaf(x[i], c, -M), -1e38f), e = exp2_(t);
            s += e;
            u = __builtin_fmaf(e, t, u);
        }
        const float f = exp2_(-off);
        u = (u - off * s) * f;
        s *= f;
    } else if (c > 0.0f) {
#pragma unroll
        for (uint32_t i = 0; i < kHeld; i++) {
            const float t = exponent(x[i], m, c), e = exp2_(t);
            s += e;
            u += e * t;
        }
    }
    // before the token in the order: larger ones, and equal ones of lower tokens, which are
    // above the next smaller f32.  One comparison a logit, but for the load the token is in.
    uint32_t above = 0;
    if (given) {
        const float below = next_below(xt);
#pragma unroll
        for (uint32_t j = 0; j < LOADS; j++) {
            const int64_t i = first + j * kThreads * U;
            const float bound = i + U <= tok ? below : xt;
#pragma unroll
            for (uint32_t e = 0; e < U; e++) above += (uint32_t)__popcll(__ballot(x[j * U + e] > bound));
        }
        uint32_t more = 0;
        if (xt == -kInf) {  // nothing is below: all before it that are not above
#pragma unroll
            for (uint32_t j = 0; j < LOADS; j++) {
                const int64_t i = first + j * kThreads * U;
#pragma unroll
                for (uint32_t e = 0; e < U; e++)
                    more += !(x[j * U + e] > xt) && i + (int64_t)e >= 0 && i + (int64_t)e < tok;
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < LOADS; j++) {
                const int64_t i = first + j * kThreads * U;
                if (i <= tok && tok < i + U) {
#pragma unroll
                    for (uint32_t e = 0; e < U; e++) more += x[j * U + e] == xt && i + (int64_t)e < tok;
                }
            }
        }
        // the loads of the row's edges hold -inf where it has no logit, which is above nothing
        if (__ballot(more != 0)) above += (uint32_t)wave_sum((float)more);
    }
    s = wave_sum(s);
    u = wave_sum(u);
    if (lane == 0) part[1][wave] = s, part[2][wave] = u, counts[wave] = above;
    __syncthreads();
    if (threadIdx.x == 0) {
        Stats st = {m, 0.0f, 0.0f, 0u};
#pragma unroll
        for (uint32_t i = 0; i < kWaves; i++) st.s += part[1][i], st.u += part[2][i], st.above += counts[i];
        *gptr_mut<u32x4>(a.stats + 4 * (size_t)blockIdx.x) =
            u32x4{__float_as_uint(st.m), __float_as_uint(st.s), __float_as_uint(st.u), st.above};
    }
    if constexpr (TOP) {
        auto each = [&](auto f) {
#pragma unroll
            for (uint32_t j = 0; j < LOADS; j++)
#pragma unroll
                for (uint32_t e = 0; e < U; e++) {
                    const float y = x[j * U + e];
                    f(y > -kInf ? key_of(y + 0.0f, (uint32_t)(first + j * kThreads * U + e)) : 0ull);
                }
        };
        select_top(top, a.top, ordered(most + 0.0f), each, a.keys + (size_t)blockIdx.x * a.top);
    }
}

// Workgroup: a row's pieces joined.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void join_kernel(LogprobArgs a, uint32_t pieces) {
    __shared__ float part[3][kWaves];
    __shared__ uint32_t counts[kWaves];
    __shared__ TopLds top;
    __shared__ u64 out[kMostTop];
    const uint32_t row = blockIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x / 64;
    const float c = factor(a.temperature, row);
    const float* const stats = a.stats + 4 * (size_t)row * pieces;
    float m = -kInf;
    for (uint32_t i = threadIdx.x; i < pieces; i += kThreads) m = fmaxf(m, gptr<float>(stats)[4 * (size_t)i]);
    m = wave_max(m);
    if (lane == 0) part[0][wave] = m;
    __syncthreads();
    m = part[0][0];
#pragma unroll
    for (uint32_t i = 1; i < kWaves; i++) m = fmaxf(m, part[0][i]);
    float s = 0.0f, u = 0.0f;
    uint32_t above = 0;
    for (uint32_t i = threadIdx.x; i < pieces; i += kThreads) {
        const u32x4 w = *gptr<u32x4>(stats + 4 * (size_t)i);
        const float t = exponent(__uint_as_float(w.x), m, c), e = exp2_(t), ps = __uint_as_float(w.y);
        if (e > 0.0f) {  // else t ps may leave f32
            s += ps * e;
            u += (__uint_as_float(w.z) + t * ps) * e;
        }
        above += w.w;
    }
    s = wave_sum(s);
    u = wave_sum(u);
#pragma unroll
    for (int d = 32; d; d /= 2) above += (uint32_t)__shfl_xor((int)above, d);
    if (lane == 0) part[1][wave] = s, part[2][wave] = u, counts[wave] = above;
    __syncthreads();
    s = u = 0.0f;
    above = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; i++) s += part[1][i], u += part[2][i], above += counts[i];
    const float log_s = logf(s);
    const float inv = a.temperature ? c * kLn2 : 1.0f;
    auto logp = [&](float x) { return x == -kInf ? -kInf : (x - m) * inv - log_s; };
    if (a.top) {
        const u64* const keys = a.keys + (size_t)row * pieces * a.top;
        const u64 total = (u64)pieces * a.top;
        uint32_t largest = 0;
        for (u64 i = threadIdx.x; i < total; i += kThreads) largest = max(largest, (uint32_t)(*gptr<u64>(keys + i) >> 32));
        auto each = [&](auto f) {
            for (u64 i = 0; i < total; i += kThreads) f(i + threadIdx.x < total ? *gptr<u64>(keys + i + threadIdx.x) : 0ull);
        };
        select_top(top, a.top, largest, each, out);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < a.top; i += kThreads) {
            const u64 key = out[i];
            const size_t to = (size_t)row * a.top + i;
            const float x = unordered((uint32_t)(key >> 32));
            a.top_tokens[to] = key ? (int64_t)(uint32_t)~(uint32_t)key : -1;
            a.top_logprobs[to] = !key ? -kInf : c < 0.0f ? (i ? -kInf : 0.0f) : logp(x);
        }
    }
    if (threadIdx.x == 0) {
        if (a.entropy) {
            const float h = log_s - u / s * kLn2;
            a.entropy[row] = c < 0.0f || m == -kInf || h < 0.0f ? 0.0f : h;
        }
        const int64_t tok = a.tokens ? a.tokens[row] : -1;
        const bool given = tok >= 0 && tok < (int64_t)a.vocab;
        if (a.ranks) a.ranks[row] = given ? (int32_t)above : -1;
        if (a.logprobs) {
            float y = -kInf;
            if (given) {
                const uint64_t at = (uint64_t)((int64_t)row * a.stride + tok);
                const float x = plain(BF16 ? bf16_bits_to_f32(gptr<uint16_t>(a.logits)[at]) : gptr<float>(a.logits)[at]);
                y = c < 0.0f ? (above == 0 && x > -kInf ? 0.0f : -kInf) : logp(x);
            }
            a.logprobs[row] = y;
        }
    }
}

uint32_t pieces_of(uint32_t vocab, bool bf16) {
    return (uint32_t)(((uint64_t)vocab + (bf16 ? 7 : 3) + kPiece - 1) / kPiece);
}

}  // namespace

LogprobPlan logprob_plan(uint32_t rows, uint32_t vocab, uint32_t top, bool bf16) {
    LogprobPlan p;
    p.pieces = pieces_of(vocab, bf16);
    const uint64_t n = (uint64_t)rows * p.pieces;
    p.keys_at = 16 * n;
    p.bytes = (p.keys_at + 8 * n * top + 255) / 256 * 256;
    return p;
}

hipError_t logprob_launch(LogprobArgs a, const LogprobPlan& plan, uint8_t* work, hipStream_t st) {
    a.stats = reinterpret_cast<float*>(work);
    a.keys = reinterpret_cast<unsigned long long*>(work + plan.keys_at);
    const uint64_t grid = (uint64_t)a.rows * plan.pieces;
    if (!launchable(grid, kThreads) || !launchable(a.rows, kThreads)) return kTooManyThreads;
    auto go = [&](auto bf16, auto top) {
        piece_kernel<decltype(bf16)::value, decltype(top)::value><<<(uint32_t)grid, kThreads, 0, st>>>(a, plan.pieces);
    };
    using Y = std::true_type;
    using N = std::false_type;
    if (a.bf16) {
        a.top ? go(Y(), Y()) : go(Y(), N());
        join_kernel<true><<<a.rows, kThreads, 0, st>>>(a, plan.pieces);
    } else {
        a.top ? go(N(), Y()) : go(N(), N());
        join_kernel<false><<<a.rows, kThreads, 0, st>>>(a, plan.pieces);
    }
    return hipGetLastError();
}

}  // namespace dmx
