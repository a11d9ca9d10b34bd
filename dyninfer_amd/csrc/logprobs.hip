// Log probabilities of given tokens, their ranks, the entropy and the likeliest
// alternatives of logits [rows, vocab].
//
//   t_i = (x_i - m) / T with m = max x,  S = sum e^t_i,  U = sum e^t_i t_i
//   log p_i = t_i - ln S,  entropy = ln S - U / S
//
// S is held as R = S - 1, the sum without the largest logit's own 1, and ln S as log1p R: of a token that has nearly all of
// the probability the logarithm is -R, which S itself holds to 2^-24 of 1 only.
//
// One pass: a workgroup holds a piece of a row in registers (256 threads x 32 logits; 16 or 64
// logits a thread, 128 or 512 threads were slower), so its maximum is known before the exponentials and
// every logit is read once; a second small launch joins a row's pieces.  A row of up to
// 2048 logits is one wave's, in one launch (8000 rows of 1000 in bf16 18 us with a launch for each row's
// joining 76).  Bound by the logits' bytes where rows are many (2047 rows of 151936 in bf16, 622 MB:
// 130 to 135 us without tokens, 4.6 to 4.8 TB/s, nearly the rate of a copy; some eleven vector instructions a logit, the
// exponential counted as four, fill four fifths of that), by two launches where they are few (one
// row 7 us).
//
// The order is that of (logit, lower token first), held as one 64-bit key: the
// float's bits as a whole number of the same order, and the token's complement.
// A piece's largest `top`: of its threads' largest logits one wave finds a bound
// that `top` of them reach; what reaches it is gathered in LDS, in each wave's own order and
// quarter, and one wave puts it in order.  That is latency, not bytes: the 2047 rows with tokens take 131 to 148 us by
// card, with 1, 5, 20, 64 alternatives 161, 164, 194, 352.  Few more than `top` reach the bound, unless many logits tie, or
// fewer than `top` threads hold any that count: then all of them reach it, and where one wave has more than its
// quarter holds, `top` rounds over the piece find one after another.  So with 64 alternatives where a piece's logits
// lie in few threads: 1000 rows of 24576 in bf16 take 55 us, of 24976, whose last piece has 400, 290, and under a mask
// that leaves 300 in a row 990 (300 here and there: 54).
#include "kvcache.hpp"

#include <type_traits>

namespace dmx {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

constexpr uint32_t kHeld = 32;        // logits a thread holds
constexpr uint32_t kGathered = 512;   // keys that LDS has room for
constexpr float kInf = __builtin_inff();
constexpr float kMost = 3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Sums of a piece up to this are taken again without the largest logit; of larger ones S - 1 has no more than five times the
// relative error of S.  A row's nearly certain piece is one of many, and where logits are spread there is none; if every
// piece had one logit far above its others, 2047 rows of 151936 in bf16 would take 170 us instead of 130 (with 5
// alternatives 204 instead of 165).
constexpr float kCertain = 1.25f;

struct Stats {
    float m, r, u;   // largest logit, R and U from it, exponents in powers of two; of nothing above -inf R = -1
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

// ln(1 + r).  A small r, of a nearly certain row, by 2 artanh(r / (2 + r)), whose series ends at 2^-34 here.
__device__ __forceinline__ float log_sum(float r) {
    if (!(fabsf(r) < kCertain - 1.0f)) return logf(1.0f + r);
    const float z = r / (2.0f + r), q = z * z;
    return 2.0f * z * __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, 1.0f / 9, 1.0f / 7), 0.2f), 1.0f / 3), 1.0f);
}

// (x - m) c, not below what a product with 0 survives; also for x = m = -inf.
__device__ __forceinline__ float exponent(float x, float m, float c) { return fmaxf((x - m) * c, -1e38f); }

// f over all 64 lanes, the same in each: within rows of 16 by DPP, then by swaps of rows, no step through LDS.
template <class T, class F>
__device__ __forceinline__ T wave_all(T x, F f) {
    static_assert(sizeof(T) == 4, "one register");
    auto bits = [](T v) { return __builtin_bit_cast(uint32_t, v); };
    auto moved = [&](T v, auto ctrl) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, (int)bits(v), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    x = f(x, moved(x, std::integral_constant<int, 0xB1>()));   // lane ^ 1
    x = f(x, moved(x, std::integral_constant<int, 0x4E>()));   // lane ^ 2
    x = f(x, moved(x, std::integral_constant<int, 0x141>()));  // mirrored in 8
    x = f(x, moved(x, std::integral_constant<int, 0x140>()));  // mirrored in 16
    const auto r = __builtin_amdgcn_permlane16_swap(bits(x), bits(x), false, false);  // rows 0 0 2 2 and 1 1 3 3
    x = f(__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(bits(x), bits(x), false, false);  // lower and upper half
    return f(__builtin_bit_cast(T, (uint32_t)h[0]), __builtin_bit_cast(T, (uint32_t)h[1]));
}
__device__ __forceinline__ float wave_max(float x) {
    return wave_all(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
    return wave_all(x, [](float a, float b) { return a + b; });
}

template <int THREADS>
struct TopLds {
    static constexpr uint32_t WAVES = THREADS / 64, EACH = kGathered / WAVES;
    uint32_t most[THREADS];
    u64 keys[kGathered];  // EACH for every wave
    u64 best[WAVES];
    uint32_t count[WAVES], bound;
};

// A bound on the high half of keys that at least `top` of the threads' largest (l.most, behind a
// barrier) reach, and not many more if there is such a one.  By one wave, for all behind the next barrier.
template <int THREADS>
__device__ __forceinline__ void find_bound(TopLds<THREADS>& l, uint32_t top) {
    static_assert(kMostTop <= 64, "no more than a wave has lanes");
    constexpr uint32_t N = THREADS / 64;
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t v[N], hi = 0, lo = ~0u;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) v[i] = l.most[lane + 64 * i], hi = max(hi, v[i]), lo = min(lo, v[i]);
    hi = wave_all(hi, [](uint32_t a, uint32_t b) { return max(a, b); });
    lo = wave_all(lo, [](uint32_t a, uint32_t b) { return min(a, b); });
    hi = __builtin_amdgcn_readfirstlane(hi);
    lo = max((uint32_t)__builtin_amdgcn_readfirstlane(lo), kNothing + 1);
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        uint32_t n = 0;
#pragma unroll
        for (uint32_t i = 0; i < N; i++) n += (uint32_t)__popcll(__ballot(v[i] >= mid));
        if (n >= top) {
            lo = mid;
            if (n <= top + top / 4 + 6) break;  // exactly `top`: 2047 rows of 151936 with 20 203 us; up to 2 top + 32: 209; so 193
        } else {
            hi = mid - 1;
        }
    }
    if (lane == 0) l.bound = lo;
}

// The `top` largest of n different keys, 64 PER at most, held by one wave (0: none), into
// out[0..top-1], descending, 0 where there are fewer.  room: LDS for 64 keys.
template <uint32_t PER>
__device__ __forceinline__ void finish_top(const u64 (&k)[PER], uint32_t n, uint32_t top, u64* room, u64* out) {
    const uint32_t lane = threadIdx.x & 63u;
    u64 from = 1;
    if (n > 64) {  // a bound that `top` to 64 of them reach: by their high halves, then, where those tie, by all bits
        uint32_t hi = 0;
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) hi = max(hi, (uint32_t)(k[i] >> 32));
        hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)wave_all(hi, [](uint32_t a, uint32_t b) { return max(a, b); }));
        uint32_t lo = kNothing + 1;
        while (n > 64 && lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            uint32_t some = 0;
#pragma unroll
            for (uint32_t i = 0; i < PER; i++) some += (uint32_t)__popcll(__ballot((uint32_t)(k[i] >> 32) >= mid));
            if (some >= top) {
                lo = mid;
                n = some;
            } else {
                hi = mid - 1;
            }
        }
        from = (u64)lo << 32;
        u64 to = from | 0xFFFFFFFFull;
        while (n > 64) {
            const u64 mid = from + (to - from) / 2 + 1;
            uint32_t some = 0;
#pragma unroll
            for (uint32_t i = 0; i < PER; i++) some += (uint32_t)__popcll(__ballot(k[i] >= mid));
            if (some >= top) {
                from = mid;
                n = some;
            } else {
                to = mid - 1;
            }
        }
    }
    uint32_t at = 0;
#pragma unroll
    for (uint32_t i = 0; i < PER; i++) {  // side by side
        const bool in = k[i] >= from;
        const u64 mask = __ballot(in);
        if (in) room[at + (uint32_t)__popcll(mask & ((1ull << lane) - 1ull))] = k[i];
        at += (uint32_t)__popcll(mask);
    }
    __builtin_amdgcn_wave_barrier();
    // a key a lane: its place is the number of larger ones
    const u64 key = lane < n ? room[lane] : 0ull;
    const int lo32 = (int)(uint32_t)key, hi32 = (int)(uint32_t)(key >> 32);
    uint32_t place = 0;
    for (uint32_t j = 0; j < n; j++)
        place += ((u64)(uint32_t)__builtin_amdgcn_readlane(hi32, (int)j) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo32, (int)j)) > key;
    if (lane < n && place < top) out[place] = key;
    if (lane >= n && lane < top) out[lane] = 0;
}

// The `top` largest keys in out[0..top-1], descending, 0 where there are fewer; behind the barrier after find_bound.
// each(reaches, f) calls f(key) in the same order in all threads of a wave, for the keys whose high half
// reaches `reaches`; it may leave out others, or give 0; again(f) for all keys, without holding them in registers.
// Keys differ, those that count are above kNothing's.
template <int THREADS, class E, class A>
__device__ __forceinline__ void select_top(TopLds<THREADS>& l, uint32_t top, const E& each, const A& again, u64* out) {
    using L = TopLds<THREADS>;
    constexpr uint32_t N = L::WAVES;
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64));
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)l.bound);
    uint32_t found = 0;  // of this wave
    each(lo, [&](u64 key) {
        const bool in = (uint32_t)(key >> 32) >= lo;
        const u64 mask = __ballot(in);
        const uint32_t at = found + (uint32_t)__popcll(mask & ((1ull << lane) - 1ull));
        if (in && at < L::EACH) l.keys[wave * L::EACH + at] = key;
        found += (uint32_t)__popcll(mask);
    });
    if (lane == 0) l.count[wave] = found;
    __syncthreads();
    uint32_t n = 0, widest = 0, ends[N];
#pragma unroll
    for (uint32_t w = 0; w < N; w++) {
        const uint32_t k = (uint32_t)__builtin_amdgcn_readfirstlane((int)l.count[w]);
        n += k;
        widest = max(widest, k);
        ends[w] = n;
    }
    auto gathered = [&](uint32_t i) {  // number i of them
        uint32_t at = i;
#pragma unroll
        for (uint32_t w = 0; w + 1 < N; w++)
            if (i >= ends[w]) at = (w + 1) * L::EACH + i - ends[w];
        return l.keys[at];
    };
    if (widest <= L::EACH) {  // by one wave
        if (wave != 0) return;
        auto finish = [&](auto per) {
            constexpr uint32_t PER = decltype(per)::value;
            u64 k[PER];
#pragma unroll
            for (uint32_t i = 0; i < PER; i++) k[i] = 64 * i + lane < n ? gathered(64 * i + lane) : 0ull;
            finish_top(k, n, top, l.keys, out);
        };
        if (n <= 64)
            finish(std::integral_constant<uint32_t, 1>());
        else if (n <= 128)
            finish(std::integral_constant<uint32_t, 2>());
        else
            finish(std::integral_constant<uint32_t, kGathered / 64>());
        return;
    }
    // too many for a wave's quarter: one after another, each the largest below the one before
    u64 last = ~0ull;
    for (uint32_t i = 0; i < top; i++) {
        u64 best = 0;
        again([&](u64 key) {
            if ((uint32_t)(key >> 32) > kNothing && key < last && key > best) best = key;
        });
#pragma unroll
        for (int d = 32; d; d /= 2) {
            const u64 o = __shfl_xor(best, d);
            best = o > best ? o : best;
        }
        if (lane == 0) l.best[wave] = best;
        __syncthreads();
        best = l.best[0];
#pragma unroll
        for (uint32_t w = 1; w < N; w++) best = l.best[w] > best ? l.best[w] : best;
        __syncthreads();
        if (threadIdx.x == 0) out[i] = best;
        last = best;  // 0: nothing is below it
    }
}

// A row's outputs from its statistics and its largest keys (in LDS, behind a barrier).
template <int THREADS, bool BF16>
__device__ __forceinline__ void write_row(const LogprobArgs& a, uint32_t row, const Stats& st, float c, const u64* keys) {
    const float m = st.m, log_s = log_sum(st.r), inv = a.temperature ? c * kLn2 : 1.0f;
    auto logp = [&](float x) {
        if (x == -kInf) return -kInf;
        const float d = x - m;  // may leave f32 where d / T does not
        return (d == -kInf ? (0.5f * x - 0.5f * m) * (2.0f * inv) : d * inv) - log_s;
    };
    for (uint32_t i = threadIdx.x; i < a.top; i += THREADS) {
        const u64 key = keys[i];
        const size_t to = (size_t)row * a.top + i;
        gptr_mut<int64_t>(a.top_tokens)[to] = key ? (int64_t)(uint32_t)~(uint32_t)key : -1;
        gptr_mut<float>(a.top_logprobs)[to] = !key ? -kInf : c < 0.0f ? (i ? -kInf : 0.0f) : logp(unordered((uint32_t)(key >> 32)));
    }
    if (threadIdx.x != 0) return;
    if (a.entropy) {
        const float h = log_s - st.u / (1.0f + st.r) * kLn2;
        gptr_mut<float>(a.entropy)[row] = c < 0.0f || m == -kInf || h < 0.0f ? 0.0f : h;
    }
    const int64_t tok = a.tokens ? gptr<int64_t>(a.tokens)[row] : -1;
    const bool given = tok >= 0 && tok < (int64_t)a.vocab;
    if (a.ranks) gptr_mut<int32_t>(a.ranks)[row] = given ? (int32_t)st.above : -1;
    if (a.logprobs) {
        float y = -kInf;
        if (given) {
            const uint64_t at = (uint64_t)((int64_t)row * a.stride + tok);
            const float x = plain(BF16 ? bf16_bits_to_f32(gptr<uint16_t>(a.logits)[at]) : gptr<float>(a.logits)[at]);
            y = c < 0.0f ? (st.above == 0 && x > -kInf ? 0.0f : -kInf) : logp(x);
        }
        gptr_mut<float>(a.logprobs)[row] = y;
    }
}

// Workgroup (row, piece).  Pieces are whole 16-byte units of memory: a row that does not begin
// at one has its first piece begin before the row, and the last may end behind it (units without
// a logit of the row are not read; what lies beside it in one is not looked at).  ONE: a row is one
// piece, and finished here.
template <int THREADS, bool BF16, bool TOP, bool ONE>
__global__ __launch_bounds__(THREADS, BF16 ? 6 : 1) void piece_kernel(LogprobArgs a, uint32_t pieces) {
    constexpr uint32_t U = BF16 ? 8 : 4, LOADS = kHeld / U;  // logits of a load
    constexpr uint32_t W = THREADS / 64, PIECE = THREADS * kHeld;
    __shared__ float part[3][W];
    __shared__ uint32_t counts[W];
    __shared__ std::conditional_t<TOP, TopLds<THREADS>, char> top;
    __shared__ u64 best[TOP && ONE ? kMostTop : 1];
    const uint32_t row = ONE ? blockIdx.x : blockIdx.x / pieces, piece = ONE ? 0u : blockIdx.x % pieces;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64;
    const uintptr_t base = reinterpret_cast<uintptr_t>(a.logits) + (uint64_t)((int64_t)row * a.stride) * (BF16 ? 2 : 4);
    const uint32_t shift = (uint32_t)(base & 15u) / (BF16 ? 2 : 4);
    const char* const src = reinterpret_cast<const char*>(base & ~(uintptr_t)15);
    // this thread's load j holds logits first + j * THREADS * U ..
    const int64_t first = (int64_t)piece * PIECE + threadIdx.x * U - shift;
    float x[kHeld];
    u32x4 w[LOADS];
#pragma unroll
    for (uint32_t j = 0; j < LOADS; j++) {
        const bool there = first + j * THREADS * U < (int64_t)a.vocab;
        w[j] = there ? *gptr<u32x4>(src + 16 * ((uint64_t)piece * (PIECE / U) + j * THREADS + threadIdx.x)) : u32x4{};
    }
    const int64_t tok = a.tokens ? gptr<int64_t>(a.tokens)[row] : -1;
    const bool given = tok >= 0 && tok < (int64_t)a.vocab;
    float xt = kInf;
    if (given) {
        const char* p = reinterpret_cast<const char*>(base) + tok * (BF16 ? 2 : 4);
        xt = plain(BF16 ? bf16_bits_to_f32(*gptr<uint16_t>(p)) : *gptr<float>(p));
    }
    const float c = factor(a.temperature, row);
    float some[LOADS], most = -kInf;  // the largest of each load, of all
#pragma unroll
    for (uint32_t j = 0; j < LOADS; j++) {
        const int64_t i = first + j * THREADS * U;
#pragma unroll
        for (uint32_t e = 0; e < U; e++)
            x[j * U + e] = BF16 ? __uint_as_float(e & 1u ? w[j][e / 2] & 0xFFFF0000u : w[j][e / 2] << 16) : __uint_as_float(w[j][e]);
        if (i < 0 || i + U > (int64_t)a.vocab) {  // the row's edges
#pragma unroll
            for (uint32_t e = 0; e < U; e++)
                if (i + (int64_t)e < 0 || i + (int64_t)e >= (int64_t)a.vocab) x[j * U + e] = -kInf;
        }
        some[j] = -kInf;
#pragma unroll
        for (uint32_t e = 0; e < U; e++) some[j] = fmaxf(some[j], x[j * U + e]);  // of a NaN and a number the number
        most = fmaxf(most, some[j]);
    }
    float m = wave_max(most);
    if (lane == 0) part[0][wave] = m;
    if constexpr (TOP) {
        top.most[threadIdx.x] = ordered(plain(most));
    }
    __syncthreads();
    if constexpr (TOP) {
        if (wave == 0) find_bound(top, a.top);
    }
    m = part[0][0];
#pragma unroll
    for (uint32_t i = 1; i < W; i++) m = fmaxf(m, part[0][i]);
    if (m == kInf) {  // an infinity among them
#pragma unroll
        for (uint32_t i = 0; i < kHeld; i++) x[i] = plain(x[i]);
        m = kMost;
    }
    float s = 0.0f, u = 0.0f;
    // one product a logit where nothing leaves f32: x c - M with M = m c rounded, which then
    // is taken off by what it was rounded by
    const float M = m * c, off = __builtin_fmaf(m, c, -M);
    const bool near = c > 0.0f && fabsf(M) < 1e30f;
    if (near) {
#pragma unroll
        for (uint32_t i = 0; i < kHeld; i++) {
            const float t = __builtin_fmaf(x[i], c, -M), e = exp2_(t);
            s += e;
            u = __builtin_fmaf(e, t, u);
        }
        const float f = exp2_(-off);
        u = (u - off * s) * f;
        s *= f;
    }
    // -inf or a NaN among them (0 times -inf), or numbers too far apart
    if (c > 0.0f && (!near || __any(u != u))) {
        s = u = 0.0f;
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
            const float bound = first + j * THREADS * U + U <= tok ? below : xt;
#pragma unroll
            for (uint32_t e = 0; e < U; e++) above += (uint32_t)__popcll(__ballot(x[j * U + e] > bound));
        }
        uint32_t more = 0;
        if (xt == -kInf) {  // nothing is below: all before it that are not above
#pragma unroll
            for (uint32_t j = 0; j < LOADS; j++) {
                const int64_t i = first + j * THREADS * U;
#pragma unroll
                for (uint32_t e = 0; e < U; e++)
                    more += !(x[j * U + e] > xt) && i + (int64_t)e >= 0 && i + (int64_t)e < tok;
            }
        } else if (tok >= (int64_t)piece * PIECE - shift && tok < (int64_t)(piece + 1) * PIECE - shift) {
#pragma unroll
            for (uint32_t j = 0; j < LOADS; j++) {
                const int64_t i = first + j * THREADS * U;
                if (i <= tok && tok < i + U) {
#pragma unroll
                    for (uint32_t e = 0; e < U; e++) more += x[j * U + e] == xt && i + (int64_t)e < tok;
                }
            }
        }
        // the loads of the row's edges hold -inf where it has no logit, which is above nothing
        if (__any(more != 0)) above += (uint32_t)wave_sum((float)more);
    }
    s = wave_sum(s);
    u = wave_sum(u);
    if (lane == 0) part[1][wave] = s, part[2][wave] = u, counts[wave] = above;
    __syncthreads();
    auto joined = [&](uint32_t k) {
        float sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < W; i++) sum += part[k][i];
        return sum;
    };
    Stats st = {m, joined(1) - 1.0f, joined(2), 0u};
#pragma unroll
    for (uint32_t i = 0; i < W; i++) st.above += counts[i];
    if (c > 0.0f && m > -kInf && st.r < kCertain - 1.0f) {  // the same in all threads; one logit is m
        s = u = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kHeld; i++) {
            const float t = exponent(x[i], m, c), e = x[i] == m ? 0.0f : exp2_(t);
            s += e;
            u += e * t;
        }
        s = wave_sum(s);
        u = wave_sum(u);
        if constexpr (W > 1) __syncthreads();
        if (lane == 0) part[1][wave] = s, part[2][wave] = u;
        __syncthreads();
        st.r = joined(1);
        st.u = joined(2);
    }
    if constexpr (TOP) {
        auto each = [&](uint32_t reaches, auto f) {
            const float bound = unordered(reaches);
            if (!__any(most >= bound)) return;
#pragma unroll
            for (uint32_t j = 0; j < LOADS; j++) {
                if (!__any(some[j] >= bound)) continue;
#pragma unroll
                for (uint32_t e = 0; e < U; e++) {
                    const float y = x[j * U + e];
                    const bool in = y >= bound;
                    if (__any(in)) f(in ? key_of(y + 0.0f, (uint32_t)first + j * THREADS * U + e) : 0ull);
                }
            }
        };
        auto again = [&](auto f) {
#pragma unroll 1
            for (uint32_t j = 0; j < LOADS; j++) {
                const int64_t i = first + j * THREADS * U;
                if (i >= (int64_t)a.vocab) continue;
                const u32x4 y = *gptr<u32x4>(src + 16 * ((uint64_t)piece * (PIECE / U) + j * THREADS + threadIdx.x));
#pragma unroll
                for (uint32_t e = 0; e < U; e++) {
                    const float z = plain(BF16 ? __uint_as_float(e & 1u ? y[e / 2] & 0xFFFF0000u : y[e / 2] << 16) : __uint_as_float(y[e]));
                    if (i + (int64_t)e >= 0 && i + (int64_t)e < (int64_t)a.vocab) f(key_of(z, (uint32_t)i + e));
                }
            }
        };
        select_top<THREADS>(top, a.top, each, again, ONE ? best : a.keys + (size_t)blockIdx.x * a.top);
        __syncthreads();
    }
    if constexpr (ONE) {
        write_row<THREADS, BF16>(a, row, st, c, best);
    } else if (threadIdx.x == 0) {
        *gptr_mut<u32x4>(a.stats + 4 * (size_t)blockIdx.x) =
            u32x4{__float_as_uint(st.m), __float_as_uint(st.r), __float_as_uint(st.u), st.above};
    }
}

// Workgroup: a row's pieces joined.  Up to 64 kMany keys (20 pieces of 64) are one wave's, in registers; up to 64 kFew
// (19 pieces of 20) in as few as that takes (by kMany 2047 rows of 151936 with 20 alternatives 197 us instead of
// 193, one row with 5 13.8 instead of 11).
constexpr uint32_t kJoin = 256, kFew = 6, kMany = 20;
template <bool BF16, bool TOP>
__global__ __launch_bounds__(kJoin) void join_kernel(LogprobArgs a, uint32_t pieces) {
    constexpr uint32_t W = kJoin / 64;
    __shared__ float part[4][W];
    __shared__ uint32_t counts[W];
    __shared__ std::conditional_t<TOP, TopLds<kJoin>, char> top;
    __shared__ u64 best[TOP ? kMostTop : 1];
    const uint32_t row = blockIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x / 64;
    const u64* const keys = a.keys + (size_t)row * pieces * a.top;
    const u64 total = (u64)pieces * a.top;
    const float c = factor(a.temperature, row);
    const float* const stats = a.stats + 4 * (size_t)row * pieces;
    const u32x4 mine = threadIdx.x < pieces ? *gptr<u32x4>(stats + 4 * threadIdx.x) : u32x4{0xFF800000u, 0xBF800000u, 0u, 0u};  // -inf, -1
    if constexpr (TOP) {
        auto by_one = [&](auto per) {
            constexpr uint32_t PER = decltype(per)::value;
            u64 k[PER];
            uint32_t n = 0;
#pragma unroll
            for (uint32_t i = 0; i < PER; i++) k[i] = 64 * i + lane < total ? *gptr<u64>(keys + 64 * i + lane) : 0ull;
#pragma unroll
            for (uint32_t i = 0; i < PER; i++) n += (uint32_t)__popcll(__ballot(k[i] != 0));
            finish_top(k, n, a.top, top.keys, best);
        };
        if (total > 64 * kMany) {
            uint32_t largest = 0;
            for (u64 i = threadIdx.x; i < total; i += kJoin) largest = max(largest, (uint32_t)(*gptr<u64>(keys + i) >> 32));
            top.most[threadIdx.x] = largest;
        } else if (wave == W - 1) {  // the others see to the statistics
            if (total <= 64 * kFew)
                by_one(std::integral_constant<uint32_t, kFew>());
            else
                by_one(std::integral_constant<uint32_t, kMany>());
        }
    }
    float m = __uint_as_float(mine.x);
    for (uint32_t i = threadIdx.x + kJoin; i < pieces; i += kJoin) m = fmaxf(m, gptr<float>(stats)[4 * (size_t)i]);
    m = wave_max(m);
    if (lane == 0) part[0][wave] = m;
    __syncthreads();
    if constexpr (TOP) {
        if (total > 64 * kMany && wave == 0) find_bound(top, a.top);
    }
    m = part[0][0];
#pragma unroll
    for (uint32_t i = 1; i < W; i++) m = fmaxf(m, part[0][i]);
    float s = 0.0f, u = 0.0f, ones = 0.0f;  // R without the largest logits' ones, and those
    uint32_t above = 0;
    auto join = [&](u32x4 w) {
        const float pm = __uint_as_float(w.x), pr = __uint_as_float(w.y), pu = __uint_as_float(w.z);
        const float t = exponent(pm, m, c), e = exp2_(t), ps = 1.0f + pr;
        if (pm == m) {
            s += pr;
            u += pu;
            ones += 1.0f;
        } else if (e > 0.0f) {  // else t ps may leave f32
            s += ps * e;
            u += (pu + t * ps) * e;
        }
        above += w.w;
    };
    join(mine);
    for (uint32_t i = threadIdx.x + kJoin; i < pieces; i += kJoin) join(*gptr<u32x4>(stats + 4 * (size_t)i));
    s = wave_sum(s);
    u = wave_sum(u);
    ones = wave_sum(ones);
    above = wave_all(above, [](uint32_t x, uint32_t y) { return x + y; });
    if (lane == 0) part[1][wave] = s, part[2][wave] = u, part[3][wave] = ones, counts[wave] = above;
    if constexpr (TOP) {
        if (total > 64 * kMany) {
            auto each = [&](uint32_t, auto f) {
                for (u64 i = 0; i < total; i += kJoin) f(i + threadIdx.x < total ? *gptr<u64>(keys + i + threadIdx.x) : 0ull);
            };
            auto again = [&](auto f) {
#pragma unroll 1
                for (u64 i = threadIdx.x; i < total; i += kJoin) f(*gptr<u64>(keys + i));
            };
            __syncthreads();
            select_top<kJoin>(top, a.top, each, again, best);
        }
    }
    __syncthreads();
    Stats st = {m, 0.0f, 0.0f, 0u};
    ones = -1.0f;
#pragma unroll
    for (uint32_t i = 0; i < W; i++) st.r += part[1][i], st.u += part[2][i], ones += part[3][i], st.above += counts[i];
    st.r += ones;
    write_row<kJoin, BF16>(a, row, st, c, best);
}

// Rows of up to 2048 logits are one wave's, without a second launch; longer ones pieces of 8192.
constexpr uint32_t kSmall = 64 * kHeld, kPiece = 256 * kHeld;

}  // namespace

LogprobPlan logprob_plan(uint32_t rows, uint32_t vocab, uint32_t top, bool bf16) {
    LogprobPlan p = {};
    const uint64_t n = (uint64_t)vocab + (bf16 ? 7 : 3);  // with what may lie before a row's first
    p.small = n <= kSmall;
    p.pieces = p.small ? 1u : (uint32_t)((n + kPiece - 1) / kPiece);
    if (p.pieces > 1) {
        const uint64_t all = (uint64_t)rows * p.pieces;
        p.keys_at = 16 * all;
        p.bytes = (p.keys_at + 8 * all * top + 255) / 256 * 256;
    }
    return p;
}

hipError_t logprob_launch(LogprobArgs a, const LogprobPlan& plan, uint8_t* work, hipStream_t st) {
    a.stats = reinterpret_cast<float*>(work);
    a.keys = reinterpret_cast<unsigned long long*>(work + plan.keys_at);
    const uint64_t grid = (uint64_t)a.rows * plan.pieces;
    if (!launchable(grid, plan.small ? 64 : 256) || !launchable(a.rows, plan.small ? 64 : kJoin)) return kTooManyThreads;
    auto go = [&](auto bf16, auto top) {
        constexpr bool B = decltype(bf16)::value, T = decltype(top)::value;
        if (plan.small) {
            piece_kernel<64, B, T, true><<<(uint32_t)grid, 64, 0, st>>>(a, 1);
        } else if (plan.pieces == 1) {
            piece_kernel<256, B, T, true><<<(uint32_t)grid, 256, 0, st>>>(a, 1);
        } else {
            piece_kernel<256, B, T, false><<<(uint32_t)grid, 256, 0, st>>>(a, plan.pieces);
            join_kernel<B, T><<<a.rows, kJoin, 0, st>>>(a, plan.pieces);
        }
        return hipGetLastError();
    };
    using Y = std::true_type;
    using N = std::false_type;
    if (a.bf16) return a.top ? go(Y(), Y()) : go(Y(), N());
    return a.top ? go(N(), Y()) : go(N(), N());
}

}  // namespace dmx
