// Verification of drafted tokens (the rule stands in include/dyninfer_mi355x.h).
//
// Three launches: the softmax statistics of every row, a workgroup a piece of a
// row (bound by reading the logits once); the walk down each tree, one
// workgroup a sequence; and the draw from what is left of the last node's
// distribution, pieces again.
//
// What is left after rejections at a node needs no stored row.  With p the
// target's and q the drafts' distribution, R_0 = p and R_k+1 = max(R_k - q, 0) /
// sum, every R_k is max(p - a_k q, 0) / w_k with a_0 = 0, w_0 = 1,
// a_k+1 = a_k + w_k and w_k+1 = sum max(p - a_k+1 q, 0).  Without q, R_k is p
// without the rejected tokens over what they leave of 1.  So the walk reads a
// node's p and q at its token only, all nodes at once, and goes on in LDS; it
// reads a whole row only for the w of a node that tries another child after a
// rejection (without q: where the difference from 1 would be inexact).
#include "kvcache.hpp"

namespace dmx {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Logits of a workgroup of the statistics.  Few rows are cut finer, for the
// latency of one pass: 5 bf16 rows of 151936 in 16384s took 9.3 us, in 4096s 5.4
// (4.8 with four loads in flight); 376 f32 rows, 228 MB, take 38 to 43 us, 49.8 with one
// load in flight and an accurate exponential of every element.
constexpr uint32_t kPiece = 16384, kSmallPiece = 4096;
constexpr uint32_t kManyPieces = 1024;  // workgroups from which the large pieces are taken
constexpr uint32_t kDraw = 4096;        // logits of a workgroup of the draw
constexpr uint32_t kNodes = 256;        // nodes the walk holds in LDS at a time
constexpr float kFltMax = 3.402823466e38f;

// Statistics of a piece of a row, or of a row.
struct Stat {
    float m;     // largest logit (NaN as -inf, +inf as the largest f32)
    float s;     // sum of exp((x - m) / temperature); greedy rows: not used
    uint32_t i;  // the lowest index of the largest
    uint32_t pad;
};

// What the draw needs of a sequence, written by the walk.
struct Left {
    uint32_t row;    // of the logits; ~0: nothing to draw (greedy, or no rows)
    uint32_t gone;   // rejected tokens (no draft probabilities), in the list of row0 + j
    float m, inv_t;  // p = exp((x - m) inv_t) / s
    float s, a;      // scores (e - a s q) / noise
    uint32_t done;   // workgroups of the draw that have brought their best
    unsigned long long best;
};

// NaN as -inf, +inf as the largest f32.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -__builtin_inff()), kFltMax); }

__device__ __forceinline__ float at(const void* p, uint32_t bf16, int64_t i) {
    return bf16 ? bf16_bits_to_f32(gptr<uint16_t>(p)[i]) : gptr<float>(p)[i];
}

// exp((x - m) / t), 0 for an x of -inf also where m is.
__device__ __forceinline__ float weight(float x, float m, float inv_t) {
    return x == -__builtin_inff() ? 0.0f : expf((x - m) * inv_t);
}

// Two statistics of disjoint pieces.
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float inv_t) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    r.i = a.m > b.m ? a.i : b.m > a.m ? b.i : min(a.i, b.i);
    r.s = a.s * weight(a.m, r.m, inv_t) + b.s * weight(b.m, r.m, inv_t);
    r.pad = 0;
    return r;
}

__device__ __forceinline__ Stat shuffle(const Stat& a, int x) {
    return {__shfl_xor(a.m, x), __shfl_xor(a.s, x), (uint32_t)__shfl_xor((int)a.i, x), 0u};
}

// The sequence that row `row` belongs to (the last whose start is not above it).
__device__ __forceinline__ uint32_t seq_of(const int32_t* starts, uint32_t seqs, uint32_t row) {
    uint32_t lo = 0, hi = seqs - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (starts[mid] <= (int32_t)row) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ float temperature(const VerifyArgs& a, uint32_t seq) {
    return a.temperature ? gptr<float>(a.temperature)[seq] : 1.0f;
}

// 1 / t of a positive temperature, neither infinite nor 0: -inf times it is -inf.
__device__ __forceinline__ float inverse(float t) { return fmaxf(fminf(1.0f / t, kFltMax), 1.2e-38f); }

template <bool BF16>
__global__ __launch_bounds__(256) void stats_kernel(VerifyArgs a, Stat* out, uint32_t pieces, uint32_t size) {
    const uint32_t piece = blockIdx.x % pieces, row = blockIdx.x / pieces;
    const float t = temperature(a, seq_of(a.starts, a.seqs, row));
    const bool greedy = !(t > 0.0f);
    const float inv_t = greedy ? 0.0f : inverse(t);
    const uint32_t lo = piece * size, hi = min(a.vocab, lo + size);
    constexpr uint32_t E = BF16 ? 2 : 4, V = 16 / E;  // elements of a 16-byte load
    const uint8_t* base = static_cast<const uint8_t*>(a.logits) + (int64_t)row * a.logits_stride * (int64_t)E;
    // 16-byte steps from the first boundary at or after lo
    const uint32_t off = (uint32_t)((uintptr_t)(base + (size_t)lo * E) & 15u) / E;
    const uint32_t first = min(hi, lo + (off ? V - off : 0u));
    const float scale = fminf(inv_t * 1.44269504f, kFltMax);
    Stat st = {-__builtin_inff(), 0.0f, ~0u, 0u};
    auto take = [&](const float (&x)[V], uint32_t i0, uint32_t n) {
        float m = -__builtin_inff();
#pragma unroll
        for (uint32_t j = 0; j < V; j++)
            if (j < n) m = fmaxf(m, x[j]);
        if (m > st.m) {
            st.s *= weight(st.m, m, inv_t);
            st.m = m;
#pragma unroll
            for (int j = V - 1; j >= 0; j--)
                if ((uint32_t)j < n && x[j] == m) st.i = i0 + j;
        }
        if (!greedy && st.m != -__builtin_inff()) {
            // the sum is its largest terms', whose arguments are small: 2^y as the
            // instruction gives it, of the one product
#pragma unroll
            for (uint32_t j = 0; j < V; j++)
                if (j < n) st.s += __builtin_amdgcn_exp2f((x[j] - st.m) * scale);
        }
    };
    // the ends that are no whole step, by one thread each
    auto ends = [&](uint32_t b, uint32_t e) {
        float x[V] = {};
        for (uint32_t j = 0; j < V; j++)
            if (b + j < e) x[j] = clean(at(base, BF16, b + j));
        take(x, b, e - b);
    };
    if (threadIdx.x == 0 && first > lo) ends(lo, first);
    const uint32_t steps = (hi - first) / V;
    constexpr uint32_t N = 4;  // loads in flight
    for (uint32_t i0 = threadIdx.x; i0 < steps; i0 += 256 * N) {
        u32x4 ww[N];
#pragma unroll
        for (uint32_t k = 0; k < N; k++) {
            const uint32_t i = min(i0 + 256 * k, steps - 1);
            ww[k] = *gptr<u32x4>(base + ((size_t)first + (size_t)i * V) * E);
        }
#pragma unroll
        for (uint32_t k = 0; k < N; k++) {
            const uint32_t i = i0 + 256 * k;
            if (i >= steps) break;
            float x[V];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (BF16) {
                    x[2 * j] = clean(bf16_bits_to_f32(ww[k][j] & 0xFFFFu));
                    x[2 * j + 1] = clean(__uint_as_float(ww[k][j] & 0xFFFF0000u));
                } else {
                    x[j] = clean(__uint_as_float(ww[k][j]));
                }
            }
            take(x, first + i * V, V);
        }
    }
    if (threadIdx.x == 255 && first + steps * V < hi) ends(first + steps * V, hi);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) st = join(st, shuffle(st, x), inv_t);
    __shared__ Stat sm[4];
    if ((threadIdx.x & 63u) == 0) sm[threadIdx.x >> 6] = st;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; w++) st = join(st, sm[w], inv_t);
        out[(size_t)row * pieces + piece] = st;
    }
}

// Sum over the workgroup, the same in every thread.
__device__ float block_sum(float x, float* sm) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) x += __shfl_xor(x, s);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) sm[threadIdx.x >> 6] = x;
    __syncthreads();
    float r = 0.0f;
    for (uint32_t w = 0; w < blockDim.x / 64; w++) r += sm[w];
    return r;
}

// A node as the walk sees it: its parent, the target's and the drafts'
// probability of its token there (greedy: p is 1 at the parent's best token).
struct Node {
    uint32_t parent;
    int32_t token;  // -1: outside the vocabulary
    float p, q, u;
};

// Eight elements from i on, 16-byte aligned.
__device__ __forceinline__ void eight(const void* p, uint32_t bf16, int64_t i, float (&x)[8]) {
    if (bf16) {
        const u32x4 w = *gptr<u32x4>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[2 * j] = bf16_bits_to_f32(w[j] & 0xFFFFu);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const u32x4 w = *gptr<u32x4>(static_cast<const float*>(p) + i + 4 * k);
#pragma unroll
            for (int j = 0; j < 4; j++) x[4 * k + j] = __uint_as_float(w[j]);
        }
    }
}

// This thread's share of sum max(p - aq q, 0) over a row, or, without q, of what the
// rejected tokens leave of p.  One workgroup reads the row, bound by its instructions, some 17 us
// for 151936 tokens: 15 siblings that all miss, 14 such sums, take 246 us of a call's 271 with f32
// probabilities, 258 of 285 with bf16.  (Calls of 8 trees of 8 took 181 and 240 us with loads of one
// element and an accurate exponential, so 78 and 84 on the same drafts.)
__device__ float left_of_row(const VerifyArgs& a, uint32_t row, const Stat& st, float inv_t, float aq, const int32_t* gone,
                             uint32_t rejected) {
    if (st.m == -__builtin_inff()) return 0.0f;
    const float inv_s = 1.0f / st.s, scale = fminf(inv_t * 1.44269504f, kFltMax);
    const int64_t lr = (int64_t)row * a.logits_stride, pr = (int64_t)row * a.probs_stride;
    const bool wide = (((uintptr_t)a.logits + lr * (a.logits_bf16 ? 2 : 4)) & 15u) == 0 &&
                      (!a.probs || (((uintptr_t)a.probs + pr * (a.probs_bf16 ? 2 : 4)) & 15u) == 0);
    float sum = 0.0f;
    auto take = [&](float x, float q, uint32_t v) {
        const float y = clean(x);
        float e = y == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((y - st.m) * scale) * inv_s;
        if (a.probs) {
            e = fmaxf(e - aq * q, 0.0f);
        } else {
            for (uint32_t g = 0; g < rejected; g++)
                if (gone[g] == (int32_t)v) e = 0.0f;
        }
        sum += e;
    };
    const uint32_t whole = wide ? a.vocab & ~7u : 0u;
    constexpr uint32_t N = 2;  // eights of a thread on their way together
    for (uint32_t v0 = 8 * threadIdx.x; v0 < whole; v0 += 8 * N * blockDim.x) {
        float x[N][8], q[N][8] = {};
#pragma unroll
        for (uint32_t k = 0; k < N; k++) {
            const uint32_t v = min(v0 + 8 * k * blockDim.x, whole - 8);
            eight(a.logits, a.logits_bf16, lr + v, x[k]);
            if (a.probs) eight(a.probs, a.probs_bf16, pr + v, q[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < N; k++) {
            const uint32_t v = v0 + 8 * k * blockDim.x;
            if (v >= whole) break;
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) take(x[k][j], q[k][j], v + j);
        }
    }
    for (uint32_t v = whole + threadIdx.x; v < a.vocab; v += blockDim.x)
        take(at(a.logits, a.logits_bf16, lr + v), a.probs ? at(a.probs, a.probs_bf16, pr + v) : 0.0f, v);
    return sum;
}

// Every thread follows the same path (all it branches on is the same in all of
// them); all of them work on the rows' statistics, the nodes, and sums over a row.
// Latency: 6 us for a chain of five, 11 for 32 trees of up to 16 (reading the nodes ahead
// of the statistics: 6.2 and 10.7).
__global__ __launch_bounds__(1024) void walk_kernel(VerifyArgs a, const Stat* stats, uint32_t pieces, Stat* rows,
                                                    int32_t* gone_list, Left* left) {
    const uint32_t seq = blockIdx.x;
    __shared__ float sm[16];
    __shared__ Node nodes[kNodes];
    const int32_t r0 = a.starts[seq], r1 = a.starts[seq + 1];
    const uint32_t row0 = r0 < 0 ? 0u : min((uint32_t)r0, a.tokens), end = r1 < 0 ? 0u : min((uint32_t)r1, a.tokens);
    const uint32_t n = end > row0 ? min(end - row0, a.max_new) : 0u;
    int32_t* path = a.path + (size_t)seq * a.max_new;
    for (uint32_t i = threadIdx.x; i < a.max_new; i += blockDim.x) path[i] = -1;
    Left out = {};
    if (n == 0) {
        if (threadIdx.x == 0) {
            a.counts[seq] = 0;
            a.next[seq] = -1;
            out.row = ~0u;
            left[seq] = out;
        }
        return;
    }
    const float t = temperature(a, seq);
    const bool greedy = !(t > 0.0f);
    const float inv_t = greedy ? 0.0f : inverse(t);
    int32_t* gone = gone_list + row0;  // the rejected tokens of the current node

    // a row's statistics from its pieces', a wave a row
    for (uint32_t r = threadIdx.x >> 6; r < n; r += blockDim.x / 64) {
        Stat st = {-__builtin_inff(), 0.0f, ~0u, 0u};
        for (uint32_t i = threadIdx.x & 63u; i < pieces; i += 64)
            st = join(st, stats[(size_t)(row0 + r) * pieces + i], inv_t);
#pragma unroll
        for (int x = 1; x < 64; x *= 2) st = join(st, shuffle(st, x), inv_t);
        if ((threadIdx.x & 63u) == 0) rows[row0 + r] = st;
    }
    __syncthreads();

    uint32_t cur = 0, count = 1, rejected = 0;
    float aq = 0.0f, w = 1.0f;
    bool w_known = true, spent = false;
    if (threadIdx.x == 0) path[0] = 0;
    for (uint32_t c0 = 1; c0 < n; c0 += kNodes) {
        const uint32_t cn = min(kNodes, n - c0);
        __syncthreads();
        if (threadIdx.x < cn) {
            const uint32_t i = c0 + threadIdx.x;
            Node nd = {a.parents ? (uint32_t)a.parents[row0 + i] : i - 1, -1, 0.0f, 1.0f, 0.0f};
            if (nd.parent >= i) nd.parent = ~0u;  // no such node: never tried
            const int64_t tok = a.tokens_in[row0 + i];
            if (!greedy) nd.u = gptr<float>(a.uniform)[row0 + i];
            if (nd.parent != ~0u && tok >= 0 && tok < (int64_t)a.vocab) {
                const uint32_t row = row0 + nd.parent;
                const Stat st = rows[row];
                nd.token = (int32_t)tok;
                if (greedy) {
                    nd.p = st.m != -__builtin_inff() && (uint32_t)tok == st.i ? 1.0f : 0.0f;
                } else {
                    const float x = clean(at(a.logits, a.logits_bf16, (int64_t)row * a.logits_stride + tok));
                    if (st.s > 0.0f) nd.p = weight(x, st.m, inv_t) / st.s;
                    if (a.probs) nd.q = at(a.probs, a.probs_bf16, (int64_t)row * a.probs_stride + tok);
                }
            }
            nodes[threadIdx.x] = nd;
        }
        __syncthreads();
        for (uint32_t k = 0; k < cn; k++) {
            if (nodes[k].parent != cur || spent) continue;
            const Node nd = nodes[k];
            float p = nd.p;
            if (rejected && !greedy) {
                if (!a.probs) {
                    for (uint32_t j = 0; j < rejected; j++)
                        if (gone[j] == nd.token) p = 0.0f;
                } else {
                    p = fmaxf(p - aq * nd.q, 0.0f);
                }
                if (!w_known) {  // what earlier siblings left of the row
                    const uint32_t row = row0 + cur;
                    const Stat st = rows[row];
                    w = block_sum(left_of_row(a, row, st, inv_t, aq, gone, rejected), sm);
                    w_known = true;
                    if (!(w > 0.0f)) {
                        spent = true;
                        continue;
                    }
                }
                p /= w;
            }
            if (nd.token >= 0 && nd.u * nd.q < p) {
                cur = c0 + k;
                if (threadIdx.x == 0) path[count] = (int32_t)cur;
                count++;
                rejected = 0;
                aq = 0.0f;
                w = 1.0f;
                w_known = true;
            } else if (!greedy) {
                if (a.probs) {
                    aq += w;
                    w_known = false;
                    rejected++;
                } else if (nd.token >= 0) {
                    __syncthreads();
                    if (threadIdx.x == 0) gone[rejected] = nd.token;
                    __syncthreads();
                    rejected++;
                    // p is already over w here: w (1 - p) is left.  Below 1/16 of the
                    // row the difference has lost too many bits, and it is summed
                    w -= p * w;
                    w_known = w > 0.0625f;
                }
            }
        }
    }
    if (threadIdx.x == 0) {
        const Stat st = rows[row0 + cur];
        a.counts[seq] = (int32_t)count;
        if (greedy) {
            a.next[seq] = st.m == -__builtin_inff() ? -1 : (int64_t)st.i;
            out.row = ~0u;
        } else {
            out.row = row0 + cur;
            out.gone = spent || a.probs ? 0u : rejected;
            out.m = st.m;
            out.s = st.s;
            out.inv_t = inv_t;
            out.a = spent ? 0.0f : aq;
        }
        left[seq] = out;
    }
}

// Score and the lowest token that has it, as one number whose largest is the
// draw: scores from what is left come before those from p itself, and one that
// is not positive counts for nothing.
__device__ __forceinline__ unsigned long long pack(float left, float full, uint32_t v) {
    const uint32_t top = left > 0.0f ? __float_as_uint(left) | 0x80000000u : full > 0.0f ? __float_as_uint(full) : 0u;
    return top ? ((unsigned long long)top << 32) | (0xFFFFFFFFu - v) : 0ull;
}

// 32 rows of 151936 logits and their noise, 39 MB: 12.6 us.
__global__ __launch_bounds__(512) void draw_kernel(VerifyArgs a, const int32_t* gone_list, Left* left, uint32_t pieces) {
    const uint32_t seq = blockIdx.x / pieces, piece = blockIdx.x % pieces;
    const uint32_t lo = piece * kDraw + threadIdx.x;
    constexpr uint32_t N = kDraw / 512;  // all loads of a thread in flight together
    float x[N], z[N], q[N];
#pragma unroll
    for (uint32_t j = 0; j < N; j++) {
        const uint32_t v = lo + 512 * j;
        z[j] = v < a.vocab ? gptr<float>(a.noise)[(int64_t)seq * a.noise_stride + v] : 1.0f;
    }
    const Left l = left[seq];
    if (l.row == ~0u) return;
    const int32_t r0 = a.starts[seq];
    const int32_t* gone = gone_list + (r0 < 0 ? 0 : r0);
    const float as = l.a * l.s, scale = fminf(l.inv_t * 1.44269504f, kFltMax);
    const bool minus = a.probs && as > 0.0f;
    const int64_t lr = (int64_t)l.row * a.logits_stride, pr = (int64_t)l.row * a.probs_stride;
#pragma unroll
    for (uint32_t j = 0; j < N; j++) {
        const uint32_t v = lo + 512 * j;
        x[j] = v < a.vocab ? at(a.logits, a.logits_bf16, lr + v) : -__builtin_inff();
        q[j] = minus && v < a.vocab ? at(a.probs, a.probs_bf16, pr + v) : 0.0f;
    }
    unsigned long long best = 0;
#pragma unroll
    for (uint32_t j = 0; j < N; j++) {
        const uint32_t v = lo + 512 * j;
        const float y = clean(x[j]);
        const float e = y == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((y - l.m) * scale);
        float r = minus ? e - as * q[j] : e;
        for (uint32_t g = 0; g < l.gone; g++)
            if (gone[g] == (int32_t)v) r = 0.0f;
        const float inv = __builtin_amdgcn_rcpf(z[j]);
        best = max(best, pack(r * inv, e * inv, v));
    }
#pragma unroll
    for (int s = 1; s < 64; s *= 2) best = max(best, (unsigned long long)__shfl_xor((long long)best, s));
    __shared__ unsigned long long sm[8];
    if ((threadIdx.x & 63u) == 0) sm[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 8; w++) best = max(best, sm[w]);
    // The largest does not depend on the order of these; the last workgroup reads it.
    // Only this number passes between workgroups, by an atomic that has returned
    // before the count goes up, so no cache need be written back: with release and
    // acquire on the count 2400 workgroups took 40.4 us, without 17.6 (1216 of 512
    // threads: 12.6).
    const unsigned long long old = __hip_atomic_fetch_max(&left[seq].best, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::"v"(old) : "memory");
    const uint32_t before = __hip_atomic_fetch_add(&left[seq].done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before + 1 == pieces) {
        best = __hip_atomic_load(&left[seq].best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        a.next[seq] = best ? (int64_t)(0xFFFFFFFFu - (uint32_t)best) : -1;
    }
}

// Size of the statistics' pieces.
uint32_t piece_size(uint32_t tokens, uint32_t vocab) {
    return (uint64_t)tokens * ((vocab + kPiece - 1) / kPiece) >= kManyPieces ? kPiece : kSmallPiece;
}
uint32_t piece_count(uint32_t tokens, uint32_t vocab) {
    const uint32_t s = piece_size(tokens, vocab);
    return (vocab + s - 1) / s;
}

uint64_t round256(uint64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

uint64_t verify_workspace_bytes(uint32_t seqs, uint32_t tokens, uint32_t vocab) {
    return round256((uint64_t)tokens * piece_count(tokens, vocab) * sizeof(Stat)) + round256((uint64_t)tokens * sizeof(Stat)) +
           round256((uint64_t)tokens * 4) + (uint64_t)seqs * sizeof(Left);
}

hipError_t verify_launch(const VerifyArgs& a, uint8_t* work, hipStream_t st) {
    if (a.seqs == 0) return hipSuccess;
    const uint32_t size = piece_size(a.tokens, a.vocab), pieces = piece_count(a.tokens, a.vocab);
    const uint32_t draws = (a.vocab + kDraw - 1) / kDraw;
    if (!launchable((uint64_t)a.tokens * pieces, 256) || !launchable(a.seqs, 1024) ||
        !launchable((uint64_t)a.seqs * draws, 512))
        return kTooManyThreads;
    Stat* stats = reinterpret_cast<Stat*>(work);
    work += round256((uint64_t)a.tokens * pieces * sizeof(Stat));
    Stat* rows = reinterpret_cast<Stat*>(work);
    work += round256((uint64_t)a.tokens * sizeof(Stat));
    int32_t* gone = reinterpret_cast<int32_t*>(work);
    work += round256((uint64_t)a.tokens * 4);
    Left* left = reinterpret_cast<Left*>(work);
    if (a.tokens) {
        if (a.logits_bf16)
            stats_kernel<true><<<a.tokens * pieces, 256, 0, st>>>(a, stats, pieces, size);
        else
            stats_kernel<false><<<a.tokens * pieces, 256, 0, st>>>(a, stats, pieces, size);
    }
    walk_kernel<<<a.seqs, 1024, 0, st>>>(a, stats, pieces, rows, gone, left);
    draw_kernel<<<a.seqs * draws, 512, 0, st>>>(a, gone, left, draws);
    return hipGetLastError();
}

}  // namespace dmx
