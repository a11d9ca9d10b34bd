// Verification of drafted tokens (the rule stands in include/dyninfer_mi355x.h).
//
// Three launches: the softmax statistics of every row, a workgroup a piece of a
// row (bound by reading the logits once); the walk down each tree, one
// workgroup a sequence, which reads single probabilities (and the whole row
// only where a node's second child is tried after a rejection); and the draw
// from what is left of the last node's distribution, pieces again.
//
// What is left after rejections at a node needs no stored row.  With p the
// target's and q the drafts' distribution, R_0 = p and R_k+1 = max(R_k - q, 0) /
// sum, every R_k is max(p - a_k q, 0) / w_k with a_0 = 0, w_0 = 1,
// a_k+1 = a_k + w_k and w_k+1 = sum max(p - a_k+1 q, 0).  Without q, R_k is p
// without the rejected tokens over what they leave of 1.
#include "kvcache.hpp"

namespace dmx {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kPiece = 16384;  // logits of a workgroup
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
    uint32_t row;    // of the logits; ~0: no rows
    uint32_t gone;   // rejected tokens (no draft probabilities), in the list of row0 + j
    float m, inv_t;  // p = exp((x - m) inv_t) / s
    float s, a;      // scores (e - a s q) / noise
    uint32_t greedy, done;
    unsigned long long best[2];  // of what is left, and of p
};

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

template <bool BF16>
__global__ __launch_bounds__(256) void stats_kernel(VerifyArgs a, Stat* out, uint32_t pieces) {
    const uint32_t piece = blockIdx.x % pieces, row = blockIdx.x / pieces;
    const float t = temperature(a, seq_of(a.starts, a.seqs, row));
    const bool greedy = !(t > 0.0f);
    const float inv_t = greedy ? 0.0f : fminf(1.0f / t, kFltMax);
    const uint32_t lo = piece * kPiece, hi = min(a.vocab, lo + kPiece);
    constexpr uint32_t E = BF16 ? 2 : 4, V = 16 / E;  // elements of a 16-byte load
    const uint8_t* base = static_cast<const uint8_t*>(a.logits) + (int64_t)row * a.logits_stride * (int64_t)E;
    // 16-byte steps from the first boundary at or after lo
    const uint32_t off = (uint32_t)((uintptr_t)(base + (size_t)lo * E) & 15u) / E;
    const uint32_t first = min(hi, lo + (off ? V - off : 0u));
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
        if (!greedy) {
#pragma unroll
            for (uint32_t j = 0; j < V; j++)
                if (j < n) st.s += weight(x[j], st.m, inv_t);
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
    for (uint32_t i = threadIdx.x; i < steps; i += 256) {
        const u32x4 ww = *gptr<u32x4>(base + ((size_t)first + (size_t)i * V) * E);
        float x[V];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (BF16) {
                x[2 * j] = clean(bf16_bits_to_f32(ww[j] & 0xFFFFu));
                x[2 * j + 1] = clean(__uint_as_float(ww[j] & 0xFFFF0000u));
            } else {
                x[j] = clean(__uint_as_float(ww[j]));
            }
        }
        take(x, first + i * V, V);
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

__device__ __forceinline__ Stat row_stat(const Stat* stats, uint32_t pieces, uint32_t row, float inv_t) {
    Stat st = {-__builtin_inff(), 0.0f, ~0u, 0u};
    for (uint32_t i = threadIdx.x & 63u; i < pieces; i += 64) st = join(st, stats[(size_t)row * pieces + i], inv_t);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) st = join(st, shuffle(st, x), inv_t);
    return st;
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

// Every thread follows the same path (all it branches on is the same in all of
// them); all of them join in only for a sum over a row.
__global__ __launch_bounds__(1024) void walk_kernel(VerifyArgs a, const Stat* stats, uint32_t pieces, int32_t* gone_list,
                                                    Left* left) {
    const uint32_t seq = blockIdx.x;
    __shared__ float sm[16];
    const int32_t r0 = a.starts[seq], r1 = a.starts[seq + 1];
    const uint32_t row0 = r0 < 0 ? 0u : min((uint32_t)r0, a.tokens), end = r1 < 0 ? 0u : min((uint32_t)r1, a.tokens);
    const uint32_t n = end > row0 ? min(end - row0, a.max_new) : 0u;
    int32_t* path = a.path + (size_t)seq * a.max_new;
    for (uint32_t i = threadIdx.x; i < a.max_new; i += blockDim.x) path[i] = -1;
    __syncthreads();
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
    const float inv_t = greedy ? 0.0f : fminf(1.0f / t, kFltMax);
    int32_t* gone = gone_list + row0;  // the rejected tokens of the current node
    uint32_t cur = 0, count = 1, rejected = 0;
    float aq = 0.0f, w = 1.0f;
    bool w_known = true, spent = false;
    Stat st = row_stat(stats, pieces, row0, inv_t);
    if (threadIdx.x == 0) path[0] = 0;
    for (uint32_t i = 1; i < n; i++) {
        const uint32_t parent = a.parents ? (uint32_t)a.parents[row0 + i] : i - 1;
        if (parent != cur || spent) continue;
        const int64_t tok = a.tokens_in[row0 + i];
        const uint32_t row = row0 + cur;
        const bool inside = tok >= 0 && tok < (int64_t)a.vocab;
        bool yes;
        if (greedy) {
            yes = inside && st.m != -__builtin_inff() && (uint32_t)tok == st.i;
        } else {
            if (!w_known) {  // a sibling was rejected: what is left of the row
                float sum = 0.0f;
                const int64_t lr = (int64_t)row * a.logits_stride, pr = (int64_t)row * a.probs_stride;
                for (uint32_t v = threadIdx.x; v < a.vocab; v += blockDim.x) {
                    float e = weight(clean(at(a.logits, a.logits_bf16, lr + v)), st.m, inv_t) / st.s;
                    if (a.probs) {
                        e = fmaxf(e - aq * at(a.probs, a.probs_bf16, pr + v), 0.0f);
                    } else {
                        for (uint32_t j = 0; j < rejected; j++)
                            if (gone[j] == (int32_t)v) e = 0.0f;
                    }
                    sum += e;
                }
                w = block_sum(sum, sm);
                w_known = true;
                if (!(w > 0.0f)) {
                    spent = true;
                    continue;
                }
            }
            float p = 0.0f, q = 1.0f;
            if (inside && st.s > 0.0f) {
                p = weight(clean(at(a.logits, a.logits_bf16, (int64_t)row * a.logits_stride + tok)), st.m, inv_t) / st.s;
                if (a.probs) {
                    q = at(a.probs, a.probs_bf16, (int64_t)row * a.probs_stride + tok);
                    p = fmaxf(p - aq * q, 0.0f);
                } else {
                    for (uint32_t j = 0; j < rejected; j++)
                        if (gone[j] == (int32_t)tok) p = 0.0f;
                }
                p /= w;
            } else if (a.probs && inside) {
                q = at(a.probs, a.probs_bf16, (int64_t)row * a.probs_stride + tok);
            }
            yes = gptr<float>(a.uniform)[row0 + i] * q < p;
        }
        if (yes) {
            cur = i;
            if (threadIdx.x == 0) path[count] = (int32_t)i;
            count++;
            rejected = 0;
            aq = 0.0f;
            w = 1.0f;
            w_known = true;
            st = row_stat(stats, pieces, row0 + cur, inv_t);
        } else if (!greedy) {
            if (a.probs) {
                aq += w;
                w_known = false;
            } else if (inside) {
                __syncthreads();
                if (threadIdx.x == 0) gone[rejected] = (int32_t)tok;
                __syncthreads();
                rejected++;
                w_known = false;
            }
        }
    }
    if (threadIdx.x == 0) {
        a.counts[seq] = (int32_t)count;
        if (greedy) {
            a.next[seq] = st.m == -__builtin_inff() ? -1 : (int64_t)st.i;
            out.row = ~0u;
        } else {
            out.row = row0 + cur;
            out.gone = spent ? 0u : rejected;
            out.m = st.m;
            out.s = st.s;
            out.inv_t = inv_t;
            out.a = spent ? 0.0f : aq;
        }
        left[seq] = out;
    }
}

// Score (not negative) and the lowest token that has it, as one number.
__device__ __forceinline__ unsigned long long pack(float score, uint32_t v) {
    return score > 0.0f ? ((unsigned long long)__float_as_uint(score) << 32) | (0xFFFFFFFFu - v) : 0ull;
}

__global__ __launch_bounds__(256) void draw_kernel(VerifyArgs a, const int32_t* gone_list, Left* left, uint32_t pieces) {
    const uint32_t seq = blockIdx.x / pieces, piece = blockIdx.x % pieces;
    const Left l = left[seq];
    if (l.row == ~0u) return;
    const int32_t r0 = a.starts[seq];
    const int32_t* gone = gone_list + (r0 < 0 ? 0 : r0);
    const float as = l.a * l.s;
    const uint32_t lo = piece * kPiece, hi = min(a.vocab, lo + kPiece);
    unsigned long long best0 = 0, best1 = 0;
    for (uint32_t v = lo + threadIdx.x; v < hi; v += 256) {
        const float e = weight(clean(at(a.logits, a.logits_bf16, (int64_t)l.row * a.logits_stride + v)), l.m, l.inv_t);
        const float z = gptr<float>(a.noise)[(int64_t)seq * a.noise_stride + v];
        float x = e;
        if (a.probs) {
            x = as > 0.0f ? e - as * at(a.probs, a.probs_bf16, (int64_t)l.row * a.probs_stride + v) : e;
        } else {
            for (uint32_t j = 0; j < l.gone; j++)
                if (gone[j] == (int32_t)v) x = 0.0f;
        }
        best0 = max(best0, pack(x / z, v));
        best1 = max(best1, pack(e / z, v));
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
        best0 = max(best0, (unsigned long long)__shfl_xor((long long)best0, x));
        best1 = max(best1, (unsigned long long)__shfl_xor((long long)best1, x));
    }
    // the largest does not depend on the order of these; the last workgroup reads it
    if ((threadIdx.x & 63u) == 0) {
        __hip_atomic_fetch_max(&left[seq].best[0], best0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_fetch_max(&left[seq].best[1], best1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t before = __hip_atomic_fetch_add(&left[seq].done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        if (before + 1 == pieces) {
            best0 = __hip_atomic_load(&left[seq].best[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            best1 = __hip_atomic_load(&left[seq].best[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const unsigned long long b = best0 ? best0 : best1;  // nothing left: the target's own
            a.next[seq] = b ? (int64_t)(0xFFFFFFFFu - (uint32_t)b) : -1;
        }
    }
}

uint64_t stats_bytes(uint32_t tokens, uint32_t vocab) {
    return ((uint64_t)tokens * verify_pieces(vocab) * sizeof(Stat) + 255) / 256 * 256;
}

}  // namespace

uint32_t verify_pieces(uint32_t vocab) { return (vocab + kPiece - 1) / kPiece; }

uint64_t verify_workspace_bytes(uint32_t seqs, uint32_t tokens, uint32_t vocab, uint32_t max_new) {
    (void)max_new;
    return stats_bytes(tokens, vocab) + ((uint64_t)tokens * 4 + 255) / 256 * 256 + (uint64_t)seqs * sizeof(Left);
}

hipError_t verify_launch(const VerifyArgs& a, uint8_t* work, hipStream_t st) {
    if (a.seqs == 0) return hipSuccess;
    const uint32_t pieces = verify_pieces(a.vocab);
    Stat* stats = reinterpret_cast<Stat*>(work);
    int32_t* gone = reinterpret_cast<int32_t*>(work + stats_bytes(a.tokens, a.vocab));
    Left* left = reinterpret_cast<Left*>(reinterpret_cast<uint8_t*>(gone) + ((uint64_t)a.tokens * 4 + 255) / 256 * 256);
    if (a.tokens) {
        if (a.logits_bf16)
            stats_kernel<true><<<a.tokens * pieces, 256, 0, st>>>(a, stats, pieces);
        else
            stats_kernel<false><<<a.tokens * pieces, 256, 0, st>>>(a, stats, pieces);
    }
    walk_kernel<<<a.seqs, 1024, 0, st>>>(a, stats, pieces, gone, left);
    draw_kernel<<<a.seqs * pieces, 256, 0, st>>>(a, gone, left, pieces);
    return hipGetLastError();
}

}  // namespace dmx
