// C ABI of the calls around attention (include/dyninfer_mi355x.h): rotary
// positions, the quantized paged cache, attention of drafted tokens over it,
// and their verification.  Checks here keep every kernel inside the buffers
// described; what the host cannot see (device tables) the kernels check.
#include <algorithm>
#include <cmath>
#include <utility>

#include "capi_common.hpp"
#include "kvcache.hpp"

using dmx::aligned;
using dmx::check_ctx;
using dmx::DeviceGuard;
using dmx::fail;
using dmx::hip_fail;

namespace {

constexpr int BAD = DYNINFER_MI355X_ERR_INVALID_ARGUMENT;
constexpr int UNSUPPORTED = DYNINFER_MI355X_ERR_UNSUPPORTED;

bool dim_ok(uint32_t d) { return d == 64 || d == 96 || d == 128 || d == 256; }

uint32_t bits_of(uint32_t enc) { return enc == DYNINFER_KV_Q8 ? 8 : enc == DYNINFER_KV_Q4 ? 4 : 0; }

int check_dim(uint32_t d) {
    return dim_ok(d) ? 0 : fail(UNSUPPORTED, "head_dim " + std::to_string(d) + " is not 64, 96, 128 or 256");
}

// The cache's shape, without its buffers.
int check_shape(const dyninfer_kvcache_t* c) {
    if (!c) return fail(BAD, "cache is NULL");
    if (!bits_of(c->k_encoding) || !bits_of(c->v_encoding)) return fail(UNSUPPORTED, "cache encodings must be KV_Q8 or KV_Q4");
    if (int rc = check_dim(c->head_dim)) return rc;
    if (c->kv_heads == 0 || c->pages == 0) return fail(BAD, "cache has no heads or no pages");
    if (c->kv_heads > 4096) return fail(UNSUPPORTED, "more than 4096 kv heads");
    if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
        return fail(UNSUPPORTED, "page_size must be a power of two, 16..4096");
    if (c->pages > 0x7FFFFFFFull) return fail(UNSUPPORTED, "more pages than 32-bit page ids can name");
    return 0;
}

// Slots (tokens of one head) of the cache: at most 2^31 * 2^12 * 2^12.
uint64_t slots(const dyninfer_kvcache_t* c) { return c->pages * c->kv_heads * c->page_size; }

uint64_t k_codes(const dyninfer_kvcache_t* c) { return slots(c) * (c->head_dim * bits_of(c->k_encoding) / 8); }
uint64_t v_codes(const dyninfer_kvcache_t* c) { return slots(c) * (c->head_dim * bits_of(c->v_encoding) / 8); }
uint64_t k_total(const dyninfer_kvcache_t* c) { return k_codes(c) + slots(c) * (c->head_dim / 32 * 2); }
uint64_t v_total(const dyninfer_kvcache_t* c) { return v_codes(c) + slots(c) * 2; }

int check_cache(const dyninfer_kvcache_t* c, dmx::KvView& kv) {
    if (int rc = check_shape(c)) return rc;
    if (!c->k || !c->v) return fail(BAD, "cache buffers are NULL");
    if (!aligned(c->k, 256) || !aligned(c->v, 256)) return fail(BAD, "cache buffers must be 256-byte aligned");
    if (c->k_bytes != k_total(c) || c->v_bytes != v_total(c))
        return fail(BAD, "cache buffers must be " + std::to_string(k_total(c)) + " and " + std::to_string(v_total(c)) +
                             " bytes, got " + std::to_string(c->k_bytes) + " and " + std::to_string(c->v_bytes));
    kv.k = static_cast<uint8_t*>(c->k);
    kv.v = static_cast<uint8_t*>(c->v);
    kv.k_scales = k_codes(c);
    kv.v_scales = v_codes(c);
    kv.pages = c->pages;
    kv.heads = c->kv_heads;
    kv.dim = c->head_dim;
    kv.page_shift = (uint32_t)__builtin_ctz(c->page_size);
    kv.k_bits = bits_of(c->k_encoding);
    kv.v_bits = bits_of(c->v_encoding);
    return 0;
}

// `tables`: the device tables are needed (not for a size query).
int check_batch(const dyninfer_kvbatch_t* b, bool tables, dmx::KvBatch& out) {
    if (!b) return fail(BAD, "batch is NULL");
    if (tables && b->sequences) {
        if ((b->table_pages && !b->page_table) || !b->lengths || !b->starts) return fail(BAD, "batch tables are NULL");
        if (!aligned(b->page_table, 4) || !aligned(b->lengths, 4) || !aligned(b->starts, 4))
            return fail(BAD, "batch tables must be 4-byte aligned");
    }
    if (b->tokens > 0x7FFFFFFFu || b->max_new > b->tokens)
        return fail(BAD, "batch: max_new must not be above tokens, nor tokens above 2^31 - 1");
    if (b->sequences > (1u << 24)) return fail(UNSUPPORTED, "batch: more than 2^24 sequences; split the call");
    if (b->max_length > 0x7FFFFFFFull) return fail(UNSUPPORTED, "batch: sequences are limited to 2^31 - 1 positions");
    out = {b->page_table, b->lengths, b->starts, b->sequences, b->table_pages, b->tokens, b->max_new};
    return 0;
}

int check_rows(const dyninfer_rows_t* r, const char* what, dmx::KvRows& out) {
    const std::string w(what);
    if (!r || !r->data) return fail(BAD, w + " is NULL");
    if (r->dtype != DYNINFER_DTYPE_F32 && r->dtype != DYNINFER_DTYPE_BF16) return fail(UNSUPPORTED, w + " must be f32 or bf16");
    const uint32_t e = r->dtype == DYNINFER_DTYPE_BF16 ? 2 : 4;
    if (!aligned(r->data, e)) return fail(BAD, w + " is misaligned");
    if (r->heads == 0) return fail(BAD, w + " has no heads");
    if (r->token_stride < 0 || r->head_stride < 0) return fail(BAD, w + ": strides must not be negative");
    out.p = r->data;
    out.ts = r->token_stride;
    out.hs = r->head_stride;
    out.bf16 = e == 2;
    out.vec = aligned(r->data, 16) && r->token_stride * e % 16 == 0 && (r->heads == 1 || r->head_stride * e % 16 == 0);
    return 0;
}

// Rows that are written: no two heads or tokens may share an element.
int check_out(const dyninfer_rows_t* r, uint32_t dim, uint32_t tokens, const char* what, dmx::KvRows& out) {
    if (int rc = check_rows(r, what, out)) return rc;
    const int64_t d = dim, h = r->heads, n = tokens;
    const bool token_major = (h <= 1 || r->head_stride >= d) && (n <= 1 || r->token_stride >= (h > 1 ? (h - 1) * r->head_stride + d : d));
    const bool head_major = (n <= 1 || r->token_stride >= d) && (h <= 1 || r->head_stride >= (n > 1 ? (n - 1) * r->token_stride + d : d));
    return token_major || head_major ? 0 : fail(BAD, std::string(what) + ": heads or tokens overlap");
}

int check_rope(const dyninfer_rope_t* r, uint32_t dim, uint32_t tokens, dmx::RopeView& out) {
    if (!r) return fail(BAD, "rope is NULL");
    if (!r->table || !aligned(r->table, 16)) return fail(BAD, "rope table is NULL or not 16-byte aligned");
    if (tokens && (!r->positions || !aligned(r->positions, 4))) return fail(BAD, "rope positions are NULL or misaligned");
    if (r->rot_dim < 2 || r->rot_dim % 2 || r->rot_dim > dim)
        return fail(BAD, "rot_dim must be even, 2.." + std::to_string(dim));
    if (r->layout != DYNINFER_ROPE_INTERLEAVED && r->layout != DYNINFER_ROPE_HALF) return fail(BAD, "unknown rope layout");
    out = {r->table, r->positions, r->table_positions, r->rot_dim, r->layout == DYNINFER_ROPE_HALF};
    return 0;
}

int same_place(const dyninfer_rows_t* a, const dyninfer_rows_t* b) {
    return a->data == b->data && a->token_stride == b->token_stride && a->head_stride == b->head_stride;
}

// First and last byte of rows, and whether two sets of rows may meet.
bool meet(const dyninfer_rows_t* a, const dyninfer_rows_t* b, uint32_t tokens, uint32_t dim) {
    if (!tokens) return false;
    auto span = [&](const dyninfer_rows_t* r) {
        const uint64_t e = r->dtype == DYNINFER_DTYPE_BF16 ? 2 : 4;
        return e * ((uint64_t)(tokens - 1) * (uint64_t)r->token_stride + (uint64_t)(r->heads - 1) * (uint64_t)r->head_stride + dim);
    };
    const uintptr_t x = (uintptr_t)a->data, y = (uintptr_t)b->data;
    return x < y + span(b) && y < x + span(a);
}

// Whether the elements of two sets of rows lie apart although their spans meet:
// slices of one fused tensor (equal strides, another range of heads).
bool interleaved(const dyninfer_rows_t* a, const dyninfer_rows_t* b, uint32_t dim) {
    if (a->dtype != b->dtype || a->token_stride != b->token_stride) return false;
    const int64_t e = a->dtype == DYNINFER_DTYPE_BF16 ? 2 : 4;
    const dyninfer_rows_t *lo = a, *hi = b;
    if ((uintptr_t)lo->data > (uintptr_t)hi->data) std::swap(lo, hi);
    const uint64_t gap = ((uintptr_t)hi->data - (uintptr_t)lo->data);
    const uint64_t lo_row = (uint64_t)e * ((lo->heads - 1) * (uint64_t)lo->head_stride + dim);
    const uint64_t hi_row = (uint64_t)e * ((hi->heads - 1) * (uint64_t)hi->head_stride + dim);
    return gap >= lo_row && gap + hi_row <= (uint64_t)e * (uint64_t)lo->token_stride;
}

// y (out of x) may be x, or lie apart from it.
int check_apart(const dyninfer_rows_t* x, const dyninfer_rows_t* y, uint32_t tokens, uint32_t dim, const char* what) {
    if (same_place(x, y) || !meet(x, y, tokens, dim) || interleaved(x, y, dim)) return 0;
    return fail(BAD, std::string(what) + " overlaps its input");
}

int check_workspace(const void* p, uint64_t bytes, uint64_t need, const char* what) {
    if (!need) return 0;
    if (!p || bytes < need)
        return fail(BAD, std::string(what) + " needs a device workspace of " + std::to_string(need) + " bytes (got " +
                             (p ? std::to_string(bytes) + " bytes" : std::string("NULL")) + ")");
    if (!aligned(p, 256)) return fail(BAD, std::string("the workspace of ") + what + " must be 256-byte aligned");
    return 0;
}

int launched(hipError_t e) {
    if (e == dmx::kTooManyThreads)
        return fail(UNSUPPORTED, "the call needs 2^32 threads or more in a launch; split it");
    return e == hipSuccess ? DYNINFER_MI355X_OK : hip_fail(e, "kernel launch");
}

}  // namespace

extern "C" {

int dyninfer_mi355x_rope_table(dyninfer_mi355x_ctx_t* ctx, const dyninfer_rope_params_t* p, uint32_t positions,
                               float* table, void* stream) {
    if (int rc = check_ctx(ctx)) return rc;
    if (!p) return fail(BAD, "rope parameters are NULL");
    if (p->rot_dim < 2 || p->rot_dim % 2 || p->rot_dim > 256) return fail(BAD, "rot_dim must be even, 2..256");
    if (!(p->theta > 1.0) || !std::isfinite(p->theta)) return fail(BAD, "theta must be above 1");
    double lo = 0, hi = 0, attn = 1;
    if (p->scaling > DYNINFER_ROPE_BANDS) return fail(BAD, "unknown rope scaling");
    if (p->scaling != DYNINFER_ROPE_PLAIN && (!(p->factor > 0) || !std::isfinite(p->factor)))
        return fail(BAD, "factor must be above 0");
    if (p->scaling >= DYNINFER_ROPE_YARN && (!(p->original_length > 0) || !std::isfinite(p->original_length)))
        return fail(BAD, "original_length must be above 0");
    if (p->scaling == DYNINFER_ROPE_YARN) {
        if (!(p->beta_slow > 0) || !(p->beta_fast > p->beta_slow)) return fail(BAD, "beta_fast must be above beta_slow, above 0");
        if (!(p->attn_factor >= 0) || !std::isfinite(p->attn_factor)) return fail(BAD, "attn_factor must not be negative");
        // the pair that makes `beta` turns over the original length
        auto pair = [&](double beta) {
            return p->rot_dim * std::log(p->original_length / (beta * 2 * M_PI)) / (2 * std::log(p->theta));
        };
        lo = std::fmax(std::floor(pair(p->beta_fast)), 0);
        hi = std::fmin(std::ceil(pair(p->beta_slow)), p->rot_dim - 1.0);
        attn = p->attn_factor > 0 ? p->attn_factor : p->factor > 1 ? 0.1 * std::log(p->factor) + 1 : 1;
    } else if (p->scaling == DYNINFER_ROPE_BANDS) {
        if (!(p->low_turns >= 0) || !(p->high_turns > p->low_turns)) return fail(BAD, "high_turns must be above low_turns");
        lo = p->low_turns;
        hi = p->high_turns;
    }
    if (positions == 0) return DYNINFER_MI355X_OK;
    if (!table || !aligned(table, 16)) return fail(BAD, "rope table is NULL or not 16-byte aligned");
    DeviceGuard g(ctx->device);
    if (g.err != hipSuccess) return hip_fail(g.err, "hipSetDevice");
    return launched(dmx::rope_table_launch(p->rot_dim, p->scaling, p->theta, p->factor, p->original_length, lo, hi, attn,
                                           positions, table, static_cast<hipStream_t>(stream)));
}

int dyninfer_mi355x_rope(dyninfer_mi355x_ctx_t* ctx, const dyninfer_rows_t* x, const dyninfer_rows_t* y,
                         uint32_t tokens, uint32_t head_dim, const dyninfer_rope_t* rope, void* stream) {
    if (int rc = check_ctx(ctx)) return rc;
    if (int rc = check_dim(head_dim)) return rc;
    dmx::RopeView rp;
    if (int rc = check_rope(rope, head_dim, tokens, rp)) return rc;
    if (tokens == 0) return DYNINFER_MI355X_OK;
    dmx::KvRows in, out;
    if (int rc = check_rows(x, "x", in)) return rc;
    if (int rc = check_out(y, head_dim, tokens, "y", out)) return rc;
    if (x->dtype != y->dtype || x->heads != y->heads) return fail(BAD, "x and y must share dtype and heads");
    if (int rc = check_apart(x, y, tokens, head_dim, "y")) return rc;
    DeviceGuard g(ctx->device);
    if (g.err != hipSuccess) return hip_fail(g.err, "hipSetDevice");
    return launched(dmx::rope_launch(in, out, tokens, x->heads, head_dim, rp, static_cast<hipStream_t>(stream)));
}

int dyninfer_mi355x_kv_cache_bytes(const dyninfer_kvcache_t* cache, uint64_t* k_bytes, uint64_t* v_bytes) {
    if (!k_bytes || !v_bytes) return fail(BAD, "outputs are NULL");
    *k_bytes = *v_bytes = 0;
    if (int rc = check_shape(cache)) return rc;
    *k_bytes = k_total(cache);
    *v_bytes = v_total(cache);
    return DYNINFER_MI355X_OK;
}

int dyninfer_mi355x_kv_append(dyninfer_mi355x_ctx_t* ctx, const dyninfer_kvcache_t* cache,
                              const dyninfer_kvbatch_t* batch, const dyninfer_rows_t* k, const dyninfer_rows_t* v,
                              const dyninfer_rope_t* rope, const dyninfer_rows_t* q, const dyninfer_rows_t* q_out,
                              void* stream) {
    if (int rc = check_ctx(ctx)) return rc;
    dmx::KvView kv;
    dmx::KvBatch b;
    if (int rc = check_cache(cache, kv)) return rc;
    if (int rc = check_batch(batch, true, b)) return rc;
    if ((q || q_out) && !rope) return fail(BAD, "queries are given but no rope to rotate them by");
    if (!q != !q_out) return fail(BAD, "q and q_out go together");
    dmx::RopeView rp = {};
    if (rope)
        if (int rc = check_rope(rope, kv.dim, b.tokens, rp)) return rc;
    if (b.tokens == 0 || b.seqs == 0) return DYNINFER_MI355X_OK;
    dmx::KvRows kr, vr, qr = {}, qo = {};
    if (int rc = check_rows(k, "k", kr)) return rc;
    if (int rc = check_rows(v, "v", vr)) return rc;
    if (k->heads != kv.heads || v->heads != kv.heads) return fail(BAD, "k and v must have the cache's heads");
    if (k->dtype != v->dtype) return fail(BAD, "k and v must share a dtype");
    if (q) {
        if (int rc = check_rows(q, "q", qr)) return rc;
        if (int rc = check_out(q_out, kv.dim, b.tokens, "q_out", qo)) return rc;
        if (q->dtype != q_out->dtype || q->heads != q_out->heads) return fail(BAD, "q and q_out must share dtype and heads");
        if (int rc = check_apart(q, q_out, b.tokens, kv.dim, "q_out")) return rc;
        // its rows are written while k and v are read
        if ((meet(q_out, k, b.tokens, kv.dim) && !interleaved(q_out, k, kv.dim)) ||
            (meet(q_out, v, b.tokens, kv.dim) && !interleaved(q_out, v, kv.dim)))
            return fail(BAD, "q_out overlaps k or v");
    }
    DeviceGuard g(ctx->device);
    if (g.err != hipSuccess) return hip_fail(g.err, "hipSetDevice");
    return launched(dmx::kv_append_launch(kv, b, kr, vr, rp, qr, qo, q ? q->heads : 0, static_cast<hipStream_t>(stream)));
}

int dyninfer_mi355x_kv_read(dyninfer_mi355x_ctx_t* ctx, const dyninfer_kvcache_t* cache,
                            const dyninfer_kvbatch_t* batch, const dyninfer_rows_t* k, const dyninfer_rows_t* v,
                            void* stream) {
    if (int rc = check_ctx(ctx)) return rc;
    dmx::KvView kv;
    dmx::KvBatch b;
    if (int rc = check_cache(cache, kv)) return rc;
    if (int rc = check_batch(batch, true, b)) return rc;
    if (b.tokens == 0 || b.seqs == 0 || (!k && !v)) return DYNINFER_MI355X_OK;
    dmx::KvRows kr = {}, vr = {};
    if (k)
        if (int rc = check_out(k, kv.dim, b.tokens, "k", kr)) return rc;
    if (v)
        if (int rc = check_out(v, kv.dim, b.tokens, "v", vr)) return rc;
    if ((k && k->heads != kv.heads) || (v && v->heads != kv.heads)) return fail(BAD, "k and v must have the cache's heads");
    if (k && v && meet(k, v, b.tokens, kv.dim) && !interleaved(k, v, kv.dim)) return fail(BAD, "k and v overlap");
    DeviceGuard g(ctx->device);
    if (g.err != hipSuccess) return hip_fail(g.err, "hipSetDevice");
    return launched(dmx::kv_read_launch(kv, b, kr, vr, static_cast<hipStream_t>(stream)));
}

int dyninfer_mi355x_kv_commit(dyninfer_mi355x_ctx_t* ctx, const dyninfer_kvcache_t* cache,
                              const dyninfer_kvbatch_t* batch, const int32_t* path, uint32_t path_stride,
                              const int32_t* counts, void* stream) {
    if (int rc = check_ctx(ctx)) return rc;
    dmx::KvView kv;
    dmx::KvBatch b;
    if (int rc = check_cache(cache, kv)) return rc;
    if (int rc = check_batch(batch, true, b)) return rc;
    if (b.tokens == 0 || b.seqs == 0) return DYNINFER_MI355X_OK;
    if ((path_stride && !path) || !counts || !aligned(path, 4) || !aligned(counts, 4))
        return fail(BAD, "path / counts are NULL or misaligned");
    DeviceGuard g(ctx->device);
    if (g.err != hipSuccess) return hip_fail(g.err, "hipSetDevice");
    return launched(dmx::kv_commit_launch(kv, b, path, path_stride, counts, static_cast<hipStream_t>(stream)));
}

int dyninfer_mi355x_tree_attention_workspace_bytes(const dyninfer_kvcache_t* cache, const dyninfer_kvbatch_t* batch,
                                                   uint32_t q_heads, uint32_t dtype, uint64_t* out_bytes) {
    if (!out_bytes) return fail(BAD, "out_bytes is NULL");
    *out_bytes = 0;
    dmx::KvBatch b;
    if (int rc = check_shape(cache)) return rc;
    if (int rc = check_batch(batch, false, b)) return rc;
    if (dtype != DYNINFER_DTYPE_F32 && dtype != DYNINFER_DTYPE_BF16) return fail(UNSUPPORTED, "q must be f32 or bf16");
    if (q_heads == 0 || q_heads % cache->kv_heads) return fail(BAD, "query heads must be a multiple of the kv heads");
    if (b.tokens == 0 || b.seqs == 0 || b.max_new == 0) return DYNINFER_MI355X_OK;
    dmx::KvView kv = {};
    kv.heads = cache->kv_heads;
    kv.dim = cache->head_dim;
    for (bool chain : {false, true})  // enough with a mask and without
        *out_bytes = std::max(*out_bytes, dmx::attn_plan(kv, b, batch->max_length, q_heads, dtype == DYNINFER_DTYPE_BF16, chain).bytes);
    return DYNINFER_MI355X_OK;
}

int dyninfer_mi355x_tree_attention(dyninfer_mi355x_ctx_t* ctx, const dyninfer_kvcache_t* cache,
                                   const dyninfer_kvbatch_t* batch, const dyninfer_rows_t* q, const int64_t* mask,
                                   uint32_t mask_words, float scale, const dyninfer_rows_t* out, float* lse,
                                   void* workspace, uint64_t workspace_bytes, void* stream) {
    if (int rc = check_ctx(ctx)) return rc;
    dmx::AttnArgs a = {};
    if (int rc = check_cache(cache, a.kv)) return rc;
    if (int rc = check_batch(batch, true, a.b)) return rc;
    if (a.b.tokens == 0 || a.b.seqs == 0 || a.b.max_new == 0) return DYNINFER_MI355X_OK;
    if (int rc = check_rows(q, "q", a.q)) return rc;
    if (int rc = check_out(out, a.kv.dim, a.b.tokens, "out", a.out)) return rc;
    if (q->dtype != out->dtype || q->heads != out->heads) return fail(BAD, "q and out must share dtype and heads");
    if (meet(q, out, a.b.tokens, a.kv.dim) && !interleaved(q, out, a.kv.dim)) return fail(BAD, "out overlaps q");
    if (q->heads % a.kv.heads) return fail(BAD, "query heads must be a multiple of the kv heads");
    if (q->heads > 65535) return fail(UNSUPPORTED, "more than 65535 query heads");
    if (mask && !aligned(mask, 8)) return fail(BAD, "mask must be 8-byte aligned");
    if (mask && (uint64_t)mask_words * 64 < a.b.max_new) return fail(BAD, "mask has fewer bits than max_new");
    if (lse && !aligned(lse, 4)) return fail(BAD, "lse must be 4-byte aligned");
    if (!std::isfinite(scale)) return fail(BAD, "scale must be finite");
    a.group = q->heads / a.kv.heads;
    if ((uint64_t)a.b.max_new * a.group > 0x7FFFFFFFull) return fail(UNSUPPORTED, "too many rows of one kv head");
    const dmx::AttnPlan plan = dmx::attn_plan(a.kv, a.b, batch->max_length, q->heads, a.q.bf16, !mask);
    if (int rc = check_workspace(workspace, workspace_bytes, plan.bytes, "tree_attention")) return rc;
    a.mask = mask;
    a.mask_words = mask_words;
    a.lse = lse;
    a.scale = scale;
    DeviceGuard g(ctx->device);
    if (g.err != hipSuccess) return hip_fail(g.err, "hipSetDevice");
    return launched(dmx::attn_launch(a, plan, static_cast<uint8_t*>(workspace), static_cast<hipStream_t>(stream)));
}

int dyninfer_mi355x_draft_verify_workspace_bytes(uint32_t sequences, uint32_t tokens, uint32_t vocab, uint32_t max_new,
                                                 uint64_t* out_bytes) {
    if (!out_bytes) return fail(BAD, "out_bytes is NULL");
    *out_bytes = 0;
    if (vocab == 0) return fail(BAD, "vocab must be above 0");
    if (max_new > tokens) return fail(BAD, "max_new must not be above tokens");
    *out_bytes = dmx::verify_workspace_bytes(sequences, tokens, vocab);
    return DYNINFER_MI355X_OK;
}

int dyninfer_mi355x_draft_verify(dyninfer_mi355x_ctx_t* ctx, const dyninfer_verify_t* v, void* workspace,
                                 uint64_t workspace_bytes, void* stream) {
    if (int rc = check_ctx(ctx)) return rc;
    if (!v) return fail(BAD, "arguments are NULL");
    if (v->vocab == 0 || v->vocab > 0x7FFFFFFFu) return fail(BAD, "vocab must be 1..2^31 - 1");
    if (v->tokens > 0x7FFFFFFFu || v->max_new > v->tokens)
        return fail(BAD, "max_new must not be above tokens, nor tokens above 2^31 - 1");
    if (v->sequences == 0) return DYNINFER_MI355X_OK;
    auto float_type = [](uint32_t t) { return t == DYNINFER_DTYPE_F32 || t == DYNINFER_DTYPE_BF16; };
    if (!float_type(v->logits_dtype) || (v->draft_probs && !float_type(v->probs_dtype)))
        return fail(UNSUPPORTED, "logits and draft_probs must be f32 or bf16");
    auto size = [](uint32_t t) { return t == DYNINFER_DTYPE_BF16 ? 2u : 4u; };
    // without rows (max_new 0) path has no elements
    if (!v->starts || !aligned(v->starts, 4) || (v->max_new && !v->path) || !aligned(v->path, 4) || !v->counts ||
        !aligned(v->counts, 4) || !v->next_token || !aligned(v->next_token, 8) || (v->temperature && !aligned(v->temperature, 4)))
        return fail(BAD, "starts, temperature or an output is NULL or misaligned");
    if (!v->noise || !aligned(v->noise, 4)) return fail(BAD, "noise is NULL or misaligned");
    if (v->noise_stride < (int64_t)v->vocab && v->sequences > 1) return fail(BAD, "noise rows overlap");
    if (v->tokens) {
        if (!v->logits || !aligned(v->logits, size(v->logits_dtype))) return fail(BAD, "logits are NULL or misaligned");
        if (v->draft_probs && !aligned(v->draft_probs, size(v->probs_dtype))) return fail(BAD, "draft_probs are misaligned");
        if (v->tokens > 1 && (v->logits_stride < (int64_t)v->vocab || (v->draft_probs && v->probs_stride < (int64_t)v->vocab)))
            return fail(BAD, "rows of logits or draft_probs overlap");
        if (!v->draft_tokens || !aligned(v->draft_tokens, 8) || !v->uniform || !aligned(v->uniform, 4) ||
            (v->parents && !aligned(v->parents, 4)))
            return fail(BAD, "draft_tokens, uniform or parents are NULL or misaligned");
    }
    const uint64_t need = dmx::verify_workspace_bytes(v->sequences, v->tokens, v->vocab);
    if (int rc = check_workspace(workspace, workspace_bytes, need, "draft_verify")) return rc;
    dmx::VerifyArgs a = {};
    a.logits = v->logits;
    a.probs = v->draft_probs;
    a.logits_stride = v->logits_stride;
    a.probs_stride = v->probs_stride;
    a.noise_stride = v->noise_stride;
    a.logits_bf16 = v->logits_dtype == DYNINFER_DTYPE_BF16;
    a.probs_bf16 = v->probs_dtype == DYNINFER_DTYPE_BF16;
    a.tokens_in = v->draft_tokens;
    a.parents = v->parents;
    a.starts = v->starts;
    a.temperature = v->temperature;
    a.uniform = v->uniform;
    a.noise = v->noise;
    a.vocab = v->vocab;
    a.seqs = v->sequences;
    a.tokens = v->tokens;
    a.max_new = v->max_new;
    a.path = v->path;
    a.counts = v->counts;
    a.next = v->next_token;
    DeviceGuard g(ctx->device);
    if (g.err != hipSuccess) return hip_fail(g.err, "hipSetDevice");
    return launched(dmx::verify_launch(a, static_cast<uint8_t*>(workspace), static_cast<hipStream_t>(stream)));
}

}  // extern "C"
