// C-ABI of attention heads and of the paged cache: norms with rotation, cache
// appends and attention.  Checks on the host, kernels on the caller's stream.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/minirun_hip.h"
#include "capi_util.hpp"
#include "mr_kernels.hpp"

namespace {

using mrc::fail;
using mrc::hip_fail;

constexpr int64_t FAR = int64_t(1) << 40;   // the longest stride, in elements
constexpr int64_t PITCH = int64_t(1) << 32;  // a cache's pages lie nearer, in bytes
constexpr int64_t MOST = int64_t(1) << 30;  // keys of a sequence, rows of queries: the kernels count past them in 32 bits

bool act(mr_dtype d) { return d == MR_BF16 || d == MR_F32; }
int size_of(mr_dtype d) { return d == MR_F32 ? 4 : 2; }
bool elem_aligned(const void* p, mr_dtype d) { return reinterpret_cast<uintptr_t>(p) % size_of(d) == 0; }
mr_status done(hipError_t e, const char* what) { return e == hipSuccess ? MR_OK : hip_fail(e, what); }
// nothing lies a stride away along an axis of one entry
int64_t stride_of(int64_t entries, int64_t stride) { return entries > 1 ? stride : 0; }
bool stride_in(int64_t s) { return s >= 0 && s <= FAR; }

int64_t lanes_of(int dim) {
    int64_t n = 1;
    while (8 * n < dim) n *= 2;
    return n;
}

// [tokens][heads][dim] that is written: no two rows meet, whichever axis is the outer one
bool rows_apart(int64_t tokens, int64_t heads, int64_t dim, int64_t ts, int64_t hs) {
    if (!stride_in(ts) || !stride_in(hs)) return false;
    if (tokens == 1) return heads == 1 || hs >= dim;
    if (heads == 1) return ts >= dim;
    return hs <= ts ? hs >= dim && ts >= hs * (heads - 1) + dim : ts >= dim && hs >= ts * (tokens - 1) + dim;
}

mr_status check_rope(const char* what, const mr_rotary& r, int64_t tokens, int dim, mr::HeadRope& out) {
    out = mr::HeadRope{};
    if (r.dim == 0) return MR_OK;
    if (r.dim < 0 || r.dim % 2 || r.col0 < 0 || r.col0 > dim - r.dim)
        return fail(MR_INVALID_SHAPE, "%s: rotated columns %d .. %d + %d of heads of %d (an even number inside the head)", what,
                    r.col0, r.col0, r.dim, dim);
    if (r.pairs != MR_ROPE_ADJACENT && r.pairs != MR_ROPE_HALVES)
        return fail(MR_INVALID_ARGUMENT, "%s: rotary pairs %d", what, (int)r.pairs);
    if (r.table_rows <= 0 || r.table_rows > INT32_MAX || (!r.positions && r.table_rows < tokens))
        return fail(MR_INVALID_SHAPE, "%s: rotary tables of %lld rows for %lld tokens%s", what, (long long)r.table_rows,
                    (long long)tokens, r.positions ? "" : " without positions");
    if (!r.cos_t || !r.sin_t || !mrc::aligned4(r.cos_t) || !mrc::aligned4(r.sin_t) || !mrc::aligned4(r.positions))
        return fail(MR_INVALID_ARGUMENT, "%s: NULL or misaligned rotary tables or positions", what);
    out = mr::HeadRope{r.cos_t, r.sin_t, r.positions, r.table_rows, r.dim / 2, r.col0, r.pairs == MR_ROPE_HALVES};
    return MR_OK;
}

mr_status check_eps(const char* what, float eps) {
    return eps >= 0 && std::isfinite(eps) ? MR_OK : fail(MR_INVALID_ARGUMENT, "%s: eps must be finite, >= 0", what);
}

mr_status head_norm_sizes(const mr_head_norm_args* a, const char* what) {
    if (a->tokens < 0 || a->dim < 1 || a->dim > 512 || a->q.heads < 0 || a->k.heads < 0 ||
        int64_t(a->q.heads) + a->k.heads < 1)
        return fail(MR_INVALID_SHAPE, "%s: %d tokens of %d + %d heads of %d (1 to 512)", what, a->tokens, a->q.heads, a->k.heads,
                    a->dim);
    const int64_t heads = int64_t(a->q.heads) + a->k.heads;
    if (heads > INT32_MAX || a->tokens * heads > INT32_MAX ||
        a->tokens * heads * lanes_of(a->dim) >= (int64_t(1) << 32) - 1024)
        return fail(MR_INVALID_SHAPE, "%s: %d tokens of %lld heads are more than one launch takes", what, a->tokens,
                    (long long)heads);
    return MR_OK;
}

mr_status head_norm(const mr_head_norm_args* a, bool backward, void* stream) {
    const char* what = backward ? "head norm backward" : "head norm";
    if (!a) return fail(MR_INVALID_ARGUMENT, "%s: args is NULL", what);
    mr_status st = head_norm_sizes(a, what);
    if (st != MR_OK) return st;
    if (!act(a->x_dtype) || !act(a->out_dtype) || !act(a->weight_dtype))
        return fail(MR_INVALID_DTYPE, "%s: types must be bf16 or f32, got x %s, weight %s, out %s", what,
                    mrc::dtype_name(a->x_dtype), mrc::dtype_name(a->weight_dtype), mrc::dtype_name(a->out_dtype));
    if ((st = check_eps(what, a->eps)) != MR_OK) return st;
    mr::HeadNormParams p{};
    if ((st = check_rope(what, a->rope, a->tokens, a->dim, p.rope)) != MR_OK) return st;
    const mr_head_rows* rows[2] = {&a->q, &a->k};
    bool weights = false;
    for (int i = 0; i < 2; ++i) {
        const mr_head_rows& r = *rows[i];
        mr::HeadSegment& s = p.seg[i];
        s.heads = r.heads;
        s.dw = backward ? r.d_weight : nullptr;  // (also without heads: zeros)
        weights = weights || s.dw;
        if (!mrc::aligned4(s.dw)) return fail(MR_INVALID_ARGUMENT, "%s: a misaligned weight", what);
        if (!r.heads) continue;
        s.w = r.weight;
        if (!elem_aligned(r.weight, a->weight_dtype)) return fail(MR_INVALID_ARGUMENT, "%s: a misaligned weight", what);
        if (!a->tokens) continue;
        if (!r.x || !r.out || (backward && !r.d_out)) return fail(MR_INVALID_ARGUMENT, "%s: NULL rows", what);
        if (!elem_aligned(r.x, a->x_dtype) || !elem_aligned(r.out, a->out_dtype) ||
            (backward && !elem_aligned(r.d_out, a->x_dtype)))
            return fail(MR_INVALID_ARGUMENT, "%s: misaligned rows", what);
        s.x = r.x;
        s.x_ts = stride_of(a->tokens, r.x_token_stride);
        s.x_hs = stride_of(r.heads, r.x_head_stride);
        s.out = r.out;
        s.out_ts = stride_of(a->tokens, r.out_token_stride);
        s.out_hs = stride_of(r.heads, r.out_head_stride);
        if (backward) {
            s.dy = r.d_out;
            s.dy_ts = stride_of(a->tokens, r.d_out_token_stride);
            s.dy_hs = stride_of(r.heads, r.d_out_head_stride);
        }
        if (!stride_in(s.x_ts) || !stride_in(s.x_hs) || !stride_in(s.dy_ts) || !stride_in(s.dy_hs))
            return fail(MR_INVALID_ARGUMENT, "%s: strides must be 0 to 2^40", what);
        if (!rows_apart(a->tokens, r.heads, a->dim, s.out_ts, s.out_hs))
            return fail(MR_INVALID_ARGUMENT, "%s: strides %lld and %lld of the output make rows of %d meet", what,
                        (long long)r.out_token_stride, (long long)r.out_head_stride, a->dim);
    }
    if (p.seg[0].dw && p.seg[0].dw == p.seg[1].dw)
        return fail(MR_INVALID_ARGUMENT, "%s: one d_weight for queries and keys (it is written, not added to)", what);
    p.tokens = a->tokens;
    p.dim = a->dim;
    p.x_f32 = a->x_dtype == MR_F32;
    p.w_f32 = a->weight_dtype == MR_F32;
    p.out_f32 = a->out_dtype == MR_F32;
    p.eps = a->eps;
    if (backward) {
        mr::head_norm_blocks(a->tokens, {a->q.heads, a->k.heads}, a->dim, p.blocks);
        if (weights) {
            const size_t need = mr_head_norm_rope_backward_workspace_size(a);
            if (a->workspace_bytes < need)
                return fail(MR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu needed", what, a->workspace_bytes, need);
            if (need && (!a->workspace || !mrc::aligned4(a->workspace)))
                return fail(MR_INVALID_ARGUMENT, "%s: NULL or misaligned workspace", what);
            p.partial = (float*)a->workspace;
        }
    }
    if (!a->tokens && !weights) return MR_OK;
    return done(mr::launch_head_norm(p, backward, (hipStream_t)stream), backward ? "head norm backward launch" : "head norm launch");
}

mr_status check_cache(const char* what, const mr_kv_cache& c) {
    if (c.pages < 0 || c.page_size <= 0 || c.page_size % 16 || c.kv_heads <= 0 || c.head_dim <= 0 || c.head_dim > 256 ||
        c.head_dim % 32)
        return fail(MR_INVALID_SHAPE,
                    "%s: %d pages of %d rows of %d heads of %d (rows a multiple of 16, heads a multiple of 32 up to 256)", what,
                    c.pages, c.page_size, c.kv_heads, c.head_dim);
    if (int64_t(c.page_size) * c.kv_heads > (int64_t(1) << 28) / c.head_dim || int64_t(c.pages) * c.page_size > INT32_MAX)
        return fail(MR_INVALID_SHAPE, "%s: pages of more than 2^28 values, or 2^31 rows or more in all", what);
    const bool mx = c.k_scales || c.v_scales;
    const int64_t rows = int64_t(c.page_size) * c.kv_heads;
    if (c.pages > 1 && (c.page_stride < rows * c.head_dim / (mx ? 8 : 1) || c.page_stride >= (mx ? PITCH / 4 : PITCH / 2) ||
                        c.page_stride % (mx ? 4 : 8) ||
                        (mx && (c.scale_page_stride < rows * c.head_dim / 32 || c.scale_page_stride >= PITCH))))
        return fail(MR_INVALID_ARGUMENT, "%s: pages must be apart, by a multiple of 16 bytes below 2^32", what);
    if (c.pages && (!c.k || !c.v || (mx && (!c.k_scales || !c.v_scales)) || !mrc::aligned16(c.k) || !mrc::aligned16(c.v)))
        return fail(MR_INVALID_ARGUMENT, "%s: NULL or misaligned cache (16 bytes)", what);
    return MR_OK;
}

// What the sizes of an attention call decide; MR_OK and a route, or why not
mr_status attention_route(const mr_kv_attention_args* a, mr::KvAttnRoute& r) {
    const char* what = "kv attention";
    const mr_kv_cache& c = a->cache;
    mr_status st = check_cache(what, c);
    if (st != MR_OK) return st;
    if (a->batch < 0 || a->tokens < 0 || a->heads <= 0 || a->heads % c.kv_heads || int64_t(a->tokens) * a->heads > MOST)
        return fail(MR_INVALID_SHAPE, "%s: %d sequences, %d tokens of %d heads over %d key heads", what, a->batch, a->tokens,
                    a->heads, c.kv_heads);
    if (!a->q_offsets && a->tokens != a->batch)
        return fail(MR_INVALID_SHAPE, "%s: %d tokens of %d sequences need q_offsets", what, a->tokens, a->batch);
    if (a->max_pages < 0 || int64_t(a->max_pages) * c.page_size > MOST || a->max_kv_len < 0 || a->window < 0)
        return fail(MR_INVALID_SHAPE, "%s: %d pages a sequence, %d keys, window %d", what, a->max_pages, a->max_kv_len, a->window);
    const int64_t holds = int64_t(a->max_pages) * c.page_size;
    const int64_t keys = a->max_kv_len ? std::min<int64_t>(a->max_kv_len, holds) : holds;
    if (!a->batch || !a->tokens) {
        r = mr::KvAttnRoute{false, 16, 0, 1, 64, 256};
        return MR_OK;
    }
    r = mr::kv_attention_route(a->tokens, a->batch, a->q_offsets != nullptr, c.kv_heads, a->heads / c.kv_heads, c.head_dim,
                               a->window, keys, mrc::cu_count());
    if (r.tiles * c.kv_heads * r.splits >= (int64_t(1) << 32) / r.threads)
        return fail(MR_INVALID_SHAPE, "%s: %lld tiles of %d key heads are more than one launch takes", what, (long long)r.tiles,
                    c.kv_heads);
    return MR_OK;
}

}  // namespace

extern "C" {

mr_status mr_head_norm_rope(const mr_head_norm_args* a, void* stream) { return head_norm(a, false, stream); }

size_t mr_head_norm_rope_backward_workspace_size(const mr_head_norm_args* a) {
    if (!a || head_norm_sizes(a, "head norm backward") != MR_OK) return 0;
    int blocks[2];
    mr::head_norm_blocks(a->tokens, {a->q.heads, a->k.heads}, a->dim, blocks);
    return size_t(blocks[0] + blocks[1]) * a->dim * sizeof(float);
}

mr_status mr_head_norm_rope_backward(const mr_head_norm_args* a, void* stream) { return head_norm(a, true, stream); }

mr_status mr_kv_append(const mr_kv_append_args* a, void* stream) {
    const char* what = "kv append";
    if (!a) return fail(MR_INVALID_ARGUMENT, "%s: args is NULL", what);
    const mr_kv_cache& c = a->cache;
    mr_status st = check_cache(what, c);
    if (st != MR_OK) return st;
    if (a->tokens < 0 || int64_t(a->tokens) * c.kv_heads > INT32_MAX / lanes_of(c.head_dim))
        return fail(MR_INVALID_SHAPE, "%s: %d tokens of %d heads are more than one launch takes", what, a->tokens, c.kv_heads);
    if (!act(a->dtype) || (a->normalize && !act(a->norm_w_dtype)))
        return fail(MR_INVALID_DTYPE, "%s: keys, values and norm weights must be bf16 or f32, got %s and %s", what,
                    mrc::dtype_name(a->dtype), mrc::dtype_name(a->norm_w_dtype));
    if (a->normalize && (st = check_eps(what, a->eps)) != MR_OK) return st;
    mr::KvAppendParams p{};
    if ((st = check_rope(what, a->rope, a->tokens, c.head_dim, p.rope)) != MR_OK) return st;
    if (!a->tokens) return MR_OK;
    if (!a->k || !a->v || !a->slots) return fail(MR_INVALID_ARGUMENT, "%s: k, v and slots must be non-NULL", what);
    if (!elem_aligned(a->k, a->dtype) || !elem_aligned(a->v, a->dtype) || !mrc::aligned4(a->slots) ||
        (a->normalize && !elem_aligned(a->norm_w, a->norm_w_dtype)))
        return fail(MR_INVALID_ARGUMENT, "%s: a misaligned pointer", what);
    p.k_ts = stride_of(a->tokens, a->k_token_stride);
    p.k_hs = stride_of(c.kv_heads, a->k_head_stride);
    p.v_ts = stride_of(a->tokens, a->v_token_stride);
    p.v_hs = stride_of(c.kv_heads, a->v_head_stride);
    if (!stride_in(p.k_ts) || !stride_in(p.k_hs) || !stride_in(p.v_ts) || !stride_in(p.v_hs))
        return fail(MR_INVALID_ARGUMENT, "%s: strides must be 0 to 2^40", what);
    if (!c.pages) return MR_OK;
    p.k = a->k;
    p.v = a->v;
    p.tokens = a->tokens;
    p.heads = c.kv_heads;
    p.dim = c.head_dim;
    p.f32 = a->dtype == MR_F32;
    p.slots = a->slots;
    p.slot_end = c.pages * c.page_size;
    p.page_size = c.page_size;
    p.norm = a->normalize != 0;
    p.w = a->normalize ? a->norm_w : nullptr;
    p.w_f32 = a->norm_w_dtype == MR_F32;
    p.eps = a->eps;
    p.k_pages = c.k;
    p.v_pages = c.v;
    p.k_scales = c.k_scales;
    p.v_scales = c.v_scales;
    p.page_stride = c.pages > 1 ? c.page_stride : 0;
    p.scale_stride = c.pages > 1 ? c.scale_page_stride : 0;
    return done(mr::launch_kv_append(p, (hipStream_t)stream), "kv append launch");
}

size_t mr_kv_attention_workspace_size(const mr_kv_attention_args* a) {
    mr::KvAttnRoute r;
    if (!a || attention_route(a, r) != MR_OK) return 0;
    return mr::kv_attention_workspace(r, a->tokens, a->heads, a->cache.head_dim);
}

mr_status mr_kv_attention(const mr_kv_attention_args* a, void* stream) {
    const char* what = "kv attention";
    if (!a) return fail(MR_INVALID_ARGUMENT, "%s: args is NULL", what);
    const mr_kv_cache& c = a->cache;
    mr::KvAttnRoute r;
    mr_status st = attention_route(a, r);
    if (st != MR_OK) return st;
    if (!act(a->out_dtype))
        return fail(MR_INVALID_DTYPE, "%s: out must be bf16 or f32, got %s", what, mrc::dtype_name(a->out_dtype));
    if (!(a->scale > 0) || !std::isfinite(a->scale * 1.4426950408889634f)) return fail(MR_INVALID_SHAPE, "%s: scale must be finite, > 0", what);
    if (!a->tokens || !a->batch) return MR_OK;
    if (!a->q || !a->out || !a->kv_lens || (a->max_pages && !a->page_table))
        return fail(MR_INVALID_ARGUMENT, "%s: q, out, kv_lens and page_table must be non-NULL", what);
    const int64_t q_ts = stride_of(a->tokens, a->q_token_stride), q_hs = stride_of(a->heads, a->q_head_stride);
    const int64_t out_ts = stride_of(a->tokens, a->out_token_stride), out_hs = stride_of(a->heads, a->out_head_stride);
    if (!mrc::aligned16(a->q) || !mrc::aligned16(a->out) || q_ts % 8 || q_hs % 8 || out_ts % 8 || out_hs % 8)
        return fail(MR_INVALID_ARGUMENT, "%s: q and out must be 16-byte aligned, their strides multiples of 8", what);
    if (!stride_in(q_ts) || !stride_in(q_hs) || !rows_apart(a->tokens, a->heads, c.head_dim, out_ts, out_hs))
        return fail(MR_INVALID_ARGUMENT, "%s: strides of q must be 0 to 2^40, and rows of out apart", what);
    if (!mrc::aligned4(a->page_table) || !mrc::aligned4(a->kv_lens) || !mrc::aligned4(a->q_offsets) ||
        !mrc::aligned4(a->sinks) || !mrc::aligned4(a->lse) ||
        (a->batch > 1 && (a->page_table_stride < 0 || a->page_table_stride > FAR)))
        return fail(MR_INVALID_ARGUMENT, "%s: a misaligned pointer, or a page table stride outside 0 to 2^40", what);
    const size_t need = mr::kv_attention_workspace(r, a->tokens, a->heads, c.head_dim);
    if (a->workspace_bytes < need)
        return fail(MR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu needed", what, a->workspace_bytes, need);
    if (need && (!a->workspace || !mrc::aligned16(a->workspace)))
        return fail(MR_INVALID_ARGUMENT, "%s: NULL or misaligned workspace (16 bytes)", what);
    mr::KvAttnParams p{};
    p.q = (const uint16_t*)a->q;
    p.q_ts = q_ts;
    p.q_hs = q_hs;
    p.k = (const char*)c.k;
    p.v = (const char*)c.v;
    p.k_scales = c.k_scales;
    p.v_scales = c.v_scales;
    p.page_bytes = c.pages > 1 ? (uint32_t)(c.page_stride * (c.k_scales ? 4 : 2)) : 0;
    p.scale_bytes = c.pages > 1 ? (uint32_t)c.scale_page_stride : 0;
    p.pages = c.pages;
    p.page_size = c.page_size;
    p.kv_heads = c.kv_heads;
    p.group = a->heads / c.kv_heads;
    p.dim = c.head_dim;
    p.table = a->page_table;
    p.table_stride = a->page_table_stride;
    p.max_keys = c.pages ? a->max_pages * c.page_size : 0;  // (without pages nothing is read)
    p.lens = a->kv_lens;
    p.q_offsets = a->q_offsets;
    p.batch = a->batch;
    p.tokens = a->tokens;
    p.window = a->window < int64_t(a->max_pages) * c.page_size ? a->window : 0;  // (a longer one hides nothing)
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.sinks = a->sinks;
    p.out = a->out;
    p.out_ts = out_ts;
    p.out_hs = out_hs;
    p.out_f32 = a->out_dtype == MR_F32;
    p.lse = a->lse;
    p.splits = r.splits;
    p.chunk = r.chunk;
    p.part_o = (float*)a->workspace;
    p.part_ml = p.part_o + size_t(a->tokens) * a->heads * r.splits * c.head_dim;
    return done(mr::launch_kv_attention(p, r, (hipStream_t)stream), "kv attention launch");
}

}  // extern "C"
