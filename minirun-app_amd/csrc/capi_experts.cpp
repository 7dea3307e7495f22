// C-ABI of MXFP4 matrices and of the way of tokens to routed experts and back:
// checks on the host, kernels on the caller's stream.
#include <hip/hip_runtime.h>

#include "../../include/minirun_hip.h"
#include "capi_util.hpp"
#include "mr_kernels.hpp"

namespace {

using mrc::fail;
using mrc::hip_fail;

bool act(mr_dtype d) { return d == MR_BF16 || d == MR_F32; }

mr_status done(hipError_t e, const char* what) { return e == hipSuccess ? MR_OK : hip_fail(e, what); }

// values of a matrix: rows and cols positive, whole blocks, sizes that 64-bit
// byte offsets hold
mr_status check_extent(int64_t rows, int64_t cols, const char* what) {
    if (rows < 0 || cols <= 0 || cols % 32)
        return fail(MR_INVALID_SHAPE, "%s: %lld rows of %lld columns; the columns are blocks of 32", what,
                    (long long)rows, (long long)cols);
    if (rows > 0 && cols > (int64_t(1) << 37) / rows)
        return fail(MR_INVALID_SHAPE, "%s: %lld x %lld values are more than 2^37", what, (long long)rows, (long long)cols);
    return MR_OK;
}

// tokens, slots and row widths that the routing entry points share
mr_status check_rows(int32_t tokens, int32_t per_token, int64_t dim, mr_dtype dtype, const char* what) {
    if (tokens < 0 || per_token <= 0 || int64_t(tokens) * per_token > (1 << 24))
        return fail(MR_INVALID_SHAPE, "%s: %d tokens of %d experts (at most 2^24 pairs)", what, tokens, per_token);
    if (dim <= 0 || dim > (1 << 24)) return fail(MR_INVALID_SHAPE, "%s: rows of %lld values", what, (long long)dim);
    if (!act(dtype)) return fail(MR_INVALID_DTYPE, "%s: rows must be bf16 or f32, got %s", what, mrc::dtype_name(dtype));
    // at most a thread per 8 values, and a wave, for a token (row_launch in
    // experts.hip), in a grid of less than 2^32
    if (int64_t(tokens) * std::max<int64_t>(64, (dim + 7) / 8) >= (int64_t(1) << 32))
        return fail(MR_INVALID_SHAPE, "%s: %d tokens of %lld values are more than one launch takes", what, tokens,
                    (long long)dim);
    return MR_OK;
}

// element pointers on their element's boundary
bool elem_aligned(const void* p, mr_dtype d) { return (reinterpret_cast<uintptr_t>(p) & (d == MR_F32 ? 3 : 1)) == 0; }

bool stride_ok(int64_t stride, int64_t dim) { return stride >= dim && stride <= (int64_t(1) << 40); }

}  // namespace

extern "C" {

mr_status mr_mxfp4_validate(mr_dtype packed_dtype, int32_t packed_rank, const int64_t* packed_shape,
                            mr_dtype scales_dtype, int32_t scales_rank, const int64_t* scales_shape, int64_t* experts,
                            int64_t* rows, int64_t* cols) {
    if (packed_dtype != MR_U32)
        return fail(MR_INVALID_DTYPE, "MXFP4 packed weights must be uint32, got %s", mrc::dtype_name(packed_dtype));
    if (scales_dtype != MR_U8)
        return fail(MR_INVALID_DTYPE, "MXFP4 scales must be uint8 (E8M0), got %s", mrc::dtype_name(scales_dtype));
    if ((packed_rank != 2 && packed_rank != 3) || scales_rank != packed_rank)
        return fail(MR_INVALID_SHAPE, "MXFP4 operands need two equal ranks of 2 or 3 (a stack of experts), got %d and %d",
                    packed_rank, scales_rank);
    if (!packed_shape || !scales_shape) return fail(MR_INVALID_ARGUMENT, "mr_mxfp4_validate: NULL shape");
    const int lead = packed_rank - 2;
    for (int i = 0; i < packed_rank; ++i)
        if (packed_shape[i] < (i == lead ? 0 : 1) || packed_shape[i] > (int64_t(1) << 37))
            return fail(MR_INVALID_SHAPE, "MXFP4 packed weights have an axis of %lld", (long long)packed_shape[i]);
    for (int i = 0; i <= lead; ++i)
        if (packed_shape[i] != scales_shape[i])
            return fail(MR_INVALID_SHAPE, "MXFP4 operands disagree on axis %d: packed %lld, scales %lld", i,
                        (long long)packed_shape[i], (long long)scales_shape[i]);
    const int64_t n = packed_shape[lead + 1] * 8;
    if (n % 32 || scales_shape[lead + 1] != n / 32)
        return fail(MR_INVALID_SHAPE, "MXFP4 rows of %lld values need %lld scales in whole blocks of 32, got %lld",
                    (long long)n, (long long)(n / 32), (long long)scales_shape[lead + 1]);
    if (experts) *experts = lead ? packed_shape[0] : 0;
    if (rows) *rows = packed_shape[lead];
    if (cols) *cols = n;
    return MR_OK;
}

mr_status mr_mxfp4_quantize(const void* x, mr_dtype x_dtype, int64_t rows, int64_t cols, int64_t x_stride,
                            uint32_t* packed, uint8_t* scales, void* stream) {
    const mr_status st = check_extent(rows, cols, "MXFP4 quantization");
    if (st != MR_OK) return st;
    if (!act(x_dtype))
        return fail(MR_INVALID_DTYPE, "MXFP4 quantization: x must be bf16 or f32, got %s", mrc::dtype_name(x_dtype));
    if (rows == 0) return MR_OK;
    if (!x || !packed || !scales) return fail(MR_INVALID_ARGUMENT, "MXFP4 quantization: x, packed and scales must be non-NULL");
    if (!stride_ok(x_stride, cols) || !elem_aligned(x, x_dtype) || !mrc::aligned4(packed))
        return fail(MR_INVALID_ARGUMENT, "MXFP4 quantization: a stride shorter than the rows, or a misaligned pointer");
    mr::Mxfp4QuantizeParams p{x, x_dtype == MR_F32, rows, cols, x_stride, packed, scales};
    return done(mr::launch_mxfp4_quantize(p, (hipStream_t)stream), "MXFP4 quantization launch");
}

mr_status mr_mxfp4_dequantize(const mr_mxfp4_matrix* w, void* out, mr_dtype out_dtype, int64_t out_stride,
                              void* stream) {
    if (!w) return fail(MR_INVALID_ARGUMENT, "MXFP4 dequantization: w is NULL");
    const mr_status st = check_extent(w->rows, w->cols, "MXFP4 dequantization");
    if (st != MR_OK) return st;
    if (!act(out_dtype))
        return fail(MR_INVALID_DTYPE, "MXFP4 dequantization: out must be bf16 or f32, got %s", mrc::dtype_name(out_dtype));
    if (w->rows == 0) return MR_OK;
    if (!w->packed || !w->scales || !out)
        return fail(MR_INVALID_ARGUMENT, "MXFP4 dequantization: packed, scales and out must be non-NULL");
    if (!stride_ok(out_stride, w->cols) || !elem_aligned(out, out_dtype) || !mrc::aligned4(w->packed))
        return fail(MR_INVALID_ARGUMENT, "MXFP4 dequantization: a stride shorter than the rows, or a misaligned pointer");
    mr::Mxfp4DequantizeParams p{w->packed, w->scales, w->rows, w->cols, out, out_dtype == MR_F32, out_stride};
    return done(mr::launch_mxfp4_dequantize(p, (hipStream_t)stream), "MXFP4 dequantization launch");
}

// what the products ask of x, w and y; fills what they share
static mr_status gemm_params(const char* what, const void* x, mr_dtype x_dtype, const uint8_t* x_scales, int64_t x_rows,
                             int64_t x_stride, const mr_mxfp4_matrix* w, int64_t y_rows, void* y, mr_dtype y_dtype,
                             int64_t y_stride, mr::Mxfp4GemmParams& p) {
    const mr_status st = check_extent(w->rows, w->cols, what);
    if (st != MR_OK) return st;
    const bool mx = x_dtype == MR_U32;
    if (w->rows == 0 || w->rows > mr::MXFP4_MAX_OUT || w->cols > (1 << 20))
        return fail(MR_INVALID_SHAPE, "%s: a weight of %lld x %lld (at most 2^22 x 2^20)", what, (long long)w->rows,
                    (long long)w->cols);
    if (x_rows < 0 || x_rows > INT32_MAX) return fail(MR_INVALID_SHAPE, "%s: x has %lld rows", what, (long long)x_rows);
    if ((!mx && !act(x_dtype)) || !act(y_dtype))
        return fail(MR_INVALID_DTYPE, "%s: x must be bf16, f32 or MXFP4 and y bf16 or f32, got %s and %s", what,
                    mrc::dtype_name(x_dtype), mrc::dtype_name(y_dtype));
    if (x_rows == 0 || y_rows == 0) return MR_OK;
    if (!x || (mx && !x_scales) || !w->packed || !w->scales || !y)
        return fail(MR_INVALID_ARGUMENT, "%s: x, w and y must be non-NULL", what);
    const int size = x_dtype == MR_F32 ? 4 : 2;
    if (!mrc::aligned16(x) || !mrc::aligned16(w->packed) || (!mx && x_rows > 1 && x_stride * size % 16))
        return fail(MR_INVALID_ARGUMENT, "%s: x and w->packed must be 16-byte aligned, x's rows a multiple of 16 bytes apart",
                    what);
    // byte offsets of the rows of a tile in 32 bits
    if (!mx && x_rows > 1 && x_stride > (1 << 23) / size)
        return fail(MR_INVALID_ARGUMENT, "%s: rows of x more than 2^23 bytes apart", what);
    if ((!mx && x_rows > 1 && x_stride < w->cols) || (y_rows > 1 && !stride_ok(y_stride, w->rows)) ||
        !elem_aligned(y, y_dtype))
        return fail(MR_INVALID_ARGUMENT, "%s: a stride shorter than the rows, or a misaligned y", what);
    p.x = x;
    p.x_scales = x_scales;
    p.x_kind = mx ? mr::MX_X_MXFP4 : (x_dtype == MR_F32 ? mr::MX_X_F32 : mr::MX_X_BF16);
    p.ldx = x_rows > 1 ? x_stride : w->cols;
    p.packed = w->packed;
    p.scales = w->scales;
    p.y = y;
    p.y_f32 = y_dtype == MR_F32;
    p.ldy = y_rows > 1 ? y_stride : w->rows;
    p.M = (int)x_rows;
    p.N = (int)w->rows;
    p.K = (int)w->cols;
    return MR_OK;
}

mr_status mr_mxfp4_matmul(const void* x, mr_dtype x_dtype, int32_t tokens, int64_t x_stride, const mr_mxfp4_matrix* w,
                          void* y, mr_dtype y_dtype, int64_t y_stride, void* stream) {
    if (!w) return fail(MR_INVALID_ARGUMENT, "MXFP4 matmul: w is NULL");
    if (x_dtype == MR_U32)
        return fail(MR_INVALID_DTYPE, "MXFP4 matmul: x must be bf16 or f32 (mr_mxfp4_matmul_quantized takes MXFP4)");
    mr::Mxfp4GemmParams p{};
    const mr_status st = gemm_params("MXFP4 matmul", x, x_dtype, nullptr, tokens, x_stride, w, tokens, y, y_dtype, y_stride, p);
    if (st != MR_OK || tokens == 0) return st;
    return done(mr::launch_mxfp4_gemm(p, mrc::cu_count(), (hipStream_t)stream), "MXFP4 matmul launch");
}

mr_status mr_mxfp4_matmul_quantized(const mr_mxfp4_matrix* x, const mr_mxfp4_matrix* w, void* y, mr_dtype y_dtype,
                                    int64_t y_stride, void* stream) {
    if (!x || !w) return fail(MR_INVALID_ARGUMENT, "MXFP4 matmul: x or w is NULL");
    if (x->cols != w->cols)
        return fail(MR_INVALID_SHAPE, "MXFP4 matmul: x has %lld columns, w %lld", (long long)x->cols, (long long)w->cols);
    mr::Mxfp4GemmParams p{};
    const mr_status st = gemm_params("MXFP4 matmul", x->packed, MR_U32, x->scales, x->rows, 0, w, x->rows, y, y_dtype, y_stride, p);
    if (st != MR_OK || x->rows == 0) return st;
    return done(mr::launch_mxfp4_gemm(p, mrc::cu_count(), (hipStream_t)stream), "MXFP4 matmul launch");
}

mr_status mr_mxfp4_expert_matmul(const mr_mxfp4_expert_args* a, void* stream) {
    const char* what = "MXFP4 expert matmul";
    if (!a) return fail(MR_INVALID_ARGUMENT, "mr_mxfp4_expert_matmul: args is NULL");
    if (a->experts <= 0 || a->experts > mr::EXPERT_MAX)
        return fail(MR_INVALID_SHAPE, "%s: %d experts (1 to %d)", what, a->experts, mr::EXPERT_MAX);
    if (a->rows < 0 || a->rows > (1 << 24) || (a->pair_of_row && (a->per_token <= 0 || a->rows % a->per_token)))
        return fail(MR_INVALID_SHAPE, "%s: %d rows (at most 2^24) of tokens with %d experts each", what, a->rows, a->per_token);
    const int32_t x_rows = a->pair_of_row ? a->rows / a->per_token : a->rows;
    if (a->x_rows != x_rows)
        return fail(MR_INVALID_SHAPE, "%s: x has %d rows, %d are asked for", what, a->x_rows, x_rows);
    if ((a->x_dtype == MR_U32) != (a->x_scales != nullptr) && a->rows > 0)
        return fail(MR_INVALID_ARGUMENT, "%s: x_scales goes with MXFP4 words, and only with them", what);
    mr::Mxfp4GemmParams p{};
    const mr_status st = gemm_params(what, a->x, a->x_dtype, a->x_scales, a->x_rows, a->x_stride, &a->w, a->rows, a->y,
                                     a->y_dtype, a->y_stride, p);
    if (st != MR_OK || a->rows == 0) return st;
    if (!a->offsets || !mrc::aligned4(a->offsets) || !mrc::aligned4(a->pair_of_row))
        return fail(MR_INVALID_ARGUMENT, "%s: offsets is NULL, or a misaligned pointer", what);
    p.offsets = a->offsets;
    p.experts = a->experts;
    p.pairs = a->rows;
    p.pair_of_row = a->pair_of_row;
    p.per_token = a->per_token;
    // byte offsets of all rows of x in 32 bits
    const int64_t x_row = p.x_kind == mr::MX_X_MXFP4 ? p.K / 2 : p.ldx * (p.x_kind == mr::MX_X_F32 ? 4 : 2);
    if (a->pair_of_row && p.M * x_row >= 0xffff0000ll)
        return fail(MR_INVALID_SHAPE, "%s: x of %d rows by token is 2^32 bytes or more; give its rows in expert order", what, p.M);
    if (!mr::mxfp4_gemm_fits(p))
        return fail(MR_INVALID_SHAPE, "%s: %d rows of %lld outputs are more than one launch takes", what, a->rows,
                    (long long)a->w.rows);
    return done(mr::launch_mxfp4_gemm(p, mrc::cu_count(), (hipStream_t)stream), "MXFP4 expert matmul launch");
}

static mr_status check_sort(int32_t tokens, int32_t per_token, int32_t experts) {
    if (tokens < 0 || per_token <= 0 || int64_t(tokens) * per_token > (1 << 24))
        return fail(MR_INVALID_SHAPE, "expert sort: %d tokens of %d experts (at most 2^24 pairs)", tokens, per_token);
    if (experts <= 0 || experts > mr::EXPERT_MAX)
        return fail(MR_INVALID_SHAPE, "expert sort: %d experts (1 to %d)", experts, mr::EXPERT_MAX);
    return MR_OK;
}

static size_t sort_workspace(int32_t tokens, int32_t per_token, int32_t experts) {
    const int blocks = mr::expert_sort_blocks(int64_t(tokens) * per_token);
    return blocks > 1 ? mrc::align256(size_t(blocks) * size_t(experts) * 4) : 0;
}

size_t mr_expert_sort_workspace_size(int32_t tokens, int32_t per_token, int32_t experts) {
    return check_sort(tokens, per_token, experts) == MR_OK ? sort_workspace(tokens, per_token, experts) : 0;
}

mr_status mr_expert_sort(const int32_t* ids, int32_t tokens, int32_t per_token, int32_t experts, int32_t* offsets,
                         int32_t* pair_of_row, int32_t* row_of_pair, void* workspace, size_t workspace_bytes,
                         void* stream) {
    const mr_status st = check_sort(tokens, per_token, experts);
    if (st != MR_OK) return st;
    const int32_t pairs = tokens * per_token;
    if (!offsets || (pairs > 0 && (!ids || !pair_of_row || !row_of_pair)))
        return fail(MR_INVALID_ARGUMENT, "expert sort: ids, offsets, pair_of_row and row_of_pair must be non-NULL");
    if (!mrc::aligned4(ids) || !mrc::aligned4(offsets) || !mrc::aligned4(pair_of_row) || !mrc::aligned4(row_of_pair) ||
        !mrc::aligned4(workspace))
        return fail(MR_INVALID_ARGUMENT, "expert sort: a misaligned pointer");
    const size_t need = sort_workspace(tokens, per_token, experts);
    if (need && (!workspace || workspace_bytes < need))
        return fail(MR_WORKSPACE_TOO_SMALL, "expert sort: workspace %zu bytes < %zu required", workspace_bytes, need);
    mr::ExpertSortParams p{ids, pairs, experts, offsets, pair_of_row, row_of_pair, (int32_t*)workspace};
    return done(mr::launch_expert_sort(p, (hipStream_t)stream), "expert sort launch");
}

mr_status mr_expert_dispatch(const void* x, mr_dtype dtype, int32_t tokens, int64_t dim, int64_t x_stride,
                             const int32_t* row_of_pair, int32_t per_token, void* rows, int64_t rows_stride,
                             void* stream) {
    const mr_status st = check_rows(tokens, per_token, dim, dtype, "expert dispatch");
    if (st != MR_OK) return st;
    if (tokens == 0) return MR_OK;
    if (!x || !row_of_pair || !rows)
        return fail(MR_INVALID_ARGUMENT, "expert dispatch: x, row_of_pair and rows must be non-NULL");
    if (!stride_ok(x_stride, dim) || !stride_ok(rows_stride, dim) || !elem_aligned(x, dtype) ||
        !elem_aligned(rows, dtype) || !mrc::aligned4(row_of_pair))
        return fail(MR_INVALID_ARGUMENT, "expert dispatch: a stride shorter than the rows, or a misaligned pointer");
    mr::ExpertRowsParams p{};
    p.tokens = x;
    p.ld_tokens = x_stride;
    p.out = rows;
    p.ld_out = rows_stride;
    p.f32 = dtype == MR_F32;
    p.dim = dim;
    p.n_tokens = tokens;
    p.per_token = per_token;
    p.row_of_pair = row_of_pair;
    return done(mr::launch_expert_dispatch(p, mrc::cu_count(), (hipStream_t)stream), "expert dispatch launch");
}

mr_status mr_expert_combine(const void* rows, mr_dtype dtype, int64_t rows_stride, int64_t dim,
                            const int32_t* row_of_pair, const float* weights, int32_t tokens, int32_t per_token,
                            void* out, int64_t out_stride, void* stream) {
    const mr_status st = check_rows(tokens, per_token, dim, dtype, "expert combine");
    if (st != MR_OK) return st;
    if (tokens == 0) return MR_OK;
    if (!rows || !row_of_pair || !out)
        return fail(MR_INVALID_ARGUMENT, "expert combine: rows, row_of_pair and out must be non-NULL");
    if (!stride_ok(rows_stride, dim) || !stride_ok(out_stride, dim) || !elem_aligned(rows, dtype) ||
        !elem_aligned(out, dtype) || !mrc::aligned4(row_of_pair) || !mrc::aligned4(weights))
        return fail(MR_INVALID_ARGUMENT, "expert combine: a stride shorter than the rows, or a misaligned pointer");
    mr::ExpertRowsParams p{};
    p.rows = rows;
    p.ld_rows = rows_stride;
    p.out = out;
    p.ld_out = out_stride;
    p.f32 = dtype == MR_F32;
    p.dim = dim;
    p.n_tokens = tokens;
    p.per_token = per_token;
    p.row_of_pair = row_of_pair;
    p.weights = weights;
    return done(mr::launch_expert_combine(p, mrc::cu_count(), (hipStream_t)stream), "expert combine launch");
}

mr_status mr_expert_combine_backward(const void* d_out, mr_dtype dtype, int64_t d_out_stride, int64_t dim,
                                     const void* rows, int64_t rows_stride, const int32_t* row_of_pair,
                                     const float* weights, int32_t tokens, int32_t per_token, void* d_rows,
                                     int64_t d_rows_stride, float* d_weights, void* stream) {
    const mr_status st = check_rows(tokens, per_token, dim, dtype, "expert combine backward");
    if (st != MR_OK) return st;
    if (tokens == 0 || (!d_rows && !d_weights)) return MR_OK;
    if (!d_out || !row_of_pair || (d_weights && !rows))
        return fail(MR_INVALID_ARGUMENT, "expert combine backward: d_out, row_of_pair and (for d_weights) rows must be non-NULL");
    if (!stride_ok(d_out_stride, dim) || (d_weights && !stride_ok(rows_stride, dim)) ||
        (d_rows && !stride_ok(d_rows_stride, dim)) || !elem_aligned(d_out, dtype) || !elem_aligned(rows, dtype) ||
        !elem_aligned(d_rows, dtype) || !mrc::aligned4(row_of_pair) || !mrc::aligned4(weights) ||
        !mrc::aligned4(d_weights))
        return fail(MR_INVALID_ARGUMENT, "expert combine backward: a stride shorter than the rows, or a misaligned pointer");
    mr::ExpertRowsParams p{};
    p.tokens = d_out;
    p.ld_tokens = d_out_stride;
    p.rows = d_weights ? rows : nullptr;
    p.ld_rows = d_weights ? rows_stride : dim;
    p.out = d_rows;
    p.ld_out = d_rows ? d_rows_stride : dim;
    p.f32 = dtype == MR_F32;
    p.dim = dim;
    p.n_tokens = tokens;
    p.per_token = per_token;
    p.row_of_pair = row_of_pair;
    p.weights = weights;
    p.d_weights = d_weights;
    return done(mr::launch_expert_combine_backward(p, mrc::cu_count(), (hipStream_t)stream), "expert combine backward launch");
}

}  // extern "C"
