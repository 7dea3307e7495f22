// RMSNorm of every head of the queries and keys with the rotation by their
// positions, in one pass, and its gradients.
//
// For a head's row x, weight w and the rotation R of the row's position:
//   r = 1 / sqrt(mean(x^2) + eps),  y = R (w * (x * r))
// and with g = R^T dy:
//   dw = sum over rows of g * (x r)
//   dx = r * (g * w - (x r) * mean(g * w * (x r)))
// so the backward pass needs x and dy only; r is computed again.
//
// What bounds it: HBM, rows read and written once.  A group of 8 to 64 lanes
// has one row, eight columns a lane (head_rows.hpp), so a wave's loads and
// stores are whole lines; a row's sum is a butterfly inside its group, and the
// rotation's partners pass through the wave's own part of LDS.  Queries and
// keys of a token are neighbouring rows of one launch, so that their angles
// come from the caches.
//
// The weights' gradients are sums over all rows: a workgroup of the backward
// pass walks rows of the queries or of the keys, keeps its sums in registers
// and leaves one partial row; a second launch adds the partial rows in their
// order, so the result does not depend on timing.
#include <algorithm>

#include "head_rows.hpp"

namespace mr {

namespace {

constexpr int HN_WAVES = 4;

// One row a group of lanes: row `id` is head id % (heads of q and k) of token
// id / that; the heads of q come first.
template <bool F32, bool VEC, int KIND>
__global__ void __launch_bounds__(64 * HN_WAVES) head_norm_kernel(HeadNormParams p, uint32_t rows) {
    __shared__ __attribute__((aligned(16))) float sh[HN_WAVES][512];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, group = l >> p.lpr_log2, c = 8 * (l & (p.lpr - 1));
    const uint32_t id = ((blockIdx.x * HN_WAVES + w) << (6 - p.lpr_log2)) + group;
    if ((id & ~(uint32_t)group) >= rows) return;  // (a whole wave)
    const bool in = id < rows;
    const uint32_t heads = (uint32_t)(p.seg[0].heads + p.seg[1].heads), my = in ? id : rows - 1;
    const uint32_t token = my / heads, h = my - token * heads;
    const bool key = h >= (uint32_t)p.seg[0].heads;
    const HeadSegment s = key ? p.seg[1] : p.seg[0];
    const int64_t head = key ? h - p.seg[0].heads : h;
    const int n = in ? p.dim : 0;
    float x[8], wt[8];
    head_load<F32, VEC>(s.x, token * s.x_ts + head * s.x_hs, c, n, x);
    if (s.w) {
        head_load<VEC>(s.w, p.w_f32, 0, c, p.dim, wt);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) wt[j] = 1.f;
    }
    const int64_t at = rope_row(p.rope, token);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
    ss = group_sum(ss, p.lpr);
    const float inv = 1.f / sqrtf(ss / (float)p.dim + p.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = wt[j] * (x[j] * inv);
    head_rotate<KIND, false>(x, p.rope, at, c, &sh[w][8 * (group << p.lpr_log2)]);
    head_store<VEC>(s.out, p.out_f32, token * s.out_ts + head * s.out_hs, c, n, x);
}

// blocks[i] workgroups walk the rows of segment i (token-major); each leaves
// its sums for the weights' gradient in partial[workgroup][dim].
template <bool F32, bool VEC, int KIND>
__global__ void __launch_bounds__(64 * HN_WAVES) head_norm_backward_kernel(HeadNormParams p) {
    __shared__ __attribute__((aligned(16))) float sh[HN_WAVES][512];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, group = l >> p.lpr_log2, c = 8 * (l & (p.lpr - 1));
    const bool key = blockIdx.x >= (unsigned)p.blocks[0];
    const HeadSegment s = key ? p.seg[1] : p.seg[0];
    const uint32_t block = key ? blockIdx.x - p.blocks[0] : blockIdx.x, blocks = key ? p.blocks[1] : p.blocks[0];
    const uint32_t rows = (uint32_t)(p.tokens * s.heads), per_wave = 64u >> p.lpr_log2;
    float wt[8], dw[8];
    if (s.w) {
        head_load<VEC>(s.w, p.w_f32, 0, c, p.dim, wt);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) wt[j] = 1.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[j] = 0.f;
    const uint32_t step = blocks * HN_WAVES * per_wave;
    for (uint32_t first = (block * HN_WAVES + w) * per_wave; first < rows; first += step) {
        const bool in = first + group < rows;
        const uint32_t my = in ? first + group : rows - 1;
        const uint32_t token = my / (uint32_t)s.heads;
        const int64_t head = my - token * (uint32_t)s.heads;
        const int n = in ? p.dim : 0;
        float x[8], g[8];
        head_load<F32, VEC>(s.x, token * s.x_ts + head * s.x_hs, c, n, x);
        head_load<F32, VEC>(s.dy, token * s.dy_ts + head * s.dy_hs, c, n, g);
        const int64_t at = rope_row(p.rope, token);
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
        ss = group_sum(ss, p.lpr);
        const float inv = 1.f / sqrtf(ss / (float)p.dim + p.eps);
        head_rotate<KIND, true>(g, p.rope, at, c, &sh[w][8 * (group << p.lpr_log2)]);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] *= inv;
            if (in) dw[j] = fmaf(g[j], x[j], dw[j]);
            g[j] *= wt[j];
            dot = fmaf(g[j], x[j], dot);
        }
        dot = group_sum(dot, p.lpr) / (float)p.dim;
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = inv * (g[j] - x[j] * dot);
        head_store<VEC>(s.out, p.out_f32, token * s.out_ts + head * s.out_hs, c, n, g);
    }
    if (!s.dw) return;
    // the groups of a wave by lane exchange, then the waves
#pragma unroll
    for (int j = 0; j < 8; ++j)
        for (int d = p.lpr; d < 64; d *= 2) dw[j] += __shfl_xor(dw[j], d);
    if (l < p.lpr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sh[w][c + j] = dw[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.dim; i += 64 * HN_WAVES)
        p.partial[(int64_t)blockIdx.x * p.dim + i] = (sh[0][i] + sh[1][i]) + (sh[2][i] + sh[3][i]);
}

// dw[i] = the sum of a segment's partial rows: 16 columns a workgroup, 16
// threads a column, each of which adds every 16th row.
__global__ void __launch_bounds__(256) head_norm_weight_kernel(HeadNormParams p) {
    __shared__ float sh[16][16];
    const HeadSegment s = p.seg[blockIdx.y];
    if (!s.dw) return;
    const int i = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
    const int first = blockIdx.y ? p.blocks[0] : 0, blocks = p.blocks[blockIdx.y];
    float sum = 0.f;
    if (i < p.dim)
        for (int b = part; b < blocks; b += 16) sum += p.partial[(int64_t)(first + b) * p.dim + i];
    sh[part][threadIdx.x & 15] = sum;
    __syncthreads();
    if (part == 0 && i < p.dim) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += sh[k][threadIdx.x];
        s.dw[i] = t;
    }
}

int lanes_log2(int dim) {
    int n = 0;
    while ((8 << n) < dim) ++n;
    return n;
}

}  // namespace

RopeKind head_rope_kind(const HeadRope& r) {
    const bool whole = r.col0 % 8 == 0 && ((uintptr_t)r.cos_t & 15) == 0 && ((uintptr_t)r.sin_t & 15) == 0;
    if (r.half == 0) return ROPE_ADJACENT;  // (no columns: nothing is read)
    if (whole && r.halves && r.half % 8 == 0) return ROPE_HALVES;
    if (whole && !r.halves && r.half % 4 == 0) return ROPE_ADJACENT;
    return ROPE_ANY;
}

// Partial rows for the weights' gradients: workgroups for about 16 rows of each
// group of lanes, at most 1024 for both segments.
void head_norm_blocks(int64_t tokens, const int (&heads)[2], int dim, int (&blocks)[2]) {
    const int64_t per_block = int64_t(HN_WAVES) * (64 >> lanes_log2(dim));
    const int64_t most = 1024, all = tokens * (heads[0] + heads[1]);
    for (int i = 0; i < 2; ++i) {
        const int64_t rows = tokens * heads[i];
        const int64_t full = (rows + per_block - 1) / per_block, share = all ? most * rows / all : 0;
        blocks[i] = (int)std::min(full, std::max<int64_t>(share, 1));
    }
}

namespace {

template <bool F32, bool VEC, int KIND>
hipError_t head_norm_run(const HeadNormParams& p, bool backward, hipStream_t st) {
    if (!backward) {
        const int64_t rows = p.tokens * (p.seg[0].heads + p.seg[1].heads), per = HN_WAVES * (64 >> p.lpr_log2);
        hipLaunchKernelGGL((head_norm_kernel<F32, VEC, KIND>), dim3((unsigned)((rows + per - 1) / per)), dim3(64 * HN_WAVES),
                           0, st, p, (uint32_t)rows);
        return hipGetLastError();
    }
    if (p.blocks[0] + p.blocks[1] > 0) {
        hipLaunchKernelGGL((head_norm_backward_kernel<F32, VEC, KIND>), dim3((unsigned)(p.blocks[0] + p.blocks[1])),
                           dim3(64 * HN_WAVES), 0, st, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.seg[0].dw || p.seg[1].dw) {
        hipLaunchKernelGGL(head_norm_weight_kernel, dim3((unsigned)((p.dim + 15) / 16), 2), dim3(256), 0, st, p);
        return hipGetLastError();
    }
    return hipSuccess;
}

template <bool F32, bool VEC>
hipError_t head_norm_kind(const HeadNormParams& p, bool backward, hipStream_t st) {
    switch (head_rope_kind(p.rope)) {
        case ROPE_ADJACENT: return head_norm_run<F32, VEC, ROPE_ADJACENT>(p, backward, st);
        case ROPE_HALVES: return head_norm_run<F32, VEC, ROPE_HALVES>(p, backward, st);
        default: return head_norm_run<F32, VEC, ROPE_ANY>(p, backward, st);
    }
}

}  // namespace

hipError_t launch_head_norm(HeadNormParams p, bool backward, hipStream_t st) {
    p.lpr_log2 = lanes_log2(p.dim);
    p.lpr = 1 << p.lpr_log2;
    // 16-byte pieces need every row of every tensor on a 16-byte boundary
    const int xs = p.x_f32 ? 4 : 2, os = p.out_f32 ? 4 : 2;
    bool vec = p.dim % 8 == 0;
    auto piece = [&](const void* q, int64_t ts, int64_t hs, int size) {
        vec = vec && ((uintptr_t)q & 15) == 0 && ts * size % 16 == 0 && hs * size % 16 == 0;
    };
    for (const HeadSegment& s : p.seg) {
        if (!s.heads) continue;
        piece(s.x, s.x_ts, s.x_hs, xs);
        piece(s.out, s.out_ts, s.out_hs, os);
        piece(s.w, 0, 0, 1);
        if (backward) piece(s.dy, s.dy_ts, s.dy_hs, xs);
    }
    if (p.x_f32) return vec ? head_norm_kind<true, true>(p, backward, st) : head_norm_kind<true, false>(p, backward, st);
    return vec ? head_norm_kind<false, true>(p, backward, st) : head_norm_kind<false, false>(p, backward, st);
}

}  // namespace mr
