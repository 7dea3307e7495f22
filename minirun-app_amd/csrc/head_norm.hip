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
// rotation's partners pass through the wave's own part of LDS.  The heads of a
// token are neighbouring rows, so that their angles come from the caches.
//
// The weights' gradients are sums over all rows: a workgroup of the backward
// pass walks rows of the queries or of the keys with the next ones in flight (8192
// tokens of 32 + 8 heads of 128, bf16: 57 us a call among others, 49 of them here, 5.2
// TB/s; where the two took 54, one row at a time with nothing in flight took 76), keeps
// its sums in registers and leaves one partial row; a second launch adds the partial rows
// in their order, so the result does not depend on timing.
#include <algorithm>

#include "head_rows.hpp"

namespace mr {

namespace {

constexpr int HN_WAVES = 4;
constexpr int HN_PARTIALS = 1024;  // partial rows of a segment at most
constexpr int HN_ROWS = 2;         // that a group of the backward pass takes a step

// A row, (token, head) in order, a group of lanes: the keys' workgroups follow the
// queries'.  (4096 tokens of 32 + 4 heads of 128, bf16: 18.9 us a call among others, 4.1
// TB/s; 20.2 in a profiler's trace.  A copy of these bytes takes 16.2.  Where this form
// took 20.5, two, four and eight rows a group loaded together took 21.2, 22.0 and 24.4,
// waves that walk rows with the next ones in flight 23.3, stores past the caches 20.9.)
template <bool F32, bool VEC, int KIND>
__global__ void __launch_bounds__(64 * HN_WAVES) head_norm_kernel(HeadNormParams p, uint32_t q_blocks) {
    __shared__ __attribute__((aligned(16))) float sh[HN_WAVES][512];
    const int l = threadIdx.x & 63, group = l >> p.lpr_log2, c = 8 * (l & (p.lpr - 1));
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool key = blockIdx.x >= q_blocks;
    const HeadSegment s = key ? p.seg[1] : p.seg[0];
    const uint32_t groups = 64u >> p.lpr_log2, rows = (uint32_t)(p.tokens * s.heads);
    const uint32_t first = ((blockIdx.x - (key ? q_blocks : 0)) * HN_WAVES + w) * groups;
    if (first >= rows) return;  // (a whole wave)
    const uint32_t id = first + group, my = min(id, rows - 1), token = my / (uint32_t)s.heads;
    const int64_t head = my - token * (uint32_t)s.heads;
    const int n = id < rows ? p.dim : 0;
    float v[8], wt[8];
    head_load<F32, VEC>(s.x, token * s.x_ts + head * s.x_hs, c, n, v);
    HeadAngles<KIND> angles;
    angles.load(p.rope, rope_row(p.rope, token), c);
    if (s.w) {
        head_load<VEC>(s.w, p.w_f32, 0, c, p.dim, wt);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) wt[j] = 1.f;
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
    ss = group_sum(ss, p.lpr);
    const float inv = rsqrtf(fmaf(ss, p.inv_dim, p.eps));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = wt[j] * (v[j] * inv);
    head_rotate<KIND, false>(v, p.rope, angles, c, &sh[w][8 * (group << p.lpr_log2)]);
    head_store<VEC>(s.out, p.out_f32, token * s.out_ts + head * s.out_hs, c, n, v);
}

// blocks[i] workgroups walk the rows of segment i (token-major), a group of lanes U rows
// at a time, the next ones in flight; each leaves its sums for the weights' gradient in
// partial[workgroup][dim].
template <bool F32, bool VEC, int KIND>
__global__ void __launch_bounds__(64 * HN_WAVES) head_norm_backward_kernel(HeadNormParams p) {
    constexpr int U = HN_ROWS;
    __shared__ __attribute__((aligned(16))) float sh[HN_WAVES][512];
    const int l = threadIdx.x & 63, group = l >> p.lpr_log2, c = 8 * (l & (p.lpr - 1));
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool key = blockIdx.x >= (unsigned)p.blocks[0];
    const HeadSegment s = key ? p.seg[1] : p.seg[0];
    const uint32_t block = key ? blockIdx.x - p.blocks[0] : blockIdx.x, blocks = key ? p.blocks[1] : p.blocks[0];
    const uint32_t rows = (uint32_t)(p.tokens * s.heads), groups = 64u >> p.lpr_log2;
    float wt[8], dw[8];
    if (s.w) {
        head_load<VEC>(s.w, p.w_f32, 0, c, p.dim, wt);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) wt[j] = 1.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[j] = 0.f;
    using Walk = HeadWalk<3>;
    const int64_t ts[3] = {s.x_ts, s.out_ts, s.dy_ts}, hs[3] = {s.x_hs, s.out_hs, s.dy_hs};
    const typename Walk::Step near = Walk::step(groups, s.heads, ts, hs);
    struct Rows {
        HeadEight<F32, VEC> x[U], g[U];
        Walk row[U];
    };
    const uint32_t last = (uint32_t)p.tokens - 1;
    auto load = [&](const Walk& first, Rows& r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            r.row[u] = u ? r.row[u - 1] : first;
            if (u) r.row[u].next(near);
            const int n = r.row[u].token <= last ? p.dim : 0;
            r.x[u].load(s.x, r.row[u].at[0], c, n);
            r.g[u].load(s.dy, r.row[u].at[2], c, n);
        }
    };
    const bool one_token = (uint32_t)s.heads % (groups * U) == 0;
    auto work = [&](const Rows& r) {
        HeadAngles<KIND> angles;
        angles.load(p.rope, rope_row(p.rope, min(r.row[0].token, last)), c);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = r.row[u].token <= last;
            if (u && !one_token) angles.load(p.rope, rope_row(p.rope, min(r.row[u].token, last)), c);
            float x[8], g[8];
            r.x[u].values(x);
            r.g[u].values(g);
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
            ss = group_sum(ss, p.lpr);
            const float inv = rsqrtf(fmaf(ss, p.inv_dim, p.eps));
            head_rotate<KIND, true>(g, p.rope, angles, c, &sh[w][8 * (group << p.lpr_log2)]);
            float dot = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] *= inv;
                if (in) dw[j] = fmaf(g[j], x[j], dw[j]);
                g[j] *= wt[j];
                dot = fmaf(g[j], x[j], dot);
            }
            dot = group_sum(dot, p.lpr) * p.inv_dim;
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = inv * (g[j] - x[j] * dot);
            head_store<VEC>(s.out, p.out_f32, r.row[u].at[1], c, in ? p.dim : 0, g);
        }
    };
    const uint32_t step = blocks * HN_WAVES * groups * U;
    uint32_t at = (block * HN_WAVES + w) * groups * U;
    if (at < rows) {
        const typename Walk::Step far = Walk::step(step, s.heads, ts, hs);
        Walk walk;
        walk.start(at + group, s.heads, ts, hs);
        Rows now;
        load(walk, now);
        for (; at + step < rows; at += step) {
            walk.next(far);
            Rows next;
            load(walk, next);
            work(now);
            now = next;
        }
        work(now);
    }
    if (!s.dw) return;
    // the groups of a wave by lane exchange, then the waves
#pragma unroll
    for (int j = 0; j < 8; ++j)
        for (int d = p.lpr; d < 64; d *= 2) dw[j] += __shfl_xor(dw[j], d);
    wave_lds_fence();
    if (l < p.lpr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sh[w][c + j] = dw[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.dim; i += 64 * HN_WAVES)
        p.partial[(int64_t)blockIdx.x * p.dim + i] = (sh[0][i] + sh[1][i]) + (sh[2][i] + sh[3][i]);
}

// dw[i] = the sum of a segment's partial rows: 16 columns a workgroup, 64 threads a
// column, each of which adds every 64th row (16 at most, loaded together).
__global__ void __launch_bounds__(1024) head_norm_weight_kernel(HeadNormParams p) {
    __shared__ float sh[64][17];
    const HeadSegment s = p.seg[blockIdx.y];
    if (!s.dw) return;
    const int col = threadIdx.x & 15, i = blockIdx.x * 16 + col, part = threadIdx.x >> 4;
    const int first = blockIdx.y ? p.blocks[0] : 0, blocks = p.blocks[blockIdx.y];
    float v[HN_PARTIALS / 64], sum = 0.f;
#pragma unroll
    for (int k = 0; k < HN_PARTIALS / 64; ++k) {
        const int b = part + 64 * k;
        v[k] = b < blocks && i < p.dim ? p.partial[(int64_t)(first + b) * p.dim + i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < HN_PARTIALS / 64; ++k) sum += v[k];
    sh[part][col] = sum;
    __syncthreads();
    if (part) return;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 64; ++k) t += sh[k][col];
    if (i < p.dim) s.dw[i] = t;
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

// Partial rows for the weights' gradients: workgroups of both segments by their rows (none
// without), about HN_PARTIALS in all.
void head_norm_blocks(int64_t tokens, const int (&heads)[2], int dim, int (&blocks)[2]) {
    const int64_t per_block = int64_t(HN_WAVES) * (64 >> lanes_log2(dim)) * HN_ROWS, all = tokens * (int64_t(heads[0]) + heads[1]);
    for (int i = 0; i < 2; ++i) {
        const int64_t rows = tokens * heads[i];
        const int64_t full = (rows + per_block - 1) / per_block, share = all ? HN_PARTIALS * rows / all : 0;
        blocks[i] = (int)std::min(full, std::max<int64_t>(share, 1));
    }
}

namespace {

template <bool F32, bool VEC, int KIND>
hipError_t head_norm_run(const HeadNormParams& p, bool backward, hipStream_t st) {
    if (!backward) {
        const int64_t per = HN_WAVES * (64 >> p.lpr_log2);
        const int64_t q = (p.tokens * p.seg[0].heads + per - 1) / per, k = (p.tokens * p.seg[1].heads + per - 1) / per;
        hipLaunchKernelGGL((head_norm_kernel<F32, VEC, KIND>), dim3((unsigned)(q + k)), dim3(64 * HN_WAVES), 0, st, p,
                           (uint32_t)q);
        return hipGetLastError();
    }
    if (p.blocks[0] + p.blocks[1] > 0) {
        hipLaunchKernelGGL((head_norm_backward_kernel<F32, VEC, KIND>), dim3((unsigned)(p.blocks[0] + p.blocks[1])),
                           dim3(64 * HN_WAVES), 0, st, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.seg[0].dw || p.seg[1].dw) {
        hipLaunchKernelGGL(head_norm_weight_kernel, dim3((unsigned)((p.dim + 15) / 16), 2), dim3(1024), 0, st, p);
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
    p.inv_dim = 1.f / (float)p.dim;
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
