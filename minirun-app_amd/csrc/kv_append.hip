// New tokens' keys and values into the pages of a cache, the keys normalised
// and rotated on the way, as bf16 or as MXFP4 (blocks of 32 values along a
// head: mxfp4.hip's rule).
//
//   key = R (w * (k / sqrt(mean(k^2) + eps))), value = v; each stored value is
//   rounded once, from the unrounded one
//
// A value next to a border of the 4-bit grid goes the wrong way if it is off by
// a rounding of f32, and a block's power with it, so keys are computed in f64 and
// handed to the instructions that round as f32 "to odd": cut off, the last bit set
// if that lost anything, which no later rounding to fewer bits can tell from the
// f64 value.
//
// What bounds it: HBM (8192 tokens of 8 heads of 128 as they are, bf16: 15.4 us,
// 4.6 TB/s) and, with norm and rotation, the vector units: the norm in f64 takes 4.2
// us of it, the rotation 6.6 (25.4 us in all; in MXFP4 22.2).  A group of dim / 8
// lanes has one head's row, as in head_norm.hip; the four lanes of a block
// find its largest magnitude by two DPP steps.  Keys and values in one workgroup
// took 21.5 us in MXFP4 and 13.3 instead of 11.4 for 4001 tokens in bf16.
#include "head_rows.hpp"

namespace mr {

namespace {

constexpr int KA_WAVES = 4;

__device__ __forceinline__ float to_odd(double d) {
    const float f = (float)d;
    const double back = (double)f;
    uint32_t u = __float_as_uint(f);
    if (back == d || d != d) return f;
    if (__builtin_fabs(back) > __builtin_fabs(d)) --u;
    return __uint_as_float(u | 1u);
}

__device__ __forceinline__ uint32_t block_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));
}

// blockIdx.y: 0 keys, 1 values.  Row `id` is head id % heads of token id / heads.
template <bool F32, bool VEC, int KIND>
__global__ void __launch_bounds__(64 * KA_WAVES) kv_append_kernel(KvAppendParams p, uint32_t rows) {
    __shared__ __attribute__((aligned(16))) double sh[KA_WAVES][512];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, group = l >> p.lpr_log2, c = 8 * (l & (p.lpr - 1));
    const uint32_t id = ((blockIdx.x * KA_WAVES + w) << (6 - p.lpr_log2)) + group;
    if ((id & ~(uint32_t)group) >= rows) return;  // (a whole wave)
    const uint32_t my = min(id, rows - 1), token = my / (uint32_t)p.heads;
    const int64_t head = my - token * (uint32_t)p.heads;
    const int32_t slot = p.slots[token];
    // rows past the last and slots outside the pages: nothing is read or stored
    const bool in = id < rows && slot >= 0 && slot < p.slot_end;
    const int n = in ? p.dim : 0;
    const bool key = blockIdx.y == 0;
    float v[8];
    head_load<F32, VEC>(key ? p.k : p.v, token * (key ? p.k_ts : p.v_ts) + head * (key ? p.k_hs : p.v_hs), c, n, v);
    if (key && p.turn) {
        double y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = v[j];
        if (p.norm) {
            double ss = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += y[j] * y[j];
            for (int d = 1; d < p.lpr; d *= 2) ss += __shfl_xor(ss, d);
            const double inv = 1.0 / sqrt(ss / p.dim + (double)p.eps);
            float wt[8];
            if (p.w) {
                head_load<VEC>(p.w, p.w_f32, 0, c, p.dim, wt);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) wt[j] = 1.f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = wt[j] * (y[j] * inv);
        }
        if (p.rope.half) {
            HeadAngles<KIND> angles;
            angles.load(p.rope, rope_row(p.rope, token), c);
            head_rotate<KIND, false>(y, p.rope, angles, c, &sh[w][8 * (group << p.lpr_log2)]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_odd(y[j]);
    }
    const uint32_t page = (uint32_t)slot / (uint32_t)p.page_size;
    const int64_t row = head * p.page_size + ((uint32_t)slot - page * (uint32_t)p.page_size);
    if (!p.k_scales) {
        uint16_t* to = (uint16_t*)(key ? p.k_pages : p.v_pages) + page * p.page_stride + row * p.dim + c;
        if (c < n)
            *(u32x4*)to = u32x4{pack_bf16x2_hw(v[0], v[1]), pack_bf16x2_hw(v[2], v[3]), pack_bf16x2_hw(v[4], v[5]),
                                pack_bf16x2_hw(v[6], v[7])};
        return;
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = block_max(top);
    const bool finite = top < 0x7f800000u;
    const uint32_t e = top >> 23, byte = finite ? (e > 2 ? e - 2 : 0) : 255u;
    const float scale = __uint_as_float(finite ? byte << 23 : 0x3f800000u);
    uint32_t word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], scale, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], scale, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], scale, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], scale, 3);
    if (c >= n) return;
    ((uint32_t*)(key ? p.k_pages : p.v_pages))[page * p.page_stride + (row * p.dim + c) / 8] = finite ? word : 0u;
    if ((l & 3) == 0) (key ? p.k_scales : p.v_scales)[page * p.scale_stride + (row * p.dim + c) / 32] = (uint8_t)byte;
}

template <bool F32, bool VEC>
hipError_t append_kind(const KvAppendParams& p, RopeKind kind, dim3 grid, uint32_t rows, hipStream_t st) {
    const dim3 block(64 * KA_WAVES);
    switch (kind) {
        case ROPE_ADJACENT: hipLaunchKernelGGL((kv_append_kernel<F32, VEC, ROPE_ADJACENT>), grid, block, 0, st, p, rows); break;
        case ROPE_HALVES: hipLaunchKernelGGL((kv_append_kernel<F32, VEC, ROPE_HALVES>), grid, block, 0, st, p, rows); break;
        default: hipLaunchKernelGGL((kv_append_kernel<F32, VEC, ROPE_ANY>), grid, block, 0, st, p, rows);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_append(KvAppendParams p, hipStream_t st) {
    p.lpr_log2 = 2;
    while ((8 << p.lpr_log2) < p.dim) ++p.lpr_log2;
    p.lpr = 1 << p.lpr_log2;
    p.turn = p.norm || p.rope.half;
    const int size = p.f32 ? 4 : 2;
    auto piece = [&](const void* q, int64_t ts, int64_t hs) {
        return ((uintptr_t)q & 15) == 0 && ts * size % 16 == 0 && hs * size % 16 == 0;
    };
    const bool vec = piece(p.k, p.k_ts, p.k_hs) && piece(p.v, p.v_ts, p.v_hs) && ((uintptr_t)p.w & 15) == 0;
    const uint32_t rows = (uint32_t)(p.tokens * p.heads), per = KA_WAVES * (64 >> p.lpr_log2);
    const dim3 grid((rows + per - 1) / per, 2);
    const RopeKind kind = head_rope_kind(p.rope);
    if (p.f32) return vec ? append_kind<true, true>(p, kind, grid, rows, st) : append_kind<true, false>(p, kind, grid, rows, st);
    return vec ? append_kind<false, true>(p, kind, grid, rows, st) : append_kind<false, false>(p, kind, grid, rows, st);
}

}  // namespace mr
