// MXFP4 quantisation and its inverse: blocks of 32 values along a row, one
// power of two (E8M0) and 32 e2m1 numbers each, the storage of
// MXFP4Weights.swift:36-60 (element j of a word in bits 4j .. 4j + 3).
//
// Per block, with A the largest magnitude:
//   byte = max(0, floor(log2 A) - 2 + 127), so that A / 2^(byte - 127) is in
//          [4, 8), or below 4 where the byte is clamped (A < 2^-125)
//   code = the e2m1 number (0, .5, 1, 1.5, 2, 3, 4, 6) nearest to
//          |x| / 2^(byte - 127), the even code of two equally near ones, 6
//          above it; the sign is x's
// floor(log2 A) is A's exponent field, so nothing is computed in floating
// point before v_cvt_scalef32_pk_fp4, which divides by the power of two and
// rounds (subnormal values and byte 0 included; pinned against the rule on
// hardware).  A block with a NaN or an infinity gets byte 255 and codes 0: all
// of its values are NaN.
//
// What bounds it: HBM (2 or 4 bytes read, 17 / 32 of a byte written per
// value).  A lane owns 8 values (16 or 32 bytes of loads, one word stored), so
// every load and store of a wave covers whole lines; the four lanes of a block
// find A by two DPP steps.  Each lane has the loads of MX_U such pieces in
// flight before it uses the first.  24576 x 1536 in f32: 37 us (4.6 TB/s), and
// back 28 us (6.2 TB/s).
#include <algorithm>
#include <type_traits>

#include "mr_kernels.hpp"

namespace mr {

namespace {

constexpr int MX_U = 4;      // pieces of 512 values per wave
constexpr int MX_WAVES = 4;  // waves per workgroup

// Eight values of a row as stored, from or to a buffer at a byte offset.  What lies
// past the end of a buffer is zeros or is not stored, without a branch, behind
// which the compiler would wait for the loads before it.
template <bool F32, bool VEC>
struct MxEight {
    using Elem = std::conditional_t<F32, uint32_t, uint16_t>;
    static constexpr int N16 = F32 ? 2 : 1, SIZE = F32 ? 4 : 2;
    std::conditional_t<VEC, u32x4[N16], Elem[8]> v;
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t row, int at) {
#pragma unroll
        for (int k = 0; k < (VEC ? N16 : 8); ++k) {
            if constexpr (VEC)
                v[k] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(row, at + 16 * k, 0, 0));
            else if constexpr (F32)
                v[k] = __builtin_amdgcn_raw_buffer_load_b32(row, at + 4 * k, 0, 0);
            else
                v[k] = __builtin_amdgcn_raw_buffer_load_b16(row, at + 2 * k, 0, 0);
        }
    }
    // value k's bits as those of an f32
    __device__ __forceinline__ uint32_t bits(int k) const {
        if constexpr (!VEC)
            return F32 ? (uint32_t)v[k] : (uint32_t)v[k] << 16;
        else if constexpr (F32)
            return v[k >> 2][k & 3];
        else
            return k & 1 ? v[0][k >> 1] & 0xffff0000u : v[0][k >> 1] << 16;
    }
    __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t row, int at) const {
#pragma unroll
        for (int k = 0; k < (VEC ? N16 : 8); ++k) {
            if constexpr (VEC)
                __builtin_amdgcn_raw_buffer_store_b128(v[k], row, at + 16 * k, 0, 0);
            else if constexpr (F32)
                __builtin_amdgcn_raw_buffer_store_b32(v[k], row, at + 4 * k, 0, 0);
            else
                __builtin_amdgcn_raw_buffer_store_b16(v[k], row, at + 2 * k, 0, 0);
        }
    }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_buffer(const void* p, int64_t bytes_before, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((char*)p + bytes_before, 0, bytes, 0x00020000);
}

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));
}

// Wave `unit` (of this launch's from `first` on) takes values 512 MX_U (unit % per_row) .. of row
// unit / per_row.  cols is a multiple of 32, so the four lanes of a block are
// all inside the row or all past it.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(64 * MX_WAVES) mxfp4_quantize_kernel(Mxfp4QuantizeParams p, int64_t first, int64_t per_row) {
    const int64_t unit = first + (int64_t)blockIdx.x * MX_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = p.rows == 1 ? 0 : unit / per_row;
    if (row >= p.rows) return;
    const int l = threadIdx.x & 63;
    const int64_t c0 = (unit - row * per_row) * (512 * MX_U), o = row * p.cols + c0;
    if (c0 >= p.cols) return;  // (one long row: a wave past its end)
    const int n = (int)min(p.cols - c0, (int64_t)512 * MX_U);  // of this wave
    using E = MxEight<F32, VEC>;
    const __amdgpu_buffer_rsrc_t x = mx_buffer(p.x, (row * p.x_stride + c0) * E::SIZE, n * E::SIZE);
    const __amdgpu_buffer_rsrc_t packed = mx_buffer(p.packed, o / 2, n / 2), scales = mx_buffer(p.scales, o / 32, n / 32);
    E v[MX_U];
#pragma unroll
    for (int u = 0; u < MX_U; ++u) v[u].load(x, (512 * u + 8 * l) * E::SIZE);
#pragma unroll
    for (int u = 0; u < MX_U; ++u) {
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = max(top, v[u].bits(k) & 0x7fffffffu);
        top = quad_max(top);
        const bool finite = top < 0x7f800000u;
        const uint32_t e = top >> 23, byte = finite ? (e > 2 ? e - 2 : 0) : 255u;
        const float scale = __uint_as_float(finite ? byte << 23 : 0x3f800000u);
        auto f = [&](int k) { return __uint_as_float(v[u].bits(k)); };
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(0), f(1), scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(2), f(3), scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(4), f(5), scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(6), f(7), scale, 3);
        __builtin_amdgcn_raw_buffer_store_b32(finite ? w : 0u, packed, 256 * u + 4 * l, 0, 0);
        // (one lane of a block's four; the others' offset is past the end)
        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)byte, scales, l & 3 ? 64 * MX_U : 16 * u + l / 4, 0, 0);
    }
}

// value = (+-) e2m1 * 2^(byte - 127), exact in f32 and bf16 (subnormal there
// below byte 1 or 2, infinite where it passes the type's largest); NaN at byte
// 255.  A lane owns a word: 8 values.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(64 * MX_WAVES) mxfp4_dequantize_kernel(Mxfp4DequantizeParams p, int64_t first, int64_t per_row) {
    const int64_t unit = first + (int64_t)blockIdx.x * MX_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = p.rows == 1 ? 0 : unit / per_row;
    if (row >= p.rows) return;
    const int l = threadIdx.x & 63;
    const int64_t c0 = (unit - row * per_row) * (512 * MX_U), o = row * p.cols + c0;
    if (c0 >= p.cols) return;  // (one long row: a wave past its end)
    const int n = (int)min(p.cols - c0, (int64_t)512 * MX_U);  // of this wave
    using E = MxEight<F32, VEC>;
    const __amdgpu_buffer_rsrc_t out = mx_buffer(p.out, (row * p.out_stride + c0) * E::SIZE, n * E::SIZE);
    const __amdgpu_buffer_rsrc_t packed = mx_buffer(p.packed, o / 2, n / 2), scales = mx_buffer(p.scales, o / 32, n / 32);
    uint32_t w[MX_U];
    uint32_t b[MX_U];
#pragma unroll
    for (int u = 0; u < MX_U; ++u) {
        w[u] = __builtin_amdgcn_raw_buffer_load_b32(packed, 256 * u + 4 * l, 0, 0);
        b[u] = __builtin_amdgcn_raw_buffer_load_b8(scales, 16 * u + l / 4, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < MX_U; ++u) {
        const float scale = __uint_as_float(b[u] << 23);
        E y;
        if constexpr (F32) {
            const f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], scale, 0),
                                __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], scale, 1),
                                __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], scale, 2),
                                __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], scale, 3)};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if constexpr (VEC)
                    y.v[k >> 2][k & 3] = __float_as_uint(v[k >> 1][k & 1]);
                else
                    y.v[k] = __float_as_uint(v[k >> 1][k & 1]);
            }
        } else {
            const u32x4 v = __builtin_bit_cast(u32x4, mxfp4_bf16(w[u], scale));
            if constexpr (VEC) {
                y.v[0] = v;
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) y.v[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
            }
        }
        y.store(out, (512 * u + 8 * l) * E::SIZE);
    }
}

// rows laid out without gaps are one long row
template <typename P>
int64_t mx_units(P& p, int64_t& stride, int64_t& per_row) {
    if (stride == p.cols) {
        p.cols *= p.rows;
        stride = p.cols;
        p.rows = 1;
    }
    per_row = (p.cols + 512 * MX_U - 1) / (512 * MX_U);
    return per_row * p.rows;
}

template <typename K, typename P>
hipError_t mx_launch(K kern, const P& p, int64_t units, int64_t per_row, hipStream_t st) {
    // grids of less than 2^32 threads
    constexpr int64_t MOST = (1ll << 23) * MX_WAVES;
    for (int64_t first = 0; first < units; first += MOST) {
        const int64_t grid = (std::min(MOST, units - first) + MX_WAVES - 1) / MX_WAVES;
        hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * MX_WAVES), 0, st, p, first, per_row);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_mxfp4_quantize(Mxfp4QuantizeParams p, hipStream_t st) {
    const int size = p.x_f32 ? 4 : 2;
    const bool vec = ((uintptr_t)p.x & 15) == 0 && (p.rows == 1 || p.x_stride * size % 16 == 0);
    if (p.rows == 1) p.x_stride = p.cols;
    int64_t per_row;
    const int64_t units = mx_units(p, p.x_stride, per_row);
    if (p.x_f32)
        return vec ? mx_launch(mxfp4_quantize_kernel<true, true>, p, units, per_row, st)
                   : mx_launch(mxfp4_quantize_kernel<true, false>, p, units, per_row, st);
    return vec ? mx_launch(mxfp4_quantize_kernel<false, true>, p, units, per_row, st)
               : mx_launch(mxfp4_quantize_kernel<false, false>, p, units, per_row, st);
}

hipError_t launch_mxfp4_dequantize(Mxfp4DequantizeParams p, hipStream_t st) {
    const int size = p.out_f32 ? 4 : 2;
    const bool vec = ((uintptr_t)p.out & 15) == 0 && (p.rows == 1 || p.out_stride * size % 16 == 0);
    if (p.rows == 1) p.out_stride = p.cols;
    int64_t per_row;
    const int64_t units = mx_units(p, p.out_stride, per_row);
    if (p.out_f32)
        return vec ? mx_launch(mxfp4_dequantize_kernel<true, true>, p, units, per_row, st)
                   : mx_launch(mxfp4_dequantize_kernel<true, false>, p, units, per_row, st);
    return vec ? mx_launch(mxfp4_dequantize_kernel<false, true>, p, units, per_row, st)
               : mx_launch(mxfp4_dequantize_kernel<false, false>, p, units, per_row, st);
}

}  // namespace mr
