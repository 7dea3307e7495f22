// A head's row in lanes: what the norms, rotations and cache appends of
// attention heads share.  A group of `lpr` lanes (a power of two) has one row,
// lane c of it columns 8 c .. 8 c + 7; lanes past the row hold zeros.
#pragma once

#include "mr_kernels.hpp"

namespace mr {

// Eight values of a row of n from column c as f32.  VEC: whole 16-byte loads
// (c and n multiples of 8, the row aligned); else one by one, up to n.
template <bool F32, bool VEC>
__device__ __forceinline__ void head_load(const void* base, int64_t at, int c, int n, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if constexpr (VEC) {
        if (c < n) {
            if constexpr (F32) {
                const f32x4* p = (const f32x4*)((const float*)base + at + c);
                const f32x4 a = p[0], b = p[1];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
            } else {
                const u32x4 a = *(const u32x4*)((const uint16_t*)base + at + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(j & 1 ? a[j >> 1] & 0xffff0000u : a[j >> 1] << 16);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < n)
                v[j] = F32 ? ((const float*)base)[at + c + j] : bf16_bits_to_f32(((const uint16_t*)base)[at + c + j]);
    }
}

template <bool VEC>
__device__ __forceinline__ void head_load(const void* base, int f32, int64_t at, int c, int n, float (&v)[8]) {
    if (f32)
        head_load<true, VEC>(base, at, c, n, v);
    else
        head_load<false, VEC>(base, at, c, n, v);
}

template <bool VEC>
__device__ __forceinline__ void head_store(void* base, int f32, int64_t at, int c, int n, const float (&v)[8]) {
    if constexpr (VEC) {
        if (c >= n) return;
        if (f32) {
            f32x4* p = (f32x4*)((float*)base + at + c);
            p[0] = f32x4{v[0], v[1], v[2], v[3]};
            p[1] = f32x4{v[4], v[5], v[6], v[7]};
        } else {
            *(u32x4*)((uint16_t*)base + at + c) = u32x4{pack_bf16x2_hw(v[0], v[1]), pack_bf16x2_hw(v[2], v[3]),
                                                        pack_bf16x2_hw(v[4], v[5]), pack_bf16x2_hw(v[6], v[7])};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < n) {
                if (f32)
                    ((float*)base)[at + c + j] = v[j];
                else
                    ((uint16_t*)base)[at + c + j] = f32_to_bf16_bits(v[j]);
            }
    }
}

// This wave's LDS writes before its own LDS reads of other lanes' values (a
// wave's LDS operations are done in order; the compiler has to keep them so).
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The row of the angle tables for a token: positions[token], or the token
// itself; -1 where the tables have no such row.
__device__ __forceinline__ int64_t rope_row(const HeadRope& r, int64_t token) {
    const int64_t at = r.positions ? (int64_t)r.positions[token] : token;
    return at >= 0 && at < r.rows ? at : -1;
}

// v (columns c .. c + 7 of a row) with columns [col0, col0 + 2 half) rotated by
// the angles of table row `at` (INV: by the negated ones):
//   (a, b) -> (a cos - b sin, a sin + b cos)
// for adjacent pairs, or for column i and column i + half.  KIND: how the
// columns lie.  ROPE_ADJACENT and ROPE_HALVES: col0 and half such that the
// lane's eight columns are four whole pairs, or all on one side with their
// partners in one other lane, and table rows of whole 16-byte pieces;
// ROPE_ANY: anything.  `row` is the group's part of LDS (8 lpr values), which
// ROPE_HALVES and ROPE_ANY use to hand partners over.  T: float rounds every
// operation as written; double.
template <int KIND, bool INV, typename T>
__device__ __forceinline__ void head_rotate(T (&v)[8], const HeadRope& r, int64_t at, int c, T* row) {
    if constexpr (KIND != ROPE_ADJACENT) {
#pragma unroll
        for (int j = 0; j < 8; ++j) row[c + j] = v[j];
        wave_lds_fence();
    }
    const float nan = __builtin_nanf("");
    auto turn = [&](T a, T p, float co, float si, bool second) -> T {
        const T cc = at < 0 ? nan : co, ss = at < 0 ? nan : (INV ? -si : si);
        if constexpr (sizeof(T) == 4)
            return second ? add_rn(mul_rn(p, ss), mul_rn(a, cc)) : sub_rn(mul_rn(a, cc), mul_rn(p, ss));
        else
            return second ? p * ss + a * cc : a * cc - p * ss;
    };
    const int64_t table = max(at, (int64_t)0) * r.half;
    if constexpr (KIND == ROPE_ADJACENT) {
        const int k = c - r.col0;
        if (k >= 0 && k < 2 * r.half) {
            const f32x4 co = *(const f32x4*)(r.cos_t + table + k / 2), si = *(const f32x4*)(r.sin_t + table + k / 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const T a = v[2 * j], b = v[2 * j + 1];
                v[2 * j] = turn(a, b, co[j], si[j], false);
                v[2 * j + 1] = turn(b, a, co[j], si[j], true);
            }
        }
    } else if constexpr (KIND == ROPE_HALVES) {
        const int k = c - r.col0;
        if (k >= 0 && k < 2 * r.half) {
            const bool second = k >= r.half;
            const int i = second ? k - r.half : k;
            const T* partner = row + (second ? c - r.half : c + r.half);
            const f32x4 c0 = *(const f32x4*)(r.cos_t + table + i), c1 = *(const f32x4*)(r.cos_t + table + i + 4);
            const f32x4 s0 = *(const f32x4*)(r.sin_t + table + i), s1 = *(const f32x4*)(r.sin_t + table + i + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = turn(v[j], partner[j], c0[j], s0[j], second);
                v[4 + j] = turn(v[4 + j], partner[4 + j], c1[j], s1[j], second);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = c + j - r.col0;
            if (k < 0 || k >= 2 * r.half) continue;
            const bool second = r.halves ? k >= r.half : (k & 1);
            const int i = r.halves ? (second ? k - r.half : k) : k >> 1;
            const int d = r.halves ? r.half : 1;
            v[j] = turn(v[j], row[second ? c + j - d : c + j + d], r.cos_t[table + i], r.sin_t[table + i], second);
        }
    }
    if constexpr (KIND != ROPE_ADJACENT) wave_lds_fence();  // the next row's values come after these reads
}

}  // namespace mr
