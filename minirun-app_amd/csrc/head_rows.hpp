// A head's row in lanes: what the norms, rotations and cache appends of
// attention heads share.  A group of `lpr` lanes (a power of two) has one row,
// lane c of it columns 8 c .. 8 c + 7; lanes past the row hold zeros.
#pragma once

#include "mr_kernels.hpp"

namespace mr {

// Eight values of a row of n from column c, as stored: loaded first, widened where
// they are used.  VEC: whole 16-byte loads (c and n multiples of 8, the row aligned);
// else one by one, up to n.
template <bool F32, bool VEC>
struct HeadEight {
    u32x4 raw[F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* base, int64_t at, int c, int n) {
#pragma unroll
        for (int k = 0; k < (F32 ? 2 : 1); ++k) raw[k] = u32x4{};
        if constexpr (VEC) {
            if (c < n) {
                const u32x4* p = (const u32x4*)((const char*)base + (at + c) * (F32 ? 4 : 2));
#pragma unroll
                for (int k = 0; k < (F32 ? 2 : 1); ++k) raw[k] = p[k];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < n) {
                    if constexpr (F32)
                        raw[j >> 2][j & 3] = ((const uint32_t*)base)[at + c + j];
                    else
                        raw[0][j >> 1] |= (uint32_t)((const uint16_t*)base)[at + c + j] << (16 * (j & 1));
                }
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (F32)
                v[j] = __uint_as_float(raw[j >> 2][j & 3]);
            else
                v[j] = __uint_as_float(j & 1 ? raw[0][j >> 1] & 0xffff0000u : raw[0][j >> 1] << 16);
        }
    }
};

template <bool F32, bool VEC>
__device__ __forceinline__ void head_load(const void* base, int64_t at, int c, int n, float (&v)[8]) {
    HeadEight<F32, VEC> e;
    e.load(base, at, c, n);
    e.values(v);
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

// A row (token, head) of a tensor set and the offsets of its values, and the way to a
// row `by` further: no division, and one 64-bit addition or two for each tensor.
template <int N>
struct HeadWalk {
    struct Step {  // wave-uniform
        uint32_t token, head, heads;
        int64_t by[N], wrap[N];
    };
    uint32_t token, head;
    int64_t at[N];

    __device__ __forceinline__ static Step step(uint32_t by, uint32_t heads, const int64_t (&ts)[N], const int64_t (&hs)[N]) {
        Step s;
        s.token = by / heads;
        s.head = by - s.token * heads;
        s.heads = heads;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s.by[i] = s.token * ts[i] + s.head * hs[i];
            s.wrap[i] = ts[i] - heads * hs[i];
        }
        return s;
    }
    __device__ __forceinline__ void start(uint32_t id, uint32_t heads, const int64_t (&ts)[N], const int64_t (&hs)[N]) {
        token = id / heads;
        head = id - token * heads;
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] = token * ts[i] + head * hs[i];
    }
    __device__ __forceinline__ void next(const Step& s) {
        token += s.token;
        head += s.head;
        const bool wrap = head >= s.heads;
        if (wrap) head -= s.heads, ++token;
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] += s.by[i] + (wrap ? s.wrap[i] : 0);
    }
};

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

// How far into the rotated columns a lane's eight are, as angles lie: KIND says how
// the columns do.  ROPE_ADJACENT and ROPE_HALVES: col0 and half such that the eight
// columns are four whole pairs, or all on one side with their partners in one other
// lane, and table rows of whole 16-byte pieces; ROPE_ANY: anything.
template <int KIND>
struct HeadAngles {
    static constexpr int N = KIND == ROPE_ADJACENT ? 4 : 8;
    float co[N], si[N];
    // table row `at` (rope_row), columns c .. c + 7
    __device__ __forceinline__ void load(const HeadRope& r, int64_t at, int c) {
        const int k = c - r.col0;
        const int64_t table = max(at, (int64_t)0) * r.half;
        if constexpr (KIND == ROPE_ANY) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int x = k + j;
                if (x < 0 || x >= 2 * r.half) continue;
                const int i = r.halves ? (x >= r.half ? x - r.half : x) : x >> 1;
                co[j] = r.cos_t[table + i], si[j] = r.sin_t[table + i];
            }
        } else {
            if (k < 0 || k >= 2 * r.half) return;
            const int i = KIND == ROPE_ADJACENT ? k / 2 : (k >= r.half ? k - r.half : k);
#pragma unroll
            for (int x = 0; x < N; x += 4) {
                const f32x4 a = *(const f32x4*)(r.cos_t + table + i + x), b = *(const f32x4*)(r.sin_t + table + i + x);
#pragma unroll
                for (int j = 0; j < 4; ++j) co[x + j] = a[j], si[x + j] = b[j];
            }
        }
        if (at < 0) {  // the tables have no such row
#pragma unroll
            for (int j = 0; j < N; ++j) co[j] = si[j] = __builtin_nanf("");
        }
    }
};

// v (columns c .. c + 7 of a row) with columns [col0, col0 + 2 half) rotated (INV: by
// the negated angles):
//   (a, b) -> (a cos - b sin, a sin + b cos)
// for adjacent pairs, or for column i and column i + half.  `row` is the group's part
// of LDS (8 lpr values), through which ROPE_HALVES and ROPE_ANY hand partners over.
// T: float rounds every operation as written; double.  sum: if given, the magnitudes of
// the two terms of each result, added; of columns that stay, the value's.
template <int KIND, bool INV, typename T>
__device__ __forceinline__ void head_rotate(T (&v)[8], const HeadRope& r, const HeadAngles<KIND>& g, int c, T* row,
                                            float* sum = nullptr) {
    if (sum)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = __builtin_fabsf((float)v[j]);
    if constexpr (KIND != ROPE_ADJACENT) {
#pragma unroll
        for (int j = 0; j < 8; ++j) row[c + j] = v[j];
        wave_lds_fence();
    }
    auto turn = [&](T a, T p, float co, float si, bool second, int j) -> T {
        const T cc = co, ss = INV ? -si : si;
        if (sum) sum[j] = __builtin_fabsf((float)a * co) + __builtin_fabsf((float)p * si);
        if constexpr (sizeof(T) == 4)
            return second ? add_rn(mul_rn(p, ss), mul_rn(a, cc)) : sub_rn(mul_rn(a, cc), mul_rn(p, ss));
        else
            return second ? p * ss + a * cc : a * cc - p * ss;
    };
    const int k = c - r.col0;
    if constexpr (KIND == ROPE_ADJACENT) {
        if (k >= 0 && k < 2 * r.half) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const T a = v[2 * j], b = v[2 * j + 1];
                v[2 * j] = turn(a, b, g.co[j], g.si[j], false, 2 * j);
                v[2 * j + 1] = turn(b, a, g.co[j], g.si[j], true, 2 * j + 1);
            }
        }
    } else if constexpr (KIND == ROPE_HALVES) {
        if (k >= 0 && k < 2 * r.half) {
            const bool second = k >= r.half;
            const T* partner = row + (second ? c - r.half : c + r.half);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = turn(v[j], partner[j], g.co[j], g.si[j], second, j);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int x = k + j;
            if (x < 0 || x >= 2 * r.half) continue;
            const bool second = r.halves ? x >= r.half : (x & 1);
            const int d = r.halves ? r.half : 1;
            v[j] = turn(v[j], row[second ? c + j - d : c + j + d], g.co[j], g.si[j], second, j);
        }
    }
    if constexpr (KIND != ROPE_ADJACENT) wave_lds_fence();  // the next row's values come after these reads
}

}  // namespace mr
