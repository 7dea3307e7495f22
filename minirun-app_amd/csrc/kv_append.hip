// New tokens' keys and values into the pages of a cache, the keys normalised
// and rotated on the way, as bf16 or as MXFP4 (blocks of 32 values along a
// head: mxfp4.hip's rule).
//
//   key = R (w * (k / sqrt(mean(k^2) + eps))), value = v; each stored value is
//   rounded once, from the unrounded one
//
// A value next to a border of the 4-bit grid goes the wrong way if it is off by
// a rounding of f32, and a block's power with it.  So keys are computed in f32 with a
// bound of their error first, and rounded from both ends of what they may be: where
// these agree, so does the exact value between them.  A wave that has a value where
// they don't (of four rows of 128 one in 340 in MXFP4; in bf16, whose borders are nearer,
// one in 5 with the rotation alone, every other one with the norm too) computes its rows
// in f64 and hands them to the instructions that round as f32 "to odd": cut
// off, the last bit set if that lost anything, which no later rounding to fewer bits
// can tell from the f64 value.
//
// What bounds it, by 8192 tokens of 8 heads of 128 in bf16, not in the caches: HBM where
// they are stored as they are (in bf16 15.1 us, 4.4 TB/s); with norm and rotation the
// vector units (in MXFP4 19.4 to 20.5 us, 15 of them the issue of 9.2 million
// instructions; where it took 18.6, all keys in f64 22.2, f32's terms kept for it 20.5; in
// bf16, half of the waves in f64, 25.7 to 27, f64 alone 0.5 less).  The rotation alone in
// bf16, 20.2 to 21.1, is held by neither: 3.3 TB/s, and half of the time instructions; the
// registers (67) keep more rows from being under way.
//
// A group of dim / 8 lanes has one head's row, as in head_norm.hip; the four lanes of a
// block find its largest magnitude by two DPP steps.  Everything a row needs is asked for
// at once.
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

// Eight values as they are stored: bf16, or codes and the scale of the block that four
// lanes have.  `most`: the largest magnitude of the eight, or more in the same binade.
// The values of an MXFP4 block stand for 2^lift times as much (one lift for all of it).
struct Stored {
    u32x4 bf16;
    uint32_t codes, byte;
};

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ Stored narrow(bool mx, const float (&v)[8], uint32_t most, uint32_t lift = 0) {
    Stored s{};
    if (!mx) {
        s.bf16 = u32x4{pack_bf16x2_hw(v[0], v[1]), pack_bf16x2_hw(v[2], v[3]), pack_bf16x2_hw(v[4], v[5]),
                       pack_bf16x2_hw(v[6], v[7])};
        return s;
    }
    most = block_max(most);
    const bool finite = most < 0x7f800000u;
    const uint32_t e = most >> 23;
    s.byte = finite ? min((e > 2 ? e - 2 : 0) + lift, 254u) : 255u;
    const float scale = __uint_as_float(finite ? (s.byte - lift) << 23 : 0x3f800000u);
    uint32_t word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], scale, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], scale, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], scale, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], scale, 3);
    s.codes = finite ? word : 0u;
    return s;
}

__device__ __forceinline__ uint32_t most_of(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, magnitude(v[j]));
    return m;
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
    // everything is asked for at once, also for padding
    const bool key = blockIdx.y == 0, turn = key && p.turn, mx = p.k_scales;
    const int32_t slot = p.slots[token];
    HeadEight<F32, VEC> own;
    own.load(key ? p.k : p.v, token * (key ? p.k_ts : p.v_ts) + head * (key ? p.k_hs : p.v_hs), c, p.dim);
    HeadAngles<KIND> angles;
    float wt[8];
    auto terms = [&]() {
        if (p.rope.half) angles.load(p.rope, rope_row(p.rope, token), c);
        if (p.w) {
            head_load<VEC>(p.w, p.w_f32, 0, c, p.dim, wt);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) wt[j] = 1.f;
        }
    };
    if (turn) terms();
    // rows past the last and slots outside the pages: nothing is stored
    const int n = id < rows && slot >= 0 && slot < p.slot_end ? p.dim : 0;
    float x[8];
    own.values(x);
    Stored s;
    if (turn) {
        const int at = 8 * (group << p.lpr_log2);
        // With u = 2^-24: the sum of squares is off by 14 u of it (8 and 6 roundings), the
        // mean and eps by 17, the root (1 ulp of the instruction) by 8.5 + 2, so y by 12.5;
        // a rotation's result by 12.5 + 1 and 1 of its two terms' magnitudes, and each end
        // by one more: 15.5 u, 3 u without the norm.  That holds for normal numbers: a product
        // below them is off by 2^-150, which a large weight makes too much if it comes before
        // it, so such rows (zeros too, which it may have become) are left to f64, like rows
        // whose squares could leave f32's range and results that could; later ones are within
        // 2^-140, with cosines.
        float y[8], sum[8], ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[j];
        bool sure = true;
        if (p.norm) {
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
            for (int d = 1; d < p.lpr; d *= 2) ss += __shfl_xor(ss, d);
            sure = ss > 0x1p-100f && ss < 0x1p100f;
            const float inv = __builtin_amdgcn_rsqf(fmaf(ss, p.inv_dim, p.eps));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[j] *= inv;
                sure = sure && !__builtin_amdgcn_classf(y[j], 0xF0);  // (zeros and subnormal numbers)
                y[j] *= wt[j];
            }
        }
        if (p.rope.half) {
            head_rotate<KIND, false>(y, p.rope, angles, c, (float*)&sh[w][0] + at, sum);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] = __builtin_fabsf(y[j]);
        }
        const float u = p.norm ? 17 * 0x1p-24f : 4 * 0x1p-24f;
        float ends[2][8];
        uint32_t near = 0, far = 0;  // the largest magnitude is between these
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float off = fmaf(sum[j], u, 0x1p-140f);
            ends[0][j] = y[j] - off, ends[1][j] = y[j] + off;
            near = max(near, min(magnitude(ends[0][j]), magnitude(ends[1][j])));
            far = max(far, max(magnitude(ends[0][j]), magnitude(ends[1][j])));
        }
        sure = sure && far < 0x7e800000u;  // 2^126
        s = narrow(mx, ends[0], far);
        const Stored t = narrow(mx, ends[1], far);
        if (mx)
            sure = sure && s.codes == t.codes && block_max(near) >> 23 == block_max(far) >> 23;
        else
            sure = sure && ((s.bf16[0] ^ t.bf16[0]) | (s.bf16[1] ^ t.bf16[1]) | (s.bf16[2] ^ t.bf16[2]) | (s.bf16[3] ^ t.bf16[3])) == 0;
        if (__builtin_amdgcn_ballot_w64(c < n && !sure)) {
            asm volatile("" ::: "memory");  // (read again, rather than kept in registers that other waves could use)
            terms();
            own.load(p.k, token * p.k_ts + head * p.k_hs, c, p.dim);
            own.values(x);
            double z[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = x[j];
            if (p.norm) {
                double sq = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) sq += z[j] * z[j];
                for (int d = 1; d < p.lpr; d *= 2) sq += __shfl_xor(sq, d);
                const double inv = 1.0 / sqrt(sq / p.dim + (double)p.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] = wt[j] * (z[j] * inv);
            }
            if (p.rope.half) head_rotate<KIND, false>(z, p.rope, angles, c, &sh[w][at]);
            // A block of values of 2^126 or more, which may pass f32, takes part 2^-8 times as
            // large (what that cuts off its small values has code 0 beside the large one).
            uint32_t lift = 0;
            if (mx) {
                uint32_t top = 0;  // sign, exponent and first bits of an f64, without the sign
#pragma unroll
                for (int j = 0; j < 8; ++j) top = max(top, (uint32_t)(__builtin_bit_cast(uint64_t, z[j]) >> 32) & 0x7fffffffu);
                top = block_max(top);
                if (top >= 1149u << 20 && top < 0x7ff00000u) lift = 8;
            }
            const double by = lift ? 0x1p-8 : 1.0;
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = to_odd(z[j] * by);
            s = narrow(mx, y, most_of(y), lift);
        }
    } else {
        s = narrow(mx, x, most_of(x));
    }
    if (c >= n) return;
    const uint32_t page = (uint32_t)slot / (uint32_t)p.page_size;
    const int64_t row = head * p.page_size + ((uint32_t)slot - page * (uint32_t)p.page_size);
    if (!mx) {
        *(u32x4*)((uint16_t*)(key ? p.k_pages : p.v_pages) + page * p.page_stride + row * p.dim + c) = s.bf16;
        return;
    }
    ((uint32_t*)(key ? p.k_pages : p.v_pages))[page * p.page_stride + (row * p.dim + c) / 8] = s.codes;
    if ((l & 3) == 0) (key ? p.k_scales : p.v_scales)[page * p.scale_stride + (row * p.dim + c) / 32] = (uint8_t)s.byte;
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
    p.inv_dim = 1.f / p.dim;
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
