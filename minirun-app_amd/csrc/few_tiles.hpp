// What the MFMA kernels for few tokens share (skinny.hip, affine_gemm.hip,
// mxfp4_few.hip): buffer offsets past every row, and the sum of the waves' parts.
#pragma once
#include "mr_kernels.hpp"

namespace mr {

namespace {

// byte offsets outside every buffer (host check: buffers under 2^30 bytes), of
// a lane's row and of a k-block past the row's end; their sum is outside too
constexpr uint32_t SK_OOB_ROW = 0x40000000u, SK_OOB_K = 0x80000000u;

// the resource in scalar registers (its inputs are uniform, but may have been
// computed in vector registers)
__device__ __forceinline__ i32x4 uniform_rsrc(const void* base, uint32_t bytes) {
    i32x4 r = buffer_rsrc(base, bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_readfirstlane(r[i]);
    return r;
}

// partial sums of the waves -> LDS -> one f32x4 per (tile, lane): emit(r, t,
// lane, value) of row tile r, token tile t
template <int RT, int TT, int NW, typename F>
__device__ __forceinline__ void sk_reduce(char* lds, const f32x4 (&acc)[RT][TT], F emit) {
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    constexpr int P = RT * TT * 64;
    f32x4* d = (f32x4*)lds;
    __syncthreads();  // every wave is done with its ring
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) d[w * P + (r * TT + t) * 64 + l] = acc[r][t];
    __syncthreads();
    for (int i = tid; i < P; i += 64 * NW) {
        f32x4 v[NW];
#pragma unroll
        for (int k = 0; k < NW; ++k) v[k] = d[k * P + i];
#pragma unroll
        for (int n = 1; n < NW; n *= 2)
#pragma unroll
            for (int k = 0; k + n < NW; k += 2 * n) v[k] += v[k + n];
        const int rt = __builtin_amdgcn_readfirstlane(i >> 6);
        emit(rt / TT, rt % TT, i & 63, v[0]);
    }
}

}  // namespace

}  // namespace mr
