// What the MXFP4 products share: the scaled MFMA, and which
// expert, rows and weight rows a workgroup of a routed product has.
#pragma once
#include <algorithm>

#include "mr_kernels.hpp"

namespace mr {

namespace {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

// D[16][16] += A . B^T over 128 k, both operands e2m1 codes with a scale byte
// per 32: lane l holds row l % 16 and block l / 16 (16 bytes of codes, element
// 0 in the low bits of the first word; its scale in byte SEL of the word).  D as
// v_mfma_f32_16x16x32_bf16's.
template <int SEL>
__device__ __forceinline__ f32x4 mfma16_mxfp4(const u32x4& a, uint32_t sa, const u32x4& b, uint32_t sb, const f32x4& c) {
    const i32x8 va = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i32x8 vb = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, SEL, (int)sa, SEL, (int)sb);
}

// D[32][32] += A . B^T over 64 k: lane l holds row l % 32 and block l / 32, and
// its scale in byte SEL of the word.  D as v_mfma_f32_32x32x16_bf16's.
template <int SEL>
__device__ __forceinline__ f32x16 mfma32_mxfp4(const u32x4& a, uint32_t sa, const u32x4& b, uint32_t sb, const f32x16& c) {
    const i32x8 va = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i32x8 vb = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, c, 4, 4, SEL, (int)sa, SEL, (int)sb);
}

struct MxTile {
    int expert, row, rows;  // rows row .. row + rows - 1 of y are the expert's
    int n_tile;             // of its weight rows
};

// Tiles of BM rows of one expert each, counted by expert; each has n_tiles
// tiles of weight rows.  The grid covers the most tiles that any offsets need;
// the tiles that there are go to the XCDs in equal runs of neighbours (blocks
// go to the 8 XCDs in turn), so that those of one expert mostly share an L2.
// Every wave finds its own tile: a lane counts the tiles of `run` experts.
// False: none is left for this workgroup.  Offsets are taken as they are, but
// no tile leaves [0, pairs).
template <int BM>
__device__ __forceinline__ bool mx_find_tile(const int32_t* offsets, int experts, int pairs, int n_tiles, MxTile& t) {
    constexpr int R = 4;  // experts per lane whose offsets stay in registers
    const int l = threadIdx.x & 63, run = (experts + 63) / 64;
    auto at = [&](int e) { return min(max(offsets[min(e, experts)], 0), pairs); };
    auto count = [](int lo, int hi) { return hi > lo ? (hi - lo + BM - 1) / BM : 0; };
    int off[R + 1], mine = 0;
#pragma unroll
    for (int k = 0; k <= R; ++k) off[k] = at(l * run + min(k, run));  // (in flight together)
#pragma unroll
    for (int k = 0; k < R; ++k) mine += count(off[k], off[k + 1]);
    for (int k = R, lo = off[R]; k < run; ++k) {
        const int hi = at(l * run + k + 1);
        mine += count(lo, hi);
        lo = hi;
    }
    const int incl = (int)wave_scan_incl((uint32_t)mine);
    const int64_t total = (int64_t)__builtin_amdgcn_readlane(incl, 63) * n_tiles;
    const int64_t per = (total + 7) / 8, j = blockIdx.x >> 3, id = (blockIdx.x & 7) * per + j;
    if (j >= per || id >= total) return false;
    const int i = (int)(id / n_tiles);
    int e = -1, row = 0, rows = 0;
    if (i >= incl - mine && i < incl) {
        int left = i - (incl - mine);
        auto look = [&](int k, int lo, int hi) {
            const int c = count(lo, hi);
            if (e < 0 && left < c) {
                e = l * run + k;
                row = lo + left * BM;
                rows = min(BM, hi - row);
            }
            left -= c;
        };
#pragma unroll
        for (int k = 0; k < R; ++k) look(k, off[k], off[k + 1]);
        for (int k = R, lo = off[R]; k < run && e < 0; ++k) {
            const int hi = at(l * run + k + 1);
            look(k, lo, hi);
            lo = hi;
        }
    }
    const uint64_t found = __ballot(e >= 0);
    if (!found) return false;
    const int from = __builtin_ctzll(found);
    t.expert = __builtin_amdgcn_readlane(e, from);
    t.row = __builtin_amdgcn_readlane(row, from);
    t.rows = __builtin_amdgcn_readlane(rows, from);
    t.n_tile = __builtin_amdgcn_readfirstlane((int)(id - (int64_t)i * n_tiles));
    return true;
}

// Rows of x for N rows of a tile that starts at row m0 of y and has `rows`
// (row_of(u): row u's place in the tile; past the last, the last): the place
// itself, or where rows come by token, the token's row.  The pairs' loads are in
// flight together: one after the other they were a third of a small call.
template <int N, typename F>
__device__ __forceinline__ void mx_x_rows(const Mxfp4GemmParams& p, bool by_token, int m0, int rows, uint32_t (&out)[N], F row_of) {
#pragma unroll
    for (int u = 0; u < N; ++u) out[u] = (uint32_t)min(row_of(u), rows - 1);
    if (by_token) {
#pragma unroll
        for (int u = 0; u < N; ++u) out[u] = (uint32_t)p.pair_of_row[m0 + (int)out[u]];
#pragma unroll
        for (int u = 0; u < N; ++u) out[u] = min(out[u] / (uint32_t)p.per_token, (uint32_t)(p.M - 1));
    }
}

// the most tiles of bm rows that `pairs` rows of `experts` experts can make
inline int64_t mx_tile_bound(const Mxfp4GemmParams& p, int bm) {
    return ((int64_t)p.pairs + (int64_t)std::min(p.experts, p.pairs) * (bm - 1)) / bm;
}

}  // namespace

}  // namespace mr
