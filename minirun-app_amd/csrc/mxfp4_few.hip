// Products with MXFP4 weights for few rows: y[t][o] = sum_i x[t][i] w[o][i],
// for the tokens of one matrix, or for rows in expert order, each expert's rows
// times its own matrix of a stack.  x is bf16, f32, or MXFP4 itself.
//
// What bounds it: the weights' bytes from HBM, 17 / 32 of a byte each, read
// once per 16 TT rows of x; then x's lines from L2, about two clocks each; and
// for small matrices the chain of a workgroup (find the tile, load, sum).  A
// workgroup owns 16 RT weight rows and 16 TT rows of x, and its NW waves split
// K: wave w takes the entries w, w + NW, ... of 256 k.  Each wave streams its
// entries into a ring of S entries in LDS by DMA and waits for its own loads
// alone; the waves' sums meet in LDS once, at the end, in a fixed order.
//
// An entry is one 128-byte line of each weight row, the 16 bytes with the row's
// eight scale bytes, and 256 values of each row of x.  A lane of the MFMA holds
// weight row l % 16 and blocks 2 (l / 16) + 0..1 of the entry's eight: 16 bytes
// of codes and one scale byte each, so nothing is exchanged between lanes.
//   x in bf16: the block's four words become bf16 with their scale (exact: two
//     significant bits), one v_mfma_f32_16x16x32_bf16 each, with the eight
//     values of x that belong to the word.
//   x in f32: the same with x cut into three bf16 parts by truncation, whose
//     sum is x exactly.
//   x in MXFP4: v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands' codes
//     and scale bytes as they are.
// Chains start from zero per entry and are added to the running sums in f32.
//
// K is a multiple of 32.  In an entry that the row ends in, codes of W and x
// past the end are loaded as zeros (through the buffers' bounds), and scale
// bytes past the end, which may be the next row's, are replaced by that of 1.
// Scale rows start on any byte: the 16 bytes start on the word before.
#include <algorithm>

#include "few_tiles.hpp"
#include "mxfp4_tiles.hpp"

namespace mr {

namespace {

template <int XT>
struct XEntry {  // of 256 k
    static constexpr int BYTES = XT == MX_X_BF16 ? 512 : (XT == MX_X_F32 ? 1024 : 128);
    static constexpr int CHUNKS = BYTES / 16;  // of 16 bytes per row
    static constexpr int RPI = 64 / CHUNKS;    // rows per DMA instruction
    static constexpr int KPC = 256 / CHUNKS;   // values per chunk
    // chunk c of row r is in slot c ^ swizzle(r), so that the 16 rows of a
    // read of one chunk lie in 16 bank groups
    static __device__ __forceinline__ int swizzle(int r) { return XT == MX_X_MXFP4 ? (r >> 1) & 7 : r & 15; }
};

// the three bf16 parts of eight f32 values, by truncation
__device__ __forceinline__ void split3(const u32x4& a, const u32x4& b, bf16x8 (&part)[3]) {
    u32x4 v[3];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t x[2] = {k < 2 ? a[2 * k] : b[2 * k - 4], k < 2 ? a[2 * k + 1] : b[2 * k - 3]};
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            v[n][k] = (x[0] >> 16) | (x[1] & 0xffff0000u);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float f = __uint_as_float(x[h]), top = __uint_as_float(x[h] & 0xffff0000u);
                x[h] = fabsf(f) == INFINITY ? 0u : __float_as_uint(f - top);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < 3; ++n) part[n] = __builtin_bit_cast(bf16x8, v[n]);
}

template <int XT, int RT, int TT, int XI, int S, int NW>
struct FewShape {
    using X = XEntry<XT>;
    static constexpr int XS = XT == MX_X_MXFP4 ? 1 : 0;  // DMA instructions of x's scales (W's: one)
    static constexpr int NI = 2 * RT + 1 + XI + XS;
    static constexpr int SOFF = 2048 * RT, XOFF = SOFF + 1024, XSOFF = XOFF + 1024 * XI, ENTRY = XSOFF + 1024 * XS;
    static constexpr int ROWS = XI * X::RPI;             // rows of x in an entry
    static constexpr int BM = ROWS < 16 * TT ? ROWS : 16 * TT;  // rows of x per workgroup
    static constexpr size_t LDS = std::max<size_t>((size_t)NW * S * ENTRY, (size_t)NW * RT * TT * 1024);
    static_assert((S - 1) * NI < 64, "vmcnt range");
    static_assert(RT <= 4 && TT <= 4 && (ROWS >= 16 * TT || (TT == 1 && (ROWS & (ROWS - 1)) == 0)), "rows of an entry");
    static_assert(LDS <= 163840, "LDS");
};

template <int XT, int RT, int TT, int XI, int S, int NW, bool ROUTED>
__global__ void __launch_bounds__(64 * NW) mxfp4_few_kernel(Mxfp4GemmParams p, int blocks) {
    using F = FewShape<XT, RT, TT, XI, S, NW>;
    using X = XEntry<XT>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int l = threadIdx.x & 63, q = l >> 4, lr = l & 15;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n_tiles = (p.N + 16 * RT - 1) / (16 * RT);
    int tile, m0, toks;
    int64_t first_row = 0;  // weight row 0 of the expert
    if constexpr (ROUTED) {
        MxTile t;
        if (!mx_find_tile<F::BM>(p.offsets, p.experts, p.pairs, n_tiles, t)) return;
        tile = t.n_tile;
        m0 = t.row;
        toks = t.rows;
        first_row = (int64_t)t.expert * p.N;
    } else {
        int tb;
        sk_tile(blockIdx.x, blocks, tile, tb);
        if (tile >= n_tiles) return;
        m0 = tb * F::BM;
        toks = min(F::BM, p.M - m0);
    }
    const int n0 = tile * 16 * RT, rows = min(16 * RT, p.N - n0);
    const uint32_t K = (uint32_t)p.K, wrow = K / 2, srow = K / 32;
    const int64_t xrow = XT == MX_X_MXFP4 ? wrow : p.ldx * (XT == MX_X_F32 ? 4 : 2);
    const i32x4 wres = uniform_rsrc((const char*)p.packed + (first_row + n0) * wrow, (uint32_t)rows * wrow);
    // scales through aligned words
    const uint64_t wsa = (uint64_t)(uintptr_t)p.scales + (first_row + n0) * srow;
    const uint32_t ws0 = (uint32_t)wsa & 3u;
    const i32x4 sres = uniform_rsrc((const void*)(uintptr_t)(wsa & ~3ull), (ws0 + (uint32_t)rows * srow + 3u) & ~3u);
    // x: from this workgroup's first row, or (rows by token) from row 0
    const bool by_token = ROUTED && p.pair_of_row != nullptr;
    const int64_t x_from = by_token ? 0 : m0, x_rows = by_token ? p.M : toks;
    const i32x4 xres = uniform_rsrc((const char*)p.x + x_from * xrow,
                                    (uint32_t)((x_rows - 1) * xrow + X::BYTES * (int64_t)K / 256));
    auto x_index = [&](int r) -> uint32_t {  // of this workgroup's -> row of the buffer
        r = min(r, toks - 1);
        if (by_token) return min((uint32_t)p.pair_of_row[m0 + r] / (uint32_t)p.per_token, (uint32_t)(p.M - 1));
        return (uint32_t)r;
    };
    const int nent = (int)((K + 255) / 256);
    const int n = w < nent ? (nent - 1 - w) / NW + 1 : 0;  // this wave's entries

    constexpr uint32_t PAST = 0xfffffff0u;  // an offset that reads zeros
    // W: lane l of an instruction fills slot l % 8 of row 8 i + l / 8 (odd i:
    // chunk ^ 4); its scales: lane l, row l
    const uint32_t ch8 = (l & 7) ^ (l >> 4);
    uint32_t wo[2 * RT], xo[XI], xso = 0, xsh[TT];
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) {
        const int r = 8 * i + (l >> 3);
        wo[i] = r < rows ? (uint32_t)r * wrow + 16u * (ch8 ^ (4 * (i & 1))) : SK_OOB_ROW;
    }
    const uint32_t so = l < rows ? (ws0 + (uint32_t)l * srow) & ~3u : SK_OOB_ROW;
    auto x_chunk = [&](int u) { return (uint32_t)((l % X::CHUNKS) ^ X::swizzle(X::RPI * u + l / X::CHUNKS)); };
#pragma unroll
    for (int u = 0; u < XI; ++u) xo[u] = x_index(X::RPI * u + l / X::CHUNKS) * (uint32_t)xrow + 16u * x_chunk(u);
    i32x4 xsres{};
    if constexpr (XT == MX_X_MXFP4) {
        const uint64_t xa = (uint64_t)(uintptr_t)p.x_scales + x_from * srow;
        const uint32_t xs0 = (uint32_t)xa & 3u;
        xsres = uniform_rsrc((const void*)(uintptr_t)(xa & ~3ull), (xs0 + (uint32_t)x_rows * srow + 3u) & ~3u);
        xso = (xs0 + x_index(l) * srow) & ~3u;
#pragma unroll
        for (int t = 0; t < TT; ++t) xsh[t] = ((xs0 + x_index(16 * t + lr) * srow) & 3u) + 2u * q;
    }

    char* ring = lds + w * S * F::ENTRY;
    auto issue = [&](int i, int slot) {
        const uint32_t ent = w + NW * i;
        const bool live = i < n;
        char* e = ring + slot * F::ENTRY;
#pragma unroll
        for (int c = 0; c < 2 * RT; ++c) {
            const bool in = live && 256u * ent + 32u * (ch8 ^ (4 * (c & 1))) < K;
            dma16_buf(wres, wo[c] + (in ? 128u * ent : SK_OOB_K), e + 1024 * c);
        }
        dma16_buf(sres, so + (live ? 8u * ent : SK_OOB_K), e + F::SOFF);
#pragma unroll
        for (int u = 0; u < XI; ++u) {
            const bool in = live && 256u * ent + X::KPC * x_chunk(u) < K && X::RPI * u + l / X::CHUNKS < toks;
            dma16_buf(xres, in ? xo[u] + (uint32_t)X::BYTES * ent : PAST, e + F::XOFF + 1024 * u);
        }
        if constexpr (XT == MX_X_MXFP4) dma16_buf(xsres, live && l < toks ? xso + 8u * ent : PAST, e + F::XSOFF);
    };
    f32x4 tot[RT][TT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) tot[r][t] = f32x4{};
    uint32_t wsh[RT];  // byte of the lane's first block in its row's 16
#pragma unroll
    for (int r = 0; r < RT; ++r) wsh[r] = ((ws0 + (uint32_t)(16 * r + lr) * srow) & 3u) + 2u * q;
#pragma unroll
    for (int s = 0; s < S; ++s) issue(s, s);
    // scale bytes of the lane's two blocks, those of 1 past the row's end
    auto scale_bytes = [&](const char* row, uint32_t at, bool in0, bool in1) -> uint32_t {
        const uint32_t* v = (const uint32_t*)row + (at >> 2);
        const uint32_t d = __builtin_amdgcn_alignbyte(v[1], v[0], at & 3u);
        return in1 ? d : (in0 ? (d & 0xffu) | 0x7f00u : 0x7f7fu);
    };
    int slot = 0;
    for (int i = 0; i < n; ++i) {
        wait_vmcnt<(S - 1) * F::NI>();
        const char* e = ring + slot * F::ENTRY;
        const uint32_t k0 = 256u * (w + NW * i) + 64u * q;
        const bool in0 = k0 < K, in1 = k0 + 32 < K;
        u32x4 fw[RT][2];
        uint32_t bw[RT], bx[TT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int u = 0; u < 2; ++u) fw[r][u] = *(const u32x4*)(e + 2048 * r + 128 * lr + 16 * ((2 * q + u) ^ (lr >> 1)));
            bw[r] = scale_bytes(e + F::SOFF + 16 * (16 * r + lr), wsh[r], in0, in1);
        }
        constexpr int XF = XT == MX_X_MXFP4 ? 1 : (XT == MX_X_F32 ? 8 : 4);  // 16-byte pieces per block
        u32x4 fx[TT][XF];
        auto read_x = [&](int u) {
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const int row = (16 * t + lr) % F::ROWS;
#pragma unroll
                for (int s = 0; s < XF; ++s)
                    fx[t][s] = *(const u32x4*)(e + F::XOFF + X::BYTES * row + 16 * ((XF * (2 * q + u) + s) ^ X::swizzle(row)));
            }
        };
        if constexpr (XT == MX_X_MXFP4) {
#pragma unroll
            for (int t = 0; t < TT; ++t) bx[t] = scale_bytes(e + F::XSOFF + 16 * (16 * t + lr), xsh[t], in0, in1);
        }
        // the slot is free once everything is in registers
        auto refill = [&] {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xc07f);  // the same, known to the compiler
            __builtin_amdgcn_sched_barrier(0);
            issue(i + S, slot);
        };
        f32x4 part[RT][TT];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < TT; ++t) part[r][t] = f32x4{};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            read_x(u);
            if (u == 1) refill();
            if constexpr (XT == MX_X_MXFP4) {
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int t = 0; t < TT; ++t)
                        part[r][t] = u ? mfma16_mxfp4<1>(fx[t][0], bx[t], fw[r][1], bw[r], part[r][t])
                                       : mfma16_mxfp4<0>(fx[t][0], bx[t], fw[r][0], bw[r], part[r][t]);
            } else {
                float sc[RT];
#pragma unroll
                for (int r = 0; r < RT; ++r) sc[r] = __uint_as_float(((bw[r] >> (8 * u)) & 255u) << 23);
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    bf16x8 wf[RT];
#pragma unroll
                    for (int r = 0; r < RT; ++r) wf[r] = mxfp4_bf16(fw[r][u][s], sc[r]);
#pragma unroll
                    for (int t = 0; t < TT; ++t) {
                        if constexpr (XT == MX_X_F32) {
                            bf16x8 xf[3];
                            split3(fx[t][2 * s], fx[t][2 * s + 1], xf);
#pragma unroll
                            for (int r = 0; r < RT; ++r)  // small parts first
                                part[r][t] = mfma16(xf[0], wf[r], mfma16(xf[1], wf[r], mfma16(xf[2], wf[r], part[r][t])));
                        } else {
#pragma unroll
                            for (int r = 0; r < RT; ++r) part[r][t] = mfma16(__builtin_bit_cast(bf16x8, fx[t][s]), wf[r], part[r][t]);
                        }
                    }
                }
            }
        }
        slot = slot + 1 == S ? 0 : slot + 1;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < TT; ++t) tot[r][t] += part[r][t];
    }
    wait_vmcnt<0>();
    sk_reduce<RT, TT, NW>(lds, tot, [&](int r, int t, int lane, f32x4 v) {
        const int nn = 16 * r + (lane & 15);
        if (nn >= rows) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = 16 * t + 4 * (lane >> 4) + e;
            if (m >= toks) break;
            const int64_t o = (int64_t)(m0 + m) * p.ldy + n0 + nn;
            if (p.y_f32)
                ((float*)p.y)[o] = v[e];
            else
                ((uint16_t*)p.y)[o] = f32_to_bf16_bits(v[e]);
        }
    });
}

template <int XT, int RT, int TT, int XI, int S, int NW>
hipError_t launch_few(const Mxfp4GemmParams& p, hipStream_t st) {
    using F = FewShape<XT, RT, TT, XI, S, NW>;
    constexpr size_t lds = F::LDS;
    const bool routed = p.offsets != nullptr;
    const auto kern = routed ? mxfp4_few_kernel<XT, RT, TT, XI, S, NW, true> : mxfp4_few_kernel<XT, RT, TT, XI, S, NW, false>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const int64_t tiles = (p.N + 16 * RT - 1) / (16 * RT), blocks = ((int64_t)p.M + F::BM - 1) / F::BM;
    const int64_t grid = routed ? (mx_tile_bound(p, F::BM) * tiles + 7) / 8 * 8 : (tiles + 7) / 8 * 8 * blocks;
    if (grid * 64 * NW >= (1ll << 32)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * NW), lds, st, p, (int)blocks);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mxfp4_few(const Mxfp4GemmParams& p, hipStream_t st) {
    // rows of x that one workgroup takes: all, or for experts about the mean
    const int m = p.offsets ? (p.pairs + p.experts - 1) / p.experts : p.M;
    if (p.x_kind == MX_X_MXFP4) return m <= 16 ? launch_few<2, 2, 1, 2, 2, 8>(p, st) : launch_few<2, 2, 4, 8, 1, 8>(p, st);
    if (p.x_kind == MX_X_F32) return m <= 16 ? launch_few<1, 2, 1, 16, 1, 4>(p, st) : launch_few<1, 2, 2, 32, 1, 4>(p, st);
    if (m <= 2 && (!p.offsets || p.pairs <= 4096)) return launch_few<0, 2, 1, 1, 3, 8>(p, st);
    return m <= 16 ? launch_few<0, 2, 1, 8, 1, 8>(p, st) : launch_few<0, 2, 4, 32, 1, 4>(p, st);
}

// as many workgroups as a routed call can need in a grid of less than 2^32
// threads
bool mxfp4_gemm_fits(const Mxfp4GemmParams& p) {
    return !p.offsets || (mx_tile_bound(p, 16) * ((p.N + 31) / 32) + 7) * 512 < (1ll << 32);
}

// Rows per large tile (0: the kernel for few rows).
static int tile_rows(const Mxfp4GemmParams& p, int cu_count) {
    if (p.x_kind == MX_X_F32) return 0;
    const int64_t m = p.offsets ? (p.pairs + p.experts - 1) / p.experts : p.M;
    if (m < 64) return 0;
    const int64_t n_tiles = (p.N + 255) / 256, m_tiles = (m + 255) / 256 * (p.offsets ? p.experts : 1);
    return m > 128 && n_tiles * m_tiles >= cu_count ? 256 : 128;
}

// A matrix's tokens in as many launches as grids of less than 2^32 threads
// take (one, up to 2^23 workgroups of 16 tokens x 32 weight rows).
hipError_t launch_mxfp4_gemm(const Mxfp4GemmParams& p, int cu_count, hipStream_t st) {
    const int tm = tile_rows(p, cu_count);
    if (p.offsets) return tm ? launch_mxfp4_tiles(p, tm, st) : launch_mxfp4_few(p, st);
    const int64_t most = (((int64_t)1 << 23) / ((p.N + 31) / 32 + 7) - 1) * 16 / 256 * 256;
    for (int64_t m = 0; m < p.M; m += most) {
        Mxfp4GemmParams q = p;
        q.M = (int)std::min<int64_t>(most, p.M - m);
        const int64_t row = p.x_kind == MX_X_MXFP4 ? p.K / 2 : p.ldx * (p.x_kind == MX_X_F32 ? 4 : 2);
        q.x = (const char*)p.x + m * row;
        if (p.x_scales) q.x_scales = p.x_scales + m * (p.K / 32);
        q.y = (char*)p.y + m * p.ldy * (p.y_f32 ? 4 : 2);
        const hipError_t e = tm ? launch_mxfp4_tiles(q, tm, st) : launch_mxfp4_few(q, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace mr
