// Products with MXFP4 weights for few rows: y[t][o] = sum_i x[t][i] w[o][i],
// for the tokens of one matrix, or for rows in expert order, each expert's rows
// times its own matrix of a stack.  x is bf16, f32, or MXFP4 itself.
//
// What bounds it: the weights' bytes from HBM, 17 / 32 of a byte each, read
// once per 16 TT rows of x; then x's lines from L2, about two clocks each; and
// for small matrices the chain of a workgroup (find the tile, load, sum).  A
// workgroup owns 16 RT weight rows and 16 TT rows of x, and its NW waves split
// K: wave w takes the entries w, w + NW, ... of 256 k.  Each wave has room for one
// entry in LDS, filled by DMA: once it is in registers the next one goes out, and
// the products of this one, the other waves and the other workgroups of the CU
// cover its way.  A wave waits for its own loads alone; the waves' sums meet in LDS
// once, at the end, in a fixed order.
//
// An entry is one 128-byte line of each weight row, the 16 bytes with the row's
// eight scale bytes, and 256 values of each row of x.  A lane of the MFMA holds
// weight row l % 16 and blocks 2 (l / 16) + 0..1 of the entry's eight: 16 bytes
// of codes and one scale byte each, so nothing is exchanged between lanes.
//   x in bf16: the block's four words become bf16 with their scale (exact: two
//     significant bits), one v_mfma_f32_16x16x32_bf16 each, with the eight
//     values of x that belong to the word.
//   x in f32: the same with x cut into three bf16 parts by truncation, whose
//     sum is x exactly.  Against an infinite weight (scale bytes 253 and 254) a
//     part that is zero makes the sum NaN: outputs that are NaN, of weight rows
//     that have such bytes, are computed again, x uncut.
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
    // Chunk c of row r is in slot c ^ swizzle(r), so that the 16 rows of a read of
    // one chunk lie in 16 bank groups.  bf16: with bits 3 and 4 of c exchanged, so
    // that lanes of the first two of a read's four blocks, which it takes together,
    // have the same groups for the same rows (four clocks less a read; with the two
    // rows of one token's kernels four more, beside a wait for the weights).
    static __device__ __forceinline__ int swizzle(int r) { return XT == MX_X_MXFP4 ? (r >> 1) & 7 : r & 15; }
    static __device__ __forceinline__ int swap(int c) { return XT == MX_X_BF16 ? (c & 7) | (c & 8) << 1 | (c & 16) >> 1 : c; }
    static __device__ __forceinline__ int slot(int c, int r) { return swap(c) ^ swizzle(r); }
    static __device__ __forceinline__ int chunk(int slot, int r) { return swap(slot ^ swizzle(r)); }
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

// One output of f32 activations again, by a whole wave: the sum over a row of x
// and one of W, weights as bf16.  It ends at the first NaN.
__device__ __forceinline__ float mx_f32_again(const float* x, const uint32_t* packed, const uint8_t* scales, int K) {
    float d = 0.f;
#pragma unroll 1
    for (int k = 8 * (threadIdx.x & 63); k < (K + 511) / 512 * 512; k += 512) {
        if (k < K) {
            const u32x4 v[2] = {*(const u32x4*)(x + k), *(const u32x4*)(x + k + 4)};
            const u32x4 wv = __builtin_bit_cast(u32x4, mxfp4_bf16(packed[k >> 3], __uint_as_float((uint32_t)scales[k >> 5] << 23)));
#pragma unroll
            for (int i = 0; i < 8; ++i)
                d = fmaf(__uint_as_float(v[i >> 2][i & 3]), __uint_as_float(i & 1 ? wv[i >> 1] & 0xffff0000u : wv[i >> 1] << 16), d);
        }
        if (__ballot(d != d)) return NAN;
    }
    return wave_sum(d);
}

// Those that are NaN of a wave's outputs again, if any of the weight rows that they
// are of may hold infinite weights: `words` has those rows' scale bytes, n of them
// words.  Of lane l, bit i of `again` is an output in row m of the tile from m0 on and
// weight row n of the expert, m and n from at(l, i); stored by that lane through
// store(m, n, value).
template <typename At, typename Store>
__device__ __forceinline__ void mx_f32_nans(const Mxfp4GemmParams& p, bool by_token, int64_t first_row, int m0,
                                            const uint32_t* words, int n_words, uint32_t again, At at, Store store) {
    const int l = threadIdx.x & 63;
    uint64_t lanes = __ballot(again != 0);
    if (__builtin_expect(lanes == 0, 1)) return;
    bool mine = false;
#pragma unroll 4
    for (int i = l; i < n_words; i += 64) {
        const uint32_t v = words[i];
#pragma unroll
        for (int k = 0; k < 32; k += 8) mine |= ((v >> k) & 255u) - 253u < 2u;
    }
    if (!__ballot(mine)) return;
#pragma unroll 1
    while (lanes) {
        const int from = __builtin_ctzll(lanes);
        lanes &= lanes - 1;
        uint32_t bits = __builtin_amdgcn_readlane(again, from);
#pragma unroll 1
        for (; bits; bits &= bits - 1) {
            int m, n;
            at(from, __builtin_ctz(bits), m, n);
            uint32_t row[1];
            mx_x_rows<1>(p, by_token, m0, m + 1, row, [&](int) { return m; });
            const int64_t x_row = by_token ? row[0] : m0 + m, w_row = first_row + n;
            const float y = mx_f32_again((const float*)p.x + x_row * p.ldx, p.packed + w_row * (p.K / 8),
                                         p.scales + w_row * (p.K / 32), p.K);
            if (l == from) store(m, n, y);
        }
    }
}

// Weight tile and block of x's rows of this workgroup: neighbours, which share a
// weight tile, on one XCD (consecutive workgroups go to the 8 XCDs in turn), and
// as many on each (whole weight tiles per XCD left some with half of the work
// again: 273 x 4096, 200 tokens, 18 tiles, 8.6 us).
__device__ __forceinline__ bool mx_tile(int n_tiles, int blocks, int& tile, int& tb) {
    const uint32_t total = (uint32_t)n_tiles * (uint32_t)blocks, per = (total + 7) / 8, j = blockIdx.x >> 3;
    const uint32_t id = (blockIdx.x & 7) * per + j;
    if (j >= per || id >= total) return false;
    tile = (int)(id / (uint32_t)blocks);
    tb = (int)(id - (uint32_t)tile * (uint32_t)blocks);
    return true;
}

template <int XT, int RT, int TT, int XI, int NW>
struct FewShape {
    using X = XEntry<XT>;
    static constexpr int XS = XT == MX_X_MXFP4 ? 1 : 0;  // DMA instructions of x's scales (W's: one)
    static constexpr int SOFF = 2048 * RT, XOFF = SOFF + 1024, XSOFF = XOFF + 1024 * XI, ENTRY = XSOFF + 1024 * XS;
    static constexpr int ROWS = XI * X::RPI;             // rows of x in an entry
    static constexpr int BM = ROWS < 16 * TT ? ROWS : 16 * TT;  // rows of x per workgroup
    static constexpr size_t LDS = std::max<size_t>((size_t)NW * ENTRY, (size_t)NW * RT * TT * 1024);
    static_assert(RT <= 4 && TT <= 4 && (ROWS >= 16 * TT || (TT == 1 && (ROWS & (ROWS - 1)) == 0)), "rows of an entry");
    static_assert(LDS <= 163840, "LDS");
};

template <int XT, int RT, int TT, int XI, int NW, bool ROUTED>
__global__ void __launch_bounds__(64 * NW) mxfp4_few_kernel(Mxfp4GemmParams p, int blocks) {
    using F = FewShape<XT, RT, TT, XI, NW>;
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
        if (!mx_tile(n_tiles, blocks, tile, tb)) return;
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
    // rows of x that this lane loads from, then (MXFP4) whose scales it loads and
    // that its fragments are of
    constexpr int NX = XI + (XT == MX_X_MXFP4 ? 1 + TT : 0);
    uint32_t xr[NX];
    mx_x_rows<NX>(p, by_token, m0, toks, xr, [&](int u) {
        return u < XI ? X::RPI * u + l / X::CHUNKS : (u == XI ? l : 16 * (u - XI - 1) + lr);
    });
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
    auto x_chunk = [&](int u) { return (uint32_t)X::chunk(l % X::CHUNKS, X::RPI * u + l / X::CHUNKS); };
#pragma unroll
    for (int u = 0; u < XI; ++u) xo[u] = xr[u] * (uint32_t)xrow + 16u * x_chunk(u);
    i32x4 xsres{};
    if constexpr (XT == MX_X_MXFP4) {
        const uint64_t xa = (uint64_t)(uintptr_t)p.x_scales + x_from * srow;
        const uint32_t xs0 = (uint32_t)xa & 3u;
        xsres = uniform_rsrc((const void*)(uintptr_t)(xa & ~3ull), (xs0 + (uint32_t)x_rows * srow + 3u) & ~3u);
        xso = (xs0 + xr[XI] * srow) & ~3u;
#pragma unroll
        for (int t = 0; t < TT; ++t) xsh[t] = ((xs0 + xr[XI + 1 + t] * srow) & 3u) + 2u * q;
    }

    char* const e = lds + w * F::ENTRY;
    auto issue = [&](int i) {
        const uint32_t ent = w + NW * i;
        const bool live = i < n;
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
    issue(0);
    // scale bytes of the lane's two blocks, those of 1 past the row's end
    auto scale_bytes = [&](const char* row, uint32_t at, bool in0, bool in1) -> uint32_t {
        const uint32_t* v = (const uint32_t*)row + (at >> 2);
        const uint32_t d = __builtin_amdgcn_alignbyte(v[1], v[0], at & 3u);
        return in1 ? d : (in0 ? (d & 0xffu) | 0x7f00u : 0x7f7fu);
    };
    for (int i = 0; i < n; ++i) {
        wait_vmcnt<0>();
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
                    fx[t][s] = *(const u32x4*)(e + F::XOFF + X::BYTES * row + 16 * X::slot(XF * (2 * q + u) + s, row));
            }
        };
        if constexpr (XT == MX_X_MXFP4) {
#pragma unroll
            for (int t = 0; t < TT; ++t) bx[t] = scale_bytes(e + F::XSOFF + 16 * (16 * t + lr), xsh[t], in0, in1);
        }
        // the entry's place is free once everything is in registers
        auto refill = [&] {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xc07f);  // the same, known to the compiler
            __builtin_amdgcn_sched_barrier(0);
            issue(i + 1);
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
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < TT; ++t) tot[r][t] += part[r][t];
    }
    wait_vmcnt<0>();
    auto store = [&](int m, int n, float y) {
        const int64_t o = (int64_t)(m0 + m) * p.ldy + n;
        if (p.y_f32)
            ((float*)p.y)[o] = y;
        else
            ((uint16_t*)p.y)[o] = f32_to_bf16_bits(y);
    };
    sk_reduce<RT, TT, NW>(lds, tot, [&](int r, int t, int lane, f32x4 v) {
        const int nn = 16 * r + (lane & 15);
        if constexpr (XT == MX_X_F32) {
            uint32_t again = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = 16 * t + 4 * (lane >> 4) + e;
                if (nn >= rows || m >= toks) continue;
                store(m, n0 + nn, v[e]);
                if (v[e] != v[e]) again |= 1u << e;
            }
            mx_f32_nans(p, by_token, first_row, m0, (const uint32_t*)(uintptr_t)(wsa & ~3ull),
                        (int)((ws0 + (uint32_t)rows * srow + 3u) >> 2), again,
                        [&](int from, int e, int& m, int& n) {
                            m = 16 * t + 4 * (from >> 4) + e;
                            n = n0 + 16 * r + (from & 15);
                        },
                        store);
        } else {
            if (nn >= rows) return;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = 16 * t + 4 * (lane >> 4) + e;
                if (m >= toks) break;
                store(m, n0 + nn, v[e]);
            }
        }
    });
}

// The same products for more rows of x, where reading x once per 16 or 32 weight
// rows would cost more than the weights: the NW waves of a workgroup own 16 RT
// weight rows each and share the 16 TT rows of x.  K streams through a ring of S
// stages of 256 k (x once, W and its scales per wave), one barrier per stage: it
// says that every wave's part of the stage has landed and that the slot of the
// last one is free, into which stage s + S - 1 then goes.  Up to S - 1 stages are
// in flight.  S = 1: a second barrier, after the reads of a stage, frees it for the
// next, and the workgroups of a CU cover each other's waits.  No sum crosses a wave.
template <int XT, int RT, int TT, int S, int NW>
struct MidShape {
    using X = XEntry<XT>;
    static constexpr int XI = 16 * TT / X::RPI;           // DMA instructions of x
    static constexpr int XPW = XI / NW;                   // of a wave
    static constexpr int XS = XT == MX_X_MXFP4 ? 1 : 0;   // of x's scales: a copy per wave
    static constexpr int NI = XPW + 2 * RT + 1 + XS;
    static constexpr int WAVE = 2048 * RT + 1024 + 1024 * XS;  // bytes of a wave's part
    static constexpr int STAGE = 1024 * XI + NW * WAVE;
    static constexpr size_t LDS = (size_t)S * STAGE;
    static_assert(XI % NW == 0 && (S - 1) * NI < 64 && LDS <= 163840 && RT <= 4 && TT <= 4, "stages");
};

template <int XT, int RT, int TT, int S, int NW, bool ROUTED>
__global__ void __launch_bounds__(64 * NW) mxfp4_mid_kernel(Mxfp4GemmParams p, int blocks) {
    using F = MidShape<XT, RT, TT, S, NW>;
    using X = XEntry<XT>;
    constexpr int BM = 16 * TT, BN = 16 * RT * NW;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int l = threadIdx.x & 63, q = l >> 4, lr = l & 15;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n_tiles = (p.N + BN - 1) / BN;
    int tile, m0, toks;
    int64_t first_row = 0;  // weight row 0 of the expert
    if constexpr (ROUTED) {
        MxTile t;
        if (!mx_find_tile<BM>(p.offsets, p.experts, p.pairs, n_tiles, t)) return;
        tile = t.n_tile;
        m0 = t.row;
        toks = t.rows;
        first_row = (int64_t)t.expert * p.N;
    } else {
        int tb;
        if (!mx_tile(n_tiles, blocks, tile, tb)) return;
        m0 = tb * BM;
        toks = min(BM, p.M - m0);
    }
    // this wave's rows; none for a wave past N, which still loads its part of x
    const int n0 = tile * BN + 16 * RT * w, rows = min(16 * RT, p.N - n0);
    const uint32_t K = (uint32_t)p.K, wrow = K / 2, srow = K / 32;
    const int64_t xrow = XT == MX_X_MXFP4 ? wrow : p.ldx * (XT == MX_X_F32 ? 4 : 2);
    const int64_t w_first = first_row + min(n0, p.N - 1);
    const uint32_t wrows = (uint32_t)max(rows, 0);
    const i32x4 wres = uniform_rsrc((const char*)p.packed + w_first * wrow, wrows * wrow);
    const uint64_t wsa = (uint64_t)(uintptr_t)p.scales + w_first * srow;
    const uint32_t ws0 = (uint32_t)wsa & 3u;
    const i32x4 sres = uniform_rsrc((const void*)(uintptr_t)(wsa & ~3ull), wrows ? (ws0 + wrows * srow + 3u) & ~3u : 0u);
    const bool by_token = ROUTED && p.pair_of_row != nullptr;
    const int64_t x_from = by_token ? 0 : m0, x_rows = by_token ? p.M : toks;
    const i32x4 xres = uniform_rsrc((const char*)p.x + x_from * xrow,
                                    (uint32_t)((x_rows - 1) * xrow + X::BYTES * (int64_t)K / 256));
    const int nst = (int)((K + 255) / 256);

    constexpr uint32_t PAST = 0xfffffff0u;  // an offset that reads zeros
    const uint32_t ch8 = (l & 7) ^ (l >> 4);
    uint32_t wo[2 * RT], xo[F::XPW], xso = 0, xsh[TT];
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) {
        const int r = 8 * i + (l >> 3);
        wo[i] = r < rows ? (uint32_t)r * wrow + 16u * (ch8 ^ (4 * (i & 1))) : SK_OOB_ROW;
    }
    const uint32_t so = l < rows ? (ws0 + (uint32_t)l * srow) & ~3u : SK_OOB_ROW;
    // x: this wave's instruction u of XPW
    auto x_instr = [&](int u) { return F::XPW * w + u; };
    auto x_row = [&](int u) { return X::RPI * x_instr(u) + l / X::CHUNKS; };
    auto x_chunk = [&](int u) { return (uint32_t)X::chunk(l % X::CHUNKS, x_row(u)); };
    constexpr int NX = F::XPW + (XT == MX_X_MXFP4 ? 1 + TT : 0);
    uint32_t xr[NX];
    mx_x_rows<NX>(p, by_token, m0, toks, xr,
                  [&](int u) { return u < F::XPW ? x_row(u) : (u == F::XPW ? l : 16 * (u - F::XPW - 1) + lr); });
#pragma unroll
    for (int u = 0; u < F::XPW; ++u) xo[u] = xr[u] * (uint32_t)xrow + 16u * x_chunk(u);
    i32x4 xsres{};
    if constexpr (XT == MX_X_MXFP4) {
        const uint64_t xa = (uint64_t)(uintptr_t)p.x_scales + x_from * srow;
        const uint32_t xs0 = (uint32_t)xa & 3u;
        xsres = uniform_rsrc((const void*)(uintptr_t)(xa & ~3ull), (xs0 + (uint32_t)x_rows * srow + 3u) & ~3u);
        xso = (xs0 + xr[F::XPW] * srow) & ~3u;
#pragma unroll
        for (int t = 0; t < TT; ++t) xsh[t] = ((xs0 + xr[F::XPW + 1 + t] * srow) & 3u) + 2u * q;
    }
    const int woff = 1024 * F::XI + w * F::WAVE;  // of the wave's part in a stage
    auto issue = [&](int s, int slot) {
        const uint32_t st = s;
        const bool live = s < nst;
        char* e = lds + slot * F::STAGE;
#pragma unroll
        for (int u = 0; u < F::XPW; ++u) {
            const bool in = live && 256u * st + X::KPC * x_chunk(u) < K && x_row(u) < toks;
            dma16_buf(xres, in ? xo[u] + (uint32_t)X::BYTES * st : PAST, e + 1024 * x_instr(u));
        }
        e += woff;
#pragma unroll
        for (int c = 0; c < 2 * RT; ++c) {
            const bool in = live && 256u * st + 32u * (ch8 ^ (4 * (c & 1))) < K;
            dma16_buf(wres, wo[c] + (in ? 128u * st : SK_OOB_K), e + 1024 * c);
        }
        dma16_buf(sres, so + (live ? 8u * st : SK_OOB_K), e + 2048 * RT);
        if constexpr (XT == MX_X_MXFP4) dma16_buf(xsres, live && l < toks ? xso + 8u * st : PAST, e + 2048 * RT + 1024);
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
    for (int s = 0; s < (S == 1 ? 1 : S - 1); ++s) issue(s, s);
    auto scale_bytes = [&](const char* row, uint32_t at, bool in0, bool in1) -> uint32_t {
        const uint32_t* v = (const uint32_t*)row + (at >> 2);
        const uint32_t d = __builtin_amdgcn_alignbyte(v[1], v[0], at & 3u);
        return in1 ? d : (in0 ? (d & 0xffu) | 0x7f00u : 0x7f7fu);
    };
    int slot = 0;
#pragma unroll 1
    for (int s = 0; s < nst; ++s) {
        wait_vmcnt<(S == 1 ? 0 : S - 2) * F::NI>();
        lds_barrier();
        if constexpr (S > 1) issue(s + S - 1, slot ? slot - 1 : S - 1);
        const char* e = lds + slot * F::STAGE;
        const char* ew = e + woff;
        const uint32_t k0 = 256u * s + 64u * q;
        const bool in0 = k0 < K, in1 = k0 + 32 < K;
        u32x4 fw[RT][2];
        uint32_t bw[RT], bx[TT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int u = 0; u < 2; ++u) fw[r][u] = *(const u32x4*)(ew + 2048 * r + 128 * lr + 16 * ((2 * q + u) ^ (lr >> 1)));
            bw[r] = scale_bytes(ew + 2048 * RT + 16 * (16 * r + lr), wsh[r], in0, in1);
        }
        if constexpr (XT == MX_X_MXFP4) {
#pragma unroll
            for (int t = 0; t < TT; ++t) bx[t] = scale_bytes(ew + 2048 * RT + 1024 + 16 * (16 * t + lr), xsh[t], in0, in1);
        }
        constexpr int XF = XT == MX_X_MXFP4 ? 1 : (XT == MX_X_F32 ? 8 : 4);  // 16-byte pieces per block
        f32x4 part[RT][TT];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < TT; ++t) part[r][t] = f32x4{};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            u32x4 fx[TT][XF];
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int c = 0; c < XF; ++c)
                    fx[t][c] = *(const u32x4*)(e + X::BYTES * (16 * t + lr) + 16 * X::slot(XF * (2 * q + u) + c, 16 * t + lr));
            if (S == 1 && u == 1) {
                lds_barrier();  // every wave has read the stage
                if (s + 1 < nst) issue(s + 1, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            // W is the first operand: a lane then holds four outputs of one row of y
            if constexpr (XT == MX_X_MXFP4) {
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int t = 0; t < TT; ++t)
                        part[r][t] = u ? mfma16_mxfp4<1>(fw[r][1], bw[r], fx[t][0], bx[t], part[r][t])
                                       : mfma16_mxfp4<0>(fw[r][0], bw[r], fx[t][0], bx[t], part[r][t]);
            } else {
                float sc[RT];
#pragma unroll
                for (int r = 0; r < RT; ++r) sc[r] = __uint_as_float(((bw[r] >> (8 * u)) & 255u) << 23);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    bf16x8 wf[RT];
#pragma unroll
                    for (int r = 0; r < RT; ++r) wf[r] = mxfp4_bf16(fw[r][u][c], sc[r]);
#pragma unroll
                    for (int t = 0; t < TT; ++t) {
                        if constexpr (XT == MX_X_F32) {
                            bf16x8 xf[3];
                            split3(fx[t][2 * c], fx[t][2 * c + 1], xf);
#pragma unroll
                            for (int r = 0; r < RT; ++r)  // small parts first
                                part[r][t] = mfma16(wf[r], xf[0], mfma16(wf[r], xf[1], mfma16(wf[r], xf[2], part[r][t])));
                        } else {
#pragma unroll
                            for (int r = 0; r < RT; ++r) part[r][t] = mfma16(wf[r], __builtin_bit_cast(bf16x8, fx[t][c]), part[r][t]);
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
    wait_vmcnt<0>();  // (loads of zeros past the last stage)
    // tot[r][t][e]: y row m0 + 16 t + l % 16, column n0 + 16 r + 4 (l / 16) + e
    const int size = p.y_f32 ? 4 : 2;
    const bool vec = ((uintptr_t)p.y & (4 * size - 1)) == 0 && (p.ldy & 3) == 0;
    uint32_t again = 0;  // x in f32: which are NaN
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        const int m = 16 * t + lr;
        if (m >= toks) continue;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int c = 16 * r + 4 * q;
            const int64_t o = (int64_t)(m0 + m) * p.ldy + n0 + c;
            const f32x4 v = tot[r][t];
            if constexpr (XT == MX_X_F32) {
                static_assert(4 * RT * TT <= 32, "a bit per output");
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < rows && v[e] != v[e]) again |= 1u << (4 * (RT * t + r) + e);
            }
            if (vec && c + 4 <= rows) {
                if (p.y_f32)
                    *(f32x4*)((float*)p.y + o) = v;
                else
                    *(u32x2*)((uint16_t*)p.y + o) = u32x2{pack_bf16x2_hw(v[0], v[1]), pack_bf16x2_hw(v[2], v[3])};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < rows) {
                        if (p.y_f32)
                            ((float*)p.y)[o + e] = v[e];
                        else
                            ((uint16_t*)p.y)[o + e] = f32_to_bf16_bits(v[e]);
                    }
            }
        }
    }
    if constexpr (XT == MX_X_F32)
        mx_f32_nans(p, by_token, first_row, m0, (const uint32_t*)(uintptr_t)(wsa & ~3ull),
                    (int)((ws0 + wrows * srow + 3u) >> 2), again,
                    [&](int from, int i, int& m, int& n) {
                        m = 16 * (i / (4 * RT)) + (from & 15);
                        n = n0 + 16 * (i / 4 % RT) + 4 * (from >> 4) + i % 4;
                    },
                    [&](int m, int n, float y) {
                        const int64_t o = (int64_t)(m0 + m) * p.ldy + n;
                        if (p.y_f32)
                            ((float*)p.y)[o] = y;
                        else
                            ((uint16_t*)p.y)[o] = f32_to_bf16_bits(y);
                    });
}

// The kernels as a call chooses among them: launch, or say which it is
template <int XT, int RT, int TT, int XI, int NW, bool ROUTED = false>
struct Few {
    using F = FewShape<XT, RT, TT, XI, NW>;
    static constexpr Mxfp4Route ROUTE = {MX_FEW, 16 * RT, F::BM, NW, 1};
    static constexpr int BN = 16 * RT, BM = F::BM, THREADS = 64 * NW;
    static constexpr size_t LDS = F::LDS;
    static constexpr auto KERNEL = mxfp4_few_kernel<XT, RT, TT, XI, NW, ROUTED>;
    static constexpr bool BY_EXPERT = ROUTED;
};
template <int XT, int RT, int TT, int S, int NW, bool ROUTED = false>
struct Mid {
    using F = MidShape<XT, RT, TT, S, NW>;
    static constexpr Mxfp4Route ROUTE = {MX_MID, 16 * RT * NW, 16 * TT, NW, S};
    static constexpr int BN = 16 * RT * NW, BM = 16 * TT, THREADS = 64 * NW;
    static constexpr size_t LDS = F::LDS;
    static constexpr auto KERNEL = mxfp4_mid_kernel<XT, RT, TT, S, NW, ROUTED>;
    static constexpr bool BY_EXPERT = ROUTED;
};

template <typename C>
hipError_t launch(const Mxfp4GemmParams& p, hipStream_t st) {
    if (C::LDS > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)C::KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, (int)C::LDS);
        if (e != hipSuccess) return e;
    }
    const int64_t tiles = (p.N + C::BN - 1) / C::BN, blocks = ((int64_t)p.M + C::BM - 1) / C::BM;
    const int64_t grid = C::BY_EXPERT ? (mx_tile_bound(p, C::BM) * tiles + 7) / 8 * 8 : (tiles * blocks + 7) / 8 * 8;
    if (grid * C::THREADS >= (1ll << 32)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(C::KERNEL, dim3((unsigned)grid), dim3(C::THREADS), C::LDS, st, p, (int)blocks);
    return hipGetLastError();
}

// Which kernel and tile.  Both split a call into workgroups of some weight rows
// x some rows of x; small ones fill the GPU, large ones read less, and rows that
// are short leave waves that split them idle.  In us, one call among others with
// the weights in the caches, unless it says otherwise (from HBM 5 to 25% more, and
// more for kernels that read the weights more than once):
//   matrix, x in bf16, one round of workgroups of the smallest tile that gives no
//     more than one a CU, with 8 waves: 576 x 7168, 96 tokens, 16 x 16 7.4, 32 x
//     16 8.4; 1536 x 7168, 64 tokens, 32 x 16 8.5, 16 x 16 12.3; 2048 x 12608, 100
//     tokens, 64 x 16 16.5, 32 x 16 with 4 waves 20.4; with 4 waves where a row is
//     short: 273 x 1024, 300 tokens, 4.8 and 6.9.  Then one round of 64 x 48 (4096 x
//     4096, 150 tokens, 14.6, mid 18) or, for long rows, of 64 x 64 with 3 waves
//     (1536 x 12608, 600 tokens, 51 and 67), else mid, 128 x 32: 24576 x 1536, 37
//     tokens, 10.5, 64 x 16 17 (64 x 48, which fits 33 to 48 tokens: 10.3, but with
//     the weights from HBM 12.7 and 128 x 32 12.3; 65536 x 2048, 48 tokens, 34.9
//     and 30.1; 20000 x 1536, 34 tokens, 12.5 and 11.8)
//   x in MXFP4, which costs a quarter to read: 7168 x 4096, 16 tokens, 32 x 16 with
//     8 waves 4.8, 16 x 16 5.8, 64 x 16 5.7; 1024 x 4096, 200 tokens, 64 x 16 with 8
//     waves 5.9, 64 x 32 6.5, x 1024 32 x 16 with 4 4.1, 64 x 32 4.9; 1024 x 2048,
//     600 tokens, 64 x 32 with 4 waves 6.6, mid 7.9 (24576 x 1536, 16 tokens, 6.5
//     and mid 5.5); 7168 x 16384, 64 tokens, 64 x
//     32 with 8 waves 18.7, 64 x 64 24.4; 2048 x 12608, 600 tokens, 64 x 64 with 4
//     waves 33, with 8 42; 12000 x 1024, 100 tokens, mid 128 x 32 6.0, 128 x 64 6.9
//   experts by their mean rows, x in bf16: 128 of 2048 x 768, 6 rows, mid 128 x 16
//     20.2, 128 x 32 22.4, 12 rows 21.2 and 22.9, 19 rows 25.5 and 24.0; one stage
//     in the ring, which leaves room for four or five workgroups a CU, where there
//     are more than two a CU: these, with two stages 24.1, 28.1 (12 rows, 128 x
//     32) and 29.3; 32 of 1536 x 7168, 6 rows, 384 workgroups, 34.0 and 31.0
//   MXFP4, with two waves: 128 of 2048 x 768, 9 rows, 64 x 16 18.9, 128 x 16 19.3
//     (two stages 23.9), 16 rows, 64 x 32 20.9, 64 x 16 21.1; 32 of 1536 x 7168, 12
//     rows, 29.3 and 34.4; 24576 x 1536, 16 tokens, 64 x 16 5.5, 64 x 32 6.4
// and few pairs, two rows of x staged per 16 weight rows, 8 of 128 experts 4.8,
// mid 8.3; 64 pairs 10.9 and 11.5, 96 13.4 and 12.1; 2048 x 768, 4 pairs 4.3 and
// 5.2, 16 pairs 6.6 and 5.4; 32 of 1536 x 7168, 24 pairs 20.8 and 23.5, 64 pairs 35
// and 30; 192 x 1024, 64 pairs 5.0 and 6.0, 192 pairs 7.6 and 6.2.
bool few_pairs(const Mxfp4GemmParams& p) {
    return p.pairs <= 2 * p.experts && (int64_t)p.pairs * ((p.N + 15) / 16) * 4 <= 3 * (int64_t)p.K;
}

// about how many tiles of 128 weight rows x `bm` rows of x a routed call has
int64_t routed_tiles(const Mxfp4GemmParams& p, int bm) {
    return ((int64_t)p.N + 127) / 128 * (p.pairs * 4ll <= p.experts * 3ll * bm ? std::min(p.experts, p.pairs) : p.pairs / bm + p.experts / 2);
}

template <typename Go>
auto choose_bf16(const Mxfp4GemmParams& p, int cus, Go go) {
    const int entries = (p.K + 255) / 256;
    if (p.offsets) {
        if (few_pairs(p)) return go(Few<0, 1, 1, 1, 4, true>{});
        if (p.pairs <= 12 * p.experts) return routed_tiles(p, 16) > 2 * cus ? go(Mid<0, 2, 1, 1, 4, true>{}) : go(Mid<0, 2, 1, 2, 4, true>{});
        return routed_tiles(p, 32) > 2 * cus ? go(Mid<0, 2, 2, 1, 4, true>{}) : go(Mid<0, 2, 2, 2, 4, true>{});
    }
    if (p.M <= 2) {
        if (entries >= 16) return go(Few<0, 1, 1, 1, 8>{});
        return entries >= 8 ? go(Few<0, 1, 1, 1, 4>{}) : go(Few<0, 1, 1, 1, 2>{});
    }
    const int64_t b = ((int64_t)p.M + 15) / 16, n16 = (p.N + 15) / 16, n32 = (p.N + 31) / 32, n64 = (p.N + 63) / 64;
    if (n16 * b <= cus) return entries > 4 ? go(Few<0, 1, 1, 8, 8>{}) : go(Few<0, 1, 1, 8, 4>{});
    if (n32 * b <= cus && entries > 4) return go(Few<0, 2, 1, 8, 8>{});
    if (n64 * b <= cus && entries >= 8) return go(Few<0, 4, 1, 8, 8>{});
    if (n32 * b <= 2 * cus) return go(Few<0, 2, 1, 8, 4>{});
    if (n64 * b <= 2 * cus) return go(Few<0, 4, 1, 8, 4>{});
    if (n64 * (((int64_t)p.M + 47) / 48) <= cus) return go(Few<0, 4, 3, 24, 4>{});
    if (n64 * (((int64_t)p.M + 63) / 64) <= cus && p.K > 4096) return go(Few<0, 4, 4, 32, 3>{});
    if (b == 1) return go(Mid<0, 2, 1, 2, 4>{});
    return go(Mid<0, 2, 2, 2, 4>{});
}

template <typename Go>
auto choose_mxfp4(const Mxfp4GemmParams& p, int cus, Go go) {
    if (p.offsets) {
        if (few_pairs(p)) return go(Few<2, 1, 1, 2, 4, true>{});
        return p.pairs <= 10 * p.experts ? go(Mid<2, 2, 1, 1, 2, true>{}) : go(Mid<2, 2, 2, 1, 2, true>{});
    }
    const int64_t b = ((int64_t)p.M + 15) / 16, n16 = (p.N + 15) / 16, n32 = (p.N + 31) / 32, n64 = (p.N + 63) / 64;
    if (n16 * b <= cus) return go(Few<2, 1, 1, 2, 8>{});
    if (n32 * b <= cus) return go(Few<2, 2, 1, 2, 8>{});
    if (n64 * b <= cus && p.K > 2048) return go(Few<2, 4, 1, 2, 8>{});
    if (n32 * b <= 2 * cus && p.K <= 2048) return go(Few<2, 2, 1, 2, 4>{});
    if (n64 * ((b + 1) / 2) <= cus) return go(Few<2, 4, 2, 4, 8>{});
    if (b > 4 && n64 * ((b + 1) / 2) <= 2 * cus && p.K <= 2048) return go(Few<2, 4, 2, 4, 4>{});
    if (n64 * ((b + 3) / 4) <= cus && p.K > 2048) return go(Few<2, 4, 4, 8, 8>{});
    if (n64 * ((b + 3) / 4) <= 2 * cus && p.K > 2048) return go(Few<2, 4, 4, 8, 4>{});
    return b <= 4 ? go(Mid<2, 2, 1, 1, 2>{}) : go(Mid<2, 2, 2, 1, 4>{});
}

// f32: the cuts of x cost more than its bytes, so a cut serves 32 or 64 weight
// rows where there are workgroups enough (mid 64 and 32 rows a wave: 24576 x 1536,
// 37 tokens, 576 tiles of 128, 29 and 32 us, 5 tokens 19 and 16.6; 128 experts of
// 768 x 2048, 12 rows, 40 and 53; 64 of 512 x 512, one row, 9.0 and 8.1); few of
// them split K instead: 1536 x 7168, 64 tokens, 32 x 16 with 4 waves 23, mid 62,
// 2048 x 2048 9 and 20
template <typename Go>
auto choose_f32(const Mxfp4GemmParams& p, int cus, Go go) {
    if (p.offsets) {
        const int64_t tiles = routed_tiles(p, 16);
        if (2 * tiles <= cus) return go(Mid<1, 1, 1, 1, 4, true>{});
        return tiles <= cus ? go(Mid<1, 2, 1, 1, 4, true>{}) : go(Mid<1, 4, 1, 1, 4, true>{});
    }
    if (p.M == 1) return go(Few<1, 4, 1, 1, 4>{});
    const int64_t b = ((int64_t)p.M + 15) / 16;
    if ((p.N + 31) / 32 * b <= 2 * cus) return go(Few<1, 2, 1, 16, 4>{});
    return (p.N + 127) / 128 * b <= cus ? go(Mid<1, 2, 1, 1, 4>{}) : go(Mid<1, 4, 1, 1, 4>{});
}

template <typename Go>
auto choose(const Mxfp4GemmParams& p, int cus, Go go) {
    if (p.x_kind == MX_X_MXFP4) return choose_mxfp4(p, cus, go);
    return p.x_kind == MX_X_F32 ? choose_f32(p, cus, go) : choose_bf16(p, cus, go);
}

hipError_t launch_mxfp4_few(const Mxfp4GemmParams& p, int cus, hipStream_t st) {
    return choose(p, cus, [&](auto c) { return launch<decltype(c)>(p, st); });
}

// Large tiles (mxfp4_gemm.hip), or none.  Those of 128 x 128 pay once they cover
// the larger part of the GPU and the kernels of few rows would read W more than
// once.  In us, one call among others, weights from HBM (from the caches 5 to 30%
// less, with the same sides ahead except where noted), 128 and few rows:
//   bf16: 24576 x 1536, 65 tokens, 192 tiles, 16.2 and 18.4, 64 tokens 16.1 and
//     12.6; 7168 x 16384, 300 tokens, 168 tiles, 122 and 135, 200 tokens, 112 tiles,
//     123 and 86; 16384 x 4096, 65 tokens, 128 tiles, 35 and 25
//   MXFP4: 24576 x 1536, 64 tokens, 10.2 and 12.2, 37 tokens 9.9 and 10.5; 16384 x
//     4096, 65 tokens, 19.8 and 17.5; 4096 x 12608, 400 tokens, 128 tiles, 68 and 42
// and for experts from some rows each: bf16, 128 of 768 x 2048, 62 rows, 52 and 49,
// 50 rows 52 and 44, 31 rows 50 and 38; 32 of 1536 x 7168, 88 rows, 99 and 110, 62
// rows 96 and 89; MXFP4, 128 of 768 x 2048, 31 rows, 25.0 and 35.2, 19 rows 24.7 and
// 26.1 (from the caches 20.4 and 19.4).  The border of 60 rows in bf16 is early by
// about 10.
// Between the tiles, by rounds of workgroups, in units of a sixth of the time of a
// round of two a CU (bf16: a last round of at most one a CU takes 4): three a CU 8,
// 256 x 256 12 (MXFP4) or 10.5 (bf16).
//   MXFP4, three, two, 256: 24576 x 1536, 300 tokens, 16.1, 21.0 and 19.9, 4096
//     tokens 121, 146 and 121; 16384 x 4096, 1000 tokens, 55, 52 and 41; 4096 tokens
//     to 8 of 128 experts of 768 x 2048 54 and 62; 1024 to 8 of 32 of 1536 x 7168 98
//     and 89; 7168 x 16384, 400 tokens, 72 and 64
//   bf16, two and 256: 24576 x 1536, 600 tokens, 48 and 74, 4096 tokens 268 and 254;
//     16384 x 4096, 1000 tokens, 120 and 102
MxTiles tiles_of(const Mxfp4GemmParams& p, int cus) {
    if (p.x_kind == MX_X_F32) return MX_TILES_NONE;
    const bool mx = p.x_kind == MX_X_MXFP4;
    auto cols = [&](int size) { return ((int64_t)p.N + size - 1) / size; };
    int64_t small;  // tiles of 128
    if (p.offsets) {
        if (p.pairs < (mx ? 24 : 60) * (int64_t)p.experts) return MX_TILES_NONE;
        small = routed_tiles(p, 128);
    } else {
        if (p.M <= (mx ? 32 : 64)) return MX_TILES_NONE;
        small = cols(128) * (((int64_t)p.M + 127) / 128);
    }
    if (small * 8 < (!mx || p.K > 4096 ? 5 : !p.offsets && p.M <= 64 ? 6 : 4) * cus) return MX_TILES_NONE;
    const int64_t left = small % (2 * cus);
    const int64_t two = small / (2 * cus) * 6 + (left == 0 ? 0 : left <= cus && !mx ? 4 : 6);
    const int64_t three = mx ? (small + 3 * cus - 1) / (3 * cus) * 8 : INT64_MAX;
    if (!p.offsets) {
        const int64_t rounds = (cols(256) * (((int64_t)p.M + 255) / 256) + cus - 1) / cus;
        if (mx ? 12 * rounds <= std::min(two, three) : 21 * rounds <= 2 * two) return MX_TILES_256;
    }
    return three <= two ? MX_TILES_128x3 : MX_TILES_128x2;
}

}  // namespace

// as many workgroups as a routed call can need (of 256 threads, 16 rows of x and
// 128 weight rows; of few pairs no more than 2^20) in a grid of less than 2^32
// threads
bool mxfp4_gemm_fits(const Mxfp4GemmParams& p) {
    return !p.offsets || (mx_tile_bound(p, 16) * ((p.N + 127) / 128) + 7) * 256 < (1ll << 32);
}

Mxfp4Route mxfp4_route(const Mxfp4GemmParams& p, int cu_count) {
    const MxTiles tile = tiles_of(p, cu_count);
    if (tile == MX_TILES_NONE) return choose(p, cu_count, [](auto c) { return decltype(c)::ROUTE; });
    const int size = tile == MX_TILES_256 ? 256 : 128;
    return {MX_TILES, size, size, 4, tile == MX_TILES_128x3 ? 1 : 2};
}

// A matrix's tokens in as many launches as grids of less than 2^32 threads take:
// one, up to 2^23 workgroups of 16 tokens x 16 weight rows (MXFP4_MAX_OUT weight
// rows leave 256 tokens each).
hipError_t launch_mxfp4_gemm(const Mxfp4GemmParams& p, int cu_count, hipStream_t st) {
    const MxTiles tile = tiles_of(p, cu_count);
    if (p.offsets) return tile ? launch_mxfp4_tiles(p, tile, st) : launch_mxfp4_few(p, cu_count, st);
    const int64_t most = ((int64_t)1 << 23) / ((p.N + 15) / 16 + 8) * 16 / 256 * 256;
    for (int64_t m = 0; m < p.M; m += most) {
        Mxfp4GemmParams q = p;
        q.M = (int)std::min<int64_t>(most, p.M - m);
        const int64_t row = p.x_kind == MX_X_MXFP4 ? p.K / 2 : p.ldx * (p.x_kind == MX_X_F32 ? 4 : 2);
        q.x = (const char*)p.x + m * row;
        if (p.x_scales) q.x_scales = p.x_scales + m * (p.K / 32);
        q.y = (char*)p.y + m * p.ldy * (p.y_f32 ? 4 : 2);
        const hipError_t e = tile ? launch_mxfp4_tiles(q, tile, st) : launch_mxfp4_few(q, cu_count, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace mr
