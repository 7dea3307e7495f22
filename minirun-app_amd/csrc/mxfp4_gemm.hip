// Products with MXFP4 weights for many rows: y[t][o] = sum_i x[t][i] w[o][i]
// in tiles of TM x TN rows of x and W, 256 x 256 or 128 x 128, for the tokens of
// one matrix or for rows in expert order (tiles of 128, each of one expert's rows).
// x is bf16, or MXFP4 itself; y bf16 or f32.
//
// What bounds it: the matrix pipe, and the way of the operands to it.  One
// workgroup of 4 waves computes a tile, each wave a quarter of it in 32x32 MFMA
// tiles; each operand fragment serves MI or JN of them.  With 256 x 256 (the
// accumulators are half of the registers, one workgroup a CU) a prompt of 4096
// tokens runs at 1.2 PFLOP/s in bf16 (24576 x 1536, 254 us) and 4.1 PFLOP/s in
// MXFP4 (7168 x 16384, 232 us; 217 with the operands in the caches; 230 to 255 from
// card to card).  128 x 128 reads twice as much per operation, but two or three
// workgroups a CU cover each other's waits, ends of tiles and starts: 4096 tokens to
// 8 of 128 experts of 768 x 2048, MXFP4, three 54 us, two 62 (weights from HBM; from
// the caches 47 and 54; 31 us is the time of the bytes; eight stages a tile leave
// latency in view: of the 30000 clocks of a tile with two workgroups 19000 were its
// stages', whose matrix instructions take 5800, 7500 its start and 3500 its end).
// Operands come by global -> LDS DMA, issued between the MFMAs.  A load costs by
// the lines it touches, about two clocks each, whether it takes 4 or 128 bytes of
// a line, so rows come in whole lines of 128 bytes and scales 16 bytes of a row
// at a time (64-byte pieces and four scale bytes per load kept the matrix pipe
// waiting: 4096 x 7168 x 16384 in MXFP4 took 312 us, its loads alone 264).
//
//   x in MXFP4: v_mfma_scale_f32_32x32x64_f8f6f4 on the codes and scale bytes
//     as stored.  A stage is 256 k: a line of each row of x and W, in a ring of
//     two.  In step s of four, lane half h has block 4 h + s, so that its four
//     scale bytes of a stage are one word and the step picks its byte (op_sel).
//     The barrier that ends stage t, before its last step, frees its buffer:
//     half of stage t + 2 is issued in that step, half in the next one, and two
//     steps are left for it to land.  Scales come for two stages together.
//     ONE: a ring of one.  The barrier after the reads of a stage's last step
//     frees it, the next stage is issued at once, and what the MFMAs that follow
//     leave of its way is the other workgroups' time.  It takes less LDS and fewer
//     registers, which makes room for a third workgroup; where there are not that
//     many, or for bf16 (a third one gained nothing there: 112 and 111 us), the
//     ring of two is faster (7168 x 16384, 400 tokens, 64 and 72 us).
//   x in bf16: a stage is 64 k: a line of each row of x, in a ring of three; W's
//     rows come 64 bytes (two stages) at a time, in a ring of two.  Lane half h
//     has block h of the stage's two: the block's four words, one per 16-deep
//     step, become bf16 with their scale (exact) beside the MFMAs; for x, step s
//     of half h takes the chunk 4 h + s.
// Each step's fragments are read a step ahead; one barrier per stage (ONE: two).
// Past the last stage the issues repeat it into stages that are not read, or load
// zeros, so that the waits are constants.  Chunk c of a 128-byte row r is in slot c ^
// ((r >> 1) & 7), of a 64-byte one in c ^ ((r >> 2) & 3): the 16 lanes of a read
// (16 neighbouring rows, one chunk) hit 16 bank groups.
//
// RAGGED: K is no multiple of a stage (256, or 128 for W's pieces), or the scales
// do not start on a word.  Scale rows then start on any byte and come with the
// word that follows; chunks past the end of the rows are loaded as zeros
// (through the buffer's bounds), and their scale bytes, which may be the next
// row's, are replaced by that of 1.
//
// Rows past the tile's last (of x) or N (of W) repeat the last row; their
// outputs are not stored.
#include <algorithm>

#include "few_tiles.hpp"
#include "mxfp4_tiles.hpp"

namespace mr {

namespace {

constexpr int MG_THREADS = 256;

__device__ __forceinline__ int slot128(int r, int c) { return 8 * r + (c ^ ((r >> 1) & 7)); }
__device__ __forceinline__ int slot64(int r, int c) { return 4 * r + (c ^ ((r >> 2) & 3)); }

template <int XT, int TM, int TN, bool ONE, bool RAGGED>
struct MgShape {
    static constexpr bool MX = XT == MX_X_MXFP4;
    static constexpr int A = TM * 128;                // bytes of x in a stage
    static constexpr int B = TN * (MX ? 128 : 64);    // of W in its pieces
    static constexpr int NA = MX ? (ONE ? 1 : 2) : 3, NB = ONE ? 1 : 2;  // stages of x in the ring, of W and the scales
    static_assert(MX || !ONE, "one stage: MXFP4");
    // scales: 16 bytes (MXFP4: x's rows first) or 4 per row, and RAGGED the word
    // after them; rows in whole instructions of the four waves
    static constexpr int SROWS = MX ? (TM + TN + 255) / 256 * 256 : TN, SROW = MX ? 16 : 4;
    static constexpr int S = SROWS * (SROW + (RAGGED ? 4 : 0));
    static constexpr int RING = NA * A + NB * B + NB * S;
    // DMA instructions per wave: x and W of a stage or piece, scales
    static constexpr int DA = A / 4096, DB = B / 4096, SQ = MX ? SROWS / 256 : 1, DS = SQ * (RAGGED ? 2 : 1);
    static constexpr size_t LDS_BF16 = std::max<size_t>(RING, (size_t)TM * TN * 2);
    static constexpr size_t LDS_F32 = std::max<size_t>(RING, (size_t)TM / 2 * TN * 4);
    static constexpr int PER_CU = TN == 256 ? 1 : (ONE ? 3 : 2);  // workgroups
    static_assert(PER_CU * LDS_BF16 <= 163840 && PER_CU * LDS_F32 <= 163840, "LDS");
};

template <int XT, int TM, int TN, bool ONE, bool ROUTED, bool YF32, bool RAGGED>
__global__ void __launch_bounds__(MG_THREADS, (MgShape<XT, TM, TN, ONE, RAGGED>::PER_CU)) mxfp4_gemm_kernel(Mxfp4GemmParams p) {
    using S = MgShape<XT, TM, TN, ONE, RAGGED>;
    constexpr bool MX = S::MX;
    constexpr int DA = S::DA, DB = S::DB, DS = S::DS, SQ = S::SQ;
    constexpr int WM = TM / 2, MI = WM / 32;  // rows and 32-row MFMA tiles per wave
    constexpr int WN = TN / 2, JN = WN / 32;  // columns and 32-column ones
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_tiles = (p.N + TN - 1) / TN;
    int m0, rows, nt;
    int64_t first = 0;  // weight row 0 of the expert
    if constexpr (ROUTED) {
        MxTile t;
        if (!mx_find_tile<TM>(p.offsets, p.experts, p.pairs, n_tiles, t)) return;
        nt = t.n_tile;
        m0 = t.row;
        rows = t.rows;
        first = (int64_t)t.expert * p.N;
    } else {
        // XCD-aware order: consecutive workgroups go to the 8 XCDs in turn, so
        // XCD x gets tile ids x * total / 8 ..; ids run over groups of 4 row
        // tiles, W tiles outer, so one XCD's resident workgroups share rows of
        // x and W in its L2
        const int m_tiles = (p.M + TM - 1) / TM, total = m_tiles * n_tiles;
        int bid = blockIdx.x;
        if ((total & 7) == 0) bid = (bid & 7) * (total >> 3) + (bid >> 3);
        constexpr int GM = 4;
        const int group = bid / (GM * n_tiles), first_m = group * GM;
        const int gsize = min(m_tiles - first_m, GM);
        m0 = (first_m + (bid % (GM * n_tiles)) % gsize) * TM;
        nt = (bid % (GM * n_tiles)) / gsize;
        rows = min(TM, p.M - m0);
    }
    const int n0 = nt * TN;
    const uint32_t wrow = (uint32_t)p.K / 2, srow = (uint32_t)p.K / 32;
    const uint32_t xrow = MX ? wrow : (uint32_t)p.ldx * 2u;
    const int wrows = min(TN, p.N - n0);

    // x: from the tile's first row, or (rows by token) from row 0 with the
    // token's offset; a byte offset past the buffer reads zeros
    const bool by_token = ROUTED && p.pair_of_row != nullptr;
    const int64_t x_from = by_token ? 0 : m0;
    const int64_t x_rows = by_token ? p.M : rows;
    const uint32_t x_bytes = (uint32_t)((x_rows - 1) * (MX ? wrow : p.ldx * 2) + (MX ? wrow : 2 * p.K));
    const i32x4 xres = uniform_rsrc((const char*)p.x + x_from * (MX ? wrow : p.ldx * 2), x_bytes);
    const i32x4 wres = uniform_rsrc((const char*)p.packed + (first + n0) * wrow, (uint32_t)wrows * wrow);
    // rows of x that this lane loads from, and (q >= DA) whose scales it loads, or
    // (RAGGED) that its fragments are of
    constexpr int NX = DA + (MX ? SQ + (RAGGED ? MI : 0) : 0);
    const int wm = w >> 1, wn = w & 1;
    uint32_t xr[NX];
    mx_x_rows<NX>(p, by_token, m0, rows, xr, [&](int u) {
        if (u < DA) return 8 * (DA * w + u) + (l >> 3);
        if (u < DA + SQ) return 64 * (SQ * w + u - DA) + l;
        return wm * WM + (u - DA - SQ) * 32 + (l & 31);
    });
    // scales: through aligned words
    const uint64_t wsa = (uint64_t)(uintptr_t)p.scales + (first + n0) * srow;
    const uint32_t ws0 = (uint32_t)wsa & 3u;
    const i32x4 wsres = uniform_rsrc((const void*)(uintptr_t)(wsa & ~3ull), (ws0 + (uint32_t)wrows * srow + 3u) & ~3u);
    uint64_t xsa = 0;
    uint32_t xs0 = 0;
    i32x4 xsres{};
    if constexpr (MX) {
        xsa = (uint64_t)(uintptr_t)p.x_scales + x_from * srow;
        xs0 = (uint32_t)xsa & 3u;
        xsres = uniform_rsrc((const void*)(uintptr_t)(xsa & ~3ull), (xs0 + (uint32_t)x_rows * srow + 3u) & ~3u);
    }

    // lane l of a DMA instruction over 128-byte rows fills slot l % 8 of row 8 i
    // + l / 8 (odd i: chunk ^ 4), over 64-byte rows slot l % 4 of row 16 i + l / 4
    const uint32_t ch8 = (l & 7) ^ (l >> 4), ch4 = (l & 3) ^ ((l >> 4) & 3);
    uint32_t ao[DA], bo[DB], so[SQ];
    i32x4 sres[SQ];
#pragma unroll
    for (int q = 0; q < DA; ++q) ao[q] = xr[q] * xrow + 16u * (ch8 ^ (4 * (q & 1)));
#pragma unroll
    for (int q = 0; q < DB; ++q) {
        const int r = MX ? 8 * (DB * w + q) + (l >> 3) : 16 * (DB * w + q) + (l >> 2);
        bo[q] = (uint32_t)min(r, wrows - 1) * wrow + 16u * (MX ? ch8 ^ (4 * (q & 1)) : ch4);
    }
#pragma unroll
    for (int q = 0; q < SQ; ++q) {  // scales: a row per lane, x's rows first
        const int first_r = MX ? 64 * (SQ * w + q) : 64 * (w % (TN / 64));
        const bool of_x = MX && first_r < TM;
        const int r = first_r + l - (MX && !of_x ? TM : 0);
        sres[q] = of_x ? xsres : wsres;
        so[q] = (of_x ? xs0 + xr[MX ? DA + q : 0] * srow : ws0 + (uint32_t)min(r, wrows - 1) * srow) & ~3u;
    }
    const uint32_t K = (uint32_t)p.K;
    constexpr uint32_t PAST = 0xfffffff0u;  // an offset that reads zeros
    // instruction q of x's stage t, into ring slot `st`
    const int AT = MX ? (p.K + 255) / 256 : (p.K + 127) / 128 * 2;  // stages
    auto dma_a = [&](int t, char* st, int q) {
        t = min(t, AT - 1);
        const uint32_t ch = ch8 ^ (4 * (q & 1));
        const bool past = RAGGED && (MX ? 256u * t + 32u * ch : 64u * t + 8u * ch) >= K;
        dma16_buf(xres, past ? PAST : ao[q] + 128u * t, st + 1024 * (DA * w + q));
    };
    // instruction q of W's piece t (MXFP4: stage t)
    const int BT = MX ? AT : AT / 2;
    auto dma_b = [&](int t, char* st, int q) {
        t = min(t, BT - 1);
        const uint32_t ch = MX ? ch8 ^ (4 * (q & 1)) : ch4;
        const bool past = RAGGED && (MX ? 256u : 128u) * t + 32u * ch >= K;
        dma16_buf(wres, past ? PAST : bo[q] + (MX ? 128u : 64u) * t, st + 1024 * (DB * w + q));
    };
    // instruction q of scale group t (of 512 or 128 k)
    const int ST = (p.K + (MX ? 511 : 127)) / (MX ? 512 : 128);
    auto dma_s = [&](int t, char* st, int q) {
        t = min(t, ST - 1);
        if constexpr (MX) {
            if (q < SQ)
                dma16_buf(sres[q], so[q] + 16u * t, st + 1024 * (SQ * w + q));
            else
                dma4_buf(sres[q - SQ], so[q - SQ] + 16u * t + 16u, st + 16 * S::SROWS + 256 * (SQ * w + q - SQ));
        } else {
            dma4_buf(sres[0], so[0] + 4u * t + 4u * q, st + 4 * TN * q + 256 * (w % (TN / 64)));
        }
    };

    f32x16 acc[MI][JN];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < JN; ++j) acc[i][j] = f32x16{};
    // the rows' first scale byte in their words
    uint32_t ash[MI], bsh[JN];
    if constexpr (RAGGED) {
#pragma unroll
        for (int i = 0; i < MI; ++i) ash[i] = MX ? (xs0 + xr[MX ? DA + SQ + i : 0] * srow) & 3u : 0u;
#pragma unroll
        for (int j = 0; j < JN; ++j) bsh[j] = (ws0 + (uint32_t)min(wn * WN + j * 32 + (l & 31), wrows - 1) * srow) & 3u;
    }
    struct Frag {
        u32x4 a[MI];
        u32x4 b[MX ? JN : 1];
    };
    struct Scales {
        uint32_t a[MX ? MI : 1], b[JN];
    };
    char* const ring_b = lds + S::NA * S::A;
    char* const ring_s = ring_b + S::NB * S::B;
    auto read_a = [&](const char* st, int ks, Frag& f) {
#pragma unroll
        for (int i = 0; i < MI; ++i) f.a[i] = *(const u32x4*)(st + 16 * slot128(wm * WM + i * 32 + (l & 31), 4 * h + ks));
    };
    // DMA that goes with MFMA m of NM of a step: `n` instructions, evenly
    auto spread = [](int m, int nm, int n, auto issue) {
#pragma unroll
        for (int r = 0; r < n; ++r)
            if (m == (r + 1) * nm / n - 1) {
                issue(r);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    constexpr int NM = MI * JN;
    Frag fr[2];

    if constexpr (MX) {
        Scales sg[2];
        auto read_b = [&](const char* st, int ks, Frag& f) {
#pragma unroll
            for (int j = 0; j < JN; ++j) f.b[j] = *(const u32x4*)(st + 16 * slot128(wn * WN + j * 32 + (l & 31), 4 * h + ks));
        };
        // stage t's word of row r: of the group's four, number 2 (t % 2) + h
        auto word = [&](int t, int r, uint32_t sh) -> uint32_t {
            const char* st = ring_s + (ONE ? 0 : (t >> 1) & 1) * S::S;
            const int d = 2 * (t & 1) + h;
            const uint32_t v = *(const uint32_t*)(st + 16 * r + 4 * d);
            if constexpr (!RAGGED) return v;
            const uint32_t next = *(const uint32_t*)(d == 3 ? st + 16 * S::SROWS + 4 * r : st + 16 * r + 4 * d + 4);
            const uint32_t all = __builtin_amdgcn_alignbyte(next, v, sh);
            // blocks of the row that are left from this lane's first on
            const int left = max(p.K / 32 - 8 * min(t, AT - 1) - 4 * h, 0);
            return left >= 4 ? all : (all & ~(~0u << (8 * left))) | (0x7f7f7f7fu << (8 * left));
        };
        auto read_scales = [&](int t, Scales& s) {
#pragma unroll
            for (int i = 0; i < MI; ++i) s.a[i] = word(t, wm * WM + i * 32 + (l & 31), RAGGED ? ash[i] : 0u);
#pragma unroll
            for (int j = 0; j < JN; ++j) s.b[j] = word(t, TM + wn * WN + j * 32 + (l & 31), RAGGED ? bsh[j] : 0u);
        };
        constexpr int NQ = DA + DB, H0 = NQ / 2;  // instructions of a stage; those that go with its predecessor's last step
        auto dma = [&](int t, int q) {
            if (q < DA)
                dma_a(t, lds + (ONE ? 0 : t & 1) * S::A, q);
            else
                dma_b(t, ring_b + (ONE ? 0 : t & 1) * S::B, q - DA);
        };
        auto step = [&](const Frag& f, const Scales& s, auto ks_, int n, auto issue) {
            constexpr int ks = decltype(ks_)::value;
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const int i = m % MI, j = m / MI;
                acc[i][j] = mfma32_mxfp4<ks>(f.b[j], s.b[j], f.a[i], s.a[i], acc[i][j]);
                spread(m, NM, n, issue);
            }
        };
        auto none = [](int) {};
        if constexpr (ONE) {
            auto load = [&](int t) {
                if (!(t & 1)) {
#pragma unroll
                    for (int q = 0; q < DS; ++q) dma_s(t >> 1, ring_s, q);
                }
#pragma unroll
                for (int q = 0; q < NQ; ++q) dma(t, q);
            };
            load(0);
#pragma unroll 1
            for (int t = 0; t < AT; ++t) {
                wait_vmcnt<0>();
                lds_barrier();  // the stage has landed
                Scales& now = sg[0];
                read_scales(t, now);
                auto read = [&](int ks) {
                    read_a(lds, ks, fr[0]);
                    read_b(ring_b, ks, fr[0]);
                };
                read(0);
                step(fr[0], now, std::integral_constant<int, 0>{}, 0, none);
                read(1);
                step(fr[0], now, std::integral_constant<int, 1>{}, 0, none);
                read(2);
                step(fr[0], now, std::integral_constant<int, 2>{}, 0, none);
                read(3);
                lds_barrier();  // every wave has read it
                if (t + 1 < AT) load(t + 1);
                __builtin_amdgcn_sched_barrier(0);
                step(fr[0], now, std::integral_constant<int, 3>{}, 0, none);
            }
        } else {
#pragma unroll
        for (int q = 0; q < DS; ++q) dma_s(0, ring_s, q);
#pragma unroll
        for (int q = 0; q < NQ; ++q) dma(0, q);
        wait_vmcnt<0>();
        lds_barrier();
#pragma unroll
        for (int q = 0; q < H0; ++q) dma(1, q);
        read_a(lds, 0, fr[0]);
        read_b(ring_b, 0, fr[0]);
        read_scales(0, sg[0]);
        auto stage = [&](int t, Scales& now, Scales& next) {
            const char *sa = lds + (t & 1) * S::A, *sb = ring_b + (t & 1) * S::B;
            read_a(sa, 1, fr[1]);
            read_b(sb, 1, fr[1]);
            step(fr[0], now, std::integral_constant<int, 0>{}, NQ - H0, [&](int r) { dma(t + 1, H0 + r); });
            read_a(sa, 2, fr[0]);
            read_b(sb, 2, fr[0]);
            if (t & 1)
                step(fr[1], now, std::integral_constant<int, 1>{}, 0, none);
            else  // the next group's scales
                step(fr[1], now, std::integral_constant<int, 1>{}, DS,
                     [&](int r) { dma_s((t >> 1) + 1, ring_s + (((t >> 1) + 1) & 1) * S::S, r); });
            read_a(sa, 3, fr[1]);
            read_b(sb, 3, fr[1]);
            step(fr[0], now, std::integral_constant<int, 2>{}, 0, none);
            wait_vmcnt<0>();  // this wave's part of stage t + 1 landed
            lds_barrier();    // every wave's; every wave is done reading stage t
            read_a(lds + (~t & 1) * S::A, 0, fr[0]);
            read_b(ring_b + (~t & 1) * S::B, 0, fr[0]);
            read_scales(t + 1, next);
            step(fr[1], now, std::integral_constant<int, 3>{}, H0, [&](int r) { dma(t + 2, r); });
        };
        int t = 0;
#pragma unroll 1
        for (; t + 1 < AT; t += 2) {
            stage(t, sg[0], sg[1]);
            stage(t + 1, sg[1], sg[0]);
        }
        if (t < AT) stage(t, sg[0], sg[1]);
        }
    } else {
        struct Weights {
            u32x4 b[JN];
            float s[JN];
        } wr[2];
        // W of stage t: block 2 (t % 2) + h of piece t / 2
        auto read_w = [&](int t, Weights& v) {
            const char* st = ring_b + ((t >> 1) & 1) * S::B;
            const char* ss = ring_s + ((t >> 1) & 1) * S::S;
            const int c = 2 * (t & 1) + h;
#pragma unroll
            for (int j = 0; j < JN; ++j) {
                const int r = wn * WN + j * 32 + (l & 31);
                v.b[j] = *(const u32x4*)(st + 16 * slot64(r, c));
                uint32_t d = *(const uint32_t*)(ss + 4 * r);
                if constexpr (RAGGED) d = __builtin_amdgcn_alignbyte(*(const uint32_t*)(ss + 4 * TN + 4 * r), d, bsh[j]);
                const bool past = RAGGED && 64u * (uint32_t)min(t, AT - 1) + 32u * h >= K;
                v.s[j] = __uint_as_float(past ? 127u << 23 : ((d >> (8 * c)) & 255u) << 23);
            }
        };
        auto step = [&](const Frag& f, const Weights& v, auto ks_, int n, auto issue) {
            constexpr int ks = decltype(ks_)::value;
            bf16x8 wv;
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const int i = m % MI, j = m / MI;
                if (i == 0) wv = mxfp4_bf16(v.b[j][ks], v.s[j]);
                acc[i][j] = mfma32(wv, __builtin_bit_cast(bf16x8, f.a[i]), acc[i][j]);
                spread(m, NM, n, issue);
            }
        };
        // ring slots of x's stages t, t + 1, t + 2
        char *a0 = lds, *a1 = lds + S::A, *a2 = lds + 2 * S::A;
#pragma unroll
        for (int q = 0; q < DA; ++q) dma_a(0, a0, q);
#pragma unroll
        for (int q = 0; q < DB; ++q) dma_b(0, ring_b, q);
#pragma unroll
        for (int q = 0; q < DS; ++q) dma_s(0, ring_s, q);
#pragma unroll
        for (int q = 0; q < DA; ++q) dma_a(1, a1, q);
        wait_vmcnt<DA>();
        lds_barrier();
        read_a(a0, 0, fr[0]);
        read_w(0, wr[0]);
        // stage t of piece t / 2: x of stage t + 2 goes out with the first two
        // steps, and in a piece's first stage the next piece with the third
        auto stage = [&](int t, auto first, Weights& now, Weights& next) {
            constexpr bool FIRST = decltype(first)::value;
            const int g = (t >> 1) + 1;
            read_a(a0, 1, fr[1]);
            step(fr[0], now, std::integral_constant<int, 0>{}, DA / 2, [&](int r) { dma_a(t + 2, a2, r); });
            read_a(a0, 2, fr[0]);
            step(fr[1], now, std::integral_constant<int, 1>{}, DA / 2, [&](int r) { dma_a(t + 2, a2, DA / 2 + r); });
            read_a(a0, 3, fr[1]);
            step(fr[0], now, std::integral_constant<int, 2>{}, FIRST ? DB + DS : 0, [&](int r) {
                if (r < DB)
                    dma_b(g, ring_b + (g & 1) * S::B, r);
                else
                    dma_s(g, ring_s + (g & 1) * S::S, r - DB);
            });
            wait_vmcnt<DA + (FIRST ? DB + DS : 0)>();  // what this stage issued may be under way
            lds_barrier();  // stage t + 1 whole; every wave is done reading stage t
            read_a(a1, 0, fr[0]);
            read_w(t + 1, next);
            step(fr[1], now, std::integral_constant<int, 3>{}, 0, [](int) {});
            char* const freed = a0;
            a0 = a1;
            a1 = a2;
            a2 = freed;
        };
#pragma unroll 1
        for (int t = 0; t < AT; t += 2) {
            stage(t, std::true_type{}, wr[0], wr[1]);
            stage(t + 1, std::false_type{}, wr[1], wr[0]);
        }
    }
    wait_vmcnt<0>();
    lds_barrier();  // the ring is free

    // acc[i][j][4g + e]: y row wm*WM + i*32 + l%32, column wn*WN + j*32 + 8g +
    // 4 (l/32) + e of the tile; through LDS to row-contiguous stores of 16 bytes
    // (y not on 16 bytes, or the last columns of a ragged N: one by one)
    const int size = YF32 ? 4 : 2;
    const bool vec = ((uintptr_t)p.y & 15) == 0 && (p.ldy * size & 15) == 0;
    if constexpr (YF32) {
        // half a tile at a time; 16-byte chunk q of row r at q ^ (r & 15)
        float* ly = (float*)lds;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (wm == half) {
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const int row = i * 32 + (l & 31);
#pragma unroll
                    for (int j = 0; j < JN; ++j)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const int q = (wn * WN + j * 32 + 8 * g + 4 * h) >> 2;
                            *(f32x4*)(ly + row * TN + 4 * (q ^ (row & 15))) =
                                f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                        }
                }
            }
            __syncthreads();
            float* yf = (float*)p.y + (int64_t)(m0 + half * WM) * p.ldy + n0;
            constexpr int PER = WM * TN / 4 / MG_THREADS;
#pragma unroll 4
            for (int it = 0; it < PER; ++it) {
                const int idx = tid + MG_THREADS * it, row = idx / (TN / 4), q = idx % (TN / 4);
                const f32x4 v = *(const f32x4*)(ly + row * TN + 4 * (q ^ (row & 15)));
                if (half * WM + row >= rows) continue;
                float* o = yf + (int64_t)row * p.ldy + 4 * q;
                if (vec && n0 + 4 * q + 4 <= p.N) {
                    *(f32x4*)o = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n0 + 4 * q + e < p.N) o[e] = v[e];
                }
            }
            __syncthreads();
        }
    } else {
        // 16-byte chunk q of row r at q ^ r
        uint16_t* ly = (uint16_t*)lds;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int row = wm * WM + i * 32 + (l & 31);
#pragma unroll
            for (int j = 0; j < JN; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int col = wn * WN + j * 32 + 8 * g + 4 * h;
                    const int q = (col >> 3) ^ (row & (TN / 8 - 1));
                    u32x2 v;
                    v[0] = pack_bf16x2_hw(acc[i][j][4 * g], acc[i][j][4 * g + 1]);
                    v[1] = pack_bf16x2_hw(acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
                    *(u32x2*)(ly + row * TN + 8 * q + (col & 7)) = v;
                    __builtin_amdgcn_sched_barrier(0);  // (registers)
                }
        }
        __syncthreads();
        uint16_t* yb = (uint16_t*)p.y + (int64_t)m0 * p.ldy + n0;
        constexpr int PER = TM * TN / 8 / MG_THREADS;
#pragma unroll 4
        for (int it = 0; it < PER; ++it) {
            const int idx = tid + MG_THREADS * it, row = idx / (TN / 8), q = idx % (TN / 8);
            const u32x4 v = *(const u32x4*)(ly + row * TN + 8 * (q ^ (row & (TN / 8 - 1))));
            if (row >= rows) continue;
            uint16_t* o = yb + (int64_t)row * p.ldy + 8 * q;
            if (vec && n0 + 8 * q + 8 <= p.N) {
                *(u32x4*)o = v;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n0 + 8 * q + e < p.N) o[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
            }
        }
    }
}

template <int XT, int TM, int TN, bool ONE, bool ROUTED, bool YF32, bool RAGGED>
hipError_t mg_launch(const Mxfp4GemmParams& p, hipStream_t st) {
    using S = MgShape<XT, TM, TN, ONE, RAGGED>;
    constexpr size_t lds = YF32 ? S::LDS_F32 : S::LDS_BF16;
    const auto kern = mxfp4_gemm_kernel<XT, TM, TN, ONE, ROUTED, YF32, RAGGED>;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
    const int64_t n_tiles = (p.N + TN - 1) / TN;
    const int64_t grid = ROUTED ? (mx_tile_bound(p, TM) * n_tiles + 7) / 8 * 8 : (p.M + (int64_t)TM - 1) / TM * n_tiles;
    if (grid * MG_THREADS >= (1ll << 32)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(MG_THREADS), lds, st, p);
    return hipGetLastError();
}

template <int XT, int TM, int TN, bool ONE, bool ROUTED>
hipError_t mg_launch_y(const Mxfp4GemmParams& p, hipStream_t st) {
    const bool ragged = p.K % (XT == MX_X_MXFP4 ? 256 : 128) || ((uintptr_t)p.scales & 3) || ((uintptr_t)p.x_scales & 3);
    if (p.y_f32)
        return ragged ? mg_launch<XT, TM, TN, ONE, ROUTED, true, true>(p, st) : mg_launch<XT, TM, TN, ONE, ROUTED, true, false>(p, st);
    return ragged ? mg_launch<XT, TM, TN, ONE, ROUTED, false, true>(p, st) : mg_launch<XT, TM, TN, ONE, ROUTED, false, false>(p, st);
}

template <int XT, bool ONE>
hipError_t mg_launch_128(const Mxfp4GemmParams& p, hipStream_t st) {
    return p.offsets ? mg_launch_y<XT, 128, 128, ONE, true>(p, st) : mg_launch_y<XT, 128, 128, ONE, false>(p, st);
}

}  // namespace

hipError_t launch_mxfp4_tiles(const Mxfp4GemmParams& p, MxTiles kind, hipStream_t st) {
    if (p.x_kind == MX_X_MXFP4) {
        if (kind == MX_TILES_256) return mg_launch_y<MX_X_MXFP4, 256, 256, false, false>(p, st);
        return kind == MX_TILES_128x3 ? mg_launch_128<MX_X_MXFP4, true>(p, st) : mg_launch_128<MX_X_MXFP4, false>(p, st);
    }
    return kind == MX_TILES_256 ? mg_launch_y<MX_X_BF16, 256, 256, false, false>(p, st) : mg_launch_128<MX_X_BF16, false>(p, st);
}

}  // namespace mr
