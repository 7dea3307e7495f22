// Attention of a few queries of each sequence over a paged cache of keys and
// values, in bf16 or MXFP4, and the joining of partial results.
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j   over the keys j that i sees
//
// with the softmax in one pass: a running maximum m, l = sum 2^(s_j - m) and
// o = sum 2^(s_j - m) v_j, in f32; a sink enters l at the end.
//
// What bounds it: the cache's bytes from HBM (a key head's rows are read once
// for all of its query heads), and for short sequences the chain of loads.
// So a wave works alone: it walks keys of its own in steps of 32, has the next
// step's loads in flight, and never meets a barrier before the end.  A step:
//   - the packed rows arrive in registers, whole neighbouring rows a load;
//     keys go to the wave's part of LDS as stored, values as bf16;
//   - S^T = K . Q^T on 16x16x32 MFMA.  Lane (n, g) holds dims DP/4 g .. of
//     key n, so that an MXFP4 key is one 16-byte read (of 128 dims) and its
//     scale one byte; q's registers hold the same dims;
//   - the lane that has query n's scores keeps its maximum and sum;
//   - O^T += V^T . P^T: the scores' registers are the second operand as they
//     are, V^T comes by transposed reads.  P is rounded to bf16 (at most 2^-8 of
//     each term, whose errors average out); sums stay in f32.
// The waves of a workgroup split its keys and meet once, in LDS.  A tile's keys
// are split over workgroups where that fills the GPU (kv_attention_route),
// which leave (m, l, o) in the workspace for the join.
//   Measured (8 query heads a key head of 128, MXFP4 unless said; us): 64 sequences of
// 4000 keys, 8 key heads, 56, 4.9 TB/s, in bf16 186, 5.6 TB/s; one of 131072, 8 key heads,
// 30 and the join 4; 64 of 1000 to 12000, 4 key heads, 39 and the join 4 (about 10 of them
// while the last parts leave CUs idle).  A wave alone takes 0.9 a step, mostly the issue
// of its instructions (150 vector, about 70 scalar, 32 LDS): the loads of a second step in
// flight changed nothing (the last two, with their joins, 43 and 51 for 38 and 44, since
// fewer waves fit), nor did eight waves a workgroup (38 and 49), nor keys as codes on the
// scaled matrix instructions against q in two e4m3 parts (38 and 45, and scores 100 times
// less exact).
//
// Scores of keys that a row does not see become -inf, values that no row may see zeros
// where they are loaded.  Infinities and NaN of values that some rows of a step see and
// others do not, or whose probability left f32's range, take a way of their own
// (kv_add_infinite).
#include <algorithm>

#include "kv_tiles.hpp"

namespace mr {

namespace {

constexpr int KD_WAVES = 4, KD_STEP = 32;

template <int DP, bool MX>
struct KvDecodeLds {
    // rows apart by an odd number of 16-byte (K) and 32-byte (V) pieces, so that 16
    // rows read at one column, and 8 rows read by transposed reads, meet all banks
    static constexpr int K_STRIDE = MX ? DP / 2 + 16 : DP * 2 + 16;  // bytes
    static constexpr int V_STRIDE = DP + 16;                         // values
    static constexpr int V_BYTES = KD_STEP * V_STRIDE * 2, K_BYTES = KD_STEP * K_STRIDE;
    static constexpr int S_BYTES = MX ? KD_STEP * DP / 32 : 0;  // the keys' scales
    static constexpr int O_STRIDE = DP + 4;                     // f32, the end's sums of 16 rows
    // the keys are in registers again before the values take their place
    static constexpr int ALL_K = K_BYTES + S_BYTES, WAVE = ((V_BYTES > ALL_K ? V_BYTES : ALL_K) + 15) / 16 * 16;
    static_assert(16 * O_STRIDE * 4 <= WAVE, "the sums of 16 rows fit");
};

// A wave's LDS operations are done in order; the compiler has to keep them so
// where lanes hand values over.
__device__ __forceinline__ void kd_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int DP, int R, bool MX>
__global__ void __launch_bounds__(64 * KD_WAVES) kv_decode_kernel(KvAttnParams p) {
    using L = KvDecodeLds<DP, MX>;
    constexpr int ROWS = 16 * R, KS = DP / 32, DT = DP / 16, CPL = DP / 4, DN = DP / 64;
    __shared__ __attribute__((aligned(16))) char lds[KD_WAVES * L::WAVE];
    __shared__ float sm[KD_WAVES][ROWS], sl[KD_WAVES][ROWS];
    const int l = threadIdx.x & 63, n = l & 15, g = l >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // first parts first: the parts that short sequences do not have are spread over the XCDs
    const int unit = blockIdx.x / p.kv_heads, kv_head = blockIdx.x - unit * p.kv_heads;
    const int tiles = gridDim.x / (p.kv_heads * p.splits);
    const int split = unit / tiles, tile_id = unit - split * tiles;
    KvTile t;
    if (!kv_find<ROWS>(p, tile_id, t)) return;

    // this workgroup's keys, and this wave's
    int kb = t.kbeg, ke = t.kend;
    if (p.splits > 1) {
        const int64_t at = (int64_t)t.kbeg + (int64_t)split * p.chunk;
        kb = (int)min(at, (int64_t)t.kend);
        if (split + 1 < p.splits) ke = (int)min(at + p.chunk, (int64_t)t.kend);
    }
    const int per = ((max(ke - kb, 0) + KD_WAVES - 1) / KD_WAVES + KD_STEP - 1) / KD_STEP * KD_STEP;
    const int wb = min(kb + w * per, ke), we = min(wb + per, ke);

    char* mine = lds + w * L::WAVE;
    uint16_t* vt = (uint16_t*)mine;
    char* kt = mine;
    uint8_t* ksc = (uint8_t*)(kt + L::K_BYTES);

    KvRow row[R];
    bf16x8 q[R][KS];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        row[r] = kv_row(p, t, kv_head, t.first_row + 16 * r + n);
        const uint16_t* qp = p.q + row[r].token * p.q_ts + row[r].head * p.q_hs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = CPL * g + 8 * s;
            q[r][s] = row[r].ok && d < p.dim ? *(const bf16x8*)(qp + d) : bf16x8{};
        }
    }

    float m[R], sum[R];
    f32x4 o[R][DT];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        sum[r] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] = f32x4{};
    }

    int apart_from = we, apart_to = 0;  // keys whose infinite values were left out
    if (wb < we) {
        // the two groups of a step: their pages, a step ahead of their loads (past the last
        // key again its page, whose rows are cut and masked)
        const char* table = (const char*)(p.table + t.b * p.table_stride);
        const uint32_t last = 4u * ((uint32_t)(we - 1) / (uint32_t)p.page_size);
        uint32_t entry = 4u * ((uint32_t)wb / (uint32_t)p.page_size);  // bytes
        int offset = wb - (int)(entry / 4) * p.page_size;
        int id[2], off[2];
        auto look = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                off[h] = offset;
                id[h] = s_load((const int32_t*)(table + min(entry, last)));
                offset += 16;
                const int same = (offset - p.page_size) >> 31;  // -1, or 0 at a page's end
                offset &= same;
                entry += 4 + 4 * same;
            }
        };
        using Group = KvGroup<DP, MX>;
        const typename Group::At at = Group::at(p.dim, l);
        Group k[2], v[2];
        int have[2];
        auto load = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                have[h] = kv_page(p, id[h]);
                k[h].load(kv_from<MX>(p, true, kv_head, id[h], off[h]), at);
                v[h].load(kv_from<MX>(p, false, kv_head, id[h], off[h]), at);
            }
        };
        look();
        load();
        look();
        for (int k0 = wb; k0 < we; k0 += KD_STEP) {
            const int seen[2] = {have[0], have[1]};
            const bool all = k0 >= t.all_lo && k0 + KD_STEP <= min(t.all_hi, we) && (seen[0] & seen[1]);
            if (!all) {
#pragma unroll
                for (int h = 0; h < 2; ++h)  // (of a page that does not exist, all rows)
                    if (k0 + 16 * h + 16 > we || !seen[h]) v[h].cut(seen[h] ? we - k0 - 16 * h : 0, l);
                const bool apart = __builtin_amdgcn_ballot_w64(v[0].not_finite() || v[1].not_finite()) != 0;
                if (apart) {
                    apart_to = k0 + KD_STEP, apart_from = min(apart_from, k0);
#pragma unroll
                    for (int h = 0; h < 2; ++h) v[h].clean();
                }
            }
            if (p.dim < DP) {
#pragma unroll
                for (int h = 0; h < 2; ++h) k[h].narrow(at), v[h].narrow(at);
            }
            // keys through LDS, as they are stored, into the operands' registers
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (MX) {
#pragma unroll
                    for (int i = 0; i < Group::N; ++i)
                        if (Group::active(l)) {
                            const int rr = 16 * h + Group::row(l, i);
                            *(u32x4*)(kt + rr * L::K_STRIDE + 16 * Group::piece(l)) = k[h].v[i];
                            ksc[rr * (DP / 32) + Group::piece(l)] = k[h].scale[i];
                        }
                } else {
                    k[h].put((uint16_t*)kt + 16 * h * (L::K_STRIDE / 2), L::K_STRIDE / 2, l);
                }
            }
            kd_fence();
            constexpr int KW = MX ? KS / 4 + (KS < 4) : KS;  // 16-byte pieces of a lane (DP 64 in MXFP4: half of one)
            u32x4 kw[2][KW];
            uint32_t ks[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char* kr = kt + (16 * h + n) * L::K_STRIDE + g * (MX ? CPL / 2 : CPL * 2);
                if constexpr (MX && KS == 2) {
                    const u32x2 x = *(const u32x2*)kr;
                    kw[h][0] = u32x4{x[0], x[1], 0, 0};
                } else {
#pragma unroll
                    for (int i = 0; i < KW; ++i) kw[h][i] = *(const u32x4*)(kr + 16 * i);
                }
                if constexpr (MX) {  // the lane's dims lie in one block, or (DP 256) in two
                    const uint8_t* sc = ksc + (16 * h + n) * (DP / 32) + CPL * g / 32;
                    ks[h][0] = sc[0];
                    ks[h][1] = DP == 256 ? sc[1] : 0;
                }
            }
            kd_fence();
            // values to where the keys were
#pragma unroll
            for (int h = 0; h < 2; ++h) v[h].put(vt + 16 * h * L::V_STRIDE, L::V_STRIDE, l);
            if (k0 + KD_STEP < we) {
                load();
                look();
            }

            f32x4 s[2][R];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int r = 0; r < R; ++r) s[h][r] = f32x4{};
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    bf16x8 a;
                    if constexpr (MX)
                        a = mxfp4_bf16(kw[h][i / 4][i % 4], __uint_as_float(ks[h][i / 4] << 23));
                    else
                        a = __builtin_bit_cast(bf16x8, kw[h][i]);
#pragma unroll
                    for (int r = 0; r < R; ++r) s[h][r] = mfma16(a, q[r][i], s[h][r]);
                }
            }

            bf16x8 pb[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (!all) {
                    int lo = row[r].lo - k0 - 4 * g, hi = min(row[r].hi, we) - k0 - 4 * g;
                    asm volatile("" : "+v"(lo), "+v"(hi));  // (behind the branch)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i)  // key 4 g + this of the step
                            if (16 * h + i < lo || 16 * h + i >= hi || !seen[h]) s[h][r][i] = -INFINITY;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[h][r][i]);
                mx = xor32_max(xor16_max(mx)) * p.scale_log2;  // (the scale is positive)
                const bool raise = mx > m[r] + KV_TAU;
                if (__builtin_amdgcn_ballot_w64(raise)) {
                    const float up = raise ? mx : m[r];
                    const float alpha = raise ? __builtin_amdgcn_exp2f(m[r] - up) : 1.f;
                    m[r] = up;
                    sum[r] *= alpha;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[r][d] *= alpha;
                }
                const float ref = m[r] == -INFINITY ? 0.f : m[r];  // (no key yet: every score is -inf)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float e = __builtin_amdgcn_exp2f(fmaf(s[h][r][i], p.scale_log2, -ref));
                        sum[r] += e;
                        pb[r][4 * h + i] = (__bf16)e;
                    }
            }

            kd_fence();
            // key 4 g + e of group 0 and 4 g + e - 4 of group 1 are k-slot 8 g + e
            auto values = [&](int d) {
                const uint16_t* at = vt + (4 * g + (n >> 2)) * L::V_STRIDE + 16 * d + 4 * (n & 3);
                const bf16x4 lo = ds_read_tr16(at), hi = ds_read_tr16(at + 16 * L::V_STRIDE);
                return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            };
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const bf16x8 a = values(d);
#pragma unroll
                for (int r = 0; r < R; ++r) o[r][d] = mfma16(a, pb[r], o[r][d]);
            }
            kd_fence();
        }
    }

    // infinite values that were left out (kv_add_infinite)
    kv_each_infinite<DP, MX>(
        p, t.b, kv_head, apart_from, min(apart_to, we), l, [](int) { return true; },
        [&](int first, int last) {
            for (int key = first; key < last; ++key)
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int d = 0; d < DT; ++d)
                        kv_add_infinite<MX>(p, t.b, kv_head, key, key >= row[r].lo && key < row[r].hi, 16 * d + 4 * g,
                                            [&](int j, float v) { o[r][d][j] += v; });
        });

    // the waves' sums
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float all = xor32_sum(xor16_sum(sum[r]));
        if (g == 0) {
            sm[w][16 * r + n] = m[r];
            sl[w][16 * r + n] = all;
        }
    }
    __syncthreads();
    const int rn = threadIdx.x >> 4, dn = 4 * (threadIdx.x & 15);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float* part = (float*)mine;
#pragma unroll
        for (int d = 0; d < DT; ++d) *(f32x4*)(part + n * L::O_STRIDE + 16 * d + 4 * g) = o[r][d];
        __syncthreads();
        // thread: row rn, dims dn + 64 i
        float top = -INFINITY, total = 0.f, a[KD_WAVES];
#pragma unroll
        for (int x = 0; x < KD_WAVES; ++x) top = fmaxf(top, sm[x][16 * r + rn]);
#pragma unroll
        for (int x = 0; x < KD_WAVES; ++x) {
            const float mw = sm[x][16 * r + rn];
            a[x] = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - top);
            total = fmaf(sl[x][16 * r + rn], a[x], total);
        }
        const KvRow to = kv_row(p, t, kv_head, t.first_row + 16 * r + rn);
        f32x4 x[DN];
#pragma unroll
        for (int i = 0; i < DN; ++i) {
            x[i] = f32x4{};
#pragma unroll
            for (int y = 0; y < KD_WAVES; ++y)
                x[i] += a[y] * *(const f32x4*)((const float*)(lds + y * L::WAVE) + rn * L::O_STRIDE + dn + 64 * i);
        }
        bool nan = false;
#pragma unroll
        for (int i = 0; i < DN; ++i) nan |= kv_nan(x[i]);
        nan &= to.ok & (total == total);
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(nan) != 0, 0)) {  // (kv_add_infinite)
            f32x4 y[DN];
#pragma unroll
            for (int i = 0; i < DN; ++i) y[i] = f32x4{};
            bool left = true;
            kv_each_infinite<DP, MX>(
                p, t.b, kv_head, kb, ke, l, [&](int) { return left; },
                [&](int first, int last) {
                    for (int key = first; key < last; ++key)
#pragma unroll
                        for (int i = 0; i < DN; ++i)
                            kv_add_infinite<MX>(p, t.b, kv_head, key, nan && key >= to.lo && key < to.hi, dn + 64 * i,
                                                [&](int j, float v) { y[i][j] += v; });
                    bool more = false;
#pragma unroll
                    for (int i = 0; i < 4 * DN; ++i) more |= (x[i / 4][i % 4] != x[i / 4][i % 4]) & (y[i / 4][i % 4] == y[i / 4][i % 4]);
                    left = __builtin_amdgcn_ballot_w64(nan && more) != 0;
                });
#pragma unroll
            for (int i = 0; i < 4 * DN; ++i)  // (none: sums of finite values have left f32's range)
                if (nan && x[i / 4][i % 4] != x[i / 4][i % 4] && !(__builtin_fabsf(y[i / 4][i % 4]) < INFINITY)) x[i / 4][i % 4] = y[i / 4][i % 4];
        }
        if (to.ok) {
            const int64_t at = (int64_t)to.token * (p.kv_heads * p.group) + to.head;
            float inv = 1.f;
            if (p.splits == 1) {
                const KvEnd end = kv_end(top, total, p.sinks, to.head);
                inv = end.inv;
                if (p.lse && dn == 0) p.lse[at] = end.lse;
            } else if (dn == 0) {
                float* ml = p.part_ml + 2 * (at * p.splits + split);
                ml[0] = top;
                ml[1] = total;
            }
            if (p.splits == 1 || total != 0.f) {
#pragma unroll
                for (int i = 0; i < DN; ++i) {
                    const int d = dn + 64 * i;
                    if (d >= p.dim) break;
                    if (p.splits > 1) {
                        *(f32x4*)(p.part_o + (at * p.splits + split) * p.dim + d) = x[i];
                        continue;
                    }
                    const f32x4 y = total == 0.f ? f32x4{} : kv_weighted(x[i], inv);  // (0 times an infinity is not)
                    if (p.out_f32)
                        *(f32x4*)((float*)p.out + to.token * p.out_ts + to.head * p.out_hs + d) = y;
                    else
                        *(u32x2*)((uint16_t*)p.out + to.token * p.out_ts + to.head * p.out_hs + d) =
                            u32x2{pack_bf16x2_hw(y[0], y[1]), pack_bf16x2_hw(y[2], y[3])};
                }
            }
        }
        __syncthreads();
    }
}

// The parts of a row joined: blockIdx.x is the (query, head), blockIdx.y a span of
// `cols` dims; 4 dims a thread, threads that are left over share the parts.
constexpr int KJ_MAX = 1024;  // parts
constexpr int KJ_FEW = 32;    // of them where a row has a group of lanes alone
constexpr int KJ_EARLY = 4;

__global__ void __launch_bounds__(256) kv_join_kernel(KvAttnParams p, int span) {
    __shared__ float weight[KJ_MAX];
    __shared__ __attribute__((aligned(16))) float add[256 * 4];
    __shared__ float red[4];
    const int heads = p.kv_heads * p.group;
    const int64_t at = blockIdx.x;
    const int token = (int)(at / heads), head = (int)(at - (int64_t)token * heads);
    // tokens that no sequence has are left as they are
    if (p.q_offsets && (token < s_load(p.q_offsets) || token >= s_load(p.q_offsets + p.batch))) return;
    const f32x2* ml = (const f32x2*)p.part_ml + at * p.splits;
    const int w = threadIdx.x >> 6;
    const int d0 = blockIdx.y * span, cols = min(span, p.dim - d0) / 4;
    const int shares = 256 / cols, share = threadIdx.x / cols, c = threadIdx.x - share * cols;
    float top = -INFINITY;
    f32x2 mine[KJ_MAX / 256];
    // the first sums of this thread's share are under way while the weights are found
    const float* o = p.part_o + at * p.splits * p.dim + d0 + 4 * c;
    f32x4 early[KJ_EARLY];
#pragma unroll
    for (int i = 0; i < KJ_EARLY; ++i) {
        const int s = share + shares * i;
        early[i] = share < shares && s < p.splits ? *(const f32x4*)(o + (int64_t)s * p.dim) : f32x4{};
    }
#pragma unroll
    for (int i = 0; i < KJ_MAX / 256; ++i) {
        const int s = threadIdx.x + 256 * i;
        mine[i] = s < p.splits ? ml[s] : f32x2{-INFINITY, 0.f};
    }
#pragma unroll
    for (int i = 0; i < KJ_MAX / 256; ++i) top = fmaxf(top, mine[i][0]);
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) red[w] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < KJ_MAX / 256; ++i) {
        const float a = mine[i][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine[i][0] - top);
        total = fmaf(mine[i][1], a, total);
        weight[threadIdx.x + 256 * i] = mine[i][1] == 0.f ? -1.f : a;  // (no sums were left: not read)
    }
    total = wave_sum(total);
    if ((threadIdx.x & 63) == 0) red[w] = total;
    __syncthreads();
    total = (red[0] + red[1]) + (red[2] + red[3]);
    const KvEnd end = kv_end(top, total, p.sinks, head);
    const float inv = end.inv;
    if (p.lse && threadIdx.x == 0 && blockIdx.y == 0) p.lse[at] = end.lse;
    f32x4 x{};
    if (share < shares) {
#pragma unroll
        for (int i = 0; i < KJ_EARLY; ++i) {
            const int s = share + shares * i;
            if (s < p.splits && !(weight[s] < 0.f)) x += weight[s] * early[i];
        }
#pragma unroll 8
        for (int s = share + KJ_EARLY * shares; s < p.splits; s += shares)
            if (!(weight[s] < 0.f)) x += weight[s] * *(const f32x4*)(o + (int64_t)s * p.dim);
        if (__builtin_expect(kv_nan(x) && total == total, 0)) {  // (an infinity of a part whose weight is 0)
            x = f32x4{};
            for (int s = share; s < p.splits; s += shares)
                if (!(weight[s] < 0.f)) x += kv_weighted(*(const f32x4*)(o + (int64_t)s * p.dim), weight[s]);
        }
    }
    *(f32x4*)(add + 4 * threadIdx.x) = x;
    __syncthreads();
    if (share) return;
    for (int s = 1; s < shares; ++s) x += *(const f32x4*)(add + 4 * (s * cols + c));
    const int64_t to = token * p.out_ts + head * p.out_hs + d0 + 4 * c;
    x = kv_weighted(x, inv);
    if (p.out_f32)
        *(f32x4*)((float*)p.out + to) = x;
    else
        *(u32x2*)((uint16_t*)p.out + to) = u32x2{pack_bf16x2_hw(x[0], x[1]), pack_bf16x2_hw(x[2], x[3])};
}

// The same for many rows of few parts: 2^lanes_log2 lanes have a row, 4 dims a lane, and
// read its parts one after another (8192 rows of 8 parts of 128 dims, attention with its
// join: 39 us, 50 with a workgroup a row; 1024 rows of 32 parts 47 and 43).
__global__ void __launch_bounds__(256) kv_join_rows_kernel(KvAttnParams p, int lanes_log2) {
    const int heads = p.kv_heads * p.group, c = 4 * (threadIdx.x & ((1 << lanes_log2) - 1));
    const int64_t at = ((int64_t)blockIdx.x << (8 - lanes_log2)) + (threadIdx.x >> lanes_log2);
    if (at >= (int64_t)p.tokens * heads) return;
    const int token = (int)(at / heads), head = (int)(at - (int64_t)token * heads);
    // tokens that no sequence has are left as they are
    if (p.q_offsets && (token < s_load(p.q_offsets) || token >= s_load(p.q_offsets + p.batch))) return;
    const f32x2* ml = (const f32x2*)p.part_ml + at * p.splits;
    float top = -INFINITY;
    int first = p.splits, last = 0;  // the parts that left sums are among these
    for (int s = 0; s < p.splits; ++s) {
        const f32x2 x = ml[s];
        top = fmaxf(top, x[0]);
        if (x[1] != 0.f) first = min(first, s), last = s + 1;
    }
    float total = 0.f;
    f32x4 x{};
    const float* o = p.part_o + at * p.splits * p.dim + (c < p.dim ? c : 0);
#pragma unroll 4
    for (int s = first; s < last; ++s) {
        const f32x2 y = ml[s];
        const f32x4 v = *(const f32x4*)(o + (int64_t)s * p.dim);
        const float a = y[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(y[0] - top);
        total = fmaf(y[1], a, total);
        if (y[1] != 0.f) x += a * v;
    }
    if (__builtin_expect(kv_nan(x) && total == total, 0)) {  // (an infinity of a part whose weight is 0)
        x = f32x4{};
        for (int s = first; s < last; ++s) {
            const f32x2 y = ml[s];
            if (y[1] != 0.f)
                x += kv_weighted(*(const f32x4*)(o + (int64_t)s * p.dim), __builtin_amdgcn_exp2f(y[0] - top));
        }
    }
    const KvEnd end = kv_end(top, total, p.sinks, head);
    const float inv = end.inv;
    if (p.lse && c == 0) p.lse[at] = end.lse;
    if (c >= p.dim) return;
    const int64_t to = token * p.out_ts + head * p.out_hs + c;
    x = kv_weighted(x, inv);
    if (p.out_f32)
        *(f32x4*)((float*)p.out + to) = x;
    else
        *(u32x2*)((uint16_t*)p.out + to) = u32x2{pack_bf16x2_hw(x[0], x[1]), pack_bf16x2_hw(x[2], x[3])};
}

template <int DP, bool MX>
hipError_t decode_rows(const KvAttnParams& p, int rows, unsigned grid, hipStream_t st) {
    const dim3 block(64 * KD_WAVES);
    if (rows == 16)
        hipLaunchKernelGGL((kv_decode_kernel<DP, 1, MX>), dim3(grid), block, 0, st, p);
    else if (rows == 32)
        hipLaunchKernelGGL((kv_decode_kernel<DP, 2, MX>), dim3(grid), block, 0, st, p);
    else if constexpr (DP <= 128)
        hipLaunchKernelGGL((kv_decode_kernel<DP, 4, MX>), dim3(grid), block, 0, st, p);
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

template <bool MX>
hipError_t decode_dim(const KvAttnParams& p, int rows, unsigned grid, hipStream_t st) {
    if (p.dim <= 64) return decode_rows<64, MX>(p, rows, grid, st);
    if (p.dim <= 128) return decode_rows<128, MX>(p, rows, grid, st);
    return decode_rows<256, MX>(p, rows, grid, st);
}

}  // namespace

// `keys`: the most that a sequence has (an estimate is enough: a longer one's last
// part takes what is left).  Parts of equal length, so that long sequences weigh no
// more than their keys.  A workgroup costs about 4 us around its keys and 0.95 us per
// 128 of them while HBM is not the bound, the join 3 to 5 us, more with many parts or
// rows; measured with 8 heads a key head of 128 dims, MXFP4 (us):
//   16 rows, little work: one workgroup a CU, parts of 128 keys or more (4 key heads: 4000
//     keys in parts of 128 / 512 / whole 8.7 / 11.5 / 34.7; 32000 in 128 / 512 / 2048
//     17.8 / 13.8 / 24.3)
//   16 rows, much: parts of 512 keys or more, three workgroups a CU, all of a length (131072
//     keys, 8 key heads, by 3 / 3.5 / 4 / 5 a CU 35.6 / 38.8 / 37.4 / 40.3; bf16, 32
//     sequences of 2000 to 8000, by 3 / 4 59 / 67), four of up to 64 dims (27.3 / 28.2 /
//     25.6 / 26.4), but of 1536 keys at most, since lengths differ (64 of 1000 to 12000, 4
//     key heads, in 1024 / 1536 / 2048 49 / 45 / 48)
//   32 and 64 rows leave more sums and fill a CU with two workgroups (24 rows, 32
//     sequences of 1000 to 6000, in 512 / 1024 / 2048 38 / 32 / 36) or one (40 rows: 72 /
//     57 / 48; 24 rows of 256 dims 77 / 64 / 52)
//   no parts up to 512 keys (1 query of 500 in 128 / whole 8.6 / 7.8, 6 queries of 300
//     14.5 / 13.4), nor for two workgroups a CU without them unless sequences are long and
//     may differ (64 of 4000, 8 key heads, whole / in 2048 57 / 61; 8 queries of 64 x 3000
//     113 / 137)
//   prompts: one workgroup a CU, and sums of many rows are dear: parts where whole tiles
//     leave half of the CUs idle (256 tiles, 100 queries of 16 x 600 keys, in 512 / whole
//     68 / 33; 64 tiles, 512 queries behind 16000, in 1024 / 4096 / whole 185 / 144 / 411;
//     4 tiles, 16 queries behind 2000, in 128 / 256 / 512 17.7 / 18.9 / 23.2), and few keys
//     in one (16 queries of 250 in 128 / whole 16.1 / 12.1, of 400 16.7 / 17.2; 512 queries
//     of 512, 64 tiles, 30 / 23)
//   at most 32 workgroups a CU in parts: more of them cost more than what unequal lengths leave
//     idle, and workspace without end (64 sequences, 8 key heads, of 8000 to 65536 keys, by
//     8 / 16 / 32 / 64 / any 395 / 378 / 383 / 401 / 423; of 1 to 65536, each 1.25 times the
//     next, 202 / 131 / 115 / 122 / 138; 256 of 4000 to 32768 662 / 727 / 713 / 741 / 818)
// A tile of the few-query kernel has at most 64 rows (32 of 256 dims: registers).  More
// are prompts: 128 rows behind 16000 keys 27.8 us as such, 32.6 in tiles of 64.
constexpr int KV_PARTS = 32;  // workgroups a CU, where there are parts

KvAttnRoute kv_attention_route(int64_t tokens, int batch, bool ragged, int kv_heads, int group, int dim, int window,
                               int64_t keys, int cu_count) {
    KvAttnRoute r;
    const int64_t rows = ragged ? (tokens * group + batch - 1) / batch : group;  // of a sequence, on average
    r.prompt = rows > (dim > 128 ? 32 : 64);
    // tiles of as few rows as hold a sequence's
    r.rows = r.prompt ? (dim > 128 ? 128 : 256) : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    r.threads = r.prompt ? 2 * r.rows : 64 * KD_WAVES;  // (a wave has 32 rows of a prompt)
    r.tiles = ragged ? (tokens * group + r.rows - 1) / r.rows + batch : int64_t(batch) * ((group + r.rows - 1) / r.rows);
    const int64_t groups = batch * ((rows + r.rows - 1) / r.rows) * kv_heads;  // workgroups without parts
    // a tile's queries span at most its rows' positions
    if (window) keys = std::min<int64_t>(keys, (int64_t)window + r.rows + 16);
    const int64_t cus = cu_count, work = std::min(groups, KV_PARTS * cus) * std::max<int64_t>(keys, 1);
    int64_t chunk;
    if (r.prompt) {
        chunk = std::max<int64_t>(128, groups >= cus ? keys : (keys + cus / groups - 1) / (cus / groups));
        if (keys <= 256 || (keys <= 512 && 8 * groups >= cus)) chunk = keys;
    } else {
        const int fit = r.rows * dim > 32 * 128 ? 1 : 2;  // workgroups a CU
        if (r.rows == 16)
            chunk = std::max({std::min<int64_t>(work / cus, 512), work / ((dim > 64 ? 3 : 4) * cus), int64_t(128)});
        else
            chunk = std::max<int64_t>(256, work / (fit * cus));
        chunk = std::min<int64_t>(chunk, r.rows > 16 && fit == 1 ? 2048 : 1536);
        if (keys <= 512 || (groups >= 2 * cus && keys <= 4096)) chunk = keys;
    }
    const int64_t most = std::min<int64_t>(KJ_MAX, std::max<int64_t>(1, KV_PARTS * cus / groups));
    chunk = std::max(chunk, (keys + most - 1) / most);
    chunk = std::max<int64_t>(64, (chunk + 63) / 64 * 64);
    r.splits = (int)std::max<int64_t>(1, (keys + chunk - 1) / chunk);
    if (tokens * kv_heads * group > (1 << 20)) r.splits = 1;  // (the join has a workgroup per row)
    r.chunk = (int)std::min<int64_t>(chunk, INT32_MAX - 63);
    return r;
}

size_t kv_attention_workspace(const KvAttnRoute& r, int64_t tokens, int heads, int dim) {
    return r.splits == 1 ? 0 : size_t(tokens) * heads * r.splits * (size_t(dim) + 2) * 4;
}

hipError_t launch_kv_attention(const KvAttnParams& p, const KvAttnRoute& r, hipStream_t st) {
    const unsigned grid = (unsigned)(r.tiles * p.kv_heads * r.splits);
    hipError_t e;
    if (r.prompt)
        e = launch_kv_prompt(p, grid, st);
    else
        e = p.k_scales ? decode_dim<true>(p, r.rows, grid, st) : decode_dim<false>(p, r.rows, grid, st);
    if (e != hipSuccess || r.splits == 1) return e;
    const int64_t rows = (int64_t)p.tokens * p.kv_heads * p.group;
    if (r.splits <= KJ_FEW && rows >= 2048) {
        int lanes_log2 = 3;
        while ((4 << lanes_log2) < p.dim) ++lanes_log2;
        const int64_t per = 256 >> lanes_log2;
        hipLaunchKernelGGL(kv_join_rows_kernel, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, st, p, lanes_log2);
        return hipGetLastError();
    }
    // few rows: 32 dims a workgroup, so that more of them read
    const int span = rows < 1024 ? 32 : p.dim;
    hipLaunchKernelGGL(kv_join_kernel, dim3((unsigned)rows, (unsigned)((p.dim + span - 1) / span)), dim3(256), 0, st, p, span);
    return hipGetLastError();
}

}  // namespace mr
