// Attention of many queries of a sequence over a paged cache (kv_attention.hip
// has the formula, the small form and what is shared).
//
// A workgroup of four waves has 128 (query, head) rows of one sequence and key
// head, heads of a query next to each other, so that a tile spans few positions
// and all heads of a group share the keys.  Tiles of 64 keys come through two
// LDS buffers as bf16 (MXFP4 values are converted once a workgroup): a tile's
// rows are loaded into registers a whole tile ahead, 16 rows of one page a
// wave, and written while the tile before is in use; one barrier a tile.
//   S^T = K . Q^T and O^T = V^T . P^T on 32x32x16 MFMA: a lane owns one query,
// whose maximum and sum stay in it but for one exchange between the halves of
// the wave.
// What bounds it: the products (4 dim flops a pair of query and key) with the
// softmax on the vector units beside them.
#include <type_traits>

#include "kv_tiles.hpp"

namespace mr {

namespace {

constexpr int KP_ROWS = 128, KP_KEYS = 64;

template <int DP>
struct KvPromptLds {
    // rows read at one column (K) lie 16 bytes apart modulo all banks, the four rows
    // of a transposed read (V) 64 bytes
    static constexpr int K_STRIDE = DP + 8, V_STRIDE = DP + 32;
    static constexpr int K_SIZE = KP_KEYS * K_STRIDE, V_SIZE = KP_KEYS * V_STRIDE, BUF = K_SIZE + V_SIZE;
    static constexpr int BYTES = 2 * BUF * 2 + 64;
    static_assert(KP_ROWS * DP * 2 <= BYTES, "the output's tile fits");
};

// keys of tile index kb * 32 + 8 * (i / 4) + 4 * half + i % 4 are score i of block kb

template <int DP, bool MX>
__global__ void __launch_bounds__(256, DP == 256 ? 1 : 2) kv_prompt_kernel(KvAttnParams p) {
    using L = KvPromptLds<DP>;
    constexpr int KS = DP / 16, DB = DP / 32;
    extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
    int* flags = (int*)(lds + 2 * L::BUF);  // [2][4]: a wave's rows of the tile hold infinities or NaN
    const int l = threadIdx.x & 63, lq = l & 31, hh = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads_splits = p.kv_heads * p.splits;
    // the last tiles of a sequence, which have the most keys, go first
    const int tiles = gridDim.x / heads_splits;
    const int order = blockIdx.x / heads_splits, rest = blockIdx.x - order * heads_splits;
    const int split = rest / p.kv_heads, kv_head = rest - split * p.kv_heads;
    KvTile t;
    if (!kv_find<KP_ROWS>(p, tiles - 1 - order, t)) return;
    int kb = t.kbeg, ke = t.kend;
    if (p.splits > 1) {
        const int64_t at = (int64_t)t.kbeg + (int64_t)split * p.chunk;
        kb = (int)min(at, (int64_t)t.kend);
        if (split + 1 < p.splits) ke = (int)min(at + p.chunk, (int64_t)t.kend);
    }

    const KvRow row = kv_row(p, t, kv_head, t.first_row + 32 * w + lq);
    // keys that some, and that all of this wave's rows see
    const int w0 = t.first_row + 32 * w, i0 = min(w0 / p.group, t.qn - 1), i1 = min((w0 + 31) / p.group, t.qn - 1);
    const int pos0 = t.len - t.qn + i0, pos1 = t.len - t.qn + i1;
    const int wave_hi = w0 < t.qn * p.group ? min(max(pos1 + 1, 0), ke) : 0, all_hi = max(pos0 + 1, 0);
    const int wave_lo = p.window ? max(pos0 + 1 - p.window, 0) : 0, all_lo = p.window ? max(pos1 + 1 - p.window, 0) : 0;

    bf16x8 qf[KS];
    {
        const uint16_t* qp = p.q + row.token * p.q_ts + row.head * p.q_hs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 16 * s + 8 * hh;
            qf[s] = row.ok && d < p.dim ? *(const bf16x8*)(qp + d) : bf16x8{};
        }
    }
    float m_run = -INFINITY, l_part = 0.f;
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x16{};

    // wave w brings keys 16 w .. of each tile
    const int steps = (max(ke - kb, 0) + KP_KEYS - 1) / KP_KEYS;
    KvGroup<DP, MX> kreg, vreg;
    KvWalk walk;
    walk.start(p, t.b, steps ? kb + 16 * w : 0);
    int id = -1, off = 0, ahead = kb + 16 * w;  // the next group to load, its page
    auto look = [&]() {
        off = walk.offset;
        id = ahead < ke ? s_load(walk.entry) : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) walk.next(p.page_size);
    };
    bool have = false;
    int from = 0;
    auto load = [&]() {
        from = ahead;
        have = kv_page(p, id, ahead < ke);
        kv_load<DP, MX>(p, kv_head, id, off, have, l, kreg, vreg);
        ahead += KP_KEYS;
    };
    // what was loaded goes to buffer `to`
    auto put = [&](int to) {
        if (from + 16 > ke) kreg.cut(ke - from, l), vreg.cut(ke - from, l);
        uint16_t* kt = lds + to * L::BUF;
        kreg.put(kt + 16 * w * L::K_STRIDE, L::K_STRIDE, l);
        vreg.put(kt + L::K_SIZE + 16 * w * L::V_STRIDE, L::V_STRIDE, l);
        // bit 0: infinities or NaN; bit 1: the rows do not exist
        const int bad = (__builtin_amdgcn_ballot_w64(vreg.not_finite()) ? 1 : 0) | (have ? 0 : 2);
        if (l == 0) flags[4 * to + w] = bad;
    };

    const int tr_key = 4 * hh + ((l & 15) >> 2), tr_d = 16 * ((l >> 4) & 1) + 4 * (l & 3);
    auto tile = [&](auto masked_tag, const uint16_t* kt, const int* fl, int k0) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        const uint16_t* vt = kt + L::K_SIZE;
        f32x16 s[2] = {f32x16{}, f32x16{}};
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < KS; ++x)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const bf16x8 a = *(const bf16x8*)(kt + (32 * b + lq) * L::K_STRIDE + 16 * x + 8 * hh);
                s[b] = mfma32(a, qf[x], s[b]);
            }
        __builtin_amdgcn_s_setprio(0);
        float mx = -INFINITY;
        bool apart = false;
        uint32_t gone = 0;  // bit per group of 16 keys
        if constexpr (MASKED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int f = __builtin_amdgcn_readfirstlane(fl[i]);
                apart |= (f & 1) != 0;
                gone |= (f & 2 ? 1u : 0u) << i;
            }
        }
        const int hi = min(row.hi, ke) - k0 - 4 * hh, lo = row.lo - k0 - 4 * hh;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int at = 32 * b + 8 * (i >> 2) + (i & 3);  // + 4 hh
                if (MASKED && (at >= hi || at < lo || (gone >> (at >> 4) & 1))) s[b][i] = -INFINITY;
                mx = fmaxf(mx, s[b][i]);
            }
        mx = xor32_max(mx) * p.scale_log2;  // (the scale is positive)
        const bool raise = mx > m_run + KV_TAU;
        if (__builtin_amdgcn_ballot_w64(raise)) {
            const float up = raise ? mx : m_run;
            const float alpha = raise ? __builtin_amdgcn_exp2f(m_run - up) : 1.f;
            m_run = up;
            l_part *= alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= alpha;
        }
        const float ref = m_run == -INFINITY ? 0.f : m_run;  // (no key yet: every score is -inf)
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[b][i], p.scale_log2, -ref));
                s[b][i] = e;
                ls[i & 3] += e;
            }
        l_part += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        auto values = [&](int x, int d) {
            const uint16_t* at = vt + (16 * x + tr_key) * L::V_STRIDE + 32 * d + tr_d;
            const bf16x4 a = ds_read_tr16(at), b = ds_read_tr16(at + 8 * L::V_STRIDE);
            return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        };
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            bf16x8 pb;
#pragma unroll
            for (int e = 0; e < 8; ++e) pb[e] = (__bf16)s[x >> 1][8 * (x & 1) + e];
            if (!MASKED || !apart) {
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = mfma32(values(x, d), pb, o[d]);
            } else {
                // one key at a time, added where it is seen
                if (gone >> x & 1) continue;
                for (int key = 0; key < 16; ++key) {
                    const int at = 16 * x + key - 4 * hh;
                    const bool mine = at < hi && at >= lo;
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        bf16x8 a = values(x, d);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (8 * (e >> 2) + 4 * hh + (e & 3) != key) a[e] = (__bf16)0.f;
                        const f32x16 one = mfma32(a, pb, f32x16{});
                        if (mine) o[d] += one;
                    }
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
    };

    if (steps > 0) {
        look();
        load();
        look();
        put(0);
        if (steps > 1) {
            load();
            look();
        }
        __syncthreads();
        for (int i = 0; i < steps; ++i) {
            if (i + 1 < steps) put((i + 1) & 1);
            if (i + 2 < steps) {
                load();
                look();
            }
            const int k0 = kb + KP_KEYS * i;
            const uint16_t* kt = lds + (i & 1) * L::BUF;
            const int* fl = flags + 4 * (i & 1);
            if (k0 < wave_hi && k0 + KP_KEYS > wave_lo) {
                const bool whole = (__builtin_amdgcn_readfirstlane((fl[0] | fl[1]) | (fl[2] | fl[3])) & 2) == 0;
                if (whole && k0 >= all_lo && k0 + KP_KEYS <= min(all_hi, ke))
                    tile(std::false_type{}, kt, fl, k0);
                else
                    tile(std::true_type{}, kt, fl, k0);
            }
            __syncthreads();
        }
    }

    float total = xor32_sum(l_part);
    const int64_t at = (int64_t)row.token * (p.kv_heads * p.group) + row.head;
    if (p.splits > 1) {
        if (!row.ok) return;
        if (hh == 0) {
            float* ml = p.part_ml + 2 * (at * p.splits + split);
            ml[0] = m_run;
            ml[1] = total;
        }
        if (total == 0.f) return;
        float* to = p.part_o + (at * p.splits + split) * p.dim;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 32 * d + 8 * i + 4 * hh;
                if (c < p.dim) *(f32x4*)(to + c) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            }
        return;
    }
    float top = m_run, was = 1.f;
    if (p.sinks && row.ok) {
        const float sink = p.sinks[row.head] * 1.4426950408889634f;
        top = fmaxf(m_run, sink);
        was = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - top);
        if (top != -INFINITY) total = fmaf(total, was, __builtin_amdgcn_exp2f(sink - top));
    }
    const float inv = total == 0.f ? 0.f : was / total;  // (no key is seen: zeros)
    if (p.lse && row.ok && hh == 0)
        p.lse[at] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
    if (p.out_f32) {
        if (!row.ok) return;
        float* to = (float*)p.out + row.token * p.out_ts + row.head * p.out_hs;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 32 * d + 8 * i + 4 * hh;
                if (c < p.dim)
                    *(f32x4*)(to + c) = f32x4{o[d][4 * i] * inv, o[d][4 * i + 1] * inv, o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv};
            }
        return;
    }
    // bf16: the wave's 32 rows through its part of LDS (free since the last barrier),
    // 16-byte piece c of row r at c ^ (r & 7), then whole rows
    uint16_t* st = lds + w * 32 * DP;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *(u32x2*)(st + lq * DP + (((4 * d + i) ^ (lq & 7)) << 3) + 4 * hh) =
                u32x2{pack_bf16x2_hw(o[d][4 * i] * inv, o[d][4 * i + 1] * inv),
                      pack_bf16x2_hw(o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv)};
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    constexpr int PIECES = DP / 8;
#pragma unroll
    for (int i = 0; i < 32 * PIECES / 64; ++i) {
        const int x = l + 64 * i, r = x / PIECES, c = x % PIECES;
        const KvRow to = kv_row(p, t, kv_head, w0 + r);
        const u32x4 v = *(const u32x4*)(st + r * DP + ((c ^ (r & 7)) << 3));
        if (to.ok && 8 * c < p.dim)
            *(u32x4*)((uint16_t*)p.out + to.token * p.out_ts + to.head * p.out_hs + 8 * c) = v;
    }
}

template <int DP, bool MX>
hipError_t prompt_launch(const KvAttnParams& p, unsigned grid, hipStream_t st) {
    const void* f = (const void*)kv_prompt_kernel<DP, MX>;
    constexpr int bytes = KvPromptLds<DP>::BYTES;
    const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((kv_prompt_kernel<DP, MX>), dim3(grid), dim3(256), bytes, st, p);
    return hipGetLastError();
}

template <bool MX>
hipError_t prompt_dim(const KvAttnParams& p, unsigned grid, hipStream_t st) {
    if (p.dim <= 64) return prompt_launch<64, MX>(p, grid, st);
    if (p.dim <= 128) return prompt_launch<128, MX>(p, grid, st);
    return prompt_launch<256, MX>(p, grid, st);
}

}  // namespace

hipError_t launch_kv_prompt(const KvAttnParams& p, unsigned grid, hipStream_t st) {
    return p.k_scales ? prompt_dim<true>(p, grid, st) : prompt_dim<false>(p, grid, st);
}

}  // namespace mr
