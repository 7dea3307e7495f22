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

// Every wave's LDS traffic is done; loads into registers stay in flight.  (The
// builtin tells the compiler that earlier LDS reads have landed.)
__device__ __forceinline__ void kp_barrier() {
    __builtin_amdgcn_s_waitcnt(0xC07F);
    lds_barrier();
}

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
    using Group = KvGroup<DP, MX>;
    const typename Group::At at = Group::at(p.dim, l);
    Group kreg, vreg;
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
        have = kv_page(p, id);
        kv_load<DP, MX>(p, kv_head, id, off, at, kreg, vreg);
        ahead += KP_KEYS;
    };
    // what was loaded goes to buffer `to`; flags say of the wave's 16 rows, in bit 0,
    // that infinities or NaN among their values were left out (where not every row of the
    // workgroup sees the tile), in bit 1 that their page does not exist
    auto put = [&](int to) {
        if (from + 16 > ke || !have) vreg.cut(have ? ke - from : 0, l);
        if (p.dim < DP) kreg.narrow(at), vreg.narrow(at);
        uint16_t* kt = lds + to * L::BUF;
        const int k0 = from - 16 * w;
        const bool apart = (k0 < t.all_lo || k0 + KP_KEYS > t.all_hi) && __builtin_amdgcn_ballot_w64(vreg.not_finite()) != 0;
        kreg.put(kt + 16 * w * L::K_STRIDE, L::K_STRIDE, l);
        if (apart)
            vreg.template put<true>(kt + L::K_SIZE + 16 * w * L::V_STRIDE, L::V_STRIDE, l);
        else
            vreg.put(kt + L::K_SIZE + 16 * w * L::V_STRIDE, L::V_STRIDE, l);
        if (l == 0) flags[4 * to + w] = (apart ? 1 : 0) | (have ? 0 : 2);
    };

    const int tr_key = 4 * hh + ((l & 15) >> 2), tr_d = 16 * ((l >> 4) & 1) + 4 * (l & 3);
    // one tile for this wave's 32 rows; masked: not every row sees every key (a branch
    // around the masking alone: two forms of the whole cost 40 spilled registers)
    auto tile = [&](bool masked, const uint16_t* kt, int gone, int k0) {
        const uint16_t* vt = kt + L::K_SIZE;
        f32x16 s[2] = {f32x16{}, f32x16{}};
        // operands come in two sets, so that one's reads overlap the other's products
        // (the fences keep the scheduler from reading them all at once)
        bf16x8 ka[2][4];
        auto keys = [&](int x, bf16x8(&a)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                a[e] = *(const bf16x8*)(kt + (32 * (e & 1) + lq) * L::K_STRIDE + 32 * x + 16 * (e >> 1) + 8 * hh);
        };
        keys(0, ka[0]);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < KS / 2; ++x) {
            if (x + 1 < KS / 2) keys(x + 1, ka[(x + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e & 1] = mfma32(ka[x & 1][e], qf[2 * x + (e >> 1)], s[e & 1]);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        float mx = -INFINITY;
        if (masked) {
            const int hi = min(row.hi, ke) - k0 - 4 * hh, lo = row.lo - k0 - 4 * hh;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int at = 32 * b + 8 * (i >> 2) + (i & 3);  // + 4 hh
                    if (at >= hi || at < lo || (gone >> (at >> 4) & 1)) s[b][i] = -INFINITY;
                }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
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
        __builtin_amdgcn_s_setprio(1);
        // DB blocks of 32 dims of 16 keys, in two sets of at most four
        constexpr int VB = DB < 4 ? DB : 4, VN = 4 * (DB / VB);
        bf16x8 va[2][VB];
        auto values = [&](int x, bf16x8(&a)[VB]) {
            const uint16_t* at = vt + (16 * (x & 3) + tr_key) * L::V_STRIDE + 32 * VB * (x >> 2) + tr_d;
#pragma unroll
            for (int d = 0; d < VB; ++d) {
                const bf16x4 u = ds_read_tr16(at + 32 * d), v = ds_read_tr16(at + 32 * d + 8 * L::V_STRIDE);
                a[d] = bf16x8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
            }
        };
        values(0, va[0]);
#pragma unroll
        for (int x = 0; x < VN; ++x) {
            if (x + 1 < VN) values(x + 1, va[(x + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
            bf16x8 pb;
#pragma unroll
            for (int e = 0; e < 8; ++e) pb[e] = (__bf16)s[(x & 3) >> 1][8 * (x & 1) + e];
#pragma unroll
            for (int d = 0; d < VB; ++d) o[VB * (x >> 2) + d] = mfma32(va[x & 1][d], pb, o[VB * (x >> 2) + d]);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
    };

    int apart_from = ke, apart_to = 0;  // keys whose infinite values were left out
    if (steps > 0) {
        look();
        load();
        look();
        put(0);
        if (steps > 1) {
            load();
            look();
        }
        kp_barrier();
        for (int i = 0; i < steps; ++i) {
            if (i + 1 < steps) put((i + 1) & 1);
            if (i + 2 < steps) {
                load();
                look();
            }
            const int k0 = kb + KP_KEYS * i;
            const uint16_t* kt = lds + (i & 1) * L::BUF;
            if (k0 < wave_hi && k0 + KP_KEYS > wave_lo) {
                // (four flags of two bits)
                const u32x4 f = *(const u32x4*)(flags + 4 * (i & 1));
                const int fl = __builtin_amdgcn_readfirstlane((int)(f[0] | f[1] << 2 | f[2] << 4 | f[3] << 6));
                const int gone = (fl >> 1 & 1) | (fl >> 2 & 2) | (fl >> 3 & 4) | (fl >> 4 & 8);
                tile(gone || k0 < all_lo || k0 + KP_KEYS > min(all_hi, ke), kt, gone, k0);
                if (fl & 0x55) apart_to = k0 + KP_KEYS, apart_from = min(apart_from, k0);
            }
            kp_barrier();
        }
    }

    for (int key = apart_from; key < min(apart_to, ke); ++key)
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                kv_add_infinite<MX>(p, t.b, kv_head, key, key >= row.lo && key < row.hi, 32 * d + 8 * c + 4 * hh,
                                    [&](int j, float v) { o[d][4 * c + j] += v; });

    float total = xor32_sum(l_part);
    const int64_t place = (int64_t)row.token * (p.kv_heads * p.group) + row.head;
    if (p.splits > 1) {
        if (!row.ok) return;
        if (hh == 0) {
            float* ml = p.part_ml + 2 * (place * p.splits + split);
            ml[0] = m_run;
            ml[1] = total;
        }
        if (total == 0.f) return;
        float* to = p.part_o + (place * p.splits + split) * p.dim;
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
        p.lse[place] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
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
