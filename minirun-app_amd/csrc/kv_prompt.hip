// Attention of many queries of a sequence over a paged cache (kv_attention.hip
// has the formula, the small form and what is shared).
//
// A workgroup of eight waves has 256 (query, head) rows of one sequence and key
// head (four waves and 128 rows for heads of more than 128 dims, whose sums take
// twice the registers), heads of a query next to each other, so that a tile spans few
// positions and all heads of a group share the keys.  Tiles of 64 keys come through
// two LDS buffers as bf16: rows are loaded into registers a whole tile ahead of their
// way to LDS, 16 rows of keys or values of one page a wave.
//   S^T = K . Q^T and O^T = V^T . P^T on 32x32x16 MFMA: a lane owns one query,
// whose maximum and sum stay in it but for one exchange between the halves of
// the wave.
// What bounds it: the products (4 dim flops a pair of query and key) and, beside
// them, the softmax and the conversions on the vector units and the way of operands from
// LDS, each of which is about half busy.  An exp2 and a conversion of two MXFP4 values
// take 16 clocks of a wave's vector unit, other instructions 4: for a wave's 32 products
// of 32 clocks a tile, 32 exp2, about 120 others and 16 conversions.  (With four waves a
// workgroup every wave has 32 of these, which cost 44 us of 230.)  Two waves a SIMD alone
// ran products and softmax one after the other, so a wave's own are interleaved: while the
// products of the next tile's scores run, the scores of this one become probabilities, and
// while its values are multiplied, the next scores' maximum is found and rows go to LDS.
// So keys are a tile ahead of values, and one barrier ends a tile.
//   Measured: 4096 queries of 32 heads behind 1000 keys, 4 key heads of 128 in MXFP4,
// 199 us, 1.03 PFLOP/s (4-wave workgroups 245 without and 231 with the interleaving).  Keys
// as codes on the scaled matrix instructions, a quarter of the LDS reads for keys and no
// conversion of them, took 200.
#include <type_traits>

#include "kv_tiles.hpp"

namespace mr {

namespace {

constexpr int KP_KEYS = 64;
constexpr int kp_waves(int dp) { return dp == 256 ? 4 : 8; }

template <int DP>
struct KvPromptLds {
    // rows read at one column (K) lie 16 bytes apart modulo all banks, the four rows
    // of a transposed read (V) 64 bytes
    static constexpr int K_STRIDE = DP + 8, V_STRIDE = DP + 32;
    static constexpr int K_SIZE = KP_KEYS * K_STRIDE, V_SIZE = KP_KEYS * V_STRIDE;
    static constexpr int V_AT = 2 * K_SIZE, FLAGS_AT = V_AT + 2 * V_SIZE;  // two buffers of each
    static constexpr int BYTES = FLAGS_AT * 2 + 16;
    static_assert(32 * kp_waves(DP) * DP * 2 <= BYTES, "the output's tile fits");
};

// Every wave's LDS traffic is done; loads into registers stay in flight.  (The
// builtin tells the compiler that earlier LDS reads have landed.)
__device__ __forceinline__ void kp_barrier() {
    __builtin_amdgcn_s_waitcnt(0xC07F);
    lds_barrier();
}

// score e of block b (32 keys) is key 32 b + 8 (e / 4) + 4 hh + e % 4 of its tile

template <int DP, bool MX>
__global__ void __launch_bounds__(64 * kp_waves(DP), kp_waves(DP) / 4) kv_prompt_kernel(KvAttnParams p) {
    using L = KvPromptLds<DP>;
    constexpr int W = kp_waves(DP), KP_ROWS = 32 * W, KS = DP / 16, DB = DP / 32;
    extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
    // a byte per 16 rows and buffer, of keys and of values: their page does not exist, or
    // infinities or NaN were left out of them
    uint8_t* const key_flags = (uint8_t*)(lds + L::FLAGS_AT);
    uint8_t* const value_flags = key_flags + 8;
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

    const KvRow own = kv_row(p, t, kv_head, t.first_row + 32 * w + lq);
    // keys that all of this wave's rows see
    const int w0 = t.first_row + 32 * w, i0 = min(w0 / p.group, t.qn - 1), i1 = min((w0 + 31) / p.group, t.qn - 1);
    const int pos0 = t.len - t.qn + i0, pos1 = t.len - t.qn + i1;
    const int all_hi = min(max(pos0 + 1, 0), ke), all_lo = p.window ? max(pos1 + 1 - p.window, 0) : 0;

    bf16x8 qf[KS];
    {
        const uint16_t* qp = p.q + own.token * p.q_ts + own.head * p.q_hs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 16 * s + 8 * hh;
            qf[s] = own.ok && d < p.dim ? *(const bf16x8*)(qp + d) : bf16x8{};
        }
    }
    float m_run = -INFINITY, l_part = 0.f;
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x16{};

    // Tiles go by twos (a last one may have no keys), so that no branch divides the
    // accumulators' way.
    const int steps = (max(ke - kb, 0) + 2 * KP_KEYS - 1) / (2 * KP_KEYS) * 2;
    // Wave w brings 16 keys, w % 4, of each tile: their keys or their values, or both in
    // turn (TASKS).
    constexpr int TASKS = 8 / W;
    using Group = KvGroup<DP, MX>;
    const typename Group::At at = Group::at(p.dim, l);
    const int part16 = w & 3;
    struct Rows {
        Group v;
        int from;   // the first row's key
        bool have;  // their page exists
        KvWalk walk;
        int ahead, id;  // the next tile's first key, its page
        KvFrom next;    // and where it is
        bool next_have;
    };
    Rows task[TASKS];
    auto is_values = [&](int j) { return TASKS == 1 ? w >= 4 : j == 1; };  // (wave-uniform)
    auto look = [&](Rows& r) { r.id = r.ahead < ke ? s_load(r.walk.entry) : -1; };
    // the next tile's place, and a look at the one after it; then its rows.  (Tiles past
    // the last read page 0.)
    auto prepare = [&](int j) {
        Rows& r = task[j];
        r.next = kv_from<MX>(p, !is_values(j), kv_head, r.id, r.walk.offset);
        r.next_have = kv_page(p, r.id);
        r.ahead += KP_KEYS;
        r.walk.next();
        look(r);
    };
    auto load = [&](int j) {
        Rows& r = task[j];
        r.from = r.ahead - KP_KEYS;
        r.have = r.next_have;
        r.v.load(r.next, at);
    };
    // rows of values lie 64 bytes apart modulo all banks, as a lane's blocks do: four rows'
    // lanes take other quarters of them (KvGroup::turn)
    auto turned = [&](int j) { return is_values(j) ? Group::row(l, 0) & 3 : 0; };
    // what is left to do to loaded rows before they go to a buffer (rarely more)
    auto ready = [&](int j, int buffer) {
        Rows& r = task[j];
        if (p.dim < DP) r.v.narrow(at);
        uint32_t flag = r.have ? 0 : 1;
        if (is_values(j)) {
            if (r.from + 16 > ke || !r.have) r.v.cut(r.have ? ke - r.from : 0, l);
            const int k0 = r.from - 16 * part16;
            flag = 0;
            if (k0 < t.all_lo || k0 + KP_KEYS > t.all_hi) {  // not every row of the workgroup sees the tile
                flag = __builtin_amdgcn_ballot_w64(r.v.not_finite()) != 0;
                if (flag) r.v.clean();
            }
        }
        if (l == 0) (is_values(j) ? value_flags : key_flags)[4 * buffer + part16] = (uint8_t)flag;
        r.v.turn(turned(j));
    };
    // a quarter of them, or all, to the buffer
    auto put = [&](int j, int buffer, int part) {
        uint16_t* to = lds + (is_values(j) ? L::V_AT + buffer * L::V_SIZE + 16 * part16 * L::V_STRIDE
                                           : buffer * L::K_SIZE + 16 * part16 * L::K_STRIDE);
        task[j].v.put_part(to, is_values(j) ? L::V_STRIDE : L::K_STRIDE, l, part, turned(j));
    };
    auto put_all = [&](int j, int buffer) {
        ready(j, buffer);
#pragma unroll
        for (int x = 0; x < 4; ++x) put(j, buffer, x);
    };

    // operands: keys 32 b + lq of a buffer, dims 16 x + 8 hh ..; values of 16 keys, four
    // blocks (or all) of 32 dims
    constexpr int VB = DB < 4 ? DB : 4, VN = 4 * (DB / VB);
    const int tr_key = 4 * hh + ((l & 15) >> 2), tr_d = 16 * ((l >> 4) & 1) + 4 * (l & 3);
    auto keys = [&](int buffer, int x, bf16x8(&a)[2]) {
        const uint16_t* from = lds + buffer * L::K_SIZE + lq * L::K_STRIDE + 16 * x + 8 * hh;
        a[0] = *(const bf16x8*)from;
        a[1] = *(const bf16x8*)(from + 32 * L::K_STRIDE);
    };
    auto values = [&](int buffer, int x, bf16x8(&a)[VB]) {
        const uint16_t* from = lds + L::V_AT + buffer * L::V_SIZE + (16 * (x & 3) + tr_key) * L::V_STRIDE +
                               32 * VB * (x >> 2) + tr_d;
#pragma unroll
        for (int d = 0; d < VB; ++d) {
            const bf16x4 lo = ds_read_tr16(from + 32 * d), hi = ds_read_tr16(from + 32 * d + 8 * L::V_STRIDE);
            a[d] = bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
    };
    // scores that a row does not see become -inf; tile `i`, its keys' flags
    auto mask = [&](int i, int flags, f32x16(&s)[2]) {
        const int k0 = kb + KP_KEYS * i;
        const uint32_t f = __builtin_amdgcn_readfirstlane(flags);
        if (!f && k0 >= all_lo && k0 + KP_KEYS <= all_hi) return;
        int hi = min(own.hi, ke) - k0 - 4 * hh, lo = own.lo - k0 - 4 * hh;
        asm volatile("" : "+v"(hi), "+v"(lo));  // (behind the branch, not 64 compares a tile)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int key = 32 * b + 8 * (e >> 2) + (e & 3);  // + 4 hh
                if (key >= hi || key < lo || (f >> (8 * (key >> 4)) & 1)) s[b][e] = -INFINITY;
            }
    };

    int apart_from = ke, apart_to = 0;  // keys whose infinite values were left out
    float mx = -INFINITY;               // of the tile in turn, this lane's 32 scores
    // Tile i: its scores are s, its values in buffer B, the next one's keys in B ^ 1.
    // Leaves the next tile's scores in n and their maximum in mx, keys i + 2 and values
    // i + 1 in LDS, keys i + 3 and values i + 2 under way.
    auto buffer_of = [&](int j, int B) { return is_values(j) ? B ^ 1 : B; };
    auto tile = [&](auto buffer_tag, int i, f32x16(&s)[2], f32x16(&n)[2]) {
        constexpr int B = decltype(buffer_tag)::value;
        const float top = xor32_max(mx) * p.scale_log2;  // (the scale is positive)
        const bool raise = top > m_run + KV_TAU;
        if (__builtin_amdgcn_ballot_w64(raise)) {
            const float up = raise ? top : m_run;
            const float alpha = raise ? __builtin_amdgcn_exp2f(m_run - up) : 1.f;
            m_run = up;
            l_part *= alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= alpha;
        }
        const float ref = m_run == -INFINITY ? 0.f : m_run;  // (no key yet: every score is -inf)
        const int k0 = kb + KP_KEYS * i;
        if (k0 < t.all_lo || k0 + KP_KEYS > t.all_hi)  // (else no values were left out)
            if (__builtin_amdgcn_readfirstlane(*(const int*)(value_flags + 4 * B)))
                apart_to = k0 + KP_KEYS, apart_from = min(apart_from, k0);
        const int flags = *(const int*)(key_flags + 4 * (B ^ 1));  // (used after the products)

        // (the fences keep each product's share of the other work beside it)
        bf16x8 ka[2][2];
        u32x4 pb[4];  // probabilities as bf16: word e / 2 % 4 of the 16 keys e / 8
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
        keys(B ^ 1, 0, ka[0]);
#pragma unroll
        for (int x = 0; x < KS; ++x) {
            if (x + 1 < KS) keys(B ^ 1, x + 1, ka[(x + 1) & 1]);
            if (x < TASKS) prepare(x);
#pragma unroll
            for (int b = 0; b < 2; ++b) n[b] = mfma32(ka[x & 1][b], qf[x], x ? n[b] : f32x16{});
#pragma unroll
            for (int e = 32 * x / KS; e < 32 * (x + 1) / KS; e += 2) {
                const float y = __builtin_amdgcn_exp2f(fmaf(s[e >> 4][e & 15], p.scale_log2, -ref));
                const float z = __builtin_amdgcn_exp2f(fmaf(s[e >> 4][(e & 15) + 1], p.scale_log2, -ref));
                ls[e & 3] += y;
                ls[(e & 3) + 1] += z;
                uint32_t two = pack_bf16x2_hw(y, z);
                asm volatile("" : "+v"(two));  // (here, not where it is used)
                pb[e >> 3][e >> 1 & 3] = two;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l_part += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        mask(i + 1, flags, n);
#pragma unroll
        for (int j = 0; j < TASKS; ++j) ready(j, buffer_of(j, B));
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        bf16x8 va[2][VB];
        values(B, 0, va[0]);
#pragma unroll
        for (int x = 0; x < VN; ++x) {
            if (x + 1 < VN) values(B, x + 1, va[(x + 1) & 1]);
#pragma unroll
            for (int d = 0; d < VB; ++d) o[VB * (x >> 2) + d] = mfma32(va[x & 1][d], __builtin_bit_cast(bf16x8, pb[x & 3]), o[VB * (x >> 2) + d]);
            if (x < 4) {
#pragma unroll
                for (int j = 0; j < TASKS; ++j) put(j, buffer_of(j, B), x);
#pragma unroll
                for (int e = 8 * x; e < 8 * x + 8; ++e) m4[e & 3] = fmaxf(m4[e & 3], n[e >> 4][e & 15]);
                asm volatile("" : "+v"(m4[0]), "+v"(m4[1]), "+v"(m4[2]), "+v"(m4[3]));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
#pragma unroll
        for (int j = 0; j < TASKS; ++j) load(j);
        kp_barrier();
    };

    if (steps > 0) {
        // keys 0 and 1 and values 0 go to their buffers, keys 2 and values 1 are under way
#pragma unroll
        for (int j = 0; j < TASKS; ++j) {
            Rows& r = task[j];
            r.ahead = kb + 16 * part16;
            r.walk.start(p, t.b, r.ahead, KP_KEYS);
            look(r);
            prepare(j);
            load(j);
        }
#pragma unroll
        for (int j = 0; j < TASKS; ++j) {
            put_all(j, 0);
            prepare(j);
            load(j);
            if (!is_values(j)) {
                put_all(j, 1);
                prepare(j);
                load(j);
            }
        }
        kp_barrier();
        if (w0 >= t.qn * p.group) {
            // a wave without rows of its own only brings the others' keys and values
            kp_barrier();
            for (int i = 0; i < steps; ++i) {
#pragma unroll
                for (int j = 0; j < TASKS; ++j) {
                    put_all(j, buffer_of(j, i & 1));
                    prepare(j);
                    load(j);
                }
                kp_barrier();
            }
        } else {
            f32x16 s[2] = {f32x16{}, f32x16{}}, n[2];
            bf16x8 a[2];
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                keys(0, x, a);
#pragma unroll
                for (int b = 0; b < 2; ++b) s[b] = mfma32(a[b], qf[x], s[b]);
            }
            mask(0, *(const int*)key_flags, s);
#pragma unroll
            for (int e = 0; e < 32; ++e) mx = fmaxf(mx, s[e >> 4][e & 15]);
            kp_barrier();
            for (int i = 0; i < steps; i += 2) {
                tile(std::integral_constant<int, 0>{}, i, s, n);
                tile(std::integral_constant<int, 1>{}, i + 1, n, s);
            }
        }
    }

    const float total = xor32_sum(l_part);
    // infinities and NaN (kv_add_infinite): dims that are NaN begin again from 0
    float any[4] = {};  // (NaN if a dim is, or if some are infinities of both signs)
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) any[e & 3] += o[d][e];
    const float z = (any[0] + any[1]) + (any[2] + any[3]);
    const bool nan = z != z && own.hi > 0 && total == total;
    const bool again = __builtin_amdgcn_ballot_w64(nan) != 0;
    bool left = again;
    uint32_t lost[DB] = {};  // these dims, a bit each
    if (__builtin_expect(again, 0)) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (nan && o[d][e] != o[d][e]) lost[d] |= 1u << e, o[d][e] = 0.f;
    }
    kv_each_infinite<DP, MX>(
        p, t.b, kv_head, again ? kb : apart_from, again ? ke : min(apart_to, ke), l,
        [&](int k0) { return left || (k0 >= apart_from && k0 < apart_to); },
        [&](int first, int last) {
            for (int key = first; key < last; ++key)
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        kv_add_infinite<MX>(p, t.b, kv_head, key, key >= own.lo && key < own.hi, 32 * d + 8 * c + 4 * hh,
                                            [&](int j, float v) { o[d][4 * c + j] += v; });
            if (!left) return;
            bool more = false;  // dims that are not NaN again
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) more = more || ((lost[d] >> e & 1) && o[d][e] == o[d][e]);
            left = __builtin_amdgcn_ballot_w64(more) != 0;
        });
    if (__builtin_expect(again, 0)) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e)  // (sums of finite values that left f32's range)
                if ((lost[d] >> e & 1) && __builtin_fabsf(o[d][e]) < INFINITY) o[d][e] = __builtin_nanf("");
    }

    auto mine = [&]() {  // this lane's row, found again rather than kept in registers
        int at = lq;
        asm volatile("" : "+v"(at));
        return kv_row(p, t, kv_head, t.first_row + 32 * w + at);
    };
    if (p.splits > 1) {
        const KvRow row = mine();
        if (!row.ok) return;
        const int64_t place = (int64_t)row.token * (p.kv_heads * p.group) + row.head;
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
    int head = 0;
    if (p.sinks) {
        const KvRow row = mine();
        head = row.ok ? row.head : 0;
    }
    const KvEnd end = kv_end(m_run, total, p.sinks, head);
    const float inv = end.inv;
    if (total == 0.f)
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = f32x16{};  // (0 times an infinity is not)
    if (__builtin_expect(inv != 0.f, 1)) {
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= inv;
    } else {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = kv_weighted(o[d][e], inv);
    }
    if (p.lse && hh == 0) {
        const KvRow row = mine();
        if (row.ok) p.lse[(int64_t)row.token * (p.kv_heads * p.group) + row.head] = end.lse;
    }
    if (p.out_f32) {
        const KvRow row = mine();
        if (!row.ok) return;
        float* to = (float*)p.out + row.token * p.out_ts + row.head * p.out_hs;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 32 * d + 8 * i + 4 * hh;
                if (c < p.dim)
                    *(f32x4*)(to + c) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
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
                u32x2{pack_bf16x2_hw(o[d][4 * i], o[d][4 * i + 1]), pack_bf16x2_hw(o[d][4 * i + 2], o[d][4 * i + 3])};
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
    hipLaunchKernelGGL((kv_prompt_kernel<DP, MX>), dim3(grid), dim3(64 * kp_waves(DP)), bytes, st, p);
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
