// What the two kernels of attention over a paged cache share: which rows and
// keys a workgroup has, and the way of 16 keys of a page into its registers.
//
// A tile's rows are (query, head) pairs of one sequence and one key head: row
// r is query r / group and the group's head r % group.  Query i of a sequence
// of n queries and `len` keys sits at position len - n + i and sees the keys
// up to there, or the last `window` of them.
#pragma once

#include "mr_kernels.hpp"

namespace mr {

constexpr float KV_TAU = 8.f;  // log2 headroom of the running maximum: sums are rescaled when a score passes it

struct KvTile {
    int b, q0, qn, len;  // sequence, its first query, queries and keys
    int first_row;
    int kbeg, kend;      // keys that some row sees (kbeg a multiple of 16); none: kbeg >= kend
    int all_lo, all_hi;  // keys that every row sees
};

// int32 read through the scalar cache (nothing in these kernels writes them)
__device__ __forceinline__ int s_load(const int32_t* p) {
    return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
}

__device__ __forceinline__ int kv_queries(const KvAttnParams& p, int b, int& q0) {
    q0 = p.q_offsets[b];
    const int q1 = p.q_offsets[b + 1];
    return q0 >= 0 && q1 <= p.tokens && q1 > q0 ? q1 - q0 : 0;
}

// The tile `tile` of all sequences' tiles of ROWS rows; false: there is no such.
template <int ROWS>
__device__ __forceinline__ bool kv_find(const KvAttnParams& p, int tile, KvTile& t) {
    if (!p.q_offsets) {
        const int per = (p.group + ROWS - 1) / ROWS;
        t.b = tile / per;
        t.first_row = (tile - t.b * per) * ROWS;
        t.q0 = t.b;
        t.qn = 1;
    } else {
        // lanes count the tiles of 64 sequences, a scan finds the one that has this tile.  (A
        // search over places with room for any offsets needs no scan, but leaves gaps that
        // fall on the same XCDs: 256 sequences of 2 x 8 rows 20 us so, 30 with the search,
        // 1024 90 and 103; from some 2000 on the scan is the slower one, 4096 115 and 51.)
        const int l = threadIdx.x & 63;
        uint32_t left = (uint32_t)tile;
        int at = -1;
        for (int b0 = 0; b0 < p.batch; b0 += 64) {
            uint32_t n = 0;
            int q0;
            if (b0 + l < p.batch) n = ((uint32_t)kv_queries(p, b0 + l, q0) * (uint32_t)p.group + ROWS - 1) / ROWS;
            const uint32_t end = wave_scan_incl(n), all = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
            if (left < all) {
                const int i = __builtin_ctzll(__builtin_amdgcn_ballot_w64(end > left));
                left -= (uint32_t)__builtin_amdgcn_readlane((int)(end - n), i);
                at = b0 + i;
                break;
            }
            left -= all;
        }
        if (at < 0) return false;
        t.b = at;
        const int q0 = s_load(p.q_offsets + at), q1 = s_load(p.q_offsets + at + 1);
        t.q0 = q0;
        t.qn = q1 - q0;
        if (left >= ((uint32_t)t.qn * (uint32_t)p.group + ROWS - 1) / ROWS) return false;
        t.first_row = (int)left * ROWS;
    }
    t.len = min(max(s_load(p.lens + t.b), 0), p.max_keys);
    const int i0 = t.first_row / p.group, i1 = min((t.first_row + ROWS - 1) / p.group, t.qn - 1);
    const int p0 = t.len - t.qn + i0, p1 = t.len - t.qn + i1;  // positions of the first and the last query
    t.kend = max(p1 + 1, 0);
    t.all_hi = max(p0 + 1, 0);
    t.kbeg = p.window ? max(p0 + 1 - p.window, 0) & ~15 : 0;
    t.all_lo = p.window ? max(p1 + 1 - p.window, 0) : 0;
    return true;
}

// A row's keys [lo, hi), and where its query, output and sink are
struct KvRow {
    bool ok;
    int token, head, lo, hi;
};
__device__ __forceinline__ KvRow kv_row(const KvAttnParams& p, const KvTile& t, int kv_head, int row) {
    KvRow r;
    const int i = row / p.group;
    r.ok = i < t.qn;
    r.token = t.q0 + min(i, t.qn - 1);
    r.head = kv_head * p.group + row - i * p.group;
    const int pos = t.len - t.qn + i;
    r.hi = r.ok ? max(pos + 1, 0) : 0;
    r.lo = p.window ? max(pos + 1 - p.window, 0) : 0;
    return r;
}

// What a row's sums come to with its head's sink (sinks null: none): the factor of its output
// and the logarithm, from the running maximum of its scores in base 2 and their sum.  The sink
// is met in natural units, since it may be any f32 and many would leave f32 in base 2.
struct KvEnd {
    float inv, lse;
};
__device__ __forceinline__ KvEnd kv_end(float top, float total, const float* sinks, int head) {
    constexpr float LN2 = 0.6931471805599453f, LOG2E = 1.4426950408889634f;
    if (!sinks) return total == 0.f ? KvEnd{0.f, -INFINITY} : KvEnd{1.f / total, (top + __builtin_amdgcn_logf(total)) * LN2};
    const float sink = sinks[head];
    if (total == 0.f) return KvEnd{0.f, sink};  // no key is seen, or none with a score above -inf: zeros
    const float m = top * LN2, up = fmaxf(m, sink);
    const float was = __builtin_amdgcn_exp2f((m - up) * LOG2E);
    const float all = fmaf(total, was, __builtin_amdgcn_exp2f((sink - up) * LOG2E));
    return KvEnd{was / all, up + __builtin_amdgcn_logf(all) * LN2};
}

// The groups of 16 keys of a sequence, one after another: a page holds a whole
// number of them.  Wave-uniform.
struct KvWalk {
    const int32_t* entry;  // of the page table
    int offset;            // of the group in its page
    int pages, rest, page_size;  // a step's whole pages and rows
    __device__ __forceinline__ void start(const KvAttnParams& p, int b, int key, int step) {
        const int page = key / p.page_size;
        entry = p.table + b * p.table_stride + page;
        offset = key - page * p.page_size;
        page_size = p.page_size;
        pages = step / page_size;
        rest = step - pages * page_size;
    }
    __device__ __forceinline__ void next() {
        entry += pages;
        offset += rest;
        if (offset >= page_size) {
            offset -= page_size;
            ++entry;
        }
    }
};

__device__ __forceinline__ bool kv_page(const KvAttnParams& p, int id) { return (uint32_t)id < (uint32_t)p.pages; }

// Where the group at `offset` of page `id` begins, its keys or its values (in page 0
// where there is no such page: whoever loads it hides the keys and clears the values)
struct KvFrom {
    const char* rows;
    const uint8_t* scales;
};
template <bool MX>
__device__ __forceinline__ KvFrom kv_from(const KvAttnParams& p, bool keys, int kv_head, int id, int offset) {
    const uint64_t page = kv_page(p, id) ? (uint32_t)id : 0u;
    const uint32_t row = (uint32_t)(kv_head * p.page_size + offset);  // (a page has at most 2^28 values)
    const uint64_t bytes = page * p.page_bytes + row * (uint32_t)(MX ? p.dim / 2 : p.dim * 2);
    const uint64_t sc = MX ? page * p.scale_bytes + row * (uint32_t)(p.dim / 32) : 0;
    return KvFrom{(keys ? p.k : p.v) + bytes, (keys ? p.k_scales : p.v_scales) + sc};
}

// Pairs of bf16 with zeros for infinities and NaN
__device__ __forceinline__ u32x4 kv_finite(u32x4 x) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if ((x[k] & 0x7f80u) == 0x7f80u) x[k] &= 0xffff0000u;
        if ((x[k] & 0x7f800000u) == 0x7f800000u) x[k] &= 0xffffu;
    }
    return x;
}

// 16 keys (or values) of one head as a wave loads them: 16-byte pieces, RPL
// rows a load, so that a load covers whole neighbouring rows; MXFP4: a piece is
// a block of 32 values, and its scale comes with it.  Lanes without a piece of
// their own (heads of fewer dims than DP) read the row's first.
template <int DP, bool MX>
struct KvGroup {
    static constexpr int LPR = MX ? DP / 32 : DP / 8;          // pieces of a row
    static constexpr int RPL = 64 / LPR < 16 ? 64 / LPR : 16;  // rows of a load
    static constexpr int N = 16 / RPL;
    u32x4 v[N];
    uint8_t scale[MX ? N : 1];  // (widened where it is used: sooner would wait for the load)

    __device__ __forceinline__ static int row(int l, int i) { return i * RPL + l / LPR; }
    __device__ __forceinline__ static int piece(int l) { return l % LPR; }
    __device__ __forceinline__ static bool active(int l) { return RPL * LPR == 64 || l < RPL * LPR; }

    // A lane's byte offsets in a group's rows and scales; the next load's rows follow
    struct At {
        uint32_t bytes, scale, step, scale_step;
        bool mine;
    };
    __device__ __forceinline__ static At at(int dim, int l) {
        const uint32_t row_bytes = MX ? dim / 2 : dim * 2, blocks = dim / 32, r = active(l) ? l / LPR : 0;
        At a;
        a.mine = piece(l) * (MX ? 32 : 8) < dim;
        a.bytes = r * row_bytes + (a.mine ? 16 * piece(l) : 0);
        a.scale = r * blocks + (a.mine ? piece(l) : 0);
        a.step = RPL * row_bytes;
        a.scale_step = RPL * blocks;
        return a;
    }
    // from: the group's first row (wave-uniform)
    __device__ __forceinline__ void load(const KvFrom& from, const At& a) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = *(const u32x4*)(from.rows + (a.bytes + i * a.step));
        if constexpr (MX) {
#pragma unroll
            for (int i = 0; i < N; ++i) scale[i] = from.scales[a.scale + i * a.scale_step];
        }
    }
    __device__ __forceinline__ void clear(int i) {
        v[i] = u32x4{};
        if constexpr (MX) scale[i] = 0;
    }
    // rows from `n` on become zeros
    __device__ __forceinline__ void cut(int n, int l) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (row(l, i) >= n) clear(i);
    }
    // dims past a head's become zeros
    __device__ __forceinline__ void narrow(const At& a) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!a.mine) clear(i);
    }
    // a value of this lane may be infinite or NaN (MXFP4: its block's scale says so)
    __device__ __forceinline__ bool not_finite() const {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (MX) {
                bad |= scale[i] >= 253;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    bad |= (v[i][k] & 0x7f80u) == 0x7f80u || (v[i][k] & 0x7f800000u) == 0x7f800000u;
            }
        }
        return bad;
    }
    // zeros for infinities and NaN (as bf16 values)
    __device__ __forceinline__ void clean() {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (MX) {
                // 2^126 and 2^127 leave the numbers below 4 and below 2 finite
                const uint32_t e = scale[i];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t w = v[i][k], two = w >> 2 & 0x11111111u, four = two & w >> 1;
                    v[i][k] = e == 255 ? 0 : w & ~(15u * (e == 254 ? two : (e == 253 ? four : 0)));
                }
                if (e == 255) scale[i] = 0;
            } else {
                v[i] = kv_finite(v[i]);
            }
        }
    }
    // MXFP4: words k ^ turn in place of word k, so that lanes of neighbouring rows write
    // other pieces of their blocks at a time
    __device__ __forceinline__ void turn(int turn) {
        if constexpr (MX) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const u32x4 a = v[i], b = turn & 1 ? u32x4{a[1], a[0], a[3], a[2]} : a;
                v[i] = turn & 2 ? u32x4{b[2], b[3], b[0], b[1]} : b;
            }
        }
    }
    // into bf16 rows of `stride` values; part: a quarter of it; turned: by how much
    __device__ __forceinline__ void put_part(uint16_t* rows, int stride, int l, int part, int turned = 0) const {
        if (!active(l)) return;
        if constexpr (MX) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                *(bf16x8*)(rows + row(l, i) * stride + 32 * piece(l) + 8 * (part ^ turned)) =
                    mxfp4_bf16(v[i][part], __uint_as_float((uint32_t)scale[i] << 23));
        } else {
#pragma unroll
            for (int i = part; i < N; i += 4) *(u32x4*)(rows + row(l, i) * stride + 8 * piece(l)) = v[i];
        }
    }
    __device__ __forceinline__ void put(uint16_t* rows, int stride, int l) const {
#pragma unroll
        for (int part = 0; part < 4; ++part) put_part(rows, stride, l, part);
    }
};

// An infinite or NaN value of a key that a row sees makes its dim of the row so, however
// small the key's probability.  A product does not always say that:
//   - where some rows of a tile see a key and others do not, 0 times such a value would
//     reach the others: it is a zero in LDS (KvGroup::clean);
//   - where a probability, or a factor that sums are rescaled by, has left f32's range, 0
//     times an infinity is NaN for the row that sees it too.
// So at the end the keys of the former, and all of a row's keys where a dim is NaN, are
// looked through again, and what they hold is added: the infinity or NaN itself.  (Again
// where the product had it, which changes nothing.)  add(j, v): to dims d0 + j (j < 4) of
// the lane's row.  `key` and the sequence are wave-uniform, d0 is the lane's.
template <bool MX, typename F>
__device__ __forceinline__ void kv_add_infinite(const KvAttnParams& p, int b, int kv_head, int key, bool sees, int d0, F&& add) {
    const int page = key / p.page_size, id = s_load(p.table + b * p.table_stride + page);
    if ((uint32_t)id >= (uint32_t)p.pages || !sees || d0 >= p.dim) return;
    const int64_t row = (int64_t)kv_head * p.page_size + (key - page * p.page_size);
    uint32_t lo, hi;
    if constexpr (MX) {
        const uint16_t w = *(const uint16_t*)(p.v + (uint64_t)id * p.page_bytes + (row * p.dim + d0) / 2);
        const uint8_t e = p.v_scales[(uint64_t)id * p.scale_bytes + (row * p.dim + d0) / 32];
        const u32x4 x = __builtin_bit_cast(u32x4, mxfp4_bf16(w, __uint_as_float((uint32_t)e << 23)));
        lo = x[0], hi = x[1];
    } else {
        const u32x2 x = *(const u32x2*)(p.v + (uint64_t)id * p.page_bytes + (row * p.dim + d0) * 2);
        lo = x[0], hi = x[1];
    }
    const uint32_t v[4] = {lo << 16, lo & 0xffff0000u, hi << 16, hi & 0xffff0000u};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if ((v[j] & 0x7f800000u) == 0x7f800000u) add(j, __uint_as_float(v[j]));
}

// Groups of 16 keys (`from` a multiple of 16) with values of this head that are infinite or
// NaN: each(first, last).  wanted(first): whether to look at a group.  A wave together.
template <int DP, bool MX, typename W, typename F>
__device__ __forceinline__ void kv_each_infinite(const KvAttnParams& p, int b, int kv_head, int from, int to, int l, W&& wanted,
                                                 F&& each) {
    using Group = KvGroup<DP, MX>;
    const typename Group::At at = Group::at(p.dim, l);
    if (__builtin_expect(from >= to, 1)) return;
    for (int k0 = from; k0 < to; k0 += 16) {
        if (!wanted(k0)) continue;
        const int page = k0 / p.page_size, id = s_load(p.table + b * p.table_stride + page);
        if (!kv_page(p, id)) continue;
        Group v;
        v.load(kv_from<MX>(p, false, kv_head, id, k0 - page * p.page_size), at);
        if (__builtin_amdgcn_ballot_w64(v.not_finite())) each(k0, min(k0 + 16, to));
    }
}

// v times a weight or factor that may have left f32's range
__device__ __forceinline__ float kv_weighted(float v, float a) {
    return a == 0.f && !(__builtin_fabsf(v) < INFINITY) ? v : a * v;
}
__device__ __forceinline__ f32x4 kv_weighted(f32x4 v, float a) {
    if (__builtin_expect(a != 0.f, 1)) return a * v;
    return f32x4{kv_weighted(v[0], a), kv_weighted(v[1], a), kv_weighted(v[2], a), kv_weighted(v[3], a)};
}
__device__ __forceinline__ bool kv_nan(f32x4 v) {
    return __builtin_isunordered(v[0], v[1]) | __builtin_isunordered(v[2], v[3]);
}

}  // namespace mr
