// The way of tokens to their experts and back: the pairs (token, slot) in
// expert order, the tokens' rows laid out in it, the experts' results added up
// with the router's weights, and the gradients of the last two.
//
//   sort      rows are the pairs with an id in [0, experts), by expert, inside
//             an expert by pair index (a stable counting sort)
//   dispatch  rows[row_of_pair[t][j]] = x[t]
//   combine   out[t] = sum_j w[t][j] * rows[row_of_pair[t][j]]
//   backward  d_rows[row] = w[t][j] * d_out[t],
//             d_w[t][j] = <d_out[t], rows[row_of_pair[t][j]]>
// and the gradient of the dispatch is a combine with all weights 1.
//
// A pair whose id is outside [0, experts) has no row (row_of_pair -1): it adds
// nothing, its d_w is 0.  No result depends on the order in which anything
// runs: there is no atomic whose order could show.
#include <algorithm>
#include <type_traits>

#include "mr_kernels.hpp"

namespace mr {

namespace {

// ---------------------------------------------------------------- sort
constexpr int ES_WAVES = 8, ES_THREADS = 64 * ES_WAVES;
constexpr int ES_STEPS = EXPERT_SORT_PAIRS / ES_THREADS;  // pairs per lane

// pair u of lane l of wave w: wave w has the 64 ES_STEPS pairs from
// 64 ES_STEPS w of the workgroup's, lanes next to each other
__device__ __forceinline__ int es_pair(int w, int l, int u) { return 64 * (ES_STEPS * w + u) + l; }

__device__ __forceinline__ void es_load(const ExpertSortParams& p, int first, int (&bin)[ES_STEPS]) {
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < ES_STEPS; ++u) {
        const int i = first + es_pair(w, l, u);
        bin[u] = i < p.pairs ? p.ids[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < ES_STEPS; ++u) bin[u] = (uint32_t)bin[u] < (uint32_t)p.experts ? bin[u] : -1;
}

// counts[block][expert], more than one workgroup only
__global__ void __launch_bounds__(ES_THREADS) expert_count_kernel(ExpertSortParams p) {
    extern __shared__ int32_t bins[];
    for (int e = threadIdx.x; e < p.experts; e += ES_THREADS) bins[e] = 0;
    __syncthreads();
    int bin[ES_STEPS];
    es_load(p, blockIdx.x * EXPERT_SORT_PAIRS, bin);
#pragma unroll
    for (int u = 0; u < ES_STEPS; ++u)
        if (bin[u] >= 0) atomicAdd(&bins[bin[u]], 1);  // a count: the order does not show
    __syncthreads();
    int32_t* out = p.counts + (int64_t)blockIdx.x * p.experts;
    for (int e = threadIdx.x; e < p.experts; e += ES_THREADS) out[e] = bins[e];
}

// counts[block][expert] becomes the expert's pairs up to and in the workgroup
// that counted it.  A workgroup has 64 experts (or what is
// left): `groups` threads per expert share the workgroups' counts in runs.
constexpr int EX_THREADS = 1024;
__global__ void __launch_bounds__(EX_THREADS) expert_scan_kernel(ExpertSortParams p, int blocks) {
    __shared__ int32_t part[EX_THREADS];
    const int tid = threadIdx.x, e0 = 64 * blockIdx.x, left = min(p.experts - e0, 64), groups = EX_THREADS / left;
    const int g = tid / left, e = tid - g * left, run = (blocks + groups - 1) / groups;
    const int lo = min(g * run, blocks), hi = g < groups ? min(lo + run, blocks) : lo;
    int32_t* at = p.counts + e0 + e;
    int sum = 0;
#pragma unroll 8
    for (int b = lo; b < hi; ++b) sum += at[(int64_t)b * p.experts];
    part[tid] = sum;
    __syncthreads();
    int before = 0;
    for (int k = 0; k < g; ++k) before += part[k * left + e];
    for (int b = lo; b < hi; b += 8) {
        int c[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) c[k] = b + k < hi ? at[(int64_t)(b + k) * p.experts] : 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            before += c[k];
            if (b + k < hi) at[(int64_t)(b + k) * p.experts] = before;
        }
    }
}

// One workgroup places 2048 pairs (4096: 2 us more at 32768 pairs).  LDS:
// cursor[wave][expert], at first the wave's count of the expert, then the row
// that the wave's next pair of it gets: the expert's first row, plus its pairs in
// earlier workgroups (SCANNED: read; else summed over their counts), plus those
// in earlier waves.  A wave then takes its pairs in order, 64 at a time;
// lanes of one expert find each other by one ballot per bit of the id, so a
// lane's rank among them is a count of bits.
template <bool SCANNED>
__global__ void __launch_bounds__(ES_THREADS) expert_place_kernel(ExpertSortParams p) {
    extern __shared__ int32_t cursor[];
    __shared__ int32_t sums[ES_WAVES];
    __shared__ int32_t group_sums[2][ES_THREADS];
    const int tid = threadIdx.x, l = tid & 63, E = p.experts;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int blocks = gridDim.x, first = blockIdx.x * EXPERT_SORT_PAIRS;
    int bin[ES_STEPS];
    es_load(p, first, bin);
    for (int i = tid; i < ES_WAVES * E; i += ES_THREADS) cursor[i] = 0;
    __syncthreads();
    int32_t* mine = cursor + w * E;
#pragma unroll
    for (int u = 0; u < ES_STEPS; ++u)
        if (bin[u] >= 0) atomicAdd(&mine[bin[u]], 1);
    __syncthreads();
    // ES_THREADS experts at a time: first rows by a scan over the experts
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += ES_THREADS) {
        const int e = e0 + tid;
        int before = 0, total = 0;  // of the expert: in earlier workgroups, in all
        if (SCANNED) {
            if (e < E) {
                if (blockIdx.x > 0) before = p.counts[((int64_t)blockIdx.x - 1) * E + e];
                total = p.counts[((int64_t)blocks - 1) * E + e];
            }
        } else if (blocks == 1) {
            if (e < E) {
#pragma unroll
                for (int k = 0; k < ES_WAVES; ++k) total += cursor[k * E + e];
            }
        } else {
            // `groups` threads per expert share the workgroups' counts
            const int left = min(E - e0, ES_THREADS), groups = ES_THREADS / left;
            const int g = tid / left, own = e0 + tid - g * left;
            if (g < groups) {
#pragma unroll 8
                for (int b = g; b < blocks; b += groups) {
                    const int c = p.counts[(int64_t)b * E + own];
                    total += c;
                    before += b < (int)blockIdx.x ? c : 0;
                }
            }
            group_sums[0][tid] = total;
            group_sums[1][tid] = before;
            __syncthreads();
            total = before = 0;
            for (int k = 0; e < E && k < groups; ++k) {
                total += group_sums[0][k * left + tid];
                before += group_sums[1][k * left + tid];
            }
        }
        const int incl = (int)wave_scan_incl((uint32_t)total);
        if (l == 63) sums[w] = incl;
        __syncthreads();
        int at = carry + incl - total;
#pragma unroll
        for (int k = 0; k < ES_WAVES; ++k) {
            const int c = sums[k];
            if (k < w) at += c;
            carry += c;
        }
        if (e < E) {
            if (blockIdx.x == 0) p.offsets[e] = at;
            at += before;
#pragma unroll
            for (int k = 0; k < ES_WAVES; ++k) {
                const int c = cursor[k * E + e];
                cursor[k * E + e] = at;
                at += c;
            }
        }
        __syncthreads();  // sums are free; at the end, the cursors are whole
    }
    if (blockIdx.x == 0 && tid == 0) p.offsets[E] = carry;
    int bits = 0;
    while ((1 << bits) < E) ++bits;
#pragma unroll 1
    for (int u = 0; u < ES_STEPS; ++u) {
        int b = bin[0];  // bin[u], without indexed registers
#pragma unroll
        for (int k = 1; k < ES_STEPS; ++k) b = u == k ? bin[k] : b;
        const int i = first + es_pair(w, l, u);
        if (first + es_pair(w, 0, u) >= p.pairs) break;
        uint64_t same = __ballot(b >= 0);
        for (int k = 0; k < bits; ++k) {
            const uint64_t set = __ballot((b >> k) & 1);
            same &= (b >> k) & 1 ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << l) - 1)), n = __popcll(same);
        int row = -1;
        if (b >= 0) {
            row = mine[b] + rank;
            p.pair_of_row[row] = i;
        }
        // every lane has read its cursor before the last of an expert moves it
        __builtin_amdgcn_wave_barrier();
        if (b >= 0 && rank == n - 1) mine[b] = row + 1;
        __builtin_amdgcn_wave_barrier();
        if (i < p.pairs) p.row_of_pair[i] = row;
    }
    // rows past the last: no pair
    for (int r = carry + blockIdx.x * ES_THREADS + tid; r < p.pairs; r += blocks * ES_THREADS) p.pair_of_row[r] = -1;
}

// ---------------------------------------------------------------- rows
// A row as a buffer of its `dim` values, or (live false) of none: loads past its
// end give zeros and stores there nothing, so that neither needs a branch, behind
// which the compiler waits for the loads before it (the backward of one token of
// 7168: 12.9 us with branches, 7.1 without).
template <bool F32>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const void* p, int64_t row, int64_t ld, int64_t dim, bool live = true) {
    constexpr int SIZE = F32 ? 4 : 2;
    return __builtin_amdgcn_make_buffer_rsrc((char*)p + (live ? row : 0) * ld * SIZE, 0, live ? (int)dim * SIZE : 0, 0x00020000);
}

// Eight values of a row as stored: VEC, 16 bytes next to each other (f32: twice,
// at a distance of the workgroup's), rows 16-byte aligned; otherwise 8 at a
// distance of the workgroup's threads.  Every instruction of a wave covers whole
// lines.  Loads are streaming (a row is read once), and so are the stores of
// results: of 142 us for sort, dispatch and combine of 4096 tokens of 7168, 4 rows
// each, that took 15.  Dispatched rows, which the experts' products read next, are
// stored plainly (past the caches 2 us less, but the products after them take 20
// of 480 more).
template <bool F32, bool VEC>
struct Eight {
    using Elem = std::conditional_t<F32, uint32_t, uint16_t>;
    static constexpr int N16 = F32 ? 2 : 1, E16 = F32 ? 4 : 8;  // 16-byte units, values of one
    static constexpr int STEP = VEC ? E16 : 1;                  // values of a load or store
    static constexpr int NT = 2;                                // the instructions' streaming bit
    std::conditional_t<VEC, u32x4[N16], Elem[8]> v;
    static __device__ __forceinline__ int at(int c, int k) { return (c + k * STEP * (int)blockDim.x) * (F32 ? 4 : 2); }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t row, int c) {
#pragma unroll
        for (int k = 0; k < (VEC ? N16 : 8); ++k) {
            if constexpr (VEC)
                v[k] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(row, at(c, k), 0, NT));
            else if constexpr (F32)
                v[k] = __builtin_amdgcn_raw_buffer_load_b32(row, at(c, k), 0, 0);
            else
                v[k] = __builtin_amdgcn_raw_buffer_load_b16(row, at(c, k), 0, 0);
        }
    }
    template <bool STREAM>
    __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t row, int c) const {
#pragma unroll
        for (int k = 0; k < (VEC ? N16 : 8); ++k) {
            if constexpr (VEC)
                __builtin_amdgcn_raw_buffer_store_b128(v[k], row, at(c, k), 0, STREAM ? NT : 0);
            else if constexpr (F32)
                __builtin_amdgcn_raw_buffer_store_b32(v[k], row, at(c, k), 0, 0);
            else
                __builtin_amdgcn_raw_buffer_store_b16(v[k], row, at(c, k), 0, 0);
        }
    }
    __device__ __forceinline__ float get(int k) const {
        if constexpr (VEC) {
            if constexpr (F32) return __uint_as_float(v[k >> 2][k & 3]);
            return __uint_as_float(k & 1 ? v[0][k >> 1] & 0xffff0000u : v[0][k >> 1] << 16);
        } else {
            return F32 ? __uint_as_float(v[k]) : __uint_as_float((uint32_t)v[k] << 16);
        }
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
            if constexpr (F32) {
                if constexpr (VEC) {
                    v[k >> 2][k & 3] = __float_as_uint(f[k]);
                    v[k >> 2][(k & 3) + 1] = __float_as_uint(f[k + 1]);
                } else {
                    v[k] = __float_as_uint(f[k]);
                    v[k + 1] = __float_as_uint(f[k + 1]);
                }
            } else {
                const uint32_t two = pack_bf16x2_hw(f[k], f[k + 1]);
                if constexpr (VEC) {
                    v[0][k >> 1] = two;
                } else {
                    v[k] = (uint16_t)two;
                    v[k + 1] = (uint16_t)(two >> 16);
                }
            }
        }
    }
};

// the first value of this thread's piece `i` of a row (of 8 blockDim.x values)
template <bool F32, bool VEC>
__device__ __forceinline__ int piece_col(int i) {
    return 8 * i * (int)blockDim.x + Eight<F32, VEC>::STEP * (int)threadIdx.x;
}

// The rows of a token's slots j0 .. j0 + 63: lane j has that of slot j0 + j
// (-1: none, and for what no sort writes), and its weight.  `has`: the slots
// that have one.  Batches of rows are read off with readlane, so that their
// addresses and the branches round them are scalar.
struct Slots {
    int row;
    float weight;
    uint64_t has;
    __device__ __forceinline__ void load(const ExpertRowsParams& p, int64_t t, int j0) {
        const int j = j0 + (threadIdx.x & 63);
        const int64_t i = t * p.per_token + j;
        row = -1;
        weight = 1.f;
        if (j < p.per_token) {
            row = p.row_of_pair[i];
            if ((int64_t)(uint32_t)row >= (int64_t)p.n_tokens * p.per_token) row = -1;
            if (p.weights) weight = p.weights[i];
        }
        has = __ballot(row >= 0);
    }
    __device__ __forceinline__ int row_of(int j) const { return __builtin_amdgcn_readlane(row, j); }
    __device__ __forceinline__ float weight_of(int j) const {
        return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), j));
    }
};

// One workgroup per token and span of a row: the piece is read once and stored
// once per slot that has a row, bit for bit.  Bound by its stores (4096 tokens of
// 7168, 4 rows each: 294 MB in 56 us).
template <bool F32, bool VEC, int U>
__global__ void __launch_bounds__(512) expert_dispatch_kernel(ExpertRowsParams p, int spans) {
    const int64_t t = blockIdx.x / (unsigned)spans, s = blockIdx.x - t * spans;
    const __amdgpu_buffer_rsrc_t xr = row_buffer<F32>(p.tokens, t, p.ld_tokens, p.dim);
    Eight<F32, VEC> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].load(xr, piece_col<F32, VEC>(s * U + u));
    for (int j0 = 0; j0 < p.per_token; j0 += 64) {
        Slots sl;
        sl.load(p, t, j0);
        for (uint64_t m = sl.has; m; m &= m - 1) {
            const __amdgpu_buffer_rsrc_t row = row_buffer<F32>(p.out, sl.row_of(__builtin_ctzll(m)), p.ld_out, p.dim);
#pragma unroll
            for (int u = 0; u < U; ++u) x[u].template store<false>(row, piece_col<F32, VEC>(s * U + u));
        }
    }
}

constexpr int EC_ROWS = 8;  // rows of a token in flight together

// One workgroup per token and span; sums in f32, in slot order.  Bound by its loads
// (4096 tokens of 7168, 4 rows each: 294 MB in 53 us).
template <bool F32, bool VEC, int U>
__global__ void __launch_bounds__(512) expert_combine_kernel(ExpertRowsParams p, int spans) {
    const int64_t t = blockIdx.x / (unsigned)spans, s = blockIdx.x - t * spans;
    float sum[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[u][k] = 0.f;
    for (int j0 = 0; j0 < p.per_token; j0 += 64) {
        Slots sl;
        sl.load(p, t, j0);
        uint64_t m = sl.has;
        while (m) {
            Eight<F32, VEC> y[EC_ROWS][U];
            float w[EC_ROWS];
            const int n = min(__popcll(m), EC_ROWS);
#pragma unroll
            for (int b = 0; b < EC_ROWS; ++b) {
                const int j = b < n ? __builtin_ctzll(m) : 0;
                m &= m - 1;  // (0 stays 0)
                w[b] = sl.weight_of(j);
                const __amdgpu_buffer_rsrc_t row = row_buffer<F32>(p.rows, sl.row_of(j), p.ld_rows, p.dim, b < n);
#pragma unroll
                for (int u = 0; u < U; ++u) y[b][u].load(row, piece_col<F32, VEC>(s * U + u));
            }
#pragma unroll
            for (int b = 0; b < EC_ROWS; ++b) {
                if (b >= n) continue;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < 8; ++k) sum[u][k] = fmaf(w[b], y[b][u].get(k), sum[u][k]);
            }
        }
    }
    const __amdgpu_buffer_rsrc_t out = row_buffer<F32>(p.out, t, p.ld_out, p.dim);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        Eight<F32, VEC> o;
        o.set(sum[u]);
        o.template store<true>(out, piece_col<F32, VEC>(s * U + u));
    }
}

// One workgroup per token, all spans: d_out[t] is read once per batch of rows,
// each row once, each d_row written once; the dot products are summed per thread
// over the spans, then over the workgroup in a fixed order.  Bound by HBM (2001
// tokens of 2048, 6 rows each: 106 MB in 23 us).
template <bool F32, bool VEC, int U>
__global__ void __launch_bounds__(512) expert_combine_backward_kernel(ExpertRowsParams p, int spans) {
    __shared__ float part[8][EC_ROWS];
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, waves = blockDim.x >> 6;
    const __amdgpu_buffer_rsrc_t gr = row_buffer<F32>(p.tokens, t, p.ld_tokens, p.dim);
    for (int j0 = 0; j0 < p.per_token; j0 += 64) {
        Slots sl;
        sl.load(p, t, j0);
        if (p.d_weights && w == 0 && j0 + l < p.per_token && sl.row < 0) p.d_weights[t * p.per_token + j0 + l] = 0.f;
        uint64_t m = sl.has;
        while (m) {
            const uint64_t before = m;
            const int n = min(__popcll(m), EC_ROWS);
            float wt[EC_ROWS], dot[EC_ROWS];
            int r[EC_ROWS];
#pragma unroll
            for (int b = 0; b < EC_ROWS; ++b) {
                const int j = b < n ? __builtin_ctzll(m) : 0;
                m &= m - 1;  // (0 stays 0)
                r[b] = sl.row_of(j);
                wt[b] = sl.weight_of(j);
                dot[b] = 0.f;
            }
            for (int s = 0; s < spans; ++s) {
                Eight<F32, VEC> g[U], y[EC_ROWS][U];
                int c[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    c[u] = piece_col<F32, VEC>(s * U + u);
                    g[u].load(gr, c[u]);
                }
                if (p.d_weights) {
#pragma unroll
                    for (int b = 0; b < EC_ROWS; ++b) {
                        const __amdgpu_buffer_rsrc_t row = row_buffer<F32>(p.rows, r[b], p.ld_rows, p.dim, b < n);
#pragma unroll
                        for (int u = 0; u < U; ++u) y[b][u].load(row, c[u]);
                    }
                }
                if (p.out) {
#pragma unroll
                    for (int b = 0; b < EC_ROWS; ++b) {
                        if (b >= n) continue;
                        const __amdgpu_buffer_rsrc_t row = row_buffer<F32>(p.out, r[b], p.ld_out, p.dim);
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            float d[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) d[k] = wt[b] * g[u].get(k);
                            Eight<F32, VEC> o;
                            o.set(d);
                            o.template store<true>(row, c[u]);
                        }
                    }
                }
                if (p.d_weights) {  // (past the row's end both are zeros)
#pragma unroll
                    for (int b = 0; b < EC_ROWS; ++b) {
                        if (b >= n) continue;
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            float d = 0.f;
#pragma unroll
                            for (int k = 0; k < 8; ++k) d = fmaf(g[u].get(k), y[b][u].get(k), d);
                            dot[b] += d;
                        }
                    }
                }
            }
            if (p.d_weights) {
#pragma unroll
                for (int b = 0; b < EC_ROWS; ++b) dot[b] = wave_sum(dot[b]);
                if (l == 0) {
#pragma unroll
                    for (int b = 0; b < EC_ROWS; ++b) part[w][b] = dot[b];
                }
                __syncthreads();
                if (w == 0 && ((before & ~m) >> l & 1)) {  // the lanes of the batch's slots
                    const int b = __popcll(before & ((1ull << l) - 1));
                    float d = 0.f;
                    for (int k = 0; k < waves; ++k) d += part[k][b];
                    p.d_weights[t * p.per_token + j0 + l] = d;
                }
                __syncthreads();  // the parts are read before they are written again
            }
        }
    }
}

bool row_aligned(const void* p, int64_t ld, int size) { return !p || (((uintptr_t)p & 15) == 0 && ld * size % 16 == 0); }

// Threads of a workgroup and pieces of 8 values per thread (U): two pieces and
// up to 512 threads, so that most rows are one workgroup's; where there are few
// tokens, one piece and a wave each, to have the work on many CUs (per_span)
struct RowLaunch {
    bool vec, two;
    int threads, spans;
};
RowLaunch row_launch(const ExpertRowsParams& p, bool per_span, int cus) {
    const int size = p.f32 ? 4 : 2;
    RowLaunch r;
    r.vec = p.dim % 8 == 0 && row_aligned(p.tokens, p.ld_tokens, size) && row_aligned(p.rows, p.ld_rows, size) &&
            row_aligned(p.out, p.ld_out, size);
    const int64_t pieces = (p.dim + 7) / 8;
    const bool few = per_span && p.n_tokens < cus;
    r.two = !few && pieces > 64;
    const int u = r.two ? 2 : 1;
    r.threads = few ? 64 : (int)std::min<int64_t>(512, (pieces + 64 * u - 1) / (64 * u) * 64);
    r.spans = (int)((pieces + (int64_t)r.threads * u - 1) / ((int64_t)r.threads * u));
    return r;
}

}  // namespace

#define MR_ROW_KERNEL(KERNEL, PER_SPAN)                                                          \
    const RowLaunch r = row_launch(p, PER_SPAN, cu_count);                                       \
    const int64_t grid = (int64_t)p.n_tokens * (PER_SPAN ? r.spans : 1);                         \
    if (grid * r.threads >= (1ll << 32)) return hipErrorInvalidValue;                            \
    const auto kern = p.f32 ? (r.vec ? (r.two ? KERNEL<true, true, 2> : KERNEL<true, true, 1>)   \
                                     : (r.two ? KERNEL<true, false, 2> : KERNEL<true, false, 1>)) \
                            : (r.vec ? (r.two ? KERNEL<false, true, 2> : KERNEL<false, true, 1>) \
                                     : (r.two ? KERNEL<false, false, 2> : KERNEL<false, false, 1>)); \
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(r.threads), 0, st, p, r.spans);          \
    return hipGetLastError()

hipError_t launch_expert_dispatch(const ExpertRowsParams& p, int cu_count, hipStream_t st) { MR_ROW_KERNEL(expert_dispatch_kernel, true); }
hipError_t launch_expert_combine(const ExpertRowsParams& p, int cu_count, hipStream_t st) { MR_ROW_KERNEL(expert_combine_kernel, true); }
hipError_t launch_expert_combine_backward(const ExpertRowsParams& p, int cu_count, hipStream_t st) {
    MR_ROW_KERNEL(expert_combine_backward_kernel, false);
}

#undef MR_ROW_KERNEL

// Every workgroup of the placement reads all counts, unless they are scanned
// first, in a launch more (a call in us: 2^20 pairs of 1024 experts 94 -> 27, 2^24
// pairs of 128 2135 -> 161, of 8 210 -> 80; 32768 pairs of 4096 26 -> 21; 2^17
// pairs of 256 15 without)
bool scan_counts(int64_t blocks, int64_t experts) { return blocks > 512 || blocks * experts >= 1 << 16; }

hipError_t launch_expert_sort(const ExpertSortParams& p, hipStream_t st) {
    const int blocks = std::max(1, expert_sort_blocks(p.pairs));
    const size_t lds = (size_t)ES_WAVES * p.experts * 4;
    const bool scan = scan_counts(blocks, p.experts);
    const auto place = scan ? expert_place_kernel<true> : expert_place_kernel<false>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)place, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    if (blocks > 1) {
        hipLaunchKernelGGL(expert_count_kernel, dim3(blocks), dim3(ES_THREADS), (size_t)p.experts * 4, st, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (scan) {
        hipLaunchKernelGGL(expert_scan_kernel, dim3((p.experts + 63) / 64), dim3(EX_THREADS), 0, st, p, blocks);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(place, dim3(blocks), dim3(ES_THREADS), lds, st, p);
    return hipGetLastError();
}

}  // namespace mr
