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

// One workgroup places 4096 pairs.  LDS: cursor[wave][expert], at first the
// wave's count of the expert, then the row that the wave's next pair of it
// gets: the expert's first row, plus its pairs in earlier workgroups, plus
// those in earlier waves.  A wave then takes its pairs in order, 64 at a time;
// lanes of one expert find each other by one ballot per bit of the id, so a
// lane's rank among them is a count of bits.
__global__ void __launch_bounds__(ES_THREADS) expert_place_kernel(ExpertSortParams p) {
    extern __shared__ int32_t cursor[];
    __shared__ int32_t sums[ES_WAVES];
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
        if (e < E) {
            if (blocks == 1) {
#pragma unroll
                for (int k = 0; k < ES_WAVES; ++k) total += cursor[k * E + e];
            } else {
#pragma unroll 8
                for (int b = 0; b < blocks; ++b) {
                    const int c = p.counts[(int64_t)b * E + e];
                    total += c;
                    before += b < (int)blockIdx.x ? c : 0;
                }
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
// Eight values of a row per thread: VEC, 8 next to each other (16 or 32
// bytes, rows 16-byte aligned); otherwise 8 at a distance of the workgroup's
// threads, so that a wave still reads whole lines.
template <bool F32, bool VEC>
struct Eight {
    float v[8];
    __device__ __forceinline__ void load(const void* p, int64_t c, int step, int64_t dim) {
        if constexpr (VEC) {
            if constexpr (F32) {
                const f32x4 a = *(const f32x4*)((const float*)p + c), b = *(const f32x4*)((const float*)p + c + 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = a[k], v[4 + k] = b[k];
            } else {
                const u32x4 a = *(const u32x4*)((const uint16_t*)p + c);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[2 * k] = __uint_as_float(a[k] << 16), v[2 * k + 1] = __uint_as_float(a[k] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t i = c + (int64_t)k * step;
                v[k] = i >= dim ? 0.f : (F32 ? ((const float*)p)[i] : bf16_bits_to_f32(((const uint16_t*)p)[i]));
            }
        }
    }
    __device__ __forceinline__ void store(void* p, int64_t c, int step, int64_t dim) const {
        if constexpr (VEC) {
            if constexpr (F32) {
                *(f32x4*)((float*)p + c) = f32x4{v[0], v[1], v[2], v[3]};
                *(f32x4*)((float*)p + c + 4) = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                *(u32x4*)((uint16_t*)p + c) = u32x4{pack_bf16x2_hw(v[0], v[1]), pack_bf16x2_hw(v[2], v[3]),
                                                    pack_bf16x2_hw(v[4], v[5]), pack_bf16x2_hw(v[6], v[7])};
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t i = c + (int64_t)k * step;
                if (i < dim) {
                    if (F32)
                        ((float*)p)[i] = v[k];
                    else
                        ((uint16_t*)p)[i] = f32_to_bf16_bits(v[k]);
                }
            }
        }
    }
};

template <bool F32>
__device__ __forceinline__ const char* row_at(const void* p, int64_t row, int64_t ld) {
    return (const char*)p + row * ld * (F32 ? 4 : 2);
}

// the first value of this thread's eight in span `s` of 8 blockDim.x values
template <bool VEC>
__device__ __forceinline__ int64_t span_col(int64_t s) {
    return 8 * s * blockDim.x + (VEC ? 8 : 1) * (int64_t)threadIdx.x;
}

// row of pair i, -1 for none (and for what no sort writes)
__device__ __forceinline__ int pair_row(const ExpertRowsParams& p, int64_t i) {
    const int r = p.row_of_pair[i];
    return (int64_t)(uint32_t)r < (int64_t)p.n_tokens * p.per_token ? r : -1;
}

// One workgroup per token and span: the token's piece is read once and stored
// per_token times, bit for bit.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256) expert_dispatch_kernel(ExpertRowsParams p, int spans) {
    using Elem = std::conditional_t<F32, uint32_t, uint16_t>;
    const int64_t t = blockIdx.x / (unsigned)spans;
    const int64_t c = span_col<VEC>(blockIdx.x - t * spans);
    if (c >= p.dim) return;
    const Elem* x = (const Elem*)row_at<F32>(p.tokens, t, p.ld_tokens) + c;
    const int n = VEC ? 8 : (int)std::min<int64_t>(8, (p.dim - c + blockDim.x - 1) / blockDim.x);
    u32x4 v[F32 ? 2 : 1];
    Elem e[8];
    if constexpr (VEC) {
#pragma unroll
        for (int k = 0; k < (F32 ? 2 : 1); ++k) v[k] = ((const u32x4*)x)[k];
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) e[k] = x[(int64_t)k * blockDim.x];
    }
    for (int j = 0; j < p.per_token; ++j) {
        const int r = pair_row(p, t * p.per_token + j);
        if (r < 0) continue;
        Elem* y = (Elem*)row_at<F32>(p.out, r, p.ld_out) + c;
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < (F32 ? 2 : 1); ++k) ((u32x4*)y)[k] = v[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < n) y[(int64_t)k * blockDim.x] = e[k];
        }
    }
}

constexpr int EC_U = 8;  // slots whose rows are in flight together

// One workgroup per token and span; sums in f32, in slot order.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256) expert_combine_kernel(ExpertRowsParams p, int spans) {
    const int64_t t = blockIdx.x / (unsigned)spans;
    const int64_t c = span_col<VEC>(blockIdx.x - t * spans);
    if (c >= p.dim) return;
    Eight<F32, VEC> sum;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum.v[k] = 0.f;
    for (int j0 = 0; j0 < p.per_token; j0 += EC_U) {
        Eight<F32, VEC> y[EC_U];
        int r[EC_U];
        float w[EC_U];
#pragma unroll
        for (int j = 0; j < EC_U; ++j) {
            const int64_t i = t * p.per_token + j0 + j;
            r[j] = j0 + j < p.per_token ? pair_row(p, i) : -1;
            w[j] = r[j] >= 0 && p.weights ? p.weights[i] : 1.f;
        }
#pragma unroll
        for (int j = 0; j < EC_U; ++j)
            if (r[j] >= 0) y[j].load(row_at<F32>(p.rows, r[j], p.ld_rows), c, blockDim.x, p.dim);
#pragma unroll
        for (int j = 0; j < EC_U; ++j)
            if (r[j] >= 0) {
#pragma unroll
                for (int k = 0; k < 8; ++k) sum.v[k] = fmaf(w[j], y[j].v[k], sum.v[k]);
            }
    }
    sum.store((char*)row_at<F32>(p.out, t, p.ld_out), c, blockDim.x, p.dim);
}

// One workgroup per token, all spans: d_out[t] is read once per EC_U slots,
// each slot's row once, each d_row written once; the dot products are summed
// per thread over the spans, then over the workgroup in a fixed order.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256) expert_combine_backward_kernel(ExpertRowsParams p, int spans) {
    __shared__ float part[4][EC_U];
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x, w = tid >> 6, waves = blockDim.x >> 6;
    for (int j0 = 0; j0 < p.per_token; j0 += EC_U) {
        int r[EC_U];
        float wt[EC_U], dot[EC_U];
#pragma unroll
        for (int j = 0; j < EC_U; ++j) {
            const int64_t i = t * p.per_token + j0 + j;
            r[j] = j0 + j < p.per_token ? pair_row(p, i) : -1;
            wt[j] = r[j] >= 0 && p.weights ? p.weights[i] : 1.f;
            dot[j] = 0.f;
        }
        for (int s = 0; s < spans; ++s) {
            const int64_t c = span_col<VEC>(s);
            if (c >= p.dim) break;
            Eight<F32, VEC> g, y[EC_U];
            g.load(row_at<F32>(p.tokens, t, p.ld_tokens), c, blockDim.x, p.dim);
            if (p.d_weights) {
#pragma unroll
                for (int j = 0; j < EC_U; ++j)
                    if (r[j] >= 0) y[j].load(row_at<F32>(p.rows, r[j], p.ld_rows), c, blockDim.x, p.dim);
#pragma unroll
                for (int j = 0; j < EC_U; ++j)
                    if (r[j] >= 0) {
                        float d = 0.f;
#pragma unroll
                        for (int k = 0; k < 8; ++k) d = fmaf(g.v[k], y[j].v[k], d);
                        dot[j] += d;
                    }
            }
            if (p.out) {
#pragma unroll
                for (int j = 0; j < EC_U; ++j)
                    if (r[j] >= 0) {
                        Eight<F32, VEC> d;
#pragma unroll
                        for (int k = 0; k < 8; ++k) d.v[k] = wt[j] * g.v[k];
                        d.store((char*)row_at<F32>(p.out, r[j], p.ld_out), c, blockDim.x, p.dim);
                    }
            }
        }
        if (p.d_weights) {
#pragma unroll
            for (int j = 0; j < EC_U; ++j) dot[j] = wave_sum(dot[j]);
            if ((tid & 63) == 0) {
#pragma unroll
                for (int j = 0; j < EC_U; ++j) part[w][j] = dot[j];
            }
            __syncthreads();
            if (tid < EC_U && j0 + tid < p.per_token) {
                float d = 0.f;
                for (int k = 0; k < waves; ++k) d += part[k][tid];
                p.d_weights[t * p.per_token + j0 + tid] = d;
            }
            __syncthreads();  // the parts are read before they are written again
        }
    }
}

// threads of a workgroup: eight values each, no more waves than the row has
// work for
int row_threads(int64_t dim) { return (int)std::min<int64_t>(256, (dim + 511) / 512 * 64); }

bool row_aligned(const void* p, int64_t ld, int64_t rows, int size) {
    return !p || (((uintptr_t)p & 15) == 0 && (rows == 1 || ld * size % 16 == 0));
}

template <typename L>
hipError_t row_launch(const ExpertRowsParams& p, bool per_span, L launch) {
    const int size = p.f32 ? 4 : 2, threads = row_threads(p.dim);
    const bool vec = p.dim % 8 == 0 && row_aligned(p.tokens, p.ld_tokens, 2, size) &&
                     row_aligned(p.rows, p.ld_rows, 2, size) && row_aligned(p.out, p.ld_out, 2, size);
    const int64_t spans = (p.dim + 8 * threads - 1) / (8 * threads), grid = p.n_tokens * (per_span ? spans : 1);
    if (grid * threads >= (1ll << 32)) return hipErrorInvalidValue;
    launch(vec, dim3((unsigned)grid), dim3((unsigned)threads), (int)spans);
    return hipGetLastError();
}

}  // namespace

#define MR_ROW_KERNEL(KERNEL, PER_SPAN)                                                                      \
    return row_launch(p, PER_SPAN, [&](bool vec, dim3 g, dim3 b, int spans) {                                \
        if (p.f32)                                                                                           \
            vec ? KERNEL<true, true><<<g, b, 0, st>>>(p, spans) : KERNEL<true, false><<<g, b, 0, st>>>(p, spans);   \
        else                                                                                                 \
            vec ? KERNEL<false, true><<<g, b, 0, st>>>(p, spans) : KERNEL<false, false><<<g, b, 0, st>>>(p, spans); \
    })

hipError_t launch_expert_dispatch(const ExpertRowsParams& p, hipStream_t st) { MR_ROW_KERNEL(expert_dispatch_kernel, true); }
hipError_t launch_expert_combine(const ExpertRowsParams& p, hipStream_t st) { MR_ROW_KERNEL(expert_combine_kernel, true); }
hipError_t launch_expert_combine_backward(const ExpertRowsParams& p, hipStream_t st) {
    MR_ROW_KERNEL(expert_combine_backward_kernel, false);
}

#undef MR_ROW_KERNEL

hipError_t launch_expert_sort(const ExpertSortParams& p, hipStream_t st) {
    const int blocks = std::max(1, expert_sort_blocks(p.pairs));
    const size_t lds = (size_t)ES_WAVES * p.experts * 4;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)expert_place_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    if (blocks > 1) {
        hipLaunchKernelGGL(expert_count_kernel, dim3(blocks), dim3(ES_THREADS), (size_t)p.experts * 4, st, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(expert_place_kernel, dim3(blocks), dim3(ES_THREADS), lds, st, p);
    return hipGetLastError();
}

}  // namespace mr
