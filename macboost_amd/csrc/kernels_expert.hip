// kernels_expert.hip — rows sorted by expert and back (mbk_expert_*): a stable
// counting sort of the assignments by expert, the rows' features in that order,
// the experts' outputs summed back for each row, and the gradient of that sum.
// All of them move data; none has work worth counting.
#include <algorithm>

#include "mbk.h"
#include "ops.h"

namespace mbk {

namespace {

__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

// ---------------------------------------------------------------------------
// The sort.  Wavefront u owns the assignments [u * per, (u + 1) * per): it
// counts them by expert, the counts are summed over the wavefronts before it
// and the experts below, and it then hands out slots in ascending order: every
// step is ordered, so the sort is stable and needs no atomic on global memory.
// Counters of one wavefront lie in LDS.
// ---------------------------------------------------------------------------
constexpr int SORT_WAVES = 4;

// table[e * units + u]: assignments of wavefront u to expert e.
__global__ __launch_bounds__(64 * SORT_WAVES) void k_expert_count(
    const int32_t *__restrict__ expert, int64_t slots, int32_t experts, int64_t per, int32_t units,
    uint32_t *__restrict__ table) {
    extern __shared__ uint32_t lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t *count = lds + (size_t)wave * experts;
    const int32_t u = blockIdx.x * SORT_WAVES + wave;
    for (int e = lane; e < experts; e += 64) count[e] = 0;
    __syncthreads();
    if (u < units) {
        const int64_t a = u * per, b = min(slots, a + per);
        for (int64_t i = a + lane; i < b; i += 64) {
            const uint32_t e = (uint32_t)expert[i];
            if (e < (uint32_t)experts) atomicAdd(&count[e], 1u);
        }
    }
    __syncthreads();
    if (u < units)
        for (int e = lane; e < experts; e += 64) table[(int64_t)e * units + u] = count[e];
}

// One wavefront per expert: its counts become sums over the wavefronts before,
// total[e] their sum.
__global__ __launch_bounds__(256) void k_expert_scan(uint32_t *__restrict__ table, int32_t experts,
                                                     int32_t units, uint32_t *__restrict__ total) {
    const int e = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (e >= experts) return;
    uint32_t *row = table + (int64_t)e * units;
    uint32_t sum = 0;
    for (int u0 = 0; u0 < units; u0 += 64) {
        const uint32_t c = u0 + lane < units ? row[u0 + lane] : 0;
        uint32_t x = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(x, o, 64);
            if (lane >= o) x += y;
        }
        if (u0 + lane < units) row[u0 + lane] = sum + x - c;
        sum += __shfl(x, 63, 64);
    }
    if (lane == 0) total[e] = sum;
}

// offsets[e] = assignments to experts below e, by one workgroup.
__global__ __launch_bounds__(1024) void k_expert_offsets(const uint32_t *__restrict__ total,
                                                         int32_t experts,
                                                         int32_t *__restrict__ offsets) {
    __shared__ uint32_t wave_sum[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (int e0 = 0; e0 < experts; e0 += 1024) {
        const int e = e0 + threadIdx.x;
        const uint32_t c = e < experts ? total[e] : 0;
        uint32_t x = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(x, o, 64);
            if (lane >= o) x += y;
        }
        if (lane == 63) wave_sum[wave] = x;
        __syncthreads();
        uint32_t below = 0, all = 0;
        for (int w = 0; w < 16; ++w) {
            if (w < wave) below += wave_sum[w];
            all += wave_sum[w];
        }
        if (e < experts) offsets[e] = (int32_t)(before + below + x - c);
        before += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) offsets[experts] = (int32_t)before;
}

__global__ __launch_bounds__(64 * SORT_WAVES) void k_expert_place(
    const int32_t *__restrict__ expert, int64_t slots, int32_t experts, int32_t key_bits,
    int64_t per, int32_t units, const uint32_t *__restrict__ table,
    const int32_t *__restrict__ offsets, int32_t *__restrict__ source,
    int32_t *__restrict__ slot) {
    extern __shared__ uint32_t lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t *next = lds + (size_t)wave * experts;
    const int32_t u = blockIdx.x * SORT_WAVES + wave;
    if (u >= units) return;                     // no barrier below
    for (int e = lane; e < experts; e += 64)
        next[e] = (uint32_t)offsets[e] + table[(int64_t)e * units + u];
    const int64_t a = u * per, b = min(slots, a + per);
    for (int64_t i0 = a; i0 < b; i0 += 64) {
        const int64_t i = i0 + lane;
        const uint32_t e = i < b ? (uint32_t)expert[i] : 0xFFFFFFFFu;
        const bool kept = e < (uint32_t)experts;
        uint64_t same = __ballot(kept);         // lanes with this lane's expert
        for (int k = 0; k < key_bits; ++k) {
            const uint64_t ones = __ballot((e >> k) & 1u);
            same &= (e >> k) & 1u ? ones : ~ones;
        }
        uint32_t at = 0;
        if (kept) at = next[e] + lanes_below(same);
        __builtin_amdgcn_wave_barrier();
        if (kept && lanes_below(same) == 0) next[e] = at + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (kept) source[at] = (int32_t)i;
        if (i < b) slot[i] = kept ? (int32_t)at : -1;
    }
    // the places behind the last kept assignment
    const int64_t kept = offsets[experts];
    for (int64_t i = a + lane; i < b; i += 64)
        if (i >= kept) source[i] = -1;
}

struct SortShape {
    int64_t per;
    int32_t units;
};
// At least 1024 assignments a wavefront, at most 8 wavefronts a CU and 4M counters.
SortShape sort_shape(const ExpertPlan &p, int num_cus) {
    const int64_t slots = p.rows * p.k;
    int64_t units = std::min<int64_t>((slots + 1023) / 1024, 8 * (int64_t)num_cus);
    units = std::max<int64_t>(1, std::min<int64_t>(units, ((int64_t)4 << 20) / p.experts));
    const int64_t per = std::max<int64_t>(64, ((slots + units - 1) / units + 63) / 64 * 64);
    return {per, (int32_t)std::max<int64_t>(1, (slots + per - 1) / per)};
}

// ---------------------------------------------------------------------------
// Moving rows.  Assignment a of slot s lies in the sorted matrix at
// base + f * step: [slots][cols] has base s * cols and step 1, blocks (the
// expert's [cols][n_e] at cols * offsets[e]) have base cols * offsets[e] + s -
// offsets[e] and step n_e.
// ---------------------------------------------------------------------------
struct Place {
    int64_t base;                // -1: dropped
    int64_t step;
};
__device__ __forceinline__ Place place_of(const ExpertPlan &p, int64_t a, int32_t cols,
                                          bool blocked) {
    const int32_t s = p.slot[a];
    if (s < 0) return {-1, 0};
    if (!blocked) return {(int64_t)s * cols, 1};
    const int32_t e = p.expert[a];
    const int32_t first = p.offsets[e];
    return {(int64_t)first * cols + (s - first), p.offsets[e + 1] - first};
}

constexpr int TILE = 64;

// A tile of 64 rows x 64 columns at a time, 256 threads; XCOLS / SCOLS: the lanes of a
// wavefront run along the columns of the rows' matrix / of the sorted matrix, else
// along the rows; LDS turns the tile where the two differ.
template <typename T, bool XCOLS, bool SCOLS>
__global__ __launch_bounds__(256) void k_expert_gather(ExpertPlan p, ExpertMatrix x,
                                                       T *__restrict__ sorted) {
    __shared__ T tile[TILE][TILE + 1];
    const int64_t i0 = (int64_t)blockIdx.x * TILE;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T *data = static_cast<const T *>(x.data);
    for (int32_t f0 = blockIdx.y * TILE; f0 < x.cols; f0 += gridDim.y * TILE) {
        for (int q = wave; q < TILE; q += 4) {
            const int64_t i = i0 + (XCOLS ? q : lane);
            const int32_t f = f0 + (XCOLS ? lane : q);
            if (i < p.rows && f < x.cols)
                tile[XCOLS ? q : lane][XCOLS ? lane : q] =
                    data[i * x.row_stride + f * x.col_stride];
        }
        __syncthreads();
        if (SCOLS) {
            for (int q = wave; q < TILE; q += 4) {
                if (i0 + q >= p.rows || f0 + lane >= x.cols) continue;
                for (int j = 0; j < p.k; ++j) {
                    const Place at = place_of(p, (i0 + q) * p.k + j, x.cols, x.blocked);
                    if (at.base >= 0) sorted[at.base + (f0 + lane) * at.step] = tile[q][lane];
                }
            }
        } else if (i0 + lane < p.rows) {
            for (int j = 0; j < p.k; ++j) {
                const Place at = place_of(p, (i0 + lane) * p.k + j, x.cols, x.blocked);
                if (at.base < 0) continue;
                for (int q = wave; q < TILE && f0 + q < x.cols; q += 4)
                    sorted[at.base + (f0 + q) * at.step] = tile[lane][q];
            }
        }
        __syncthreads();
    }
}

// out[i] = sum over j, ascending, of weight[i][j] * sorted[slot[i][j]], in f32.
template <typename T, bool XCOLS, bool SCOLS>
__global__ __launch_bounds__(256) void k_expert_combine(ExpertPlan p, const T *__restrict__ sorted,
                                                        const float *__restrict__ weights,
                                                        ExpertMatrix out) {
    __shared__ float tile[TILE][TILE + 1];
    const int64_t i0 = (int64_t)blockIdx.x * TILE;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T *data = static_cast<T *>(out.data);
    for (int32_t f0 = blockIdx.y * TILE; f0 < out.cols; f0 += gridDim.y * TILE) {
        for (int q = wave; q < TILE; q += 4) {
            const int r = SCOLS ? q : lane, c = SCOLS ? lane : q;
            if (i0 + r >= p.rows || f0 + c >= out.cols) continue;
            float sum = 0.0f;
            for (int j = 0; j < p.k; ++j) {
                const int64_t a = (i0 + r) * p.k + j;
                const Place at = place_of(p, a, out.cols, out.blocked);
                if (at.base < 0) continue;
                const float v = to_f32(sorted[at.base + (f0 + c) * at.step]);
                sum += weights ? weights[a] * v : v;
            }
            tile[r][c] = sum;
        }
        __syncthreads();
        for (int q = wave; q < TILE; q += 4) {
            const int r = XCOLS ? q : lane, c = XCOLS ? lane : q;
            if (i0 + r < p.rows && f0 + c < out.cols)
                data[(i0 + r) * out.row_stride + (f0 + c) * out.col_stride] = (T)tile[r][c];
        }
        __syncthreads();
    }
}

// d_sorted[slot[i][j]] = weight[i][j] * dout[i] and d_weights[i][j] = dout[i] .
// sorted[slot[i][j]].  A workgroup has all columns of its rows: each thread sums its
// own columns in f32, and the threads of a row are added in a fixed order.
template <typename T, bool XCOLS, bool SCOLS>
__global__ __launch_bounds__(256) void k_expert_combine_grad(
    ExpertPlan p, ExpertMatrix dout, const T *__restrict__ sorted,
    const float *__restrict__ weights, T *__restrict__ d_sorted, float *__restrict__ d_weights) {
    constexpr int ROWS = 16;
    __shared__ T tile[ROWS][TILE + 2];
    __shared__ float sums[ROWS][17];
    const int64_t i0 = (int64_t)blockIdx.x * ROWS;
    const T *data = static_cast<const T *>(dout.data);
    // 16 threads a row; along the rows the row is the thread's fast index
    const int xr = XCOLS ? threadIdx.x >> 4 : threadIdx.x & 15;
    const int xc = XCOLS ? threadIdx.x & 15 : threadIdx.x >> 4;
    const int sr = SCOLS ? threadIdx.x >> 4 : threadIdx.x & 15;
    const int sc = SCOLS ? threadIdx.x & 15 : threadIdx.x >> 4;
    for (int j = 0; j < p.k; ++j) {
        const int64_t a = (i0 + sr) * p.k + j;
        const bool row = i0 + sr < p.rows;
        const Place at = row ? place_of(p, a, dout.cols, dout.blocked) : Place{-1, 0};
        const float w = row && weights ? weights[a] : 1.0f;
        float dot = 0.0f;
        for (int32_t f0 = 0; f0 < dout.cols; f0 += TILE) {
            __syncthreads();
            for (int c = xc; c < TILE; c += 16)
                if (i0 + xr < p.rows && f0 + c < dout.cols)
                    tile[xr][c] = data[(i0 + xr) * dout.row_stride + (f0 + c) * dout.col_stride];
            __syncthreads();
            if (at.base >= 0)
                for (int c = sc; c < TILE && f0 + c < dout.cols; c += 16) {
                    const float g = to_f32(tile[sr][c]);
                    const int64_t k = at.base + (f0 + c) * at.step;
                    dot += g * to_f32(sorted[k]);
                    d_sorted[k] = (T)(w * g);
                }
        }
        sums[sr][sc] = dot;
        __syncthreads();
        if (threadIdx.x < ROWS && i0 + threadIdx.x < p.rows) {
            float s = 0.0f;
            for (int c = 0; c < 16; ++c) s += sums[threadIdx.x][c];
            d_weights[(i0 + threadIdx.x) * p.k + j] = s;
        }
        __syncthreads();
    }
}

bool along_columns(const ExpertMatrix &x) { return x.col_stride <= x.row_stride; }

dim3 tile_grid(int64_t rows, int32_t cols) {
    return dim3((uint32_t)((rows + TILE - 1) / TILE),
                (uint32_t)std::min<int32_t>((cols + TILE - 1) / TILE, 1024));
}

template <typename T>
hipError_t gather(hipStream_t s, const ExpertPlan &p, const ExpertMatrix &x, void *sorted) {
    const dim3 g = tile_grid(p.rows, x.cols), b(256);
    T *out = static_cast<T *>(sorted);
    if (along_columns(x)) {
        if (x.blocked) hipLaunchKernelGGL((k_expert_gather<T, true, false>), g, b, 0, s, p, x, out);
        else hipLaunchKernelGGL((k_expert_gather<T, true, true>), g, b, 0, s, p, x, out);
    } else {
        if (x.blocked) hipLaunchKernelGGL((k_expert_gather<T, false, false>), g, b, 0, s, p, x, out);
        else hipLaunchKernelGGL((k_expert_gather<T, false, true>), g, b, 0, s, p, x, out);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t combine(hipStream_t s, const ExpertPlan &p, const void *sorted, const float *w,
                   const ExpertMatrix &x) {
    const dim3 g = tile_grid(p.rows, x.cols), b(256);
    const T *y = static_cast<const T *>(sorted);
    if (along_columns(x)) {
        if (x.blocked) hipLaunchKernelGGL((k_expert_combine<T, true, false>), g, b, 0, s, p, y, w, x);
        else hipLaunchKernelGGL((k_expert_combine<T, true, true>), g, b, 0, s, p, y, w, x);
    } else {
        if (x.blocked) hipLaunchKernelGGL((k_expert_combine<T, false, false>), g, b, 0, s, p, y, w, x);
        else hipLaunchKernelGGL((k_expert_combine<T, false, true>), g, b, 0, s, p, y, w, x);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t combine_grad(hipStream_t s, const ExpertPlan &p, const ExpertMatrix &x,
                        const void *sorted, const float *w, void *d_sorted, float *d_weights) {
    const dim3 g((uint32_t)((p.rows + 15) / 16)), b(256);
    const T *y = static_cast<const T *>(sorted);
    T *dy = static_cast<T *>(d_sorted);
    if (along_columns(x)) {
        if (x.blocked)
            hipLaunchKernelGGL((k_expert_combine_grad<T, true, false>), g, b, 0, s, p, x, y, w, dy,
                               d_weights);
        else
            hipLaunchKernelGGL((k_expert_combine_grad<T, true, true>), g, b, 0, s, p, x, y, w, dy,
                               d_weights);
    } else {
        if (x.blocked)
            hipLaunchKernelGGL((k_expert_combine_grad<T, false, false>), g, b, 0, s, p, x, y, w,
                               dy, d_weights);
        else
            hipLaunchKernelGGL((k_expert_combine_grad<T, false, true>), g, b, 0, s, p, x, y, w, dy,
                               d_weights);
    }
    return hipGetLastError();
}

}  // namespace

size_t expert_scratch(const ExpertPlan &p, int num_cus) {
    const SortShape sh = sort_shape(p, num_cus);
    return ((size_t)p.experts * sh.units + p.experts) * sizeof(uint32_t);
}

hipError_t launch_expert_sort(hipStream_t s, const ExpertPlan &p, int num_cus, char *scratch) {
    const SortShape sh = sort_shape(p, num_cus);
    const int64_t slots = p.rows * p.k;
    uint32_t *table = reinterpret_cast<uint32_t *>(scratch);
    uint32_t *total = table + (size_t)p.experts * sh.units;
    int bits = 0;
    while (bits < 31 && (1 << bits) < p.experts) ++bits;
    const dim3 g((uint32_t)((sh.units + SORT_WAVES - 1) / SORT_WAVES)), b(64 * SORT_WAVES);
    const size_t lds = (size_t)SORT_WAVES * p.experts * sizeof(uint32_t);
    hipError_t e = allow_all_lds(reinterpret_cast<const void *>(k_expert_count));
    if (e == hipSuccess) e = allow_all_lds(reinterpret_cast<const void *>(k_expert_place));
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_expert_count, g, b, lds, s, p.expert, slots, p.experts, sh.per, sh.units,
                       table);
    hipLaunchKernelGGL(k_expert_scan, dim3((uint32_t)((p.experts + 3) / 4)), dim3(256), 0, s,
                       table, p.experts, sh.units, total);
    hipLaunchKernelGGL(k_expert_offsets, dim3(1), dim3(1024), 0, s, total, p.experts, p.offsets);
    hipLaunchKernelGGL(k_expert_place, g, b, lds, s, p.expert, slots, p.experts, bits, sh.per,
                       sh.units, table, p.offsets, p.source, p.slot);
    return hipGetLastError();
}

hipError_t launch_expert_gather(hipStream_t s, const ExpertPlan &p, const ExpertMatrix &x,
                                void *sorted) {
    return x.bf16 ? gather<__bf16>(s, p, x, sorted) : gather<float>(s, p, x, sorted);
}

hipError_t launch_expert_combine(hipStream_t s, const ExpertPlan &p, const void *sorted,
                                 const float *weights, const ExpertMatrix &out) {
    return out.bf16 ? combine<__bf16>(s, p, sorted, weights, out)
                    : combine<float>(s, p, sorted, weights, out);
}

hipError_t launch_expert_combine_grad(hipStream_t s, const ExpertPlan &p,
                                      const ExpertMatrix &dout, const void *sorted,
                                      const float *weights, void *d_sorted, float *d_weights) {
    return dout.bf16 ? combine_grad<__bf16>(s, p, dout, sorted, weights, d_sorted, d_weights)
                     : combine_grad<float>(s, p, dout, sorted, weights, d_sorted, d_weights);
}

}  // namespace mbk
