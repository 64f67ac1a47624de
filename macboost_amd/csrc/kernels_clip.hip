// kernels_clip.hip — the norm of many gradients together, and each of them scaled so that it is
// at most a given one (mbk_grad_clip).  Both passes are bound by memory: the factor needs every
// element, so the gradients are read twice unless they fit a cache.
#include <algorithm>

#include "mbk.h"
#include "ops.h"

namespace mbk {

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;

// Visits the elements of a piece, E at a time: take(offset of the first, how many of them).
// E > 1 only where the piece's addresses and stride are multiples of 16 bytes.
template <int E, class Take>
__device__ __forceinline__ void each_of(const ClipPiece &p, Take take) {
    if (p.rows == 1) {
        for (int i = threadIdx.x * E; i < p.cols; i += THREADS * E) take((int64_t)i, p.cols - i);
        return;
    }
    const uint32_t chunks = (uint32_t)(p.cols + E - 1) / E, all = chunks * (uint32_t)p.rows;
    for (uint32_t i = threadIdx.x; i < all; i += THREADS) {
        const uint32_t r = i / chunks, c = (i - r * chunks) * E;
        take(r * p.stride + c, p.cols - (int)c);
    }
}

template <typename T, int E>
__device__ __forceinline__ double squares(const ClipPiece &p) {
    typedef T V __attribute__((ext_vector_type(E)));
    const T *g = static_cast<const T *>(p.grad);
    double sum = 0.0;
    each_of<E>(p, [&](int64_t at, int n) {
        if (n >= E) {
            const V v = *reinterpret_cast<const V *>(g + at);
#pragma unroll
            for (int e = 0; e < E; ++e) sum = __builtin_fma((double)v[e], (double)v[e], sum);
        } else {
            for (int e = 0; e < n; ++e) sum = __builtin_fma((double)g[at + e], (double)g[at + e], sum);
        }
    });
    return sum;
}

// A product in 64 bits, rounded to f32 and from there to the type.
template <typename T> __device__ __forceinline__ T scaled(T v, double by) {
    return (T)(float)((double)v * by);
}

template <typename T, int E>
__device__ __forceinline__ void scale(const ClipPiece &p, double by) {
    typedef T V __attribute__((ext_vector_type(E)));
    const T *g = static_cast<const T *>(p.grad);
    T *o = static_cast<T *>(p.out);
    each_of<E>(p, [&](int64_t at, int n) {
        if (n >= E) {
            V v = *reinterpret_cast<const V *>(g + at);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = scaled<T>(v[e], by);
            *reinterpret_cast<V *>(o + at) = v;
        } else {
            for (int e = 0; e < n; ++e) o[at + e] = scaled<T>(g[at + e], by);
        }
    });
}

// The sum of v over the workgroup, in every thread.
__device__ __forceinline__ double sum_all(double v, double *wave_sum) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += wave_sum[w];
    __syncthreads();
    return sum;
}

__global__ __launch_bounds__(THREADS) void k_clip_norm(const ClipPiece *__restrict__ pieces,
                                                       int64_t count,
                                                       double *__restrict__ partial) {
    __shared__ double wave_sum[WAVES];
    double sum = 0.0;
    for (int64_t i = blockIdx.x; i < count; i += gridDim.x) {
        const ClipPiece p = pieces[i];
        if (p.bf16) sum += p.wide ? squares<__bf16, 8>(p) : squares<__bf16, 1>(p);
        else sum += p.wide ? squares<float, 4>(p) : squares<float, 1>(p);
    }
    sum = sum_all(sum, wave_sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// Every workgroup sums up the partial sums by itself.  Pieces come in the other order than in the
// first pass, so that the last ones read are still in a cache.
__global__ __launch_bounds__(THREADS) void k_clip_scale(const ClipPiece *__restrict__ pieces,
                                                        int64_t count,
                                                        const double *__restrict__ partial,
                                                        int32_t partials, float max_norm,
                                                        float *__restrict__ norm, bool outputs) {
    __shared__ double wave_sum[WAVES];
    double sum = 0.0;
    for (int i = threadIdx.x; i < partials; i += THREADS) sum += partial[i];
    sum = sum_all(sum, wave_sum);
    const double all = __builtin_sqrt(sum);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)all;
    if (!outputs) return;
    const bool clip = all > (double)max_norm && all < __builtin_inf();
    const double by = clip ? (double)max_norm / all : 1.0;
    for (int64_t i = blockIdx.x; i < count; i += gridDim.x) {
        const ClipPiece p = pieces[count - 1 - i];
        if (!p.out || (!clip && p.out == p.grad)) continue;
        if (p.bf16) {
            if (p.wide) scale<__bf16, 8>(p, by);
            else scale<__bf16, 1>(p, by);
        } else {
            if (p.wide) scale<float, 4>(p, by);
            else scale<float, 1>(p, by);
        }
    }
}

int groups_of(int64_t pieces, int num_cus) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(pieces, 8 * (int64_t)num_cus));
}

}  // namespace

size_t clip_scratch(int64_t pieces, int num_cus) {
    return sizeof(double) * (size_t)groups_of(pieces, num_cus);
}

hipError_t launch_clip(hipStream_t s, const ClipCall &c, char *scratch) {
    const int groups = groups_of(c.pieces, c.num_cus);
    double *partial = reinterpret_cast<double *>(scratch);
    hipLaunchKernelGGL(k_clip_norm, dim3(groups), dim3(THREADS), 0, s, c.piece, c.pieces, partial);
    hipLaunchKernelGGL(k_clip_scale, dim3(c.outputs ? groups : 1), dim3(THREADS), 0, s, c.piece,
                       c.pieces, partial, groups, c.max_norm, c.norm, c.outputs);
    return hipGetLastError();
}

}  // namespace mbk
