// kernels_clip.hip — the norm of many gradients together, and each of them scaled so that it is
// at most a given one (mbk_grad_clip).  Both passes are bound by memory: the factor needs every
// element, so the gradients are read twice unless they fit a cache.
#include <algorithm>

#include "mbk.h"
#include "ops.h"

namespace mbk {

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;

// 16 bytes at any address that holds an element.
template <typename T, int E> using Run = T __attribute__((ext_vector_type(E), aligned(sizeof(T))));

// Visits a piece 16 bytes at a time, AT_ONCE of them on the way: take(runs, where they are, how
// many elements of each count).  Where a row ends inside a run only its elements are read.
constexpr int AT_ONCE = 4;
template <typename T, int E, class Take>
__device__ __forceinline__ void each_run(const ClipPiece &p, Take take) {
    const T *g = static_cast<const T *>(p.grad);
    const uint32_t chunks = (uint32_t)(p.cols + E - 1) / E, all = chunks * (uint32_t)p.rows;
    for (uint32_t i0 = threadIdx.x; i0 < all; i0 += AT_ONCE * THREADS) {
        Run<T, E> v[AT_ONCE];
        int64_t at[AT_ONCE];
        int n[AT_ONCE];
#pragma unroll
        for (int q = 0; q < AT_ONCE; ++q) {
            const uint32_t i = i0 + q * THREADS;
            const uint32_t r = p.rows == 1 ? 0 : i / chunks, c = (i - r * chunks) * E;
            at[q] = r * p.stride + c;
            n[q] = i < all ? p.cols - (int)c : 0;
            if (n[q] >= E) v[q] = *reinterpret_cast<const Run<T, E> *>(g + at[q]);
        }
#pragma unroll
        for (int q = 0; q < AT_ONCE; ++q)
            if (n[q] < E)
#pragma unroll
                for (int e = 0; e < E; ++e) v[q][e] = e < n[q] ? g[at[q] + e] : (T)0.0f;
        take(v, at, n);
    }
}

template <typename T, int E>
__device__ __forceinline__ double squares(const ClipPiece &p) {
    double sum = 0.0;
    each_run<T, E>(p, [&](const Run<T, E> (&v)[AT_ONCE], const int64_t (&)[AT_ONCE],
                          const int (&)[AT_ONCE]) {
#pragma unroll
        for (int q = 0; q < AT_ONCE; ++q)
#pragma unroll
            for (int e = 0; e < E; ++e) sum = __builtin_fma((double)v[q][e], (double)v[q][e], sum);
    });
    return sum;
}

// Products in 64 bits, rounded to f32 and from there to the type.
template <typename T, int E>
__device__ __forceinline__ void scale(const ClipPiece &p, double by, bool streamed) {
    T *o = static_cast<T *>(p.out);
    each_run<T, E>(p, [&](const Run<T, E> (&v)[AT_ONCE], const int64_t (&at)[AT_ONCE],
                          const int (&n)[AT_ONCE]) {
#pragma unroll
        for (int q = 0; q < AT_ONCE; ++q) {
            Run<T, E> x;
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = (T)(float)((double)v[q][e] * by);
            if (n[q] >= E) {
                put(o + at[q], x, streamed);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (e < n[q]) o[at[q] + e] = x[e];
            }
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

// 353 MB of both types take 55 us, 6.5 TB/s with what the call before left in the last cache; six
// tensors of 75000 elements 3.5, a launch and two reads one after the other.
__global__ __launch_bounds__(THREADS) void k_clip_norm(const ClipPiece *__restrict__ pieces,
                                                       int64_t count,
                                                       double *__restrict__ partial) {
    __shared__ double wave_sum[WAVES];
    double sum = 0.0;
    for (int64_t i = blockIdx.x; i < count; i += gridDim.x) {
        const ClipPiece p = pieces[i];
        sum += p.bf16 ? squares<__bf16, 8>(p) : squares<float, 4>(p);
    }
    sum = sum_all(sum, wave_sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// Every workgroup sums up the partial sums by itself.  Pieces come in the other order than in the
// first pass, so that the last ones read are still in a cache (353 MB forwards 120 us, 117 so);
// stores of many outputs go past it (the next call's first pass: 82 us after ordinary ones, 54).
// 353 MB take 119 us, 5.9 TB/s of reading and writing.
__global__ __launch_bounds__(THREADS) void k_clip_scale(const ClipPiece *__restrict__ pieces,
                                                        int64_t count,
                                                        const double *__restrict__ partial,
                                                        int32_t partials, float max_norm,
                                                        float *__restrict__ norm, bool outputs,
                                                        bool streamed) {
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
        if (p.bf16) scale<__bf16, 8>(p, by, streamed);
        else scale<float, 4>(p, by, streamed);
    }
}

// Few elements: both passes by one workgroup in one launch, a wavefront up to ONE_EACH pieces of at
// most 256 runs, which stay in its registers between the passes (32,700 f32 elements 7.7 us a
// call, 10.9 by two launches; 64 pieces, 65,000 elements, take one workgroup 10.1).
constexpr int ONE_WAVES = 16, ONE_EACH = CLIP_ONE / ONE_WAVES;
typedef uint32_t Raw __attribute__((ext_vector_type(4)));

template <typename T> constexpr int RUN = 16 / sizeof(T);
// Where run i of a piece lies and how many of its elements are real.
template <typename T>
__device__ __forceinline__ int run_at(const ClipPiece &p, uint32_t i, int64_t &at) {
    const uint32_t chunks = (uint32_t)(p.cols + RUN<T> - 1) / RUN<T>;
    const uint32_t r = p.rows == 1 ? 0 : i / chunks, c = (i - r * chunks) * RUN<T>;
    at = r * p.stride + c;
    return i < chunks * (uint32_t)p.rows ? p.cols - (int)c : 0;
}
template <typename T>
__device__ __forceinline__ void load_runs(const ClipPiece &p, Raw (&raw)[4]) {
    typedef Run<T, RUN<T>> V;
    const T *g = static_cast<const T *>(p.grad);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        int64_t at;
        const int n = run_at<T>(p, q * 64 + (threadIdx.x & 63), at);
        V v;
        if (n >= RUN<T>) {
            v = *reinterpret_cast<const V *>(g + at);
        } else {
#pragma unroll
            for (int e = 0; e < RUN<T>; ++e) v[e] = e < n ? g[at + e] : (T)0.0f;
        }
        raw[q] = __builtin_bit_cast(Raw, v);
    }
}
template <typename T> __device__ __forceinline__ double sum_runs(const Raw (&raw)[4]) {
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const auto v = __builtin_bit_cast(T __attribute__((ext_vector_type(16 / sizeof(T)))), raw[q]);
#pragma unroll
        for (int e = 0; e < RUN<T>; ++e) sum = __builtin_fma((double)v[e], (double)v[e], sum);
    }
    return sum;
}
template <typename T>
__device__ __forceinline__ void store_runs(const ClipPiece &p, const Raw (&raw)[4], double by) {
    typedef Run<T, RUN<T>> V;
    T *o = static_cast<T *>(p.out);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        int64_t at;
        const int n = run_at<T>(p, q * 64 + (threadIdx.x & 63), at);
        V v = __builtin_bit_cast(V, raw[q]);
#pragma unroll
        for (int e = 0; e < RUN<T>; ++e) v[e] = (T)(float)((double)v[e] * by);
        if (n >= RUN<T>) {
            *reinterpret_cast<V *>(o + at) = v;
        } else {
#pragma unroll
            for (int e = 0; e < RUN<T>; ++e)
                if (e < n) o[at + e] = v[e];
        }
    }
}

__global__ __launch_bounds__(64 * ONE_WAVES) void k_clip_one(const ClipPiece *__restrict__ pieces,
                                                             int32_t count, float max_norm,
                                                             float *__restrict__ norm) {
    __shared__ double wave_sum[ONE_WAVES];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Raw raw[ONE_EACH][4];
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < ONE_EACH; ++k) {
        if (k * ONE_WAVES + wave >= count) continue;
        const ClipPiece p = pieces[k * ONE_WAVES + wave];
        if (p.bf16) load_runs<__bf16>(p, raw[k]);
        else load_runs<float>(p, raw[k]);
    }
#pragma unroll
    for (int k = 0; k < ONE_EACH; ++k) {
        if (k * ONE_WAVES + wave >= count) continue;
        sum += pieces[k * ONE_WAVES + wave].bf16 ? sum_runs<__bf16>(raw[k]) : sum_runs<float>(raw[k]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if ((threadIdx.x & 63) == 0) wave_sum[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < ONE_WAVES; ++w) sum += wave_sum[w];
    const double all = __builtin_sqrt(sum);
    if (threadIdx.x == 0) *norm = (float)all;
    const bool clip = all > (double)max_norm && all < __builtin_inf();
    const double by = clip ? (double)max_norm / all : 1.0;
#pragma unroll
    for (int k = 0; k < ONE_EACH; ++k) {
        if (k * ONE_WAVES + wave >= count) continue;
        const ClipPiece p = pieces[k * ONE_WAVES + wave];
        if (!p.out || (!clip && p.out == p.grad)) continue;
        if (p.bf16) store_runs<__bf16>(p, raw[k], by);
        else store_runs<float>(p, raw[k], by);
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
    if (c.one) {
        hipLaunchKernelGGL(k_clip_one, dim3(1), dim3(64 * ONE_WAVES), 0, s, c.piece,
                           (int32_t)c.pieces, c.max_norm, c.norm);
        return hipGetLastError();
    }
    const int groups = groups_of(c.pieces, c.num_cus);
    double *partial = reinterpret_cast<double *>(scratch);
    hipLaunchKernelGGL(k_clip_norm, dim3(groups), dim3(THREADS), 0, s, c.piece, c.pieces, partial);
    hipLaunchKernelGGL(k_clip_scale, dim3(c.outputs ? groups : 1), dim3(THREADS), 0, s, c.piece,
                       c.pieces, partial, groups, c.max_norm, c.norm, c.outputs, c.streamed);
    return hipGetLastError();
}

}  // namespace mbk
