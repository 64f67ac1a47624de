// kernels_adjust.hip — scores with penalties for the classes of a row's history, biases and
// masks of allowed classes (mbk_adjust).  Each score is read and written once.
#include "grid.hpp"
#include "mbk.h"
#include "ops.h"

namespace mbk {

namespace {

// A workgroup takes up to CLASSES classes of a row: it counts in LDS how often the row's history
// holds each of them, and then passes over their scores.  The history is read once for each of
// a row's workgroups.
template <int E, int THREADS, int CLASSES>
__global__ __launch_bounds__(THREADS) void k_adjust(AdjustCall c, int32_t parts) {
    extern __shared__ uint32_t count[];              // [class], where there are penalties
    const int64_t id = group_id();
    const int64_t row = id / parts;
    if (row >= c.rows) return;
    const int64_t first = (id - row * parts) * CLASSES;
    const int here = (int)min((int64_t)CLASSES, c.classes - first);
    int32_t len = 0;
    if (c.penalties) {
        len = c.lengths ? min(max(c.lengths[row], 0), c.history) : c.history;
        for (int i = threadIdx.x; i < here; i += THREADS) count[i] = 0;
        __syncthreads();
        const int32_t *ids = c.ids + row * c.history_stride;
        for (int32_t i = threadIdx.x; i < len; i += THREADS) {
            const int64_t at = ids[i] - first;
            if (at >= 0 && at < here) atomicAdd(&count[at], 1u);
        }
        __syncthreads();
    }
    typedef float V __attribute__((ext_vector_type(E)));
    const float *scores = c.scores + row * c.score_stride + first;
    float *out = c.out + row * c.out_stride + first;
    const float *bias = c.bias ? c.bias + first : nullptr;
    const uint32_t *allowed = c.allowed ? c.allowed + row * c.mask_stride + first / 32 : nullptr;
    for (int i = threadIdx.x * E; i < here; i += THREADS * E) {
        const int n = here - i;
        float z[E], b[E];
        if (E > 1 && n >= E) {
            const V v = *reinterpret_cast<const V *>(scores + i);
#pragma unroll
            for (int e = 0; e < E; ++e) z[e] = v[e];
            if (bias) {
                const V w = *reinterpret_cast<const V *>(bias + i);
#pragma unroll
                for (int e = 0; e < E; ++e) b[e] = w[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                z[e] = e < n ? scores[i + e] : 0.0f;
                if (bias) b[e] = e < n ? bias[i + e] : 0.0f;
            }
        }
        const uint32_t bits = allowed ? allowed[i >> 5] >> (i & 31) : ~0u;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (len > 0 && e < n) {
                const uint32_t times = count[i + e];
                if (times) {
                    z[e] = z[e] > 0.0f ? z[e] / c.repetition : z[e] * c.repetition;
                    z[e] -= __builtin_fmaf(c.frequency, (float)times, c.presence);
                }
            }
            if (bias) z[e] += b[e];
            if (!((bits >> e) & 1u)) z[e] = -__builtin_inff();
        }
        if (E > 1 && n >= E) {
            V v;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = z[e];
            *reinterpret_cast<V *>(out + i) = v;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < n) out[i + e] = z[e];
        }
    }
}

bool aligned(const void *p, int64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 4 == 0;
}

template <int E>
hipError_t adjust(hipStream_t s, const AdjustCall &c) {
    constexpr int CLASSES = 4096;
    const int32_t parts = (int32_t)((c.classes + CLASSES - 1) / CLASSES);
    const size_t lds = c.penalties ? CLASSES * sizeof(uint32_t) : 0;
    hipLaunchKernelGGL((k_adjust<E, 256, CLASSES>), grid_of(c.rows * parts), dim3(256), lds, s, c,
                       parts);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_adjust(hipStream_t s, const AdjustCall &c) {
    const bool wide = aligned(c.scores, c.score_stride) && aligned(c.out, c.out_stride) &&
                      (!c.bias || aligned(c.bias, 0));
    return wide ? adjust<4>(s, c) : adjust<1>(s, c);
}

}  // namespace mbk
