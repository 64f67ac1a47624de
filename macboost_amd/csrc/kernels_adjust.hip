// kernels_adjust.hip — scores with penalties for the classes of a row's history, biases and
// masks of allowed classes (mbk_adjust).  Each score is read and written once, which bounds it:
// 256 x 100000 take 39 us, 5.3 TB/s; 1 x 1003 3.3, a launch and three reads one after the other.
#include "grid.hpp"
#include "mbk.h"
#include "ops.h"

namespace mbk {

namespace {

// A workgroup takes up to CLASSES classes of a row: it counts in LDS how often the row's history
// holds each of them, with their scores on the way, and then passes over the scores, four a lane at
// any address of a float.  The history is read once for each of a row's workgroups: 256 x 100000
// scores with histories of up to 2000 take 38 us by 4096 classes, 40 by 2048 and 37 by 16384, which
// leaves CUs idle where there are fewer (1000 x 20000: 32, 34 and 37).
constexpr int THREADS = 256, CLASSES = 4096, EACH = CLASSES / (4 * THREADS);
typedef float Run __attribute__((ext_vector_type(4), aligned(4)));

__global__ __launch_bounds__(THREADS) void k_adjust(AdjustCall c, int32_t parts) {
    __shared__ uint32_t count[CLASSES];              // [class], where there are penalties
    const int64_t id = group_id();
    const int64_t row = id / parts;
    if (row >= c.rows) return;
    const int64_t first = (id - row * parts) * CLASSES;
    const int here = (int)min((int64_t)CLASSES, c.classes - first);
    const float *scores = c.scores + row * c.score_stride + first;
    float *out = c.out + row * c.out_stride + first;
    const float *bias = c.bias ? c.bias + first : nullptr;
    const uint32_t *allowed = c.allowed ? c.allowed + row * c.mask_stride + first / 32 : nullptr;
    const auto load = [&](const float *p, int i) {
        if (i + 4 <= here) return *reinterpret_cast<const Run *>(p + i);
        Run v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < here ? p[i + e] : 0.0f;
        return v;
    };
    Run z[EACH];
#pragma unroll
    for (int x = 0; x < EACH; ++x) z[x] = load(scores, (x * THREADS + threadIdx.x) * 4);
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
#pragma unroll
    for (int x = 0; x < EACH; ++x) {
        const int i = (x * THREADS + threadIdx.x) * 4;
        if (i >= here) break;
        if (len > 0)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t times = i + e < here ? count[i + e] : 0;
                if (times) {
                    const float v = z[x][e] > 0.0f ? z[x][e] / c.repetition : z[x][e] * c.repetition;
                    z[x][e] = v - __builtin_fmaf(c.frequency, (float)times, c.presence);
                }
            }
        if (bias) {
            const Run b = load(bias, i);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[x][e] += b[e];
        }
        if (allowed) {
            const uint32_t bits = allowed[i >> 5] >> (i & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!((bits >> e) & 1u)) z[x][e] = -__builtin_inff();
        }
        if (i + 4 <= here) {
            put(out + i, z[x], c.streamed);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < here) out[i + e] = z[x][e];
        }
    }
}

}  // namespace

hipError_t launch_adjust(hipStream_t s, const AdjustCall &call) {
    AdjustCall c = call;
    c.streamed = c.rows * c.classes * 4 > STREAMED;
    const int32_t parts = (int32_t)((c.classes + CLASSES - 1) / CLASSES);
    hipLaunchKernelGGL(k_adjust, grid_of(c.rows * parts), dim3(THREADS), 0, s, c, parts);
    return hipGetLastError();
}

}  // namespace mbk
