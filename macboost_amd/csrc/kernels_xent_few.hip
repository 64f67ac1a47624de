// kernels_xent_few.hip — the many-class loss of up to 32 rows without gradients, as in
// serving: what bounds it is reading W once, so W is not packed first.
//
// h lies in LDS whole, as operands of the matrix instruction.  Each wavefront takes tiles
// of 32 classes by itself: their rows are copied straight into its own LDS buffers, 128
// bytes of each at a time and two steps ahead, so that eight wavefronts keep 64 KB
// of a CU on the way and no barrier holds them.  (Rows of odd bf16 elements go through
// registers, one step ahead.)  The product is W h' (classes down,
// rows across): a lane has scores of one row, and keeps its maximum and sum over all
// tiles.  f32 operands go into the f32 matrix instruction as they are: at 1/16 of
// the bf16 rate it still takes less time than W's bytes.
#include <algorithm>

#include "mbk.h"
#include "xent.hpp"

namespace mbk {

namespace {

constexpr int WAVES = 8, BUFS = 3;
constexpr int STEP = 32 * 128;                       // bytes of a wavefront's step
constexpr int H_BYTES = LDS_BYTES - WAVES * BUFS * STEP;     // 64 KB
constexpr int ROWS = 32;

__device__ __forceinline__ void join2(float &top, float &sum, float t2, float s2) {
    const float now = fmaxf(top, t2), ref = now == -INFINITY ? 0.0f : now;
    sum = sum * __builtin_amdgcn_exp2f(top - ref) + s2 * __builtin_amdgcn_exp2f(t2 - ref);
    top = now;
}

// part[workgroup][row]: the maximum of z log2 e and the sum of its powers of 2.
// B: bytes of W a lane copies at a time, what its rows' alignment allows (2: by registers).
template <typename T, int B>
__global__ __launch_bounds__(64 * WAVES, 2) void k_few_stats(XentCall c, int64_t tiles, int32_t steps,
                                                             float2 *__restrict__ part) {
    constexpr int PER = 16 / sizeof(T);              // elements of a chunk of 16 bytes
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char *h = lds, *buf = lds + H_BYTES + wave * BUFS * STEP;
    // h: chunk q of row i at (q * 32 + i) * 16, zeros behind its sizes
    for (int q = threadIdx.x; q < steps * 8 * ROWS; q += 64 * WAVES) {
        const int i = q % ROWS, k = q / ROWS * PER;
        T x[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e)
            x[e] = i < c.rows && k + e < c.dim
                       ? static_cast<const T *>(c.h)[i * c.h_stride + k + e] : (T)0.0f;
        *reinterpret_cast<u32x4 *>(h + q * 16) = *reinterpret_cast<const u32x4 *>(x);
    }
    __syncthreads();
    // The chunks of a row are permuted by the row so that 16 rows x 1 chunk fall on all
    // banks.
    const auto permute = [](int row) { return ((row >> 1) & 1) * 4 + ((row >> 2) & 3); };
    const int64_t first = (int64_t)blockIdx.x * WAVES + wave, hop = (int64_t)gridDim.x * WAVES;
    const int64_t mine = first < tiles ? (tiles - first + hop - 1) / hop : 0;
    const int64_t total = mine * steps;
    int64_t tile = first;                            // of the next copy
    int32_t step = 0;
    const T *w_all = static_cast<const T *>(c.w);
    const auto next_step = [&] {
        if (++step == steps) {
            step = 0;
            tile += hop;
        }
    };
    // Where row `row` of the next step has its element k; behind the row, an element that
    // zeros of h go with.
    const auto element = [&](int row, int k) {
        const int64_t v = min(tile * 32 + row, c.classes - 1);
        return w_all + v * c.w_stride + (k < c.dim ? k : 0);
    };
    constexpr int COPIES = B == 2 ? 0 : 4096 / (64 * B);
    const auto copy = [&](int to) {
        if constexpr (B != 2) {
#pragma unroll
            for (int j = 0; j < COPIES; ++j) {
                const int at = j * 64 * B + lane * B, row = at / 128, in = at % 128;
                const int k = (step * 8 + ((in / 16) ^ permute(row))) * PER + in % 16 / (int)sizeof(T);
                global_void *from = (global_void *)element(row, k);
                lds_void *dst = (lds_void *)(buf + to * STEP + j * 64 * B);
                if constexpr (B == 16) __builtin_amdgcn_global_load_lds(from, dst, 16, 0, 0);
                else __builtin_amdgcn_global_load_lds(from, dst, 4, 0, 0);
            }
            next_step();
        }
    };
    T ahead[B == 2 ? 32 : 1];
    const auto load = [&] {
        if constexpr (B == 2) {
#pragma unroll
            for (int row = 0; row < 32; ++row) ahead[row] = *element(row, step * 64 + lane);
            next_step();
        }
    };
    if (B == 2 && total > 0) load();
    if (total > 0) copy(0);
    if (total > 1) copy(1);
    float top = -INFINITY, sum = 0.0f;
    int at = 0;
    for (int64_t t = 0, i = 0; i < mine; ++i) {
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
        for (int32_t k = 0; k < steps; ++k, ++t) {
            if constexpr (B == 2) {
#pragma unroll
                for (int row = 0; row < 32; ++row)
                    *reinterpret_cast<T *>(buf + at * STEP + row * 128 +
                                           ((lane >> 3) ^ permute(row)) * 16 + (lane & 7) * 2) =
                        ahead[row];
                if (t + 1 < total) load();
            } else {
                // this step's copies are there when at most the next step's are not
                if (t + 1 < total) {
                    if constexpr (COPIES == 4) __builtin_amdgcn_s_waitcnt(0x0F74);
                    else __builtin_amdgcn_s_waitcnt(0x4F70);
                }
                else __builtin_amdgcn_s_waitcnt(0x0F70);
                __builtin_amdgcn_sched_barrier(0);
                if (t + 2 < total) copy(at >= 1 ? at - 1 : BUFS - 1);
            }
            const char *w = buf + at * STEP;
            at = at == BUFS - 1 ? 0 : at + 1;
            const int row = lane & 31;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const u32x4 a = *reinterpret_cast<const u32x4 *>(
                    w + row * 128 + ((2 * q + half) ^ permute(row)) * 16);
                const u32x4 b = *reinterpret_cast<const u32x4 *>(
                    h + ((k * 8 + 2 * q + half) * ROWS + row) * 16);
                if constexpr (sizeof(T) == 2) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                                __builtin_bit_cast(bf16x8, b), s, 0,
                                                                0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s = __builtin_amdgcn_mfma_f32_32x32x2f32(
                            __uint_as_float(a[e]), __uint_as_float(b[e]), s, 0, 0, 0);
                }
            }
        }
        const int64_t v0 = (first + i * hop) * 32 + half * 4;
        float m = top;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int64_t v = v0 + (r >> 2) * 8 + (r & 3);
            float b = 0.0f;
            if (v >= c.classes) b = -INFINITY;
            else if (c.bias) b = c.bias[v];
            // a class that is not offered, whatever its w gave
            s[r] = b == -INFINITY ? -INFINITY : __builtin_fmaf(s[r], LOG2E, b * LOG2E);
            m = fmaxf(m, s[r]);
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        sum *= __builtin_amdgcn_exp2f(top - ref);
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(s[r] - ref);
        top = m;
    }
    join2(top, sum, __shfl_xor(top, 32, 64), __shfl_xor(sum, 32, 64));
    __syncthreads();
    float2 *all = reinterpret_cast<float2 *>(lds);
    if (half == 0) all[wave * ROWS + lane] = make_float2(top, sum);
    __syncthreads();
    if (threadIdx.x < ROWS) {
        for (int w = 1; w < WAVES; ++w) {
            const float2 o = all[w * ROWS + threadIdx.x];
            join2(top, sum, o.x, o.y);
        }
        part[blockIdx.x * ROWS + threadIdx.x] = make_float2(top, sum);
    }
}

// One wavefront a row: the parts joined, and the label's score from h and W.
template <typename T>
__global__ __launch_bounds__(64) void k_few_join(XentCall c, int32_t parts,
                                                 const float2 *__restrict__ part) {
    const int lane = threadIdx.x;
    const int64_t i = blockIdx.x;
    const int32_t y = c.labels[i];
    const float wt = c.weights ? c.weights[i] : 1.0f;
    const float by = y < 0 || y >= c.classes ? -INFINITY : c.bias ? c.bias[y] : 0.0f;
    float dot = 0.0f;
    if (by != -INFINITY)
        for (int32_t f = lane; f < c.dim; f += 64)
            dot += (float)static_cast<const T *>(c.h)[i * c.h_stride + f] *
                   (float)static_cast<const T *>(c.w)[y * c.w_stride + f];
    float top = -INFINITY, sum = 0.0f;
    for (int p = lane; p < parts; p += 64) join2(top, sum, part[p * ROWS + i].x, part[p * ROWS + i].y);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        join2(top, sum, __shfl_xor(top, o, 64), __shfl_xor(sum, o, 64));
        dot += __shfl_xor(dot, o, 64);
    }
    if (lane != 0) return;
    const bool none = top == -INFINITY && sum == 0.0f;
    const float lse = log_sum(top, sum).natural;
    c.lse[i] = lse;
    const bool out = y < 0 || y >= c.classes || wt == 0.0f || none;
    c.loss[i] = out ? 0.0f : wt * (lse - (dot + by));
}

template <typename T, int B> hipError_t run(hipStream_t s, const XentCall &c, char *scratch) {
    const hipError_t e = allow_all_lds(reinterpret_cast<const void *>(k_few_stats<T, B>));
    if (e != hipSuccess) return e;
    const int64_t tiles = (c.classes + 31) / 32;
    const int32_t steps = (int32_t)((c.dim * sizeof(T) + 127) / 128);
    const uint32_t groups = (uint32_t)std::min<int64_t>(c.num_cus, (tiles + WAVES - 1) / WAVES);
    float2 *part = reinterpret_cast<float2 *>(scratch);
    hipLaunchKernelGGL((k_few_stats<T, B>), dim3(groups), dim3(64 * WAVES), LDS_BYTES, s, c, tiles,
                       steps, part);
    hipLaunchKernelGGL((k_few_join<T>), dim3((uint32_t)c.rows), dim3(64), 0, s, c, (int32_t)groups,
                       part);
    return hipGetLastError();
}

}  // namespace

// h must fit the LDS beside the buffers.
bool xent_few(const XentCall &c) {
    const int64_t size = c.bf16 ? 2 : 4;
    return !c.grad && c.rows <= ROWS && (c.dim * size + 127) / 128 * 128 * ROWS <= H_BYTES;
}

size_t xent_few_scratch(const XentCall &c) { return (size_t)c.num_cus * ROWS * sizeof(float2); }

hipError_t launch_xent_few(hipStream_t s, const XentCall &c, char *scratch) {
    const int64_t size = c.bf16 ? 2 : 4;
    const uint64_t all = (uint64_t)(c.dim * size) | (uint64_t)(c.w_stride * size) |
                         reinterpret_cast<uintptr_t>(c.w);
    if (all % 16 == 0)
        return c.bf16 ? run<__bf16, 16>(s, c, scratch) : run<float, 16>(s, c, scratch);
    if (all % 4 == 0) return c.bf16 ? run<__bf16, 4>(s, c, scratch) : run<float, 4>(s, c, scratch);
    return run<__bf16, 2>(s, c, scratch);
}

}  // namespace mbk
