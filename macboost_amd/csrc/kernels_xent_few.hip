// kernels_xent_few.hip — the many-class loss of up to 32 rows, as in serving or small
// batches: what bounds it is reading W (and writing dW), so W is not packed first.
//
// h lies in LDS whole, as operands of the matrix instruction.  Each wavefront takes tiles
// of 32 classes by itself: their rows are copied straight into its own LDS buffers, 128
// bytes of each at a time and two steps ahead, so that eight wavefronts keep 64 KB
// of a CU on the way and no barrier holds them.  (Rows of odd bf16 elements go through
// registers, one step ahead.)  The product is W h' (classes down,
// rows across): a lane has scores of one row, and keeps its maximum and sum over all
// tiles.  f32 operands go into the f32 matrix instruction as they are: at 1/16 of
// the bf16 rate it still takes less time than W's bytes.  16 x 1024 x 100000 bf16: 55 us, W at
// 4.9 TB/s by the first kernel.  (32 rows are one operand of the instruction: with gradients,
// 32 x 512 x 100000 f32 239 us here and 494 by the kernels for more rows, 32 x 64 x 1000 22 and 37.)
// Copies of 16 bytes a lane where W's rows are aligned to them, else of 4, or by registers:
// 16 x 512 x 100000 f32 63 us by 16 bytes, 84 by 4.
//
// The gradients take a second kernel, with a tile of 32 classes of W in LDS at a time: its
// scores again, G (32 x 32, f32), dW = G' h written at once, and dh += G W kept in
// registers over the tiles and summed over the workgroups at the end.  All of its
// products are of the f32 instruction, so nothing is rounded before the outputs.
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
    sum = sum * exp_of(top - ref) + s2 * exp_of(t2 - ref);
    top = now;
}

// part[workgroup][row]: the maximum of z and the sum of exp(z - it).
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
            s[r] = b == -INFINITY ? -INFINITY : s[r] + b;
            m = fmaxf(m, s[r]);
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        sum *= exp_of(top - ref);
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += exp_of(s[r] - ref);
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

// One wavefront a row: the parts joined, and the label's score from h and W.  lse2: the
// reference and log2 of the sum, +inf for a row that is out (NULL: not wanted).
template <typename T>
__global__ __launch_bounds__(64) void k_few_join(XentCall c, int32_t parts,
                                                 const float2 *__restrict__ part,
                                                 float2 *__restrict__ lse2) {
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
    const LogSum l = log_sum(sum);
    c.lse[i] = lse_of(top, l);
    const bool out = y < 0 || y >= c.classes || wt == 0.0f || none;
    c.loss[i] = out ? 0.0f : wt * loss_of(top, l, dot + by);
    if (lse2) lse2[i] = out ? make_float2(0.0f, INFINITY) : make_float2(top, l.base2);
}

// ---- gradients -------------------------------------------------------------------------
// Element (x, k) of h or of a tile of W in LDS: chunks of 16 bytes of k, each with its 32
// rows; the chunks 528 bytes apart, so that reads along x and along k fall on all banks.
constexpr int CHUNK_BYTES = ROWS * 16 + 16;
constexpr int GRAD_WAVES = 8;
constexpr int G_STRIDE = 33;
template <typename T>
__device__ __forceinline__ float element_of(const char *m, int x, int k) {
    constexpr int PER = 16 / sizeof(T);
    return (float)*reinterpret_cast<const T *>(m + k / PER * CHUNK_BYTES + x * 16 +
                                               k % PER * (int)sizeof(T));
}
// 32 rows of a matrix on their way to LDS, 16 lanes a row: element k of the lane's row is
// row[k], NULL for zeros.  B: bytes that the rows are aligned to.
template <int N> struct Staged {
    u32x4 v[N];
};
template <typename T, int B, int N>
__device__ __forceinline__ void load(Staged<N> &s, int chunks, int dim, const T *row) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = (threadIdx.x & 15) + n * 16, k = c * PER;
        if (c >= chunks) break;
        u32x4 v = {0, 0, 0, 0};
        if (row) {
            if (B == 16) {
                v = *reinterpret_cast<const u32x4 *>(row + k);
            } else if (B == 4 && k + PER <= dim) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = reinterpret_cast<const uint32_t *>(row + k)[i];
            } else {
                T e[PER];
#pragma unroll
                for (int i = 0; i < PER; ++i) e[i] = k + i < dim ? row[k + i] : (T)0.0f;
                __builtin_memcpy(&v, e, sizeof v);
            }
        }
        s.v[n] = v;
    }
}
template <int N>
__device__ __forceinline__ void store(char *m, const Staged<N> &s, int chunks) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = (threadIdx.x & 15) + n * 16;
        if (c >= chunks) break;
        *reinterpret_cast<u32x4 *>(m + c * CHUNK_BYTES + (threadIdx.x >> 4) * 16) = s.v[n];
    }
}

// part_dh[workgroup][row][dim].
// The next tile of W is asked for while this one is worked on.  NB: blocks of 32 columns
// that a wavefront keeps of dh; with one, two workgroups fit a CU's registers (grad_groups).
template <typename T, int B, int NB>
__global__ __launch_bounds__(64 * GRAD_WAVES, NB == 1 ? 4 : 2) void k_few_grad(XentCall c, int64_t tiles,
                                                                 int32_t chunks,
                                                                 const float2 *__restrict__ lse2,
                                                                 float *__restrict__ part_dh) {
    constexpr int PER = 16 / sizeof(T);
    extern __shared__ char lds[];
    char *h = lds, *w = lds + chunks * CHUNK_BYTES;
    float *sums = reinterpret_cast<float *>(w + chunks * CHUNK_BYTES);   // [4][16][64]
    float *g = sums + 4 * 16 * 64;                                       // [row][class]
    const int lane = threadIdx.x & 63, half = lane >> 5, l = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (c.dim + 31) / 32;
    // A row that is out is zeros here: what it holds reaches nothing.  So is one whose lse is not
    // finite: its G is NaN where a class is offered, and 0 times what it holds where none is.
    const int x0 = threadIdx.x >> 4;                 // the row that this lane brings
    Staged<NB * (int)sizeof(T)> staged;
    load<T, sizeof(T)>(staged, chunks, c.dim,
                       x0 < c.rows && fabsf(lse2[x0].y) < INFINITY
                           ? static_cast<const T *>(c.h) + x0 * c.h_stride : nullptr);
    store(h, staged, chunks);
    const auto ask = [&](int64_t t) {
        const int64_t v = t * 32 + x0;
        load<T, B>(staged, chunks, c.dim,
                   v < c.classes && !(c.bias && c.bias[v] == -INFINITY)
                       ? static_cast<const T *>(c.w) + v * c.w_stride : nullptr);
    };
    if (blockIdx.x < tiles) ask(blockIdx.x);
    const float ref = l < c.rows ? lse2[l].x : 0.0f, l2 = l < c.rows ? lse2[l].y : INFINITY;
    const int32_t label = l < c.rows ? c.labels[l] : -1;
    const float wt = l2 == INFINITY ? 0.0f : c.weights ? c.weights[l] : 1.0f;
    f32x16 dh[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) dh[b][r] = 0.0f;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t v0 = t * 32;
        __syncthreads();                             // the last tile's reads
        store(w, staged, chunks);
        __syncthreads();
        if (t + gridDim.x < tiles) ask(t + gridDim.x);
        // scores, classes down and rows across, k in parts of the wavefronts
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
        for (int q = wave; q < (chunks + 1) / 2; q += GRAD_WAVES) {
            const int at = 2 * q + half;
            u32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (at < chunks) {
                a = *reinterpret_cast<const u32x4 *>(w + at * CHUNK_BYTES + l * 16);
                b = *reinterpret_cast<const u32x4 *>(h + at * CHUNK_BYTES + l * 16);
            }
            T x[PER], y[PER];
            __builtin_memcpy(x, &a, 16);
            __builtin_memcpy(y, &b, 16);
#pragma unroll
            for (int e = 0; e < PER; ++e)
                s = __builtin_amdgcn_mfma_f32_32x32x2f32((float)x[e], (float)y[e], s, 0, 0, 0);
        }
        // their sum over the wavefronts, in three rounds of halves, in the first one
#pragma unroll
        for (int n = GRAD_WAVES / 2; n > 0; n >>= 1) {
            if (wave >= n && wave < 2 * n)
#pragma unroll
                for (int r = 0; r < 16; ++r) sums[((wave - n) * 16 + r) * 64 + lane] = s[r];
            __syncthreads();
            if (wave < n)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] += sums[(wave * 16 + r) * 64 + lane];
            __syncthreads();
        }
        if (wave == 0)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int x = (r >> 2) * 8 + half * 4 + (r & 3);
                const int64_t v = v0 + x;
                float b = -INFINITY;
                if (v < c.classes) b = c.bias ? c.bias[v] : 0.0f;
                float p = 0.0f;
                if (l2 != INFINITY && b != -INFINITY) {
                    p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r] + b - ref, LOG2E, -l2));
                    if (v == label) p -= 1.0f;
                    p *= wt;
                }
                g[l * G_STRIDE + x] = p;
            }
        __syncthreads();
        if (c.dbias && threadIdx.x < 32 && v0 + threadIdx.x < c.classes) {
            float sum = 0.0f;
            for (int i = 0; i < ROWS; ++i) sum += g[i * G_STRIDE + threadIdx.x];
            c.dbias[v0 + threadIdx.x] = sum;
        }
        // dW and dh, blocks of 32 columns in turn
        if (c.dw)
            for (int b = wave; b < blocks; b += GRAD_WAVES) {
                const int j = min(b * 32 + l, chunks * PER - 1);
                f32x16 o;
#pragma unroll
                for (int r = 0; r < 16; ++r) o[r] = 0.0f;
#pragma unroll 4
                for (int k = 0; k < ROWS; k += 2)
                    o = __builtin_amdgcn_mfma_f32_32x32x2f32(g[(k + half) * G_STRIDE + l],
                                                             element_of<T>(h, k + half, j), o, 0, 0,
                                                             0);
                if (b * 32 + l < c.dim)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int64_t v = v0 + (r >> 2) * 8 + half * 4 + (r & 3);
                        if (v < c.classes)
                            static_cast<T *>(c.dw)[v * c.w_stride + b * 32 + l] = (T)o[r];
                    }
            }
        if (c.dh)
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int b = wave + n * GRAD_WAVES;
                if (b >= blocks) break;
                const int j = min(b * 32 + l, chunks * PER - 1);
#pragma unroll 4
                for (int k = 0; k < 32; k += 2)
                    dh[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(g[l * G_STRIDE + k + half],
                                                                 element_of<T>(w, k + half, j),
                                                                 dh[n], 0, 0, 0);
            }
    }
    if (!c.dh) return;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int j = (wave + n * GRAD_WAVES) * 32 + l;
        if (j >= c.dim) continue;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = (r >> 2) * 8 + half * 4 + (r & 3);
            if (i < c.rows) part_dh[((int64_t)blockIdx.x * c.rows + i) * c.dim + j] = dh[n][r];
        }
    }
}

// The workgroups' parts of 64 elements of dh added, by four wavefronts.
template <typename T>
__global__ __launch_bounds__(256) void k_few_join_dh(XentCall c, int32_t parts,
                                                     const float *__restrict__ part) {
    __shared__ float sums[256];
    const int64_t at = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63), all = c.rows * c.dim;
    float sum = 0.0f;
    if (at < all)
#pragma unroll 8
        for (int p = threadIdx.x >> 6; p < parts; p += 4) sum += part[p * all + at];
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x >= 64 || at >= all) return;
    for (int w = 1; w < 4; ++w) sum += sums[w * 64 + threadIdx.x];
    static_cast<T *>(c.dh)[at / c.dim * c.h_stride + at % c.dim] = (T)sum;
}

// Scratch: the parts of the rows, lse2, the parts of dh.
size_t part_bytes(const XentCall &c) { return (size_t)c.num_cus * ROWS * sizeof(float2); }

// Columns that a workgroup of k_few_grad keeps with one block a wavefront.
constexpr int ONE_BLOCK = 32 * GRAD_WAVES;
int32_t grad_chunks(const XentCall &c) { return (c.dim * (c.bf16 ? 2 : 4) + 15) / 16; }
size_t grad_lds(const XentCall &c) {
    return (size_t)2 * grad_chunks(c) * CHUNK_BYTES + 4 * (4 * 16 * 64 + ROWS * G_STRIDE);
}
// Two workgroups a CU where they fit its LDS, too (f32: up to 232 outputs).
int grad_groups(const XentCall &c) {
    return (c.dim <= ONE_BLOCK && 2 * grad_lds(c) <= LDS_BYTES ? 2 : 1) * c.num_cus;
}

template <typename T, int B, int NB>
hipError_t run_grad(hipStream_t s, const XentCall &c, const float2 *lse2, float *part_dh) {
    const hipError_t e = allow_all_lds(reinterpret_cast<const void *>(k_few_grad<T, B, NB>));
    if (e != hipSuccess) return e;
    const int32_t chunks = grad_chunks(c);
    const int64_t tiles = (c.classes + 31) / 32;
    const uint32_t groups = (uint32_t)std::min<int64_t>(grad_groups(c), tiles);
    hipLaunchKernelGGL((k_few_grad<T, B, NB>), dim3(groups), dim3(64 * GRAD_WAVES), grad_lds(c), s, c,
                       tiles, chunks, lse2, part_dh);
    if (c.dh)
        hipLaunchKernelGGL((k_few_join_dh<T>), dim3((uint32_t)((c.rows * c.dim + 63) / 64)),
                           dim3(256), 0, s, c, (int32_t)groups, part_dh);
    return hipGetLastError();
}

template <typename T, int B> hipError_t run(hipStream_t s, const XentCall &c, char *scratch) {
    const hipError_t e = allow_all_lds(reinterpret_cast<const void *>(k_few_stats<T, B>));
    if (e != hipSuccess) return e;
    const int64_t tiles = (c.classes + 31) / 32;
    const int32_t steps = (int32_t)((c.dim * sizeof(T) + 127) / 128);
    const uint32_t groups = (uint32_t)std::min<int64_t>(c.num_cus, (tiles + WAVES - 1) / WAVES);
    float2 *part = reinterpret_cast<float2 *>(scratch);
    float2 *lse2 = reinterpret_cast<float2 *>(scratch + part_bytes(c));
    float *part_dh = reinterpret_cast<float *>(lse2 + ROWS);
    hipLaunchKernelGGL((k_few_stats<T, B>), dim3(groups), dim3(64 * WAVES), LDS_BYTES, s, c, tiles,
                       steps, part);
    hipLaunchKernelGGL((k_few_join<T>), dim3((uint32_t)c.rows), dim3(64), 0, s, c, (int32_t)groups,
                       part, c.grad ? lse2 : nullptr);
    if (!c.grad) return hipGetLastError();
    if (c.dim <= ONE_BLOCK) return run_grad<T, B, 1>(s, c, lse2, part_dh);
    if constexpr (sizeof(T) == 2)
        if (c.dim > 2 * ONE_BLOCK) return run_grad<T, B, 4>(s, c, lse2, part_dh);
    return run_grad<T, B, 2>(s, c, lse2, part_dh);
}

}  // namespace

// h must fit the LDS beside the buffers.
bool xent_few(const XentCall &c) {
    const int64_t size = c.bf16 ? 2 : 4;
    return c.rows <= ROWS && (c.dim * size + 127) / 128 * 128 * ROWS <= H_BYTES;
}

size_t xent_few_scratch(const XentCall &c) {
    return part_bytes(c) + 8 * ROWS + (c.grad ? (size_t)4 * grad_groups(c) * c.rows * c.dim : 0);
}

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
