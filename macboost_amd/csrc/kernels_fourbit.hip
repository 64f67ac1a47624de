// kernels_fourbit.hip — scores of many classes with class vectors in 4 bits and a scale for each
// group of a vector's elements (mbk_fourbit_pack, mbk_fourbit_scores).
//
// An element is code * scale with a code of -8..7 and a scale of bf16: 3 bits (or a power of
// two) times 8, which f16 holds without rounding once a power of two has brought a class's
// largest scale near the top of f16's range.  So the scores are one product on the 16-bit
// matrix instruction over all of dim, with codes turned into f16 in registers; the powers of two
// of the class and of the row of h come back in the end.
//
// Layout of W in 4 bits, tiles of 16 classes by blocks of 128 elements, as the matrix
// instruction's lanes take them: lane q * 16 + c of a block holds 16 bytes of class c, its word j
// the elements 32 j + 8 q + i, i = 0..7, in nibble (i >> 1) + 4 (i & 1), a code plus 8.
// Behind them the scales as f16, [tile][block][class][groups of the block], and behind those each
// class's exponent as int32, [tile][class].
#include <algorithm>

#include "grid.hpp"
#include "mbk.h"
#include "ops.h"

namespace mbk {

namespace {

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int BLOCK = 128;           // elements of a class in a block
constexpr int TILE = 16;             // classes
// The largest scale of a class lies in [2^TOP, 2^(TOP + 1)): 8 of them are below f16's largest.
constexpr int TOP = 11;
// The largest |h| of a row likewise.
constexpr int H_TOP = 14;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

__device__ __forceinline__ float bf16_rounded(float v) { return (float)(__bf16)v; }

// floor(log2 |v|), 0 for 0, 127 for an infinity.
__device__ __forceinline__ int exponent(float v) {
    return v == 0.0f ? 0 : v < __builtin_inff() ? ilogbf(v) : 127;
}

// A workgroup a tile and a run of its blocks; a wavefront a block: two passes over W, the
// first for the largest scale of each class.
template <typename T>
__global__ __launch_bounds__(256) void k_fourbit_pack(FourbitShape s, const T *__restrict__ w,
                                                 int64_t stride, uint32_t *__restrict__ codes,
                                                 _Float16 *__restrict__ scales,
                                                 int32_t *__restrict__ exponents) {
    __shared__ float most[256];
    const int64_t tile = group_id();
    if (tile * TILE >= s.classes) return;
    const int c = threadIdx.x & 15, part = threadIdx.x >> 4;       // 16 parts a class
    const int64_t cls = tile * TILE + c;
    const bool real = cls < s.classes;
    const T *row = w + (real ? cls : 0) * stride;
    const int blocks = s.blocks, per = BLOCK / s.group, groups = blocks * per;
    const auto scale_of = [&](int g) {
        float m = 0.0f;
        bool finite = true;
        if (real)
            for (int k = g * s.group; k < min(s.dim, (g + 1) * s.group); ++k) {
                const float v = fabsf(to_f32(row[k]));
                finite &= v < __builtin_inff();
                m = fmaxf(m, v);
            }
        // f32(1 / 7); NaN reaches every score of the class
        return finite ? bf16_rounded(m * 0x1.24924ap-3f) : __builtin_nanf("");
    };
    float m = 0.0f;
    for (int g = part; g < groups; g += 16) m = fmaxf(m, scale_of(g));
    most[threadIdx.x] = m;
    __syncthreads();
    for (int p = 0; p < 16; ++p) m = fmaxf(m, most[p * 16 + c]);
    const int e = exponent(m) - TOP;
    if (part == 0) exponents[cls] = e;
    for (int g = part; g < groups; g += 16) {
        const float scale = scale_of(g);
        scales[((tile * blocks + g / per) * TILE + c) * per + g % per] =
            (_Float16)ldexpf(scale, -e);
        for (int k0 = g * s.group; k0 < (g + 1) * s.group; k0 += 8) {
            uint32_t word = 0;
            for (int i = 0; i < 8; ++i) {
                float code = 0.0f;
                if (real && k0 + i < s.dim && scale > 0.0f)
                    code = rintf(to_f32(row[k0 + i]) / scale);
                const uint32_t n = (uint32_t)((int)fminf(fmaxf(code, -8.0f), 7.0f) + 8);
                word |= n << (4 * ((i >> 1) + 4 * (i & 1)));
            }
            const int block = k0 / BLOCK, j = k0 % BLOCK / 32, q = k0 % 32 / 8;
            codes[(((tile * blocks + block) * 64) + q * 16 + c) * 4 + j] = word;
        }
    }
}

// h as columns of f16 terms: column r of bf16 rows, columns 2 r and 2 r + 1 of f32 rows (the row
// and 2^11 times what its f16 leaves, 22 bits together), a power of two apart that brings the row's
// largest near the top of f16's range.  As the matrix instruction takes them: [column tile][32
// elements][lane][8], lane q * 16 + column.  A workgroup a row.
template <typename T>
__global__ __launch_bounds__(256) void k_fourbit_columns(const T *__restrict__ h, int64_t stride,
                                                    int64_t rows, int32_t dim, int32_t steps,
                                                    _Float16 *__restrict__ columns,
                                                    int32_t *__restrict__ exponents) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
    __shared__ float most[4];
    const int64_t r = group_id();                    // rows of whole tiles of columns
    if (r * TERMS >= (rows * TERMS + 15) / 16 * 16) return;
    const T *row = h + (r < rows ? r : 0) * stride;
    const int n = r < rows ? dim : 0;
    float m = 0.0f;
    for (int k = threadIdx.x; k < n; k += 256) m = fmaxf(m, fabsf(to_f32(row[k])));
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    const int e = exponent(m) - H_TOP;
    if (threadIdx.x == 0 && r < rows) exponents[r] = e;
    for (int k = threadIdx.x; k < steps * 32; k += 256) {
        const float v = k < n ? ldexpf(to_f32(row[k]), -e) : 0.0f;
        const int64_t col = r * TERMS;
        _Float16 *to = columns + (((col / 16) * steps + k / 32) * 64 + k % 32 / 8 * 16 + col % 16) * 8 +
                       k % 8;
        const _Float16 t = (_Float16)v;
        to[0] = t;
        if constexpr (TERMS == 2) to[8] = (_Float16)((v - (float)t) * 2048.0f);
    }
}

// Eight codes of a word times the scale, exact.
__device__ __forceinline__ half8 weights(uint32_t word, _Float16 scale) {
    const half2 s = {scale, scale};
    half8 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // 1024 + n or 1024 + 16 n in the low bits of an f16
        const uint32_t w = i < 2 ? word : word >> 8;
        const uint32_t bits = (w & (i & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
        half2 v = __builtin_bit_cast(half2, bits);
        if (i & 1) {
            const half2 by = {(_Float16)0.0625f, (_Float16)0.0625f};
            const half2 minus = {(_Float16)-72.0f, (_Float16)-72.0f};
            v = __builtin_elementwise_fma(v, by, minus);
        } else {
            const half2 minus = {(_Float16)-1032.0f, (_Float16)-1032.0f};
            v = v + minus;
        }
        v = v * s;
        out[2 * i] = v[0];
        out[2 * i + 1] = v[1];
    }
    return out;
}

// A wavefront two tiles of classes by CT tiles of columns.
template <int TERMS, int CT>
__global__ __launch_bounds__(256) void k_fourbit_scores(FourbitCall c, const _Float16 *__restrict__ columns,
                                                   const int32_t *__restrict__ row_exponents) {
    constexpr int TC = 2;
    const int lane = threadIdx.x & 63;
    const int64_t tiles = (c.shape.classes + TILE - 1) / TILE;
    const int64_t tile0 = ((int64_t)group_id() * 4 + (threadIdx.x >> 6)) * TC;
    if (tile0 >= tiles) return;
    const int blocks = c.shape.blocks, per = BLOCK / c.shape.group;
    const int64_t col_tiles = (c.rows * TERMS + 15) / 16;
    for (int64_t ct0 = (int64_t)blockIdx.y * CT; ct0 < col_tiles; ct0 += (int64_t)gridDim.y * CT) {
        float4v acc[TC][CT];
#pragma unroll
        for (int t = 0; t < TC; ++t)
#pragma unroll
            for (int x = 0; x < CT; ++x) acc[t][x] = float4v{0, 0, 0, 0};
        for (int b = 0; b < blocks; ++b) {
            uint4v word[TC];
            _Float16 scale[TC][4];
#pragma unroll
            for (int t = 0; t < TC; ++t) {
                const int64_t at = min(tile0 + t, tiles - 1) * blocks + b;
                word[t] = reinterpret_cast<const uint4v *>(c.codes)[at * 64 + lane];
                const _Float16 *s = c.scales + (at * TILE + (lane & 15)) * per;
#pragma unroll
                for (int j = 0; j < 4; ++j) scale[t][j] = s[j * per / 4];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                half8 a[TC];
#pragma unroll
                for (int t = 0; t < TC; ++t) a[t] = weights(word[t][j], scale[t][j]);
#pragma unroll
                for (int x = 0; x < CT; ++x) {
                    const int64_t ct = min(ct0 + x, col_tiles - 1);
                    const half8 h = reinterpret_cast<const half8 *>(
                        columns)[(ct * blocks * 4 + b * 4 + j) * 64 + lane];
#pragma unroll
                    for (int t = 0; t < TC; ++t)
                        acc[t][x] =
                            __builtin_amdgcn_mfma_f32_16x16x32_f16(a[t], h, acc[t][x], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < TC; ++t) {
            const int64_t cls = (tile0 + t) * TILE + (lane >> 4) * 4;
#pragma unroll
            for (int x = 0; x < CT; ++x) {
                float4v z = acc[t][x];
                if constexpr (TERMS == 2)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        z[i] = __builtin_fmaf(__shfl_xor(z[i], 1, 64), 0x1p-11f, z[i]);
                const int64_t row = ((ct0 + x) * 16 + (lane & 15)) / TERMS;
                const bool mine = (TERMS == 1 || !(lane & 1)) && row < c.rows;
                if (mine && tile0 + t < tiles) {
                    const int re = row_exponents[row];
                    float *to = c.scores + row * c.score_stride + cls;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (cls + i < c.shape.classes) {
                            float v = ldexpf(z[i], c.exponents[cls + i] + re);
                            if (c.bias) {
                                const float b = c.bias[cls + i];
                                v = b == -__builtin_inff() ? b : v + b;
                            }
                            to[i] = v;
                        }
                }
            }
        }
    }
}

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

size_t code_bytes(const FourbitShape &s) {
    return (size_t)((s.classes + TILE - 1) / TILE) * s.blocks * 1024;
}
size_t scale_bytes(const FourbitShape &s) {
    return (size_t)((s.classes + TILE - 1) / TILE) * s.blocks * TILE * (BLOCK / s.group) * 2;
}

// Columns of h that are held: 64 MB of them, or 16 rows.
int64_t rows_a_turn(const FourbitCall &c) {
    const int64_t row = (int64_t)c.shape.blocks * BLOCK * (c.bf16 ? 2 : 4);
    return std::max<int64_t>(16, std::min<int64_t>(16384, ((int64_t)64 << 20) / row) / 16 * 16);
}
size_t column_bytes(const FourbitCall &c, size_t rows) {
    return (rows * (c.bf16 ? 1 : 2) + 15) / 16 * c.shape.blocks * 4096;
}

template <int TERMS, int CT>
hipError_t scores(hipStream_t st, const FourbitCall &c, const _Float16 *columns, const int32_t *e) {
    const int64_t tiles = (c.shape.classes + TILE - 1) / TILE;
    const int64_t col_tiles = (c.rows * TERMS + 15) / 16;
    const int64_t turns = (col_tiles + CT - 1) / CT;
    hipLaunchKernelGGL((k_fourbit_scores<TERMS, CT>), grid_of((tiles + 7) / 8, (uint32_t)std::min<int64_t>(turns, 32768)),
                       dim3(256), 0, st, c, columns, e);
    return hipGetLastError();
}

template <typename T>
hipError_t run(hipStream_t st, const FourbitCall &c, char *scratch) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
    _Float16 *columns = reinterpret_cast<_Float16 *>(scratch);
    const int64_t col_tiles = (c.rows * TERMS + 15) / 16;
    const int steps = c.shape.blocks * 4;
    int32_t *e = reinterpret_cast<int32_t *>(scratch + column_bytes(c, (size_t)c.rows));
    hipLaunchKernelGGL((k_fourbit_columns<T>), grid_of(col_tiles * 16 / TERMS), dim3(256), 0, st,
                       static_cast<const T *>(c.h), c.h_stride, c.rows, c.shape.dim, steps, columns,
                       e);
    if (col_tiles <= 1) return scores<TERMS, 1>(st, c, columns, e);
    if (col_tiles <= 2) return scores<TERMS, 2>(st, c, columns, e);
    return scores<TERMS, 4>(st, c, columns, e);
}

}  // namespace

FourbitShape fourbit_shape(int64_t classes, int32_t dim, int32_t group) {
    return {classes, dim, group, (dim + BLOCK - 1) / BLOCK};
}

size_t fourbit_bytes(const FourbitShape &s) {
    return code_bytes(s) + rounded(scale_bytes(s)) +
           (size_t)((s.classes + TILE - 1) / TILE) * TILE * 4;
}

void fourbit_parts(const FourbitShape &s, char *packed, uint32_t **codes, _Float16 **scales,
              int32_t **exponents) {
    *codes = reinterpret_cast<uint32_t *>(packed);
    *scales = reinterpret_cast<_Float16 *>(packed + code_bytes(s));
    *exponents = reinterpret_cast<int32_t *>(packed + code_bytes(s) + rounded(scale_bytes(s)));
}

hipError_t launch_fourbit_pack(hipStream_t st, const FourbitShape &s, bool bf16, const void *w,
                          int64_t stride, char *packed) {
    uint32_t *codes;
    _Float16 *scales;
    int32_t *exponents;
    fourbit_parts(s, packed, &codes, &scales, &exponents);
    const dim3 g = grid_of((s.classes + TILE - 1) / TILE);
    if (bf16)
        hipLaunchKernelGGL((k_fourbit_pack<__bf16>), g, dim3(256), 0, st, s,
                           static_cast<const __bf16 *>(w), stride, codes, scales, exponents);
    else
        hipLaunchKernelGGL((k_fourbit_pack<float>), g, dim3(256), 0, st, s,
                           static_cast<const float *>(w), stride, codes, scales, exponents);
    return hipGetLastError();
}

size_t fourbit_scratch(const FourbitCall &c) {
    const size_t rows = (size_t)std::min(c.rows, rows_a_turn(c));
    return column_bytes(c, rows) + 4 * rows;
}

hipError_t launch_fourbit_scores(hipStream_t st, const FourbitCall &c, char *scratch) {
    const int64_t each = rows_a_turn(c);
    const int64_t row = c.h_stride * (c.bf16 ? 2 : 4);
    for (int64_t r = 0; r < c.rows; r += each) {
        FourbitCall part = c;
        part.rows = std::min(each, c.rows - r);
        part.h = static_cast<const char *>(c.h) + r * row;
        part.scores = c.scores + r * c.score_stride;
        const hipError_t e = c.bf16 ? run<__bf16>(st, part, scratch) : run<float>(st, part, scratch);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace mbk
