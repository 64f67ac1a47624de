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
// Behind them the scales as f16, [tile][four blocks][class][groups of the four blocks], so that a
// lane loads those of four blocks at once, and behind those each class's exponent as int32,
// [tile][class].
#include <algorithm>
#include <type_traits>

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

// Eight elements of a row from k on, 0 behind its end.
template <typename T>
__device__ __forceinline__ void eight(const T *row, int k, int dim, bool wide, float (&v)[8]) {
    if (wide && k + 8 <= dim) {
        constexpr int N = 16 / sizeof(T);
        typedef T V __attribute__((ext_vector_type(N)));
#pragma unroll
        for (int x = 0; x < 8 / N; ++x) {
            const V part = reinterpret_cast<const V *>(row + k)[x];
#pragma unroll
            for (int i = 0; i < N; ++i) v[x * N + i] = to_f32(part[i]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < dim ? to_f32(row[k + i]) : 0.0f;
}

// A workgroup a tile of classes, a wavefront a block of it at a time, in the lanes that hold its
// codes: the scales first, for the class's exponent, and then all again.  100000 x 1024 bf16 90
// us, f32 149, the second reading from L2.
constexpr int PACK_WAVES = 4;
template <typename T, int PER>
__global__ __launch_bounds__(64 * PACK_WAVES) void k_fourbit_pack(
    FourbitShape s, const T *__restrict__ w, int64_t stride, bool wide, uint4v *__restrict__ codes,
    _Float16 *__restrict__ scales, int32_t *__restrict__ exponents) {
    __shared__ float most[PACK_WAVES][TILE];
    const int64_t tile = group_id();
    if (tile * TILE >= s.classes) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    const int64_t cls = tile * TILE + c;
    const T *row = w + (cls < s.classes ? cls : 0) * stride;
    const int dim = cls < s.classes ? s.dim : 0;
    const int quads = (s.blocks + 3) / 4;
    // The lane's 32 elements of a block and the scales of its groups.
    const auto block = [&](int b, float (&v)[4][8], float (&scale)[PER]) {
        float m[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            eight(row, b * BLOCK + j * 32 + q * 8, dim, wide, v[j]);
            m[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = fabsf(v[j][i]);
                m[j] = fmaxf(m[j], x < __builtin_inff() ? x : __builtin_inff());
            }
            m[j] = fmaxf(m[j], __shfl_xor(m[j], 16, 64));
            m[j] = fmaxf(m[j], __shfl_xor(m[j], 32, 64));
        }
#pragma unroll
        for (int g = 0; g < PER; ++g) {
            float all = 0.0f;
#pragma unroll
            for (int j = g * 4 / PER; j < (g + 1) * 4 / PER; ++j) all = fmaxf(all, m[j]);
            // f32(1 / 7); what is not finite reaches every score of the class
            scale[g] = all < __builtin_inff() ? bf16_rounded(all * 0x1.24924ap-3f)
                                              : __builtin_nanf("");
        }
    };
    float v[4][8], scale[PER], m = 0.0f;
    for (int b = wave; b < s.blocks; b += PACK_WAVES) {
        block(b, v, scale);
#pragma unroll
        for (int g = 0; g < PER; ++g) m = fmaxf(m, scale[g]);
    }
    if (q == 0) most[wave][c] = m;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < PACK_WAVES; ++x) m = fmaxf(m, most[x][c]);
    const int e = exponent(m) - TOP;
    if (wave == 0 && q == 0) exponents[cls] = e;
    for (int b = wave; b < quads * 4; b += PACK_WAVES) {
#pragma unroll
        for (int g = 0; g < PER; ++g) scale[g] = 0.0f;
        if (b < s.blocks) {
            block(b, v, scale);
            uint4v words;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float by = scale[j * PER / 4];
                words[j] = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float code = by > 0.0f ? rintf(v[j][i] / by) : 0.0f;
                    words[j] |= (uint32_t)((int)fminf(fmaxf(code, -8.0f), 7.0f) + 8)
                                << (4 * ((i >> 1) + 4 * (i & 1)));
                }
            }
            codes[(tile * s.blocks + b) * 64 + lane] = words;
        }
        if (q == 0)
#pragma unroll
            for (int g = 0; g < PER; ++g)
                scales[(((tile * quads + b / 4) * TILE + c) * 4 + b % 4) * PER + g] =
                    (_Float16)ldexpf(scale[g], -e);
    }
}

// h as columns of f16 terms: column r of bf16 rows, columns 2 r and 2 r + 1 of f32 rows (the row
// and 2^11 times what its f16 leaves, 22 bits together), a power of two apart that brings the row's
// largest near the top of f16's range.  As the matrix instruction takes them: [column tile][32
// elements][lane][8], lane q * 16 + column with the elements 8 q + i.
template <typename T> constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;

// A wavefront's part of a tile of columns: the steps first, first + each, ... of the largest |h|
// of the lane's row, over all of its lanes.
template <typename T>
__device__ __forceinline__ float largest(const T *row, int dim, bool wide, int steps, int first,
                                         int each) {
    const int q = (threadIdx.x & 63) >> 4;
    float m = 0.0f;
    for (int s = first; s < steps; s += each) {
        float v[8];
        eight(row, s * 32 + q * 8, dim, wide, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
    }
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    return fmaxf(m, __shfl_xor(m, 32, 64));
}

// The same steps as terms, a KB a step.
template <typename T>
__device__ __forceinline__ void terms(const T *row, int dim, bool wide, int steps, int first,
                                      int each, int e, half8 *to) {
    const int lane = threadIdx.x & 63;
    for (int s = first; s < steps; s += each) {
        float v[8];
        eight(row, s * 32 + (lane >> 4) * 8, dim, wide, v);
        half8 out;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = ldexpf(v[i], -e);
            const _Float16 t = (_Float16)x;
            out[i] = TERMS<T> == 2 && (lane & 1) ? (_Float16)((x - (float)t) * 2048.0f) : t;
        }
        to[s * 64 + lane] = out;
    }
}

// Where many columns are made for all workgroups: a workgroup a tile of columns, two passes over its
// rows (201 x 777 f32 as 26 tiles: 5 us, the latency of both).
constexpr int COLUMN_WAVES = 16;
template <typename T>
__global__ __launch_bounds__(64 * COLUMN_WAVES) void k_fourbit_columns(
    const T *__restrict__ h, int64_t stride, int64_t rows, int32_t dim, bool wide, int32_t steps,
    half8 *__restrict__ columns, int32_t *__restrict__ exponents) {
    __shared__ float most[COLUMN_WAVES][16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t tile = group_id(), r = (tile * 16 + (lane & 15)) / TERMS<T>;
    if (tile * 16 >= rows * TERMS<T>) return;
    const T *row = h + (r < rows ? r : 0) * stride;
    const int n = r < rows ? dim : 0;
    const float m = largest(row, n, wide, steps, wave, COLUMN_WAVES);
    if (lane < 16) most[wave][lane] = m;
    __syncthreads();
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < COLUMN_WAVES; ++w) all = fmaxf(all, most[w][lane & 15]);
    const int e = exponent(all) - H_TOP;
    if (wave == 0 && lane < 16 && r < rows) exponents[r] = e;
    terms(row, n, wide, steps, wave, COLUMN_WAVES, e, columns + tile * steps * 64);
}

// Constants of weights() in registers, so that a mask and the exponent's bits are one instruction
// (which takes no literals).
struct Unpack {
    uint32_t low, high;              // masks of the nibbles
    uint32_t exponent;               // f16's 1024
    __device__ __forceinline__ Unpack() {
        asm("s_mov_b32 %0, 0x000F000F" : "=s"(low));
        asm("s_mov_b32 %0, 0x00F000F0" : "=s"(high));
        asm("v_mov_b32 %0, 0x64006400" : "=v"(exponent));
    }
};

// Eight codes of a word times the scale, exact.
__device__ __forceinline__ half8 weights(const Unpack &u, uint32_t word, _Float16 scale) {
    const half2 s = {scale, scale};
    half8 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // 1024 + n or 1024 + 16 n in the low bits of an f16
        const uint32_t bits = ((i < 2 ? word : word >> 8) & (i & 1 ? u.high : u.low)) | u.exponent;
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

// Words and scales of a class tile's blocks.
template <int PER> struct Scales {
    half8 x[PER < 2 ? 1 : PER / 2];                  // of four blocks; PER 1: half of it
};
template <int PER>
__device__ __forceinline__ Scales<PER> scales_of(const _Float16 *scales, int64_t quad) {
    const _Float16 *s = scales + (quad * TILE + (threadIdx.x & 15)) * 4 * PER;
    Scales<PER> out;
    if constexpr (PER == 1) {
        typedef _Float16 half4 __attribute__((ext_vector_type(4)));
        const half4 v = *reinterpret_cast<const half4 *>(s);
        out.x[0] = half8{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
    } else {
#pragma unroll
        for (int i = 0; i < PER / 2; ++i) out.x[i] = reinterpret_cast<const half8 *>(s)[i];
    }
    return out;
}
// Of word j of block i.
template <int PER>
__device__ __forceinline__ _Float16 scale_at(const Scales<PER> &s, int i, int j) {
    const int at = i * PER + j * PER / 4;
    return s.x[at / 8][at % 8];
}

__device__ __forceinline__ float other_term(float v) {       // the neighbouring column's
    return __builtin_bit_cast(
        float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
}

// What the scores of a tile of classes end with: a lane's classes, their exponents and biases.  N
// terms a row: with two a column's lanes have two of its four classes each.  Loaded before the
// first scores are written, since loads between the stores wait one by one.
template <int N> struct Ends {
    static constexpr int EACH = 4 / N;
    int64_t cls;
    int e[EACH];
    float b[EACH];
};
template <int N>
__device__ __forceinline__ Ends<N> ends_of(const FourbitCall &c, int64_t tile) {
    const int lane = threadIdx.x & 63;
    Ends<N> out;
    out.cls = tile * TILE + (lane >> 4) * 4 + (N == 2 && (lane & 1) ? 2 : 0);
#pragma unroll
    for (int i = 0; i < Ends<N>::EACH; ++i) {
        const bool real = out.cls + i < c.shape.classes;
        out.e[i] = real ? c.exponents[out.cls + i] : 0;
        out.b[i] = real && c.bias ? c.bias[out.cls + i] : 0.0f;
    }
    return out;
}

// The scores of a lane's classes and row.
template <int N>
__device__ __forceinline__ void scores_of(const FourbitCall &c, const float4v &z,
                                          const Ends<N> &end, int row_exponent,
                                          float (&v)[Ends<N>::EACH]) {
    if constexpr (N == 2) {
        const bool odd = threadIdx.x & 1;
        const float a = other_term(odd ? z[0] : z[2]), b = other_term(odd ? z[1] : z[3]);
        v[0] = odd ? __builtin_fmaf(z[2], 0x1p-11f, a) : __builtin_fmaf(a, 0x1p-11f, z[0]);
        v[1] = odd ? __builtin_fmaf(z[3], 0x1p-11f, b) : __builtin_fmaf(b, 0x1p-11f, z[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = z[i];
    }
#pragma unroll
    for (int i = 0; i < Ends<N>::EACH; ++i) {
        v[i] = ldexpf(v[i], end.e[i] + row_exponent);
        if (c.bias) v[i] = end.b[i] == -__builtin_inff() ? end.b[i] : v[i] + end.b[i];
    }
}

// E scores of a row from class cls on, at any address of a float.
template <int E>
__device__ __forceinline__ void put_scores(const FourbitCall &c, int64_t row, int64_t cls,
                                           const float (&v)[E], bool streamed) {
    if (row >= c.rows) return;
    float *to = c.scores + row * c.score_stride + cls;
    if (cls + E <= c.shape.classes) {
        typedef float V __attribute__((ext_vector_type(E), aligned(4)));
        V out;
#pragma unroll
        for (int i = 0; i < E; ++i) out[i] = v[i];
        put(to, out, streamed);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (cls + i < c.shape.classes) to[i] = v[i];
    }
}

template <int N>
__device__ __forceinline__ void write_scores(const FourbitCall &c, const float4v &z,
                                             const Ends<N> &end, int64_t column,
                                             int row_exponent) {
    float v[Ends<N>::EACH];
    scores_of<N>(c, z, end, row_exponent, v);
    put_scores(c, column / N, end.cls, v, false);
}

// ---- few columns: reading W is the work ------------------------------------------------
// All columns lie in LDS, made there by each workgroup: [step][q][column], without the columns
// that no row has, in whose place the matrix instruction gets the last one's.  A wavefront streams
// its tiles of classes, four blocks at a time and two such reads ahead; `ks` wavefronts share a
// tile's blocks where there are few tiles.  Tiles go to the workgroups in turn, so that no CU has
// two more than another.
// 16 x 1024 by 100000 classes, 53 MB of W: 18.3 us with changing inputs, 19.4 under the
// profiler, of which 4 are the columns and about 4 unpacking that does not hide behind the stream;
// vector units busy 28 %, the matrix cores 5.  1 x 64 by 1000: 5.3 us, latency.
constexpr int FEW_WAVES = 8, FEW_THREADS = 64 * FEW_WAVES;
constexpr int FEW_HEAD = 1024;       // bytes of LDS before the columns, for up to 32 rows' exponents
constexpr int KEPT = 4;              // eights of h that a thread keeps from the maximum on
template <typename T, int CT, int PER>
__global__ __launch_bounds__(FEW_THREADS, 4) void k_fourbit_few(FourbitCall c, int32_t ks,
                                                                int32_t log2_rows) {
    extern __shared__ half8 lds[];
    int *exponents = reinterpret_cast<int *>(lds);   // [row]
    half8 *columns = lds + FEW_HEAD / 16;
    constexpr int N = TERMS<T>;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t tiles = (c.shape.classes + TILE - 1) / TILE;
    const int blocks = c.shape.blocks, quads = (blocks + 3) / 4;
    const int part = wave % ks;
    const int first = part * quads / ks, last = (part + 1) * quads / ks;
    const int64_t turn = (int64_t)gridDim.x * (FEW_WAVES / ks);
    const int width = (int)c.rows * N;               // columns
    const Unpack unpack;

    // a thread's row of h, and its eights of it: the first ones stay in registers
    const int my_row = threadIdx.x & ((1 << log2_rows) - 1);
    const int eights = blocks * (BLOCK / 8), each = FEW_THREADS >> log2_rows;
    const int first_eight = threadIdx.x >> log2_rows;
    const bool has_row = my_row < c.rows;
    const T *row = static_cast<const T *>(c.h) + (has_row ? my_row : 0) * c.h_stride;
    const int n = has_row ? c.shape.dim : 0;
    float kept[KEPT][8], most = 0.0f;
#pragma unroll
    for (int i = 0; i < KEPT; ++i) eight(row, (first_eight + i * each) * 8, n, c.wide_h, kept[i]);

    struct Place {
        int64_t tile;
        int quad;
    };
    struct Buffer {
        uint4v word[4];
        Scales<PER> scale;
    };
    const auto after = [&](Place p) {
        return p.quad + 1 < last ? Place{p.tile, p.quad + 1} : Place{p.tile + turn, first};
    };
    const auto fetch = [&](Buffer &b, const Place &p) {
        if (p.tile >= tiles) return;
        const uint4v *from =
            reinterpret_cast<const uint4v *>(c.codes) + (p.tile * blocks + p.quad * 4) * 64;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p.quad * 4 + i < blocks) b.word[i] = from[i * 64 + lane];
        b.scale = scales_of<PER>(c.scales, p.tile * quads + p.quad);
    };
    Place at{(int64_t)(wave / ks) * gridDim.x + blockIdx.x, first};
    Place ahead = after(at);
    Buffer x0, x1, x2;
    fetch(x0, at);
    fetch(x1, ahead);

#pragma unroll
    for (int i = 0; i < KEPT; ++i)
#pragma unroll
        for (int x = 0; x < 8; ++x) most = fmaxf(most, fabsf(kept[i][x]));
    for (int g = first_eight + KEPT * each; g < eights; g += each) {
        float v[8];
        eight(row, g * 8, n, c.wide_h, v);
#pragma unroll
        for (int x = 0; x < 8; ++x) most = fmaxf(most, fabsf(v[x]));
    }
    for (int o = 1 << log2_rows; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    // [wave][row] where the columns come
    float *meet = reinterpret_cast<float *>(columns);
    if (lane < 1 << log2_rows) meet[(wave << log2_rows) + lane] = most;
    __syncthreads();
    for (int w = 0; w < FEW_WAVES; ++w) most = fmaxf(most, meet[(w << log2_rows) + my_row]);
    __syncthreads();
    const int e = exponent(most) - H_TOP;
    if (threadIdx.x < c.rows) exponents[threadIdx.x] = e;
    const auto put = [&](int g, const float (&v)[8]) {
        half8 t, rest;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const float y = ldexpf(v[x], -e);
            t[x] = (_Float16)y;
            rest[x] = (_Float16)((y - (float)t[x]) * 2048.0f);
        }
        half8 *to = columns + g * width + my_row * N;
        to[0] = t;
        if constexpr (N == 2) to[1] = rest;
    };
    if (has_row) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i)
            if (first_eight + i * each < eights) put(first_eight + i * each, kept[i]);
        for (int g = first_eight + KEPT * each; g < eights; g += each) {
            float v[8];
            eight(row, g * 8, n, c.wide_h, v);
            put(g, v);
        }
    }
    __syncthreads();
    const half8 *mine[CT];                           // the lane's column of step 0
    int re[CT];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
        const int column = min(x * 16 + (lane & 15), width - 1);
        mine[x] = columns + (lane >> 4) * width + column;
        re[x] = exponents[column / N];
    }

    float4v acc[CT];
#pragma unroll
    for (int x = 0; x < CT; ++x) acc[x] = float4v{0, 0, 0, 0};
    Ends<N> end;
    // One read's blocks; false behind the last one.
    const auto step = [&](const Buffer &b, Buffer &next) {
        if (at.tile >= tiles) return false;
        const Place then = after(ahead);
        fetch(next, then);
        if (at.quad == first) end = ends_of<N>(c, at.tile);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (at.quad * 4 + i >= blocks) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j && (at.quad * 4 + i) * BLOCK + j * 32 >= c.shape.dim) break;
                const half8 a = weights(unpack, b.word[i][j], scale_at<PER>(b.scale, i, j));
#pragma unroll
                for (int x = 0; x < CT; ++x)
                    acc[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        a, mine[x][((at.quad * 4 + i) * 4 + j) * 4 * width], acc[x], 0, 0, 0);
            }
        }
        if (at.quad + 1 == last && ks == 1) {
#pragma unroll
            for (int x = 0; x < CT; ++x) {
                write_scores<N>(c, acc[x], end, x * 16 + (lane & 15), re[x]);
                acc[x] = float4v{0, 0, 0, 0};
            }
        }
        at = ahead;
        ahead = then;
        return true;
    };
    while (step(x0, x2) && step(x1, x0) && step(x2, x1)) {}
    if (ks == 1) return;
    // a tile a group of wavefronts: their sums meet in LDS, in the order of the blocks
    __syncthreads();                                 // the columns are read
    float4v *sums = reinterpret_cast<float4v *>(columns);
#pragma unroll
    for (int x = 0; x < CT; ++x) sums[(wave * CT + x) * 64 + lane] = acc[x];
    __syncthreads();
    const int64_t tile = (int64_t)(wave / ks) * gridDim.x + blockIdx.x;
    if (part != 0 || tile >= tiles) return;
#pragma unroll
    for (int x = 0; x < CT; ++x) {
        float4v z = acc[x];
        for (int p = 1; p < ks; ++p) {
            const float4v y = sums[((wave + p) * CT + x) * 64 + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] += y[i];
        }
        write_scores<N>(c, z, end, x * 16 + (lane & 15), re[x]);
    }
}

// ---- more columns: tiles of 256 classes by CT * 16 columns --------------------------------
// A wavefront four tiles of classes, whose codes it turns into f16 in registers; the four share the
// columns of a block of W, copied to LDS while the block before is worked on.
// Bound by issue: a block's unpacking is shared by CT products only, and a wavefront waits at each
// block for its columns.  201 x 777 f32 by 50003 classes of groups of 32: 50 us, 0.7 PFLOP/s of padded
// products of two terms; matrix cores busy 29 %, vector units 38, wavefronts waiting 34.  bf16 31,
// and 512 x 1024 by 32000 40, 0.84 PFLOP/s.
typedef __attribute__((address_space(1))) void global_void;
typedef __attribute__((address_space(3))) void lds_void;
constexpr int WIDE_WAVES = 4, WIDE_TILES = 4;
template <int N, int CT, int PER>
__global__ __launch_bounds__(64 * WIDE_WAVES, 2) void k_fourbit_tiles(
    FourbitCall c, const half8 *__restrict__ columns, const int32_t *__restrict__ row_exponents,
    int64_t column_tiles, int32_t turns) {
    extern __shared__ half8 lds[];                   // [buffer][column tile][step of the block][lane]
    constexpr int BUFFER = CT * 4 * 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t tiles = (c.shape.classes + TILE - 1) / TILE;
    const int blocks = c.shape.blocks, quads = (blocks + 3) / 4;
    const int64_t id = group_id();
    const int64_t tile0 = (id / turns * WIDE_WAVES + wave) * WIDE_TILES;
    const int64_t column0 = id % turns * CT;
    if (id / turns * WIDE_WAVES * WIDE_TILES >= tiles) return;
    const auto copy = [&](int b) {
#pragma unroll
        for (int x = 0; x < CT; ++x) {
            const int64_t t = min(column0 + x, column_tiles - 1);
            __builtin_amdgcn_global_load_lds(
                (global_void *)(columns + ((t * blocks + b) * 4 + wave) * 64 + lane),
                (lds_void *)(lds + (b & 1) * BUFFER + (x * 4 + wave) * 64), 16, 0, 0);
        }
    };
    const Unpack unpack;
    int64_t at[WIDE_TILES];
#pragma unroll
    for (int t = 0; t < WIDE_TILES; ++t) at[t] = min(tile0 + t, tiles - 1);
    uint4v word[WIDE_TILES], ahead[WIDE_TILES];
    const auto fetch = [&](int b) {
#pragma unroll
        for (int t = 0; t < WIDE_TILES; ++t)
            ahead[t] = reinterpret_cast<const uint4v *>(c.codes)[(at[t] * blocks + b) * 64 + lane];
    };
    typedef _Float16 halves __attribute__((ext_vector_type(PER)));
    halves scale[WIDE_TILES], scale_ahead[WIDE_TILES];
    const auto fetch_scales = [&](int b) {
#pragma unroll
        for (int t = 0; t < WIDE_TILES; ++t)
            scale_ahead[t] = reinterpret_cast<const halves *>(
                c.scales)[((at[t] * quads + b / 4) * TILE + (lane & 15)) * 4 + b % 4];
    };
    float4v acc[WIDE_TILES][CT];
#pragma unroll
    for (int t = 0; t < WIDE_TILES; ++t)
#pragma unroll
        for (int x = 0; x < CT; ++x) acc[t][x] = float4v{0, 0, 0, 0};
    copy(0);
    fetch(0);
    fetch_scales(0);
    for (int b = 0; b < blocks; ++b) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                             // the block is there; the other buffer is read
#pragma unroll
        for (int t = 0; t < WIDE_TILES; ++t) {
            word[t] = ahead[t];
            scale[t] = scale_ahead[t];
        }
        if (b + 1 < blocks) {
            copy(b + 1);
            fetch(b + 1);
            fetch_scales(b + 1);
        }
        const half8 *here = lds + (b & 1) * BUFFER + lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (b * BLOCK + j * 32 >= c.shape.dim) break;
            half8 a[WIDE_TILES];
#pragma unroll
            for (int t = 0; t < WIDE_TILES; ++t) a[t] = weights(unpack, word[t][j], scale[t][j * PER / 4]);
#pragma unroll
            for (int x = 0; x < CT; ++x) {
                const half8 h = here[(x * 4 + j) * 64];
#pragma unroll
                for (int t = 0; t < WIDE_TILES; ++t)
                    acc[t][x] =
                        __builtin_amdgcn_mfma_f32_16x16x32_f16(a[t], h, acc[t][x], 0, 0, 0);
            }
        }
    }
    int e[CT];
#pragma unroll
    for (int x = 0; x < CT; ++x)
        e[x] = row_exponents[min(((column0 + x) * 16 + (lane & 15)) / N, c.rows - 1)];
    Ends<N> end[WIDE_TILES];
#pragma unroll
    for (int t = 0; t < WIDE_TILES; ++t) end[t] = ends_of<N>(c, tile0 + t);
    // a wavefront's 64 classes of a tile of columns meet in LDS, so that a row's go out 256 bytes
    // together: where rows are at odd addresses, 64 at a time leave parts of lines
    constexpr int ROWS = 16 / N, ROW = WIDE_TILES * TILE + 4;
    float *meet = reinterpret_cast<float *>(lds) + wave * ROWS * ROW;
    __syncthreads();                                 // the columns are read
#pragma unroll
    for (int x = 0; x < CT; ++x) {
#pragma unroll
        for (int t = 0; t < WIDE_TILES; ++t) {
            float v[Ends<N>::EACH];
            scores_of<N>(c, acc[t][x], end[t], e[x], v);
            float *to = meet + (lane & 15) / N * ROW + (int)(end[t].cls - tile0 * TILE);
#pragma unroll
            for (int i = 0; i < Ends<N>::EACH; ++i) to[i] = v[i];
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < ROWS / 4; ++i) {
            const int row = i * 4 + (lane >> 4);
            const float4v z = *reinterpret_cast<const float4v *>(meet + row * ROW + (lane & 15) * 4);
            const float v[4] = {z[0], z[1], z[2], z[3]};
            put_scores(c, (column0 + x) * 16 / N + row, tile0 * TILE + (lane & 15) * 4, v,
                       c.streamed);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

size_t code_bytes(const FourbitShape &s) {
    return (size_t)((s.classes + TILE - 1) / TILE) * s.blocks * 1024;
}
size_t scale_bytes(const FourbitShape &s) {
    return (size_t)((s.classes + TILE - 1) / TILE) * ((s.blocks + 3) / 4) * 4 * TILE *
           (BLOCK / s.group) * 2;
}

// Columns of h that are held: 64 MB of them, or 16 rows.
int64_t rows_a_turn(const FourbitCall &c) {
    const int64_t row = (int64_t)c.shape.blocks * BLOCK * (c.bf16 ? 2 : 4);
    return std::max<int64_t>(16, std::min<int64_t>(16384, ((int64_t)64 << 20) / row) / 16 * 16);
}
size_t column_bytes(const FourbitCall &c, size_t rows) {
    return (rows * (c.bf16 ? 1 : 2) + 15) / 16 * c.shape.blocks * 4096;
}

template <typename T> int64_t column_tiles(const FourbitCall &c) {
    return (c.rows * TERMS<T> + 15) / 16;
}
// LDS of the columns, or of the wavefronts' sums or maxima in their place.
constexpr size_t FEW_LDS = 159 << 10;
size_t few_lds(const FourbitCall &c) {
    const size_t width = (size_t)c.rows * (c.bf16 ? 1 : 2);
    return FEW_HEAD + std::max(width * c.shape.blocks * (BLOCK * 2),
                               (size_t)FEW_WAVES * ((width + 15) / 16 == 1 ? 1 : 2) * 1024);
}
constexpr int FEW_TILES = 2;
bool few(const FourbitCall &c) {
    return (c.bf16 ? column_tiles<__bf16>(c) : column_tiles<float>(c)) <= FEW_TILES &&
           few_lds(c) <= FEW_LDS;
}

template <typename T, int CT, int PER> hipError_t run_few(hipStream_t st, const FourbitCall &c) {
    const void *f = reinterpret_cast<const void *>(k_fourbit_few<T, CT, PER>);
    const hipError_t e = allow_all_lds(f);
    if (e != hipSuccess) return e;
    const int64_t tiles = (c.shape.classes + TILE - 1) / TILE;
    const int quads = (c.shape.blocks + 3) / 4;
    const size_t lds = few_lds(c);
    const int64_t most = (int64_t)c.num_cus * (lds <= (80 << 10) ? 2 : 1);      // workgroups at once
    // wavefronts a tile: as many as fill them
    int ks = 1;
    while (ks < FEW_WAVES && 2 * ks <= quads && 2 * ks * tiles <= most * FEW_WAVES) ks *= 2;
    const int64_t groups = (tiles * ks + FEW_WAVES - 1) / FEW_WAVES;
    int log2_rows = 0;
    while ((1 << log2_rows) < c.rows) ++log2_rows;
    hipLaunchKernelGGL((k_fourbit_few<T, CT, PER>), dim3((uint32_t)std::min(groups, most)),
                       dim3(FEW_THREADS), lds, st, c, ks, log2_rows);
    return hipGetLastError();
}

template <typename T, int CT, int PER>
hipError_t run_tiles(hipStream_t st, const FourbitCall &c, const half8 *columns, const int32_t *e,
                     int64_t column_tiles, int turns) {
    const hipError_t bad =
        allow_all_lds(reinterpret_cast<const void *>(k_fourbit_tiles<TERMS<T>, CT, PER>));
    if (bad != hipSuccess) return bad;
    const int64_t tiles = (c.shape.classes + TILE - 1) / TILE;
    const int64_t groups = (tiles + WIDE_WAVES * WIDE_TILES - 1) / (WIDE_WAVES * WIDE_TILES) * turns;
    hipLaunchKernelGGL((k_fourbit_tiles<TERMS<T>, CT, PER>), grid_of(groups), dim3(64 * WIDE_WAVES),
                       std::max((size_t)CT * 8192, (size_t)WIDE_WAVES * (16 / TERMS<T>) *
                                                       (WIDE_TILES * TILE + 4) * 4),
                       st,
                       c, columns, e, column_tiles, turns);
    return hipGetLastError();
}

template <typename T, int PER> hipError_t run(hipStream_t st, const FourbitCall &c, char *scratch) {
    const int64_t tiles = column_tiles<T>(c);
    if (few(c))
        return tiles <= 1 ? run_few<T, 1, PER>(st, c) : run_few<T, 2, PER>(st, c);
    half8 *columns = reinterpret_cast<half8 *>(scratch);
    const int steps = c.shape.blocks * 4;
    int32_t *e = reinterpret_cast<int32_t *>(scratch + column_bytes(c, (size_t)c.rows));
    hipLaunchKernelGGL((k_fourbit_columns<T>), grid_of(tiles), dim3(64 * COLUMN_WAVES), 0, st,
                       static_cast<const T *>(c.h), c.h_stride, c.rows, c.shape.dim, c.wide_h, steps,
                       columns, e);
    // tiles of columns a turn: the time is that of the CU with most turns, each its tiles' products
    // and about two tiles' worth of unpacking, beginning and end
    const int64_t groups =
        ((c.shape.classes + TILE - 1) / TILE + WIDE_WAVES * WIDE_TILES - 1) / (WIDE_WAVES * WIDE_TILES);
    int64_t best = 0, least = 0;
    for (int64_t ct = 1; ct <= 8; ++ct) {
        const int64_t each = (groups * ((tiles + ct - 1) / ct) + c.num_cus - 1) / c.num_cus;
        if (!best || each * (ct + 2) <= least) best = ct, least = each * (ct + 2);
    }
    const int turns = (int)((tiles + best - 1) / best);
    switch (best) {
    case 1: return run_tiles<T, 1, PER>(st, c, columns, e, tiles, turns);
    case 2: return run_tiles<T, 2, PER>(st, c, columns, e, tiles, turns);
    case 3: return run_tiles<T, 3, PER>(st, c, columns, e, tiles, turns);
    case 4: return run_tiles<T, 4, PER>(st, c, columns, e, tiles, turns);
    case 5: return run_tiles<T, 5, PER>(st, c, columns, e, tiles, turns);
    case 6: return run_tiles<T, 6, PER>(st, c, columns, e, tiles, turns);
    case 7: return run_tiles<T, 7, PER>(st, c, columns, e, tiles, turns);
    default: return run_tiles<T, 8, PER>(st, c, columns, e, tiles, turns);
    }
}

template <typename T> hipError_t run(hipStream_t st, const FourbitCall &c, char *scratch) {
    switch (c.shape.group) {
    case 32: return run<T, 4>(st, c, scratch);
    case 64: return run<T, 2>(st, c, scratch);
    default: return run<T, 1>(st, c, scratch);
    }
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
    const bool wide = reinterpret_cast<uintptr_t>(w) % 16 == 0 && stride * (bf16 ? 2 : 4) % 16 == 0;
    const dim3 g = grid_of((s.classes + TILE - 1) / TILE);
    const auto launch = [&](auto type, auto per) {
        using T = decltype(type);
        hipLaunchKernelGGL((k_fourbit_pack<T, decltype(per)::value>), g, dim3(64 * PACK_WAVES), 0, st,
                           s, static_cast<const T *>(w), stride, wide,
                           reinterpret_cast<uint4v *>(codes), scales, exponents);
    };
    const auto typed = [&](auto type) {
        if (s.group == 32) launch(type, std::integral_constant<int, 4>{});
        else if (s.group == 64) launch(type, std::integral_constant<int, 2>{});
        else launch(type, std::integral_constant<int, 1>{});
    };
    if (bf16) typed(__bf16{});
    else typed(float{});
    return hipGetLastError();
}

size_t fourbit_scratch(const FourbitCall &c) {
    if (few(c)) return 0;
    const size_t rows = (size_t)std::min(c.rows, rows_a_turn(c));
    return column_bytes(c, rows) + 4 * rows;
}

hipError_t launch_fourbit_scores(hipStream_t st, const FourbitCall &c, char *scratch) {
    const int64_t each = rows_a_turn(c);
    const int64_t row = c.h_stride * (c.bf16 ? 2 : 4);
    const bool wide_h = reinterpret_cast<uintptr_t>(c.h) % 16 == 0 && row % 16 == 0;
    for (int64_t r = 0; r < c.rows; r += each) {
        FourbitCall part = c;
        part.rows = std::min(each, c.rows - r);
        part.wide_h = wide_h;
        part.streamed = part.rows * c.shape.classes * 4 > STREAMED;
        part.h = static_cast<const char *>(c.h) + r * row;
        part.scores = c.scores + r * c.score_stride;
        const hipError_t e = c.bf16 ? run<__bf16>(st, part, scratch) : run<float>(st, part, scratch);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace mbk
