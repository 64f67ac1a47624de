// kernels_xent.hip — cross entropy of scores h W' + b over many classes, and its
// gradient (mbk_xent, mbk_xent_grad), without keeping the scores.
//
//   z_iv = h_i . W_v + b_v,  lse_i = log sum_v exp z_iv
//   loss_i = w_i (lse_i - z_i,y_i),  G_iv = w_i (exp(z_iv - lse_i) - [v = y_i])
//   dh = G W,  dW = G' h,  db = column sums of G
//
// The classes are taken in pieces: one pass over all of them keeps each row's
// running maximum and sum; a second one makes the scores of a piece again, writes
// its G, and two products turn that into dh and dW before the next piece overwrites
// it.
//
// Operands.  The matrix instructions take 16-bit operands and add in f32.  All operands go
// in as f16 terms of x 2^s:
//   W: s is its column's, and puts the column's largest element below 2^14.
//   h, for the scores: the columns' powers of W are taken back, and one of the row puts the
//   largest h_ij max_v |W_vj| below 2^14.
//   w h, for dW: s is its column's.
// So columns may be of very different sizes.
//   bf16 inputs: one term, which holds their 8 bits as they are down to 2^-30 of that
//   largest.  G is rounded to one f16 term, too, 11 bits, and w h again where there are weights: as
//   bf16 terms they would add as much error again to dh and dW as their own rounding to bf16
//   (measured 2.8e-3 in place of 1.7e-3 of their norm), at the same rate.
//   f32 inputs: two terms, hi + lo, 22 bits, and three products hi hi + hi lo + lo hi: what is
//   dropped, lo lo and the bits behind lo, is at most 2^-21 of an element's product and
//   random in sign, the size of what an f32 sum over the same length rounds away.  (f32
//   operands have an instruction of 1/16 of the rate; three of these cost 3/16.)
// That holds for elements from 2^-16 of the largest on (f16 has no smaller exponents); below,
// they are off by up to 2^-38 of it, so that a score is by 2^-21 sum_j |h_ij W_vj| + 2^-37 d
// max_j (|h_ij| max_v |W_vj|) at most.  G / w is off by up to 2^-40 where that is more.
//
// Classes not offered (bias -inf) are packed as zeros, and so are rows that are out
// (label outside [0, V), weight 0, or no class offered) and hold NaN, infinities or values
// that could overflow: what they hold reaches nothing, and a finite row that is out is
// multiplied by zeros.
//
// 16384 x 1024 x 65536 bf16 takes 2.1 ms for the statistics (1.05 PFLOP/s), 2.55 for G (0.86; it
// writes 2.1 GB) and 4.27 for dh and dW (1.03); a library product of bf16 reaches 1.23 to 1.56.
// The matrix cores are busy 50 to 53 % of the cycles (G 41 %), at 1.85 to 1.9 GHz, where the
// kernels that pack run at 2.4; the wavefronts wait for 38 to 47 % of theirs, at the ends of steps
// of copies and of LDS reads.  Without their copies the products take 17 % less.
#include <algorithm>

#include "mbk.h"
#include "ops.h"
#include "xent.hpp"

namespace mbk {

namespace {

typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;

constexpr int LD_PAD = 128;              // operands' rows are padded to it
constexpr int G_EXP = 15;                // |G / w| <= 1 goes in times 2^this

// Eight of an array whose length is padded.
template <typename V> __device__ __forceinline__ void load8(const V *p, int f, V (&x)[8]) {
    typedef __attribute__((ext_vector_type(4))) V V4;
    const V4 a = *reinterpret_cast<const V4 *>(p + f), b = *reinterpret_cast<const V4 *>(p + f + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = a[e];
        x[e + 4] = b[e];
    }
}
template <typename T> __device__ __forceinline__ float load_f32(const void *p, int64_t i) {
    return (float)static_cast<const T *>(p)[i];
}

// What the rows of a matrix are aligned to: 16, 4, or an element.
template <typename T> __device__ __forceinline__ int alignment(const void *p, int64_t stride) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(stride * sizeof(T));
    return all & 15 ? (all & 3 ? 2 : 4) : 16;
}
// Eight elements of a row from f on, zeros behind its d.
template <typename T>
__device__ __forceinline__ void load8(const void *p, int64_t row, int f, int d, int align,
                                      float (&x)[8]) {
    const T *from = static_cast<const T *>(p) + row + f;
    T y[8];
    if (align == 16 && f + 8 <= d) {
        u32x4 v[sizeof(T) / 2];
#pragma unroll
        for (int q = 0; q < (int)sizeof(T) / 2; ++q) v[q] = reinterpret_cast<const u32x4 *>(from)[q];
        __builtin_memcpy(y, v, sizeof y);
    } else if (sizeof(T) == 2 && align != 2 && f + 8 <= d) {
        uint32_t v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = reinterpret_cast<const uint32_t *>(from)[q];
        __builtin_memcpy(y, v, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = f + e < d ? from[e] : (T)0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)y[e];
}
// Eight elements times 2^s into the planes.
template <typename T>
__device__ __forceinline__ void pack8(const float (&x)[8], const int (&s)[8], u16 *to,
                                      int64_t plane) {
    u16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        u16 a, b;
        split_f16(ldexpf(x[e], s[e]), a, b);
        hi[e] = a;
        lo[e] = b;
    }
    *reinterpret_cast<u16x8 *>(to) = hi;
    if (sizeof(T) == 4) *reinterpret_cast<u16x8 *>(to + plane) = lo;
}
constexpr int MAX_WAVES = 8;              // of the kernels that prepare
// A weight, its exponent apart: times h it may pass f32, where G is small.
struct Apart {
    float mantissa;
    int exp;
};
__device__ __forceinline__ Apart apart(float w) {
    const int e = exponent_of(w);
    return e != NO_EXP ? Apart{__builtin_amdgcn_frexp_mantf(w), e} : Apart{w, 0};
}
// Whether row i counts.  A class offered is looked for elsewhere.
__device__ __forceinline__ bool row_in(const XentPack &k, const XentCall &c, int64_t i, float &wt) {
    const int32_t y = c.labels[i];
    wt = c.weights ? c.weights[i] : 1.0f;
    return y >= 0 && y < k.v && wt != 0.0f;
}

// The columns' largest: workgroups of W, then (gradients) of the rows' w h, 256 columns
// each, eight a lane, and two rows a wavefront, in turns.  Those of W also leave the padded bias
// and whether a class is offered.
constexpr int COLUMNS = 256, COLUMN_ROWS = 2 * MAX_WAVES, ROWS_AHEAD = 4;
template <typename T>
__global__ __launch_bounds__(64 * MAX_WAVES) void k_xent_columns(XentPack k, XentCall c) {
    __shared__ int32_t most[COLUMN_ROWS][COLUMNS];
    const int lane = threadIdx.x & 31, r = threadIdx.x >> 5;
    const bool of_w = (int32_t)blockIdx.x < k.w_groups;
    const int32_t group = of_w ? blockIdx.x : blockIdx.x - k.w_groups;
    const int64_t stride = of_w ? c.w_stride : c.h_stride, rows = of_w ? k.v_pad : k.n;
    const void *from = of_w ? c.w : c.h;
    const int align = alignment<T>(from, stride);
    const int32_t f = blockIdx.y * COLUMNS + lane * 8;
    int m[8] = {NO_EXP, NO_EXP, NO_EXP, NO_EXP, NO_EXP, NO_EXP, NO_EXP, NO_EXP};
    bool any = false;
    // four rows at a time, so that as many loads are on the way
    const int64_t hop = (int64_t)(of_w ? k.w_groups : k.hg_groups) * COLUMN_ROWS;
    for (int64_t v0 = (int64_t)group * COLUMN_ROWS + r; v0 < rows; v0 += ROWS_AHEAD * hop) {
        float wt[ROWS_AHEAD], x[ROWS_AHEAD][8];
#pragma unroll
        for (int q = 0; q < ROWS_AHEAD; ++q) {
            const int64_t v = v0 + q * hop;
            const bool here = v < (of_w ? k.v : k.n);
            load8<T>(from, (here ? v : 0) * stride, f, here ? k.d : 0, align, x[q]);
            wt[q] = 0.0f;
            if (of_w) {
                const float b = here ? (c.bias ? c.bias[v] : 0.0f) : -INFINITY;
                if (b != -INFINITY) wt[q] = 1.0f;
                if (lane == 0 && blockIdx.y == 0 && v < k.v_pad) k.bias[v] = b;
            } else if (here && !row_in(k, c, v, wt[q])) {
                wt[q] = 0.0f;
            }
            any = any || wt[q] != 0.0f;
        }
        // times 0 a value that is not finite is none either
#pragma unroll
        for (int q = 0; q < ROWS_AHEAD; ++q) {
            const Apart w = apart(wt[q]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                m[e] = max(m[e], exponent_of(x[q][e] * w.mantissa) + w.exp);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) most[r][lane * 8 + e] = m[e];
    const bool offered = __syncthreads_or(any);
    if (of_w && blockIdx.y == 0 && threadIdx.x == 0) k.ctl->offered.part[group] = offered;
    const int64_t col = (int64_t)blockIdx.y * COLUMNS + threadIdx.x;
    if (threadIdx.x >= COLUMNS || col >= k.ld) return;
    int v = NO_EXP;
#pragma unroll
    for (int q = 0; q < COLUMN_ROWS; ++q) v = max(v, most[q][threadIdx.x]);
    (of_w ? k.w_part : k.hg_part)[group * (int64_t)k.ld + col] = v;
}

// A column's power of two, of its largest exponent.  A column of W that is all zeros has one
// that keeps h's column from its rows' scales.
constexpr int ZERO_COLUMN = 1000;
__device__ __forceinline__ int32_t column_exp(int e, bool of_w) {
    return e > NO_EXP / 2 ? TOP_EXP - e : of_w ? ZERO_COLUMN : 0;
}
// All of them: 64 columns a workgroup, whose wavefronts go over the groups in turns.
constexpr int SCALE_WAVES = 16;
__global__ __launch_bounds__(64 * SCALE_WAVES) void k_xent_scales(XentPack k) {
    __shared__ int32_t most[SCALE_WAVES][64];
    __shared__ uint32_t words[SCALE_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t cols = k.ld / 64;
    const bool of_w = (int32_t)blockIdx.x < cols;
    const int64_t col = (int64_t)(of_w ? blockIdx.x : blockIdx.x - cols) * 64 + lane;
    const int32_t *part = of_w ? k.w_part : k.hg_part;
    const int32_t groups = of_w ? k.w_groups : k.hg_groups;
    int m = NO_EXP;
#pragma unroll 8
    for (int g = wave; g < groups; g += SCALE_WAVES) m = max(m, part[(int64_t)g * k.ld + col]);
    most[wave][lane] = m;
    if (blockIdx.x == 0) {
        const uint32_t any = largest_of<SCALE_WAVES>(k.ctl->offered, k.w_groups, words);
        if (threadIdx.x == 0) k.ctl->offered.all = any;
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < SCALE_WAVES; ++w) m = max(m, most[w][lane]);
    (of_w ? k.w_exp : k.hg_exp)[col] = column_exp(m, of_w);
}
// Of few groups and columns, by each workgroup of the next kernel, without a launch: W's in LDS,
// and both in memory by the first one (2000 x 256 x 2000 f32, 32 groups, 29 us and 30.5 with
// the launch, 4000 x 256 x 4000, 63 groups, 52.5 and 51).
constexpr int FEW_GROUPS = 32, FEW_COLUMNS = 64 * MAX_WAVES;
__device__ __forceinline__ bool few_scales(const XentPack &k, int32_t *exps, uint32_t *words) {
    const int32_t col = threadIdx.x;
    if (col < k.ld) {
        int w = NO_EXP, h = NO_EXP;
#pragma unroll 8
        for (int g = 0; g < k.w_groups; ++g) w = max(w, k.w_part[g * k.ld + col]);
        exps[col] = column_exp(w, true);
        if (blockIdx.x == 0) {
#pragma unroll 8
            for (int g = 0; g < k.hg_groups; ++g) h = max(h, k.hg_part[g * k.ld + col]);
            k.w_exp[col] = exps[col];
            k.hg_exp[col] = column_exp(h, false);
        }
    }
    return largest_of<MAX_WAVES>(k.ctl->offered, k.w_groups, words);
}
// Eight columns' powers of W.
__device__ __forceinline__ void load_exps(const XentPack &k, const int32_t *few, int f,
                                          int (&s)[8]) {
    if (k.few) load8<int32_t>(few, f, s);
    else load8<int32_t>(k.w_exp, f, s);
}

// The kernels that pack take a wavefront a row, over the rows in turns.
template <typename T>
__device__ __forceinline__ void pack_w(const XentPack &k, const void *w, int64_t stride,
                                       const int32_t *exps) {
    const int lane = threadIdx.x & 63;
    const int align = alignment<T>(w, stride);
    constexpr int ROWS = 2;
    const int64_t hop = (int64_t)k.pack_w_groups * MAX_WAVES;
    for (int64_t v0 = (int64_t)blockIdx.x * MAX_WAVES + (threadIdx.x >> 6); v0 < k.v_pad;
         v0 += ROWS * hop) {
        int32_t d[ROWS];
#pragma unroll
        for (int q = 0; q < ROWS; ++q)
            d[q] = v0 + q * hop < k.v && k.bias[v0 + q * hop] != -INFINITY ? k.d : 0;
        for (int32_t f = lane * 8; f < k.ld; f += 512) {
            float x[ROWS][8];
            int s[8];
#pragma unroll
            for (int q = 0; q < ROWS; ++q)
                load8<T>(w, (d[q] ? v0 + q * hop : 0) * stride, f, d[q], align, x[q]);
            load_exps(k, exps, f, s);
#pragma unroll
            for (int q = 0; q < ROWS; ++q)
                if (v0 + q * hop < k.v_pad)
                    pack8<T>(x[q], s, k.w + (v0 + q * hop) * k.ld + f, k.v_pad * k.ld);
        }
    }
}

// W packed, and by the workgroups behind those, the rows: label and weight (-1 and 0 where
// the row is out) and h.  A row that is out and whose scores may not be finite is packed as
// zeros, its label -2.
template <typename T>
__global__ __launch_bounds__(64 * MAX_WAVES) void k_xent_pack(XentPack k, XentCall c) {
    __shared__ int32_t exps[FEW_COLUMNS];
    __shared__ uint32_t words[MAX_WAVES];
    const bool offered = k.few ? few_scales(k, exps, words) : k.ctl->offered.all != 0;
    if ((int32_t)blockIdx.x < k.pack_w_groups) {
        pack_w<T>(k, c.w, c.w_stride, exps);
        return;
    }
    const int32_t group = blockIdx.x - k.pack_w_groups;
    const int lane = threadIdx.x & 63;
    const int align = alignment<T>(c.h, c.h_stride);
    for (int64_t i = (int64_t)group * MAX_WAVES + (threadIdx.x >> 6); i < k.n_pad;
         i += (int64_t)k.pack_h_groups * MAX_WAVES) {
        int32_t d = i < k.n ? k.d : 0;
        float wt = 0.0f;
        const bool in = i < k.n && row_in(k, c, i, wt) && offered;
        int m = NO_EXP;
        uint32_t most = 0;
        for (int32_t f = lane * 8; f < d; f += 512) {
            float x[8];
            int s[8];
            load8<T>(c.h, i * c.h_stride, f, d, align, x);
            load_exps(k, exps, f, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                m = max(m, exponent_of(x[e]) - s[e]);
                most = max(most, __float_as_uint(fabsf(x[e])));
            }
        }
        m = wave_max(m);
        int s = m > NO_EXP / 2 ? TOP_EXP - m : 0;
        int32_t y = -1;
        if (in) {
            y = c.labels[i];
        } else {
            wt = 0.0f;
            if (wave_max(most) >= XENT_HUGE || s < FAR_ROW) {
                y = -2;
                s = 0;
                d = 0;
            }
        }
        if (lane == 0) {
            k.row_scale[i] = power_of_2(-s);
            k.label[i] = y;
            k.weight[i] = wt;
        }
        for (int32_t f = lane * 8; f < k.ld; f += 512) {
            float x[8];
            int e[8];
            load8<T>(c.h, i * c.h_stride, f, d, align, x);
            load_exps(k, exps, f, e);
#pragma unroll
            for (int q = 0; q < 8; ++q) e[q] = s - e[q];
            pack8<T>(x, e, k.h + i * k.ld + f, k.n_pad * k.ld);
        }
    }
}

// ---- products --------------------------------------------------------------------
// C[m][n] = sum_k A[m][k] B[n][k].  An operand lies with k contiguous (KC: element (m, k)
// at m * ld + k) or with m contiguous (k * ld + m); the second kind is turned by the LDS
// reads (ds_read_tr16_b64: 16 lanes read 4 rows of 16 elements, lane i gets column i).
// P planes of f16 terms.
//
// A workgroup has a tile of 256 x 256 in eight wavefronts (Wide: 128 x 64 each) or of
// 128 x 128 in four (Narrow: 64 x 64 each).  Steps of k are copied into LDS directly, one
// step ahead, 64 of one plane or 32 of two.
template <int WM_, int WN_, int MT_, int NT_> struct Tiling {
    static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_;     // wavefronts, blocks of 32
    static constexpr int WAVES = WM * WN, T = WM * MT * 32;
    static_assert(T == WN * NT * 32, "square tiles");
};
using Wide = Tiling<2, 4, 4, 2>;
using Narrow = Tiling<2, 2, 2, 2>;

template <int P> constexpr int BK = 64 / P;          // k of a step
template <int P, class C> constexpr int OP_BYTES = P * C::T * BK<P> * 2;
template <int P, class C> constexpr int LDS_TILES = 4 * OP_BYTES<P, C>;      // A and B, twice

struct Operand {
    const u16 *p;
    int64_t plane, ld;
};

// The chunks of 16 bytes of an LDS row are permuted by the row.  Rows of k (KC, 64 or 128
// bytes): the 16 rows x 1 chunk of a read fall on all banks.  Rows of m: the 4 rows x 4
// chunks of a read across do.
template <int P, bool KC> __device__ __forceinline__ int chunk_xor(int row) {
    if constexpr (!KC) return (row & 3) * 4;
    else if constexpr (P == 1) return ((row >> 1) & 1) * 4 + ((row >> 2) & 3);
    else return (row >> 2) & 3;
}

// Starts the copies of a step of an operand from m0, k0 on.
template <int P, bool KC, class C>
__device__ __forceinline__ void copy_step(const Operand &o, int64_t m0, int64_t k0, char *lds,
                                          int wave) {
    constexpr int ROW = (KC ? BK<P> : C::T) * 2, PLANE = C::T * BK<P> * 2;
    constexpr int ROWS = 1024 / ROW;                 // of a wavefront's copy
    const int lane = threadIdx.x & 63;
    const int row = wave * ROWS + lane * 16 / ROW;
    const int chunk = (lane * 16 % ROW / 16) ^ chunk_xor<P, KC>(row);
    const uint32_t mine = (uint32_t)row * (uint32_t)o.ld * 2 + chunk * 16;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const char *from = reinterpret_cast<const char *>(o.p + p * o.plane +
                                                          (KC ? m0 * o.ld + k0 : k0 * o.ld + m0));
#pragma unroll
        for (int q = 0; q < PLANE / 1024 / C::WAVES; ++q)
            __builtin_amdgcn_global_load_lds(
                (global_void *)(from + (int64_t)q * C::WAVES * ROWS * o.ld * 2 + mine),
                (lds_void *)(lds + p * PLANE + (q * C::WAVES + wave) * 1024), 16, 0, 0);
    }
}

// Operands of the matrix instruction, lane l with element m0 + l % 32 of a block and k =
// 16 SLAB + l / 32 * 8 .. + 7, for N blocks of 32 from m0 on.
template <int P, class C, int SLAB, int N>
__device__ __forceinline__ void along(const char *lds, int m0, u32x4 (&f)[N][P]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int t = 0; t < N; ++t) {
        const int row = m0 + t * 32 + (lane & 31);
        const int chunk = (SLAB * 2 + (lane >> 5)) ^ chunk_xor<P, true>(row);
#pragma unroll
        for (int p = 0; p < P; ++p)
            f[t][p] = *reinterpret_cast<const u32x4 *>(lds + p * (C::T * BK<P> * 2) +
                                                       row * (BK<P> * 2) + chunk * 16);
    }
}
// Across: m0 is a multiple of 32 N, so that the blocks differ in chunk bits alone.  The
// reads wait for themselves: see kernels_xent_fused.hip.
template <class C> __device__ __forceinline__ uint32_t across_at(int m0) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    const int row = (g >> 1) * 8 + (i >> 2), m = m0 + (g & 1) * 16 + (i & 3) * 4;
    return row * (C::T * 2) + ((m >> 3) ^ ((row & 3) * 4)) * 16 + (m & 7) * 2;
}
#define TR(dst, addr, off) "ds_read_b64_tr_b16 " dst ", " addr " offset:" off "\n\t"
#define TR2(d0, d1, addr, o0, o1) TR(d0, addr, o0) TR(d1, addr, o1)
template <int N, int P> struct AcrossReads {
    u32x2 x[N][P][2];
    __device__ __forceinline__ void get(u32x4 (&f)[N][P]) const {
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int p = 0; p < P; ++p)
                f[t][p] = u32x4{x[t][p][0][0], x[t][p][0][1], x[t][p][1][0], x[t][p][1][1]};
    }
};
template <int P, class C, int SLAB>
__device__ __forceinline__ void across(uint32_t at, u32x4 (&f)[2][P]) {
    constexpr int ROW = C::T * 2, O = SLAB * 16 * ROW, O4 = O + 4 * ROW, PLANE = C::T * BK<P> * 2;
    AcrossReads<2, P> r;
#pragma unroll
    for (int p = 0; p < P; ++p)
        asm volatile(TR2("%0", "%1", "%4", "%6", "%7") TR2("%2", "%3", "%5", "%6", "%7")
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(r.x[0][p][0]), "=&v"(r.x[0][p][1]), "=&v"(r.x[1][p][0]),
                       "=&v"(r.x[1][p][1])
                     : "v"(at + p * PLANE), "v"((at ^ 64) + p * PLANE), "n"(O), "n"(O4)
                     : "memory");
    r.get(f);
}
// Both operands across: one wait for all reads of a plane.
template <int P, class C, int SLAB>
__device__ __forceinline__ void across_both(uint32_t a, uint32_t b, u32x4 (&fa)[C::MT][P],
                                            u32x4 (&fb)[C::NT][P]) {
    constexpr int ROW = C::T * 2, O = SLAB * 16 * ROW, O4 = O + 4 * ROW, PLANE = C::T * BK<P> * 2;
    AcrossReads<C::MT, P> ra;
    AcrossReads<C::NT, P> rb;
    static_assert(C::NT == 2 && (C::MT == 2 || C::MT == 4), "reads of 2 or 4 and 2 blocks");
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const uint32_t ap = a + p * PLANE, bp = b + p * PLANE;
        if constexpr (C::MT == 4)
            asm volatile(TR2("%0", "%1", "%12", "%18", "%19") TR2("%2", "%3", "%13", "%18", "%19")
                         TR2("%4", "%5", "%14", "%18", "%19") TR2("%6", "%7", "%15", "%18", "%19")
                         TR2("%8", "%9", "%16", "%18", "%19")
                         TR2("%10", "%11", "%17", "%18", "%19") "s_waitcnt lgkmcnt(0)"
                         : "=&v"(ra.x[0][p][0]), "=&v"(ra.x[0][p][1]), "=&v"(ra.x[1][p][0]),
                           "=&v"(ra.x[1][p][1]), "=&v"(ra.x[2][p][0]), "=&v"(ra.x[2][p][1]),
                           "=&v"(ra.x[3][p][0]), "=&v"(ra.x[3][p][1]), "=&v"(rb.x[0][p][0]),
                           "=&v"(rb.x[0][p][1]), "=&v"(rb.x[1][p][0]), "=&v"(rb.x[1][p][1])
                         : "v"(ap), "v"(ap ^ 64), "v"(ap ^ 128), "v"(ap ^ 192), "v"(bp),
                           "v"(bp ^ 64), "n"(O), "n"(O4)
                         : "memory");
        else
            asm volatile(TR2("%0", "%1", "%8", "%12", "%13") TR2("%2", "%3", "%9", "%12", "%13")
                         TR2("%4", "%5", "%10", "%12", "%13") TR2("%6", "%7", "%11", "%12", "%13")
                         "s_waitcnt lgkmcnt(0)"
                         : "=&v"(ra.x[0][p][0]), "=&v"(ra.x[0][p][1]), "=&v"(ra.x[1][p][0]),
                           "=&v"(ra.x[1][p][1]), "=&v"(rb.x[0][p][0]), "=&v"(rb.x[0][p][1]),
                           "=&v"(rb.x[1][p][0]), "=&v"(rb.x[1][p][1])
                         : "v"(ap), "v"(ap ^ 64), "v"(bp), "v"(bp ^ 64), "n"(O), "n"(O4)
                         : "memory");
    }
    ra.get(fa);
    rb.get(fb);
}
#undef TR2
#undef TR

template <class C> using Acc = f32x16[C::MT][C::NT];
template <class C> __device__ __forceinline__ void clear(Acc<C> &acc) {
#pragma unroll
    for (int x = 0; x < C::MT; ++x)
#pragma unroll
        for (int y = 0; y < C::NT; ++y)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
}

// The product over the steps [first, last) of k of a sequence of tiles: next(i, m0, n0)
// gives tile i, done(i) takes its sums from acc.  The copies run ahead over the ends of
// tiles.
template <int P, bool AK, bool BKC, class C, class Next, class Done>
__device__ __forceinline__ void products(const Operand &a, const Operand &b, int64_t tiles,
                                         int64_t first, int64_t last, char *lds, Acc<C> &acc,
                                         Next next, Done done) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / C::WN * C::MT * 32, wn = wave % C::WN * C::NT * 32;
    const uint32_t base = lds_address(lds);
    const uint32_t a_at = AK ? 0 : across_at<C>(wm);
    const uint32_t b_at = BKC ? 0 : across_at<C>(wn);
    if (first >= last) {                 // a split without a step: no copy is left behind
        clear<C>(acc);
        return;
    }
    int64_t m0, n0;
    next(0, m0, n0);
    copy_step<P, AK, C>(a, m0, first * BK<P>, lds, wave);
    copy_step<P, BKC, C>(b, n0, first * BK<P>, lds + OP_BYTES<P, C>, wave);
    int buf = 0;
    for (int64_t i = 0; i < tiles; ++i) {
        clear<C>(acc);
        for (int64_t t = first; t < last; ++t) {
            copies_done();
            __syncthreads();             // the step is there; the other buffer is read
            const int cur = buf * 2 * OP_BYTES<P, C>, nxt = 2 * OP_BYTES<P, C> - cur;
            buf ^= 1;
            const bool end = t + 1 == last;
            if (end && i + 1 < tiles) next(i + 1, m0, n0);
            if (!end || i + 1 < tiles) {
                const int64_t k0 = (end ? first : t + 1) * BK<P>;
                copy_step<P, AK, C>(a, m0, k0, lds + nxt, wave);
                copy_step<P, BKC, C>(b, n0, k0, lds + nxt + OP_BYTES<P, C>, wave);
            }
            const auto slab = [&](auto which) {
                constexpr int S = decltype(which)::value;
                u32x4 fa[C::MT][P], fb[C::NT][P];
                if constexpr (!AK && !BKC) {
                    across_both<P, C, S>(base + cur + a_at, base + cur + OP_BYTES<P, C> + b_at, fa,
                                         fb);
                } else {
                    static_assert(AK, "A across goes with B across");
                    along<P, C, S>(lds + cur, wm, fa);
                    if constexpr (BKC) along<P, C, S>(lds + cur + OP_BYTES<P, C>, wn, fb);
                    else across<P, C, S>(base + cur + OP_BYTES<P, C> + b_at, fb);
                }
#pragma unroll
                for (int x = 0; x < C::MT; ++x)
#pragma unroll
                    for (int y = 0; y < C::NT; ++y) acc[x][y] = mma<P>(fa[x], fb[y], acc[x][y]);
            };
            slab(At<0>{});
            slab(At<1>{});
            if constexpr (BK<P> == 64) {
                slab(At<2>{});
                slab(At<3>{});
            }
        }
        done(i);
    }
}

// Workgroups go to the 8 XCDs in turn; each XCD gets a run of tiles, in groups of 8
// rows of tiles, so that what its L2 holds is used by many.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t total, uint32_t tiles_m,
                                        uint32_t tiles_n, uint32_t &tm, uint32_t &tn) {
    const uint32_t xcd = id & 7, per = total >> 3, more = total & 7;
    const uint32_t at = xcd * per + min(xcd, more) + (id >> 3);
    const uint32_t group = at / (8 * tiles_n), in = at % (8 * tiles_n);
    const uint32_t rows = min(8u, tiles_m - group * 8);
    tm = group * 8 + in % rows;
    tn = in / rows;
}

// ---- pass 1: each row's maximum and sum ---------------------------------------------
// The product is W h' (classes down, rows across), so that a lane has scores of one
// row: the maximum and sum stay in registers over the classes of a split, and only
// two lanes and two wavefronts have parts of a row.  part[2 * split + half][row]: the
// maximum of z, and the sum of exp(z - it).
template <int P, class C>
__global__ __launch_bounds__(C::WAVES * 64, 2) void k_xent_stats(XentPack k, int32_t row_tiles,
                                                                 int32_t class_tiles,
                                                                 int32_t splits,
                                                                 float2 *__restrict__ part) {
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t row_tile, split;
    tile_of(blockIdx.x, gridDim.x, row_tiles, splits, row_tile, split);
    const int64_t i0 = (int64_t)row_tile * C::T;
    const Operand a{k.w, k.v_pad * k.ld, k.ld}, b{k.h, k.n_pad * k.ld, k.ld};
    float m[C::NT], s[C::NT], sc[C::NT];
    int64_t row[C::NT];
#pragma unroll
    for (int y = 0; y < C::NT; ++y) {
        row[y] = i0 + wave % C::WN * C::NT * 32 + y * 32 + (lane & 31);
        m[y] = -INFINITY;
        s[y] = 0.0f;
        sc[y] = k.row_scale[row[y]];
    }
    Acc<C> acc;
    const auto next = [&](int64_t i, int64_t &m0, int64_t &n0) {
        m0 = (split + i * splits) * C::T;
        n0 = i0;
    };
    const auto done = [&](int64_t i) {
        const float *bias = k.bias + (split + i * splits) * C::T + wave / C::WN * C::MT * 32 +
                            (lane >> 5) * 4;
        float top[C::NT];
#pragma unroll
        for (int y = 0; y < C::NT; ++y) top[y] = m[y];
#pragma unroll
        for (int x = 0; x < C::MT; ++x)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 b = *reinterpret_cast<const f32x4 *>(bias + x * 32 + q * 8);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int y = 0; y < C::NT; ++y) {
                        const float z = __builtin_fmaf(acc[x][y][q * 4 + e], sc[y], b[e]);
                        acc[x][y][q * 4 + e] = z;
                        top[y] = fmaxf(top[y], z);
                    }
            }
#pragma unroll
        for (int y = 0; y < C::NT; ++y) {
            const float ref = top[y] == -INFINITY ? 0.0f : top[y];
            float sum[2] = {s[y] * exp_of(m[y] - ref), 0.0f};
#pragma unroll
            for (int x = 0; x < C::MT; ++x)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sum[r & 1] += exp_of(acc[x][y][r] - ref);
            m[y] = top[y];
            s[y] = sum[0] + sum[1];
        }
    };
    const int64_t tiles = (class_tiles - (int64_t)split + splits - 1) / splits;
    products<P, true, true, C>(a, b, tiles, 0, (k.d + BK<P> - 1) / BK<P>, lds, acc, next, done);
#pragma unroll
    for (int y = 0; y < C::NT; ++y) {
        const float m2 = __shfl_xor(m[y], 32, 64), s2 = __shfl_xor(s[y], 32, 64);
        const float top = fmaxf(m[y], m2), ref = top == -INFINITY ? 0.0f : top;
        const float sum = s[y] * exp_of(m[y] - ref) + s2 * exp_of(m2 - ref);
        if (lane < 32)
            part[(2 * split + wave / C::WN) * k.n_pad + row[y]] = make_float2(top, sum);
    }
}

// The parts of a row joined, one wavefront a row: lse, as reference and log2 of the sum for
// the gradients, and loss.  The label's score is summed in f32 from h and W themselves.  For
// gradients, h is packed once more as dW's product takes it, times the row's weight and with
// powers of two of its columns (the rows are summed over).
template <typename T>
__global__ __launch_bounds__(256) void k_xent_join(XentPack k, XentCall c, int32_t parts,
                                                   const float2 *__restrict__ part,
                                                   float2 *__restrict__ lse2) {
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)group_id() * 4 + (threadIdx.x >> 6);
    if (i >= k.n_pad) return;
    float top = -INFINITY, sum = 0.0f;
    for (int p = lane; p < parts; p += 64) {
        const float2 q = part[p * k.n_pad + i];
        const float now = fmaxf(top, q.x), ref = now == -INFINITY ? 0.0f : now;
        sum = sum * exp_of(top - ref) + q.y * exp_of(q.x - ref);
        top = now;
    }
    const int32_t y = k.label[i];
    const bool open = y >= 0 && k.bias[y] != -INFINITY;
    float dot = 0.0f;
    if (open)
        for (int32_t f = lane; f < k.d; f += 64)
            dot += load_f32<T>(c.h, i * c.h_stride + f) * load_f32<T>(c.w, y * c.w_stride + f);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float t2 = __shfl_xor(top, o, 64), s2 = __shfl_xor(sum, o, 64);
        const float now = fmaxf(top, t2), ref = now == -INFINITY ? 0.0f : now;
        sum = sum * exp_of(top - ref) + s2 * exp_of(t2 - ref);
        top = now;
        dot += __shfl_xor(dot, o, 64);
    }
    if (k.hg) {
        const int align = alignment<T>(c.h, c.h_stride);
        const int32_t d = y >= 0 ? k.d : 0;
        const Apart wt = apart(k.weight[i]);
        for (int32_t f = lane * 8; f < k.ld; f += 512) {
            float x[8];
            int s[8];
            load8<T>(c.h, i * c.h_stride, f, d, align, x);
            load8<int32_t>(k.hg_exp, f, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] *= wt.mantissa;
                s[e] += wt.exp;
            }
            pack8<T>(x, s, k.hg + i * k.ld + f, k.n_pad * k.ld);
        }
    }
    if (lane != 0) return;
    const LogSum l = log_sum(sum);
    lse2[i] = make_float2(top, l.base2);
    if (i >= k.n) return;
    const float z = open ? dot + (c.bias ? c.bias[y] : 0.0f) : -INFINITY;
    c.lse[i] = y == -2 ? NAN : lse_of(top, l);
    c.loss[i] = y < 0 ? 0.0f : k.weight[i] * loss_of(top, l, z);
}

// ---- pass 2: G of a piece ------------------------------------------------------------
// g[v - v0][i - r0], rows of rows_pad: G / w times 2^15.  part_db[part of the rows][v]: sums
// of G itself.
// A workgroup has a tile of rows and every splits-th tile of classes.
template <int P, class C>
__global__ __launch_bounds__(C::WAVES * 64, 2) void k_xent_g(XentPack k, int64_t v0, int64_t r0,
                                                             int64_t rows_pad, int64_t plane,
                                                             int32_t row_tiles,
                                                             int32_t class_tiles, int32_t splits,
                                                             const float2 *__restrict__ lse2,
                                                             u16 *__restrict__ g,
                                                             float *__restrict__ part_db) {
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t row_tile, split;
    tile_of(blockIdx.x, gridDim.x, row_tiles, splits, row_tile, split);
    const int64_t i0 = r0 + (int64_t)row_tile * C::T;
    const Operand a{k.w, k.v_pad * k.ld, k.ld}, b{k.h, k.n_pad * k.ld, k.ld};
    const int64_t iw = i0 + wave % C::WN * C::NT * 32;
    float sc[C::NT], ref[C::NT], l[C::NT], wt[C::NT];
    int32_t label[C::NT];
#pragma unroll
    for (int y = 0; y < C::NT; ++y) {
        const int64_t i = iw + y * 32 + (lane & 31);
        sc[y] = k.row_scale[i];
        label[y] = k.label[i];
        const float2 lse = lse2[i];
        ref[y] = label[y] < 0 ? 0.0f : lse.x;
        l[y] = label[y] < 0 ? INFINITY : lse.y;          // a row that is out: 2^-inf
        wt[y] = k.weight[i];
    }
    const uint32_t mine = half * 4 * (uint32_t)rows_pad + (lane & 31);
    Acc<C> acc;
    const auto next = [&](int64_t i, int64_t &m0, int64_t &n0) {
        m0 = v0 + (split + i * splits) * C::T;
        n0 = i0;
    };
    const auto done = [&](int64_t i) {
        const int64_t c0 = v0 + (split + i * splits) * C::T + wave / C::WN * C::MT * 32;
#pragma unroll
        for (int x = 0; x < C::MT; ++x) {
            const int64_t c = c0 + x * 32;
            float db[16];
#pragma unroll
            for (int y = 0; y < C::NT; ++y) {
                const int64_t at = label[y] - c - half * 4;      // 8 q + e if the label is here
                const bool hot = __any(at >= 0 && at < 32);
                u16 *to = g + (c - v0) * rows_pad + (iw - r0) + y * 32;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 b =
                        *reinterpret_cast<const f32x4 *>(k.bias + c + half * 4 + q * 8);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float z = __builtin_fmaf(acc[x][y][q * 4 + e], sc[y], b[e]);
                        float p = __builtin_amdgcn_exp2f(
                            __builtin_fmaf(z - ref[y], LOG2E, -l[y]));
                        if (hot && at == q * 8 + e) p -= 1.0f;
                        db[q * 4 + e] = y == 0 ? p * wt[y]
                                               : __builtin_fmaf(p, wt[y], db[q * 4 + e]);
                        u16 hi, lo;
                        split_f16(p * (float)(1 << G_EXP), hi, lo);
                        to[mine] = hi;
                        if constexpr (P == 2) to[plane + mine] = lo;
                        to += e < 3 ? rows_pad : 5 * rows_pad;
                    }
                }
            }
            // The sums over the rows: each exchange halves the classes a lane holds, and
            // lane l % 32 ends with the class of register l >> 1 & 15.
            if (part_db) {
#pragma unroll
                for (int n = 8, o = 16; n > 0; n >>= 1, o >>= 1) {
                    const bool upper = lane & o;
#pragma unroll
                    for (int r = 0; r < n; ++r) {
                        const float keep = upper ? db[r + n] : db[r];
                        db[r] = keep + __shfl_xor(upper ? db[r] : db[r + n], o, 64);
                    }
                }
                db[0] += __shfl_xor(db[0], 1, 64);
                const int r = lane >> 1 & 15;
                if (!(lane & 1))
                    part_db[((int64_t)row_tile * C::WN + wave % C::WN) * k.v_pad + c +
                            (r >> 2) * 8 + half * 4 + (r & 3)] = db[0];
            }
        }
    };
    const int64_t tiles = (class_tiles - (int64_t)split + splits - 1) / splits;
    products<P, true, true, C>(a, b, tiles, 0, (k.d + BK<P> - 1) / BK<P>, lds, acc, next, done);
}

// Where a product over the pieces goes: the f32 sums so far, [split][m_pad][ld], and, with
// the last piece and no splits, the output.
struct Out {
    float *acc;
    int64_t m_pad;
    bool first, last;
    int32_t splits;
    void *out;
    int64_t rows, stride;        // of the output; its columns are k.d
    bool classes;                // dW: rows whose bias is -inf are 0; dh: times weight
};
// The power of two of column n of a product with G.
__device__ __forceinline__ int out_exp(const XentPack &k, bool classes, int64_t n) {
    return n < k.d ? -G_EXP - (classes ? k.hg_exp : k.w_exp)[n] : 0;
}
template <int P>
__device__ __forceinline__ void put(const XentPack &k, const Out &o, int64_t m, int64_t n, float v,
                                    int exp) {
    if (m >= o.rows || n >= k.d) return;
    v = ldexpf(v, exp);
    if (!o.classes) v *= k.weight[m];
    else if (k.bias[m] == -INFINITY) v = 0.0f;
    if constexpr (P == 1) static_cast<__bf16 *>(o.out)[m * o.stride + n] = (__bf16)v;
    else static_cast<float *>(o.out)[m * o.stride + n] = v;
}

// A product with G: its first row is m_first of the output.
struct Product {
    Operand a, b;
    int32_t tiles_m, tiles_n;
    int64_t steps, m_first;
    Out o;
};
template <int P, bool AK, class C>
__device__ __forceinline__ void product(const XentPack &k, const Product &q, uint32_t id, char *lds) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Out &o = q.o;
    const uint32_t per = q.tiles_m * q.tiles_n, split = id / per;
    uint32_t tm, tn;
    tile_of(id % per, per, q.tiles_m, q.tiles_n, tm, tn);
    Acc<C> acc;
    const auto next = [&](int64_t, int64_t &m0, int64_t &n0) {
        m0 = (int64_t)tm * C::T;
        n0 = (int64_t)tn * C::T;
    };
    products<P, AK, false, C>(q.a, q.b, 1, q.steps * split / o.splits,
                              q.steps * (split + 1) / o.splits, lds, acc, next, [](int64_t) {});
    int exp[C::NT];
#pragma unroll
    for (int y = 0; y < C::NT; ++y)
        exp[y] = out_exp(k, o.classes,
                         (int64_t)tn * C::T + wave % C::WN * C::NT * 32 + y * 32 + (lane & 31));
    float *sums = o.acc + split * o.m_pad * k.ld;
#pragma unroll
    for (int x = 0; x < C::MT; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int64_t m = q.m_first + (int64_t)tm * C::T + wave / C::WN * C::MT * 32 + x * 32 +
                              (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
#pragma unroll
            for (int y = 0; y < C::NT; ++y) {
                const int64_t n = (int64_t)tn * C::T + wave % C::WN * C::NT * 32 + y * 32 +
                                  (lane & 31);
                float v = acc[x][y][r];
                if (o.first && o.last && o.splits == 1) {
                    put<P>(k, o, m, n, v, exp[y]);
                } else if (n < k.ld) {
                    if (!o.first) v += sums[m * k.ld + n];
                    if (o.last && o.splits == 1) put<P>(k, o, m, n, v, exp[y]);
                    else sums[m * k.ld + n] = v;
                }
            }
        }
}

// Both products, dh (A = G across, m the rows) by the first workgroups and dW (A = G along, m
// the classes), B = W or h across: where neither fills the chip they run side by side (bf16
// 194 x 216 x 835 with gradients: 50 us, 69 with a launch for each and for each sum).
template <int P, class C>
__global__ __launch_bounds__(C::WAVES * 64, 2) void k_xent_products(XentPack k, Product dh,
                                                                    uint32_t dh_groups, Product dw) {
    extern __shared__ char lds[];
    if (blockIdx.x < dh_groups) product<P, false, C>(k, dh, blockIdx.x, lds);
    else product<P, true, C>(k, dw, blockIdx.x - dh_groups, lds);
}

// The splits of a product's row added, in order.
template <int P>
__device__ __forceinline__ void join_splits(const XentPack &k, int64_t m, const Out &o) {
    for (int32_t n = threadIdx.x; n < k.d; n += 256) {
        float v = 0.0f;
#pragma unroll 4
        for (int s = 0; s < o.splits; ++s) v += o.acc[(s * o.m_pad + m) * k.ld + n];
        put<P>(k, o, m, n, v, out_exp(k, o.classes, n));
    }
}
// A workgroup a row of dh_rows and of dw_rows, whose splits it adds, and then one for 256 classes
// from v0 on: db[v] += the parts' sums, in order.
template <int P>
__global__ __launch_bounds__(256) void k_xent_finish(XentPack k, uint32_t dh_rows, int64_t dh_first,
                                                     Out dh, uint32_t dw_rows, int64_t dw_first,
                                                     Out dw, int64_t v0, int64_t classes,
                                                     int32_t parts,
                                                     const float *__restrict__ part_db, bool first,
                                                     float *__restrict__ db) {
    if (blockIdx.x < dh_rows) {
        join_splits<P>(k, dh_first + blockIdx.x, dh);
        return;
    }
    if (blockIdx.x < dh_rows + dw_rows) {
        join_splits<P>(k, dw_first + (blockIdx.x - dh_rows), dw);
        return;
    }
    const int64_t c = (int64_t)(blockIdx.x - dh_rows - dw_rows) * 256 + threadIdx.x;
    if (c >= classes) return;
    double sum = 0.0;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) sum += part_db[p * k.v_pad + v0 + c];
    if (k.bias[v0 + c] == -INFINITY) sum = 0.0;
    db[v0 + c] = first ? (float)sum : (float)(db[v0 + c] + sum);
}

// Zeros where there is no row to sum over.
template <typename T>
__global__ __launch_bounds__(256) void k_xent_zero(T *out, int64_t rows, int32_t cols,
                                                   int64_t stride) {
    const int64_t v = (int64_t)group_id() * 4 + (threadIdx.x >> 6);
    if (v >= rows) return;
    for (int32_t f = threadIdx.x & 63; f < cols; f += 64) out[v * stride + f] = (T)0.0f;
}

// ---- the call -------------------------------------------------------------------------
int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
uint32_t blocks(int64_t x, int64_t per) { return (uint32_t)((x + per - 1) / per); }

// G of a piece: 32k rows and 512 MB at most.  16384 x 1024 x 65536 bf16 with gradients: 8.8
// ms; with 256 MB, which the memory-side cache would hold, 9.3 (half the tiles of dW, so
// that k is split), with 1 GB 8.7.
constexpr int64_t PIECE_ROWS = 32768;
constexpr int64_t PIECE_BYTES = (int64_t)512 << 20;

// What a k step of a workgroup of 256 x 256 takes, in us, at the rate that the large products
// reach (1.1 PFLOP/s), and one of 128 x 128 with another beside it on its CU: half of a
// quarter of the CU's work each, at 0.85 of the rate (8191 x 768 x 50000 bf16: 0.62 ms by wide
// tiles, 0.70 by narrow ones; 16384 x 1024 x 65536 with gradients 8.7 and 10.4).
double step_us(bool wide, int P) { return (P == 1 ? 1.95 : 2.9) * (wide ? 1.0 : 0.5 / 0.85); }
int64_t slots_of(bool wide, int num_cus) { return (wide ? 1 : 2) * (int64_t)num_cus; }

// Workgroups that share a tile of rows: one wide workgroup a CU or two narrow ones.
int32_t splits_of(bool wide, int64_t row_tiles, int64_t class_tiles, int num_cus) {
    return (int32_t)std::max<int64_t>(1, std::min(class_tiles, slots_of(wide, num_cus) / row_tiles));
}

// Wide tiles where the tiles that a workgroup gets then take less time: padding and the last
// round, in which few have one, count (f32, loss: 1024 x 512 x 16384 117 us wide, 124
// narrow; 300 x 512 x 33000 148 and 127; 400 x 1024 x 33000 250 and 217).
bool wide_tiles(int64_t rows, int64_t classes, int num_cus) {
    double us[2];
    for (const bool wide : {false, true}) {
        const int64_t t = wide ? 256 : 128;
        const int64_t row_tiles = up(rows, t) / t, class_tiles = up(classes, t) / t;
        const int64_t splits = splits_of(wide, row_tiles, class_tiles, num_cus);
        const int64_t slots = slots_of(wide, num_cus);
        us[wide] = step_us(wide, 1) * (double)((class_tiles + splits - 1) / splits) *
                   (double)((row_tiles * splits + slots - 1) / slots);
    }
    return us[1] <= us[0];
}

// How a product over k of m x n is cut.
struct Cut {
    bool wide;
    int32_t tiles_n, splits;
};
// The least time, four steps a workgroup at least, by the steps of the workgroups' rounds, 3 us for a workgroup's start and
// end, and what the parts of a split k take to be written, read and joined.  (f32, with
// gradients: 256 x 512 x 40000 360 us, 1115 without splits.)
Cut cut_of(bool wide_allowed, int P, int64_t m, int64_t n, int64_t steps, int num_cus) {
    Cut best{};
    double least = 1e300;
    for (const bool wide : {true, false}) {
        if (wide && !wide_allowed) continue;
        const int64_t t = wide ? 256 : 128, slots = slots_of(wide, num_cus);
        const int64_t tiles_m = m / t, tiles_n = up(n, t) / t, tiles = tiles_m * tiles_n;
        const int64_t most = std::max<int64_t>(
            1, std::min<int64_t>({steps / 4, 64, 2 * slots / tiles}));
        for (int64_t s = 1; s <= most; ++s) {
            const double join = s == 1 ? 0.0 : 4.0 + (double)(s * m) * (double)n * 8.0 / 4.5e6;
            const double us = (double)((tiles * s + slots - 1) / slots) *
                                  ((double)((steps + s - 1) / s) * step_us(wide, P) + 3.0) + join;
            if (us < least) {
                least = us;
                best = {wide, (int32_t)tiles_n, (int32_t)s};
            }
        }
    }
    return best;
}

struct Plan {
    int P;
    bool wide, wide_g;           // tiles of the statistics (and padding), of G
    int64_t n_pad, v_pad, ld, piece_rows, piece_classes;
    int32_t splits;
    Cut dh, dw;                  // of whole pieces
    int32_t w_groups, hg_groups;
    size_t ctl, w_part, hg_part, w_exp, hg_exp, h, hg, w, bias, scale, label, weight, lse, part, g,
        db, dh_acc, dw_acc, end;
};

Plan plan_of(const XentCall &c) {
    Plan p{};
    p.P = c.bf16 ? 1 : 2;
    p.wide = wide_tiles(c.rows, c.classes, c.num_cus);
    const int64_t t = p.wide ? 256 : 128, step = 64 / p.P;
    p.n_pad = up(c.rows, t);
    p.v_pad = up(c.classes, t);
    p.ld = up(c.dim, LD_PAD);
    const int64_t row_tiles = p.n_pad / t, class_tiles = p.v_pad / t;
    p.splits = splits_of(p.wide, row_tiles, class_tiles, c.num_cus);
    p.piece_rows = std::min(p.n_pad, PIECE_ROWS);
    p.piece_classes = std::min(
        p.v_pad, std::max<int64_t>(t, PIECE_BYTES / (2 * p.P * p.piece_rows) / t * t));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    // a wide tile may read 128 elements past the last packed row
    const size_t past = 512;
    // workgroups of k_xent_columns: four a CU over all columns
    const int64_t most = std::max<int64_t>(
        1, std::min(4 * c.num_cus, MOST_GROUPS) / (up(c.dim, COLUMNS) / COLUMNS));
    const auto groups = [&](int64_t rows) {
        return (int32_t)std::min(blocks(rows, COLUMN_ROWS * ROWS_AHEAD), (uint32_t)most);
    };
    p.w_groups = groups(p.v_pad);
    p.hg_groups = c.grad ? groups(p.n_pad) : 0;
    p.ctl = take(sizeof(XentCtl));
    p.w_part = take((size_t)4 * p.w_groups * p.ld);
    p.hg_part = take((size_t)4 * p.hg_groups * p.ld);
    p.w_exp = take((size_t)4 * p.ld);
    p.hg_exp = take((size_t)4 * p.ld);
    p.h = take((size_t)2 * p.P * p.n_pad * p.ld + past);
    p.w = take((size_t)2 * p.P * p.v_pad * p.ld + past);
    p.bias = take((size_t)4 * p.v_pad);
    p.scale = take((size_t)4 * p.n_pad);
    p.label = take((size_t)4 * p.n_pad);
    p.weight = take((size_t)4 * p.n_pad);
    p.lse = take((size_t)8 * p.n_pad);
    p.part = take((size_t)16 * p.splits * p.n_pad);
    if (c.grad) {
        p.wide_g = p.wide && wide_tiles(p.piece_rows, p.piece_classes, c.num_cus);
        p.hg = take((size_t)2 * p.P * p.n_pad * p.ld + past);
        if (c.dbias) p.db = take((size_t)4 * (p.piece_rows / 64) * p.v_pad);
        p.g = take((size_t)2 * p.P * p.piece_rows * p.piece_classes);
        p.dh = cut_of(p.wide, p.P, p.piece_rows, c.dim, p.piece_classes / step, c.num_cus);
        p.dw = cut_of(p.wide, p.P, p.piece_classes, c.dim, p.piece_rows / step, c.num_cus);
        if (p.dh.splits > 1 || p.piece_classes < p.v_pad)
            p.dh_acc = take((size_t)4 * p.dh.splits * p.n_pad * p.ld);
        if (p.dw.splits > 1 || p.piece_rows < p.n_pad)
            p.dw_acc = take((size_t)4 * p.dw.splits * p.v_pad * p.ld);
    }
    p.end = at;
    return p;
}

// Workgroups of a product of m rows.
uint32_t product_groups(const Cut &c, int64_t m) {
    return (uint32_t)(m / (c.wide ? 256 : 128)) * c.tiles_n * c.splits;
}
Product product_of(const Operand &a, const Operand &b, const Cut &c, int64_t m, int64_t steps,
                   int64_t m_first, Out o) {
    o.splits = c.splits;
    return {a, b, (int32_t)(m / (c.wide ? 256 : 128)), c.tiles_n, steps, m_first, o};
}
// Rows of it that a later kernel joins.
uint32_t rows_to_join(const Product &q, int64_t m) {
    return q.o.last && q.o.splits > 1 && q.m_first < q.o.rows
               ? (uint32_t)std::min(m, q.o.rows - q.m_first) : 0;
}
template <int P>
void launch_products(hipStream_t s, const XentPack &k, bool wide, const Product &dh,
                     uint32_t dh_groups, const Product &dw, uint32_t dw_groups) {
    const dim3 g(dh_groups + dw_groups);
    if (wide)
        hipLaunchKernelGGL((k_xent_products<P, Wide>), g, dim3(512), (LDS_TILES<P, Wide>), s, k, dh,
                           dh_groups, dw);
    else
        hipLaunchKernelGGL((k_xent_products<P, Narrow>), g, dim3(256), (LDS_TILES<P, Narrow>), s, k,
                           dh, dh_groups, dw);
}

template <int P, class C>
void launch_stats(hipStream_t s, const XentPack &k, int32_t splits, float2 *part) {
    const int32_t rt = (int32_t)(k.n_pad / C::T), vt = (int32_t)(k.v_pad / C::T);
    hipLaunchKernelGGL((k_xent_stats<P, C>), dim3((uint32_t)rt * splits), dim3(C::WAVES * 64),
                       (LDS_TILES<P, C>), s, k, rt, vt, splits, part);
}
template <int P, class C>
void launch_g(hipStream_t s, const XentPack &k, int64_t v0, int64_t nv, int64_t r0, int64_t nr,
              int64_t plane, int num_cus, const float2 *lse2, u16 *g, float *part_db) {
    const int32_t rt = (int32_t)(nr / C::T), vt = (int32_t)(nv / C::T);
    const int32_t splits = splits_of(C::T == 256, rt, vt, num_cus);
    hipLaunchKernelGGL((k_xent_g<P, C>), dim3((uint32_t)rt * splits), dim3(C::WAVES * 64),
                       (LDS_TILES<P, C>), s, k, v0, r0, nr, plane, rt, vt, splits, lse2, g, part_db);
}

template <int P, typename T>
hipError_t run(hipStream_t s, const XentCall &c, const Plan &p, char *m) {
    XentPack k{};
    k.n = c.rows;
    k.v = c.classes;
    k.n_pad = p.n_pad;
    k.v_pad = p.v_pad;
    k.d = c.dim;
    k.ld = (int32_t)p.ld;
    k.ctl = reinterpret_cast<XentCtl *>(m + p.ctl);
    k.w_groups = p.w_groups;
    k.hg_groups = p.hg_groups;
    k.few = p.w_groups <= FEW_GROUPS && p.hg_groups <= FEW_GROUPS && p.ld <= FEW_COLUMNS;
    k.w_part = reinterpret_cast<int32_t *>(m + p.w_part);
    k.hg_part = reinterpret_cast<int32_t *>(m + p.hg_part);
    k.w_exp = reinterpret_cast<int32_t *>(m + p.w_exp);
    k.hg_exp = reinterpret_cast<int32_t *>(m + p.hg_exp);
    k.h = reinterpret_cast<u16 *>(m + p.h);
    k.hg = c.grad ? reinterpret_cast<u16 *>(m + p.hg) : nullptr;
    k.w = reinterpret_cast<u16 *>(m + p.w);
    k.bias = reinterpret_cast<float *>(m + p.bias);
    k.row_scale = reinterpret_cast<float *>(m + p.scale);
    k.label = reinterpret_cast<int32_t *>(m + p.label);
    k.weight = reinterpret_cast<float *>(m + p.weight);
    float2 *lse2 = reinterpret_cast<float2 *>(m + p.lse);
    float2 *part = reinterpret_cast<float2 *>(m + p.part);
    const dim3 b(256);
    const void *big[] = {reinterpret_cast<const void *>(k_xent_stats<P, Wide>),
                         reinterpret_cast<const void *>(k_xent_stats<P, Narrow>),
                         reinterpret_cast<const void *>(k_xent_g<P, Wide>),
                         reinterpret_cast<const void *>(k_xent_g<P, Narrow>),
                         reinterpret_cast<const void *>(k_xent_products<P, Wide>),
                         reinterpret_cast<const void *>(k_xent_products<P, Narrow>)};
    for (const void *f : big) {
        const hipError_t e = allow_all_lds(f);
        if (e != hipSuccess) return e;
    }
    const auto groups = [&](int64_t rows) {
        return (int32_t)std::min<int64_t>((rows + MAX_WAVES - 1) / MAX_WAVES, 4 * c.num_cus);
    };
    k.pack_w_groups = groups(k.v_pad);
    k.pack_h_groups = groups(k.n_pad);
    hipLaunchKernelGGL((k_xent_columns<T>),
                       dim3((uint32_t)(k.w_groups + k.hg_groups), blocks(c.dim, COLUMNS)),
                       dim3(64 * MAX_WAVES), 0, s, k, c);
    if (!k.few)
        hipLaunchKernelGGL(k_xent_scales, dim3((uint32_t)(k.ld / 64 * (c.grad ? 2 : 1))),
                           dim3(64 * SCALE_WAVES), 0, s, k);
    hipLaunchKernelGGL((k_xent_pack<T>), dim3((uint32_t)(k.pack_w_groups + k.pack_h_groups)),
                       dim3(64 * MAX_WAVES), 0, s, k, c);
    if (p.wide) launch_stats<P, Wide>(s, k, p.splits, part);
    else launch_stats<P, Narrow>(s, k, p.splits, part);
    hipLaunchKernelGGL((k_xent_join<T>), grid_of(blocks(k.n_pad, 4)), b, 0, s, k, c, 2 * p.splits,
                       part, lse2);
    if (!c.grad) return hipGetLastError();
    u16 *g = reinterpret_cast<u16 *>(m + p.g);
    float *part_db = c.dbias ? reinterpret_cast<float *>(m + p.db) : nullptr;
    const int64_t plane = p.piece_rows * p.piece_classes, step = BK<P>;
    for (int64_t v0 = 0; v0 < k.v_pad; v0 += p.piece_classes)
        for (int64_t r0 = 0; r0 < k.n_pad; r0 += p.piece_rows) {
            const int64_t nv = std::min(p.piece_classes, k.v_pad - v0);
            const int64_t nr = std::min(p.piece_rows, k.n_pad - r0);
            if (p.wide_g) launch_g<P, Wide>(s, k, v0, nv, r0, nr, plane, c.num_cus, lse2, g, part_db);
            else launch_g<P, Narrow>(s, k, v0, nv, r0, nr, plane, c.num_cus, lse2, g, part_db);
            const Operand ag{g, plane, nr};
            const Product dh = product_of(
                ag, {k.w + v0 * k.ld, k.v_pad * k.ld, k.ld}, p.dh, nr, nv / step, r0,
                Out{reinterpret_cast<float *>(m + p.dh_acc), k.n_pad, v0 == 0, v0 + nv == k.v_pad, 1,
                    c.dh, k.n, c.h_stride, false});
            const Product dw = product_of(
                ag, {k.hg + r0 * k.ld, k.n_pad * k.ld, k.ld}, p.dw, nv, nr / step, v0,
                Out{reinterpret_cast<float *>(m + p.dw_acc), k.v_pad, r0 == 0, r0 + nr == k.n_pad, 1,
                    c.dw, k.v, c.w_stride, true});
            const uint32_t dh_groups = c.dh ? product_groups(p.dh, nr) : 0;
            const uint32_t dw_groups = c.dw ? product_groups(p.dw, nv) : 0;
            if (p.dh.wide == p.dw.wide && dh_groups && dw_groups) {
                launch_products<P>(s, k, p.dh.wide, dh, dh_groups, dw, dw_groups);
            } else {
                if (dh_groups) launch_products<P>(s, k, p.dh.wide, dh, dh_groups, dw, 0);
                if (dw_groups) launch_products<P>(s, k, p.dw.wide, dh, 0, dw, dw_groups);
            }
            const uint32_t dh_rows = c.dh ? rows_to_join(dh, nr) : 0;
            const uint32_t dw_rows = c.dw ? rows_to_join(dw, nv) : 0;
            const int64_t live = std::min(nv, k.v - v0);
            const uint32_t db_groups = c.dbias ? blocks(live, 256) : 0;
            // a part of db is 64 rows, of either tiling
            if (dh_rows + dw_rows + db_groups)
                hipLaunchKernelGGL((k_xent_finish<P>), dim3(dh_rows + dw_rows + db_groups), b, 0, s,
                                   k, dh_rows, r0, dh.o, dw_rows, v0, dw.o, v0, live,
                                   (int32_t)(nr / 64), part_db, r0 == 0, c.dbias);
        }
    return hipGetLastError();
}

}  // namespace

size_t xent_scratch(const XentCall &c) {
    if (!c.rows) return 0;
    if (xent_few(c)) return xent_few_scratch(c);
    return c.dim <= XENT_FUSED_DIM ? xent_fused_scratch(c) : plan_of(c).end;
}

hipError_t launch_xent(hipStream_t s, const XentCall &c, char *scratch) {
    if (c.rows && xent_few(c)) return launch_xent_few(s, c, scratch);
    if (c.rows && c.dim <= XENT_FUSED_DIM) return launch_xent_fused(s, c, scratch);
    if (c.rows) {
        const Plan p = plan_of(c);
        return c.bf16 ? run<1, __bf16>(s, c, p, scratch) : run<2, float>(s, c, p, scratch);
    }
    // no row: no loss, and gradients that are empty sums
    if (c.grad && c.dw) {
        const dim3 g = grid_of(blocks(c.classes, 4)), b(256);
        if (c.bf16)
            hipLaunchKernelGGL((k_xent_zero<__bf16>), g, b, 0, s, static_cast<__bf16 *>(c.dw),
                               c.classes, c.dim, c.w_stride);
        else
            hipLaunchKernelGGL((k_xent_zero<float>), g, b, 0, s, static_cast<float *>(c.dw),
                               c.classes, c.dim, c.w_stride);
    }
    if (c.grad && c.dbias)
        hipLaunchKernelGGL((k_xent_zero<float>), grid_of(blocks(c.classes, 4)), dim3(256), 0, s,
                           c.dbias, c.classes, 1, (int64_t)1);
    return hipGetLastError();
}

}  // namespace mbk
