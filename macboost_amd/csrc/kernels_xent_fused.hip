// kernels_xent_fused.hip — the many-class loss for few outputs (dim <= 128): a
// workgroup keeps 128 rows of one operand in registers and streams the other through
// LDS, so neither the scores nor G ever leave the registers.
//
//   rows pass:    X = 128 rows of h, Y = the classes of a split.  S' = Y X' gives a lane
//                 scores of one row: running maximum, sum, and O' += Y' P' with
//                 P = exp(S - maximum).  The splits' parts of a row are joined into lse,
//                 loss and dh = w (O / sum - W_label).
//   classes pass: X = 128 classes, Y = the rows of a split.  P = exp(S - lse) less the
//                 label's 1, times the row's weight; O' += Y' P' is dW, parts summed in
//                 order.
//
// Both products of a tile read the same LDS rows: the first along them, the second
// across (ds_read_tr16_b64).  S' comes out with a lane's values 8 (r / 4) + 4 half +
// r % 4 of Y; the second product's sum over Y may take them in any order, so the
// lane's own registers, rounded, are its operand, and the read across picks Y's
// rows in that order: no value moves between lanes.
//
// Operands are one f16 term (bf16) or two (f32), as kernels_xent.hip says, but one packed h
// serves the scores and dW.  So a column of W is packed times 2^c and h's times 2^-c, half the
// difference of their sizes (h's over the rows, each brought to the size 1): both columns'
// largest are then 2^-k of the largest of all if their product is 2^-2k of the largest product,
// and are held with 22 bits up to k = 16, with 38 - k from there on.  P carries the rows' weights
// over their powers of two into dW, off by 2^-40 of the largest.
//
// 20000 x 100 x 10000 f32 takes 262 and 275 us, 1.12 and 1.06 PFLOP/s of f16 products (112 columns
// of the first and 128 of the second, three terms), with the matrix cores busy 51 to 54 % of the
// cycles at 1.92 to 1.96 GHz.  Without the exponentials the rows pass takes 6 % less, without the
// split of P into terms 5 %.  bf16, with a third of the products and as many exponentials, takes
// 128 and 146 us: matrix cores busy 34 and 29 %, vector instructions 41 and 37 %.
#include <algorithm>

#include "mbk.h"
#include "xent.hpp"

namespace mbk {

namespace {

typedef __attribute__((ext_vector_type(4))) unsigned short u16x4;

constexpr int XB = 128;                  // X rows of a workgroup, 32 a wavefront
constexpr int TY = 64;                   // Y rows of a tile
// p = exp(z - maximum) is kept times 2^13, and the maximum may lag by 2 log 2, so that p as
// f16 terms is at most 2^15 and keeps steps of 2^-38.
constexpr int P_EXP = 13;
constexpr float LAG = 1.38f;
// exp(z - ref) is 2^(z log2 e + c), c = -ref log2 e, in two instructions, else in three (bf16 20000
// x 32 x 10000 with gradients 187 us, by three always 195).  c's rounding is a relative error of
// |ref| 2^-24, no more than z's own: up to here 2^-16.
constexpr float FAR = 256.0f;

// Elements of a packed row for KS slabs of 16.
__host__ __device__ constexpr int row_ld(int ks) { return ks <= 2 ? 32 : ks <= 4 ? 64 : 128; }

struct Fused {
    int64_t n, v, n_pad, v_pad;
    int32_t d;
    int32_t w_groups, h_groups, pack_groups;     // that look at W's and h's columns, pack
    bool few;                            // of the first two: those that pack sum them up
    XentCtl *ctl;
    int32_t *part, *col;                 // [group][ld] and [W, h][ld] largest exponents of columns
    int32_t *exp2;                       // [ld] a column of W is packed times 2^this
    u16 *h, *w;                          // planes of n_pad * ld, v_pad * ld
    float *bias;                         // [v_pad] the bias, -inf: not offered
    // of the rows, [n_pad]:
    float *sc;                           // the scale of a score
    int32_t *exp;                        // h is packed times 2^(exp - its column's exp2)
    int32_t *label;                      // -1: out, -2: out and not finite
    float *weight;                       // 0: out
    float *ref, *l2;                     // lse as a score and log2 of the sum, +inf: out
    float *c2;                           // -lse log2 e, where no row's is far
    float *wq;                           // weight as the classes pass multiplies with it
};

// The classes pass multiplies P with a row's weight over its power of two; E, of the largest
// of them, puts that below 2^15.  Words of XentMax hold E + ROW_BIAS, 0 for no row.
constexpr int ROW_BIAS = 1 << 14;
__device__ __forceinline__ int wq_exp(uint32_t row_max) {
    return row_max ? 15 - ((int)row_max - ROW_BIAS) : 0;
}

template <typename T> __device__ __forceinline__ float load_f32(const void *p, int64_t i) {
    return (float)static_cast<const T *>(p)[i];
}

// Up to four elements of a row from f on, zeros behind the row.
template <typename T>
__device__ __forceinline__ void load4(const void *p, int64_t row, int f, int d, float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = f + e < d ? load_f32<T>(p, row + f + e) : 0.0f;
}
// LD / 4 lanes a row in the kernels that prepare and join, and a grid that goes over
// the rows in turns.
template <int LANES> __device__ __forceinline__ int row_max(int m) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o, 64));
    return m;
}
// The largest exponents of the columns: of W by the first workgroups, which also leave the
// padded bias and whether a class is offered, and of h, less the row's largest, by those behind.
template <typename T, int LD>
__global__ __launch_bounds__(256) void k_fused_columns(Fused k, XentCall c) {
    constexpr int LANES = LD / 4, ROWS = 256 / LANES;
    __shared__ int32_t most[ROWS][LD];
    const int f = threadIdx.x % LANES * 4, r = threadIdx.x / LANES;
    int m[4] = {NO_EXP, NO_EXP, NO_EXP, NO_EXP};
    bool any = false;
    // four rows at a time, so that as many loads are on the way
    constexpr int AHEAD = 4;
    float x[AHEAD][4];
    bool in[AHEAD];
    if ((int32_t)blockIdx.x < k.w_groups) {
        const int64_t hop = (int64_t)k.w_groups * ROWS;
        for (int64_t v0 = (int64_t)blockIdx.x * ROWS + r; v0 < k.v_pad; v0 += AHEAD * hop) {
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int64_t v = v0 + q * hop;
                const float b = v < k.v ? (c.bias ? c.bias[v] : 0.0f) : -INFINITY;
                if (f == 0 && v < k.v_pad) k.bias[v] = b;
                in[q] = b != -INFINITY;
                any = any || in[q];
                load4<T>(c.w, (v < k.v ? v : 0) * c.w_stride, f, v < k.v ? k.d : 0, x[q]);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (in[q]) m[e] = max(m[e], exponent_of(x[q][e]));
        }
    } else {
        const int64_t hop = (int64_t)k.h_groups * ROWS;
        for (int64_t i0 = (int64_t)(blockIdx.x - k.w_groups) * ROWS + r; i0 < k.n;
             i0 += AHEAD * hop) {
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int64_t i = i0 + q * hop;
                const int32_t y = i < k.n ? c.labels[i] : -1;
                in[q] = y >= 0 && y < k.v && !(c.weights && c.weights[i] == 0.0f);
                load4<T>(c.h, (i < k.n ? i : 0) * c.h_stride, f, i < k.n ? k.d : 0, x[q]);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                int at[4], top = NO_EXP;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    at[e] = exponent_of(x[q][e]);
                    top = max(top, at[e]);
                }
                top = row_max<LANES>(top);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (in[q] && at[e] != NO_EXP) m[e] = max(m[e], at[e] - top);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) most[r][f + e] = m[e];
    const bool offered = __syncthreads_or(any);
    if ((int32_t)blockIdx.x < k.w_groups && threadIdx.x == 0)
        k.ctl->offered.part[blockIdx.x] = offered;
    if (threadIdx.x >= LD) return;
    int all = NO_EXP;
#pragma unroll
    for (int q = 0; q < ROWS; ++q) all = max(all, most[q][threadIdx.x]);
    k.part[(int64_t)blockIdx.x * LD + threadIdx.x] = all;
}

// Over the groups: 32 columns a workgroup, and 32 threads a column in turns.
__global__ __launch_bounds__(1024) void k_fused_scales(Fused k, int32_t ld) {
    __shared__ int32_t most[32][32];
    __shared__ uint32_t words[16];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const bool of_w = (int32_t)blockIdx.x < ld / 32;
    const int32_t col = (of_w ? blockIdx.x : blockIdx.x - ld / 32) * 32 + lane;
    const int32_t first = of_w ? 0 : k.w_groups, groups = of_w ? k.w_groups : k.h_groups;
    int m = NO_EXP;
#pragma unroll 8
    for (int g = slice; g < groups; g += 32) m = max(m, k.part[(int64_t)(first + g) * ld + col]);
    most[slice][lane] = m;
    if (blockIdx.x == 0) {
        const uint32_t any = largest_of<16>(k.ctl->offered, k.w_groups, words);
        if (threadIdx.x == 0) k.ctl->offered.all = any;
    }
    __syncthreads();
    if (slice != 0) return;
#pragma unroll
    for (int q = 1; q < 32; ++q) m = max(m, most[q][lane]);
    k.col[(of_w ? 0 : ld) + col] = m;
}

// The same of few groups, by each workgroup of the next kernel, without a launch (2000 x 64 x
// 2000 f32, 64 groups, 24.4 us and 25.1 with the launch, 3500 x 128 x 4000, 235 groups, 45 and
// 40): whether a class is offered.
constexpr int FEW_GROUPS = 64;
template <int LD>
__device__ __forceinline__ bool few_columns(const Fused &k, int32_t *col, int32_t (&part)[2][256]) {
    const int32_t c = threadIdx.x % LD, slice = threadIdx.x / LD;
    const int32_t *from = k.part + c;
    int w = NO_EXP, h = NO_EXP;
#pragma unroll 4
    for (int g = slice; g < k.w_groups; g += 256 / LD) w = max(w, from[g * LD]);
    from += k.w_groups * LD;
#pragma unroll 4
    for (int g = slice; g < k.h_groups; g += 256 / LD) h = max(h, from[g * LD]);
    const bool any = (int32_t)threadIdx.x < k.w_groups && k.ctl->offered.part[threadIdx.x];
    part[0][threadIdx.x] = w;
    part[1][threadIdx.x] = h;
    const bool offered = __syncthreads_or(any);
    if (threadIdx.x < 2 * LD) {
        const int32_t *p = part[threadIdx.x / LD] + c;
        int m = p[0];
#pragma unroll
        for (int q = 1; q < 256 / LD; ++q) m = max(m, p[q * LD]);
        col[threadIdx.x] = m;
    }
    __syncthreads();
    return offered;
}

// Column threadIdx.x's power of two, by the first LD threads: a, b are the largest exponents
// of W's and h's column; 2^c for W and 2^-c for h leave both at level (a + b) / 2, and the
// largest level goes to TOP_EXP.  A column that only one of them has goes to that level.
template <int LD>
__device__ __forceinline__ int column_exp(const int32_t *col, int32_t *words) {
    int a = NO_EXP, b = NO_EXP;
    if (threadIdx.x < LD) {
        a = col[threadIdx.x];
        b = col[LD + threadIdx.x];
    }
    const bool both = a != NO_EXP && b != NO_EXP;
    const int c = (b - a) >> 1;
    int level = largest<4>(both ? a + c : NO_EXP, words);
    if (level == NO_EXP) level = 0;
    return both ? c + TOP_EXP - level : a != NO_EXP ? TOP_EXP - a
                                      : b != NO_EXP ? b + TOP_EXP - 2 * level : 0;
}

// The packed rows of W and then of h.  A row that is out and whose scores may not be finite
// is packed as zeros, its label -2.
constexpr int ZERO_ROW = 1 << 20;        // of exp: nothing but zeros
template <typename T, int LD>
__global__ __launch_bounds__(256) void k_fused_pack(Fused k, XentCall c) {
    constexpr int LANES = LD / 4, ROWS = 256 / LANES;
    const int f = threadIdx.x % LANES * 4;
    __shared__ int32_t words[4], exps[LD], cols[2 * LD], part[2][256];
    const bool any = k.few ? few_columns<LD>(k, cols, part) : k.ctl->offered.all != 0;
    const int mine = column_exp<LD>(k.few ? cols : k.col, words);
    if (threadIdx.x < LD) {
        exps[threadIdx.x] = mine;
        if (blockIdx.x == 0) k.exp2[threadIdx.x] = mine;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) k.ctl->far = 0;
    __syncthreads();
    int ex[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ex[e] = exps[f + e];
    uint32_t row = 0;
    for (int64_t at = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; at < k.v_pad + k.n_pad;
         at += (int64_t)k.pack_groups * ROWS) {
        const bool of_w = at < k.v_pad;
        const int64_t i = of_w ? at : at - k.v_pad;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        int s[4] = {ex[0], ex[1], ex[2], ex[3]};
        if (of_w) {
            if (k.bias[i] != -INFINITY) load4<T>(c.w, i * c.w_stride, f, k.d, x);
        } else {
            if (i < k.n) load4<T>(c.h, i * c.h_stride, f, k.d, x);
            int32_t y = i < k.n ? c.labels[i] : -1;
            float wt = i < k.n ? (c.weights ? c.weights[i] : 1.0f) : 0.0f;
            int m = NO_EXP;
            bool huge = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m = max(m, exponent_of(x[e]) - ex[e]);
                huge = huge || __float_as_uint(fabsf(x[e])) >= XENT_HUGE;
            }
            m = row_max<LANES>(m);
            huge = row_max<LANES>(huge);
            const bool zeros = m < NO_EXP / 2;
            int exp = zeros ? 0 : TOP_EXP - m;
            if (y < 0 || y >= k.v || wt == 0.0f || !any) {
                wt = 0.0f;
                y = -1;
                if (huge || exp < FAR_ROW) {
                    y = -2;
                    exp = 0;
                    x[0] = x[1] = x[2] = x[3] = 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = exp - ex[e];
            if (f == 0) {
                k.label[i] = y;
                k.weight[i] = wt;
                k.exp[i] = zeros ? ZERO_ROW : exp;
                k.sc[i] = power_of_2(-exp);
                const int e = exponent_of(wt);
                if (!zeros && e != NO_EXP) row = max(row, (uint32_t)(e - exp + ROW_BIAS));
            }
        }
        u16 *to = (of_w ? k.w : k.h) + i * LD + f;
        u16 hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split_f16(ldexpf(x[e], s[e]), hi[e], lo[e]);
        *reinterpret_cast<u16x4 *>(to) = u16x4{hi[0], hi[1], hi[2], hi[3]};
        if (sizeof(T) == 4)
            *reinterpret_cast<u16x4 *>(to + (of_w ? k.v_pad : k.n_pad) * LD) =
                u16x4{lo[0], lo[1], lo[2], lo[3]};
    }
    const uint32_t most = largest<4>(row, reinterpret_cast<uint32_t *>(words));
    if (threadIdx.x == 0) k.ctl->row.part[blockIdx.x] = most;
}

// ---- a tile in LDS -----------------------------------------------------------------
// TY rows of LD elements a plane, the 16-byte chunks of a row permuted by the row so
// that the 16 rows x 1 chunk of a read along and the 4 rows x 4 chunks of a read
// across fall on all 64 banks.  Rows 8 apart differ in bit 1 alone, rows 16 apart not
// at all.
template <int LD> __device__ __forceinline__ int chunk_xor(int row) {
    const int low = (row >> 2) & 3;
    if constexpr (LD == 32) return low;
    else if constexpr (LD == 64) return ((row >> 1) & 1) * 4 + low;
    else return (row & 3) * 4 + low;
}
template <int P, int LD> constexpr int TILE_BYTES = P * TY * LD * 2;

// Starts the copies of a tile's operand; the LDS side is linear, so the source is
// read in the permuted order.
template <int P, int LD>
__device__ __forceinline__ void load_tile(const u16 *src, int64_t plane, char *lds, int wave) {
    constexpr int ROW = LD * 2, PLANE = TY * ROW;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int q = 0; q < PLANE / 4096; ++q) {
            const int at = (q * 4 + wave) * 1024, o = at + lane * 16;
            const int row = o / ROW, chunk = (o % ROW / 16) ^ chunk_xor<LD>(row);
            __builtin_amdgcn_global_load_lds(
                (global_void *)(src + p * plane + row * LD + chunk * 8),
                (lds_void *)(lds + p * PLANE + at), 16, 0, 0);
        }
}

template <int P, int LD>
__device__ __forceinline__ void along(const char *lds, int row, int slab, u32x4 (&f)[P]) {
    const int lane = threadIdx.x & 63, r = row + (lane & 31);
    const int chunk = (slab * 2 + (lane >> 5)) ^ chunk_xor<LD>(r);
#pragma unroll
    for (int p = 0; p < P; ++p)
        f[p] = *reinterpret_cast<const u32x4 *>(lds + p * (TY * LD * 2) + r * (LD * 2) + chunk * 16);
}

typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

// Eight values as the second product's operand.
template <int P> __device__ __forceinline__ void pack8(const float (&x)[8], u32x4 (&f)[P]) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const f16x2 hi = {(_Float16)x[e], (_Float16)x[e + 1]};
        const uint32_t h = __builtin_bit_cast(uint32_t, hi);
        f[0][e / 2] = h;
        if constexpr (P == 2) {
            float r0, r1;                // x - hi in one instruction each
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(h), "v"(x[e]));
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
                : "=v"(r1) : "v"(h), "v"(x[e + 1]));
            const f16x2 lo = {(_Float16)r0, (_Float16)r1};
            f[1][e / 2] = __builtin_bit_cast(uint32_t, lo);
        }
    }
}

// The reads across, for the columns of two blocks of 32 (one with LD == 32): lane l gets
// column l % 32 of the block and rows 4 (l / 32) + 0..3 and 8 + that.  They wait for
// themselves: the compiler would have the builtin wait for the copies of the next
// tile too, which no read here depends on.
template <int LD> __device__ __forceinline__ int across_at() {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    const int r = (g >> 1) * 4 + (i >> 2), c = (g & 1) * 16 + (i & 3) * 4;
    return r * (LD * 2) + ((c >> 3) ^ chunk_xor<LD>(r)) * 16 + (c & 7) * 2;
}
#define TR(dst, addr, off) "ds_read_b64_tr_b16 " dst ", " addr " offset:" off "\n\t"
template <int P, int LD, int ROW, int COL>
__device__ __forceinline__ void across(uint32_t at, u32x4 (&f)[2][P]) {
    constexpr int R = LD * 2, O = ROW * R, O8 = O + 8 * R, PLANE = TY * R;
    // the block's columns, its rows 8 further, and both for the pair's other block
    const uint32_t a0 = at ^ (COL * 2), a8 = a0 ^ 32, b0 = a0 ^ 64, b8 = a0 ^ 96;
    u32x2 x[2][P][2];
    if constexpr (LD == 32 && P == 1) {
        asm volatile(TR("%0", "%2", "%4") TR("%1", "%3", "%5") "s_waitcnt lgkmcnt(0)"
                     : "=&v"(x[0][0][0]), "=&v"(x[0][0][1])
                     : "v"(a0), "v"(a8), "n"(O), "n"(O8)
                     : "memory");
    } else if constexpr (LD == 32) {
        asm volatile(TR("%0", "%4", "%6") TR("%1", "%5", "%7") TR("%2", "%4", "%8")
                     TR("%3", "%5", "%9") "s_waitcnt lgkmcnt(0)"
                     : "=&v"(x[0][0][0]), "=&v"(x[0][0][1]), "=&v"(x[0][1][0]), "=&v"(x[0][1][1])
                     : "v"(a0), "v"(a8), "n"(O), "n"(O8), "n"(PLANE + O), "n"(PLANE + O8)
                     : "memory");
    } else if constexpr (P == 1) {
        asm volatile(TR("%0", "%4", "%8") TR("%1", "%5", "%9") TR("%2", "%6", "%8")
                     TR("%3", "%7", "%9") "s_waitcnt lgkmcnt(0)"
                     : "=&v"(x[0][0][0]), "=&v"(x[0][0][1]), "=&v"(x[1][0][0]), "=&v"(x[1][0][1])
                     : "v"(a0), "v"(a8), "v"(b0), "v"(b8), "n"(O), "n"(O8)
                     : "memory");
    } else {
        asm volatile(TR("%0", "%8", "%12") TR("%1", "%9", "%13") TR("%2", "%8", "%14")
                     TR("%3", "%9", "%15") TR("%4", "%10", "%12") TR("%5", "%11", "%13")
                     TR("%6", "%10", "%14") TR("%7", "%11", "%15") "s_waitcnt lgkmcnt(0)"
                     : "=&v"(x[0][0][0]), "=&v"(x[0][0][1]), "=&v"(x[0][1][0]), "=&v"(x[0][1][1]),
                       "=&v"(x[1][0][0]), "=&v"(x[1][0][1]), "=&v"(x[1][1][0]), "=&v"(x[1][1][1])
                     : "v"(a0), "v"(a8), "v"(b0), "v"(b8), "n"(O), "n"(O8), "n"(PLANE + O),
                       "n"(PLANE + O8)
                     : "memory");
    }
#pragma unroll
    for (int j = 0; j < (LD == 32 ? 1 : 2); ++j)
#pragma unroll
        for (int p = 0; p < P; ++p)
            f[j][p] = u32x4{x[j][p][0][0], x[j][p][0][1], x[j][p][1][0], x[j][p][1][1]};
}
#undef TR

// O' += Y' P' for the 32 rows of Y from row Y on, P in p.
template <int P, int KS, int Y>
__device__ __forceinline__ void second_product(uint32_t at, const float (&p)[2][8],
                                               f32x16 (&o)[(KS + 1) / 2]) {
    constexpr int LD = row_ld(KS), JT = (KS + 1) / 2;
    u32x4 b[2][P];
    pack8<P>(p[0], b[0]);
    pack8<P>(p[1], b[1]);
    u32x4 a[2][P];
    across<P, LD, Y, 0>(at, a);
    o[0] = mma<P>(a[0], b[0], o[0]);
    if constexpr (JT > 1) o[1] = mma<P>(a[1], b[0], o[1]);
    if constexpr (JT > 2) {
        across<P, LD, Y, 64>(at, a);
        o[2] = mma<P>(a[0], b[0], o[2]);
        if constexpr (JT > 3) o[3] = mma<P>(a[1], b[0], o[3]);
    }
    across<P, LD, Y + 16, 0>(at, a);
    o[0] = mma<P>(a[0], b[1], o[0]);
    if constexpr (JT > 1) o[1] = mma<P>(a[1], b[1], o[1]);
    if constexpr (JT > 2) {
        across<P, LD, Y + 16, 64>(at, a);
        o[2] = mma<P>(a[0], b[1], o[2]);
        if constexpr (JT > 3) o[3] = mma<P>(a[1], b[1], o[3]);
    }
}

// S' of the 32 rows of Y from row y on: all of the operand is asked for first.
template <int P, int KS>
__device__ __forceinline__ f32x16 first_product(const char *tile, int y, const u32x4 (&x)[KS][P]) {
    constexpr int LD = row_ld(KS), STEP = KS < 4 ? KS : 4;
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int q0 = 0; q0 < KS; q0 += STEP) {
        u32x4 a[STEP][P];
#pragma unroll
        for (int q = 0; q < STEP; ++q)
            if (q0 + q < KS) along<P, LD>(tile, y, q0 + q, a[q]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < STEP; ++q)
            if (q0 + q < KS) s = mma<P>(a[q], x[q0 + q], s);
    }
    return s;
}
// The values of 16 rows of Y that go with a lane's registers of S'.
template <typename V> __device__ __forceinline__ void of_rows(const V *rows, int y, V (&out)[16]) {
    typedef __attribute__((ext_vector_type(4))) V V4;
    const V *from = rows + y + ((threadIdx.x & 63) >> 5) * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const V4 v = *reinterpret_cast<const V4 *>(from + 8 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[q * 4 + e] = v[e];
    }
}
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// ---- rows pass ----------------------------------------------------------------------
// part_o[split][row][ld], part_ms[split][row] = (reference, sum): sum and O are of
// 2^13 exp(z - reference).
template <int P, int KS, bool GRAD>
__global__ __launch_bounds__(256, 2) void k_fused_rows(Fused k, int32_t splits,
                                                       float *__restrict__ part_o,
                                                       float2 *__restrict__ part_ms) {
    constexpr int LD = row_ld(KS), JT = (KS + 1) / 2;
    constexpr int BUF = TILE_BYTES<P, LD> + TY * 4;      // a multiple of 256: see across
    extern __shared__ char lds[];
    if (GRAD && blockIdx.x == 0) {       // for the kernels behind this one
        const uint32_t most = largest_of<4>(k.ctl->row, k.pack_groups,
                                            reinterpret_cast<uint32_t *>(lds));
        if (threadIdx.x == 0) k.ctl->row.all = most;
    }
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t x0 = (int64_t)(blockIdx.x / splits) * XB;
    const int32_t split = blockIdx.x % splits;
    const int64_t tiles = k.v_pad / TY, first = tiles * split / splits,
                  last = tiles * (split + 1) / splits;
    const int64_t row = x0 + wave * 32 + (lane & 31);
    u32x4 x[KS][P];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int p = 0; p < P; ++p)
            x[s][p] = *reinterpret_cast<const u32x4 *>(k.h + p * k.n_pad * LD + row * LD + s * 16 +
                                                       half * 8);
    const float sc = k.sc[row];
    float ref = 0.0f, top = -INFINITY, sum = 0.0f, c2 = P_EXP;
    bool far = false;                    // of the wavefront
    f32x16 o[GRAD ? JT : 1];
#pragma unroll
    for (int j = 0; j < (GRAD ? JT : 1); ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[j][r] = 0.0f;

    auto load = [&](int64_t t, int buf) {
        char *to = lds + buf * BUF;
        load_tile<P, LD>(k.w + t * TY * LD, k.v_pad * LD, to, wave);
        if (wave == 0)
            __builtin_amdgcn_global_load_lds((global_void *)(k.bias + t * TY + lane),
                                             (lds_void *)(to + TILE_BYTES<P, LD>), 4, 0, 0);
    };
    if (first < last) load(first, 0);
    for (int64_t t = first; t < last; ++t) {
        const int buf = (t - first) & 1;
        copies_done();
        __syncthreads();                 // the tile is there; the other one is read
        if (t + 1 < last) load(t + 1, buf ^ 1);
        const char *tile = lds + buf * BUF;
        const float *bias = reinterpret_cast<const float *>(tile + TILE_BYTES<P, LD>);
        const uint32_t at = lds_address(tile) + across_at<LD>();
        static_assert(BUF % 256 == 0, "reads across xor the low bits of the address");
        auto block = [&](auto where) {
            constexpr int y = decltype(where)::value;
            float b[16];
            of_rows(bias, y, b);
            f32x16 s = first_product<P, KS>(tile, y, x);
            float m = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = __builtin_fmaf(s[r], sc, b[r]);
                m = fmaxf(m, s[r]);
            }
            // a new maximum: what was summed so far is brought to it, of the rows that have
            // one, so that no row's bits depend on another's
            if (__any(m > top + LAG)) {
                const float now = fmaxf(m, other_half(m));
                if (now > top + LAG) {
                    const float scale = top == -INFINITY ? 0.0f : exp_of(top - now);
                    sum *= scale;
                    if constexpr (GRAD)
#pragma unroll
                        for (int j = 0; j < JT; ++j)
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[j][r] *= scale;
                    ref = top = now;
                    c2 = __builtin_fmaf(-ref, LOG2E, (float)P_EXP);
                }
                far = __any(fabsf(ref) >= FAR);
            }
            float p[2][8], part[2] = {0.0f, 0.0f};
            if (far) {
                const bool mine = fabsf(ref) >= FAR;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[r] = mine ? __builtin_fmaf(s[r] - ref, LOG2E, (float)P_EXP)
                                : __builtin_fmaf(s[r], LOG2E, c2);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], LOG2E, c2);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[r >> 3][r & 7] = __builtin_amdgcn_exp2f(s[r]);
                part[r & 1] += p[r >> 3][r & 7];
            }
            sum += part[0] + part[1];
            if constexpr (GRAD) second_product<P, KS, y>(at, p, o);
        };
        block(At<0>{});
        block(At<32>{});
    }
    sum += other_half(sum);
    const int64_t at = split * k.n_pad + row;
    if (half == 0) part_ms[at] = make_float2(top, sum);
    if constexpr (GRAD) {
        float *out = part_o + at * LD;
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4 *>(out + j * 32 + q * 8 + half * 4) =
                    make_float4(o[j][q * 4], o[j][q * 4 + 1], o[j][q * 4 + 2], o[j][q * 4 + 3]);
    }
}

// The splits of a row joined, LD / 4 lanes a row; its label's score is summed in f32
// from h and W themselves.
template <typename T, int LD, bool GRAD>
__global__ __launch_bounds__(256) void k_fused_join_rows(Fused k, XentCall c, int32_t splits,
                                                         const float *__restrict__ part_o,
                                                         const float2 *__restrict__ part_ms) {
    constexpr int LANES = LD / 4;
    const int64_t i = (int64_t)group_id() * (256 / LANES) + threadIdx.x / LANES;
    if (i >= k.n_pad) return;
    const int f = threadIdx.x % LANES * 4;
    const int32_t y = k.label[i];
    const bool open = y >= 0 && k.bias[y] != -INFINITY;
    const float wt = k.weight[i];
    const int32_t exp = k.exp[i];
    int32_t ex[4] = {0, 0, 0, 0}, row_exp = 0;       // asked for ahead of the stores
    if constexpr (GRAD) {
#pragma unroll
        for (int e = 0; e < 4; ++e) ex[e] = k.exp2[f + e];
        row_exp = wq_exp(k.ctl->row.all);
    }
    float wy[4] = {0.0f, 0.0f, 0.0f, 0.0f}, dot = 0.0f;
    if (open)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (f + e < k.d) {
                wy[e] = load_f32<T>(c.w, y * c.w_stride + f + e);
                dot += wy[e] * load_f32<T>(c.h, i * c.h_stride + f + e);
            }
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) dot += __shfl_xor(dot, m, 64);
    float ref = -INFINITY;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) ref = fmaxf(ref, part_ms[s * k.n_pad + i].x);
    const bool none = ref == -INFINITY;
    float sum = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float2 ms = part_ms[s * k.n_pad + i];
        const float scale = none ? 1.0f : exp_of(ms.x - ref);
        sum += ms.y * scale;
        if constexpr (GRAD) {
            const float4 p = *reinterpret_cast<const float4 *>(part_o + (s * k.n_pad + i) * LD + f);
            o[0] += p.x * scale;
            o[1] += p.y * scale;
            o[2] += p.z * scale;
            o[3] += p.w * scale;
        }
    }
    const LogSum l = log_sum(sum, P_EXP);
    if (f == 0) {
        if (i < k.n) {
            const float z = open ? dot + (c.bias ? c.bias[y] : 0.0f) : -INFINITY;
            c.lse[i] = y == -2 ? NAN : lse_of(ref, l);
            c.loss[i] = y < 0 ? 0.0f : wt * loss_of(ref, l, z);
        }
        if constexpr (GRAD) {
            k.ref[i] = y < 0 ? 0.0f : ref;
            k.l2[i] = y < 0 ? INFINITY : l.base2;
            k.c2[i] = y < 0 ? -INFINITY : -__builtin_fmaf(ref, LOG2E, l.base2);
            if (y >= 0 && fabsf(ref) >= FAR) k.ctl->far = 1;
            // a row of zeros has no power of two; a weight that is not finite stays so
            k.wq[i] = exp != ZERO_ROW ? ldexpf(wt, row_exp - exp)
                                      : fabsf(wt) < INFINITY ? 0.0f : wt;
        }
    }
    if constexpr (GRAD) {
        if (!c.dh || i >= k.n) return;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (f + e < k.d) {
                // divided first: the sum of 2^13 p W is beyond f32 for W that is not
                const float g = y < 0 ? 0.0f : wt * (ldexpf(o[e] / sum, -ex[e]) - wy[e]);
                static_cast<T *>(c.dh)[i * c.h_stride + f + e] = (T)g;
            }
    }
}

// ---- classes pass ---------------------------------------------------------------------
// part[split][class][ld] of dW, part_db[split][class]
constexpr int ROW_ARRAYS = 5;            // of a tile's rows: sc, c2, wq, label, weight
template <int P, int KS>
__global__ __launch_bounds__(256, 2) void k_fused_classes_pass(Fused k, int32_t splits,
                                                               float *__restrict__ part,
                                                               float *__restrict__ part_db) {
    constexpr int LD = row_ld(KS), JT = (KS + 1) / 2;
    constexpr int ROWS_AT = TILE_BYTES<P, LD>;           // ROW_ARRAYS of them
    constexpr int BUF = ROWS_AT + ROW_ARRAYS * TY * 4;
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t x0 = (int64_t)(blockIdx.x / splits) * XB + wave * 32;
    const int32_t split = blockIdx.x % splits;
    const int64_t tiles = k.n_pad / TY, first = tiles * split / splits,
                  last = tiles * (split + 1) / splits;
    const int64_t v = x0 + (lane & 31);
    u32x4 x[KS][P];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int p = 0; p < P; ++p)
            x[s][p] = *reinterpret_cast<const u32x4 *>(k.w + p * k.v_pad * LD + v * LD + s * 16 +
                                                       half * 8);
    const float b = k.bias[v];
    const bool far = k.ctl->far;
    double db = 0.0;                     // of sums over 32 rows
    f32x16 o[JT];
#pragma unroll
    for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[j][r] = 0.0f;

    auto load = [&](int64_t t, int buf) {
        char *to = lds + buf * BUF;
        load_tile<P, LD>(k.h + t * TY * LD, k.n_pad * LD, to, wave);
        const void *rows[ROW_ARRAYS] = {k.sc, k.c2, k.wq, k.label, k.weight};
#pragma unroll
        for (int q = 0; q < ROW_ARRAYS; ++q)
            if (wave == (q & 3))
                __builtin_amdgcn_global_load_lds(
                    (global_void *)(static_cast<const float *>(rows[q]) + t * TY + lane),
                    (lds_void *)(to + ROWS_AT + q * TY * 4), 4, 0, 0);
    };
    if (first < last) load(first, 0);
    for (int64_t t = first; t < last; ++t) {
        const int buf = (t - first) & 1;
        copies_done();
        __syncthreads();
        if (t + 1 < last) load(t + 1, buf ^ 1);
        const char *tile = lds + buf * BUF;
        const float *sc = reinterpret_cast<const float *>(tile + ROWS_AT), *c2 = sc + TY,
                    *wq = sc + 2 * TY, *weight = sc + 4 * TY;
        const int32_t *label = reinterpret_cast<const int32_t *>(sc + 3 * TY);
        const uint32_t at = lds_address(tile) + across_at<LD>();
        static_assert(BUF % 256 == 0, "reads across xor the low bits of the address");
        auto block = [&](auto where) {
            constexpr int y = decltype(where)::value;
            const int64_t mine = label[y + (lane & 31)] - x0;
            const bool hot = __any(mine >= 0 && mine < 32);
            f32x16 s = first_product<P, KS>(tile, y, x);
            float p[2][8], of[16], of2[16];
            of_rows(c2, y, of);
            of_rows(sc, y, of2);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], of2[r], b);
            if (far) {
                float ref[16];
                of_rows(k.ref + t * TY, y, ref);
                of_rows(k.l2 + t * TY, y, of2);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[r] = fabsf(ref[r]) >= FAR ? __builtin_fmaf(s[r] - ref[r], LOG2E, -of2[r])
                                                : __builtin_fmaf(s[r], LOG2E, of[r]);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], LOG2E, of[r]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r >> 3][r & 7] = __builtin_amdgcn_exp2f(s[r]);
            if (hot) {
                int32_t l[16];
                of_rows(label, y, l);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (l[r] == v) p[r >> 3][r & 7] -= 1.0f;
            }
            if (part_db) {
                float sum = 0.0f;
                of_rows(weight, y, of);
#pragma unroll
                for (int r = 0; r < 16; ++r) sum = __builtin_fmaf(p[r >> 3][r & 7], of[r], sum);
                db += sum;
            }
            of_rows(wq, y, of);
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r >> 3][r & 7] *= of[r];
            second_product<P, KS, y>(at, p, o);
        };
        block(At<0>{});
        block(At<32>{});
    }
    const int64_t at = split * k.v_pad + v;
    if (part_db) {
        db += __shfl_xor(db, 32, 64);
        if (half == 0) part_db[at] = (float)db;
    }
    float *out = part + at * LD;
#pragma unroll
    for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4 *>(out + j * 32 + q * 8 + half * 4) =
                make_float4(o[j][q * 4], o[j][q * 4 + 1], o[j][q * 4 + 2], o[j][q * 4 + 3]);
}

// LD / 4 lanes a class, and where there are many splits SPLIT_GROUPS of them, whose sums
// are added in order.
constexpr int SPLIT_GROUPS = 8;
template <typename T, int LD, bool GROUPS>
__global__ __launch_bounds__(256) void k_fused_join_classes(Fused k, XentCall c, int32_t splits,
                                                            const float *__restrict__ part,
                                                            const float *__restrict__ part_db) {
    constexpr int LANES = LD / 4, G = GROUPS ? SPLIT_GROUPS : 1, CLASSES = 256 / LANES / G;
    __shared__ float4 sums[GROUPS ? 256 : 1];
    __shared__ double dbs[GROUPS ? 256 : 1];
    const int l = threadIdx.x % LANES, f = l * 4;
    const int g = threadIdx.x / LANES % G;
    const int64_t v = (int64_t)group_id() * CLASSES + threadIdx.x / (LANES * G);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    double db = 0.0;
    if (v < k.v) {
#pragma unroll 4
        for (int s = g; s < splits; s += G) {
            const float4 p = *reinterpret_cast<const float4 *>(part + (s * k.v_pad + v) * LD + f);
            sum.x += p.x;
            sum.y += p.y;
            sum.z += p.z;
            sum.w += p.w;
            if (c.dbias && l == 0) db += part_db[s * k.v_pad + v];
        }
    }
    if constexpr (GROUPS) {
        sums[threadIdx.x] = sum;
        dbs[threadIdx.x] = db;
        __syncthreads();
        if (g != 0) return;
        for (int o = 1; o < G; ++o) {
            const float4 p = sums[threadIdx.x + o * LANES];
            sum.x += p.x;
            sum.y += p.y;
            sum.z += p.z;
            sum.w += p.w;
            db += dbs[threadIdx.x + o * LANES];
        }
    }
    if (v >= k.v) return;
    const bool open = k.bias[v] != -INFINITY;
    const int exp = wq_exp(k.ctl->row.all);
    int32_t ex[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ex[e] = k.exp2[f + e];
    const float x[4] = {sum.x, sum.y, sum.z, sum.w};
    if (c.dw)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (f + e < k.d)
                static_cast<T *>(c.dw)[v * c.w_stride + f + e] =
                    (T)(open ? ldexpf(x[e], ex[e] - exp) : 0.0f);
    if (c.dbias && l == 0) c.dbias[v] = open ? (float)db : 0.0f;
}

// ---- the call ---------------------------------------------------------------------------
int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
uint32_t blocks(int64_t x, int64_t per) { return (uint32_t)((x + per - 1) / per); }

// Workgroups for `blocks` X blocks over `tiles` Y tiles: two run on a CU at once, and
// the last round of them should be full.  At least 4 tiles a split, and at most 512 MB of
// parts, unless one takes more: past that a fuller last round is a few percent of many (1M x 128
// x 1M f32: 11 splits and 5.6 GB for 4 %).
constexpr int64_t PART_BYTES = (int64_t)512 << 20;
int32_t pick_splits(int64_t x_blocks, int64_t tiles, int64_t part_bytes, int num_cus) {
    const int64_t slots = 2 * (int64_t)num_cus;
    const int64_t most =
        std::max<int64_t>(1, std::min<int64_t>({tiles / 4, 64, PART_BYTES / part_bytes}));
    int64_t best = 1;
    double cost = 1e30;
    for (int64_t s = 1; s <= most; ++s) {
        // rounds of workgroups times a workgroup's tiles, and its start and end
        const double c = (double)((x_blocks * s + slots - 1) / slots) *
                         ((double)((tiles + s - 1) / s) + 3.0);
        if (c < cost) {
            cost = c;
            best = s;
        }
    }
    return (int32_t)best;
}

struct Plan {
    int P, ks;
    int64_t n_pad, v_pad, ld;
    int32_t row_splits, class_splits;
    int32_t w_groups, h_groups;
    size_t ctl, col_part, col, exp2, h, w, bias, rows, part_ms, part, part_db, end;
};

Plan plan_of(const XentCall &c) {
    Plan p{};
    p.P = c.bf16 ? 1 : 2;
    p.ks = (c.dim + 15) / 16;
    p.ld = row_ld(p.ks);
    p.n_pad = up(c.rows, XB);
    p.v_pad = up(c.classes, XB);
    // of the loss alone as with gradients, so that its bits are the same
    const int64_t part_row = 4 * p.ld;
    p.row_splits = pick_splits(p.n_pad / XB, p.v_pad / TY, part_row * p.n_pad, c.num_cus);
    p.class_splits = pick_splits(p.v_pad / XB, p.n_pad / TY, part_row * p.v_pad, c.num_cus);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    // workgroups of k_fused_columns: eight a CU, four rows a thread or more
    const auto groups = [&](int64_t rows) {
        return (int32_t)std::max<int64_t>(
            1, std::min<int64_t>((rows * p.ld + 4095) / 4096, std::min(4 * c.num_cus, MOST_GROUPS)));
    };
    p.w_groups = groups(p.v_pad);
    p.h_groups = groups(p.n_pad);
    p.ctl = take(sizeof(XentCtl));
    p.col_part = take((size_t)4 * (p.w_groups + p.h_groups) * p.ld);
    p.col = take((size_t)8 * p.ld);
    p.exp2 = take((size_t)4 * p.ld);
    p.h = take((size_t)2 * p.P * p.n_pad * p.ld);
    p.w = take((size_t)2 * p.P * p.v_pad * p.ld);
    p.bias = take((size_t)4 * p.v_pad);
    p.rows = take((size_t)8 * 4 * p.n_pad);
    p.part_ms = take((size_t)8 * p.row_splits * p.n_pad);
    if (c.grad) {
        p.part = take((size_t)4 * p.ld * std::max(p.row_splits * p.n_pad, p.class_splits * p.v_pad));
        p.part_db = take((size_t)4 * p.class_splits * p.v_pad);
    }
    p.end = at;
    return p;
}

template <int P, int KS, typename T>
hipError_t run(hipStream_t s, const XentCall &c, const Plan &p, char *m) {
    constexpr int LD = row_ld(KS);
    Fused k{};
    k.n = c.rows;
    k.v = c.classes;
    k.n_pad = p.n_pad;
    k.v_pad = p.v_pad;
    k.d = c.dim;
    k.ctl = reinterpret_cast<XentCtl *>(m + p.ctl);
    k.w_groups = p.w_groups;
    k.h_groups = p.h_groups;
    k.few = k.w_groups + k.h_groups <= FEW_GROUPS;
    k.part = reinterpret_cast<int32_t *>(m + p.col_part);
    k.col = reinterpret_cast<int32_t *>(m + p.col);
    k.exp2 = reinterpret_cast<int32_t *>(m + p.exp2);
    k.h = reinterpret_cast<u16 *>(m + p.h);
    k.w = reinterpret_cast<u16 *>(m + p.w);
    k.bias = reinterpret_cast<float *>(m + p.bias);
    float *rows = reinterpret_cast<float *>(m + p.rows);
    k.sc = rows;
    k.exp = reinterpret_cast<int32_t *>(rows + p.n_pad);
    k.label = reinterpret_cast<int32_t *>(rows + 2 * p.n_pad);
    k.weight = rows + 3 * p.n_pad;
    k.ref = rows + 4 * p.n_pad;
    k.l2 = rows + 5 * p.n_pad;
    k.wq = rows + 6 * p.n_pad;
    k.c2 = rows + 7 * p.n_pad;
    float2 *part_ms = reinterpret_cast<float2 *>(m + p.part_ms);
    float *part = reinterpret_cast<float *>(m + p.part);
    float *part_db = reinterpret_cast<float *>(m + p.part_db);
    const dim3 b(256);
    const size_t lds_rows = 2 * (TILE_BYTES<P, LD> + TY * 4);
    const size_t lds_classes = 2 * (TILE_BYTES<P, LD> + ROW_ARRAYS * TY * 4);
    const void *big[] = {reinterpret_cast<const void *>(k_fused_rows<P, KS, true>),
                         reinterpret_cast<const void *>(k_fused_rows<P, KS, false>),
                         reinterpret_cast<const void *>(k_fused_classes_pass<P, KS>)};
    for (const void *f : big) {
        const hipError_t e = allow_all_lds(f);
        if (e != hipSuccess) return e;
    }
    k.pack_groups = (int32_t)std::min<int64_t>(((k.v_pad + k.n_pad) * LD + 1023) / 1024,
                                               std::min(8 * c.num_cus, MOST_GROUPS));
    hipLaunchKernelGGL((k_fused_columns<T, LD>), dim3((uint32_t)(k.w_groups + k.h_groups)), b, 0, s,
                       k, c);
    if (!k.few)
        hipLaunchKernelGGL(k_fused_scales, dim3(2 * LD / 32), dim3(1024), 0, s, k, LD);
    hipLaunchKernelGGL((k_fused_pack<T, LD>), dim3((uint32_t)k.pack_groups), b, 0, s, k, c);
    const dim3 gr((uint32_t)(k.n_pad / XB * p.row_splits));
    const dim3 gj = grid_of(blocks(k.n_pad, 1024 / LD));
    if (!c.grad) {
        hipLaunchKernelGGL((k_fused_rows<P, KS, false>), gr, b, lds_rows, s, k, p.row_splits,
                           static_cast<float *>(nullptr), part_ms);
        hipLaunchKernelGGL((k_fused_join_rows<T, LD, false>), gj, b, 0, s, k, c, p.row_splits, part,
                           part_ms);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((k_fused_rows<P, KS, true>), gr, b, lds_rows, s, k, p.row_splits, part,
                       part_ms);
    hipLaunchKernelGGL((k_fused_join_rows<T, LD, true>), gj, b, 0, s, k, c, p.row_splits, part,
                       part_ms);
    if (c.dw || c.dbias) {
        hipLaunchKernelGGL((k_fused_classes_pass<P, KS>),
                           dim3((uint32_t)(k.v_pad / XB * p.class_splits)), b, lds_classes, s, k,
                           p.class_splits, part, c.dbias ? part_db : nullptr);
        if (p.class_splits >= 2 * SPLIT_GROUPS)
            hipLaunchKernelGGL((k_fused_join_classes<T, LD, true>),
                               grid_of(blocks(k.v, 1024 / LD / SPLIT_GROUPS)), b, 0, s, k, c,
                               p.class_splits, part, part_db);
        else
            hipLaunchKernelGGL((k_fused_join_classes<T, LD, false>), grid_of(blocks(k.v, 1024 / LD)),
                               b, 0, s, k, c, p.class_splits, part, part_db);
    }
    return hipGetLastError();
}

template <int P, typename T>
hipError_t run_dim(hipStream_t s, const XentCall &c, const Plan &p, char *m) {
    switch (p.ks) {
    case 1: return run<P, 1, T>(s, c, p, m);
    case 2: return run<P, 2, T>(s, c, p, m);
    case 3: return run<P, 3, T>(s, c, p, m);
    case 4: return run<P, 4, T>(s, c, p, m);
    case 5: return run<P, 5, T>(s, c, p, m);
    case 6: return run<P, 6, T>(s, c, p, m);
    case 7: return run<P, 7, T>(s, c, p, m);
    default: return run<P, 8, T>(s, c, p, m);
    }
}

}  // namespace

size_t xent_fused_scratch(const XentCall &c) { return plan_of(c).end; }

hipError_t launch_xent_fused(hipStream_t s, const XentCall &c, char *scratch) {
    const Plan p = plan_of(c);
    return c.bf16 ? run_dim<1, __bf16>(s, c, p, scratch) : run_dim<2, float>(s, c, p, scratch);
}

}  // namespace mbk
