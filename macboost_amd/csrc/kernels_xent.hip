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
// Operands.  The matrix instructions take 16-bit operands and add in f32.  bf16
// inputs go in as they are, and G is rounded to bf16 (half a step, 2^-8 of each
// element at most, random in sign: what the outputs' own rounding to bf16 costs).  f32
// inputs go in as two f16 terms, x 2^s = hi + lo, which hold 22 bits of it, and
// three products hi hi + hi lo + lo hi: what is dropped, lo lo and the bits behind
// lo, is at most 2^-21 of an element's product and random in sign, the size of
// what an f32 sum over the same length rounds away.  (f32 operands have an
// instruction of 1/16 of the bf16 rate; three of these cost 3/16.)  s is a power of
// two that puts the largest element of h's row, or of all of W, below 2^14, so that
// elements down to 2^-38 of it keep a step of their own.
//
// Classes not offered (bias -inf) are packed as zeros, and so are rows that are out
// (label outside [0, V), weight 0, or no class offered) and hold NaN, infinities or values
// that could overflow: what they hold reaches nothing, and a finite row that is out is
// multiplied by zeros.
#include <algorithm>

#include "mbk.h"
#include "ops.h"
#include "xent.hpp"

namespace mbk {

namespace {

constexpr int TILE = 128;                // rows and columns of a workgroup's product
constexpr int LD_PAD = 128;              // operands' rows are padded to it
constexpr float G_SCALE = 32768.0f;      // f32: |G / w| <= 1 as f16 terms

__global__ void k_xent_init(XentCtl *ctl) {
    ctl->w_max = ctl->hg_max = ctl->open = 0;
}

template <typename T> __device__ __forceinline__ float load_f32(const void *p, int64_t i) {
    return (float)static_cast<const T *>(p)[i];
}

// Classes: the padded bias, whether any is offered, the largest |W|.
template <typename T>
__global__ __launch_bounds__(256) void k_xent_classes(XentPack k, const void *w, int64_t stride,
                                                      const float *__restrict__ bias) {
    const int lane = threadIdx.x & 63;
    const int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (v >= k.v_pad) return;
    const float b = v < k.v ? (bias ? bias[v] : 0.0f) : -INFINITY;
    const bool open = b != -INFINITY;
    if (lane == 0) {
        k.bias[v] = b * LOG2E;
        if (open && !k.ctl->open) k.ctl->open = 1u;
    }
    if (sizeof(T) == 2 || !open) return;
    uint32_t m = 0;
    for (int32_t f = lane; f < k.d; f += 64) m = max(m, finite_bits(load_f32<T>(w, v * stride + f)));
    m = wave_max(m);
    if (lane == 0) raise(&k.ctl->w_max, m);
}

template <typename T>
__global__ __launch_bounds__(256) void k_xent_pack_w(XentPack k, const void *w, int64_t stride) {
    const int lane = threadIdx.x & 63;
    const int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (v >= k.v_pad) return;
    const bool open = k.bias[v] != -INFINITY;
    const int s = sizeof(T) == 4 ? scale_exp(k.ctl->w_max) : 0;
    u16 *row = k.w + v * k.ld;
    for (int32_t f = lane; f < k.ld; f += 64) {
        const bool in = open && f < k.d;
        if (sizeof(T) == 2) {
            row[f] = in ? static_cast<const u16 *>(w)[v * stride + f] : 0;
        } else {
            u16 hi, lo;
            split_f16(in ? ldexpf(load_f32<T>(w, v * stride + f), s) : 0.0f, hi, lo);
            row[f] = hi;
            row[k.v_pad * k.ld + f] = lo;
        }
    }
}

// Rows: label and weight (-1 and 0 where the row is out), h scaled by row.  A row that
// is out and not finite is packed as zeros, its label -2.
template <typename T>
__global__ __launch_bounds__(256) void k_xent_rows(XentPack k, const void *h, int64_t stride,
                                                   const int32_t *__restrict__ labels,
                                                   const float *__restrict__ weights) {
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= k.n_pad) return;
    int32_t y = i < k.n ? labels[i] : -1;
    float wt = i < k.n ? (weights ? weights[i] : 1.0f) : 0.0f;
    const bool out = y < 0 || y >= k.v || wt == 0.0f || !k.ctl->open;
    int s = 0;
    bool zeros = i >= k.n;
    if (out) {
        y = -1;
        wt = 0.0f;
    }
    if ((out || sizeof(T) == 4) && i < k.n) {
        uint32_t m = 0, most = 0;
        for (int32_t f = lane; f < k.d; f += 64) {
            const float x = load_f32<T>(h, i * stride + f);
            m = max(m, finite_bits(x));
            most = max(most, __float_as_uint(fabsf(x)));
        }
        m = wave_max(m);
        if (out && wave_max(most) >= XENT_HUGE) {
            y = -2;
            m = 0;
            zeros = true;
        }
        if (sizeof(T) == 4) s = scale_exp(m);
        if (sizeof(T) == 4 && lane == 0 && wt != 0.0f)
            raise(&k.ctl->hg_max, finite_bits(wt * __uint_as_float(m)));
    }
    if (lane == 0) {
        if (sizeof(T) == 4) k.row_scale[i] = ldexpf(LOG2E, -(s + scale_exp(k.ctl->w_max)));
        k.label[i] = y;
        k.weight[i] = wt;
    }
    u16 *row = k.h + i * k.ld;
    for (int32_t f = lane; f < k.ld; f += 64) {
        const bool in = !zeros && f < k.d;
        if (sizeof(T) == 2) {
            row[f] = in ? static_cast<const u16 *>(h)[i * stride + f] : 0;
        } else {
            u16 hi, lo;
            split_f16(in ? ldexpf(load_f32<T>(h, i * stride + f), s) : 0.0f, hi, lo);
            row[f] = hi;
            row[k.n_pad * k.ld + f] = lo;
        }
    }
}

// f32: h as dW's product takes it, times the row's weight and with one scale for all
// rows (they are summed over).
__global__ __launch_bounds__(256) void k_xent_pack_hg(XentPack k, const float *h, int64_t stride) {
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= k.n_pad) return;
    const bool live = k.label[i] >= 0;
    const float wt = k.weight[i];
    const int s = scale_exp(k.ctl->hg_max);
    u16 *row = k.hg + i * k.ld;
    for (int32_t f = lane; f < k.ld; f += 64) {
        u16 hi, lo;
        split_f16(live && f < k.d ? ldexpf(wt * h[i * stride + f], s) : 0.0f, hi, lo);
        row[f] = hi;
        row[k.n_pad * k.ld + f] = lo;
    }
}

// ---- products --------------------------------------------------------------------
// C[m][n] = sum_k A[m][k] B[n][k], a tile of 128 x 128 by 4 wavefronts of 64 x 64.
// An operand lies with k contiguous (KC: element (m, k) at m * ld + k) or with m
// contiguous (k * ld + m); the second kind is turned by the LDS reads
// (ds_read_tr16_b64: 16 lanes read 4 rows of 16 elements, lane i gets column i).
// P == 1: bf16; P == 2: f16 in two planes, three products.
template <int P> constexpr int BK = 64 / P;          // k of a step
template <int P> constexpr int OP_BYTES = P * TILE * BK<P> * 2;
template <int P> constexpr int LDS_TILES = 4 * OP_BYTES<P>;      // A and B, twice

struct Operand {
    const u16 *p;
    int64_t plane, ld;
};

// Bytes of 16-byte chunk c of row r in LDS.  A read of the matrix instruction's
// operand takes one chunk of 8 rows at a time (KC) or 32 bytes of 4 rows: the chunks
// are permuted so that these fall on different banks.
template <int P, bool KC> __device__ __forceinline__ int lds_at(int r, int c) {
    if constexpr (KC) {
        constexpr int CH = BK<P> / 8;
        const int x = CH == 8 ? r & 7 : (r >> 1) & 3;
        return (r * CH + (c ^ x)) * 16;
    } else {
        return (r * 16 + ((((c >> 1) ^ (r & 7)) << 1) | (c & 1))) * 16;
    }
}

template <int P, bool KC> struct Stage {
    static constexpr int NQ = BK<P> / 16;            // chunks a thread and plane
    u32x4 r[P][NQ];
    __device__ __forceinline__ void load(const Operand &o, int64_t m0, int64_t k0) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const int idx = threadIdx.x + 256 * q;
                int64_t at;
                if constexpr (KC) {
                    constexpr int CH = BK<P> / 8;
                    at = (m0 + idx / CH) * o.ld + k0 + idx % CH * 8;
                } else {
                    at = (k0 + idx / 16) * o.ld + m0 + idx % 16 * 8;
                }
                r[p][q] = *reinterpret_cast<const u32x4 *>(o.p + p * o.plane + at);
            }
    }
    __device__ __forceinline__ void store(char *lds) const {
        constexpr int CH = KC ? BK<P> / 8 : 16;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const int idx = threadIdx.x + 256 * q;
                *reinterpret_cast<u32x4 *>(lds + p * (TILE * BK<P> * 2) +
                                           lds_at<P, KC>(idx / CH, idx % CH)) = r[p][q];
            }
    }
};

// The operand of the matrix instruction: lane l has element m0 + l % 32, k =
// k0 + l / 32 * 8 .. + 7.
template <int P, bool KC>
__device__ __forceinline__ void fragment(const char *lds, int m0, int k0, u32x4 (&f)[P]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const char *plane = lds + p * (TILE * BK<P> * 2);
        if constexpr (KC) {
            f[p] = *reinterpret_cast<const u32x4 *>(
                plane + lds_at<P, true>(m0 + (lane & 31), k0 / 8 + (lane >> 5)));
        } else {
            typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
            const int g = lane >> 4, i = lane & 15;
            const int m = m0 + (g & 1) * 16 + (i & 3) * 4, k = k0 + (g >> 1) * 8 + (i >> 2);
            union {
                i16x4 h[2];
                u32x4 v;
            } u;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                u.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_i16x4 *)(plane + lds_at<P, false>(k + 4 * t, m / 8) + (m & 7) * 2));
            f[p] = u.v;
        }
    }
}

// Adds the product of steps [0, steps) into acc[mt][nt]: wavefront w has rows
// (w >> 1) * 64 + mt * 32 and columns (w & 1) * 64 + nt * 32 of the tile.
template <int P, bool AK, bool BKC>
__device__ __forceinline__ void tile_product(const Operand &a, const Operand &b, int64_t m0,
                                             int64_t n0, int64_t steps, char *lds,
                                             f32x16 (&acc)[2][2]) {
    const int wave = threadIdx.x >> 6;
    Stage<P, AK> sa;
    Stage<P, BKC> sb;
    sa.load(a, m0, 0);
    sb.load(b, n0, 0);
    __syncthreads();                     // the last tile's reads
    sa.store(lds);
    sb.store(lds + OP_BYTES<P>);
    __syncthreads();
    for (int64_t t = 0; t < steps; ++t) {
        const char *cur = lds + (t & 1) * 2 * OP_BYTES<P>;
        char *nxt = lds + ((t + 1) & 1) * 2 * OP_BYTES<P>;
        if (t + 1 < steps) {
            sa.load(a, m0, (t + 1) * BK<P>);
            sb.load(b, n0, (t + 1) * BK<P>);
        }
#pragma unroll
        for (int k = 0; k < BK<P>; k += 16) {
            u32x4 fa[2][P], fb[2][P];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                fragment<P, AK>(cur, (wave >> 1) * 64 + x * 32, k, fa[x]);
                fragment<P, BKC>(cur + OP_BYTES<P>, (wave & 1) * 64 + x * 32, k, fb[x]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) acc[x][y] = mma<P>(fa[x], fb[y], acc[x][y]);
        }
        if (t + 1 < steps) {
            sa.store(nxt);
            sb.store(nxt + OP_BYTES<P>);
        }
        __syncthreads();
    }
}

__device__ __forceinline__ void clear(f32x16 (&acc)[2][2]) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
}

// Row of register r in a 32 x 32 block; its column is lane % 32.
__device__ __forceinline__ int block_row(int r) {
    return (r >> 2) * 8 + ((threadIdx.x & 63) >> 5) * 4 + (r & 3);
}

// ---- pass 1: each row's maximum and sum ---------------------------------------------
// The product is W h' (classes down, rows across), so that a lane has scores of one
// row: the maximum and sum stay in registers over the classes of a split, and only
// two lanes and two wavefronts have parts of a row.  part[2 * split + half][row]: the
// maximum of z log2 e, and the sum of its powers of 2.
template <int P>
__global__ __launch_bounds__(256, 2) void k_xent_stats(XentPack k, int64_t class_tiles,
                                                       int32_t splits,
                                                       float2 *__restrict__ part) {
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i0 = (int64_t)(blockIdx.x / splits) * TILE;
    const int32_t split = blockIdx.x % splits;
    const Operand a{k.w, k.v_pad * k.ld, k.ld}, b{k.h, k.n_pad * k.ld, k.ld};
    const int64_t steps = (k.d + BK<P> - 1) / BK<P>;
    float m[2], s[2], sc[2];
    int64_t row[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        row[y] = i0 + (wave & 1) * 64 + y * 32 + (lane & 31);
        m[y] = -INFINITY;
        s[y] = 0.0f;
        sc[y] = P == 2 ? k.row_scale[row[y]] : LOG2E;
    }
    for (int64_t t = split; t < class_tiles; t += splits) {
        f32x16 acc[2][2];
        clear(acc);
        tile_product<P, true, true>(a, b, t * TILE, i0, steps, lds, acc);
        const float *bias = k.bias + t * TILE + (wave >> 1) * 64 + (lane >> 5) * 4;
        float4 b2[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                b2[x][q] = *reinterpret_cast<const float4 *>(bias + x * 32 + q * 8);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            float top = m[y];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float4 q = b2[x][r >> 2];
                    const float b = (r & 3) == 0 ? q.x : (r & 3) == 1 ? q.y : (r & 3) == 2 ? q.z : q.w;
                    acc[x][y][r] = __builtin_fmaf(acc[x][y][r], sc[y], b);
                    top = fmaxf(top, acc[x][y][r]);
                }
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum[2] = {s[y] * __builtin_amdgcn_exp2f(m[y] - ref), 0.0f};
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sum[r & 1] += __builtin_amdgcn_exp2f(acc[x][y][r] - ref);
            m[y] = top;
            s[y] = sum[0] + sum[1];
        }
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        const float m2 = __shfl_xor(m[y], 32, 64), s2 = __shfl_xor(s[y], 32, 64);
        const float top = fmaxf(m[y], m2), ref = top == -INFINITY ? 0.0f : top;
        const float sum = s[y] * __builtin_amdgcn_exp2f(m[y] - ref) +
                          s2 * __builtin_amdgcn_exp2f(m2 - ref);
        if (lane < 32)
            part[(2 * split + (wave >> 1)) * k.n_pad + row[y]] = make_float2(top, sum);
    }
}

// The parts of a row joined, one wavefront a row: lse and loss.  The label's score is
// summed in f32 from h and W themselves.
template <typename T>
__global__ __launch_bounds__(256) void k_xent_join(XentPack k, XentCall c, int32_t parts,
                                                   const float2 *__restrict__ part,
                                                   float *__restrict__ lse2) {
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= k.n_pad) return;
    float top = -INFINITY, sum = 0.0f;
    for (int p = lane; p < parts; p += 64) {
        const float2 q = part[p * k.n_pad + i];
        const float now = fmaxf(top, q.x), ref = now == -INFINITY ? 0.0f : now;
        sum = sum * __builtin_amdgcn_exp2f(top - ref) + q.y * __builtin_amdgcn_exp2f(q.x - ref);
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
        sum = sum * __builtin_amdgcn_exp2f(top - ref) + s2 * __builtin_amdgcn_exp2f(t2 - ref);
        top = now;
        dot += __shfl_xor(dot, o, 64);
    }
    const float l2 = (top == -INFINITY ? 0.0f : top) + log2f(sum);
    if (lane != 0) return;
    lse2[i] = l2;
    if (i >= k.n) return;
    const float lse = y == -2 ? NAN : l2 * LN2, z = open ? dot + (c.bias ? c.bias[y] : 0.0f) : -INFINITY;
    c.lse[i] = lse;
    c.loss[i] = y < 0 ? 0.0f : k.weight[i] * (lse - z);
}

// ---- pass 2: G of a piece ------------------------------------------------------------
// g[v - v0][i - r0], rows of rows_pad; f32: G / w in two f16 terms times 2^15.
template <int P>
__global__ __launch_bounds__(256, 2) void k_xent_g(XentPack k, int64_t v0, int64_t r0, int64_t rows_pad,
                                                int64_t plane, int32_t row_tiles,
                                                const float *__restrict__ lse2,
                                                u16 *__restrict__ g) {
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i0 = r0 + (int64_t)(blockIdx.x % row_tiles) * TILE;
    const int64_t c0 = v0 + (int64_t)(blockIdx.x / row_tiles) * TILE;
    const Operand a{k.w, k.v_pad * k.ld, k.ld}, b{k.h, k.n_pad * k.ld, k.ld};
    f32x16 acc[2][2];
    clear(acc);
    tile_product<P, true, true>(a, b, c0, i0, (k.d + BK<P> - 1) / BK<P>, lds, acc);
    const int64_t c = c0 + (wave >> 1) * 64 + (lane >> 5) * 4;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        const int64_t i = i0 + (wave & 1) * 64 + y * 32 + (lane & 31);
        const float sc = P == 2 ? k.row_scale[i] : LOG2E;
        const int32_t label = k.label[i];
        // a row that is out: 2^-inf
        const float l = label < 0 ? INFINITY : lse2[i], wt = k.weight[i];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int64_t here = c + x * 32;
            const int64_t mine = label - here;           // 8 q + e if the label is here
            const bool hot = __any(mine >= 0 && mine < 32);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 b4 = *reinterpret_cast<const float4 *>(k.bias + here + q * 8);
                const float b2[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float p = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(acc[x][y][q * 4 + e], sc, b2[e] - l));
                    if (hot && mine == q * 8 + e) p -= 1.0f;
                    u16 *at = g + (here + q * 8 + e - v0) * rows_pad + (i - r0);
                    if constexpr (P == 1) {
                        *at = bits_of((__bf16)(wt * p));
                    } else {
                        u16 hi, lo;
                        split_f16(p * G_SCALE, hi, lo);
                        at[0] = hi;
                        at[plane] = lo;
                    }
                }
            }
        }
    }
}

// Where a product's tile goes: the f32 sums of the pieces so far, and, with the last
// piece, the output.
struct Out {
    float *acc;                  // [m][ld]
    bool first, last;
    const float *bias;           // dW: rows of bias -inf are 0
    void *out;
    int64_t rows, stride;        // of the output; its columns are d
};

template <int P>
__device__ __forceinline__ void put(const Out &o, int32_t d, int32_t ld, int64_t m, int64_t n,
                                    float v, float scale) {
    float *acc = o.acc + m * ld + n;
    if (!o.first) v += *acc;
    if (!o.last) {
        *acc = v;
    } else if (m < o.rows && n < d) {
        if (o.bias && o.bias[m] == -INFINITY) v = 0.0f;
        if constexpr (P == 1) static_cast<__bf16 *>(o.out)[m * o.stride + n] = (__bf16)v;
        else static_cast<float *>(o.out)[m * o.stride + n] = v * scale;
    }
}

// dh[i][j] += sum over the piece's v of g[v][i] W[v][j].
template <int P>
__global__ __launch_bounds__(256, 2) void k_xent_dh(XentPack k, int64_t v0, int64_t classes_pad,
                                                 int64_t r0, int64_t rows_pad, int64_t plane,
                                                 int32_t row_tiles, const u16 *__restrict__ g,
                                                 Out o) {
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m0 = (int64_t)(blockIdx.x % row_tiles) * TILE;
    const int64_t n0 = (int64_t)(blockIdx.x / row_tiles) * TILE;
    const Operand a{g, plane, rows_pad}, b{k.w + v0 * k.ld, k.v_pad * k.ld, k.ld};
    const float ws = P == 2 ? ldexpf(1.0f, -scale_exp(k.ctl->w_max)) / G_SCALE : 1.0f;
    f32x16 acc[2][2];
    clear(acc);
    tile_product<P, false, false>(a, b, m0, n0, classes_pad / BK<P>, lds, acc);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int64_t i = r0 + m0 + (wave >> 1) * 64 + x * 32 + block_row(r);
            const float scale = P == 2 ? ws * k.weight[i] : 1.0f;
#pragma unroll
            for (int y = 0; y < 2; ++y)
                put<P>(o, k.d, k.ld, i, n0 + (wave & 1) * 64 + y * 32 + (lane & 31), acc[x][y][r],
                       scale);
        }
}

// dW[v][j] += sum over the rows of g[v][i] hg[i][j].
template <int P>
__global__ __launch_bounds__(256, 2) void k_xent_dw(XentPack k, int64_t v0, int64_t r0, int64_t rows_pad,
                                                 int64_t plane, int32_t class_tiles,
                                                 const u16 *__restrict__ g, Out o) {
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m0 = (int64_t)(blockIdx.x % class_tiles) * TILE;
    const int64_t n0 = (int64_t)(blockIdx.x / class_tiles) * TILE;
    const Operand a{g, plane, rows_pad}, b{k.hg + r0 * k.ld, k.n_pad * k.ld, k.ld};
    const float scale = P == 2 ? ldexpf(1.0f, -scale_exp(k.ctl->hg_max)) / G_SCALE : 1.0f;
    f32x16 acc[2][2];
    clear(acc);
    tile_product<P, true, false>(a, b, m0, n0, rows_pad / BK<P>, lds, acc);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int y = 0; y < 2; ++y)
                put<P>(o, k.d, k.ld, v0 + m0 + (wave >> 1) * 64 + x * 32 + block_row(r),
                       n0 + (wave & 1) * 64 + y * 32 + (lane & 31), acc[x][y][r], scale);
}

// db[v] += sum over the rows of G, one wavefront a class.
template <int P>
__global__ __launch_bounds__(256) void k_xent_db(XentPack k, int64_t v0, int64_t classes, int64_t r0,
                                                 int64_t rows_pad, int64_t plane,
                                                 const u16 *__restrict__ g, bool first,
                                                 float *__restrict__ db) {
    const int lane = threadIdx.x & 63;
    const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (c >= classes) return;
    float sum = 0.0f;
    for (int64_t i = lane; i < rows_pad; i += 64) {
        const u16 *at = g + c * rows_pad + i;
        if constexpr (P == 1) {
            sum += (float)__builtin_bit_cast(__bf16, *at);
        } else {
            const float p = (float)__builtin_bit_cast(_Float16, at[0]) +
                            (float)__builtin_bit_cast(_Float16, at[plane]);
            if (k.label[r0 + i] >= 0) sum += p * k.weight[r0 + i];
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) {
        if (P == 2) sum *= 1.0f / G_SCALE;
        if (k.bias[v0 + c] == -INFINITY) sum = 0.0f;
        db[v0 + c] = first ? sum : db[v0 + c] + sum;
    }
}

// Zeros where there is no row to sum over.
template <typename T>
__global__ __launch_bounds__(256) void k_xent_zero(T *out, int64_t rows, int32_t cols,
                                                   int64_t stride) {
    const int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (v >= rows) return;
    for (int32_t f = threadIdx.x & 63; f < cols; f += 64) out[v * stride + f] = (T)0.0f;
}

// ---- the call -------------------------------------------------------------------------
int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
uint32_t blocks(int64_t x, int64_t per) { return (uint32_t)((x + per - 1) / per); }

// G of a piece: 32k rows and 256 MB at most (what the memory-side cache holds).
constexpr int64_t PIECE_ROWS = 32768;
constexpr int64_t PIECE_BYTES = (int64_t)256 << 20;

struct Plan {
    int P;
    int64_t n_pad, v_pad, ld, piece_rows, piece_classes;
    int32_t splits;
    size_t ctl, h, hg, w, bias, scale, label, weight, lse, part, g, dh_acc, dw_acc, end;
};

Plan plan_of(const XentCall &c) {
    Plan p{};
    p.P = c.bf16 ? 1 : 2;
    p.n_pad = up(c.rows, TILE);
    p.v_pad = up(c.classes, TILE);
    p.ld = up(c.dim, LD_PAD);
    const int64_t row_tiles = p.n_pad / TILE, class_tiles = p.v_pad / TILE;
    // three workgroups a CU, if there are as many tiles
    p.splits = (int32_t)std::max<int64_t>(
        1, std::min<int64_t>(class_tiles, (3 * (int64_t)c.num_cus + row_tiles - 1) / row_tiles));
    p.piece_rows = std::min(p.n_pad, PIECE_ROWS);
    p.piece_classes = std::min(
        p.v_pad, std::max<int64_t>(TILE, PIECE_BYTES / (2 * p.P * p.piece_rows) / TILE * TILE));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.ctl = take(sizeof(XentCtl));
    p.h = take((size_t)2 * p.P * p.n_pad * p.ld);
    p.w = take((size_t)2 * p.P * p.v_pad * p.ld);
    p.bias = take((size_t)4 * p.v_pad);
    p.scale = take((size_t)4 * p.n_pad);
    p.label = take((size_t)4 * p.n_pad);
    p.weight = take((size_t)4 * p.n_pad);
    p.lse = take((size_t)4 * p.n_pad);
    p.part = take((size_t)16 * p.splits * p.n_pad);
    if (c.grad) {
        p.hg = c.bf16 ? p.h : take((size_t)2 * p.P * p.n_pad * p.ld);
        p.g = take((size_t)2 * p.P * p.piece_rows * p.piece_classes);
        if (p.piece_classes < p.v_pad) p.dh_acc = take((size_t)4 * p.n_pad * p.ld);
        if (p.piece_rows < p.n_pad) p.dw_acc = take((size_t)4 * p.v_pad * p.ld);
    }
    p.end = at;
    return p;
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
    k.h = reinterpret_cast<u16 *>(m + p.h);
    k.hg = reinterpret_cast<u16 *>(m + p.hg);
    k.w = reinterpret_cast<u16 *>(m + p.w);
    k.bias = reinterpret_cast<float *>(m + p.bias);
    k.row_scale = reinterpret_cast<float *>(m + p.scale);
    k.label = reinterpret_cast<int32_t *>(m + p.label);
    k.weight = reinterpret_cast<float *>(m + p.weight);
    float *lse = reinterpret_cast<float *>(m + p.lse);
    float2 *part = reinterpret_cast<float2 *>(m + p.part);
    const dim3 b(256);
    constexpr int LDS = LDS_TILES<P>;
    const void *big[] = {reinterpret_cast<const void *>(k_xent_stats<P>),
                         reinterpret_cast<const void *>(k_xent_g<P>),
                         reinterpret_cast<const void *>(k_xent_dh<P>),
                         reinterpret_cast<const void *>(k_xent_dw<P>)};
    for (const void *f : big) {
        const hipError_t e = allow_all_lds(f);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(k_xent_init, dim3(1), dim3(1), 0, s, k.ctl);
    hipLaunchKernelGGL((k_xent_classes<T>), dim3(blocks(k.v_pad, 4)), b, 0, s, k, c.w, c.w_stride,
                       c.bias);
    hipLaunchKernelGGL((k_xent_pack_w<T>), dim3(blocks(k.v_pad, 4)), b, 0, s, k, c.w, c.w_stride);
    hipLaunchKernelGGL((k_xent_rows<T>), dim3(blocks(k.n_pad, 4)), b, 0, s, k, c.h, c.h_stride,
                       c.labels, c.weights);
    hipLaunchKernelGGL((k_xent_stats<P>), dim3((uint32_t)(k.n_pad / TILE * p.splits)), b, LDS, s, k,
                       k.v_pad / TILE, p.splits, part);
    hipLaunchKernelGGL((k_xent_join<T>), dim3(blocks(k.n_pad, 4)), b, 0, s, k, c, 2 * p.splits,
                       part, lse);
    if (!c.grad) return hipGetLastError();
    if constexpr (P == 2)
        hipLaunchKernelGGL(k_xent_pack_hg, dim3(blocks(k.n_pad, 4)), b, 0, s, k,
                           static_cast<const float *>(c.h), c.h_stride);
    u16 *g = reinterpret_cast<u16 *>(m + p.g);
    const int64_t plane = p.piece_rows * p.piece_classes;
    const uint32_t cols = (uint32_t)(p.ld / TILE);
    for (int64_t v0 = 0; v0 < k.v_pad; v0 += p.piece_classes)
        for (int64_t r0 = 0; r0 < k.n_pad; r0 += p.piece_rows) {
            const int64_t nv = std::min(p.piece_classes, k.v_pad - v0);
            const int64_t nr = std::min(p.piece_rows, k.n_pad - r0);
            const int32_t vt = (int32_t)(nv / TILE), rt = (int32_t)(nr / TILE);
            hipLaunchKernelGGL((k_xent_g<P>), dim3((uint32_t)(vt * rt)), b, LDS, s, k, v0, r0, nr,
                               plane, rt, lse, g);
            if (c.dh) {
                const Out o{reinterpret_cast<float *>(m + p.dh_acc), v0 == 0, v0 + nv == k.v_pad,
                            nullptr, c.dh, k.n, c.h_stride};
                hipLaunchKernelGGL((k_xent_dh<P>), dim3((uint32_t)rt * cols), b, LDS, s, k, v0, nv,
                                   r0, nr, plane, rt, g, o);
            }
            if (c.dw) {
                const Out o{reinterpret_cast<float *>(m + p.dw_acc), r0 == 0, r0 + nr == k.n_pad,
                            k.bias, c.dw, k.v, c.w_stride};
                hipLaunchKernelGGL((k_xent_dw<P>), dim3((uint32_t)vt * cols), b, LDS, s, k, v0, r0,
                                   nr, plane, vt, g, o);
            }
            if (c.dbias) {
                const int64_t live = std::min(nv, k.v - v0);
                hipLaunchKernelGGL((k_xent_db<P>), dim3(blocks(live, 4)), b, 0, s, k, v0, live, r0,
                                   nr, plane, g, r0 == 0, c.dbias);
            }
        }
    return hipGetLastError();
}

}  // namespace

size_t xent_scratch(const XentCall &c) {
    if (!c.rows) return 0;
    return c.dim <= XENT_FUSED_DIM ? xent_fused_scratch(c) : plan_of(c).end;
}

hipError_t launch_xent(hipStream_t s, const XentCall &c, char *scratch) {
    if (c.rows && c.dim <= XENT_FUSED_DIM) return launch_xent_fused(s, c, scratch);
    if (c.rows) {
        const Plan p = plan_of(c);
        return c.bf16 ? run<1, __bf16>(s, c, p, scratch) : run<2, float>(s, c, p, scratch);
    }
    // no row: no loss, and gradients that are empty sums
    if (c.grad && c.dw) {
        const dim3 g(blocks(c.classes, 4)), b(256);
        if (c.bf16)
            hipLaunchKernelGGL((k_xent_zero<__bf16>), g, b, 0, s, static_cast<__bf16 *>(c.dw),
                               c.classes, c.dim, c.w_stride);
        else
            hipLaunchKernelGGL((k_xent_zero<float>), g, b, 0, s, static_cast<float *>(c.dw),
                               c.classes, c.dim, c.w_stride);
    }
    if (c.grad && c.dbias)
        hipLaunchKernelGGL((k_xent_zero<float>), dim3(blocks(c.classes, 4)), dim3(256), 0, s,
                           c.dbias, c.classes, 1, (int64_t)1);
    return hipGetLastError();
}

}  // namespace mbk
