// ops.h — kernel launchers of the seam's many-class loss (kernels_xent.hip), of
// rows sorted by expert (kernels_expert.hip), of category vectors (kernels_embed.hip), of the
// norm of gradients (kernels_clip.hip) and of scores from class vectors in 4 bits and their
// penalties (kernels_fourbit.hip, kernels_adjust.hip); ops.cpp checks the arguments.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mbk {

// ---- cross entropy over many classes ----------------------------------------

struct XentCall {
    int64_t rows, classes;
    int32_t dim;
    bool bf16;                       // h, w, dh, dw: bf16, else f32
    int64_t h_stride, w_stride;
    const void *h, *w;
    const float *bias;               // NULL: none
    const int32_t *labels;
    const float *weights;            // NULL: 1
    float *loss, *lse;
    bool grad;
    void *dh, *dw;                   // NULL: not asked for
    float *dbias;
    int num_cus;
};
// Bytes of scratch that the call takes.
size_t xent_scratch(const XentCall &c);
hipError_t launch_xent(hipStream_t s, const XentCall &c, char *scratch);

// ---- rows sorted by expert ---------------------------------------------------

struct ExpertPlan {
    int64_t rows;
    int32_t k, experts;
    const int32_t *expert;           // [rows][k]
    int32_t *offsets, *source, *slot;
};
// The rows' matrix: element (i, f) at data[i * row_stride + f * col_stride].
struct ExpertMatrix {
    void *data;
    int64_t row_stride, col_stride;
    int32_t cols;
    bool bf16;                       // else f32
    bool blocked;                    // layout of the sorted matrix
};
size_t expert_scratch(const ExpertPlan &p, int num_cus);
hipError_t launch_expert_sort(hipStream_t s, const ExpertPlan &p, int num_cus, char *scratch);
hipError_t launch_expert_gather(hipStream_t s, const ExpertPlan &p, const ExpertMatrix &x,
                                void *sorted);
hipError_t launch_expert_combine(hipStream_t s, const ExpertPlan &p, const void *sorted,
                                 const float *weights, const ExpertMatrix &out);
hipError_t launch_expert_combine_grad(hipStream_t s, const ExpertPlan &p,
                                      const ExpertMatrix &dout, const void *sorted,
                                      const float *weights, void *d_sorted, float *d_weights);

// Outputs of more bytes than all XCDs' L2 hold are stored past it: they would drive out what is
// read, and what takes them next finds little of them there (65536 x 1024 bf16 rows looked up and
// added: 70 us by ordinary stores, 57 so).
constexpr int64_t STREAMED = (int64_t)32 << 20;
#ifdef __HIP_DEVICE_COMPILE__
// Stores a vector at any address that holds one of its elements.  (A template's argument leaves a
// type's alignment behind, so that it is given here.)  The empty statements keep the compiler from
// making one ordinary store of both.
template <typename V> __device__ __forceinline__ void put(void *to, const V &v, bool streamed) {
    typedef V Loose __attribute__((aligned(sizeof(v[0]))));
    Loose *at = static_cast<Loose *>(to);
    if (streamed) {
        __builtin_nontemporal_store(v, at);
    } else {
        asm volatile("" ::: "memory");
        *at = v;
        asm volatile("" ::: "memory");
    }
}
#else
template <typename V> __device__ void put(void *, const V &, bool) {}
#endif

// ---- category vectors ---------------------------------------------------------

struct EmbedCall {
    int64_t rows, entries;
    int32_t dim;
    bool bf16;                       // table, base, out, dout, dtable: bf16, else f32
    int64_t row_stride, table_stride;
    float scale;
    const int32_t *ids;
    const void *table, *base;        // base NULL: 0
    void *out;
    const void *dout;                // of the gradient
    void *dtable;
    int num_cus;
    bool streamed;                   // set by the launchers
};
hipError_t launch_embed(hipStream_t s, const EmbedCall &c);
size_t embed_grad_scratch(const EmbedCall &c);
hipError_t launch_embed_grad(hipStream_t s, const EmbedCall &c, char *scratch);

// ---- the norm of many gradients -------------------------------------------------

// A part of a gradient: rows of cols elements; one row, or short ones.
struct ClipPiece {
    const void *grad;
    void *out;                       // NULL: none
    int64_t stride;
    int32_t rows, cols;
    bool bf16;
};
// Elements of a piece: short ones where all gradients together leave CUs without one (75,000
// elements: two kernels of 12.2 us together in pieces of 8192, 7.9 in pieces of 1024).
constexpr int64_t clip_piece(int64_t elements) {
    return elements < ((int64_t)1 << 18) ? 1024 : elements < ((int64_t)1 << 21) ? 2048 : 8192;
}
constexpr int CLIP_ONE = 32;             // pieces of at most 256 runs of 16 bytes that one workgroup takes
constexpr int CLIP_RUNS = 256;
struct ClipCall {
    const ClipPiece *piece;
    int64_t pieces;
    bool one;                        // at most CLIP_ONE such pieces
    bool outputs, streamed;
    float max_norm;
    float *norm;
    int num_cus;
};
size_t clip_scratch(int64_t pieces, int num_cus);
hipError_t launch_clip(hipStream_t s, const ClipCall &c, char *scratch);

// ---- scores from class vectors in 4 bits, and their penalties -----------------------

struct FourbitShape {
    int64_t classes;
    int32_t dim, group;
    int32_t blocks;                  // of 128 elements
};
FourbitShape fourbit_shape(int64_t classes, int32_t dim, int32_t group);
size_t fourbit_bytes(const FourbitShape &s);
void fourbit_parts(const FourbitShape &s, char *packed, uint32_t **codes, _Float16 **scales,
              int32_t **exponents);
hipError_t launch_fourbit_pack(hipStream_t st, const FourbitShape &s, bool bf16, const void *w,
                          int64_t stride, char *packed);
struct FourbitCall {
    FourbitShape shape;
    int64_t rows;
    bool bf16;                       // h: bf16, else f32
    const void *h;
    int64_t h_stride;
    const uint32_t *codes;
    const _Float16 *scales;
    const int32_t *exponents;
    const float *bias;               // NULL: none
    float *scores;
    int64_t score_stride;
    bool wide_h;                     // rows at multiples of 16 bytes; set by the launcher,
    bool streamed;                   // as this is
    int num_cus;
};
size_t fourbit_scratch(const FourbitCall &c);
hipError_t launch_fourbit_scores(hipStream_t st, const FourbitCall &c, char *scratch);

struct AdjustCall {
    int64_t rows, classes, score_stride, out_stride;
    int32_t history;                 // ids a row, at most
    int64_t history_stride, mask_stride;
    float repetition, presence, frequency;
    bool penalties;                  // there are a history and a penalty
    const float *scores;
    const int32_t *ids, *lengths;    // lengths NULL: history
    const float *bias;               // NULL: none
    const uint32_t *allowed;         // NULL: all
    float *out;
    bool streamed;                   // set by the launcher
};
hipError_t launch_adjust(hipStream_t s, const AdjustCall &c);

}  // namespace mbk
