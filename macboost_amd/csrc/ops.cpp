// ops.cpp — the seam's operators beside the tree build: the loss over many classes
// (mbk_xent, mbk_xent_grad), rows sorted by expert (mbk_expert_*), category vectors
// (mbk_embed*), the norm of gradients (mbk_tensors_*, mbk_grad_clip), scores from class vectors
// in 4 bits (mbk_fourbit_*) and their penalties (mbk_adjust).  Each call
// checks its arguments (the context last), queues its kernels on the context's stream and
// returns; it allocates only when it needs more scratch than the context holds.  Calls that
// use scratch are queued whole, one after another, whichever threads make them.
#include <algorithm>
#include <cmath>
#include <functional>
#include <initializer_list>
#include <vector>

#include "../../include/macboost.h"
#include "abi.hpp"
#include "core.hpp"
#include "ops.h"

namespace {

void need(bool ok, const char *what) {
    if (!ok) mb::invalid(what);
}

constexpr int64_t MOST_ROWS = 0x7FFFFF00;
constexpr int32_t MOST_EXPERTS = 8192;       // counters of four wavefronts in LDS
constexpr int64_t MOST_STRIDE = (int64_t)1 << 40;
constexpr int64_t MOST_ELEMENTS = (int64_t)1 << 38;

bool is_bf16(int32_t type) {
    need(type == MBK_F32 || type == MBK_BF16, "type must be MBK_F32 or MBK_BF16");
    return type == MBK_BF16;
}

// Every one a multiple of `size` bytes (NULL is).
void need_multiple(size_t size, std::initializer_list<const void *> arrays) {
    for (const void *p : arrays)
        need(reinterpret_cast<uintptr_t>(p) % size == 0,
             "arrays must be at multiples of their elements' size");
}
size_t size_of(bool bf16) { return bf16 ? 2 : 4; }

mbk::XentCall xent_call(const mbk_xent_shape *sh, const void *h,
                        const void *w, const float *bias, const int32_t *labels,
                        const float *weights, float *loss, float *lse) {
    need(sh != nullptr, "null shape");
    need(sh->rows >= 0 && sh->rows <= MOST_ROWS, "rows must be in 0..2^31-256");
    need(sh->classes >= 1 && sh->classes <= MOST_ROWS, "classes must be in 1..2^31-256");
    need(sh->dim >= 1 && sh->dim <= (1 << 20), "dim must be in 1..2^20");
    need(sh->h_stride >= sh->dim && sh->w_stride >= sh->dim,
         "h_stride and w_stride must be at least dim");
    need(sh->h_stride <= MOST_STRIDE && sh->w_stride <= MOST_STRIDE,
         "h_stride and w_stride must be at most 2^40");
    need(w && (!sh->rows || (h && labels && loss && lse)), "null argument");
    mbk::XentCall c{};
    c.rows = sh->rows;
    c.classes = sh->classes;
    c.dim = sh->dim;
    c.bf16 = is_bf16(sh->type);
    c.h_stride = sh->h_stride;
    c.w_stride = sh->w_stride;
    c.h = h;
    c.w = w;
    c.bias = bias;
    c.labels = labels;
    c.weights = weights;
    c.loss = loss;
    c.lse = lse;
    return c;
}

void run_xent(mbk_context *ctx, mbk::XentCall c) {
    need(ctx != nullptr, "null kernel-seam context");
    c.num_cus = mb::context_cus(ctx);
    mb::OnDevice here(mb::context_device(ctx));
    std::lock_guard<std::mutex> lock(mb::context_scratch_mutex(ctx));
    char *scratch = mb::context_scratch(ctx, mbk::xent_scratch(c));
    MB_HIP(mbk::launch_xent(mb::context_stream(ctx), c, scratch));
}

mbk::ExpertPlan expert_plan(const mbk_expert_plan *p) {
    need(p != nullptr, "null plan");
    need(p->rows >= 0 && p->k >= 1 && p->rows <= MOST_ROWS / p->k,
         "rows must be >= 0, k >= 1 and rows * k at most 2^31-256");
    need(p->experts >= 1 && p->experts <= MOST_EXPERTS, "experts must be in 1..8192");
    need(p->offsets && (!p->rows || (p->expert && p->source && p->slot)), "null plan array");
    return {p->rows, p->k, p->experts, p->expert, p->offsets, p->source, p->slot};
}

mbk::ExpertMatrix expert_matrix(const mbk_expert_matrix *m, int64_t rows) {
    need(m != nullptr, "null matrix");
    need(m->cols >= 1, "cols must be positive");
    need(m->cols <= (1 << 30), "cols must be at most 2^30");
    need(m->data || !rows, "null matrix data");
    // no element twice: rows apart by a row's columns, or columns by a column's rows
    const int64_t rs = m->row_stride, cs = m->col_stride;
    need(rs >= 1 && cs >= 1 && rs <= MOST_STRIDE && cs <= MOST_STRIDE &&
             ((m->cols - 1) <= (rs - 1) / cs || rows - 1 <= (cs - 1) / rs),
         "row_stride and col_stride must be in 1..2^40 and keep the elements apart");
    return {m->data, m->row_stride, m->col_stride, m->cols, is_bf16(m->type), m->blocked != 0};
}

mbk::EmbedCall embed_call(const mbk_embed_shape *sh, const int32_t *ids, const void *base) {
    need(sh != nullptr, "null shape");
    need(sh->rows >= 0 && sh->rows <= MOST_ROWS, "rows must be in 0..2^31-256");
    need(sh->entries >= 1 && sh->entries <= MOST_ROWS, "entries must be in 1..2^31-256");
    need(sh->dim >= 1 && sh->dim <= (1 << 20), "dim must be in 1..2^20");
    need(sh->row_stride >= sh->dim && sh->table_stride >= sh->dim &&
             sh->row_stride <= MOST_STRIDE && sh->table_stride <= MOST_STRIDE,
         "row_stride and table_stride must be in dim..2^40");
    need(std::isfinite(sh->scale), "scale must be finite");
    mbk::EmbedCall c{};
    c.rows = sh->rows;
    c.entries = sh->entries;
    c.dim = sh->dim;
    c.bf16 = is_bf16(sh->type);
    c.row_stride = sh->row_stride;
    c.table_stride = sh->table_stride;
    c.scale = sh->scale;
    c.ids = ids;
    c.base = base;
    return c;
}

// The pieces of one gradient of the list: short rows together, long ones and gradients without
// gaps in runs of `most` elements.  runs: 16-byte runs of short rows a piece, at most.
void add_pieces(const mbk_tensor &t, int64_t most, int64_t runs, std::vector<mbk::ClipPiece> &out) {
    const bool bf16 = t.type == MBK_BF16;
    const int64_t size = bf16 ? 2 : 4;
    const auto add = [&](int64_t at, int64_t rows, int64_t cols) {
        const char *g = static_cast<const char *>(t.grad) + at * size;
        char *o = t.out ? static_cast<char *>(t.out) + at * size : nullptr;
        out.push_back({g, o, t.stride, (int32_t)rows, (int32_t)cols, bf16});
    };
    if (!t.rows || !t.cols) return;
    const bool whole = t.rows == 1 || t.stride == t.cols;
    const int64_t rows = whole ? 1 : t.rows, cols = whole ? t.rows * t.cols : t.cols;
    if (cols >= most || whole) {
        for (int64_t r = 0; r < rows; ++r)
            for (int64_t c = 0; c < cols; c += most)
                add(r * t.stride + c, 1, std::min(most, cols - c));
        return;
    }
    const int64_t chunks = (cols * size + 15) / 16;
    const int64_t each = std::max<int64_t>(1, std::min(most / cols, runs / chunks));
    for (int64_t r = 0; r < rows; r += each) add(r * t.stride, std::min(each, rows - r), cols);
}

// Two outs at one place would be scaled twice, and an out that is another's gradient be read after
// that.  (A gradient without an out is read before all stores.)
void need_apart(const mbk_tensor *list, int32_t count) {
    const auto some = [&](int32_t i) { return list[i].rows && list[i].cols; };
    std::vector<const void *> outs;
    for (int32_t i = 0; i < count; ++i)
        if (list[i].out && some(i)) outs.push_back(list[i].out);
    std::sort(outs.begin(), outs.end(), std::less<>());
    bool apart = std::adjacent_find(outs.begin(), outs.end()) == outs.end();
    for (int32_t i = 0; i < count && apart; ++i)
        apart = !some(i) || !list[i].out || list[i].out == list[i].grad ||
                !std::binary_search(outs.begin(), outs.end(), list[i].grad, std::less<>());
    need(apart, "an out is also another gradient or its out");
}

mbk::FourbitShape fourbit_shape(const mbk_fourbit_shape *sh) {
    need(sh != nullptr, "null shape");
    need(sh->classes >= 1 && sh->classes <= MOST_ROWS, "classes must be in 1..2^31-256");
    need(sh->dim >= 1 && sh->dim <= (1 << 20), "dim must be in 1..2^20");
    need(sh->group == 32 || sh->group == 64 || sh->group == 128, "group must be 32, 64 or 128");
    return mbk::fourbit_shape(sh->classes, sh->dim, sh->group);
}

void need_packed(const void *packed) {
    need(packed != nullptr, "null argument");
    need(reinterpret_cast<uintptr_t>(packed) % 16 == 0, "packed must be a multiple of 16 bytes");
}

}  // namespace

extern "C" {

int mbk_xent(mbk_context *ctx, const mbk_xent_shape *shape, const void *h, const void *w,
             const float *bias, const int32_t *labels, const float *weights, float *loss,
             float *lse, char **err) {
    return mb::guarded(err, [&]() -> int {
        run_xent(ctx, xent_call(shape, h, w, bias, labels, weights, loss, lse));
        return 0;
    }, -1);
}

int mbk_xent_grad(mbk_context *ctx, const mbk_xent_shape *shape, const void *h, const void *w,
                  const float *bias, const int32_t *labels, const float *weights, float *loss,
                  float *lse, void *dh, void *dw, float *dbias, char **err) {
    return mb::guarded(err, [&]() -> int {
        mbk::XentCall c = xent_call(shape, h, w, bias, labels, weights, loss, lse);
        c.grad = dh || dw || dbias;
        c.dh = dh;
        c.dw = dw;
        c.dbias = dbias;
        run_xent(ctx, c);
        return 0;
    }, -1);
}

int mbk_expert_sort(mbk_context *ctx, const mbk_expert_plan *plan, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk::ExpertPlan p = expert_plan(plan);
        need(ctx != nullptr, "null kernel-seam context");
        mb::OnDevice here(mb::context_device(ctx));
        const int cus = mb::context_cus(ctx);
        std::lock_guard<std::mutex> lock(mb::context_scratch_mutex(ctx));
        char *scratch = mb::context_scratch(ctx, mbk::expert_scratch(p, cus));
        MB_HIP(mbk::launch_expert_sort(mb::context_stream(ctx), p, cus, scratch));
        return 0;
    }, -1);
}

int mbk_expert_gather(mbk_context *ctx, const mbk_expert_plan *plan, const mbk_expert_matrix *x,
                      void *sorted, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk::ExpertPlan p = expert_plan(plan);
        const mbk::ExpertMatrix m = expert_matrix(x, p.rows);
        need(sorted || !p.rows, "null argument");
        need(ctx != nullptr, "null kernel-seam context");
        if (!p.rows) return 0;
        mb::OnDevice here(mb::context_device(ctx));
        MB_HIP(mbk::launch_expert_gather(mb::context_stream(ctx), p, m, sorted));
        return 0;
    }, -1);
}

int mbk_expert_combine(mbk_context *ctx, const mbk_expert_plan *plan, const void *sorted,
                       const float *weights, const mbk_expert_matrix *out, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk::ExpertPlan p = expert_plan(plan);
        const mbk::ExpertMatrix m = expert_matrix(out, p.rows);
        need(sorted || !p.rows, "null argument");
        need(ctx != nullptr, "null kernel-seam context");
        if (!p.rows) return 0;
        mb::OnDevice here(mb::context_device(ctx));
        MB_HIP(mbk::launch_expert_combine(mb::context_stream(ctx), p, sorted, weights, m));
        return 0;
    }, -1);
}

int mbk_expert_combine_grad(mbk_context *ctx, const mbk_expert_plan *plan,
                            const mbk_expert_matrix *dout, const void *sorted,
                            const float *weights, void *d_sorted, float *d_weights, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk::ExpertPlan p = expert_plan(plan);
        const mbk::ExpertMatrix m = expert_matrix(dout, p.rows);
        need((sorted && d_sorted && d_weights) || !p.rows, "null argument");
        need(ctx != nullptr, "null kernel-seam context");
        if (!p.rows) return 0;
        mb::OnDevice here(mb::context_device(ctx));
        MB_HIP(mbk::launch_expert_combine_grad(mb::context_stream(ctx), p, m, sorted, weights,
                                               d_sorted, d_weights));
        return 0;
    }, -1);
}

int mbk_embed(mbk_context *ctx, const mbk_embed_shape *shape, const void *table,
              const int32_t *ids, const void *base, void *out, char **err) {
    return mb::guarded(err, [&]() -> int {
        mbk::EmbedCall c = embed_call(shape, ids, base);
        need(table && (!c.rows || (ids && out)), "null argument");
        need_multiple(size_of(c.bf16), {table, base, out});
        need_multiple(sizeof *ids, {ids});
        need(ctx != nullptr, "null kernel-seam context");
        if (!c.rows) return 0;
        c.table = table;
        c.out = out;
        mb::OnDevice here(mb::context_device(ctx));
        MB_HIP(mbk::launch_embed(mb::context_stream(ctx), c));
        return 0;
    }, -1);
}

int mbk_embed_grad(mbk_context *ctx, const mbk_embed_shape *shape, const int32_t *ids,
                   const void *dout, const void *base, void *dtable, char **err) {
    return mb::guarded(err, [&]() -> int {
        mbk::EmbedCall c = embed_call(shape, ids, base);
        need(dtable && (!c.rows || (ids && dout)), "null argument");
        need_multiple(size_of(c.bf16), {dout, base, dtable});
        need_multiple(sizeof *ids, {ids});
        need(ctx != nullptr, "null kernel-seam context");
        if (!c.rows && base == dtable) return 0;
        c.dout = dout;
        c.dtable = dtable;
        c.num_cus = mb::context_cus(ctx);
        mb::OnDevice here(mb::context_device(ctx));
        std::lock_guard<std::mutex> lock(mb::context_scratch_mutex(ctx));
        char *scratch = mb::context_scratch(ctx, mbk::embed_grad_scratch(c));
        MB_HIP(mbk::launch_embed_grad(mb::context_stream(ctx), c, scratch));
        return 0;
    }, -1);
}

int mbk_tensors_create(mbk_context *ctx, const mbk_tensor *list, int32_t count, mbk_tensors **out,
                       char **err) {
    return mb::guarded(err, [&]() -> int {
        need(count >= 0 && count <= (1 << 24), "count must be in 0..2^24");
        need(out && (!count || list), "null argument");
        int64_t elements = 0;
        for (int32_t i = 0; i < count; ++i) {
            const mbk_tensor &t = list[i];
            (void)is_bf16(t.type);
            need(t.rows >= 0 && t.cols >= 0 && t.rows <= MOST_ELEMENTS && t.cols <= MOST_ELEMENTS,
                 "rows and cols must be in 0..2^38");
            need(t.stride >= t.cols && t.stride <= MOST_STRIDE, "stride must be in cols..2^40");
            need(!t.cols || t.rows <= (MOST_ELEMENTS - elements) / t.cols,
                 "gradients must have at most 2^38 elements together");
            elements += t.rows * t.cols;
            need(t.grad || !t.rows || !t.cols, "null gradient");
            const size_t size = size_of(t.type == MBK_BF16);
            need(reinterpret_cast<uintptr_t>(t.grad) % size == 0 &&
                     reinterpret_cast<uintptr_t>(t.out) % size == 0,
                 "grad and out must be multiples of their elements' size");
        }
        need_apart(list, count);
        std::vector<mbk::ClipPiece> pieces;
        auto made = std::make_unique<mbk_tensors>();
        int64_t written = 0;
        for (int32_t i = 0; i < count; ++i) {
            if (list[i].out) written += list[i].rows * list[i].cols * (list[i].type == MBK_BF16 ? 2 : 4);
            made->outputs |= list[i].out != nullptr;
        }
        const auto cut = [&](int64_t most, int64_t runs) {
            pieces.clear();
            for (int32_t i = 0; i < count; ++i) add_pieces(list[i], most, runs, pieces);
        };
        if (elements <= 4 * mbk::CLIP_ONE * mbk::CLIP_RUNS) {
            cut(4 * mbk::CLIP_RUNS, mbk::CLIP_RUNS);
            made->one = pieces.size() <= (size_t)mbk::CLIP_ONE;
        }
        if (!made->one) cut(mbk::clip_piece(elements), INT64_MAX);
        need(ctx != nullptr, "null kernel-seam context");
        need(!mb::context_captured(ctx), "the context's stream is being captured");
        mb::OnDevice here(mb::context_device(ctx));
        made->pieces = (int64_t)pieces.size();
        made->streamed = written > mbk::STREAMED;
        made->piece.alloc(pieces.size());
        hipStream_t s = mb::context_stream(ctx);
        if (!pieces.empty())
            MB_HIP(hipMemcpyAsync(made->piece.ptr, pieces.data(),
                                  pieces.size() * sizeof(mbk::ClipPiece), hipMemcpyHostToDevice, s));
        MB_HIP(hipStreamSynchronize(s));
        std::lock_guard<std::mutex> lock(mb::context_scratch_mutex(ctx));
        mb::context_lists(ctx).push_back(std::move(made));
        *out = mb::context_lists(ctx).back().get();
        return 0;
    }, -1);
}

void mbk_tensors_destroy(mbk_context *ctx, mbk_tensors *list) {
    (void)mb::guarded(nullptr, [&]() -> int {
        if (!ctx || !list) return 0;
        mb::OnDevice here(mb::context_device(ctx));
        std::lock_guard<std::mutex> lock(mb::context_scratch_mutex(ctx));
        auto &lists = mb::context_lists(ctx);
        const auto at = std::find_if(lists.begin(), lists.end(),
                                     [&](const auto &l) { return l.get() == list; });
        if (at == lists.end()) return 0;
        // what a graph has captured must stay, and a wait would end the capture
        list->gone = true;
        if (list->captured || mb::context_captured(ctx)) return 0;
        (void)hipStreamSynchronize(mb::context_stream(ctx));
        lists.erase(at);
        return 0;
    }, -1);
}

int mbk_grad_clip(mbk_context *ctx, mbk_tensors *list, float max_norm, float *norm, char **err) {
    return mb::guarded(err, [&]() -> int {
        need(max_norm >= 0.0f, "max_norm must be >= 0");
        need(list && norm, "null argument");
        need_multiple(sizeof *norm, {norm});
        need(ctx != nullptr, "null kernel-seam context");
        std::lock_guard<std::mutex> lock(mb::context_scratch_mutex(ctx));
        const auto &lists = mb::context_lists(ctx);
        need(std::any_of(lists.begin(), lists.end(),
                         [&](const auto &l) { return l.get() == list && !l->gone; }),
             "the list is not one of the context's");
        mb::OnDevice here(mb::context_device(ctx));
        const int cus = mb::context_cus(ctx);
        char *scratch = mb::context_scratch(ctx, mbk::clip_scratch(list->pieces, cus));
        list->captured |= mb::context_captured(ctx);
        MB_HIP(mbk::launch_clip(mb::context_stream(ctx),
                                {list->piece.ptr, list->pieces, list->one, list->outputs,
                                 list->streamed, max_norm, norm, cus},
                                scratch));
        return 0;
    }, -1);
}

int64_t mbk_fourbit_bytes(const mbk_fourbit_shape *shape) {
    return mb::guarded(nullptr, [&]() -> int64_t { return (int64_t)mbk::fourbit_bytes(fourbit_shape(shape)); },
                       -1);
}

int mbk_fourbit_pack(mbk_context *ctx, const mbk_fourbit_shape *shape, int32_t type, const void *w,
                int64_t w_stride, void *packed, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk::FourbitShape s = fourbit_shape(shape);
        need(w_stride >= s.dim && w_stride <= MOST_STRIDE, "w_stride must be in dim..2^40");
        const bool bf16 = is_bf16(type);
        need(w != nullptr, "null argument");
        need_multiple(size_of(bf16), {w});
        need_packed(packed);
        need(ctx != nullptr, "null kernel-seam context");
        mb::OnDevice here(mb::context_device(ctx));
        MB_HIP(mbk::launch_fourbit_pack(mb::context_stream(ctx), s, bf16, w, w_stride,
                                   static_cast<char *>(packed)));
        return 0;
    }, -1);
}

int mbk_fourbit_scores(mbk_context *ctx, const mbk_fourbit_shape *shape, int64_t rows, int32_t type,
                  const void *h, int64_t h_stride, const void *packed, const float *bias,
                  float *scores, int64_t score_stride, char **err) {
    return mb::guarded(err, [&]() -> int {
        mbk::FourbitCall c{};
        c.shape = fourbit_shape(shape);
        need(rows >= 0 && rows <= MOST_ROWS, "rows must be in 0..2^31-256");
        need(h_stride >= c.shape.dim && h_stride <= MOST_STRIDE, "h_stride must be in dim..2^40");
        need(score_stride >= c.shape.classes && score_stride <= MOST_STRIDE,
             "score_stride must be in classes..2^40");
        c.bf16 = is_bf16(type);
        need(!rows || (h && scores), "null argument");
        need_multiple(size_of(c.bf16), {h});
        need_multiple(sizeof *scores, {bias, scores});
        need_packed(packed);
        need(ctx != nullptr, "null kernel-seam context");
        if (!rows) return 0;
        uint32_t *codes;
        _Float16 *scales;
        int32_t *exponents;
        mbk::fourbit_parts(c.shape, static_cast<char *>(const_cast<void *>(packed)), &codes, &scales,
                      &exponents);
        c.rows = rows;
        c.h = h;
        c.h_stride = h_stride;
        c.codes = codes;
        c.scales = scales;
        c.exponents = exponents;
        c.bias = bias;
        c.scores = scores;
        c.score_stride = score_stride;
        c.num_cus = mb::context_cus(ctx);
        mb::OnDevice here(mb::context_device(ctx));
        std::lock_guard<std::mutex> lock(mb::context_scratch_mutex(ctx));
        char *scratch = mb::context_scratch(ctx, mbk::fourbit_scratch(c));
        MB_HIP(mbk::launch_fourbit_scores(mb::context_stream(ctx), c, scratch));
        return 0;
    }, -1);
}

int mbk_adjust(mbk_context *ctx, const mbk_adjust_shape *shape, const float *scores,
               const int32_t *ids, const int32_t *lengths, const float *bias,
               const uint32_t *allowed, float *out, char **err) {
    return mb::guarded(err, [&]() -> int {
        const mbk_adjust_shape *sh = shape;
        need(sh != nullptr, "null shape");
        need(sh->rows >= 0 && sh->rows <= MOST_ROWS, "rows must be in 0..2^31-256");
        need(sh->classes >= 1 && sh->classes <= MOST_ROWS, "classes must be in 1..2^31-256");
        need(sh->rows <= MOST_STRIDE / sh->classes, "rows * classes must be at most 2^40");
        need(sh->score_stride >= sh->classes && sh->out_stride >= sh->classes &&
                 sh->score_stride <= MOST_STRIDE && sh->out_stride <= MOST_STRIDE,
             "score_stride and out_stride must be in classes..2^40");
        need(sh->history >= 0 && sh->history <= (1 << 24), "history must be in 0..2^24");
        need(sh->history_stride >= sh->history && sh->history_stride <= MOST_STRIDE,
             "history_stride must be in history..2^40");
        need(sh->mask_stride == 0 || (sh->mask_stride >= (sh->classes + 31) / 32 &&
                                      sh->mask_stride <= MOST_STRIDE),
             "mask_stride must be 0 or in classes / 32..2^40");
        need(sh->repetition > 0.0f && std::isfinite(sh->repetition),
             "repetition must be positive and finite");
        need(std::isfinite(sh->presence) && std::isfinite(sh->frequency),
             "presence and frequency must be finite");
        need(!sh->rows || (scores && out && (!sh->history || ids)), "null argument");
        need_multiple(sizeof *scores, {scores, ids, lengths, bias, allowed, out});
        need(scores != out || sh->score_stride == sh->out_stride,
             "scores that are out must have its stride");
        need(ctx != nullptr, "null kernel-seam context");
        if (!sh->rows) return 0;
        mbk::AdjustCall c{};
        c.rows = sh->rows;
        c.classes = sh->classes;
        c.score_stride = sh->score_stride;
        c.out_stride = sh->out_stride;
        c.history = sh->history;
        c.history_stride = sh->history_stride;
        c.mask_stride = sh->mask_stride;
        c.repetition = sh->repetition;
        c.presence = sh->presence;
        c.frequency = sh->frequency;
        c.penalties = sh->history > 0 && (sh->repetition != 1.0f || sh->presence != 0.0f ||
                                          sh->frequency != 0.0f);
        c.scores = scores;
        c.ids = ids;
        c.lengths = lengths;
        c.bias = bias;
        c.allowed = allowed;
        c.out = out;
        mb::OnDevice here(mb::context_device(ctx));
        MB_HIP(mbk::launch_adjust(mb::context_stream(ctx), c));
        return 0;
    }, -1);
}

}  // extern "C"
