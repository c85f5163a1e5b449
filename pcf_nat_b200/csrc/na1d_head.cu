// C ABI of the losses of a classification head: checks of the arguments, where the pieces lie in the caller's buffers, order of the passes.
#include "na1d_head.cuh"

#include <climits>
#include <cmath>

namespace na1d {
namespace head {

Shape shape_of(const na1d_head& h) {
    Shape s = {};
    s.N = h.rows; s.D = h.dim; s.V = h.classes; s.k = h.top;
    s.Np = round_up(s.N, kTile);
    s.Dp = round_up(s.D, 8);
    s.parts = (s.V + kTile - 1) / kTile * (kTile / kPart);
    s.x_stride = h.x_stride; s.w_stride = h.weight_stride;
    s.norm = h.normalize != 0;
    const bool fp16 = h.dtype == NA1D_FP16;
    // the weight is read where it is if its rows are whole 16-byte pieces, and need no powers of two of their own
    s.copy_w = (fp16 && s.norm) || h.weight_type != h.dtype || s.D % 8 != 0 || h.weight_stride % 8 != 0 || h.weight_stride < s.D || (reinterpret_cast<uintptr_t>(h.weight) & 15) != 0;
    s.cs = kLog2e * h.scale / (s.k ? h.temperature : 1.f);
    // fp16 holds 6e-5 to 65504 in full: probabilities times 2^14. Those of cosines carry the inverse lengths, up to 2^-lift each, and
    // |p - 1| or |p - q| of up to 1 times the margin's slope cos m + c / sin a sin m: 445 at a margin of 0.2, 2236 at a right angle.
    const double slope = s.k || h.margin == 0.f ? 1.0 : std::fabs(std::cos((double)h.margin)) + std::fabs(std::sin((double)h.margin)) / std::sqrt((double)kSineFloor);
    const int room = s.norm ? 2 * lift(true) + (int)std::floor(std::log2(65504.0 / (1.01 * slope))) : 14;   // (1 %: rounded cosines and lengths)
    s.up = fp16 ? std::ldexp(1.f, room) : 1.f;
    return s;
}

Saved saved_at(const na1d_head& h, const Shape& s, void* base) {
    Saved v = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        uint8_t* p = static_cast<uint8_t*>(base) + at;   // (with base null: sizes alone)
        at += round_up(bytes, 256);
        return static_cast<void*>(p);
    };
    v.words = static_cast<Words*>(take(sizeof(Words)));
    v.own_count = static_cast<int*>(take(round_up(s.V, kTile) * 4));
    v.place = static_cast<int*>(take(s.N * 4));
    v.row = static_cast<int*>(take(s.Np * 4));
    v.lse2 = static_cast<float*>(take(s.Np * 4));
    v.target = static_cast<int*>(take(s.Np * 4));
    v.slope = static_cast<float*>(take(s.Np * 4));
    v.own = static_cast<int*>(take(s.V * kOwn * 4));
    if (s.norm) {
        v.ix = static_cast<float*>(take(s.Np * 4));
        v.iw = static_cast<float*>(take(round_up(s.V, kTile) * 4));
        v.x_up = static_cast<float*>(take(s.Np * 4));
        if (s.copy_w) v.w_up = static_cast<float*>(take(s.V * 4));
    }
    if (s.k) {
        v.q = static_cast<float*>(take(s.N * s.k * 4));
        v.index = static_cast<int*>(take(s.N * s.k * 4));
        v.entry = static_cast<float*>(take(s.N * s.k * 4));
    }
    v.x = take(s.Np * s.Dp * 2);
    if (s.copy_w) v.w = take(s.V * s.Dp * 2);
    v.bytes = at;
    return v;
}

// A piece of the classes has gradients of at most kPieceBytes, or four tiles where those are more. Smaller pieces would stay in L2, but cost more than that
// saves; larger ones gain little for their memory. 64, 128, 256, 512 MB: 3152, 3182, 3012, 3157 us a pass at 8192 x 1024 x 50000 (all rows counted);
// 261, 203, 205, 204 at 4099 x 192 x 17982; 650, 639, 613, 592 at 1024 x 256 x 200003; 3458, 3028, 2870, 2767 at 6400 x 192 x 200000.
constexpr int64_t kPieceBytes = 256ll << 20;
// when the last pair is through with its items, in steps (as the products' kernel shares them out)
static int64_t last_end(int64_t items_x, int64_t item_x, int64_t items_w, int64_t item_w, int64_t pairs) {
    const int64_t more = items_w % pairs, busy1 = items_w / pairs * item_w, busy0 = busy1 + item_w, average = (items_w * item_w + items_x * item_x) / pairs;
    auto fill = [&](int64_t end, int64_t busy) { return end > busy ? (end - busy) / item_x : 0; };
    int64_t best = -1;
    for (int k = 0; k < 32; ++k) {
        const int64_t busy = k & 1 ? busy1 : busy0, end = busy + ((average > busy ? average - busy : 0) / item_x + (k >> 1)) * item_x;
        if (more * fill(end, busy0) + (pairs - more) * fill(end, busy1) >= items_x && (best < 0 || end < best)) best = end;
    }
    return best > (more ? busy0 : busy1) ? best : more ? busy0 : busy1;
}
Pieces pieces_of(const Shape& s, bool want_x, bool want_w) {
    Pieces p = {};
    const int64_t pairs = device_sm_count() / 2;
    p.tiles = (s.V + kTile - 1) / kTile;
    int64_t most = kPieceBytes / (s.Np * kTile * 2);
    most = most < 4 ? 4 : most;
    p.count = (p.tiles + most - 1) / most;
    p.piece_tiles = (p.tiles + p.count - 1) / p.count;
    p.count = (p.tiles + p.piece_tiles - 1) / p.piece_tiles;
    // Whole rounds of the pairs, where the limit allows (6400 x 192 x 200000: 2870 us in pieces of 79 tiles, 2804 in ones of 148, which are 462 MB, 2915 in ones of 74).
    if (p.piece_tiles > pairs && p.count > 1 && round_up(p.piece_tiles, pairs) <= most) {
        p.piece_tiles = round_up(p.piece_tiles, pairs);
        p.count = (p.tiles + p.piece_tiles - 1) / p.piece_tiles;
    }
    p.pitch = p.piece_tiles * kTile;
    p.d_tiles = (int)((s.D + kTile - 1) / kTile);
    p.d_width = (int)round_up((s.D + p.d_tiles - 1) / p.d_tiles, 32);
    // Steps of 64 of the two contractions, and a pair's share of all of them. The weight's tiles are whole where that leaves no pair with much more
    // than its share; then their gradients leave at once, unless the way back through the normalisation needs more than one tile of a row.
    const int64_t steps_x = p.pitch / 64, steps_w = s.Np / 64;
    const int64_t items_x = want_x ? s.Np / kTile * p.d_tiles : 0, tiles_w = want_w ? p.piece_tiles * p.d_tiles : 0;
    const int64_t share = (items_x * steps_x + tiles_w * steps_w + pairs - 1) / pairs, whole = share + share / 4 < 16 ? 16 : share + share / 4;
    p.splits_w = (int)(whole >= steps_w ? 1 : (steps_w + whole - 1) / whole < 16 ? (steps_w + whole - 1) / whole : 16);
    p.direct_w = want_w && p.splits_w == 1 && (!s.norm || p.d_tiles == 1);
    // Splits of the rows' contraction, which fill up what the weight's items leave of the pairs' time: the end of the last pair (a step takes about
    // half a microsecond) against the partial sums' way to memory and back (4 TB/s; the normalised ones of wide rows are read twice).
    const int64_t items_w = tiles_w * p.splits_w, item_w = (steps_w + p.splits_w - 1) / p.splits_w;
    const double each = (double)s.Np * s.Dp * 4 * (s.norm && s.Dp > 256 ? 3 : 2) / 4e6;
    double best = 0;
    p.splits_x = 1;
    for (int n = 1; items_x && n <= 32 && n <= steps_x / 4 + 1; ++n) {
        const double cost = 0.5 * last_end(items_x * n, (steps_x + n - 1) / n, items_w, item_w, pairs) + n * each;
        if (n == 1 || cost < best) { best = cost; p.splits_x = n; }
    }
    return p;
}

namespace {

bool type_ok(int t) { return t == NA1D_BF16 || t == NA1D_FP16 || t == NA1D_FP32; }
bool bad_align(const void* p, int64_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

int check(const na1d_head* h) {
    if (!h) return NA1D_ERR_NULL_POINTER;
    if (h->dtype != NA1D_BF16 && h->dtype != NA1D_FP16) return NA1D_ERR_BAD_DTYPE;
    if (!type_ok(h->x_type) || !type_ok(h->weight_type)) return NA1D_ERR_BAD_DTYPE;
    if ((h->x_type != NA1D_FP32 && h->x_type != h->dtype) || (h->weight_type != NA1D_FP32 && h->weight_type != h->dtype)) return NA1D_ERR_BAD_DTYPE;
    if (h->rows <= 0 || h->dim <= 0 || h->classes <= 0 || h->top < 0) return NA1D_ERR_BAD_SHAPE;
    if (h->rows > NA1D_HEAD_MAX_ROWS || h->dim > NA1D_HEAD_MAX_DIM || h->classes > NA1D_HEAD_MAX_CLASSES || h->top > NA1D_HEAD_MAX_TOP) return NA1D_ERR_TOO_LARGE;
    if (h->x_stride < 0 || h->weight_stride < 0) return NA1D_ERR_BAD_STRIDE;
    if (h->reduction != NA1D_HEAD_MEAN && h->reduction != NA1D_HEAD_SUM && h->reduction != NA1D_HEAD_NONE) return NA1D_ERR_BAD_SHAPE;
    if (!(h->scale > 0.f) || !std::isfinite(h->scale) || !std::isfinite(h->margin)) return NA1D_ERR_BAD_SCALE;
    if (!(h->scale < 0x1p118f)) return NA1D_ERR_BAD_SCALE;
    if (h->top > 0) {
        if (!(h->temperature > 0.f) || !std::isfinite(h->temperature)) return NA1D_ERR_BAD_SCALE;
        // the factors of logits, gradients and losses are held in fp32
        const double tau = h->temperature, factors[3] = {h->scale / tau, h->scale * tau, tau * tau};
        for (double f : factors)
            if (!(f > 0x1p-118 && f < 0x1p118)) return NA1D_ERR_BAD_SCALE;
    }
    if ((h->top > 0 || !h->normalize) && h->margin != 0.f) return NA1D_ERR_BAD_SCALE;
    if (!h->x || !h->weight || (h->top ? !h->teacher_logits || !h->teacher_index : !h->labels)) return NA1D_ERR_NULL_POINTER;
    if (bad_align(h->x, h->x_type == NA1D_FP32 ? 4 : 2) || bad_align(h->weight, h->weight_type == NA1D_FP32 ? 4 : 2) || bad_align(h->labels, 8) ||
        bad_align(h->teacher_index, 8) || bad_align(h->teacher_logits, 4))
        return NA1D_ERR_MISALIGNED;
    return NA1D_OK;
}

// the forward pass's scratch: partial maxima and sums, the blocks' losses, which rows have a teacher
struct Forward {
    float2* part;
    float* block_sums;
    int* flags;
    int64_t bytes;
};
Forward forward_at(const Shape& s, void* base) {
    Forward f = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        uint8_t* p = static_cast<uint8_t*>(base) + at;
        at += round_up(bytes, 256);
        return static_cast<void*>(p);
    };
    f.part = static_cast<float2*>(take(s.parts * s.Np * 8));
    f.block_sums = static_cast<float*>(take((s.N + 7) / 8 * 4));
    if (s.k) f.flags = static_cast<int*>(take(s.N * 4));
    f.bytes = at;
    return f;
}
// the backward pass's: gradients of a piece's logits, partial sums of both products, the rows' factors
struct Backward {
    void* grad;
    float *part_x, *part_w, *coef;
    int64_t bytes;
};
Backward backward_at(const na1d_head& h, const Shape& s, const Pieces& p, bool want_x, bool want_w, void* base) {
    Backward b = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        uint8_t* q = static_cast<uint8_t*>(base) + at;
        at += round_up(bytes, 256);
        return static_cast<void*>(q);
    };
    b.grad = take(s.Np * p.pitch * 2);
    if (want_x) b.part_x = static_cast<float*>(take(p.splits_x * s.Np * s.Dp * 4));
    if (want_w) b.part_w = static_cast<float*>(take((p.direct_w ? s.Np : p.splits_w * p.pitch) * s.Dp * 4));   // (direct: rows' own classes alone)
    if (h.reduction == NA1D_HEAD_NONE) b.coef = static_cast<float*>(take((s.Np + 1) * 4));
    b.bytes = at;
    return b;
}
#define NA1D_HEAD_TRY(call)                                   \
    do {                                                      \
        if (cudaError_t e = (call)) return api_cuda_status(e); \
    } while (0)

int forward(const na1d_head& h, float* loss, void* saved, void* scratch, cudaStream_t st) {
    bind_primary_context();
    const Shape s = shape_of(h);
    const Saved sv = saved_at(h, s, saved);
    const Forward f = forward_at(s, scratch);
    const void* w = s.copy_w ? sv.w : h.weight;
    const int64_t ldw = s.copy_w ? s.Dp : h.weight_stride;
    NA1D_HEAD_TRY(prepare(h, s, sv, f.flags, loss, st));
    NA1D_HEAD_TRY(stats(h, s, sv, f.part, w, ldw, st));
    NA1D_HEAD_TRY(combine(h, s, sv, f.part, f.block_sums, loss, w, ldw, st));
    return NA1D_OK;
}

int backward(const na1d_head& h, void* dx, void* dw, const float* d_loss, void* saved, void* scratch, cudaStream_t st) {
    bind_primary_context();
    const Shape s = shape_of(h);
    const Saved sv = saved_at(h, s, saved);
    const Pieces p = pieces_of(s, dx != nullptr, dw != nullptr);
    const Backward b = backward_at(h, s, p, dx != nullptr, dw != nullptr, scratch);
    const void* w = s.copy_w ? sv.w : h.weight;
    const int64_t ldw = s.copy_w ? s.Dp : h.weight_stride;
    if (b.coef) NA1D_HEAD_TRY(coefficients(h, s, sv, d_loss, b.coef, st));
    for (int64_t i = 0; i < p.count; ++i) {
        const int64_t v0 = i * p.pitch, cols = s.V - v0 < p.pitch ? s.V - v0 : p.pitch;
        const bool last = i + 1 == p.count;
        FinishArgs f = finish_args(h, s, sv, last ? dx : nullptr, dw, b.part_x, b.part_w, d_loss, b.coef, p, v0, p.direct_w || !dw ? 0 : cols, w, ldw);
        f.own_classes = p.direct_w && last;
        const bool after = i > 0 || b.coef != nullptr;
        NA1D_HEAD_TRY(gradients(h, s, sv, b.coef, b.grad, p.pitch, v0, (cols + kTile - 1) / kTile, w, ldw, after, st));
        NA1D_HEAD_TRY(products(h, s, sv, b.grad, p, v0, cols, i > 0, b.part_x, b.part_w, f, w, ldw, st));
        if (f.dx || f.cols || f.own_classes) NA1D_HEAD_TRY(finish(h, f, st));
    }
    return NA1D_OK;
}

}  // namespace
}  // namespace head
}  // namespace na1d

extern "C" {

int64_t na1d_head_saved_bytes(const na1d_head* head) {
    if (int s = na1d::head::check(head)) return s;
    const na1d::head::Shape s = na1d::head::shape_of(*head);
    return na1d::head::saved_at(*head, s, nullptr).bytes;
}
int64_t na1d_head_forward_scratch(const na1d_head* head) {
    if (int s = na1d::head::check(head)) return s;
    return na1d::head::forward_at(na1d::head::shape_of(*head), nullptr).bytes;
}
int64_t na1d_head_backward_scratch(const na1d_head* head, int want_x, int want_weight) {
    if (int s = na1d::head::check(head)) return s;
    const na1d::head::Shape s = na1d::head::shape_of(*head);
    return na1d::head::backward_at(*head, s, na1d::head::pieces_of(s, want_x != 0, want_weight != 0), want_x != 0, want_weight != 0, nullptr).bytes;
}
int na1d_head_weight_in_place(const na1d_head* head) {
    if (int s = na1d::head::check(head)) return s;
    return !na1d::head::shape_of(*head).copy_w;
}
int na1d_head_forward(const na1d_head* head, float* loss, void* saved, void* scratch, void* stream) {
    if (int s = na1d::head::check(head)) return s;
    if (!loss || !saved || !scratch) return NA1D_ERR_NULL_POINTER;
    if (na1d::head::bad_align(saved, 256) || na1d::head::bad_align(scratch, 256) || na1d::head::bad_align(loss, 4)) return NA1D_ERR_MISALIGNED;
    return na1d::head::forward(*head, loss, saved, scratch, (cudaStream_t)stream);
}
int na1d_head_backward(const na1d_head* head, void* d_x, void* d_weight, const float* d_loss, void* saved, void* scratch, void* stream) {
    if (int s = na1d::head::check(head)) return s;
    if (!d_loss || !saved || !scratch || (!d_x && !d_weight)) return NA1D_ERR_NULL_POINTER;
    if (na1d::head::bad_align(saved, 256) || na1d::head::bad_align(scratch, 256) || na1d::head::bad_align(d_x, 32) || na1d::head::bad_align(d_weight, 32) ||
        na1d::head::bad_align(d_loss, 4))
        return NA1D_ERR_MISALIGNED;
    return na1d::head::backward(*head, d_x, d_weight, d_loss, saved, scratch, (cudaStream_t)stream);
}

}  // extern "C"
