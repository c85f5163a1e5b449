// The losses of a classification head (na1d_head*.cu): what a call is made of, and where its pieces lie in the caller's buffers.
//
// Rows x (N, D) and weight w (V, D), products s = x w^T, logits z = scale s (or scale s / (|x| |w|)). The (N, V) logits are never stored:
//   forward   rows that count side by side (head_rows) -> s tile by tile, a running maximum and sum per row and 128 classes (head_stats)
//             -> log-sum-exp, the target's terms, the loss (head_combine)
//   backward  for a piece of the classes at a time: s again, its gradient in 16 bits (head_logits, gradient form) -> the products with
//             w and x (head_grad) -> sums over splits, the way back through the normalisation (head_finish)
#pragma once
#include "../../include/na1d_b200.h"
#include "na1d_tc_common.cuh"
#include "na1d_internal.h"

namespace na1d {

int api_cuda_status(cudaError_t e);   // a status code, and the error kept for na1d_last_cuda_error()

namespace head {

constexpr int kTile = 256;            // rows and classes of a product tile (a pair of CTAs)
constexpr int kPart = 128;            // classes that one partial maximum and sum stand for
constexpr float kSineFloor = 2e-7f;   // of the squared sine in the margin's formula
constexpr int kIgnored = -1, kBad = -2;
constexpr int kNoClass = 0x7fffffff;  // behind a row's entries, which are sorted by class
constexpr int kOwn = 8;               // rows of a class whose own gradients' roundings are made good

inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// words at the start of `saved`
struct Words {
    int counted;                // rows that count
    int ticket;                 // blocks of the combining kernel that are done
    int most_ix, most_iw;       // largest inverse norms (their bits), for the range of fp16
};

// Pointers into `saved`. Rows that count are numbered c = 0 .. counted - 1 in their order.
struct Saved {
    Words* words;
    int* place;        // (N)  c of a row, or kIgnored
    int* row;          // (Np) row of c
    float* lse2;       // (Np) log2 of the softmax's sum
    int* target;       // (Np) the row's own class: its label (or kBad), or the entry with the largest gradient
    float* slope;      // (Np) gradient of that class's logit: (p - 1) psi', or p - q
    int* own_count;    // (V rounded up) rows whose own class it is
    int* own;          // (V, kOwn) and the first of them to come
    float* ix;         // (Np) 1 / |x| (normalised)
    float* iw;         // (V rounded up) 1 / |w|
    float* q;          // (N, k) teacher's probabilities, sorted by class
    int* index;        // (N, k) classes in their order, kNoClass behind them
    float* entry;      // (N, k) the entry's logit as a power of two, then its gradient p - q
    void* x;           // (Np, Dp) 16 bits, zeros behind the rows that count
    void* w;           // (V, Dp) 16 bits, where the weight is not used in its place
    int64_t zeros, bytes;   // the first of them start as zeros
};

struct Shape {
    int64_t N, D, V, k, Np, Dp, parts;
    int64_t x_stride, w_stride;
    bool norm, train_classes, copy_w;
    float cs;                   // log2(e) scale / temperature: from a product (or cosine) to a power of two
};

Shape shape_of(const na1d_head& h);
Saved saved_at(const na1d_head& h, const Shape& s, void* base);

// how the backward pass is cut up
struct Pieces {
    int64_t tiles, piece_tiles, count, pitch;   // tiles of classes; of a piece; pieces; row pitch of a piece's gradients
    int d_tiles, d_width;                       // tiles over D and their width
    int splits_x, splits_w;
};
Pieces pieces_of(const Shape& s, bool want_x, bool want_w);

// ---- passes (na1d_head_rows.cu)
cudaError_t teacher(const na1d_head& h, const Shape& s, const Saved& sv, int* flags, cudaStream_t st);
cudaError_t rows(const na1d_head& h, const Shape& s, const Saved& sv, const int* flags, float* loss, cudaStream_t st);
cudaError_t weight(const na1d_head& h, const Shape& s, const Saved& sv, cudaStream_t st);
cudaError_t combine(const na1d_head& h, const Shape& s, const Saved& sv, const float2* part, float* block_sums, float* loss, const void* w, int64_t ldw,
                    cudaStream_t st);
cudaError_t coefficients(const na1d_head& h, const Shape& s, const Saved& sv, const float* d_loss, float* coef, cudaStream_t st);
// gradients of rows v0 .. v0 + cols of the weight (cols may be 0) and, where dx is given, of the rows
cudaError_t finish(const na1d_head& h, const Shape& s, const Saved& sv, void* dx, void* dw, const float* part_x, const float* part_w, const float* d_loss,
                   const float* coef, int splits_x, int splits_w, int64_t v0, int64_t cols, int64_t piece_rows, const void* w, int64_t ldw, cudaStream_t st);

// ---- products (na1d_head_logits.cu, na1d_head_grad.cu)
cudaError_t stats(const na1d_head& h, const Shape& s, const Saved& sv, float2* part, const void* w, int64_t ldw, cudaStream_t st);
cudaError_t gradients(const na1d_head& h, const Shape& s, const Saved& sv, const float* coef, void* grad, int64_t pitch, int64_t v0, int64_t tiles, const void* w,
                      int64_t ldw, cudaStream_t st);
cudaError_t products(const na1d_head& h, const Shape& s, const Saved& sv, const void* grad, const Pieces& p, int64_t v0, int64_t cols, bool add, float* part_x,
                     float* part_w, const void* w, int64_t ldw, cudaStream_t st);
int logits_read_status();
int grad_read_status();

// power of two that a 16-bit gradient of logits is multiplied with. bf16: none. fp16 holds 6e-5 to 65504 in full: probabilities times 2^14;
// normalised ones also carry the inverse norms, at most `most`, and the margin's slope (at most 450).
__device__ __forceinline__ float gradient_scale(const Words* w, bool fp16, bool norm) {
    if (!fp16) return 1.f;
    if (!norm) return 16384.f;
    const float most = __int_as_float(w->most_ix) * __int_as_float(w->most_iw);
    if (!(most > 0.f) || most > 1e30f) return 1.f;
    int e;
    frexpf(most, &e);
    e = 6 - e;
    return ldexpf(1.f, e < -100 ? -100 : e > 100 ? 100 : e);
}

// The gradient of a row's own class as it is rounded to 16 bits, in one order of operations: `out` = row_factor(..)
__device__ __forceinline__ float row_factor(float up, float ix, float coef, bool norm) { return norm ? up * ix * coef : up * coef; }
__device__ __forceinline__ float own_gradient(float slope, float out, float iw, bool norm) { return norm ? (slope * out) * iw : slope * out; }

}  // namespace head
}  // namespace na1d
