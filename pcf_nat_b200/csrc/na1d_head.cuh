// The losses of a classification head (na1d_head*.cu): what a call is made of, and where its pieces lie in the caller's buffers.
//
// Rows x (N, D) and weight w (V, D), products s = x w^T, logits z = scale s (or scale s / (|x| |w|)). The (N, V) logits are never stored:
//   forward   rows that count side by side (prepare) -> s tile by tile, a running maximum and sum per row and 64 classes (stats)
//             -> log-sum-exp, the target's terms, the loss (combine)
//   backward  for a piece of the classes at a time: s again, its gradient in 16 bits (gradients) -> the products with
//             w and x (products) -> sums over splits, the way back through the normalisation (finish)
#pragma once
#include "../../include/na1d_b200.h"
#include "na1d_tc_common.cuh"
#include "na1d_internal.h"

#include <atomic>
#include <utility>

namespace na1d {

int api_cuda_status(cudaError_t e);   // a status code, and the error kept for na1d_last_cuda_error()

namespace head {

// Launch of one of a head's kernels. Each of them starts while its predecessor in the stream ends (programmatic dependent launch): it sets itself up, waits
// until everything before it is done (ptx::grid_dependency_wait, before it reads or writes anything), and lets its own successor start. `after`: false for
// the first kernel of a pass, whose predecessor is somebody else's.
template <typename... P, typename... A>
inline cudaError_t launch(void (*kern)(P...), int64_t blocks, int threads, size_t smem, cudaStream_t st, bool after, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = after ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
}
// dynamic shared memory beyond the default for a kernel, once for each device
template <typename K>
inline cudaError_t allow_smem(K kern, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
    done.fetch_or(bit, std::memory_order_relaxed);
    return cudaSuccess;
}
__device__ __forceinline__ void wait_for_predecessor() {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr int kTile = 256;            // rows and classes of a product tile (a pair of CTAs)
constexpr int kPart = 64;             // classes that one partial maximum and sum stand for
constexpr float kSineFloor = 2e-7f;   // of the squared sine in the margin's formula
constexpr int kIgnored = -1, kBad = -2;
constexpr int kNoClass = 0x7fffffff;  // behind a row's entries, which are sorted by class
constexpr int kOwn = 4;               // rows of a class whose own gradients' roundings are made good
// Normalised rows (and classes, where the weight is copied) are kept times a power of two that leaves them a length of 2^lift(..) to twice that. A cosine's
// gradient carries both inverse lengths: so its range in fp16 is the same for every row and class, whatever the others' lengths are. 2^7 keeps elements of
// 2^-21 of a row's length out of fp16's subnormals, and the longest elements far from its end.
__host__ __device__ constexpr int lift(bool fp16) { return fp16 ? 7 : 0; }

inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// words at the start of `saved`
struct Words {
    int counted;                // rows that count
    int ticket;                 // blocks of the combining kernel that are done
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
    float* ix;         // (Np) 1 / |x| of the kept row (normalised)
    float* iw;         // (V rounded up) 1 / |w|, of the kept class where there is a copy
    float* x_up;       // (Np) the power of two that the kept row is x times
    float* w_up;       // (V) of the kept class; null where the weight stays where it is
    float* q;          // (N, k) teacher's probabilities, sorted by class
    int* index;        // (N, k) classes in their order, kNoClass behind them
    float* entry;      // (N, k) the entry's logit as a power of two, then its gradient p - q
    void* x;           // (Np, Dp) 16 bits, zeros behind the rows that count
    void* w;           // (V, Dp) 16 bits, where the weight is not used in its place
    int64_t bytes;
};

struct Shape {
    int64_t N, D, V, k, Np, Dp, parts;
    int64_t x_stride, w_stride;
    bool norm, copy_w;
    float cs;                   // log2(e) scale / temperature: from a product (or cosine) to a power of two
    float up;                   // power of two that a 16-bit gradient of logits is multiplied with
};

Shape shape_of(const na1d_head& h);
Saved saved_at(const na1d_head& h, const Shape& s, void* base);

// how the backward pass is cut up
struct Pieces {
    int64_t tiles, piece_tiles, count, pitch;   // tiles of classes; of a piece; pieces; row pitch of a piece's gradients
    int d_tiles, d_width;                       // tiles over D and their width
    int splits_x, splits_w;                     // of the contractions
    bool direct_w;                              // the weight's gradient leaves the products as it is: no partial sums
};
Pieces pieces_of(const Shape& s, bool want_x, bool want_w);

// ---- passes (na1d_head_rows.cu)
cudaError_t prepare(const na1d_head& h, const Shape& s, const Saved& sv, int* flags, float* loss, cudaStream_t st);
cudaError_t combine(const na1d_head& h, const Shape& s, const Saved& sv, const float2* part, float* block_sums, float* loss, const void* w, int64_t ldw,
                    cudaStream_t st);
cudaError_t coefficients(const na1d_head& h, const Shape& s, const Saved& sv, const float* d_loss, float* coef, cudaStream_t st);
// What the last step of both gradients needs: sums times the common factor, what rounding took from a row's own class, the way back through
// the normalisation.
struct FinishArgs {
    void *dx, *dw;
    const float *part_x, *part_w, *d_loss, *coef;
    const void *x, *w;
    const float *ix, *iw, *x_up, *w_up, *slope;
    const int *place, *target, *own_count, *own;
    const Words* words;
    long long Np, piece_rows, ldw;
    int N, D, Dp, cols, v0, splits_x, splits_w, x_type, w_type, reduction;
    float factor, up;
    bool norm;
    bool own_classes;           // part_w has the sums of classes that are rows' own, at such a row
};
FinishArgs finish_args(const na1d_head& h, const Shape& s, const Saved& sv, void* dx, void* dw, const float* part_x, const float* part_w, const float* d_loss,
                       const float* coef, const Pieces& p, int64_t v0, int64_t cols, const void* w, int64_t ldw);
// the rows' gradients (dx) and, from partial sums, those of a piece of the weight (cols > 0)
cudaError_t finish(const na1d_head& h, const FinishArgs& a, cudaStream_t st);

// ---- products (na1d_head_logits.cu, na1d_head_grad.cu)
cudaError_t stats(const na1d_head& h, const Shape& s, const Saved& sv, float2* part, const void* w, int64_t ldw, cudaStream_t st);
cudaError_t gradients(const na1d_head& h, const Shape& s, const Saved& sv, const float* coef, void* grad, int64_t pitch, int64_t v0, int64_t tiles, const void* w,
                      int64_t ldw, bool after, cudaStream_t st);
cudaError_t products(const na1d_head& h, const Shape& s, const Saved& sv, const void* grad, const Pieces& p, int64_t v0, int64_t cols, bool add, float* part_x,
                     float* part_w, const FinishArgs& f, const void* w, int64_t ldw, cudaStream_t st);
int logits_read_status();
int grad_read_status();

// The gradient of a row's own class as it is rounded to 16 bits, in one order of operations: `out` = row_factor(..)
__device__ __forceinline__ float row_factor(float up, float ix, float coef, bool norm) { return norm ? up * ix * coef : up * coef; }
__device__ __forceinline__ float own_gradient(float slope, float out, float iw, bool norm) { return norm ? (slope * out) * iw : slope * out; }

// element i of a tensor of one of the three types
__device__ __forceinline__ float load_any(const void* p, int type, long long i) {
    if (type == NA1D_FP32) return static_cast<const float*>(p)[i];
    const unsigned short raw = static_cast<const unsigned short*>(p)[i];
    return type == NA1D_BF16 ? Cvt<__nv_bfloat16>::from_bits(raw) : Cvt<__half>::from_bits(raw);
}
__device__ __forceinline__ void store_any(void* p, int type, long long i, float v) {
    if (type == NA1D_FP32) static_cast<float*>(p)[i] = v;
    else if (type == NA1D_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
// What rounding took from the gradient of row c's own class (the largest of the row, mostly): it is made good in fp32
template <typename E>
__device__ __forceinline__ float own_rest(const FinishArgs& a, int c) {
    const int v = a.target[c];
    const float f = own_gradient(a.slope[c], row_factor(a.up, a.norm ? a.ix[c] : 1.f, a.coef ? a.coef[c] : 1.f, a.norm), a.norm ? a.iw[v] : 1.f, a.norm);
    const float rest = f - (float)E(f);
    return fabsf(rest) < INFINITY ? rest : 0.f;
}
// what both gradients are multiplied with
__device__ __forceinline__ float common_factor(const FinishArgs& a, int counted) {
    const float f = a.factor / a.up;
    return a.reduction == NA1D_HEAD_NONE ? f * a.coef[a.Np] : f * (a.d_loss[0] / (a.reduction == NA1D_HEAD_MEAN ? (float)max(counted, 1) : 1.f));
}

}  // namespace head
}  // namespace na1d
