// The passes around the products of a head's losses: each reads its inputs once, a warp to a row or a class. prepare, combine and finish are 4 % of the kernels' time
// at 8192 x 1024 x 50000 (12, 16 and 43 us) and a sixth at 4099 x 192 x 17982 (9, 9 and 15 us); at 1024 x 256 x 200003 the weight's lengths take prepare 25 us
// where its 102 MB need 16, and in fp16, with the copy that its powers of two need, a pass takes 621 us instead of 585.
#include "na1d_head.cuh"

namespace na1d {
namespace head {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }   // -126 <= e <= 127
template <typename E> __device__ __forceinline__ float squares(const uint4& v, float ss) {
    float f[8];
    Cvt<E>::unpack(v, f);
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fmaf(f[k], f[k], ss);
    return ss;
}
// Inverse length of a row. `up`: 2^up times the row has a length of 2^lift to twice that, and `kept` is 1 / its length then
struct Length {
    float inverse, kept;
    int up;
};
// from an inverse length of the row times 2^-less
__device__ __forceinline__ Length length_from(float inverse, int less, int lift) {
    const int e = ((__float_as_int(inverse) >> 23) & 255) - 126;   // inverse = m 2^e, m from 1/2 to 1: the length is 2^-e to twice that
    return Length{inverse, inverse * power_of_two(-e - lift), e - less + lift};
}
// Squares outside fp32's range, or nearly: taken again of the row against its largest element. Rows of zeros, and ones shorter than 2^-126: all 0; a row with an
// infinity or NaN has no length: NaN. (A call of its own: inlined, it took 12 registers from the rows of ordinary length: 31.9 us instead of 26.1 at 1024 x 256 x 200003.)
template <typename E>
__device__ __noinline__ Length far_length(const void* src, int type, long long at, int D, int lift, int lane) {
    float most = 0.f, ss = 0.f;
    bool number = true;
    auto element = [&](int j) { return (float)E(load_any(src, type, at + j)); };   // (fp32 rows are rounded first)
    for (int j = lane; j < D; j += 32) {
        const float f = fabsf(element(j));
        number &= f < INFINITY;
        most = fmaxf(most, f);
    }
    most = warp_max(most);
    if (!__all_sync(0xffffffffu, number)) return Length{NAN, NAN, 0};
    if (most == 0.f) return Length{0.f, 0.f, 0};
    int less;
    frexpf(most, &less);
    for (int j = lane; j < D; j += 32) {
        const float f = ldexpf(element(j), -less);
        ss = fmaf(f, f, ss);
    }
    Length l = length_from(rsqrtf(warp_sum(ss)), less, lift);
    if (l.up - lift > 126) return Length{0.f, 0.f, 0};
    l.inverse = ldexpf(l.inverse, -less);
    return l;
}
__device__ __forceinline__ bool has_squares(float ss) { return ss >= 0x1p-100f && ss <= 0x1p100f; }
// of a row of D elements whose sum of squares is `ss`
template <typename E>
__device__ __forceinline__ Length length_of(float ss, const void* src, int type, long long at, int D, int lift, int lane) {
    return has_squares(ss) ? length_from(rsqrtf(ss), 0, lift) : far_length<E>(src, type, at, D, lift, lane);
}
// eight elements times 2^l.up (in two steps: it may be beyond fp32); zeros, or NaN, where the row has no direction
template <typename E> __device__ __forceinline__ uint4 kept_piece(const uint4& v, const Length& l) {
    const float p = power_of_two(l.up / 2), q = l.kept > 0.f ? power_of_two(l.up - l.up / 2) : l.kept;
    float f[8];
    Cvt<E>::unpack(v, f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = f[k] * p * q;
    return Cvt<E>::pack(f);
}
// One row of D elements to 16 bits at dst (Dp of them, zeros behind D; null: not stored), times a power of two where it is normalised.
// wide: rows start on 16 bytes, D is a multiple of 8.
template <typename E>
__device__ __forceinline__ Length copy_row(E* dst, const void* src, int type, long long at, int D, int Dp, bool wide, bool norm, int lift, int lane) {
    // eight elements to a lane at a time in every form, so that a row's length has the same bits in all of them
    auto piece = [&](int j) {
        if (wide && type != NA1D_FP32) return __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(src) + at) + j);
        float f[8];
        if (wide) {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(src) + at) + 2 * j;
            const float4 a = __ldg(p), b = __ldg(p + 1);
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = 8 * j + k < D ? load_any(src, type, at + 8 * j + k) : 0.f;
        }
        return Cvt<E>::pack(f);
    };
    const int n = Dp / 8;
    if (!norm) {
        for (int j = lane; j < n; j += 32) reinterpret_cast<uint4*>(dst)[j] = piece(j);
        return Length{1.f, 1.f, 0};
    }
    float ss = 0.f;
    uint4 last = make_uint4(0, 0, 0, 0);   // (all of a row of up to 256: it is loaded once)
    for (int j = lane; j < n; j += 32) {
        last = piece(j);
        ss = squares<E>(last, ss);
    }
    const Length l = length_of<E>(warp_sum(ss), src, type, at, D, lift, lane);
    if (dst)
        for (int j = lane; j < n; j += 32) reinterpret_cast<uint4*>(dst)[j] = kept_piece<E>(n <= 32 ? last : piece(j), l);
    return l;
}

// ---------------------------------------------------------------- a teacher's probabilities
struct TeacherArgs {
    const float* logits;
    const int64_t* index;
    float* q;
    int *out, *flags;          // flags (N): rows that count; null where the rows' kernel finds out by itself
    long long V;
    int N, k;
    float rt;                  // 1 / temperature
};
// Softmax over row i's entries, and the entries in the order of their classes, so that a tile of classes finds its own; a warp, `classes`: k ints of its
// own. An entry counts with a class in [0, V); one beyond (or a logit that is no number) makes the row's probabilities NaN.
__device__ __forceinline__ bool teacher_row(const TeacherArgs& a, int i, int* classes, int lane) {
    const size_t at = (size_t)i * a.k;
    float most = -INFINITY;
    bool bad = false;
    for (int j = lane; j < a.k; j += 32) {
        const int64_t v = a.index[at + j];
        classes[j] = v < 0 ? kNoClass : v < a.V ? (int)v : kNoClass - 1;
        if (v < 0) continue;
        const float t = a.logits[at + j] * a.rt;
        bad |= v >= a.V || t != t || t == INFINITY;
        most = fmaxf(most, t);
    }
    most = warp_max(most);
    bad = __any_sync(0xffffffffu, bad);
    auto weight = [&](int j) { return classes[j] != kNoClass && most > -INFINITY ? expf(a.logits[at + j] * a.rt - most) : 0.f; };
    float sum = 0.f;
    for (int j = lane; j < a.k; j += 32) sum += weight(j);
    sum = warp_sum(sum);
    const float r = 1.f / sum;
    __syncwarp();
    for (int j = lane; j < a.k; j += 32) {
        const int v = classes[j];
        int rank = 0;
#pragma unroll 4
        for (int o = 0; o < a.k; ++o) {
            const int u = classes[o];
            rank += u < v || (u == v && o < j);
        }
        a.q[at + rank] = v == kNoClass ? 0.f : bad ? NAN : most > -INFINITY ? weight(j) * r : 0.f;
        a.out[at + rank] = v < kNoClass - 1 ? v : kNoClass;
    }
    __syncwarp();
    return bad || most > -INFINITY;
}
__global__ void __launch_bounds__(kThreads) teacher_kernel(const __grid_constant__ TeacherArgs a) {
    extern __shared__ int classes_s[];
    wait_for_predecessor();
    const int i = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= a.N) return;
    const bool on = teacher_row(a, i, classes_s + (threadIdx.x >> 5) * a.k, lane);
    if (lane == 0) a.flags[i] = on;
}

// ---------------------------------------------------------------- rows that count, side by side; the weight
struct PrepareArgs {
    const void *x, *w;
    const int64_t* labels;
    float* loss;               // (N) zeros for rows that do not count; null where the loss is one number
    Words* words;
    int *place, *row, *target, *own_count;
    float *ix, *iw, *x_up, *w_up;
    void *out, *w_out;         // w_out: null where the weight stays where it is
    long long x_stride, w_stride, ignore;
    int N, Np, V, D, Dp, x_type, w_type, per_block, row_blocks, lift;
    bool wide, w_wide, norm;
    TeacherArgs t;
    bool top;
};
// whether row i counts: by its label, or by an entry with a class and a logit above minus infinity (as teacher_row finds)
__device__ __forceinline__ bool row_counts(const PrepareArgs& a, int i) {
    if (!a.top) return a.labels[i] != a.ignore;
    if (a.t.flags) return a.t.flags[i] != 0;
    for (int j = 0; j < a.t.k; ++j) {
        const size_t at = (size_t)i * a.t.k + j;
        if (a.t.index[at] >= 0 && (a.t.index[at] >= a.t.V || !(a.t.logits[at] * a.t.rt <= -INFINITY))) return true;
    }
    return false;
}
// Blocks below row_blocks take `per_block` rows each. Such a block counts the rows before its own itself: labels are few bytes, and no block waits for
// another. The others take the weight: a copy in 16 bits where the products cannot read it as it is, and its rows' lengths.
template <typename E>
__global__ void __launch_bounds__(kThreads) prepare_kernel(const __grid_constant__ PrepareArgs a) {
    __shared__ int sums[kWarps], places[kThreads], base_s;
    extern __shared__ int classes_s[];
    wait_for_predecessor();
    if (blockIdx.x == 0 && threadIdx.x == 0) a.words->ticket = 0;
    for (int v = blockIdx.x * kThreads + threadIdx.x; v < a.V; v += gridDim.x * kThreads) a.own_count[v] = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if ((int)blockIdx.x >= a.row_blocks) {
        const int step = (gridDim.x - a.row_blocks) * kWarps;
        int v = (blockIdx.x - a.row_blocks) * kWarps + warp;
        if (!a.w_out && a.D <= 256) {   // lengths alone: four rows' loads at a time
            for (; v + 3 * step < a.V; v += 4 * step) {
                uint4 r[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    r[i] = lane < a.D / 8 ? __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(a.w) + (v + i * step) * a.w_stride) + lane) : make_uint4(0, 0, 0, 0);
                float ss[4];
                bool near = true;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ss[i] = warp_sum(squares<E>(r[i], 0.f));
                    near &= has_squares(ss[i]);
                }
                if (!near) break;   // (one by one from here on)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (lane == 0) a.iw[v + i * step] = rsqrtf(ss[i]);
            }
        }
        for (; v < a.V; v += step) {
            const Length l = copy_row<E>(a.w_out ? static_cast<E*>(a.w_out) + (size_t)v * a.Dp : nullptr, a.w, a.w_type, v * a.w_stride, a.D, a.Dp, a.w_wide, a.norm, a.lift, lane);
            if (a.norm && lane == 0) {
                a.iw[v] = a.w_up ? l.kept : l.inverse;
                if (a.w_up) a.w_up[v] = ldexpf(1.f, l.up);
            }
        }
        return;
    }
    const int r0 = min(a.N, (int)blockIdx.x * a.per_block), r1 = min(a.N, r0 + a.per_block);
    int before = 0;
    for (int i = threadIdx.x; i < r0; i += kThreads) before += row_counts(a, i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (lane == 0) sums[warp] = before;
    __syncthreads();
    if (threadIdx.x == 0) {
        int s = 0;
        for (int w = 0; w < kWarps; ++w) s += sums[w];
        base_s = s;
    }
    __syncthreads();
    int base = base_s;
    E* out = static_cast<E*>(a.out);
    for (int c0 = r0; c0 < r1; c0 += kThreads) {
        const int i = c0 + threadIdx.x;
        const bool in = i < r1, on = in && row_counts(a, i);
        const unsigned mask = __ballot_sync(0xffffffffu, on);
        __syncthreads();
        if (lane == 0) sums[warp] = __popc(mask);
        __syncthreads();
        int c = base + __popc(mask & ((1u << lane) - 1));
        for (int w = 0; w < warp; ++w) c += sums[w];
        int total = 0;
        for (int w = 0; w < kWarps; ++w) total += sums[w];
        if (in) {
            // a row that does not count: the free places from the end are filled with zeros in the order of such rows
            places[threadIdx.x] = on ? c : -1 - (a.N - 1 - (i - c));
            a.place[i] = on ? c : kIgnored;
            if (on) {
                a.row[c] = i;
                if (!a.top) {
                    const int64_t v = a.labels[i];
                    a.target[c] = v >= 0 && v < a.V ? (int)v : kBad;
                }
            } else if (a.loss) a.loss[i] = 0.f;
        }
        __syncthreads();
        const int n = min(kThreads, r1 - c0);
        for (int j = warp; j < n; j += kWarps) {
            const int p = places[j];
            if (p >= 0) {
                const Length l = copy_row<E>(out + (size_t)p * a.Dp, a.x, a.x_type, (c0 + j) * a.x_stride, a.D, a.Dp, a.wide, a.norm, a.lift, lane);
                if (a.norm && lane == 0) {
                    a.ix[p] = l.kept;
                    a.x_up[p] = ldexpf(1.f, l.up);
                }
                if (a.top && !a.t.flags) teacher_row(a.t, c0 + j, classes_s + warp * a.t.k, lane);
            } else {
                for (int e = lane; e < a.Dp / 8; e += 32) reinterpret_cast<uint4*>(out + (size_t)(-1 - p) * a.Dp)[e] = make_uint4(0, 0, 0, 0);
            }
        }
        base += total;
        __syncthreads();
    }
    const long long pad = (long long)(a.Np - a.N) * (a.Dp / 8);   // 16-byte pieces behind the last row
    for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < pad; e += (long long)a.row_blocks * kThreads)
        reinterpret_cast<uint4*>(out + (size_t)a.N * a.Dp)[e] = make_uint4(0, 0, 0, 0);
    if (r0 < a.N && r1 == a.N && threadIdx.x == 0) a.words->counted = base;
}

// ---------------------------------------------------------------- single logits
// x (a 16-bit row of Dp, zeros behind D) times a row of the weight: one warp, every lane gets the sum
template <typename E>
__device__ __forceinline__ float dot_row(const E* x, const E* w, int D8, int lane) {
    float s = 0.f;
    for (int j = lane; j < D8; j += 32) {
        float a[8], b[8];
        Cvt<E>::unpack(__ldg(reinterpret_cast<const uint4*>(x) + j), a);
        Cvt<E>::unpack(__ldg(reinterpret_cast<const uint4*>(w) + j), b);
#pragma unroll
        for (int k = 0; k < 8; ++k) s = fmaf(a[k], b[k], s);
    }
    return warp_sum(s);
}
struct Products {
    const void *x, *w;
    const float *ix, *iw;
    long long ldw;
    int Dp;
    float cs;
    bool norm;
};
// the logit of row c and class v as a product or a cosine
template <typename E>
__device__ __forceinline__ float logit_of(const Products& p, int c, int v, int lane) {
    const float s = dot_row(static_cast<const E*>(p.x) + (size_t)c * p.Dp, static_cast<const E*>(p.w) + (size_t)v * p.ldw, p.Dp / 8, lane);
    return p.norm ? s * p.ix[c] * p.iw[v] : s;
}
// ---------------------------------------------------------------- log-sum-exp and loss
struct CombineArgs {
    const float2* part;
    Words* words;
    const int *row, *index;
    int *target, *own_count, *own;
    const float *q, *entry;
    float *gradient, *lse2, *slope, *block_sums, *loss;
    int parts, k, reduction;
    float cos_m, sin_m, tau2;
    bool margin;
    Products p;
};
// A warp takes a row: its partial sums, then what belongs to the target or the teacher's entries. The last block to finish adds up the
// blocks' sums in their order.
template <typename E>
__global__ void __launch_bounds__(kThreads) combine_kernel(const __grid_constant__ CombineArgs a) {
    __shared__ float loss_s[kWarps];
    __shared__ int last;
    wait_for_predecessor();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, counted = a.words->counted, c = blockIdx.x * kWarps + warp;
    auto own_row = [&](int v, int c) {   // (in whatever order: they are sorted before they are added up)
        const int n = atomicAdd(a.own_count + v, 1);
        if (n < kOwn) a.own[(size_t)v * kOwn + n] = c;
    };
    float loss = 0.f;
    if (c < counted) {
        float m = -INFINITY, s = 0.f;
        const float2* part = a.part + (size_t)c * a.parts;
        int p = lane;
        for (; p + 96 < a.parts; p += 128) {   // four loads at a time
            float2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = part[p + 32 * i];
            const float to = fmaxf(fmaxf(fmaxf(v[0].x, v[1].x), fmaxf(v[2].x, v[3].x)), m), by = to > -INFINITY ? to : 0.f;
            s *= exp2_fast(m - by);
#pragma unroll
            for (int i = 0; i < 4; ++i) s = fmaf(v[i].y, exp2_fast(v[i].x - by), s);
            m = to;
        }
        for (; p < a.parts; p += 32) {
            const float2 v = part[p];
            const float to = fmaxf(m, v.x), by = to > -INFINITY ? to : 0.f;
            s = s * exp2_fast(m - by) + v.y * exp2_fast(v.x - by);
            m = to;
        }
        const float top = warp_max(m), by = top > -INFINITY ? top : 0.f;
        s = warp_sum(s * exp2_fast(m - by));
        m = top;
        if (a.k == 0) {
            const int target = a.target[c];
            if (target < 0) {
                loss = NAN;
                if (lane == 0) a.lse2[c] = NAN;
            } else {
                float z = logit_of<E>(a.p, c, target, lane), slope = 1.f;
                if (a.margin) {   // cos(angle + m) and its derivative
                    const float sine2 = fmaf(-z, z, 1.f), sine = sqrtf(fmaxf(sine2, kSineFloor));
                    slope = a.cos_m + (sine2 > kSineFloor ? z / sine : 0.f) * a.sin_m;
                    z = z * a.cos_m - sine * a.sin_m;
                }
                z *= a.p.cs;
                // the other classes' sum against the target's term: a small loss is this ratio, with its relative accuracy
                const float above = m - z, ratio = s * exp2f(above);
                const bool small = ratio < 1e30f || ratio != ratio;
                loss = small ? log1pf(ratio) : fmaf(above, kLn2, logf(s));
                if (lane == 0) {
                    a.lse2[c] = small ? z + log2f(1.f + ratio) : m + log2f(s);
                    a.slope[c] = -(small ? ratio / (1.f + ratio) : 1.f) * slope;
                    own_row(target, c);
                }
            }
        } else {
            const size_t at = (size_t)a.row[c] * a.k;
            // everything against the largest entry, near which the sum's logarithm is small: log p = z - top - log(sum / 2^top)
            float top = -INFINITY;
            for (int e = lane; e < a.k; e += 32)
                if (a.index[at + e] != kNoClass) top = fmaxf(top, a.entry[at + e]);
            top = warp_max(top);
            if (!(top > -INFINITY)) top = m;
            const float over = exp2f(m - top) * s < 1e30f ? log2f(exp2f(m - top) * s) : (m - top) + log2f(s), lse2 = top + over;
            // (a class that comes twice has its entries side by side: all of them take the gradient of the class)
            float best = -1.f, own = 0.f;
            int own_class = kBad;
            for (int e = lane; e < a.k; e += 32) {
                const int v = a.index[at + e];
                const float q = a.q[at + e];
                if (q != q) loss = q;
                if (v == kNoClass) continue;
                const float z2 = (a.entry[at + e] - top) - over;
                if (q > 0.f) loss += q * (logf(q) - z2 * kLn2);
                float all = q;
                for (int o = e - 1; o >= 0 && a.index[at + o] == v; --o) all += a.q[at + o];
                for (int o = e + 1; o < a.k && a.index[at + o] == v; ++o) all += a.q[at + o];
                const float g = exp2_fast(z2) - all;
                if (fabsf(g) > best) { best = fabsf(g); own = g; own_class = v; }
                a.gradient[at + e] = g;
            }
            for (int o = 16; o > 0; o >>= 1) {   // the largest of all, the lowest class of equals
                const float b = __shfl_xor_sync(0xffffffffu, best, o), g = __shfl_xor_sync(0xffffffffu, own, o);
                const int v = __shfl_xor_sync(0xffffffffu, own_class, o);
                if (b > best || (b == best && v < own_class)) { best = b; own = g; own_class = v; }
            }
            if (lane == 0) {
                a.target[c] = own_class;
                a.slope[c] = own;
                if (own_class >= 0) own_row(own_class, c);
            }
            loss = warp_sum(loss) * a.tau2;
            if (lane == 0) a.lse2[c] = loss == loss ? lse2 : NAN;   // (an entry that is no class: nothing of the row counts)
        }
        if (a.reduction == NA1D_HEAD_NONE && lane == 0) a.loss[a.row[c]] = loss;
    }
    if (a.reduction == NA1D_HEAD_NONE) return;
    if (lane == 0) loss_s[warp] = loss;
    __syncthreads();
    if (warp == 0) {
        const float s = warp_sum(lane < kWarps ? loss_s[lane] : 0.f);
        if (lane == 0) {
            a.block_sums[blockIdx.x] = s;
            __threadfence();
            last = atomicAdd(&a.words->ticket, 1) == (int)gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    float s = 0.f;
    for (int b = threadIdx.x; b < (int)gridDim.x; b += kThreads) s += __ldcg(a.block_sums + b);
    s = warp_sum(s);
    if (lane == 0) loss_s[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.f;
        for (int w = 0; w < kWarps; ++w) s += loss_s[w];
        *a.loss = a.reduction == NA1D_HEAD_MEAN ? s / (float)max(counted, 1) : s;
    }
}

// ---------------------------------------------------------------- backward
// factors of single rows' losses, side by side as the rows; fp16: relative to the largest finite one (of 2^-120 at least: its inverse is a number), which follows
// them. A probability times its row's factor keeps all digits down to 2^-28 of the largest factor (cosines: 2^-19 at a margin of 0.2).
__global__ void __launch_bounds__(1024) coefficients_kernel(const float* __restrict__ d_loss, const Words* __restrict__ words, const int* __restrict__ row, long long Np,
                                                            bool relative, float* __restrict__ coef) {
    __shared__ float most_s[32];
    wait_for_predecessor();
    const int counted = words->counted;
    float most = 0.f;
    if (relative) {
        for (int c = threadIdx.x; c < counted; c += 1024) {
            const float f = fabsf(d_loss[row[c]]);
            if (f < INFINITY) most = fmaxf(most, f);
        }
        most = warp_max(most);
        if ((threadIdx.x & 31) == 0) most_s[threadIdx.x >> 5] = most;
        __syncthreads();
        most = warp_max(most_s[threadIdx.x & 31]);
    }
    most = most > 0.f ? fmaxf(most, 0x1p-120f) : 1.f;
    const float r = 1.f / most;
    for (int c = threadIdx.x; c < counted; c += 1024) coef[c] = relative ? d_loss[row[c]] * r : d_loss[row[c]];
    if (threadIdx.x == 0) coef[Np] = most;
}
template <typename E>
__device__ __forceinline__ void unpack_row(const E* row, int j, float* f) { Cvt<E>::unpack(__ldg(reinterpret_cast<const uint4*>(row) + j), f); }
// One row of a gradient: the splits' sum and what rounding took (`n` rows of the other operand times `rest`: `other(i)`), without its part along the row it
// belongs to where that is normalised, times the common factor and the power of two that the row is kept with.
template <typename E, typename Other>
__device__ __forceinline__ void finish_row(void* out, int type, long long at, const float* part, long long split, int splits, const E* own, float inverse, float f, float back,
                                           int n, const float* rest, Other other, bool norm, int D, int Dp, int lane) {
    auto sum = [&](int j, float* s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = 0.f;
        for (int k = 0; k < splits; ++k) {
            const float4* p = reinterpret_cast<const float4*>(part + k * split) + 2 * j;
            const float4 u = p[0], v = p[1];
            s[0] += u.x; s[1] += u.y; s[2] += u.z; s[3] += u.w; s[4] += v.x; s[5] += v.y; s[6] += v.z; s[7] += v.w;
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            if (i >= n) break;
            float x[8];
            unpack_row(other(i), j, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = fmaf(rest[i], x[e], s[e]);
        }
    };
    float along = 0.f, kept[8];   // (rows of up to 256: a lane has eight columns, which are added up once)
    if (norm) {
        for (int j = lane; j < Dp / 8; j += 32) {
            float x[8], s[8];
            unpack_row(own, j, x);
            sum(j, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) kept[e] = s[e];
#pragma unroll
            for (int e = 0; e < 8; ++e) along = fmaf(x[e], 8 * j + e < D ? s[e] : 0.f, along);
        }
        along = warp_sum(along) * inverse;   // (a length of 1e-20 has no square in fp32)
    }
    const bool wide = D % 8 == 0 && type != NA1D_FP32;
    for (int j = lane; j < Dp / 8; j += 32) {
        float s[8];
        if (norm && Dp <= 256) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = kept[e];
        } else {
            sum(j, s);
        }
        if (norm) {
            float x[8];
            unpack_row(own, j, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = fmaf(-along, x[e] * inverse, s[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = s[e] * f * back;
        if (wide) reinterpret_cast<uint4*>(static_cast<E*>(out) + at)[j] = Cvt<E>::pack(s);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (8 * j + e < D) store_any(out, type, at + 8 * j + e, s[e]);
    }
}
template <typename E>
__global__ void __launch_bounds__(kThreads, 3) finish_kernel(const __grid_constant__ FinishArgs a) {
    wait_for_predecessor();
    const int lane = threadIdx.x & 31, counted = a.words->counted, first = a.cols + (a.dx ? a.N : 0), n = first + (a.own_classes ? a.N : 0);
    const float f = common_factor(a, counted);
    const E *x = static_cast<const E*>(a.x), *w = static_cast<const E*>(a.w);
    auto class_row = [&](int v, const float* part, long long split, int splits) {
        float rest[kOwn];
        int rows_in_order[kOwn];
        const int count = a.own_count[v], rows = count <= kOwn ? count : 0;   // (of many rows the roundings average out)
        if (rows) {
            const int mine = lane < rows ? a.own[(size_t)v * kOwn + lane] : kNoClass;
            int rank = 0;
#pragma unroll
            for (int o = 0; o < kOwn; ++o) rank += __shfl_sync(0xffffffffu, mine, o) < mine;
#pragma unroll
            for (int o = 0; o < kOwn; ++o) {
                const unsigned who = __ballot_sync(0xffffffffu, lane < rows && rank == o);
                rows_in_order[o] = __shfl_sync(0xffffffffu, mine, who ? __ffs(who) - 1 : 0);
                rest[o] = o < rows ? own_rest<E>(a, rows_in_order[o]) : 0.f;
            }
        }
        finish_row<E>(a.dw, a.w_type, (long long)v * a.D, part, split, splits, w + (size_t)v * a.ldw, a.norm ? a.iw[v] : 1.f, f, a.w_up ? a.w_up[v] : 1.f, rows, rest,
                      [&](int o) { return x + (size_t)rows_in_order[o] * a.Dp; }, a.norm, a.D, a.Dp, lane);
    };
    for (int i = blockIdx.x * kWarps + (threadIdx.x >> 5); i < n; i += gridDim.x * kWarps) {
        if (i < a.cols) {
            class_row(a.v0 + i, a.part_w + (size_t)i * a.Dp, a.piece_rows * a.Dp, a.splits_w);
            continue;
        }
        if (i >= first) {   // the class of a row, if it is the one that has the class's sums
            const int c = a.place[i - first], v = c < 0 ? c : a.target[c];
            if (v >= 0 && a.own_count[v] <= kOwn && a.own[(size_t)v * kOwn] == c) class_row(v, a.part_w + (size_t)c * a.Dp, 0, 1);
            continue;
        }
        const int r = i - a.cols, c = a.place[r];
        if (c < 0) {
            for (int j = lane; j < a.D; j += 32) store_any(a.dx, a.x_type, (long long)r * a.D + j, 0.f);
            continue;
        }
        const int v = a.target[c];
        const float rest[kOwn] = {v >= 0 ? own_rest<E>(a, c) : 0.f};
        finish_row<E>(a.dx, a.x_type, (long long)r * a.D, a.part_x + (size_t)c * a.Dp, a.Np * a.Dp, a.splits_x, x + (size_t)c * a.Dp, a.norm ? a.ix[c] : 1.f, f,
                      a.norm ? a.x_up[c] : 1.f, v >= 0 ? 1 : 0, rest, [&](int) { return w + (size_t)v * a.ldw; }, a.norm, a.D, a.Dp, lane);
    }
}

int blocks_for(int64_t warps, int64_t most = 148 * 8) {
    const int64_t b = (warps + kWarps - 1) / kWarps;
    return (int)(b < 1 ? 1 : b < most ? b : most);
}
Products products_of(const Shape& s, const Saved& sv, const void* w, int64_t ldw) {
    return Products{sv.x, w, sv.ix, sv.iw, ldw, (int)s.Dp, s.cs, s.norm};
}

}  // namespace

namespace {
TeacherArgs teacher_args(const na1d_head& h, const Shape& s, const Saved& sv, int* flags) {
    return TeacherArgs{h.teacher_logits, h.teacher_index, sv.q, sv.index, flags, (long long)s.V, (int)s.N, (int)s.k, 1.f / h.temperature};
}
bool whole_pieces(const void* p, int64_t stride, int64_t D) { return D % 8 == 0 && stride % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
}  // namespace
cudaError_t prepare(const na1d_head& h, const Shape& s, const Saved& sv, int* flags, float* loss, cudaStream_t st) {
    PrepareArgs a = {};
    a.x = h.x; a.w = h.weight; a.labels = h.labels; a.top = s.k > 0;
    a.loss = h.reduction == NA1D_HEAD_NONE ? loss : nullptr;
    a.words = sv.words; a.place = sv.place; a.row = sv.row; a.target = sv.target; a.own_count = sv.own_count; a.ix = sv.ix; a.iw = sv.iw; a.x_up = sv.x_up; a.w_up = sv.w_up;
    a.out = sv.x; a.w_out = s.copy_w ? sv.w : nullptr;
    a.x_stride = h.x_stride; a.w_stride = h.weight_stride; a.ignore = h.ignore_index;
    a.N = (int)s.N; a.Np = (int)s.Np; a.V = (int)s.V; a.D = (int)s.D; a.Dp = (int)s.Dp; a.x_type = h.x_type; a.w_type = h.weight_type;
    a.norm = s.norm; a.lift = lift(h.dtype == NA1D_FP16);
    a.wide = whole_pieces(h.x, h.x_stride, s.D);
    a.w_wide = whole_pieces(h.weight, h.weight_stride, s.D);
    a.per_block = (int)round_up((s.N + 295) / 296, kWarps);
    a.row_blocks = (int)((s.N + a.per_block - 1) / a.per_block);
    a.row_blocks = a.row_blocks < 16 ? 16 : a.row_blocks;   // (a few rows: the others fill up the tile with zeros)
    // Few rows find out by themselves which of them have a teacher (a row's first entry tells, mostly): a launch less. Many would look at all rows
    // before theirs once for each block (a pass in a graph: 85 us against 75 with the launch at 1003 rows of up to 20 entries,
    // 49.8 against 49.2 at 256 of 32, 45.1 either way at 16 of 8).
    const bool early = s.N * s.k > 8192;
    size_t smem = 0;
    if (s.k) {
        a.t = teacher_args(h, s, sv, early ? flags : nullptr);
        smem = (size_t)kWarps * s.k * 4;
        if (early)
            if (cudaError_t e = launch(teacher_kernel, (s.N + kWarps - 1) / kWarps, kThreads, smem, st, false, a.t)) return e;
    }
    const int64_t blocks = a.row_blocks + (s.copy_w || s.norm ? blocks_for(s.V) : 0);
    return launch(h.dtype == NA1D_BF16 ? prepare_kernel<__nv_bfloat16> : prepare_kernel<__half>, blocks, kThreads, early ? 0 : smem, st, early, a);
}
cudaError_t combine(const na1d_head& h, const Shape& s, const Saved& sv, const float2* part, float* block_sums, float* loss, const void* w, int64_t ldw,
                    cudaStream_t st) {
    CombineArgs a = {};
    a.part = part; a.words = sv.words; a.row = sv.row; a.target = sv.target; a.own_count = sv.own_count; a.own = sv.own; a.index = sv.index; a.q = sv.q;
    a.entry = a.gradient = sv.entry; a.lse2 = sv.lse2; a.slope = sv.slope; a.block_sums = block_sums; a.loss = loss;
    a.parts = (int)s.parts; a.k = (int)s.k; a.reduction = h.reduction;
    a.margin = s.norm && h.margin != 0.f;
    a.cos_m = (float)cos((double)h.margin); a.sin_m = (float)sin((double)h.margin);
    a.tau2 = h.temperature * h.temperature;
    a.p = products_of(s, sv, w, ldw);
    const unsigned blocks = (unsigned)((s.N + kWarps - 1) / kWarps);
    return launch(h.dtype == NA1D_BF16 ? combine_kernel<__nv_bfloat16> : combine_kernel<__half>, blocks, kThreads, 0, st, true, a);
}
cudaError_t coefficients(const na1d_head& h, const Shape& s, const Saved& sv, const float* d_loss, float* coef, cudaStream_t st) {
    return launch(coefficients_kernel, 1, 1024, 0, st, false, d_loss, sv.words, sv.row, s.Np, h.dtype == NA1D_FP16, coef);
}
FinishArgs finish_args(const na1d_head& h, const Shape& s, const Saved& sv, void* dx, void* dw, const float* part_x, const float* part_w, const float* d_loss,
                       const float* coef, const Pieces& p, int64_t v0, int64_t cols, const void* w, int64_t ldw) {
    FinishArgs a = {};
    a.dx = dx; a.dw = dw; a.part_x = part_x; a.part_w = part_w; a.d_loss = d_loss; a.coef = coef;
    a.x = sv.x; a.w = w; a.ix = sv.ix; a.iw = sv.iw; a.x_up = sv.x_up; a.w_up = sv.w_up; a.place = sv.place; a.words = sv.words;
    a.slope = sv.slope; a.target = sv.target; a.own_count = sv.own_count; a.own = sv.own;
    a.Np = s.Np; a.piece_rows = p.pitch; a.ldw = ldw;
    a.N = (int)s.N; a.D = (int)s.D; a.Dp = (int)s.Dp; a.cols = (int)cols; a.v0 = (int)v0; a.splits_x = p.splits_x; a.splits_w = p.splits_w;
    a.x_type = h.x_type; a.w_type = h.weight_type; a.reduction = h.reduction; a.norm = s.norm; a.up = s.up;
    a.factor = s.k ? h.scale * h.temperature : h.scale;
    return a;
}
cudaError_t finish(const na1d_head& h, const FinishArgs& a, cudaStream_t st) {
    const int blocks = blocks_for((int64_t)(a.dx ? a.N : 0) + (a.own_classes ? a.N : 0) + a.cols);
    return launch(h.dtype == NA1D_BF16 ? finish_kernel<__nv_bfloat16> : finish_kernel<__half>, blocks, kThreads, 0, st, true, a);
}

}  // namespace head
}  // namespace na1d
