// Rows of up to 256 channels with labels: the gradient of the logits and the weight's gradient in one kernel, so that the former is read only once
// (by the product for the rows), not twice.
//
// A pair of CTAs takes 256 classes, whose rows of the weight stay in shared memory, and walks over the rows, 128 at a time:
//   S^T = w x^T      (256 classes x 128 rows) into tensor memory: a lane is a class
//   H^T              2^(z - lse) less the targets, in 16 bits: back to tensor memory as the left operand of the next product, and out for the rows'
//   dw += H^T x      (256 classes x D), the rows' tile once more, now contracted across its rows
// A class's factors are its lane's own; a row's come from 256 bytes of shared memory that a warp fills for itself. The sum of H s over the rows is the
// part of dw along w, which the way back through the normalisation takes out. Sixteen warps turn S^T into H^T and empty the accumulators when the
// rows are through; products are issued one step ahead of them.
// Bound: the arithmetic of H^T (about 2600 SM cycles a step, two products 1536 at 192 channels, 48 KB from L2).
#include "na1d_head.cuh"
#include "na1d_mlp.cuh"

namespace na1d {
namespace head {
namespace {

__device__ int g_head_status = 0;

constexpr int kEpilogue = 16;                        // warps 0-15: 32 classes (tensor-memory lanes) and a quarter of a step's rows each
constexpr int kThreads = (kEpilogue + 4) * 32;       // 16: loads, 17: MMA issue, 18: tensor memory
constexpr int kRows = 128;                           // rows of a step
constexpr int kHalf = 128;                           // classes of a CTA
constexpr int kClassBox = 64 * kHalf * 2;            // 64 channels of a CTA's classes
constexpr int kFirstBox = 64 * (kRows / 2) * 2;      // 64 channels of a CTA's half of a step's rows
constexpr int kSecondBox = 64 * kRows * 2;           // 64 channels of a step's rows
constexpr int kSlots = 2;
// Tensor-memory columns: dw (256), S^T (128), two H^T of 16 bits (64 each). As everywhere, a product writes columns only behind a barrier that covers
// whatever may still read them: S^T of step j + 1 waits until all warps have read S^T of step j, and H^T of step j lies where that of step j - 2 was, whose product
// is among those that the signal for S^T of step j waits for.
constexpr uint32_t kAcc = 0, kLogits = 256, kOperand = 384, kOperandCols = 64;

struct Barriers {
    uint64_t w_full, w_free, first_full[kSlots], first_free[kSlots], second_full[kSlots], second_free[kSlots], s_full, s_free, h_ready[2], acc_full, acc_free, along;
    uint32_t tmem;
    int abort;
};
struct Maps { CUtensorMap w, first, second; };
struct Args {
    const Words* words;
    const int* target;
    const float *ix, *iw, *lse2, *slope, *coef;
    void* grad;                // H^T: (classes of the piece, pitch), or null
    long long pitch, Dq;
    float* part_w;             // sums of classes that are rows' own, at such a row
    int v0, cols, tiles, D, boxes, width, first_bytes, second_boxes;
    float cs;
    bool fp16;
    FinishArgs f;
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// sixteen columns of a class's gradient as they are wanted
template <typename E>
__device__ __forceinline__ void store_columns(const FinishArgs& f, int v, int col, const float* d) {
    const long long at = (long long)v * f.D + col;
    if (f.w_type != NA1D_FP32 && f.D % 16 == 0) {
        if (col < f.D) {
            const uint4 a = Cvt<E>::pack(d), b = Cvt<E>::pack(d + 8);
            const uint32_t s[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            store_sector(static_cast<E*>(f.dw) + at, s);
        }
    } else if (f.D % 8 == 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (col + 8 * j < f.D) {
                if (f.w_type == NA1D_FP32) store_sector(static_cast<float*>(f.dw) + at + 8 * j, reinterpret_cast<const uint32_t*>(d + 8 * j));
                else *reinterpret_cast<uint4*>(static_cast<E*>(f.dw) + at + 8 * j) = Cvt<E>::pack(d + 8 * j);
            }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (col + j < f.D) store_any(f.dw, f.w_type, at + j, d[j]);
    }
}

template <typename E, bool NORM>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) both_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args g) {
    extern __shared__ uint8_t raw[];
    uint8_t* classes = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* firsts = classes + g.boxes * kClassBox;
    uint8_t* seconds = firsts + kSlots * g.first_bytes;
    __shared__ Barriers bar;
    __shared__ float4 factors_s[kEpilogue][kRows / 8];     // of a warp's 32 rows, pairs of (slope, shift) of the exponent
    __shared__ float along_s[2][4][kHalf];
    const int warp = ptx::warp_index(), lane = threadIdx.x & 31;
    const uint32_t rank = pair::cta_rank();
    const int pair_index = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    volatile int* abort_flag = &bar.abort;
#define NA1D_BOTH_FAIL(code) { atomicExch(&g_head_status, code); *abort_flag = 1; ok = false; break; }

    if (warp == kEpilogue) {
        if (lane < kSlots) {
            ptx::mbar_init(&bar.first_full[lane], 1); ptx::mbar_init(&bar.first_free[lane], 1);
            ptx::mbar_init(&bar.second_full[lane], 1); ptx::mbar_init(&bar.second_free[lane], 1);
            ptx::mbar_init(&bar.h_ready[lane], 2 * kEpilogue);
        } else if (lane == kSlots) {
            ptx::mbar_init(&bar.w_full, 1); ptx::mbar_init(&bar.w_free, 1);
            ptx::mbar_init(&bar.s_full, 1); ptx::mbar_init(&bar.s_free, 2 * kEpilogue);
            ptx::mbar_init(&bar.acc_full, 1); ptx::mbar_init(&bar.acc_free, 2 * kEpilogue);
            ptx::mbar_init(&bar.along, kEpilogue);
            bar.abort = 0;
        } else if (lane < kSlots + 4) {
            ptx::prefetch_tensormap(lane == kSlots + 1 ? &maps.w : lane == kSlots + 2 ? &maps.first : &maps.second);
        }
        ptx::fence_mbar_init();
    }
    if (warp == kEpilogue + 2) { pair::tmem_alloc(&bar.tmem, 512); pair::tmem_relinquish(); }
    ptx::tc_fence_before_sync();
    __syncthreads();
    pair::cluster_sync();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = bar.tmem;
    wait_for_predecessor();
    const int counted = g.words->counted, steps = (counted + kRows - 1) / kRows;
    bool ok = true;

    if (warp < kEpilogue) {
        const int q = warp & 3, part = warp >> 2, row = q * 32 + lane;   // the class is lane `row` of the CTA's; rows 32 part .. + 31 of a step
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const uint32_t s_free = pair::in_leader(&bar.s_free), h_ready0 = pair::in_leader(&bar.h_ready[0]), h_ready1 = pair::in_leader(&bar.h_ready[1]);
        const uint32_t s = tmem + lanes + kLogits + part * 32;
        const float up = gradient_scale(g.words, g.fp16, NORM), factor = common_factor(g.f, counted, up);
        float4* factors = factors_s[warp];
        // what belongs to this lane's row of a step: asked for while the step before is worked on
        struct Row {
            bool live;
            int target;
            float ix, lse2, coef, slope;
        };
        auto row_of = [&](int t) {
            const int c = t * kRows + part * 32 + lane;
            Row r = {c < counted, kIgnored, 1.f, 0.f, 1.f, 0.f};
            if (r.live) {
                r.target = g.target[c];
                r.lse2 = g.lse2[c];
                r.slope = g.slope[c];
                if (NORM) r.ix = g.ix[c];
                if (g.coef) r.coef = g.coef[c];
            }
            return r;
        };
        Row next_row = row_of(0);
        int j = 0, items = 0;
        for (int i = pair_index; ok && i < g.tiles; i += pairs, ++items) {
            const int local = i * kTile + (int)rank * kHalf + row, v = g.v0 + local, v_warp = v - lane;
            const bool live = local < g.cols, all_live = local - lane + 32 <= g.cols;
            const float iw = NORM && live ? g.iw[v] : 0.f;
            // a class that is some rows' own (and not that of many, whose roundings average out) gets what rounding took in the last step
            const int own_rows = live ? g.f.own_count[v] : 0;
            const bool whole = own_rows > 0 && own_rows <= kOwn;
            float* dst = whole ? g.part_w + (size_t)g.f.own[(size_t)v * kOwn] * g.Dq : nullptr;
            float along = 0.f;
            for (int t = 0; t < steps; ++t, ++j) {
                // this lane's row: what the exponent is made of, and whether its target is among this warp's classes
                const Row r = next_row;
                next_row = row_of(t + 1 < steps ? t + 1 : 0);
                float a = 0.f, b = -INFINITY, at_target = 0.f;
                int hit = -1;
                bool negative = false;
                if (r.live) {
                    const float out = row_factor(up, r.ix, r.coef, NORM);
                    a = r.ix > 0.f ? g.cs * r.ix : g.cs;
                    b = log2f(fabsf(out)) - r.lse2;
                    negative = out < 0.f;
                    hit = r.target - v_warp;
                    if ((unsigned)hit < 32u) at_target = own_gradient(r.slope, out, NORM ? g.iw[v_warp + hit] : 1.f, NORM);
                    else hit = -1;
                }
                const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), negatives = __ballot_sync(0xffffffffu, negative);
                __syncwarp();
                reinterpret_cast<float2*>(factors)[lane] = make_float2(a, b);
                __syncwarp();
                if (!ptx::mbar_wait(&bar.s_full, j & 1) || *abort_flag) NA1D_BOTH_FAIL(1)
                ptx::tc_fence_after_sync();
                float d[32];
                pair::tmem_ld32(s, d);
                ptx::tmem_ld_wait();
                ptx::tc_fence_before_sync();   // the next step's first product may have these columns
                __syncwarp();
                if (lane == 0) pair::arrive_cluster(s_free);
                uint32_t packed[16];
                float2 sum = both(0.f);
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float4 f = factors[k];
                    const float2 product = make_float2(d[2 * k], d[2 * k + 1]);
                    float2 z = NORM ? mul2(product, both(iw)) : product;
                    z = fma2(z, make_float2(f.x, f.z), make_float2(f.y, f.w));
                    float2 e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
                    if constexpr (NORM) {
                        e = mul2(e, both(iw));
                        sum = fma2(e, product, sum);
                    }
                    packed[k] = Cvt<E>::pack2(e.x, e.y);
                }
                if (negatives) {   // (seldom: the signs, and the sum once more with them)
                    sum = both(0.f);
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        packed[k] ^= ((negatives >> (2 * k) & 1u) << 15) | ((negatives >> (2 * k + 1) & 1u) << 31);
                        if constexpr (NORM) {
                            const float4 f = factors[k];
                            const float2 product = make_float2(d[2 * k], d[2 * k + 1]), z = fma2(mul2(product, both(iw)), make_float2(f.x, f.z), make_float2(f.y, f.w));
                            const float2 e = mul2(make_float2(exp2_fast(z.x), exp2_fast(z.y)), both(iw));
                            sum = fma2(make_float2(negatives >> (2 * k) & 1u ? -e.x : e.x, negatives >> (2 * k + 1) & 1u ? -e.y : e.y), product, sum);
                        }
                    }
                }
                for (unsigned left = hits; left; left &= left - 1) {
                    const unsigned bit = left & -left;   // (by its bit: indexed, the values would go to local memory)
                    const int from = __ffs(left) - 1, at = __shfl_sync(0xffffffffu, hit, from);
                    const float value = __shfl_sync(0xffffffffu, at_target, from), fa = __shfl_sync(0xffffffffu, a, from), fb = __shfl_sync(0xffffffffu, b, from);
                    if (at == lane) {
                        const uint32_t rounded = Cvt<E>::pack2(value, value);
                        float product = 0.f;
#pragma unroll
                        for (int k = 0; k < 32; ++k) product = bit & (1u << k) ? d[k] : product;
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            packed[k] = bit & (1u << (2 * k)) ? (packed[k] & 0xffff0000u) | (rounded & 0x0000ffffu) : packed[k];
                            packed[k] = bit & (2u << (2 * k)) ? (packed[k] & 0x0000ffffu) | (rounded & 0xffff0000u) : packed[k];
                        }
                        if constexpr (NORM) {   // in the place of what was added for it
                            const float was = exp2_fast(fmaf(product * iw, fa, fb)) * iw;
                            sum.x = fmaf(value - (negatives & bit ? -was : was), product, sum.x);
                        }
                    }
                }
                if (!all_live && !live) {   // classes that are not there: zeros, whatever was staged
                    sum = both(0.f);
#pragma unroll
                    for (int k = 0; k < 16; ++k) packed[k] = 0u;
                }
                along += sum.x + sum.y;
                pair::tmem_st16(tmem + lanes + kOperand + (j & 1) * kOperandCols + part * 16, packed);
                ptx::tmem_st_wait();
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) pair::arrive_cluster(j & 1 ? h_ready1 : h_ready0);
                if (g.grad) {
                    E* out = static_cast<E*>(g.grad) + (size_t)local * g.pitch + t * kRows + part * 32;
                    store_sector(out, packed);
                    store_sector(out + 16, packed + 8);
                }
            }
            if (!ok) break;
            // the classes' gradients
            const E* own = static_cast<const E*>(g.f.w) + (size_t)(live ? v : 0) * g.f.ldw;
            uint4 w[NORM ? 8 : 1];
            if constexpr (NORM) {   // the columns that this warp takes of the classes' own rows, all of them at once
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int n = 16 * part + 64 * (k >> 1) + 8 * (k & 1);
                    w[k] = live && !whole && n < g.D ? __ldg(reinterpret_cast<const uint4*>(own + n)) : make_uint4(0, 0, 0, 0);
                }
            }
            if (NORM) {
                along_s[items & 1][part][row] = along;
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&bar.along);
                if (!ptx::mbar_wait(&bar.along, items & 1) || *abort_flag) NA1D_BOTH_FAIL(2)
                const float(*sums)[kHalf] = along_s[items & 1];
                along = ((sums[0][row] + sums[1][row]) + (sums[2][row] + sums[3][row])) * iw * iw;
            }
            if (steps > 0) {
                if (!ptx::mbar_wait(&bar.acc_full, items & 1) || *abort_flag) NA1D_BOTH_FAIL(3)
                ptx::tc_fence_after_sync();
            }
#pragma unroll
            for (int chunk = 0; chunk < 4; ++chunk) {
                const int n = 16 * part + 64 * chunk;
                if (n >= g.width) break;
                float d[16] = {};
                if (steps > 0) {
                    pair::tmem_ld16(tmem + lanes + kAcc + n, d);
                    ptx::tmem_ld_wait();
                }
                if (whole) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (n + 8 * k < g.D) store_sector(dst + n + 8 * k, reinterpret_cast<const uint32_t*>(d + 8 * k));
                } else if (live) {
                    if (NORM) {
                        float e[16];
                        Cvt<E>::unpack(w[NORM ? 2 * chunk : 0], e);
                        Cvt<E>::unpack(w[NORM ? 2 * chunk + 1 : 0], e + 8);
#pragma unroll
                        for (int k = 0; k < 16; ++k) d[k] = fmaf(-along, e[k], d[k]);
                    }
#pragma unroll
                    for (int k = 0; k < 16; ++k) d[k] *= factor;
                    store_columns<E>(g.f, v, n, d);
                }
            }
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) pair::arrive_cluster(pair::in_leader(&bar.acc_free));
        }
    } else if (warp == kEpilogue) {
        if (ptx::elect_one()) {
            int j = 0, items = 0;
            const bool two = g.second_boxes > 1;
            for (int i = pair_index; ok && i < g.tiles; i += pairs, ++items) {
                if (steps == 0) continue;
                if (!ptx::mbar_wait_relaxed(&bar.w_free, (items & 1) ^ 1) || *abort_flag) NA1D_BOTH_FAIL(4)
                if (rank == 0) ptx::mbar_expect_tx(&bar.w_full, 2 * g.boxes * kClassBox);
                for (int b = 0; b < g.boxes; ++b) pair::load_2d(classes + b * kClassBox, &maps.w, pair::in_leader(&bar.w_full), b * 64, g.v0 + i * kTile + (int)rank * kHalf);
                for (int t = 0; t < steps; ++t, ++j) {
                    const int slot = j % kSlots;
                    const uint32_t phase = ((j / kSlots) & 1) ^ 1;   // the first round finds the slots empty
                    if (!ptx::mbar_wait_relaxed(&bar.first_free[slot], phase) || *abort_flag) NA1D_BOTH_FAIL(5)
                    if (rank == 0) ptx::mbar_expect_tx(&bar.first_full[slot], 2 * g.first_bytes);
                    for (int b = 0; b < g.boxes; ++b)
                        pair::load_2d(firsts + slot * g.first_bytes + b * kFirstBox, &maps.first, pair::in_leader(&bar.first_full[slot]), b * 64, t * kRows + (int)rank * (kRows / 2));
                    if (!ptx::mbar_wait_relaxed(&bar.second_free[slot], phase) || *abort_flag) { 
                        atomicExch(&g_head_status, 6); *abort_flag = 1; ok = false; ++j; break;
                    }
                    if (rank == 0) ptx::mbar_expect_tx(&bar.second_full[slot], 2 * g.second_boxes * kSecondBox);
                    uint8_t* to = seconds + slot * g.second_boxes * kSecondBox;
                    pair::load_2d(to, &maps.second, pair::in_leader(&bar.second_full[slot]), (int)rank * (g.width / 2), t * kRows);
                    if (two) pair::load_2d(to + kSecondBox, &maps.second, pair::in_leader(&bar.second_full[slot]), (int)rank * (g.width / 2) + 64, t * kRows);
                }
            }
            if (!ok && rank == 0) {   // loads that are on their way arrive before the CTAs leave
                for (int k = j - 1; k >= 0 && k >= j - kSlots; --k) {
                    ptx::mbar_wait(&bar.first_full[k % kSlots], (k / kSlots) & 1, 1u << 14);
                    ptx::mbar_wait(&bar.second_full[k % kSlots], (k / kSlots) & 1, 1u << 14);
                }
                for (int k = items; k >= 0 && k >= items - 1; --k) ptx::mbar_wait(&bar.w_full, k & 1, 1u << 14);
            }
        }
    } else if (warp == kEpilogue + 1) {
        if (rank == 0 && ptx::elect_one()) {
            constexpr uint32_t fmt = tc::Fmt<E>::v;
            const uint32_t idesc1 = ptx::instr_desc(fmt, 0, 0, 256, kRows), idesc2 = ptx::instr_desc(fmt, 0, 1, 256, g.width);
            const uint64_t a = pair::k_major(ptx::smem_u32(classes));
            int j = 0, items = 0;
            // dw of step jj, the first of its item (`item`-th) or the last
            auto second = [&](int jj, int item, bool opens, bool closes) {
                const int slot = jj % kSlots;
                if (opens && (!ptx::mbar_wait(&bar.acc_free, (item & 1) ^ 1) || *abort_flag)) { atomicExch(&g_head_status, 7); *abort_flag = 1; ok = false; return; }
                if (!ptx::mbar_wait(&bar.h_ready[jj & 1], (jj >> 1) & 1) || *abort_flag) { atomicExch(&g_head_status, 8); *abort_flag = 1; ok = false; return; }
                if (!ptx::mbar_wait(&bar.second_full[slot], (jj / kSlots) & 1) || *abort_flag) { atomicExch(&g_head_status, 9); *abort_flag = 1; ok = false; return; }
                ptx::tc_fence_after_sync();
                const uint64_t b = pair::mn_major(ptx::smem_u32(seconds + slot * g.second_boxes * kSecondBox), kSecondBox);
                const uint32_t h = tmem + kOperand + (jj & 1) * kOperandCols;
#pragma unroll
                for (int k = 0; k < kRows / 16; ++k) pair::mma_ts(tmem + kAcc, h + k * 8, tc::desc_advance(b, k * 2048), idesc2, !opens || k > 0);
                pair::commit(&bar.second_free[slot]);
                if (closes) pair::commit(&bar.acc_full);
            };
            int open_item = 0;
            bool opens = false;   // of the step before
            for (int i = pair_index; ok && i < g.tiles; i += pairs, ++items) {
                if (steps == 0) continue;
                if (!ptx::mbar_wait(&bar.w_full, items & 1) || *abort_flag) NA1D_BOTH_FAIL(10)
                ptx::tc_fence_after_sync();
                for (int t = 0; ok && t < steps; ++t, ++j) {
                    const int slot = j % kSlots;
                    if (!ptx::mbar_wait(&bar.s_free, (j & 1) ^ 1) || *abort_flag) NA1D_BOTH_FAIL(11)
                    if (!ptx::mbar_wait(&bar.first_full[slot], (j / kSlots) & 1) || *abort_flag) NA1D_BOTH_FAIL(12)
                    ptx::tc_fence_after_sync();
                    const uint64_t b = pair::k_major(ptx::smem_u32(firsts + slot * g.first_bytes));
                    for (int k = 0; k < (g.D + 15) / 16; ++k)
                        pair::mma_ss(tmem + kLogits, tc::desc_advance(a, (k >> 2) * kClassBox + (k & 3) * 32), tc::desc_advance(b, (k >> 2) * kFirstBox + (k & 3) * 32), idesc1, k > 0);
                    pair::commit(&bar.first_free[slot]);
                    pair::commit(&bar.s_full);   // (and all that was issued before, the second product of the step two back among it)
                    if (t == steps - 1) pair::commit(&bar.w_free);
                    if (j > 0) second(j - 1, open_item, opens, t == 0);
                    opens = t == 0;
                    open_item = items;
                }
            }
            if (ok && j > 0) second(j - 1, open_item, opens, true);
        }
    }
#undef NA1D_BOTH_FAIL
    __syncwarp();
    ptx::tc_fence_before_sync();
    __syncthreads();
    pair::cluster_sync();   // neither CTA leaves while the other may still signal it or read its operands
    if (warp == kEpilogue + 2) pair::tmem_dealloc(tmem, 512);
}

template <typename E, bool NORM>
cudaError_t run(const Shape& s, const Saved& sv, Args a, const void* w, int64_t ldw, bool after, int dtype, cudaStream_t st) {
    Maps maps;
    const int64_t dx[2] = {s.D, s.Np}, sx[1] = {s.Dp}, dw[2] = {s.D, s.V}, sw[1] = {ldw};
    const int tall[2] = {64, kHalf}, low[2] = {64, kRows / 2};
    if (!make_matrix_map(&maps.w, w, dtype, 2, dw, sw, tall) || !make_matrix_map(&maps.first, sv.x, dtype, 2, dx, sx, low) ||
        !make_matrix_map(&maps.second, sv.x, dtype, 2, dx, sx, tall))
        return cudaErrorInvalidValue;
    a.boxes = (int)((s.D + 63) / 64);
    a.width = (int)round_up(s.D, 32);
    a.first_bytes = a.boxes * kFirstBox;
    a.second_boxes = a.width / 2 > 64 ? 2 : 1;
    const int smem = a.boxes * kClassBox + kSlots * (a.first_bytes + a.second_boxes * kSecondBox) + 1024;
    auto* kern = both_kernel<E, NORM>;
    static std::atomic<uint64_t> allowed{0};
    if (cudaError_t e = allow_smem(kern, 4 * kClassBox + kSlots * (4 * kFirstBox + 2 * kSecondBox) + 1024, allowed)) return e;
    const int64_t pairs = device_sm_count() / 2;
    return launch(kern, 2 * (a.tiles < pairs ? a.tiles : pairs), kThreads, smem, st, after, maps, a);
}

}  // namespace

cudaError_t gradients_and_weight(const na1d_head& h, const Shape& s, const Saved& sv, const float* coef, void* grad, int64_t pitch, int64_t v0, int64_t cols, float* part_w,
                                 const FinishArgs& f, const void* w, int64_t ldw, bool after, cudaStream_t st) {
    Args a = {};
    a.words = sv.words; a.target = sv.target; a.ix = sv.ix; a.iw = sv.iw; a.lse2 = sv.lse2; a.slope = sv.slope; a.coef = coef;
    a.grad = grad; a.pitch = pitch; a.Dq = s.Dp; a.part_w = part_w; a.v0 = (int)v0; a.cols = (int)cols; a.tiles = (int)((cols + kTile - 1) / kTile); a.D = (int)s.D;
    a.cs = s.cs; a.fp16 = h.dtype == NA1D_FP16; a.f = f;
    using B = __nv_bfloat16;
    if (h.dtype == NA1D_BF16) return s.norm ? run<B, true>(s, sv, a, w, ldw, after, 0, st) : run<B, false>(s, sv, a, w, ldw, after, 0, st);
    return s.norm ? run<__half, true>(s, sv, a, w, ldw, after, 1, st) : run<__half, false>(s, sv, a, w, ldw, after, 1, st);
}
int both_read_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_head_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_head_status, &zero, sizeof(int));
    return v;
}

}  // namespace head
}  // namespace na1d
