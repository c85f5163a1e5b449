// Products of a head's rows and weight, s = x w^T, tile by tile on CTA pairs (cta_group::2), that never leave the chip as they are:
//   stats      a running maximum and sum of 2^z per row, over 64 classes at a time; a teacher's entries
//   gradient   the gradient of the logits in 16 bits, p minus the target's, for a piece of the classes
// A pair takes 256 rows and 256 classes: each CTA stages its 128 rows of x and half of the tile's rows of w by TMA (stages of 64 channels), the leader
// issues the products, and sixteen warps of each CTA read the accumulators back, a row per lane and a quarter of the columns, while the next tile's
// products fill the other half of tensor memory.
// The softmax's maximum and sum stay in 32 bits; the gradient is rounded to 16 bits once, as an operand of the products that follow.
// Bound, forward: at 1024 channels the tensor pipe (8192 x 1024 x 50000, 6144 rows counted: 372 to 391 us, 1.6 to 1.7 PFLOP/s, pipe active 97 % of the
// cycles at 1.53 GHz). At 192 and 256 channels a 256 x 256 tile takes 4400 and 4000 SM cycles where its products take 1536 and 2048 and its exponentials
// 2048 (4099 x 192 x 17982: 41 us; 1024 x 256 x 200003: 98 to 103 us). In an earlier build the tile lost a tenth without exponentials, and a quarter without the epilogue.
// Bound, gradient: the epilogue, 5700 to 5800 cycles a tile there (54 us; 137 us in two pieces), of which that build lost half without it and 2 % without
// exponentials; at 1024 channels the pipe is active 75 % of the cycles (458 us in four pieces).
#include "na1d_head.cuh"
#include "na1d_mlp.cuh"

namespace na1d {
namespace head {
namespace {

__device__ int g_head_status = 0;

constexpr int kEpilogue = 16;                       // warps; each reaches 32 lanes of tensor memory, and takes a quarter of a tile's columns
constexpr int kThreads = 64 + 32 * kEpilogue;       // warp 0: tensor memory and loads, 1: MMA issue, from 2 on: epilogue
constexpr int kWidth = kTile * 4 / kEpilogue;       // columns of a warp
constexpr int kStep = 64, kHalf = 128;
constexpr int kOperand = kHalf * kStep * 2;         // 16 KB: 128 rows of 64 channels
constexpr int kStageBytes = 2 * kOperand;
constexpr int kMostStages = 6;
constexpr int kOut = 32 * 128;                      // a warp's rows of 64 gradients
// The gradients leave through shared memory, by TMA: a sector of each row at a time straight from the lanes took 60 us instead of 55 at
// 4099 x 192 x 17982 and 150 instead of 138 at 1024 x 256 x 200003.
template <bool GRAD> struct Form {
    static constexpr int stages = GRAD ? 5 : kMostStages, smem = stages * kStageBytes + (GRAD ? kEpilogue * kOut : 0) + 1024;
};
constexpr uint32_t kCols = 512;
constexpr int kBand = 16;                           // row tiles that are walked together through the classes

static_assert(kWidth == kPart, "a warp leaves one partial maximum and sum of a row");

struct Barriers {
    uint64_t full[kMostStages], empty[kMostStages], acc_full[2], acc_empty[2];
    uint32_t tmem;
    int abort;
};
struct Maps { CUtensorMap x, w, out; };
struct Args {
    const Words* words;
    const int *row, *target, *index;
    const float *ix, *iw, *lse2, *slope, *coef;
    float* entry;
    float2* part;               // stats: (Np, parts)
    void* grad;                 // gradient: (Np, pitch)
    long long pitch;
    int parts;
    int V, v0, tiles, k, steps, tail;   // first class and tiles of classes of this launch; stages of a tile, products of 16 channels in the last one
    float cs, up;
};

__device__ __forceinline__ float log2_fast(float x) {   // (2^-22 of the logarithm: less than 16 bits of a gradient show)
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void store_tile(const CUtensorMap* map, const void* src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(src)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void prefetch_line(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
// Tiles in the order in which the pairs take them: bands of kBand row tiles, in a band the classes outside and its row tiles inside, so that the pairs
// at work share both operands in L2. A pair takes every `step`-th; from one to its next inside a band there is nothing to divide.
struct Walk {
    int m, n, left;             // this tile; tiles behind it that are in the list
    int first, height, dm, dn;  // its band; the step in it
    int index, step, row_tiles, tiles;
    __device__ __forceinline__ Walk(int index_, int step_, int row_tiles_, int tiles_) : index(index_), step(step_), row_tiles(row_tiles_), tiles(tiles_) {
        left = row_tiles * tiles - index;
        find();
    }
    __device__ __forceinline__ void find() {
        if (left <= 0) return;
        const int band = index / (kBand * tiles), r = index - band * kBand * tiles;
        first = band * kBand;
        height = min(kBand, row_tiles - first);
        n = r / height;
        m = first + (r - n * height);
        dn = step / height;
        dm = step - dn * height;
    }
    __device__ __forceinline__ bool any() const { return left > 0; }
    __device__ __forceinline__ void next() {
        left -= step;
        index += step;
        m += dm;
        n += dn;
        if (m >= first + height) { m -= height; ++n; }
        if (n >= tiles) find();
    }
};

// TOP: the rows have a teacher's entries, sorted by class, instead of a label. A lane has the place of its row's next entry at hand, and the
// class of the one after it.
// FIXED: scaled cosines whose whole range fits fp32's exponents: the scale stands for the maximum.
template <typename E, bool GRAD, bool NORM, bool TOP, bool FIXED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) logits_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args g) {
    constexpr int kStages = Form<GRAD>::stages;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    __shared__ Barriers bar;
    const int warp = ptx::warp_index(), lane = threadIdx.x & 31;
    const uint32_t rank = pair::cta_rank();
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    volatile int* abort_flag = &bar.abort;

    if (warp == 0) {
        if (lane < kStages) { ptx::mbar_init(&bar.full[lane], 1); ptx::mbar_init(&bar.empty[lane], 1); }
        else if (lane < kStages + 2) { ptx::mbar_init(&bar.acc_full[lane - kStages], 1); ptx::mbar_init(&bar.acc_empty[lane - kStages], 2 * kEpilogue); }
        else if (lane == kStages + 2) bar.abort = 0;
        ptx::fence_mbar_init();
    } else if (warp == 1 && lane < 2) {
        ptx::prefetch_tensormap(lane ? &maps.w : &maps.x);
        if (GRAD && lane == 0) ptx::prefetch_tensormap(&maps.out);
    }
    if (warp == 0) { __syncwarp(); pair::tmem_alloc(&bar.tmem, kCols); pair::tmem_relinquish(); }
    ptx::tc_fence_before_sync();
    __syncthreads();
    pair::cluster_sync();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = bar.tmem;
    wait_for_predecessor();
    const int counted = g.words->counted, row_tiles = (counted + kTile - 1) / kTile, items = row_tiles * g.tiles;

    if (warp == 0) {
        if (ptx::elect_one()) {
            int slot = 0, n = 0;
            uint32_t phase = 1;   // the first round finds the slots empty
            bool ok = true;
            for (Walk t(first, step, row_tiles, g.tiles); ok && t.any(); t.next()) {
                const int m = t.m * kTile + rank * kHalf, v = g.v0 + t.n * kTile + rank * kHalf;
                for (int k = 0; k < g.steps; ++k) {
                    if (!ptx::mbar_wait_relaxed(&bar.empty[slot], phase) || *abort_flag) { atomicExch(&g_head_status, 1); *abort_flag = 1; ok = false; break; }
                    const uint32_t full = pair::in_leader(&bar.full[slot]);
                    uint8_t* s = smem + slot * kStageBytes;
                    if (rank == 0) ptx::mbar_expect_tx(&bar.full[slot], 2 * kStageBytes);
                    pair::load_2d(s, &maps.x, full, k * kStep, m);
                    pair::load_2d(s + kOperand, &maps.w, full, k * kStep, v);
                    ++n;
                    if (++slot == kStages) { slot = 0; phase ^= 1; }
                }
            }
            if (!ok && rank == 0)   // loads that are on their way arrive before the CTAs leave
                for (int j = n - 1; j >= 0 && j >= n - kStages; --j) ptx::mbar_wait(&bar.full[j % kStages], (j / kStages) & 1, 1u << 14);
        }
    } else if (warp == 1) {
        if (rank == 0 && ptx::elect_one()) {
            constexpr uint32_t idesc = ptx::instr_desc(tc::Fmt<E>::v, 0, 0, 256, kTile);
            int slot = 0, it = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = first; ok && i < items; i += step, ++it) {
                const uint32_t d = tmem + (it & 1) * kTile;
                if (!ptx::mbar_wait(&bar.acc_empty[it & 1], ((it >> 1) & 1) ^ 1) || *abort_flag) { atomicExch(&g_head_status, 2); *abort_flag = 1; break; }
                ptx::tc_fence_after_sync();
                for (int k = 0; k < g.steps; ++k) {
                    if (!ptx::mbar_wait(&bar.full[slot], phase) || *abort_flag) { atomicExch(&g_head_status, 3); *abort_flag = 1; ok = false; break; }
                    ptx::tc_fence_after_sync();
                    const uint32_t s = ptx::smem_u32(smem + slot * kStageBytes);
                    const uint64_t a = pair::k_major(s), b = pair::k_major(s + kOperand);
                    const int products = k + 1 < g.steps ? kStep / 16 : g.tail;
#pragma unroll
                    for (int j = 0; j < kStep / 16; ++j)
                        if (j < products) pair::mma_ss(d, tc::desc_advance(a, j * 32), tc::desc_advance(b, j * 32), idesc, k > 0 || j > 0);
                    pair::commit(&bar.empty[slot]);
                    if (++slot == kStages) { slot = 0; phase ^= 1; }
                }
                if (ok) pair::commit(&bar.acc_full[it & 1]);
            }
        }
    } else {
        const int q = warp & 3, h = (warp - 2) >> 2;   // tensor-memory lanes 32 q .. + 31 (those a warp reaches), quarter h of the columns
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const float up = GRAD ? g.up : 1.f;
        uint8_t* out_rows = smem + kStages * kStageBytes + (warp - 2) * kOut;
        // what belongs to a tile's row: asked for while the tile before is worked on
        struct Row {
            int target, place;
            float ix, lse2, coef, slope;
        };
        auto row_of = [&](const Walk& t) {
            Row r = {kIgnored, 0, 0.f, 0.f, 1.f, 0.f};
            const int c = t.m * kTile + rank * kHalf + q * 32 + lane;
            if (t.any() && c < counted) {
                if (TOP) r.place = g.row[c];
                else r.target = g.target[c];
                if (NORM) r.ix = g.ix[c];
                if (GRAD) {
                    r.lse2 = g.lse2[c];
                    if (!TOP) r.slope = g.slope[c];
                    if (g.coef) r.coef = g.coef[c];
                }
            }
            if (NORM && t.any() && lane < kWidth * 4 / 128) prefetch_line(g.iw + g.v0 + t.n * kTile + h * kWidth + lane * 32);
            return r;
        };
        int it = 0;
        Walk ahead(first, step, row_tiles, g.tiles);
        Row next_row = row_of(ahead);
        while (ahead.any()) {
            const int c = ahead.m * kTile + rank * kHalf + q * 32 + lane, v = g.v0 + ahead.n * kTile + h * kWidth;
            const Row row = next_row;
            ahead.next();
            next_row = row_of(ahead);
            const bool live = c < counted;
            const int target = row.target;
            // (a row of zeros has no direction: its products are 0 whatever they are multiplied with, and it gets no gradient)
            const float ix = NORM ? row.ix : 1.f, cs = ix > 0.f ? g.cs * ix : g.cs;
            // the gradient's factor goes into the exponent, but for its sign
            float shift = 0.f, out = 0.f, at_target = 0.f;
            bool negative = false;
            if (GRAD && live) {
                out = row_factor(up, ix, row.coef, NORM);
                shift = log2_fast(fabsf(out)) - row.lse2;
                negative = out < 0.f;
                if (!TOP && target >= 0) at_target = own_gradient(row.slope, out, NORM ? g.iw[target] : 1.f, NORM);
            }
            const int* classes = nullptr;
            float* entry = nullptr;
            int next = kNoClass, after = kNoClass, pos = 0;
            if (TOP && live) {
                classes = g.index + (size_t)row.place * g.k;
                entry = g.entry + (size_t)row.place * g.k;
                for (int end = g.k; pos < end;) {   // the first entry whose class is v or more
                    const int mid = (pos + end) >> 1;
                    if (__ldg(classes + mid) < v) pos = mid + 1;
                    else end = mid;
                }
                if (pos < g.k) next = __ldg(classes + pos);
                if (pos + 1 < g.k) after = __ldg(classes + pos + 1);
            }
            auto advance = [&]() {
                ++pos;
                next = after;
                after = pos + 1 < g.k ? __ldg(classes + pos + 1) : kNoClass;
            };
            if (!ptx::mbar_wait(&bar.acc_full[it & 1], (it >> 1) & 1) || *abort_flag) { atomicExch(&g_head_status, 4); *abort_flag = 1; break; }
            ptx::tc_fence_after_sync();
            const uint32_t acc = tmem + lanes + (it & 1) * kTile + h * kWidth;
            float most = FIXED ? g.cs : -INFINITY, sum = 0.f;
            // (rows behind the last that counts are nobody's: the products contract over whole steps of 64)
            const bool any_row = c - lane < (GRAD ? (counted + 63) / 64 * 64 : counted);
#pragma unroll(GRAD ? 1 : 2)
            for (int n = 0; n < kWidth; n += 32) {
                if (!any_row) break;
                float d[32];
                float2 iw[NORM ? 16 : 1];
                const int col = v + n;
                if constexpr (NORM) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 f = __ldg(reinterpret_cast<const float4*>(g.iw + col) + j);
                        iw[2 * j] = make_float2(f.x, f.y);
                        iw[2 * j + 1] = make_float2(f.z, f.w);
                    }
                }
                pair::tmem_ld32(acc + n, d);
                ptx::tmem_ld_wait();
                const bool hit = !TOP && (unsigned)(target - col) < 32u;
                if constexpr (NORM) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float2 z = mul2(make_float2(d[2 * j], d[2 * j + 1]), iw[j]);
                        d[2 * j] = z.x;
                        d[2 * j + 1] = z.y;
                    }
                }
                if constexpr (!GRAD) {
                    if (col + 32 > g.V) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (col + j >= g.V) d[j] = -INFINITY;
                    }
                    if (hit) {   // the target's logit is added in its own form
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (j == target - col) d[j] = -INFINITY;
                    }
                    if constexpr (TOP) {
                        while (__any_sync(0xffffffffu, next < col + 32)) {
                            if (next < col + 32) {
                                // (by its bit: indexed, the row would go to local memory)
                                const uint32_t bit = 1u << (next - col);
                                float z = 0.f;
#pragma unroll
                                for (int j = 0; j < 32; ++j) z = bit & (1u << j) ? d[j] : z;
                                entry[pos] = z * cs;
                                advance();
                            }
                        }
                    }
                    float by = most;
                    if constexpr (!FIXED) {
                        float m[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) m[j] = fmaxf(fmaxf(d[j], d[j + 8]), fmaxf(d[j + 16], d[j + 24]));
                        const float top = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), fmaxf(fmaxf(m[4], m[5]), fmaxf(m[6], m[7])));
                        const float to = fmaxf(most, top * cs);
                        by = to > -INFINITY ? to : 0.f;
                        sum *= exp2_fast(most - by);
                        most = to;
                    }
                    float2 s0 = both(0.f), s1 = both(0.f);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float2 z = fma2(make_float2(d[2 * j], d[2 * j + 1]), both(cs), both(-by)), e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
                        if (j & 1) s1 = add2(s1, e);
                        else s0 = add2(s0, e);
                    }
                    s0 = add2(s0, s1);
                    sum += s0.x + s0.y;
                } else {
                    uint32_t packed[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float2 z = fma2(make_float2(d[2 * j], d[2 * j + 1]), both(cs), both(shift));
                        float2 e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
                        if constexpr (NORM) e = mul2(e, iw[j]);
                        d[2 * j] = e.x;
                        d[2 * j + 1] = e.y;
                    }
                    if (negative) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) d[j] = -d[j];
                    }
                    if (hit) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (j == target - col) d[j] = at_target;
                    }
                    if constexpr (TOP) {
                        while (__any_sync(0xffffffffu, next < col + 32)) {
                            if (next < col + 32) {
                                const float f = own_gradient(entry[pos], out, NORM ? __ldg(g.iw + next) : 1.f, NORM);
                                const uint32_t bit = 1u << (next - col);
#pragma unroll
                                for (int j = 0; j < 32; ++j) d[j] = bit & (1u << j) ? f : d[j];
                                advance();
                            }
                        }
                    }
                    if (!live || col + 32 > g.V) {   // rows and classes that are not there: zeros, whatever was staged
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (!live || col + j >= g.V) d[j] = 0.f;
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) packed[j] = Cvt<E>::pack2(d[2 * j], d[2 * j + 1]);
                    if (n == 0) {   // the tile before has left
                        if (lane == 0) ptx::tma_store_wait_read();
                        __syncwarp();
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<uint4*>(out_rows + lane * 128 + ((((n >> 3) + j) ^ (lane & 7)) << 4)) = make_uint4(packed[4 * j], packed[4 * j + 1], packed[4 * j + 2], packed[4 * j + 3]);
                }
            }
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) pair::arrive_cluster(pair::in_leader(&bar.acc_empty[it & 1]));
            if (GRAD && any_row) {
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    store_tile(&maps.out, out_rows, v - g.v0, c);
                    ptx::tma_store_commit();
                }
            }
            if (!GRAD && live) g.part[(size_t)c * g.parts + v / kPart] = make_float2(most, sum);
            ++it;
        }
        if (GRAD && lane == 0) ptx::tma_store_wait_all();
    }
    __syncwarp();
    ptx::tc_fence_before_sync();
    __syncthreads();
    pair::cluster_sync();   // neither CTA leaves while the other may still signal it or read its operands
    if (warp == 0) pair::tmem_dealloc(tmem, kCols);
}

template <typename E, bool GRAD, bool NORM, bool TOP, bool FIXED = false>
cudaError_t run(const Shape& s, const Saved& sv, const Args& a, const void* w, int64_t ldw, bool after, int dtype, cudaStream_t st) {
    Maps maps;
    const int64_t dx[2] = {s.D, s.Np}, sx[1] = {s.Dp}, dw[2] = {s.D, s.V}, sw[1] = {ldw};
    const int box[2] = {kStep, kHalf};
    if (!make_matrix_map(&maps.x, sv.x, dtype, 2, dx, sx, box) || !make_matrix_map(&maps.w, w, dtype, 2, dw, sw, box)) return cudaErrorInvalidValue;
    const int64_t dout[2] = {a.pitch, s.Np}, sout[1] = {a.pitch};
    const int out_box[2] = {64, 32};
    if (GRAD && !make_matrix_map(&maps.out, a.grad, dtype, 2, dout, sout, out_box)) return cudaErrorInvalidValue;
    if (!GRAD) maps.out = maps.x;
    constexpr int kSmem = Form<GRAD>::smem;
    auto* kern = logits_kernel<E, GRAD, NORM, TOP, FIXED>;
    static std::atomic<uint64_t> allowed{0};
    if (cudaError_t e = allow_smem(kern, kSmem, allowed)) return e;
    const int64_t items = s.Np / kTile * a.tiles, pairs = device_sm_count() / 2;
    return launch(kern, 2 * (items < pairs ? items : pairs), kThreads, kSmem, st, after, maps, a);
}
template <bool GRAD>
cudaError_t start(const na1d_head& h, const Shape& s, const Saved& sv, Args a, const void* w, int64_t ldw, bool after, cudaStream_t st) {
    a.words = sv.words; a.row = sv.row; a.target = sv.target; a.index = sv.index; a.entry = sv.entry;
    a.ix = sv.ix; a.iw = sv.iw; a.lse2 = sv.lse2; a.slope = sv.slope;
    a.parts = (int)s.parts; a.V = (int)s.V; a.k = (int)s.k; a.cs = s.cs; a.up = s.up;
    a.steps = (int)((s.D + kStep - 1) / kStep);
    a.tail = (int)((s.D - (int64_t)(a.steps - 1) * kStep + 15) / 16);
    // scaled cosines of at most +-48 powers of two: the smallest term is 2^-96 of the one that the scale stands for
    const bool fixed = !GRAD && s.norm && s.cs <= 48.f;
#define NA1D_HEAD_RUN(E, NORM, TOP, code) \
    return fixed && NORM ? run<E, GRAD, NORM, TOP, !GRAD && NORM>(s, sv, a, w, ldw, after, code, st) : run<E, GRAD, NORM, TOP>(s, sv, a, w, ldw, after, code, st)
    const bool bf16 = h.dtype == NA1D_BF16, top = s.k > 0;
    using B = __nv_bfloat16;
    using H = __half;
    if (bf16 && s.norm && top) NA1D_HEAD_RUN(B, true, true, 0);
    if (bf16 && s.norm) NA1D_HEAD_RUN(B, true, false, 0);
    if (bf16 && top) NA1D_HEAD_RUN(B, false, true, 0);
    if (bf16) NA1D_HEAD_RUN(B, false, false, 0);
    if (s.norm && top) NA1D_HEAD_RUN(H, true, true, 1);
    if (s.norm) NA1D_HEAD_RUN(H, true, false, 1);
    if (top) NA1D_HEAD_RUN(H, false, true, 1);
    NA1D_HEAD_RUN(H, false, false, 1);
#undef NA1D_HEAD_RUN
}

}  // namespace

cudaError_t stats(const na1d_head& h, const Shape& s, const Saved& sv, float2* part, const void* w, int64_t ldw, cudaStream_t st) {
    Args a = {};
    a.part = part;
    a.tiles = (int)((s.V + kTile - 1) / kTile);
    return start<false>(h, s, sv, a, w, ldw, true, st);
}
cudaError_t gradients(const na1d_head& h, const Shape& s, const Saved& sv, const float* coef, void* grad, int64_t pitch, int64_t v0, int64_t tiles, const void* w,
                      int64_t ldw, bool after, cudaStream_t st) {
    Args a = {};
    a.coef = coef; a.grad = grad; a.pitch = pitch; a.v0 = (int)v0; a.tiles = (int)tiles;
    return start<true>(h, s, sv, a, w, ldw, after, st);
}
int logits_read_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_head_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_head_status, &zero, sizeof(int));
    return v;
}

}  // namespace head
}  // namespace na1d
