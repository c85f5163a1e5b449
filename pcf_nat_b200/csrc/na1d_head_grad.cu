// The two products of a head's backward pass, from the gradient G of the logits of a piece of the classes (rows x classes, 16 bits):
//   rows      dx += G w     contraction over the piece's classes
//   weight    dw  = G^T x   contraction over the rows that count
// in one launch of CTA pairs over 256 x (up to 256) tiles. G's tile is staged as it lies: its contraction index runs along its rows for the
// first product and across them for the second; w and x contract across their rows in both. The rows' results leave as
// fp32 partial sums, one for each split of the contraction: the pieces' shares of dx are added up there in the order of the pieces. The weight's are
// complete in a tile (unless there are too few tiles for the SMs) and leave as they are wanted.
// Bound: at 1024 channels the tensor pipe, active 75 % of the cycles (8192 x 1024 x 50000, 6144 rows counted: 1007 to 1020 us in four pieces, 1.25 PFLOP/s).
// At 192 and 256 channels mostly memory, since both products read G: 4.4 and 5.2 TB/s from and to HBM, pipe active 45 % (4099 x 192 x 17982: 72 to 74 us;
// 1024 x 256 x 200003: 238 us). One kernel for the gradient of the logits and the weight's, with G as an operand from tensor memory, gained nothing: it and the
// rows' products took 119 us where the two kernels take 126, and 390 where they take 375.
#include "na1d_head.cuh"
#include "na1d_mlp.cuh"

namespace na1d {
namespace head {
namespace {

__device__ int g_head_status = 0;

constexpr int kEpilogue = 16;                       // warps; each reaches 32 lanes of tensor memory, and takes every fourth 16 columns
constexpr int kThreads = 128 + 32 * kEpilogue;      // warp 0: loads, 1: MMA issue, 2: tensor memory, 3: the plan, from 4 on: results
constexpr int kStep = 64, kHalf = 128;              // contraction steps of a stage; rows of G's side in one CTA
constexpr int kBox = 64 * kStep * 2;                // 64 columns of a stage
constexpr int kOperand = 2 * kBox;
constexpr int kStageBytes = 2 * kOperand;
constexpr int kOwnBox = 64 * kHalf * 2;             // 64 columns of the classes' own rows
constexpr int kMostStages = 6;
constexpr int kMostSmem = 232448 - 5 * 1024;        // (static: barriers, the plan, sums of four warps)
constexpr uint32_t kCols = 512;

struct Barriers {
    uint64_t full[kMostStages], empty[kMostStages], acc_full[2], acc_empty[2], own_full, own_free, along;
    uint32_t tmem;
    int abort;
};
struct Maps { CUtensorMap g_rows, g_cols, x, w, own; };   // G with its contraction along and across its rows; w for a product, and as it is
struct Args {
    const Words* words;
    float *part_x, *part_w;
    long long Np, Dq, piece_rows;                    // rows of a split's partial sums and their pitch
    int D, d_tiles, d_width, v0, cols, tiles, splits_x, splits_w, stages;
    bool want_x, want_w, add, direct;
    FinishArgs f;
};
struct Item {
    int m0, n0, k0, k1, split;
    bool rows;                                       // a tile of dx
};
// The weight's items go to the pairs in turn, the rows' fill up what those leave of the pairs' time: pairs below `more` have one item of the weight's
// more than the others, and take fill0 items of the rows', the others fill1.
struct Plan {
    int items_x, items_w, steps_x, steps_w, more, fill0, fill1;
};
// (a warp)
__device__ __forceinline__ Plan plan_of(const Args& g, int pairs) {
    const int counted = g.words->counted;
    Plan p;
    p.items_x = g.want_x ? (counted + kTile - 1) / kTile * g.d_tiles * g.splits_x : 0;
    p.items_w = g.want_w ? g.tiles * g.d_tiles * g.splits_w : 0;
    p.steps_x = (g.cols + kStep - 1) / kStep;
    p.steps_w = (counted + kStep - 1) / kStep;
    p.more = p.items_w % pairs;
    // a pair's end: the smallest by which all of the rows' items are done, each of them taking the longest one's time. It lies a whole number of
    // them behind the weight's items of some pairs, and within one of the average: each lane tries one such end.
    const int item_x = (p.steps_x + g.splits_x - 1) / g.splits_x, item_w = (p.steps_w + g.splits_w - 1) / g.splits_w;
    const int busy1 = p.items_w / pairs * item_w, busy0 = busy1 + item_w, lane = threadIdx.x & 31;
    const int average = (int)(((long long)p.items_w * item_w + (long long)p.items_x * item_x) / pairs), busy = lane & 1 ? busy1 : busy0;
    const int end = busy + (max(average - busy, 0) / item_x + (lane >> 1)) * item_x;
    const int fill0 = max(end - busy0, 0) / item_x, fill1 = max(end - busy1, 0) / item_x;
    const bool enough = (long long)p.more * fill0 + (long long)(pairs - p.more) * fill1 >= p.items_x;
    const unsigned best = __reduce_min_sync(0xffffffffu, enough ? (unsigned)end : 0xffffffffu);
    const int who = __ffs(__ballot_sync(0xffffffffu, enough && (unsigned)end == best)) - 1;
    p.fill0 = __shfl_sync(0xffffffffu, fill0, who);
    p.fill1 = __shfl_sync(0xffffffffu, fill1, who);
    return p;
}
// a pair's items, one after the other: the weight's, then the rows'
struct Walk {
    int next_w, next_x, end_x;
};
__device__ __forceinline__ Walk walk_of(const Plan& p, int pair) {
    Walk w;
    w.next_w = pair;
    const long long first = pair < p.more ? (long long)pair * p.fill0 : (long long)p.more * p.fill0 + (long long)(pair - p.more) * p.fill1;
    const long long end = first + (pair < p.more ? p.fill0 : p.fill1);
    w.next_x = first < p.items_x ? (int)first : p.items_x;
    w.end_x = end < p.items_x ? (int)end : p.items_x;
    return w;
}
__device__ __forceinline__ bool next_item(const Args& g, const Plan& p, Walk& w, int pairs, Item& t) {
    int i;
    if (w.next_w < p.items_w) {
        t.rows = false;
        i = w.next_w;
        w.next_w += pairs;
    } else if (w.next_x < w.end_x) {
        t.rows = true;
        i = w.next_x++;
    } else {
        return false;
    }
    const int splits = t.rows ? g.splits_x : g.splits_w, steps = t.rows ? p.steps_x : p.steps_w;
    const int tile = i / splits;
    t.split = i - tile * splits;
    t.m0 = tile / g.d_tiles * kTile;
    t.n0 = tile % g.d_tiles * g.d_width;
    t.k0 = (int)((long long)steps * t.split / splits);
    t.k1 = (int)((long long)steps * (t.split + 1) / splits);
    return true;
}

__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {   // this CTA's own
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(ptx::smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(c0), "r"(c1) : "memory");
}
// one addition to each of four places that nothing else in the launch touches: nothing waits for what was there
__device__ __forceinline__ void add4(float* p, const float* d) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(d[0]), "f"(d[1]), "f"(d[2]), "f"(d[3]) : "memory");
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

// PROJECT: the classes' own rows are staged too, for the way back through the normalisation
template <typename E, bool PROJECT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) grad_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args g) {
    const int kStages = PROJECT ? g.stages : kMostStages;   // (the staged classes take the others' place)
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* own_rows = smem + kStages * kStageBytes;
    __shared__ Barriers bar;
    __shared__ Plan plan_s;
    __shared__ float along_s[2][4][kHalf];
    const int warp = ptx::warp_index(), lane = threadIdx.x & 31;
    const uint32_t rank = pair::cta_rank();
    const int pair_index = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    volatile int* abort_flag = &bar.abort;

    if (warp == 0) {
        if (lane < kStages) { ptx::mbar_init(&bar.full[lane], 1); ptx::mbar_init(&bar.empty[lane], 1); }
        else if (lane < kStages + 2) { ptx::mbar_init(&bar.acc_full[lane - kStages], 1); ptx::mbar_init(&bar.acc_empty[lane - kStages], 2 * kEpilogue); }
        else if (lane == kStages + 2) { ptx::mbar_init(&bar.own_full, 1); ptx::mbar_init(&bar.own_free, kEpilogue); ptx::mbar_init(&bar.along, kEpilogue); bar.abort = 0; }
        ptx::fence_mbar_init();
    } else if (warp == 1 && lane < 5) {
        ptx::prefetch_tensormap(lane == 0 ? &maps.g_rows : lane == 1 ? &maps.g_cols : lane == 2 ? &maps.x : lane == 3 ? &maps.w : &maps.own);
    }
    if (warp == 2) { pair::tmem_alloc(&bar.tmem, kCols); pair::tmem_relinquish(); }
    wait_for_predecessor();
    if (warp == 3) {
        const Plan made = plan_of(g, pairs);
        if (lane == 0) plan_s = made;
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    pair::cluster_sync();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = bar.tmem;
    const Plan p = plan_s;
    Walk walk = walk_of(p, pair_index);
    Item t;
    const int half_width = g.d_width / 2;               // columns of w or x in one CTA

    if (warp == 0) {
        if (ptx::elect_one()) {
            int slot = 0, n = 0, projected = 0;
            uint32_t phase = 1;   // the first round finds the slots empty
            bool ok = true;
            const bool two = half_width > 64;
            const int own_boxes = (g.D + 63) / 64;
            while (ok && next_item(g, p, walk, pairs, t)) {
                const CUtensorMap* mb = t.rows ? &maps.w : &maps.x;
                const int m = t.m0 + rank * kHalf, d = t.n0 + rank * half_width, r0 = t.rows ? g.v0 : 0;
                for (int k = t.k0; k < t.k1; ++k) {
                    if (!ptx::mbar_wait_relaxed(&bar.empty[slot], phase) || *abort_flag) { atomicExch(&g_head_status, 1); *abort_flag = 1; ok = false; break; }
                    const uint32_t full = pair::in_leader(&bar.full[slot]);
                    uint8_t* s = smem + slot * kStageBytes;
                    if (rank == 0) ptx::mbar_expect_tx(&bar.full[slot], 2 * (kOperand + (two ? 2 : 1) * kBox));
                    if (t.rows) {
                        pair::load_2d(s, &maps.g_rows, full, k * kStep, m);
                    } else {
                        pair::load_2d(s, &maps.g_cols, full, m, k * kStep);
                        pair::load_2d(s + kBox, &maps.g_cols, full, m + 64, k * kStep);
                    }
                    pair::load_2d(s + kOperand, mb, full, d, r0 + k * kStep);
                    if (two) pair::load_2d(s + kOperand + kBox, mb, full, d + 64, r0 + k * kStep);
                    ++n;
                    if (++slot == kStages) { slot = 0; phase ^= 1; }
                }
                if (PROJECT && ok && !t.rows) {   // (last: the epilogue of the item before may still read the rows that were there)
                    if (!ptx::mbar_wait_relaxed(&bar.own_free, (projected & 1) ^ 1) || *abort_flag) { atomicExch(&g_head_status, 5); *abort_flag = 1; ok = false; break; }
                    ptx::mbar_expect_tx(&bar.own_full, own_boxes * kOwnBox);
                    for (int b = 0; b < own_boxes; ++b) load_tile(own_rows + b * kOwnBox, &maps.own, &bar.own_full, b * 64, g.v0 + m);
                    ++projected;
                }
            }
            if (!ok) {   // loads that are on their way arrive before the CTAs leave
                if (rank == 0)
                    for (int j = n - 1; j >= 0 && j >= n - kStages; --j) ptx::mbar_wait(&bar.full[j % kStages], (j / kStages) & 1, 1u << 14);
                if (projected > 0) ptx::mbar_wait(&bar.own_full, (projected - 1) & 1, 1u << 14);
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && ptx::elect_one()) {
            const uint32_t rows_desc = ptx::instr_desc(tc::Fmt<E>::v, 0, 1, 256, g.d_width), cols_desc = ptx::instr_desc(tc::Fmt<E>::v, 1, 1, 256, g.d_width);
            int slot = 0, it = 0;
            uint32_t phase = 0;
            bool ok = true;
            while (ok && next_item(g, p, walk, pairs, t)) {
                if (t.k0 == t.k1) continue;
                const uint32_t d = tmem + (it & 1) * kTile, idesc = t.rows ? rows_desc : cols_desc, a_step = t.rows ? 32 : 2048;
                if (!ptx::mbar_wait(&bar.acc_empty[it & 1], ((it >> 1) & 1) ^ 1) || *abort_flag) { atomicExch(&g_head_status, 2); *abort_flag = 1; break; }
                ptx::tc_fence_after_sync();
                for (int k = t.k0; k < t.k1; ++k) {
                    if (!ptx::mbar_wait(&bar.full[slot], phase) || *abort_flag) { atomicExch(&g_head_status, 3); *abort_flag = 1; ok = false; break; }
                    ptx::tc_fence_after_sync();
                    const uint32_t s = ptx::smem_u32(smem + slot * kStageBytes);
                    const uint64_t a = t.rows ? pair::k_major(s) : pair::mn_major(s, kBox), b = pair::mn_major(s + kOperand, kBox);
#pragma unroll
                    for (int j = 0; j < kStep / 16; ++j)
                        pair::mma_ss(d, tc::desc_advance(a, j * a_step), tc::desc_advance(b, j * 2048), idesc, k > t.k0 || j > 0);
                    pair::commit(&bar.empty[slot]);
                    if (++slot == kStages) { slot = 0; phase ^= 1; }
                }
                if (ok) pair::commit(&bar.acc_full[it & 1]);
                ++it;
            }
        }
    } else if (warp >= 4) {
        const int q = warp & 3, h = (warp - 4) >> 2;   // tensor-memory lanes 32 q .. + 31 (those a warp reaches); columns 16 h, 16 h + 64, ..
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const int counted = g.words->counted, row = q * 32 + lane;
        const float factor = g.direct ? common_factor(g.f, counted) : 1.f;
        const uint8_t* own_row = own_rows + row * 128;
        int it = 0, projected = 0;
        while (next_item(g, p, walk, pairs, t)) {
            const bool empty = t.k0 == t.k1;           // a split without steps: zeros
            if (empty && t.rows && g.add) continue;
            const int r = t.m0 + rank * kHalf + row, v = g.v0 + r;
            const bool live = r < (t.rows ? counted : g.cols), direct = g.direct && !t.rows;
            float* dst = t.rows ? g.part_x + (size_t)t.split * g.Np * g.Dq + (size_t)r * g.Dq : g.part_w + (size_t)t.split * g.piece_rows * g.Dq + (size_t)r * g.Dq;
            bool whole = !direct;                      // an fp32 sum at dst
            float iw = 0.f, back = 1.f;
            if (direct && live) {
                // a class that is some rows' own (and not that of many, whose roundings average out) gets what rounding took in the last step
                const int count = g.f.own_count[v];
                whole = count > 0 && count <= kOwn;
                if (whole) dst = g.part_w + (size_t)g.f.own[(size_t)v * kOwn] * g.Dq;
                if (PROJECT) {
                    iw = g.f.iw[v];
                    if (g.f.w_up) back = g.f.w_up[v];
                }
            }
            if (!empty) {
                if (!ptx::mbar_wait_relaxed(&bar.acc_full[it & 1], (it >> 1) & 1) || *abort_flag) { atomicExch(&g_head_status, 4); *abort_flag = 1; break; }
                ptx::tc_fence_after_sync();
            }
            const uint32_t acc = tmem + lanes + (it & 1) * kTile;
            auto columns = [&](int n, float* d) {
                if (empty) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) d[j] = 0.f;
                } else {
                    pair::tmem_ld16(acc + n, d);
                    ptx::tmem_ld_wait();
                }
            };
            auto own_columns = [&](int n, float* e) {   // of the staged row: 16-byte pieces, swizzled
                const uint8_t* box = own_row + (n >> 6) * kOwnBox;
#pragma unroll
                for (int j = 0; j < 2; ++j) Cvt<E>::unpack(*reinterpret_cast<const uint4*>(box + (((((n & 63) >> 3) + j) ^ (row & 7)) << 4)), e + 8 * j);
            };
            float along = 0.f;
            if (PROJECT && direct) {
                if (!ptx::mbar_wait_relaxed(&bar.own_full, projected & 1) || *abort_flag) { atomicExch(&g_head_status, 6); *abort_flag = 1; break; }
#pragma unroll 1
                for (int n = 16 * h; n < g.d_width; n += 64) {
                    float d[16], e[16];
                    columns(n, d);
                    own_columns(n, e);
#pragma unroll
                    for (int j = 0; j < 16; ++j) along = fmaf(d[j], e[j], along);
                }
                along_s[projected & 1][h][row] = along;
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&bar.along);
                if (!ptx::mbar_wait(&bar.along, projected & 1) || *abort_flag) { atomicExch(&g_head_status, 7); *abort_flag = 1; break; }
                const float(*sums)[kHalf] = along_s[projected & 1];
                along = ((sums[0][row] + sums[1][row]) + (sums[2][row] + sums[3][row])) * iw;
            }
#pragma unroll 1
            for (int n = 16 * h; n < g.d_width; n += 64) {
                float d[16];
                columns(n, d);
                const int col = t.n0 + n;
                if (live && whole) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (col + 8 * j < g.D) {
                            if (t.rows && g.add) {
                                add4(dst + col + 8 * j, d + 8 * j);
                                add4(dst + col + 8 * j + 4, d + 8 * j + 4);
                            } else {
                                store_sector(dst + col + 8 * j, reinterpret_cast<const uint32_t*>(d + 8 * j));
                            }
                        }
                } else if (live) {
                    if (PROJECT) {
                        float e[16];
                        own_columns(n, e);
#pragma unroll
                        for (int j = 0; j < 16; ++j) d[j] = fmaf(-along, e[j] * iw, d[j]);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) d[j] = PROJECT ? d[j] * factor * back : d[j] * factor;
                    store_columns<E>(g.f, v, col, d);
                }
            }
            if (PROJECT && direct) {
                ++projected;
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&bar.own_free);
            }
            if (!empty) {
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) pair::arrive_cluster(pair::in_leader(&bar.acc_empty[it & 1]));
                ++it;
            }
        }
    }
    __syncwarp();
    ptx::tc_fence_before_sync();
    __syncthreads();
    pair::cluster_sync();   // neither CTA leaves while the other may still signal it or read its operands
    if (warp == 2) pair::tmem_dealloc(tmem, kCols);
}

template <typename E, bool PROJECT>
cudaError_t run(const Shape& s, const Saved& sv, const void* grad, Args a, int64_t pitch, const void* w, int64_t ldw, int dtype, cudaStream_t st) {
    Maps maps;
    const int64_t dg[2] = {pitch, s.Np}, sg[1] = {pitch}, dx[2] = {s.D, s.Np}, sx[1] = {s.Dp}, dw[2] = {s.D, s.V}, sw[1] = {ldw};
    const int along[2] = {64, kHalf}, across[2] = {64, kStep};
    if (!make_matrix_map(&maps.g_rows, grad, dtype, 2, dg, sg, along) || !make_matrix_map(&maps.g_cols, grad, dtype, 2, dg, sg, across) ||
        !make_matrix_map(&maps.x, sv.x, dtype, 2, dx, sx, across) || !make_matrix_map(&maps.w, w, dtype, 2, dw, sw, across) ||
        !make_matrix_map(&maps.own, w, dtype, 2, dw, sw, along))
        return cudaErrorInvalidValue;
    auto* kern = grad_kernel<E, PROJECT>;
    const int own_bytes = PROJECT ? (int)((s.D + 63) / 64) * kOwnBox : 0, fit = (kMostSmem - 1024 - own_bytes) / kStageBytes;
    a.stages = fit < kMostStages ? fit : kMostStages;
    const int smem = a.stages * kStageBytes + own_bytes + 1024;
    static std::atomic<uint64_t> allowed{0};
    if (cudaError_t e = allow_smem(kern, kMostSmem, allowed)) return e;
    const int64_t items = (a.want_x ? s.Np / kTile * a.d_tiles * a.splits_x : 0) + (a.want_w ? (int64_t)a.tiles * a.d_tiles * a.splits_w : 0);
    const int64_t pairs = device_sm_count() / 2;
    return launch(kern, 2 * (items < pairs ? items : pairs), kThreads, smem, st, true, maps, a);
}

}  // namespace

cudaError_t products(const na1d_head& h, const Shape& s, const Saved& sv, const void* grad, const Pieces& p, int64_t v0, int64_t cols, bool add, float* part_x,
                     float* part_w, const FinishArgs& f, const void* w, int64_t ldw, cudaStream_t st) {
    Args a = {};
    a.words = sv.words; a.part_x = part_x; a.part_w = part_w;
    a.Np = s.Np; a.Dq = s.Dp; a.piece_rows = p.pitch;
    a.D = (int)s.D; a.d_tiles = p.d_tiles; a.d_width = p.d_width; a.v0 = (int)v0; a.cols = (int)cols;
    a.tiles = (int)((cols + kTile - 1) / kTile); a.splits_x = p.splits_x; a.splits_w = p.splits_w;
    a.want_x = part_x != nullptr; a.want_w = part_w != nullptr; a.add = add; a.direct = p.direct_w;
    a.f = f;
    const bool project = p.direct_w && s.norm;
    if (h.dtype == NA1D_BF16) return project ? run<__nv_bfloat16, true>(s, sv, grad, a, p.pitch, w, ldw, 0, st) : run<__nv_bfloat16, false>(s, sv, grad, a, p.pitch, w, ldw, 0, st);
    return project ? run<__half, true>(s, sv, grad, a, p.pitch, w, ldw, 1, st) : run<__half, false>(s, sv, grad, a, p.pitch, w, ldw, 1, st);
}
int grad_read_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_head_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_head_status, &zero, sizeof(int));
    return v;
}

}  // namespace head
}  // namespace na1d
