// The two products of a head's backward pass, from the gradient G of the logits of a piece of the classes (rows x classes, 16 bits):
//   rows      dx += G w     contraction over the piece's classes
//   weight    dw  = G^T x   contraction over the rows that count
// in one launch of CTA pairs over 256 x (up to 256) tiles. G's tile is staged as it lies: its contraction index runs along its rows for the
// first product and across them for the second; w and x contract across their rows in both. The rows' results leave as
// fp32 partial sums, one for each split of the contraction: the pieces' shares of dx are added up there in the order of the pieces. The weight's are
// complete in a tile (unless there are too few tiles for the SMs) and leave as they are wanted.
#include "na1d_head.cuh"
#include "na1d_mlp.cuh"

namespace na1d {
namespace head {
namespace {

__device__ int g_head_status = 0;

constexpr int kThreads = 384;                       // warp 0: loads, 1: MMA issue, 2: tensor memory, 4-11: results
constexpr int kStep = 64, kHalf = 128;              // contraction steps of a stage; rows of G's side in one CTA
constexpr int kBox = 64 * kStep * 2;                // 64 columns of a stage
constexpr int kOperand = 2 * kBox;
constexpr int kStageBytes = 2 * kOperand;
constexpr int kStages = 6;
constexpr int kSmem = kStages * kStageBytes + 1024;
constexpr uint32_t kCols = 512;

struct Barriers {
    uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2];
    uint32_t tmem;
    int abort;
};
struct Maps { CUtensorMap g_rows, g_cols, x, w; };   // G with its contraction along and across its rows
struct Args {
    const Words* words;
    float *part_x, *part_w;
    long long Np, Dq, piece_rows;                    // rows of a split's partial sums and their pitch
    int D, d_tiles, d_width, v0, cols, tiles, splits_x, splits_w;
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
__device__ __forceinline__ Plan plan_of(const Args& g, int pairs) {
    const int counted = g.words->counted;
    Plan p;
    p.items_x = g.want_x ? (counted + kTile - 1) / kTile * g.d_tiles * g.splits_x : 0;
    p.items_w = g.want_w ? g.tiles * g.d_tiles * g.splits_w : 0;
    p.steps_x = (g.cols + kStep - 1) / kStep;
    p.steps_w = (counted + kStep - 1) / kStep;
    p.more = p.items_w % pairs;
    // a pair's end: the smallest by which all of the rows' items are done, each of them taking the longest one's time
    const int item_x = (p.steps_x + g.splits_x - 1) / g.splits_x, item_w = (p.steps_w + g.splits_w - 1) / g.splits_w;
    const int busy1 = p.items_w / pairs * item_w, busy0 = busy1 + item_w;
    auto fill = [&](int end, int busy) { return end > busy ? (end - busy) / item_x : 0; };
    int low = 0, high = busy0 + (p.items_x / pairs + 1) * item_x;      // (enough: every pair could take its share)
    while (low < high) {
        const int mid = (low + high) >> 1;
        const long long n = (long long)p.more * fill(mid, busy0) + (long long)(pairs - p.more) * fill(mid, busy1);
        if (n >= p.items_x) high = mid;
        else low = mid + 1;
    }
    p.fill0 = fill(low, busy0);
    p.fill1 = fill(low, busy1);
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

// A class's gradient straight from the accumulators: what rounding took from the rows whose own class it is, the way back through the
// normalisation (both warps of a row go through all of its columns for that), the common factor. Lane: a row of the tile.
template <typename E>
__device__ __forceinline__ void direct_rows(const Args& g, const Item& t, int r, bool live, float factor, float up, uint32_t acc, int n0, int n1, bool empty) {
    const FinishArgs& f = g.f;
    const int v = g.v0 + r;
    const int count = live ? f.own_count[v] : 0, rows = count <= kOwn ? count : 0;   // (of many rows the roundings average out)
    const E *x = static_cast<const E*>(f.x), *own = static_cast<const E*>(f.w) + (size_t)(live ? v : 0) * f.ldw;
    const int* mine = f.own + (size_t)(live ? v : 0) * kOwn;
    // sixteen columns of the sum, the rows' shares in the order of the rows
    auto columns = [&](int n, float* d) {
#pragma unroll
        for (int j = 0; j < 16; ++j) d[j] = 0.f;
        if (!empty) {
            pair::tmem_ld16(acc + n, d);
            ptx::tmem_ld_wait();
        }
        int before = -1;
        for (int i = 0; i < rows; ++i) {
            int c = kNoClass;
            for (int o = 0; o < rows; ++o) {
                const int m = __ldg(mine + o);
                if (m > before && m < c) c = m;
            }
            before = c;
            const float rest = own_rest<E>(f, c, up);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (t.n0 + n + 8 * j < f.D) {
                    float e[8];
                    Cvt<E>::unpack(__ldg(reinterpret_cast<const uint4*>(x + (size_t)c * f.Dp + t.n0 + n) + j), e);
#pragma unroll
                    for (int k = 0; k < 8; ++k) d[8 * j + k] = fmaf(rest, e[k], d[8 * j + k]);
                }
        }
    };
    auto own_columns = [&](int n, float* e) {   // (rows of D up to a multiple of 8 are there, zeros behind D)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (live && t.n0 + n + 8 * j < f.D) Cvt<E>::unpack(__ldg(reinterpret_cast<const uint4*>(own + t.n0 + n) + j), e + 8 * j);
            else
#pragma unroll
                for (int k = 0; k < 8; ++k) e[8 * j + k] = 0.f;
        }
    };
    float along = 0.f;
    if (f.norm) {
#pragma unroll 1
        for (int n = 0; n < g.d_width; n += 16) {
            float d[16], e[16];
            columns(n, d);
            own_columns(n, e);
#pragma unroll
            for (int j = 0; j < 16; ++j) along = fmaf(d[j], e[j], along);
        }
        const float iw = live ? f.iw[v] : 0.f;
        along *= iw * iw;
    }
#pragma unroll 1
    for (int n = n0; n < n1; n += 16) {
        float d[16];
        columns(n, d);
        if (f.norm) {
            float e[16];
            own_columns(n, e);
#pragma unroll
            for (int j = 0; j < 16; ++j) d[j] = fmaf(-along, e[j], d[j]);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) d[j] *= factor;
        const int col = t.n0 + n;
        const long long at = (long long)v * f.D + col;
        if (!live) continue;
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
}

template <typename E>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) grad_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args g) {
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    __shared__ Barriers bar;
    const int warp = ptx::warp_index(), lane = threadIdx.x & 31;
    const uint32_t rank = pair::cta_rank();
    __shared__ Plan plan_s;
    const int pair_index = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    volatile int* abort_flag = &bar.abort;

    if (warp == 0) {
        if (lane < kStages) { ptx::mbar_init(&bar.full[lane], 1); ptx::mbar_init(&bar.empty[lane], 1); }
        else if (lane < kStages + 2) { ptx::mbar_init(&bar.acc_full[lane - kStages], 1); ptx::mbar_init(&bar.acc_empty[lane - kStages], 16); }
        else if (lane == kStages + 2) bar.abort = 0;
        ptx::fence_mbar_init();
    } else if (warp == 1 && lane < 4) {
        ptx::prefetch_tensormap(lane == 0 ? &maps.g_rows : lane == 1 ? &maps.g_cols : lane == 2 ? &maps.x : &maps.w);
    }
    if (warp == 2) { pair::tmem_alloc(&bar.tmem, kCols); pair::tmem_relinquish(); }
    if (warp == 3 && lane == 0) plan_s = plan_of(g, pairs);
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
            int slot = 0, n = 0;
            uint32_t phase = 1;   // the first round finds the slots empty
            bool ok = true;
            const bool two = half_width > 64;
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
            }
            if (!ok && rank == 0)   // loads that are on their way arrive before the CTAs leave
                for (int j = n - 1; j >= 0 && j >= n - kStages; --j) ptx::mbar_wait(&bar.full[j % kStages], (j / kStages) & 1, 1u << 14);
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
        const int q = warp & 3, h = (warp - 4) >> 2;   // tensor-memory lanes 32 q .. + 31 (those a warp reaches), half h of the columns
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const int counted = g.words->counted;
        const float up = gradient_scale(g.words, g.f.fp16, g.f.norm), factor = g.direct ? common_factor(g.f, counted, up) : 1.f;
        int it = 0;
        while (next_item(g, p, walk, pairs, t)) {
            const bool empty = t.k0 == t.k1;           // a split without steps: zeros
            if (empty && t.rows && g.add) continue;
            const int r = t.m0 + rank * kHalf + q * 32 + lane;
            const bool live = r < (t.rows ? counted : g.cols);
            float* dst = (t.rows ? g.part_x + (size_t)t.split * g.Np * g.Dq : g.part_w + (size_t)t.split * g.piece_rows * g.Dq) + (size_t)r * g.Dq + t.n0;
            if (!empty) {
                if (!ptx::mbar_wait_relaxed(&bar.acc_full[it & 1], (it >> 1) & 1) || *abort_flag) { atomicExch(&g_head_status, 4); *abort_flag = 1; break; }
                ptx::tc_fence_after_sync();
            }
            if (g.direct && !t.rows) {
                direct_rows<E>(g, t, r, live, factor, up, tmem + lanes + (it & 1) * kTile, h * half_width, (h + 1) * half_width, empty);
                if (!empty) {
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) pair::arrive_cluster(pair::in_leader(&bar.acc_empty[it & 1]));
                    ++it;
                }
                continue;
            }
#pragma unroll 1
            for (int n = h * half_width; n < (h + 1) * half_width; n += 16) {
                float d[16] = {};
                if (!empty) {
                    pair::tmem_ld16(tmem + lanes + (it & 1) * kTile + n, d);
                    ptx::tmem_ld_wait();
                }
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (live && t.n0 + n + 8 * j < g.D) {
                        float* at = dst + n + 8 * j;
                        if (t.rows && g.add) {
                            const float4 a = reinterpret_cast<const float4*>(at)[0], b = reinterpret_cast<const float4*>(at)[1];
                            d[8 * j] += a.x; d[8 * j + 1] += a.y; d[8 * j + 2] += a.z; d[8 * j + 3] += a.w;
                            d[8 * j + 4] += b.x; d[8 * j + 5] += b.y; d[8 * j + 6] += b.z; d[8 * j + 7] += b.w;
                        }
                        store_sector(at, reinterpret_cast<const uint32_t*>(d + 8 * j));
                    }
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

template <typename E>
cudaError_t run(const Shape& s, const Saved& sv, const void* grad, const Args& a, int64_t pitch, const void* w, int64_t ldw, int dtype, cudaStream_t st) {
    Maps maps;
    const int64_t dg[2] = {pitch, s.Np}, sg[1] = {pitch}, dx[2] = {s.D, s.Np}, sx[1] = {s.Dp}, dw[2] = {s.D, s.V}, sw[1] = {ldw};
    const int along[2] = {64, kHalf}, across[2] = {64, kStep};
    if (!make_matrix_map(&maps.g_rows, grad, dtype, 2, dg, sg, along) || !make_matrix_map(&maps.g_cols, grad, dtype, 2, dg, sg, across) ||
        !make_matrix_map(&maps.x, sv.x, dtype, 2, dx, sx, across) || !make_matrix_map(&maps.w, w, dtype, 2, dw, sw, across))
        return cudaErrorInvalidValue;
    auto* kern = grad_kernel<E>;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)) return e;
    const int64_t items = (a.want_x ? s.Np / kTile * a.d_tiles * a.splits_x : 0) + (a.want_w ? (int64_t)a.tiles * a.d_tiles * a.splits_w : 0);
    const int64_t pairs = device_sm_count() / 2;
    kern<<<2 * (int)(items < pairs ? items : pairs), kThreads, kSmem, st>>>(maps, a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t products(const na1d_head& h, const Shape& s, const Saved& sv, const void* grad, const Pieces& p, int64_t v0, int64_t cols, bool add, float* part_x,
                     float* part_w, const FinishArgs& f, const void* w, int64_t ldw, cudaStream_t st) {
    Args a = {};
    a.words = sv.words; a.part_x = part_x; a.part_w = part_w;
    a.Np = s.Np; a.Dq = s.Dp; a.piece_rows = p.pitch;
    a.D = (int)s.D; a.d_tiles = p.d_tiles; a.d_width = p.d_width; a.v0 = (int)v0; a.cols = (int)cols;
    a.tiles = (int)((cols + kTile - 1) / kTile); a.splits_x = p.splits_x; a.splits_w = p.splits_w;
    a.want_x = part_x != nullptr; a.want_w = p.direct_w || part_w != nullptr; a.add = add; a.direct = p.direct_w;
    a.f = f;
    return h.dtype == NA1D_BF16 ? run<__nv_bfloat16>(s, sv, grad, a, p.pitch, w, ldw, 0, st) : run<__half>(s, sv, grad, a, p.pitch, w, ldw, 1, st);
}
int grad_read_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_head_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_head_status, &zero, sizeof(int));
    return v;
}

}  // namespace head
}  // namespace na1d
