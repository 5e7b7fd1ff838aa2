// Products of routed rows on the tensor cores (tcgen05), 16-bit types.
//
// tc_rows_kernel: out[slot, f] = sum_i W[g(slot)][f, i] x[row(slot), i].  The matrix is the first operand, so its result rows
// fill the 128 lanes of TMEM whatever the number of routed rows is; the slots are the columns, NT of them per tile (16 where a
// few rows meet each matrix and its bytes are what counts, 256 where the arithmetic does).  Both operands come by TMA in
// 64-deep slices through a ring of stages, the gathered rows by row number (four per instruction), straight into the swizzled
// layout the tensor cores read; rows behind a group's end are named out of range and arrive as zeros.  Two accumulators in
// TMEM alternate, so a tile is stored while the next one is summed.
//
// A tile's sum may go on with a second product (`rank` > 0): the group's low-rank matrix times rows u that were computed before,
// kept as hi + lo pairs of the 16-bit type (two planes), so that the intermediate's rounding (2^-16 in bf16, 2^-22 in fp16)
// stays below the result's.
//
// Few tiles with long sums are cut along the sum over the blocks of a cluster; the partial results meet in distributed shared
// memory, added in the order of the blocks.
#pragma once
#include "mps_routed_plain.cuh"
#include "mps_tc.cuh"

namespace mps {

constexpr int kTcThreads = 256;  // warps: 0 matrix loads, 1 products, 2 row loads, 3 idle, 4-7 results
constexpr int kTcFeatures = 128;
constexpr int kTcDepth = 64;
constexpr int kTcRing = 192 * 1024;  // shared memory of the stages

struct TcRows {
    CUtensorMap w, x, w2, u;  // matrices {i, f, group} or {f, i, group}; rows {i, row}; the low-rank pair's matrix and rows
    const int *group_ptr;     // NULL: one group of all slots
    const int *slot_row;      // row behind a slot; NULL: the slot itself
    int n_groups, n_slots, n_x_rows;
    int k, n;                 // summed index, result features
    int rank, rank_groups;    // depth of the second product; groups that have one (the first rank_groups)
    const void *u_base;       // rows of the second product (host side)
    int u_plane;              // rows between the hi and the lo plane of u
    int w_rows;               // rows of a matrix box (features, where they are its rows)
    bool w_shared, mn_major, gather, bf16, scatter, pair;  // pair: result stored as hi + lo planes of out
    const float *group_scale;
    void *out;
    long long out_plane;
    int split;                // blocks of a cluster, each with its part of the sum
    int *status;
};

struct TcPipe {
    uint64_t full[16], empty[16], tmem_full[2], tmem_empty[2];
    uint32_t tmem;
    int gave_up;
};

template <int NT>
struct TcShape {
    static constexpr uint32_t kStage = kTcFeatures * 128 + NT * 128;
    static constexpr int kStages = kTcRing / kStage < 12 ? kTcRing / kStage : 12;
    static constexpr uint32_t kColumns = 2 * NT < 32 ? 32 : 2 * NT;
    static constexpr uint32_t kReduce = NT <= 64 ? NT * kTcFeatures * 4 : 0;  // only small tiles are split
    static constexpr int kSplitStages = (kTcRing - (int)kReduce) / kStage < 12 ? (kTcRing - (int)kReduce) / kStage : 12;
    static size_t bytes(int n_groups) { return 1024 + kTcRing + (size_t)(3 * n_groups + 1) * sizeof(int); }
};

// A cursor over the tiles of all groups: tile numbers only rise, so the group is found by walking on.
struct TcCursor {
    const int *first, *lo, *hi;  // first tile of every group (n_groups + 1), its slots
    int group = 0;
    __device__ __forceinline__ void seek(int tile) {
        while (tile >= first[group + 1]) ++group;
    }
};

template <int NT>
__global__ void __launch_bounds__(kTcThreads, 1) tc_rows_kernel(const __grid_constant__ TcRows a) {
    using S = TcShape<NT>;
    extern __shared__ uint8_t s_raw[];
    __shared__ TcPipe pipe;
    __shared__ int s_sum[kTcThreads / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = (smem_addr(s_raw) + 1023) & ~1023u;
    int *first = reinterpret_cast<int *>(s_raw + (ring - smem_addr(s_raw)) + kTcRing);
    int *lo = first + a.n_groups + 1, *hi = lo + a.n_groups;
    const int split = a.split, part = split > 1 ? (int)cluster_rank() : 0;
    const int stages = split > 1 ? S::kSplitStages : S::kStages;
    const uint32_t partial = ring + (uint32_t)S::kSplitStages * S::kStage;  // split only

    // ---- tiles of the groups
    {
        constexpr int PER = kMaxRowGroups / kTcThreads + 1;  // a list with the ungrouped rows has one group more
        int tiles[PER], sum = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int g = tid * PER + i;
            tiles[i] = 0;
            if (g < a.n_groups) {
                int2 r = make_int2(0, a.n_slots);
                if (a.group_ptr) r = group_range(a.group_ptr, g, a.n_slots, a.status);
                lo[g] = r.x;
                hi[g] = r.y;
                tiles[i] = (r.y - r.x + NT - 1) / NT;
            }
            sum += tiles[i];
        }
        int scan = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, scan, d);
            if (lane >= d) scan += o;
        }
        if (lane == 31) s_sum[warp] = scan;
        if (tid == 0) {
            for (int i = 0; i < stages; ++i) {
                mbar_init(smem_addr(&pipe.full[i]), 1);
                mbar_init(smem_addr(&pipe.empty[i]), 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(smem_addr(&pipe.tmem_full[i]), 1);
                mbar_init(smem_addr(&pipe.tmem_empty[i]), 128);
            }
            pipe.gave_up = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        if (warp == 1) tmem_alloc(smem_addr(&pipe.tmem), S::kColumns);
        __syncthreads();
        for (int w = 0; w < warp; ++w) scan += s_sum[w];
        int at = scan - sum;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int g = tid * PER + i;
            if (g < a.n_groups) first[g] = at;
            at += tiles[i];
            if (g == a.n_groups - 1) first[a.n_groups] = at;
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    }
    const uint32_t tmem = pipe.tmem;
    volatile int *gave_up = &pipe.gave_up;
    const int feature_tiles = (a.n + kTcFeatures - 1) / kTcFeatures, main_steps = (a.k + kTcDepth - 1) / kTcDepth;
    const int rank_steps = 2 * ((a.rank + kTcDepth - 1) / kTcDepth);
    const long long n_tiles = (long long)first[a.n_groups] * feature_tiles;
    const long long worker = blockIdx.x / split, workers = gridDim.x / split;
    TcCursor cur = {first, lo, hi};

    // steps of this block for a tile of group g
    auto range = [&](int g, int &s0, int &s1) {
        const int total = main_steps + (g < a.rank_groups ? rank_steps : 0);
        s0 = (int)((long long)total * part / split);
        s1 = (int)((long long)total * (part + 1) / split);
    };

    int it = 0;        // stages used so far, this warp's count
    int turn = 0;      // tiles done so far
    for (long long tile = worker; tile < n_tiles; tile += workers, ++turn) {
        const int tt = (int)(tile / feature_tiles), f0 = (int)(tile - (long long)tt * feature_tiles) * kTcFeatures;
        cur.seek(tt);
        const int g = cur.group, slot0 = lo[g] + (tt - first[g]) * NT, slot1 = min(slot0 + NT, hi[g]);
        int s0, s1;
        range(g, s0, s1);
        const int buf = turn & 1;
        if (warp == 0) {
            if (lane == 0) {
                const int z = a.w_shared ? 0 : g;
                const int halves = a.n - f0 > 64 ? 2 : 1;  // MN-major: boxes of 64 features
                const uint32_t bytes = (a.mn_major ? halves * kBlock64 : a.w_rows * 128u) + NT * 128u;
                for (int s = s0; s < s1; ++s, ++it) {
                    const int st = it % stages;
                    mbar_wait(smem_addr(&pipe.empty[st]), ((it / stages) & 1) ^ 1, gave_up, a.status);
                    const uint32_t bar = smem_addr(&pipe.full[st]), dst = ring + st * S::kStage;
                    const bool second = s >= main_steps;
                    const int e = s - main_steps, i0 = (second ? e >> 1 : s) * kTcDepth;
                    mbar_expect(bar, bytes);
                    const CUtensorMap *m = second ? &a.w2 : &a.w;
                    if (a.mn_major)
                        for (int h = 0; h < halves; ++h) tma_3d(dst + h * kBlock64, m, f0 + h * 64, i0, second ? g : z, bar);
                    else tma_3d(dst, m, i0, f0, second ? g : z, bar);
                    if (second) tma_2d(dst + kTcFeatures * 128, &a.u, i0, (e & 1) * a.u_plane + slot0, bar);
                    else if (!a.gather) tma_2d(dst + kTcFeatures * 128, &a.x, i0, slot0, bar);
                }
            }
        } else if (warp == 1) {
            if (lane == 0) {
                mbar_wait(smem_addr(&pipe.tmem_empty[buf]), ((turn >> 1) & 1) ^ 1, gave_up, a.status);
                tc_fence_after();
                const uint32_t d = tmem + buf * NT, idesc = mma_desc(a.bf16, a.mn_major, false, NT);
                const uint64_t a_step = operand_step(a.mn_major), b_step = operand_step(false);
                for (int s = s0; s < s1; ++s, ++it) {
                    const int st = it % stages;
                    mbar_wait(smem_addr(&pipe.full[st]), (it / stages) & 1, gave_up, a.status);
                    tc_fence_after();
                    const uint32_t src = ring + st * S::kStage;
                    const uint64_t da = operand(src, a.mn_major), db = operand(src + kTcFeatures * 128, false);
                    const int left = s >= main_steps ? a.rank - ((s - main_steps) >> 1) * kTcDepth : a.k - s * kTcDepth;
                    const int steps = min(4, (left + 15) >> 4);
                    for (int i = 0; i < steps; ++i) tc_mma(d, da + i * a_step, db + i * b_step, idesc, s > s0 || i > 0);
                    tc_commit(smem_addr(&pipe.empty[st]));
                }
                tc_commit(smem_addr(&pipe.tmem_full[buf]));
            }
        } else if (warp == 2) {
            if (a.gather) {
                constexpr int SETS = (NT / 4 + 31) / 32;
                int r[SETS][4];
#pragma unroll
                for (int q = 0; q < SETS; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int slot = slot0 + (lane + 32 * q) * 4 + i;
                        r[q][i] = a.n_x_rows;  // out of range: zeros
                        if (slot < slot1) {
                            const int row = a.slot_row[slot];
                            if ((unsigned)row < (unsigned)a.n_x_rows) r[q][i] = row;
                            else atomicOr(a.status, kStatusBadIndex);
                        }
                    }
                for (int s = s0; s < s1; ++s, ++it) {
                    const int st = it % stages;
                    // every use of a stage is waited for, also where nothing is loaded: a parity tells neighbouring uses apart only
                    mbar_wait(smem_addr(&pipe.empty[st]), ((it / stages) & 1) ^ 1, gave_up, a.status);
                    __syncwarp();  // nor may a lane without rows fall behind the others
                    if (s >= main_steps) continue;
                    const uint32_t dst = ring + st * S::kStage + kTcFeatures * 128;
#pragma unroll
                    for (int q = 0; q < SETS; ++q)
                        if (lane + 32 * q < NT / 4) tma_rows(dst + (lane + 32 * q) * 512, &a.x, s * kTcDepth, r[q], smem_addr(&pipe.full[st]));
                }
                __syncwarp();
            }
        } else if (warp >= 4) {
            mbar_wait(smem_addr(&pipe.tmem_full[buf]), (turn >> 1) & 1, gave_up, a.status);
            tc_fence_after();
            const int quad = warp & 3, f = f0 + quad * 32 + lane;
            const float scale = a.group_scale ? a.group_scale[g] : 1.0f;
            uint16_t *out = (uint16_t *)a.out;
            auto store = [&](int slot, int row, float v) {
                if (f >= a.n) return;
                v *= scale;
                const long long at = (long long)(a.scatter ? row : slot) * a.n + f;
                const uint16_t h = to_16(v, a.bf16);
                out[at] = h;
                if (a.pair) out[at + a.out_plane] = to_16(v - from_16(h, a.bf16), a.bf16);
            };
#pragma unroll 1
            for (int c0 = 0; c0 < NT; c0 += 16) {
                if (slot0 + c0 >= slot1) break;
                float v[16];
                tmem_load(tmem + ((uint32_t)(quad * 32) << 16) + buf * NT + c0, v);
                if (split > 1) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(partial + ((c0 + j) * kTcFeatures + quad * 32 + lane) * 4), "f"(v[j]) : "memory");
                    continue;
                }
                int rows = 0;
                if (a.scatter && slot0 + c0 + (lane & 15) < slot1) {
                    rows = a.slot_row[slot0 + c0 + (lane & 15)];
                    if ((unsigned)rows >= (unsigned)a.n_x_rows) rows = -1;
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int row = __shfl_sync(0xffffffffu, rows, j);
                    if (slot0 + c0 + j < slot1 && row >= 0) store(slot0 + c0 + j, row, v[j]);
                }
            }
            tc_fence_before();
            mbar_arrive(smem_addr(&pipe.tmem_empty[buf]));
            if (split > 1) {
                // every block of the cluster adds up and stores its share of the columns
                cluster_sync();
                for (int c = part; slot0 + c < slot1; c += split) {
                    float v = 0.0f;
                    for (int p = 0; p < split; ++p) v += load_peer(partial + (c * kTcFeatures + quad * 32 + lane) * 4, p);
                    int row = 0;
                    if (a.scatter) {
                        row = a.slot_row[slot0 + c];
                        if ((unsigned)row >= (unsigned)a.n_x_rows) row = -1;
                    }
                    if (row >= 0) store(slot0 + c, row, v);
                }
                cluster_sync();  // the partial results may be overwritten, and no block leaves while one still reads its own
            }
        }
        if (split > 1 && warp < 4) {
            __syncwarp();
            cluster_sync();
            cluster_sync();
        }
    }
    if (*gave_up) __nanosleep(1000000);  // copies in flight land before the block's memory is given back
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, S::kColumns);
    }
}

// tc_outer_kernel: out[g][f, c] = sum over the slots s of group g of P[.., f] Q[s, c] - the gradient by a group's matrix.  The
// summed index is the slot, so both operands lie across it (MN-major): a stage holds 64 slots of 128 features of P and of up
// to NT columns of Q in blocks of 64.  Whole slices of rows in slot order come as one box per block, gathered rows and the
// last slice of a group by row number, with the rows behind the group's end named out of range: zeros, whatever lies there.
// With `pair` a block of columns of Q is a hi and a lo plane, added up when the result is stored.
struct TcOuter {
    CUtensorMap p_rows, p_tile, q_rows, q_tile;  // boxes of one row / of 64
    const int *group_ptr, *slot_row;             // slot_row: rows of P (NULL: in slot order)
    int n_groups, n_slots, n_p_rows;
    int i, j;                                    // features of P, columns of Q
    int q_plane, q_rows_all;                     // rows between the planes of Q; rows of the tensor
    bool bf16, pair;
    void *out;
    long long out_group, out_f, out_c;
    int split;
    int *status;
};

template <int NT>
struct TcOuterShape {
    static constexpr uint32_t kStage = 2 * kBlock64 + NT / 64 * kBlock64;
    static constexpr int kStages = kTcRing / kStage;
    static constexpr uint32_t kReduce = NT <= 128 ? NT * kTcFeatures * 4 : 0;
    static constexpr int kSplitStages = (kTcRing - (int)kReduce) / kStage;
    static constexpr size_t kBytes = 1024 + kTcRing;
};

template <int NT>
__global__ void __launch_bounds__(kTcThreads, 1) tc_outer_kernel(const __grid_constant__ TcOuter a) {
    using S = TcOuterShape<NT>;
    extern __shared__ uint8_t s_raw[];
    __shared__ TcPipe pipe;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = (smem_addr(s_raw) + 1023) & ~1023u;
    const int split = a.split, part = split > 1 ? (int)cluster_rank() : 0;
    const int stages = split > 1 ? S::kSplitStages : S::kStages;
    const uint32_t partial = ring + (uint32_t)S::kSplitStages * S::kStage;
    if (tid == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(smem_addr(&pipe.full[i]), 1);
            mbar_init(smem_addr(&pipe.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_addr(&pipe.tmem_full[i]), 1);
            mbar_init(smem_addr(&pipe.tmem_empty[i]), 128);
        }
        pipe.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_addr(&pipe.tmem), 2 * NT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = pipe.tmem;
    volatile int *gave_up = &pipe.gave_up;
    constexpr int COLS = NT;
    const int cols = a.pair ? COLS / 2 : COLS;  // result columns per tile
    const int i_tiles = (a.i + kTcFeatures - 1) / kTcFeatures, j_tiles = (a.j + cols - 1) / cols;
    const long long n_tiles = (long long)a.n_groups * i_tiles * j_tiles;
    const long long worker = blockIdx.x / split, workers = gridDim.x / split;
    int it = 0, turn = 0;
    for (long long tile = worker; tile < n_tiles; tile += workers, ++turn) {
        const int g = (int)(tile / ((long long)i_tiles * j_tiles)), rest = (int)(tile - (long long)g * i_tiles * j_tiles);
        const int f0 = rest / j_tiles * kTcFeatures, c0 = rest % j_tiles * cols;
        const int2 slots = group_range(a.group_ptr, g, a.n_slots, a.status);
        const int total = (slots.y - slots.x + kTcDepth - 1) / kTcDepth;
        const int s0 = (int)((long long)total * part / split), s1 = (int)((long long)total * (part + 1) / split);
        const int buf = turn & 1;
        const int p_blocks = a.i - f0 > 64 ? 2 : 1, q_blocks = a.pair ? 2 : min(NT / 64, (a.j - c0 + 63) / 64);
        if (warp == 0) {
            if (lane == 0) {
                for (int s = s0; s < s1; ++s, ++it) {
                    const int st = it % stages, slot = slots.x + s * kTcDepth;
                    mbar_wait(smem_addr(&pipe.empty[st]), ((it / stages) & 1) ^ 1, gave_up, a.status);
                    const uint32_t bar = smem_addr(&pipe.full[st]), dst = ring + st * S::kStage;
                    mbar_expect(bar, (p_blocks + q_blocks) * kBlock64);
                    if (slot + kTcDepth > slots.y) continue;  // a part of a slice: by row number
                    if (!a.slot_row)
                        for (int b = 0; b < p_blocks; ++b) tma_2d(dst + b * kBlock64, &a.p_tile, f0 + b * 64, slot, bar);
                    for (int b = 0; b < q_blocks; ++b)
                        tma_2d(dst + (2 + b) * kBlock64, &a.q_tile, a.pair ? c0 : c0 + b * 64, a.pair ? b * a.q_plane + slot : slot, bar);
                }
            }
        } else if (warp == 1) {
            if (lane == 0) {
                mbar_wait(smem_addr(&pipe.tmem_empty[buf]), ((turn >> 1) & 1) ^ 1, gave_up, a.status);
                tc_fence_after();
                const uint32_t d = tmem + buf * NT, idesc = mma_desc(a.bf16, true, true, q_blocks * 64);
                const uint64_t step = operand_step(true);
                for (int s = s0; s < s1; ++s, ++it) {
                    const int st = it % stages;
                    mbar_wait(smem_addr(&pipe.full[st]), (it / stages) & 1, gave_up, a.status);
                    tc_fence_after();
                    const uint32_t src = ring + st * S::kStage;
                    const uint64_t da = operand(src, true), db = operand(src + 2 * kBlock64, true);
                    const int steps = min(4, (slots.y - slots.x - s * kTcDepth + 15) >> 4);
                    for (int i = 0; i < steps; ++i) tc_mma(d, da + i * step, db + i * step, idesc, s > s0 || i > 0);
                    tc_commit(smem_addr(&pipe.empty[st]));
                }
                tc_commit(smem_addr(&pipe.tmem_full[buf]));
            }
        } else if (warp == 2) {
            const int q = lane & 15, half = lane >> 4;  // four slots of a slice; every other block
            int next[4];
            auto fetch = [&](int s) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int slot = slots.x + s * kTcDepth + q * 4 + i;
                    next[i] = a.n_p_rows;
                    if (s < s1 && slot < slots.y) {
                        const int row = a.slot_row ? a.slot_row[slot] : slot;
                        if ((unsigned)row < (unsigned)a.n_p_rows) next[i] = row;
                        else atomicOr(a.status, kStatusBadIndex);
                    }
                }
            };
            fetch(s0);
            for (int s = s0; s < s1; ++s, ++it) {
                int r[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = next[i];
                const int st = it % stages, slot = slots.x + s * kTcDepth;
                const bool part_slice = slot + kTcDepth > slots.y;
                if (a.slot_row) fetch(s + 1);
                else {  // the last slice of rows in slot order
#pragma unroll
                    for (int i = 0; i < 4; ++i) r[i] = slot + q * 4 + i < slots.y ? slot + q * 4 + i : a.n_p_rows;
                }
                // every use of a stage is waited for, also where nothing is loaded: a parity tells neighbouring uses apart only
                mbar_wait(smem_addr(&pipe.empty[st]), ((it / stages) & 1) ^ 1, gave_up, a.status);
                __syncwarp();  // nor may a lane without rows fall behind the others
                if (!a.slot_row && !part_slice) continue;
                const uint32_t bar = smem_addr(&pipe.full[st]), dst = ring + st * S::kStage + q * 512;
                if (half < p_blocks) tma_rows(dst + half * kBlock64, &a.p_rows, f0 + half * 64, r, bar);
                if (part_slice) {
                    for (int b = half; b < q_blocks; b += 2) {
                        int rq[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int at = slot + q * 4 + i;
                            rq[i] = at < slots.y ? (a.pair ? b * a.q_plane : 0) + at : a.q_rows_all;
                        }
                        tma_rows(dst + (2 + b) * kBlock64, &a.q_rows, a.pair ? c0 : c0 + b * 64, rq, bar);
                    }
                }
            }
            __syncwarp();
        } else if (warp >= 4) {
            mbar_wait(smem_addr(&pipe.tmem_full[buf]), (turn >> 1) & 1, gave_up, a.status);
            tc_fence_after();
            const int quad = warp & 3, f = f0 + quad * 32 + lane;
            uint16_t *out = (uint16_t *)a.out + g * a.out_group + f * a.out_f;
            const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16) + buf * NT;
            const bool none = s0 == s1;
#pragma unroll 1
            for (int c = 0; c < cols && c0 + c < a.j; c += 16) {
                float v[16] = {}, w[16];
                if (!none) {
                    tmem_load(lanes + c, v);
                    if (a.pair) {
                        tmem_load(lanes + cols + c, w);
#pragma unroll
                        for (int x = 0; x < 16; ++x) v[x] += w[x];
                    }
                }
                if (split > 1) {
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(partial + ((c + x) * kTcFeatures + quad * 32 + lane) * 4), "f"(v[x]) : "memory");
                } else {
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        if (f < a.i && c0 + c + x < a.j) out[(c0 + c + x) * a.out_c] = to_16(v[x], a.bf16);
                }
            }
            tc_fence_before();
            mbar_arrive(smem_addr(&pipe.tmem_empty[buf]));
            if (split > 1) {
                cluster_sync();
                for (int c = part; c < cols && c0 + c < a.j; c += split) {
                    float v = 0.0f;
                    for (int p = 0; p < split; ++p) v += load_peer(partial + (c * kTcFeatures + quad * 32 + lane) * 4, p);
                    if (f < a.i) out[(c0 + c) * a.out_c] = to_16(v, a.bf16);
                }
                cluster_sync();
            }
        }
        if (split > 1 && warp < 4) {
            __syncwarp();
            cluster_sync();
            cluster_sync();
        }
    }
    if (*gave_up) __nanosleep(1000000);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, 2 * NT);
    }
}

}  // namespace mps
