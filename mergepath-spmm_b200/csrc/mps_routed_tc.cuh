// Products of routed rows on the tensor cores (tcgen05), 16-bit types.
//
// tc_rows_kernel: out[slot, f] = sum_i W[g(slot)][f, i] x[row(slot), i].  The matrix is the first operand, so its result rows
// fill the 128 lanes of TMEM whatever the number of routed rows is; the slots are the columns, NT of them per tile (32 where a
// few rows meet each matrix and its bytes are what counts, 256 where the arithmetic does).  The matrices come by TMA in 64-deep
// slices through a ring of stages, rows in slot order too; gathered rows by number, four per TMA instruction, issued by one
// elected lane of each of eight warps: 0.29 us for 128 rows of a slice, about what the TMA unit gives (0.35 us from four warps,
// 0.45 us as 16-byte asynchronous copies by 128 threads, 1.2 us from 32 diverged lanes of one warp).  Two accumulators in TMEM
// alternate, so a tile is stored while the next one is summed; results go through shared memory, where 64 slots by 128 features
// become whole 256-byte rows.
//
// A tile's sum may go on with a second product (RANK): the group's low-rank matrix times rows u that were computed before, in two
// planes whose sum has fp32's range.  In bf16 they are bf16 values (off by 2^-16 of u at most) and meet the matrix as it is.  A pair
// of fp16 values has no digits left below 2^-24 and ends at 65504, and intermediates next to nothing are what training starts from
// (the second matrix begins at zero); so in fp16 they are tf32 values (2^-21), and the matrix, exactly, is in fp32
// (adapter_prepare_kernel).
//
// The widest tiles (NT = 256) belong to a pair of neighbouring blocks (cta_group::2): 256 features by 256 slots, each block
// loading its 128 features and half of the slots, so that a block's slice is 32 KB instead of 48 and six of them are in flight.
// Both blocks' loads arrive at the first one's barriers; it issues the products for both, and each stores the features it holds.
//
// Every warp that loads has something to load into every stage: the products of a slice wait for it, so it cannot fall behind
// the ring.  A warp that only waited for a stage could be lapped, and a barrier's parity does not tell uses two apart.
//
// Few tiles with long sums are cut along the sum over the blocks of a cluster; the partial results meet in distributed shared
// memory, added in the order of the blocks by the warps that store results, while the others are at the next tile.
//
// For a few rows of many adapters the shared matrix must not be read once per adapter.  Then the tiles hold rows of any adapter,
// and the result warps add u times the row's own low-rank matrix themselves (`delta`), computed in fp32 while the slices of
// the shared matrix are still coming.
#pragma once
#include "mps_routed_plain.cuh"
#include "mps_tc.cuh"

namespace mps {

constexpr int kTcThreads = 512;  // warps: 0 TMA, 1 products, 2-3 none, 4-7 results (TMEM lanes go by warp number mod 4), 8-15 row loads
constexpr int kTcFeatures = 128;
constexpr int kTcDepth = 64;
// What a launch of the row products is for.  Each is a form of its own: a short launch waits for its code to arrive, so that what one
// use needs costs the others a microsecond or two, and long ones their loops' registers (all in one form: 32,768 slots 303 us, of
// their own 286; adapters of 4096 rows 165 and 153).
enum TcUse {
    kProduct,   // rows, gathered or not, times their group's matrix
    kNarrow,    // gathered rows times narrow matrices, results in fp32 (or pairs that stand for it)
    kByRow,     // rows in order times one matrix, plus u times the matrix of each row's own adapter, by the warps that store results
    kWide16,    // rows listed by adapter times one matrix, plus a second product of the 16-bit type
    kWideTf32,  // or of tf32
};
constexpr int kTcRing = 192 * 1024;            // shared memory of the stages
constexpr int kOutPitch = kTcFeatures * 2 + 16;  // a result row in shared memory; the pad spreads 16-byte reads over the banks
constexpr int kOutBytes = 64 * kOutPitch;        // 64 rows at a time
constexpr int kF32Pitch = kTcFeatures * 4 + 16;  // 32 rows in fp32
static_assert(32 * kF32Pitch <= kOutBytes);
constexpr int kOutTotal = (kOutBytes + 1023) / 1024 * 1024;

struct TcRows {
    CUtensorMap w, x, w2, u;  // matrices {i, f, group} or {f, i, group}; rows {i, row}; the second product's {rank, f, group}, {rank, row}
    CUtensorMap x_run, u_run; // gathered rows: as many neighbouring ones as a warp loads
    const int *group_ptr;     // NULL: one group of all slots
    const int *slot_row;      // row behind a slot; NULL: the slot itself
    int n_groups, n_slots, n_x_rows;
    int k, n;                 // summed index, result features
    int rank, rank_groups;    // depth of the second product; groups that have one (the first rank_groups)
    const void *u_base, *w2_base;  // its rows, two planes of n_x_rows, and matrices (host side)
    int w_rows;               // rows of a matrix box (features, where they are its rows)
    bool mn_major, gather, bf16;
    void *out;
    float *out_f32;             // instead of out, each where not NULL: the result in fp32, by row,
    void *out_wide;             //   as two planes by row for a second product,
    uint16_t *out_slots;        //   as two planes of bf16 by slot,
    unsigned *maxima;           //   and the largest finite magnitudes of it, see finite_bits
    const float *group_scale;   // factor of a group's results then (NULL: 1)
    const int *ids;           // delta (kByRow): adapter of a row,
    const float *delta_u;     //   the rows' intermediates (by row, delta_rank each),
    const uint16_t *delta_m;  //   the adapters' matrices with their strides by adapter, feature and rank index
    int delta_adapters, delta_rank;
    long long delta_group, delta_f, delta_r;
    bool ahead;               // only delta_u comes from the launch before this one
    bool apart;               // nothing does: waited for at the end, for the launches behind
    bool next_after;          // the launch behind starts once the one before has ended (it needs that one's results, not these)
    int split;                // blocks of a cluster, each with its part of the sum (a power of two)
    bool follows;             // the launch before is one of the same call (host side)
    int *status;
};

// What a launch works on: one product or (TWO) two side by side, the second one from block `second` on, a multiple of the
// cluster.  A kernel of its own: reading every argument by index cost the single product 5 percent.
struct TcRowsLaunch {
    TcRows p[2];
    int second;
};

struct TcPipe {
    uint64_t full[12], empty[12], tmem_full[2], tmem_empty[2];  // of a pair's full and tmem_empty the first block's count
    uint64_t partials, freed;                                   // split: every block's part is in its shared memory / has been read
    uint64_t summed;                                            // the products before a tile's second one are done
    uint32_t tmem;
    int gave_up;
};

__device__ __forceinline__ void pipe_init(TcPipe &pipe, int stages, bool paired, int split) {
    for (int i = 0; i < stages; ++i) {
        mbar_init(smem_addr(&pipe.full[i]), 1);
        mbar_init(smem_addr(&pipe.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
        mbar_init(smem_addr(&pipe.tmem_full[i]), 1);
        mbar_init(smem_addr(&pipe.tmem_empty[i]), paired ? 256 : 128);
    }
    mbar_init(smem_addr(&pipe.partials), 4 * split);  // a lane of each of the four result warps of every block
    mbar_init(smem_addr(&pipe.freed), 4 * split);
    mbar_init(smem_addr(&pipe.summed), 1);
    pipe.gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

// One of the result warps tells those of all blocks of the cluster.
__device__ __forceinline__ void tell_cluster(uint32_t bar, int split, int lane) {
    fence_cluster();
    __syncwarp();
    if (lane < split) mbar_arrive_at(bar, lane);
}

// Where the parts of a tile's sums meet: block o of the cluster adds up the o-th of `split` equal runs of columns, in the order
// of the blocks.  Every block writes its part of a run into block o's shared memory (reading the others' from there took a
// microsecond a round: 13 us for 32 columns).
struct Meeting {
    uint32_t buffer;  // [blocks][columns of a run][features]
    int split, part, run;
    __device__ __forceinline__ uint32_t at(int block, int column) const { return buffer + (block * run + column % run) * (kTcFeatures * 4); }
    // eight columns from c (a multiple of eight) of one feature; start: the buffer holds something to start from where this
    // block adds up
    __device__ __forceinline__ void give(int c, int feature, const float *v, bool start) const {
        const int owner = c / run;
        const uint32_t to = at(part, c) + feature * 4;
        if (owner == part) {
#pragma unroll
            for (int j = 0; j < 8; ++j) store_shared_f32(to + j * (kTcFeatures * 4), start ? v[j] + load_shared_f32(to + j * (kTcFeatures * 4)) : v[j]);
        } else {
            const uint32_t remote = in_block(to, owner);
#pragma unroll
            for (int j = 0; j < 8; ++j) store_cluster_f32(remote + j * (kTcFeatures * 4), v[j]);
        }
    }
    __device__ __forceinline__ float sum(int column, int feature) const {
        float v = 0.0f;
        for (int p = 0; p < split; ++p) v += load_shared_f32(at(p, column) + feature * 4);
        return v;
    }
    __device__ __forceinline__ void sum8(int column, int feature, float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        for (int p = 0; p < split; ++p) {
            const uint32_t from = at(p, column) + feature * 4;
            const float4 x = load_shared_float4(from), y = load_shared_float4(from + 16);
            v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
        }
    }
};

__device__ __forceinline__ uint4 pack_16(const float (&v)[8], bool bf16) {
    return bf16 ? make_uint4(to_16x2<true>(v[0], v[1]), to_16x2<true>(v[2], v[3]), to_16x2<true>(v[4], v[5]), to_16x2<true>(v[6], v[7]))
                : make_uint4(to_16x2<false>(v[0], v[1]), to_16x2<false>(v[2], v[3]), to_16x2<false>(v[4], v[5]), to_16x2<false>(v[6], v[7]));
}

// 32 columns of one feature into 32 rows of shared memory, kOutPitch apart.  What the four result warps issue per tile is what a
// short sum waits for, so the rounding takes two values an instruction and the type is no branch per value.
template <bool BF16>
__device__ __forceinline__ void spread_column(const float (&v)[32], uint32_t to) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        const uint32_t w = to_16x2<BF16>(v[j], v[j + 1]);
        store_shared_16(to + j * kOutPitch, (uint16_t)w);
        store_shared_16(to + (j + 1) * kOutPitch, (uint16_t)(w >> 16));
    }
}

// Four values of an fp32 result from feature f, of a slot and its row (outside of x where the list is wrong: nothing by row).
__device__ __forceinline__ void store_f32(const TcRows &a, int row, int slot, int f, float4 v) {
    const bool by_row = (unsigned)row < (unsigned)a.n_x_rows;
    const long long at = (long long)row * a.n + f, plane = (long long)a.n_x_rows * a.n;
    if (a.out_f32 && by_row) *reinterpret_cast<float4 *>(a.out_f32 + at) = v;
    if (a.bf16) {
        uint2 first, second;
        split_bf16(v, first, second);
        if (a.out_wide && by_row) {
            uint16_t *to = (uint16_t *)a.out_wide + at;
            *reinterpret_cast<uint2 *>(to) = first;
            *reinterpret_cast<uint2 *>(to + plane) = second;
        }
        if (a.out_slots) {
            uint16_t *to = a.out_slots + (long long)slot * a.n + f;
            *reinterpret_cast<uint2 *>(to) = first;
            *reinterpret_cast<uint2 *>(to + (long long)a.n_slots * a.n) = second;
        }
    } else if (a.out_wide && by_row) {
        float *to = (float *)a.out_wide + at;
        *reinterpret_cast<float4 *>(to) = make_float4(tf32_first(v.x), tf32_first(v.y), tf32_first(v.z), tf32_first(v.w));
        *reinterpret_cast<float4 *>(to + plane) = make_float4(tf32_second(v.x), tf32_second(v.y), tf32_second(v.z), tf32_second(v.w));
    }
}

// Largest finite magnitudes of an fp32 result, for who scales it: of every 32 features and `span` slots of a group, counted from its
// first, an entry at [feature / 32][first of the slots].  span: kSpan, or 2 where the blocks of a cluster share a tile.
constexpr int kSpan = 32;
__device__ __forceinline__ unsigned finite_bits(float v) {
    const unsigned bits = __float_as_uint(v) & 0x7fffffffu;
    return bits < 0x7f800000u ? bits : 0u;
}

// v[j] += <u of column c + j, the feature's row of that column's matrix> over `ranks` (a multiple of eight): u in shared memory (64
// floats a column), m[j] the matrices' addresses, `stride` elements between ranks.
template <bool BF16>
__device__ __forceinline__ void add_low_rank(float (&v)[4], const uint32_t (&u)[4], const uint16_t *const (&m)[4], int ranks, long long stride) {
    for (int r = 0; r < ranks; r += 8) {
        uint32_t w[4][4];
        if (stride == 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4 *>(w[j]) = *reinterpret_cast<const uint4 *>(m[j] + r);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[j][i] = m[j][(r + 2 * i) * stride] | (uint32_t)m[j][(r + 2 * i + 1) * stride] << 16;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 x = load_shared_float4(u[j] + (r + 4 * h) * 4);
                const float2 p = from_16x2<BF16>(w[j][2 * h]), q = from_16x2<BF16>(w[j][2 * h + 1]);
                v[j] = fmaf(x.w, q.y, fmaf(x.z, q.x, fmaf(x.y, p.y, fmaf(x.x, p.x, v[j]))));
            }
    }
}

constexpr int stages_for(int bytes, int stage) { return bytes / stage < 12 ? bytes / stage : 12; }

template <int NT>
struct TcShape {
    static constexpr bool kPaired = NT == 256;
    static constexpr int kRows = kPaired ? NT / 2 : NT;  // slots a block loads
    static constexpr int kSlice = kTcFeatures * 128 + kRows * 128;  // bytes of a slice
    // Slices per stage: waiting for a stage and handing it back take a thread about 200 ns, more than the products of a slice of
    // few slots.
    static constexpr int kSlices = NT <= 64 ? 2 : 1;
    static constexpr int kStage = kSlices * kSlice;
    static constexpr int kStages = stages_for(kTcRing, kStage);
    static constexpr int kColumns = 2 * NT;
    static constexpr int kReduce = NT <= 64 ? NT * kTcFeatures * 4 : 0;  // only small tiles are split
    static constexpr int kSplitStages = stages_for(kTcRing - kReduce, kStage);
    static size_t bytes(int n_groups) { return 1024 + kTcRing + kOutTotal + (size_t)(4 * n_groups + 2) * sizeof(int); }
};

// A cursor over the tiles of all groups that have slots (a few rows of many experts leave most without, and a walk past those
// costs 40 ns each: 32 slots of 256 matrices of 2048 x 1024 40 -> 28 us).  Tile numbers only rise, so the group is found by
// walking on.  Where the matrix is shared the whole tiles of every group come first and then the groups' rests: blocks take tiles
// in turn, and the short ones at the end even out what the long ones leave (4096 rows of 8 adapters: 160 -> 152 us).  With a
// matrix per group a group's tiles stay together, its rest counted among them, or the matrices would be read twice (32 groups:
// 257 -> 270 us).
struct TcCursor {
    const int *whole, *rest, *lo, *hi;  // whole tiles before every group and (rests before it | its number << 16), n_groups + 1 each; its slots
    int n_groups, group, slot0, slot1;
    bool rests;
    __device__ __forceinline__ int number() const { return rest[group] >> 16; }
    __device__ __forceinline__ void seek(int tile, int nt) {
        const int n_whole = whole[n_groups];
        if (tile >= n_whole) {
            if (!rests) group = 0;
            rests = true;
            while (tile - n_whole >= (rest[group + 1] & 0xffff)) ++group;
            slot0 = lo[group] + (whole[group + 1] - whole[group]) * nt;
        } else {
            while (tile >= whole[group + 1]) ++group;
            slot0 = lo[group] + (tile - whole[group]) * nt;
        }
        slot1 = min(slot0 + nt, hi[group]);
    }
};

// A worker's tiles: tiles of slots by tiles of features, the features fastest; counted up, a division each is 200 cycles.
struct TileWalk {
    int tile, feature, tiles, features, step_tile, step_feature;
    __device__ __forceinline__ TileWalk(int tiles_, int features_, unsigned worker, unsigned workers)
        : tile((int)(worker / (unsigned)features_)),
          feature((int)(worker % (unsigned)features_)),
          tiles(tiles_),
          features(features_),
          step_tile((int)(workers / (unsigned)features_)),
          step_feature((int)(workers % (unsigned)features_)) {}
    __device__ __forceinline__ bool more() const { return tile < tiles; }
    __device__ __forceinline__ void next() {
        tile += step_tile;
        feature += step_feature;
        if (feature >= features) {
            feature -= features;
            ++tile;
        }
    }
};

template <int NT, TcUse USE, bool TWO>
__global__ void __launch_bounds__(kTcThreads, 1) tc_rows_kernel(const __grid_constant__ TcRowsLaunch launch) {
    const bool is_second = TWO && (int)blockIdx.x >= launch.second;
    const TcRows &a = launch.p[is_second];
    const unsigned block = blockIdx.x - (is_second ? launch.second : 0), blocks = is_second ? gridDim.x - launch.second : TWO ? launch.second : gridDim.x;
    using S = TcShape<NT>;
    extern __shared__ uint8_t s_raw[];
    __shared__ TcPipe pipe;
    __shared__ int s_sum[3][kTcThreads / 32], s_active;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = (smem_addr(s_raw) + 1023) & ~1023u, staging = ring + kTcRing;
    int *whole = reinterpret_cast<int *>(s_raw + (ring - smem_addr(s_raw)) + kTcRing + kOutTotal);
    int *rest = whole + a.n_groups + 1, *lo = rest + a.n_groups + 1, *hi = lo + a.n_groups;
    const int split = a.split, part = split > 1 ? (int)cluster_rank() : 0;
    constexpr bool RANK = USE == kWide16 || USE == kWideTf32, TF32 = USE == kWideTf32, F32 = USE == kNarrow, DELTA = USE == kByRow;
    constexpr bool SHARED = RANK || DELTA;  // one matrix
    const bool gather = USE == kProduct ? a.gather : !DELTA;
    const bool reduce = DELTA || (S::kReduce > 0 && split > 1);  // results meet in shared memory before they are stored
    const int stages = reduce ? S::kSplitStages : S::kStages;
    const uint32_t partial = ring + (uint32_t)S::kSplitStages * S::kStage;
    constexpr bool PAIRED = S::kPaired;
    const int half = PAIRED ? (int)cluster_rank() : 0, group_blocks = PAIRED ? 2 : split;

    if (!a.next_after) let_next_launch_start();
    if (warp == 0 && lane < (RANK ? 6 : 3)) {
        const CUtensorMap *maps[6] = {&a.w, &a.x, &a.x_run, &a.w2, &a.u, &a.u_run};
        if (lane != 2 || gather) tma_prefetch(maps[lane]);
    }
    if (!a.ahead && !a.apart) wait_for_launch_before();
    if (a.next_after) let_next_launch_start();
    // ---- tiles of the groups
    {
        constexpr int PER = (kMaxRowGroups + 1 + kTcThreads - 1) / kTcThreads;  // a list with the ungrouped rows has one group more
        int2 slots[PER];
        int tiles[PER], sum = 0, sum_rest = 0, active = 0;  // a whole tile counts 2, a rest 1
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int g = tid * PER + i;
            tiles[i] = 0;
            if (g < a.n_groups) {
                slots[i] = make_int2(0, a.n_slots);
                if (a.group_ptr) slots[i] = group_range(a.group_ptr, g, a.n_slots, a.status);
                const int n = slots[i].y - slots[i].x;
                tiles[i] = SHARED ? n / NT * 2 + (n % NT ? 1 : 0) : (n + NT - 1) / NT * 2;
            }
            sum += tiles[i] >> 1;
            sum_rest += tiles[i] & 1;
            active += tiles[i] > 0;
        }
        int scan = sum, scan_rest = sum_rest, scan_active = active;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, scan, d), q = __shfl_up_sync(0xffffffffu, scan_rest, d), n = __shfl_up_sync(0xffffffffu, scan_active, d);
            if (lane >= d) {
                scan += o;
                scan_rest += q;
                scan_active += n;
            }
        }
        if (lane == 31) {
            s_sum[0][warp] = scan;
            s_sum[1][warp] = scan_rest;
            s_sum[2][warp] = scan_active;
        }
        if (tid == 0) pipe_init(pipe, stages, PAIRED, split);
        if (warp == 1) tmem_alloc<PAIRED>(smem_addr(&pipe.tmem), S::kColumns);
        __syncthreads();
        const bool before = lane < warp;
        int at = scan - sum + __reduce_add_sync(0xffffffffu, before ? s_sum[0][lane] : 0);
        int at_rest = scan_rest - sum_rest + __reduce_add_sync(0xffffffffu, before ? s_sum[1][lane] : 0);
        int to = scan_active - active + __reduce_add_sync(0xffffffffu, before ? s_sum[2][lane] : 0);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int g = tid * PER + i;
            if (tiles[i] > 0) {
                whole[to] = at;
                rest[to] = at_rest | g << 16;
                lo[to] = slots[i].x;
                hi[to] = slots[i].y;
                ++to;
            }
            at += tiles[i] >> 1;
            at_rest += tiles[i] & 1;
            if (g == a.n_groups - 1) {
                whole[to] = at;
                rest[to] = at_rest;
                s_active = to;
            }
        }
        tc_fence_before();
        __syncthreads();
        if (PAIRED || split > 1) cluster_sync();  // the cluster's barriers exist before anyone arrives at them
        tc_fence_after();
    }
    const uint32_t tmem = pipe.tmem;
    volatile int *gave_up = &pipe.gave_up;
    constexpr int TILE_F = PAIRED ? 2 * kTcFeatures : kTcFeatures;
    constexpr int kRankDepth = TF32 ? 32 : 64;  // of the rank in a slice: 128 bytes
    const int main_steps = (a.k + kTcDepth - 1) / kTcDepth;
    const int rank_steps = RANK ? 2 * ((a.rank + kRankDepth - 1) / kRankDepth) : 0;  // of each plane in turn
    const int shift = split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3;
    const int n_active = s_active;
    TileWalk walk(whole[n_active] + (rest[n_active] & 0xffff), (a.n + TILE_F - 1) / TILE_F, block / group_blocks, blocks / group_blocks);
    TcCursor cur = {whole, rest, lo, hi, n_active, 0, 0, 0, false};

    // steps of this block for a tile of group g
    auto range = [&](int g, int &s0, int &s1) {
        const int total = main_steps + (RANK && g < a.rank_groups ? rank_steps : 0);
        s0 = total * part >> shift;
        s1 = total * (part + 1) >> shift;
    };

    // columns of a tile's products: only as many as there are slots, so that the last tile of a group costs what it holds
    auto columns_of = [](const TcCursor &c) { return PAIRED ? (c.slot1 - c.slot0 + 31) & ~31 : (c.slot1 - c.slot0 + 15) & ~15; };

    // gathered rows: a warp loads an eighth of a slice's, a lane holding one row's number.  Of a group's last tile only as many as
    // its products read, four at least (each warp has to load into every stage): a short tile's loads would take as long as a
    // whole one's.
    constexpr int RPW = S::kRows / 8;
    auto rows_per_warp = [&](int columns) { return min(RPW, ((PAIRED ? columns / 2 : columns) + 31) / 32 * 4); };
    int row = 0, next_row = 0;
    TcCursor ahead = cur;
    auto fetch_rows = [&](const TileWalk &w) {
        next_row = a.n_x_rows;  // out of range: zeros
        if (!w.more()) return;
        ahead.seek(w.tile, NT);
        const int columns = columns_of(ahead), mine = rows_per_warp(columns);
        const int at = (warp - 8) * mine + lane, slot = ahead.slot0 + half * columns / 2 + at;
        if (lane < mine && slot < ahead.slot1 && (!PAIRED || at < columns / 2)) {
            const int r = a.slot_row[slot];
            if ((unsigned)r < (unsigned)a.n_x_rows) next_row = r;
            else atomicOr(a.status, kStatusBadIndex);
        }
    };
    const bool loads_rows = warp >= 8 && gather;
    if (loads_rows) fetch_rows(walk);
    const uint32_t full0 = PAIRED ? in_block(smem_addr(&pipe.full[0]), 0) : smem_addr(&pipe.full[0]);  // where loads are reported
    RingAt pos;  // this warp's place in the ring
    uint32_t summed_parity = 0;

    int turn = 0;  // tiles done so far
    for (; walk.more(); walk.next(), ++turn) {
        const int f0 = walk.feature * TILE_F + half * kTcFeatures;
        cur.seek(walk.tile, NT);
        const int g = cur.number(), slot0 = cur.slot0, slot1 = cur.slot1, columns = columns_of(cur);
        int s0, s1;
        range(g, s0, s1);
        const int buf = turn & 1;
        if (warp == 0) {
            if (elect_one()) {
                const int z = SHARED ? 0 : g;
                const int halves = PAIRED || a.n - f0 > 64 ? 2 : 1;  // MN-major: boxes of 64 features (as many in both blocks)
                const uint32_t w_bytes = a.mn_major ? halves * kBlock64 : a.w_rows * 128u, own = slot0 + half * columns / 2;
                const uint32_t x_bytes = gather ? rows_per_warp(columns) * 1024u : S::kRows * 128u;
                for (int s = s0; s < s1; s += S::kSlices, pos.next(stages)) {
                    mbar_wait(smem_addr(&pipe.empty[pos.stage]), pos.parity ^ 1, gave_up, a.status);
                    const uint32_t bar = full0 + pos.stage * 8;
                    if (half == 0) {
                        uint32_t bytes = 0;
#pragma unroll
                        for (int d = 0; d < S::kSlices; ++d)
                            if (s + d < s1) bytes += (!TF32 || s + d < main_steps ? w_bytes : a.w_rows * 128u) + x_bytes;
                        mbar_expect(bar, (PAIRED ? 2 : 1) * bytes);
                    }
#pragma unroll
                    for (int d = 0; d < S::kSlices; ++d) {
                        if (d > 0 && s + d >= s1) break;
                        const uint32_t dst = ring + pos.stage * S::kStage + d * S::kSlice;
                        auto load = [&](const CUtensorMap *map, bool mn_major, int i0, int number) {
                            if (mn_major)
                                for (int h = 0; h < halves; ++h) tma_3d<PAIRED>(dst + h * kBlock64, map, f0 + h * 64, i0, number, bar);
                            else tma_3d<PAIRED>(dst, map, i0, f0, number, bar);
                        };
                        if (RANK && s + d >= main_steps) {
                            load(&a.w2, !TF32 && a.mn_major, ((s + d - main_steps) >> 1) * kRankDepth, g);
                            continue;
                        }
                        const int i0 = (s + d) * kTcDepth;
                        load(&a.w, a.mn_major, i0, z);
                        if (!gather) tma_2d<PAIRED>(dst + kTcFeatures * 128, &a.x, i0, own, bar);
                    }
                }
            }
        } else if (warp == 1) {
            if (half == 0 && elect_one()) {
                mbar_wait(smem_addr(&pipe.tmem_empty[buf]), ((turn >> 1) & 1) ^ 1, gave_up, a.status);
                tc_fence_after();
                const uint32_t d = tmem + buf * NT, idesc = mma_desc(a.bf16, a.mn_major, false, TILE_F, columns);
                const uint64_t a_step = operand_step(a.mn_major), b_step = operand_step(false);
                const uint64_t a0 = operand(ring, a.mn_major), b0 = operand(ring + kTcFeatures * 128, false), m0 = operand(ring, false);
                for (int s = s0; s < s1; s += S::kSlices, pos.next(stages)) {
                    mbar_wait(smem_addr(&pipe.full[pos.stage]), pos.parity, gave_up, a.status);
                    tc_fence_after();
#pragma unroll
                    for (int d2 = 0; d2 < S::kSlices; ++d2) {
                        if (d2 > 0 && s + d2 >= s1) break;
                        const uint32_t from = pos.stage * S::kStage + d2 * S::kSlice;
                        const bool add = s > s0 || d2 > 0;
                        const int e = s + d2 - main_steps;
                        if (!TF32 || e < 0) {
                            const int left = RANK && e >= 0 ? a.rank - (e >> 1) * kRankDepth : a.k - (s + d2) * kTcDepth;
                            tc_slice<PAIRED>(d, operand_at(a0, from), operand_at(b0, from), a_step, b_step, idesc, min(4, (left + 15) >> 4), add);
                            continue;
                        }
                        if (e == 0 && add) {  // products of another kind follow those before only once they are done
                            tc_commit<PAIRED>(smem_addr(&pipe.summed));
                            mbar_wait(smem_addr(&pipe.summed), summed_parity, gave_up, a.status);
                            summed_parity ^= 1;
                            tc_fence_after();
                        }
                        tc_slice<PAIRED, true>(d, operand_at(m0, from), operand_at(b0, from), b_step, b_step, mma_desc_tf32(TILE_F, columns),
                                               min(4, (a.rank - (e >> 1) * kRankDepth + 7) >> 3), add);
                    }
                    tc_commit<PAIRED>(smem_addr(&pipe.empty[pos.stage]));
                }
                tc_commit<PAIRED>(smem_addr(&pipe.tmem_full[buf]));
            }
        } else if (loads_rows) {
            row = next_row;
            // neighbouring rows in order (a request's, listed by adapter) come as one box
            const int row0 = __shfl_sync(0xffffffffu, row, 0);
            const int n_rows = rows_per_warp(columns);
            const bool run = n_rows == RPW && __all_sync(0xffffffffu, lane >= RPW || row == row0 + lane);
            TileWalk then = walk;
            then.next();
            fetch_rows(then);  // under way while this tile is loaded
            for (int s = s0; s < s1; s += S::kSlices, pos.next(stages)) {
                mbar_wait(smem_addr(&pipe.empty[pos.stage]), pos.parity ^ 1, gave_up, a.status);
                __syncwarp();
#pragma unroll
                for (int d = 0; d < S::kSlices; ++d) {
                    if (s + d >= s1) break;
                    const uint32_t rows = ring + pos.stage * S::kStage + d * S::kSlice + kTcFeatures * 128, bar = full0 + pos.stage * 8;
                    auto load = [&](const CUtensorMap *one, const CUtensorMap *several, int i0, int plane) {
                        if (run) {
                            if (elect_one()) tma_2d<PAIRED>(rows + (warp - 8) * RPW * 128, several, i0, plane + row0, bar);
                            return;
                        }
#pragma unroll
                        for (int q = 0; q < RPW / 4; ++q) {
                            if (4 * q >= n_rows) break;
                            const int r0 = __shfl_sync(0xffffffffu, row, 4 * q), r1 = __shfl_sync(0xffffffffu, row, 4 * q + 1);
                            const int r2 = __shfl_sync(0xffffffffu, row, 4 * q + 2), r3 = __shfl_sync(0xffffffffu, row, 4 * q + 3);
                            if (elect_one())
                                tma_rows<PAIRED>(rows + ((warp - 8) * n_rows + 4 * q) * 128, one, i0, plane + r0, plane + r1, plane + r2, plane + r3, bar);
                        }
                    };
                    const int e = s + d - main_steps;
                    if (!RANK || e < 0) load(&a.x, &a.x_run, (s + d) * kTcDepth, 0);
                    else load(&a.u, &a.u_run, (e >> 1) * kRankDepth, e & 1 ? a.n_x_rows : 0);  // the same rows of one plane of u
                }
            }
        } else if (warp >= 4 && warp < 8) {
            const int quad = warp & 3, f = f0 + quad * 32 + lane, mine = tid - 128;
            const float scale = F32 && a.group_scale ? a.group_scale[g] : 1.0f;
            uint16_t *out = (uint16_t *)a.out;
            auto out_row = [&](int slot) {  // where a slot's result goes, or -1
                if (!RANK && !F32) return slot;
                const int r = a.slot_row[slot];
                return (unsigned)r < (unsigned)a.n_x_rows ? r : -1;
            };
            auto store = [&](int slot, float v) {
                const int r = out_row(slot);
                if (f >= a.n || r < 0) return;
                out[(long long)r * a.n + f] = to_16(v, a.bf16);
            };
            // Where rows of results go is read ahead, a lane holding one of the 16 rows (of 64) that its warp stores: a load between
            // two stores would wait for both.
            auto line_ahead = [&](int c0) {
                const int slot = slot0 + c0 + 2 * (warp - 4) + (lane & 1) + 8 * ((lane & 15) >> 1);
                return slot < slot1 ? out_row(slot) : -1;
            };
            const Meeting meeting = {partial, split, part, NT / split};
            const int feature = quad * 32 + lane;
            if (reduce) {
                mbar_wait(smem_addr(&pipe.freed), (turn & 1) ^ 1, gave_up, a.status);
                if constexpr (DELTA) {
                    // The columns this block adds up start from u times the adapter's matrix.  The matrices are asked for before
                    // the wait for u; u goes through shared memory, 64 of the rank at a time; four columns' loads are in flight.
                    const int first_slot = slot0 + part * meeting.run, own = min(max(slot1 - first_slot, 0), meeting.run);
                    int id[2];  // of the columns lane and lane + 32
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        id[h] = lane + 32 * h < own ? a.ids[first_slot + lane + 32 * h] : -1;
                        if (id[h] >= a.delta_adapters) {
                            atomicOr(a.status, kStatusBadIndex);
                            id[h] = -1;
                        }
                    }
                    const int fc = min(f, a.n - 1);
                    auto matrix = [&](int c) {  // of column c; some adapter's where it has none
                        const int i = __shfl_sync(0xffffffffu, c < 32 ? id[0] : id[1], c & 31);
                        return a.delta_m + max(i, 0) * a.delta_group + fc * a.delta_f;
                    };
                    if (turn == 0) {
                        for (int c = 0; c < own; ++c) {
                            const uint16_t *m = matrix(c);
                            for (int r = 0; r < a.delta_rank; r += a.delta_r == 1 ? 64 : 1) asm volatile("prefetch.global.L2 [%0];" ::"l"(m + r * a.delta_r));
                        }
                        if (a.ahead) wait_for_launch_before();
                    }
                    for (int r0 = 0; r0 < a.delta_rank; r0 += 64) {
                        const int ranks = min(64, a.delta_rank - r0);  // multiples of eight here
                        for (int i = mine * 4; i < own * ranks; i += 128 * 4) {
                            const int c = i / ranks, r = i - c * ranks;
                            const float4 q = *reinterpret_cast<const float4 *>(a.delta_u + (long long)(first_slot + c) * a.delta_rank + r0 + r);
                            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(staging + (c * 64 + r) * 4), "f"(q.x), "f"(q.y), "f"(q.z), "f"(q.w)
                                         : "memory");
                        }
                        results_sync();
                        for (int c = 0; c < own; c += 4) {
                            const uint16_t *m[4];
                            uint32_t u[4];
                            float v[4] = {};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int cc = min(c + j, own - 1);
                                m[j] = matrix(cc) + r0 * a.delta_r;
                                u[j] = staging + cc * 64 * 4;
                            }
                            if (a.bf16) add_low_rank<true>(v, u, m, ranks, a.delta_r);
                            else add_low_rank<false>(v, u, m, ranks, a.delta_r);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int cc = c + j;
                                const bool live = __shfl_sync(0xffffffffu, cc < 32 ? id[0] : id[1], cc & 31) >= 0;
                                if (cc >= own) continue;
                                const uint32_t to = meeting.at(part, cc) + feature * 4;
                                const float have = r0 ? load_shared_f32(to) : 0.0f;
                                store_shared_f32(to, live ? have + v[j] : have);  // whatever was read for a column without one stays out
                            }
                        }
                        results_sync();  // before the next ranks' u
                    }
                }
            }
            const bool rows_of_16 = F32 || (a.n % 8 == 0 && ((uintptr_t)a.out & 15) == 0), wide = rows_of_16 && !reduce;
            int line = wide && !F32 ? line_ahead(0) : 0;
            mbar_wait(smem_addr(&pipe.tmem_full[buf]), (turn >> 1) & 1, gave_up, a.status);
            tc_fence_after();
            const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16) + buf * NT;
            if (F32 && !reduce) {
#pragma unroll 1
                for (int c0 = 0; c0 < NT && slot0 + c0 < slot1; c0 += 32) {
                    float v[32];
                    const int slot = slot0 + c0 + warp - 4 + 4 * (lane & 7);  // of the rows this warp stores
                    const int at = slot < slot1 ? out_row(slot) : -1;
                    tmem_load(lanes + c0, v);
                    unsigned largest = 0;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        v[j] *= scale;
                        if (f < a.n && slot0 + c0 + j < slot1) largest = max(largest, finite_bits(v[j]));
                    }
                    if (a.maxima) {
                        largest = __reduce_max_sync(0xffffffffu, largest);
                        if (lane == 0 && f < a.n) a.maxima[(long long)(f >> 5) * a.n_slots + slot0 + c0] = largest;
                    }
                    results_sync();  // the rows before these have been read
#pragma unroll
                    for (int j = 0; j < 32; ++j) store_shared_f32(staging + j * kF32Pitch + feature * 4, v[j]);
                    results_sync();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int to = __shfl_sync(0xffffffffu, at, j), from = slot0 + c0 + warp - 4 + 4 * j;
                        if (from < slot1 && f0 + lane * 4 < a.n)
                            store_f32(a, to, from, f0 + lane * 4, load_shared_float4(staging + (warp - 4 + 4 * j) * kF32Pitch + lane * 16));
                    }
                }
            } else if (!F32 && wide) {
                // 64 columns at a time: a result warp is alone on its scheduler, so two loads and 64 roundings in flight take little
                // more time than half of them
#pragma unroll 1
                for (int c0 = 0; c0 < NT && slot0 + c0 < slot1; c0 += 64) {
                    float v[2][32];
                    if (c0) line = line_ahead(c0);
                    tmem_start(lanes + c0, v[0]);
                    if (NT > 32) tmem_start(lanes + c0 + 32, v[1]);
                    tmem_wait(v[0]);
                    if (NT > 32) tmem_wait(v[1]);
                    results_sync();  // the rows before these have been read
#pragma unroll
                    for (int h = 0; h < (NT > 32 ? 2 : 1); ++h) {
                        if (a.bf16) spread_column<true>(v[h], staging + h * 32 * kOutPitch + feature * 2);
                        else spread_column<false>(v[h], staging + h * 32 * kOutPitch + feature * 2);
                    }
                    results_sync();
#pragma unroll
                    for (int j = 0; j < (NT > 32 ? 8 : 4); ++j) {
                        const int c = (mine >> 4) + 8 * j, fc = (mine & 15) * 8;
                        const uint4 q = load_shared_128(staging + c * kOutPitch + fc * 2);
                        const int r = __shfl_sync(0xffffffffu, line, 2 * j + (lane >> 4));
                        if (r >= 0 && f0 + fc < a.n) *reinterpret_cast<uint4 *>(out + (long long)r * a.n + f0 + fc) = q;
                    }
                }
            } else
#pragma unroll 1
            for (int c0 = 0; c0 < NT && slot0 + c0 < slot1; c0 += 32) {
                float v[32] = {};
                if (s0 < s1) tmem_load(lanes + c0, v);  // a block may have no part in a short sum
                if (reduce) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        if (slot0 + c0 + j < slot1) meeting.give(c0 + j, feature, v + j, DELTA);
                } else if (!F32) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (slot0 + c0 + j < slot1) store(slot0 + c0 + j, v[j]);
                }
            }
            tc_fence_before();
            if (PAIRED) mbar_arrive_at(smem_addr(&pipe.tmem_empty[buf]), 0);
            else mbar_arrive(smem_addr(&pipe.tmem_empty[buf]));
            if (reduce) {
                // every block of the cluster adds up and stores its share of the columns; their rows are looked up meanwhile
                const int first = part * meeting.run, own = min(max(slot1 - slot0 - first, 0), meeting.run);
                const int rows_here = rows_of_16 ? line_ahead(first) : -1;
                tell_cluster(smem_addr(&pipe.partials), split, lane);
                mbar_wait(smem_addr(&pipe.partials), turn & 1, gave_up, a.status);
                fence_cluster();
                if (rows_of_16) {
                    const int fc = (mine & 15) * 8;
                    // a half warp per column; a run is a multiple of eight, so it has the second half's column even behind the last
#pragma unroll 1
                    for (int c0 = 2 * (warp - 4), i = lane >> 4; c0 < own; c0 += 8, i += 2) {
                        const int c = c0 + (lane >> 4), slot = slot0 + first + c, r = __shfl_sync(0xffffffffu, rows_here, i);
                        const bool live = c < own && f0 + fc < a.n;
                        float v[8];
                        meeting.sum8(c, fc, v);
                        if constexpr (F32) {
                            unsigned largest = 0;
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                v[j] *= scale;
                                if (live) largest = max(largest, finite_bits(v[j]));
                            }
                            if (a.maxima) {  // of four lanes' features and both columns
                                largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                                largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                                largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 16));
                                if ((lane & 19) == 0 && f0 + fc < a.n) a.maxima[(long long)((f0 + fc) >> 5) * a.n_slots + slot0 + first + c0] = largest;
                            }
                            if (live) {
                                store_f32(a, r, slot, f0 + fc, make_float4(v[0], v[1], v[2], v[3]));
                                store_f32(a, r, slot, f0 + fc + 4, make_float4(v[4], v[5], v[6], v[7]));
                            }
                        } else if (live && r >= 0) *reinterpret_cast<uint4 *>(out + (long long)r * a.n + f0 + fc) = pack_16(v, a.bf16);
                    }
                } else
                    for (int c = 0; c < own; ++c) store(slot0 + first + c, meeting.sum(c, feature));
                tell_cluster(smem_addr(&pipe.freed), split, lane);
            }
        }
    }
    if (a.apart) wait_for_launch_before();
    if (*gave_up) __nanosleep(1000000);  // copies in flight land before the block's memory is given back
    tc_fence_before();
    __syncthreads();
    if (PAIRED || split > 1) cluster_sync();  // no block leaves while another's products, reads or arrivals still reach it
    if (warp == 1) {
        tc_fence_after();
        tmem_free<PAIRED>(tmem, S::kColumns);
    }
}

// u[row, r] = scale * <x[row], the row's adapter matrix [r]> in fp32, for a few rows: a warp per value, eight ranks per block.  The
// launch behind it may start at once; it waits for these values where it needs them.
__global__ void __launch_bounds__(256) adapter_dots_kernel(int k, int rank, int n_adapters, bool bf16, const int *__restrict__ ids,
                                                           const float *__restrict__ scale, const uint16_t *__restrict__ x,
                                                           const uint16_t *__restrict__ m, float *__restrict__ u, int *status) {
    let_next_launch_start();
    const int row = blockIdx.x, r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, id = ids[row];
    if (id < 0 || r >= rank) return;
    if (id >= n_adapters) {
        if (lane == 0) atomicOr(status, kStatusBadIndex);
        return;
    }
    const uint16_t *p = x + (long long)row * k, *q = m + ((long long)id * rank + r) * k;
    float sum = 0.0f;
#pragma unroll 8
    for (int i = lane * 8; i < k; i += 256) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p + i), b = *reinterpret_cast<const uint4 *>(q + i);
        const uint32_t v[4] = {a.x, a.y, a.z, a.w}, w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            sum = fmaf(from_16((uint16_t)(v[j >> 1] >> (j & 1) * 16), bf16), from_16((uint16_t)(w[j >> 1] >> (j & 1) * 16), bf16), sum);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) u[(long long)row * rank + r] = scale ? sum * scale[id] : sum;
}

// What the adapters' products read in another form than it came in, in fp16.  First the matrices of the groups that have slots, in
// fp32 with the rank contiguous (exact, and what a tf32 product reads by TMA); they are beside the launch before.  Behind that
// launch, for the matrix gradients, its two fp32 results as hi + lo planes in slot order (off by 2^-22 of a value; of an infinite
// value lo is zero).  fp16 has not fp32's range: a group's values of 64 columns are multiplied by the power of two that brings the
// largest of them, out of `maxima`, just below 2^15, so that what fp16 rounds away is 2^-40 of that largest at most.  Bound by
// latency and bytes: 2 read and 4 written per element of a matrix, 4 and 4 per value (8 matrices of 4096 x 64, 12 MB: 8 us by itself, on
// the SMs that the narrow product leaves).
struct PrepareArgs {
    const int *group_ptr, *slot_row;
    int n_groups, n_slots, n_rows, rank;
    const uint16_t *m;        // matrices by group, features x rank (by_rank: rank x features); NULL: none
    float *m_f32;
    int features;
    bool by_rank;
    const float *values[2];   // by row; NULL: none
    uint16_t *planes[2];
    const unsigned *maxima[2];
    int *exponents[2];
    int span, run;            // run: slots per warp, at most 32
    int *status;
};

__device__ __forceinline__ void split_fp16(float4 v, uint2 &hi, uint2 &lo) {
    hi = make_uint2(to_16x2<false>(v.x, v.y), to_16x2<false>(v.z, v.w));
    const float2 h = from_16x2<false>(hi.x), q = from_16x2<false>(hi.y);
    auto rest = [](float x, float first) { return fabsf(first) < INFINITY ? x - first : 0.0f; };
    lo = make_uint2(to_16x2<false>(rest(v.x, h.x), rest(v.y, h.y)), to_16x2<false>(rest(v.z, q.x), rest(v.w, q.y)));
}

__global__ void __launch_bounds__(256) adapter_prepare_kernel(const PrepareArgs a) {
    constexpr int N = 4;  // loads in flight
    __shared__ int s_ptr[kMaxRowGroups + 1];
    __shared__ uint16_t s_active[kMaxRowGroups];
    __shared__ int s_count[8];
    let_next_launch_start();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int g = tid; g <= a.n_groups; g += 256) s_ptr[g] = a.group_ptr[g];
    __syncthreads();
    auto range = [&](int g) { return group_range(make_int2(s_ptr[g], s_ptr[g + 1]), a.n_slots, a.status); };
    if (a.m) {
        int n_active = 0;  // groups with slots, in order
        for (int g0 = 0; g0 < a.n_groups; g0 += 256) {
            const int g = g0 + tid;
            bool active = false;
            if (g < a.n_groups) {
                const int2 slots = range(g);
                active = slots.x < slots.y;
            }
            const unsigned lanes = __ballot_sync(0xffffffffu, active);
            if (lane == 0) s_count[warp] = __popc(lanes);
            __syncthreads();
            int at = n_active + __popc(lanes & ((1u << lane) - 1));
            for (int w = 0; w < 8; ++w) {
                if (w < warp) at += s_count[w];
                n_active += s_count[w];
            }
            if (active) s_active[at] = (uint16_t)g;
            __syncthreads();
        }
        const long long size = (long long)a.features * a.rank, per = size / 8, all = n_active * per, step = (long long)gridDim.x * 256;
        for (long long i0 = (long long)blockIdx.x * 256 + tid; i0 < all; i0 += N * step) {
            uint32_t w[N][4];
            long long to[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const long long i = i0 + n * step;
                to[n] = -1;
                if (i >= all) continue;
                const int which = (int)(i / per);
                const long long first = s_active[which] * size, rest = i - which * per;
                if (a.by_rank) {  // eight ranks of a feature, neighbouring threads at neighbouring features
                    const int r = (int)(rest / a.features) * 8, f = (int)(rest - (long long)(r / 8) * a.features);
                    const uint16_t *q = a.m + first + (long long)r * a.features + f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[n][j] = q[(long long)(2 * j) * a.features] | (uint32_t)q[(long long)(2 * j + 1) * a.features] << 16;
                    to[n] = first + (long long)f * a.rank + r;
                } else {
                    const uint4 q = *reinterpret_cast<const uint4 *>(a.m + first + rest * 8);
                    w[n][0] = q.x, w[n][1] = q.y, w[n][2] = q.z, w[n][3] = q.w;
                    to[n] = first + rest * 8;
                }
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (to[n] < 0) continue;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 x = from_16x2<false>(w[n][2 * j]), y = from_16x2<false>(w[n][2 * j + 1]);
                    *reinterpret_cast<float4 *>(a.m_f32 + to[n] + 4 * j) = make_float4(x.x, x.y, y.x, y.y);
                }
            }
        }
    }
    // a warp per run of slots of either result, cut where groups end
    const int used = min(max(s_ptr[a.n_groups], 0), a.n_slots), runs = a.values[0] ? (used + a.run - 1) / a.run : 0, blocks_of_rank = (a.rank + 63) / 64;
    const int step = gridDim.x * 8;
    int run = blockIdx.x * 8 + warp;
    // Who has nothing to split makes room for the next launch's blocks; one stays, so that what waits for this launch waits for the
    // one before, too.
    if (blockIdx.x > 0 && (long long)blockIdx.x * 8 >= 2ll * runs) return;
    auto row_of = [&](int n) {  // the row of this lane's slot
        const int slot = (n >= runs ? n - runs : n) * a.run + lane, row = n < 2 * runs && lane < a.run && slot < used ? a.slot_row[slot] : -1;
        return (unsigned)row < (unsigned)a.n_rows ? row : -1;
    };
    int row = row_of(run);
    wait_for_launch_before();
    for (; run < 2 * runs; run += step, row = row_of(run)) {
        const int which = run >= runs, first = (which ? run - runs : run) * a.run, end = min(first + a.run, used);
        const float *values = a.values[which];
        const unsigned *maxima = a.maxima[which];
        int s = first;
        while (s < end) {
            int g = 0, above = a.n_groups;  // the last group that starts at s or before it
            while (above - g > 1) {
                const int mid = (g + above) >> 1;
                if (s_ptr[mid] <= s) g = mid;
                else above = mid;
            }
            const int2 slots = range(g);
            const int stop = max(min(end, slots.y), s + 1);
            for (int j = 0; j < blocks_of_rank; ++j) {
                const int pieces = min(64, a.rank - 64 * j) / 4, count = (stop - s) * pieces;
                float4 v[N];
                auto load = [&](int i0) {
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        const int i = i0 + 32 * n, r = __shfl_sync(0xffffffffu, row, (s - first + i / pieces) & 31);
                        v[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (i < count && r >= 0) v[n] = __ldcg(reinterpret_cast<const float4 *>(values + (long long)r * a.rank + 64 * j + i % pieces * 4));
                    }
                };
                load(lane);
                unsigned largest = 0;
                for (int b = 2 * j; b < 2 * j + 2 && b * 32 < a.rank; ++b)
                    for (int i = slots.x + lane * a.span; i < slots.y; i += 32 * a.span) largest = max(largest, __ldcg(maxima + (long long)b * a.n_slots + i));
                largest = __reduce_max_sync(0xffffffffu, largest);
                const int exponent = largest ? min(268 - (int)(largest >> 23), 253) : 127;  // 2^e .. 2^(e+1) to 2^14 .. 2^15; one
                const float scale = __uint_as_float((uint32_t)exponent << 23);
                if (s == slots.x && lane == 0) a.exponents[which][(long long)g * blocks_of_rank + j] = exponent;
                for (int i0 = 0; i0 < count; i0 += 32 * N) {
                    if (i0) load(i0 + lane);
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        const int i = i0 + lane + 32 * n;
                        if (i >= count) continue;
                        uint2 hi, lo;
                        split_fp16(make_float4(v[n].x * scale, v[n].y * scale, v[n].z * scale, v[n].w * scale), hi, lo);
                        uint16_t *to = a.planes[which] + (long long)(s + i / pieces) * a.rank + 64 * j + i % pieces * 4;
                        *reinterpret_cast<uint2 *>(to) = hi;
                        *reinterpret_cast<uint2 *>(to + (long long)a.n_slots * a.rank) = lo;
                    }
                }
            }
            s = stop;
        }
    }
}

// tc_outer_kernel: out[g][f, c] = sum over the slots s of group g of P[.., f] Q[s, c] - the gradient by a group's matrix.  The
// summed index is the slot, so both operands lie across it (MN-major): a stage holds 64 slots of 128 features of P and of up
// to NT columns of Q in blocks of 64.  Whole slices of rows in slot order come as a box per block; gathered rows and the last
// slice of a group by row number, those behind the group's end named out of range: zeros, whatever lies there.
// In a launch of two products (a `pair`) a block of columns of Q is a hi and a lo plane of n_slots rows, added up when the result is stored; in fp16 each group's values have
// been multiplied by a power of two (adapter_prepare_kernel), and the result is by its inverse.
struct TcOuter {
    CUtensorMap p_rows, p_tile, q_rows, q_tile;  // boxes of one row / of 64
    const int *group_ptr, *slot_row;  // slot_row: rows of P (NULL: in slot order)
    int n_groups, n_slots, n_p_rows;
    int i, j;                         // features of P, columns of Q
    bool bf16;
    const int *exponents;             // pair: the exponent field of the power of two by [group][column / 64] (NULL: one)
    void *out;
    long long out_group, out_f, out_c;
    int split;
    bool follows;
    bool apart;                       // needs nothing of the launch before, which has waited for the one before itself
    int *status;
};

struct TcOuterLaunch {
    TcOuter p[2];
    int second;
};

template <int NT>
struct TcOuterShape {
    static constexpr bool kPaired = NT == 256;
    static constexpr int kStage = 2 * kBlock64 + 2 * kBlock64;  // a block of a pair loads half of the columns
    static constexpr int kStages = stages_for(kTcRing, kStage);
    static constexpr int kReduce = NT <= 128 ? NT * kTcFeatures * 4 : 0;
    static constexpr int kSplitStages = stages_for(kTcRing - kReduce, kStage);
    static constexpr size_t kBytes = 1024 + kTcRing + kOutTotal;
};

template <int NT, bool TWO>
__global__ void __launch_bounds__(kTcThreads, 1) tc_outer_kernel(const __grid_constant__ TcOuterLaunch launch) {
    const bool is_second = TWO && (int)blockIdx.x >= launch.second;
    const TcOuter &a = launch.p[is_second];
    const int block = blockIdx.x - (is_second ? launch.second : 0), blocks = is_second ? gridDim.x - launch.second : TWO ? launch.second : gridDim.x;
    using S = TcOuterShape<NT>;
    extern __shared__ uint8_t s_raw[];
    __shared__ TcPipe pipe;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = (smem_addr(s_raw) + 1023) & ~1023u, staging = ring + kTcRing;
    const int split = S::kReduce > 0 ? a.split : 1, part = split > 1 ? (int)cluster_rank() : 0;
    const int stages = split > 1 ? S::kSplitStages : S::kStages;
    const uint32_t partial = ring + (uint32_t)S::kSplitStages * S::kStage;
    constexpr bool PAIRED = S::kPaired;
    constexpr int TILE_F = PAIRED ? 2 * kTcFeatures : kTcFeatures;
    const int half = PAIRED ? (int)cluster_rank() : 0, group_blocks = PAIRED ? 2 : split;
    let_next_launch_start();
    if (warp == 0 && lane < 4) {
        const CUtensorMap *maps[4] = {&a.p_rows, &a.p_tile, &a.q_rows, &a.q_tile};
        tma_prefetch(maps[lane]);
    }
    if (tid == 0) pipe_init(pipe, stages, PAIRED, split);
    if (warp == 1) tmem_alloc<PAIRED>(smem_addr(&pipe.tmem), 2 * NT);
    if (!a.apart) wait_for_launch_before();
    tc_fence_before();
    __syncthreads();
    if (PAIRED || split > 1) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = pipe.tmem;
    volatile int *gave_up = &pipe.gave_up;
    constexpr bool pair = TWO;
    constexpr int cols = pair ? NT / 2 : NT;  // result columns per tile
    const int i_tiles = (a.i + TILE_F - 1) / TILE_F, j_tiles = (a.j + cols - 1) / cols;
    const int per_group = i_tiles * j_tiles, n_tiles = a.n_groups * per_group;  // below 2^31 (host)
    const int worker = block / group_blocks, workers = blocks / group_blocks, shift = split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3;
    const bool gather = pair || a.slot_row != nullptr;
    const uint32_t full0 = PAIRED ? in_block(smem_addr(&pipe.full[0]), 0) : smem_addr(&pipe.full[0]);
    RingAt pos;
    int turn = -1;  // tiles with products before this one
    const int q_end = (pair ? 2 : 1) * a.n_slots;  // out of range of Q
    const bool on_16 = ((uintptr_t)a.out & 15) == 0;
    const bool wide = a.out_f == 1 && a.i % 8 == 0 && on_16, own_rows = a.out_c == 1 && a.j % 8 == 0 && on_16;  // rows of features / of columns
    int2 ends = make_int2(0, 0);  // of the next tile's group: read a tile ahead
    if (worker < n_tiles) ends = make_int2(a.group_ptr[worker / per_group], a.group_ptr[worker / per_group + 1]);
    for (int tile = worker; tile < n_tiles; tile += workers) {
        const int g = tile / per_group, rest = tile - g * per_group;
        const int2 slots = group_range(ends, a.n_slots, a.status);
        if (tile + workers < n_tiles) ends = make_int2(a.group_ptr[(tile + workers) / per_group], a.group_ptr[(tile + workers) / per_group + 1]);
        const int f0 = rest / j_tiles * TILE_F + half * kTcFeatures, c0 = rest % j_tiles * cols;
        uint16_t *out = (uint16_t *)a.out + g * a.out_group;
        if (slots.x == slots.y && split == 1 && (wide || own_rows)) {
            // a group without slots: zeros, by all warps and past the pipeline (114 groups of 128 x 3472, 112 of them without: 45 -> 24 us)
            const int n_c = min(cols, a.j - c0), n_f = min(kTcFeatures, a.i - f0), pieces = n_c >> 3;
            if (wide) {
                for (int i = tid; i < n_c * 16; i += kTcThreads)
                    if ((i & 15) * 8 < n_f) *reinterpret_cast<uint4 *>(out + (c0 + (i >> 4)) * a.out_c + f0 + (i & 15) * 8) = make_uint4(0, 0, 0, 0);
            } else
                for (int f = warp; f < n_f; f += kTcThreads / 32)
                    for (int c = lane; c < pieces; c += 32) *reinterpret_cast<uint4 *>(out + (f0 + f) * a.out_f + c0 + c * 8) = make_uint4(0, 0, 0, 0);
            continue;
        }
        ++turn;
        const int total = (slots.y - slots.x + kTcDepth - 1) / kTcDepth;
        const int s0 = (int)((long long)total * part >> shift), s1 = (int)((long long)total * (part + 1) >> shift);
        const int buf = turn & 1;
        const int p_blocks = PAIRED || a.i - f0 > 64 ? 2 : 1, q_blocks = pair || a.j - c0 > NT / 2 ? 2 : 1;
        const int q0 = c0 + half * q_blocks * 64;  // the columns this block loads
        if (warp == 0) {
            if (elect_one()) {
                const int whole = min(s1, (slots.y - slots.x) / kTcDepth);  // the slices before this one are whole
                const uint32_t bytes = (PAIRED ? 2 : 1) * (p_blocks + q_blocks) * kBlock64;
                for (int s = s0; s < whole; ++s, pos.next(stages)) {
                    const int st = pos.stage, slot = slots.x + s * kTcDepth;
                    mbar_wait(smem_addr(&pipe.empty[st]), pos.parity ^ 1, gave_up, a.status);
                    const uint32_t bar = full0 + st * 8, dst = ring + st * S::kStage;
                    if (half == 0) mbar_expect(bar, bytes);
                    if (!gather)
                        for (int b = 0; b < p_blocks; ++b) tma_2d<PAIRED>(dst + b * kBlock64, &a.p_tile, f0 + b * 64, slot, bar);
                    for (int b = 0; b < q_blocks; ++b)
                        tma_2d<PAIRED>(dst + (2 + b) * kBlock64, &a.q_tile, pair ? c0 : q0 + b * 64, pair ? b * a.n_slots + slot : slot, bar);
                }
                if (max(s0, whole) < s1) {  // part of a slice: by row number, zeros behind the group's end up to what the products read
                    const int st = pos.stage, slot = slots.x + (s1 - 1) * kTcDepth;
                    mbar_wait(smem_addr(&pipe.empty[st]), pos.parity ^ 1, gave_up, a.status);
                    const uint32_t bar = full0 + st * 8, dst = ring + st * S::kStage;
                    const int n_read = min(kTcDepth, (slots.y - slot + 15) & ~15);
                    if (half == 0) mbar_expect(bar, (PAIRED ? 2 : 1) * 128 * (p_blocks * (gather ? kTcDepth : n_read) + q_blocks * n_read));
#pragma unroll 1
                    for (int b = gather ? 2 : 0; b < 2 + q_blocks; ++b) {
                        if (b >= p_blocks && b < 2) continue;
                        const bool q = b >= 2;
                        const int x = !q ? f0 + b * 64 : pair ? c0 : q0 + (b - 2) * 64, plane = q && pair ? (b - 2) * a.n_slots : 0;
#pragma unroll 1
                        for (int i = 0; i < n_read; i += 4) {
                            auto line = [&](int j) { return slot + i + j < slots.y ? plane + slot + i + j : q ? q_end : a.n_p_rows; };
                            tma_rows<PAIRED>(dst + b * kBlock64 + i * 128, q ? &a.q_rows : &a.p_rows, x, line(0), line(1), line(2), line(3), bar);
                        }
                    }
                    pos.next(stages);
                }
            }
        } else if (warp == 1) {
            if (half == 0 && elect_one()) {
                mbar_wait(smem_addr(&pipe.tmem_empty[buf]), ((turn >> 1) & 1) ^ 1, gave_up, a.status);
                tc_fence_after();
                const uint32_t d = tmem + buf * NT, idesc = mma_desc(a.bf16, true, true, TILE_F, q_blocks * (PAIRED ? 128 : 64));
                const uint64_t step = operand_step(true), a0 = operand(ring, true), b0 = operand(ring + 2 * kBlock64, true);
                for (int s = s0; s < s1; ++s, pos.next(stages)) {
                    const int st = pos.stage;
                    mbar_wait(smem_addr(&pipe.full[st]), pos.parity, gave_up, a.status);
                    tc_fence_after();
                    tc_slice<PAIRED>(d, operand_at(a0, st * S::kStage), operand_at(b0, st * S::kStage), step, step, idesc,
                                     min(4, (slots.y - slots.x - s * kTcDepth + 15) >> 4), s > s0);
                    tc_commit<PAIRED>(smem_addr(&pipe.empty[st]));
                }
                tc_commit<PAIRED>(smem_addr(&pipe.tmem_full[buf]));
            }
        } else if (warp >= 8 && gather) {
            // rows by number, an eighth of a slice's per warp.  The numbers are read eight slices ahead: a lane holds one of the
            // warp's eight of four neighbouring slices.
            auto fetch = [&](int s) {
                const int slot = slots.x + (s + (lane >> 3)) * kTcDepth + (warp - 8) * 8 + (lane & 7);
                int r = a.n_p_rows;  // out of range: zeros
                if (s + (lane >> 3) < s1 && slot < slots.y) {
                    r = a.slot_row[slot];
                    if ((unsigned)r >= (unsigned)a.n_p_rows) {
                        atomicOr(a.status, kStatusBadIndex);
                        r = a.n_p_rows;
                    }
                }
                return r;
            };
            int now = fetch(s0), next = fetch(s0 + 4);
            for (int s = s0; s < s1; ++s, pos.next(stages)) {
                const int which = (s - s0) & 3;
                if (which == 0 && s > s0) {
                    now = next;
                    next = fetch(s + 4);
                }
                const int st = pos.stage;
                mbar_wait(smem_addr(&pipe.empty[st]), pos.parity ^ 1, gave_up, a.status);
                __syncwarp();
                const uint32_t dst = ring + st * S::kStage + (warp - 8) * 8 * 128, bar = full0 + st * 8;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int from = which * 8 + 4 * q;
                    const int r0 = __shfl_sync(0xffffffffu, now, from), r1 = __shfl_sync(0xffffffffu, now, from + 1);
                    const int r2 = __shfl_sync(0xffffffffu, now, from + 2), r3 = __shfl_sync(0xffffffffu, now, from + 3);
                    if (elect_one()) {
                        tma_rows<PAIRED>(dst + q * 512, &a.p_rows, f0, r0, r1, r2, r3, bar);
                        if (p_blocks > 1) tma_rows<PAIRED>(dst + kBlock64 + q * 512, &a.p_rows, f0 + 64, r0, r1, r2, r3, bar);
                    }
                }
            }
        } else if (warp >= 4 && warp < 8) {
            if (split > 1) mbar_wait(smem_addr(&pipe.freed), (turn & 1) ^ 1, gave_up, a.status);
            mbar_wait(smem_addr(&pipe.tmem_full[buf]), (turn >> 1) & 1, gave_up, a.status);
            tc_fence_after();
            const int quad = warp & 3, f = f0 + quad * 32 + lane, mine = tid - 128;
            const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16) + buf * NT;
            const Meeting meeting = {partial, split, part, cols / split};
            const int feature = quad * 32 + lane;
            const bool none = s0 == s1;
            float inverse = 1.0f;
            if (pair && a.exponents && slots.x < slots.y) inverse = __uint_as_float((uint32_t)(254 - __ldcg(a.exponents + (long long)g * ((a.j + 63) / 64) + (c0 >> 6))) << 23);
            // an infinite sum of hi values is the result, whatever an infinite factor made of the lo ones
            auto join = [&](float hi, float lo) {
                const float sum = hi + lo;
                return (sum == sum ? sum : hi) * inverse;
            };
            if (wide && split == 1) {
#pragma unroll 1
                for (int c = 0; c < cols && c0 + c < a.j; c += 64) {
                    float v[2][32];
#pragma unroll
                    for (int h = 0; h < 2; ++h) tmem_start(lanes + c + 32 * h, v[h]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) tmem_wait(v[h]);
                    if (pair) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float w[32];
                            tmem_load(lanes + cols + c + 32 * h, w);
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[h][x] = join(v[h][x], w[x]);
                        }
                    }
                    results_sync();  // the rows before these have been read
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (a.bf16) spread_column<true>(v[h], staging + h * 32 * kOutPitch + feature * 2);
                        else spread_column<false>(v[h], staging + h * 32 * kOutPitch + feature * 2);
                    }
                    results_sync();
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int cc = (mine >> 4) + 8 * x, fc = (mine & 15) * 8;
                        const uint4 q = load_shared_128(staging + cc * kOutPitch + fc * 2);
                        if (c0 + c + cc < a.j && f0 + fc < a.i) *reinterpret_cast<uint4 *>(out + (c0 + c + cc) * a.out_c + f0 + fc) = q;
                    }
                }
            } else
#pragma unroll 1
            for (int c = 0; c < cols && c0 + c < a.j; c += 32) {
                float v[32] = {};
                if (!none) {
                    tmem_load(lanes + c, v);
                    if (pair) {
                        float w[32];
                        tmem_load(lanes + cols + c, w);
#pragma unroll
                        for (int x = 0; x < 32; ++x) v[x] = join(v[x], w[x]);
                    }
                }
                if (split > 1) {
#pragma unroll
                    for (int x = 0; x < 32; x += 8) meeting.give(c + x, feature, v + x, false);
                } else if (own_rows) {
#pragma unroll
                    for (int x = 0; x < 32; x += 8) {
                        const float w[8] = {v[x], v[x + 1], v[x + 2], v[x + 3], v[x + 4], v[x + 5], v[x + 6], v[x + 7]};
                        if (f < a.i && c0 + c + x < a.j) *reinterpret_cast<uint4 *>(out + f * a.out_f + c0 + c + x) = pack_16(w, a.bf16);
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if (f < a.i && c0 + c + x < a.j) out[f * a.out_f + (c0 + c + x) * a.out_c] = to_16(v[x], a.bf16);
                }
            }
            tc_fence_before();
            if (PAIRED) mbar_arrive_at(smem_addr(&pipe.tmem_empty[buf]), 0);
            else mbar_arrive(smem_addr(&pipe.tmem_empty[buf]));
            if (split > 1) {
                tell_cluster(smem_addr(&pipe.partials), split, lane);
                mbar_wait(smem_addr(&pipe.partials), turn & 1, gave_up, a.status);
                fence_cluster();
                const int first = part * meeting.run, own = min(max(a.j - c0 - first, 0), meeting.run);
                for (int c = 0; c < own; ++c) {
                    const float v = meeting.sum(c, feature);
                    if (f < a.i) out[f * a.out_f + (c0 + first + c) * a.out_c] = to_16(v, a.bf16);
                }
                tell_cluster(smem_addr(&pipe.freed), split, lane);
            }
        }
    }
    if (a.apart) wait_for_launch_before();
    if (*gave_up) __nanosleep(1000000);
    tc_fence_before();
    __syncthreads();
    if (PAIRED || split > 1) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_free<PAIRED>(tmem, 2 * NT);
    }
}

}  // namespace mps
