// Products of rows with the matrix each is routed to, on the CUDA cores: any element type, any width, any alignment.
//
// One block computes a 64 x 64 tile of the result from 16-deep slices of both operands in shared memory, each thread a 4 x 4
// patch in fp32 registers.  Bound by fp32 multiply-adds; it serves fp32 and the widths a tensor map cannot describe.
#pragma once
#include "mps_types.cuh"

namespace mps {

constexpr int kPlainTile = 64, kPlainDepth = 16, kPlainThreads = 256;
constexpr int kMaxRowGroups = 1024;  // groups a block scans at once

// Start and end of group g inside [0, n_slots): whatever group_ptr holds, no slot outside the arrays is named.
__device__ __forceinline__ int2 group_range(int2 ends, int n_slots, int *status) {
    const int a = min(max(ends.x, 0), n_slots), b = min(max(ends.y, a), n_slots);
    if (a != ends.x || b != ends.y) atomicOr(status, kStatusBadIndex);
    return make_int2(a, b);
}
__device__ __forceinline__ int2 group_range(const int *group_ptr, int g, int n_slots, int *status) {
    return group_range(make_int2(group_ptr[g], group_ptr[g + 1]), n_slots, status);
}

// Group and slot range of tile number `tile` when every group is cut into tiles of `rows` slots.  Called by all THREADS
// threads of a block; false when there is no such tile.
template <int THREADS>
__device__ __forceinline__ bool find_tile(const int *group_ptr, int n_groups, int n_slots, int rows, long long tile, int *status, int &group,
                                          int &lo, int &hi) {
    constexpr int PER = kMaxRowGroups / THREADS;
    __shared__ int s_warp[THREADS / 32];
    __shared__ int s_hit[3];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int tiles[PER], sum = 0;
    if (tid == 0) s_hit[0] = -1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int g = tid * PER + i;
        tiles[i] = 0;
        if (g < n_groups) {
            const int2 r = group_range(group_ptr, g, n_slots, status);
            tiles[i] = (r.y - r.x + rows - 1) / rows;
        }
        sum += tiles[i];
    }
    int scan = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += o;
    }
    if (lane == 31) s_warp[warp] = scan;
    __syncthreads();
    for (int w = 0; w < warp; ++w) scan += s_warp[w];
    int first = scan - sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (tile >= first && tile < first + tiles[i]) {
            const int g = tid * PER + i;
            const int2 r = group_range(group_ptr, g, n_slots, status);
            s_hit[0] = g;
            s_hit[1] = r.x + (int)(tile - first) * rows;
            s_hit[2] = r.y;
        }
        first += tiles[i];
    }
    __syncthreads();
    group = s_hit[0];
    lo = s_hit[1];
    hi = min(s_hit[1] + rows, s_hit[2]);
    return group >= 0;
}

struct RowsArgs {
    const int *group_ptr;        // NULL: one group of all n_slots rows
    const int *slot_row;         // row of x behind a slot; NULL: the slot itself
    int n_groups, n_slots, n_x_rows, k, n;
    long long w_group, w_k, w_n;  // strides of the matrix by group, by summed index, by result column
    const float *group_scale;    // NULL: 1
    bool out_by_row;             // result row = row of x instead of the slot
    // low-rank part: out[row, :] += u[row, :] times the adapter's matrix
    const int *ids;
    const float *u;
    int n_adapters, rank;
    long long b_group, b_r, b_n;
    int *status;
};

template <typename T, typename TO, bool LOWRANK>
__global__ void __launch_bounds__(kPlainThreads) plain_rows_kernel(RowsArgs a, const T *__restrict__ x, const T *__restrict__ w, const T *__restrict__ b,
                                                                  TO *__restrict__ out) {
    __shared__ float s_x[kPlainDepth][kPlainTile + 4], s_w[kPlainDepth][kPlainTile + 4];
    __shared__ int s_row[kPlainTile];
    const int tid = threadIdx.x;
    int group = 0, lo = (int)blockIdx.x * kPlainTile, hi = min(lo + kPlainTile, a.n_slots);
    if (a.group_ptr && !find_tile<kPlainThreads>(a.group_ptr, a.n_groups, a.n_slots, kPlainTile, blockIdx.x, a.status, group, lo, hi)) return;
    if (tid < kPlainTile) {
        int r = -1;
        if (lo + tid < hi) {
            r = a.slot_row ? a.slot_row[lo + tid] : lo + tid;
            if ((unsigned)r >= (unsigned)a.n_x_rows) {
                atomicOr(a.status, kStatusBadIndex);
                r = -1;
            }
        }
        s_row[tid] = r;
    }
    __syncthreads();
    const T *wg = w + group * a.w_group;
    const int col0 = blockIdx.y * kPlainTile, tx = tid & 15, ty = tid >> 4;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < a.k; k0 += kPlainDepth) {
        for (int i = tid; i < kPlainTile * kPlainDepth; i += kPlainThreads) {
            const int d = i & (kPlainDepth - 1), m = i / kPlainDepth;
            const int r = s_row[m];
            s_x[d][m] = r >= 0 && k0 + d < a.k ? to_f32(x[(long long)r * a.k + k0 + d]) : 0.0f;
            // neighbouring threads walk whichever index of the matrix is contiguous
            const int wd = a.w_k == 1 ? d : i / kPlainTile, wn = a.w_k == 1 ? m : i & (kPlainTile - 1);
            s_w[wd][wn] = k0 + wd < a.k && col0 + wn < a.n ? to_f32(wg[(k0 + wd) * a.w_k + (col0 + wn) * a.w_n]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < kPlainDepth; ++d) {
            float p[4], q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { p[i] = s_x[d][ty * 4 + i]; q[i] = s_w[d][tx + 16 * i]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(p[i], q[j], acc[i][j]);
        }
        __syncthreads();
    }
    const float scale = a.group_scale ? a.group_scale[group] : 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = ty * 4 + i;
        if (lo + m >= hi) continue;
        const int r = s_row[m];
        if (a.out_by_row && r < 0) continue;
        int adapter = -1;
        if (LOWRANK) {
            adapter = a.ids[lo + m];
            if (adapter >= a.n_adapters) {
                atomicOr(a.status, kStatusBadIndex);
                adapter = -1;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = col0 + tx + 16 * j;
            if (c >= a.n) continue;
            float v = acc[i][j] * scale;
            if (LOWRANK && adapter >= 0) {
                const float *u = a.u + (long long)r * a.rank;
                const T *bb = b + adapter * a.b_group + c * a.b_n;
                for (int d = 0; d < a.rank; ++d) v = fmaf(u[d], to_f32(bb[d * a.b_r]), v);
            }
            out[(long long)(a.out_by_row ? r : lo + m) * a.n + c] = from_f32<TO>(v);
        }
    }
}

// out[g][i][j] = sum over the slots s of group g of p[.., i] q[.., j], each operand read by slot or by the slot's row.
struct OuterArgs {
    const int *group_ptr, *slot_row;
    int n_groups, n_slots, n_rows, i, j;
    bool p_by_row, q_by_row;
    int *status;
};

template <typename TP, typename TQ, typename TO>
__global__ void __launch_bounds__(kPlainThreads) plain_outer_kernel(OuterArgs a, const TP *__restrict__ p, const TQ *__restrict__ q, TO *__restrict__ out) {
    __shared__ float s_p[kPlainDepth][kPlainTile + 4], s_q[kPlainDepth][kPlainTile + 4];
    __shared__ int s_row[kPlainDepth];
    const int tid = threadIdx.x, group = blockIdx.z, tx = tid & 15, ty = tid >> 4;
    const int i0 = blockIdx.x * kPlainTile, j0 = blockIdx.y * kPlainTile;
    const int2 range = group_range(a.group_ptr, group, a.n_slots, a.status);
    float acc[4][4] = {};
    for (int s0 = range.x; s0 < range.y; s0 += kPlainDepth) {
        if (tid < kPlainDepth) {
            int r = -1;
            if (s0 + tid < range.y) {
                r = a.slot_row ? a.slot_row[s0 + tid] : s0 + tid;
                if ((unsigned)r >= (unsigned)a.n_rows) {
                    atomicOr(a.status, kStatusBadIndex);
                    r = -1;
                }
            }
            s_row[tid] = r;
        }
        __syncthreads();
        for (int e = tid; e < kPlainTile * kPlainDepth; e += kPlainThreads) {
            const int d = e / kPlainTile, m = e & (kPlainTile - 1), r = s_row[d];
            const long long rp = a.p_by_row ? r : s0 + d, rq = a.q_by_row ? r : s0 + d;
            s_p[d][m] = r >= 0 && i0 + m < a.i ? to_f32(p[rp * a.i + i0 + m]) : 0.0f;
            s_q[d][m] = r >= 0 && j0 + m < a.j ? to_f32(q[rq * a.j + j0 + m]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < kPlainDepth; ++d) {
            float u[4], v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { u[i] = s_p[d][ty * 4 + i]; v[i] = s_q[d][tx + 16 * i]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(u[i], v[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int ii = i0 + ty * 4 + i, jj = j0 + tx + 16 * j;
            if (ii < a.i && jj < a.j) out[((long long)group * a.i + ii) * a.j + jj] = from_f32<TO>(acc[i][j]);
        }
}

}  // namespace mps
