// Entry points of the products of routed rows: experts' products, their combination, low-rank adapters, and the gradients.
#include "mps.h"

#include <cuda_runtime.h>

#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "mps_internal.h"
#include "mps_routed_plain.cuh"
#include "mps_routed_tc.cuh"
#include "mps_types.cuh"

using mps::fail;
using mps::sm_count;
using mps::OuterArgs;
using mps::RowsArgs;
using mps::TcOuter;
using mps::TcRows;

namespace {

#define RD_CUDA(call)                                                                               \
    do {                                                                                            \
        cudaError_t e_ = (call);                                                                    \
        if (e_ != cudaSuccess) return fail(MPS_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_));  \
    } while (0)

__device__ int g_status;
__global__ void clear_status(int bits) { atomicAnd(&g_status, ~bits); }

int status_pointer(int **p) {
    static mps::PerDevice<int *> known;
    int dev = 0;
    RD_CUDA(cudaGetDevice(&dev));
    if ((*p = known.get(dev))) return MPS_OK;
    RD_CUDA(cudaGetSymbolAddress((void **)p, g_status));
    known.put(dev, *p);
    return MPS_OK;
}

bool misaligned(const void *p, size_t size) { return ((uintptr_t)p & (size - 1)) != 0; }
size_t size_of(int dtype) { return dtype == MPS_F32 ? 4 : 2; }

struct Span {
    const void *at;
    long long elements;
};
// Whether a result shares memory with an operand (or a result named after it), which other blocks may still have to read.
bool overlap(int dtype, std::initializer_list<Span> results, std::initializer_list<Span> operands) {
    const uintptr_t size = size_of(dtype);
    auto meet = [&](const Span &a, const Span &b) {
        const uintptr_t p = (uintptr_t)a.at, q = (uintptr_t)b.at;
        return p && q && a.elements > 0 && b.elements > 0 && p < q + (uintptr_t)b.elements * size && q < p + (uintptr_t)a.elements * size;
    };
    for (const Span *r = results.begin(); r != results.end(); ++r) {
        for (const Span &o : operands)
            if (meet(*r, o)) return true;
        for (const Span *q = r + 1; q != results.end(); ++q)
            if (meet(*r, *q)) return true;
    }
    return false;
}
bool known(int dtype) { return dtype == MPS_F32 || dtype == MPS_F16 || dtype == MPS_BF16; }

// ---------------------------------------------------------------------------------------------- combine

// 16 bytes of elements from any element's address p inside [lo, hi).  Where p is not on a 16-byte boundary two aligned loads are
// shifted into place; at the edges of the buffer, where those would reach outside, the elements come one by one.
template <typename T>
__device__ __forceinline__ mps::Pack<T> load_any(const T *p, const T *lo, const T *hi) {
    const uintptr_t at = (uintptr_t)p, m = at & 15, q = at - m;
    mps::Pack<T> out;
    if (m == 0) return *reinterpret_cast<const mps::Pack<T> *>(p);
    if (q < (uintptr_t)lo || q + 32 > (uintptr_t)hi) {
#pragma unroll
        for (int i = 0; i < mps::Pack<T>::N; ++i) out.v[i] = p[i];
        return out;
    }
    const uint4 x = *reinterpret_cast<const uint4 *>(q), y = *reinterpret_cast<const uint4 *>(q + 16);
    uint32_t a[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) a[i] = m & 8 ? a[i + 2] : a[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) a[i] = m & 4 ? a[i + 1] : a[i];
    uint32_t *o = reinterpret_cast<uint32_t *>(&out);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = m & 2 ? __funnelshift_r(a[i], a[i + 1], 16) : a[i];
    return out;
}

// A row of `dim` elements from dst in pieces: piece 0 up to dst's first 16-byte boundary, then whole 16 bytes, then what is left.
template <typename T>
struct Pieces {
    static constexpr int N = mps::Pack<T>::N;
    int head, dim;
    __device__ __forceinline__ Pieces(const T *dst, int dim_) : head((int)((16 - ((uintptr_t)dst & 15)) & 15) / (int)sizeof(T)), dim(dim_) {}
    __device__ __forceinline__ int start(int piece) const { return piece ? head + (piece - 1) * N : 0; }
    __device__ __forceinline__ int count(int piece) const { return min(piece ? N : head, dim - start(piece)); }
};
// as many as any row can have
template <typename T>
int most_pieces(int dim, bool aligned) { return (dim + mps::Pack<T>::N - 1) / mps::Pack<T>::N + (aligned ? 0 : 1); }

// y[t] = sum over j of weight[t, j] * rows[slot[t, j]].  Moves bytes only: a thread owns 16 bytes of a row of y and keeps the loads
// of several of the row's terms in flight.  ALIGNED: every row starts on a 16-byte boundary; else the pieces lie on those of y
// and the terms are shifted (14,210 rows of 8 terms of 549 fp16: 61 us, 139 element by element).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) combine_kernel(int n_rows, int per_row, int n_slots, int dim, int pieces, const int *__restrict__ slot_of,
                                                      const float *__restrict__ weights, const T *__restrict__ rows, T *__restrict__ y, int *status) {
    // blockIdx.x: rows (as many as fill 256 threads), blockIdx.y: stretches of a long row
    constexpr int N = mps::Pack<T>::N;
    const int rows_here = pieces < 256 ? 256 / pieces : 1, local = pieces < 256 ? (int)threadIdx.x / pieces : 0;
    const int piece = (int)threadIdx.x - local * pieces + (int)blockIdx.y * 256;
    if (local >= rows_here || piece >= pieces) return;
    const T *end = rows + (long long)n_slots * dim;
    for (long long t = (long long)blockIdx.x * rows_here + local; t < n_rows; t += (long long)gridDim.x * rows_here) {
        T *dst = y + t * dim;
        int from = piece * N, n = N;
        if (!ALIGNED) {
            const Pieces<T> p(dst, dim);
            from = p.start(piece);
            n = p.count(piece);
            if (n <= 0) continue;
        }
        float acc[N] = {};
#pragma unroll 4
        for (int j = 0; j < per_row; ++j) {
            const int s = slot_of[t * per_row + j];
            if (s < 0) continue;
            if (s >= n_slots) {
                atomicOr(status, mps::kStatusBadIndex);
                continue;
            }
            const float w = weights ? weights[t * per_row + j] : 1.0f;
            const T *src = rows + (long long)s * dim + from;
            if (ALIGNED || n == N) {
                const mps::Pack<T> p = ALIGNED ? *reinterpret_cast<const mps::Pack<T> *>(src) : load_any(src, rows, end);
#pragma unroll
                for (int v = 0; v < N; ++v) acc[v] = fmaf(w, mps::to_f32(p.v[v]), acc[v]);
            } else {
#pragma unroll
                for (int v = 0; v < N; ++v)
                    if (v < n) acc[v] = fmaf(w, mps::to_f32(src[v]), acc[v]);
            }
        }
        mps::Pack<T> p;
#pragma unroll
        for (int v = 0; v < N; ++v) p.v[v] = mps::from_f32<T>(acc[v]);
        if (ALIGNED || n == N) *reinterpret_cast<mps::Pack<T> *>(dst + from) = p;
        else
#pragma unroll
            for (int v = 0; v < N; ++v)
                if (v < n) dst[from + v] = p.v[v];
    }
}

// d_rows[slot[t, j]] = weight[t, j] * dy[t] and d_weights[t, j] = <dy[t], rows[slot[t, j]]>, `lanes` lanes (a power of two, as many
// as a row has pieces, 32 at most) per (t, j): rows is read and d_rows written once, the repeated reads of dy[t] meet the cache.
// ALIGNED as above, the pieces on d_rows' boundaries.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) combine_backward_kernel(int n_rows, int per_row, int n_slots, int dim, int pieces, int lanes,
                                                               const int *__restrict__ slot_of, const float *__restrict__ weights, const T *__restrict__ dy,
                                                               const T *__restrict__ rows, T *__restrict__ d_rows, float *__restrict__ d_weights, int *status) {
    constexpr int N = mps::Pack<T>::N;
    const int lane = threadIdx.x & (lanes - 1), per_warp = 32 / lanes;
    const T *end = rows + (long long)n_slots * dim, *dy_end = dy + (long long)n_rows * dim;
    const long long pairs = (long long)n_rows * per_row;
    // the lanes of a warp stay together for the sums: whole warps of pairs, some of them behind the last
    for (long long i0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * per_warp; i0 < pairs; i0 += (long long)gridDim.x * 8 * per_warp) {
        const long long i = i0 + (threadIdx.x & 31) / lanes, t = i / per_row;
        int s = i < pairs ? slot_of[i] : -1;
        if (s >= n_slots) {
            if (lane == 0) atomicOr(status, mps::kStatusBadIndex);
            s = -1;
        }
        float dot = 0.0f;
        if (s >= 0) {
            const float w = weights ? weights[i] : 1.0f;
            const T *g = dy + t * dim, *src = rows + (long long)s * dim;
            T *dst = d_rows + (long long)s * dim;
            const Pieces<T> cut(dst, dim);
#pragma unroll 4
            for (int piece = lane; piece < pieces; piece += lanes) {
                const int from = ALIGNED ? piece * N : cut.start(piece), n = ALIGNED ? N : cut.count(piece);
                if (ALIGNED || n == N) {
                    const mps::Pack<T> p = ALIGNED ? *reinterpret_cast<const mps::Pack<T> *>(g + from) : load_any(g + from, dy, dy_end);
                    mps::Pack<T> q = {}, o;
                    if (d_weights) q = ALIGNED ? *reinterpret_cast<const mps::Pack<T> *>(src + from) : load_any(src + from, rows, end);
#pragma unroll
                    for (int v = 0; v < N; ++v) {
                        const float d = mps::to_f32(p.v[v]);
                        dot = fmaf(d, mps::to_f32(q.v[v]), dot);
                        o.v[v] = mps::from_f32<T>(w * d);
                    }
                    *reinterpret_cast<mps::Pack<T> *>(dst + from) = o;
                } else {
                    for (int v = 0; v < n; ++v) {
                        const float d = mps::to_f32(g[from + v]);
                        if (d_weights) dot = fmaf(d, mps::to_f32(src[from + v]), dot);
                        dst[from + v] = mps::from_f32<T>(w * d);
                    }
                }
            }
        }
        if (d_weights) {
            for (int d = lanes >> 1; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
            if (lane == 0 && i < pairs) d_weights[i] = dot;
        }
    }
}

template <typename T>
int launch_combine(int n_rows, int per_row, int n_slots, int dim, const int *slot_of, const float *weights, const void *rows, void *y, cudaStream_t st) {
    int *status;
    if (int rc = status_pointer(&status)) return rc;
    const bool aligned = dim % mps::Pack<T>::N == 0 && !misaligned(rows, 16) && !misaligned(y, 16);
    const int pieces = most_pieces<T>(dim, aligned), rows_here = pieces < 256 ? 256 / pieces : 1;
    const long long blocks = ((long long)n_rows + rows_here - 1) / rows_here;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20), (unsigned)((pieces + 255) / 256));
    if (aligned) combine_kernel<T, true><<<grid, 256, 0, st>>>(n_rows, per_row, n_slots, dim, pieces, slot_of, weights, (const T *)rows, (T *)y, status);
    else combine_kernel<T, false><<<grid, 256, 0, st>>>(n_rows, per_row, n_slots, dim, pieces, slot_of, weights, (const T *)rows, (T *)y, status);
    RD_CUDA(cudaGetLastError());
    return MPS_OK;
}

template <typename T>
int launch_combine_backward(int n_rows, int per_row, int n_slots, int dim, const int *slot_of, const float *weights, const void *dy, const void *rows,
                            void *d_rows, float *d_weights, cudaStream_t st) {
    int *status;
    if (int rc = status_pointer(&status)) return rc;
    const bool aligned = dim % mps::Pack<T>::N == 0 && !misaligned(rows, 16) && !misaligned(dy, 16) && !misaligned(d_rows, 16);
    const int pieces = most_pieces<T>(dim, aligned);
    int lanes = 4;
    while (lanes < 32 && lanes < pieces) lanes *= 2;
    const long long blocks = ((long long)n_rows * per_row + 8 * (32 / lanes) - 1) / (8 * (32 / lanes));
    const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : 1 << 20);
    if (aligned)
        combine_backward_kernel<T, true><<<grid, 256, 0, st>>>(n_rows, per_row, n_slots, dim, pieces, lanes, slot_of, weights, (const T *)dy, (const T *)rows,
                                                               (T *)d_rows, d_weights, status);
    else
        combine_backward_kernel<T, false><<<grid, 256, 0, st>>>(n_rows, per_row, n_slots, dim, pieces, lanes, slot_of, weights, (const T *)dy, (const T *)rows,
                                                                (T *)d_rows, d_weights, status);
    RD_CUDA(cudaGetLastError());
    return MPS_OK;
}

// ---------------------------------------------------------------------------------------------- products

template <typename T, typename TO, bool LOWRANK>
int launch_plain_rows(RowsArgs a, const void *x, const void *w, const void *b, void *out, cudaStream_t st) {
    if (int rc = status_pointer(&a.status)) return rc;
    const long long tiles = (a.n_slots + mps::kPlainTile - 1) / mps::kPlainTile + (a.group_ptr ? a.n_groups : 0);  // every group ends in a part of a tile
    const dim3 grid((unsigned)tiles, (unsigned)((a.n + mps::kPlainTile - 1) / mps::kPlainTile));
    mps::plain_rows_kernel<T, TO, LOWRANK><<<grid, mps::kPlainThreads, 0, st>>>(a, (const T *)x, (const T *)w, (const T *)b, (TO *)out);
    RD_CUDA(cudaGetLastError());
    return MPS_OK;
}

template <typename TP, typename TQ, typename TO>
int launch_plain_outer(OuterArgs a, const void *p, const void *q, void *out, cudaStream_t st) {
    if (int rc = status_pointer(&a.status)) return rc;
    const dim3 grid((unsigned)((a.i + mps::kPlainTile - 1) / mps::kPlainTile), (unsigned)((a.j + mps::kPlainTile - 1) / mps::kPlainTile),
                    (unsigned)a.n_groups);
    mps::plain_outer_kernel<TP, TQ, TO><<<grid, mps::kPlainThreads, 0, st>>>(a, (const TP *)p, (const TQ *)q, (TO *)out);
    RD_CUDA(cudaGetLastError());
    return MPS_OK;
}

// ---- tensor cores

// Tensor map of `dims` sizes (innermost first, rows packed) of one of the types, read in boxes of 128 bytes by box_rows.
int tensor_map(CUtensorMap *map, int dtype, const void *base, int dims, unsigned long long d0, unsigned long long d1, unsigned long long d2, int box_rows) {
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                               const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess) fn = nullptr;
        return (Encode)fn;
    }();
    if (!encode) return fail(MPS_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const unsigned bytes = (unsigned)size_of(dtype);
    const cuuint64_t size[3] = {d0, d1, d2}, pitch[2] = {d0 * bytes, d0 * d1 * bytes};
    const cuuint32_t box[3] = {128 / bytes, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const CUtensorMapDataType type = dtype == MPS_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == MPS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult rc = encode(map, type, dims, const_cast<void *>(base), size, pitch,
                               box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(MPS_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %llu x %llu x %llu", (int)rc, d0, d1, d2);
    return MPS_OK;
}

// Lets the kernel have the device's shared memory, once per device.
template <auto Kernel>
int allow_smem() {
    static mps::PerDevice<int> allowed;  // shared memory the kernel may ask for
    int dev = 0;
    RD_CUDA(cudaGetDevice(&dev));
    if (allowed.get(dev) == 0) {
        int most = 0;
        RD_CUDA(cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev));
        cudaFuncAttributes at;
        RD_CUDA(cudaFuncGetAttributes(&at, Kernel));
        RD_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)at.sharedSizeBytes));
        allowed.put(dev, most);
    }
    return MPS_OK;
}

// Clusters of that size that the device runs at once, one block per SM.  Fewer than SMs / size: a cluster lies in one GPC (a B200
// runs 33 of four and 15 of eight).  Tiles are dealt out by block number, so a cluster that starts behind another doubles the time.
template <auto Kernel>
int clusters_at_once(int cluster, size_t smem, int sms, int *n) {
    static mps::PerDevice<int> known[4];  // of 1, 2, 4 and 8 blocks
    const int which = cluster == 1 ? 0 : cluster == 2 ? 1 : cluster == 4 ? 2 : 3;
    int dev = 0;
    RD_CUDA(cudaGetDevice(&dev));
    if ((*n = known[which].get(dev)) == 0) {
        if (int rc = allow_smem<Kernel>()) return rc;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = cluster;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(cluster);
        cfg.blockDim = dim3(mps::kTcThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        RD_CUDA(cudaOccupancyMaxActiveClusters(n, Kernel, &cfg));
        if (*n < 1) *n = 1;
        known[which].put(dev, *n);
    }
    if (*n > sms / cluster) *n = sms / cluster;  // of those left to this launch
    return MPS_OK;
}

// A launch of `blocks` blocks in clusters; `follows`: the launch before it on the stream is one of the same call, and this one may
// start before that has ended.
template <auto Kernel, typename Args>
int launch_tc(const Args &args, long long blocks, int cluster, size_t smem, bool follows, cudaStream_t st) {
    if (int rc = allow_smem<Kernel>()) return rc;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(mps::kTcThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = follows ? 2 : 1;
    RD_CUDA(cudaLaunchKernelEx(&cfg, Kernel, args));
    return MPS_OK;
}

int steps_of(int summed) { return (summed + mps::kTcDepth - 1) / mps::kTcDepth; }

// Blocks that share a tile's sum: as many as leave no SM without work, but two slices each at least.
int split_of(long long tiles, int steps, int sms) {
    int split = 1;
    while (split < 8 && tiles * split * 2 <= sms && split * 4 <= steps) split *= 2;
    return split;
}

// How the rows of a product are cut: slots per tile and blocks per tile's sum, by an estimate of the time in SM cycles.  A step of
// 64 summed elements takes the longest of its products (2 cycles a slot and 128 features), its bytes (64 a cycle and SM out of
// L2), its gathered rows (4.3 cycles each) and what its issue takes (330); a tile costs 1,500 cycles more where nothing overlaps its first loads and last
// stores, 2,500 where a cluster adds its parts.  Measured: 32,768 slots of 32 groups, 2048 x 2048: 250 us with 256 slots per
// tile; 32 slots of 64 groups, 1024 x 2048: 28 us with 32.
struct Cut {
    int nt, split;
    double cycles;
};
Cut best_cut(int slots, int groups, int features, int steps, bool gather, int sms, int most_nt) {
    const double active = groups == 1 ? 1.0 : groups * (1.0 - std::pow(1.0 - 1.0 / groups, (double)slots));  // groups that slots chosen evenly meet
    Cut best = {32, 1, 1e30};
    for (int nt = 32; nt <= most_nt; nt *= 2) {
        const bool paired = nt == 256;
        const int loaded = paired ? mps::TcShape<256>::kRows : nt, tile_f = paired ? 256 : 128;
        const double per = slots / active, tiles_of_group = groups == 1 ? std::ceil(per / nt) : std::fmax(1.0, per / nt + 0.5);
        const double tiles = active * tiles_of_group * ((features + tile_f - 1) / tile_f);
        const double bytes = 128.0 * ((features < 128 ? features : 128) + loaded);
        const double step = std::fmax(std::fmax(330.0, std::fmax(2.0 * nt + 20, bytes / 64)), gather ? 4.3 * loaded : 0.0);
        for (int split = 1; split <= (nt <= 64 ? nt / 8 : 1); split *= 2) {  // a block adds up eight columns at least
            if (split > 1 && steps < 2 * split) break;  // two slices each at least
            const double waves = std::fmax(1.0, std::ceil(tiles / (sms / (paired ? 2 : split)) - 0.05));
            const double cycles = waves * (std::ceil((double)steps / split) * step + (split > 1 ? 2500 : 1500));
            if (cycles < best.cycles) best = {nt, split, cycles};
        }
    }
    return best;
}

// Blocks for two products side by side, in proportion to their work; each at least a cluster, none more than it has tiles for.
void share_blocks(long long clusters, int cluster, const long long (&tiles)[2], const double (&work)[2], long long (&blocks)[2]) {
    if (tiles[1] && clusters < 2) clusters = 2;  // one each, whatever the device has room for
    long long first = tiles[1] ? (long long)(clusters * work[0] / (work[0] + work[1]) + 0.5) : clusters;
    if (tiles[1]) first = first < 1 ? 1 : first > clusters - 1 ? clusters - 1 : first;
    const long long second = tiles[1] < clusters - first ? tiles[1] : clusters - first;  // what one has no use for goes to the other
    first = tiles[0] < clusters - second ? tiles[0] : clusters - second;
    blocks[0] = first * cluster;
    blocks[1] = second * cluster;
}

int type_of(bool bf16) { return bf16 ? MPS_BF16 : MPS_F16; }

template <int NT, mps::TcUse USE, bool TWO = false>
int launch_tc_rows(const mps::TcRowsLaunch &in, int sms, int *used, cudaStream_t st) {
    mps::TcRowsLaunch l = in;
    const int tile_f = mps::kTcFeatures * (mps::TcShape<NT>::kPaired ? 2 : 1), cluster = mps::TcShape<NT>::kPaired ? 2 : l.p[0].split;
    long long tiles[2] = {}, blocks[2];
    double work[2] = {};
    for (int i = 0; i < (TWO ? 2 : 1); ++i) {
        const TcRows &a = l.p[i];
        const long long most = a.n_slots / NT + (a.n_groups < a.n_slots ? a.n_groups : a.n_slots);  // a group ends in a part of a tile
        tiles[i] = most * ((a.n + tile_f - 1) / tile_f);
        work[i] = (double)tiles[i] * a.k;
        if (tiles[i] >= 1LL << 31) return fail(MPS_ERR_UNSUPPORTED, "routed product: %lld tiles", tiles[i]);
    }
    const size_t smem = mps::TcShape<NT>::bytes(l.p[0].n_groups);
    int clusters;
    if (int rc = clusters_at_once<mps::tc_rows_kernel<NT, USE, TWO>>(cluster, smem, sms, &clusters)) return rc;
    share_blocks(clusters, cluster, tiles, work, blocks);
    l.second = (int)blocks[0];
    if (used) *used = (int)(blocks[0] + blocks[1]);
    return launch_tc<mps::tc_rows_kernel<NT, USE, TWO>>(l, blocks[0] + blocks[1], cluster, smem, l.p[0].follows, st);
}

// The matrices of a: stored features x summed (MN-major: summed x features), `groups` of them.
int tc_matrix(CUtensorMap *map, TcRows *a, const void *w, int summed, int features, long long groups) {
    a->w_rows = features < mps::kTcFeatures ? (features + 7) / 8 * 8 : mps::kTcFeatures;
    return a->mn_major ? tensor_map(map, type_of(a->bf16), w, 3, features, summed, groups, mps::kTcDepth)
                       : tensor_map(map, type_of(a->bf16), w, 3, summed, features, groups, a->w_rows);
}

// One product, or two narrow ones of the same groups side by side (at most 64 slots per tile): what every use has in common filled in.
// x_rows: rows of each x.  used (or NULL): the launch's blocks, each with an SM to itself.
template <mps::TcUse USE>
int tc_rows(const TcRows *products, int n, const Cut &cut, const void *const *x, long long x_rows, int sms, cudaStream_t st, int *used = nullptr) {
    mps::TcRowsLaunch l = {};
    const int loaded = cut.nt == 256 ? mps::TcShape<256>::kRows : cut.nt;  // slots a block loads
    for (int i = 0; i < n; ++i) {
        TcRows &a = l.p[i];
        a = products[i];
        if (int rc = status_pointer(&a.status)) return rc;
        a.split = cut.split;
        if (int rc = tensor_map(&a.x, type_of(a.bf16), x[i], 2, a.k, x_rows, 1, a.gather ? 1 : loaded)) return rc;
        if (a.gather)
            if (int rc = tensor_map(&a.x_run, type_of(a.bf16), x[i], 2, a.k, x_rows, 1, loaded / 8)) return rc;
        if (a.rank) {
            const int type = a.bf16 ? MPS_BF16 : MPS_F32;
            if (int rc = tensor_map(&a.u, type, a.u_base, 2, a.rank, 2ull * x_rows, 1, 1)) return rc;
            if (int rc = tensor_map(&a.u_run, type, a.u_base, 2, a.rank, 2ull * x_rows, 1, loaded / 8)) return rc;
            if (a.bf16) {
                if (int rc = tc_matrix(&a.w2, &a, a.w2_base, a.rank, a.n, a.rank_groups)) return rc;
            } else if (int rc = tensor_map(&a.w2, MPS_F32, a.w2_base, 3, a.rank, a.n, a.rank_groups, a.w_rows)) return rc;
        }
    }
    if constexpr (USE == mps::kNarrow)
        if (n == 2) return cut.nt == 32 ? launch_tc_rows<32, USE, true>(l, sms, used, st) : launch_tc_rows<64, USE, true>(l, sms, used, st);
    if (cut.nt == 32) return launch_tc_rows<32, USE>(l, sms, used, st);
    if constexpr (USE == mps::kByRow) return launch_tc_rows<64, USE>(l, sms, used, st);
    else {
        if (cut.nt == 64) return launch_tc_rows<64, USE>(l, sms, used, st);
        if (cut.nt == 128) return launch_tc_rows<128, USE>(l, sms, used, st);
        return launch_tc_rows<256, USE>(l, sms, used, st);
    }
}

template <int NT, bool TWO>
int launch_tc_outer(const mps::TcOuterLaunch &in, int sms, cudaStream_t st) {
    mps::TcOuterLaunch l = in;
    const int tile_f = mps::kTcFeatures * (mps::TcOuterShape<NT>::kPaired ? 2 : 1);
    long long tiles[2] = {}, blocks[2];
    for (int i = 0; i < (TWO ? 2 : 1); ++i) {
        const TcOuter &a = l.p[i];
        const int cols = TWO ? NT / 2 : NT;
        tiles[i] = (long long)a.n_groups * ((a.i + tile_f - 1) / tile_f) * ((a.j + cols - 1) / cols);
        if (tiles[i] >= 1LL << 31) return fail(MPS_ERR_UNSUPPORTED, "routed matrix gradient: %lld tiles", tiles[i]);
    }
    const TcOuter &a = l.p[0];
    const int steps = steps_of(a.n_slots / a.n_groups);  // of the mean group
    const int split = NT <= 128 ? split_of(tiles[0] + tiles[1], steps, sms) : 1, cluster = mps::TcOuterShape<NT>::kPaired ? 2 : split;
    l.p[0].split = l.p[1].split = split;
    const double work[2] = {(double)tiles[0], (double)tiles[1]};
    int clusters;
    if (int rc = clusters_at_once<mps::tc_outer_kernel<NT, TWO>>(cluster, mps::TcOuterShape<NT>::kBytes, sms, &clusters)) return rc;
    share_blocks(clusters, cluster, tiles, work, blocks);
    l.second = (int)blocks[0];
    return launch_tc<mps::tc_outer_kernel<NT, TWO>>(l, blocks[0] + blocks[1], cluster, mps::TcOuterShape<NT>::kBytes, a.follows, st);
}

// One gradient by the matrices, or two of the same groups side by side (of pairs of planes).  P: n_p_rows rows of a.i, by a.slot_row or in slot order;
// Q: rows of a.j in slot order (pair: two planes of them).
int tc_outer(const TcOuter *products, int n, const void *const *p, const void *const *q, int sms, cudaStream_t st) {
    mps::TcOuterLaunch l = {};
    for (int i = 0; i < n; ++i) {
        TcOuter &a = l.p[i];
        a = products[i];
        if (int rc = status_pointer(&a.status)) return rc;
        const unsigned long long q_rows = n * (unsigned long long)a.n_slots;
        if (int rc = tensor_map(&a.p_rows, type_of(a.bf16), p[i], 2, a.i, a.n_p_rows, 1, 1)) return rc;
        if (int rc = tensor_map(&a.p_tile, type_of(a.bf16), p[i], 2, a.i, a.n_p_rows, 1, mps::kTcDepth)) return rc;
        if (int rc = tensor_map(&a.q_rows, type_of(a.bf16), q[i], 2, a.j, q_rows, 1, 1)) return rc;
        if (int rc = tensor_map(&a.q_tile, type_of(a.bf16), q[i], 2, a.j, q_rows, 1, mps::kTcDepth)) return rc;
    }
    if (n == 2) return launch_tc_outer<128, true>(l, sms, st);
    return l.p[0].j <= 128 ? launch_tc_outer<128, false>(l, sms, st) : launch_tc_outer<256, false>(l, sms, st);
}

// Whether tensor maps can describe the operands: a 16-bit type, row pitches and addresses in multiples of 16 bytes.
bool tc_widths(int dtype, std::initializer_list<int> pitches, std::initializer_list<const void *> pointers) {
    if (dtype == MPS_F32) return false;
    for (int p : pitches)
        if (p % 8) return false;
    for (const void *p : pointers)
        if (misaligned(p, 16)) return false;
    return true;
}

int check_product(const char *who, int n_slots, int n_rows, int n_groups, int k, int n, int dtype) {
    if (n_slots < 0 || n_rows < 0 || n_groups < 1 || k < 1 || n < 1)
        return fail(MPS_ERR_ARG, "%s: %d slots, %d rows, %d groups, k = %d, n = %d", who, n_slots, n_rows, n_groups, k, n);
    if (!known(dtype)) return fail(MPS_ERR_ARG, "%s: unknown dtype %d", who, dtype);
    if (n_groups > mps::kMaxRowGroups) return fail(MPS_ERR_UNSUPPORTED, "%s: at most %d groups", who, mps::kMaxRowGroups);
    if (k > 1 << 21 || n > 1 << 21) return fail(MPS_ERR_UNSUPPORTED, "%s: k and n may be up to %d", who, 1 << 21);
    constexpr int most = INT32_MAX - 1024;  // the end of a tile or slice that starts before the last one is still a 32-bit number
    if (n_slots > most || n_rows > most) return fail(MPS_ERR_UNSUPPORTED, "%s: at most %d slots and rows", who, most);
    return MPS_OK;
}

// ---------------------------------------------------------------------------------------------- adapters

struct AdapterShape {
    int n_rows, k, n, n_adapters, rank, dtype;
    const int *ids, *group_ptr, *slot_row;
    const float *scale;
};

// u[row] = scale * (x[row] times the row's adapter matrix), fp32, rows without an adapter left as they were
template <typename T>
int adapter_narrow(const AdapterShape &s, int k, const void *x, const void *m, long long m_k, long long m_r, float *u, cudaStream_t st) {
    RowsArgs a = {};
    a.group_ptr = s.group_ptr;
    a.slot_row = s.slot_row;
    a.n_groups = s.n_adapters;
    a.n_slots = a.n_x_rows = s.n_rows;
    a.k = k;
    a.n = s.rank;
    a.w_group = (long long)k * s.rank;
    a.w_k = m_k;
    a.w_n = m_r;
    a.group_scale = s.scale;
    a.out_by_row = true;
    return launch_plain_rows<T, float, false>(a, x, m, nullptr, u, st);
}

// out = x times the shared matrix + u times the row's adapter matrix
template <typename T>
int adapter_wide(const AdapterShape &s, int k, int n, const void *x, const void *w, long long w_k, long long w_n, const float *u, const void *m,
                 long long m_r, long long m_n, void *out, cudaStream_t st) {
    RowsArgs a = {};
    a.n_slots = a.n_x_rows = s.n_rows;
    a.k = k;
    a.n = n;
    a.w_k = w_k;
    a.w_n = w_n;
    a.ids = s.ids;
    a.u = u;
    a.n_adapters = s.n_adapters;
    a.rank = s.rank;
    a.b_group = (long long)n * s.rank;
    a.b_r = m_r;
    a.b_n = m_n;
    return launch_plain_rows<T, T, true>(a, x, w, m, out, st);
}

// Whether the shared matrix is read once for rows of any adapter, the low-rank part added in fp32 by the warps that store the
// results (six multiply-adds a cycle and SM, 1.5 from matrices stored by rank, as measured), or per adapter, the low-rank part
// summed on the tensor cores.  Measured at 4096 x 4096 in bf16, rank 16: 64 rows of 24 adapters 20 us by rows and 81 us by
// adapter, 256 rows of 64 adapters 41 and 207, 1024 rows of 8 adapters 125 and 76; 4096 rows of 8 adapters of rank 64 1046 and 129.
// Made for the SMs of a B200 whatever the device has free, so that a call decides as its workspace's size was decided.
bool by_rows(const AdapterShape &s, int k, int n, bool by_rank, Cut *cut) {
    constexpr int sms = 148;
    const Cut grouped = best_cut(s.n_rows, s.n_adapters + 1, n, steps_of(k) + 2 * steps_of(s.rank), true, sms, 256);
    const Cut rows = best_cut(s.n_rows, 1, n, steps_of(k), false, sms, 64);
    const double low_rank = (double)s.n_rows * n * s.rank / ((by_rank ? 1.5 : 6.0) * sms);
    *cut = rows.cycles + low_rank < grouped.cycles ? rows : grouped;
    return rows.cycles + low_rank < grouped.cycles;
}

// Workspace.  The intermediates in fp32, by row; where rows are tiled by adapter the one that the wide product reads in two planes,
// by row, and in fp16 the adapters' matrices in fp32 with the rank contiguous; for the matrix gradients both intermediates in two
// planes of the type in slot order, in fp16 with their exponents and the magnitudes that these come from; then the rows listed with
// those that ask for no adapter behind the others.  Where no tensor map describes the operands the first two are all.
struct AdapterSpace {
    float *u, *v, *m;
    char *wide;
    uint16_t *u_slots, *v_slots;
    unsigned *u_maxima, *v_maxima;
    int *u_exponents, *v_exponents, *ptr, *row;
    bool rows;  // see by_rows
    Cut cut;
    int64_t bytes;
    AdapterSpace(void *base, const AdapterShape &s, bool backward) {
        char *at = (char *)base;
        auto take = [&](auto *&p, bool wanted, int64_t count) {
            p = wanted ? (std::remove_reference_t<decltype(p)>)at : nullptr;
            if (wanted) at += (count * (int64_t)sizeof(*p) + 255) / 256 * 256;
        };
        const int64_t values = (int64_t)s.n_rows * s.rank;
        const bool tc = s.dtype != MPS_F32 && s.k % 8 == 0 && s.rank % 8 == 0 && (!backward || s.n % 8 == 0), fp16 = s.dtype == MPS_F16;
        const int summed = backward ? s.n : s.k, features = backward ? s.k : s.n;  // of the wide product
        rows = by_rows(s, summed, features, backward, &cut);
        take(u, true, values);
        take(v, backward, values);
        take(wide, tc && !rows, 2 * values * (fp16 ? 4 : 2));
        take(m, tc && !rows && fp16, (int64_t)s.n_adapters * features * s.rank);
        for (int i = 0; i < 2; ++i) {
            take(i ? v_slots : u_slots, tc && backward, 2 * values);
            take(i ? v_maxima : u_maxima, tc && backward && fp16, (int64_t)s.n_rows * ((s.rank + 31) / 32));
            take(i ? v_exponents : u_exponents, tc && backward && fp16, (int64_t)s.n_adapters * ((s.rank + 63) / 64));
        }
        take(ptr, tc && !rows, s.n_adapters + 2);
        take(row, tc && !rows, s.n_rows);
        bytes = at - (char *)base;
    }
};

// The narrow product of rows of x with the adapters' matrices (mn_major: stored summed x rank): scale * x A, stored as its out_...
// pointers ask.
int tc_adapter_narrow(const AdapterShape &s, int k, const void *m, bool mn_major, TcRows *a) {
    a->bf16 = s.dtype == MPS_BF16;
    a->mn_major = mn_major;
    a->group_ptr = s.group_ptr;
    a->slot_row = s.slot_row;
    a->n_groups = s.n_adapters;
    a->n_slots = a->n_x_rows = s.n_rows;
    a->k = k;
    a->n = s.rank;
    a->gather = true;
    a->group_scale = s.scale;
    return tc_matrix(&a->w, a, m, k, s.rank, s.n_adapters);
}

// What the products behind the narrow one read in fp16, see adapter_prepare_kernel.  m (or NULL): the wide product's adapter matrices.
int tc_adapter_prepare(const AdapterShape &s, const AdapterSpace &ws, const void *m, bool by_rank, int features, bool backward, int span, int sms, cudaStream_t st) {
    mps::PrepareArgs a = {};
    a.group_ptr = s.group_ptr;
    a.slot_row = s.slot_row;
    a.n_groups = s.n_adapters;
    a.n_slots = a.n_rows = s.n_rows;
    a.rank = s.rank;
    a.m = (const uint16_t *)m;
    a.m_f32 = ws.m;
    a.features = features;
    a.by_rank = by_rank;
    a.run = 1;
    if (backward) {
        // as many slots per warp as a group has on average: a warp takes one group after the other, about a microsecond each, and
        // reads what a large one's exponent comes from again for every run of its slots
        while (a.run < 32 && 2 * a.run * s.n_adapters <= s.n_rows) a.run *= 2;
        a.values[0] = ws.u, a.values[1] = ws.v;
        a.planes[0] = ws.u_slots, a.planes[1] = ws.v_slots;
        a.maxima[0] = ws.u_maxima, a.maxima[1] = ws.v_maxima;
        a.exponents[0] = ws.u_exponents, a.exponents[1] = ws.v_exponents;
        a.span = span;
    }
    if (int rc = status_pointer(&a.status)) return rc;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * sms);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    RD_CUDA(cudaLaunchKernelEx(&cfg, mps::adapter_prepare_kernel, a));
    return MPS_OK;
}

// out = x times the shared matrix plus u times the row's adapter matrix m: of rows of any adapter (ws.rows), with u by row, or by
// adapter with the planes and matrices of the workspace.  used (or NULL): its blocks, where the launch behind it needs nothing of
// it and runs beside it.
int tc_adapter_wide(const AdapterShape &s, const AdapterSpace &ws, int k, int n, const void *x, const void *w, const float *u, const void *m, bool mn_major,
                    void *out, bool ahead, int sms, cudaStream_t st, int *used = nullptr) {
    TcRows a = {};
    a.next_after = used != nullptr;
    a.bf16 = s.dtype == MPS_BF16;
    a.mn_major = mn_major;
    a.n_slots = a.n_x_rows = s.n_rows;
    a.k = k;
    a.n = n;
    a.follows = true;
    a.out = out;
    if (int rc = tc_matrix(&a.w, &a, w, k, n, 1)) return rc;
    if (ws.rows) {
        a.n_groups = 1;
        a.ids = s.ids;
        a.delta_u = u;
        a.delta_m = (const uint16_t *)m;
        a.delta_adapters = s.n_adapters;
        a.delta_rank = s.rank;
        a.delta_group = (long long)n * s.rank;
        a.delta_f = mn_major ? 1 : s.rank;
        a.delta_r = mn_major ? n : 1;
        a.ahead = ahead;
        return tc_rows<mps::kByRow>(&a, 1, ws.cut, &x, s.n_rows, sms, st, used);
    }
    a.group_ptr = ws.ptr;
    a.slot_row = ws.row;
    a.n_groups = s.n_adapters + 1;
    a.rank = s.rank;
    a.rank_groups = s.n_adapters;
    a.u_base = ws.wide;
    a.w2_base = a.bf16 ? m : ws.m;
    a.gather = true;
    return a.bf16 ? tc_rows<mps::kWide16>(&a, 1, ws.cut, &x, s.n_rows, sms, st, used) : tc_rows<mps::kWideTf32>(&a, 1, ws.cut, &x, s.n_rows, sms, st, used);
}

TcOuter tc_adapter_outer(const AdapterShape &s, int features, const int *exponents, void *out, long long out_f, long long out_c) {
    TcOuter a = {};
    a.bf16 = s.dtype == MPS_BF16;
    a.group_ptr = s.group_ptr;
    a.slot_row = s.slot_row;
    a.n_groups = s.n_adapters;
    a.n_slots = a.n_p_rows = s.n_rows;
    a.i = features;
    a.j = s.rank;
    a.follows = a.apart = true;  // beside the rows' gradient
    a.exponents = exponents;
    a.out = out;
    a.out_group = (long long)features * s.rank;
    a.out_f = out_f;
    a.out_c = out_c;
    return a;
}

template <typename T>
int adapters(const AdapterShape &s, const void *x, const void *w, const void *a, const void *b, void *y, void *workspace, cudaStream_t st) {
    const AdapterSpace ws(workspace, s, false);
    if (tc_widths(s.dtype, {s.k, s.rank}, {x, w, a, b})) {
        int sms, *status;
        if (int rc = sm_count(&sms)) return rc;
        if (int rc = status_pointer(&status)) return rc;
        if (ws.rows) {
            const dim3 grid((unsigned)s.n_rows, (unsigned)((s.rank + 7) / 8));
            mps::adapter_dots_kernel<<<grid, 256, 0, st>>>(s.k, s.rank, s.n_adapters, s.dtype == MPS_BF16, s.ids, s.scale, (const uint16_t *)x,
                                                           (const uint16_t *)a, ws.u, status);
            RD_CUDA(cudaGetLastError());
        } else {
            if (int rc = mps::list_rows_and_rest(s.n_rows, s.n_adapters, s.ids, ws.ptr, ws.row, st)) return rc;
            TcRows narrow = {};
            if (int rc = tc_adapter_narrow(s, s.k, a, false, &narrow)) return rc;
            narrow.out_wide = ws.wide;
            narrow.follows = narrow.apart = true;  // beside the listing
            if (int rc = tc_rows<mps::kNarrow>(&narrow, 1, best_cut(s.n_rows, s.n_adapters, s.rank, steps_of(s.k), true, sms, 256), &x, s.n_rows, sms, st)) return rc;
            if (s.dtype == MPS_F16)
                if (int rc = tc_adapter_prepare(s, ws, b, false, s.n, false, 0, sms, st)) return rc;
        }
        return tc_adapter_wide(s, ws, s.k, s.n, x, w, ws.u, b, false, y, ws.rows, sms, st);
    }
    if (int rc = adapter_narrow<T>(s, s.k, x, a, 1, s.k, ws.u, st)) return rc;
    return adapter_wide<T>(s, s.k, s.n, x, w, 1, s.k, ws.u, b, 1, s.rank, y, st);
}

template <typename T>
int adapters_backward(const AdapterShape &s, const void *dy, const void *x, const void *w, const void *a, const void *b, void *dx, void *da, void *db,
                      void *workspace, cudaStream_t st) {
    const AdapterSpace ws(workspace, s, true);
    if (tc_widths(s.dtype, {s.k, s.n, s.rank}, {dy, x, w, a, b})) {
        int sms, used = 0;
        if (int rc = sm_count(&sms)) return rc;
        if (!ws.rows)
            if (int rc = mps::list_rows_and_rest(s.n_rows, s.n_adapters, s.ids, ws.ptr, ws.row, st)) return rc;
        const bool fp16 = s.dtype == MPS_F16;
        TcRows narrow[2] = {};  // side by side, and beside the listing: scale * x A^T and scale * dy B
        if (int rc = tc_adapter_narrow(s, s.k, a, false, &narrow[0])) return rc;
        if (int rc = tc_adapter_narrow(s, s.n, b, true, &narrow[1])) return rc;
        narrow[1].out_wide = ws.wide;
        if (fp16) {  // split once all of an adapter's are there
            narrow[0].out_f32 = ws.u, narrow[1].out_f32 = ws.v;
            narrow[0].maxima = ws.u_maxima, narrow[1].maxima = ws.v_maxima;
        } else {
            narrow[0].out_slots = ws.u_slots, narrow[1].out_slots = ws.v_slots;
            if (ws.rows) narrow[1].out_f32 = ws.v;
        }
        narrow[0].follows = narrow[0].apart = narrow[1].apart = !ws.rows;
        const void *const in[2] = {x, dy};
        const Cut half = best_cut(s.n_rows, s.n_adapters, s.rank, steps_of(s.k > s.n ? s.k : s.n), true, sms / 2, 64);
        if (int rc = tc_rows<mps::kNarrow>(narrow, 2, half, in, s.n_rows, sms, st)) return rc;
        if (fp16)
            if (int rc = tc_adapter_prepare(s, ws, ws.rows ? nullptr : a, true, s.k, true, half.split > 1 ? 2 : mps::kSpan, sms, st)) return rc;
        if (int rc = tc_adapter_wide(s, ws, s.n, s.k, dy, w, ws.v, a, true, dx, false, sms, st, &used)) return rc;
        const TcOuter outer[2] = {tc_adapter_outer(s, s.k, fp16 ? ws.v_exponents : nullptr, da, 1, s.k),
                                  tc_adapter_outer(s, s.n, fp16 ? ws.u_exponents : nullptr, db, s.rank, 1)};
        const void *const q[2] = {ws.v_slots, ws.u_slots};
        // beside few blocks of that on the SMs they leave, else on each as it gets free
        return tc_outer(outer, 2, in, q, used <= sms / 2 ? sms - used : sms, st);
    }
    if (int rc = adapter_narrow<T>(s, s.k, x, a, 1, s.k, ws.u, st)) return rc;
    if (int rc = adapter_narrow<T>(s, s.n, dy, b, s.rank, 1, ws.v, st)) return rc;
    if (int rc = adapter_wide<T>(s, s.n, s.k, dy, w, s.k, 1, ws.v, a, s.k, 1, dx, st)) return rc;
    OuterArgs o = {};
    o.group_ptr = s.group_ptr;
    o.slot_row = s.slot_row;
    o.n_groups = s.n_adapters;
    o.n_slots = o.n_rows = s.n_rows;
    o.p_by_row = o.q_by_row = true;
    o.i = s.rank;
    o.j = s.k;
    if (int rc = launch_plain_outer<float, T, T>(o, ws.v, x, da, st)) return rc;
    o.i = s.n;
    o.j = s.rank;
    return launch_plain_outer<T, float, T>(o, dy, ws.u, db, st);
}

int check_adapter_sizes(const char *who, const AdapterShape &s) {
    if (s.n_rows < 0 || s.k < 1 || s.n < 1 || s.n_adapters < 1 || s.rank < 1)
        return fail(MPS_ERR_ARG, "%s: %d rows, k = %d, n = %d, %d adapters of rank %d", who, s.n_rows, s.k, s.n, s.n_adapters, s.rank);
    if (!known(s.dtype)) return fail(MPS_ERR_ARG, "%s: unknown dtype %d", who, s.dtype);
    if (s.n_adapters > mps::kMaxRowGroups) return fail(MPS_ERR_UNSUPPORTED, "%s: at most %d adapters", who, mps::kMaxRowGroups);
    if (s.k > 1 << 21 || s.n > 1 << 21 || s.rank > 1 << 12) return fail(MPS_ERR_UNSUPPORTED, "%s: k and n may be up to %d, the rank up to %d", who, 1 << 21, 1 << 12);
    if (s.n_rows >= 1 << 30) return fail(MPS_ERR_UNSUPPORTED, "%s: at most %d rows", who, (1 << 30) - 1);
    return MPS_OK;
}

int check_adapters(const char *who, const AdapterShape &s, const void *workspace, int64_t bytes, bool backward) {
    if (int rc = check_adapter_sizes(who, s)) return rc;
    if (!s.group_ptr || (s.n_rows > 0 && (!s.ids || !s.slot_row))) return fail(MPS_ERR_ARG, "%s: NULL pointer", who);
    if (misaligned(s.ids, 4) || misaligned(s.group_ptr, 4) || misaligned(s.slot_row, 4) || misaligned(s.scale, 4))
        return fail(MPS_ERR_ALIGN, "%s: a pointer is not aligned to its element size", who);
    if (s.n_rows > 0) {
        const int64_t need = AdapterSpace(nullptr, s, backward).bytes;
        if (!workspace || bytes < need) return fail(MPS_ERR_ARG, "%s: the workspace needs %lld bytes, %lld given", who, (long long)need, (long long)bytes);
        if (misaligned(workspace, 256)) return fail(MPS_ERR_ALIGN, "%s: the workspace must be 256-byte aligned", who);
    }
    return MPS_OK;
}

}  // namespace

#define RD_BY_TYPE(dtype, call)                     \
    do {                                            \
        if ((dtype) == MPS_F32) { using T = float; return call; }      \
        if ((dtype) == MPS_F16) { using T = __half; return call; }     \
        using T = __nv_bfloat16;                    \
        return call;                                \
    } while (0)

extern "C" int mps_routed_product(int32_t n_slots, int32_t n_rows, int32_t n_groups, int32_t k, int32_t n, int dtype, int transpose,
                                  const int32_t *d_group_ptr, const int32_t *d_slot_row, const void *d_x, const void *d_w, void *d_y, void *stream) {
    if (int rc = check_product("mps_routed_product", n_slots, n_rows, n_groups, k, n, dtype)) return rc;
    if (n_slots == 0) return MPS_OK;
    if (!d_group_ptr || !d_x || !d_w || !d_y) return fail(MPS_ERR_ARG, "mps_routed_product: NULL pointer");
    if (!d_slot_row && n_rows < n_slots) return fail(MPS_ERR_ARG, "mps_routed_product: %d rows for %d slots read in order", n_rows, n_slots);
    const size_t size = size_of(dtype);
    if (misaligned(d_group_ptr, 4) || misaligned(d_slot_row, 4) || misaligned(d_x, size) || misaligned(d_w, size) || misaligned(d_y, size))
        return fail(MPS_ERR_ALIGN, "mps_routed_product: a pointer is not aligned to its element size");
    const int summed = transpose ? n : k, features = transpose ? k : n;
    if (overlap(dtype, {{d_y, (long long)n_slots * features}}, {{d_x, (long long)n_rows * summed}, {d_w, (long long)n_groups * k * n}}))
        return fail(MPS_ERR_ARG, "mps_routed_product: the result overlaps an operand");
    if (n_rows > 0 && tc_widths(dtype, {k, summed}, {d_x, d_w})) {
        TcRows a = {};
        a.bf16 = dtype == MPS_BF16;
        a.mn_major = transpose != 0;
        a.group_ptr = d_group_ptr;
        a.slot_row = d_slot_row;
        a.n_groups = n_groups;
        a.n_slots = n_slots;
        a.n_x_rows = n_rows;
        a.k = summed;
        a.n = features;
        a.gather = d_slot_row != nullptr;
        a.out = d_y;
        int sms;
        if (int rc = sm_count(&sms)) return rc;
        if (int rc = tc_matrix(&a.w, &a, d_w, summed, features, n_groups)) return rc;
        return tc_rows<mps::kProduct>(&a, 1, best_cut(n_slots, n_groups, features, steps_of(summed), a.gather, sms, 256), &d_x, n_rows, sms, (cudaStream_t)stream);
    }
    RowsArgs a = {};
    a.group_ptr = d_group_ptr;
    a.slot_row = d_slot_row;
    a.n_groups = n_groups;
    a.n_slots = n_slots;
    a.n_x_rows = n_rows;
    a.k = summed;
    a.n = features;
    a.w_group = (long long)k * n;
    a.w_k = transpose ? k : 1;
    a.w_n = transpose ? 1 : k;
    RD_BY_TYPE(dtype, (launch_plain_rows<T, T, false>(a, d_x, d_w, nullptr, d_y, (cudaStream_t)stream)));
}

extern "C" int mps_routed_wgrad(int32_t n_slots, int32_t n_rows, int32_t n_groups, int32_t k, int32_t n, int dtype, const int32_t *d_group_ptr,
                                const int32_t *d_slot_row, const void *d_x, const void *d_dy, void *d_dw, void *stream) {
    if (int rc = check_product("mps_routed_wgrad", n_slots, n_rows, n_groups, k, n, dtype)) return rc;
    if (!d_group_ptr || !d_dw || (n_slots > 0 && (!d_x || !d_dy))) return fail(MPS_ERR_ARG, "mps_routed_wgrad: NULL pointer");
    if (!d_slot_row && n_rows < n_slots) return fail(MPS_ERR_ARG, "mps_routed_wgrad: %d rows for %d slots read in order", n_rows, n_slots);
    const size_t size = size_of(dtype);
    if (misaligned(d_group_ptr, 4) || misaligned(d_slot_row, 4) || misaligned(d_x, size) || misaligned(d_dy, size) || misaligned(d_dw, size))
        return fail(MPS_ERR_ALIGN, "mps_routed_wgrad: a pointer is not aligned to its element size");
    if (overlap(dtype, {{d_dw, (long long)n_groups * k * n}}, {{d_x, (long long)n_rows * k}, {d_dy, (long long)n_slots * n}}))
        return fail(MPS_ERR_ARG, "mps_routed_wgrad: the result overlaps an operand");
    if (n_slots > 0 && n_rows > 0 && tc_widths(dtype, {k, n}, {d_x, d_dy})) {
        int sms;
        if (int rc = sm_count(&sms)) return rc;
        TcOuter a = {};
        a.bf16 = dtype == MPS_BF16;
        a.group_ptr = d_group_ptr;
        a.slot_row = d_slot_row;
        a.n_groups = n_groups;
        a.n_slots = n_slots;
        a.n_p_rows = n_rows;
        a.i = k;
        a.j = n;
        a.out = d_dw;
        a.out_group = (long long)k * n;
        a.out_f = 1;
        a.out_c = k;
        return tc_outer(&a, 1, &d_x, &d_dy, sms, (cudaStream_t)stream);
    }
    OuterArgs a = {};
    a.group_ptr = d_group_ptr;
    a.slot_row = d_slot_row;
    a.n_groups = n_groups;
    a.n_slots = n_slots;
    a.n_rows = n_rows;
    a.i = n;
    a.j = k;
    a.q_by_row = true;
    RD_BY_TYPE(dtype, (launch_plain_outer<T, T, T>(a, d_dy, d_x, d_dw, (cudaStream_t)stream)));
}

static int check_combine(const char *who, int n_rows, int per_row, int n_slots, int dim, int dtype) {
    if (n_rows < 0 || per_row < 1 || n_slots < 0 || dim < 1) return fail(MPS_ERR_ARG, "%s: %d rows of %d terms, %d slots, dim %d", who, n_rows, per_row, n_slots, dim);
    if (!known(dtype)) return fail(MPS_ERR_ARG, "%s: unknown dtype %d", who, dtype);
    if ((long long)n_rows * per_row >= 1LL << 31) return fail(MPS_ERR_UNSUPPORTED, "%s: rows * per_row does not fit 31 bits", who);
    if (dim > 1 << 24) return fail(MPS_ERR_UNSUPPORTED, "%s: dim may be up to %d", who, 1 << 24);  // stretches of a row are the grid's y
    return MPS_OK;
}

extern "C" int mps_routed_combine(int32_t n_rows, int32_t per_row, int32_t n_slots, int32_t dim, int dtype, const int32_t *d_slot_of,
                                  const float *d_weights, const void *d_rows, void *d_y, void *stream) {
    if (int rc = check_combine("mps_routed_combine", n_rows, per_row, n_slots, dim, dtype)) return rc;
    if (n_rows == 0) return MPS_OK;
    if (!d_slot_of || !d_y || (n_slots > 0 && !d_rows)) return fail(MPS_ERR_ARG, "mps_routed_combine: NULL pointer");
    const size_t size = size_of(dtype);
    if (misaligned(d_slot_of, 4) || misaligned(d_weights, 4) || misaligned(d_rows, size) || misaligned(d_y, size))
        return fail(MPS_ERR_ALIGN, "mps_routed_combine: a pointer is not aligned to its element size");
    if (overlap(dtype, {{d_y, (long long)n_rows * dim}}, {{d_rows, (long long)n_slots * dim}}))
        return fail(MPS_ERR_ARG, "mps_routed_combine: the result overlaps an operand");
    RD_BY_TYPE(dtype, launch_combine<T>(n_rows, per_row, n_slots, dim, d_slot_of, d_weights, d_rows, d_y, (cudaStream_t)stream));
}

extern "C" int mps_routed_combine_backward(int32_t n_rows, int32_t per_row, int32_t n_slots, int32_t dim, int dtype, const int32_t *d_slot_of,
                                           const float *d_weights, const void *d_dy, const void *d_rows, void *d_drows, float *d_dweights, void *stream) {
    if (int rc = check_combine("mps_routed_combine_backward", n_rows, per_row, n_slots, dim, dtype)) return rc;
    if (n_rows == 0) return MPS_OK;
    if (!d_slot_of || !d_dy || (n_slots > 0 && (!d_drows || (d_dweights && !d_rows)))) return fail(MPS_ERR_ARG, "mps_routed_combine_backward: NULL pointer");
    const size_t size = size_of(dtype);
    if (misaligned(d_slot_of, 4) || misaligned(d_weights, 4) || misaligned(d_dweights, 4) || misaligned(d_dy, size) || misaligned(d_rows, size) ||
        misaligned(d_drows, size))
        return fail(MPS_ERR_ALIGN, "mps_routed_combine_backward: a pointer is not aligned to its element size");
    if (overlap(dtype, {{d_drows, (long long)n_slots * dim}}, {{d_dy, (long long)n_rows * dim}, {d_rows == d_drows ? nullptr : d_rows, (long long)n_slots * dim}}))
        return fail(MPS_ERR_ARG, "mps_routed_combine_backward: the result overlaps an operand");
    RD_BY_TYPE(dtype, launch_combine_backward<T>(n_rows, per_row, n_slots, dim, d_slot_of, d_weights, d_dy, d_rows, d_drows, d_dweights, (cudaStream_t)stream));
}

extern "C" int64_t mps_adapters_workspace(int32_t n_rows, int32_t k, int32_t n, int32_t n_adapters, int32_t rank, int dtype, int backward) {
    const AdapterShape s = {n_rows, k, n, n_adapters, rank, dtype, nullptr, nullptr, nullptr, nullptr};
    if (int rc = check_adapter_sizes("mps_adapters_workspace", s)) return rc;
    return n_rows == 0 ? 0 : AdapterSpace(nullptr, s, backward != 0).bytes;
}

extern "C" int mps_adapters(int32_t n_rows, int32_t k, int32_t n, int32_t n_adapters, int32_t rank, int dtype, const int32_t *d_ids,
                            const int32_t *d_group_ptr, const int32_t *d_slot_row, const float *d_scale, const void *d_x, const void *d_w,
                            const void *d_a, const void *d_b, void *d_y, void *d_workspace, int64_t workspace_bytes, void *stream) {
    const AdapterShape s = {n_rows, k, n, n_adapters, rank, dtype, d_ids, d_group_ptr, d_slot_row, d_scale};
    if (int rc = check_adapters("mps_adapters", s, d_workspace, workspace_bytes, false)) return rc;
    if (n_rows == 0) return MPS_OK;
    if (!d_x || !d_w || !d_a || !d_b || !d_y) return fail(MPS_ERR_ARG, "mps_adapters: NULL pointer");
    const size_t size = size_of(dtype);
    if (misaligned(d_x, size) || misaligned(d_w, size) || misaligned(d_a, size) || misaligned(d_b, size) || misaligned(d_y, size))
        return fail(MPS_ERR_ALIGN, "mps_adapters: a pointer is not aligned to its element size");
    const long long matrix = (long long)n_adapters * rank, space = (workspace_bytes + (int64_t)size - 1) / (int64_t)size;
    if (overlap(dtype, {{d_y, (long long)n_rows * n}, {d_workspace, space}},
                {{d_x, (long long)n_rows * k}, {d_w, (long long)n * k}, {d_a, matrix * k}, {d_b, matrix * n}}))
        return fail(MPS_ERR_ARG, "mps_adapters: the result or the workspace overlaps an operand");
    RD_BY_TYPE(dtype, adapters<T>(s, d_x, d_w, d_a, d_b, d_y, d_workspace, (cudaStream_t)stream));
}

extern "C" int mps_adapters_backward(int32_t n_rows, int32_t k, int32_t n, int32_t n_adapters, int32_t rank, int dtype, const int32_t *d_ids,
                                     const int32_t *d_group_ptr, const int32_t *d_slot_row, const float *d_scale, const void *d_dy, const void *d_x,
                                     const void *d_w, const void *d_a, const void *d_b, void *d_dx, void *d_da, void *d_db, void *d_workspace,
                                     int64_t workspace_bytes, void *stream) {
    const AdapterShape s = {n_rows, k, n, n_adapters, rank, dtype, d_ids, d_group_ptr, d_slot_row, d_scale};
    if (int rc = check_adapters("mps_adapters_backward", s, d_workspace, workspace_bytes, true)) return rc;
    if (!d_w || !d_a || !d_b || !d_da || !d_db || (n_rows > 0 && (!d_dy || !d_x || !d_dx))) return fail(MPS_ERR_ARG, "mps_adapters_backward: NULL pointer");
    const size_t size = size_of(dtype);
    if (misaligned(d_dy, size) || misaligned(d_x, size) || misaligned(d_w, size) || misaligned(d_a, size) || misaligned(d_b, size) ||
        misaligned(d_dx, size) || misaligned(d_da, size) || misaligned(d_db, size))
        return fail(MPS_ERR_ALIGN, "mps_adapters_backward: a pointer is not aligned to its element size");
    const long long matrix = (long long)n_adapters * rank, space = n_rows ? (workspace_bytes + (int64_t)size - 1) / (int64_t)size : 0;
    if (overlap(dtype, {{d_dx, (long long)n_rows * k}, {d_da, matrix * k}, {d_db, matrix * n}, {d_workspace, space}},
                {{d_dy, (long long)n_rows * n}, {d_x, (long long)n_rows * k}, {d_w, (long long)n * k}, {d_a, matrix * k}, {d_b, matrix * n}}))
        return fail(MPS_ERR_ARG, "mps_adapters_backward: a result or the workspace overlaps an operand");
    if (n_rows == 0) {  // no rows: the adapters' gradients are zero
        const size_t bytes = (size_t)n_adapters * rank * size;
        RD_CUDA(cudaMemsetAsync(d_da, 0, bytes * k, (cudaStream_t)stream));
        RD_CUDA(cudaMemsetAsync(d_db, 0, bytes * n, (cudaStream_t)stream));
        return MPS_OK;
    }
    RD_BY_TYPE(dtype, adapters_backward<T>(s, d_dy, d_x, d_w, d_a, d_b, d_dx, d_da, d_db, d_workspace, (cudaStream_t)stream));
}

extern "C" int mps_routed_check(void *stream) {
    cudaStream_t st = (cudaStream_t)stream;
    int routed = 0, route = 0;
    RD_CUDA(cudaMemcpyFromSymbolAsync(&routed, g_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
    RD_CUDA(cudaStreamSynchronize(st));
    if (routed) {  // what was read and nothing else: another stream may have reported something since; done when this returns
        clear_status<<<1, 1, 0, st>>>(routed);
        RD_CUDA(cudaGetLastError());
        RD_CUDA(cudaStreamSynchronize(st));
    }
    if (int rc = mps::take_route_status(st, &route)) return rc;
    const int status = routed | route;
    if (status & mps::kStatusTimeout) return fail(MPS_ERR_DEVICE, "mps_routed_check: a kernel gave up a wait");
    if (status & mps::kStatusBadIndex) return fail(MPS_ERR_ARG, "mps_routed_check: an id, a slot or a group offset was out of range");
    return MPS_OK;
}
