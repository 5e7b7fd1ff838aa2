// Blackwell building blocks of the routed products: mbarriers with bounded waits, TMA loads, tcgen05 products into TMEM.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "mps_types.cuh"

namespace mps {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// one lane of a converged warp, in the form the compiler knows to be a single thread (products and their descriptors then stay
// in uniform registers)
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}

// The stage a warp is at in the ring, and the parity of its use.  Counted up: a division per slice costs the thread that issues
// the products more than the products take.
struct RingAt {
    int stage = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next(int stages) {
        if (++stage == stages) {
            stage = 0;
            parity ^= 1;
        }
    }
};

constexpr long long kWaitLimit = 1ll << 34;  // SM cycles, nine seconds: no wait of a working kernel comes near

// Waits for the phase; after kWaitLimit (or once another thread of the block gave up) it records that and returns.  The block
// then runs through its remaining steps without waiting, and its result counts as undefined.  Counted in the SM's own cycles,
// which only rise; the global timer is read in two halves and may be set.
__device__ __forceinline__ void mbar_wait(uint32_t bar, uint32_t parity, volatile int *gave_up, int *status) {
    if (mbar_try(bar, parity)) return;
    const long long start = clock64();
    for (;;) {
        for (int i = 0; i < 64; ++i)
            if (mbar_try(bar, parity)) return;
        if (*gave_up) return;
        if (clock64() - start > kWaitLimit) {
            *gave_up = 1;
            atomicOr(status, kStatusTimeout);
            return;
        }
    }
}

// ---- TMA: boxes of 64 elements of a 16-bit type or 32 of fp32 (128 bytes, 128-byte swizzle) by some rows.  The x coordinate is a
// multiple of as many throughout, so every copy starts on a 128-byte multiple of its row.
// PAIRED: the barrier may be the other block's.
template <bool PAIRED>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    if constexpr (PAIRED)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(bar)
                     : "memory");
    else asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x),
                 "r"(y), "r"(bar)
                 : "memory");
}
template <bool PAIRED>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    if constexpr (PAIRED)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                     : "memory");
    else asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
// four rows by number, one under the other; a row number outside the tensor gives zeros
template <bool PAIRED>
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap *map, int x, int r0, int r1, int r2, int r3, uint32_t bar) {
    if constexpr (PAIRED)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
                dst),
            "l"(map), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
            "l"(map), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
            : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// ---- tcgen05; PAIRED: by two neighbouring blocks of a cluster as one, the products issued by the first for both
template <bool PAIRED>
__device__ __forceinline__ void tmem_alloc(uint32_t where, uint32_t columns) {
    if constexpr (PAIRED) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <bool PAIRED>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    if constexpr (PAIRED) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// arrives at the barrier (PAIRED: at both blocks' barriers of that address) once the products issued so far are done
template <bool PAIRED>
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    if constexpr (PAIRED)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                     : "memory");
    else asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// TF32: 32-bit operands with ten bits of fraction, eight summed elements at a time; else a 16-bit type, sixteen
template <bool PAIRED, bool TF32>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    if constexpr (PAIRED && TF32)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
            "r"(idesc), "r"((uint32_t)add)
            : "memory");
    else if constexpr (PAIRED)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
            "r"(idesc), "r"((uint32_t)add)
            : "memory");
    else if constexpr (TF32)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
            "r"(idesc), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
            "r"(idesc), "r"((uint32_t)add)
            : "memory");
}

// Shared-memory operand in 128-byte swizzled atoms of eight 128-byte rows.  Summed index contiguous: the rows are the tile's
// rows, atoms 1024 bytes apart.  Summed index across the rows (MN-major): an atom holds 64 tile rows by 8 summed ones, the
// next 8 summed ones follow after 1024 bytes, the next 64 tile rows after kBlock64.
constexpr uint32_t kBlock64 = 64 * 128;  // 64 summed rows of 128 bytes
__device__ __forceinline__ uint64_t operand(uint32_t addr, bool mn_major) {
    const uint64_t lead = mn_major ? kBlock64 >> 4 : 1, stride = 1024 >> 4;
    return (uint64_t)((addr >> 4) & 0x3fff) | lead << 16 | stride << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// 16 summed elements further, in units of the descriptor's address field
__device__ __forceinline__ uint64_t operand_step(bool mn_major) { return mn_major ? (16 * 128) >> 4 : 32 >> 4; }
// the same operand `bytes` further on (addresses stay below 2^18, so the field does not overflow)
__device__ __forceinline__ uint64_t operand_at(uint64_t first, uint32_t bytes) { return first + (bytes >> 4); }

// fp32 result, both operands of one 16-bit type, m result rows (128; 256 by a pair of blocks) by n columns
__device__ __forceinline__ uint32_t mma_desc(bool bf16, bool a_mn, bool b_mn, int m, int n) {
    return 1u << 4 | (uint32_t)bf16 << 7 | (uint32_t)bf16 << 10 | (uint32_t)a_mn << 15 | (uint32_t)b_mn << 16 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// the same of two tf32 operands, their summed index contiguous
__device__ __forceinline__ uint32_t mma_desc_tf32(int m, int n) { return 1u << 4 | 2u << 7 | 2u << 10 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24; }

// 32 consecutive columns of the calling warp's 32 TMEM lanes, one lane per thread; there after tmem_wait
__device__ __forceinline__ void tmem_start(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
        "%23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// The values pass through the wait, so that nothing uses them before it.
__device__ __forceinline__ void tmem_wait(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32]) {
    tmem_start(addr, v);
    tmem_wait(v);
}

__device__ __forceinline__ uint16_t to_16(float v, bool bf16) {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
// two values rounded into one 32-bit word, the first below
template <bool BF16>
__device__ __forceinline__ uint32_t to_16x2(float a, float b) {
    uint32_t r;
    if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// two values of a 32-bit word, the lower half first
template <bool BF16>
__device__ __forceinline__ float2 from_16x2(uint32_t v) {
    if constexpr (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    else return __half22float2(__halves2half2(__ushort_as_half((uint16_t)v), __ushort_as_half((uint16_t)(v >> 16))));
}
__device__ __forceinline__ float from_16(uint16_t v, bool bf16) { return bf16 ? __bfloat162float(__ushort_as_bfloat16(v)) : __half2float(__ushort_as_half(v)); }

__device__ __forceinline__ void store_shared_16(uint32_t addr, uint16_t v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(v) : "memory"); }
__device__ __forceinline__ uint4 load_shared_128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void results_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // the four warps that store results

// ---- clusters
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of block `rank`'s variable of that address in this block, and a store to it
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    return remote;
}
__device__ __forceinline__ void store_cluster_f32(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
// Arrives at a barrier of either block.  (With .release.cluster the arrival waits for the thread's writes to reach the cluster,
// about a microsecond; it follows no writes here that the other block reads.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// the same at block `rank`'s barrier of that address
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar, uint32_t rank) {
    mbar_arrive_cluster(in_block(bar, rank));
}
__device__ __forceinline__ void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
// Launches of one call follow one another with programmatic serialization: every kernel lets the next one start at once (its
// blocks take the SMs that fall free, its set-up overlaps the end of this one) and waits for the launch before it, and with it
// all earlier ones, before it touches memory.  Nothing where a launch was an ordinary one.
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_launch_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ float load_shared_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_shared_float4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void store_shared_f32(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }

// An fp32 value as the sum of two tf32 values, off by 2^-21 of it at most: its first eleven bits, and what is left rounded to
// eleven.  The second has the first's sign and (from 2^-100 up, where the least normal number is nothing) is no zero, so that an
// infinite factor gives the infinity that the value would; of an infinite value it is next to nothing.
__device__ __forceinline__ float tf32_first(float v) { return v != v ? v : __uint_as_float(__float_as_uint(v) & 0xffffe000u); }
__device__ __forceinline__ float tf32_second(float v) {
    const uint32_t rest = fabsf(v) < INFINITY ? (__float_as_uint(fabsf(v - tf32_first(v))) + 0x1000u) & 0xffffe000u : 0u;
    return copysignf(__uint_as_float(rest < 0x00800000u && fabsf(v) >= 0x1p-100f ? 0x00800000u : rest), v);
}

// The same of four values in bf16, two to a word: 2^-16 of a value lost.
__device__ __forceinline__ uint32_t bf16_first(float v) { return v != v ? 0x7fffu : __float_as_uint(v) >> 16; }
__device__ __forceinline__ uint32_t bf16_second(float v) {
    const float rest = fabsf(v) < INFINITY ? v - __uint_as_float(bf16_first(v) << 16) : 0.0f;
    const uint32_t bits = __bfloat16_as_ushort(__float2bfloat16_rn(fabsf(rest)));
    return (bits < 0x0080u && fabsf(v) >= 0x1p-100f ? 0x0080u : bits) | (__float_as_uint(v) >> 16 & 0x8000u);
}
__device__ __forceinline__ void split_bf16(float4 v, uint2 &first, uint2 &second) {
    first = make_uint2(bf16_first(v.x) | bf16_first(v.y) << 16, bf16_first(v.z) | bf16_first(v.w) << 16);
    second = make_uint2(bf16_second(v.x) | bf16_second(v.y) << 16, bf16_second(v.z) | bf16_second(v.w) << 16);
}

// the products of one slice: `steps` (1..4) times 32 bytes of summed elements, the first overwriting the accumulator unless `add`
template <bool PAIRED, bool TF32 = false>
__device__ __forceinline__ void tc_slice(uint32_t d, uint64_t a, uint64_t b, uint64_t a_step, uint64_t b_step, uint32_t idesc, int steps, bool add) {
    if (steps == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) tc_mma<PAIRED, TF32>(d, a + i * a_step, b + i * b_step, idesc, add || i > 0);
    } else {
        for (int i = 0; i < steps; ++i) tc_mma<PAIRED, TF32>(d, a + i * a_step, b + i * b_step, idesc, add || i > 0);
    }
}

}  // namespace mps
