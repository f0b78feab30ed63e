// sm100.cuh -- the asynchronous copies, barriers, tensor-core instructions
// and launch attributes of sm_100a that the decode-step kernels use.
//
// Every wait ends: after kWaitCycles the waiting thread counts the event in
// g_expired_waits, marks its CTA (`dead`) so that the CTA's other waits end
// too, and the kernel returns without the results of that CTA.
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace tsg {

// Tensor map of a row-major matrix [rows][cols], or of `count` of them one
// behind the other, in boxes of box_cols x box_rows; boxes 64 bytes wide have
// the 64-byte swizzle, others (128 bytes) the 128-byte one (k_project.cu).
cudaError_t tensor_map(CUtensorMap* out, CUtensorMapDataType type, const void* p, uint64_t cols, uint64_t rows, uint64_t row_bytes,
                       uint32_t box_cols, uint32_t box_rows, uint64_t count = 0);

namespace {

constexpr long long kWaitCycles = 4000000000ll;  // 2 s and more

__device__ unsigned long long g_expired_waits;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity)
        : "memory");
    return ok;
}
// Waits for the phase `parity` of b to end; false when it did not in time.
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, uint32_t* dead) {
    if (mbar_try(b, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; i++)
            if (mbar_try(b, parity)) return true;
        if (*reinterpret_cast<volatile uint32_t*>(dead)) return false;
        if (clock64() - t0 > kWaitCycles) {
            atomicAdd(&g_expired_waits, 1ull);
            atomicExch(dead, 1u);
            return false;
        }
    }
}
// After an expired wait: a bounded time for what is in flight.
__device__ __forceinline__ void settle() {
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000) __nanosleep(1000);
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
// The two halves of a cluster barrier that orders no memory: behind the wait,
// every CTA of the cluster has started.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }
// Address of the same shared-memory variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_rank(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Without ordering what came before: a release to the cluster costs some
// hundred cycles, which a thread that only starts copies need not pay.
__device__ __forceinline__ void mbar_arrive_relaxed_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t cluster_addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
    return v;
}

__device__ __forceinline__ void st_shared2b(uint32_t at, uint16_t v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(v) : "memory"); }
__device__ __forceinline__ uint16_t ld_shared2b(uint32_t at) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ float2 ld_cluster2(uint32_t cluster_addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr) : "memory");
    return v;
}

// Position in a ring of barriers and the parity of its current phase.
struct Ring {
    int i = 0, n;
    uint32_t phase;
    __device__ __forceinline__ Ring(int n_, uint32_t phase_) : n(n_), phase(phase_) {}
    __device__ __forceinline__ void next() {
        if (++i == n) i = 0, phase ^= 1;
    }
    __device__ __forceinline__ void skip(int by) {
        i += by;
        phase ^= (uint32_t)(i / n) & 1;
        i %= n;
    }
};

// `bytes` from global to this CTA's shared memory, both on 16-byte boundaries
// and bytes a multiple of 16.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}
// One box of a tensor map to this CTA's shared memory; `bar` (a cluster
// address) may be the other CTA's of a pair (CG = 2).
template <int CG>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
            : "memory");
}

template <int CG>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}
// The other way: one box from this CTA's shared memory, as a bulk group of
// the calling thread.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x),
                 "r"(y), "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until the stores have read their shared memory, but for the last N groups.
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t t, uint32_t cols) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(cols));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(cols));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// Barrier of `threads` threads that returns whether any of them passed true.
__device__ __forceinline__ bool bar_or(int id, int threads, bool v) {
    uint32_t any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n barrier.cta.red.or.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
        : "=r"(any)
        : "r"(id), "r"(threads), "r"((uint32_t)v)
        : "memory");
    return any;
}

// Shared-memory operand descriptors (version 1): start >> 4, leading and
// stride byte offsets >> 4, swizzle.  K-major rows of 128 / 64 bytes in
// groups of eight; MN-major blocks of 64 elements x 8, `mn` bytes apart.
__device__ __forceinline__ uint64_t desc_of(uint32_t addr, uint32_t lead, uint32_t stride, uint64_t swizzle) {
    return (uint64_t)(addr >> 4 & 0x3fff) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | swizzle << 61;
}
__device__ __forceinline__ uint64_t desc_k128(uint32_t addr) { return desc_of(addr, 16, 1024, 2); }
__device__ __forceinline__ uint64_t desc_k64(uint32_t addr) { return desc_of(addr, 16, 512, 4); }
__device__ __forceinline__ uint64_t desc_mn128(uint32_t addr, uint32_t mn) { return desc_of(addr, mn, 1024, 2); }

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (CG == 2)
        asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                     "l"(a), "l"(b), "r"(idesc), "r"(add)
                     : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                     "l"(a), "l"(b), "r"(idesc), "r"(add)
                     : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_tf32(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (CG == 2)
        asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::tf32 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                     "l"(a), "l"(b), "r"(idesc), "r"(add)
                     : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                     "l"(a), "l"(b), "r"(idesc), "r"(add)
                     : "memory");
}
// Arrives at b (in both CTAs of a pair) when the instructions so far are done.
template <int CG>
__device__ __forceinline__ void mma_commit(uint64_t* b) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(b)),
                     "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
}
// 32 columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t t, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

// f32 rounded to TF32 (11 significant bits, nearest, ties away).
__device__ __forceinline__ uint32_t to_tf32(float v) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}
// v as two bf16 terms of one sign, neither of them zero: the upper one is one
// step below v's first 8 bits, the lower one the rest, rounded, so that their
// sum is within 2^-15 v.  An infinity times such a v has the sign of their
// product and not the NaN of an infinity times zero or of two signs; values
// that round to infinity in 8 bits stay finite.  Infinities and NaNs are both
// terms.  (v below bf16's second least value, 2^-132, counts as zero there.)
__device__ __forceinline__ void bf16_terms(float v, uint32_t& high, uint32_t& low) {
    const uint32_t u = __float_as_uint(v), m = u >> 16 & 0x7fffu;
    const bool special = m >= 0x7f80u;
    high = special ? (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)) : (u >> 16 & 0x8000u) | (m > 0u ? m - 1u : 0u);
    low = special ? high : (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v - __uint_as_float(high << 16)));
}

// What a TF32 instruction leaves out of v, which it cuts to 11 significant
// bits; zero where v is not finite.
__device__ __forceinline__ uint32_t tf32_rest(float v) {
    const uint32_t u = __float_as_uint(v);
    return (u & 0x7f800000u) == 0x7f800000u ? 0u : __float_as_uint(v - __uint_as_float(u & 0xffffe000u));
}

// v = high + low for TF32 instructions, low zero where v is not finite (the
// upper term then is v): products with the lower terms have to leave out what
// is not finite.  Returns whether v is not.  Values that would round to
// infinity are cut instead.
__device__ __forceinline__ bool tf32_terms(float v, uint32_t& high, uint32_t& low) {
    const uint32_t u = __float_as_uint(v), m = u & 0x7fffffffu;
    const bool special = m >= 0x7f800000u;
    high = special ? (m > 0x7f800000u ? 0x7fffffffu : u) : (m >= 0x7f7ff000u ? u : u + 0x1000u) & 0xffffe000u;
    low = special ? 0u : to_tf32(v - __uint_as_float(high));
    return special;
}
__device__ __forceinline__ void st_shared4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint4 ld_shared4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// Programmatic dependent launch: the dependent kernel may start once every
// CTA of the one before it has called release_dependents, and sees that
// kernel's results after grid_dependency_wait.
__device__ __forceinline__ void release_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[2];
    // cx x cy: cluster; dependent: programmatically dependent on the launch before
    Launch(int cx, int cy, bool dependent, dim3 grid, unsigned block, size_t smem, cudaStream_t s) {
        cfg.gridDim = grid;
        cfg.blockDim = dim3(block, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = s;
        cfg.attrs = at;
        if (dependent) {
            at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
        }
        if (cx * cy > 1) {
            at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
            at[cfg.numAttrs].val.clusterDim.x = (unsigned)cx;
            at[cfg.numAttrs].val.clusterDim.y = (unsigned)cy;
            at[cfg.numAttrs++].val.clusterDim.z = 1;
        }
    }
};

template <class... KArgs, class... Args>
cudaError_t launch_dependent(int cluster, void (*kern)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t s, Args... args) {
    const Launch l(cluster, 1, true, grid, block, smem, s);
    return cudaLaunchKernelEx(&l.cfg, kern, args...);
}

// Clusters along y.
template <class... KArgs, class... Args>
cudaError_t launch_split_y(int cluster, bool dependent, void (*kern)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t s,
                           Args... args) {
    const Launch l(1, cluster, dependent, grid, block, smem, s);
    return cudaLaunchKernelEx(&l.cfg, kern, args...);
}

}  // namespace
}  // namespace tsg
