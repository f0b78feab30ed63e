// k_lowrank.cu -- kernels of the low-rank adapters beside a shared
// projection, and of their gradients, but for the tensor-core projection of
// many tokens (k_project.cu).
//
// For token m with adapter e (or none):
//   low[m]  = s_e x[m] A_e^T                              (r values, f32)
//   y[m]    = base[m] + x[m] W^T + bias + low[m] B_e^T
// and, for the gradient dy of y with W frozen,
//   u[m]    = s_e dy[m] B_e
//   dx[m]   = dy[m] W + u[m] A_e
//   dA_e    = sum over e's tokens of u[m]^T x[m]
//   dB_e    = sum over e's tokens of dy[m]^T low[m]
// The kernels below are these lines; a factor's strides turn the forward
// form into the backward one.  Sums are held in f32 and each result is
// rounded to its type once.
#include <climits>
#include <type_traits>

#include "launch.cuh"
#include "lowrank.cuh"
#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace tsg {

namespace {

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// Two 16-bit elements as floats.
template <class T>
__device__ __forceinline__ float2 pair_f(uint32_t v) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

template <class T>
__device__ __forceinline__ uint4 whole16(const T* row, int k) { return *reinterpret_cast<const uint4*>(row + k); }

// Elements [k, k + 16 / sizeof(T)) of a row of `n`, zeros behind it.  Loops
// take whole16 while they can: loads under a condition do not overlap.
template <class T>
__device__ __forceinline__ uint4 load16(const T* row, int k, int n) {
    constexpr int V = 16 / sizeof(T);
    if (k + V <= n) return *reinterpret_cast<const uint4*>(row + k);
    T v[V];
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = k + i < n ? row[k + i] : from_f<T>(0.f);
    uint4 r;
    memcpy(&r, v, 16);
    return r;
}

template <class T>
__device__ __forceinline__ float dot16(uint4 a, uint4 b, float v) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            v = fmaf(__uint_as_float(x[i]), __uint_as_float(y[i]), v);
        } else {
            const float2 p = pair_f<T>(x[i]), q = pair_f<T>(y[i]);
            v = fmaf(p.y, q.y, fmaf(p.x, q.x, v));
        }
    }
    return v;
}

// D = A B + C on 16 x 8 x 16 of a 16-bit type, f32 sums.
template <class T>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma8_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------- packing

// 32 rows x 128 columns of a job through shared memory, read along whichever
// axis of src is contiguous, written along k.  Factors of 14 adapters, rank 64,
// over 8960 (transposed) and 1536 (as f32): 15 us; 32 x 32 tiles took 32.
__device__ __forceinline__ void pack_tile(const PackJob& a, const uint16_t* src, uint16_t* dst, long long j0, int k0) {
    __shared__ __align__(4) uint16_t tile[32][130];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const bool along = a.sk == 1;
    const auto row = [&](int i) { return along ? ty + 8 * (i >> 2) : tx; };
    const auto col = [&](int i) { return along ? tx + 32 * (i & 3) : ty + 8 * i; };
    uint16_t v[16];
#pragma unroll
    for (int i = 0; i < 16; i++)  // loads from clamped places overlap, loads under a condition do not
        v[i] = src[min(j0 + row(i), a.rows - 1) * a.sj + min(k0 + col(i), a.cols - 1) * a.sk];
#pragma unroll
    for (int i = 0; i < 16; i++) tile[row(i)][col(i)] = k0 + col(i) < a.cols ? v[i] : (uint16_t)0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int j = ty + 8 * (i >> 1), k = (tx + 32 * (i & 1)) * 2;
        if (j0 + j < a.rows && k0 + k < a.dst_cols)
            *reinterpret_cast<uint32_t*>(dst + (j0 + j) * a.dst_cols + k0 + k) = *reinterpret_cast<const uint32_t*>(&tile[j][k]);
    }
}

// 128 rows x 16 columns of a factor as f32; returns whether an element is not
// finite.  A thread takes 8 neighbours along whichever axis of src is
// contiguous, in one load where they are on a 16-byte boundary.
__device__ __forceinline__ bool pack_f32(const PackJob& a, const uint16_t* src, float* dst, long long j0, int k0, int dtype) {
    __shared__ float tile[128][17];
    const bool along = a.sk == 1;  // k is the contiguous axis
    const int j = along ? threadIdx.x >> 1 : (threadIdx.x & 15) * 8, k = along ? (threadIdx.x & 1) * 8 : threadIdx.x >> 4;
    const long long jj = j0 + j;
    const int kk = k0 + k, left = along ? (jj < a.rows ? a.cols - kk : 0) : (kk < a.cols ? (int)min(8ll, a.rows - jj) : 0);
    const uint16_t* from = src + (left > 0 ? jj * a.sj + kk * a.sk : 0);
    uint16_t v[8];
    if (left >= 8 && (reinterpret_cast<uintptr_t>(from) & 15) == 0) {
        const uint4 u = *reinterpret_cast<const uint4*>(from);
        memcpy(v, &u, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = from[i < left ? i : 0];
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i >= left) v[i] = 0;
    }
    bool bad = false;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        f[i] = dtype == DT_BF16 ? __uint_as_float((uint32_t)v[i] << 16) : __half2float(__ushort_as_half(v[i]));
        if ((__float_as_uint(f[i]) & 0x7f800000u) == 0x7f800000u) f[i] = copysignf(1.f, f[i]), bad = true;
    }
    if (along) {
        if (jj < a.rows) {
            float4* to = reinterpret_cast<float4*>(dst + jj * a.dst_cols + kk);
            to[0] = make_float4(f[0], f[1], f[2], f[3]), to[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) tile[j + i][k] = f[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int row = (threadIdx.x >> 2) + 64 * i, col = (threadIdx.x & 3) * 4;
            if (j0 + row < a.rows)
                *reinterpret_cast<float4*>(dst + (j0 + row) * a.dst_cols + k0 + col) =
                    make_float4(tile[row][col], tile[row][col + 1], tile[row][col + 2], tile[row][col + 3]);
        }
    }
    return bad;
}

// Adapter e's tokens in order, and the number of tokens of lower adapters:
// each block looks through all indexes, a warp through neighbouring ones.
__device__ void pack_lists(const PackJob& a, int e) {
    __shared__ int warp_own[8], warp_less[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int* first = static_cast<int*>(a.dst);
    int* list = first + a.count + 1;
    // four neighbouring tokens a lane, in one load where the indexes allow
    const long long each = (a.rows + 1023) / 1024 * 128, m0 = min(warp * each, a.rows), m1 = min(m0 + each, a.rows);
    const bool quads = a.id.per == 1 && (reinterpret_cast<uintptr_t>(a.id.ids) & 15) == 0;
    const auto scan = [&](auto see) {
        const auto known = [&](int id) { return (unsigned)id < (unsigned)a.id.count ? id : -1; };
        long long m = m0 + lane * 4;
        if (quads)
            for (; m - lane * 4 + 512 <= m1; m += 512) {
                int4 id[4];
#pragma unroll
                for (int q = 0; q < 4; q++) id[q] = *reinterpret_cast<const int4*>(a.id.ids + m + q * 128);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int v[4] = {known(id[q].x), known(id[q].y), known(id[q].z), known(id[q].w)};
                    see(v, m + q * 128);
                }
            }
        for (; m - lane * 4 < m1; m += 128) {
            int v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = m + i < m1 ? a.id.of(m + i) : -1;
            see(v, m);
        }
    };
    int less = 0, own = 0;  // tokens of lower adapters, of this one
    scan([&](const int (&id)[4], long long) {
#pragma unroll
        for (int i = 0; i < 4; i++) less += id[i] >= 0 && id[i] < e, own += id[i] == e;
    });
    less = __reduce_add_sync(0xffffffffu, less), own = __reduce_add_sync(0xffffffffu, own);
    if (lane == 0) warp_own[warp] = own, warp_less[warp] = less;
    __syncthreads();
    int at = 0, total = 0;
    less = 0;
#pragma unroll
    for (int w = 0; w < 8; w++) less += warp_less[w], at += w < warp ? warp_own[w] : 0, total += warp_own[w];
    if (threadIdx.x == 0) {
        first[e] = less;
        if (e + 1 == a.count) first[a.count] = less + total;
    }
    at += less;
    if (own) scan([&](const int (&id)[4], long long m) {
        unsigned ball[4];
        int before = at;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            ball[i] = __ballot_sync(0xffffffffu, id[i] == e);
            before += __popc(ball[i] & ((1u << lane) - 1)), at += __popc(ball[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (id[i] == e) list[before++] = (int)m + i;
    });
}

__global__ void __launch_bounds__(256) k_pack(const __grid_constant__ PackJobs jobs) {
    release_dependents();
    long long b = blockIdx.x;
    int q = 0;
    while (b >= jobs.job[q].blocks) b -= jobs.job[q++].blocks;
    const PackJob& a = jobs.job[q];
    if (a.kind == PackJob::LISTS) {
        pack_lists(a, (int)b);
    } else if (a.kind == PackJob::COPY) {
        const long long tr = (a.rows + 31) / 32, tc = (a.dst_cols + 127) / 128, e = b / (tr * tc), in = b % (tr * tc);
        pack_tile(a, static_cast<const uint16_t*>(a.src) + e * a.se, static_cast<uint16_t*>(a.dst) + e * a.rows * a.dst_cols, in % tr * 32,
                  (int)(in / tr) * 128);
    } else {
        const int tc = a.dst_cols / 16;
        const long long tr = (a.rows + 127) / 128, e = b / (tr * tc);
        const bool bad = pack_f32(a, static_cast<const uint16_t*>(a.src) + e * a.se, static_cast<float*>(a.dst) + e * a.rows * a.dst_cols,
                                  b / tc % tr * 128, (int)(b % tc) * 16, jobs.dtype);
        const int any = __syncthreads_or(bad);
        if (threadIdx.x == 0) a.bad[b] = any;
    }
}

// ---------------------------------------------------------------- low

// Token by token: WPJ warps share one rank index of NT neighbouring tokens,
// whose factor row is read once where they have one adapter.  Bound: reading
// each token's own factor (r k elements), from L2 where tokens share it.  48
// tokens of 64 adapters, rank 30 over 8960: 8.1 us, 4.2 TB/s.
template <class T, bool VEC, int WPJ, int NT>
__global__ void __launch_bounds__(256) k_low_token(const LowPair both) {
    release_dependents();
    if (both.after_pack[blockIdx.z] == 2) grid_dependency_wait();
    const LowArgs a = both.a[blockIdx.z];
    const long long m0 = (long long)blockIdx.x * NT;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % WPJ;
    const int j = blockIdx.y * (8 / WPJ) + warp / WPJ, rs = low_stride(a.r);
    int e[NT];
    bool one = true;
#pragma unroll
    for (int i = 0; i < NT; i++) {
        e[i] = m0 + i < a.n ? a.id.of(m0 + i) : -1;
        one &= e[i] == e[0];
    }
    float v[NT] = {};
    const T* f[NT];
    const T* x[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) {  // clamped places: what they give is not kept
        x[i] = static_cast<const T*>(a.x) + min(m0 + i, a.n - 1) * a.x_stride;
        f[i] = static_cast<const T*>(a.f.p) + max(e[i], 0) * a.f.se + min(j, a.r - 1) * a.f.sj;
    }
    if (!(one && e[0] < 0)) {
        if constexpr (VEC) {
            constexpr int V = 16 / sizeof(T);
            int k = (part * 32 + lane) * V;
            if (one) {
#pragma unroll 4
                for (; k + V <= a.k; k += 32 * V * WPJ) {
                    const uint4 fk = whole16(f[0], k);
#pragma unroll
                    for (int i = 0; i < NT; i++) v[i] = dot16<T>(whole16(x[i], k), fk, v[i]);
                }
            } else {
#pragma unroll 2
                for (; k + V <= a.k; k += 32 * V * WPJ)
#pragma unroll
                    for (int i = 0; i < NT; i++) v[i] = dot16<T>(whole16(x[i], k), whole16(f[i], k), v[i]);
            }
            if (k < a.k)
#pragma unroll
                for (int i = 0; i < NT; i++) v[i] = dot16<T>(load16(x[i], k, a.k), load16(f[i], k, a.k), v[i]);
        } else {
#pragma unroll 4
            for (int k = part * 32 + lane; k < a.k; k += 32 * WPJ)
#pragma unroll
                for (int i = 0; i < NT; i++) v[i] = fmaf(to_f(x[i][k]), to_f(f[i][k * a.f.sk]), v[i]);
        }
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int q = 16; q; q >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], q);
    }
    if constexpr (WPJ > 1) {
        __shared__ float part_sum[8][NT];
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < NT; i++) part_sum[warp][i] = v[i];
        __syncthreads();
        if (part == 0)
#pragma unroll
            for (int i = 0; i < NT; i++) {
                v[i] = 0.f;
#pragma unroll
                for (int q = 0; q < WPJ; q++) v[i] += part_sum[warp + q][i];
            }
    }
    if (part == 0 && lane == 0 && j < rs) {
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const long long m = m0 + i;
            if (m >= a.n) break;
            const float low = e[i] >= 0 && j < a.r ? (a.scale ? a.scale[e[i]] * v[i] : v[i]) : 0.f;
            if (a.low) a.low[m * rs + j] = a.tf32 ? __uint_as_float(to_tf32(low)) : low;
            if (a.split) {
                uint32_t h, l;
                bf16_terms(low, h, l);
                a.split[m * 2 * rs + j] = (uint16_t)h, a.split[(m * 2 + 1) * rs + j] = (uint16_t)l;
            }
        }
    }
    // what the next launch reads behind its own wait for this one then comes
    // behind the packing too
    if (both.after_pack[blockIdx.z] == 1) grid_dependency_wait();
}

// f32 factors whose contiguous axis is the rank's (the backward call's B):
// 32 rank indexes of four neighbouring tokens a CTA, a lane each, the
// contraction over the warps.  Bound: reading the factor, from L2.  284 tokens,
// rank 64 over 1536: 17 us, about 110 with lanes along the contraction, which
// takes less below rank 32 (634 tokens, rank 13: 13 us, 43 so).
__global__ void __launch_bounds__(1024) k_low_cols(const LowArgs a) {
    constexpr int NT = 4, U = 4;  // U: rows of the factor under way
    __shared__ float part[32][NT][32];
    const long long m0 = (long long)blockIdx.x * NT;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.y * 32 + lane, rs = low_stride(a.r);
    int e[NT];
    const float *f[NT], *x[NT];
    bool one = true;
#pragma unroll
    for (int i = 0; i < NT; i++) {  // clamped places: what they give is not kept
        e[i] = m0 + i < a.n ? a.id.of(m0 + i) : -1;
        one &= e[i] == e[0];
        x[i] = static_cast<const float*>(a.x) + min(m0 + i, a.n - 1) * a.x_stride;
        f[i] = static_cast<const float*>(a.f.p) + max(e[i], 0) * a.f.se + min(j, a.r - 1) * a.f.sj;
    }
    float v[NT] = {};
    if (!(one && e[0] < 0)) {
        const int k0 = (int)((long long)a.k * warp / 32), k1 = (int)((long long)a.k * (warp + 1) / 32);
        for (int k = k0; k < k1; k += U) {
            float fk[U];
            if (one) {
                float xk[U][NT];
#pragma unroll
                for (int q = 0; q < U; q++) {
                    const int at = min(k + q, k1 - 1);
                    fk[q] = f[0][at * a.f.sk];
#pragma unroll
                    for (int i = 0; i < NT; i++) xk[q][i] = x[i][at];
                }
#pragma unroll
                for (int q = 0; q < U; q++)
                    if (k + q < k1)
#pragma unroll
                        for (int i = 0; i < NT; i++) v[i] = fmaf(xk[q][i], fk[q], v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    float xk[U];
#pragma unroll
                    for (int q = 0; q < U; q++) {
                        const int at = min(k + q, k1 - 1);
                        fk[q] = f[i][at * a.f.sk], xk[q] = x[i][at];
                    }
#pragma unroll
                    for (int q = 0; q < U; q++)
                        if (k + q < k1) v[i] = fmaf(xk[q], fk[q], v[i]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NT; i++) part[warp][i][lane] = v[i];
    __syncthreads();
    const int i = threadIdx.x >> 5;  // the first four warps finish a token each
    if (i >= NT || m0 + i >= a.n || j >= rs) return;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 32; w++) sum += part[w][i][lane];
    const int own = a.id.of(m0 + i);
    a.low[(m0 + i) * rs + j] = own >= 0 && j < a.r ? (a.scale ? a.scale[own] * sum : sum) : 0.f;
}

// ---------------------------------------------------------------- projection

// f32: BM x BN outputs per CTA, TM x TN per thread in two halves, 16 of the
// contraction at a time, the next D times as many on their way in registers.  The
// adapters' terms are more of the same contraction, one after the other for
// up to kF32Adapters adapters of the tile, each added to its own tokens' sums
// only; with more of them each output takes its token's own.  A
// cluster of S CTAs shares both where the tiles are few, and each finishes
// some of the rows.  On the FMA pipe: the tensor cores' TF32 would need
// three products and rounds its sums towards zero.  1024 tokens of 1536 -> 1536:
// 170 us, 28 TFLOP/s; 201 of 1001 -> 771 (14 tiles, eight CTAs each): 30 us.
constexpr int kF32Adapters = 8;

template <int BM, int BN>
struct F32Tile {
    static constexpr int BK = 16, kTiles = 2 * BK * (BM + 4 + BN + 4) * 4, kSums = BM * (BN + 1) * 4;
    static constexpr int kSmem = kTiles > kSums ? kTiles : kSums;
};

template <int BM, int BN, int TM, int TN, int D>
__global__ void __launch_bounds__(256, BM == 64 ? 2 : 1) k_project_f32(const ProjectArgs a, int vec_x, int vec_w, int vec_g) {
    constexpr int BK = F32Tile<BM, BN>::BK, LX = BM * BK / 1024, LW = BN * BK / 1024;  // float4 loads of a thread
    static_assert((BM / TM) * (BN / TN) == 256, "one thread per TM x TN outputs");
    extern __shared__ __align__(16) float room[];
    float (*const xs)[BK][BM + 4] = reinterpret_cast<float (*)[BK][BM + 4]>(room);
    float (*const ws)[BK][BN + 4] = reinterpret_cast<float (*)[BK][BN + 4]>(room + 2 * BK * (BM + 4));
    float (*const part)[BN + 1] = reinterpret_cast<float (*)[BN + 1]>(room);  // behind the contraction
    __shared__ __align__(16) int ids[BM];
    cg::cluster_group cluster = cg::this_cluster();
    const int S = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long m0 = (long long)(blockIdx.x / S) * BM;
    const int o0 = blockIdx.y * BN;
    static_assert(BN / TN == 16, "16 x 16 threads");
    // a warp is 4 x 8 of them: its reads of w fill the banks once
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tx = (warp & 1) * 8 + (lane & 7), ty = (warp >> 1) * 4 + (lane >> 3);
    const auto row_of = [&](int i) { return ty * 4 + i / 4 * (BM / (TM / 4)) + i % 4; };
    const auto col_of = [&](int j) { return tx * 4 + j / 4 * (BN / (TN / 4)) + j % 4; };
    if (threadIdx.x < BM) ids[threadIdx.x] = m0 + threadIdx.x < a.n ? a.id.of(m0 + threadIdx.x) : -1;
    float acc[TM][TN] = {};
    // acc += rows x [n][k] times w [o][k], or [k][o] where `w_t`, over blocks
    // [b0, b1) of k; of an adapter's factor for the rows in `mine` only
    const auto contract = [&](const float* x, long long x_stride, bool vx, const float* w, long long w_stride, bool w_t, bool vw, int kk,
                              int b0, int b1, auto one, unsigned mine) {
        float4 nx[D][LX], nw[D][LW];
        // four neighbours of a row that ends at `n`, from clamped places: what
        // is behind the end is replaced by zeros on the way to shared memory,
        // since a use of the values here would wait for them
        const auto quad = [](const float* row, int at, int n, bool vec) {
            if (vec && at + 4 <= n) return *reinterpret_cast<const float4*>(row + at);
            return make_float4(row[min(at, n - 1)], row[min(at + 1, n - 1)], row[min(at + 2, n - 1)], row[min(at + 3, n - 1)]);
        };
        const auto load = [&](int b, float4 (&nx)[LX], float4 (&nw)[LW]) {
            const int k0 = b * BK;
#pragma unroll
            for (int i = 0; i < LX; i++) {
                const int q = threadIdx.x + 256 * i;
                nx[i] = quad(x + min(m0 + q / 4, a.n - 1) * x_stride, k0 + q % 4 * 4, kk, vx);
            }
#pragma unroll
            for (int i = 0; i < LW; i++) {
                const int q = threadIdx.x + 256 * i;
                if (w_t) nw[i] = quad(w + (long long)min(k0 + q / (BN / 4), kk - 1) * w_stride, o0 + q % (BN / 4) * 4, a.o, vw);
                else nw[i] = quad(w + (long long)min(o0 + q / 4, a.o - 1) * w_stride, k0 + q % 4 * 4, kk, vw);
            }
        };
        const auto store = [&](int b, int s, float4 (&nx)[LX], float4 (&nw)[LW]) {
            const int left = kk - b * BK;
            const auto cut = [&](float4 v, int k) {
                return make_float4(k < left ? v.x : 0.f, k + 1 < left ? v.y : 0.f, k + 2 < left ? v.z : 0.f, k + 3 < left ? v.w : 0.f);
            };
#pragma unroll
            for (int i = 0; i < LX; i++) {
                const int q = threadIdx.x + 256 * i, m = q / 4, k = q % 4 * 4;
                const float4 v = cut(nx[i], k);
                xs[s][k][m] = v.x, xs[s][k + 1][m] = v.y, xs[s][k + 2][m] = v.z, xs[s][k + 3][m] = v.w;
            }
#pragma unroll
            for (int i = 0; i < LW; i++) {
                const int q = threadIdx.x + 256 * i;
                if (w_t) {
                    const bool in = q / (BN / 4) < left;
                    *reinterpret_cast<float4*>(&ws[s][q / (BN / 4)][q % (BN / 4) * 4]) = in ? nw[i] : make_float4(0.f, 0.f, 0.f, 0.f);
                } else {
                    const int o = q / 4, k = q % 4 * 4;
                    const float4 v = cut(nw[i], k);
                    ws[s][k][o] = v.x, ws[s][k + 1][o] = v.y, ws[s][k + 2][o] = v.z, ws[s][k + 3][o] = v.w;
                }
            }
        };
        if (b0 >= b1) return;
#pragma unroll
        for (int d = 0; d < D; d++)
            if (b0 + d < b1) load(b0 + d, nx[d], nw[d]);
        store(b0, 0, nx[0], nw[0]);
        __syncthreads();
        for (int c = b0; c < b1; c += D) {
#pragma unroll
            for (int d = 0; d < D; d++) {
                const int b = c + d, s = (b - b0) & 1;
                if (b >= b1) break;
                if (b + D < b1) load(b + D, nx[d], nw[d]);
#pragma unroll(BM == 64 ? BK : BK / 2)
                for (int k = 0; k < BK; k++) {  // 128: whole, it would take the registers of the loads under way
                    float xv[TM], wv[TN];
#pragma unroll
                    for (int i = 0; i < TM; i += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&xs[s][k][ty * 4 + i / 4 * (BM / (TM / 4))]);
                        xv[i] = f.x, xv[i + 1] = f.y, xv[i + 2] = f.z, xv[i + 3] = f.w;
                    }
#pragma unroll
                    for (int i = 0; i < TN; i += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&ws[s][k][tx * 4 + i / 4 * (BN / (TN / 4))]);
                        wv[i] = f.x, wv[i + 1] = f.y, wv[i + 2] = f.z, wv[i + 3] = f.w;
                    }
#pragma unroll
                    for (int i = 0; i < TM; i++)
                        if (!decltype(one)::value || (mine >> i & 1))
#pragma unroll
                            for (int j = 0; j < TN; j++) acc[i][j] = fmaf(xv[i], wv[j], acc[i][j]);
                }
                if (b + 1 < b1) store(b + 1, s ^ 1, nx[(d + 1) % D], nw[(d + 1) % D]);
                __syncthreads();
            }
        }
    };
    if (a.w) {
        const int blocks = (a.k + BK - 1) / BK;
        contract(static_cast<const float*>(a.x), a.x_stride, vec_x, static_cast<const float*>(a.w), a.w_stride, a.w_t, vec_w, a.k,
                 blocks * rank / S, blocks * (rank + 1) / S, std::false_type(), 0);
    }
    __syncthreads();
    const bool g_t = a.g.sk == 1 && a.g.sj != 1;  // [r][o], else [o][r]
    int distinct = 0;
    const auto above = [&](int e) {  // the tile's next adapter; every thread looks for itself
        int next = INT_MAX;
#pragma unroll 4
        for (int i = 0; i < BM; i += 4) {
            const int4 q = *reinterpret_cast<const int4*>(ids + i);
            next = min(min(next, q.x > e ? q.x : INT_MAX), min(q.y > e ? q.y : INT_MAX, min(q.z > e ? q.z : INT_MAX, q.w > e ? q.w : INT_MAX)));
        }
        return next;
    };
    for (int e = above(-1); e != INT_MAX && distinct <= kF32Adapters; e = above(e)) distinct++;
    const bool each = distinct > kF32Adapters;
    for (int e = above(-1), at = 0; !each && e != INT_MAX; e = above(e), at++) {
        if (at % S != rank) continue;
        unsigned mine = 0;
#pragma unroll
        for (int i = 0; i < TM; i++) mine |= (unsigned)(ids[row_of(i)] == e) << i;
        contract(a.low, low_stride(a.r), true, static_cast<const float*>(a.g.p) + e * a.g.se, g_t ? a.g.sj : a.g.sk, g_t, vec_g, a.r, 0,
                 (a.r + BK - 1) / BK, std::true_type(), mine);
    }
    const auto finish = [&](long long m, int o, float v) {
        if (a.bias) v += static_cast<const float*>(a.bias)[o];
        if (a.base) v += static_cast<const float*>(a.base)[m * a.base_stride + o];
        if (each && ids[m - m0] >= 0) {
            const float *low = a.low + m * low_stride(a.r), *g = static_cast<const float*>(a.g.p) + ids[m - m0] * a.g.se + o * a.g.sk;
            constexpr int U = 8;  // blocks of loads from clamped places
            for (int j = 0; j < a.r; j += U) {
                float l[U], f[U];
#pragma unroll
                for (int i = 0; i < U; i++) l[i] = low[min(j + i, a.r - 1)], f[i] = g[min(j + i, a.r - 1) * a.g.sj];
#pragma unroll
                for (int i = 0; i < U; i++)
                    if (j + i < a.r) v = fmaf(l[i], f[i], v);
            }
        }
        static_cast<float*>(a.out)[m * a.out_stride + o] = v;
    };
    if (S > 1 || each) {
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++) part[row_of(i)][col_of(j)] = acc[i][j];
        if (S > 1) cluster.sync();
        else __syncthreads();
        const int row0 = BM * rank / S, rows = BM * (rank + 1) / S - row0;
        for (int q = threadIdx.x; q < rows * BN; q += 256) {
            const int row = row0 + q / BN, col = q % BN;
            if (m0 + row >= a.n || o0 + col >= a.o) continue;
            float v = 0.f;
            for (int c = 0; c < S; c++) v += *cluster.map_shared_rank(&part[row][col], c);
            finish(m0 + row, o0 + col, v);
        }
        if (S > 1) cluster.sync();
    } else {
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++)
                if (m0 + row_of(i) < a.n && o0 + col_of(j) < a.o) finish(m0 + row_of(i), o0 + col_of(j), acc[i][j]);
    }
}

// sum_j low[j] b[j] for a row of a factor; 16 bytes at a time where r and the
// row allow, else 4, else 2.
template <class T>
__device__ __forceinline__ float dot_low(const float* low, const T* b, int r, float v) {
    if ((r & 7) == 0 && (reinterpret_cast<uintptr_t>(b) & 15) == 0) {
#pragma unroll 4
        for (int j = 0; j < r; j += 8) {
            const uint4 u = *reinterpret_cast<const uint4*>(b + j);
            const float4 p = *reinterpret_cast<const float4*>(low + j), q = *reinterpret_cast<const float4*>(low + j + 4);
            const float2 f0 = pair_f<T>(u.x), f1 = pair_f<T>(u.y), f2 = pair_f<T>(u.z), f3 = pair_f<T>(u.w);
            v = fmaf(p.x, f0.x, v), v = fmaf(p.y, f0.y, v), v = fmaf(p.z, f1.x, v), v = fmaf(p.w, f1.y, v);
            v = fmaf(q.x, f2.x, v), v = fmaf(q.y, f2.y, v), v = fmaf(q.z, f3.x, v), v = fmaf(q.w, f3.y, v);
        }
    } else if ((r & 1) == 0 && (reinterpret_cast<uintptr_t>(b) & 3) == 0) {
        // blocks of unconditional loads, from clamped places behind the last rank
        for (int j = 0; j < r; j += 16) {
            float2 l[8];
            uint32_t q[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int at = min(j + 2 * i, r - 2);
                q[i] = *reinterpret_cast<const uint32_t*>(b + at), l[i] = *reinterpret_cast<const float2*>(low + at);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 f = pair_f<T>(q[i]);
                if (j + 2 * i < r) v = fmaf(l[i].x, f.x, v), v = fmaf(l[i].y, f.y, v);
            }
        }
    } else {
        for (int j = 0; j < r; j += 8) {
            float l[8], f[8];
#pragma unroll
            for (int i = 0; i < 8; i++) l[i] = low[min(j + i, r - 1)], f[i] = to_f(b[min(j + i, r - 1)]);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (j + i < r) v = fmaf(l[i], f[i], v);
        }
    }
    return v;
}

// f32, few tokens: a warp for each output of four tokens.  Bound: reading W,
// and the launches' latency: one token of 1536 -> 1536 takes 6 us, 23 as a tile;
// 31 of them take 37 us, 28 as tiles.
__global__ void __launch_bounds__(256) k_project_f32_few(const ProjectArgs a, int vec) {
    constexpr int NT = 4, U = 4;  // U: loads of a row under way
    const int lane = threadIdx.x & 31, o = blockIdx.x * 8 + (threadIdx.x >> 5), m0 = blockIdx.y * NT;
    float v[NT] = {};
    if (a.w && o < a.o) {
        const float* w = static_cast<const float*>(a.w) + o * a.w_stride;
        const float* x[NT];
#pragma unroll
        for (int i = 0; i < NT; i++) x[i] = static_cast<const float*>(a.x) + min((long long)m0 + i, a.n - 1) * a.x_stride;
        const int whole = vec ? a.k / 4 * 4 : 0;
        for (int k = lane * 4; k < whole; k += 128 * U) {
            float4 f[U];
#pragma unroll
            for (int q = 0; q < U; q++) f[q] = *reinterpret_cast<const float4*>(w + min(k + 128 * q, whole - 4));
#pragma unroll
            for (int q = 0; q < U; q++)
                if (k + 128 * q < whole)
#pragma unroll
                    for (int i = 0; i < NT; i++) {
                        const float4 g = *reinterpret_cast<const float4*>(x[i] + k + 128 * q);
                        v[i] = fmaf(f[q].x, g.x, v[i]), v[i] = fmaf(f[q].y, g.y, v[i]), v[i] = fmaf(f[q].z, g.z, v[i]), v[i] = fmaf(f[q].w, g.w, v[i]);
                    }
        }
        for (int k = whole + lane; k < a.k; k += 32 * 2 * U) {
            float f[2 * U];
#pragma unroll
            for (int q = 0; q < 2 * U; q++) f[q] = w[min(k + 32 * q, a.k - 1)];
#pragma unroll
            for (int q = 0; q < 2 * U; q++)
                if (k + 32 * q < a.k)
#pragma unroll
                    for (int i = 0; i < NT; i++) v[i] = fmaf(f[q], x[i][k + 32 * q], v[i]);
        }
    }
    grid_dependency_wait();
    if (o >= a.o) return;
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const int m = m0 + i, e = m < a.n ? a.id.of(m) : -1;
        if (e >= 0) {
            const float *low = a.low + m * low_stride(a.r), *g = static_cast<const float*>(a.g.p) + e * a.g.se + o * a.g.sk;
            for (int j = lane; j < a.r; j += 32) v[i] = fmaf(low[j], g[j], v[i]);
        }
#pragma unroll
        for (int q = 16; q; q >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], q);
        if (lane == i && m < a.n) {
            float y = v[i];
            if (a.bias) y += static_cast<const float*>(a.bias)[o];
            if (a.base) y += static_cast<const float*>(a.base)[m * a.base_stride + o];
            static_cast<float*>(a.out)[m * a.out_stride + o] = y;
        }
    }
}

// Few tokens: a cluster of S CTAs streams 16 rows of W once past NB * 8
// tokens, its 8 S warps sharing the contraction in 32-wide blocks.  Operands go
// from global memory to the matrix instructions' registers: a thread's 16
// bytes of a row are the k indexes of two instructions, in the same (permuted)
// order for W and x.  Bound: reading W, and the launch's latency; the stream
// starts before low is there, and waits for it only to add the adapters' terms.
// One token of 1536 -> 1536 with rank 16: 9.0 us with low.
template <class T, int NB>
__global__ void __launch_bounds__(256) k_project_small(const ProjectArgs a) {
    cg::cluster_group cluster = cg::this_cluster();
    const int S = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int o0 = (blockIdx.x / S) * 16;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    extern __shared__ float red[];  // [8][16][RS], the sums over the warps in the first
    constexpr int RS = NB * 8 + 1;
    if (a.w) {
        float acc[NB][4] = {};
        const T* wr[2];
#pragma unroll
        for (int i = 0; i < 2; i++) wr[i] = static_cast<const T*>(a.w) + (long long)min(o0 + g + 8 * i, a.o - 1) * a.w_stride;
        const T* xr[NB];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) xr[nb] = static_cast<const T*>(a.x) + min((long long)nb * 8 + g, a.n - 1) * a.x_stride;
        const auto block = [&](auto load, int k) {
            uint4 w[2], x[NB];
#pragma unroll
            for (int i = 0; i < 2; i++) w[i] = load(wr[i], k);
#pragma unroll
            for (int nb = 0; nb < NB; nb++) x[nb] = load(xr[nb], k);
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                mma16<T>(acc[nb], w[0].x, w[1].x, w[0].y, w[1].y, x[nb].x, x[nb].y);
                mma16<T>(acc[nb], w[0].z, w[1].z, w[0].w, w[1].w, x[nb].z, x[nb].w);
            }
        };
        int k = (rank * 8 + warp) * 32;
#pragma unroll 4
        for (; k + 32 <= a.k; k += S * 256) block([](const T* row, int at) { return whole16(row, at); }, k + 8 * t);
        if (k < a.k) block([&](const T* row, int at) { return load16(row, at, a.k); }, k + 8 * t);
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int c = 0; c < 4; c++) red[(warp * 16 + g + (c >> 1) * 8) * RS + nb * 8 + 2 * t + (c & 1)] = acc[nb][c];
        __syncthreads();
        if (S > 1) {
            for (int i = threadIdx.x; i < 16 * NB * 8; i += 256) {
                float* p = red + (i / (NB * 8)) * RS + i % (NB * 8);
                float v = 0.f;
#pragma unroll
                for (int q = 0; q < 8; q++) v += p[q * 16 * RS];
                *p = v;
            }
            cluster.sync();
        }
    }
    grid_dependency_wait();
    const int rs = low_stride(a.r), per = 16 * NB * 8 / S;
    for (int i = rank * per + threadIdx.x; i < (rank + 1) * per; i += 256) {
        const int row = i % 16, m = i / 16, o = o0 + row;
        if (o >= a.o || m >= a.n) continue;
        float v = a.bias ? to_f(static_cast<const T*>(a.bias)[o]) : 0.f;
        if (a.base) v += to_f(static_cast<const T*>(a.base)[m * a.base_stride + o]);
        const int e = a.id.of(m);
        if (e >= 0) v = dot_low(a.low + m * rs, static_cast<const T*>(a.g.p) + e * a.g.se + o * a.g.sk, a.r, v);
        if (a.w) {
            float* p = red + row * RS + m;
            if (S > 1)
                for (int q = 0; q < S; q++) v += *cluster.map_shared_rank(p, q);
            else
#pragma unroll
                for (int q = 0; q < 8; q++) v += p[q * 16 * RS];
        }
        static_cast<T*>(a.out)[m * a.out_stride + o] = from_f<T>(v);
    }
    if (S > 1) cluster.sync();
}

// ---------------------------------------------------------------- gradients of the factors


constexpr int kGradChunk = 32;  // groups whose tokens are listed in shared memory at a time

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <class T, int RB>
struct GradTile {
    static constexpr bool kSplit = std::is_same<T, __nv_bfloat16>::value;  // low as two bf16 terms
    // 128 features; rows four (split: 16 bytes; else 8 banks) apart from a multiple of all banks
    static constexpr int kRow = kSplit ? 272 : sizeof(T) == 4 ? 136 * 4 : 288;
    static constexpr int kURow = kSplit ? RB * 32 + 16 : RB * 32 + 32;  // bytes
    static constexpr int kX = 32 * kRow, kU = 32 * kURow;
    static constexpr int kStages = sizeof(T) == 4 || RB == 8 ? 4 : 5;
    static constexpr int kPerSm = sizeof(T) == 4 || RB == 8 ? 2 : 3;  // CTAs
    static constexpr int kSmem = kStages * (kX + kU);
};

__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

// A window of W places of the tokens' list (adapter by adapter), 128 features and RB * 8
// rank indexes per CTA, so that CTAs have the same work however the tokens are spread
// over the adapters.  For each adapter in the window, in groups of 32 tokens, the rows
// are gathered and low^T x summed with matrix instructions whose 16-row axis are the
// features and whose contraction the tokens.  bf16: 16 x 8 x 16 products with low's two
// bf16 terms, which hold it to 2^-15, operands transposed on the way from shared memory.
// Else 16 x 8 x 8 TF32 products: low is split into two TF32 parts, which leaves 2^-20
// beside fp16 x, exact in TF32 (65 us beside a base for 4096 tokens of 1536 and 1536,
// rank 64; 57 with low in 11 bits alone), and 2^-22 beside f32 x, which is split as well
// (their products of infinities left apart cost 1 to 3 % of an f32 call: 1024 tokens of
// 1536 -> 1536, rank 16: 258 us, 255 with NaNs for them).  An adapter that lies in one
// window is written here; the others' sums over a window go to the workspace, and
// k_grad_sum adds them in the windows' order.  Bound: reading x once per 64 rank
// indexes.  8192 tokens of 1536 and 1536, rank 16, three adapters: 18 us, 2.8 TB/s; 2048
// of 8960 and 1536, rank 32: 26 us.
template <class T, int RB>
__global__ void __launch_bounds__(256, (GradTile<T, RB>::kPerSm)) k_grad(const GradPair both, int tiles0, int window, float* partial, int dependent) {
    using L = GradTile<T, RB>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int own[kGradChunk * 32], start;
    release_dependents();
    const int tile = blockIdx.x;
    const GradArgs a = both.g[tile >= tiles0];
    const int k0 = (tile >= tiles0 ? tile - tiles0 : tile) * 128, j0 = blockIdx.y * RB * 8;
    const int rs = low_stride(both.r);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int wf = warp & 3, wt = warp >> 2;
    // what is read here was complete before the launch before this one let it
    // start (k_project.cu); that launch itself is waited for in the end
    const int* first = both.first;
    const int pos0 = blockIdx.z * window, total = first[both.adapters], pos1 = min(pos0 + window, total);
    for (int e = threadIdx.x; e < both.adapters; e += 256)
        if (first[e] <= pos0 && pos0 < first[e + 1]) start = e;
    __syncthreads();

    // this thread's part of every group: 16 bytes at one place of some rows
    constexpr int C = 128 * (int)sizeof(T) / 16, kRows = 256 / C, kXParts = 32 / kRows;  // of x
    constexpr int CU = RB * 2, kURows = 256 / CU < 32 ? 256 / CU : 32, kUParts = 32 / kURows;  // of low
    const int xc = threadIdx.x % C, xrow = threadIdx.x / C, uc = threadIdx.x % CU, urow = threadIdx.x / CU;
    const int xbytes = min(16, max(0, (a.k - k0) * (int)sizeof(T) - xc * 16));
    // split: RB parts of the high terms, RB of the low ones
    const int uj = L::kSplit ? j0 + uc % RB * 8 : j0 + uc * 4, ufirst = L::kSplit ? (uc / RB * rs + uj) * 2 : uj * 4;
    const int ubytes = uj < rs && urow < 32 ? 16 : 0;
    const char* xfrom = static_cast<const char*>(a.x) + (xbytes ? (size_t)k0 * sizeof(T) + xc * 16 : 0);
    const char* ufrom = static_cast<const char*>(a.low) + (ubytes ? ufirst : 0);
    const long long xpitch = a.x_stride * (long long)sizeof(T);
    const uint32_t base = smem_u32(smem), xto = base + xrow * L::kRow + xc * 16, uto = base + L::kX + urow * L::kURow + uc * 16;

    int e = start;
    for (int pos = pos0; pos < pos1; e++) {
        const int e0 = first[e], e1 = first[e + 1], end = min(e1, pos1);
        if (e1 <= pos) continue;
        float acc[2][RB][4] = {};
        const int all = (end - pos + 31) / 32;
        for (int q0 = 0; q0 < all; q0 += kGradChunk) {
            const int groups = min(kGradChunk, all - q0);
            for (int i = threadIdx.x; i < groups * 32; i += 256) {
                const int at = pos + q0 * 32 + i;
                own[i] = at < end ? both.list[at] : -1;
            }
            __syncthreads();
            uint32_t put = 0, take = 0;  // stages' offsets
            const auto next = [](uint32_t at) { return at + (L::kX + L::kU) == L::kSmem ? 0u : at + (L::kX + L::kU); };
            const auto fetch = [&](int q) {
                if (q < groups) {
#pragma unroll
                    for (int i = 0; i < kXParts; i++) {
                        const int m = own[q * 32 + xrow + i * kRows];
                        cp_async16(xto + put + i * kRows * L::kRow, xfrom + max(m, 0) * xpitch, m >= 0 ? xbytes : 0);
                    }
                    if (urow < 32)
#pragma unroll
                        for (int i = 0; i < kUParts; i++) {
                            const int m = own[q * 32 + urow + i * kURows];
                            cp_async16(uto + put + i * kURows * L::kURow, ufrom + max(m, 0) * (long long)(rs * 4), m >= 0 ? ubytes : 0);
                        }
                }
                put = next(put);
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll
            for (int q = 0; q < L::kStages - 1; q++) fetch(q);
            for (int q = 0; q < groups; q++, take = next(take)) {
                asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 2) : "memory");
                __syncthreads();
                fetch(q + L::kStages - 1);
                const uint8_t* sx = smem + take;
                if constexpr (L::kSplit) {
                    // 16 tokens a warp; lanes address rows of 8 x 8 blocks: tokens down, features / rank indexes across
                    const uint32_t xat = base + take + (wt * 16 + (lane >> 4) * 8 + (lane & 7)) * L::kRow + (wf * 32 + (lane >> 3 & 1) * 8) * 2;
                    const uint32_t uat = base + take + L::kX + (wt * 16 + (lane & 15)) * L::kURow + (lane >> 4) * 16;
                    uint32_t f[2][4];
                    ldmatrix4_trans(f[0], xat);
                    ldmatrix4_trans(f[1], xat + 32);
#pragma unroll
                    for (int term = 0; term < 2; term++)
#pragma unroll
                        for (int nb = 0; nb < RB; nb += 2) {
                            uint32_t u[4];
                            ldmatrix4_trans(u, uat + term * RB * 16 + nb * 16);
#pragma unroll
                            for (int q = 0; q < 2; q++) {
                                mma16<T>(acc[q][nb], f[q][0], f[q][1], f[q][2], f[q][3], u[0], u[1]);
                                mma16<T>(acc[q][nb + 1], f[q][0], f[q][1], f[q][2], f[q][3], u[2], u[3]);
                            }
                        }
                    continue;
                }
                const float* su = reinterpret_cast<const float*>(sx + L::kX);
                constexpr int UR = L::kURow / 4;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int tok = (wt * 2 + h) * 8 + t;
                    // four features of two tokens per thread: rows g and g + 8 of two products
                    float f[2][4];
                    uint32_t odd = 0;  // fp16: signs of exponents that are full
#pragma unroll
                    for (int z = 0; z < 2; z++) {
                        const uint8_t* p = sx + (tok + 4 * z) * L::kRow + (wf * 32 + 4 * g) * sizeof(T);
                        if constexpr (sizeof(T) == 4) {
                            const float4 v = *reinterpret_cast<const float4*>(p);
                            f[z][0] = v.x, f[z][1] = v.y, f[z][2] = v.z, f[z][3] = v.w;
                        } else {
                            const uint2 v = *reinterpret_cast<const uint2*>(p);
                            const float2 lo = pair_f<T>(v.x), hi = pair_f<T>(v.y);
                            odd |= ((v.x & 0x7c007c00u) + 0x04000400u) | ((v.y & 0x7c007c00u) + 0x04000400u);
                            f[z][0] = lo.x, f[z][1] = lo.y, f[z][2] = hi.x, f[z][3] = hi.y;
                        }
                    }
                    uint32_t am[2][4], al[2][4];
                    bool special = odd & 0x80008000u;
#pragma unroll
                    for (int q2 = 0; q2 < 2; q2++)
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            const float v = f[z >> 1][q2 * 2 + (z & 1)];
                            if constexpr (sizeof(T) == 4) special |= tf32_terms(v, am[q2][z], al[q2][z]);
                            else am[q2][z] = __float_as_uint(v);
                        }
                    // an infinity of x times the lower term of low would be a NaN
                    // where that is zero or of the other sign
                    special = __any_sync(0xffffffffu, special);
#pragma unroll
                    for (int nb = 0; nb < RB; nb++) {
                        const float b0 = su[tok * UR + nb * 8 + g], b1 = su[(tok + 4) * UR + nb * 8 + g];
                        uint32_t m0b, m1b, l0, l1;
                        bool s0 = false, s1 = false;
                        if constexpr (sizeof(T) == 4) s0 = tf32_terms(b0, m0b, l0), s1 = tf32_terms(b1, m1b, l1);
                        else m0b = __float_as_uint(b0), m1b = __float_as_uint(b1), l0 = tf32_rest(b0), l1 = tf32_rest(b1);
#pragma unroll
                        for (int q2 = 0; q2 < 2; q2++) {
                            if constexpr (sizeof(T) == 4) mma8_tf32(acc[q2][nb], al[q2], s0 ? 0u : m0b, s1 ? 0u : m1b);
                            if (!special) mma8_tf32(acc[q2][nb], am[q2], l0, l1);
                            mma8_tf32(acc[q2][nb], am[q2], m0b, m1b);
                        }
                    }
                    if (special) {
#pragma unroll
                        for (int q2 = 0; q2 < 2; q2++)
#pragma unroll
                            for (int z = 0; z < 4; z++)
                                if ((am[q2][z] & 0x7f800000u) == 0x7f800000u) am[q2][z] = 0u;
#pragma unroll
                        for (int nb = 0; nb < RB; nb++) {
                            const float b0 = su[tok * UR + nb * 8 + g], b1 = su[(tok + 4) * UR + nb * 8 + g];
                            uint32_t m0b, m1b, l0, l1;
                            if constexpr (sizeof(T) == 4) tf32_terms(b0, m0b, l0), tf32_terms(b1, m1b, l1);
                            else l0 = tf32_rest(b0), l1 = tf32_rest(b1);
#pragma unroll
                            for (int q2 = 0; q2 < 2; q2++) mma8_tf32(acc[q2][nb], am[q2], l0, l1);
                        }
                    }
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();
        }

        // the two token halves: sum[rank index][feature]
        float* sum = reinterpret_cast<float*>(smem);
        constexpr int SR = 129;
        static_assert(RB * 8 * SR * 4 <= L::kSmem, "the sums fit where the tiles were");
#pragma unroll
        for (int half = 1; half >= 0; half--) {
            if (wt == half)
#pragma unroll
                for (int q = 0; q < 2; q++)
#pragma unroll
                    for (int nb = 0; nb < RB; nb++)
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const int feature = L::kSplit ? 16 * q + g + 8 * (c >> 1) : 4 * g + 2 * q + (c >> 1);
                            float* p = sum + (nb * 8 + 2 * t + (c & 1)) * SR + wf * 32 + feature;
                            *p = half ? acc[q][nb][c] : *p + acc[q][nb][c];
                        }
            __syncthreads();
        }
        const bool whole = e0 >= pos0 && e1 <= pos1;
        float* to = partial + ((((long long)blockIdx.z * 2 + (e0 >= pos0)) * gridDim.y + blockIdx.y) * gridDim.x + tile) * (RB * 8 * 128);
        for (int i = threadIdx.x; i < RB * 8 * 128; i += 256) {
            // consecutive threads along whichever axis of the result is contiguous
            const int j = a.sk == 1 ? i >> 7 : i % (RB * 8), k = a.sk == 1 ? i & 127 : i / (RB * 8);
            const float v = sum[j * SR + k];
            if (!whole) to[i] = v;
            else if (j0 + j < both.r && k0 + k < a.k)
                static_cast<T*>(a.out)[e * a.se + (j0 + j) * a.sj + (long long)(k0 + k) * a.sk] = from_f<T>(v);
        }
        __syncthreads();
        pos = end;
    }
    if (dependent) grid_dependency_wait();
}

// Four neighbouring results of one thread, 1024 of a CTA at a time.
template <class T>
__device__ __forceinline__ void put4(T* to, const float (&r)[4]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(to) = make_float4(r[0], r[1], r[2], r[3]);
    } else {
        T h[4] = {from_f<T>(r[0]), from_f<T>(r[1]), from_f<T>(r[2]), from_f<T>(r[3])};
        uint2 u;
        memcpy(&u, h, 8);
        *reinterpret_cast<uint2*>(to) = u;
    }
}

// The gradients of adapters whose tokens lie in several windows, and zeros for
// those without tokens; `chunks` times 1024 results of a tile per CTA.  Bound:
// latency behind k_grad, 4 us at 8192 tokens.
template <class T, int RB>
__global__ void __launch_bounds__(256) k_grad_sum(const GradPair both, int tiles0, int window, int chunks, const float* partial) {
    grid_dependency_wait();
    constexpr int kChunks = RB * 8 * 128 / 1024;
    const int tile = blockIdx.x, e = blockIdx.z, groups = kChunks / chunks, pass = blockIdx.y / groups;
    const GradArgs a = both.g[tile >= tiles0];
    const int k0 = (tile >= tiles0 ? tile - tiles0 : tile) * 128, j0 = pass * RB * 8;
    const int e0 = both.first[e], e1 = both.first[e + 1], w0 = e0 / window, w1 = e1 > e0 ? (e1 - 1) / window : w0 - 1;
    if (w0 == w1) return;
    const long long each = (long long)(gridDim.y / groups) * gridDim.x * (RB * 8 * 128);  // between a window's two sums
    for (int chunk = blockIdx.y % groups * chunks, last = chunk + chunks; chunk < last; chunk++) {
        const int i = (chunk * 256 + threadIdx.x) * 4;
        const float* from = partial + ((long long)pass * gridDim.x + tile) * (RB * 8 * 128) + i;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        const auto add = [&](float4 f) { v.x += f.x, v.y += f.y, v.z += f.z, v.w += f.w; };
        // the adapter begins in its first window and goes on in the others
        if (w1 > w0) add(*reinterpret_cast<const float4*>(from + (w0 * 2 + 1) * each));
        int w = w0 + 1;
        for (; w + 7 <= w1; w += 8) {
            float4 f[8];
#pragma unroll
            for (int q = 0; q < 8; q++) f[q] = *reinterpret_cast<const float4*>(from + (w + q) * 2 * each);
#pragma unroll
            for (int q = 0; q < 8; q++) add(f[q]);
        }
        for (; w <= w1; w++) add(*reinterpret_cast<const float4*>(from + w * 2 * each));
        const float r[4] = {v.x, v.y, v.z, v.w};
        // along whichever axis of the result is contiguous
        const int j = a.sk == 1 ? i >> 7 : i % (RB * 8), k = a.sk == 1 ? i & 127 : i / (RB * 8), left = a.sk == 1 ? a.k - (k0 + k) : both.r - (j0 + j);
        if (a.sk == 1 ? j0 + j >= both.r : k0 + k >= a.k) continue;
        T* to = static_cast<T*>(a.out) + e * a.se + (j0 + j) * a.sj + (long long)(k0 + k) * a.sk;
        if (left >= 4 && reinterpret_cast<uintptr_t>(to) % (4 * sizeof(T)) == 0) put4(to, r);
        else
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (q < left) to[q] = from_f<T>(r[q]);
    }
}

int sm_count() {
    int dev = 0, sms = 1;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

template <class T>
cudaError_t low_launch(const LowArgs* a, int count, bool vec, const int* after_pack, cudaStream_t s) {
    const long long n = a[0].n;
    if (sizeof(T) == 2 && !low_by_token(n, a[0].k, a[count - 1].k, a[0].r, a[0].id.count))
        return launch_low_tc(a, count, std::is_same<T, __half>::value ? DT_F16 : DT_BF16, after_pack, s);
    if (sizeof(T) == 4 && a[count - 1].f.sk >= 32) {
        const LowArgs& u = a[count - 1];
        const cudaError_t e = count == 2 ? low_launch<T>(a, 1, vec, after_pack, s) : cudaSuccess;
        if (e != cudaSuccess) return e;
        KScope ks("adapter_low", s);
        return launch_cl(1, k_low_cols, dim3((unsigned)((n + 3) / 4), (u.r + 31) / 32), 1024, 0, s, u);
    }
    const LowPair both{{a[0], a[count - 1]}, {after_pack[0], after_pack[count - 1]}};
    const int kmax = a[0].k > a[count - 1].k ? a[0].k : a[count - 1].k;
    KScope ks("adapter_low", s);
    // long contractions over more warps, to have more loads in flight
    const int rs = low_stride(a[0].r);
    const auto go = [&](auto kern, int ranks, int tokens) {
        const dim3 grid((unsigned)((n + tokens - 1) / tokens), (rs + ranks - 1) / ranks, count);
        return after_pack[0] ? launch_dependent(1, kern, grid, 256, 0, s, both) : launch_cl(1, kern, grid, 256, 0, s, both);
    };
    // four tokens a warp once that leaves eight CTAs for every SM (48 tokens with
    // adapters of their own over 8960: 8 us one by one, 16 us by fours)
    const bool longk = kmax * sizeof(T) > 4096;
    if (n * rs / (longk ? 8 : 32) >= 8 * sm_count()) {
        if (longk) return vec ? go(k_low_token<T, true, 4, 4>, 2, 4) : go(k_low_token<T, false, 4, 4>, 2, 4);
        return vec ? go(k_low_token<T, true, 1, 4>, 8, 4) : go(k_low_token<T, false, 1, 4>, 8, 4);
    }
    if (longk) return vec ? go(k_low_token<T, true, 4, 1>, 2, 1) : go(k_low_token<T, false, 4, 1>, 2, 1);
    return vec ? go(k_low_token<T, true, 1, 1>, 8, 1) : go(k_low_token<T, false, 1, 1>, 8, 1);
}

template <class T, int NB>
cudaError_t small_launch(const ProjectArgs& a, cudaStream_t s) {
    // as many CTAs share a contraction as it takes to give every SM one,
    // while each of their warps has four blocks
    const int tiles = (a.o + 15) / 16;
    int S = 1;
    while (S < 8 && a.w && tiles * S < sm_count() && a.k >= S * 2048) S *= 2;
    const size_t smem = (size_t)8 * 16 * (NB * 8 + 1) * 4;
    KScope ks("adapter_project", s);
    const cudaError_t e = ensure_smem(k_project_small<T, NB>, smem);
    return e != cudaSuccess ? e : launch_dependent(S, k_project_small<T, NB>, dim3((unsigned)(tiles * S)), 256, smem, s, a);
}

template <class T>
cudaError_t small_width(const ProjectArgs& a, cudaStream_t s) { return a.n <= 8 ? small_launch<T, 1>(a, s) : small_launch<T, 2>(a, s); }

template <class T, int RB>
cudaError_t grad_launch(const GradPair& a, long long n, bool dependent, float* partial, cudaStream_t s) {
    using L = GradTile<T, RB>;
    const int t0 = (a.g[0].k + 127) / 128, t1 = (a.g[1].k + 127) / 128, passes = (a.r + RB * 8 - 1) / (RB * 8);
    const int window = grad_window(n, a.g[0].k, a.g[1].k, a.r, a.adapters);
    cudaError_t e = ensure_smem(k_grad<T, RB>, L::kSmem + 1024);  // own[] is beside the tiles
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)(t0 + t1), passes, (unsigned)((n + window - 1) / window));
    // larger parts of a tile per CTA as long as eight CTAs for every SM are left
    constexpr int kChunks = RB * 8 * 128 / 1024;
    int chunks = 1;
    while (chunks < kChunks && (long long)(t0 + t1) * passes * a.adapters * kChunks / (2 * chunks) >= 8 * sm_count()) chunks *= 2;
    const dim3 sums((unsigned)(t0 + t1), passes * (kChunks / chunks), a.adapters);
    KScope ks("adapter_grad", s, 2);
    e = dependent ? launch_dependent(1, k_grad<T, RB>, grid, 256, L::kSmem, s, a, t0, window, partial, 1)
                  : launch_cl(1, k_grad<T, RB>, grid, 256, L::kSmem, s, a, t0, window, partial, 0);
    return e != cudaSuccess ? e : launch_dependent(1, k_grad_sum<T, RB>, sums, 256, 0, s, a, t0, window, chunks, static_cast<const float*>(partial));
}

template <class T>
cudaError_t grad_width(const GradPair& a, long long n, bool dependent, float* partial, cudaStream_t s) {
    if (a.r <= 16) return grad_launch<T, 2>(a, n, dependent, partial, s);
    if (a.r <= 32) return grad_launch<T, 4>(a, n, dependent, partial, s);
    return grad_launch<T, 8>(a, n, dependent, partial, s);
}

}  // namespace

#define TSG_DTYPE_SWITCH(dtype, ...)                                   \
    switch (dtype) {                                                   \
        case DT_F32: { using T = float; __VA_ARGS__; } break;          \
        case DT_BF16: { using T = __nv_bfloat16; __VA_ARGS__; } break; \
        case DT_F16: { using T = __half; __VA_ARGS__; } break;         \
    }                                                                  \
    return cudaErrorInvalidValue;

cudaError_t launch_pack(const PackJobs& a, cudaStream_t s) {
    long long blocks = 0;
    for (int q = 0; q < a.jobs; q++) blocks += a.job[q].blocks;
    if (blocks > INT_MAX) return cudaErrorInvalidConfiguration;
    KScope ks("adapter_pack", s);
    k_pack<<<(unsigned)blocks, 256, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_low(const LowArgs* a, int count, int dtype, bool vec, const int* after_pack, cudaStream_t s) {
    TSG_DTYPE_SWITCH(dtype, return low_launch<T>(a, count, vec, after_pack, s));
}

cudaError_t launch_project_f32(const ProjectArgs& a, cudaStream_t s) {
    const auto vec = [](const void* p, long long stride, long long rows) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows < 2 || stride % 4 == 0); };
    const int vx = vec(a.x, a.x_stride, a.n), vw = vec(a.w, a.w_stride, a.w_t ? a.k : a.o);
    KScope ks("adapter_project", s);
    if (a.n <= kSmallTokens && !a.w_t)
        return launch_dependent(1, k_project_f32_few, dim3((a.o + 7) / 8, (unsigned)((a.n + 3) / 4)), 256, 0, s, a, vx && vw);
    // a factor's rows: r rows of o elements, or o rows of r
    const int vg = vec(a.g.p, a.g.sk == 1 && a.g.sj != 1 ? a.g.sj : a.g.sk, 2) && (a.id.count == 1 || a.g.se % 4 == 0);
    // The tile and the number of CTAs that share a contraction with the least
    // time on the SM with the most CTAs: a 64 x 64 tile takes 0.35 of a
    // 128 x 128 one, whose operands' way from shared memory costs half, and
    // clusters of four and more leave some SMs of each group out.
    int tile = 64, S = 1;
    double least = 1e300;
    for (int size = 64; size <= 128; size *= 2) {
        const long long tiles = (a.n + size - 1) / size * ((a.o + size - 1) / size);
        for (int c = 1; c <= 8 && (c == 1 || (a.w && a.k >= 64 * c)); c *= 2) {
            const int sms = c < 4 ? sm_count() : sm_count() * 128 / 148;
            const double cost = ((double)((tiles * c + sms - 1) / sms) / c + 0.005 * c) * (size == 64 ? 0.35 : 1);
            if (cost < least) tile = size, S = c, least = cost;
        }
    }
    const auto go = [&](auto kern, size_t smem) {
        const cudaError_t e = ensure_smem(kern, smem);
        return e != cudaSuccess ? e : launch_cl(S, kern, dim3((unsigned)((a.n + tile - 1) / tile * S), (a.o + tile - 1) / tile), 256, smem, s, a, vx, vw, vg);
    };
    return tile == 64 ? go(k_project_f32<64, 64, 4, 4, 4>, F32Tile<64, 64>::kSmem) : go(k_project_f32<128, 128, 8, 8, 1>, F32Tile<128, 128>::kSmem);
}

cudaError_t launch_project_small(const ProjectArgs& a, int dtype, cudaStream_t s) {
    return dtype == DT_BF16 ? small_width<__nv_bfloat16>(a, s) : small_width<__half>(a, s);
}

cudaError_t launch_grads(const GradPair& a, long long n, int dtype, bool dependent, float* partial, cudaStream_t s) {
    TSG_DTYPE_SWITCH(dtype, return grad_width<T>(a, n, dependent, partial, s));
}

}  // namespace tsg
