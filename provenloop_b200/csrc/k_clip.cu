// k_clip.cu -- norms over many tensors, for each group of a stack, and the
// clipping of the tensors by them.
//
// Group e has the e-th part of every tensor:
//   norm_e = sqrt(sum over its elements of g^2)
//   out = g min(1, max_e / norm_e), rounded once
// A group whose norm is not finite is left as it is.
//
// The bound is the tensors' traffic.  Parts go in chunks; each chunk's sum of
// squares is a 64-bit value of its own, and a group's are added in an order
// that depends on the sizes alone.
#include "launch.cuh"
#include "sm100.cuh"
#include "train.cuh"

namespace tsg {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kChunk = 16384;  // elements of a part that a CTA takes
constexpr int kTable = 128;         // tensors in a launch's arguments

struct ClipEntry {
    const void* grad;
    void* out;
    uint64_t part;
    uint32_t chunk0;  // chunks of a group in the entries before
    int16_t dtype, out_dtype;
};
struct ClipTable {
    ClipEntry t[kTable];
    int count;
    uint32_t chunks;      // of a group in this launch
    uint32_t group_chunks, at;  // of a group in all launches, and in those before
    double* partial;      // [groups][group_chunks]
    const float* factor;  // [groups]
};

__device__ __forceinline__ const ClipEntry& entry_of(const ClipTable& a, uint32_t chunk) {
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (chunk < a.t[mid].chunk0) hi = mid;
        else lo = mid;
    }
    return a.t[lo];
}

template <class T>
__device__ __forceinline__ float value(T v) { return (float)v; }

template <int N>
__device__ double block_total(double v) {
    __shared__ double warp_sum[N / 32];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int i = 0; i < N / 32; i++) v += warp_sum[i];
    return v;
}

// Sum of the squares of n elements.  Those of a vector are added in 32 bits,
// and once more in 64 where that may overflow or lose what is small.
template <class T>
__device__ double squares(const T* x, uint32_t n) {
    constexpr uint32_t N = 16 / sizeof(T);
    const uint32_t head = (uint32_t)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)), end = head + n;
    double total = 0.0;
    for (uint32_t p = threadIdx.x * N; p < end; p += kThreads * N) {
        if (p >= head && p + N <= end) {
            const uint4 z = *reinterpret_cast<const uint4*>(x + p - head);
            const T* e = reinterpret_cast<const T*>(&z);
            float s = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < N; i++) s = fmaf(value(e[i]), value(e[i]), s);
            if (s > 1e-30f && s < 1e37f) {
                total += s;
            } else {
                for (uint32_t i = 0; i < N; i++) total += (double)value(e[i]) * value(e[i]);
            }
        } else {
            for (uint32_t i = 0; i < N; i++)
                if (p + i >= head && p + i < end) total += (double)value(x[p + i - head]) * value(x[p + i - head]);
        }
    }
    return total;
}

template <class T, class O>
__device__ void scaled(const T* x, O* out, uint32_t n, float by) {
    constexpr uint32_t N = 16 / sizeof(T);
    const uint32_t head = (uint32_t)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)), end = head + n;
    const bool whole = (reinterpret_cast<uintptr_t>(out) - head * sizeof(O)) % 16 == 0;
    for (uint32_t p = threadIdx.x * N; p < end; p += kThreads * N) {
        if (whole && p >= head && p + N <= end) {
            const uint4 z = *reinterpret_cast<const uint4*>(x + p - head);
            const T* e = reinterpret_cast<const T*>(&z);
            uint4 r[sizeof(O) / sizeof(T)];
            O* o = reinterpret_cast<O*>(r);
#pragma unroll
            for (uint32_t i = 0; i < N; i++) o[i] = (O)(value(e[i]) * by);
#pragma unroll
            for (uint32_t i = 0; i < sizeof(O) / sizeof(T); i++) reinterpret_cast<uint4*>(out + p - head)[i] = r[i];
        } else {
            for (uint32_t i = 0; i < N; i++)
                if (p + i >= head && p + i < end) out[p + i - head] = (O)(value(x[p + i - head]) * by);
        }
    }
}

__global__ void __launch_bounds__(kThreads) k_squares(const __grid_constant__ ClipTable a) {
    const uint32_t group = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const ClipEntry& t = entry_of(a, chunk);
    const uint64_t at = (uint64_t)(chunk - t.chunk0) * kChunk, from = group * t.part + at;
    const uint32_t n = (uint32_t)min((unsigned long long)kChunk, (unsigned long long)(t.part - at));
    double v;
    if (t.dtype == DT_F32) v = squares(static_cast<const float*>(t.grad) + from, n);
    else if (t.dtype == DT_BF16) v = squares(static_cast<const __nv_bfloat16*>(t.grad) + from, n);
    else v = squares(static_cast<const __half*>(t.grad) + from, n);
    v = block_total<kThreads>(v);
    if (threadIdx.x == 0) a.partial[(uint64_t)group * a.group_chunks + a.at + chunk] = v;
}

// A group's norm and factor.  One CTA for each group.
__global__ void __launch_bounds__(1024) k_norms(const double* partial, uint32_t chunks, const float* max_norms, float max_norm, int one_max,
                                                float* norms, float* factor) {
    grid_dependency_wait();
    const double* p = partial + (uint64_t)blockIdx.x * chunks;
    double v = 0.0;
    for (uint32_t i = threadIdx.x; i < chunks; i += 1024) v += p[i];
    v = block_total<1024>(v);
    if (threadIdx.x) return;
    const double root = sqrt(v), most = max_norms ? max_norms[one_max ? 0 : blockIdx.x] : max_norm;
    const float norm = (float)root;
    norms[blockIdx.x] = norm;
    factor[blockIdx.x] = isfinite(norm) && root > most ? (float)(fmax(most, 0.0) / root) : 1.f;
}

__global__ void __launch_bounds__(kThreads) k_scale(const __grid_constant__ ClipTable a) {
    grid_dependency_wait();
    const uint32_t group = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const ClipEntry& t = entry_of(a, chunk);
    const float by = a.factor[group];
    if (by == 1.f && t.grad == t.out) return;
    const uint64_t at = (uint64_t)(chunk - t.chunk0) * kChunk, from = group * t.part + at;
    const uint32_t n = (uint32_t)min((unsigned long long)kChunk, (unsigned long long)(t.part - at));
    if (t.dtype == DT_F32) scaled(static_cast<const float*>(t.grad) + from, static_cast<float*>(t.out) + from, n, by);
    else if (t.dtype == DT_BF16 && t.out_dtype == DT_BF16)
        scaled(static_cast<const __nv_bfloat16*>(t.grad) + from, static_cast<__nv_bfloat16*>(t.out) + from, n, by);
    else if (t.dtype == DT_BF16) scaled(static_cast<const __nv_bfloat16*>(t.grad) + from, static_cast<float*>(t.out) + from, n, by);
    else if (t.out_dtype == DT_F16) scaled(static_cast<const __half*>(t.grad) + from, static_cast<__half*>(t.out) + from, n, by);
    else scaled(static_cast<const __half*>(t.grad) + from, static_cast<float*>(t.out) + from, n, by);
}

uint64_t chunks_of(const ClipTensor* t, uint64_t count) {
    uint64_t c = 0;
    for (uint64_t i = 0; i < count; i++) c += (t[i].part + kChunk - 1) / kChunk;
    return c;
}

}  // namespace

uint64_t clip_partials(const ClipTensor* t, uint64_t count, uint32_t groups) { return chunks_of(t, count) * groups + (groups + 1) / 2; }

cudaError_t launch_clip(const ClipArgs& a, cudaStream_t s) {
    const uint64_t chunks = chunks_of(a.tensors, a.count);
    float* factor = reinterpret_cast<float*>(a.partial + chunks * a.groups);
    cudaError_t e = cudaSuccess;
    KScope ks("clip_gradients", s, 1);
    for (int pass = 0; pass < 2; pass++) {
        uint64_t at = 0;
        for (uint64_t i = 0; i < a.count && e == cudaSuccess;) {
            ClipTable t{};
            t.group_chunks = (uint32_t)chunks, t.at = (uint32_t)at, t.partial = a.partial, t.factor = factor;
            for (; i < a.count && t.count < kTable; i++) {
                const ClipTensor& c = a.tensors[i];
                if (!c.part) continue;
                t.t[t.count++] = {c.grad, c.out, c.part, t.chunks, (int16_t)c.dtype, (int16_t)c.out_dtype};
                t.chunks += (uint32_t)((c.part + kChunk - 1) / kChunk);
            }
            if (!t.count) break;
            at += t.chunks;
            const dim3 grid(t.chunks * a.groups);
            if (pass) {
                e = launch_dependent(1, k_scale, grid, kThreads, 0, s, t);
            } else {
                k_squares<<<grid, kThreads, 0, s>>>(t);
                e = cudaGetLastError();
            }
            ks.kernels++;
        }
        if (pass == 0 && e == cudaSuccess)
            e = launch_dependent(1, k_norms, dim3(a.groups), 1024, 0, s, (const double*)a.partial, (uint32_t)chunks, a.max_norms, a.max_norm,
                                 a.one_max, a.norms, factor);
    }
    return e;
}

}  // namespace tsg
