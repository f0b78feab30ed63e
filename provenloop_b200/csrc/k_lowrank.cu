// k_lowrank.cu -- kernels of the low-rank adapters beside a shared
// projection, and of their gradients.
//
// For token m with adapter e (or none):
//   low[m]  = s_e x[m] A_e^T                              (r values, f32)
//   y[m]    = base[m] + x[m] W^T + bias + low[m] B_e^T
// and, for the gradient dy of y with W frozen,
//   u[m]    = s_e dy[m] B_e
//   dx[m]   = dy[m] W + u[m] A_e
//   dA_e    = sum over e's tokens of u[m]^T x[m]
//   dB_e    = sum over e's tokens of dy[m]^T low[m]
// The three kernels below are these lines; a factor's strides turn the
// forward form into the backward one.  Sums are held in f32 and each result
// is rounded to its type once.
#include "launch.cuh"
#include "lowrank.cuh"

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

// One CTA per token, one warp per rank index in turn.
template <class T>
__global__ void __launch_bounds__(256) k_low(const LowArgs a) {
    const long long m = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int e = a.id.of(m);
    float* low = a.low + m * a.r;
    if (e < 0) {
        for (int j = threadIdx.x; j < a.r; j += blockDim.x) low[j] = 0.f;
        return;
    }
    const T* x = static_cast<const T*>(a.x) + m * a.x_stride;
    const T* f = static_cast<const T*>(a.f.p) + e * a.f.se;
    const float s = a.scale ? a.scale[e] : 1.f;
    for (int j = warp; j < a.r; j += 8) {
        float v = 0.f;
        for (int k = lane; k < a.k; k += 32) v = fmaf(to_f(x[k]), to_f(f[j * a.f.sj + k * a.f.sk]), v);
#pragma unroll
        for (int q = 16; q; q >>= 1) v += __shfl_xor_sync(0xffffffffu, v, q);
        if (lane == 0) low[j] = s * v;
    }
}

// 64 x 64 outputs per CTA, 4 x 4 per thread, 16 of the contraction at a time.
template <class T>
__global__ void __launch_bounds__(256) k_project(const ProjectArgs a) {
    constexpr int BM = 64, BN = 64, BK = 16;
    __shared__ float xs[BK][BM + 1], ws[BK][BN + 1];
    const long long m0 = (long long)blockIdx.x * BM;
    const int o0 = blockIdx.y * BN;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    if (a.w) {
        const T* x = static_cast<const T*>(a.x);
        const T* w = static_cast<const T*>(a.w);
        for (int k0 = 0; k0 < a.k; k0 += BK) {
            for (int i = threadIdx.x; i < BM * BK; i += 256) {
                const int k = i % BK, m = i / BK;
                xs[k][m] = m0 + m < a.n && k0 + k < a.k ? to_f(x[(m0 + m) * a.x_stride + k0 + k]) : 0.f;
            }
            for (int i = threadIdx.x; i < BN * BK; i += 256) {
                // consecutive threads along whichever axis of W is contiguous
                const int k = a.w_sk == 1 ? i % BK : i / BN, o = a.w_sk == 1 ? i / BK : i % BN;
                ws[k][o] = o0 + o < a.o && k0 + k < a.k ? to_f(w[(o0 + o) * a.w_so + (k0 + k) * a.w_sk]) : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < BK; k++) {
                float xv[4], wv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) xv[i] = xs[k][ty + 16 * i], wv[i] = ws[k][tx + 16 * i];
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i][j] = fmaf(xv[i], wv[j], acc[i][j]);
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const long long m = m0 + ty + 16 * i;
        if (m >= a.n) continue;
        const int e = a.id.of(m);
        const float* low = a.low + m * a.r;
        const T* g = static_cast<const T*>(a.g.p) + (e < 0 ? 0 : e) * a.g.se;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int o = o0 + tx + 16 * j;
            if (o >= a.o) continue;
            float v = acc[i][j];
            if (a.bias) v += to_f(static_cast<const T*>(a.bias)[o]);
            if (e >= 0)
                for (int q = 0; q < a.r; q++) v = fmaf(low[q], to_f(g[q * a.g.sj + o * a.g.sk]), v);
            if (a.base) v += to_f(static_cast<const T*>(a.base)[m * a.base_stride + o]);
            static_cast<T*>(a.out)[m * a.out_stride + o] = from_f<T>(v);
        }
    }
}

// One thread per element of the gradient, all tokens in order.
template <class T>
__global__ void __launch_bounds__(256) k_grad(const GradArgs a) {
    const int k = blockIdx.x * 256 + threadIdx.x;
    const int j = blockIdx.y, e = blockIdx.z;
    if (k >= a.k) return;
    const T* x = static_cast<const T*>(a.x);
    float v = 0.f;
    for (long long m = 0; m < a.n; m++)
        if (a.id.of(m) == e) v = fmaf(a.low[m * a.r + j], to_f(x[m * a.x_stride + k]), v);
    static_cast<T*>(a.out)[e * a.se + j * a.sj + k * a.sk] = from_f<T>(v);
}

}  // namespace

#define TSG_DTYPE_SWITCH(dtype, ...)                                   \
    switch (dtype) {                                                   \
        case DT_F32: { using T = float; __VA_ARGS__; } break;          \
        case DT_BF16: { using T = __nv_bfloat16; __VA_ARGS__; } break; \
        case DT_F16: { using T = __half; __VA_ARGS__; } break;         \
        default: return cudaErrorInvalidValue;                         \
    }

cudaError_t launch_low(const LowArgs& a, int dtype, cudaStream_t s) {
    KScope ks("adapter_low", s);
    TSG_DTYPE_SWITCH(dtype, k_low<T><<<(unsigned)a.n, 256, 0, s>>>(a));
    return cudaGetLastError();
}

cudaError_t launch_project(const ProjectArgs& a, int dtype, cudaStream_t s) {
    KScope ks("adapter_project", s);
    const dim3 grid((unsigned)((a.n + 63) / 64), (a.o + 63) / 64);
    TSG_DTYPE_SWITCH(dtype, k_project<T><<<grid, 256, 0, s>>>(a));
    return cudaGetLastError();
}

cudaError_t launch_grad(const GradArgs& a, int dtype, cudaStream_t s) {
    KScope ks("adapter_grad", s);
    const dim3 grid((a.k + 255) / 256, a.r, a.id.count);
    TSG_DTYPE_SWITCH(dtype, k_grad<T><<<grid, 256, 0, s>>>(a));
    return cudaGetLastError();
}

}  // namespace tsg
