// lowrank.cuh -- internal interface between the C entry points of the
// plaintext decode-step operators (decode_ops.cu) and their kernels
// (k_lowrank.cu, k_rules.cu).  Not part of the public ABI.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace tsg {

enum Dtype : int { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

inline size_t dtype_size(int t) { return t == DT_F32 ? 4 : 2; }

// Adapter of each token: ids[m / per], none where it is outside [0, count).
struct AdapterIds {
    const int32_t* ids;
    long long per;
    int count;
#ifdef __CUDACC__
    __device__ __forceinline__ int of(long long m) const {
        const int e = ids[per == 1 ? m : m / per];
        return (unsigned)e < (unsigned)count ? e : -1;
    }
#endif
};

// A stack of low-rank factors seen as F[e][j][k]: element (j, k) of adapter
// e at p + e * se + j * sj + k * sk.  A ([E][r][d_in]) has (sj, sk) =
// (d_in, 1); B ([E][d_out][r]), contracted over d_out, has (1, r).
struct Factor {
    const void* p;
    long long se, sj, sk;
};

// low[m][j] = scale_e * sum_k x[m][k] F[e][j][k] (f32 [n][r]; zero rows where
// a token has no adapter).
struct LowArgs {
    const void* x;
    long long x_stride;
    long long n;
    int k, r;
    Factor f;
    AdapterIds id;
    const float* scale;
    float* low;
};

// out[m][o] = base[m][o] + sum_k x[m][k] W(o, k) + bias[o]
//           + sum_j low[m][j] G[e][j][o];  W(o, k) at w + o * w_so + k * w_sk,
// each term but the last optional.
struct ProjectArgs {
    const void* x;
    long long x_stride;
    long long n;
    int k, o, r;
    const void* w;
    long long w_so, w_sk;
    const void* bias;
    const void* base;
    long long base_stride;
    const float* low;
    Factor g;  // sk here is the stride of o
    AdapterIds id;
    void* out;
    long long out_stride;
};

// Gradient of one factor: out[e][j][k] = sum over the tokens m of adapter e
// of low[m][j] x[m][k], written at out + e * se + j * sj + k * sk.
struct GradArgs {
    const void* x;
    long long x_stride;
    long long n;
    int k, r;
    const float* low;
    AdapterIds id;
    void* out;
    long long se, sj, sk;
};

cudaError_t launch_low(const LowArgs& a, int dtype, cudaStream_t s);
cudaError_t launch_project(const ProjectArgs& a, int dtype, cudaStream_t s);
cudaError_t launch_grad(const GradArgs& a, int dtype, cudaStream_t s);

struct RulesArgs {
    const void* logits;
    long long logits_stride;
    long long n;
    uint32_t vocab;
    const void* tokens;  // int32 or int64 [n][token_cols]
    long long tokens_stride;
    uint32_t token_cols;
    int tokens64;
    const int32_t *lengths, *prompt_lengths;
    const float *repetition, *frequency, *presence;
    const void* bias_ids;  // int32 or int64 [n][bias_cols]
    const float* bias_values;
    long long bias_ids_stride, bias_values_stride;
    uint32_t bias_cols;
    int bias64;
    const uint32_t* mask;
    long long mask_stride;
    void* out;
    long long out_stride;
    long long* pick;
};

cudaError_t launch_rules(const RulesArgs& a, int dtype, int out_dtype, cudaStream_t s);

}  // namespace tsg
