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

// Rows of low are padded to a multiple of four, zero behind r.
#ifdef __CUDACC__
__host__ __device__
#endif
inline int low_stride(int r) { return (r + 3) & ~3; }

// low[m][j] = scale_e * sum_k x[m][k] F[e][j][k] (f32 [n][low_stride(r)];
// zero rows where a token has no adapter).
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
//           + sum_j low[m][j] G[e][j][o], each term but the last optional.
// W(o, k) is w[o][k], or w[k][o] where w_t is set (the backward call).
struct ProjectArgs {
    const void* x;
    long long x_stride;
    long long n;
    int k, o, r;
    const void* w;
    long long w_stride;
    int w_t;
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
    int k;
    const float* low;
    void* out;
    long long se, sj, sk;
};
struct GradPair {
    GradArgs g[2];
    long long n;
    int r;
    AdapterIds id;
};

// dst[e][j][k] (rows of `dst_cols` 16-bit elements, zeros behind `cols`) =
// src[e * se + j * sj + k * sk].
struct PackArgs {
    const void* src;
    long long se, sj, sk;
    long long rows;
    int count, cols, dst_cols;
    void* dst;
};

// The kernels that a call takes go by its sizes; decode_ops.cu lays out the
// workspace with the same rules.
constexpr int kTokenLow = 128;    // up to here, and for f32, low is computed token by token
constexpr int kSmallTokens = 64;  // up to here W is streamed once past all tokens

cudaError_t launch_pack(const PackArgs& a, cudaStream_t s);
// one or two of them (the same n, r and id) in one launch; `vec`: rows of x
// and f start on 16-byte boundaries and f.sk is 1
cudaError_t launch_low(const LowArgs* a, int count, int dtype, bool vec, cudaStream_t s);
// f32, any strides
cudaError_t launch_project_f32(const ProjectArgs& a, cudaStream_t s);
// 16-bit types, at most kSmallTokens tokens; x and w (not transposed) on 16-byte boundaries
cudaError_t launch_project_small(const ProjectArgs& a, int dtype, cudaStream_t s);
// 16-bit types; x and w rows on 16-byte boundaries (k_project.cu)
cudaError_t launch_project_tc(const ProjectArgs& a, int dtype, cudaStream_t s);
// rows of x on 16-byte boundaries, but for f32 (`vec`: they are)
cudaError_t launch_grads(const GradPair& a, int dtype, bool vec, cudaStream_t s);
// waits of k_project.cu that ran out on the current device so far
cudaError_t expired_waits(unsigned long long* out);

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
