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

// Rows of low are padded to a multiple of 16, zero behind r.
#ifdef __CUDACC__
__host__ __device__
#endif
inline int low_stride(int r) { return (r + 15) & ~15; }

// low[m][j] = scale_e * sum_k x[m][k] F[e][j][k] (f32 [n][low_stride(r)];
// zero rows where a token has no adapter).  What multiplies them by FMA takes
// them as they are; matrix instructions take them rounded to TF32 (k_project_tc:
// 11 significant bits, the range of f32; nothing else may read them then), as two such terms (gradients of f32
// and fp16 inputs) or as two bf16 terms (of bf16 inputs).
struct LowArgs {
    const void* x;
    long long x_stride;
    long long n;
    int k, r;
    Factor f;
    AdapterIds id;
    const float* scale;
    float* low;      // or null
    uint16_t* split; // or null; bf16 inputs: the same values as bf16_terms, [n][2][low_stride(r)]
    int tf32;        // low is rounded to TF32 when it is written (here that hides; in k_project_tc it costs 1 % of a prefill)
};

struct LowPair {
    LowArgs a[2];
    int after_pack[2];  // launch_low
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
    int low_tf32;  // as LowArgs' tf32
    Factor g;  // sk here is the stride of o
    const float* g32;     // g as f32 [e][o][low_stride(r)], elements that are not finite replaced by 1 of their sign (k_project.cu only)
    const uint32_t* bad;  // [e][ceil(o / 128)][low_stride(r) / 16]: some of them are
    AdapterIds id;
    void* out;
    long long out_stride;
    // x or w lies in the workspace, written by launch_pack.  launch_low, which
    // stands between the two, lets the projection start before the packing is
    // over (it only waits for it before it ends), so what loads x and w has to
    // wait for launch_low first; other operands' loads start at once.
    int packed;
};

// Gradient of one factor: out[e][j][k] = sum over the tokens m of adapter e
// of low[m][j] x[m][k], written at out + e * se + j * sj + k * sk.
struct GradArgs {
    const void* x;
    long long x_stride;
    int k;
    const void* low;  // LowArgs' split for bf16 x, else its low: rows of 4 low_stride(r) bytes
    void* out;
    long long se, sj, sk;
};
struct GradPair {
    GradArgs g[2];
    int r, adapters;
    const int* first;  // [adapters + 1]: adapter e's tokens, in order, are list[first[e] .. first[e + 1])
    const int* list;
};

// What a call lays out in its workspace first, in one launch: copies of
// operands whose rows are not on 16-byte boundaries (or factors transposed),
// factors as f32, the tokens of each adapter.
struct PackJob {
    enum Kind : int { COPY, TO_F32, LISTS } kind;
    const void* src;  // COPY, TO_F32: element (e, j, k) at e * se + j * sj + k * sk
    long long se, sj, sk;
    long long rows;  // j
    int count, cols, dst_cols;
    void* dst;      // [count][rows][dst_cols], zeros behind cols: 16-bit elements / f32
    uint32_t* bad;  // TO_F32: [count][ceil(rows / 128)][dst_cols / 16]
    AdapterIds id;  // LISTS: dst is first [count + 1], then the list [rows]
    long long blocks;
};
constexpr int kMaxPack = 7;
struct PackJobs {
    PackJob job[kMaxPack];
    int jobs, dtype;
    void add(PackJob j) {
        j.blocks = j.kind == PackJob::LISTS ? j.count : j.kind == PackJob::TO_F32 ? (j.rows + 127) / 128 * (j.dst_cols / 16) * j.count : ((j.rows + 31) / 32) * ((j.dst_cols + 127) / 128) * j.count;
        job[jobs++] = j;
    }
};

// The kernels that a call takes go by its sizes; decode_ops.cu lays out the
// workspace with the same rules.
// Low token by token reads each token's factor (from L2 where tokens share
// it): for f32 always, else up to 48 MiB of such reads, and up to 256 MiB where
// a tile of the matrix form may have to go past x more than four times for its
// tokens' adapters (739 tokens of 47 adapters of rank 64 over 1536: 26 us token
// by token, 157 us as a matrix; 3453 tokens in 23 requests of rank 16: 31 and 10).
inline bool low_by_token(long long n, long long k0, long long k1, long long r, long long adapters) {
    const long long bytes = n * r * (k0 > k1 ? k0 : k1) * 2, tile = n < 128 ? n : 128;
    const long long units = (adapters < tile ? adapters : tile) * (low_stride((int)r) / 16);
    return bytes <= (units > 32 ? 256ll : 48ll) << 20;
}
constexpr int kSms = 148;  // the workspace's rules and the gradients' order of sums go by a B200's, whatever device is current
constexpr int kSmallTokens = 16;  // up to here W is streamed once past all tokens
// The projection takes each token's factor from where it is, n o r elements
// in all, up to 32 MiB of them; above that the factors are converted first
// and shared by the tokens of a tile.  Tiles too few for half of the SMs with
// a long contraction (k, 0 without a shared projection) take it all the same,
// since only that way shares a contraction (217 tokens, 8960 -> 1536, rank 64:
// 80 us for the backward call, 85 with converted factors).
inline bool factor_by_token(long long n, long long o, long long r, long long k) {
    return n * o * r * 2 <= 32ll << 20 || (k >= 4096 && ((n + 127) / 128) * ((o + 63) / 64) < kSms / 2);
}

// Places of the tokens' list that a CTA of the gradients takes: three CTAs for
// each SM over the tiles of 128 features and up to 64 rank indexes, and at least
// 128 places each, or down to 8 while they hold two adapters or more (each
// costs a CTA 3 to 10 us however few its tokens: 72 tokens of 42 adapters of
// rank 64 over 1536 + 1536 take 57 us so and 147 us in windows of 32).
inline int grad_ranks(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : (r + 63) / 64 * 64; }  // padded
inline long long grad_tiles(long long k0, long long k1) { return (k0 + 127) / 128 + (k1 + 127) / 128; }
inline int grad_window(long long n, long long k0, long long k1, int r, int adapters) {
    const long long ctas = grad_tiles(k0, k1) * (r <= 64 ? 1 : (r + 63) / 64);
    long long windows = (3 * kSms + ctas - 1) / ctas;
    long long most = (n + 7) / 8 < adapters / 2 ? (n + 7) / 8 : adapters / 2;
    if (most < (n + 127) / 128) most = (n + 127) / 128;
    if (windows > most) windows = most;
    if (windows * 32 > n) return (int)((n + windows * 8 - 1) / (windows * 8) * 8);
    return (int)((n + windows * 32 - 1) / (windows * 32) * 32);
}
inline uint64_t grad_partial_bytes(long long n, long long k0, long long k1, int r, int adapters) {
    const int w = grad_window(n, k0, k1, r, adapters);
    return (uint64_t)((n + w - 1) / w) * 2 * grad_tiles(k0, k1) * 128 * grad_ranks(r) * 4;
}

cudaError_t launch_pack(const PackJobs& a, cudaStream_t s);
// one or two of them (the same n, r and id) in one launch; `vec`: rows of x
// and f start on 16-byte boundaries and f.sk is 1; `after_pack`, for each:
// launch_pack was queued directly before, and its results are used here (2)
// or by the next launch only (1), else 0
cudaError_t launch_low(const LowArgs* a, int count, int dtype, bool vec, const int* after_pack, cudaStream_t s);
// 16-bit types, x and f on 16-byte boundaries, many tokens (k_project.cu)
cudaError_t launch_low_tc(const LowArgs* a, int count, int dtype, const int* after_pack, cudaStream_t s);
// f32, any strides
cudaError_t launch_project_f32(const ProjectArgs& a, cudaStream_t s);
// 16-bit types, at most kSmallTokens tokens; x and w (not transposed) on 16-byte boundaries
cudaError_t launch_project_small(const ProjectArgs& a, int dtype, cudaStream_t s);
// 16-bit types; x and w rows on 16-byte boundaries (k_project.cu); a.g32 is
// null where factor_by_token
cudaError_t launch_project_tc(const ProjectArgs& a, int dtype, cudaStream_t s);
// rows of x on 16-byte boundaries; `dependent`: launch_project_tc was queued
// directly before, and behind it what is read here; partial: grad_partial_bytes
cudaError_t launch_grads(const GradPair& a, long long n, int dtype, bool dependent, float* partial, cudaStream_t s);
// waits of k_project.cu / k_rules.cu that ran out on the current device so far
cudaError_t expired_waits_project(unsigned long long* out);
cudaError_t expired_waits_rules(unsigned long long* out);

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
