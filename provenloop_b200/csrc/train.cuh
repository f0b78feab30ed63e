// train.cuh -- internal interface between the C entry points of the training
// operators (train_ops.cu) and their kernels (k_loss.cu, k_clip.cu).  Not part
// of the public ABI.
#pragma once
#include "lowrank.cuh"

namespace tsg {

// Rows of logits, what of each counts, and where they lie.
struct LossRows {
    const void* logits;
    long long stride;
    long long n;
    uint32_t vocab;
    int targets64;
    const void* targets;
    uint32_t sequences;
    const int32_t* starts;  // or null: `per` rows each
    long long per;
#ifdef __CUDACC__
    // The row's target, or -1: it does not count.
    __device__ __forceinline__ int target(long long row) const {
        const long long y = targets64 ? static_cast<const long long*>(targets)[row] : (long long)static_cast<const int32_t*>(targets)[row];
        return (unsigned long long)y < vocab ? (int)y : -1;
    }
    // The row's sequence, or -1: it is in none (with `starts` alone).
    __device__ __forceinline__ int sequence(long long row) const {
        if (!starts) return (int)((uint32_t)row / (uint32_t)per);  // fewer than 2^32 rows
        if (row < starts[0] || row >= starts[sequences]) return -1;
        uint32_t lo = 0, hi = sequences;  // starts[lo] <= row < starts[hi]
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (row < starts[mid]) hi = mid;
            else lo = mid;
        }
        return (int)lo;
    }
#endif
};

// max of a row and the sum of exp(z - max).
struct RowStats {
    float max, sum;
};

struct PolicyTerms {
    const float *old, *ref, *advantages;
    int advantage_rows, kind;
    float low, high, kl;  // 1 - clip_low, 1 + clip_high
};

struct PreferTerms {
    const float* ref;
    int kind, average;
    float beta, smoothing;
};

// A loss is the sum of its parts by groups of so many, and of the groups.
constexpr uint32_t kLossGroup = 1024;
__host__ __device__ constexpr uint64_t loss_groups(uint64_t parts) { return (parts + kLossGroup - 1) / kLossGroup; }
// Sums for `parts`: those, and the groups' of each level above.
constexpr uint64_t loss_sums(uint64_t parts) { return parts + (parts > kLossGroup ? loss_sums(loss_groups(parts)) : 0); }
constexpr uint64_t loss_tickets(uint64_t parts) { return loss_groups(parts) + (parts > kLossGroup ? loss_tickets(loss_groups(parts)) : 0); }

// What a loss's launches hand to one another, in the workspace.
struct LossWork {
    int* order;        // [n + 1], or null: loss_orders
    int* counts;       // [sequences + 1]: rows that count, and all of them (policy)
    RowStats* stats;   // [n] (preference)
    double* logs;      // [n]: log-probabilities (preference)
    float* slope;      // [sequences]: d loss / d log-probability (preference)
    double* parts;     // loss_sums(n) (policy; by cluster or by row) or (pairs) (preference)
    unsigned* ticket;  // [tickets]: parts of each group that are there
    uint32_t tickets;  // loss_tickets(n) or (pairs), 0 where there is no loss
};

struct LossOut {
    float *loss, *margins, *logprobs;
    void* grad;
    long long grad_stride;
    const float* grad_scale;
};

// Whether k_order puts the rows in order first: long ones of persistent clusters, if they are more
// than the CTAs do by themselves.
// both: a call that goes over them once without a gradient too.
bool loss_orders(uint64_t n, uint32_t vocab, int dtype, bool grad, bool both);
cudaError_t launch_logprobs(const LossRows& r, const LossWork& w, float* logprobs, int dtype, cudaStream_t s);
cudaError_t launch_logprobs_backward(const LossRows& r, const float* g, const LossWork& w, const LossOut& o, int dtype, cudaStream_t s);
cudaError_t launch_policy(const LossRows& r, const PolicyTerms& p, const LossWork& w, const LossOut& o, int dtype, cudaStream_t s);
cudaError_t launch_preference(const LossRows& r, const PreferTerms& p, const LossWork& w, const LossOut& o, int dtype, cudaStream_t s);

// waits of k_loss.cu that ran out on the current device so far
cudaError_t expired_waits_loss(unsigned long long* out);

// One group's part of one tensor.
struct ClipTensor {
    const void* grad;
    void* out;
    uint64_t part;  // elements of a group
    int dtype, out_dtype;
};
struct ClipArgs {
    const ClipTensor* tensors;  // host memory
    uint64_t count;
    uint32_t groups;
    const float* max_norms;
    float max_norm;
    int one_max;
    float* norms;
    double* partial;  // clip_partials(...) of them
};
uint64_t clip_partials(const ClipTensor* t, uint64_t count, uint32_t groups);
cudaError_t launch_clip(const ClipArgs& a, cudaStream_t s);

}  // namespace tsg
