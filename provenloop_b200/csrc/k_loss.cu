// k_loss.cu -- log-probabilities of given tokens, losses on them, and the
// gradients for the logits.
//
// Row t with logits z, target y:
//   m = max_v z_v,  s = sum_v exp(z_v - m),  l = z_y - m - log s
//   d loss / d z_v = g ([v = y] - exp(z_v - m) / s),  g = d loss / d l
// A row whose target lies outside the vocabulary, or which belongs to no
// sequence, does not count: l = 0 and its gradient is zeros; neither it nor a
// row with g = 0 is read for its gradient.
//
// The bound is the logits' traffic: each is read once, and its gradient
// written once.
#include "../../include/tsgpu.h"
#include "launch.cuh"
#include "sm100.cuh"
#include "train.cuh"

namespace cg = cooperative_groups;

namespace tsg {

namespace {

constexpr int kThreads = 512;
constexpr int kCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;

// What k_rows does with a row: its log-probability; the gradient for a given
// g; the policy loss's g; the gradient for known statistics and a g by sequence.
enum RowMode : int { LOGPROBS, GIVEN, POLICY, KNOWN };

struct RowArgs {
    LossRows r;
    PolicyTerms p;
    LossWork w;
    LossOut o;
    const float* g;   // GIVEN: [n]
};

__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// 16 bytes of a row as f32, and back.
template <class T>
struct Lane;
template <>
struct Lane<float> {
    static constexpr uint32_t N = 4, kLow = 0xff800000u;
    static __device__ __forceinline__ void open(const uint4& z, float (&f)[4]) {
        f[0] = __uint_as_float(z.x), f[1] = __uint_as_float(z.y), f[2] = __uint_as_float(z.z), f[3] = __uint_as_float(z.w);
    }
    static __device__ __forceinline__ uint4 close(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    static __device__ __forceinline__ float top(const uint4& z) {
        return fmaxf(fmaxf(__uint_as_float(z.x), __uint_as_float(z.y)), fmaxf(__uint_as_float(z.z), __uint_as_float(z.w)));
    }
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Lane<__nv_bfloat16> {
    static constexpr uint32_t N = 8, kLow = 0xff80ff80u;
    static __device__ __forceinline__ void open(const uint4& z, float (&f)[8]) {
        const uint32_t w[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int i = 0; i < 4; i++) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    static __device__ __forceinline__ uint4 close(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float top(const uint4& z) {
        const uint32_t m = max2(max2(z.x, z.y), max2(z.z, z.w));
        return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
    static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Lane<__half> {
    static constexpr uint32_t N = 8, kLow = 0xfc00fc00u;
    static __device__ __forceinline__ void open(const uint4& z, float (&f)[8]) {
        const uint32_t w[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = v.x, f[2 * i + 1] = v.y;
        }
    }
    static __device__ __forceinline__ uint4 close(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float top(const uint4& z) {
        const uint32_t m = max2(max2(z.x, z.y), max2(z.z, z.w));
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&m));
        return fmaxf(v.x, v.y);
    }
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

// exp(a - b) for a <= b, 1 where they are the same infinity.
__device__ __forceinline__ float weight(float a, float b) { return a == b ? 1.f : exp2_fast((a - b) * kLog2e); }

// Statistics of two parts of a row as one.  A NaN is in the sum.
__device__ __forceinline__ RowStats join(const RowStats& a, const RowStats& b) {
    const float m = fmaxf(a.max, b.max);
    return {m, a.sum * weight(a.max, m) + b.sum * weight(b.max, m)};
}

// l = log-probability of a row's target with logit z, in 64 bits: the row's
// one value that all of its gradient hangs on.
__device__ __forceinline__ double logprob(float z, const RowStats& s) {
    return z == -INFINITY ? (double)-INFINITY : ((double)z - (double)s.max) - log((double)s.sum);
}

// The policy loss's term of a row and its derivative by l, without the row's weight.
__device__ __forceinline__ double policy_term(const PolicyTerms& p, long long row, double l, double a, double* slope) {
    const double rho = p.old ? exp(l - (double)p.old[row]) : l == l ? 1.0 : l, cut = rho < p.low ? (double)p.low : rho > p.high ? (double)p.high : rho;
    const double whole = rho * a, held = cut * a;
    const bool clipped = whole > held;  // not where one is a NaN
    double term = clipped ? -held : -whole, by = clipped ? 0.0 : -whole;
    if (p.ref && p.kl != 0.f) {
        const double d = (double)p.ref[row] - l, e = expm1(d);
        // exp(d) - 1 - d, by its series where that cancels (rest below 2^-50 of it)
        const double k = fabs(d) < 1e-3 ? d * d * (0.5 + d * (1.0 / 6 + d * (1.0 / 24 + d * (1.0 / 120 + d / 720)))) : e - d;
        term += p.kl * k;
        by -= p.kl * e;
    }
    *slope = by;
    return term;
}

// The share of a row of sequence q in the policy loss.
__device__ __forceinline__ double policy_weight(int kind, const int* counts, uint32_t sequences, int q) {
    return kind == TS_REDUCE_TOKEN ? 1.0 / counts[sequences] : kind == TS_REDUCE_SEQUENCE ? 1.0 / ((double)counts[q] * sequences) : 1.0;
}

// A CTA's part [first, last) of a row whose elements are addressed by
// p = v + head, head being the row's offset from a 16-byte boundary.
template <class T>
struct Span {
    const T* x;
    uint32_t head, first, last;
    __device__ __forceinline__ Span(const T* x_, uint32_t vocab, int rank, int cl) : x(x_) {
        head = (uint32_t)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
        const uint32_t end = head + vocab, span = ((end + cl - 1) / cl + 127) / 128 * 128;
        first = min(end, rank * span), last = min(end, first + span);
    }
    // The vector at p < last; -inf for what lies outside.
    __device__ __forceinline__ uint4 load(uint32_t p) const {
        constexpr uint32_t N = Lane<T>::N;
        if (p >= head && p + N <= last) return *reinterpret_cast<const uint4*>(x + p - head);
        uint4 z = make_uint4(Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow);
        T* e = reinterpret_cast<T*>(&z);
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            if (p + i >= head && p + i < last) e[i] = x[p + i - head];
        return z;
    }
    __device__ __forceinline__ void store(T* out, bool whole, uint32_t p, const uint4& z) const {
        constexpr uint32_t N = Lane<T>::N;
        if (whole && p >= head && p + N <= last) {
            *reinterpret_cast<uint4*>(out + p - head) = z;
            return;
        }
        const T* e = reinterpret_cast<const T*>(&z);
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            if (p + i >= head && p + i < last) out[p + i - head] = e[i];
    }
};

template <class T>
__device__ RowStats span_stats(const Span<T>& sp) {
    constexpr uint32_t N = Lane<T>::N, kStep = kThreads * N;
    RowStats t{-INFINITY, 0.f};
    for (uint32_t p = sp.first + threadIdx.x * N; p < sp.last; p += 4 * kStep) {
        uint4 z[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
            z[j] = p + j * kStep < sp.last ? sp.load(p + j * kStep) : make_uint4(Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow);
        const float m = fmaxf(fmaxf(Lane<T>::top(z[0]), Lane<T>::top(z[1])), fmaxf(Lane<T>::top(z[2]), Lane<T>::top(z[3])));
        if (m > t.max) t.sum *= weight(t.max, m), t.max = m;
        const float from = t.max == -INFINITY ? 0.f : t.max;
        float sum[4] = {};
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            float f[N];
            Lane<T>::open(z[j], f);
#pragma unroll
            for (uint32_t i = 0; i < N; i++) sum[j] += exp2_fast((f[i] - from) * kLog2e);
        }
        t.sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    return t;
}

template <class T, int MODE>
__global__ void __launch_bounds__(kThreads, 2) k_rows(const RowArgs a) {
    constexpr uint32_t N = Lane<T>::N, kStep = kThreads * N;
    __shared__ RowStats warp_stats[kThreads / 32], cta_stats[kCluster];
    __shared__ float coef[2];  // g and -g / s
    cg::cluster_group cluster = cg::this_cluster();
    cluster_arrive();
    const int rank = (int)cluster.block_rank(), cl = (int)cluster.num_blocks();
    const long long row = blockIdx.x / cl;
    const T* x = static_cast<const T*>(a.r.logits) + row * a.r.stride;
    const Span<T> sp(x, a.r.vocab, rank, cl);
    T* out = a.o.grad ? static_cast<T*>(a.o.grad) + row * a.o.grad_stride : nullptr;
    const bool out_vec = out && reinterpret_cast<uintptr_t>(out) % 16 == reinterpret_cast<uintptr_t>(x) % 16;

    if (MODE == POLICY) grid_dependency_wait();
    int y = a.r.target(row), q = -1;
    if (MODE == POLICY) {
        q = a.w.sequence[row];
        if (q < 0) y = -1;
    } else if (y >= 0 && (a.r.starts || MODE == KNOWN)) {
        q = a.r.sequence(row);
        if (q < 0) y = -1;
    }
    const float zy = y >= 0 ? Lane<T>::one(x[y]) : 0.f;
    float g = 0.f;
    RowStats s{0.f, 1.f};
    if (MODE == GIVEN && y >= 0) g = a.g[row];
    if (MODE == KNOWN) {
        grid_dependency_wait();
        if (y >= 0) g = a.w.slope[q], s = a.w.stats[row];
    }
    if (MODE != KNOWN && y >= 0 && (MODE != GIVEN || g != 0.f)) {
        s = span_stats<T>(sp);
#pragma unroll
        for (int o = 16; o; o >>= 1) s = join(s, {__shfl_xor_sync(0xffffffffu, s.max, o), __shfl_xor_sync(0xffffffffu, s.sum, o)});
        if ((threadIdx.x & 31) == 0) warp_stats[threadIdx.x >> 5] = s;
        __syncthreads();
        if (threadIdx.x < 32) {
            s = threadIdx.x < kThreads / 32 ? warp_stats[threadIdx.x] : RowStats{-INFINITY, 0.f};
#pragma unroll
            for (int o = kThreads / 64; o; o >>= 1) s = join(s, {__shfl_xor_sync(0xffffffffu, s.max, o), __shfl_xor_sync(0xffffffffu, s.sum, o)});
            s = {__shfl_sync(0xffffffffu, s.max, 0), __shfl_sync(0xffffffffu, s.sum, 0)};  // the same bits for every CTA
        }
        cluster_wait();  // the other CTAs have started
        if (threadIdx.x < cl) *cluster.map_shared_rank(&cta_stats[rank], (int)threadIdx.x) = s;
        cluster.sync();
        s = cta_stats[0];
        for (int i = 1; i < cl; i++) s = join(s, cta_stats[i]);
    } else {
        cluster_wait();
    }
    if (MODE == LOGPROBS || MODE == POLICY) {
        if (threadIdx.x == 0) {
            const double l = y >= 0 ? logprob(zy, s) : 0.0;
            double part = 0.0, slope = 0.0;
            if (MODE == POLICY && y >= 0) {
                const double wt = policy_weight(a.p.kind, a.w.counts, a.r.sequences, q);
                part = wt * policy_term(a.p, row, l, a.p.advantages[a.p.advantage_rows ? row : q], &slope);
                slope *= wt;
            }
            if (rank == 0) {
                if (a.o.logprobs) a.o.logprobs[row] = (float)l;
                if (MODE == LOGPROBS && a.w.stats) a.w.stats[row] = s;
                if (MODE == POLICY) a.w.parts[row] = part;
            }
            if (MODE == POLICY && out) {
                g = (float)(slope * (a.o.grad_scale ? *a.o.grad_scale : 1.f));
                coef[0] = g;
            }
        }
        if (!out) return;
        __syncthreads();
        g = coef[0];
    }
    if (MODE == LOGPROBS) return;
    if (g == 0.f) {  // not for a NaN
        for (uint32_t p = sp.first + threadIdx.x * N; p < sp.last; p += kStep) sp.store(out, out_vec, p, make_uint4(0, 0, 0, 0));
        return;
    }
    const float c = -__fdiv_rn(g, s.sum), from = s.max == -INFINITY ? 0.f : s.max;
    for (uint32_t p = sp.first + threadIdx.x * N; p < sp.last; p += 4 * kStep) {
        uint4 z[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
            if (p + j * kStep < sp.last) z[j] = sp.load(p + j * kStep);
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t at = p + j * kStep;
            if (at >= sp.last) break;
            float f[N];
            Lane<T>::open(z[j], f);
#pragma unroll
            for (uint32_t i = 0; i < N; i++) f[i] = c * exp2_fast((f[i] - from) * kLog2e);
            const uint32_t k = (uint32_t)y + sp.head - at;
            if (k < N) {
#pragma unroll
                for (uint32_t i = 0; i < N; i++) f[i] += i == k ? g : 0.f;
            }
            sp.store(out, out_vec, at, Lane<T>::close(f));
        }
    }
}

// Rows that count: the sequence of each, how many each sequence has, and how
// many there are.  One CTA.
__global__ void __launch_bounds__(1024) k_count(const LossRows r, const LossWork w) {
    for (uint32_t i = threadIdx.x; i <= r.sequences; i += 1024) w.counts[i] = 0;
    __syncthreads();
    for (long long at = 0; at < r.n; at += 1024) {
        const long long row = at + threadIdx.x;
        const int q = row < r.n && r.target(row) >= 0 ? r.sequence(row) : -1;
        if (row < r.n) w.sequence[row] = q;
        const unsigned same = __match_any_sync(0xffffffffu, q), any = __ballot_sync(0xffffffffu, q >= 0);
        if (q >= 0 && (int)(threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(w.counts + q, __popc(same));
        if ((threadIdx.x & 31) == 0 && any) atomicAdd(w.counts + r.sequences, __popc(any));
    }
}

template <int N>
__device__ double block_sum(double v) {
    __shared__ double warp_sum[N / 32];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int i = 0; i < N / 32; i++) v += warp_sum[i];
    return v;
}

// The loss from its parts, always in the same order.  One CTA.
__global__ void __launch_bounds__(1024) k_total(const double* parts, long long n, double by, float* out) {
    grid_dependency_wait();
    double v = 0.0;
    for (long long i = threadIdx.x; i < n; i += 1024) v += parts[i];
    v = block_sum<1024>(v);
    if (threadIdx.x == 0) *out = (float)(v * by);
}

// A pair's lead over the reference, its loss and the slopes of its two
// sequences.  One CTA for each pair.
template <class T>
__global__ void __launch_bounds__(256) k_pairs(const LossRows r, const PreferTerms p, const LossWork w, const LossOut o) {
    grid_dependency_wait();
    const uint32_t pairs = r.sequences / 2, pair = blockIdx.x;
    double lead[2];
    long long counted[2];
    for (int side = 0; side < 2; side++) {
        const uint32_t q = pair + side * pairs;
        const long long lo = r.starts ? max(0ll, (long long)r.starts[q]) : q * r.per;
        const long long hi = r.starts ? min(r.n, (long long)r.starts[q + 1]) : lo + r.per;
        double v = 0.0, n = 0.0;
        for (long long row = lo + threadIdx.x; row < hi; row += 256) {
            const int y = r.target(row);
            if (y < 0) continue;
            const float z = Lane<T>::one(static_cast<const T*>(r.logits)[row * r.stride + y]);
            v += logprob(z, w.stats[row]) - (p.ref ? (double)p.ref[row] : 0.0);
            n += 1.0;
        }
        lead[side] = block_sum<256>(v);
        counted[side] = (long long)block_sum<256>(n);
        if (p.average && counted[side]) lead[side] /= (double)counted[side];
    }
    if (threadIdx.x) return;
    const double d = lead[0] - lead[1], h = p.beta * d, e = p.smoothing;
    double loss, slope;  // by d
    if (p.kind == TS_PREFER_SIGMOID) {
        // log sigmoid(h) = min(h, 0) - log1p(exp(-|h|)), sigmoid'(h) / sigmoid(h) = sigmoid(-h)
        const double t = log1p(exp(-fabs(h))), up = 1.0 / (1.0 + exp(-h)), down = 1.0 / (1.0 + exp(h));
        loss = (1.0 - e) * (t - fmin(h, 0.0)) + e * (t + fmax(h, 0.0));
        if (h != h) loss = h;
        slope = p.beta * (e * up - (1.0 - e) * down);
    } else if (p.kind == TS_PREFER_HINGE) {
        loss = h >= 1.0 ? 0.0 : 1.0 - h;
        slope = h >= 1.0 ? 0.0 : h != h ? h : -(double)p.beta;
    } else {
        const double off = d - 0.5 / p.beta;
        loss = off * off;
        slope = 2.0 * off;
    }
    w.parts[pair] = loss;
    if (o.margins) o.margins[pair] = (float)h;
    slope *= (double)(o.grad_scale ? *o.grad_scale : 1.f) / pairs;
    w.slope[pair] = (float)(p.average && counted[0] ? slope / counted[0] : slope);
    w.slope[pair + pairs] = (float)-(p.average && counted[1] ? slope / counted[1] : slope);
}

template <class T, int MODE>
cudaError_t launch_rows(const RowArgs& a, bool dependent, cudaStream_t s) {
    int dev = 0, sms = 1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    int cl = 1;
    double least = 0;
    for (int c = 1; c <= kCluster; c *= 2) {
        const double cost = (double)((a.r.n * c + 2 * sms - 1) / (2 * sms)) * (1.0 / c + 0.05);
        if (c == 1 || cost < least) cl = c, least = cost;
    }
    const Launch l(cl, 1, dependent, dim3((unsigned)(a.r.n * cl)), kThreads, 0, s);
    return cudaLaunchKernelEx(&l.cfg, k_rows<T, MODE>, a);
}

template <int MODE>
cudaError_t rows(const RowArgs& a, int dtype, bool dependent, cudaStream_t s) {
    if (dtype == DT_F32) return launch_rows<float, MODE>(a, dependent, s);
    return dtype == DT_BF16 ? launch_rows<__nv_bfloat16, MODE>(a, dependent, s) : launch_rows<__half, MODE>(a, dependent, s);
}

template <class T>
cudaError_t pairs(const LossRows& r, const PreferTerms& p, const LossWork& w, const LossOut& o, cudaStream_t s) {
    return launch_dependent(1, k_pairs<T>, dim3(r.sequences / 2), 256, 0, s, r, p, w, o);
}

}  // namespace

cudaError_t launch_logprobs(const LossRows& r, float* logprobs, int dtype, cudaStream_t s) {
    RowArgs a{};
    a.r = r;
    a.o.logprobs = logprobs;
    KScope ks("token_logprobs", s);
    return rows<LOGPROBS>(a, dtype, false, s);
}

cudaError_t launch_logprobs_backward(const LossRows& r, const float* g, const LossOut& o, int dtype, cudaStream_t s) {
    RowArgs a{};
    a.r = r;
    a.o = o;
    a.g = g;
    KScope ks("token_logprobs_backward", s);
    return rows<GIVEN>(a, dtype, false, s);
}

cudaError_t launch_policy(const LossRows& r, const PolicyTerms& p, const LossWork& w, const LossOut& o, int dtype, cudaStream_t s) {
    RowArgs a{};
    a.r = r, a.p = p, a.w = w, a.o = o;
    KScope ks("policy_loss", s, r.n ? 3 : 1);
    cudaError_t e = cudaSuccess;
    if (r.n) {
        k_count<<<1, 1024, 0, s>>>(r, w);
        e = cudaGetLastError();
        if (e == cudaSuccess) e = rows<POLICY>(a, dtype, true, s);
    }
    if (e == cudaSuccess) e = launch_dependent(1, k_total, dim3(1), 1024, 0, s, (const double*)w.parts, r.n, 1.0, o.loss);
    return e;
}

cudaError_t launch_preference(const LossRows& r, const PreferTerms& p, const LossWork& w, const LossOut& o, int dtype, cudaStream_t s) {
    RowArgs a{};
    a.r = r, a.w = w, a.o = o;
    a.o.grad = nullptr;
    const uint32_t n = r.sequences / 2;
    KScope ks("preference_loss", s, 2 + (r.n > 0) + (r.n > 0 && o.grad));
    cudaError_t e = r.n ? rows<LOGPROBS>(a, dtype, false, s) : cudaSuccess;
    if (e == cudaSuccess)
        e = dtype == DT_F32 ? pairs<float>(r, p, w, o, s) : dtype == DT_BF16 ? pairs<__nv_bfloat16>(r, p, w, o, s) : pairs<__half>(r, p, w, o, s);
    if (e == cudaSuccess) e = launch_dependent(1, k_total, dim3(1), 1024, 0, s, (const double*)w.parts, (long long)n, 1.0 / n, o.loss);
    a.o.grad = o.grad;
    if (e == cudaSuccess && r.n && o.grad) e = rows<KNOWN>(a, dtype, true, s);
    return e;
}

}  // namespace tsg
