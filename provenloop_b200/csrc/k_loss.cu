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
// written once.  Rows that fit are held in registers (k_rows, k_short), of longer ones a
// persistent cluster keeps what it can in shared memory (k_ring).  On one B200, in bf16
// over 151936 tokens: 4096 rows' log-probabilities take 197 to 205 us (6.1 to 6.3 TB/s), gradients for
// given slopes 525 to 563 us (4.4 to 4.7 TB/s; 5.9 with known statistics).  Without an element's two exponentials
// and some twenty instructions the same copies take 370 us; with them neither the issue slots (54 to 56 %)
// nor the unit of exponentials (51 %) is at its limit: the rest is roles that wait for one another,
// a row's gradient for its statistics first of all.  Tried and slower: exponentials kept in
// shared memory in 32 bits (570 us: a row's gradient then waits for the next one's
// statistics), a part of them by polynomials on the FMA pipe (586 us), bulk stores of the
// gradient (750 us), more statistics warps and fewer for the gradient (600 us and more).
#include <algorithm>
#include <atomic>
#include <cfloat>

#include "../../include/tsgpu.h"
#include "launch.cuh"
#include "sm100.cuh"
#include "train.cuh"

namespace tsg {

namespace {

constexpr int kCluster = 8;
constexpr int kRowWarps = 8;  // of a CTA of k_rows
constexpr float kLog2e = 1.4426950408889634f;

// What is done with a row that counts: its log-probability; the gradient for
// a given g; the policy loss; the gradient for known statistics and a g by sequence.
enum Mode : int { LOGPROBS, GIVEN, POLICY, KNOWN };

struct RowArgs {
    LossRows r;
    PolicyTerms p;
    LossWork w;
    LossOut o;
    const float* g;  // GIVEN: [n]
    int mode;
    int backwards;   // the last rows first
    int wait;        // the launch before this one has to be waited for
    int units;       // clusters (k_ring) or rows (k_short)
    int log;         // of the CTAs in a cluster
    int own_order;   // the CTAs put the rows in order by themselves
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

// Pairs of f32 in one instruction: the issue slots bound what an element costs.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n .reg .b64 w, x, y, z;\n mov.b64 w, {%2, %3};\n mov.b64 x, {%4, %5};\n mov.b64 y, {%6, %7};\n fma.rn.f32x2 z, w, x, y;\n mov.b64 {%0, %1}, z;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
// The greater one, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// exp(a - b) for a <= b, 1 where they are equal, as 2^t with t = d log2(e), d = a - b.
// (a log2(e) - b log2(e) in one FMA would carry b's rounding, and not give 1.)
// t's rounding and constant make it off by 2^-22 + 2^-22 |d|.  In a row's sum that counts by the
// weight itself, exp(d) |d| at most; results below 2^-126 are 0.
__device__ __forceinline__ float weight(float a, float b) { return exp2_fast((a - b) * kLog2e); }
__device__ __forceinline__ float2 weight2(float2 a, float2 less) {
    const float2 d = mul2(add2(a, less), make_float2(kLog2e, kLog2e));
    return make_float2(exp2_fast(d.x), exp2_fast(d.y));
}
// The same for an element of the gradient, which hangs on its own exponential.  In 16 bits the
// error is lost in the result's rounding (at |d| = 30 a five hundredth of half a step of bf16, a
// sixtieth of fp16's); in f32 it would be most of what the result is off (2^-19 at |d| = 40).
// There 2^t is multiplied by exp(d - t ln 2), 1 + (d - t ln 2) in 32 bits since t's
// rounding is all that is left, and found by one FMA: off by 2^-21 and 2^-28 |d|, beside d's own
// 2^-24 |d|.  Gradients of 300 rows of 50257 (deviation 3) are so off by 3.5e-7 of themselves (root
// of the mean square), without it 5.2e-7; it costs 3 % (1500 rows of 151936: 385 and 375 us).  The
// rows' sums with it: log-probabilities no nearer (3.3e-7 and 3.2e-7), 2 to 5 % slower.
constexpr float kLn2 = 0.69314718f, kLeastExp = -128.f;  // exp of the latter is 0 here; an infinite d would give NaN
template <class T>
__device__ __forceinline__ float grad_weight(float a, float b) {
    if constexpr (sizeof(T) == 2) return weight(a, b);
    const float d = max_nan(a - b, kLeastExp), t = __fmul_rn(d, kLog2e), e = exp2_fast(t);
    return fmaf(e, fmaf(t, -kLn2, d), e);
}
template <class T>
__device__ __forceinline__ float2 grad_weight2(float2 a, float2 less) {
    if constexpr (sizeof(T) == 2) return weight2(a, less);
    float2 d = add2(a, less);
    d = make_float2(max_nan(d.x, kLeastExp), max_nan(d.y, kLeastExp));
    const float2 t = mul2(d, make_float2(kLog2e, kLog2e)), e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
    return fma2(e, fma2(t, make_float2(-kLn2, -kLn2), d), e);
}

// Of a warp's lanes, the same bits in all of them.
__device__ __forceinline__ RowStats join_lanes(const RowStats& s) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(s.max));
    float sum = s.sum * weight(s.max, m);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return {m, sum};
}
// Of no elements, or of such as are -inf; differences of finite maxima are never NaN.
__device__ __forceinline__ RowStats nothing() { return {-FLT_MAX, 0.f}; }

// Adds V vectors to a thread's statistics.
template <class T, int V>
__device__ __forceinline__ void see(RowStats& t, const uint4 (&z)[V]) {
    constexpr int N = Lane<T>::N;
    float m = t.max;
#pragma unroll
    for (int j = 0; j < V; j++) m = fmaxf(m, Lane<T>::top(z[j]));
    const float2 less = make_float2(-m, -m);
    float2 sum[V] = {};
#pragma unroll
    for (int j = 0; j < V; j++) {
        float f[N];
        Lane<T>::open(z[j], f);
#pragma unroll
        for (int i = 0; i < N; i += 2) sum[j] = add2(sum[j], weight2(make_float2(f[i], f[i + 1]), less));
    }
    float2 all = sum[0];
#pragma unroll
    for (int j = 1; j < V; j++) all = add2(all, sum[j]);
    t.sum = fmaf(t.sum, weight(t.max, m), all.x + all.y), t.max = m;
}

// What the gradient of a row is made of: g, -g / s, the target's logit, m.
struct Coef {
    float g, by, zy, max;
};

// -g p of one vector; the target's g is added by fix_target.
template <class T>
__device__ __forceinline__ uint4 slope_of(const uint4& z, const Coef& c) {
    constexpr int N = Lane<T>::N;
    const float2 less = make_float2(-c.max, -c.max), by = make_float2(c.by, c.by);
    float f[N];
    Lane<T>::open(z, f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 p = mul2(grad_weight2<T>(make_float2(f[i], f[i + 1]), less), by);
        f[i] = p.x, f[i + 1] = p.y;
    }
    return Lane<T>::close(f);
}
// g (1 - p) for the target, by the thread that wrote -g p there.
template <class T>
__device__ __forceinline__ void fix_target(T* out, const Coef& c) {
    *out = Lane<T>::put(fmaf(c.by, grad_weight<T>(c.zy, c.max), c.g));
}

// log s: the exponent's part in 64 bits, so that what is left has an error of 2^-24.
__device__ __forceinline__ double log_of(float s) {
    if (!(s >= 0.5f && s < INFINITY)) return log((double)s);
    const uint32_t u = __float_as_uint(s), up = (u & 0x7fffffu) > 0x400000u;  // mantissa above 1.5: halved
    return (double)((int)(u >> 23) - 127 + (int)up) * 0.69314718055994531 + (double)logf(__uint_as_float((u & 0x7fffffu) | (up ? 0x3f000000u : 0x3f800000u)));
}

// The log-probability of a row's target with logit z: the one value that all
// of the row's gradient hangs on.
__device__ __forceinline__ double logprob(float z, const RowStats& s) {
    return z == -INFINITY ? (double)-INFINITY : ((double)z - (double)s.max) - log_of(s.sum);
}

// What finishes a row, loaded before its statistics are there.
struct RowInfo {
    float zy, old, ref, a;  // a: advantage (POLICY), g (GIVEN, KNOWN)
    RowStats s;             // KNOWN
    double share, scaled;   // of the row in the policy loss, and in its gradient
};

__device__ __forceinline__ RowInfo row_info(const RowArgs& a, long long row, float zy) {
    RowInfo i{zy, 0.f, 0.f, 0.f, {0.f, 1.f}, 0.0, 0.0};
    if (a.mode == GIVEN) i.a = a.g[row];
    if (a.mode == KNOWN) {
        i.a = a.w.slope[a.r.sequence(row)];
        i.s = a.w.stats[row];
    }
    if (a.mode == POLICY) {
        const int q = a.r.sequence(row), kind = a.p.kind;
        i.a = a.p.advantages[a.p.advantage_rows ? row : q];
        if (a.p.old) i.old = a.p.old[row];
        if (a.p.ref) i.ref = a.p.ref[row];
        i.share = kind == TS_REDUCE_TOKEN ? 1.0 / a.w.counts[a.r.sequences] : kind == TS_REDUCE_SEQUENCE ? 1.0 / ((double)a.w.counts[q] * a.r.sequences) : 1.0;
        i.scaled = i.share * (a.o.grad_scale ? (double)*a.o.grad_scale : 1.0);
    }
    return i;
}

// The policy loss's term of a row, and its derivative by l.  By a whole warp, the lanes of which
// have the same row: the two exponentials, in 64 bits, are computed at once, by every other lane (5000
// rows of 8000 in bf16: 79.7 us, one after the other 83, and in 32 bits, off by 2^-24 of their arguments, 78).
__device__ __forceinline__ double policy_term(const PolicyTerms& p, const RowInfo& i, double l, double* slope) {
    const bool moves = p.ref && p.kl != 0.f;
    const double d = (double)i.ref - l, own = p.old || moves ? exp(threadIdx.x & 1 ? d : l - (double)i.old) : 0.0;
    const double rho = p.old ? __shfl_sync(0xffffffffu, own, 0) : l == l ? 1.0 : l;
    const double cut = rho < p.low ? (double)p.low : rho > p.high ? (double)p.high : rho, whole = rho * i.a, held = cut * i.a;
    const bool clipped = whole > held;  // not where one is a NaN
    double term = clipped ? -held : -whole, by = clipped ? 0.0 : -whole;
    if (moves) {
        // exp(d) - 1 - d and exp(d) - 1: by the series where they cancel (what is left out is below 2^-40 of it)
        const double e = __shfl_sync(0xffffffffu, own, 1) - 1.0;
        const double series = d * d * (1.0 / 2 + d * (1.0 / 6 + d * (1.0 / 24 + d * (1.0 / 120 + d * (1.0 / 720 + d * (1.0 / 5040 + d * (1.0 / 40320 + d / 362880)))))));
        const bool near = fabs(d) < 0.25;
        term += p.kl * (near ? series : e == INFINITY ? e : e - d);  // d may be infinite too
        by -= p.kl * (near ? d + series : e);
    }
    *slope = by;
    return term;
}

// A row's results but its gradient, written where `write` is set; returns
// what the gradient needs and adds to the loss.
__device__ __forceinline__ Coef finish_row(const RowArgs& a, const RowInfo& i, long long row, const RowStats& s, bool write, double* loss) {
    float g = i.a;
    if (a.mode == LOGPROBS || a.mode == POLICY) {
        const double l = logprob(i.zy, s);
        if (write) {
            if (a.o.logprobs) a.o.logprobs[row] = (float)l;
            if (a.mode == LOGPROBS && a.w.stats) a.w.stats[row] = s, a.w.logs[row] = l;
        }
        if (a.mode == POLICY) {
            double slope;
            *loss += i.share * policy_term(a.p, i, l, &slope);
            g = (float)(i.scaled * slope);
        }
    }
    return {g, -__fdiv_rn(g, s.sum), i.zy, s.max};
}

// The same for a row that does not count.
__device__ __forceinline__ void skip_row(const RowArgs& a, long long row) {
    if ((a.mode == LOGPROBS || a.mode == POLICY) && a.o.logprobs) a.o.logprobs[row] = 0.f;
}

// The loss from its parts in an order that depends on their number alone: the
// last warp to come to a group of them adds it up, the last of these the groups.  Part
// `part` is there.
__device__ __forceinline__ void total(const LossWork& w, uint32_t part, uint32_t parts, double by, float* out) {
    const int lane = (int)(threadIdx.x & 31);
    double* from = w.parts;
    unsigned* ticket = w.ticket;
    for (;;) {
        const uint32_t groups = (uint32_t)loss_groups(parts), group = part / kLossGroup, here = min(kLossGroup, parts - group * kLossGroup);
        unsigned before = 0;
        __syncwarp();
        if (lane == 0) {
            __threadfence();
            before = atomicAdd(ticket + group, 1u);
        }
        if (__shfl_sync(0xffffffffu, before, 0) != here - 1) return;
        __threadfence();
        double v = 0.0;
#pragma unroll 8
        for (uint32_t i = lane; i < here; i += 32) v += __ldcg(from + group * kLossGroup + i);
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (groups == 1) {
            if (lane == 0) *out = (float)(v * by);
            return;
        }
        from += parts, ticket += groups;
        if (lane == 0) from[group] = v;
        part = group, parts = groups;
    }
}
// Before any part: none has come yet.  By a whole CTA.
__device__ __forceinline__ void clear_tickets(const LossWork& w) {
    for (uint32_t i = threadIdx.x; i < w.tickets; i += blockDim.x) w.ticket[i] = 0u;
}

// The vector at p of a row (addressed as Span says) by its elements: -inf for
// what lies outside of [head, last).  Out of line, and by values: rows have two of them.
template <class T>
__device__ __noinline__ uint4 load_edge(const T* x, uint32_t head, uint32_t last, uint32_t p) {
    uint4 z = make_uint4(Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow);
    T* e = reinterpret_cast<T*>(&z);
#pragma unroll
    for (uint32_t i = 0; i < Lane<T>::N; i++)
        if (p + i >= head && p + i < last) e[i] = x[p + i - head];
    return z;
}
template <class T>
__device__ __noinline__ void store_edge(T* out, uint32_t head, uint32_t last, uint32_t p, uint4 z) {
    const T* e = reinterpret_cast<const T*>(&z);
#pragma unroll
    for (uint32_t i = 0; i < Lane<T>::N; i++)
        if (p + i >= head && p + i < last) out[p + i - head] = e[i];
}

// A CTA's part [first, last) of a row whose elements are addressed by
// p = v + head, head being the row's offset from a 16-byte boundary.
template <class T>
struct Span {
    const T* x;
    uint32_t head, first, last;
    // the part `rank` of 2^log parts
    __device__ __forceinline__ Span(const T* x_, uint32_t vocab, int rank, int log) : x(x_) {
        head = (uint32_t)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
        const uint32_t end = head + vocab, span = ((end + (1u << log) - 1 >> log) + 127) / 128 * 128;
        first = min(end, rank * span), last = min(end, first + span);
    }
    __device__ __forceinline__ bool whole(uint32_t p) const { return p >= head && p + Lane<T>::N <= last; }
    __device__ __forceinline__ uint4 edge(uint32_t p) const { return load_edge(x, head, last, p); }
    __device__ __forceinline__ void store(T* out, bool vec, uint32_t p, const uint4& z) const {
        if (vec && whole(p)) *reinterpret_cast<uint4*>(out + p - head) = z;
        else store_edge(out, head, last, p, z);
    }
};

// The target of a row that counts (for a given g of 0 it need not), else -1.
__device__ __forceinline__ int counted(const RowArgs& a, long long row, long long lo, long long hi) {
    if (row < lo || row >= hi) return -1;
    const int y = a.r.target(row);
    const float g = a.mode == GIVEN ? a.g[row] : 1.f;  // at once with the target
    return g == 0.f ? -1 : y;
}
__device__ __forceinline__ long long rows_from(const LossRows& r) { return r.starts ? max(0ll, (long long)r.starts[0]) : 0ll; }
__device__ __forceinline__ long long rows_to(const LossRows& r) { return r.starts ? min(r.n, (long long)r.starts[r.sequences]) : r.n; }

// Rows that a CTA, or a cluster of them, holds in registers, V vectors a thread.
template <class T, int THREADS, int V>
__global__ void __launch_bounds__(THREADS) k_short(const RowArgs a) {
    constexpr uint32_t N = Lane<T>::N, W = THREADS / 32;
    __shared__ RowStats warp_stats[W], cta_stats[kCluster];
    __shared__ Coef shared_coef;
    const int cl = 1 << a.log, rank = (int)cluster_rank();
    if (cl > 1) cluster_arrive();
    const long long row = blockIdx.x >> a.log;
    const int y = counted(a, row, rows_from(a.r), rows_to(a.r)), lane = (int)(threadIdx.x & 31);
    const Span<T> sp(static_cast<const T*>(a.r.logits) + row * a.r.stride, a.r.vocab, rank, a.log);
    T* const out = a.o.grad ? static_cast<T*>(a.o.grad) + row * a.o.grad_stride : nullptr;
    const bool vec = out && reinterpret_cast<uintptr_t>(out) % 16 == reinterpret_cast<uintptr_t>(sp.x) % 16;
    uint4 z[V];
    Coef c{0.f, 0.f, 0.f, 0.f};
    if (y >= 0) {
        const float zy = Lane<T>::one(sp.x[y]);  // before the row may be written
#pragma unroll
        for (uint32_t j = 0; j < V; j++) {
            const uint32_t p = sp.first + (threadIdx.x + j * THREADS) * N;
            z[j] = p >= sp.last ? make_uint4(Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow)
                   : sp.whole(p) ? *reinterpret_cast<const uint4*>(sp.x + p - sp.head) : sp.edge(p);
        }
        RowStats s = nothing();
        if (a.mode != KNOWN) {
            see<T, V>(s, z);
            s = join_lanes(s);
            if (lane == 0) warp_stats[threadIdx.x >> 5] = s;
        }
        __syncthreads();
        if (cl > 1 && a.mode != KNOWN) {
            cluster_wait();  // the other CTAs have started
            if (threadIdx.x < 32) {
                s = join_lanes(lane < (int)W ? warp_stats[lane] : nothing());
                if (lane < cl)
                    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(map_rank(&cta_stats[rank], (uint32_t)lane)), "f"(s.max), "f"(s.sum)
                                 : "memory");
            }
            cluster_sync_all();
        }
        if (threadIdx.x < 32) {
            if (a.wait) grid_dependency_wait();
            const RowInfo i = row_info(a, row, zy);
            const RowStats* const from = cl > 1 ? cta_stats : warp_stats;
            s = a.mode == KNOWN ? i.s : join_lanes(lane < (cl > 1 ? cl : (int)W) ? from[lane] : nothing());
            double loss = 0.0;
            c = finish_row(a, i, row, s, rank == 0 && lane == 0, &loss);
            if (lane == 0) {
                shared_coef = c;
                if (a.mode == POLICY && rank == 0) a.w.parts[row] = loss;
            }
        }
        if (cl > 1 && a.mode == KNOWN) cluster_wait();
        __syncthreads();
        c = shared_coef;
    } else {
        if (cl > 1) cluster_wait();
        if (threadIdx.x < 32) {
            if (a.wait) grid_dependency_wait();
            if (lane == 0 && rank == 0) {
                skip_row(a, row);
                if (a.mode == POLICY) a.w.parts[row] = 0.0;
            }
        }
    }
    if (a.mode == LOGPROBS && blockIdx.x == 0) clear_tickets(a.w);
    if (a.mode == POLICY && rank == 0 && threadIdx.x < 32) total(a.w, (uint32_t)row, (uint32_t)a.units, 1.0, a.o.loss);
    if (!out) return;
#pragma unroll
    for (uint32_t j = 0; j < V; j++) {
        const uint32_t p = sp.first + (threadIdx.x + j * THREADS) * N;
        if (p >= sp.last) continue;
        sp.store(out, vec, p, c.g == 0.f ? make_uint4(0u, 0u, 0u, 0u) : slope_of<T>(z[j], c));
        if (c.g != 0.f && (uint32_t)y + sp.head - p < N) fix_target(out + y, c);
    }
}

// Many short rows: a warp to a row, V vectors a lane, and no barriers.
template <class T, int V>
__global__ void __launch_bounds__(kRowWarps * 32) k_rows(const RowArgs a) {
    constexpr uint32_t N = Lane<T>::N;
    const int lane = (int)(threadIdx.x & 31), unit = (int)(blockIdx.x * kRowWarps + (threadIdx.x >> 5));
    if (a.mode == LOGPROBS && blockIdx.x == 0) clear_tickets(a.w);
    const long long lo = rows_from(a.r), hi = rows_to(a.r);
    const auto row_at = [&](long long i) { return a.backwards ? a.r.n - 1 - i : i; };
    double loss = 0.0;
    bool wait = a.wait;
    int y = unit < a.r.n ? counted(a, row_at(unit), lo, hi) : -1;
    for (long long i = unit; i < a.r.n; i += a.units) {
        const long long row = row_at(i);
        const Span<T> sp(static_cast<const T*>(a.r.logits) + row * a.r.stride, a.r.vocab, 0, 0);
        uint4 z[V];
        float zy = 0.f;
        if (y >= 0) {
            zy = Lane<T>::one(sp.x[y]);
#pragma unroll
            for (uint32_t j = 0; j < V; j++) {
                const uint32_t p = (lane + j * 32) * N;
                z[j] = p >= sp.last ? make_uint4(Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow)
                       : sp.whole(p) ? *reinterpret_cast<const uint4*>(sp.x + p - sp.head) : sp.edge(p);
            }
        }
        const int next = i + a.units < a.r.n ? counted(a, row_at(i + a.units), lo, hi) : -1;
        if (wait) grid_dependency_wait(), wait = false;
        Coef c{0.f, 0.f, 0.f, 0.f};
        if (y >= 0) {
            const RowInfo info = row_info(a, row, zy);
            RowStats s = info.s;
            if (a.mode != KNOWN) {
                s = nothing();
                see<T, V>(s, z);
                s = join_lanes(s);
            }
            c = finish_row(a, info, row, s, lane == 0, &loss);
        } else if (lane == 0) {
            skip_row(a, row);
        }
        __syncwarp();  // the row may be written now
        if (a.o.grad) {
            T* const out = static_cast<T*>(a.o.grad) + row * a.o.grad_stride;
            const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == reinterpret_cast<uintptr_t>(sp.x) % 16;
#pragma unroll
            for (uint32_t j = 0; j < V; j++) {
                const uint32_t p = (lane + j * 32) * N;
                if (p >= sp.last) continue;
                sp.store(out, vec, p, c.g == 0.f ? make_uint4(0u, 0u, 0u, 0u) : slope_of<T>(z[j], c));
                if (c.g != 0.f && (uint32_t)y + sp.head - p < N) fix_target(out + y, c);
            }
        }
        y = next;
    }
    if (a.mode == POLICY && unit < a.units) {
        if (wait) grid_dependency_wait();
        if (lane == 0) a.w.parts[unit] = loss;
        total(a.w, (uint32_t)unit, (uint32_t)a.units, 1.0, a.o.loss);
    }
}

// Longer rows: persistent clusters, each with every so many-th row, a CTA with
// its part of it in slots of a ring in shared memory.  Warps have roles:
//   one starts the copies into the slots,
//   S warps take the statistics of a part as it arrives,
//   one joins them, exchanges them within the cluster and finishes the row,
//   G warps write the part's gradient once that is known.
// A part keeps KEEP slots until its gradient is written from them; what there is
// more of it is copied once more (from L2) behind the rest and before the next
// row, whose statistics are taken meanwhile.  So a row comes from memory once.
// Every wait goes by one of these barriers, in the order of the rows; which it is
// waiting for is never more than one phase away (test_loss_ring.py has a model).
constexpr uint32_t kSlot = 16384;  // of half the size, the thread that starts the copies is the bound (4.0 TB/s)
constexpr uint32_t kZeros = 4096;  // bytes that rows which do not count are written from
constexpr int kTeam = 8;   // warps that take a slot together, four vectors a lane
constexpr int kDepth = 4;  // rows between two roles
// Rows that the CTAs put in order by themselves, each for itself before its first copy, where
// k_order would be another launch to wait for.  As they come, in order by k_order, and so (us, with gradients):
// 1001 rows of 151936 in bf16, 615 of which count, 140, 119 and 118; 600, 296 of which, 83, 70 and 69; 1100 rows that
// all count 160, 165 and 163; 909 rows of 50257 in f32, 391 of which, 63, 66 and 64.
constexpr int kOwnOrder = 2048;
constexpr int kStats = 2;  // rows whose lanes' statistics are waiting to be joined
// The teams of a role take the slots in turn, and every team always the same
// ones.  Where there are both roles, a slot is free again when a team of either has
// arrived, whether the load was for it or not: so no team is more than one load behind, and a
// parity wait tells the loads apart.  Statistics alone: two CTAs on an SM (4096 rows of
// 151936 in bf16: 197 us, with one of twice the slots 211).
template <bool S, bool G>
struct Roles {
    static constexpr int TS = !S ? 0 : G ? 1 : 2, TG = G ? 2 : 0, CTAS = G ? 1 : 2, SLOTS = G ? 12 : 6;
    static constexpr int KEEP = 8;  // of them; the rest is for the next row while one waits for its gradient
    static constexpr int THREADS = 64 + (TS + TG) * kTeam * 32;
    static constexpr size_t SMEM = SLOTS * kSlot + (G ? kZeros : 0);
    static_assert((!S || SLOTS % TS == 0) && (!G || SLOTS % TG == 0), "a slot's team must not change");
};

template <int S_THREADS>
struct RingShared {
    uint64_t full[12], empty[12], stats_full[kStats], stats_free[kStats], joined[kDepth], coef_full[kDepth], coef_free[kDepth];
    RowStats lane_stats[kStats][S_THREADS ? S_THREADS : 1], cta_stats[kDepth][kCluster];
    Coef coef[kDepth];
    uint32_t dead;
};

// mbar_wait with short sleeps between two looks: warps that wait would take
// issue slots from those that compute (550 and 530 us for the gradient of 4096 rows of 151936).
__device__ __forceinline__ bool sleep_wait(uint64_t* b, uint32_t parity, uint32_t* dead) {
    if (mbar_try(b, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try(b, parity)) {
        __nanosleep(20);
        if (*reinterpret_cast<volatile uint32_t*>(dead)) return false;
        if (clock64() - t0 > kWaitCycles) {
            atomicAdd(&g_expired_waits, 1ull);
            atomicExch(dead, 1u);
            return false;
        }
    }
    return true;
}
// A wait of a whole warp, whose lanes go on or give up together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t* dead) {
    return __all_sync(0xffffffffu, sleep_wait(bar, parity, dead));
}

// Before a thread says that it has read a slot: the next copy into it is of
// another proxy, which the arrival at a barrier alone does not order with loads that have
// not come back yet (they met the next row's elements in one row of 13000).
__device__ __forceinline__ void reads_done() { fence_async_shared(); }

// The rows that count, and behind them from the end the others: by k_order, by
// the CTA itself, or as they come.
struct Order {
    uint16_t own[kOwnOrder];  // if a.own_order
    int counts[32], count;
    __device__ __forceinline__ int at(const RowArgs& a, int i) const { return a.own_order ? own[i] : a.w.order[i]; }
};

// The next 32 of a cluster's rows, one a lane.  Of rows in order, every so
// many-th that counts and every so many-th other one, evenly mixed: the others only
// write, which costs next to nothing beside those that compute.
struct Batch {
    int row = 0, y = -1;
    uint32_t rows, counts;  // lanes that have a row; whose row counts
    __device__ __forceinline__ Batch(const RowArgs& a, const Order& o, int b, int lo, int hi, int cluster) {
        const int t = b * 32 + (int)(threadIdx.x & 31), n = (int)a.r.n;
        bool there;
        if (a.own_order || a.w.order) {
            const int other = a.units - 1 - cluster;
            const int mine = o.count > cluster ? (o.count - cluster - 1) / a.units + 1 : 0;
            const int rest = n - o.count > other ? (n - o.count - other - 1) / a.units + 1 : 0;
            there = t < mine + rest;
            if (there) {
                const int before = (int)((long long)t * mine / (mine + rest));
                if ((int)((t + 1ll) * mine / (mine + rest)) > before) {
                    row = o.at(a, cluster + (a.backwards ? mine - 1 - before : before) * a.units);
                    y = a.r.target(row);
                } else {
                    row = o.at(a, n - 1 - (other + (t - before) * a.units));
                }
            }
        } else {
            const long long i = (long long)t * a.units + cluster;
            there = i < n;
            if (there) {
                row = a.backwards ? n - 1 - (int)i : (int)i;
                y = counted(a, row, lo, hi);
            }
        }
        rows = __ballot_sync(0xffffffffu, there), counts = __ballot_sync(0xffffffffu, y >= 0);
    }
    __device__ __forceinline__ int row_of(int lane) const { return __shfl_sync(0xffffffffu, row, lane); }
};

template <class T, bool S, bool G>
__global__ void __launch_bounds__(Roles<S, G>::THREADS, Roles<S, G>::CTAS) k_ring(const RowArgs a) {
    constexpr uint32_t N = Lane<T>::N, SLOT = kSlot / sizeof(T);
    constexpr int TS = Roles<S, G>::TS, TG = Roles<S, G>::TG, SLOTS = Roles<S, G>::SLOTS, KEEP = Roles<S, G>::KEEP;
    constexpr uint32_t STEP = 32 * N, PIECE = 4 * STEP;  // elements of a slot that a warp takes
    static_assert(PIECE * kTeam == SLOT, "a team takes a slot");
    extern __shared__ __align__(128) unsigned char slots[];
    __shared__ RingShared<TS * kTeam * 32> sh;
    __shared__ Order order;
    const int rank = (int)cluster_rank(), warp = (int)(threadIdx.x >> 5), lane = (int)(threadIdx.x & 31);
    const int cl = 1 << a.log, cluster = (int)(blockIdx.x >> a.log);
    if (threadIdx.x == 0) {
        for (int i = 0; i < SLOTS; i++) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], S && G ? 2 * kTeam : kTeam);
        for (int i = 0; i < kStats; i++) mbar_init(&sh.stats_full[i], TS * kTeam), mbar_init(&sh.stats_free[i], 1);
        for (int i = 0; i < kDepth; i++) {
            mbar_init(&sh.joined[i], 1);
            mbar_init(&sh.coef_full[i], 1), mbar_init(&sh.coef_free[i], TG * kTeam);
        }
        sh.dead = 0;
        mbar_init_fence();
    }
    if (a.mode == LOGPROBS && blockIdx.x == 0) clear_tickets(a.w);
    if (G && threadIdx.x < kZeros / 16) {
        reinterpret_cast<uint4*>(slots + SLOTS * kSlot)[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
        fence_async_shared();
    }
    const int lo = (int)rows_from(a.r), hi = (int)rows_to(a.r);
    if (a.own_order) {
        constexpr int W = Roles<S, G>::THREADS / 32, EACH = (kOwnOrder / 32 + W - 1) / W;
        int y[EACH];
        unsigned any[EACH];
        int mine = 0;
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            const int row = (warp * EACH + j) * 32 + lane;
            y[j] = row < a.r.n ? counted(a, row, lo, hi) : -1;
        }
#pragma unroll
        for (int j = 0; j < EACH; j++) any[j] = __ballot_sync(0xffffffffu, y[j] >= 0), mine += __popc(any[j]);
        if (lane == 0) order.counts[warp] = mine;
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < W; w++) {
            if (w == warp) before = all;
            all += order.counts[w];
        }
        if (threadIdx.x == 0) order.count = all;
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            const int row = (warp * EACH + j) * 32 + lane, in_front = before + __popc(any[j] & ((1u << lane) - 1));
            if (row < a.r.n) order.own[any[j] >> lane & 1 ? in_front : (int)a.r.n - 1 - (row - in_front)] = (uint16_t)row;
            before += __popc(any[j]);
        }
    } else if (a.w.order) {
        if (a.wait) grid_dependency_wait();
        if (threadIdx.x == 0) order.count = a.w.order[a.r.n];
    }
    __syncthreads();
    cluster_arrive();  // waited for before the first access to another CTA's shared memory
    const auto span_of = [&](int row) { return Span<T>(static_cast<const T*>(a.r.logits) + row * a.r.stride, a.r.vocab, rank, a.log); };
    const auto chunks_of = [](const Span<T>& sp) { return (int)((sp.last - sp.first + SLOT - 1) / SLOT); };
    T* const data = reinterpret_cast<T*>(slots);
    T* const zeros = data + SLOTS * SLOT;  // kZeros bytes of them
    const auto again_of = [&](int n) { return S && G ? max(0, n - KEEP) : 0; };  // slots that are released after the statistics
    bool ok = true;

    if (warp == 0) {
        Ring at(SLOTS, 1);
        for (int b = 0; ok; b++) {
            const Batch rows(a, order, b, lo, hi, cluster);
            if (!rows.rows) break;
            for (uint32_t left = rows.counts; left && ok; left &= left - 1) {
                const Span<T> sp = span_of(rows.row_of(__ffs(left) - 1));
                const int n = chunks_of(sp), loads = n + again_of(n);
                for (int c = 0; c < loads && ok; c++, at.next()) {
                    if (lane) continue;
                    const uint32_t p0 = sp.first + (c < n ? c : c - n) * SLOT, p1 = min(sp.last, p0 + SLOT);
                    const uint32_t from = p0 < sp.head ? p0 + N : p0, to = p1 / N * N;
                    const uint32_t bytes = to > from ? (to - from) * (uint32_t)sizeof(T) : 0u;
                    ok = sleep_wait(&sh.empty[at.i], at.phase, &sh.dead);
                    if (!ok) break;
                    mbar_expect(&sh.full[at.i], bytes);
                    if (bytes) bulk_copy(smem_u32(data + at.i * SLOT + (from - p0)), sp.x + from - sp.head, bytes, &sh.full[at.i]);
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
        }
        if (!ok) settle();
    } else if (warp == 1) {
        Ring k(kDepth, 0), ks(kStats, 0);
        double loss = 0.0;
        bool met = false;
        if (a.wait && !a.w.order) grid_dependency_wait();
        for (int b = 0; ok; b++) {
            const Batch rows(a, order, b, lo, hi, cluster);
            if (!rows.rows) break;
            RowInfo mine{};
            if (rows.y >= 0) mine = row_info(a, rows.row, Lane<T>::one((static_cast<const T*>(a.r.logits) + rows.row * a.r.stride)[rows.y]));
            else if ((rows.rows >> lane & 1) && rank == 0) skip_row(a, rows.row);
            for (uint32_t left = rows.counts; left && ok; left &= left - 1, k.next()) {
                const int from = __ffs(left) - 1;
                RowInfo i;
                i.zy = __shfl_sync(0xffffffffu, mine.zy, from), i.old = __shfl_sync(0xffffffffu, mine.old, from);
                i.ref = __shfl_sync(0xffffffffu, mine.ref, from), i.a = __shfl_sync(0xffffffffu, mine.a, from);
                i.share = __shfl_sync(0xffffffffu, mine.share, from), i.scaled = __shfl_sync(0xffffffffu, mine.scaled, from);
                RowStats s{__shfl_sync(0xffffffffu, mine.s.max, from), __shfl_sync(0xffffffffu, mine.s.sum, from)};
                if (S) {
                    ok = warp_wait(&sh.stats_full[ks.i], ks.phase, &sh.dead);
                    if (!ok) break;
                    const RowStats* const t = sh.lane_stats[ks.i] + lane;
                    s = nothing();
#pragma unroll
                    for (int j = 0; j < TS * kTeam; j++) s.max = fmaxf(s.max, t[j * 32].max);
#pragma unroll 4
                    for (int j = 0; j < TS * kTeam; j++) s.sum = fmaf(t[j * 32].sum, weight(t[j * 32].max, s.max), s.sum);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.stats_free[ks.i]);
                    ks.next();
                    s = join_lanes(s);
                    if (cl > 1) {
                        if (!met) cluster_wait(), met = true;
                        if (lane == 0) mbar_expect(&sh.joined[k.i], (uint32_t)cl * sizeof(RowStats));
                        if (lane < cl)
                            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(
                                             map_rank(&sh.cta_stats[k.i][rank], (uint32_t)lane)),
                                         "f"(s.max), "f"(s.sum), "r"(map_rank(&sh.joined[k.i], (uint32_t)lane))
                                         : "memory");
                        ok = warp_wait(&sh.joined[k.i], k.phase, &sh.dead);
                        if (!ok) break;
                        s = join_lanes(lane < cl ? sh.cta_stats[k.i][lane] : nothing());
                    }
                }
                const Coef c = finish_row(a, i, rows.row_of(from), s, rank == 0 && lane == 0, &loss);
                if (G) {
                    ok = warp_wait(&sh.coef_free[k.i], k.phase ^ 1, &sh.dead);
                    if (!ok) break;
                    if (lane == 0) {
                        sh.coef[k.i] = c;
                        mbar_arrive(&sh.coef_full[k.i]);
                    }
                }
            }
        }
        if (a.mode == POLICY && rank == 0 && ok) {
            if (lane == 0) a.w.parts[cluster] = loss;
            total(a.w, (uint32_t)cluster, (uint32_t)a.units, 1.0, a.o.loss);
        }
        if (!met) cluster_wait();
    } else if (S && (!G || warp < 2 + TS * kTeam)) {
        const int w = (warp - 2) % kTeam, team = (warp - 2) / kTeam;
        Ring at(SLOTS, 0), k(kStats, 0);
        for (int b = 0; ok; b++) {
            const Batch rows(a, order, b, lo, hi, cluster);
            if (!rows.rows) break;
            for (uint32_t left = rows.counts; left && ok; left &= left - 1, k.next()) {
                const Span<T> sp = span_of(rows.row_of(__ffs(left) - 1));
                const int n = chunks_of(sp), again = again_of(n);
                RowStats t = nothing();
                for (int c = 0; c < n; c++, at.next()) {
                    if (at.i % TS != team) continue;
                    ok = warp_wait(&sh.full[at.i], at.phase, &sh.dead);
                    if (!ok) break;
                    const T* const here = data + at.i * SLOT + w * PIECE + lane * N;  // this lane's first vector
                    const uint32_t p0 = sp.first + c * SLOT + w * PIECE;
                    uint4 z[4];
                    if (p0 >= sp.head && p0 + PIECE <= sp.last) {
#pragma unroll
                        for (uint32_t j = 0; j < 4; j++) z[j] = *reinterpret_cast<const uint4*>(here + j * STEP);
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 4; j++) {
                            const uint32_t p = p0 + j * STEP + lane * N;
                            z[j] = p >= sp.last ? make_uint4(Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow, Lane<T>::kLow)
                                   : sp.whole(p) ? *reinterpret_cast<const uint4*>(here + j * STEP) : sp.edge(p);
                        }
                    }
                    reads_done();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.empty[at.i]);
                    if (G && c < again && lane == 0) mbar_arrive(&sh.empty[at.i]);  // in the place of the other role
                    see<T, 4>(t, z);
                }
                ok = ok && warp_wait(&sh.stats_free[k.i], k.phase ^ 1, &sh.dead);
                if (ok) sh.lane_stats[k.i][(warp - 2) * 32 + lane] = t;
                __syncwarp();
                if (lane == 0 && ok) mbar_arrive(&sh.stats_full[k.i]);
                // what arrives once more is not for this role, but it has to be seen before the slot goes on
                for (int c = 0; c < again && ok; c++, at.next()) {
                    if (at.i % TS != team) continue;
                    ok = warp_wait(&sh.full[at.i], at.phase, &sh.dead);
                    if (lane == 0 && ok) mbar_arrive(&sh.empty[at.i]);
                }
            }
        }
    } else {
        constexpr int first = 2 + TS * kTeam;
        const int w = (warp - first) % kTeam, team = (warp - first) / kTeam;
        Ring at(SLOTS, 0), k(kDepth, 0);
        for (int b = 0; ok; b++) {
            const Batch rows(a, order, b, lo, hi, cluster);
            if (!rows.rows) break;
            for (uint32_t left = rows.rows; left && ok; left &= left - 1) {
                const int of = __ffs(left) - 1;
                const int row = rows.row_of(of);
                const Span<T> sp = span_of(row);
                T* const out = static_cast<T*>(a.o.grad) + row * a.o.grad_stride;
                const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == reinterpret_cast<uintptr_t>(sp.x) % 16;
                if (!(rows.counts >> of & 1)) {
                    if (vec) {
                        // whole vectors by bulk stores of zeros, the row's ends by elements
                        const uint32_t from = sp.first < sp.head ? N : sp.first, to = sp.last / N * N;
                        if (lane == 0) {
                            for (uint32_t p = from + (uint32_t)(warp - first) * (kZeros / sizeof(T)); p < to; p += TG * kTeam * (kZeros / sizeof(T)))
                                bulk_store(out + p - sp.head, smem_u32(zeros), min(to - p, (uint32_t)(kZeros / sizeof(T))) * sizeof(T));
                            bulk_commit();
                        }
                        if (warp == first && sp.first < sp.last) {
                            const uint32_t p = lane < (int)N ? sp.first + lane : max(to, from) + lane - N;
                            if (lane < 2 * (int)N && p >= sp.head && p < sp.last && (lane < (int)N ? p < from : true)) out[p - sp.head] = Lane<T>::put(0.f);
                        }
                    } else {
                        for (uint32_t p = sp.first + (uint32_t)(warp - first) * STEP + lane * N; p < sp.last; p += TG * kTeam * STEP)
                            store_edge(out, sp.head, sp.last, p, make_uint4(0u, 0u, 0u, 0u));
                    }
                    continue;
                }
                const uint32_t y = (uint32_t)__shfl_sync(0xffffffffu, rows.y, of);
                const int n = chunks_of(sp), again = again_of(n);
                if (again) at.skip(again);
                ok = warp_wait(&sh.coef_full[k.i], k.phase, &sh.dead);
                if (!ok) break;
                const Coef c = sh.coef[k.i];
                const bool zero = c.g == 0.f;  // not for a NaN
                for (int pos = again; pos < n + again; pos++, at.next()) {
                    if (at.i % TG != team) continue;
                    const int q = pos < n ? pos : pos - n;
                    ok = warp_wait(&sh.full[at.i], at.phase, &sh.dead);
                    if (!ok) break;
                    const T* const here = data + at.i * SLOT + w * PIECE + lane * N;  // this lane's first vector
                    const uint32_t p0 = sp.first + q * SLOT + w * PIECE;
                    const bool inside = vec && p0 >= sp.head && p0 + PIECE <= sp.last;
                    T* const to = out + (p0 - sp.head) + lane * N;
                    uint4 z[4];
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) {
                        const uint32_t p = p0 + j * STEP + lane * N;
                        if (inside || sp.whole(p)) z[j] = *reinterpret_cast<const uint4*>(here + j * STEP);
                        else if (p < sp.last) z[j] = sp.edge(p);
                    }
                    reads_done();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.empty[at.i]);
                    if (!zero) {
#pragma unroll
                        for (uint32_t j = 0; j < 4; j++) z[j] = slope_of<T>(z[j], c);
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 4; j++) z[j] = make_uint4(0u, 0u, 0u, 0u);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) {
                        const uint32_t p = p0 + j * STEP + lane * N;
                        if (inside) *reinterpret_cast<uint4*>(to + j * STEP) = z[j];
                        else if (p < sp.last) sp.store(out, vec, p, z[j]);
                    }
                    // the target, by the lane that has its vector; a last slot reaches into the next CTA's part, whose
                    // target it must not touch: in place, that CTA may not have read the logit yet
                    const uint32_t v = y + sp.head - p0;
                    if (!zero && v < PIECE && y + sp.head < sp.last && v % STEP / N == (uint32_t)lane) fix_target(out + y, c);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.coef_free[k.i]);
                k.next();
            }
        }
        if (lane == 0) tma_store_wait_read<0>();
    }
    if (warp != 1) cluster_wait();
    cluster_sync_all();  // no CTA ends while another may still write to its shared memory
}

constexpr int kOrderRows = 4096;  // of a CTA of k_order at a time
// Before the rows: how many of them count (policy: by sequence, and all of
// them), and their order (order[n]: how many count, which come first, the others from
// the end), so that the clusters get as many.  By every so many-th of a padded batch's
// rows some had a quarter more than the mean (6144 rows in 16 sequences, 2996 of
// which count, on two CTAs each: 530 us, in order 506).  One CTA, or without an order several,
// whose counts then are zeros already.
__global__ void __launch_bounds__(1024) k_order(const RowArgs a) {
    constexpr int EACH = kOrderRows / 1024;
    __shared__ int before[32], found;
    release_dependents();
    const LossRows& r = a.r;
    const bool policy = a.mode == POLICY, one = gridDim.x == 1;
    const int warp = (int)(threadIdx.x >> 5), lane = (int)(threadIdx.x & 31);
    if (policy && one)
        for (uint32_t i = threadIdx.x; i <= r.sequences; i += 1024) a.w.counts[i] = 0;
    if (blockIdx.x == 0) clear_tickets(a.w);
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    const long long lo = rows_from(r), hi = rows_to(r);
    for (long long at = blockIdx.x * 1024ll * EACH; at < r.n; at += gridDim.x * 1024ll * EACH) {
        unsigned any[EACH];
        int mine = 0;
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            const long long row = at + (warp * EACH + j) * 32 + lane;
            const bool is = row < r.n && counted(a, row, lo, hi) >= 0;
            any[j] = __ballot_sync(0xffffffffu, is);
            mine += __popc(any[j]);
            if (policy) {
                const int q = is ? r.sequence(row) : -1;
                const unsigned same = __match_any_sync(0xffffffffu, q);
                if (is && lane == __ffs(same) - 1) atomicAdd(a.w.counts + q, __popc(same));
            }
        }
        if (lane == 0) before[warp] = mine;
        __syncthreads();
        if (warp == 0) {
            const int v = before[lane];
            int sum = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            before[lane] = found + sum - v;
            __syncwarp();
            if (lane == 31) found += sum;
        }
        __syncthreads();
        if (a.w.order) {
            int c = before[warp];  // rows that count in front of this warp's next 32
#pragma unroll
            for (int j = 0; j < EACH; j++) {
                const long long row = at + (warp * EACH + j) * 32 + lane;
                const int mine_before = c + __popc(any[j] & ((1u << lane) - 1));
                if (row < r.n) a.w.order[any[j] >> lane & 1 ? mine_before : r.n - 1 - (row - mine_before)] = (int)row;
                c += __popc(any[j]);
            }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (policy && one) a.w.counts[r.sequences] = found;
        else if (policy) atomicAdd(a.w.counts + r.sequences, found);
        if (a.w.order) a.w.order[r.n] = found;
    }
}

// A pair's lead over the reference, its loss and the slopes of its two
// sequences, in 64 bits: differences of long sums.  One CTA for each pair, half
// of it for each sequence, so that nothing waits but the loads, once.
__global__ void __launch_bounds__(512) k_pairs(const LossRows r, const PreferTerms p, const LossWork w, const LossOut o) {
    constexpr int HALF = 256;
    __shared__ double sums[16], numbers[16];
    release_dependents();
    grid_dependency_wait();
    const uint32_t pairs = r.sequences / 2, pair = blockIdx.x, q = pair + (threadIdx.x / HALF) * pairs;
    const int lane = (int)(threadIdx.x & 31);
    const long long lo = r.starts ? max(0ll, (long long)r.starts[q]) : q * r.per;
    const long long hi = r.starts ? min(r.n, (long long)r.starts[q + 1]) : lo + r.per;
    double v = 0.0, n = 0.0;
#pragma unroll 2
    for (long long row = lo + threadIdx.x % HALF; row < hi; row += HALF) {
        const double l = w.logs[row];  // anything where the row does not count
        const float ref = p.ref ? p.ref[row] : 0.f;
        if (r.target(row) >= 0) v += l - (double)ref, n += 1.0;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d), n += __shfl_xor_sync(0xffffffffu, n, d);
    if (lane == 0) sums[threadIdx.x >> 5] = v, numbers[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    v = sums[lane & 15], n = numbers[lane & 15];
#pragma unroll
    for (int d = 4; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d), n += __shfl_xor_sync(0xffffffffu, n, d);
    if (p.average && n > 0.0) v /= n;
    const double d = __shfl_sync(0xffffffffu, v, 0) - __shfl_sync(0xffffffffu, v, 8), h = p.beta * d, e = p.smoothing;
    double loss, slope;  // by d
    if (p.kind == TS_PREFER_SIGMOID) {
        // log sigmoid(h) = min(h, 0) - log(1 + t) and sigmoid(-|h|) = t / (1 + t) with t = exp(-|h|)
        const double t = exp(-fabs(h)), rest = log1p(t), small = t / (1.0 + t), up = h < 0.0 ? small : 1.0 - small, down = h < 0.0 ? 1.0 - small : small;
        loss = (1.0 - e) * (rest - fmin(h, 0.0));
        if (e > 0.0) loss += e * (rest + fmax(h, 0.0));  // 0, and not 0 times infinity, where h is infinite
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
    slope *= (double)(o.grad_scale ? *o.grad_scale : 1.f) / pairs;
    if (lane == 0) {
        w.parts[pair] = loss;
        if (o.margins) o.margins[pair] = (float)h;
    }
    if (lane == 0 || lane == 8) w.slope[q + (lane ? pairs : 0)] = (float)((lane ? -slope : slope) / (p.average && n > 0.0 ? n : 1.0));
    total(w, pair, pairs, 1.0 / pairs, o.loss);
}

int log2_of(int cl) { return cl == 8 ? 3 : cl / 2; }

// Clusters of `cl` CTAs of a k_ring that the current device runs at once.
template <class T, bool S, bool G>
cudaError_t clusters_at_once(int cl, int* out) {
    using R = Roles<S, G>;
    static std::atomic<int> known[64][kCluster + 1];  // by device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && (*out = known[dev][cl].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
    const Launch l(cl, 1, false, dim3((unsigned)cl), R::THREADS, R::SMEM, nullptr);
    if (cl > 1) {
        e = cudaOccupancyMaxActiveClusters(out, k_ring<T, S, G>, &l.cfg);
    } else {
        int sms = 0;
        e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        *out = sms * R::CTAS;
    }
    if (e == cudaSuccess && *out < 1) e = cudaErrorInvalidConfiguration;
    if (e == cudaSuccess && dev < 64) known[dev][cl].store(*out, std::memory_order_relaxed);
    return e;
}

// CTAs to a row: rounds of the clusters that run at once, times what one of
// them takes for a row, fixed and by the KiB of a CTA's part.  Measured, in us
// for 1500 rows on 1, 2, 4 and 8 CTAs, statistics and gradient:
//   16-bit, vocabulary  20000:  45  60  78 149      151936: 211 214 227 329
//   f32,                20000:  57  68  96 129      151936: 427 357 384 408
// (24 rows of 151936: 27 19 15 15 and 37 23 17 17; statistics alone are
// fastest on one CTA from 300 rows on, on four for few.)  A part of more than
// half of the slots overlaps less with the next row's.  What a part has beyond the
// slots that it keeps is read again, and not always found in L2: 6144 rows of 151936, half of which
// are only written, take 576 to 600 us on one CTA each and 507 on two; 1001 rows in f32, 623 of which count, 232 on
// one, 216 on two and 187 on four.
template <class T, bool S, bool G>
cudaError_t launch_ring(RowArgs a, bool dependent, cudaStream_t s) {
    using R = Roles<S, G>;
    cudaError_t e = ensure_smem(k_ring<T, S, G>, R::SMEM);
    if (e != cudaSuccess) return e;
    int cl = 1;
    double least = 0;
    for (int c = 1; c <= kCluster; c *= 2) {
        if (c > 1 && a.r.vocab < 1024u * c) break;  // no part may be empty
        int most = 1;
        e = clusters_at_once<T, S, G>(c, &most);
        if (e != cudaSuccess) return e;
        const double kib = (double)a.r.vocab * sizeof(T) / c / 1024;
        double row = !G ? 1.2 + 0.042 * kib : !S ? 1.3 + 0.047 * kib : sizeof(T) == 2 ? 1.5 + 0.055 * kib : 1.1 + (kib > 96 ? 0.05 : 0.04) * kib;
        if (S && G && kib > 170) row *= sizeof(T) == 4 ? 1.3 : 1.15;
        const double cost = (double)((a.r.n + most - 1) / most) * row;
        if (c == 1 || cost < least) cl = c, least = cost, a.units = (int)(a.r.n < most ? a.r.n : most);
    }
    a.log = log2_of(cl);
    a.own_order = !a.w.order && a.r.n > a.units && a.r.n <= kOwnOrder;
    const Launch l(cl, 1, dependent, dim3((unsigned)(a.units * cl)), R::THREADS, R::SMEM, s);
    return cudaLaunchKernelEx(&l.cfg, k_ring<T, S, G>, a);
}

template <class T, int THREADS, int V>
cudaError_t launch_short(RowArgs a, int cl, bool dependent, cudaStream_t s) {
    a.units = (int)a.r.n, a.log = log2_of(cl);
    const Launch l(cl, 1, dependent, dim3((unsigned)(a.r.n * cl)), THREADS, 0, s);
    return cudaLaunchKernelEx(&l.cfg, k_short<T, THREADS, V>, a);
}

template <class T, int V>
cudaError_t launch_rows(RowArgs a, bool dependent, cudaStream_t s) {
    const long long most = (long long)kSms * 64;  // warps that an SM has room for
    a.units = (int)(a.r.n < most ? a.r.n : most);
    const Launch l(1, 1, dependent, dim3((unsigned)(a.units + kRowWarps - 1) / kRowWarps), kRowWarps * 32, 0, s);
    return cudaLaunchKernelEx(&l.cfg, k_rows<T, V>, a);
}

// The kernel that a call's rows take: k_rows (32 threads) with so many vectors a
// lane, k_short with so many threads and CTAs to a row, or (0 threads) k_ring.
struct Path {
    int threads, cl, vectors;
};
// Short rows in registers, by a warp each if they are many (a CTA to a row is bound by the CTAs' starts,
// 2.6 ns a row): 262144 rows of 1000 in bf16 scored in 200 us and by a CTA each in 695, with gradients 299 and
// 803; 100000 rows of 2040, 128 and 275, 213 and 348; 50000 rows of 4080, 101 and 148, 189 and 211.  500 rows
// of 2040 take the same, 4800 rows of 4080 25 and 21; in f32 a lane holds no 16 vectors (50000 rows of 2040
// with gradients 235 and 181).  Longer ones too, by a CTA or a cluster, while these run at once, or
// (gradients of 16-bit types) in three rounds.  In us, so and by k_ring: 24 rows of 151936 in bf16
// with gradients 9.5 and 15, 120 rows 27 and 28, 200 rows 50 and 42; 24 rows scored 8.7 and 9.9, 48 rows
// 13 and 11; 5000 rows of 8000 63 and 32.  12 rows in f32 8.6 and 13, with gradients of 24 rows 15 and 15.
template <class T>
Path path_of(uint64_t n, uint32_t vocab, bool grad) {
    constexpr uint32_t N = Lane<T>::N;  // also what a row may be off its first vector
    const auto fits = [&](uint64_t elements, int cl) { return ((uint64_t)vocab + N + cl - 1) / cl + (cl > 1 ? 128 : 0) <= elements; };
    const auto few = [&](int cl, int threads) {
        const uint64_t at_once = kSms * 1024 / threads;
        return n * cl <= (grad && sizeof(T) == 2 ? 3 * at_once : at_once);
    };
    if (fits(32 * 4 * N, 1)) return {32, 1, 4};
    if (fits(32 * 8 * N, 1) && n > 8 * kSms) return {32, 1, 8};
    if (sizeof(T) == 2 && fits(32 * 16 * N, 1) && n > 128 * kSms) return {32, 1, 16};
    if (fits(128 * 4 * N, 1)) return {128, 1};
    if (fits(512 * 4 * N, 1)) return {few(1, 512) ? 512 : 0, 1};
    constexpr int THREADS = sizeof(T) == 2 ? 512 : 1024;
    int cl = 2;
    while (cl < kCluster && !fits(THREADS * 5 * N, cl)) cl *= 2;
    return {fits(THREADS * 5 * N, cl) && few(cl, THREADS) ? THREADS : 0, cl};
}

template <class T>
cudaError_t rows_of(RowArgs a, bool dependent, cudaStream_t s) {
    a.wait = dependent;
    const Path p = path_of<T>((uint64_t)a.r.n, a.r.vocab, a.o.grad != nullptr);
    if (p.threads == 32) {
        if (p.vectors == 4) return launch_rows<T, 4>(a, dependent, s);
        if (sizeof(T) == 4 || p.vectors == 8) return launch_rows<T, 8>(a, dependent, s);
        return launch_rows<T, sizeof(T) == 4 ? 8 : 16>(a, dependent, s);
    }
    if (p.threads == 128) return launch_short<T, 128, 4>(a, 1, dependent, s);
    if (p.threads && p.cl == 1) return launch_short<T, 512, 4>(a, 1, dependent, s);
    if (p.threads) return launch_short<T, sizeof(T) == 2 ? 512 : 1024, 5>(a, p.cl, dependent, s);
    if (!a.o.grad) return launch_ring<T, true, false>(a, dependent, s);
    return a.mode == KNOWN ? launch_ring<T, false, true>(a, dependent, s) : launch_ring<T, true, true>(a, dependent, s);
}

cudaError_t rows(const RowArgs& a, int dtype, bool dependent, cudaStream_t s) {
    return dtype == DT_F32 ? rows_of<float>(a, dependent, s) : dtype == DT_BF16 ? rows_of<__nv_bfloat16>(a, dependent, s) : rows_of<__half>(a, dependent, s);
}

// k_order, where the call needs it.
cudaError_t order(const RowArgs& a, cudaStream_t s) {
    if (!a.w.order && a.mode != POLICY) return cudaSuccess;
    unsigned ctas = 1;
    if (!a.w.order && a.r.n > 2 * kOrderRows) {
        ctas = (unsigned)std::min<long long>((a.r.n + kOrderRows - 1) / kOrderRows, kSms);
        const cudaError_t e = cudaMemsetAsync(a.w.counts, 0, (a.r.sequences + 1ull) * sizeof(int), s);
        if (e != cudaSuccess) return e;
    }
    k_order<<<ctas, 1024, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

// k_order costs a launch and 1 us for 1000 rows, whatever their length, so only long rows are put in order: those of
// 96 KiB with gradients (without known statistics), else of 256 KiB.  In us, in order and as they
// come, padded batches of which a third counts | all of which counts:
//   policy loss, 16-bit, 6144 rows of 20000: 86 89 | 157 153    50257: 171 181 | 315 309    151936: 468 485 | 856 851
//     100000 rows of 4100: 890 800 | 1775 1622    8000: 787 670 | 1252 1143    16000: 1070 948 | 1914 1806
//   policy loss, f32, 6144 rows of 20000: 140 136 | 188 187    32000: 207 207 | 303 303    151936: 873 948 | 1606 1591
//   scored, 16-bit, 6144 rows of 50257: 59 58 | 131 122    151936: 128 131 | 304 294    100000 rows of 8000: 302 205 | 572 475
//   preference loss, 16-bit, 6144 rows of 50257: 210 208 | 342 331    151936: 583 589 | 940 929
bool loss_orders(uint64_t n, uint32_t vocab, int dtype, bool grad, bool both) {
    const uint64_t row = (uint64_t)vocab * (dtype == DT_F32 ? 4 : 2), least = grad && !both ? 96 * 1024 : 256 * 1024;
    if (n <= (uint64_t)kOwnOrder || row < least) return false;
    const auto ring = [&](bool with) { return (dtype == DT_F32 ? path_of<float>(n, vocab, with) : path_of<__half>(n, vocab, with)).threads == 0; };
    return ring(grad) || (both && ring(false));
}

cudaError_t expired_waits_loss(unsigned long long* out) { return cudaMemcpyFromSymbol(out, g_expired_waits, sizeof(*out)); }

cudaError_t launch_logprobs(const LossRows& r, const LossWork& w, float* logprobs, int dtype, cudaStream_t s) {
    RowArgs a{};
    a.r = r, a.w = w, a.mode = LOGPROBS;
    a.o.logprobs = logprobs;
    KScope ks("token_logprobs", s, 1 + !!w.order);
    const cudaError_t e = order(a, s);
    return e == cudaSuccess ? rows(a, dtype, w.order, s) : e;
}

cudaError_t launch_logprobs_backward(const LossRows& r, const float* g, const LossWork& w, const LossOut& o, int dtype, cudaStream_t s) {
    RowArgs a{};
    a.r = r, a.w = w, a.o = o, a.g = g, a.mode = GIVEN;
    KScope ks("token_logprobs_backward", s, 1 + !!w.order);
    const cudaError_t e = order(a, s);
    return e == cudaSuccess ? rows(a, dtype, w.order, s) : e;
}

cudaError_t launch_policy(const LossRows& r, const PolicyTerms& p, const LossWork& w, const LossOut& o, int dtype, cudaStream_t s) {
    if (!r.n) return cudaMemsetAsync(o.loss, 0, sizeof(float), s);
    RowArgs a{};
    a.r = r, a.p = p, a.w = w, a.o = o, a.mode = POLICY;
    KScope ks("policy_loss", s, 2);
    const cudaError_t e = order(a, s);
    return e == cudaSuccess ? rows(a, dtype, true, s) : e;
}

cudaError_t launch_preference(const LossRows& r, const PreferTerms& p, const LossWork& w, const LossOut& o, int dtype, cudaStream_t s) {
    RowArgs a{};
    a.r = r, a.w = w, a.o = o, a.mode = LOGPROBS;
    a.o.grad = nullptr;
    KScope ks("preference_loss", s, 1 + (r.n > 0) + (r.n > 0 && o.grad) + !!w.order);
    cudaError_t e = order(a, s);
    if (e == cudaSuccess) e = r.n ? rows(a, dtype, w.order, s) : cudaMemsetAsync(w.ticket, 0, w.tickets * sizeof(unsigned), s);
    if (e == cudaSuccess) e = launch_dependent(1, k_pairs, dim3(r.sequences / 2), 512, 0, s, r, p, w, o);
    a.o.grad = o.grad, a.mode = KNOWN, a.backwards = 1;
    if (e == cudaSuccess && r.n && o.grad) e = rows(a, dtype, true, s);
    return e;
}

}  // namespace tsg
