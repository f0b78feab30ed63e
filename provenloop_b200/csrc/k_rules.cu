// k_rules.cu -- penalties, biases and a grammar mask on next-token logits,
// with the greedy pick, in one pass.
//
// Row i, token v with logit x, in f32 and in this order:
//   z = x
//   v is in the history:             z = z > 0 ? z / repetition : z * repetition
//   v occurs c > 0 times after the
//   prompt part of the history:      z = z - frequency * c - presence
//   v is in the row's bias list:     z = z + bias (the last entry of v counts)
//   v's mask bit is 0:               z = -inf, whatever it was
//   pick = the lowest v of the greatest z (NaN is the greatest, as in
//   torch.argmax); -1 where every z is -inf.
//
// The bound is the logits' traffic: each is read once and written once.  A
// row is split over a cluster of one to eight CTAs, so that a few rows already
// use every SM, and the pick is reduced through distributed shared memory: no
// workspace, no atomics on global memory, hence nothing that two calls or
// two captured graphs could share.  A CTA takes its part of the row in
// segments, whose asynchronous copies run two ahead of it, and goes through
// the lists (held in registers) while they arrive.
//
// What the lists say is kept in shared memory: a bitmap of the tokens that
// they name, and for those one word each, found by counting the bits before
// the token's.  The named tokens are computed first, from the lists' side; the
// stream over the segments takes them, like masked tokens, as -inf, and they
// are written over it in the end.  The stream works on pairs of 16-bit values
// and on four vectors a thread at a time, and compares them with the greatest
// value that the CTA has seen, so that hardly a warp has to look closer.
//
// What bounds it now: the lists, which keep the stream waiting for a third of
// the time (their loads queue behind the first segments), and half of the
// issue slots.  64 rows of 151936 in f32 with every rule take 27 us (2.9 TB/s),
// 256 rows in bf16 of which only the picks are wanted 35 us (2.2 TB/s; 2 us more
// when each thread compared with its own greatest), one row with 4096 tokens
// of history 12 to 14 us.
#include <climits>

#include "launch.cuh"
#include "lowrank.cuh"
#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace tsg {

namespace {

constexpr int kThreads = 512;  // and 64 registers: two CTAs per SM, one's lists beside the other's stream
constexpr int kCluster = 8;
// Tokens per segment: 32 KiB of logits, of which two CTAs on an SM hold two
// each.
template <class T>
constexpr uint32_t kSegment = 32768 / sizeof(T);
// Tokens whose lists are held at a time, or, for lists that name more tokens
// than fit beside them, half a segment.
constexpr uint32_t kBlock = 262144;
constexpr uint32_t kMaxSmem = 226 * 1024;
constexpr uint32_t kPrompt = 1u << 31;  // of a named token's word: it is in the prompt; the count behind it below

struct Best {
    float z;
    uint32_t v;
};

// The greater of b and (z, v), of equal ones the lower v; -inf is never taken.
__device__ __forceinline__ void take_any(Best& b, float z, uint32_t v) {
    const bool nz = z != z, nb = b.z != b.z;
    if (nz ? (!nb || v < b.v) : (!nb && (z > b.z || (z == b.z && v < b.v && z != -INFINITY)))) b.z = z, b.v = v;
}

// Orders values as integers, NaN above all, and back.
__device__ __forceinline__ uint32_t order_of(float z) {
    const uint32_t u = __float_as_uint(z + 0.f);  // -0 counts as 0
    return z != z ? UINT_MAX : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) && k != UINT_MAX ? k & 0x7fffffffu : k == UINT_MAX ? k : ~k); }

// Orders (z, lowest v) as an integer; 0 below everything.
__device__ __forceinline__ unsigned long long key_of(const Best& b) {
    if (b.v == UINT_MAX) return 0ull;
    return (unsigned long long)order_of(b.z) << 32 | (uint32_t)~b.v;
}

template <class T>
__device__ __forceinline__ float load_f(T v);
template <>
__device__ __forceinline__ float load_f(float v) { return v; }
template <>
__device__ __forceinline__ float load_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float load_f(__half v) { return __half2float(v); }

__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f(__half* p, float v) { *p = __float2half_rn(v); }

constexpr uint32_t kNone = UINT_MAX;

__device__ __forceinline__ long long list_at(const void* p, int is64, long long i) {
    return is64 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int32_t*>(p)[i];
}

// A token id, kNone outside the vocabulary.
__device__ __forceinline__ uint32_t place(long long v, uint32_t vocab) { return (unsigned long long)v < vocab ? (uint32_t)v : kNone; }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Eight 16-bit or four 32-bit logits: selection, maximum, one element.
template <class T>
struct Vec;
template <>
struct Vec<float> {
    static __device__ __forceinline__ void select(uint4& x, uint32_t ok) {
        constexpr uint32_t low = 0xff800000u;
        x.x = ok & 1 ? x.x : low, x.y = ok & 2 ? x.y : low, x.z = ok & 4 ? x.z : low, x.w = ok & 8 ? x.w : low;
    }
    static __device__ __forceinline__ float top(const uint4& x) {
        return max_nan(max_nan(__uint_as_float(x.x), __uint_as_float(x.y)), max_nan(__uint_as_float(x.z), __uint_as_float(x.w)));
    }
    static __device__ __forceinline__ float top4(const uint4 (&x)[4]) {
        return max_nan(max_nan(top(x[0]), top(x[1])), max_nan(top(x[2]), top(x[3])));
    }
};
template <class T>
struct Vec16 {
    static constexpr uint32_t kLow = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    // Four bits to the sign bits of a word's bytes, by one product without
    // carries, and each sign over half a word.
    static __device__ __forceinline__ void select(uint4& x, uint32_t ok) {
        const uint32_t lo = (ok & 0x0f) * 0x10204080u, hi = (ok & 0xf0) * 0x01020408u;
        const auto spread = [](uint32_t signs, uint32_t bytes) {
            uint32_t m;
            asm("prmt.b32 %0, %1, 0, %2;" : "=r"(m) : "r"(signs), "r"(bytes));
            return m;
        };
        const uint32_t m0 = spread(lo, 0x9988u), m1 = spread(lo, 0xbbaau), m2 = spread(hi, 0x9988u), m3 = spread(hi, 0xbbaau);
        x.x = (x.x & m0) | (kLow & ~m0), x.y = (x.y & m1) | (kLow & ~m1);
        x.z = (x.z & m2) | (kLow & ~m2), x.w = (x.w & m3) | (kLow & ~m3);
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t pair(const uint4& x) { return max2(max2(x.x, x.y), max2(x.z, x.w)); }
    static __device__ __forceinline__ float single(uint32_t m) {
        const T* h = reinterpret_cast<const T*>(&m);
        return max_nan(load_f(h[0]), load_f(h[1]));
    }
    static __device__ __forceinline__ float top(const uint4& x) { return single(pair(x)); }
    static __device__ __forceinline__ float top4(const uint4 (&x)[4]) {
        return single(max2(max2(pair(x[0]), pair(x[1])), max2(pair(x[2]), pair(x[3]))));
    }
};
template <>
struct Vec<__half> : Vec16<__half> {};
template <>
struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16> {};

// Where a kernel's dynamic shared memory has what, in 32-bit words.
struct RulesLayout {
    uint32_t segment, block, buffers, bits, before, count, bias, pos, ok, ok_words, buf, bytes;
    // span: tokens of a CTA's part of the row; most: entries of its lists
    RulesLayout(uint32_t span, uint32_t block_, uint64_t most, bool biases, uint32_t segment_, uint32_t size, uint32_t buffers_) {
        segment = segment_, block = span < block_ ? span : block_, buffers = buffers_;
        const uint32_t groups = (block + 127) / 128, named = (uint32_t)((most < block ? most : block) + 31) / 32 * 32;
        uint32_t at = 0;
        bits = at, at += named ? groups * 4 : 0;  // groups of 128 tokens
        before = at, at += named ? (groups + 3) / 4 * 4 : 0;
        count = at, at += named;
        bias = at, at += biases ? named : 0;
        pos = at, at += named;
        const uint32_t held = span < segment ? span : segment;  // a multiple of 128
        ok_words = held / 32;  // of one segment
        ok = at, at += ok_words * 2;
        buf = at = (at + 31) / 32 * 32;
        bytes = at * 4 + held * size * buffers;
    }
};

// T: logits, O: output (written where a.out is not null).  The row's tokens
// are addressed by p = v + head, where head is the row's offset from a 16-byte
// boundary in elements, so that vectors and bitmaps line up in rows of any
// alignment.  A CTA's part of the row goes in blocks of at most kBlock tokens,
// and these in segments.
template <class T, class O>
__global__ void __launch_bounds__(kThreads, 2) k_rules(const RulesArgs a, const RulesLayout l) {
    constexpr uint32_t VEC = 16 / sizeof(T), kPer = (kSegment<T> / 32 + kThreads - 1) / kThreads;
    constexpr int kHeld = 8;  // entries of the history that a thread keeps in registers
    extern __shared__ __align__(128) uint32_t smem[];
    __shared__ uint64_t arrived[2];
    __shared__ uint32_t dead, warp_bits[kThreads / 32], floor_of;  // the CTA's greatest before this segment
    cg::cluster_group cluster = cg::this_cluster();
    cluster_arrive();  // waited for before the first access to another CTA's shared memory
    const int rank = (int)cluster.block_rank(), cl = (int)cluster.num_blocks();
    const long long row = blockIdx.x / cl;
    const T* x = static_cast<const T*>(a.logits) + row * a.logits_stride;
    O* out = a.out ? static_cast<O*>(a.out) + row * a.out_stride : nullptr;
    const uint32_t head = (uint32_t)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    const uint32_t end = head + a.vocab;
    // whole vectors of output where the output row has the same phase
    const bool out_vec = out && reinterpret_cast<uintptr_t>(out) % 16 == head * sizeof(O) % 16;
    const uint32_t span = ((end + cl - 1) / cl + 127) / 128 * 128;
    const uint32_t first = min(end, rank * span), last = min(end, first + span);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    uint32_t *bits = smem + l.bits, *before = smem + l.before, *count = smem + l.count, *bias = smem + l.bias, *pos = smem + l.pos,
             *okw = smem + l.ok;
    T* bufs = reinterpret_cast<T*>(smem + l.buf);
    // segment s's whole vectors to one of the two buffers, by one thread
    const auto fetch = [&](uint32_t s) {
        const uint32_t lo = first + s * l.segment;
        if (lo >= last) return;
        const uint32_t hi = min(last, lo + l.segment), from = lo == 0 && head ? VEC : lo, to = hi / VEC * VEC;
        const uint32_t bytes = to > from ? (to - from) * (uint32_t)sizeof(T) : 0;
        const uint32_t at = s & (l.buffers - 1);
        mbar_expect(&arrived[at], bytes);
        if (bytes) bulk_copy(smem_u32(bufs + at * l.segment + (from - lo)), x + from - head, bytes, &arrived[at]);
    };
    if (threadIdx.x == 0) {
        mbar_init(&arrived[0], 1);
        mbar_init(&arrived[1], 1);
        dead = 0;
        floor_of = order_of(-INFINITY);
        fence_async_shared();
        fetch(0);
    }

    const uint32_t hist = a.tokens ? (uint32_t)max(0, min(a.lengths ? a.lengths[row] : INT_MAX, (int)a.token_cols)) : 0u;
    const uint32_t prompt = a.prompt_lengths ? (uint32_t)max(0, a.prompt_lengths[row]) : 0u;
    const uint32_t biases = a.bias_ids ? a.bias_cols : 0u;
    const long long tok0 = row * a.tokens_stride, bid0 = row * a.bias_ids_stride, bval0 = row * a.bias_values_stride;
    const float rho = a.repetition ? a.repetition[row] : 1.f;
    const float freq = a.frequency ? a.frequency[row] : 0.f;
    const float pres = a.presence ? a.presence[row] : 0.f;
    const uint32_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const uint32_t words = (a.vocab + 31) / 32;
    const bool lists = hist || biases, plain = !lists && !mask;
    // the mask's bits of the 32 tokens from p on, a multiple of 32; others 0
    const auto mask_at = [&](uint32_t p) {
        const long long v0 = (long long)p - head, w = v0 >> 5;  // v0 < 0 in a misaligned row's first word
        const uint32_t m0 = w >= 0 && w < words ? mask[w] : 0u, m1 = head && w + 1 < words ? mask[w + 1] : 0u;
        return __funnelshift_r(m0, m1, (uint32_t)(v0 & 31));
    };

    // the first entries of the lists, and the mask's words of the next segment
    uint32_t held[kHeld], held_bias = kNone, next_mask[kPer];
#pragma unroll
    for (int q = 0; q < kHeld; q++) held[q] = kNone;
    if (mask) {
#pragma unroll
        for (uint32_t q = 0; q < kPer; q++) next_mask[q] = mask_at(first + (threadIdx.x + q * kThreads) * 32);
    }
    if (a.tokens) {  // without waiting for the length
        long long v[kHeld];
#pragma unroll
        for (int q = 0; q < kHeld; q++) v[q] = list_at(a.tokens, a.tokens64, tok0 + min(threadIdx.x + q * kThreads, a.token_cols - 1));
#pragma unroll
        for (int q = 0; q < kHeld; q++)
            if (threadIdx.x + q * kThreads < hist) held[q] = place(v[q], a.vocab);
    }
    if (threadIdx.x < biases) held_bias = place(list_at(a.bias_ids, a.bias64, bid0 + threadIdx.x), a.vocab);
    // the second segment's copy starts once the lists' loads are through, which
    // would queue behind it (28.3 and 26.7 us for 64 rows with every rule)
    if (threadIdx.x == 0 && l.buffers == 2) {
        asm volatile("" ::"r"(held[0]));
        fetch(1);
    }

    Best named{-INFINITY, UINT_MAX}, best{-INFINITY, UINT_MAX};
    // this thread's first vector with the greatest element; which it is is found in the end
    float top = -INFINITY;
    uint32_t top_at = kNone, s = 0;  // s: segment
    uint4 top_z = make_uint4(0, 0, 0, 0);
    for (uint32_t blk = first; blk < last; blk += l.block) {
        const uint32_t blk_end = min(last, blk + l.block), size = blk_end - blk, groups = (size + 127) / 128;
        uint32_t total = 0;  // named tokens
        if (lists) {
            // f(position in the block, entry) for the block's entries of a list
            const auto each_token = [&](auto f) {
                if (!hist) return;
#pragma unroll
                for (int q = 0; q < kHeld; q++)
                    if (held[q] != kNone && held[q] + head - blk < size) f(held[q] + head - blk, threadIdx.x + q * kThreads);
                for (uint32_t i = threadIdx.x + kHeld * kThreads; i < hist; i += kThreads) {
                    const uint32_t v = place(list_at(a.tokens, a.tokens64, tok0 + i), a.vocab);
                    if (v != kNone && v + head - blk < size) f(v + head - blk, i);
                }
            };
            const auto each_bias = [&](auto f) {
                if (held_bias != kNone && held_bias + head - blk < size) f(held_bias + head - blk, threadIdx.x);
                for (uint32_t i = threadIdx.x + kThreads; i < biases; i += kThreads) {
                    const uint32_t v = place(list_at(a.bias_ids, a.bias64, bid0 + i), a.vocab);
                    if (v != kNone && v + head - blk < size) f(v + head - blk, i);
                }
            };
            const auto slot = [&](uint32_t p) {
                const uint4 w = reinterpret_cast<const uint4*>(bits)[p / 128];
                const uint32_t q = p / 32 % 4, own = q == 0 ? w.x : q == 1 ? w.y : q == 2 ? w.z : w.w;
                return before[p / 128] + (q > 0 ? __popc(w.x) : 0) + (q > 1 ? __popc(w.y) : 0) + (q > 2 ? __popc(w.z) : 0) +
                       __popc(own & ((1u << p % 32) - 1));
            };
            if (blk != first) __syncthreads();
            // bits, before, count and bias lie one behind the other
            for (uint32_t i = threadIdx.x; i < (l.pos - l.bits) / 4; i += kThreads) reinterpret_cast<uint4*>(bits)[i] = make_uint4(0u, 0u, 0u, 0u);
            __syncthreads();
            each_bias([&](uint32_t p, uint32_t) { atomicOr(bits + p / 32, 1u << p % 32); });
            each_token([&](uint32_t p, uint32_t) { atomicOr(bits + p / 32, 1u << p % 32); });
            __syncthreads();
            // bits before each group; a thread has neighbouring ones
            const uint32_t each = (groups + kThreads - 1) / kThreads, g0 = threadIdx.x * each, g1 = min(groups, g0 + each);
            uint32_t sum = 0;
            for (uint32_t g = g0; g < g1; g++) {
                const uint4 w = reinterpret_cast<const uint4*>(bits)[g];
                before[g] = sum;
                sum += __popc(w.x) + __popc(w.y) + __popc(w.z) + __popc(w.w);
            }
            uint32_t incl = sum;
#pragma unroll
            for (int q = 1; q < 32; q <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, incl, q);
                if (lane >= q) incl += y;
            }
            if (lane == 31) warp_bits[warp] = incl;
            __syncthreads();
            uint32_t below = incl - sum;
#pragma unroll
            for (int q = 0; q < kThreads / 32; q++) below += q < warp ? warp_bits[q] : 0u, total += warp_bits[q];
            for (uint32_t g = g0; g < g1; g++) before[g] += below;
            __syncthreads();
            each_bias([&](uint32_t p, uint32_t i) {
                const uint32_t at = slot(p);
                pos[at] = p;
                atomicMax(bias + at, i + 1);
            });
            each_token([&](uint32_t p, uint32_t i) {
                const uint32_t at = slot(p);
                pos[at] = p;
                if (i < prompt) atomicOr(count + at, kPrompt);
                else atomicAdd(count + at, 1u);
            });
            __syncthreads();
            // the named tokens' results, kept as bits in place of their counts
            for (uint32_t i = threadIdx.x; i < total; i += kThreads) {
                const uint32_t p = blk + pos[i], v = p - head;
                float z = load_f(x[v]);
                const uint32_t c = count[i], n = c & ~kPrompt, b = biases ? bias[i] : 0u;
                const uint32_t m = mask ? mask[v / 32] >> v % 32 : 1u;
                const float add = b ? a.bias_values[bval0 + b - 1] : 0.f;
                if (c) z = z > 0.f ? __fdiv_rn(z, rho) : __fmul_rn(z, rho);
                if (n) z = __fsub_rn(__fsub_rn(z, __fmul_rn(freq, (float)n)), pres);
                if (b) z = __fadd_rn(z, add);
                if (!(m & 1)) z = -INFINITY;
                take_any(named, z, v);
                count[i] = __float_as_uint(z);
            }
        }
        // which tokens of the segment from `lo` on the stream takes as they are,
        // and the mask's words of the segment behind it
        const auto prepare = [&](uint32_t lo, uint32_t* to) {
            const uint32_t used = (min(blk_end, lo + l.segment) - lo + 31) / 32;
#pragma unroll
            for (uint32_t q = 0; q < kPer; q++) {
                const uint32_t i = threadIdx.x + q * kThreads;
                if (i < used) to[i] = (mask ? next_mask[q] : UINT_MAX) & ~(lists ? bits[(lo - blk) / 32 + i] : 0u);
            }
            if (mask && lo + l.segment < last) {
#pragma unroll
                for (uint32_t q = 0; q < kPer; q++) next_mask[q] = mask_at(lo + l.segment + (threadIdx.x + q * kThreads) * 32);
            }
        };
        if (!plain) prepare(blk, okw + (s & 1) * l.ok_words);
        __syncthreads();  // also, every named logit has been read: out may be logits itself
        for (uint32_t lo = blk; lo < blk_end; lo += l.segment, s++) {
            const uint32_t hi = min(blk_end, lo + l.segment), at = s & (l.buffers - 1);
            const T* buf = bufs + at * l.segment;
            const uint32_t* ok_bits = okw + (s & 1) * l.ok_words;
            mbar_wait(&arrived[at], s / l.buffers & 1, &dead);
            // what all threads have seen in earlier segments, at lower ids: once a
            // few segments are through, hardly a warp finds a greater one
            const float below = value_of(*const_cast<volatile uint32_t*>(&floor_of));
            if (!(top >= below) && top == top) top = below, top_at = kNone;
            const uint32_t top_was = top_at;
            const auto see = [&](const uint4& z, uint32_t v) {
                const float m = Vec<T>::top(z);
                if (!(m <= top) && top == top) top = m, top_at = v, top_z = z;  // a NaN, once there, stays
            };
            const auto put = [&](const uint4& z, uint32_t v) {
                const T* e = reinterpret_cast<const T*>(&z);
                O* to = out + v;
                if (!out_vec) {
#pragma unroll
                    for (uint32_t i = 0; i < VEC; i++) store_f(to + i, load_f(e[i]));
                } else if constexpr (std::is_same<T, O>::value) {
                    *reinterpret_cast<uint4*>(to) = z;
                } else {
                    float4 f[VEC / 4];
#pragma unroll
                    for (uint32_t i = 0; i < VEC / 4; i++)
                        f[i] = make_float4(load_f(e[4 * i]), load_f(e[4 * i + 1]), load_f(e[4 * i + 2]), load_f(e[4 * i + 3]));
#pragma unroll
                    for (uint32_t i = 0; i < VEC / 4; i++) reinterpret_cast<float4*>(to)[i] = f[i];
                }
            };
            constexpr uint32_t kStep = kThreads * VEC;
            uint32_t q = threadIdx.x * VEC;
            // four vectors a thread at once where they lie in the segment: one
            // comparison with the greatest so far, which seldom finds a greater
            const uint32_t whole = lo >= head ? (hi - lo) / (4 * kStep) * (4 * kStep) : 0u;
            for (; q < whole; q += 4 * kStep) {
                uint4 z[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) z[j] = *reinterpret_cast<const uint4*>(buf + q + j * kStep);
                if (!plain) {
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) Vec<T>::select(z[j], ok_bits[q / 32 + j * (kStep / 32)] >> q % 32);
                }
                if (!(Vec<T>::top4(z) <= top) && top == top) {
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) see(z[j], lo + q + j * kStep - head);
                }
                if (out) {
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) put(z[j], lo + q + j * kStep - head);
                }
            }
            for (; q < hi - lo; q += kStep) {
                const uint32_t p0 = lo + q;
                // the vector's bits: VEC <= 8 of them lie in one word
                const uint32_t ok = plain ? UINT_MAX : ok_bits[q / 32] >> q % 32;
                if (p0 >= head && p0 + VEC <= hi) {
                    uint4 z = *reinterpret_cast<const uint4*>(buf + q);
                    if (!plain) Vec<T>::select(z, ok);
                    see(z, p0 - head);
                    if (out) put(z, p0 - head);
                } else {
                    // the row's ends, which did not come with the copy
#pragma unroll 1
                    for (uint32_t i = 0; i < VEC; i++) {
                        if (p0 + i < head || p0 + i >= hi) continue;
                        const uint32_t v = p0 + i - head;
                        const float z = ok >> i & 1 ? load_f(x[v]) : -INFINITY;
                        take_any(best, z, v);
                        if (out) store_f(out + v, z);
                    }
                }
            }
            const uint32_t new_floor = top_at != top_was ? order_of(top) : 0u;
            if (!plain && hi < blk_end) prepare(hi, okw + (~s & 1) * l.ok_words);
            __syncthreads();
            if (new_floor) atomicMax(&floor_of, new_floor);
            if (threadIdx.x == 0) {
                fence_async_shared();  // what was read from the buffer, before the next copy into it
                fetch(s + l.buffers);
            }
        }
        if (out)
            for (uint32_t i = threadIdx.x; i < total; i += kThreads) store_f(out + (blk + pos[i] - head), __uint_as_float(count[i]));
    }

    if (top_at != kNone) {
        const T* e = reinterpret_cast<const T*>(&top_z);
#pragma unroll
        for (uint32_t i = 0; i < VEC; i++) take_any(best, load_f(e[i]), top_at + i);
    }
    unsigned long long key = max(key_of(best), key_of(named));
#pragma unroll
    for (int q = 16; q; q >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, q));
    __shared__ unsigned long long warp_key[kThreads / 32], cta_key[kCluster];
    if ((threadIdx.x & 31) == 0) warp_key[threadIdx.x >> 5] = key;
    __syncthreads();
    cluster_wait();  // the other CTAs have started
    if (threadIdx.x < 32) {
        key = threadIdx.x < kThreads / 32 ? warp_key[threadIdx.x] : 0ull;
#pragma unroll
        for (int q = 16; q; q >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, q));
        if (threadIdx.x == 0) *cluster.map_shared_rank(&cta_key[rank], 0) = key;
    }
    cluster.sync();
    if (rank == 0 && threadIdx.x == 0 && a.pick) {
        for (int i = 1; i < cl; i++) key = max(key, cta_key[i]);
        a.pick[row] = key == 0ull ? -1ll : (long long)(uint32_t)~(uint32_t)key;
    }
}

template <class T, class O>
cudaError_t launch_one(const RulesArgs& a, cudaStream_t s) {
    // CTAs to a row: the fewest rounds of two CTAs per SM, each with its share of
    // the row and a twentieth of a row for starting and for the pick
    int dev = 0, sms = 1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    int cl = 1;
    double least = 0;
    for (int c = 1; c <= kCluster; c *= 2) {
        const double cost = (double)((a.n * c + 2 * sms - 1) / (2 * sms)) * (1.0 / c + 0.05);
        if (c == 1 || cost < least) cl = c, least = cost;
    }
    const uint64_t most = (uint64_t)(a.tokens ? a.token_cols : 0) + (a.bias_ids ? a.bias_cols : 0);
    const uint32_t span = ((a.vocab + 16 + cl - 1) / cl + 127) / 128 * 128;
    RulesLayout l(span, kBlock, most, a.bias_ids != nullptr, kSegment<T>, sizeof(T), span > kSegment<T> ? 2 : 1);
    if (l.bytes > kMaxSmem) l = RulesLayout(span, kSegment<T> / 2, most, a.bias_ids != nullptr, kSegment<T> / 2, sizeof(T), 1);
    e = ensure_smem(k_rules<T, O>, l.bytes + 1024);  // the pick's shared memory is beside it
    if (e != cudaSuccess) return e;
    KScope ks("logit_rules", s);
    return launch_cl(cl, k_rules<T, O>, dim3((unsigned)(a.n * cl)), kThreads, l.bytes, s, a, l);
}

}  // namespace

cudaError_t expired_waits_rules(unsigned long long* out) { return cudaMemcpyFromSymbol(out, g_expired_waits, sizeof(*out)); }

cudaError_t launch_rules(const RulesArgs& a, int dtype, int out_dtype, cudaStream_t s) {
    if (dtype == DT_F32) return launch_one<float, float>(a, s);
    if (dtype == DT_BF16)
        return out_dtype == DT_F32 ? launch_one<__nv_bfloat16, float>(a, s) : launch_one<__nv_bfloat16, __nv_bfloat16>(a, s);
    return out_dtype == DT_F32 ? launch_one<__half, float>(a, s) : launch_one<__half, __half>(a, s);
}

}  // namespace tsg
