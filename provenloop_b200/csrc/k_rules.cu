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
// row is split over a cluster of CTAs so that one row alone already uses
// several SMs, and the pick is reduced through distributed shared memory: no
// workspace, no atomics on global memory, hence nothing that two calls or
// two captured graphs could share.  A CTA starts the asynchronous copy of its
// segment of the row first and goes through the lists while it arrives.
//
// What the history and the biases say of the segment's tokens is kept in
// shared memory: two bitmaps (history, history or bias) read with every vector
// of logits, and for the tokens that the lists name one word each (bias entry
// + 1 << 20 | count), found by counting the bits before the token's.
#include <climits>

#include "launch.cuh"
#include "lowrank.cuh"
#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace tsg {

namespace {

constexpr int kThreads = 512;  // and 64 registers: two CTAs per SM, one's lists beside the other's stream
constexpr int kCluster = 8;
constexpr uint32_t kSegment = 19456;  // tokens per segment: an eighth of a vocabulary of 150 thousand in one go
constexpr uint32_t kWords = kSegment / 32;
constexpr uint32_t kBiasShift = 20;   // count below, bias entry + 1 above

struct Best {
    float z;
    uint32_t v;
};

// Ascending v only, so an equal z never replaces an earlier one; -inf is
// never taken.
__device__ __forceinline__ void take(Best& b, float z, uint32_t v) {
    if (z > b.z || (z != z && b.z == b.z)) b.z = z, b.v = v;
}

// Orders (z, lowest v) as an integer; 0 below everything.
__device__ __forceinline__ unsigned long long key_of(const Best& b) {
    if (b.v == UINT_MAX) return 0ull;
    const uint32_t u = __float_as_uint(b.z + 0.f);  // -0 counts as 0
    const uint32_t k = b.z != b.z ? UINT_MAX : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return (unsigned long long)k << 32 | (uint32_t)~b.v;
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

template <class T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
    T v[N];
};

__device__ __forceinline__ long long list_at(const void* p, int is64, long long i) {
    return is64 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int32_t*>(p)[i];
}

// Entries [from, to) of a list of token ids whose token lies in the segment:
// f(position in the segment, entry).
template <class F>
__device__ __forceinline__ void each_in(const void* list, int is64, long long at, uint32_t from, uint32_t to, uint32_t vocab, uint32_t shift,
                                        uint32_t size, F f) {
    uint32_t i = from + threadIdx.x;
    for (; i + 3 * kThreads < to; i += 4 * kThreads) {
        long long v[4];
#pragma unroll
        for (int q = 0; q < 4; q++) v[q] = list_at(list, is64, at + i + q * kThreads);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t p = (uint32_t)v[q] + shift;
            if ((unsigned long long)v[q] < vocab && p < size) f(p, i + q * kThreads);
        }
    }
    for (; i < to; i += kThreads) {
        const long long v = list_at(list, is64, at + i);
        const uint32_t p = (uint32_t)v + shift;
        if ((unsigned long long)v < vocab && p < size) f(p, i);
    }
}

__host__ __device__ constexpr size_t head_bytes() { return (3 * kWords + 4) * 4; }

// T: logits, O: output (written where a.out is not null).  The segment's
// tokens are addressed by p = v + head, where head is the row's offset from
// a 16-byte boundary in elements, so that vectors, bitmaps and words line up
// in rows of any alignment.  Dynamic shared memory: the bitmaps and the bit
// counts before their words, the named tokens' words, the segment's logits.
template <class T, class O>
__global__ void __launch_bounds__(kThreads, 2) k_rules(const RulesArgs a, uint32_t named) {
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ __align__(128) uint32_t smem[];
    __shared__ uint64_t arrived;
    __shared__ uint32_t dead;
    cg::cluster_group cluster = cg::this_cluster();
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

    uint32_t* seen = smem;
    uint32_t* touched = seen + kWords;
    uint32_t* before = touched + kWords;  // kWords + 4
    uint32_t* word = before + kWords + 4;
    T* buf = reinterpret_cast<T*>(word + named);
    if (threadIdx.x == 0) {
        mbar_init(&arrived, 1);
        dead = 0;
        fence_async_shared();
    }
    __syncthreads();
    // the whole vectors of [lo, hi) to buf, by one thread
    const auto fetch = [&](uint32_t lo, uint32_t hi) {
        const uint32_t from = lo == 0 && head ? VEC : lo, to = hi / VEC * VEC;
        const uint32_t bytes = to > from ? (to - from) * (uint32_t)sizeof(T) : 0;
        mbar_expect(&arrived, bytes);
        if (bytes) bulk_copy(smem_u32(buf + (from - lo)), x + from - head, bytes, &arrived);
    };
    if (threadIdx.x == 0 && first < last) fetch(first, min(last, first + kSegment));

    const uint32_t hist = a.tokens ? (uint32_t)max(0, min(a.lengths ? a.lengths[row] : INT_MAX, (int)a.token_cols)) : 0u;
    const uint32_t prompt = a.prompt_lengths ? (uint32_t)max(0, a.prompt_lengths[row]) : 0u;
    const uint32_t biases = a.bias_ids ? a.bias_cols : 0u;
    const long long tok0 = row * a.tokens_stride, bid0 = row * a.bias_ids_stride, bval0 = row * a.bias_values_stride;
    const float rho = a.repetition ? a.repetition[row] : 1.f;
    const float freq = a.frequency ? a.frequency[row] : 0.f;
    const float pres = a.presence ? a.presence[row] : 0.f;
    const uint32_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const uint32_t words = (a.vocab + 31) / 32;
    const bool lists = hist || biases;

    Best best{-INFINITY, UINT_MAX};
    uint32_t phase = 0;
    for (uint32_t lo = first; lo < last; lo += kSegment, phase ^= 1) {
        const uint32_t hi = min(last, lo + kSegment), size = hi - lo, shift = head - lo;
        if (lo != first) {
            __syncthreads();
            if (threadIdx.x == 0) {
                fence_async_shared();
                fetch(lo, hi);
            }
        }
        if (lists) {
            for (uint32_t i = threadIdx.x; i < 2 * kWords; i += kThreads) smem[i] = 0u;
            __syncthreads();
            each_in(a.bias_ids, a.bias64, bid0, 0, biases, a.vocab, shift, size, [&](uint32_t p, uint32_t) { atomicOr(touched + p / 32, 1u << p % 32); });
            each_in(a.tokens, a.tokens64, tok0, 0, hist, a.vocab, shift, size, [&](uint32_t p, uint32_t) {
                atomicOr(touched + p / 32, 1u << p % 32);
                atomicOr(seen + p / 32, 1u << p % 32);
            });
            const uint32_t most = min(named, size);
            for (uint32_t i = threadIdx.x; i < most; i += kThreads) word[i] = 0u;
            __syncthreads();
            if (threadIdx.x < 32) {
                // bits before each word: 19 words a lane
                constexpr uint32_t kEach = kWords / 32;
                static_assert(kWords % 32 == 0, "a lane has whole words");
                uint32_t sum = 0;
                for (uint32_t i = 0; i < kEach; i++) {
                    before[threadIdx.x * kEach + i] = sum;
                    sum += __popc(touched[threadIdx.x * kEach + i]);
                }
                uint32_t incl = sum;
#pragma unroll
                for (int q = 1; q < 32; q <<= 1) {
                    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, q);
                    if (threadIdx.x >= q) incl += y;
                }
                for (uint32_t i = 0; i < kEach; i++) before[threadIdx.x * kEach + i] += incl - sum;
            }
            __syncthreads();
        }
        const auto slot = [&](uint32_t p) { return before[p / 32] + __popc(touched[p / 32] & ((1u << p % 32) - 1)); };
        if (lists) {
            each_in(a.bias_ids, a.bias64, bid0, 0, biases, a.vocab, shift, size,
                    [&](uint32_t p, uint32_t i) { atomicMax(word + slot(p), (i + 1) << kBiasShift); });
            __syncthreads();
            each_in(a.tokens, a.tokens64, tok0, prompt, hist, a.vocab, shift, size, [&](uint32_t p, uint32_t) { atomicAdd(word + slot(p), 1u); });
            __syncthreads();
        }
        mbar_wait(&arrived, phase, &dead);
        for (uint32_t p0 = lo + threadIdx.x * VEC; p0 < hi; p0 += kThreads * VEC) {
            const bool whole = p0 >= head && p0 + VEC <= hi;
            Pack<T, VEC> in;
            if (whole) {
                in = *reinterpret_cast<const Pack<T, VEC>*>(buf + (p0 - lo));
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++)
                    if (p0 + i >= head && p0 + i < hi) in.v[i] = x[p0 + i - head];
            }
            // the vector's bits; a group of VEC <= 8 lies in one word, since lo is a multiple of 128
            const uint32_t q = p0 - lo;
            uint32_t tb = 0, mb = UINT_MAX;
            if (lists) tb = touched[q / 32] >> q % 32;
            if (mask) {
                // token v0 of the vector's first element; v0 < 0 in a row's first vector
                const long long v0 = (long long)p0 - head;
                const long long w = v0 >> 5;
                const uint32_t m0 = w >= 0 ? mask[w] : 0u;
                const uint32_t m1 = head && w + 1 < words ? mask[w + 1] : 0u;
                mb = __funnelshift_r(m0, m1, (uint32_t)(v0 & 31));
            }
            float z[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) z[i] = load_f(in.v[i]);
            constexpr uint32_t kAll = (1u << VEC) - 1;
            if (tb & kAll) {
                const uint32_t sb = seen[q / 32] >> q % 32;
#pragma unroll
                for (int i = 0; i < VEC; i++)
                    if (tb >> i & 1) {
                        const uint32_t c = word[slot(q + i)];
                        const uint32_t n = c & ((1u << kBiasShift) - 1), b = c >> kBiasShift;
                        if (sb >> i & 1) z[i] = z[i] > 0.f ? __fdiv_rn(z[i], rho) : __fmul_rn(z[i], rho);
                        if (n) z[i] = __fsub_rn(__fsub_rn(z[i], __fmul_rn(freq, (float)n)), pres);
                        if (b) z[i] = __fadd_rn(z[i], a.bias_values[bval0 + b - 1]);
                    }
            }
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                if (!(mb >> i & 1)) z[i] = -INFINITY;
                if (whole || (p0 + i >= head && p0 + i < hi)) take(best, z[i], p0 + i - head);
            }
            if (out) {
                Pack<O, VEC> res;
#pragma unroll
                for (int i = 0; i < VEC; i++) store_f(&res.v[i], z[i]);
                if (whole && out_vec) {
                    if constexpr (sizeof(O) * VEC > 16) {
                        const Pack<O, VEC / 2>* r2 = reinterpret_cast<const Pack<O, VEC / 2>*>(&res);
                        Pack<O, VEC / 2>* o2 = reinterpret_cast<Pack<O, VEC / 2>*>(out + (p0 - head));
                        o2[0] = r2[0], o2[1] = r2[1];
                    } else {
                        *reinterpret_cast<Pack<O, VEC>*>(out + (p0 - head)) = res;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; i++)
                        if (p0 + i >= head && p0 + i < hi) out[p0 + i - head] = res.v[i];
                }
            }
        }
    }

    unsigned long long key = key_of(best);
#pragma unroll
    for (int q = 16; q; q >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, q));
    __shared__ unsigned long long warp_key[kThreads / 32], cta_key[kCluster];
    if ((threadIdx.x & 31) == 0) warp_key[threadIdx.x >> 5] = key;
    __syncthreads();
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
    // words for as many tokens as the lists can name in a segment
    const uint64_t most = (uint64_t)(a.tokens ? a.token_cols : 0) + (a.bias_ids ? a.bias_cols : 0);
    const uint32_t span = ((a.vocab + 16 + kCluster - 1) / kCluster + 127) / 128 * 128, segment = span < kSegment ? span : kSegment;
    const uint32_t named = (uint32_t)((most < segment ? most : segment) + 31) / 32 * 32;
    const size_t smem = head_bytes() + (size_t)named * 4 + (size_t)segment * sizeof(T);
    const cudaError_t e = ensure_smem(k_rules<T, O>, smem > 48 * 1024 ? smem : smem + 48 * 1024);
    if (e != cudaSuccess) return e;
    KScope ks("logit_rules", s);
    return launch_cl(kCluster, k_rules<T, O>, dim3((unsigned)(a.n * kCluster)), kThreads, smem, s, a, named);
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
