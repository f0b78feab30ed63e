// k_clip.cu -- norms over many tensors, for each group of a stack, and the
// clipping of the tensors by them.
//
// Group e has the e-th part of every tensor:
//   norm_e = sqrt(sum over its elements of g^2)
//   out = g min(1, max_e / norm_e), rounded once
// A group whose norm is not finite is left as it is.
//
// The bound is the tensors' traffic: each element is read for the norm, and
// read and written for the clipping.  Two launches: the sums of squares of chunks of
// parts, and the scaling, which goes backwards over the chunks, since the latest
// are still in L2.  Every CTA of the second one adds up its group's sums by itself
// where there are few; where there are many, a launch between the two does.
// 295M elements in f32 (2.4 GB with the results, 3.5 GB with the second reading) take 576 us, 6.2 TB/s; the 112
// gradients of 28 layers, 6.5M elements in bf16, 15 us.
//
// A chunk's sum of squares is a 64-bit value of its own, and a group's are
// added in an order that depends on the sizes alone.
#include "launch.cuh"
#include "sm100.cuh"
#include "train.cuh"

namespace tsg {

namespace {

constexpr int kThreads = 512;
// Bytes of a part that a CTA takes: as much as its threads load at a time, or
// a quarter of that where this gives less than two CTAs to an SM (one layer's four gradients,
// 0.9 MB: 6.5 us, in larger chunks 8.6).
constexpr uint32_t kChunk = 32768, kSmallChunk = 8192;
constexpr uint32_t kFold = 4096;  // sums of a group that every CTA of the scaling adds up: eight a thread

struct ClipEntry {
    const void* grad;
    void* out;
    uint64_t part;
    int dtype, out_dtype;
};
template <int N>
struct ClipTable {
    ClipEntry t[N];
    uint32_t chunk0[N];  // chunks of a group in the entries before
    int count;
    uint32_t chunks;            // of a group in this launch
    uint32_t group_chunks, at;  // of a group in all launches, and in those before
    uint32_t chunk;             // bytes
    double* partial;            // [groups][group_chunks]
    float* factor;              // [groups], or null: the scaling finds it
};

__host__ __device__ __forceinline__ uint32_t chunk_elements(int dtype, uint32_t bytes) { return bytes / (dtype == DT_F32 ? 4 : 2); }

// Elements of one chunk.
struct Piece {
    const ClipEntry* t;
    uint64_t from;  // in the tensor
    uint32_t n;
};
template <int N>
__device__ __forceinline__ Piece piece_of(const ClipTable<N>& a, uint32_t group, uint32_t chunk) {
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (chunk < a.chunk0[mid]) hi = mid;
        else lo = mid;
    }
    const ClipEntry& t = a.t[lo];
    const uint32_t most = chunk_elements(t.dtype, a.chunk);
    const uint64_t at = (uint64_t)(chunk - a.chunk0[lo]) * most, left = t.part - at;
    return {&t, group * t.part + at, left < most ? (uint32_t)left : most};
}

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

template <class T>
__device__ __forceinline__ float value(T v) { return (float)v; }

// Sum of a vector's squares: in 32 bits, and once more in 64 where that may
// overflow or lose what is small.
template <class T>
__device__ __forceinline__ double vector_squares(const uint4& z) {
    constexpr uint32_t N = 16 / sizeof(T), ABS = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
    const T* e = reinterpret_cast<const T*>(&z);
    float s = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) s = fmaf(value(e[i]), value(e[i]), s);
    if ((s > 1e-30f && s < 1e37f) || ((z.x | z.y | z.z | z.w) & ABS) == 0) return s;
    double d = 0.0;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) d += (double)value(e[i]) * value(e[i]);
    return d;
}

// f(vector's place p, vector) and g(element's place) over n elements at x, whose
// places count from head, x's offset from a 16-byte boundary: whole vectors, four at
// a time, and the elements at the ends.
template <class T, class F, class E>
__device__ __forceinline__ void each(const T* x, uint32_t n, F vector, E element) {
    constexpr uint32_t N = 16 / sizeof(T), STEP = kThreads * N;
    const uint32_t head = (uint32_t)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)), end = head + n;
    const uint32_t lo = head ? N : 0, hi = end / N * N;  // places of whole vectors
    for (uint32_t p = lo + threadIdx.x * N; p < hi; p += 4 * STEP) {
        uint4 z[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
            if (p + j * STEP < hi) z[j] = *reinterpret_cast<const uint4*>(x + (p + j * STEP) - head);
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
            if (p + j * STEP < hi) vector(p + j * STEP - head, z[j]);
    }
    // at most N - 1 elements before and behind, or all of them where there is no whole vector
    const uint32_t i = threadIdx.x, first = min(lo, end);
    if (i >= head && i < first) element(i - head);
    const uint32_t tail = max(hi, first);
    if (tail + i < end) element(tail + i - head);
}

template <class T>
__device__ double squares(const T* x, uint32_t n) {
    double total = 0.0;
    each(x, n, [&](uint32_t, const uint4& z) { total += vector_squares<T>(z); },
         [&](uint32_t i) { total += (double)value(x[i]) * value(x[i]); });
    return total;
}

template <class T, class O>
__device__ __forceinline__ void put(O* out, const uint4& z, float by) {
    constexpr uint32_t N = 16 / sizeof(T), W = sizeof(O) / sizeof(T);
    const T* e = reinterpret_cast<const T*>(&z);
    uint4 r[W];
    O* o = reinterpret_cast<O*>(r);
#pragma unroll
    for (uint32_t i = 0; i < N; i++) o[i] = (O)(value(e[i]) * by);
    if (reinterpret_cast<uintptr_t>(out) % 16 == 0) {
#pragma unroll
        for (uint32_t i = 0; i < W; i++) reinterpret_cast<uint4*>(out)[i] = r[i];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < N; i++) out[i] = o[i];
    }
}

template <class T, class O>
__device__ void scaled(const T* x, O* out, uint32_t n, float by) {
    each(x, n, [&](uint32_t i, const uint4& z) { put<T, O>(out + i, z, by); }, [&](uint32_t i) { out[i] = (O)(value(x[i]) * by); });
}

__device__ __forceinline__ double piece_squares(const Piece& p) {
    if (p.t->dtype == DT_F32) return squares(static_cast<const float*>(p.t->grad) + p.from, p.n);
    if (p.t->dtype == DT_BF16) return squares(static_cast<const __nv_bfloat16*>(p.t->grad) + p.from, p.n);
    return squares(static_cast<const __half*>(p.t->grad) + p.from, p.n);
}
template <class T>
__device__ __forceinline__ void piece_scaled(const Piece& p, float by) {
    const T* x = static_cast<const T*>(p.t->grad) + p.from;
    if (p.t->out_dtype == DT_F32) scaled(x, static_cast<float*>(p.t->out) + p.from, p.n, by);
    else scaled(x, static_cast<T*>(p.t->out) + p.from, p.n, by);
}

// What a group is multiplied by, from its sum of squares.
struct Limit {
    const float* max_norms;
    float max_norm;
    int one_max;
    __device__ __forceinline__ float factor(uint32_t group, double sum, float* norm) const {
        const double root = sqrt(sum), most = max_norms ? max_norms[one_max ? 0 : group] : max_norm;
        *norm = (float)root;
        return isfinite(*norm) && root > most ? (float)(fmax(most, 0.0) / root) : 1.f;
    }
};

template <int N>
__global__ void __launch_bounds__(kThreads) k_squares(const __grid_constant__ ClipTable<N> a) {
    release_dependents();
    const uint32_t group = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const double v = block_total<kThreads>(piece_squares(piece_of(a, group, chunk)));
    if (threadIdx.x == 0) a.partial[(uint64_t)group * a.group_chunks + a.at + chunk] = v;
}

// A group's norm and factor.  One CTA for each group.
__global__ void __launch_bounds__(1024) k_norms(const double* partial, uint32_t chunks, const Limit l, float* norms, float* factor) {
    release_dependents();
    grid_dependency_wait();
    const double* p = partial + (uint64_t)blockIdx.x * chunks;
    double v = 0.0;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < chunks; i += 1024) v += p[i];
    v = block_total<1024>(v);
    if (threadIdx.x == 0) factor[blockIdx.x] = l.factor(blockIdx.x, v, norms + blockIdx.x);
}

template <int N>
__global__ void __launch_bounds__(kThreads) k_scale(const __grid_constant__ ClipTable<N> a, const Limit l, float* norms) {
    const uint32_t last = gridDim.x - 1 - blockIdx.x, group = last / a.chunks, chunk = last % a.chunks;
    const Piece p = piece_of(a, group, chunk);
    grid_dependency_wait();
    float by;
    if (a.factor) {
        by = a.factor[group];
    } else {
        const double* sums = a.partial + (uint64_t)group * a.group_chunks;
        double v = 0.0;
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < a.group_chunks; i += kThreads) v += sums[i];
        float norm;
        by = l.factor(group, block_total<kThreads>(v), &norm);
        if (chunk == 0 && a.at == 0 && threadIdx.x == 0) norms[group] = norm;
    }
    if (by == 1.f && p.t->grad == p.t->out) return;
    if (p.t->dtype == DT_F32) piece_scaled<float>(p, by);
    else if (p.t->dtype == DT_BF16) piece_scaled<__nv_bfloat16>(p, by);
    else piece_scaled<__half>(p, by);
}

uint64_t chunks_of(const ClipTensor* t, uint64_t count, uint32_t chunk) {
    uint64_t c = 0;
    for (uint64_t i = 0; i < count; i++) c += (t[i].part + chunk_elements(t[i].dtype, chunk) - 1) / chunk_elements(t[i].dtype, chunk);
    return c;
}

uint32_t chunk_bytes(const ClipTensor* t, uint64_t count, uint32_t groups) {
    return chunks_of(t, count, kChunk) * groups < 2 * kSms ? kSmallChunk : kChunk;
}

// The launches over the tensors, N to a launch: the squares, or the scaling.
template <int N>
cudaError_t passes(const ClipArgs& a, uint32_t chunk, uint64_t chunks, float* factor, const Limit* scale, KScope* ks, cudaStream_t s) {
    uint64_t at = 0;
    cudaError_t e = cudaSuccess;
    for (uint64_t i = 0; i < a.count && e == cudaSuccess;) {
        ClipTable<N> t;
        t.count = 0, t.chunks = 0, t.group_chunks = (uint32_t)chunks, t.at = (uint32_t)at, t.chunk = chunk, t.partial = a.partial, t.factor = factor;
        for (; i < a.count && t.count < N; i++) {
            const ClipTensor& c = a.tensors[i];
            t.chunk0[t.count] = t.chunks;
            t.t[t.count++] = {c.grad, c.out, c.part, c.dtype, c.out_dtype};
            t.chunks += (uint32_t)((c.part + chunk_elements(c.dtype, chunk) - 1) / chunk_elements(c.dtype, chunk));
        }
        at += t.chunks;
        const dim3 grid(t.chunks * a.groups);
        if (scale) {
            e = launch_dependent(1, k_scale<N>, grid, kThreads, 0, s, t, *scale, a.norms);
        } else {
            k_squares<N><<<grid, kThreads, 0, s>>>(t);
            e = cudaGetLastError();
        }
        ks->kernels++;
    }
    return e;
}

// N: the tensors in a launch's arguments, whose size the host pays for.
template <int N>
cudaError_t clip(const ClipArgs& a, cudaStream_t s) {
    const uint32_t chunk = chunk_bytes(a.tensors, a.count, a.groups);
    const uint64_t chunks = chunks_of(a.tensors, a.count, chunk);
    const Limit l{a.max_norms, a.max_norm, a.one_max};
    float* const factor = chunks <= kFold && chunks ? nullptr : reinterpret_cast<float*>(a.partial + chunks * a.groups);
    KScope ks("clip_gradients", s, 0);
    cudaError_t e = passes<N>(a, chunk, chunks, factor, nullptr, &ks, s);
    if (e == cudaSuccess && factor) {
        ks.kernels++;
        e = launch_dependent(1, k_norms, dim3(a.groups), 1024, 0, s, (const double*)a.partial, (uint32_t)chunks, l, a.norms, factor);
    }
    return e == cudaSuccess ? passes<N>(a, chunk, chunks, factor, &l, &ks, s) : e;
}

}  // namespace

uint64_t clip_partials(const ClipTensor* t, uint64_t count, uint32_t groups) {
    return chunks_of(t, count, chunk_bytes(t, count, groups)) * groups + (groups + 1) / 2;
}

cudaError_t launch_clip(const ClipArgs& a, cudaStream_t s) {
    return a.count <= 16 ? clip<16>(a, s) : a.count <= 128 ? clip<128>(a, s) : clip<448>(a, s);
}

}  // namespace tsg
