// k_project.cu -- the shared projection of many tokens with their adapters'
// second factors, on the fifth-generation tensor cores.
//
//   out[m][o] = base[m][o] + bias[o] + sum_k x[m][k] W(o, k)
//             + sum_j low[m][j] G_e(m)[j][o]
//
// One persistent CTA per SM walks tiles of 128 tokens x BN outputs.  A warp
// feeds x and W tiles by TMA through a ring of 64-wide slices, one thread
// issues the matrix instructions into one of two TMEM accumulators, four
// warps turn finished accumulators into outputs while the next tile is
// multiplied.  Bound: the tensor cores at large n; the ring is as deep as
// shared memory allows because W and x come from L2.
//
// The low-rank term is a few more steps of the same contraction.  Its axis
// lists the rank indexes of the tile's distinct adapters one adapter after the
// other; four builder warps write 16 of them at a time as TF32 operands: rows
// of low, zero except in the token's own adapter's columns, and the
// factor's columns.  So a tile whose tokens share an adapter (prefill,
// training) pays r / 16 steps and a mixed one D r / 16 for D distinct
// adapters, without sorting tokens or a second pass over out.  TF32 holds
// bf16 and fp16 factors exactly and rounds low to 11 significant bits with
// the range of f32, so that an fp16 low above 65504 does not overflow.
//
// A zero times an adapter's NaN or infinity would spread to the other
// tokens of the tile: the builders replace such elements by 0, flag the tile,
// and the epilogue adds those terms to the adapter's own tokens only.
#include <cuda.h>

#include "launch.cuh"
#include "lowrank.cuh"
#include "sm100.cuh"

namespace tsg {

namespace {

constexpr int kThreads = 320;  // warps 0-3 epilogue, 4-7 builders, 8 TMA, 9 matrix instructions
constexpr int kXK = 16;        // low-rank columns per step

template <int BN>
struct Tile {
    static constexpr int kStage = 128 * 128 + BN * 128;      // bytes: 64 16-bit elements of each row
    static constexpr int kXStage = (128 + BN) * kXK * 4;     // TF32 operands
    static constexpr int kXBufs = BN == 256 ? 1 : 2;
    static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 5 : 6;
    static constexpr int kSmem = kStages * kStage + kXBufs * kXStage + 1024 /* alignment */;
};

struct TcArgs {
    ProjectArgs p;
    int tiles_m, tiles_n, kblocks;
    int vec_out, vec_base, vec_bias;  // 16-byte accesses are aligned
};

// Everything beside the operand rings.
struct Shared {
    uint64_t full[8], empty[8], xfull[2], xempty[2], acc_full[2], acc_empty[2], drained;
    uint32_t tmem, dead;
    uint32_t xlast[2];
    uint32_t bad[4];  // by tile: an element of a factor is not finite
    alignas(16) int ids[128];
    int list[128], pos[128], warp_new[4];
};

template <class T>
__device__ __forceinline__ float elem(const void* p, long long i) {
    if constexpr (sizeof(T) == 4) return static_cast<const float*>(p)[i];
    else if constexpr (std::is_same<T, __half>::value) return __half2float(static_cast<const __half*>(p)[i]);
    else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ bool is_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// W_MN: W's outputs are contiguous (the transposed product of the backward
// call), else its contraction index.
template <class T, int BN, bool W_MN>
__global__ void __launch_bounds__(kThreads, 1)
k_project_tc(const TcArgs a, const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw) {
    using L = Tile<BN>;
    extern __shared__ uint8_t raw[];
    __shared__ Shared sh;
    const uint32_t ring = (smem_u32(raw) + 1023) & ~1023u;
    const uint32_t xring = ring + L::kStages * L::kStage;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ProjectArgs& p = a.p;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; i++) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.xfull[i], 1), mbar_init(&sh.xempty[i], 1);
            mbar_init(&sh.acc_full[i], 1), mbar_init(&sh.acc_empty[i], 128);
        }
        mbar_init(&sh.drained, 1);
        sh.dead = 0;
        mbar_init_fence();
    }
    if (warp == 9) tmem_alloc(&sh.tmem, 2 * BN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int tiles = a.tiles_m * a.tiles_n;

    if (warp == 8) {
        if (lane == 0) {
            Ring r(L::kStages, 1);
            for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
                const int m0 = t % a.tiles_m * 128, o0 = t / a.tiles_m * BN;
                for (int kb = 0; kb < a.kblocks; kb++, r.next()) {
                    if (!mbar_wait(&sh.empty[r.i], r.phase, &sh.dead)) goto tma_done;
                    const uint32_t s = ring + r.i * L::kStage;
                    mbar_expect(&sh.full[r.i], L::kStage);
                    tma_2d(s, &mx, kb * 64, m0, &sh.full[r.i]);
                    if constexpr (W_MN) {
#pragma unroll
                        for (int q = 0; q < BN / 64; q++) tma_2d(s + 16384 + q * 8192, &mw, o0 + q * 64, kb * 64, &sh.full[r.i]);
                    } else {
                        tma_2d(s + 16384, &mw, kb * 64, o0, &sh.full[r.i]);
                    }
                }
            }
        tma_done:;
        }
    } else if (warp == 9) {
        if (lane == 0) {
            constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
            constexpr uint32_t shape = 1u << 4 | (uint32_t)(BN >> 3) << 17 | (128u >> 4) << 24;
            constexpr uint32_t idesc = shape | fmt << 7 | fmt << 10 | (W_MN ? 1u << 16 : 0u);
            constexpr uint32_t xdesc = shape | 2u << 7 | 2u << 10;
            Ring r(L::kStages, 0), x(L::kXBufs, 0), acc(2, 1);
            uint32_t drain_phase = 0;
            for (int t = blockIdx.x; t < tiles; t += gridDim.x, acc.next()) {
                if (!mbar_wait(&sh.acc_empty[acc.i], acc.phase, &sh.dead)) goto mma_done;
                tc_fence_after();
                const uint32_t d = tmem + acc.i * BN;
                for (int kb = 0; kb < a.kblocks; kb++, r.next()) {
                    if (!mbar_wait(&sh.full[r.i], r.phase, &sh.dead)) goto mma_done;
                    tc_fence_after();
                    const uint32_t s = ring + r.i * L::kStage;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint64_t da = desc_k128(s + k * 32);
                        const uint64_t db = W_MN ? desc_mn128(s + 16384 + k * 2048, 8192) : desc_k128(s + 16384 + k * 32);
                        mma_f16(d, da, db, idesc, kb | k);
                    }
                    mma_commit(&sh.empty[r.i]);
                }
                if (a.kblocks) {
                    // the two kinds of instruction are ordered by waiting: once
                    // per tile, a few hundred of some ten thousand cycles
                    mma_commit(&sh.drained);
                    if (!mbar_wait(&sh.drained, drain_phase, &sh.dead)) goto mma_done;
                    drain_phase ^= 1;
                }
                for (bool first = a.kblocks == 0, last = false; !last; first = false, x.next()) {
                    if (!mbar_wait(&sh.xfull[x.i], x.phase, &sh.dead)) goto mma_done;
                    tc_fence_after();
                    last = *reinterpret_cast<volatile uint32_t*>(&sh.xlast[x.i]);
                    const uint32_t s = xring + x.i * L::kXStage;
#pragma unroll
                    for (int k = 0; k < kXK / 8; k++)
                        mma_tf32(d, desc_k64(s + k * 32), desc_k64(s + 128 * kXK * 4 + k * 32), xdesc, !first || k);
                    mma_commit(&sh.xempty[x.i]);
                }
                mma_commit(&sh.acc_full[acc.i]);
            }
        mma_done:;
        }
    } else if (warp >= 4) {
        // builders: thread i has row i of the tile and BN / 128 rows of the factor
        const int i = threadIdx.x - 128, w = warp - 4;
        grid_dependency_wait();  // low is written by the launch before this one
        Ring x(L::kXBufs, 1);
        int serial = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, serial++) {
            const long long m = (long long)(t % a.tiles_m) * 128 + i;
            const int o0 = t / a.tiles_m * BN;
            const int e = m < p.n ? p.id.of(m) : -1;
            sh.ids[i] = e;
            if (i == 0) sh.bad[serial & 3] = 0;
            bar_sync(1, 128);
            // the first row with the same adapter
            int first = (w << 5) + __ffs(__match_any_sync(0xffffffffu, e)) - 1;
#pragma unroll 4
            for (int j = w * 8 - 1; j >= 0; j--) {
                const int4 v = reinterpret_cast<const int4*>(sh.ids)[j];
                if (v.w == e) first = 4 * j + 3;
                if (v.z == e) first = 4 * j + 2;
                if (v.y == e) first = 4 * j + 1;
                if (v.x == e) first = 4 * j;
            }
            const bool lead = e >= 0 && first == i;
            const unsigned ball = __ballot_sync(0xffffffffu, lead);
            if (lane == 0) sh.warp_new[w] = __popc(ball);
            bar_sync(1, 128);
            int before = 0, distinct = 0;
#pragma unroll
            for (int q = 0; q < 4; q++) before += q < w ? sh.warp_new[q] : 0, distinct += sh.warp_new[q];
            if (lead) {
                const int at = before + __popc(ball & ((1u << lane) - 1));
                sh.list[at] = e;
                sh.pos[i] = at;
            }
            bar_sync(1, 128);
            const int own = e >= 0 ? sh.pos[first] * p.r : 1 << 30;  // this row's first column
            const int cols = distinct * p.r;
            const float* low = p.low + m * low_stride(p.r);
            bool bad = false;
            for (int c0 = 0; c0 == 0 || c0 < cols; c0 += kXK, x.next()) {
                float av[kXK], bv[BN / 128 ? BN / 128 : 1][kXK];
#pragma unroll
                for (int q = 0; q < kXK; q++) {
                    const int j = c0 + q - own;
                    av[q] = j >= 0 && j < p.r ? low[j] : 0.f;
                }
                {
                    int d = c0 / p.r, j = c0 - d * p.r;
                    long long g = d < distinct ? sh.list[d] * p.g.se : 0;
#pragma unroll
                    for (int q = 0; q < kXK; q++) {
#pragma unroll
                        for (int h = 0; h < (BN + 127) / 128; h++) {
                            const int o = o0 + i + h * 128;
                            const bool in = (BN >= 128 || i < BN) && o < p.o && d < distinct;
                            bv[h][q] = in ? elem<T>(p.g.p, g + j * p.g.sj + o * p.g.sk) : 0.f;
                        }
                        if (++j == p.r) {
                            j = 0, d++;
                            g = d < distinct ? sh.list[d] * p.g.se : 0;
                        }
                    }
                }
                const bool late = !mbar_wait(&sh.xempty[x.i], x.phase, &sh.dead);
                const uint32_t s = xring + x.i * L::kXStage;
#pragma unroll
                for (int q = 0; q < kXK / 4; q++)
                    st_shared4(s + i * 64 + ((q ^ (i >> 1 & 3)) << 4), to_tf32(av[4 * q]), to_tf32(av[4 * q + 1]), to_tf32(av[4 * q + 2]),
                               to_tf32(av[4 * q + 3]));
#pragma unroll
                for (int h = 0; h < (BN + 127) / 128; h++) {
                    if (BN < 128 && i >= BN) break;
#pragma unroll
                    for (int q = 0; q < kXK; q++)
                        if (!is_finite(bv[h][q])) bv[h][q] = 0.f, bad = true;
                    const int row = i + h * 128;
#pragma unroll
                    for (int q = 0; q < kXK / 4; q++)
                        st_shared4(s + 128 * kXK * 4 + row * 64 + ((q ^ (row >> 1 & 3)) << 4), __float_as_uint(bv[h][4 * q]),
                                   __float_as_uint(bv[h][4 * q + 1]), __float_as_uint(bv[h][4 * q + 2]), __float_as_uint(bv[h][4 * q + 3]));
                }
                if (bad) sh.bad[serial & 3] = 1;
                if (i == 0) sh.xlast[x.i] = c0 + kXK >= cols;
                fence_async_shared();
                if (bar_or(1, 128, late)) goto build_done;  // all 128 threads or none
                if (i == 0) mbar_arrive(&sh.xfull[x.i]);
            }
        }
    build_done:;
    } else {
        Ring acc(2, 0);
        int serial = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, acc.next(), serial++) {
            const long long m = (long long)(t % a.tiles_m) * 128 + threadIdx.x;
            const int o0 = t / a.tiles_m * BN;
            if (!mbar_wait(&sh.acc_full[acc.i], acc.phase, &sh.dead)) break;
            tc_fence_after();
            const uint32_t d = tmem + acc.i * BN + ((uint32_t)warp << 21);  // lane 32 * warp
            const bool row = m < p.n;
            const bool bad = *reinterpret_cast<volatile uint32_t*>(&sh.bad[serial & 3]);
            const int e = bad && row ? p.id.of(m) : -1;
            T* out = static_cast<T*>(p.out) + m * p.out_stride;
            const T* base = static_cast<const T*>(p.base) + m * p.base_stride;
#pragma unroll 1
            for (int c = 0; c < BN; c += 32) {
                float v[32];
                __syncwarp();
                tmem_ld32(d + c, v);
                if (!row || o0 + c >= p.o) continue;
                if (e >= 0) {
                    for (int q = 0; q < 32 && o0 + c + q < p.o; q++)
                        for (int j = 0; j < p.r; j++) {
                            const float g = elem<T>(p.g.p, e * p.g.se + j * p.g.sj + (o0 + c + q) * p.g.sk);
                            if (!is_finite(g)) {
                                const float add = p.low[m * low_stride(p.r) + j] * g;
#pragma unroll
                                for (int z = 0; z < 32; z++)
                                    if (z == q) v[z] += add;
                            }
                        }
                }
#pragma unroll
                for (int q = 0; q < 32; q += 8) {
                    const int o = o0 + c + q;
                    if (o >= p.o) break;
                    const bool whole = o + 8 <= p.o;
                    if (p.bias) {
                        if (whole && a.vec_bias) {
                            const uint4 b = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.bias) + o));
                            const uint32_t u[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                            for (int z = 0; z < 4; z++) {
                                const float2 f = unpack2<T>(u[z]);
                                v[q + 2 * z] += f.x, v[q + 2 * z + 1] += f.y;
                            }
                        } else {
#pragma unroll
                            for (int z = 0; z < 8; z++)
                                if (o + z < p.o) v[q + z] += elem<T>(p.bias, o + z);
                        }
                    }
                    if (p.base) {
                        if (whole && a.vec_base) {
                            const uint4 b = *reinterpret_cast<const uint4*>(base + o);
                            const uint32_t u[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                            for (int z = 0; z < 4; z++) {
                                const float2 f = unpack2<T>(u[z]);
                                v[q + 2 * z] += f.x, v[q + 2 * z + 1] += f.y;
                            }
                        } else {
#pragma unroll
                            for (int z = 0; z < 8; z++)
                                if (o + z < p.o) v[q + z] += elem<T>(base, o + z);
                        }
                    }
                    uint32_t u[4];
#pragma unroll
                    for (int z = 0; z < 4; z++) u[z] = pack2<T>(v[q + 2 * z], v[q + 2 * z + 1]);
                    if (whole && a.vec_out) {
                        *reinterpret_cast<uint4*>(out + o) = make_uint4(u[0], u[1], u[2], u[3]);
                    } else {
                        const T* h = reinterpret_cast<const T*>(u);
#pragma unroll
                        for (int z = 0; z < 8; z++)
                            if (o + z < p.o) out[o + z] = h[z];
                    }
                }
            }
            tc_fence_before();
            mbar_arrive(&sh.acc_empty[acc.i]);
        }
    }

    // A wait that ran out (sh.dead) may leave copies and instructions behind:
    // they end before the memory they write is given up.
    __syncthreads();
    if (warp == 9) {
        if (sh.dead && lane == 0) {
            mma_commit(&sh.drained);
            settle(&sh.drained);
            for (int i = 0; i < L::kStages; i++) settle(&sh.full[i]);
        }
        __syncwarp();
        tmem_free(tmem, 2 * BN);
    }
}

template <class T, int BN, bool W_MN>
cudaError_t launch_tile(const ProjectArgs& p, int sms, cudaStream_t s) {
    using L = Tile<BN>;
    TcArgs a{p};
    a.tiles_m = (int)((p.n + 127) / 128);
    a.tiles_n = (p.o + BN - 1) / BN;
    a.kblocks = p.w ? (p.k + 63) / 64 : 0;
    const auto vec = [](const void* q, long long stride) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && stride % 8 == 0; };
    a.vec_out = vec(p.out, p.out_stride);
    a.vec_base = vec(p.base, p.base_stride);
    a.vec_bias = vec(p.bias, 0);
    CUtensorMap mx{}, mw{};
    if (p.w) {
        const CUtensorMapDataType ty = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        cudaError_t e = tensor_map(&mx, ty, p.x, (uint64_t)p.k, (uint64_t)p.n, (uint64_t)p.x_stride * 2, 64, 128);
        if (e == cudaSuccess)
            e = W_MN ? tensor_map(&mw, ty, p.w, (uint64_t)p.o, (uint64_t)p.k, (uint64_t)p.w_stride * 2, 64, 64)
                     : tensor_map(&mw, ty, p.w, (uint64_t)p.k, (uint64_t)p.o, (uint64_t)p.w_stride * 2, 64, BN);
        if (e != cudaSuccess) return e;
    }
    auto kern = k_project_tc<T, BN, W_MN>;
    const cudaError_t e = ensure_smem(kern, L::kSmem);
    if (e != cudaSuccess) return e;
    KScope ks("adapter_project", s);
    const long long tiles = (long long)a.tiles_m * a.tiles_n;
    return launch_dependent(kern, dim3((unsigned)(tiles < sms ? tiles : sms)), kThreads, L::kSmem, s, a, mx, mw);
}

template <class T, bool W_MN>
cudaError_t launch_width(const ProjectArgs& p, int sms, cudaStream_t s) {
    // The tile width with the fewest (rounds over the SMs) x (cost of a tile).
    // A tile's time grows less than its width: its operands' rows, 128 of x
    // and BN of W, are what shared memory has to deliver.
    const long long tm = (p.n + 127) / 128;
    int best = 0;
    double cost = 0;
    for (const int bn : {256, 128, 64}) {
        const long long tiles = tm * ((p.o + bn - 1) / bn);
        const double c = (double)((tiles + sms - 1) / sms) * (bn + 64);
        if (!best || c < cost) best = bn, cost = c;
    }
    if (best == 256) return launch_tile<T, 256, W_MN>(p, sms, s);
    if (best == 128) return launch_tile<T, 128, W_MN>(p, sms, s);
    return launch_tile<T, 64, W_MN>(p, sms, s);
}

}  // namespace

cudaError_t tensor_map(CUtensorMap* out, CUtensorMapDataType type, const void* p, uint64_t cols, uint64_t rows, uint64_t row_bytes,
                       uint32_t box_cols, uint32_t box_rows) {
    using Encode = decltype(&cuTensorMapEncodeTiled);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess) f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {row_bytes};
    const cuuint32_t box[2] = {box_cols, box_rows}, step[2] = {1, 1};
    const CUresult r = encode(out, type, 2, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t expired_waits(unsigned long long* out) {
    return cudaMemcpyFromSymbol(out, g_expired_waits, sizeof(*out));
}

cudaError_t launch_project_tc(const ProjectArgs& p, int dtype, cudaStream_t s) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    const bool mn = p.w && p.w_t;
    if (dtype == DT_BF16) return mn ? launch_width<__nv_bfloat16, true>(p, sms, s) : launch_width<__nv_bfloat16, false>(p, sms, s);
    return mn ? launch_width<__half, true>(p, sms, s) : launch_width<__half, false>(p, sms, s);
}

}  // namespace tsg
