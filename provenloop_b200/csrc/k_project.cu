// k_project.cu -- the shared projection of many tokens with their adapters'
// second factors, on the fifth-generation tensor cores.
//
//   out[m][o] = base[m][o] + bias[o] + sum_k x[m][k] W(o, k)
//             + sum_j low[m][j] G_e(m)[j][o]
//
// Persistent CTAs, or pairs of CTAs on two SMs (CG = 2), walk tiles of
// 128 CG tokens x BN outputs.  A warp feeds x and W tiles by TMA through a
// ring of 64-wide slices, one thread issues the matrix instructions into one
// of two TMEM accumulators, four warps turn finished accumulators into
// outputs while the next tile is multiplied.  A pair shares W's rows: each
// CTA loads its 128 tokens and half of the outputs, 32 KiB a slice against
// the 48 KiB that a 128 x 256 tile of its own would need.  What bounds large
// n is these slices' way from L2 more than the tensor cores.
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

template <int CG, int BN>
struct Tile {
    static constexpr int kRows = BN / CG;                       // of W or the factor in a CTA
    static constexpr int kStage = 128 * 128 + kRows * 128;      // bytes: 64 16-bit elements of each row
    static constexpr int kXStage = (128 + kRows) * kXK * 4;     // TF32 operands
    static constexpr int kXBufs = 2;
    static constexpr int kStages = 4;
    static constexpr int kOut = 4 * 2 * 4096;                   // per epilogue warp two boxes of 32 rows x 64 outputs
    static constexpr int kSmem = kStages * kStage + kXBufs * kXStage + kOut + 1024 /* alignment */;
};

struct TcArgs {
    ProjectArgs p;
    int tiles_m, tiles_n, kblocks;
    int vec_bias, vec_g;  // 16-byte loads are aligned
    int tma_out;          // out, and base if there is one, take TMA boxes
};

// Everything beside the operand rings.
struct Shared {
    uint64_t full[8], empty[8], xfull[2], xempty[2], acc_full[2], acc_empty[2], drained, base_full[4][2];
    uint32_t tmem, dead;
    uint32_t xlast[2];
    uint32_t bad[8];  // by tile: an element of a factor is not finite
    alignas(16) int ids[256];
    int list[256], pos[256], warp_new[8];
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
template <class T, int CG, int BN, bool W_MN>
__global__ void __launch_bounds__(kThreads, 1)
k_project_tc(const TcArgs a, const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw,
             const __grid_constant__ CUtensorMap mout, const __grid_constant__ CUtensorMap mbase) {
    using L = Tile<CG, BN>;
    extern __shared__ uint8_t raw[];
    __shared__ Shared sh;
    const uint32_t ring = (smem_u32(raw) + 1023) & ~1023u;
    const uint32_t xring = ring + L::kStages * L::kStage;
    const uint32_t out_boxes = xring + L::kXBufs * L::kXStage;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ProjectArgs& p = a.p;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; i++) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.xfull[i], CG), mbar_init(&sh.xempty[i], 1);
            mbar_init(&sh.acc_full[i], 1), mbar_init(&sh.acc_empty[i], 128 * CG);
        }
        mbar_init(&sh.drained, 1);
        for (int i = 0; i < 8; i++) mbar_init(&sh.base_full[i >> 1][i & 1], 1);
        sh.dead = 0;
        for (int i = 0; i < 8; i++) sh.bad[i] = 0;
        mbar_init_fence();
    }
    if (warp == 9) tmem_alloc<CG>(&sh.tmem, 2 * BN);
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync_all();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int tiles = a.tiles_m * a.tiles_n, step = gridDim.x / CG;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;  // rank 0 issues the pair's instructions

    if (warp == 8) {
        if (lane == 0) {
            Ring r(L::kStages, 1);
            for (int t = blockIdx.x / CG; t < tiles; t += step) {
                const int m0 = (t % a.tiles_m * CG + (int)rank) * 128, o0 = t / a.tiles_m * BN + (int)rank * L::kRows;
                for (int kb = 0; kb < a.kblocks; kb++, r.next()) {
                    if (!mbar_wait(&sh.empty[r.i], r.phase, &sh.dead)) goto tma_done;
                    const uint32_t s = ring + r.i * L::kStage;
                    const uint32_t bar = CG == 2 ? map_rank(&sh.full[r.i], 0) : smem_u32(&sh.full[r.i]);
                    if (rank == 0) mbar_expect(&sh.full[r.i], CG * L::kStage);
                    tma_2d<CG>(s, &mx, kb * 64, m0, bar);
                    if constexpr (W_MN) {
#pragma unroll
                        for (int q = 0; q < L::kRows / 64; q++) tma_2d<CG>(s + 16384 + q * 8192, &mw, o0 + q * 64, kb * 64, bar);
                    } else {
                        tma_2d<CG>(s + 16384, &mw, kb * 64, o0, bar);
                    }
                }
            }
        tma_done:;
        }
    } else if (warp == 9) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
            constexpr uint32_t shape = 1u << 4 | (uint32_t)(BN >> 3) << 17 | (128u * CG >> 4) << 24;
            constexpr uint32_t idesc = shape | fmt << 7 | fmt << 10 | (W_MN ? 1u << 16 : 0u);
            constexpr uint32_t xdesc = shape | 2u << 7 | 2u << 10;
            Ring r(L::kStages, 0), x(L::kXBufs, 0), acc(2, 1);
            uint32_t drain_phase = 0;
            for (int t = blockIdx.x / CG; t < tiles; t += step, acc.next()) {
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
                        mma_f16<CG>(d, da, db, idesc, kb | k);
                    }
                    mma_commit<CG>(&sh.empty[r.i]);
                }
                if (a.kblocks) {
                    // the two kinds of instruction are ordered by waiting: once
                    // per tile, a few hundred of some ten thousand cycles
                    mma_commit<CG>(&sh.drained);
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
                        mma_tf32<CG>(d, desc_k64(s + k * 32), desc_k64(s + 128 * kXK * 4 + k * 32), xdesc, !first || k);
                    mma_commit<CG>(&sh.xempty[x.i]);
                }
                mma_commit<CG>(&sh.acc_full[acc.i]);
            }
        mma_done:;
        }
    } else if (warp >= 4) {
        // builders: thread i has row i of the CTA's tokens and kRows / 128
        // rows of the factor; both CTAs of a pair list the adapters of all
        // 128 CG tokens, in the order of their first tokens
        const int i = threadIdx.x - 128, w = warp - 4;
        grid_dependency_wait();  // low is written by the launch before this one
        Ring x(L::kXBufs, 1);
        int serial = 0;
        for (int t = blockIdx.x / CG; t < tiles; t += step, serial++) {
            const long long m0 = (long long)(t % a.tiles_m) * 128 * CG, m = m0 + rank * 128 + i;
            const int o0 = t / a.tiles_m * BN + (int)rank * L::kRows;
            int e[CG], first[CG];
            bool lead[CG];
            unsigned ball[CG];
#pragma unroll
            for (int h = 0; h < CG; h++) {
                e[h] = m0 + h * 128 + i < p.n ? p.id.of(m0 + h * 128 + i) : -1;
                sh.ids[h * 128 + i] = e[h];
            }
            // two tiles ahead: a pair's other CTA may have flagged the next tile
            // already, and the epilogue is at most five behind
            if (i == 0) sh.bad[(serial + 2) & 7] = 0;
            bar_sync(1, 128);
#pragma unroll
            for (int h = 0; h < CG; h++) {
                // the first token with the same adapter
                first[h] = h * 128 + (w << 5) + __ffs(__match_any_sync(0xffffffffu, e[h])) - 1;
#pragma unroll 4
                for (int j = h * 32 + w * 8 - 1; j >= 0; j--) {
                    const int4 v = reinterpret_cast<const int4*>(sh.ids)[j];
                    if (v.w == e[h]) first[h] = 4 * j + 3;
                    if (v.z == e[h]) first[h] = 4 * j + 2;
                    if (v.y == e[h]) first[h] = 4 * j + 1;
                    if (v.x == e[h]) first[h] = 4 * j;
                }
                lead[h] = e[h] >= 0 && first[h] == h * 128 + i;
                ball[h] = __ballot_sync(0xffffffffu, lead[h]);
                if (lane == 0) sh.warp_new[h * 4 + w] = __popc(ball[h]);
            }
            bar_sync(1, 128);
            int distinct = 0;
#pragma unroll
            for (int h = 0; h < CG; h++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    if (q == w && lead[h]) {
                        const int at = distinct + __popc(ball[h] & ((1u << lane) - 1));
                        sh.list[at] = e[h];
                        sh.pos[h * 128 + i] = at;
                    }
                    distinct += sh.warp_new[h * 4 + q];
                }
            bar_sync(1, 128);
            const int mine = CG == 2 && rank ? e[CG - 1] : e[0], mine_first = CG == 2 && rank ? first[CG - 1] : first[0];
            const int own = mine >= 0 ? sh.pos[mine_first] * p.r : 1 << 30;  // this row's first column
            const int cols = distinct * p.r;
            const float* low = p.low + (m < p.n ? m : 0) * low_stride(p.r);
            bool bad = false;
            // kAhead steps of loads are in flight in registers: every load is
            // made, from a clamped place, and selected where it is used
            constexpr int H = (L::kRows + 127) / 128, kAhead = 3;
            struct Step {
                float a[kXK];
                uint32_t b[H][kXK / 2];
            } ahead[kAhead];
            const auto load = [&](int c0, Step& st) {
                if (p.r % 4 == 0) {
#pragma unroll
                    for (int q = 0; q < kXK; q += 4) {
                        const int j = c0 + q - own;
                        const float4 f = *reinterpret_cast<const float4*>(low + (j >= 0 && j < p.r ? j : 0));
                        st.a[q] = f.x, st.a[q + 1] = f.y, st.a[q + 2] = f.z, st.a[q + 3] = f.w;
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < kXK; q++) {
                        const int j = c0 + q - own;
                        st.a[q] = low[j >= 0 && j < p.r ? j : 0];
                    }
                }
                if (a.vec_g) {
#pragma unroll
                    for (int q = 0; q < kXK; q += 8) {
                        const int d = (c0 + q) / p.r, j = c0 + q - d * p.r;
                        const T* g = static_cast<const T*>(p.g.p) + (d < distinct ? sh.list[d] * p.g.se + j : 0);
#pragma unroll
                        for (int h = 0; h < H; h++) {
                            const int o = o0 + i + h * 128;
                            const uint4 f = *reinterpret_cast<const uint4*>(g + (o < p.o ? o * p.g.sk : 0));
                            st.b[h][q / 2] = f.x, st.b[h][q / 2 + 1] = f.y, st.b[h][q / 2 + 2] = f.z, st.b[h][q / 2 + 3] = f.w;
                        }
                    }
                } else {
                    int d = c0 / p.r, j = c0 - d * p.r;
                    uint16_t v[H][kXK];
#pragma unroll
                    for (int q = 0; q < kXK; q++) {
                        const uint16_t* g = static_cast<const uint16_t*>(p.g.p) + (d < distinct ? sh.list[d] * p.g.se + j * p.g.sj : 0);
#pragma unroll
                        for (int h = 0; h < H; h++) {
                            const int o = o0 + i + h * 128;
                            v[h][q] = g[o < p.o ? o * p.g.sk : 0];
                        }
                        if (++j == p.r) j = 0, d++;
                    }
#pragma unroll
                    for (int h = 0; h < H; h++)
#pragma unroll
                        for (int q = 0; q < kXK / 2; q++) st.b[h][q] = v[h][2 * q] | (uint32_t)v[h][2 * q + 1] << 16;
                }
            };
            const int steps = max(1, (cols + kXK - 1) / kXK);
#pragma unroll
            for (int u = 0; u < kAhead; u++)
                if (u < steps) load(u * kXK, ahead[u]);
            for (int c = 0; c < steps; c += kAhead) {
#pragma unroll
                for (int u = 0; u < kAhead; u++) {
                    if (c + u >= steps) break;
                    Step& st = ahead[u];
                    const int c0 = (c + u) * kXK;
                    const bool late = !mbar_wait(&sh.xempty[x.i], x.phase, &sh.dead);
                    const uint32_t s = xring + x.i * L::kXStage;
                    uint32_t v[kXK];
#pragma unroll
                    for (int q = 0; q < kXK; q++) {
                        const int j = c0 + q - own;
                        v[q] = j >= 0 && j < p.r ? to_tf32(st.a[q]) : 0u;
                    }
#pragma unroll
                    for (int q = 0; q < kXK / 4; q++)
                        st_shared4(s + i * 64 + ((q ^ (i >> 1 & 3)) << 4), v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        if (L::kRows < 128 && i >= L::kRows) break;
                        const int row = i + h * 128;
#pragma unroll
                        for (int q = 0; q < kXK / 2; q++) {
                            const float2 f = unpack2<T>(st.b[h][q]);
                            const bool in0 = c0 + 2 * q < cols && o0 + row < p.o, in1 = c0 + 2 * q + 1 < cols && o0 + row < p.o;
                            const bool ok0 = is_finite(f.x), ok1 = is_finite(f.y);
                            v[2 * q] = in0 && ok0 ? __float_as_uint(f.x) : 0u;
                            v[2 * q + 1] = in1 && ok1 ? __float_as_uint(f.y) : 0u;
                            bad |= (in0 && !ok0) || (in1 && !ok1);
                        }
#pragma unroll
                        for (int q = 0; q < kXK / 4; q++)
                            st_shared4(s + 128 * kXK * 4 + row * 64 + ((q ^ (row >> 1 & 3)) << 4), v[4 * q], v[4 * q + 1], v[4 * q + 2],
                                       v[4 * q + 3]);
                    }
                    if (bad) {
                        sh.bad[serial & 7] = 1;
                        if constexpr (CG == 2) st_cluster(map_rank(&sh.bad[serial & 7], rank ^ 1), 1);
                    }
                    if (i == 0) sh.xlast[x.i] = c + u + 1 == steps;
                    fence_async_shared();
                    if (bar_or(1, 128, late)) goto build_done;  // all 128 threads or none
                    if (i == 0) {
                        if constexpr (CG == 2) mbar_arrive_at(map_rank(&sh.xfull[x.i], 0));
                        else mbar_arrive(&sh.xfull[x.i]);
                    }
                    x.next();
                    if (c + u + kAhead < steps) load(c0 + kAhead * kXK, st);
                }
            }
        }
    build_done:;
    } else {
        Ring acc(2, 0);
        int serial = 0;
        uint32_t base_phase = 0;  // bit: the phase of base_full[warp][buffer]
        const uint32_t boxes = out_boxes + warp * 8192;
        // This row's terms of elements of the factor that are not finite
        const auto add_bad = [&](long long m, int e, int o, float (&v)[32]) {
            for (int q = 0; q < 32 && o + q < p.o; q++)
                for (int j = 0; j < p.r; j++) {
                    const float g = elem<T>(p.g.p, e * p.g.se + j * p.g.sj + (o + q) * p.g.sk);
                    if (!is_finite(g)) {
                        const float add = p.low[m * low_stride(p.r) + j] * g;
#pragma unroll
                        for (int z = 0; z < 32; z++)
                            if (z == q) v[z] += add;
                    }
                }
        };
        const auto add_bias = [&](int o, float (&v)[32]) {
            if (a.vec_bias && o + 32 <= p.o) {
                uint4 b[4];
#pragma unroll
                for (int q = 0; q < 4; q++) b[q] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.bias) + o) + q);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t u[4] = {b[q].x, b[q].y, b[q].z, b[q].w};
#pragma unroll
                    for (int z = 0; z < 4; z++) {
                        const float2 f = unpack2<T>(u[z]);
                        v[q * 8 + 2 * z] += f.x, v[q * 8 + 2 * z + 1] += f.y;
                    }
                }
            } else {
#pragma unroll
                for (int z = 0; z < 32; z++) v[z] += elem<T>(p.bias, min(o + z, p.o - 1));
            }
        };
        for (int t = blockIdx.x / CG; t < tiles; t += step, acc.next(), serial++) {
            const int m0 = (t % a.tiles_m * CG + (int)rank) * 128 + warp * 32;  // this warp's first token
            const long long m = (long long)m0 + lane;
            const int o0 = t / a.tiles_m * BN;
            const int groups = m0 < p.n ? (min(BN, p.o - o0) + 63) / 64 : 0;  // of 64 outputs
            const bool tma_base = a.tma_out && p.base;
            const auto fetch_base = [&](int g) {  // one lane; its buffer's last store has been read
                mbar_expect(&sh.base_full[warp][g & 1], 4096);
                tma_2d<1>(boxes + (g & 1) * 4096, &mbase, o0 + g * 64, m0, smem_u32(&sh.base_full[warp][g & 1]));
            };
            if (tma_base && groups && lane == 0) {
                tma_store_wait_read<0>();
                fetch_base(0);
            }
            __syncwarp();
            if (!__all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc.i], acc.phase, &sh.dead))) break;
            tc_fence_after();
            const uint32_t d = tmem + acc.i * BN + ((uint32_t)warp << 21);  // lane 32 * warp
            const bool row = m < p.n;
            const bool bad = *reinterpret_cast<volatile uint32_t*>(&sh.bad[serial & 7]);
            const int e = bad && row ? p.id.of(m) : -1;
            if (a.tma_out) {
                // through shared memory, so that rows leave as whole boxes; base
                // comes the same way into the box that takes the result
                for (int g = 0; g < groups; g++) {
                    const uint32_t box = boxes + (g & 1) * 4096;
                    if (lane == 0) {
                        if (tma_base) {
                            tma_store_wait_read<0>();
                            if (g + 1 < groups) fetch_base(g + 1);
                        } else {
                            tma_store_wait_read<1>();
                        }
                    }
                    __syncwarp();
                    if (tma_base) {
                        mbar_wait(&sh.base_full[warp][g & 1], base_phase >> (g & 1) & 1, &sh.dead);
                        base_phase ^= 1u << (g & 1);
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int c = g * 64 + h * 32;
                        float v[32];
                        __syncwarp();
                        tmem_ld32(d + c, v);
                        if (p.bias) add_bias(o0 + c, v);
                        if (e >= 0) add_bad(m, e, o0 + c, v);
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const uint32_t at = box + lane * 128 + (((h * 4 + q) ^ (lane & 7)) << 4);
                            uint32_t u[4];
                            if (tma_base) {
                                const uint4 b = ld_shared4(at);
                                u[0] = b.x, u[1] = b.y, u[2] = b.z, u[3] = b.w;
#pragma unroll
                                for (int z = 0; z < 4; z++) {
                                    const float2 f = unpack2<T>(u[z]);
                                    v[q * 8 + 2 * z] += f.x, v[q * 8 + 2 * z + 1] += f.y;
                                }
                            }
#pragma unroll
                            for (int z = 0; z < 4; z++) u[z] = pack2<T>(v[q * 8 + 2 * z], v[q * 8 + 2 * z + 1]);
                            st_shared4(at, u[0], u[1], u[2], u[3]);
                        }
                    }
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) tma_store_2d(&mout, o0 + g * 64, m0, box);
                }
            } else {
                // rows that are not on 16-byte boundaries
                T* out = static_cast<T*>(p.out) + m * p.out_stride;
                const T* base = static_cast<const T*>(p.base) + m * p.base_stride;
                for (int c = 0; c < groups * 64 && o0 + c < p.o; c += 32) {
                    float v[32];
                    __syncwarp();
                    tmem_ld32(d + c, v);
                    if (p.bias) add_bias(o0 + c, v);
                    if (e >= 0) add_bad(m, e, o0 + c, v);
                    if (row) {
                        if (p.base) {
#pragma unroll
                            for (int z = 0; z < 32; z++) v[z] += elem<T>(base, min(o0 + c + z, p.o - 1));
                        }
#pragma unroll
                        for (int z = 0; z < 16; z++) {
                            const uint32_t u = pack2<T>(v[2 * z], v[2 * z + 1]);
                            const T* h = reinterpret_cast<const T*>(&u);
                            if (o0 + c + 2 * z < p.o) out[o0 + c + 2 * z] = h[0];
                            if (o0 + c + 2 * z + 1 < p.o) out[o0 + c + 2 * z + 1] = h[1];
                        }
                    }
                }
            }
            tc_fence_before();
            if constexpr (CG == 2) mbar_arrive_at(map_rank(&sh.acc_empty[acc.i], 0));
            else mbar_arrive(&sh.acc_empty[acc.i]);
        }
        if (lane == 0) tma_store_wait_read<0>();
    }

    // A wait that ran out (sh.dead) may leave copies and instructions behind:
    // they get a bounded time to end before the memory they write is given up.
    __syncthreads();
    if (sh.dead && threadIdx.x == 0) settle();
    if constexpr (CG == 2) cluster_sync_all();
    else __syncthreads();
    if (warp == 9) tmem_free<CG>(tmem, 2 * BN);
}

template <class T, int CG, int BN, bool W_MN>
cudaError_t launch_tile(const ProjectArgs& p, int sms, cudaStream_t s) {
    using L = Tile<CG, BN>;
    TcArgs a{p};
    a.tiles_m = (int)((p.n + 128 * CG - 1) / (128 * CG));
    a.tiles_n = (p.o + BN - 1) / BN;
    a.kblocks = p.w ? (p.k + 63) / 64 : 0;
    const auto vec = [](const void* q, long long stride) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && stride % 8 == 0; };
    const auto rows = [&](const void* q, long long stride) { return vec(q, p.n < 2 ? 0 : stride) && (p.n < 2 || (stride >= p.o && stride < (1ll << 38))); };
    a.tma_out = rows(p.out, p.out_stride) && (!p.base || rows(p.base, p.base_stride));
    a.vec_bias = vec(p.bias, 0);
    a.vec_g = p.g.sj == 1 && vec(p.g.p, p.r);
    CUtensorMap mx{}, mw{}, mout{}, mbase{};
    const CUtensorMapDataType ty = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (a.tma_out) {
        const auto pitch = [&](long long stride) { return (uint64_t)(p.n < 2 ? (p.o + 7) / 8 * 8 : stride) * 2; };
        cudaError_t e = tensor_map(&mout, ty, p.out, (uint64_t)p.o, (uint64_t)p.n, pitch(p.out_stride), 64, 32);
        if (e == cudaSuccess && p.base) e = tensor_map(&mbase, ty, p.base, (uint64_t)p.o, (uint64_t)p.n, pitch(p.base_stride), 64, 32);
        if (e != cudaSuccess) return e;
    }
    if (p.w) {
        cudaError_t e = tensor_map(&mx, ty, p.x, (uint64_t)p.k, (uint64_t)p.n, (uint64_t)p.x_stride * 2, 64, 128);
        if (e == cudaSuccess)
            e = W_MN ? tensor_map(&mw, ty, p.w, (uint64_t)p.o, (uint64_t)p.k, (uint64_t)p.w_stride * 2, 64, 64)
                     : tensor_map(&mw, ty, p.w, (uint64_t)p.k, (uint64_t)p.o, (uint64_t)p.w_stride * 2, 64, L::kRows);
        if (e != cudaSuccess) return e;
    }
    auto kern = k_project_tc<T, CG, BN, W_MN>;
    const cudaError_t e = ensure_smem(kern, L::kSmem);
    if (e != cudaSuccess) return e;
    KScope ks("adapter_project", s);
    const long long tiles = (long long)a.tiles_m * a.tiles_n, slots = sms / CG;
    return launch_dependent(CG, kern, dim3((unsigned)(tiles < slots ? tiles : slots) * CG), kThreads, L::kSmem, s, a, mx, mw, mout, mbase);
}

template <class T, bool W_MN>
cudaError_t launch_width(const ProjectArgs& p, int sms, cudaStream_t s) {
    // The tile with the least (rounds over the SMs) x (time of a tile): in
    // units of the slices' bytes, which is what a tile waits for.
    const auto cost = [&](int cg, int bn) {
        const long long tiles = ((p.n + 128 * cg - 1) / (128 * cg)) * ((p.o + bn - 1) / bn), slots = sms / cg;
        return (double)((tiles + slots - 1) / slots) * (128 + bn / cg);
    };
    const double c256 = cost(2, 256), c128 = cost(1, 128), c64 = cost(1, 64);
    if (c256 <= c128 && c256 <= c64) return launch_tile<T, 2, 256, W_MN>(p, sms, s);
    if (c128 <= c64) return launch_tile<T, 1, 128, W_MN>(p, sms, s);
    return launch_tile<T, 1, 64, W_MN>(p, sms, s);
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
