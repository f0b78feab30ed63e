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
// n is these slices' way from L2 more than the tensor cores: 4099 tokens of
// 1536 -> 8960 with rank 32 take 103 us behind low's 12 (1.1 PFLOP/s; the
// library's product alone takes 81 us), in nine rounds of tiles, the last of
// which three tokens alone ask for.
//
// The low-rank term is a few more slices of the same contraction, behind the
// shared ones in the same ring: units of 16 rank indexes of one adapter, two
// to a slice, for each distinct adapter of the tile.  Four builder warps write
// the tokens' rows of low, zero for other adapters' tokens, and TMA brings
// the factor's rows, both as TF32.  So a tile whose tokens share an adapter
// (prefill, training) pays r / 16 units and a mixed one D r / 16 for D distinct
// adapters, without sorting tokens or a second pass over out.  TF32 holds bf16 and fp16 factors exactly and low to
// 11 significant bits with the range of f32, so that an fp16 low above
// 65504 does not overflow; a second term for its other bits would double the
// units.  (Elsewhere in this file low is a factor of FMAs and keeps its 24
// bits.)  The factors are converted once per call (k_pack).
//
// A zero times an adapter's NaN or infinity would spread to the other
// tokens of the tile: k_pack replaces such elements by 1 of their sign (of which an infinite
// low gives the right infinity) and flags them, and the epilogue adds their
// terms to the adapter's own tokens only.
#include <climits>
#include <cuda.h>

#include "launch.cuh"
#include "lowrank.cuh"
#include "sm100.cuh"

namespace tsg {

namespace {

constexpr int kThreads = 448;  // warps 0-7 epilogue, 8-11 builders, 12 TMA, 13 matrix instructions
constexpr int kXK = 16;        // rank indexes per unit

template <int CG, int BN>
struct Tile {
    static constexpr int kRows = BN / CG;                       // of W or the factor in a CTA
    static constexpr int kStage = 128 * 128 + kRows * 128;      // bytes: 64 16-bit elements of each row
    static constexpr int kUnit = kStage / 2;                    // kXK TF32 values of each row
    static constexpr int kStages = 6;
    static constexpr int kOut = 8 * 2 * 2048;                   // per epilogue warp two boxes of 32 rows x 32 outputs
    static constexpr int kSmem = kStages * kStage + kOut + 1024 /* alignment */;
};

struct TcArgs {
    ProjectArgs p;
    int tiles_m, tiles_n, kblocks;
    int split, rows, x_rows;  // k_project_split
    int vec_bias;         // 16-byte loads are aligned
    int tma_out;          // out, and base if there is one, take TMA boxes
};

// The distinct adapters of a tile of up to 256 tokens, in the order of their
// first tokens.
struct TileAdapters {
    alignas(16) uint32_t next[2][4];
    int list[256];
};

// `e`: the adapters of this thread's tokens i, i + 128, ... (four warps, w this
// one).  Returns the number of distinct ones; place: each token's in the list
// (complete after the caller's next barrier), -1 without an adapter.  One
// round for each: few, mostly, and code that runs once a tile is paid by
// the instruction.
template <int W>
__device__ __forceinline__ int tile_adapters(TileAdapters& s, int w, const int (&e)[W], int (&place)[W]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < W; h++) place[h] = -1;
#pragma unroll 1
    for (int d = 0;; d++) {
        // the first token without a place: its number and adapter
        uint32_t key = UINT_MAX;
#pragma unroll
        for (int h = W - 1; h >= 0; h--) {
            const unsigned left = __ballot_sync(0xffffffffu, place[h] < 0 && e[h] >= 0);
            const int at = left ? __ffs(left) - 1 : 0;
            const int first = __shfl_sync(0xffffffffu, e[h], at);
            if (left) key = (uint32_t)(h * 128 + w * 32 + at) << 16 | (uint32_t)first;
        }
        if (lane == 0) s.next[d & 1][w] = key;
        bar_sync(1, 128);
        const uint4 all = *reinterpret_cast<const uint4*>(s.next[d & 1]);
        key = min(min(all.x, all.y), min(all.z, all.w));
        if (key == UINT_MAX) return d;
        const int found = (int)(key & 0xffffu);
#pragma unroll
        for (int h = 0; h < W; h++)
            if (e[h] == found) place[h] = d;
        if (w == 0 && lane == 0) s.list[d] = found;
    }
}

// Everything beside the operand rings.
struct Shared {
    uint64_t full[8], empty[8], counted[8], turn[2], acc_full[2], acc_empty[2], drained, base_full[8][2];
    uint32_t tmem, dead;
    uint32_t bad[16]; // by tile: an element of a factor is not finite
    int units[8];     // by tile: low-rank units, there when counted
    TileAdapters adapters;
};

template <class T>
__device__ __forceinline__ float elem(const void* p, long long i) {
    if constexpr (std::is_same<T, __half>::value) return __half2float(static_cast<const __half*>(p)[i]);
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
             const __grid_constant__ CUtensorMap mg, const __grid_constant__ CUtensorMap mout, const __grid_constant__ CUtensorMap mbase) {
    using L = Tile<CG, BN>;
    extern __shared__ uint8_t raw[];
    __shared__ Shared sh;
    const uint32_t ring = (smem_u32(raw) + 1023) & ~1023u;
    const uint32_t out_boxes = ring + L::kStages * L::kStage;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ProjectArgs& p = a.p;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; i++) mbar_init(&sh.full[i], CG), mbar_init(&sh.empty[i], 1);
        for (int i = 0; i < 8; i++) mbar_init(&sh.counted[i], 1);
        for (int i = 0; i < 2; i++) mbar_init(&sh.turn[i], 1);
        for (int i = 0; i < 2; i++) mbar_init(&sh.acc_full[i], 1), mbar_init(&sh.acc_empty[i], 8 * CG);
        mbar_init(&sh.drained, 1);
        for (int i = 0; i < 16; i++) mbar_init(&sh.base_full[i >> 1][i & 1], 1);
        sh.dead = 0;
        for (int i = 0; i < 16; i++) sh.bad[i] = 0;
        mbar_init_fence();
    }
    if (warp == 13) tmem_alloc<CG>(&sh.tmem, 2 * BN);
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync_all();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int tiles = a.tiles_m * a.tiles_n, step = gridDim.x / CG;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;  // rank 0 issues the pair's instructions
    // The TMA warp and the builders fill the ring in turns, tile by tile: a
    // barrier's parity tells a slice's use from the one before only to whom
    // comes next.  turn[0]: the shared slices of a tile have their places, the
    // builders may go on; turn[1]: so have the builders' (half as many as the
    // tile has units).  counted: the units of a tile are known; the ring is
    // less than eight tiles long.
    const bool shared_part = a.kblocks > 0;

    if (warp == 12) {
        if (lane == 0) {
            if (p.packed) grid_dependency_wait();
            Ring r(L::kStages, 1);
            int serial = 0;
            for (int t = blockIdx.x / CG; t < tiles && shared_part; t += step, serial++) {
                const int m0 = (t % a.tiles_m * CG + (int)rank) * 128, o0 = t / a.tiles_m * BN + (int)rank * L::kRows;
                for (int kb = 0; kb < a.kblocks; kb++, r.next()) {
                    if (!mbar_wait(&sh.empty[r.i], r.phase, &sh.dead)) goto tma_done;
                    const uint32_t s = ring + r.i * L::kStage;
                    const uint32_t bar = CG == 2 ? map_rank(&sh.full[r.i], 0) : smem_u32(&sh.full[r.i]);
                    if (rank == 0) mbar_expect(&sh.full[r.i], CG * L::kStage);
                    else mbar_arrive_relaxed_at(bar);
                    tma_2d<CG>(s, &mx, kb * 64, m0, bar);
                    if constexpr (W_MN) {
#pragma unroll
                        for (int q = 0; q < L::kRows / 64; q++) tma_2d<CG>(s + 16384 + q * 8192, &mw, o0 + q * 64, kb * 64, bar);
                    } else {
                        tma_2d<CG>(s + 16384, &mw, kb * 64, o0, bar);
                    }
                }
                mbar_arrive(&sh.turn[0]);
                if (!mbar_wait(&sh.turn[1], serial & 1, &sh.dead)) break;
                r.skip((*reinterpret_cast<volatile int*>(&sh.units[serial & 7]) + 1) / 2);
            }
        tma_done:;
        }
    } else if (warp == 13) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
            constexpr uint32_t shape = 1u << 4 | (uint32_t)(BN >> 3) << 17 | (128u * CG >> 4) << 24;
            constexpr uint32_t idesc = shape | fmt << 7 | fmt << 10 | (W_MN ? 1u << 16 : 0u);
            constexpr uint32_t xdesc = shape | 2u << 7 | 2u << 10;
            Ring r(L::kStages, 0), acc(2, 1);
            uint32_t drain_phase = 0;
            int serial = 0, units;
            for (int t = blockIdx.x / CG; t < tiles; t += step, acc.next(), serial++) {
                if (!mbar_wait(&sh.acc_empty[acc.i], acc.phase, &sh.dead)) goto mma_done;
                tc_fence_after();
                const uint32_t d = tmem + acc.i * BN;
                uint32_t add = 0;
                for (int kb = 0; kb < a.kblocks; kb++, r.next()) {
                    if (!mbar_wait(&sh.full[r.i], r.phase, &sh.dead)) goto mma_done;
                    tc_fence_after();
                    const uint32_t s = ring + r.i * L::kStage;
#pragma unroll
                    for (int k = 0; k < 4; k++, add = 1) {
                        const uint64_t da = desc_k128(s + k * 32);
                        const uint64_t db = W_MN ? desc_mn128(s + 16384 + k * 2048, 8192) : desc_k128(s + 16384 + k * 32);
                        mma_f16<CG>(d, da, db, idesc, add);
                    }
                    mma_commit<CG>(&sh.empty[r.i]);
                }
                if (!mbar_wait(&sh.counted[serial & 7], serial >> 3 & 1, &sh.dead)) goto mma_done;
                units = *reinterpret_cast<volatile int*>(&sh.units[serial & 7]);
                if (a.kblocks && units) {
                    // the two kinds of instruction are ordered by waiting: a few
                    // hundred of some ten thousand cycles
                    mma_commit<CG>(&sh.drained);
                    if (!mbar_wait(&sh.drained, drain_phase, &sh.dead)) goto mma_done;
                    drain_phase ^= 1;
                }
                for (int u = 0; u < units; u += 2, r.next()) {
                    if (!mbar_wait(&sh.full[r.i], r.phase, &sh.dead)) goto mma_done;
                    tc_fence_after();
                    for (int h = 0; h < 2 && u + h < units; h++) {
                        const uint32_t s = ring + r.i * L::kStage + h * L::kUnit;
#pragma unroll
                        for (int k = 0; k < kXK / 8; k++, add = 1)
                            mma_tf32<CG>(d, desc_k64(s + k * 32), desc_k64(s + 128 * kXK * 4 + k * 32), xdesc, add);
                    }
                    mma_commit<CG>(&sh.empty[r.i]);
                }
                mma_commit<CG>(&sh.acc_full[acc.i]);
            }
        mma_done:;
        }
    } else if (warp >= 8) {
        // builders: thread i has row i of the CTA's tokens; both CTAs of a
        // pair list the adapters of all 128 CG tokens, in the order of their
        // first tokens
        const int i = threadIdx.x - 256, w = warp - 8;
        const int rs = low_stride(p.r), blocks = (p.o + 127) / 128;
        grid_dependency_wait();  // low and the converted factors are written by the launches before
        release_dependents();    // what the next launch (the gradients) reads is there
        const auto load_ids = [&](int t, int (&e)[CG]) {
#pragma unroll
            for (int h = 0; h < CG; h++) {
                const long long m = ((long long)(t % a.tiles_m) * CG + h) * 128 + i;
                e[h] = t < tiles && m < p.n ? p.id.of(m) : -1;
            }
        };
        Ring r(L::kStages, 1);
        int serial = 0, e[CG];
        load_ids(blockIdx.x / CG, e);
        for (int t = blockIdx.x / CG; t < tiles; t += step, serial++) {
            const long long m0 = (long long)(t % a.tiles_m) * 128 * CG, m = m0 + rank * 128 + i;
            const int o0 = t / a.tiles_m * BN + (int)rank * L::kRows;
            int pos[CG];
            if (i == 0) sh.bad[serial & 15] = 0;  // the ring and the accumulators are less than sixteen tiles
            const int distinct = tile_adapters(sh.adapters, w, e, pos);
            const int own = CG == 2 && rank ? pos[CG - 1] : pos[0];
            // the next tile's
            load_ids(t + step, e);
            const uint4* low = reinterpret_cast<const uint4*>(p.low + (m < p.n ? m : 0) * rs);
            // the factor's flags for the tile's outputs; the first of them are looked at with low
            const int tile_o = t / a.tiles_m * BN, per = rs / kXK, flags = min((BN + 127) / 128, blocks - tile_o / 128) * per;
            const auto flag = [&](int d) { return p.bad[((long long)sh.adapters.list[d / flags] * blocks + tile_o / 128) * per + d % flags]; };
            uint32_t bad = i < distinct * flags ? flag(i) : 0u;
            for (int d = i + 128; d < distinct * flags; d += 128) bad |= flag(d);
            // without a shared product something has to clear the accumulator
            const int count = a.kblocks ? distinct : max(1, distinct), units = count * per;
            if (i == 0) {
                sh.units[serial & 7] = units;
                mbar_arrive(&sh.counted[serial & 7]);
            }
            r.skip(a.kblocks);
            bool late = shared_part && !mbar_wait(&sh.turn[0], serial & 1, &sh.dead);
            if (!units) {
                if (bar_or(1, 128, late)) goto build_done;
                if (i == 0) mbar_arrive(&sh.turn[1]);
            }
            int u = 0;
            uint4 f[4];
            for (int j = 0; j < rs; j += kXK) {
#pragma unroll
                for (int q = 0; q < 4; q++) f[q] = low[j / 4 + q];
                if (!p.low_tf32) {
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        f[q] = make_uint4(to_tf32(__uint_as_float(f[q].x)), to_tf32(__uint_as_float(f[q].y)), to_tf32(__uint_as_float(f[q].z)),
                                          to_tf32(__uint_as_float(f[q].w)));
                }
                if (bad) sh.bad[serial & 15] = 1;
                for (int d = 0; d < count; d++, u++) {
                    const uint32_t s = ring + r.i * L::kStage + (u & 1) * L::kUnit;
                    if (!(u & 1)) late |= !mbar_wait(&sh.empty[r.i], r.phase, &sh.dead);
                    if (i == 0) {
                        const uint32_t bar = CG == 2 ? map_rank(&sh.full[r.i], 0) : smem_u32(&sh.full[r.i]);
                        tma_3d<CG>(s + 128 * kXK * 4, &mg, j, o0, distinct ? sh.adapters.list[d] : 0, bar);
                    }
                    const bool in = d == own;
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        st_shared4(s + i * 64 + ((q ^ (i >> 1 & 3)) << 4), in ? f[q].x : 0u, in ? f[q].y : 0u, in ? f[q].z : 0u, in ? f[q].w : 0u);
                    if ((u & 1) || u + 1 == units) {
                        fence_async_shared();
                        if (bar_or(1, 128, late)) goto build_done;  // all 128 threads or none
                        if (i == 0) {
                            if (rank == 0) mbar_expect(&sh.full[r.i], CG * (1 + (u & 1)) * L::kRows * kXK * 4);
                            else mbar_arrive_at(map_rank(&sh.full[r.i], 0));
                            if (u + 1 == units && shared_part) mbar_arrive(&sh.turn[1]);
                        }
                        r.next();
                    }
                }
            }
        }
    build_done:;
    } else {
        Ring acc(2, 0);
        int serial = 0;
        uint32_t base_phase = 0;  // bit: the phase of base_full[warp][buffer]
        const uint32_t boxes = out_boxes + warp * 4096;
        const int quarter = warp & 3, half = warp >> 2;  // of the accumulator's lanes, of its columns
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
            const int m0 = (t % a.tiles_m * CG + (int)rank) * 128 + quarter * 32;  // this warp's first token
            const long long m = (long long)m0 + lane;
            const int o0 = t / a.tiles_m * BN + half * (BN / 2);
            const int groups = m0 < p.n ? (max(0, min(BN / 2, p.o - o0)) + 31) / 32 : 0;  // of 32 outputs
            const bool tma_base = a.tma_out && p.base;
            const auto fetch_base = [&](int g) {  // one lane; its buffer's last store has been read
                mbar_expect(&sh.base_full[warp][g & 1], 2048);
                tma_2d<1>(boxes + (g & 1) * 2048, &mbase, o0 + g * 32, m0, smem_u32(&sh.base_full[warp][g & 1]));
            };
            if (tma_base && groups && lane == 0) {
                tma_store_wait_read<0>();
                fetch_base(0);
            }
            __syncwarp();
            if (!__all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc.i], acc.phase, &sh.dead))) break;
            tc_fence_after();
            const uint32_t d = tmem + acc.i * BN + half * (BN / 2) + ((uint32_t)quarter << 21);  // lane 32 * quarter
            const bool row = m < p.n;
            const bool bad = *reinterpret_cast<volatile uint32_t*>(&sh.bad[serial & 15]);
            const int e = bad && row ? p.id.of(m) : -1;
            if (a.tma_out) {
                // through shared memory, so that rows leave as whole boxes; base
                // comes the same way into the box that takes the result
                for (int g = 0; g < groups; g++) {
                    const uint32_t box = boxes + (g & 1) * 2048;
                    if (lane == 0) {
                        if (tma_base) {
                            tma_store_wait_read<0>();
                            if (g + 1 < groups) fetch_base(g + 1);
                        } else {
                            tma_store_wait_read<1>();
                        }
                    }
                    float v[32];
                    __syncwarp();
                    tmem_ld32(d + g * 32, v);
                    if (p.bias) add_bias(o0 + g * 32, v);
                    if (e >= 0) add_bad(m, e, o0 + g * 32, v);
                    if (tma_base) {
                        mbar_wait(&sh.base_full[warp][g & 1], base_phase >> (g & 1) & 1, &sh.dead);
                        base_phase ^= 1u << (g & 1);
                    }
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const uint32_t at = box + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4);
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
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) tma_store_2d(&mout, o0 + g * 32, m0, box);
                }
            } else {
                // rows that are not on 16-byte boundaries: through the box as
                // well, and from there (to there) a row of 32 at a time
                const uint16_t* base = static_cast<const uint16_t*>(p.base);
                uint16_t* out = static_cast<uint16_t*>(p.out);
                const int rows = (int)max(0LL, min(32LL, p.n - m0));
                const auto at = [&](int i, int c) { return boxes + i * 64 + ((c >> 3 ^ (i >> 1 & 3)) << 4) + (c & 7) * 2; };
                for (int g = 0; g < groups; g++) {
                    const int o = o0 + g * 32 + lane, oc = min(o, p.o - 1);  // this lane's column
                    float v[32];
                    __syncwarp();
                    if (p.base) {
#pragma unroll 16
                        for (int i = 0; i < 32; i++) st_shared2b(at(i, lane), base[(m0 + min(i, rows - 1)) * p.base_stride + oc]);
                        __syncwarp();
                    }
                    tmem_ld32(d + g * 32, v);
                    if (p.bias) add_bias(o0 + g * 32, v);
                    if (e >= 0) add_bad(m, e, o0 + g * 32, v);
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        uint32_t u[4];
                        if (p.base) {
                            const uint4 b = ld_shared4(at(lane, q * 8));
                            u[0] = b.x, u[1] = b.y, u[2] = b.z, u[3] = b.w;
#pragma unroll
                            for (int z = 0; z < 4; z++) {
                                const float2 f = unpack2<T>(u[z]);
                                v[q * 8 + 2 * z] += f.x, v[q * 8 + 2 * z + 1] += f.y;
                            }
                        }
#pragma unroll
                        for (int z = 0; z < 4; z++) u[z] = pack2<T>(v[q * 8 + 2 * z], v[q * 8 + 2 * z + 1]);
                        st_shared4(at(lane, q * 8), u[0], u[1], u[2], u[3]);
                    }
                    __syncwarp();
#pragma unroll 16
                    for (int i = 0; i < 32; i++)
                        if (i < rows && o < p.o) out[(m0 + i) * p.out_stride + o] = ld_shared2b(at(i, lane));
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) mbar_arrive_at(map_rank(&sh.acc_empty[acc.i], 0));
                else mbar_arrive(&sh.acc_empty[acc.i]);
            }
        }
        if (lane == 0) tma_store_wait_read<0>();
    }

    // A wait that ran out (sh.dead) may leave copies and instructions behind:
    // they get a bounded time to end before the memory they write is given up.
    __syncthreads();
    if (sh.dead && threadIdx.x == 0) settle();
    if constexpr (CG == 2) cluster_sync_all();
    else __syncthreads();
    if (warp == 13) tmem_free<CG>(tmem, 2 * BN);
}

template <class T, bool W_MN>
cudaError_t operand_maps(const ProjectArgs& p, int x_rows, int w_rows, CUtensorMap* mx, CUtensorMap* mw) {
    const CUtensorMapDataType ty = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const cudaError_t e = tensor_map(mx, ty, p.x, (uint64_t)p.k, (uint64_t)p.n, (uint64_t)p.x_stride * 2, 64, x_rows);
    if (e != cudaSuccess) return e;
    return W_MN ? tensor_map(mw, ty, p.w, (uint64_t)p.o, (uint64_t)p.k, (uint64_t)p.w_stride * 2, 64, 64)
                : tensor_map(mw, ty, p.w, (uint64_t)p.k, (uint64_t)p.o, (uint64_t)p.w_stride * 2, 64, w_rows);
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
    CUtensorMap mx{}, mw{}, mg{}, mout{}, mbase{};
    const CUtensorMapDataType ty = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (a.tma_out) {
        const auto pitch = [&](long long stride) { return (uint64_t)(p.n < 2 ? (p.o + 7) / 8 * 8 : stride) * 2; };
        cudaError_t e = tensor_map(&mout, ty, p.out, (uint64_t)p.o, (uint64_t)p.n, pitch(p.out_stride), 32, 32);
        if (e == cudaSuccess && p.base) e = tensor_map(&mbase, ty, p.base, (uint64_t)p.o, (uint64_t)p.n, pitch(p.base_stride), 32, 32);
        if (e != cudaSuccess) return e;
    }
    {
        const int rs = low_stride(p.r);
        const cudaError_t e = tensor_map(&mg, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, p.g32, rs, p.o, (uint64_t)rs * 4, kXK, L::kRows, p.id.count);
        if (e != cudaSuccess) return e;
    }
    if (p.w) {
        const cudaError_t e = operand_maps<T, W_MN>(p, 128, L::kRows, &mx, &mw);
        if (e != cudaSuccess) return e;
    }
    auto kern = k_project_tc<T, CG, BN, W_MN>;
    const cudaError_t e = ensure_smem(kern, L::kSmem);
    if (e != cudaSuccess) return e;
    KScope ks("adapter_project", s);
    const long long tiles = (long long)a.tiles_m * a.tiles_n, slots = sms / CG;
    return launch_dependent(CG, kern, dim3((unsigned)(tiles < slots ? tiles : slots) * CG), kThreads, L::kSmem, s, a, mx, mw, mg, mout, mbase);
}

// v[z] += sum_j low[j] G(j, o + z) for N neighbouring outputs: the factor's
// widest loads along whichever axis is contiguous, else its elements.
template <class T, int N>
__device__ __forceinline__ void add_low(const ProjectArgs& p, const float* low, const T* g, int o, float (&v)[N]) {
    const T* at = g + o * p.g.sk;
    if (p.g.sk == 1 && o + N <= p.o && p.g.sj % N == 0 && reinterpret_cast<uintptr_t>(at) % (2 * N) == 0) {
#pragma unroll 8
        for (int j = 0; j < p.r; j++) {
            uint32_t u[N / 2];
            if constexpr (N == 8) {
                const uint4 q = *reinterpret_cast<const uint4*>(at + j * p.g.sj);
                u[0] = q.x, u[1] = q.y, u[2] = q.z, u[3] = q.w;
            } else {
                u[0] = *reinterpret_cast<const uint32_t*>(at + j * p.g.sj);
            }
            const float l = low[j];
#pragma unroll
            for (int z = 0; z < N / 2; z++) {
                const float2 f = unpack2<T>(u[z]);
                v[2 * z] = fmaf(l, f.x, v[2 * z]), v[2 * z + 1] = fmaf(l, f.y, v[2 * z + 1]);
            }
        }
    } else if (p.g.sj == 1 && (p.r & 7) == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {
#pragma unroll 2
        for (int j = 0; j < p.r; j += 8) {
            const float4 l0 = *reinterpret_cast<const float4*>(low + j), l1 = *reinterpret_cast<const float4*>(low + j + 4);
            uint4 q[N];
#pragma unroll
            for (int z = 0; z < N; z++) q[z] = *reinterpret_cast<const uint4*>(g + min(o + z, p.o - 1) * p.g.sk + j);
#pragma unroll
            for (int z = 0; z < N; z++) {
                const float2 f0 = unpack2<T>(q[z].x), f1 = unpack2<T>(q[z].y), f2 = unpack2<T>(q[z].z), f3 = unpack2<T>(q[z].w);
                v[z] = fmaf(l0.x, f0.x, v[z]), v[z] = fmaf(l0.y, f0.y, v[z]), v[z] = fmaf(l0.z, f1.x, v[z]), v[z] = fmaf(l0.w, f1.y, v[z]);
                v[z] = fmaf(l1.x, f2.x, v[z]), v[z] = fmaf(l1.y, f2.y, v[z]), v[z] = fmaf(l1.z, f3.x, v[z]), v[z] = fmaf(l1.w, f3.y, v[z]);
            }
        }
    } else if (p.g.sj == 1 && (p.r & 1) == 0 && (reinterpret_cast<uintptr_t>(g) & 3) == 0) {
        // blocks of whole unconditional loads, from clamped places behind the last rank
        constexpr int B = N == 8 ? 4 : 8;
        for (int j = 0; j < p.r; j += 2 * B) {
            float2 l[B];
            uint32_t q[B][N];
#pragma unroll
            for (int b = 0; b < B; b++) {
                const int at = min(j + 2 * b, p.r - 2);
                l[b] = *reinterpret_cast<const float2*>(low + at);
#pragma unroll
                for (int z = 0; z < N; z++) q[b][z] = *reinterpret_cast<const uint32_t*>(g + min(o + z, p.o - 1) * p.g.sk + at);
            }
#pragma unroll
            for (int b = 0; b < B; b++)
                if (j + 2 * b < p.r)
#pragma unroll
                    for (int z = 0; z < N; z++) {
                        const float2 f = unpack2<T>(q[b][z]);
                        v[z] = fmaf(l[b].x, f.x, v[z]), v[z] = fmaf(l[b].y, f.y, v[z]);
                    }
        }
    } else {
        constexpr int B = N == 8 ? 4 : 8;
        for (int j = 0; j < p.r; j += B) {
            float l[B], f[B][N];
#pragma unroll
            for (int b = 0; b < B; b++) {
                const int at = min(j + b, p.r - 1);
                l[b] = low[at];
#pragma unroll
                for (int z = 0; z < N; z++) f[b][z] = elem<T>(g, at * p.g.sj + min(o + z, p.o - 1) * p.g.sk);
            }
#pragma unroll
            for (int b = 0; b < B; b++)
                if (j + b < p.r)
#pragma unroll
                    for (int z = 0; z < N; z++) v[z] = fmaf(l[b], f[b][z], v[z]);
        }
    }
}

// Not enough tiles for all SMs: a cluster of S CTAs shares the contraction of
// a 128 x BN tile, each with a ring of its own, and the partial sums meet in
// shared memory, where each CTA finishes BN / S of the outputs.  Each token
// takes its own adapter's factor straight from memory (n o r elements in all),
// so that nothing is converted first.  Where a CTA's share is small, the six
// warps that neither load nor multiply compute these terms meanwhile (behind
// the contraction they took 5 us more).  Bound: reading W once by all SMs
// together, and the launches' latency.  48 tokens of 8960 -> 1536 with 64
// adapters of rank 30: 18 us behind low's 8, 2.5 TB/s over both; one CTA for
// each SM in clusters of six instead of eight took 23.
template <int BN>
struct SplitTile {
    static constexpr int kStages = BN == 64 ? 4 : 3;
    static constexpr int kStage = 128 * 128 + BN * 128;
    static constexpr int kRow = BN + 4;  // floats: rows of the partial sums four banks apart
    static constexpr int kEarly = 2048;  // outputs of a CTA whose other terms are computed during the contraction
    static constexpr int kSmem = kStages * kStage + kEarly * 4 + 1024;
    static_assert(128 * kRow * 4 <= kStages * kStage, "the sums fit where the ring was");
};

// Bias, base and the adapter's term of N neighbouring outputs of token m.
template <class T, int N>
__device__ __forceinline__ void other_terms(const ProjectArgs& p, long long m, int o, float (&v)[N]) {
    const int e = p.id.of(m);
    if (p.bias) {
#pragma unroll
        for (int z = 0; z < N; z++) v[z] += elem<T>(p.bias, min(o + z, p.o - 1));
    }
    if (p.base) {
        const T* base = static_cast<const T*>(p.base) + m * p.base_stride + o;
        if (o + N <= p.o && reinterpret_cast<uintptr_t>(base) % (2 * N) == 0) {
            uint32_t u[N / 2];
            if constexpr (N == 8) {
                const uint4 q = *reinterpret_cast<const uint4*>(base);
                u[0] = q.x, u[1] = q.y, u[2] = q.z, u[3] = q.w;
            } else {
                u[0] = *reinterpret_cast<const uint32_t*>(base);
            }
#pragma unroll
            for (int z = 0; z < N / 2; z++) {
                const float2 f = unpack2<T>(u[z]);
                v[2 * z] += f.x, v[2 * z + 1] += f.y;
            }
        } else {
#pragma unroll
            for (int z = 0; z < N; z++) v[z] += elem<T>(base, min(z, p.o - 1 - o));
        }
    }
    if (e >= 0) add_low<T, N>(p, p.low + m * low_stride(p.r), static_cast<const T*>(p.g.p) + e * p.g.se, o, v);
}

template <class T, int N>
__device__ __forceinline__ void put_outputs(const ProjectArgs& p, long long m, int o, const float (&v)[N]) {
    T* out = static_cast<T*>(p.out) + m * p.out_stride + o;
    uint32_t u[N / 2];
#pragma unroll
    for (int z = 0; z < N / 2; z++) u[z] = pack2<T>(v[2 * z], v[2 * z + 1]);
    if (o + N <= p.o && reinterpret_cast<uintptr_t>(out) % (2 * N) == 0) {
        if constexpr (N == 8) *reinterpret_cast<uint4*>(out) = make_uint4(u[0], u[1], u[2], u[3]);
        else *reinterpret_cast<uint32_t*>(out) = u[0];
    } else {
        const T* h = reinterpret_cast<const T*>(u);
#pragma unroll
        for (int z = 0; z < N; z++)
            if (o + z < p.o) out[z] = h[z];
    }
}

// v[z] += the partial sums of all CTAs of the cluster.
template <int N>
__device__ __forceinline__ void add_sums(const float* f, int S, float (&v)[N]) {
#pragma unroll
    for (int q = 0; q < 8; q++) {
        if (q >= S) break;
        if constexpr (N == 2) {
            const float2 w = ld_cluster2(map_rank(f, q));
            v[0] += w.x, v[1] += w.y;
        } else {
#pragma unroll
            for (int z = 0; z < N; z += 4) {
                const float4 w = ld_cluster4(map_rank(f + z, q));
                v[z] += w.x, v[z + 1] += w.y, v[z + 2] += w.z, v[z + 3] += w.w;
            }
        }
    }
}

template <class T, int BN, bool W_MN>
__global__ void __launch_bounds__(256)
k_project_split(const TcArgs a, const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw) {
    using L = SplitTile<BN>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[L::kStages], empty[L::kStages], done;
    __shared__ uint32_t tmem_at, dead;
    const uint32_t ring = (smem_u32(raw) + 1023) & ~1023u;
    float* sums = reinterpret_cast<float*>(raw + (ring - smem_u32(raw)));  // [128][kRow], when the ring is done with
    float* terms = sums + L::kStages * L::kStage / 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ProjectArgs& p = a.p;
    const int S = a.split, rank = (int)cluster_rank();
    const long long m0 = (long long)(blockIdx.x / S) * a.rows;
    const int o0 = blockIdx.y * BN, rows = (int)min((long long)a.rows, p.n - m0);
    const int per = BN / S, col0 = rank * per;  // this CTA's outputs
    const bool early = rows * per <= L::kEarly;
    const int kb0 = a.kblocks * rank / S, kb1 = a.kblocks * (rank + 1) / S;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; i++) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        mbar_init(&done, 1);
        dead = 0;
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc<1>(&tmem_at, BN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    if (warp == 0) {
        if (lane == 0) {
            if (p.packed) grid_dependency_wait();
            Ring r(L::kStages, 1);
            for (int kb = kb0; kb < kb1; kb++, r.next()) {
                if (!mbar_wait(&empty[r.i], r.phase, &dead)) break;
                const uint32_t s = ring + r.i * L::kStage, bar = smem_u32(&full[r.i]);
                mbar_expect(&full[r.i], a.x_rows * 128 + BN * 128);
                tma_2d<1>(s, &mx, kb * 64, (int)m0, bar);
                if constexpr (W_MN) {
#pragma unroll
                    for (int q = 0; q < BN / 64; q++) tma_2d<1>(s + 16384 + q * 8192, &mw, o0 + q * 64, kb * 64, bar);
                } else {
                    tma_2d<1>(s + 16384, &mw, kb * 64, o0, bar);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
            constexpr uint32_t idesc = 1u << 4 | fmt << 7 | fmt << 10 | (W_MN ? 1u << 16 : 0u) | (uint32_t)(BN >> 3) << 17 | 8u << 24;
            Ring r(L::kStages, 0);
            for (int kb = kb0; kb < kb1; kb++, r.next()) {
                if (!mbar_wait(&full[r.i], r.phase, &dead)) break;
                tc_fence_after();
                const uint32_t s = ring + r.i * L::kStage;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint64_t db = W_MN ? desc_mn128(s + 16384 + k * 2048, 8192) : desc_k128(s + 16384 + k * 32);
                    mma_f16<1>(tmem, desc_k128(s + k * 32), db, idesc, (kb - kb0) | k);
                }
                mma_commit<1>(&empty[r.i]);
            }
            mma_commit<1>(&done);
        }
    } else if (early) {
        grid_dependency_wait();  // low is written by the launch before this one
        release_dependents();
        for (int i = threadIdx.x - 64; i < rows * (per / 2); i += 192) {
            const int row = i / (per / 2), o = o0 + col0 + i % (per / 2) * 2;
            if (o >= p.o) continue;
            float v[2] = {};
            other_terms<T, 2>(p, m0 + row, o, v);
            *reinterpret_cast<float2*>(terms + 2 * i) = make_float2(v[0], v[1]);
        }
    }
    __syncwarp();
    mbar_wait(&done, 0, &dead);
    tc_fence_after();
    const int row = (warp & 3) * 32 + lane;
#pragma unroll
    for (int c = (warp >> 2) * (BN / 2); c < (warp >> 2) * (BN / 2) + BN / 2; c += 32) {
        float v[32];
        __syncwarp();
        tmem_ld32(tmem + c + ((uint32_t)(warp & 3) << 21), v);
#pragma unroll
        for (int q = 0; q < 32; q += 4)
            *reinterpret_cast<float4*>(sums + row * L::kRow + c + q) = make_float4(v[q], v[q + 1], v[q + 2], v[q + 3]);
    }
    tc_fence_before();
    if (S > 1) cluster_sync_all();
    else __syncthreads();
    if (early) {
        for (int i = threadIdx.x; i < rows * (per / 2); i += 256) {
            const int row = i / (per / 2), col = col0 + i % (per / 2) * 2;
            if (o0 + col >= p.o) continue;
            const float2 t = *reinterpret_cast<const float2*>(terms + 2 * i);
            float v[2] = {t.x, t.y};
            add_sums<2>(sums + row * L::kRow + col, S, v);
            put_outputs<T, 2>(p, m0 + row, o0 + col, v);
        }
    } else {
        grid_dependency_wait();  // low is written by the launch before this one
        release_dependents();
        for (int i = threadIdx.x; i < rows * (per / 8); i += 256) {
            const int row = i / (per / 8), col = col0 + i % (per / 8) * 8;
            if (o0 + col >= p.o) continue;
            float v[8] = {};
            add_sums<8>(sums + row * L::kRow + col, S, v);
            other_terms<T, 8>(p, m0 + row, o0 + col, v);
            put_outputs<T, 8>(p, m0 + row, o0 + col, v);
        }
    }
    if (dead && threadIdx.x == 0) settle();
    if (S > 1) cluster_sync_all();
    else __syncthreads();
    if (warp == 1) tmem_free<1>(tmem_at, BN);
}

// The adapters' term beside a base and a bias, without a shared projection:
// 32 tokens x 64 outputs a CTA.  Bound: latency, then reading base.  2048
// tokens of 256 outputs, rank 16: 16 us with low's 8.
template <class T>
__global__ void __launch_bounds__(256, 2) k_add_low(const ProjectArgs p) {
    const long long m = (long long)blockIdx.x * 32 + threadIdx.x / 8;
    const int o = blockIdx.y * 64 + threadIdx.x % 8 * 8;
    grid_dependency_wait();
    release_dependents();
    if (m >= p.n || o >= p.o) return;
    float v[8] = {};
    other_terms<T, 8>(p, m, o, v);
    put_outputs<T, 8>(p, m, o, v);
}

template <class T, int BN, bool W_MN>
cudaError_t launch_split(const ProjectArgs& p, int sms, cudaStream_t s) {
    using L = SplitTile<BN>;
    TcArgs a{p};
    a.tiles_n = (p.o + BN - 1) / BN;
    a.kblocks = (p.k + 63) / 64;
    a.tiles_m = (int)((p.n + 127) / 128);
    // as many CTAs share a tile as it takes to give every SM one, while each
    // has two slices of the contraction and eight outputs of a row
    a.split = 1;
    while (a.split < 8 && (long long)a.tiles_m * a.tiles_n * a.split < sms && a.kblocks >= 4 * a.split) a.split *= 2;
    // where that is not enough, tiles of fewer tokens, for the adapters' terms
    a.rows = 128;
    while (a.rows > 32 && p.n > a.rows / 2 && (long long)a.tiles_m * a.tiles_n * a.split < sms) {
        a.rows /= 2;
        a.tiles_m = (int)((p.n + a.rows - 1) / a.rows);
    }
    a.x_rows = p.n < a.rows ? (int)(p.n + 7) / 8 * 8 : a.rows;  // rows behind stay whatever they are: their sums are not used
    CUtensorMap mx{}, mw{};
    auto kern = k_project_split<T, BN, W_MN>;
    cudaError_t e = operand_maps<T, W_MN>(p, a.x_rows, BN, &mx, &mw);
    if (e == cudaSuccess) e = ensure_smem(kern, L::kSmem);
    if (e != cudaSuccess) return e;
    KScope ks("adapter_project", s);
    return launch_dependent(a.split, kern, dim3((unsigned)(a.tiles_m * a.split), a.tiles_n), 256, L::kSmem, s, a, mx, mw);
}

// low of many tokens: a cluster of S CTAs shares the contraction of 128
// tokens with the factors of the tile's distinct adapters, whose rank indexes,
// 16 to a unit, lie side by side as the products' columns; a token keeps its
// own adapter's.  Eight units at a time: a tile with more of them reads x
// again.  Bound: reading x, with some 60 KiB under way on each SM.  2048 tokens
// of 1536, rank 16: 8 us; both products of a training step of 8192 tokens
// (1536 and 1536): 17 us, 3 TB/s.
struct LowTile {
    static constexpr int kUnits = 8, kCols = 16 * kUnits;
    static constexpr int kStages = 3;
    static constexpr int kStage = 128 * 128 + kCols * 128;
    static constexpr int kRow = kCols + 4;
    static constexpr int kSmem = kStages * kStage + 1024;
    static_assert(128 * kRow * 4 <= kStages * kStage, "the sums fit where the ring was");
};

struct LowMaps {
    CUtensorMap x[2], f[2];
};

// Four values of token m's low.
__device__ __forceinline__ void put(const LowArgs& a, long long m, int rs, int j, float4 v) {
    if (a.low) {
        float4* to = reinterpret_cast<float4*>(a.low + m * rs + j);
        if (a.tf32)
            *reinterpret_cast<uint4*>(to) = make_uint4(to_tf32(v.x), to_tf32(v.y), to_tf32(v.z), to_tf32(v.w));
        else
            *to = v;
    }
    if (a.split) {
        uint32_t h[4], l[4];
        bf16_terms(v.x, h[0], l[0]), bf16_terms(v.y, h[1], l[1]), bf16_terms(v.z, h[2], l[2]), bf16_terms(v.w, h[3], l[3]);
        uint16_t* to = a.split + m * 2 * rs + j;
        *reinterpret_cast<uint2*>(to) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
        *reinterpret_cast<uint2*>(to + rs) = make_uint2(l[0] | l[1] << 16, l[2] | l[3] << 16);
    }
}

template <class T>
__global__ void __launch_bounds__(256) k_low_tc(const LowPair both, const __grid_constant__ LowMaps maps) {
    using L = LowTile;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[L::kStages], empty[L::kStages], done;
    __shared__ uint32_t tmem_at, dead;
    __shared__ TileAdapters adapters;
    __shared__ int place[128], found;  // each token's place in the list, its length
    release_dependents();
    const LowArgs& a = both.a[blockIdx.z];
    const uint32_t ring = (smem_u32(raw) + 1023) & ~1023u;
    float* sums = reinterpret_cast<float*>(raw + (ring - smem_u32(raw)));  // [128][kRow], when the ring is done with
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = gridDim.y, rank = (int)cluster_rank();
    const long long m0 = (long long)blockIdx.x * 128;
    const int rs = low_stride(a.r), per = rs / 16, kblocks = (a.k + 63) / 64;
    const int kb0 = kblocks * rank / S, kb1 = kblocks * (rank + 1) / S;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; i++) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        mbar_init(&done, 1);
        dead = 0;
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc<1>(&tmem_at, L::kCols);
    int e[1] = {-1}, own[1] = {-1}, distinct = 0;
    if (warp < 4) {
        if (m0 + threadIdx.x < a.n) e[0] = a.id.of(m0 + threadIdx.x);
        distinct = tile_adapters(adapters, warp, e, own);
        place[threadIdx.x] = own[0];
        if (threadIdx.x == 0) found = distinct;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    distinct = found;
    const uint32_t tmem = tmem_at;
    const int* list = adapters.list;
    if (both.after_pack[blockIdx.z] == 2) grid_dependency_wait();

    const int units = distinct * per;
    Ring fill(L::kStages, 1), drain(L::kStages, 0);
    uint32_t done_phase = 0;
    for (int u0 = 0; u0 < units; u0 += L::kUnits, done_phase ^= 1) {
        const int nu = min(L::kUnits, units - u0);
        if (warp == 0) {
            if (lane == 0)
                for (int kb = kb0; kb < kb1; kb++, fill.next()) {
                    if (!mbar_wait(&empty[fill.i], fill.phase, &dead)) break;
                    const uint32_t s = ring + fill.i * L::kStage, bar = smem_u32(&full[fill.i]);
                    mbar_expect(&full[fill.i], 16384 + nu * 2048);
                    tma_2d<1>(s, &maps.x[blockIdx.z], kb * 64, (int)m0, bar);
                    for (int u = 0; u < nu; u++)
                        tma_3d<1>(s + 16384 + u * 2048, &maps.f[blockIdx.z], kb * 64, (u0 + u) % per * 16, list[(u0 + u) / per], bar);
                }
        } else if (warp == 1) {
            if (lane == 0) {
                constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
                const uint32_t idesc = 1u << 4 | fmt << 7 | fmt << 10 | (uint32_t)(2 * nu) << 17 | 8u << 24;
                for (int kb = kb0; kb < kb1; kb++, drain.next()) {
                    if (!mbar_wait(&full[drain.i], drain.phase, &dead)) break;
                    tc_fence_after();
                    const uint32_t s = ring + drain.i * L::kStage;
#pragma unroll
                    for (int k = 0; k < 4; k++) mma_f16<1>(tmem, desc_k128(s + k * 32), desc_k128(s + 16384 + k * 32), idesc, (kb - kb0) | k);
                    mma_commit<1>(&empty[drain.i]);
                }
                mma_commit<1>(&done);
            }
        }
        __syncwarp();
        mbar_wait(&done, done_phase, &dead);
        tc_fence_after();
        const int row = (warp & 3) * 32 + lane;
        for (int c = warp >> 2 << 5; c < nu * 16; c += 64) {
            float v[32];
            __syncwarp();
            tmem_ld32(tmem + c + ((uint32_t)(warp & 3) << 21), v);
            if (kb1 > kb0) {
#pragma unroll
                for (int q = 0; q < 32; q += 4)
                    *reinterpret_cast<float4*>(sums + row * L::kRow + c + q) = make_float4(v[q], v[q + 1], v[q + 2], v[q + 3]);
            } else {
#pragma unroll
                for (int q = 0; q < 32; q += 4) *reinterpret_cast<float4*>(sums + row * L::kRow + c + q) = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        tc_fence_before();
        if (S > 1) cluster_sync_all();
        else __syncthreads();
        tc_fence_after();
        // each CTA finishes 128 / S of the tokens, four rank indexes a thread
        const int rows = 128 / S;
        for (int i = threadIdx.x; i < rows * nu * 4; i += 256) {
            const int r = rank * rows + i / (nu * 4), c = i % (nu * 4) * 4, u = u0 + c / 16;
            if (place[r] != u / per) continue;
            const int at = list[u / per], j = u % per * 16 + c % 16;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int q = 0; q < S; q++) {
                const float* p = sums + r * L::kRow + c;
                const float4 f = S > 1 ? ld_cluster4(map_rank(p, q)) : *reinterpret_cast<const float4*>(p);
                v.x += f.x, v.y += f.y, v.z += f.z, v.w += f.w;
            }
            const float scale = a.scale ? a.scale[at] : 1.f;
            const auto value = [&](float f, int jj) { return jj < a.r ? scale * f : 0.f; };
            put(a, m0 + r, rs, j, make_float4(value(v.x, j), value(v.y, j + 1), value(v.z, j + 2), value(v.w, j + 3)));
        }
        // the sums have been read before the ring's memory is filled again
        fence_async_shared();
        if (S > 1) cluster_sync_all();
        else __syncthreads();
    }
    // tokens without an adapter
    for (int i = rank * 256 + threadIdx.x; i < 128 * rs / 4; i += 256 * S) {
        const int r = i / (rs / 4);
        if (place[r] < 0 && m0 + r < a.n) put(a, m0 + r, rs, i % (rs / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    }
    if (dead && threadIdx.x == 0) settle();
    __syncthreads();
    if (warp == 1) tmem_free<1>(tmem, L::kCols);
    if (both.after_pack[blockIdx.z] == 1) grid_dependency_wait();
}

template <class T>
cudaError_t low_tc(const LowArgs* a, int count, const int* after_pack, int sms, cudaStream_t s) {
    LowPair both{{a[0], a[count - 1]}, {after_pack[0], after_pack[count - 1]}};
    LowMaps maps{};
    const CUtensorMapDataType ty = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int i = 0; i < count; i++) {
        cudaError_t e = tensor_map(&maps.x[i], ty, a[i].x, (uint64_t)a[i].k, (uint64_t)a[i].n, (uint64_t)a[i].x_stride * 2, 64, 128);
        if (e == cudaSuccess)
            e = tensor_map(&maps.f[i], ty, a[i].f.p, (uint64_t)a[i].k, (uint64_t)a[i].r, (uint64_t)a[i].f.sj * 2, 64, 16, (uint64_t)a[i].id.count);
        if (e != cudaSuccess) return e;
    }
    // as many CTAs share a contraction as still run together, two on each SM,
    // while each has two slices
    const long long tiles = (a[0].n + 127) / 128;
    const int kmax = a[0].k > a[count - 1].k ? a[0].k : a[count - 1].k;
    int S = 1;
    while (S < 8 && tiles * S * count <= sms && kmax / 64 >= 4 * S) S *= 2;
    const cudaError_t e = ensure_smem(k_low_tc<T>, LowTile::kSmem);
    if (e != cudaSuccess) return e;
    KScope ks("adapter_low", s);
    return launch_split_y(S, after_pack[0] != 0, k_low_tc<T>, dim3((unsigned)tiles, S, count), 256, LowTile::kSmem, s, both, maps);
}

template <class T, bool W_MN>
cudaError_t launch_width(const ProjectArgs& p, int sms, cudaStream_t s) {
    if (!p.g32) {
        if (!p.w) {
            KScope ks("adapter_project", s);
            return launch_dependent(1, k_add_low<T>, dim3((unsigned)((p.n + 31) / 32), (p.o + 63) / 64), 256, 0, s, p);
        }
        // 64-wide tiles as long as they do not fill the SMs twice
        const long long tiles = ((p.n + 127) / 128) * ((p.o + 63) / 64);
        return tiles <= 2 * sms ? launch_split<T, 64, W_MN>(p, sms, s) : launch_split<T, 128, W_MN>(p, sms, s);
    }
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
                       uint32_t box_cols, uint32_t box_rows, uint64_t count) {
    using Encode = decltype(&cuTensorMapEncodeTiled);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess) f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    if (!encode) return cudaErrorNotSupported;
    const uint32_t box_bytes = box_cols * (type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2);
    const cuuint64_t dims[3] = {cols, rows, count}, strides[2] = {row_bytes, row_bytes * rows};
    const cuuint32_t box[3] = {box_cols, box_rows, 1}, step[3] = {1, 1, 1};
    const CUresult r = encode(out, type, count ? 3 : 2, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              box_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t expired_waits_project(unsigned long long* out) { return cudaMemcpyFromSymbol(out, g_expired_waits, sizeof(*out)); }

cudaError_t launch_low_tc(const LowArgs* a, int count, int dtype, const int* after_pack, cudaStream_t s) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    return dtype == DT_BF16 ? low_tc<__nv_bfloat16>(a, count, after_pack, sms, s) : low_tc<__half>(a, count, after_pack, sms, s);
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
