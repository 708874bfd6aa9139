// A projection with an adapter for each row, for more rows than a decode batch
// (tvb_matmul_lora; lora.cu has the few-rows kernels).
//
// x is split once into F16 hi + lo planes with a power-of-two factor a row
// (pf_norm_split), so that F16 products are F32-faithful; the bound is the tensor
// pipe at twice the FLOPs of the projection.
//
// lora_shrink_tile_kernel (few values of t: lora_shrink_kernel, a CTA four of
// them): t[m] = scale_a A_a x[m] for 16 rows and 32 rank indexes a CTA.  x and A as
// TF32 hi + lo planes (any magnitude), three products of mma.sync m16n8k8; 8 warps,
// and the CTAs of a cluster, cut K.  Bound by the latency of its loads: 64 indexes
// a CTA, two CTAs an SM, made a call of 1400 rows 165 us, these make it 162.
// lora_gemm_kernel: 128 rows of x by 256 weight rows a tile, tcgen05 fed by TMA.
// The tensor core truncates to 24 bits as it accumulates (where all products are of
// one sign, 2^-25.4 of what a chain ends with, an MMA: 6e-7 in 30), so no chain is
// longer than 32: four k-blocks are summed in TMEM and added to registers by the
// epilogue warps while the next four go to the other half of TMEM.  After its
// k-blocks a tile takes one more such product per adapter among its rows (and 80
// rank indexes): t . B_a as TF32 hi + lo planes (any magnitude, three products), added to that adapter's
// rows alone, so one request's adapter never touches another's row, whatever it
// holds (few values of t: lora_expand_kernel does that, behind the join).  Every CTA takes an equal run of the tiles' chunks; a tile that a cut
// divides leaves F32 partial sums and lora_join_kernel adds them.
#include <algorithm>
#include <cooperative_groups.h>
#include <type_traits>

#include "lora.h"
#include "prefill.h"
#include "tcgen05.cuh"

namespace cg = cooperative_groups;

namespace tvb {

// ---- shrink -----------------------------------------------------------------------
constexpr int kLtWarps = 8, kLtRows = 16, kLtRanks = 32, kLtPerSm = 3;
// Steps of 16 k (6 products each) that the tensor core sums before the warp's sums in
// shared memory take them.  In one chain K 16384 lost 2e-5 of an adapter's product (now
// 1.3e-6); 1400 rows 2560 -> 6912 162.7 -> 164.1 us.
constexpr int kLtChain = 5;

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo, hi rounded to TF32 (11 bits), lo the rest (the product takes its first 11 bits)
__device__ __forceinline__ void tf32_planes(float x, uint32_t* hi, uint32_t* lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(*hi) : "f"(x));
    *lo = __float_as_uint(x - __uint_as_float(*hi));
}

// The next adapter after `prev` among ids[] (N a lane, -1 none), or INT_MAX.
template <int N>
__device__ __forceinline__ int next_adapter(const int (&ids)[N], int prev) {
    int v = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (ids[i] > prev) v = min(v, ids[i]);
    return __reduce_min_sync(0xffffffffu, v);
}

template <bool F16>
__device__ __forceinline__ float4 lora_load4(const void* p, size_t at) {
    if constexpr (F16) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const __half*>(p) + at));
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        return make_float4(x.x, x.y, y.x, y.y);
    } else {
        return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at));
    }
}

template <bool F16>
__global__ void __launch_bounds__(32 * kLtWarps, kLtPerSm) lora_shrink_tile_kernel(const __grid_constant__ LoraArgs a) {
    extern __shared__ float lt_red[];   // [warp][16 rows][kLtRanks + 1]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    cg::cluster_group cl = cg::this_cluster();   // its CTAs cut K
    const int rank = (int)cl.block_rank(), nsplit = (int)cl.num_blocks();
    const int m0 = blockIdx.y * kLtRows;
    int ids[1] = {-1}, rank_of = 0;
    if (lane < kLtRows && m0 + lane < a.M) ids[0] = lora_of(a, m0 + lane, &rank_of, warp == 0 && rank == 0 && blockIdx.z == 0);
    if (rank_of == 0) ids[0] = -1;
    const int parts = kLtWarps * nsplit, part = rank * kLtWarps + warp;
    const int steps = ((a.K + 15) / 16 + parts - 1) / parts;   // of 16 k, a warp
    const int s0 = part * steps, s1 = min(s0 + steps, (a.K + 15) / 16);
    for (int ad = next_adapter(ids, -1); ad != 0x7fffffff; ad = next_adapter(ids, ad)) {
        const int r = __ldg(a.rank + ad), j0 = blockIdx.z * kLtRanks;
        const void* A = a.A[ad];
        if (j0 < r) {
            const int nt = min(kLtRanks / 8, (r - j0 + 7) / 8);
            // the loads of a step (16 k) ahead of its arithmetic; k permuted so that a thread's fragments are 4
            // consecutive k
            float4 x[2], w[kLtRanks / 8];
            auto load_x = [&](int s, int h) {
                const int k = s * 16 + 4 * q, m = m0 + g + 8 * h;
                return s < s1 && k < a.K && m < a.M ? lora_load4<false>(a.x, (size_t)m * a.K + k) : make_float4(0.f, 0.f, 0.f, 0.f);
            };
            auto load_w = [&](int s, int n) {
                const int k = s * 16 + 4 * q, j = j0 + n * 8 + g;
                return s < s1 && k < a.K && j < r ? lora_load4<F16>(A, (size_t)j * a.K + k) : make_float4(0.f, 0.f, 0.f, 0.f);
            };
            x[0] = load_x(s0, 0), x[1] = load_x(s0, 1);
#pragma unroll
            for (int n = 0; n < kLtRanks / 8; ++n)
                if (n < nt) w[n] = load_w(s0, n);
            float* red = lt_red + warp * kLtRows * (kLtRanks + 1);
            int c = s0;
#pragma unroll 1
            do {
                float acc[kLtRanks / 8][4] = {};
#pragma unroll 1
                for (int s = c; s < min(c + kLtChain, s1); ++s) {
                    uint32_t xh[2][4], xl[2][4];   // [8 k][fragment]
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float v[4] = {x[h].x, x[h].y, x[h].z, x[h].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) tf32_planes(v[e], &xh[e >> 1][h + 2 * (e & 1)], &xl[e >> 1][h + 2 * (e & 1)]);
                        x[h] = load_x(s + 1, h);
                    }
#pragma unroll
                    for (int n = 0; n < kLtRanks / 8; ++n) {
                        if (n < nt) {
                            const float v[4] = {w[n].x, w[n].y, w[n].z, w[n].w};
                            uint32_t wh[4], wl[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) tf32_planes(v[e], &wh[e], &wl[e]);
                            w[n] = load_w(s + 1, n);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                mma_tf32(acc[n], xl[i], wh[2 * i], wh[2 * i + 1]);
                                mma_tf32(acc[n], xh[i], wl[2 * i], wl[2 * i + 1]);
                                mma_tf32(acc[n], xh[i], wh[2 * i], wh[2 * i + 1]);
                            }
                        }
                    }
                }
                // to this warp's sums
#pragma unroll
                for (int n = 0; n < kLtRanks / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float* to = red + (g + 8 * (e >> 1)) * (kLtRanks + 1) + n * 8 + 2 * q + (e & 1);
                        *to = c > s0 ? *to + acc[n][e] : acc[n][e];
                    }
                c += kLtChain;
            } while (c < s1);
            if (nsplit > 1) cl.sync();
            else __syncthreads();
            // the cluster's CTAs share the rows; sums in the order of K
            const float scale = __ldg(a.scale + ad);
            for (int i = rank * 32 * kLtWarps + threadIdx.x; i < kLtRows * kLtRanks; i += nsplit * 32 * kLtWarps) {
                const int m = i / kLtRanks, j = i % kLtRanks;
                const bool mine = m0 + m < a.M && __ldg(a.adapter + m0 + m) == ad && j0 + j < r;
                if (!mine) continue;
                float s = 0.f;
                for (int p = 0; p < nsplit; ++p) {
                    const float* from = cl.map_shared_rank(lt_red, p);
#pragma unroll
                    for (int w = 0; w < kLtWarps; ++w) s += from[(w * kLtRows + m) * (kLtRanks + 1) + j];
                }
                a.t[(size_t)(m0 + m) * a.max_rank + j0 + j] = s * scale;
            }
            if (nsplit > 1) cl.sync();
            else __syncthreads();
        }
    }
}

// ---- projection ---------------------------------------------------------------------
constexpr int kLgRows = 128, kLgCols = 256, kLgStages = 3, kLgChunk = 4;   // k-blocks a chunk
constexpr int kLgSoft = 8, kLgThreads = 384;
constexpr int kLgExtra = 2;   // what starting and leaving a tile costs, in chunks
constexpr int kLgPlane = kLgRows * 128, kLgStage = 2 * kLgPlane + kLgCols * 128;
constexpr int kLgLora = 2 * (kLgRows + kLgCols) * 32;   // t hi, lo, B hi, lo of 8 rank indexes

struct LgShared {
    uint64_t full[kLgStages], empty[kLgStages];
    uint64_t acc_full[2], acc_empty[2];
    uint64_t l_full, l_empty, drained;
    uint32_t tmem;
    int abort;
};
constexpr int kLgSmem = kLgStages * kLgStage + kLgLora + (int)sizeof(LgShared) + 1024;

struct LgMaps {
    CUtensorMap xh, xl, w;
};

struct LgPlan {
    int mt, tiles;      // tiles of rows, of both
    int nk, chunks;     // k-blocks, chunks a tile
    int ctas;
    int fused;          // the adapters' products are lora_gemm_kernel's too
    const int* row_exp;
    float* part;        // [CTA][2][128][256]
};

struct LgPiece {
    int m0, n0, c0, c1, slot, last_cta;
};

// The next piece from unit *u on: a tile's chunks [c0, c1).  A tile is kLgExtra +
// chunks units; CTA c takes [T c / G, T (c + 1) / G) of them.
__device__ __forceinline__ int64_t lg_begin(const LgPlan& p, int c) {
    return (int64_t)p.tiles * (p.chunks + kLgExtra) * c / p.ctas;
}
__device__ __forceinline__ bool lg_next(const LgPlan& p, int64_t* u, int64_t end, LgPiece* out) {
    const int per = p.chunks + kLgExtra;
    while (*u < end) {
        const int tile = (int)(*u / per), r = (int)(*u - (int64_t)tile * per);
        const int e = (int)min((int64_t)per, r + (end - *u)), b = max(r, kLgExtra);
        *u = (int64_t)tile * per + e;
        if (b >= e) continue;
        out->m0 = tile % p.mt * kLgRows;
        out->n0 = tile / p.mt * kLgCols;
        out->c0 = b - kLgExtra;
        out->c1 = e - kLgExtra;
        out->slot = out->c1 - out->c0 == p.chunks ? -1 : out->c0 > 0 ? 0 : 1;
        out->last_cta = (int)((((int64_t)tile + 1) * per * p.ctas - 1) / ((int64_t)p.tiles * per));
        return true;
    }
    return false;
}

__device__ __forceinline__ uint64_t sw32_desc(uint32_t saddr) {   // K-major, rows of 32 bytes, 8-row groups 256 apart
    uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)1u << 16;
    d |= (uint64_t)(256u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)6u << 61;
    return d;
}
__device__ __forceinline__ uint32_t sw32_offset(int row, int chunk) { return (uint32_t)(row * 32 + ((chunk ^ ((row >> 2) & 1)) * 16)); }

__device__ __forceinline__ void tc_mma_tf32(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// kind::tf32: D F32, A and B TF32 (2), both K-major
constexpr uint32_t umma_idesc_tf32(int M, int N) {
    return (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ uint64_t lg_pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 lg_unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t lg_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ void lg_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Steps of 8 rank indexes of an adapter, and how many the tensor core sums (3 products each).
constexpr int kLgRankSteps = 10;
__device__ __forceinline__ int lg_steps(const LoraArgs& a, int ad) { return (__ldg(a.rank + ad) + 7) / 8; }

// The adapters of rows [m0, m0 + 128): 4 rows a lane.
__device__ __forceinline__ void lg_ids(const LoraArgs& a, int m0, int (&ids)[4]) {
    const int lane = threadIdx.x & 31;
    int r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + lane * 4 + i;
        ids[i] = m < a.M ? lora_of(a, m, &r, false) : -1;
        if (ids[i] >= 0 && r == 0) ids[i] = -1;
    }
}

__global__ void __launch_bounds__(kLgThreads, 1)
lora_gemm_kernel(const __grid_constant__ LgMaps maps, const __grid_constant__ LoraArgs a, const __grid_constant__ LgPlan plan) {
    extern __shared__ unsigned char lg_raw[];
    const uint32_t raw = smem_u32(lg_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* smem = lg_raw + (base - raw);
    LgShared& sh = *reinterpret_cast<LgShared*>(smem + kLgStages * kLgStage + kLgLora);
    const uint32_t lora_s = base + kLgStages * kLgStage;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kLgStages; ++i) {
            mbar_init(sh.full + i, 1);
            mbar_init(sh.empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(sh.acc_full + i, 1);
            mbar_init(sh.acc_empty + i, kLgSoft);
        }
        mbar_init(&sh.l_full, 2);
        mbar_init(&sh.l_empty, 1);
        mbar_init(&sh.drained, 1);
        sh.abort = 0;
        fence_barrier_init();
    }
    if (warp == 9) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    volatile int* abort_flag = &sh.abort;
    auto fail = [&]() {
        *abort_flag = 1;
        if (a.status) atomicOr(a.status, TVB_DEV_TIMEOUT);
    };
    pdl_wait();   // the planes and t come from the kernels before
    int64_t u = lg_begin(plan, blockIdx.x);
    const int64_t end = lg_begin(plan, blockIdx.x + 1);
    LgPiece p;

    // registers: 128 x (200 + 200 + 104) = 384 x 168, what the CTA was launched with
    if (warp >= kLgSoft) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == 8) {
            // ---- TMA producer -----------------------------------------------------
            if (lane == 0) {
                prefetch_tmap(&maps.xh);
                prefetch_tmap(&maps.xl);
                prefetch_tmap(&maps.w);
                int it = 0;
                bool ok = true;
                while (ok && lg_next(plan, &u, end, &p)) {
                    for (int kb = p.c0 * kLgChunk; kb < min(plan.nk, p.c1 * kLgChunk); ++kb, ++it) {
                        const int s = it % kLgStages;
                        ok = mbar_wait_bounded(sh.empty + s, (uint32_t)((it / kLgStages + 1) & 1)) && !*abort_flag;
                        if (!ok) break;
                        const uint32_t st = base + s * kLgStage;
                        mbar_expect_tx(sh.full + s, kLgStage);
                        tma_load_2d(st, &maps.xh, kb * 64, p.m0, sh.full + s);
                        tma_load_2d(st + kLgPlane, &maps.xl, kb * 64, p.m0, sh.full + s);
                        tma_load_2d(st + 2 * kLgPlane, &maps.w, kb * 64, p.n0, sh.full + s);
                    }
                }
                if (!ok) {
                    fail();
                    // no TMA write may outlive the CTA
                    for (int i = max(0, it - kLgStages); i < it; ++i)
                        mbar_wait_bounded(sh.full + i % kLgStages, (uint32_t)((i / kLgStages) & 1));
                }
            }
        } else if (warp == 9) {
            // ---- MMA issuer ----------------------------------------------------------
            constexpr uint32_t idesc = umma_idesc_f16(kLgRows, kLgCols), idesc_l = umma_idesc_tf32(kLgRows, kLgCols);
            int it = 0, chunk = 0, ls = 0;
            bool ok = true;
            while (ok && lg_next(plan, &u, end, &p)) {
                if (lane == 0) {
                    for (int c = p.c0; ok && c < p.c1; ++c, ++chunk) {
                        const uint32_t d = tmem + (chunk & 1) * kLgCols;
                        ok = chunk < 2 || mbar_wait_bounded(sh.acc_empty + (chunk & 1), (uint32_t)(((chunk - 2) >> 1) & 1));
                        tc_fence_after();
                        const int k1 = min(plan.nk, (c + 1) * kLgChunk);
                        for (int kb = c * kLgChunk; ok && kb < k1; ++kb, ++it) {
                            const int s = it % kLgStages;
                            ok = mbar_wait_bounded(sh.full + s, (uint32_t)((it / kLgStages) & 1));
                            if (!ok) break;
                            tc_fence_after();
                            const uint64_t x = sw128_desc(base + s * kLgStage), w = sw128_desc(base + s * kLgStage + 2 * kLgPlane);
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) {
                                tc_mma(d, x + kk * 2, w + kk * 2, idesc, (kb != c * kLgChunk || kk) ? 1u : 0u);
                                tc_mma(d, x + (kLgPlane >> 4) + kk * 2, w + kk * 2, idesc, 1u);
                            }
                            tc_commit(sh.empty + s);
                        }
                        if (ok) tc_commit(sh.acc_full + (chunk & 1));
                    }
                }
                chunk = __shfl_sync(0xffffffffu, chunk, 0);
                ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                if (ok && plan.fused && p.c0 == 0) {
                    int ids[4];
                    lg_ids(a, p.m0, ids);
                    for (int ad = next_adapter(ids, -1); ok && ad != 0x7fffffff; ad = next_adapter(ids, ad)) {
                        const int steps = lg_steps(a, ad);
                        if (lane == 0) {
                            for (int s = 0; ok && s < steps; ++s) {
                                const uint32_t d = tmem + (chunk & 1) * kLgCols;
                                const bool begin = s % kLgRankSteps == 0;
                                if (begin) ok = chunk < 2 || mbar_wait_bounded(sh.acc_empty + (chunk & 1), (uint32_t)(((chunk - 2) >> 1) & 1));
                                ok = ok && mbar_wait_bounded(&sh.l_full, (uint32_t)((ls + s) & 1));
                                if (!ok) break;
                                tc_fence_after();
                                const uint64_t th = sw32_desc(lora_s), tl = th + (kLgRows * 32 >> 4);
                                const uint64_t bh = th + (2 * kLgRows * 32 >> 4), bl = bh + (kLgCols * 32 >> 4);
                                tc_mma_tf32(d, th, bh, idesc_l, begin ? 0u : 1u);
                                tc_mma_tf32(d, th, bl, idesc_l, 1u);
                                tc_mma_tf32(d, tl, bh, idesc_l, 1u);
                                tc_commit(&sh.l_empty);
                                if (s + 1 == steps || (s + 1) % kLgRankSteps == 0) tc_commit(sh.acc_full + (chunk++ & 1));
                            }
                        }
                        ls += steps;
                        chunk = __shfl_sync(0xffffffffu, chunk, 0);
                        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                    }
                }
            }
            if (lane == 0) {
                if (!ok) fail();
                tc_commit(&sh.drained);
                mbar_wait_bounded(&sh.drained, 0u);
            }
            __syncwarp();
        } else if (plan.fused) {
            // ---- adapters: 8 rank indexes of t and B a step, as TF32 hi + lo ------------
            const int tid = threadIdx.x - 320;   // 0 .. 63
            int ls = 0;
            bool ok = true;
            while (ok && lg_next(plan, &u, end, &p)) {
                if (p.c0 != 0) continue;
                int ids[4];
                lg_ids(a, p.m0, ids);
                // the tile's adapters, 32 at a time: lane i has the i-th's rank and factor
                for (int ad = -1; ok && ad != 0x7fffffff;) {
                    int mine = -1, count = 0;
                    while (count < 32 && (ad = next_adapter(ids, ad)) != 0x7fffffff) {
                        if (lane == count) mine = ad;
                        ++count;
                    }
                    const int my_rank = mine >= 0 ? __ldg(a.rank + mine) : 0;
                    const void* my_B = mine >= 0 ? a.B[mine] : nullptr;
                    for (int c = 0, j0 = 0; c < count; ++ls) {
                        const int rank = __shfl_sync(0xffffffffu, my_rank, c);
                        const void* B = reinterpret_cast<const void*>(__shfl_sync(0xffffffffu, reinterpret_cast<uintptr_t>(my_B), c));
                        // this thread's rows: two of t, four of B, 8 values each; nothing waits for a load before all
                        // are under way
                        float4 v[6][2];
                        const bool vec = rank % 4 == 0;
#pragma unroll
                        for (int i = 0; i < 6; ++i) {
                            const int row = i < 2 ? p.m0 + i * 64 + tid : p.n0 + (i - 2) * 64 + tid;
                            const bool in = i < 2 ? row < a.M : row < a.N;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int j = j0 + 4 * h;
                                v[i][h] = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (i < 2) {
                                    if (in && j < rank) v[i][h] = *reinterpret_cast<const float4*>(a.t + (size_t)row * a.max_rank + j);
                                } else if (vec) {
                                    if (in && j < rank)
                                        v[i][h] = a.f16 ? lora_load4<true>(B, (size_t)row * rank + j) : lora_load4<false>(B, (size_t)row * rank + j);
                                }
                            }
                        }
                        if (!vec) {
#pragma unroll
                            for (int i = 2; i < 6; ++i) {
                                const int row = p.n0 + (i - 2) * 64 + tid;
                                float f[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    f[e] = row < a.N && j0 + e < rank ? lora_elem(B, (size_t)row * rank + j0 + e, a.f16) : 0.f;
                                v[i][0] = make_float4(f[0], f[1], f[2], f[3]);
                                v[i][1] = make_float4(f[4], f[5], f[6], f[7]);
                            }
                        }
                        ok = __all_sync(0xffffffffu, (ls == 0 || mbar_wait_bounded(&sh.l_empty, (uint32_t)((ls - 1) & 1))) && !*abort_flag);
                        if (!ok) break;
#pragma unroll
                        for (int i = 0; i < 6; ++i) {
                            unsigned char* hi = smem + kLgStages * kLgStage + (i < 2 ? 0 : 2 * kLgRows * 32);
                            const int rr = (i < 2 ? i : i - 2) * 64 + tid, lo = (i < 2 ? kLgRows : kLgCols) * 32;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float f[4] = {v[i][h].x, v[i][h].y, v[i][h].z, v[i][h].w};
                                uint32_t x[4], y[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {   // t ends with the rank
                                    tf32_planes(i < 2 && j0 + 4 * h + e >= rank ? 0.f : f[e], &x[e], &y[e]);
                                }
                                *reinterpret_cast<uint4*>(hi + sw32_offset(rr, h)) = make_uint4(x[0], x[1], x[2], x[3]);
                                *reinterpret_cast<uint4*>(hi + lo + sw32_offset(rr, h)) = make_uint4(y[0], y[1], y[2], y[3]);
                            }
                        }
                        fence_proxy_async_smem_cta();
                        __syncwarp();
                        if (lane == 0) lg_arrive(&sh.l_full);
                        j0 += 8;
                        if (j0 >= rank) j0 = 0, ++c;
                    }
                }
            }
            if (!ok && lane == 0) fail();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        // ---- epilogue: two threads a row, 128 columns each, in registers ------------------
        const int r = threadIdx.x & 127, half = warp >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + half * 128;
        int chunk = 0;
        bool ok = true;
        while (lg_next(plan, &u, end, &p)) {   // (after a wait that gave up: NaN)
            const int m = p.m0 + r;
            const bool live = m < a.M;
            const float f = live ? ldexpf(1.0f, __ldg(plan.row_exp + m)) : 0.f;
            uint64_t acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0ull;
            auto add = [&](uint64_t f2, bool mine) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(sh.acc_full + (chunk & 1), (uint32_t)((chunk >> 1) & 1)) && !*abort_flag);
                if (!ok) return;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld32(lanes + (chunk & 1) * kLgCols + c * 32, v);
                    tmem_wait_ld();
                    if (mine) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            acc[c * 16 + i] = lg_fma2(lg_pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), f2, acc[c * 16 + i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) lg_arrive(sh.acc_empty + (chunk & 1));
                ++chunk;
            };
            const uint64_t f2 = lg_pack2(f, f), one = lg_pack2(1.f, 1.f);
#pragma unroll 1
            for (int c = p.c0; ok && c < p.c1; ++c) add(f2, true);
            const int n0 = p.n0 + half * 128;
            if (a.w8 && ok) {   // INT8: the weight rows' scales
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    const int n = n0 + 2 * i;
                    const float s0 = a.row_scales ? (n < a.N ? __ldg(a.row_scales + n) : 0.f) : a.tscale;
                    const float s1 = a.row_scales ? (n + 1 < a.N ? __ldg(a.row_scales + n + 1) : 0.f) : a.tscale;
                    acc[i] = lg_fma2(acc[i], lg_pack2(s0, s1), 0ull);
                }
            }
            if (ok && plan.fused && p.c0 == 0) {
                int ids[4], rank;
                lg_ids(a, p.m0, ids);
                const int id = live ? lora_of(a, m, &rank, false) : -1;
#pragma unroll 1
                for (int ad = next_adapter(ids, -1); ok && ad != 0x7fffffff; ad = next_adapter(ids, ad))
                    for (int left = lg_steps(a, ad); ok && left > 0; left -= kLgRankSteps) add(one, ad == id);
            }
            if (!ok) {
#pragma unroll
                for (int i = 0; i < 64; ++i) acc[i] = lg_pack2(NAN, NAN);
            }
            if (p.slot >= 0) {
                float* to = plan.part + ((size_t)(blockIdx.x * 2 + p.slot) * kLgRows + r) * kLgCols + half * 128;
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const float2 x = lg_unpack2(acc[i]), y = lg_unpack2(acc[i + 1]);
                    *reinterpret_cast<float4*>(to + 2 * i) = make_float4(x.x, x.y, y.x, y.y);
                }
            } else if (live) {
                float* to = a.y + (size_t)m * a.N + n0;
                if (n0 + 128 <= a.N && a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0) {
#pragma unroll
                    for (int i = 0; i < 64; i += 2) {
                        const float2 x = lg_unpack2(acc[i]), y = lg_unpack2(acc[i + 1]);
                        *reinterpret_cast<float4*>(to + 2 * i) = make_float4(x.x, x.y, y.x, y.y);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        const float2 x = lg_unpack2(acc[i]);
                        if (n0 + 2 * i < a.N) to[2 * i] = x.x;
                        if (n0 + 2 * i + 1 < a.N) to[2 * i + 1] = x.y;
                    }
                }
            }
        }
        if (!ok) fail();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Adds the pieces of the tile that CTA blockIdx.x of lora_gemm_kernel began and
// another ended, in order; 8 rows a CTA here.
__global__ void __launch_bounds__(256) lora_join_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ LgPlan plan) {
    pdl_wait();
    const int c0 = blockIdx.x;
    int64_t u = lg_begin(plan, c0);
    const int64_t end = lg_begin(plan, c0 + 1);
    LgPiece p;
    p.slot = -1;
    const int64_t per = plan.chunks + kLgExtra, start = (end - 1) / per * per;   // the run's last tile
    if (end <= u || start < u - kLgExtra) return;
    u = max(u, start);
    if (!lg_next(plan, &u, end, &p) || p.slot != 1) return;
    for (int r = blockIdx.y * 8 + (threadIdx.x >> 6); r < (int)blockIdx.y * 8 + 8; r += 4) {
        const int m = p.m0 + r, col = (threadIdx.x & 63) * 4;
        if (m >= a.M) return;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = c0; c <= p.last_cta; ++c) {
            const float4 v = *reinterpret_cast<const float4*>(plan.part + ((size_t)(c * 2 + (c == c0)) * kLgRows + r) * kLgCols + col);
            s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
        }
        const float f[4] = {s.x, s.y, s.z, s.w};
        float* to = a.y + (size_t)m * a.N + p.n0 + col;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (p.n0 + col + e < a.N) to[e] = f[e];
    }
}

// ---- expand ------------------------------------------------------------------------
// y[m] += B_a t[m] on the CUDA cores, a CTA `rows` rows (at most kLeRows) of 256
// columns, two a thread: the rows' adapters one after another, 32 rank indexes of
// their B rows in registers, t broadcast from shared memory.
// For few values of t: lora_gemm_kernel's own products cost a step for every
// adapter of a tile, this a pass over y for every 32 rank indexes.  2560 -> 6912,
// 8 adapters of rank 16 mixed: 128 rows 58 against 85 us, 512 rows 94 against 120;
// 2 of rank 64 in runs: 128 rows 66 against 56, 256 rows 93 against 65.
constexpr int kLeMaxValues = 8192;   // rows x largest rank
constexpr int kLeThreads = 128, kLeRows = 64, kLeRanks = 32, kLeGroup = 4, kLePerSm = 4;

template <bool F16>
__global__ void __launch_bounds__(kLeThreads, kLePerSm) lora_expand_kernel(const __grid_constant__ LoraArgs a, int rows) {
    __shared__ __align__(16) float ts[kLeRows + 2 * kLeGroup][kLeRanks];   // (pairs of groups are read)
    __shared__ int list[kLeRows], ids_s[kLeRows], count;
    pdl_wait();
    const int tid = threadIdx.x, m0 = blockIdx.y * rows, n0 = blockIdx.x * 2 * kLeThreads + tid;
    {
        int r = 0, id = -1;
        if (tid < rows && m0 + tid < a.M) id = lora_of(a, m0 + tid, &r, false);
        if (tid < kLeRows) ids_s[tid] = r > 0 ? id : -1;
    }
    __syncthreads();
    int ids[kLeRows / 32];
#pragma unroll
    for (int i = 0; i < kLeRows / 32; ++i) ids[i] = ids_s[i * 32 + (tid & 31)];
    for (int ad = next_adapter(ids, -1); ad != 0x7fffffff; ad = next_adapter(ids, ad)) {
        const int r = __ldg(a.rank + ad);
        const void* B = a.B[ad];
        __syncthreads();   // the list was read
        if (tid < 32) {    // the adapter's rows, in order
            int n = 0;
#pragma unroll
            for (int i = 0; i < kLeRows / 32; ++i) {
                const unsigned at = __ballot_sync(0xffffffffu, ids[i] == ad);
                if (ids[i] == ad) list[n + __popc(at & ((1u << tid) - 1))] = i * 32 + tid;
                n += __popc(at);
            }
            if (tid == 0) count = n;
        }
        for (int j0 = 0; j0 < r; j0 += kLeRanks) {
            const int rj = min(kLeRanks, r - j0);
            // 32 rank indexes of rows n0, n0 + 128 of B, as pairs
            uint64_t b[2][kLeRanks / 2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int n = n0 + c * kLeThreads;
                const size_t at = (size_t)n * r + j0;
#pragma unroll
                for (int j = 0; j < kLeRanks; j += 4) {
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (n < a.N && j < rj) {
                        if (r % 4 == 0) {
                            x = lora_load4<F16>(B, at + j);
                        } else {
                            x.x = lora_elem(B, at + j, F16);
                            if (j + 1 < rj) x.y = lora_elem(B, at + j + 1, F16);
                            if (j + 2 < rj) x.z = lora_elem(B, at + j + 2, F16);
                            if (j + 3 < rj) x.w = lora_elem(B, at + j + 3, F16);
                        }
                    }
                    b[c][j / 2] = lg_pack2(x.x, x.y);
                    b[c][j / 2 + 1] = lg_pack2(x.z, x.w);
                }
            }
            __syncthreads();   // the list is there; t of the step before was read
            const int n = count;
            for (int i = tid; i < n * kLeRanks; i += kLeThreads) {
                const int k = i / kLeRanks, j = i % kLeRanks;
                ts[k][j] = j < rj ? a.t[(size_t)(m0 + list[k]) * a.max_rank + j0 + j] : 0.f;
            }
            __syncthreads();
            // four rows at a time, the next four's y under way
            float* const y = a.y + (size_t)m0 * a.N + n0;
            const bool in[2] = {n0 < a.N, n0 + kLeThreads < a.N};
            auto fetch = [&](int k, float (&v)[kLeGroup][2]) {
#pragma unroll
                for (int i = 0; i < kLeGroup; ++i)
#pragma unroll
                    for (int c = 0; c < 2; ++c) v[i][c] = k + i < n && in[c] ? y[(size_t)list[k + i] * a.N + c * kLeThreads] : 0.f;
            };
            // (ranks of t and B behind rj are zero)
            auto add = [&](auto ranks, int k, const float (&v)[kLeGroup][2]) {
                uint64_t s[kLeGroup][2];
#pragma unroll
                for (int i = 0; i < kLeGroup; ++i) s[i][0] = s[i][1] = 0ull;
#pragma unroll
                for (int j = 0; j < decltype(ranks)::value; j += 4) {
#pragma unroll
                    for (int i = 0; i < kLeGroup; ++i) {
                        const float4 x = *reinterpret_cast<const float4*>(&ts[k + i][j]);
                        const uint64_t x0 = lg_pack2(x.x, x.y), x1 = lg_pack2(x.z, x.w);
#pragma unroll
                        for (int c = 0; c < 2; ++c) s[i][c] = lg_fma2(b[c][j / 2 + 1], x1, lg_fma2(b[c][j / 2], x0, s[i][c]));
                    }
                }
#pragma unroll
                for (int i = 0; i < kLeGroup; ++i)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float2 z = lg_unpack2(s[i][c]);
                        if (k + i < n && in[c]) y[(size_t)list[k + i] * a.N + c * kLeThreads] = v[i][c] + (z.x + z.y);
                    }
            };
            auto rows_of = [&](auto ranks) {
                float u[kLeGroup][2], v[kLeGroup][2];
                fetch(0, u);
#pragma unroll 1
                for (int k = 0; k < n; k += 2 * kLeGroup) {
                    fetch(k + kLeGroup, v);
                    add(ranks, k, u);
                    fetch(k + 2 * kLeGroup, u);
                    add(ranks, k + kLeGroup, v);
                }
            };
            if (rj <= 8) rows_of(std::integral_constant<int, 8>());
            else if (rj <= 16) rows_of(std::integral_constant<int, 16>());
            else rows_of(std::integral_constant<int, kLeRanks>());
        }
    }
}

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

tvb_status lora_many_rows(LoraArgs a, cudaStream_t st) {
    TVB_REQUIRE(a.K <= kLoraMaxK, "matmul_lora: K=%d with %d rows (at most %d above 256 rows)", a.K, a.M, kLoraMaxK);
    LgPlan plan = {};
    plan.mt = (a.M + kLgRows - 1) / kLgRows;
    plan.tiles = plan.mt * ((a.N + kLgCols - 1) / kLgCols);
    plan.nk = (a.K + 63) / 64;
    plan.chunks = (plan.nk + kLgChunk - 1) / kLgChunk;
    // every SM, unless a run would be shorter than what a tile costs by itself
    plan.ctas = (int)std::max<int64_t>(1, std::min<int64_t>(num_sms(), (int64_t)plan.tiles * (plan.chunks + kLgExtra) / (kLgExtra + 1)));
    const size_t plane = align256((size_t)a.M * a.K * 2), wide = a.w8 ? align256((size_t)a.N * a.K * 2) : 0;
    const size_t exps = align256((size_t)a.M * 4), ts = align256((size_t)a.M * a.max_rank * 4);
    const size_t parts = (size_t)plan.ctas * 2 * kLgRows * kLgCols * 4;
    Workspace ws(st);
    TVB_TRY(ws.get(2 * plane + wide + exps + ts + parts));
    uint16_t *xh = ws.at<uint16_t>(), *xl = ws.at<uint16_t>(plane), *w16 = ws.at<uint16_t>(2 * plane);
    int* row_exp = ws.at<int>(2 * plane + wide);
    a.t = ws.at<float>(2 * plane + wide + exps);
    plan.row_exp = row_exp;
    plan.part = ws.at<float>(2 * plane + wide + exps + ts);
    const uint16_t* w = a.w8 ? w16 : static_cast<const uint16_t*>(a.w);
    if (a.w8) TVB_TRY(pf_i8_to_f16(static_cast<const int8_t*>(a.w), (size_t)a.N * a.K, w16, st));
    plan.fused = a.n && (int64_t)a.M * a.max_rank > kLeMaxValues;
    if (a.n && !plan.fused) {
        TVB_TRY(lora_shrink_rows(a, st));
    } else if (a.n) {
        static int set[2][kMaxDevices];
        constexpr int smem = kLtWarps * kLtRows * (kLtRanks + 1) * 4;
        const auto kernel = a.f16 ? lora_shrink_tile_kernel<true> : lora_shrink_tile_kernel<false>;
        TVB_TRY(allow_smem(reinterpret_cast<const void*>(kernel), smem, set[a.f16]));
        const int rows = (a.M + kLtRows - 1) / kLtRows;
        const int slices = (a.max_rank + kLtRanks - 1) / kLtRanks;
        int nsplit = 1;   // CTAs that cut K: while the SMs hold them all
        while (nsplit < 8 && (int64_t)rows * slices * nsplit * 2 <= kLtPerSm * num_sms()) nsplit *= 2;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)nsplit, (unsigned)rows, (unsigned)slices);
        cfg.blockDim = dim3(32 * kLtWarps);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)nsplit;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        TVB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
        TVB_TRY(check_launch("lora_shrink_tile_kernel"));
    }
    TVB_TRY(pf_norm_split(a.x, nullptr, a.M, a.K, 0.f, xh, xl, row_exp, st));
    LgMaps maps;
    const uint64_t xd[2] = {(uint64_t)a.K, (uint64_t)a.M}, wd[2] = {(uint64_t)a.K, (uint64_t)a.N}, stride[1] = {(uint64_t)a.K * 2};
    const uint32_t xb[2] = {64u, (uint32_t)kLgRows}, wb[2] = {64u, (uint32_t)kLgCols};
    TVB_TRY(encode_f16_tiled(&maps.xh, xh, 2, xd, stride, xb));
    TVB_TRY(encode_f16_tiled(&maps.xl, xl, 2, xd, stride, xb));
    TVB_TRY(encode_f16_tiled(&maps.w, w, 2, wd, stride, wb));
    static int set[kMaxDevices];
    TVB_TRY(allow_smem(reinterpret_cast<const void*>(lora_gemm_kernel), kLgSmem, set));
    lora_gemm_kernel<<<(unsigned)plan.ctas, kLgThreads, kLgSmem, st>>>(maps, a, plan);
    TVB_TRY(check_launch("lora_gemm_kernel"));
    TVB_CUDA(launch_maybe_pdl(lora_join_kernel, dim3((unsigned)plan.ctas, kLgRows / 8), dim3(256), 0, st, true, a, plan));
    TVB_TRY(check_launch("lora_join_kernel"));
    if (!a.n || plan.fused) return TVB_OK;
    const unsigned cols = (unsigned)((a.N + 2 * kLeThreads - 1) / (2 * kLeThreads));
    // row blocks that fill the SMs once
    const int blocks = std::max(1, std::min((a.M + kLeGroup - 1) / kLeGroup, kLePerSm * num_sms() / (int)cols));
    const int rows = std::min(kLeRows, (a.M + blocks - 1) / blocks);
    const auto expand = a.f16 ? lora_expand_kernel<true> : lora_expand_kernel<false>;
    TVB_CUDA(launch_maybe_pdl(expand, dim3(cols, (unsigned)((a.M + rows - 1) / rows)), dim3(kLeThreads), 0, st, true, a, rows));
    return check_launch("lora_expand_kernel");
}

}  // namespace tvb
