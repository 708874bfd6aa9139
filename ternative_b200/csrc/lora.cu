// Adapters of many requests beside a shared projection (tvb_matmul_lora):
//   y[m] = W x[m] + scale_a B_a (A_a x[m]),  a = adapter[m]
//
// A decode batch is bound by the bytes of W and of the adapters in use, and by how
// fast weights reach the warps from L2:
//
// lora_shrink_kernel: t[m] = scale_a A_a x[m], a warp a (row, rank index).
// lora_rows_kernel: W streamed once for 16 rows through mma.sync m16n8k16 (rows
// of x are the 16-row operand and 8 weight rows the other, or, up to 8 rows, 16
// weight rows and x's; a memory-bound product that needs no more than the legacy
// tensor path).  More rows are blocks of 16 that share
// the GPU and walk the weights together, so that HBM gives them once and L2 the
// other times.  The many-rows kernels (lora_gemm.cu) take over where that would be
// more than 80 MB, or behind 256 rows: 2560 -> 6912 (35 MB) with 8 adapters of rank
// 16 among 32, 48, 64 rows 26, 34, 43 against 47, 48, 49 us, without adapters 20,
// 28, 36 against 28, 29, 29; 4096 -> 14336 (117 MB) 32 rows 113 against 67; 512 ->
// 512 256 rows 13 against 40.  x is split into F16 hi + lo
// planes with a power-of-two factor a row, so products are F32-faithful; each
// warp keeps its K slice of x in registers for the whole kernel and weights come
// straight from global memory in the operand's layout: with k permuted so that a
// thread's fragments of 2 or 4 steps are 16 contiguous bytes of a weight row.
// The CTA's warps cut K, and the CTAs of a cluster cut it further; partial sums
// meet in shared memory (distributed over the cluster), then the epilogue scales
// INT8 rows and adds t . B_a.  It is launched as the shrink kernel's dependent,
// which hides its launch; letting it start beside the shrink's CTAs was slower: the
// clusters that then found no room ran as a second wave (8 rows 4096 -> 14336: 48 us
// against 33).
#include "lora.h"

#include <algorithm>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace tvb {

constexpr int kLrWarps = 8, kLrThreads = 32 * kLrWarps;
// Largest K slice of a warp: what two CTAs an SM (one: INT8 and WIDE) have registers
// for.  (F16 and WIDE with one CTA and 160: 16 rows 4096 -> 14336 38.8 against 35.4 us.)
__host__ __device__ constexpr int lr_slice(bool w8, bool wide) { return w8 || !wide ? 128 : 96; }
// Weight rows a tile: what keeps enough loads under way (a warp's slice of an INT8
// row is half as many bytes).
__host__ __device__ constexpr int lr_cols(bool w8) { return w8 ? 32 : 16; }
// Distance of x's rows in a warp's sums of a tile: no bank conflicts as they are stored.
__host__ __device__ constexpr int lr_line(bool w8, bool wide) { return lr_cols(w8) + (wide ? 1 : 4); }
__host__ __device__ constexpr int lr_batch(bool w8) { return w8 ? 2 : 4; }   // tiles between two barriers of the CTA
// Tiles of weights under way in a warp's registers.  INT8 tiles are half the bytes;
// where one CTA has the SM to itself there are registers for two (64 rows 6912 ->
// 2560 51 -> 45 us, 16 rows 15.7 -> 14.2; F16 tiles gain nothing).
__host__ __device__ constexpr int lr_depth(bool w8, bool wide) { return w8 && wide ? 2 : 1; }
constexpr int kLrMaxSplit = 8;     // CTAs of a cluster
constexpr int kLrRows = 16;        // rows of x a CTA
constexpr int kLrMaxRows = 256;
constexpr int64_t kLrMaxAgain = 80 << 20;   // bytes of W that blocks of 16 rows read from L2

// A CTA takes 4 rank indexes of a row; its 8 warps cut K (8 k a lane), so that all
// loads of a short K are in flight at once.
constexpr int kLsRanks = 4;

template <bool F16>
__device__ __forceinline__ void lora_load8(const void* p, size_t at, float (&f)[8]) {
    if constexpr (F16) {
        h8_to_f8(__ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(p) + at)), f);
    } else {
        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
        const float4 x = __ldg(q), y = __ldg(q + 1);
        f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w, f[4] = y.x, f[5] = y.y, f[6] = y.z, f[7] = y.w;
    }
}

template <bool F16>
__global__ void __launch_bounds__(256) lora_shrink_kernel(const __grid_constant__ LoraArgs a) {
    __shared__ float part[8][kLsRanks];
    const int m = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int rank;
    const int ad = lora_of(a, m, &rank, blockIdx.y == 0 && threadIdx.x == 0);
    const int j = blockIdx.y * kLsRanks;
    if (j >= rank) return;
    const float* x = a.x + (size_t)m * a.K;
    const void* A = a.A[ad];
    float s[kLsRanks] = {};
#pragma unroll 2
    for (int k = (int)threadIdx.x * 8; k < a.K; k += 2048) {
        float v[8], f[kLsRanks][8];
#pragma unroll
        for (int i = 0; i < kLsRanks; ++i) lora_load8<F16>(A, (size_t)min(j + i, rank - 1) * a.K + k, f[i]);
        lora_load8<false>(x, k, v);
#pragma unroll
        for (int i = 0; i < kLsRanks; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[i] = fmaf(f[i][e], v[e], s[i]);
    }
#pragma unroll
    for (int i = 0; i < kLsRanks; ++i) {
        s[i] = warp_sum(s[i]);
        if (lane == 0) part[warp][i] = s[i];
    }
    __syncthreads();
    if (threadIdx.x < kLsRanks && j + (int)threadIdx.x < rank) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += part[w][threadIdx.x];
        a.t[(size_t)m * a.max_rank + j + threadIdx.x] = t * __ldg(a.scale + ad);
    }
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four int8 as two pairs of F16, exactly: the biased byte b + 128 in the low bits
// of 1024, less 1152.
__device__ __forceinline__ void i8x4_to_h2(uint32_t w, uint32_t* lo, uint32_t* hi) {
    const uint32_t u = w ^ 0x80808080u;
    uint32_t p = __byte_perm(u, 0x64646464u, 0x4140), q = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));   // 1152
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&p), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&q), bias);
    *lo = *reinterpret_cast<const uint32_t*>(&x);
    *hi = *reinterpret_cast<const uint32_t*>(&y);
}

// t . row of B from element `at` on
__device__ __forceinline__ float lora_dot(const void* Bp, size_t at, const float* t, int r, bool f16) {
    float d = 0.f;
    if (f16 && (r & 7) == 0) {
        const __half* B = static_cast<const __half*>(Bp) + at;
#pragma unroll 2
        for (int j = 0; j < r; j += 8) {
            float b[8];
            h8_to_f8(__ldg(reinterpret_cast<const uint4*>(B + j)), b);
            const float4 u = *reinterpret_cast<const float4*>(t + j), v = *reinterpret_cast<const float4*>(t + j + 4);
            d = fmaf(b[0], u.x, fmaf(b[1], u.y, fmaf(b[2], u.z, fmaf(b[3], u.w, d))));
            d = fmaf(b[4], v.x, fmaf(b[5], v.y, fmaf(b[6], v.z, fmaf(b[7], v.w, d))));
        }
    } else if (!f16 && (r & 3) == 0) {
        const float* B = static_cast<const float*>(Bp) + at;
#pragma unroll 4
        for (int j = 0; j < r; j += 4) {
            const float4 b = __ldg(reinterpret_cast<const float4*>(B + j)), u = *reinterpret_cast<const float4*>(t + j);
            d = fmaf(b.x, u.x, fmaf(b.y, u.y, fmaf(b.z, u.z, fmaf(b.w, u.w, d))));
        }
    } else {
#pragma unroll 4
        for (int j = 0; j < r; ++j) d = fmaf(lora_elem(Bp, at + j, f16), t[j], d);
    }
    return d;
}

struct LoraRowsPlan {
    int slice;    // K of a warp in a pass
    int passes;
    int tiles;    // tiles of weight rows
    int most;     // tiles of a cluster, at most
};

// W8: INT8 weights.  WIDE: 9 to 16 rows (else the upper half of the operand is
// zero and takes no registers).
template <bool W8, bool WIDE>
__global__ void __launch_bounds__(kLrThreads, WIDE && W8 ? 1 : 2)
lora_rows_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ LoraRowsPlan plan) {
    constexpr int E = W8 ? 16 : 8;                     // weights in 16 bytes
    constexpr int kBlock = 4 * E;                      // k a load of the warp
    constexpr int kBlocks = lr_slice(W8, WIDE) / kBlock;     // loads a weight row
    constexpr int kSteps = E / 4;                      // MMA steps a load
    constexpr int kHalves = WIDE ? 2 : 1;
    constexpr int kCols = lr_cols(W8), kGroups = kCols / 8, kBatch = lr_batch(W8), kRows = kLrRows / 2 * kHalves;
    constexpr int kLine = lr_line(W8, WIDE);
    constexpr int kRed = kRows * kLine;                // a warp's sums of a tile
    constexpr int kOut = kRows * kCols;
    constexpr int kDepth = lr_depth(W8, WIDE);
    static_assert(kBatch % kDepth == 0, "a tile keeps its registers");
    extern __shared__ __align__(16) float lr_smem[];   // [tile][rows][weight rows], then the warps' sums
    cg::cluster_group cl = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int rank = (int)cl.block_rank(), nsplit = (int)cl.num_blocks();
    const int group = (int)(blockIdx.x / nsplit), groups = (int)(gridDim.x / nsplit);
    const int mb = blockIdx.y * kLrRows, M = min(a.M - mb, kLrRows);   // this CTA's rows
    const int my_tiles = plan.tiles > group ? (plan.tiles - group + groups - 1) / groups : 0;
    float* warps = lr_smem + plan.most * kOut;         // [2][kBatch tiles][8 warps][rows][weight rows + 1]
    const int64_t row_bytes = (int64_t)a.K * (W8 ? 1 : 2);
    int batch = 0;

#pragma unroll 1
    for (int pass = 0; pass < plan.passes; ++pass) {
        const int k0 = ((pass * nsplit + rank) * kLrWarps + warp) * plan.slice + q * E;   // this thread's first k
        unsigned in_k = 0;   // its loads that lie inside K and the slice
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) in_k |= (unsigned)(i * kBlock < plan.slice && k0 + i * kBlock < a.K) << i;

        // this warp's weights of the tile's rows: 16 bytes of row g of each 8 a load
        uint4 w[kDepth][kGroups][kBlocks];
        int n = group * kCols + g;
        const unsigned char* wp = static_cast<const unsigned char*>(a.w) + n * row_bytes + (int64_t)k0 * (W8 ? 1 : 2);
        auto request = [&](uint4 (&w)[kGroups][kBlocks]) {
#pragma unroll
            for (int h = 0; h < kGroups; ++h) {
                const bool row = n + 8 * h < a.N;
                const unsigned char* p = wp + 8 * h * row_bytes;
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
                    w[h][i] = row && ((in_k >> i) & 1u) ? ld_stream16(p + i * 64) : make_uint4(0u, 0u, 0u, 0u);
            }
            n += groups * kCols;
            wp += groups * kCols * row_bytes;
        };
#pragma unroll
        for (int d = 0; d < kDepth; ++d)
            if (d < my_tiles) request(w[d]);

        // x of rows g (and g + 8), this thread's k, as hi + lo with a factor a row
        uint32_t xh[kBlocks][kSteps][2 * kHalves], xl[kBlocks][kSteps][2 * kHalves];
        float f[2] = {0.f, 0.f};
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf) {
            const int m = g + 8 * hf;
            float v[kBlocks][E];
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
                const bool in = m < M && ((in_k >> i) & 1u);
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    const float4 x = in ? __ldg(reinterpret_cast<const float4*>(a.x + (size_t)(mb + m) * a.K + k0 + i * kBlock + e))
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
                    v[i][e] = x.x, v[i][e + 1] = x.y, v[i][e + 2] = x.z, v[i][e + 3] = x.w;
                    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
                }
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            int e2 = 0;   // the largest / 2^e2 in [2^13, 2^14)
            if (mx > 0.f && mx < INFINITY) e2 = max(-100, min(114, (int)((__float_as_uint(mx) >> 23) & 255) - 127 - 13));
            f[hf] = __uint_as_float((uint32_t)(127 + e2) << 23);
            const float inv = __uint_as_float((uint32_t)(127 - e2) << 23);
#pragma unroll
            for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const float x0 = v[i][4 * s + 2 * p] * inv, x1 = v[i][4 * s + 2 * p + 1] * inv;
                        const __half2 hi = __floats2half2_rn(x0, x1);
                        const float2 h = __half22float2(hi);
                        const __half2 lo = __floats2half2_rn(x0 - h.x, x1 - h.y);
                        xh[i][s][p * kHalves + hf] = *reinterpret_cast<const uint32_t*>(&hi);
                        xl[i][s][p * kHalves + hf] = *reinterpret_cast<const uint32_t*>(&lo);
                    }
        }

        if constexpr (!WIDE) {   // D's columns are x's rows: their factors
            const float mine = f[0];
            f[0] = __shfl_sync(0xffffffffu, mine, 8 * q);
            f[1] = __shfl_sync(0xffffffffu, mine, 8 * q + 4);
        }
        auto step = [&](const uint4& w, int s, uint32_t (&b)[2]) {   // a thread's fragment of 16 k
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
            if constexpr (W8) i8x4_to_h2(ww[s], &b[0], &b[1]);
            else b[0] = ww[2 * s], b[1] = ww[2 * s + 1];
        };

        // kBatch tiles between barriers: the warps run apart as far as that
#pragma unroll 1
        for (int it = 0; it < my_tiles; it += kBatch, ++batch) {
            float* half = warps + (batch & 1) * (kBatch * kLrWarps * kRed);
            const int nb = min(kBatch, my_tiles - it);
            auto tile = [&](int b, uint4 (&w)[kGroups][kBlocks]) {
                // sums of the two planes apart: shorter chains.  WIDE: D's 16 rows are x's, its 8 columns weight rows; else
                // the other way round, 16 weight rows a product
                constexpr int kProds = WIDE ? kGroups : kGroups / 2;
                float hi[kProds][4] = {}, lo[kProds][4] = {};
#pragma unroll
                for (int h = 0; h < kProds; ++h)
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i) {
#pragma unroll
                        for (int s = 0; s < kSteps; ++s) {
                            if constexpr (WIDE) {
                                uint32_t b[2];
                                step(w[h][i], s, b);
                                mma_f16(hi[h], xh[i][s], b[0], b[1]);
                                mma_f16(lo[h], xl[i][s], b[0], b[1]);
                            } else {
                                uint32_t b[2], c[2];
                                step(w[2 * h][i], s, b);
                                step(w[2 * h + 1][i], s, c);
                                const uint32_t rows[4] = {b[0], c[0], b[1], c[1]};
                                mma_f16(hi[h], rows, xh[i][s][0], xh[i][s][1]);
                                mma_f16(lo[h], rows, xl[i][s][0], xl[i][s][1]);
                            }
                        }
                    }
                if (it + b + kDepth < my_tiles) request(w);
                // D: rows g, g + 8; columns 2q, 2q + 1
                float* red = half + (b * kLrWarps + warp) * kRed;
#pragma unroll
                for (int h = 0; h < kProds; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (WIDE) red[(g + 8 * (e >> 1)) * kLine + h * 8 + 2 * q + (e & 1)] = (hi[h][e] + lo[h][e]) * f[e >> 1];
                        else red[(2 * q + (e & 1)) * kLine + h * 16 + g + 8 * (e >> 1)] = (hi[h][e] + lo[h][e]) * f[e & 1];
                    }
            };
#pragma unroll 1
            for (int b = 0; b < nb; b += kDepth) {
#pragma unroll
                for (int d = 0; d < kDepth; ++d)
                    if (b + d < nb) tile(b + d, w[d]);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < nb * kOut; i += kLrThreads) {
                const int b = i / kOut, at = i % kOut / kCols * kLine + i % kCols;
                const float* r = half + b * kLrWarps * kRed + at;
                float s = r[0];
#pragma unroll
                for (int v = 1; v < kLrWarps; ++v) s += r[v * kRed];
                float* sum = lr_smem + it * kOut + i;
                *sum = pass ? *sum + s : s;
            }
        }
    }
    if (nsplit > 1) cl.sync();
    else __syncthreads();
    if (a.n) pdl_wait();   // t of the shrink kernel

    // epilogue: the cluster's CTAs share its tiles; partial sums in rank order
    // a thread keeps its row: kLrThreads / kCols rows a step
    constexpr int kStep = kLrThreads / kCols;
#pragma unroll 1
    for (int m = threadIdx.x / kCols; m < M; m += kStep) {
        const int c = threadIdx.x % kCols;
        int r;
        const int ad = lora_of(a, mb + m, &r, false);
        const float* t = a.t + (size_t)(mb + m) * a.max_rank;
        const void* Bp = ad >= 0 ? a.B[ad] : nullptr;
#pragma unroll 1
        for (int it = rank; it < my_tiles; it += nsplit) {
            const int n = (group + it * groups) * kCols + c;
            if (n >= a.N) continue;
            float s = 0.f;
            for (int p = 0; p < nsplit; ++p) s += *(cl.map_shared_rank(lr_smem, p) + it * kOut + m * kCols + c);
            s *= a.row_scales ? __ldg(a.row_scales + n) : a.tscale;
            a.y[(size_t)(mb + m) * a.N + n] = s + lora_dot(Bp, (size_t)n * r, t, r, a.f16);
        }
    }
    if (nsplit > 1) cl.sync();   // no CTA leaves while another reads its sums
}

template <bool W8, bool WIDE>
static tvb_status launch_rows_kernel(const LoraArgs& a, bool dependent, cudaStream_t st) {
    const auto kernel = lora_rows_kernel<W8, WIDE>;
    constexpr int kBlock = W8 ? 64 : 32, kMax = lr_slice(W8, WIDE);
    LoraRowsPlan plan;
    constexpr int kCols = lr_cols(W8), kOut = kCols * (WIDE ? 16 : 8);
    plan.tiles = (a.N + kCols - 1) / kCols;
    // CTAs a cluster: a power of two, which clusters pack best into the GPU, until the warps' slices hold K in one pass
    int nsplit = 1;
    while (nsplit < kLrMaxSplit && nsplit * kLrWarps * kMax < a.K) nsplit *= 2;
    plan.passes = (a.K + nsplit * kLrWarps * kMax - 1) / (nsplit * kLrWarps * kMax);
    const int per = (a.K + plan.passes * nsplit * kLrWarps - 1) / (plan.passes * nsplit * kLrWarps);
    plan.slice = (per + kBlock - 1) / kBlock * kBlock;
    constexpr int kWarpSums = 2 * lr_batch(W8) * kLrWarps * (kOut / kCols) * lr_line(W8, WIDE);

    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kLrThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)nsplit;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // clusters that fit the GPU at once: one more would be a second wave
    static int resident[kMaxDevices][kLrMaxSplit + 1];
    static int set[kMaxDevices];
    constexpr int kSmem = (WIDE && W8 ? 200 : 100) * 1024;   // one CTA an SM, or two
    TVB_TRY(allow_smem(reinterpret_cast<const void*>(kernel), kSmem, set));
    int dev = 0;
    TVB_CUDA(cudaGetDevice(&dev));
    if (!resident[dev][nsplit]) {
        int n = 0;
        cfg.gridDim = dim3((unsigned)nsplit);
        cfg.dynamicSmemBytes = kSmem;
        TVB_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
        resident[dev][nsplit] = std::max(1, n);
    }
    // as many groups as are resident, or more where a group's sums would not fit
    const int fit = (kSmem / 4 - kWarpSums) / kOut;
    const int blocks = (a.M + kLrRows - 1) / kLrRows;
    const int groups = std::min(plan.tiles, std::max(std::max(1, resident[dev][nsplit] / blocks), (plan.tiles + fit - 1) / fit));
    plan.most = (plan.tiles + groups - 1) / groups;
    cfg.gridDim = dim3((unsigned)(groups * nsplit), (unsigned)blocks);
    cfg.dynamicSmemBytes = (size_t)(plan.most * kOut + kWarpSums) * 4;
    cfg.numAttrs = dependent ? 2 : 1;
    TVB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, plan));
    return check_launch("lora_rows_kernel");
}

tvb_status lora_shrink_rows(const LoraArgs& a, cudaStream_t st) {
    const dim3 grid((unsigned)a.M, (unsigned)((a.max_rank + kLsRanks - 1) / kLsRanks));
    if (a.f16) lora_shrink_kernel<true><<<grid, 256, 0, st>>>(a);
    else lora_shrink_kernel<false><<<grid, 256, 0, st>>>(a);
    return check_launch("lora_shrink_kernel");
}

}  // namespace tvb

extern "C" tvb_status tvb_matmul_lora(float* y, const float* x, int M, int K, const tvb_weight* w, int N,
                                      const tvb_lora_table* table, const int* adapter, unsigned* status, void* stream) {
    using namespace tvb;
    TVB_REQUIRE(w && w->w && table && (M == 0 || (y && x)), "matmul_lora: null pointer");
    TVB_REQUIRE(M >= 0 && K > 0 && N > 0, "matmul_lora: bad shape %dx%dx%d", M, K, N);
    TVB_REQUIRE(M <= 65535, "matmul_lora: %d rows (at most 65535)", M);
    TVB_REQUIRE(w->dtype == TVB_F16 || w->dtype == TVB_I8_ROW || w->dtype == TVB_I8_TENSOR,
                "matmul_lora: weight dtype %d", (int)w->dtype);
    TVB_REQUIRE(w->dtype != TVB_I8_ROW || w->row_scales, "matmul_lora: row_scales is NULL");
    TVB_REQUIRE(K % (w->dtype == TVB_F16 ? 8 : 16) == 0, "matmul_lora: K=%d must be a multiple of %d", K,
                w->dtype == TVB_F16 ? 8 : 16);
    TVB_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w->w)) & 15) == 0,
                "matmul_lora: W and x must be 16-byte aligned");
    TVB_REQUIRE(table->n >= 0 && table->max_rank >= 0 && table->max_rank <= kLoraMaxRank,
                "matmul_lora: %d adapters, max_rank %d (at most %d)", table->n, table->max_rank, kLoraMaxRank);
    TVB_REQUIRE(table->n == 0 || (table->A && table->B && table->rank && table->scale && (M == 0 || adapter)),
                "matmul_lora: null adapter pointer");
    TVB_REQUIRE(table->dtype == TVB_F32 || table->dtype == TVB_F16, "matmul_lora: adapter dtype %d", (int)table->dtype);
    if (!M) return TVB_OK;
    const cudaStream_t st = as_stream(stream);
    LoraArgs a = {};
    a.x = x;
    a.y = y;
    a.M = M;
    a.K = K;
    a.N = N;
    a.w = w->w;
    a.w8 = w->dtype != TVB_F16;
    a.row_scales = w->dtype == TVB_I8_ROW ? w->row_scales : nullptr;
    a.tscale = w->dtype == TVB_I8_TENSOR ? w->tensor_scale : 1.0f;
    a.n = table->max_rank ? table->n : 0;
    a.max_rank = (table->max_rank + 3) & ~3;   // rows of t stay 16-byte aligned
    a.f16 = table->dtype == TVB_F16;
    a.A = table->A;
    a.B = table->B;
    a.rank = table->rank;
    a.scale = table->scale;
    a.adapter = adapter;
    a.status = status;
    const int64_t again = (int64_t)((M + kLrRows - 1) / kLrRows - 1) * N * K * (a.w8 ? 1 : 2);
    if (M > kLrMaxRows || (again > kLrMaxAgain && K <= kLoraMaxK)) return lora_many_rows(a, st);
    Workspace ws(st);
    if (a.n) {
        TVB_TRY(ws.get((size_t)M * a.max_rank * 4));
        a.t = ws.at<float>();
        TVB_TRY(lora_shrink_rows(a, st));
    }
    const bool wide = M > 8, dep = a.n > 0;
    if (a.w8) return wide ? launch_rows_kernel<true, true>(a, dep, st) : launch_rows_kernel<true, false>(a, dep, st);
    return wide ? launch_rows_kernel<false, true>(a, dep, st) : launch_rows_kernel<false, false>(a, dep, st);
}
