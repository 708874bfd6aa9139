// Attention of chunks of new tokens over an F16 paged cache on the tensor cores
// (tvb_attention_paged; attn_paged.cu has the formula and the split).
//
// paged_chunk_kernel: a CTA takes 128 query rows (new token x query head of the
// group) of one KV head of one sequence, and one split of its keys in tiles of
// 128.  Products in F32 accuracy from F16 operands: q (times scale log2 e, with
// a power-of-two exponent a row) and p are split into F16 hi + lo planes, K and
// V are F16 as they are, so every product takes two MMAs.
//
//   loader warps (a slot of shared memory at a time each): rows of K or V by 16-byte cp.async,
//     page by page, into the 128-byte swizzle; rows without a key become zeros
//   MMA warp: S = Q K^T (K-major operands) into one of three TMEM buffers a tile
//     ahead of the softmax, then O = P V with P from TMEM and V as the MN-major
//     operand it is in memory (no transpose)
//   softmax warps: two threads a row, each half of the tile's keys (maxima meet in
//     shared memory) and half of the dimensions; running maximum, p as hi + lo
//     over its S columns in TMEM, and O (a fresh product per tile) added to
//     registers with the rescaling, which also keeps the tensor core's truncating sums short (16
//     MMAs: 3e-7; a sum over 6000 keys in TMEM would lose 1.4e-5)
//
// A masked probability is zero but 0 x inf is not: a loader that finds a
// non-finite value in a V tile that some row does not see whole, or a page that
// does not exist, flags the CTA, which then computes its rows key by key instead.
#include "attn_paged.h"
#include "tcgen05.cuh"

namespace tvb {

constexpr int kPcRows = 128, kPcKeys = 128, kPcSlots = 4;
// Warps 0-7 softmax, 8-10 loaders, 11 MMA: 12 warps leave a thread 168 registers.
constexpr int kPcThreads = 384, kPcSoft = 8, kPcLoaders = 3, kPcMmaWarp = kPcSoft + kPcLoaders;

template <int HD>
struct PcSmem {
    static constexpr int kAtom = 128 * 128;               // 128 rows x 64 dims of F16
    static constexpr int kPlane = kAtom * (HD / 64);      // Q plane, K or V tile
    static constexpr int kQ = 0;
    static constexpr int kSlots = 2 * kPlane;
    static constexpr int kBar = kSlots + kPcSlots * kPlane;
    static constexpr int kRed = kBar + 256;                   // row maxima of the two halves, two tiles
    static constexpr int kBytes = kRed + 2 * 2 * 128 * 4 + 1024;   // alignment
};

// Shared-memory descriptor of an MN-major operand in 128-byte-swizzled atoms of
// 64 (MN) x 8 (K): atoms `lbo` bytes apart along MN, 1024 along K.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t lbo) {
    uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(lbo >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

// A from TMEM (two F16 a column), B from shared memory.
__device__ __forceinline__ void tc_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void pc_cp_async16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

template <int HD>
__global__ void __launch_bounds__(kPcThreads, 1) paged_chunk_kernel(const __grid_constant__ PagedAttnArgs a) {
    using Sm = PcSmem<HD>;
    constexpr int kO = 3 * kPcKeys;   // TMEM: S/P buffers in columns [0, 384), O behind
    extern __shared__ unsigned char pc_smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.y, split = blockIdx.z;

    int row0 = 0;
    const int b = row_block_seq<kPcRows, kPcThreads>(a.s, a.group, blockIdx.x, &row0);
    if (b >= a.s.n_seqs) return;
    const SeqView sv = seq_view(a.s, b);
    if (!sv.ok) {
        if (threadIdx.x == 0) report_bad(a.status);
        return;
    }
    const int rows = min(kPcRows, sv.n * a.group - row0);
    if (rows <= 0) return;
    const int p_first = sv.pos0 + row0 / a.group, p_last = sv.pos0 + (row0 + rows - 1) / a.group;
    const int lo = a.window ? max(0, p_first - a.window + 1) : 0;
    const int k0 = a.nsplit > 1 ? max(lo, split * a.split_len) : lo;
    const int k1 = a.nsplit > 1 ? min(p_last + 1, (split + 1) * a.split_len) : p_last + 1;
    if (k0 >= k1) return;   // no row of the block takes this split
    const int nt = (k1 - k0 + kPcKeys - 1) / kPcKeys;
    const int nitems = 2 * nt;   // K0, then K(j + 1), V(j) for every tile j

    const uint32_t raw = smem_u32(pc_smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* smem = pc_smem_raw + (base - raw);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sm::kBar);
    uint64_t* empty = full + kPcSlots;
    uint64_t* s_full = empty + kPcSlots;   // [3]
    uint64_t* p_full = s_full + 3;         // [2]
    uint64_t* o_full = p_full + 2;
    uint64_t* o_read = o_full + 1;
    uint64_t* q_full = o_read + 1;
    uint64_t* drained = q_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* poison = abort_flag + 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kPcSlots; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 3; ++i) mbar_init(s_full + i, 1);
        for (int i = 0; i < 2; ++i) mbar_init(p_full + i, 32 * kPcSoft);
        mbar_init(o_full, 1);
        mbar_init(o_read, 32 * kPcSoft);
        mbar_init(q_full, 32 * kPcSoft);
        mbar_init(drained, 1);
        *abort_flag = 0;
        *poison = 0;
        fence_barrier_init();
    }
    if (warp == kPcMmaWarp) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto fail = [&]() {
        *abort_flag = 1;
        if (a.status) atomicOr(a.status, TVB_DEV_TIMEOUT);
    };
    const int* table = a.s.table + (size_t)b * a.s.table_ld;

    if (warp >= kPcSoft && warp < kPcMmaWarp) {
        // ---- loaders ---------------------------------------------------------------
        const int w = warp - kPcSoft;
        constexpr int kLanes = HD / 8;          // 16-byte chunks, lanes a row
        constexpr int kPass = 32 / kLanes;      // rows a warp instruction
        const int c = lane % kLanes;
        for (int i = w; i < nitems; i += kPcLoaders) {
            const int sl = i % kPcSlots;
            const uint32_t slot = base + Sm::kSlots + sl * Sm::kPlane;
            const bool is_k = i == 0 || ((i & 1) && i != nitems - 1);
            const int tile = i == 0 ? 0 : is_k ? (i + 1) >> 1 : i == nitems - 1 ? nt - 1 : (i >> 1) - 1;
            const bool free_slot = mbar_wait_bounded(empty + sl, (uint32_t)((i / kPcSlots + 1) & 1));
            if (__any_sync(0xffffffffu, !free_slot || *abort_flag)) {
                fail();
                break;
            }
            const unsigned char* src = (is_k ? a.kv.k : a.kv.v) + (int64_t)kvh * a.kv.head_stride + c * 16;
            const int t0 = k0 + tile * kPcKeys;
            bool bad = false;
#pragma unroll
            for (int r0 = 0; r0 < kPcKeys; r0 += 32) {
                int64_t off = -1;
                if (t0 + r0 + lane < k1) {
                    off = paged_offset(a.kv, table, t0 + r0 + lane);
                    bad |= off < 0;
                }
#pragma unroll
                for (int r = 0; r < 32; r += kPass) {
                    const int64_t o = __shfl_sync(0xffffffffu, off, r + lane / kLanes);
                    const int row = r0 + r + lane / kLanes;
                    pc_cp_async16(slot + (c >> 3) * Sm::kAtom + sw128_offset(row, c & 7), src + (o >= 0 ? o : 0), o >= 0);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (bad) {
                *poison = 1;
                report_bad(a.status);
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            // V rows that some query row does not see must be finite
            const int t1 = min(t0 + kPcKeys, k1);
            if (!is_k && (t1 - 1 > p_first || (a.window && t0 <= p_last - a.window))) {
                __syncwarp();
                uint32_t nonfinite = 0;
                for (int j = lane; j < Sm::kPlane / 4; j += 32) {
                    const uint32_t v = *reinterpret_cast<const volatile uint32_t*>(smem + Sm::kSlots + sl * Sm::kPlane + j * 4);
                    nonfinite |= (uint32_t)((v & 0x7C00u) == 0x7C00u) | (uint32_t)((v & 0x7C000000u) == 0x7C000000u);
                }
                if (nonfinite) *poison = 1;
            }
            fence_proxy_async_smem_cta();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + sl);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == kPcMmaWarp) {
        // ---- MMA issuer --------------------------------------------------------------
        if (lane == 0) {
            constexpr uint32_t idesc_s = umma_idesc_f16(kPcRows, kPcKeys);
            constexpr uint32_t idesc_o = umma_idesc_f16(kPcRows, HD) | (1u << 16);   // B is MN-major
            int item = 0;
            auto ready = [&](int i) {
                if (!mbar_wait_bounded(full + i % kPcSlots, (uint32_t)((i / kPcSlots) & 1))) return false;
                tc_fence_after();
                return true;
            };
            auto mma_s = [&](int j) {
                const uint32_t k_s = base + Sm::kSlots + (item % kPcSlots) * Sm::kPlane, d = tmem + (j % 3) * kPcKeys;
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t o = (kk >> 2) * Sm::kAtom + (kk & 3) * 32;
                    const uint64_t kd = sw128_desc(k_s + o);
                    tc_mma(d, sw128_desc(base + Sm::kQ + o), kd, idesc_s, kk ? 1u : 0u);
                    tc_mma(d, sw128_desc(base + Sm::kQ + Sm::kPlane + o), kd, idesc_s, 1u);
                }
                tc_commit(s_full + j % 3);
            };
            bool ok = mbar_wait_bounded(q_full, 0u) && ready(0);
            if (ok) {
                tc_fence_after();
                mma_s(0);
                tc_commit(empty + 0);
                ++item;
            }
            for (int j = 0; ok && j < nt && !*abort_flag; ++j) {
                if (j + 1 < nt) {
                    ok = ready(item);
                    if (!ok) break;
                    mma_s(j + 1);
                    tc_commit(empty + item % kPcSlots);
                    ++item;
                }
                ok = mbar_wait_bounded(p_full + (j & 1), (uint32_t)((j >> 1) & 1)) && ready(item) &&
                     (j == 0 || mbar_wait_bounded(o_read, (uint32_t)((j - 1) & 1)));
                if (!ok) break;
                tc_fence_after();
                const uint32_t v_s = base + Sm::kSlots + (item % kPcSlots) * Sm::kPlane, p = tmem + (j % 3) * kPcKeys;
#pragma unroll
                for (int kk = 0; kk < kPcKeys / 16; ++kk) {
                    const uint64_t vd = sw128_mn_desc(v_s + kk * 2048, Sm::kAtom);
                    tc_mma_ts(tmem + kO, p + kk * 16, vd, idesc_o, kk ? 1u : 0u);
                    tc_mma_ts(tmem + kO, p + kk * 16 + 8, vd, idesc_o, 1u);
                }
                tc_commit(o_full);
                tc_commit(empty + item % kPcSlots);
                ++item;
            }
            if (!ok) fail();
            tc_commit(drained);   // every MMA issued above
            mbar_wait_bounded(drained, 0u);
        }
        __syncwarp();
    } else {
        // ---- softmax: two threads a row, each half of a tile's keys and of the dimensions ----
        const int r = threadIdx.x & 127, half = warp >> 2;
        const bool live = r < rows;
        const int row = row0 + min(r, rows - 1);
        const int tok = sv.row0 + row / a.group, head = kvh * a.group + row % a.group;
        const int pos = live ? sv.pos0 + row / a.group : -1;
        float* red = reinterpret_cast<float*>(smem + Sm::kRed);
        auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };
        float f = 1.f;   // q = (hi + lo) f / (scale log2 e)
        {
            const float* q = a.q + (size_t)tok * a.ldq + head * HD;
            float mx = 0.f;
#pragma unroll 4
            for (int d = 0; d < HD; d += 4) {
                const float4 x = *reinterpret_cast<const float4*>(q + d);
                mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
            }
            mx *= fabsf(a.scale2);
            // 2^e with mx / 2^e in [2^13, 2^14): both planes of every value that matters are normal F16
            int e = 0;
            if (mx > 0.f && mx < INFINITY) e = max(-100, min(100, (int)((__float_as_uint(mx) >> 23) & 255) - 127 - 13));
            f = __uint_as_float((uint32_t)(127 + e) << 23);
            const float g = a.scale2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll 2
            for (int d = half * (HD / 2); d < (half + 1) * (HD / 2); d += 8) {
                const float4 x = *reinterpret_cast<const float4*>(q + d), y = *reinterpret_cast<const float4*>(q + d + 4);
                const float v[8] = {x.x * g, x.y * g, x.z * g, x.w * g, y.x * g, y.y * g, y.z * g, y.w * g};
                __half2 hi[4], lo2[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    hi[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                    const float2 h = __half22float2(hi[i]);
                    lo2[i] = __floats2half2_rn(v[2 * i] - h.x, v[2 * i + 1] - h.y);
                }
                const int c = d >> 3;
                unsigned char* dst = smem + Sm::kQ + (c >> 3) * Sm::kAtom + sw128_offset(r, c & 7);
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(hi);
                *reinterpret_cast<uint4*>(dst + Sm::kPlane) = *reinterpret_cast<const uint4*>(lo2);
            }
            fence_proxy_async_smem_cta();
            mbar_arrive(q_full);
        }
        constexpr int kD = HD / 2;   // dimensions of this thread
        float acc[kD];
#pragma unroll
        for (int d = 0; d < kD; ++d) acc[d] = 0.f;
        float m = -INFINITY, l = 0.f, corr_prev = 1.f;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        auto add_o = [&](float c) {   // acc = acc c + O of the last product
#pragma unroll
            for (int h = 0; h < kD / 32; ++h) {
                uint32_t o[32];
                tmem_ld32(lanes + kO + half * kD + h * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[h * 32 + i] = fmaf(acc[h * 32 + i], c, __uint_as_float(o[i]));
            }
        };
        auto landed = [&](uint64_t* bar, int phase) {
            const bool in = mbar_wait_bounded(bar, (uint32_t)(phase & 1));
            return __all_sync(0xffffffffu, in && !*abort_flag) != 0;
        };
        bool ok = true;
        for (int j = 0; j < nt; ++j) {
            ok = ok && landed(s_full + j % 3, j / 3);
            // a warp that gives up tells its partner through the exchange below (a maximum is never NaN), so both leave
            if (!ok) red[((j & 1) * 2 + half) * 128 + r] = NAN;
            const uint32_t sb = lanes + (j % 3) * kPcKeys + half * 64;
            const int t0 = k0 + j * kPcKeys;
            const int t1 = min(t0 + kPcKeys, k1);
            const bool edge = t1 - t0 < kPcKeys || t1 - 1 > p_first || (a.window && t0 <= p_last - a.window);
            uint32_t s[64];
            if (ok) {
                tc_fence_after();
                tmem_ld32(sb, *reinterpret_cast<uint32_t(*)[32]>(s));
                tmem_ld32(sb + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
                tmem_wait_ld();
                if (edge) {   // keys [first, last] of this half are the row's
                    const int last = min(t1 - 1, pos) - t0 - half * 64;
                    const int first = a.window ? pos - a.window + 1 - t0 - half * 64 : 0;
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (i > last || i < first) s[i] = 0xff800000u;   // -infinity
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 64; ++i) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(s[i]));
                red[((j & 1) * 2 + half) * 128 + r] = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            }
            pair_sync();
            const float x0 = red[(j & 1) * 256 + r], x1 = red[(j & 1) * 256 + 128 + r];
            if (__any_sync(0xffffffffu, x0 != x0 || x1 != x1)) {
                ok = false;
                break;
            }
            const float mn = fmaxf(m, fmaxf(x0, x1) * f);
            const float corr = m == mn ? 1.f : ex2(m - mn);
            const float mref = mn == -INFINITY ? 0.f : mn;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 4; ++c) {   // 16 keys: 8 columns of hi, 8 of lo, in place of their scores
                uint32_t p[16];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = ex2(fmaf(__uint_as_float(s[16 * c + 2 * i]), f, -mref));
                    const float y = ex2(fmaf(__uint_as_float(s[16 * c + 2 * i + 1]), f, -mref));
                    sum[(2 * i) & 3] += x;
                    sum[(2 * i + 1) & 3] += y;
                    const __half2 hi = __floats2half2_rn(x, y);
                    const float2 h = __half22float2(hi);
                    const __half2 lw = __floats2half2_rn(x - h.x, y - h.y);
                    p[i] = *reinterpret_cast<const uint32_t*>(&hi);
                    p[8 + i] = *reinterpret_cast<const uint32_t*>(&lw);
                }
                tmem_st16(sb + 16 * c, p);
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(p_full + (j & 1));
            l = l * corr + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
            m = mn;
            if (j > 0) {
                ok = landed(o_full, j - 1);
                if (ok) {
                    tc_fence_after();
                    add_o(corr_prev);
                    tc_fence_before();
                    mbar_arrive(o_read);
                }
            }
            corr_prev = corr;
        }
        ok = ok && landed(o_full, nt - 1);
        if (ok) {
            tc_fence_after();
            add_o(corr_prev);
            tc_fence_before();
        } else {
            fail();
        }
        // the row's sum from its two halves
        red[half * 128 + r] = l;
        pair_sync();
        l = red[r] + red[128 + r];
        if (ok && live && !*poison) {
            if (a.nsplit > 1) {
                float* pp = a.part + (((size_t)split * a.s.n_tokens + tok) * a.nh + head) * (HD + 2);
                if (half == 0) *reinterpret_cast<float2*>(pp) = make_float2(l, m);
                pp += 2 + half * kD;
#pragma unroll
                for (int d = 0; d < kD; d += 2) *reinterpret_cast<float2*>(pp + d) = make_float2(acc[d], acc[d + 1]);
            } else {
                const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
                float* po = a.out + (size_t)tok * a.ldo + head * HD + half * kD;
#pragma unroll
                for (int d = 0; d < kD; d += 4)
                    *reinterpret_cast<float4*>(po + d) = make_float4(acc[d] * inv, acc[d + 1] * inv, acc[d + 2] * inv,
                                                                     acc[d + 3] * inv);
                if (a.lse && half == 0)
                    a.lse[(size_t)tok * a.nh + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kPcMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (*poison && !*abort_flag) {
        // key by key, a warp a row: lane = HD / 32 dimensions
        for (int r = warp; r < rows; r += kPcThreads / 32) paged_row_slow<__half, HD>(a, sv, table, kvh, split, row0 + r, k0, k1);
    }
}

template <int HD>
static tvb_status launch_chunk(const PagedAttnArgs& a, cudaStream_t st) {
    static int set[kMaxDevices];
    TVB_TRY(allow_smem(reinterpret_cast<const void*>(paged_chunk_kernel<HD>), PcSmem<HD>::kBytes, set));
    const int64_t blocks = ((int64_t)a.s.n_tokens * a.group) / kPcRows + a.s.n_seqs;
    paged_chunk_kernel<HD><<<dim3((unsigned)blocks, (unsigned)a.nkv, (unsigned)a.nsplit), kPcThreads, PcSmem<HD>::kBytes, st>>>(a);
    return check_launch("paged_chunk_kernel");
}

tvb_status paged_attn_chunk_f16(const PagedAttnArgs& a, int hd, cudaStream_t st) {
    return hd == 128 ? launch_chunk<128>(a, st) : launch_chunk<64>(a, st);
}

}  // namespace tvb
