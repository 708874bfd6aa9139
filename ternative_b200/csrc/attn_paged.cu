// Attention of new tokens over the paged KV cache (tvb_attention_paged).
//
//   out = sum_t p_t v_t / sum_t p_t,  p_t = 2^(s_t - m),  s_t = scale log2(e) q . k_t
//
// over the keys t in (p - window, p] of the row's position p, in one pass: a
// running maximum m per row, the sum and the weighted values rescaled by
// 2^(m_old - m_new) when it grows.
//
// paged_rows_kernel: a CTA takes its run of tiles (attn_schedule: RB query rows of
// one KV head of one sequence against 8 keys of each warp); per piece its warps take
// batches of 8 keys in turn and merge at the end.  K and V rows pass
// through a ring of cp.async stages private to each warp, so no warp waits for
// another while it streams; each lane owns head_dim / 32 dimensions.  The RB x 8
// partial dot products of a batch are summed over the lanes by a butterfly that
// halves the values it carries at each step (31 shuffles for 32 sums).
#include "attn_paged.h"

#include <algorithm>
#include <climits>

namespace tvb {

constexpr int kPrKeys = 8;   // keys a batch
// What starting and leaving a block costs, in tiles.  Decode of 32 sequences: 1, 4, 8
// take 49.3, 46.1, 49.7 us, of 4 x 61000 keys 103, 100, 101.
constexpr int kPrExtra = 4;
// Rows of a KV head from which a call may take the tensor cores (paged_chunk_kernel):
// below, its 128-row tiles are too empty.  20/5 heads, 8 sequences of 3000 keys: F16
// 24 rows 36 against 33 us there, 48 rows 46 against 33; F32 24 rows 100 against 109,
// 32 rows 126 against 109.
constexpr int kTensorRows16 = 24, kTensorRows32 = 25;
// ... unless the few-rows kernels' blocks (16 rows, F32 8) are no more than a CTA (two)
// an SM and short: more CTAs then share what one of 128 rows would do alone.  20/5
// heads, F32: 64 tokens of one sequence over 300 keys 24 against 35 us, 8 x 7 over 600
// keys 42 against 55, over 3000 126 against 109, 8 x 16 over 300 42 against 36; F16: 64
// over 300 12.8 against 18.8, 8 x 7 over 600 21 against 27, 8 x 32 over 300 26 against 17.
constexpr int kFewSpan = 1024;
// Keys up to which a CTA takes whole blocks: sharing tiles evenly costs a second
// launch.  One token, F16, 400 keys 14.2 against 16.4 us, 800 keys 20.9 against
// 17.3; 128 sequences of 1000 keys 126 against 79.
constexpr int kWholeKeys = 512;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t pr_smem(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

template <typename T, int HD>
struct PrStage {
    static constexpr int kRow = HD * (int)sizeof(T);     // bytes of a key
    static constexpr int kBytes = 2 * kPrKeys * kRow;    // K rows, then V rows
    // two CTAs an SM, so that one streams while the other starts or ends a piece; as many warps as leave each a
    // few stages of its own in shared memory
    static constexpr int kWarps = sizeof(T) == 2 ? 8 : 6, kThreads = 32 * kWarps;
    static constexpr int kStages = sizeof(T) == 2 ? 3 : 2;
    static constexpr int kTile = kPrKeys * kWarps;       // keys a tile
    static constexpr int kSmem = kWarps * kStages * kBytes;
};

// Sum over the lanes of v[0 .. NV): lane l returns the sum of v[l / (32 / NV)].
template <int NV>
__device__ __forceinline__ float pr_reduce(float (&v)[NV], int lane) {
#pragma unroll
    for (int n = NV, o = 16; o > 0; o >>= 1) {
        if (n > 1) {
            n >>= 1;
            const bool up = lane & o;
#pragma unroll
            for (int i = 0; i < NV / 2; ++i) {
                if (i < n) {
                    const float keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                }
            }
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
        }
    }
    return v[0];
}

template <typename T, int HD, int RB>
__host__ __device__ constexpr int rows_smem() {
    using St = PrStage<T, HD>;
    return St::kSmem > St::kWarps * RB * (HD + 2) * 4 ? St::kSmem : St::kWarps * RB * (HD + 2) * 4;
}

// Joins the warps' sums of a piece: [warp][row][HD + 2], maximum and sum last.  PLANES:
// the products were of two planes, where an infinity times the small one (zero, or of
// the other sign) is NaN: a row that is not finite is computed key by key, unless its
// query is not (NaN whatever the keys are).
template <int HD, int RB, int WARPS, bool PLANES>
__device__ __forceinline__ void merge_warps(const PagedAttnArgs& a, const AttnPiece& pc, const float* red) {
    constexpr int ND = HD / 32, kW = HD + 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = warp; r < pc.rows; r += WARPS) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, red[(w * RB + r) * kW + HD]);
        float L = 0.f, o[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float* x = red + (w * RB + r) * kW;
            const float c = x[HD] == -INFINITY ? (x[HD + 1] == 0.f ? 0.f : 1.f) : exp2f(x[HD] - M);   // no maximum but a sum: NaN
            if (c != 0.f) {
                L = fmaf(x[HD + 1], c, L);
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d] = fmaf(x[lane * ND + d], c, o[d]);
            }
        }
        if constexpr (PLANES) {
            bool odd = !(L < INFINITY);
#pragma unroll
            for (int d = 0; d < ND; ++d) odd |= !(fabsf(o[d]) < INFINITY);
            if (__any_sync(0xffffffffu, odd)) {
                const int t = (int)a.gdiv.div((uint32_t)(pc.row + r));
                const float* q = a.q + (size_t)(pc.tok0 + t) * a.ldq + (pc.kvh * a.group + pc.row + r - t * a.group) * HD + lane * ND;
                bool finite = true;
#pragma unroll
                for (int d = 0; d < ND; ++d) finite = finite && fabsf(q[d] * a.scale2) < INFINITY;
                if (__all_sync(0xffffffffu, finite)) {
                    attn_row_slow<__half, RB, HD>(a, pc, r);
                    continue;
                }
            }
        }
        attn_row_store<RB, HD, ND>(a, pc, r, L, M, o);
    }
}

// One piece; whole CTA.
template <typename T, int HD, int RB>
__device__ __forceinline__ void rows_piece(const PagedAttnArgs& a, const AttnPiece& pc, unsigned char* pr_smem_raw) {
    using St = PrStage<T, HD>;
    constexpr int ND = HD / 32;              // dimensions a lane
    constexpr int RG = RB < 4 ? RB : 4;      // rows reduced together
    constexpr int NG = RB / RG;
    constexpr int NV = RG * kPrKeys;         // sums of one reduction
    constexpr int LPV = 32 / NV;             // lanes that hold one
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = pc.rows, kvh = pc.kvh, k0 = max(pc.k0, pc.first), k1 = pc.k1;
    const int p_first = pc.pos0 + (int)a.gdiv.div((uint32_t)pc.row);
    const int p_last = pc.pos0 + (int)a.gdiv.div((uint32_t)(pc.row + rows - 1));

    // q (times scale log2 e) and positions of the rows
    float q[RB][ND], acc[RB][ND];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        const int row = pc.row + min(r, rows - 1), t = (int)a.gdiv.div((uint32_t)row);
        const int tok = pc.tok0 + t, head = kvh * a.group + row - t * a.group;
        pr_load<float, ND>(reinterpret_cast<const unsigned char*>(a.q + (size_t)tok * a.ldq + head * HD + lane * ND), q[r]);
#pragma unroll
        for (int d = 0; d < ND; ++d) q[r][d] *= a.scale2, acc[r][d] = 0.f;
    }
    // lane l keeps the score of row group g: row g RG + l / (8 LPV), key (l / LPV) % 8
    const int lrow = lane / (kPrKeys * LPV), lkey = (lane / LPV) % kPrKeys;
    int lpos[NG];
    float m[NG], l[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const int r = g * RG + lrow;
        lpos[g] = r < rows ? pc.pos0 + (int)a.gdiv.div((uint32_t)(pc.row + r)) : -1;
        m[g] = -INFINITY;
        l[g] = 0.f;
    }

    unsigned char* ring = pr_smem_raw + warp * St::kStages * St::kBytes;
    const unsigned char* kb = a.kv.k + (int64_t)kvh * a.kv.head_stride;
    const unsigned char* vb = a.kv.v + (int64_t)kvh * a.kv.head_stride;
    const int* table = a.s.table + (size_t)pc.b * a.s.table_ld;
    bool bad = false;

    // one batch of keys [t, t + 8) into stage st; rows that no query row sees or
    // whose page does not exist become zeros.  Returns which keys exist (bits).
    auto request = [&](int t, int st) -> unsigned {
        int64_t off = -1;
        if (lane < kPrKeys && t + lane >= k0 && t + lane < k1) {
            off = paged_offset(a.kv, table, t + lane);
            bad |= off < 0;
        }
        const unsigned have = __ballot_sync(0xffffffffu, off >= 0) & ((1u << kPrKeys) - 1);
        constexpr int kLanes = St::kRow / 16;        // lanes a row
        constexpr int kRows = 32 / kLanes;           // rows a pass
        const uint32_t dst = pr_smem(ring + st * St::kBytes) + lane * 16;
#pragma unroll
        for (int j = 0; j < kPrKeys / kRows; ++j) {
            const int key = j * kRows + lane / kLanes;
            const int64_t o = __shfl_sync(0xffffffffu, off, key);
            const int64_t at = (o >= 0 ? o : 0) + (lane % kLanes) * 16;
            cp_async16(dst + j * 512, kb + at, o >= 0);
            cp_async16(dst + kPrKeys * St::kRow + j * 512, vb + at, o >= 0);
        }
        return have;
    };

    // batches warp, warp + kWarps, ... of the keys from k0 on
    const int step = St::kTile;
    int t = k0 + warp * kPrKeys, tn = t;
    unsigned have = 0u;
    for (int i = 0; i < St::kStages - 1; ++i, tn += step) {
        have |= (tn < k1 ? request(tn, i) : 0u) << (8 * i);
        cp_async_commit();
    }
    int st = 0;
#pragma unroll 1   // the loop fits the instruction cache only once
    while (t < k1) {
        {
            const int ns = st == 0 ? St::kStages - 1 : st - 1;
            __syncwarp();   // every lane is done with the stage that is filled now
            have |= (tn < k1 ? request(tn, ns) : 0u) << (8 * (St::kStages - 1));
            cp_async_commit();
            tn += step;
            cp_async_wait<St::kStages - 1>();
            __syncwarp();
            const unsigned char* stage = ring + st * St::kBytes;
            const unsigned hv = have & 0xffu;   // keys of the stages in order, 8 bits each
            have >>= 8;
            st = st == St::kStages - 1 ? 0 : st + 1;
            float p[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float v[NV];
#pragma unroll
                for (int key = 0; key < kPrKeys; ++key) {
                    float kf[ND];
                    pr_load<T, ND>(stage + key * St::kRow + lane * ND * (int)sizeof(T), kf);
#pragma unroll
                    for (int r = 0; r < RG; ++r) {
                        float x = q[g * RG + r][0] * kf[0];
#pragma unroll
                        for (int d = 1; d < ND; ++d) x = fmaf(q[g * RG + r][d], kf[d], x);
                        v[r * kPrKeys + key] = x;
                    }
                }
                float s = pr_reduce<NV>(v, lane);
                const int kt = t + lkey;
                const bool seen = ((hv >> lkey) & 1u) && kt <= lpos[g] && (!a.window || kt > lpos[g] - a.window);
                if (!seen) s = -INFINITY;
                float mx = s;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                    if (o >= LPV && o < kPrKeys * LPV) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const float mn = fmaxf(m[g], mx);
                const float corr = m[g] == mn ? 1.f : exp2f(m[g] - mn);   // m = -inf: 0
                p[g] = s == -INFINITY ? 0.f : exp2f(s - mn);
                l[g] = l[g] * corr + p[g];
                if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
                    for (int r = 0; r < RG; ++r) {
                        const float c = __shfl_sync(0xffffffffu, corr, r * kPrKeys * LPV);
#pragma unroll
                        for (int d = 0; d < ND; ++d) acc[g * RG + r][d] *= c;
                    }
                }
                m[g] = mn;
            }
            // a key that some row does not see adds nothing to that row, even if its value is not finite
            const bool whole = hv == (1u << kPrKeys) - 1 && t + kPrKeys - 1 <= p_first && (!a.window || t > p_last - a.window);
#pragma unroll
            for (int key = 0; key < kPrKeys; ++key) {
                float vf[ND];
                pr_load<T, ND>(stage + (kPrKeys + key) * St::kRow + lane * ND * (int)sizeof(T), vf);
#pragma unroll
                for (int r = 0; r < RB; ++r) {
                    const float pr = __shfl_sync(0xffffffffu, p[r / RG], ((r % RG) * kPrKeys + key) * LPV);
                    if (whole || pr != 0.f) {
#pragma unroll
                        for (int d = 0; d < ND; ++d) acc[r][d] = fmaf(pr, vf[d], acc[r][d]);
                    }
                }
            }
            t += step;
        }
    }
    cp_async_wait<0>();
    if (bad) report_bad(a.status);

    // merge the warps: [warp][row][HD + 2] in the ring's memory
    __syncthreads();
    float* red = reinterpret_cast<float*>(pr_smem_raw);
    constexpr int kW = HD + 2;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        // sum over the row's lanes (each sum is held by LPV lanes)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            if (o >= LPV && o < kPrKeys * LPV) l[g] += __shfl_xor_sync(0xffffffffu, l[g], o);
        if (lane % (kPrKeys * LPV) == 0) {
            float* w = red + (warp * RB + g * RG + lrow) * kW;
            w[HD] = m[g];
            w[HD + 1] = l[g];
        }
    }
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int d = 0; d < ND; ++d) red[(warp * RB + r) * kW + lane * ND + d] = acc[r][d];
    __syncthreads();
    merge_warps<HD, RB, St::kWarps, false>(a, pc, red);
}

// ---- three rows or more over an F16 cache, 8 or 16 a block: mma.sync ------------------
// The rows are the 16-row operand of mma.sync m16n8k16 (a memory-bound product: the
// legacy tensor path keeps up with memory where the FP32 pipe does not, 46 against
// 62 us for 32 sequences of up to 4096 keys with 20/5 heads).  q and p (lifted, attn_lift)
// are split into F16 hi + lo planes, K and V rows come from shared memory by ldmatrix.  Every 16 keys make a fresh product that is
// added to F32 registers, so the tensor core's truncation does not add up.
template <int HD, int RB>
struct PmStage {
    static constexpr int kKeys = 16, kRow = HD * 2;
    static constexpr int kBytes = 2 * kKeys * kRow;   // K rows, then V rows, 16-byte chunk c of a row at c ^ (row % 8)
    static constexpr int kWarps = RB == 16 ? 4 : 6, kThreads = 32 * kWarps;   // (registers of 16 rows' queries)
    static constexpr int kStages = RB == 16 ? 3 : 2;
    static constexpr int kTile = kKeys * kWarps;
    static constexpr int kRing = kWarps * kStages * kBytes, kRed = kWarps * RB * (HD + 2) * 4;
    static constexpr int kSmem = kRing > kRed ? kRing : kRed;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void pm_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pm_split(float x, float y, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    *hi = *reinterpret_cast<const uint32_t*>(&h);
    *lo = *reinterpret_cast<const uint32_t*>(&l);
}

// One piece; whole CTA.  `odd` (shared): a value that some row does not see is not finite.
template <int HD, int RB>
__device__ __forceinline__ void mma_piece(const PagedAttnArgs& a, const AttnPiece& pc, unsigned char* smem, int* odd) {
    using St = PmStage<HD, RB>;
    constexpr int kHalves = RB / 8;   // 8 rows each
    constexpr int kSteps = HD / 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int rows = pc.rows, kvh = pc.kvh, k0 = max(pc.k0, pc.first), k1 = pc.k1;
    const int p_first = pc.pos0 + (int)a.gdiv.div((uint32_t)pc.row);
    const int p_last = pc.pos0 + (int)a.gdiv.div((uint32_t)(pc.row + rows - 1));
    if (threadIdx.x == 0) *odd = 0;
    __syncthreads();

    unsigned char* ring = smem + warp * St::kStages * St::kBytes;
    const unsigned char* kb = a.kv.k + (int64_t)kvh * a.kv.head_stride;
    const unsigned char* vb = a.kv.v + (int64_t)kvh * a.kv.head_stride;
    const int* table = a.s.table + (size_t)pc.b * a.s.table_ld;
    bool bad = false;
    auto request = [&](int t, int st) -> unsigned {
        int64_t off = -1;
        if (lane < St::kKeys && t + lane >= k0 && t + lane < k1) {
            off = paged_offset(a.kv, table, t + lane);
            bad |= off < 0;
        }
        const unsigned have = __ballot_sync(0xffffffffu, off >= 0) & 0xffffu;
        constexpr int kLanes = St::kRow / 16, kRows = 32 / kLanes;   // lanes a row, rows a pass
        const uint32_t dst = pr_smem(ring + st * St::kBytes);
        const int c = lane % kLanes;
#pragma unroll
        for (int j = 0; j < St::kKeys / kRows; ++j) {
            const int key = j * kRows + lane / kLanes;
            const int64_t o = __shfl_sync(0xffffffffu, off, key);
            const int64_t at = (o >= 0 ? o : 0) + c * 16;
            const uint32_t to = dst + key * St::kRow + ((c ^ (key & 7)) * 16);
            cp_async16(to, kb + at, o >= 0);
            cp_async16(to + St::kKeys * St::kRow, vb + at, o >= 0);
        }
        return have;
    };
    const int step = St::kTile;
    int t = k0 + warp * St::kKeys, tn = t;
    uint64_t have = 0;   // keys of the stages in order, 16 bits each
#pragma unroll
    for (int i = 0; i < St::kStages - 1; ++i, tn += step) {
        have |= (uint64_t)(tn < k1 ? request(tn, i) : 0u) << (16 * i);
        cp_async_commit();
    }

    // queries of rows g (and g + 8) as operand fragments, scale log2 e and a power of two a row taken out
    uint32_t qh[kSteps][2 * kHalves], ql[kSteps][2 * kHalves];
    float f[2] = {1.f, 1.f}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int pos[2] = {-1, -1};
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        const int r = g + 8 * h, row = pc.row + min(r, rows - 1), n = (int)a.gdiv.div((uint32_t)row);
        if (r < rows) pos[h] = pc.pos0 + n;
        const float* src = a.q + (size_t)(pc.tok0 + n) * a.ldq + (kvh * a.group + row - n * a.group) * HD + 2 * q;
        float2 x[kSteps][2];
        float mx = 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                float2 v = __ldg(reinterpret_cast<const float2*>(src + 16 * s + 8 * p));
                v.x *= a.scale2, v.y *= a.scale2;
                x[s][p] = v;
                mx = fmaxf(mx, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int e = 0;
        if (mx > 0.f && mx < INFINITY) e = max(-100, min(114, (int)((__float_as_uint(mx) >> 23) & 255) - 127 - 13));
        f[h] = __uint_as_float((uint32_t)(127 + e) << 23);
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int p = 0; p < 2; ++p)
                pm_split(x[s][p].x * inv, x[s][p].y * inv, &qh[s][p * kHalves + h], &ql[s][p * kHalves + h]);
    }
    float o[HD / 8][2 * kHalves];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2 * kHalves; ++e) o[n][e] = 0.f;

    const int mi = lane >> 3, r8 = lane & 7;
    int st = 0;
#pragma unroll 1
    while (t < k1) {
        const int ns = st == 0 ? St::kStages - 1 : st - 1;
        __syncwarp();   // every lane is done with the stage that is filled now
        have |= (uint64_t)(tn < k1 ? request(tn, ns) : 0u) << (16 * (St::kStages - 1));
        cp_async_commit();
        tn += step;
        cp_async_wait<St::kStages - 1>();
        __syncwarp();
        const uint32_t stage = pr_smem(ring + st * St::kBytes), vstage = stage + St::kKeys * St::kRow;
        const unsigned hv = (unsigned)have & 0xffffu;
        have >>= 16;
        const unsigned char* vrows = ring + st * St::kBytes + St::kKeys * St::kRow;
        st = st == St::kStages - 1 ? 0 : st + 1;

        float s[2][4] = {};   // 8 keys each
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
            uint32_t k[4];
            const int row = (mi >> 1) * 8 + r8, c = kk * 2 + (mi & 1);
            ldsm4(k, stage + row * St::kRow + ((c ^ (row & 7)) * 16));
            const uint32_t h0 = qh[kk][0], h1 = kHalves == 2 ? qh[kk][1] : 0u, h2 = qh[kk][kHalves], h3 = kHalves == 2 ? qh[kk][3 & (2 * kHalves - 1)] : 0u;
            const uint32_t l0 = ql[kk][0], l1 = kHalves == 2 ? ql[kk][1] : 0u, l2 = ql[kk][kHalves], l3 = kHalves == 2 ? ql[kk][3 & (2 * kHalves - 1)] : 0u;
            pm_mma(s[0], l0, l1, l2, l3, k[0], k[1]);
            pm_mma(s[1], l0, l1, l2, l3, k[2], k[3]);
            pm_mma(s[0], h0, h1, h2, h3, k[0], k[1]);
            pm_mma(s[1], h0, h1, h2, h3, k[2], k[3]);
        }
        const bool whole = hv == 0xffffu && t + St::kKeys - 1 <= p_first && (!a.window || t > p_last - a.window);
        uint32_t ph[2][2] = {}, pl[2][2] = {};   // [8 keys][rows g, g + 8]
        float corr[2] = {1.f, 1.f};
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            float v[4] = {s[0][2 * h] * f[h], s[0][2 * h + 1] * f[h], s[1][2 * h] * f[h], s[1][2 * h + 1] * f[h]};
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = (i >> 1) * 8 + 2 * q + (i & 1), kt = t + k;
                    if (!((hv >> k) & 1u) || kt > pos[h] || (a.window && kt <= pos[h] - a.window)) v[i] = -INFINITY;
                }
            }
            float mx = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(m[h], attn_lift(mx));
            corr[h] = m[h] == mn ? 1.f : exp2f(m[h] - mn);
            m[h] = mn;
            const float ref = mn == -INFINITY ? 0.f : mn;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = exp2f(v[i] - ref);
            l[h] = l[h] * corr[h] + ((v[0] + v[1]) + (v[2] + v[3]));
            pm_split(v[0], v[1], &ph[0][h], &pl[0][h]);
            pm_split(v[2], v[3], &ph[1][h], &pl[1][h]);
        }
        if (!whole) {   // zero times a value that is not finite: leave the piece to the rows' own pace
            uint32_t nonfinite = 0;
            for (int i = lane; i < St::kKeys * St::kRow / 4; i += 32) {
                const uint32_t v = reinterpret_cast<const uint32_t*>(vrows)[i];
                nonfinite |= (uint32_t)((v & 0x7C00u) == 0x7C00u) | (uint32_t)((v & 0x7C000000u) == 0x7C000000u);
            }
            if (nonfinite) *reinterpret_cast<volatile int*>(odd) = 1;
        }
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) {
            uint32_t v[4];
            const int row = (mi & 1) * 8 + r8, c = n * 2 + (mi >> 1);
            ldsm4_trans(v, vstage + row * St::kRow + ((c ^ (row & 7)) * 16));
            float d[2][4] = {};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                pm_mma(d[i], pl[0][0], pl[0][1], pl[1][0], pl[1][1], v[2 * i], v[2 * i + 1]);
                pm_mma(d[i], ph[0][0], ph[0][1], ph[1][0], ph[1][1], v[2 * i], v[2 * i + 1]);
#pragma unroll
                for (int e = 0; e < 2 * kHalves; ++e) o[2 * n + i][e] = fmaf(o[2 * n + i][e], corr[e >> 1], d[i][e]);
            }
        }
        t += step;
    }
    cp_async_wait<0>();
    if (bad) report_bad(a.status);
    __syncthreads();
    if (*odd) {
        for (int r = warp; r < rows; r += St::kWarps) attn_row_slow<__half, RB, HD>(a, pc, r);
        return;
    }
    float* red = reinterpret_cast<float*>(smem);
    constexpr int kW = HD + 2;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        float* w = red + (warp * RB + g + 8 * h) * kW;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(w + n * 8 + 2 * q) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if (q == 0) *reinterpret_cast<float2*>(w + HD) = make_float2(m[h], l[h]);
    }
    __syncthreads();
    merge_warps<HD, RB, St::kWarps, true>(a, pc, red);
}

template <int HD, int RB>
__global__ void __launch_bounds__(PmStage<HD, RB>::kThreads, 2) paged_mma_kernel(const __grid_constant__ PagedAttnArgs a) {
    using St = PmStage<HD, RB>;
    extern __shared__ __align__(128) unsigned char pr_smem_raw[];
    __shared__ AttnRun run;
    __shared__ AttnPiece pieces[St::kWarps];
    __shared__ int odd;
    if (!a.balanced) {
        AttnPiece p;
        if (attn_block<RB, St::kTile, St::kThreads>(a, 1, &p)) mma_piece<HD, RB>(a, p, pr_smem_raw, &odd);
        return;
    }
    AttnSchedule& sched = *reinterpret_cast<AttnSchedule*>(pr_smem_raw + St::kSmem);
    const int per_head = attn_schedule<RB, St::kTile, kPrExtra, St::kThreads>(a, sched, 1);
    if (threadIdx.x == 0) run = attn_run(a, per_head);
    __syncthreads();
    pdl_launch_dependents();
    bool begun = false;
    const AttnPiece& p = pieces[threadIdx.x >> 5];
    for (int64_t at = run.u; (at = attn_next<RB, St::kTile, kPrExtra>(a, sched, run, at, 1, &pieces[threadIdx.x >> 5])) != 0;) {
        mma_piece<HD, RB>(a, p, pr_smem_raw, &odd);
        __syncthreads();
        if (p.slot == 1) {
            begun = true;
            if (threadIdx.x == 0) attn_header(a, &p);
        }
    }
    if (!begun && threadIdx.x == 0) attn_header(a, nullptr);
}

template <int HD, int RB>
static tvb_status launch_mma(PagedAttnArgs a, cudaStream_t st) {
    using St = PmStage<HD, RB>;
    static int set[kMaxDevices];
    constexpr int smem = St::kSmem + (int)sizeof(AttnSchedule);
    TVB_TRY(allow_smem(reinterpret_cast<const void*>(paged_mma_kernel<HD, RB>), smem, set));
    a.min_units = 1 + kPrExtra;
    Workspace ws(st);
    dim3 grid;
    if (a.balanced) {
        grid = dim3(2u * (unsigned)num_sms());
        TVB_TRY((attn_workspace<RB, HD>(&a, (int)grid.x, &ws)));
    } else {
        grid = dim3((unsigned)(((int64_t)a.s.n_tokens * a.group) / RB + a.s.n_seqs), (unsigned)a.nkv);
    }
    paged_mma_kernel<HD, RB><<<grid, St::kThreads, smem, st>>>(a);
    TVB_TRY(check_launch("paged_mma_kernel"));
    return launch_merge<RB, HD>(a, (int)grid.x, st);
}

template <typename T, int HD, int RB>
__global__ void __launch_bounds__(PrStage<T, HD>::kThreads, 2) paged_rows_kernel(const __grid_constant__ PagedAttnArgs a) {
    extern __shared__ __align__(128) unsigned char pr_smem_raw[];
    __shared__ AttnRun run;
    using St = PrStage<T, HD>;
    __shared__ AttnPiece pieces[St::kWarps];
    if (!a.balanced) {
        AttnPiece p;
        if (attn_block<RB, St::kTile, St::kThreads>(a, 1, &p)) rows_piece<T, HD, RB>(a, p, pr_smem_raw);
        return;
    }
    AttnSchedule& sched = *reinterpret_cast<AttnSchedule*>(pr_smem_raw + rows_smem<T, HD, RB>());
    const int per_head = attn_schedule<RB, St::kTile, kPrExtra, St::kThreads>(a, sched, 1);
    if (threadIdx.x == 0) run = attn_run(a, per_head);
    __syncthreads();
    pdl_launch_dependents();
    bool begun = false;
    const AttnPiece& p = pieces[threadIdx.x >> 5];
    for (int64_t at = run.u; (at = attn_next<RB, St::kTile, kPrExtra>(a, sched, run, at, 1, &pieces[threadIdx.x >> 5])) != 0;) {
        rows_piece<T, HD, RB>(a, p, pr_smem_raw);
        __syncthreads();
        if (p.slot == 1) {
            begun = true;
            if (threadIdx.x == 0) attn_header(a, &p);
        }
    }
    if (!begun && threadIdx.x == 0) attn_header(a, nullptr);
}

template <typename T, int HD, int RB>
static tvb_status launch_rows(PagedAttnArgs a, cudaStream_t st) {
    static int set[kMaxDevices];
    using St = PrStage<T, HD>;
    constexpr int smem = rows_smem<T, HD, RB>() + (int)sizeof(AttnSchedule);
    TVB_TRY(allow_smem(reinterpret_cast<const void*>(paged_rows_kernel<T, HD, RB>), smem, set));
    a.min_units = 1 + kPrExtra;
    Workspace ws(st);
    dim3 grid;
    if (a.balanced) {
        grid = dim3(2u * (unsigned)num_sms());
        TVB_TRY((attn_workspace<RB, HD>(&a, (int)grid.x, &ws)));
    } else {
        grid = dim3((unsigned)(((int64_t)a.s.n_tokens * a.group) / RB + a.s.n_seqs), (unsigned)a.nkv);
    }
    paged_rows_kernel<T, HD, RB><<<grid, St::kThreads, smem, st>>>(a);
    TVB_TRY(check_launch("paged_rows_kernel"));
    return launch_merge<RB, HD>(a, (int)grid.x, st);
}

template <typename T, int HD>
static tvb_status launch_rows_rb(const PagedAttnArgs& a, int rows, cudaStream_t st) {
    if (rows <= 1) return launch_rows<T, HD, 1>(a, st);
    if (rows <= 2) return launch_rows<T, HD, 2>(a, st);
    if constexpr (sizeof(T) == 2) return rows <= 8 ? launch_mma<HD, 8>(a, st) : launch_mma<HD, 16>(a, st);
    else return rows <= 4 ? launch_rows<T, HD, 4>(a, st) : launch_rows<T, HD, 8>(a, st);
}

}  // namespace tvb

extern "C" tvb_status tvb_attention_paged(float* out, int ldo, float* lse, const float* q, int ldq,
                                          const tvb_kv_pages* kv, const tvb_paged_batch* batch, int nh, int nkv, int hd,
                                          float scale, int window, unsigned* status, void* stream) {
    using namespace tvb;
    TVB_REQUIRE(hd == 64 || hd == 128, "attention_paged: head_dim %d (64 and 128 are built)", hd);
    TVB_REQUIRE(nh > 0 && nkv > 0 && nh % nkv == 0 && nh <= 65535, "attention_paged: heads %d / kv heads %d", nh, nkv);
    PagedAttnArgs a = {};
    TVB_TRY(paged_cache_arg("attention_paged", kv, nkv, hd, &a.kv));
    TVB_TRY(paged_batch_arg("attention_paged", batch, kv, &a.s));
    if (!a.s.n_tokens || !a.s.n_seqs || !a.s.max_new) return TVB_OK;   // an empty buffer may have no address
    TVB_REQUIRE(out && q, "attention_paged: null pointer");
    TVB_REQUIRE(ldq >= nh * hd && ldo >= nh * hd && ((ldq | ldo) & 3) == 0, "attention_paged: leading dimensions %d, %d",
                ldq, ldo);
    TVB_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
                "attention_paged: q and out must be 16-byte aligned");
    TVB_REQUIRE(window >= 0, "attention_paged: window %d", window);
    TVB_REQUIRE(scale == scale, "attention_paged: scale is NaN");
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.ldq = ldq;
    a.ldo = ldo;
    a.nh = nh;
    a.nkv = nkv;
    a.group = nh / nkv;
    a.gdiv = FastDiv((uint32_t)a.group);
    a.scale2 = scale * 1.4426950408889634f;
    a.window = window;
    a.status = status;
    const cudaStream_t st = as_stream(stream);
    const int64_t rows64 = (int64_t)std::min(a.s.max_new, a.s.n_tokens) * a.group;
    const int rows = (int)std::min<int64_t>(rows64, 1 << 20);
    const bool f16 = kv->dtype == TVB_F16;
    const int64_t span = window ? std::min<int64_t>(a.s.max_kv, (int64_t)window + a.s.max_new) : a.s.max_kv;
    const int64_t few = (f16 ? 1 : 2) * num_sms();
    const int64_t row_blocks = ((int64_t)a.s.n_tokens * a.group / (f16 ? 16 : 8) + a.s.n_seqs) * nkv;
    const bool tensor = rows >= (f16 ? kTensorRows16 : kTensorRows32) && (row_blocks > few || row_blocks * span > few * kFewSpan);
    // many sequences or row blocks fill the SMs evenly enough block by block
    const int64_t blocks = ((int64_t)a.s.n_tokens * a.group / (tensor ? 128 : 8) + a.s.n_seqs) * nkv;
    // (the schedule's sums are 32 bits; a tile is 48 keys or more)
    a.balanced = a.s.n_seqs <= kAttnSeqs && span > kWholeKeys && blocks <= 64 * num_sms() &&
                 blocks / nkv * (span / 48 + 4) < INT_MAX;
    if (tensor) {
        TVB_TRY(paged_attn_chunk(a, hd, f16, st));
    } else if (hd == 128) {
        TVB_TRY((f16 ? launch_rows_rb<__half, 128>(a, rows, st) : launch_rows_rb<float, 128>(a, rows, st)));
    } else {
        TVB_TRY((f16 ? launch_rows_rb<__half, 64>(a, rows, st) : launch_rows_rb<float, 64>(a, rows, st)));
    }
    return TVB_OK;
}
