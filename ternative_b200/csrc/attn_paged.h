// Attention over the paged cache: what its kernels share (attn_paged.cu, one or
// few rows; attn_paged_tc.cu, chunks on the tensor cores) -- arguments, the
// split of the work over the SMs, and a row computed key by key.
#pragma once

#include "paged.cuh"

namespace tvb {

struct PagedAttnArgs {
    const float* q;
    float* out;
    float* lse;        // may be null
    int ldq, ldo;
    int nh, nkv, group;
    FastDiv gdiv;      // group
    float scale2;      // scale * log2(e): scores are kept as powers of two
    int window;        // 0: none
    int balanced;      // the grid shares the tiles evenly; else a CTA a row block
    int min_units;     // ... but no CTA gets fewer than this (tiles and blocks' extra)
    float* part;       // [CTA][2]: rows x hd weighted values, rows x (sum, maximum) of cut blocks
    int* header;       // [CTA][8]: the cut block that the CTA's last piece begins
    unsigned* status;
    PagedKV kv;
    PagedSeqs s;
};

constexpr int kAttnSeqs = 512;   // sequences that a balanced grid keeps in shared memory

// The work: row blocks (RB rows -- new token x query head of the group -- of one
// KV head of one sequence) with the tiles of TK keys that some row of the block
// sees, tile after tile, block after block, KV head after KV head; a block counts
// EX units more, before its tiles, for its start and end.  A balanced grid of G
// CTAs cuts the T units into G equal runs, whatever the lengths are; a block whose
// tiles a cut divides leaves partial sums and paged_merge_kernel joins them.
// Lengths are known on the device only, so every CTA adds up the sequences' tiles
// first (a few microseconds saved over a launch that does it).
struct AttnSchedule {
    int row0[kAttnSeqs], n[kAttnSeqs], kv[kAttnSeqs];
    int before[kAttnSeqs + 1];   // units of the earlier sequences, one KV head
};

struct AttnPiece {
    int b;              // sequence
    int tok0, pos0;     // its first row, its position
    int kvh;
    int row, rows;      // first row (token x head) of the block, rows of it
    int first, k0, k1;  // keys [max(first, k0), k1); tiles start at k0
    int tiles;
    int slot;           // -1: the whole block; else the CTA's partial 0 (continues a block) or 1 (begins one)
    int last_cta;       // slot 1: the CTA that ends the block
};

// Tiles of block i of a sequence; k0: where they start (multiples of `align`, a
// power of two, so that boxes of rows stay inside their page).
template <int RB, int TK>
__device__ __forceinline__ int attn_tiles(const PagedAttnArgs& a, int n, int pos0, int i, int align, int* first, int* k0,
                                          int* k1) {
    const int rows = min(RB, n * a.group - i * RB);
    const int p_first = pos0 + (int)a.gdiv.div((uint32_t)(i * RB));
    const int p_last = pos0 + (int)a.gdiv.div((uint32_t)(i * RB + rows - 1));
    *first = a.window ? max(0, p_first - a.window + 1) : 0;
    *k0 = *first & ~(align - 1);
    *k1 = p_last + 1;
    return (*k1 - *k0 + TK - 1) / TK;
}

// Whole warp: no rows for what is not in use.
static __device__ __noinline__ void attn_drop_unused(const PagedSeqs& s, int* n) {
    seq_scan(s, [&](int b, const SeqView&, bool used) {
        if (b < s.n_seqs && !used) n[b] = 0;
    });
}

// Whole CTA (NT threads): fills `s` and returns the units of one KV head.
template <int RB, int TK, int EX, int NT>
__device__ __forceinline__ int attn_schedule(const PagedAttnArgs& a, AttnSchedule& s, int align) {
    const int tid = threadIdx.x, lane = tid & 31;
    bool back = false;
    for (int b = tid; b < a.s.n_seqs; b += NT) {
        const SeqView v = seq_view(a.s, b);
        if (!v.ok && blockIdx.x == 0) report_bad(a.status);
        s.row0[b] = v.row0;
        s.n[b] = v.n;
        s.kv[b] = v.kv;
        back |= v.back;
    }
    if (__syncthreads_or(back)) {   // what overlaps an earlier sequence has no rows of its own
        if (tid < 32) attn_drop_unused(a.s, s.n);
        __syncthreads();
    }
    for (int b = tid >> 5; b < a.s.n_seqs; b += NT / 32) {
        const int n = s.n[b], blocks = (n * a.group + RB - 1) / RB;
        int t = 0, x, y, z;
        for (int i = lane; i < blocks; i += 32) t += attn_tiles<RB, TK>(a, n, s.kv[b] - n, i, align, &x, &y, &z) + EX;
        t = __reduce_add_sync(0xffffffffu, t);
        if (lane == 0) s.before[b + 1] = t;
    }
    __syncthreads();
    if (tid < 32) {
        int base = 0;
        for (int b0 = 0; b0 < a.s.n_seqs; b0 += 32) {
            int t = b0 + lane < a.s.n_seqs ? s.before[b0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, t, o);
                if (lane >= o) t += u;
            }
            if (b0 + lane < a.s.n_seqs) s.before[b0 + lane + 1] = base + t;
            base += __shfl_sync(0xffffffffu, t, 31);
        }
        if (lane == 0) s.before[0] = 0;
    }
    __syncthreads();
    return s.before[a.s.n_seqs];
}

// A CTA's run of units.
struct AttnRun {
    int64_t total, u, end;
    int per_head, ctas;
};

__device__ __forceinline__ AttnRun attn_run(const PagedAttnArgs& a, int per_head) {
    AttnRun r;
    r.per_head = per_head;
    r.total = (int64_t)per_head * a.nkv;
    r.ctas = (int)min((int64_t)gridDim.x, max((int64_t)1, r.total / a.min_units));
    r.u = r.total * min((int)blockIdx.x, r.ctas) / r.ctas;
    r.end = r.total * min((int)blockIdx.x + 1, r.ctas) / r.ctas;
    return r;
}

// Whole warp: the next piece from unit u of the run on, into *out (shared memory
// of this warp); returns the unit after it, 0 when the run has no more.  Not
// inlined, for the instruction cache's sake.
template <int RB, int TK, int EX>
__device__ __noinline__ int64_t attn_next(const PagedAttnArgs& a, const AttnSchedule& s, const AttnRun& r, int64_t u,
                                          int align, AttnPiece* out) {
    const int lane = threadIdx.x & 31;
    AttnPiece p;
again:
    if (u >= r.end) return 0;
    p.kvh = (int)(u / r.per_head);
    int t = (int)(u - (int64_t)p.kvh * r.per_head);
    int lo = 0, hi = a.s.n_seqs - 1;   // the last sequence that starts at or before t
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s.before[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    const int b = lo, n = s.n[b];
    p.b = b;
    p.tok0 = s.row0[b];
    p.pos0 = s.kv[b] - n;
    t -= s.before[b];
    const int blocks = (n * a.group + RB - 1) / RB;
    int i0 = 0, tiles = 0, x, y, z;
#pragma unroll 1
    for (;; i0 += 32) {   // the block that holds unit t of the sequence
        const int nt = i0 + lane < blocks ? attn_tiles<RB, TK>(a, n, p.pos0, i0 + lane, align, &x, &y, &z) + EX : 0;
        int sum = nt;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, sum > t);
        if (past || i0 + 32 >= blocks) {
            const int l = past ? __ffs(past) - 1 : 31;
            tiles = __shfl_sync(0xffffffffu, nt, l);
            t -= __shfl_sync(0xffffffffu, sum, l) - tiles;
            i0 += l;
            break;
        }
        t -= __shfl_sync(0xffffffffu, sum, 31);
    }
    // t: unit of the block, `tiles` of them; the tiles are those from EX on
    const int begin = max(t, EX), end = (int)min((int64_t)tiles, t + r.end - u);
    const int64_t first_unit = u - t;
    u = first_unit + end;
    if (begin >= end) goto again;   // the run ends, or begins, before the block's first tile
    attn_tiles<RB, TK>(a, n, p.pos0, i0, align, &p.first, &p.k0, &p.k1);
    p.row = i0 * RB;
    p.rows = min(RB, n * a.group - p.row);
    p.tiles = end - begin;
    p.slot = p.tiles == tiles - EX ? -1 : begin > EX ? 0 : 1;
    p.last_cta = (int)(((first_unit + tiles) * r.ctas - 1) / r.total);
    p.k0 += (begin - EX) * TK;
    p.k1 = min(p.k1, p.k0 + p.tiles * TK);
    __syncwarp();
    if (lane == 0) *out = p;
    __syncwarp();
    return u;
}

// The first row block of a sequence in an unbalanced grid.
template <int RB>
struct AttnFirst {
    int group;
    __device__ __forceinline__ int64_t operator()(int b, int row0) const { return ((int64_t)row0 * group) / RB + b; }
    // block x, at or behind the first, is one of the sequence's
    __device__ __forceinline__ bool has(const SeqView& v, int b, int x) const {
        return v.ok && (x - (*this)(b, v.row0)) * RB < (int64_t)v.n * group;
    }
};

// Whole CTA: the sequence of a block where starts go back (between the first `next`, or
// further on), or -1.
template <int RB, int NT>
__device__ __noinline__ int attn_odd_block(const PagedAttnArgs& a, int next, bool back) {
    if (!back && !seq_back<NT>(a.s, next)) return -1;
    const AttnFirst<RB> first = {a.group};
    const int x = (int)blockIdx.x, b = seq_last(a.s, x, first);
    return b >= 0 && first.has(seq_view(a.s, b), b, x) ? b : -1;
}

// The piece of a CTA of an unbalanced grid: row block blockIdx.x of the batch,
// whole.  Block floor(row0 g / RB) + b is the first of sequence b, so blocks of
// sequences in use never overlap and floor(T g / RB) + n of them are enough.
template <int RB, int TK, int NT>
__device__ __forceinline__ bool attn_block(const PagedAttnArgs& a, int align, AttnPiece* p) {
    if ((blockIdx.x | blockIdx.y) == 0) {   // (a sequence that cannot be is no CTA's)
        for (int b = threadIdx.x; b < a.s.n_seqs; b += NT)
            if (!seq_view(a.s, b).ok) report_bad(a.status);
    }
    const AttnFirst<RB> first = {a.group};
    const int x = (int)blockIdx.x;
    int next;
    bool back;
    int b = seq_count<NT>(a.s, x, first, &next, &back) - 1;
    back = __syncthreads_or(back);
    SeqView v = {};
    if (b >= 0) v = seq_view(a.s, b);
    if (!back && v.ok && v.n) {
        // a later sequence that starts in front of the next one starts before this one's end: it cannot claim the block
        if (!first.has(v, b, x)) return false;
    } else {
        b = attn_odd_block<RB, NT>(a, next, back);
        if (b < 0) return false;
        v = seq_view(a.s, b);
    }
    const int i = x - (int)first(b, v.row0);
    p->b = b;
    p->tok0 = v.row0;
    p->pos0 = v.pos0;
    p->kvh = blockIdx.y;
    p->row = i * RB;
    p->rows = min(RB, v.n * a.group - p->row);
    p->tiles = attn_tiles<RB, TK>(a, v.n, v.pos0, i, align, &p->first, &p->k0, &p->k1);
    p->slot = -1;
    return true;
}

// Partial (CTA, slot) of RB rows: HD weighted values of each, then each row's sum
// and maximum; partials start at multiples of 16 bytes.
template <int RB, int HD>
__host__ __device__ constexpr int attn_part_floats() {
    return (RB * (HD + 2) + 3) / 4 * 4;
}
template <int RB, int HD>
__device__ __forceinline__ float* attn_part(const PagedAttnArgs& a, int cta, int slot, int r) {
    return a.part + ((size_t)cta * 2 + slot) * attn_part_floats<RB, HD>() + (size_t)r * HD;
}
template <int RB, int HD>
__device__ __forceinline__ float* attn_part_sum(const PagedAttnArgs& a, int cta, int slot, int r) {
    return a.part + ((size_t)cta * 2 + slot) * attn_part_floats<RB, HD>() + RB * HD + 2 * r;
}

// Tells paged_merge_kernel about the cut block that this CTA begins (one thread).
__device__ __forceinline__ void attn_header(const PagedAttnArgs& a, const AttnPiece* p) {
    int* h = a.header + blockIdx.x * 8;
    h[0] = p ? p->rows : 0;
    if (p) h[1] = p->tok0, h[2] = p->row, h[3] = p->kvh, h[4] = p->last_cta;
}

template <typename T, int ND>
__device__ __forceinline__ void pr_load(const unsigned char* p, float (&f)[ND]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (ND == 4) {
            const float4 x = *reinterpret_cast<const float4*>(p);
            f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
        } else {
            const float2 x = *reinterpret_cast<const float2*>(p);
            f[0] = x.x, f[1] = x.y;
        }
    } else {
        if constexpr (ND == 4) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
            f[0] = x.x, f[1] = x.y, f[2] = y.x, f[3] = y.y;
        } else {
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(p));
            f[0] = x.x, f[1] = x.y;
        }
    }
}

// F16 planes of probabilities hold nothing below 2^-25: relative to the row's maximum
// a key 17.4 nats below it would vanish from the output while the sum counted it.  So
// the tensor-core kernels over F16 caches take powers relative to the maximum less 15:
// 2^15 at most, 2^-40 of that at least.  (A maximum so large that subtracting rounds
// stays as it is: neighbouring scores are then further apart than that.)  Sum, values
// and what they refer to go together, so nothing after them knows.
__device__ __forceinline__ float attn_lift(float mx) { return fabsf(mx) < 4194304.f ? mx - 15.f : mx; }

// log of the sum of exponentials from the sum l of powers 2^(s - m)
__device__ __forceinline__ float attn_lse(float l, float m) {
    return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}
// What the weighted values are divided by: no key gives zeros, NaN stays.
__device__ __forceinline__ float attn_inv(float l) { return l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l); }

// What a row leaves (one warp, ND dimensions a lane).
template <int RB, int HD, int ND>
__device__ __forceinline__ void attn_row_store(const PagedAttnArgs& a, const AttnPiece& p, int r, float l, float m,
                                               const float (&o)[ND]) {
    const int lane = threadIdx.x & 31;
    if (p.slot >= 0) {
        float* pp = attn_part<RB, HD>(a, blockIdx.x, p.slot, r);
        if (lane == 0) *reinterpret_cast<float2*>(attn_part_sum<RB, HD>(a, blockIdx.x, p.slot, r)) = make_float2(l, m);
#pragma unroll
        for (int d = 0; d < ND; d += 2) *reinterpret_cast<float2*>(pp + lane * ND + d) = make_float2(o[d], o[d + 1]);
    } else {
        const int t = (int)a.gdiv.div((uint32_t)(p.row + r)), tok = p.tok0 + t;
        const int head = p.kvh * a.group + p.row + r - t * a.group;
        const float inv = attn_inv(l);
        float* po = a.out + (size_t)tok * a.ldo + head * HD + lane * ND;
#pragma unroll
        for (int d = 0; d < ND; d += 2) *reinterpret_cast<float2*>(po + d) = make_float2(o[d] * inv, o[d + 1] * inv);
        if (a.lse && lane == 0) a.lse[(size_t)tok * a.nh + head] = attn_lse(l, m);
    }
}

// One row by one warp, key by key: for tiles whose masked values are not finite
// or whose pages do not exist, which the tensor cores cannot skip, and for rows that
// see something that planes cannot hold.
template <typename T, int RB, int HD>
__device__ __noinline__ void attn_row_slow(const PagedAttnArgs& a, const AttnPiece& p, int r) {
    constexpr int ND = HD / 32;
    const int lane = threadIdx.x & 31;
    const int* table = a.s.table + (size_t)p.b * a.s.table_ld;
    const int t = (int)a.gdiv.div((uint32_t)(p.row + r)), tok = p.tok0 + t, pos = p.pos0 + t;
    const int head = p.kvh * a.group + p.row + r - t * a.group;
    float q[ND], o[ND], kf[ND], vf[ND];
    pr_load<float, ND>(reinterpret_cast<const unsigned char*>(a.q + (size_t)tok * a.ldq + head * HD + lane * ND), q);
#pragma unroll
    for (int d = 0; d < ND; ++d) q[d] *= a.scale2, o[d] = 0.f;
    float m = -INFINITY, l = 0.f;
    int k0 = max(p.k0, p.first);
    if (a.window) k0 = max(k0, pos - a.window + 1);
    for (int k = k0; k < min(p.k1, pos + 1); ++k) {
        const int64_t off = paged_offset(a.kv, table, k);
        if (off < 0) continue;
        const int64_t at = off + (int64_t)p.kvh * a.kv.head_stride + lane * ND * (int)sizeof(T);
        pr_load<T, ND>(a.kv.k + at, kf);
        pr_load<T, ND>(a.kv.v + at, vf);
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) s = fmaf(q[d], kf[d], s);
        s = warp_sum(s);
        const float mn = fmaxf(m, s);
        const float c = m == mn ? 1.f : exp2f(m - mn), w = s == -INFINITY ? 0.f : exp2f(s - mn);
        l = l * c + w;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = fmaf(o[d], c, w * vf[d]);
        m = mn;
    }
    attn_row_store<RB, HD, ND>(a, p, r, l, m, o);
}

// Joins the pieces of the block that CTA blockIdx.x of the attention kernel
// began, in key order; a warp a row.
template <int RB, int HD>
__global__ void __launch_bounds__(256) paged_merge_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int ND = HD / 32;
    pdl_wait();
    const int c0 = blockIdx.x, lane = threadIdx.x & 31;
    const int* h = a.header + c0 * 8;
    const int rows = h[0];
    if (!rows) return;
    AttnPiece p;
    p.tok0 = h[1], p.row = h[2], p.kvh = h[3];
    p.slot = -1;
    const int last = h[4];
    for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.y * 8) {
        float M = -INFINITY;
        for (int c = c0 + lane; c <= last; c += 32) M = fmaxf(M, attn_part_sum<RB, HD>(a, c, c == c0, r)[1]);
        M = warp_max(M);
        float L = 0.f, o[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = 0.f;
        for (int b = c0; b <= last; b += 32) {
            // lane i: weight of piece b + i; then the pieces' values, several loads at once
            const int c = b + lane;
            float2 lm = make_float2(0.f, -INFINITY);
            if (c <= last) lm = *reinterpret_cast<const float2*>(attn_part_sum<RB, HD>(a, c, c == c0, r));
            const float w = lm.y == -INFINITY ? (lm.x == 0.f ? 0.f : 1.f) : exp2f(lm.y - M);   // no maximum but a sum: NaN
            L += warp_sum(w == 0.f ? 0.f : lm.x * w);
            const int n = min(32, last - b + 1);
#pragma unroll 8
            for (int k = 0; k < n; ++k) {
                const float wk = __shfl_sync(0xffffffffu, w, k);
                float x[ND];
                pr_load<float, ND>(reinterpret_cast<const unsigned char*>(attn_part<RB, HD>(a, b + k, b + k == c0, r) + lane * ND), x);
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d] = wk != 0.f ? fmaf(x[d], wk, o[d]) : o[d];
            }
        }
        attn_row_store<RB, HD, ND>(a, p, r, L, M, o);
    }
}

template <int RB, int HD>
tvb_status launch_merge(const PagedAttnArgs& a, int ctas, cudaStream_t st) {
    if (!a.balanced) return TVB_OK;
    TVB_CUDA(launch_maybe_pdl(paged_merge_kernel<RB, HD>, dim3((unsigned)ctas, (unsigned)((RB + 7) / 8)), dim3(256), 0, st, true, a));
    return check_launch("paged_merge_kernel");
}

// Workspace of a balanced grid.
template <int RB, int HD>
tvb_status attn_workspace(PagedAttnArgs* a, int ctas, Workspace* ws) {
    const size_t part = (size_t)ctas * 2 * attn_part_floats<RB, HD>() * 4;
    TVB_TRY(ws->get(part + (size_t)ctas * 32));
    a->part = ws->at<float>();
    a->header = ws->at<int>(part);
    return TVB_OK;
}

tvb_status paged_attn_chunk(const PagedAttnArgs& a, int hd, bool f16, cudaStream_t st);   // attn_paged_tc.cu

}  // namespace tvb
