// Attention over the paged cache: shared by its kernels (attn_paged.cu).
#pragma once

#include "paged.cuh"

namespace tvb {

struct PagedAttnArgs {
    const float* q;
    float* out;
    float* lse;        // may be null
    int ldq, ldo;
    int nh, nkv, group;
    float scale2;      // scale * log2(e): scores are kept as powers of two
    int window;        // 0: none
    int split_len;     // keys a split
    int nsplit;        // splits of the longest sequence; 1: no partials
    float* part;       // [split][token][head][hd + 2]: sum, max, weighted values
    unsigned* status;
    PagedKV kv;
    PagedSeqs s;
};

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

// Sequence and first row of row block x, RB rows a block: block floor(cu[b] g /
// RB) + b is the first of sequence b, so blocks of neighbours never overlap and
// floor(T g / RB) + n of them are enough.  Whole CTA; b = n_seqs past the end.
template <int RB, int NT>
__device__ __forceinline__ int row_block_seq(const PagedSeqs& s, int group, int x, int* first) {
    int started = 0;
    for (int b0 = 0; b0 < s.n_seqs; b0 += NT) {
        const int b = b0 + (int)threadIdx.x;
        const bool at = b < s.n_seqs && (int)(((int64_t)__ldg(s.cu + b) * group) / RB) + b <= x;
        const int n = __syncthreads_count(at);
        started += n;
        if (n < NT) break;
    }
    const int b = started - 1;
    if (b < 0) return s.n_seqs;
    *first = (x - (int)(((int64_t)__ldg(s.cu + b) * group) / RB) - b) * RB;
    return b;
}

// What a row leaves: its sum l, maximum m and weighted values o (ND dimensions a
// lane) as the partial of `split`, or divided into out and lse.
template <int HD, int ND>
__device__ __forceinline__ void paged_row_store(const PagedAttnArgs& a, int split, int tok, int head, int lane, float l,
                                                float m, const float (&o)[ND]) {
    if (a.nsplit > 1) {
        float* pp = a.part + (((size_t)split * a.s.n_tokens + tok) * a.nh + head) * (HD + 2);
        if (lane == 0) *reinterpret_cast<float2*>(pp) = make_float2(l, m);
#pragma unroll
        for (int d = 0; d < ND; ++d) pp[2 + lane * ND + d] = o[d];
    } else {
        const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);   // no key: zeros; NaN stays
        float* po = a.out + (size_t)tok * a.ldo + head * HD + lane * ND;
#pragma unroll
        for (int d = 0; d < ND; ++d) po[d] = o[d] * inv;
        if (a.lse && lane == 0)
            a.lse[(size_t)tok * a.nh + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    }
}

// One row by one warp, key by key: for tiles whose masked values are not finite
// or whose pages do not exist, which the tensor cores cannot skip.
template <typename T, int HD>
__device__ __noinline__ void paged_row_slow(const PagedAttnArgs& a, const SeqView& sv, const int* table, int kvh, int split,
                                            int row, int k0, int k1) {
    constexpr int ND = HD / 32;
    const int lane = threadIdx.x & 31;
    const int tok = sv.row0 + row / a.group, head = kvh * a.group + row % a.group, pos = sv.pos0 + row / a.group;
    float q[ND], o[ND], kf[ND], vf[ND];
    pr_load<float, ND>(reinterpret_cast<const unsigned char*>(a.q + (size_t)tok * a.ldq + head * HD + lane * ND), q);
#pragma unroll
    for (int d = 0; d < ND; ++d) q[d] *= a.scale2, o[d] = 0.f;
    float m = -INFINITY, l = 0.f;
    if (a.window) k0 = max(k0, pos - a.window + 1);
    for (int t = k0; t < min(k1, pos + 1); ++t) {
        const int64_t off = paged_offset(a.kv, table, t);
        if (off < 0) continue;
        const int64_t at = off + (int64_t)kvh * a.kv.head_stride + lane * ND * (int)sizeof(T);
        pr_load<T, ND>(a.kv.k + at, kf);
        pr_load<T, ND>(a.kv.v + at, vf);
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) s = fmaf(q[d], kf[d], s);
        s = warp_sum(s);
        const float mn = fmaxf(m, s);
        const float c = m == mn ? 1.f : exp2f(m - mn), p = s == -INFINITY ? 0.f : exp2f(s - mn);
        l = l * c + p;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = fmaf(o[d], c, p * vf[d]);
        m = mn;
    }
    paged_row_store<HD, ND>(a, split, tok, head, lane, l, m, o);
}

tvb_status paged_attn_chunk_f16(const PagedAttnArgs& a, int hd, cudaStream_t st);   // attn_paged_tc.cu

}  // namespace tvb
