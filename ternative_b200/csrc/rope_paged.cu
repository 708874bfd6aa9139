// Rotary positions of a serving step's new tokens with the append to the paged
// cache (tvb_rope_append_paged).
//
//   (a, b) -> m (a cos t - b sin t, b cos t + a sin t),   t = pos f_i
//
// for the pairs i of each head's first rot_dim dimensions, f_i = theta^(-2 i /
// rot_dim) scaled for long contexts.  The host turns f_i into turns a position
// (f_i / 2 pi, 64 bits); the kernel multiplies by the position, takes the
// fraction of a turn in [-1/2, 1/2] in 64 bits and only then goes to 32, so the
// angle's error is 2 pi 2^-26 at any position (an F32 angle at position 30,000
// is off by 1e-3).
//
// Memory bound: q is read and written once, k and v are read once and written
// in the cache's type.  A CTA takes a token: its cosines and sines go to shared
// memory once (all heads share them), then every thread moves items of 8
// dimensions as two float4.
#include <climits>
#include <cmath>

#include "paged.cuh"

namespace tvb {

constexpr int kRpThreads = 256;
constexpr int kRpMaxPairs = 128;

struct RopeArgs {
    const float *q, *k, *v;
    float* q_out;
    int ldq, ldk, ldv, ldqo;
    int nh, nkv, hd;
    int rot, interleaved;
    int f16;         // cache type
    float m;
    unsigned* status;
    PagedKV kv;
    PagedSeqs s;
    double turns[kRpMaxPairs];   // f_i / 2 pi
};

__device__ __forceinline__ void rp_store(unsigned char* p, int elem, float4 x, bool f16) {
    if (f16) {
        const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);   // the cache's rounding
        uint2 u;
        u.x = *reinterpret_cast<const uint32_t*>(&a);
        u.y = *reinterpret_cast<const uint32_t*>(&b);
        *reinterpret_cast<uint2*>(p + elem * 2) = u;
    } else {
        *reinterpret_cast<float4*>(p + elem * 4) = x;
    }
}

// The cache row and position of token `row` if it is sequence b's (one thread).  (Both
// ends are checked: before starts are known to be in order, b may begin behind the row.)
__device__ __forceinline__ bool rope_place(const RopeArgs& a, int row, int b, int64_t* off, int* pos) {
    *off = -1;
    if (b < 0) return false;
    const SeqView v = seq_view(a.s, b);
    if (!v.ok || row < v.row0 || row - v.row0 >= v.n) return false;
    *pos = v.pos0 + (row - v.row0);
    *off = paged_offset(a.kv, a.s.table + (size_t)b * a.s.table_ld, *pos);
    return *off >= 0;
}

// Whole CTA: a row that is nobody's, or whose page does not exist, or starts that go back.
__device__ __noinline__ void rope_odd_row(const RopeArgs& a, int row, int64_t* off, int* pos) {
    const bool back = seq_back<kRpThreads>(a.s, 0);
    if (back) {
        const int b = seq_last(a.s, row, [](int, int row0) { return row0; });
        __syncthreads();
        if (threadIdx.x == 0) rope_place(a, row, b, off, pos);
        __syncthreads();
    }
    // (a row behind the last sequence is nobody's, and no fault)
    if (threadIdx.x == 0 && (back || row < __ldg(a.s.cu + a.s.n_seqs))) report_bad(a.status);
}

// Whole CTA: reports sequences that cannot be; they may have no row of their own to do so.
__device__ __noinline__ void rope_report(const RopeArgs& a) {
    for (int b = threadIdx.x; b < a.s.n_seqs; b += kRpThreads)
        if (!seq_view(a.s, b).ok) report_bad(a.status);
}

__global__ void __launch_bounds__(kRpThreads) rope_append_kernel(const __grid_constant__ RopeArgs a) {
    __shared__ float4 cs[kRpMaxPairs / 2];   // cosine and sine of pairs 2i, 2i + 1; read 16 bytes at a time
    __shared__ int64_t s_off;   // the token's cache row; -1: skipped
    __shared__ int s_pos;
    const int tid = threadIdx.x, row = blockIdx.x;

    if (row == a.s.n_tokens) {   // one CTA more
        if (a.status) rope_report(a);
        return;
    }
    // the token's sequence: how many end at or before it, where starts are in order
    int ended = 0, next = 0;
    bool odd = false;   // starts go back, or the row is nobody's
    for (; next < a.s.n_seqs;) {
        const int b = next + tid;
        int row0 = INT_MIN, end = INT_MAX;
        if (b < a.s.n_seqs) row0 = __ldg(a.s.cu + b), end = __ldg(a.s.cu + b + 1);
        odd |= end < row0;
        const int n = __syncthreads_count(end <= row);
        ended += n;
        next += kRpThreads;
        if (n < kRpThreads) break;
    }
    if (tid == 0) odd |= !rope_place(a, row, ended < a.s.n_seqs ? ended : -1, &s_off, &s_pos);
    if (__syncthreads_or(odd)) rope_odd_row(a, row, &s_off, &s_pos);
    const int64_t off = s_off;
    if (off < 0) return;
    const int pos = s_pos;
    const int pairs = a.rot >> 1;
    for (int p = tid; p < pairs; p += kRpThreads) {
        const double x = (double)pos * a.turns[p];
        float sn, c;
        sincospif(2.0f * (float)(x - rint(x)), &sn, &c);
        reinterpret_cast<float2*>(cs)[p] = make_float2(c * a.m, sn * a.m);
    }
    __syncthreads();

    const int per_head = a.hd >> 3;
    const int items = (a.nh + 2 * a.nkv) * per_head;
    for (int it = tid; it < items; it += kRpThreads) {
        const int h = it / per_head, c = it - h * per_head;
        const bool is_q = h < a.nh, is_k = !is_q && h < a.nh + a.nkv;
        const bool turn = !(!is_q && !is_k) && c < (a.rot >> 3);
        const int o0 = turn && !a.interleaved ? 4 * c : 8 * c;
        const int o1 = turn && !a.interleaved ? 4 * c + (a.rot >> 1) : 8 * c + 4;
        const int kvh = is_q ? 0 : h - a.nh - (is_k ? 0 : a.nkv);
        const float* src = is_q ? a.q + (size_t)row * a.ldq + h * a.hd
                                : (is_k ? a.k + (size_t)row * a.ldk : a.v + (size_t)row * a.ldv) + kvh * a.hd;
        float4 x = *reinterpret_cast<const float4*>(src + o0);
        float4 y = *reinterpret_cast<const float4*>(src + o1);
        if (turn) {
            const float4 p = cs[2 * c], r = cs[2 * c + 1];
            // cosines p.x p.z r.x r.z, sines p.y p.w r.y r.w of pairs 4c .. 4c + 3
            if (a.interleaved) {
                x = make_float4(x.x * p.x - x.y * p.y, x.y * p.x + x.x * p.y, x.z * p.z - x.w * p.w,
                                x.w * p.z + x.z * p.w);
                y = make_float4(y.x * r.x - y.y * r.y, y.y * r.x + y.x * r.y, y.z * r.z - y.w * r.w,
                                y.w * r.z + y.z * r.w);
            } else {
                const float4 u = x, w = y;
                x = make_float4(u.x * p.x - w.x * p.y, u.y * p.z - w.y * p.w, u.z * r.x - w.z * r.y,
                                u.w * r.z - w.w * r.w);
                y = make_float4(w.x * p.x + u.x * p.y, w.y * p.z + u.y * p.w, w.z * r.x + u.z * r.y,
                                w.w * r.z + u.w * r.w);
            }
        }
        if (is_q) {
            float* dst = a.q_out + (size_t)row * a.ldqo + h * a.hd;
            *reinterpret_cast<float4*>(dst + o0) = x;
            *reinterpret_cast<float4*>(dst + o1) = y;
        } else {
            unsigned char* dst = (is_k ? a.kv.k : a.kv.v) + off + (int64_t)kvh * a.kv.head_stride;
            rp_store(dst, o0, x, a.f16);
            rp_store(dst, o1, y, a.f16);
        }
    }
}

// f_i / 2 pi of every pair, and the factor of cosine and sine.
static void rope_turns(const tvb_rope_config& r, double* turns, float* m) {
    const double two_pi = 6.283185307179586476925287;
    const double ln = std::log((double)r.theta);
    const double step = std::exp(-2.0 * ln / r.rot_dim);
    const int pairs = r.rot_dim / 2;
    *m = 1.0f;
    double lo = 0.0, width = 1.0;
    if (r.scaling == TVB_ROPE_YARN) {
        auto pair = [&](double t) { return r.rot_dim * std::log(r.original_len / (t * two_pi)) / (2.0 * ln); };
        lo = std::fmax(std::floor(pair(r.fast_turns)), 0.0);
        width = std::fmax(std::fmin(std::ceil(pair(r.slow_turns)), r.rot_dim - 1.0) - lo, 1e-3);
        *m = (float)(0.1 * std::log((double)r.factor) + 1.0);
    }
    double f = 1.0;
    for (int i = 0; i < pairs; ++i, f *= step) {
        double keep = 1.0;   // share of f that is not divided by factor
        if (r.scaling == TVB_ROPE_LINEAR) {
            keep = 0.0;
        } else if (r.scaling == TVB_ROPE_BANDS) {
            const double t = r.original_len * f / two_pi;
            keep = std::fmin(std::fmax((t - r.low_turns) / ((double)r.high_turns - r.low_turns), 0.0), 1.0);
        } else if (r.scaling == TVB_ROPE_YARN) {
            keep = 1.0 - std::fmin(std::fmax((i - lo) / width, 0.0), 1.0);
        }
        turns[i] = (f * keep + (keep < 1.0 ? f / r.factor * (1.0 - keep) : 0.0)) / two_pi;
    }
}

}  // namespace tvb

extern "C" tvb_status tvb_rope_append_paged(float* q_out, int ldqo, const float* q, int ldq, const float* k, int ldk,
                                            const float* v, int ldv, const tvb_kv_pages* kv,
                                            const tvb_paged_batch* batch, const tvb_rope_config* rope, int nh, int nkv,
                                            int hd, unsigned* status, void* stream) {
    using namespace tvb;
    TVB_REQUIRE(rope, "rope_append_paged: null pointer");
    TVB_REQUIRE(nh > 0 && nkv > 0 && hd > 0 && hd % 8 == 0 && hd <= 2 * kRpMaxPairs,
                "rope_append_paged: heads %d/%d, head_dim %d (a multiple of 8 up to %d)", nh, nkv, hd, 2 * kRpMaxPairs);
    TVB_REQUIRE(nh <= 65536 && nkv <= 65536, "rope_append_paged: heads %d/%d", nh, nkv);
    RopeArgs a;
    TVB_TRY(paged_cache_arg("rope_append_paged", kv, nkv, hd, &a.kv));
    TVB_TRY(paged_batch_arg("rope_append_paged", batch, kv, &a.s));
    if (!a.s.n_tokens || !a.s.n_seqs) return TVB_OK;   // an empty buffer may have no address
    TVB_REQUIRE(q_out && q && k && v, "rope_append_paged: null pointer");
    TVB_REQUIRE(ldq >= nh * hd && ldqo >= nh * hd && ldk >= nkv * hd && ldv >= nkv * hd &&
                    ((ldq | ldqo | ldk | ldv) & 3) == 0,
                "rope_append_paged: leading dimensions %d, %d, %d, %d", ldqo, ldq, ldk, ldv);
    TVB_REQUIRE(q_out != q || ldqo == ldq, "rope_append_paged: in place with leading dimensions %d and %d", ldqo, ldq);
    TVB_REQUIRE(((reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                  reinterpret_cast<uintptr_t>(v)) & 15) == 0,
                "rope_append_paged: buffers must be 16-byte aligned");
    TVB_REQUIRE(rope->rot_dim >= 0 && rope->rot_dim <= hd && rope->rot_dim % 8 == 0,
                "rope_append_paged: rot_dim %d (a multiple of 8 up to head_dim %d)", rope->rot_dim, hd);
    TVB_REQUIRE(rope->pairs == TVB_ROPE_HALF || rope->pairs == TVB_ROPE_INTERLEAVED, "rope_append_paged: pairs %d",
                rope->pairs);
    TVB_REQUIRE(rope->scaling >= TVB_ROPE_PLAIN && rope->scaling <= TVB_ROPE_YARN, "rope_append_paged: scaling %d",
                rope->scaling);
    TVB_REQUIRE(rope->theta > 1.0f && std::isfinite(rope->theta), "rope_append_paged: theta %g", rope->theta);
    if (rope->scaling != TVB_ROPE_PLAIN)
        TVB_REQUIRE(rope->factor >= 1.0f && std::isfinite(rope->factor), "rope_append_paged: factor %g", rope->factor);
    if (rope->scaling == TVB_ROPE_BANDS)
        TVB_REQUIRE(rope->original_len > 0 && rope->low_turns > 0.0f && rope->high_turns > rope->low_turns,
                    "rope_append_paged: original_len %d, turns %g..%g", rope->original_len, rope->low_turns,
                    rope->high_turns);
    if (rope->scaling == TVB_ROPE_YARN)
        TVB_REQUIRE(rope->original_len > 0 && rope->slow_turns > 0.0f && rope->fast_turns > rope->slow_turns,
                    "rope_append_paged: original_len %d, turns %g..%g", rope->original_len, rope->slow_turns,
                    rope->fast_turns);
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.ldqo = ldqo;
    a.nh = nh;
    a.nkv = nkv;
    a.hd = hd;
    a.rot = rope->rot_dim;
    a.interleaved = rope->pairs == TVB_ROPE_INTERLEAVED;
    a.f16 = kv->dtype == TVB_F16;
    a.status = status;
    a.m = 1.0f;
    if (a.rot) rope_turns(*rope, a.turns, &a.m);
    rope_append_kernel<<<(unsigned)a.s.n_tokens + 1u, kRpThreads, 0, as_stream(stream)>>>(a);
    return check_launch("rope_append_kernel");
}
