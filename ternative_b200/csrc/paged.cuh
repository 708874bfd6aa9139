// The paged KV cache and the ragged batch of a serving step, as the device
// reads them (tvb_kv_pages, tvb_paged_batch), and stream-ordered workspaces.
#pragma once

#include "common.cuh"
#include "paged_seq.h"

namespace tvb {

// n / d and n % d for 0 <= n < 2^31 by one high multiplication: with s =
// ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1, n / d = (mulhi(n, m) + n)
// >> s (Granlund and Montgomery's round-up method; the sum stays below 2^32).
struct FastDiv {
    uint32_t d, m, s;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div), s(0) {
        while ((1ull << s) < div) ++s;
        m = (uint32_t)(((1ull << 32) * ((1ull << s) - div)) / div + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

struct PagedKV {
    unsigned char* k;
    unsigned char* v;
    int64_t page_stride, row_stride, head_stride;   // bytes
    int n_pages;
    FastDiv page;   // page size
};

struct PagedSeqs {
    const int* cu;
    const int* kv_len;
    const int* table;
    int n_seqs, n_tokens, max_new, max_kv, table_ld;
};

// Bytes from the start of a pool to (position t, head 0) of the sequence whose
// table row is `table`; -1 where the page does not exist.
__device__ __forceinline__ int64_t paged_offset(const PagedKV& kv, const int* table, int t) {
    const uint32_t p = kv.page.div((uint32_t)t);
    const int page = __ldg(table + p);
    if ((unsigned)page >= (unsigned)kv.n_pages) return -1;
    return (int64_t)page * kv.page_stride + (int64_t)((uint32_t)t - p * kv.page.d) * kv.row_stride;
}

__device__ __forceinline__ SeqView seq_view(const PagedSeqs& s, int b) {
    return seq_numbers(__ldg(s.cu + b), __ldg(s.cu + b + 1), __ldg(s.kv_len + b), s.n_tokens, s.max_new, s.max_kv);
}

// A sequence is in use when its own numbers fit (SeqView::ok) and it starts at or
// behind the end of every earlier one that has rows and whose numbers fit: rows then
// belong to one sequence at most.  Where starts never go back the numbers alone
// decide; else a whole warp walks through the sequences, 32 a turn: f(b, view, in
// use) with a lane's b, which may lie behind the last.
template <class F>
__device__ __forceinline__ void seq_scan(const PagedSeqs& s, F f) {
    const int lane = threadIdx.x & 31;
    int ends = 0;   // the largest so far
    for (int b0 = 0; b0 < s.n_seqs; b0 += 32) {
        const int b = b0 + lane;
        SeqView v = {};
        if (b < s.n_seqs) v = seq_view(s, b);
        int end = v.n ? v.row0 + v.n : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end = max(end, u);
        }
        const int before = __shfl_up_sync(0xffffffffu, end, 1);
        f(b, v, v.ok && v.row0 >= (lane ? max(ends, before) : ends));
        ends = max(ends, __shfl_sync(0xffffffffu, end, 31));
    }
}

// Whole warp: the last sequence in use with rows whose key(b, row0) is at most x, or -1.
template <class F>
__device__ __noinline__ int seq_last(const PagedSeqs& s, int x, F key) {
    int last = -1;
    seq_scan(s, [&](int b, const SeqView& v, bool used) {
        const unsigned at = __ballot_sync(0xffffffffu, used && v.n && key(b, v.row0) <= x);
        if (at) last = (b & ~31) + 31 - __clz(at);
    });
    return last;
}

// Whole CTA (NT threads): do starts go back from sequence b0 on?
template <int NT>
__device__ __forceinline__ bool seq_back(const PagedSeqs& s, int b0) {
    bool back = false;
#pragma unroll 4
    for (int b = b0 + (int)threadIdx.x; b < s.n_seqs; b += NT) back |= __ldg(s.cu + b + 1) < __ldg(s.cu + b);
    return __syncthreads_or(back);
}

// Whole CTA (NT threads): how many sequences have key(b, cu[b]) at or before x, if starts
// do not go back (keys then do not either).  *next: the first one not looked at; *back:
// starts go back between those this thread looked at.
template <int NT, class K>
__device__ __forceinline__ int seq_count(const PagedSeqs& s, int x, K key, int* next, bool* back) {
    constexpr int kAhead = 4;   // loads of as many rounds under way: 20,000 sequences of a token 2558 -> 2208 us
    int started = 0, b0 = 0;
    *back = false;
    while (b0 < s.n_seqs) {
        int row0[kAhead], end[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int b = b0 + i * NT + (int)threadIdx.x;
            if (b < s.n_seqs) row0[i] = __ldg(s.cu + b), end[i] = __ldg(s.cu + b + 1);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int b = b0 + (int)threadIdx.x;
            bool at = false;
            if (b < s.n_seqs) {
                at = key(b, row0[i]) <= x;
                *back |= end[i] < row0[i];
            }
            const int n = __syncthreads_count(at);
            started += n;
            b0 += NT;
            if (n < NT) {
                *next = b0;
                return started;
            }
        }
    }
    *next = b0;
    return started;
}

__device__ __forceinline__ void report_bad(unsigned* status) {
    if (status) atomicOr(status, TVB_DEV_BAD_INPUT);
}

// Host checks and conversion of the descriptors (paged.cu).
tvb_status paged_cache_arg(const char* who, const tvb_kv_pages* kv, int n_kv_heads, int head_dim, PagedKV* out);
tvb_status paged_batch_arg(const char* who, const tvb_paged_batch* b, const tvb_kv_pages* kv, PagedSeqs* out);

// A workspace of this call on `st`, from a pool of the library that keeps some of
// its memory between calls (the driver orders reuse across streams; inside a
// capture it becomes the graph's own).  Freed on `st` when it goes out of scope,
// after the kernels launched until then.
class Workspace {
  public:
    explicit Workspace(cudaStream_t st) : st_(st) {}
    ~Workspace() {
        if (p_) cudaFreeAsync(p_, st_);
    }
    Workspace(const Workspace&) = delete;
    Workspace& operator=(const Workspace&) = delete;
    tvb_status get(size_t bytes);
    template <class T>
    T* at(size_t offset = 0) const {
        return reinterpret_cast<T*>(static_cast<unsigned char*>(p_) + offset);
    }

  private:
    cudaStream_t st_;
    void* p_ = nullptr;
};

// Raises a kernel's dynamic shared memory limit once per device.
constexpr int kMaxDevices = 64;
tvb_status allow_smem(const void* kernel, int bytes, int (&set)[kMaxDevices]);

}  // namespace tvb
