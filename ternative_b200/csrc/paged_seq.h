// The numbers of one sequence of a ragged batch, checked: plain C++, so that the
// check also runs on the host.
#pragma once

#ifdef __CUDACC__
#define TVB_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define TVB_HOST_DEVICE inline
#endif

namespace tvb {

// Rows [row0, row0 + n) of the token buffers at positions pos0 ... of a cache of
// kv tokens.
struct SeqView {
    int row0, n, kv, pos0;
    bool ok;     // else n and pos0 are 0
    bool back;   // it ends before it starts: starts that go back
};

// The arrays hold anything: every difference is taken after its operands were
// compared, so nothing wraps.
TVB_HOST_DEVICE SeqView seq_numbers(int row0, int end, int kv, int n_tokens, int max_new, int max_kv) {
    SeqView v;
    v.row0 = row0;
    v.kv = kv;
    v.ok = row0 >= 0 && end >= row0 && end <= n_tokens;
    v.n = v.ok ? end - row0 : 0;
    v.ok = v.ok && v.n <= max_new && kv >= v.n && kv <= max_kv;
    v.back = end < row0;
    if (!v.ok) v.n = 0;
    v.pos0 = v.ok ? kv - v.n : 0;
    return v;
}

}  // namespace tvb
