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

}  // namespace tvb
