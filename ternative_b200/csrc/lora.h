// A projection with an adapter for each row: shared by its kernels (lora.cu, few
// rows; lora_gemm.cu, many).
#pragma once

#include "paged.cuh"

namespace tvb {

constexpr int kLoraMaxRank = 256;
constexpr int kLoraMaxK = 16384;   // of the many-rows kernels

struct LoraArgs {
    const float* x;
    float* y;
    int M, K, N;
    const void* w;
    const float* row_scales;   // INT8 rows, else null
    float tscale;              // INT8 tensor, else 1
    int w8;                    // INT8 weights
    // adapters
    int n, max_rank, f16;
    const void* const* A;
    const void* const* B;
    const int* rank;
    const float* scale;
    const int* adapter;
    float* t;                  // [M][max_rank]: scale_a A_a x[m]
    unsigned* status;
};

// The adapter of row m, or -1 where it has none (or none that can be used).
__device__ __forceinline__ int lora_of(const LoraArgs& a, int m, int* rank, bool report) {
    *rank = 0;
    if (!a.n) return -1;
    const int i = __ldg(a.adapter + m);
    if (i == -1) return -1;
    int r = -1;
    if ((unsigned)i < (unsigned)a.n &&
        ((reinterpret_cast<uintptr_t>(a.A[i]) | reinterpret_cast<uintptr_t>(a.B[i])) & 15) == 0)
        r = __ldg(a.rank + i);
    if (r < 0 || r > a.max_rank) {
        if (report) report_bad(a.status);
        return -1;
    }
    *rank = r;
    return i;
}

__device__ __forceinline__ float lora_elem(const void* p, size_t i, bool f16) {
    return f16 ? __half2float(static_cast<const __half*>(p)[i]) : static_cast<const float*>(p)[i];
}

tvb_status lora_many_rows(LoraArgs a, cudaStream_t st);             // lora_gemm.cu
tvb_status lora_shrink_rows(const LoraArgs& a, cudaStream_t st);   // lora.cu

}  // namespace tvb
