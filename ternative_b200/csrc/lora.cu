// Adapters of many requests beside a shared projection (tvb_matmul_lora):
//   y[m] = W x[m] + scale_a B_a (A_a x[m]),  a = adapter[m]
#include <algorithm>

#include "paged.cuh"

namespace tvb {

constexpr int kLoraMaxRank = 256;

struct LoraArgs {
    const float* x;
    float* y;
    float* t;   // [M][max_rank]: scale_a A_a x
    int M, K, N, n, max_rank, f16;
    const void* const* A;
    const void* const* B;
    const int* rank;
    const float* scale;
    const int* adapter;
    unsigned* status;
};

// The adapter of row m, or -1 where it has none (or none that can be used).
__device__ __forceinline__ int lora_of(const LoraArgs& a, int m, int* rank) {
    const int i = __ldg(a.adapter + m);
    *rank = 0;
    if (i == -1) return -1;
    if ((unsigned)i >= (unsigned)a.n) {
        report_bad(a.status);
        return -1;
    }
    const int r = __ldg(a.rank + i);
    if (r < 0 || r > a.max_rank) {
        report_bad(a.status);
        return -1;
    }
    *rank = r;
    return i;
}

__device__ __forceinline__ float lora_elem(const void* p, size_t i, bool f16) {
    return f16 ? __half2float(static_cast<const __half*>(p)[i]) : static_cast<const float*>(p)[i];
}

// Warp per (row, rank index).
__global__ void __launch_bounds__(256) lora_shrink_kernel(const __grid_constant__ LoraArgs a) {
    const int m = blockIdx.x, lane = threadIdx.x & 31;
    int rank;
    const int ad = lora_of(a, m, &rank);
    const float* x = a.x + (size_t)m * a.K;
    for (int j = blockIdx.y * 8 + (threadIdx.x >> 5); j < rank; j += gridDim.y * 8) {
        const void* A = a.A[ad];
        float s = 0.f;
        for (int k = lane; k < a.K; k += 32) s = fmaf(x[k], lora_elem(A, (size_t)j * a.K + k, a.f16), s);
        s = warp_sum(s);
        if (lane == 0) a.t[(size_t)m * a.max_rank + j] = s * __ldg(a.scale + ad);
    }
}

// Thread per (row, output).
__global__ void __launch_bounds__(256) lora_expand_kernel(const __grid_constant__ LoraArgs a) {
    const int m = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
    int rank;
    const int ad = lora_of(a, m, &rank);
    if (ad < 0 || n >= a.N) return;
    const void* B = a.B[ad];
    float s = 0.f;
    for (int j = 0; j < rank; ++j) s = fmaf(a.t[(size_t)m * a.max_rank + j], lora_elem(B, (size_t)n * rank + j, a.f16), s);
    a.y[(size_t)m * a.N + n] += s;
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
    TVB_TRY(tvb_matmul(y, x, M, K, w, N, stream));
    if (!table->n || !table->max_rank) return TVB_OK;
    const cudaStream_t st = as_stream(stream);
    LoraArgs a = {};
    a.x = x;
    a.y = y;
    a.M = M;
    a.K = K;
    a.N = N;
    a.n = table->n;
    a.max_rank = table->max_rank;
    a.f16 = table->dtype == TVB_F16;
    a.A = table->A;
    a.B = table->B;
    a.rank = table->rank;
    a.scale = table->scale;
    a.adapter = adapter;
    a.status = status;
    Workspace ws(st);
    TVB_TRY(ws.get((size_t)M * a.max_rank * 4));
    a.t = ws.at<float>();
    lora_shrink_kernel<<<dim3((unsigned)M, (unsigned)((a.max_rank + 7) / 8)), 256, 0, st>>>(a);
    TVB_TRY(check_launch("lora_shrink_kernel"));
    lora_expand_kernel<<<dim3((unsigned)((N + 255) / 256), (unsigned)M), 256, 0, st>>>(a);
    return check_launch("lora_expand_kernel");
}
