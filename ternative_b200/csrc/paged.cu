// Host side of the paged operators: argument checks and workspaces.
#include "paged.cuh"

#include <mutex>

namespace tvb {

tvb_status paged_cache_arg(const char* who, const tvb_kv_pages* kv, int n_kv_heads, int head_dim, PagedKV* out) {
    TVB_REQUIRE(kv && kv->k && kv->v, "%s: null cache pointer", who);
    TVB_REQUIRE(kv->dtype == TVB_F32 || kv->dtype == TVB_F16, "%s: cache dtype %d (F32 or F16)", who, (int)kv->dtype);
    TVB_REQUIRE(kv->n_pages > 0 && kv->page_size > 0, "%s: %d pages of %d tokens", who, kv->n_pages, kv->page_size);
    const int64_t size = kv->dtype == TVB_F32 ? 4 : 2;
    TVB_REQUIRE(kv->page_stride > 0 && kv->row_stride >= head_dim && kv->head_stride >= (n_kv_heads > 1 ? head_dim : 0),
                "%s: cache strides (page %lld, row %lld, head %lld)", who, (long long)kv->page_stride,
                (long long)kv->row_stride, (long long)kv->head_stride);
    TVB_REQUIRE(((kv->page_stride * size) | (kv->row_stride * size) | (kv->head_stride * size)) % 16 == 0 &&
                    ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v)) & 15) == 0,
                "%s: cache addresses and strides must be multiples of 16 bytes", who);
    out->k = static_cast<unsigned char*>(kv->k);
    out->v = static_cast<unsigned char*>(kv->v);
    out->page_stride = kv->page_stride * size;
    out->row_stride = kv->row_stride * size;
    out->head_stride = kv->head_stride * size;
    out->n_pages = kv->n_pages;
    out->page = FastDiv((uint32_t)kv->page_size);
    return TVB_OK;
}

tvb_status paged_batch_arg(const char* who, const tvb_paged_batch* b, const tvb_kv_pages* kv, PagedSeqs* out) {
    TVB_REQUIRE(b && kv, "%s: null descriptor", who);
    TVB_REQUIRE(b->n_seqs >= 0 && b->n_tokens >= 0, "%s: %d sequences, %d tokens", who, b->n_seqs, b->n_tokens);
    TVB_REQUIRE(b->n_seqs == 0 || (b->cu_tokens && b->kv_len && b->block_table), "%s: null batch pointer", who);
    TVB_REQUIRE(b->n_seqs <= 65535, "%s: %d sequences (at most 65535)", who, b->n_seqs);
    TVB_REQUIRE(b->max_new >= 0 && b->max_kv >= 0, "%s: max_new %d, max_kv %d", who, b->max_new, b->max_kv);
    // a kernel's last step ends behind the longest sequence: positions stay in 32 bits
    TVB_REQUIRE(b->max_kv <= 1 << 30, "%s: max_kv %d (at most 2^30)", who, b->max_kv);
    TVB_REQUIRE(b->n_seqs == 0 || (int64_t)b->table_ld * kv->page_size >= b->max_kv,
                "%s: block_table rows of %d pages of %d tokens do not hold max_kv %d", who, b->table_ld, kv->page_size,
                b->max_kv);
    out->cu = b->cu_tokens;
    out->kv_len = b->kv_len;
    out->table = b->block_table;
    out->n_seqs = b->n_seqs;
    out->n_tokens = b->n_tokens;
    out->max_new = b->max_new;
    out->max_kv = b->max_kv;
    out->table_ld = b->table_ld;
    return TVB_OK;
}

// One-time set-up may come while the caller captures a stream, where it would end
// the capture; it touches no stream.
struct OutsideCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    OutsideCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~OutsideCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// What the pool keeps between calls: 1% of the device.  1400 rows of INT8 weights 4096 ->
// 14336 take 0.2 GB, 65,535 rows of 4096 1.1; what is held beyond it goes back to the
// device when the host next waits for it.
constexpr uint64_t kPoolKeep = 2ull << 30;

static std::mutex g_pool_mutex;
static cudaMemPool_t g_pools[kMaxDevices];

tvb_status Workspace::get(size_t bytes) {
    int dev = 0;
    TVB_CUDA(cudaGetDevice(&dev));
    TVB_REQUIRE(dev >= 0 && dev < kMaxDevices, "workspace: device %d", dev);
    {
        std::lock_guard<std::mutex> lock(g_pool_mutex);
        if (!g_pools[dev]) {
            OutsideCapture outside;
            cudaMemPoolProps props = {};
            props.allocType = cudaMemAllocationTypePinned;
            props.location.type = cudaMemLocationTypeDevice;
            props.location.id = dev;
            cudaMemPool_t pool;
            TVB_CUDA(cudaMemPoolCreate(&pool, &props));
            uint64_t keep = kPoolKeep;
            const cudaError_t e = cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep);
            if (e != cudaSuccess) {
                cudaMemPoolDestroy(pool);
                return cuda_error(e, "cudaMemPoolSetAttribute");
            }
            g_pools[dev] = pool;
        }
    }
    TVB_CUDA(cudaMallocFromPoolAsync(&p_, bytes, g_pools[dev], st_));
    return TVB_OK;
}

static std::mutex g_smem_mutex;

tvb_status allow_smem(const void* kernel, int bytes, int (&set)[kMaxDevices]) {
    int dev = 0;
    TVB_CUDA(cudaGetDevice(&dev));
    TVB_REQUIRE(dev >= 0 && dev < kMaxDevices, "device %d", dev);
    std::lock_guard<std::mutex> lock(g_smem_mutex);
    if (bytes > set[dev]) {
        OutsideCapture outside;
        TVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        set[dev] = bytes;
    }
    return TVB_OK;
}

}  // namespace tvb
