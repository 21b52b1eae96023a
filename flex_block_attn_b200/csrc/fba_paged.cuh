// What the kernels of the paged key / value cache share.
#pragma once
#include "fba_common.cuh"

namespace fba {

// Device view of fba_paged_t.
struct PagedDev {
    uint8_t *k, *v;              // [n_pages, Hkv, page_size, 128] bf16 or e4m3
    float *k_scale, *v_scale;    // [n_pages, Hkv, page_size]; null unless e4m3
    float* weight;               // likewise, or null
    int32_t* position;           // likewise, or null
    const int32_t* table;        // [B, max_pages]
    int n_pages, Hkv, page_size, page_shift, max_pages;
};

// First of the status words: what is reported there.
enum PagedReport : uint32_t { kBadPage = 2, kBadLength = 3 };
__device__ __forceinline__ void report_paged(uint32_t* status, uint32_t what, int b, int value) {
    if (atomicCAS(status + StatusWords::kFlag, 0u, what) == 0u) {
        status[StatusWords::kBx] = static_cast<uint32_t>(b);
        status[StatusWords::kTag] = static_cast<uint32_t>(value);
    }
}

// Length of sequence b, held to what its row of the table can address.
__device__ __forceinline__ int paged_length(const PagedDev& c, const int32_t* seq_lens, int b, uint32_t* status) {
    const int n = seq_lens[b], most = c.max_pages * c.page_size;   // host-checked to stay below 2^31
    if (n >= 0 && n <= most) return n;
    report_paged(status, kBadLength, b, n);
    return n < 0 ? 0 : most;
}

// Page that the table names for slot `slot` of sequence b, and the row of the pools that the slot of kv head h has in it, or
// -1 where there is no such page.  Apart, so that a thread may look up several pages at a time.
__device__ __forceinline__ int paged_page(const PagedDev& c, int b, int slot) {
    return c.table[static_cast<long long>(b) * c.max_pages + (slot >> c.page_shift)];
}
__device__ __forceinline__ long long paged_row_in(const PagedDev& c, int page, int h, int slot) {
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(c.n_pages)) return -1;
    return (static_cast<long long>(page) * c.Hkv + h) * c.page_size + (slot & (c.page_size - 1));
}
// Both, with a report.
__device__ __forceinline__ long long paged_row(const PagedDev& c, int b, int h, int slot, uint32_t* status) {
    const int page = paged_page(c, b, slot);
    const long long row = paged_row_in(c, page, h, slot);
    if (row < 0) report_paged(status, kBadPage, b, page);
    return row;
}

// Programmatic dependent launch: a kernel of this family may be set up while the one before it in the stream still runs.  Each
// waits for its predecessor's end (and with it, as the predecessor did the same, for all before) ahead of its first
// access to memory, in every thread (paged_finish_kernel but for what its predecessor reads as well).
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <class... Params, class... Args>
int launch_chained(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config, kernel, args...);
    return check_launch("launch of a paged-cache kernel");
}

// Whether two arrays of B lengths or positions share memory: what one CTA of a sequence writes, others may still have to read.
inline bool lens_overlap(const int32_t* x, const int32_t* y, int B) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
    const uintptr_t n = sizeof(int32_t) * static_cast<uintptr_t>(B);
    return x && y && a < b + n && b < a + n;
}

// Checks a cache and fills its device view (fba_paged.cu).
int paged_args(const char* who, const fba_paged_t* cache, int B, PagedDev* dev);

}  // namespace fba
