// What the kernels over a paged key/value cache share: the checked view of a catena_paged_cache_t, the lookup of a row, the
// error word, programmatic launches.  Internal — the public surface is include/catena_b200.h.
//
// A page id or a length is DATA on the device, so the host cannot check it: every kernel bounds-checks both, skips what is out of
// range and sets the thread's error word, which becomes CATENA_E_ASSERT (in blocking mode at the end of the call, otherwise at the
// next catena_b200_check_device_errors).  No table can make a kernel read or write outside the pools.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace catena {
namespace paged {

constexpr uint32_t kNoRow = 0xFFFFFFFFu;
constexpr uint32_t kErrTable = 1u, kErrLength = 2u, kErrPosition = 4u, kErrParent = 8u;

struct View {
    __nv_bfloat16* k;
    __nv_bfloat16* v;
    const int32_t* table;
    const int32_t* lengths;
    uint32_t n_pages, page_size, n_seqs, max_pages, hkv;
    uint32_t* err;

    __host__ __device__ uint32_t cap() const { return max_pages * page_size; }
#ifdef __CUDACC__
    // rows of sequence b; a length outside 0 .. cap counts as none
    __device__ __forceinline__ uint32_t length(uint32_t b) const {
        const int32_t n = lengths[b];
        if (n >= 0 && (uint32_t)n <= cap()) return (uint32_t)n;
        atomicOr(err, kErrLength);
        return 0u;
    }
    // index of row r of (sequence b, head h) among all rows of a pool (fewer than 2^32: checked on the host); kNoRow when the page
    // is none of the pool's
    __device__ __forceinline__ uint32_t row(const int32_t* tab, uint32_t pitch, uint32_t b, uint32_t h, uint32_t r) const {
        const uint32_t j = r / page_size;
        const uint32_t page = (uint32_t)tab[(size_t)b * pitch + j];
        if (page < n_pages) return (page * hkv + h) * page_size + (r - j * page_size);
        atomicOr(err, kErrTable);
        return kNoRow;
    }
    __device__ __forceinline__ uint32_t row(uint32_t b, uint32_t h, uint32_t r) const { return row(table, max_pages, b, h, r); }
#endif
};

// checks everything the host can see and fills `view`
catena_status_t check_cache(const catena_paged_cache_t* cache, const char* what, View* view);
// start of a call: binds the device, refuses a capture that the call could not survive, hands out the thread's error word
catena_status_t begin(uint32_t** err);
// end of a call: in blocking mode waits and reports what the kernels found
catena_status_t end();

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

#ifdef __CUDACC__
// Programmatic dependent launch, as in the Llama block: the next launch may begin at once, and a kernel touches memory only
// after everything launched before it has finished.
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Lets a kernel have `bytes` of dynamic shared memory; `done` belongs to the kernel (a bit per device that has been told).
template <class F>
static catena_status_t allow_smem(F kernel, size_t bytes, uint32_t* done) {
    const uint32_t bit = 1u << tls().device;
    if (*done & bit) return CATENA_OK;
    CATENA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    *done |= bit;
    return CATENA_OK;
}

struct How {
    uint32_t cluster = 1;
    bool early = true;      // may start while the launch before it still runs
};
template <class... KArgs, class... Args>
static catena_status_t launch_as(How how, const char* what, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = tls().stream;
    cudaLaunchAttribute at[2];
    cfg.attrs = at;
    if (how.early) {
        at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (how.cluster > 1) {
        at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        at[cfg.numAttrs].val.clusterDim.x = how.cluster;
        at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
    if (e != cudaSuccess) return fail_cuda(e, what);
    count_launch();
    return CATENA_OK;
}
template <class... KArgs, class... Args>
static catena_status_t launch(const char* what, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, Args... args) {
    return launch_as(How(), what, kernel, grid, block, smem, args...);
}
#endif

}  // namespace paged
}  // namespace catena
