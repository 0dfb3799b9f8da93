// What the serving operators' entry points (serving.cu) hand to their kernels.  Every pointer is device memory.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/ava_engine.h"

namespace ava {

template <typename... KArgs, typename... Args>
inline cudaError_t launch_as(void (*kernel)(KArgs...), const cudaLaunchConfig_t& cfg, Args&&... args) {
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// One launch with programmatic dependent launch (the kernels start with pdl_enter, kernels.cuh).  Unlike launch_k it
// shares nothing between threads but a word per kernel that says on which devices its shared memory has been asked for:
// these operators may be called from several threads at once.
template <auto Kernel, typename... Args>
inline cudaError_t launch_serving(int device, dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, Args&&... args) {
    static std::atomic<uint64_t> asked{0};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const uint64_t bit = 1ull << (device & 63);
    if (smem > 48 * 1024 && (device > 63 || !(asked.load(std::memory_order_relaxed) & bit))) {
        const cudaError_t rc = cudaFuncSetAttribute(reinterpret_cast<const void*>(Kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (rc != cudaSuccess) return rc;
        asked.fetch_or(bit, std::memory_order_relaxed);
    }
    return launch_as(Kernel, cfg, static_cast<Args&&>(args)...);
}

// ---- the step's lists (k_paged.cu)
struct PlanArgs {
    const int32_t *cached, *fresh, *owned, *free_count;
    int32_t *table, *owned_out, *free_list, *free_count_out, *q_start;
    int64_t* slot;
    int32_t *pos, *row;
    uint32_t* status;
    int rows, page_size, n_pages, max_pages, max_tokens, trim;
};
cudaError_t launch_paged_plan(int device, cudaStream_t st, const PlanArgs& a);

// ---- new keys and values into their pages (k_paged.cu)
struct AppendArgs {
    ava_paged_store s;
    const void *k, *v;
    int64_t token_stride, head_stride;
    const int64_t* slot;
    uint32_t* status;
    int tokens, bf16_in;
};
cudaError_t launch_paged_append(int device, cudaStream_t st, const AppendArgs& a);

// ---- the read (k_pread.cu)
struct ReadArgs {
    ava_paged_store s;
    const void* q;
    void* out;
    float* lse;
    int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
    const int32_t *table, *cached, *first, *q_start;
    uint32_t* status;
    float scale;
    int heads, group, max_pages, rows, max_tokens, max_fresh, window, bf16_q;
};
// room: paged_read_workspace bytes
cudaError_t launch_paged_read(int device, cudaStream_t st, const ReadArgs& a, void* room, int sms);
int64_t paged_read_workspace(int head_size, int sms);
// the same on tcgen05 (k_pread_tc.cu); *taken false: not its case, nothing was queued
cudaError_t launch_paged_read_tc(int device, cudaStream_t st, const ReadArgs& a, void* room, int sms, bool* taken);

// ---- drafted tokens (k_verify.cu)
struct VerifyArgs {
    const float *p, *q;
    int64_t p_stride, q_stride;
    const uint32_t* tok;
    const int32_t* q_start;
    const double* uniform;
    uint32_t* out;
    int32_t* n_out;
    uint32_t* status;
    int rows, max_tokens, vocab, max_out;
};
cudaError_t launch_verify(int device, cudaStream_t st, const VerifyArgs& a);

}  // namespace ava
