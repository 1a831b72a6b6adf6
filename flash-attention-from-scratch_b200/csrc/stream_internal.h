#pragma once
// Host/device shared definitions of the streaming-attention kernels: the paged cache
// (cache_append_sm100.cu, cache_attn_sm100.cu, tree_attn_sm100.cu, pages_sm100.cu), rotation (rotary_sm100.cu) and window attention (window_bwd_sm100.cu and the
// window build of flash_fwd_sm100.cu).

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/fa_b200.h"
#include "fa_internal.h"

namespace fa_sm100 {

// DeviceStatus::code bit: a position outside the page table or a page outside the pool was
// skipped (the kernels' own bounds check on data the host does not see).
constexpr unsigned kStatusBadPage = 1u << 5;

// A window that hides nothing (lengths are at most 2^30).
constexpr int kNoWindow = 1 << 30;

// The last key position a row at `pos` sees is pos; the first one of its window is this.
__host__ __device__ __forceinline__ int window_first(int pos, int window) {
    return (window > 0 && pos >= window) ? pos - window + 1 : 0;
}

cudaError_t launch_append(const FaAppendParams& p, DeviceStatus* status, cudaStream_t stream);

unsigned long long cached_workspace_bytes(const FaCachedParams& p, int sm_count);
cudaError_t launch_cached(const FaCachedParams& p, DeviceStatus* status, void* workspace, int sm_count,
                          cudaStream_t stream);

// Trees of at most 32 nodes in the cached attention's kernel, 16 query rows at a time (cache_attn_sm100.cu).
unsigned long long small_tree_workspace_bytes(const FaTreeParams& p, int sm_count);
cudaError_t launch_small_tree(const FaTreeParams& p, DeviceStatus* status, void* workspace, int sm_count, cudaStream_t stream);
unsigned long long tree_workspace_bytes(const FaTreeParams& p, int sm_count);
cudaError_t launch_tree(const FaTreeParams& p, DeviceStatus* status, void* workspace, int sm_count,
                        cudaStream_t stream);

cudaError_t launch_rotary(const FaRotaryParams& p, DeviceStatus* status, int sm_count, cudaStream_t stream);

cudaError_t launch_keep_tokens(const FaKeepParams& p, DeviceStatus* status, cudaStream_t stream);
cudaError_t launch_copy_pages(const FaCopyParams& p, DeviceStatus* status, cudaStream_t stream);
cudaError_t launch_fork_pages(const FaPages& p, DeviceStatus* status, cudaStream_t stream);
cudaError_t launch_free_pages(const FaPages& p, DeviceStatus* status, cudaStream_t stream);
unsigned long long reserve_workspace_bytes(const FaPages& p);
cudaError_t launch_reserve_pages(const FaPages& p, DeviceStatus* status, void* workspace, cudaStream_t stream);

cudaError_t launch_window_fwd(const FaWindowParams& p, DeviceStatus* status, unsigned epoch, int sm_count,
                              cudaStream_t stream);

unsigned long long window_bwd_workspace_bytes(const FaWindowParams& p, int sm_count);
cudaError_t launch_window_bwd(const FaWindowParams& p, DeviceStatus* status, unsigned epoch, void* workspace,
                              int sm_count, cudaStream_t stream);

}  // namespace fa_sm100
