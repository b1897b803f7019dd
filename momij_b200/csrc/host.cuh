// host.cuh -- host-side helpers that api.cu shares with the entry points of the
// attention half and the output head (kvcache.cu, attn.cu, qmm4.cu, logits.cu).
#pragma once

#include <utility>

#include "common.cuh"
#include "grant.cuh"

namespace momij {

int host_check_device();             // MOMIJ_OK or MOMIJ_ERR_NO_DEVICE
int host_sm_count();                 // of the current device, <= 0 on failure
bool host_pdl();                     // programmatic dependent launch enabled
const int32_t* host_stop_flag();     // momij_set_stop_flag's pointer
int host_stop_step();                // momij_set_stop_step's words
int host_spin_limit();               // momij_set_spin_limit's bound
void* host_tensor_map_encoder();     // cuTensorMapEncodeTiled, or NULL

inline bool host_aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline int host_cuda_status(cudaError_t e) {
    if (e == cudaSuccess) return MOMIJ_OK;
    cudaGetLastError();  // a refused launch leaves no error behind for the next call
    return MOMIJ_ERR_CUDA;
}

// Dynamic shared memory above 48 KB needs the kernel's consent, once per
// device and kernel; the attribute call is skipped when `granted` (one slot
// per device, owned by the caller) already covers the size.
template <typename K>
inline bool host_allow_smem(K kern, size_t smem, int (&granted)[64]) {
    if (smem <= 48 * 1024) return true;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    return grant_at_least(granted[dev], (int)smem, [&](int size) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, size) == cudaSuccess) return true;
        cudaGetLastError();
        return false;
    });
}

// Launch with programmatic dependent launch: the kernel starts while the
// previous one drains and waits for it (pdl_wait) before its first read.
template <typename... KArgs, typename... Args>
inline int host_launch(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, momij_stream_t st, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(st);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = host_pdl() ? 1 : 0;
    return host_cuda_status(cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...));
}

}  // namespace momij
