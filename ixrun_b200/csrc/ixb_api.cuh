// What the translation units of the library share on the host side: the calling thread's error text, the launch counter, the
// dependent-launch switch and the lookups that are made once per device.  Defined in ixb200.cu.
#pragma once
#include "../../include/ixb200.h"
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

namespace ixb {

int fail(int code, const char *fmt, ...);              // sets ixb_last_error() of this thread; returns code
int launch_check(const char *what);                    // counts a launch and reports what it left behind
int num_sms();                                         // of the current device
bool pdl_on();                                         // ixb_set_pdl
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();            // a function of the driver; null if there is none

#define IXB_CUDA(call)                                                                        \
    do {                                                                                      \
        cudaError_t e_ = (call);                                                              \
        if (e_ != cudaSuccess)                                                                \
            return fail(IXB_E_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_));          \
    } while (0)
#define IXB_GLUE(what, call)                                                                    \
    do {                                                                                      \
        cudaError_t e_ = (call);                                                              \
        if (e_ != cudaSuccess) return fail(IXB_E_CUDA, "%s launch: %s", what, cudaGetErrorString(e_)); \
        return launch_check(what);                                                            \
    } while (0)

// opt-in to more than 48 KB of dynamic shared memory, once per kernel instantiation and device
template <class K>
static cudaError_t opt_in_smem(K kernel, bool (&done)[64], int bytes)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!done[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return e;
        done[dev] = true;
    }
    return cudaSuccess;
}

// one launch, with the programmatic-stream-serialization attribute if `overlap`
template <class... KArgs, class... Args>
static cudaError_t launch_overlapped(bool overlap, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
// the same when ixb_set_pdl is on
template <class... KArgs, class... Args>
static cudaError_t launch_glue_smem(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args)
{
    return launch_overlapped(pdl_on(), kernel, grid, block, smem, st, args...);
}

}  // namespace ixb
