// What the backend's translation units share on the host: the error message behind
// mt_last_error, the per-device stream, and checks of the arrays that callers describe.
#ifndef METELLUS_MT_HOST_H
#define METELLUS_MT_HOST_H

#include <cuda_runtime.h>

#include "../../include/metellus_b200.h"

namespace mt {

// Record the calling thread's error message; fail returns 1 (the call failed), bad_argument
// 2 (nothing was done: an argument does not fit).
int fail(const char* fmt, ...);
int bad_argument(const char* fmt, ...);

// The stream a call runs on: the caller's, or (NULL) the library's own stream of `dev`,
// initialising the device at first use.
int call_stream(int dev, void* stream, cudaStream_t* out);
// Number of SMs of `dev` (looked up once per device).
int sm_count(int dev, int* out);

#define RT_CHECK(call)                                                               \
    do {                                                                             \
        cudaError_t e_ = (call);                                                     \
        if (e_ != cudaSuccess)                                                       \
            return mt::fail("%s failed: %s (%s:%d)", #call, cudaGetErrorString(e_),  \
                            __FILE__, __LINE__);                                     \
    } while (0)

// Launches a kernel that begins with `griddepcontrol.wait`: its blocks may be set up while the
// kernel before it on the stream ends, if that one is of this library too (which allow it early,
// by `griddepcontrol.launch_dependents`); the wait is for all of that kernel's memory.
// launch_clusters: in clusters of `cluster` blocks along x.
template <class... P, class... A>
cudaError_t launch_clusters(unsigned cluster, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                            A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}
template <class... P, class... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
    return launch_clusters(1, kernel, grid, block, smem, st, args...);
}

// Makes `dev` current for a call and gives the caller its own device back.
struct OnDevice {
    int caller = -1;
    cudaError_t enter(int dev) {
        int now = -1;
        cudaError_t e = cudaGetDevice(&now);
        if (e != cudaSuccess || now == dev) return e;
        caller = now;
        return cudaSetDevice(dev);
    }
    ~OnDevice() {
        if (caller >= 0) cudaSetDevice(caller);
    }
};

}  // namespace mt

#endif
