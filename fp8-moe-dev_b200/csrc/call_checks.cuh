// Checks and launches of the entry points that work without a handle (host code).
#pragma once
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/moe_fp8_b200.h"

namespace moe {

// The error text goes to the caller's buffer, if there is one.
inline int refuse(char* err, size_t err_len, int code, const char* fmt, ...)
{
    if (err && err_len) {
        va_list ap;
        va_start(ap, fmt);
        std::vsnprintf(err, err_len, fmt, ap);
        va_end(ap);
    }
    return code;
}

// Device memory of `dev`, or managed memory.  The kernels run on the current device and read no other one's memory
// through whatever peer mapping may exist.
inline bool memory_of_device(const void* p, int dev)
{
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) { cudaGetLastError(); return false; }
    if (at.type == cudaMemoryTypeManaged) return true;
    return at.type == cudaMemoryTypeDevice && at.device == dev;
}

// A strided matrix of a call, in bytes.
struct Extent {
    const char* name;
    const void* base;
    int64_t rows, row_bytes, stride_bytes;
    uintptr_t begin() const { return reinterpret_cast<uintptr_t>(base); }
    uintptr_t end() const { return begin() + (uintptr_t)((rows - 1) * stride_bytes + row_bytes); }
};

// Whether two matrices share a byte.  Column ranges of one wider matrix do not.
inline bool share_memory(const Extent& a, const Extent& b)
{
    if (!a.base || !b.base || a.rows <= 0 || b.rows <= 0 || a.row_bytes <= 0 || b.row_bytes <= 0) return false;
    if (a.begin() >= b.end() || b.begin() >= a.end()) return false;
    if (a.stride_bytes != b.stride_bytes || a.stride_bytes <= 0) return true;
    const uintptr_t s = (uintptr_t)a.stride_bytes;
    const uintptr_t d = b.begin() >= a.begin() ? (b.begin() - a.begin()) % s : (s - (a.begin() - b.begin()) % s) % s;
    return d < (uintptr_t)a.row_bytes || s - d < (uintptr_t)b.row_bytes;
}

// One launch with the programmatic-stream-serialization attribute (the kernel waits for its predecessor itself, see
// ptx.cuh), as one cluster of `cluster` CTAs per grid line if that is above 1.
template <typename... KArgs, typename... Args>
cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, unsigned cluster, cudaStream_t stream,
                         Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace moe
