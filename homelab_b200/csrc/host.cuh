// host.cuh - host side shared by the translation units of liboomb.so: per-device
// state, kernel launches with programmatic stream serialization, and the driver's
// tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>
#include <unordered_map>

#include "../../include/oomb.h"

namespace oomb {

constexpr int kMaxDevices = 64;

struct DeviceState {
    bool init = false;
    bool ok = false;
    int sms = 0;
    unsigned* err = nullptr;
};

// The current device's state, or null when it is not an sm_100 device (capi.cu).
const DeviceState* device_state();

// Sets the wait limit of the kernels in paged.cu (each translation unit's kernels
// read their own copy of the limit).
cudaError_t paged_set_wait_limit(unsigned long long ns);

// Opts a kernel into more than 48 KB of dynamic shared memory, once per
// (kernel, device): calls made later (for instance during CUDA graph capture)
// find it done and touch nothing but the stream.
inline std::mutex g_attr_mu;
inline std::unordered_map<const void*, size_t> g_attr_done[kMaxDevices];

template <typename Kernel>
bool set_smem(Kernel k, size_t bytes) {
    // the default limit covers static and dynamic shared memory together
    if (bytes <= 40 * 1024) return true;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
    const void* key = reinterpret_cast<const void*>(k);
    std::lock_guard<std::mutex> lk(g_attr_mu);
    auto it = g_attr_done[dev].find(key);
    if (it != g_attr_done[dev].end() && it->second >= bytes) return true;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) !=
        cudaSuccess)
        return false;
    g_attr_done[dev][key] = bytes;
    return true;
}

template <typename Kernel, typename... Args>
int launch(Kernel kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
    if (!set_smem(kernel, smem)) return OOMB_E_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? OOMB_OK : OOMB_E_LAUNCH;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Where a caller's buffer lives.  Pinned host memory (cudaHostAlloc,
// cudaHostRegister) is reachable from kernels at its mapped device address;
// pageable host memory and unknown pointers are reachable by no kernel.
enum class Mem { none, device, host };
inline Mem mem_kind(const void* p, const void** dev) {
    cudaPointerAttributes a{};
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        (void)cudaGetLastError();
        return Mem::none;
    }
    if (a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged) {
        *dev = p;
        return Mem::device;
    }
    if (a.type == cudaMemoryTypeHost && a.devicePointer) {
        *dev = a.devicePointer;
        return Mem::host;
    }
    return Mem::none;
}

// cuTensorMapEncodeTiled, fetched once from the driver through the runtime (the
// library links only the CUDA runtime).
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return static_cast<EncodeTiledFn>(nullptr);
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    return fn;
}

inline size_t align256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

}  // namespace oomb
