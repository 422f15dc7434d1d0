#pragma once
/* What the C ABI's entry points share (paged_host.cu, branch_host.cu): C++
 * failures as status codes, the handle's device, and workspaces. */
#include <initializer_list>
#include <mutex>
#include <new>
#include <stdexcept>
#include <string>

#include <cuda_runtime.h>

#include "../../include/nutllm_cuda.h"
#include "kernels.h"
#include "paged.h"

namespace nut {
namespace abi {

struct Failure {
    nut_status status;
    std::string message;
};

inline void cuda_check(cudaError_t e, const char *what) {
    if (e != cudaSuccess) {
        cudaGetLastError(); /* reported here: the next call's own check is not to find it */
        throw Failure{NUT_RUNTIME_ERROR,
                      std::string("cuda: ") + what + ": " + cudaGetErrorString(e)};
    }
}

template <typename F> nut_status guarded(F &&body) {
    try {
        body();
        return NUT_OK;
    } catch (const Failure &f) {
        set_last_error(f.message);
        return f.status;
    } catch (const std::bad_alloc &) {
        set_last_error("nutllm: host allocation failed");
        return NUT_RUNTIME_ERROR;
    } catch (const std::exception &e) {
        set_last_error(e.what());
        return NUT_RUNTIME_ERROR;
    }
}

/* Makes the handle's device current where it is not, and restores it. */
struct DeviceScope {
    int previous = 0, device;
    explicit DeviceScope(int d) : device(d) {
        cuda_check(cudaGetDevice(&previous), "get device");
        if (previous != device)
            cuda_check(cudaSetDevice(device), "set device");
    }
    ~DeviceScope() {
        if (previous != device)
            cudaSetDevice(previous);
    }
};

/* Workspaces come from a memory pool of this library's own on each device,
 * which keeps up to 64 MB that handles gave back: a handle is made in some 20
 * us, where cudaMalloc and cudaFree take 300 to 400 each. */
inline cudaMemPool_t workspace_pool(int device) {
    static std::mutex lock;
    static cudaMemPool_t pools[kMaxDevices] = {};
    if (device < 0 || device >= kMaxDevices)
        throw Failure{NUT_INVALID_ARGUMENT, "paged: device out of range"};
    const std::lock_guard<std::mutex> hold(lock);
    if (!pools[device]) {
        cudaMemPoolProps props{};
        props.allocType = cudaMemAllocationTypePinned;
        props.location.type = cudaMemLocationTypeDevice;
        props.location.id = device;
        cuda_check(cudaMemPoolCreate(&pools[device], &props), "create workspace pool");
        uint64_t keep = uint64_t(64) << 20;
        cuda_check(cudaMemPoolSetAttribute(pools[device], cudaMemPoolAttrReleaseThreshold, &keep),
                   "size workspace pool");
    }
    return pools[device];
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

/* Arrays of 32-bit words; NULL is aligned. */
inline bool aligned4(std::initializer_list<const void *> arrays) {
    for (const void *p : arrays)
        if (reinterpret_cast<uintptr_t>(p) & 3)
            return false;
    return true;
}

} // namespace abi
} // namespace nut
