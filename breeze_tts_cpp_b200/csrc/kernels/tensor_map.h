// The driver's tensor-map encoder, resolved once per process. Maps are filled on the host, without a driver round trip.
#pragma once
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <stdexcept>
#include <string>

namespace tts {
inline PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *entry = nullptr;
        cudaDriverEntryPointQueryResult result{};
        const cudaError_t status = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &result);
        if (status != cudaSuccess)
            throw std::runtime_error(std::string("cudaGetDriverEntryPoint(cuTensorMapEncodeTiled): ") + cudaGetErrorString(status));
        if (!entry || result != cudaDriverEntryPointSuccess)
            throw std::runtime_error("cuTensorMapEncodeTiled is unavailable in this driver");
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(entry);
    }();
    return fn;
}
} // namespace tts
