// The driver's encoder of tensor maps, looked up once.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

namespace zb {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// nullptr where the driver has none.
inline EncodeTiled encode_tiled() {
    static std::atomic<EncodeTiled> known{nullptr};
    EncodeTiled encode = known.load(std::memory_order_acquire);
    if (encode) return encode;
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn) { cudaGetLastError(); return nullptr; }
    encode = reinterpret_cast<EncodeTiled>(fn);
    known.store(encode, std::memory_order_release);
    return encode;
}

}  // namespace zb
