// Host-side launch helpers of the 8-bit floating-point kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "kernels.h"

namespace wq {

constexpr int kMaxDevices = 64;

// A kernel launch allowed to start while the previous kernel on the stream
// drains (the kernels wait with griddepcontrol.wait before they read memory).
struct LaunchConfig {
    cudaLaunchConfig_t c = {};
    cudaLaunchAttribute attr[1];
    LaunchConfig(dim3 grid, unsigned threads, size_t smem, cudaStream_t s) {
        c.gridDim = grid;
        c.blockDim = dim3(threads);
        c.dynamicSmemBytes = smem;
        c.stream = s;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        c.attrs = attr;
        c.numAttrs = 1;
    }
    LaunchConfig(const LaunchConfig&) = delete;
};

// Once per device and kernel: the shared-memory opt-in, and for kernels that
// split registers between warpgroups (`regs` > 0) the check that a launch
// gives every thread exactly `regs` (an increase would wait for registers that
// are not there).
inline cudaError_t prepare_kernel(const void* kern, size_t smem, int regs, std::atomic<int> (&ready)[kMaxDevices]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool known = dev >= 0 && dev < kMaxDevices;
    if (known && ready[dev].load(std::memory_order_acquire) == 1) return cudaSuccess;
    cudaFuncAttributes a;
    e = cudaFuncGetAttributes(&a, kern);
    if (e != cudaSuccess) return e;
    if (regs > 0 && a.numRegs != regs) return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    if (known) ready[dev].store(1, std::memory_order_release);
    return cudaSuccess;
}

// 2D map over bytes (or bf16 elements) of a row-major array in the 128-byte
// swizzle: `inner` elements per row, `outer` rows `row_bytes` apart, boxes of
// 128 bytes x box_rows; what lies outside reads as zeros.
inline bool encode_rows(CUtensorMap* map, CUtensorMapDataType dt, int elem, const void* base, int64_t inner,
                        int64_t outer, int64_t row_bytes, uint32_t box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
    const cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / elem), box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, dt, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
inline bool encode_codes(CUtensorMap* map, const void* base, int64_t inner, int64_t outer, int64_t row_bytes,
                         uint32_t box_rows) {
    return encode_rows(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, inner, outer, row_bytes, box_rows);
}

}  // namespace wq
