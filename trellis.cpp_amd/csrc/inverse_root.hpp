// The reciprocal square root of norms.
#pragma once
#include <hip/hip_runtime.h>

namespace tsp {

// 1 / sqrt(v) of a norm. (The fp32 instruction takes values below the normal range for zero.)
__device__ __forceinline__ float inverse_root(float v) {
    const bool small = v < 0x1p-126f;
    const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p64f : v);
    return small ? r * 0x1p32f : r;
}
__device__ __forceinline__ double inverse_root(double v) { return 1.0 / sqrt(v); }

}  // namespace tsp
