// mdq_ops.cuh - what the training-step operators (mdq_ops.h) share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mdq_ops.h"

// The library's error record (mdq_step.cu).
mdq_status mdq_fail(mdq_status s, const char* fmt, ...);
void mdq_clear_error();

namespace mdq_ops {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// Element i of an array whose dtype is known at run time (parameter vectors,
// which are read once per block).
__device__ __forceinline__ float load_any(const void* p, bool bf16, int64_t i) {
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_any(void* p, bool bf16, int64_t i, float v) {
    if (bf16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<float*>(p)[i] = v;
}
__device__ __forceinline__ int64_t load_id(const void* p, bool i64, int64_t i) {
    return i64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

inline bool float_type(int32_t t) { return t == MDQ_F32 || t == MDQ_BF16; }
inline bool id_type(int32_t t) { return t == MDQ_I32 || t == MDQ_I64; }

inline mdq_status launch_status(const char* what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? MDQ_OK
                            : mdq_fail(MDQ_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace mdq_ops
