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

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// ---- bulk copies into shared memory

__device__ __forceinline__ unsigned smem_at(const void* p) {
    return (unsigned)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void bar_init(void* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_at(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(void* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_at(bar)) : "memory");
}

// Whether the barrier's phase ended.  Phases last microseconds; the limit
// (hundreds of milliseconds) only keeps a lost copy from hanging the GPU.  Behind
// a wait that ran out nothing that it was for is used, nothing more is copied, and
// the results become NaN.
[[nodiscard]] __device__ __forceinline__ bool bar_wait(void* bar, unsigned parity) {
    for (int i = 0; i < 1 << 22; ++i) {
        unsigned done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(smem_at(bar)), "r"(parity) : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ unsigned long long read_once() {   // evict-first in L2
    unsigned long long policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
// Arrives at the barrier, which `bytes` of copies (may be 0) end on as well.
__device__ __forceinline__ void expect_bytes(void* bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_at(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void copy_part(void* bar, void* to, const void* from, unsigned bytes,
                                          unsigned long long policy) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1], %2, [%3], %4;" ::"r"(smem_at(to)),
        "l"(from), "r"(bytes), "r"(smem_at(bar)), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void copy_in(void* bar, void* to, const void* from, unsigned bytes,
                                        unsigned long long policy) {
    expect_bytes(bar, bytes);
    if (bytes > 0) copy_part(bar, to, from, bytes, policy);
}

inline bool float_type(int32_t t) { return t == MDQ_F32 || t == MDQ_BF16; }
inline bool id_type(int32_t t) { return t == MDQ_I32 || t == MDQ_I64; }

inline mdq_status launch_status(const char* what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? MDQ_OK
                            : mdq_fail(MDQ_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

// 16 bytes of T as floats and back.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    __device__ static __forceinline__ void unpack(uint4 w, float (&v)[4]) {
        v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y);
        v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
    }
    __device__ static __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                          __float_as_uint(v[3]));
    }
};
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&p);
}
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    __device__ static __forceinline__ void unpack(uint4 w, float (&v)[8]) {
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    __device__ static __forceinline__ uint4 pack(const float (&v)[8]) {
        return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                          pack_bf16(v[6], v[7]));
    }
};

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
inline int64_t type_size(int32_t t) { return t == MDQ_BF16 ? 2 : 4; }
// Whether rows `stride` elements apart from `p` on all start on 16 bytes.
inline bool rows16(const void* p, int64_t stride, int32_t type) {
    return aligned16(p) && stride * type_size(type) % 16 == 0;
}
inline int64_t ceil_div(int64_t a, int64_t b) { return a / b + (a % b != 0); }

// Dynamic shared memory a kernel may ask for: 227 KB less its static arrays,
// which stay below 4 KB (launch<MOST> where they do not).
constexpr int kMaxShared = 223 * 1024;

// One launch.  With `dependent` the grid may be set up while the previous
// kernel of the stream still runs; it calls wait_previous() before it reads
// what that kernel wrote (programmatic dependent launch).
template <int MOST = kMaxShared, typename... P, typename... A>
inline cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem,
                          cudaStream_t stream, int cluster, bool dependent, A... args) {
    // (48 KB with the static arrays need no leave.)  Always the same limit: calls
    // of other threads may set it as well.
    if (smem > 16 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(
            reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize,
            MOST);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchAttribute at[2];
    unsigned n = 0;
    if (cluster > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = (unsigned)cluster;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        ++n;
    }
    if (dependent) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    c.attrs = at;
    c.numAttrs = n;
    return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}

// Until the previous kernel of the stream has ended and its writes are visible
// (at once when this kernel was not launched as dependent).
__device__ __forceinline__ void wait_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

inline mdq_status status_of(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return MDQ_OK;
    cudaGetLastError();   // the error is reported here, not by a later launch
    return mdq_fail(MDQ_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace mdq_ops
