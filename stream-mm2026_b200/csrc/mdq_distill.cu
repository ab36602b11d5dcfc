// mdq_distill.cu - distillation from a teacher's top logits: loss and gradient
// (mdq_ops.h).
#include "mdq_ops.cuh"

#include <math_constants.h>

namespace {

using namespace mdq_ops;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float block_max(float v) {
    __shared__ float red[kWarps];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) v = fmaxf(v, red[i]);
    return v;
}
__device__ __forceinline__ float block_sum(float v) {
    __shared__ float red[kWarps];
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) v += red[i];
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_rows(const __grid_constant__
                                                         mdq_topk_distill_desc d) {
    __shared__ int64_t idx[MDQ_DISTILL_MAX_TOP];
    __shared__ float q[MDQ_DISTILL_MAX_TOP], lq[MDQ_DISTILL_MAX_TOP];
    const int64_t r = blockIdx.x;
    const T* z = static_cast<const T*>(d.logits) + r * d.logits_stride;
    T* out = d.grad == nullptr ? nullptr : static_cast<T*>(d.grad) + r * d.grad_stride;
    const float it = 1.0f / d.temperature, c = it * kLog2e;
    const float w = d.weight == nullptr ? 1.0f : d.weight[r];
    const float scale = d.scale * w;
    float tm = -CUDART_INF_F;
    if (w != 0.0f) {
        for (int k = threadIdx.x; k < d.top; k += kThreads) {
            int64_t i = load_id(d.index, d.index_dtype == MDQ_I64, r * d.top + k);
            float t = load_any(d.teacher, d.teacher_dtype == MDQ_BF16, r * d.top + k);
            if (i < 0 || i >= d.vocab) { i = -1; t = -CUDART_INF_F; }
            idx[k] = i;
            lq[k] = t;
            tm = fmaxf(tm, t != t ? 0.0f : t);   // a NaN is an entry: the row becomes NaN
        }
        tm = block_max(tm);
    }
    if (tm == -CUDART_INF_F) {   // weight 0, or a teacher without an entry
        if (out != nullptr)
            for (int64_t v = threadIdx.x; v < d.vocab; v += kThreads) out[v] = from_f<T>(0.0f);
        if (threadIdx.x == 0 && d.row_loss != nullptr) d.row_loss[r] = 0.0f;
        return;
    }
    float s = 0.0f;
    for (int k = threadIdx.x; k < d.top; k += kThreads) {
        lq[k] = (lq[k] - tm) * it;
        q[k] = expf(lq[k]);
        s += q[k];
    }
    s = block_sum(s);
    const float ls = logf(s), is = 1.0f / s;
    for (int k = threadIdx.x; k < d.top; k += kThreads) {
        q[k] *= is;
        lq[k] -= ls;
    }
    float m = -CUDART_INF_F, e = 0.0f;
    for (int64_t v = threadIdx.x; v < d.vocab; v += kThreads) m = fmaxf(m, to_f(z[v]));
    m = block_max(m);
    const float shift = m * c;
    for (int64_t v = threadIdx.x; v < d.vocab; v += kThreads) e += exp2f(fmaf(to_f(z[v]), c, -shift));
    e = block_sum(e);
    const float le = logf(e);
    float l = 0.0f;
    for (int k = threadIdx.x; k < d.top; k += kThreads)
        if (q[k] != 0.0f) l += q[k] * (lq[k] - ((to_f(z[idx[k]]) - m) * it - le));
    l = block_sum(l);
    if (threadIdx.x == 0 && d.row_loss != nullptr)
        d.row_loss[r] = d.temperature * d.temperature * scale * l;
    if (out == nullptr) return;
    const float u = d.upstream == nullptr ? 1.0f : d.upstream[r * d.upstream_stride];
    const float f = u * scale * d.temperature, pe = f / e;
    float own[(MDQ_DISTILL_MAX_TOP + kThreads - 1) / kThreads];
    int slot = 0;
    for (int k = threadIdx.x; k < d.top; k += kThreads, ++slot) {
        // The gradient at the entry's index, its repetitions counted; read before any is written.
        if (idx[k] < 0) continue;
        float sum = 0.0f;
        for (int j = 0; j < d.top; ++j) sum += idx[j] == idx[k] ? q[j] : 0.0f;
        own[slot] = pe * exp2f(fmaf(to_f(z[idx[k]]), c, -shift)) - f * sum;
    }
    __syncthreads();
    for (int64_t v = threadIdx.x; v < d.vocab; v += kThreads)
        out[v] = from_f<T>(pe * exp2f(fmaf(to_f(z[v]), c, -shift)));
    __syncthreads();
    slot = 0;
    for (int k = threadIdx.x; k < d.top; k += kThreads, ++slot)
        if (idx[k] >= 0) out[idx[k]] = from_f<T>(own[slot]);
}

// The sum of the rows' losses, in a fixed order.
__global__ void __launch_bounds__(kThreads) distill_total(const float* rows, int64_t n, float* out) {
    __shared__ double red[kThreads];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) s += rows[i];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) *out = (float)red[0];
}

}  // namespace

extern "C" mdq_status mdq_topk_distill(const mdq_topk_distill_desc* d, cudaStream_t stream) {
    mdq_clear_error();
    if (d == nullptr) return mdq_fail(MDQ_ERR_INVALID_ARG, "distill: null descriptor");
    if (d->rows < 0 || d->vocab < 1 || d->top < 1 || d->logits_stride < 0 || d->grad_stride < 0)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "distill: bad size");
    if (!float_type(d->logits_dtype) || !float_type(d->teacher_dtype))
        return mdq_fail(MDQ_ERR_UNSUPPORTED, "distill: logits must be MDQ_F32 or MDQ_BF16");
    if (!id_type(d->index_dtype))
        return mdq_fail(MDQ_ERR_UNSUPPORTED, "distill: indices must be MDQ_I32 or MDQ_I64");
    if (!(d->temperature > 0.0f) || d->temperature > 3.0e38f)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "distill: temperature must be positive and finite");
    if (d->upstream_stride != 0 && d->upstream_stride != 1)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "distill: upstream_stride must be 0 or 1");
    if (d->top > MDQ_DISTILL_MAX_TOP)
        return mdq_fail(MDQ_ERR_TOO_LARGE, "distill: more than %d entries a row", MDQ_DISTILL_MAX_TOP);
    if (d->rows > INT32_MAX || d->vocab > INT32_MAX)
        return mdq_fail(MDQ_ERR_TOO_LARGE, "distill: 2^31 rows or vocabulary entries or more");
    if (d->loss != nullptr && d->row_loss == nullptr && d->rows > 0)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "distill: loss needs row_loss");
    if (d->rows > 0 && (d->logits == nullptr || d->teacher == nullptr || d->index == nullptr))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "distill: null pointer");
    if (d->grad != nullptr && d->rows > 1 && d->grad_stride < d->vocab)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "distill: rows of grad overlap");
    if (d->rows == 0 && d->loss == nullptr) return MDQ_OK;
    if (d->rows > 0) {
        if (d->logits_dtype == MDQ_BF16)
            distill_rows<__nv_bfloat16><<<(unsigned)d->rows, kThreads, 0, stream>>>(*d);
        else
            distill_rows<float><<<(unsigned)d->rows, kThreads, 0, stream>>>(*d);
    }
    if (d->loss != nullptr) distill_total<<<1, kThreads, 0, stream>>>(d->row_loss, d->rows, d->loss);
    return launch_status("distill");
}
