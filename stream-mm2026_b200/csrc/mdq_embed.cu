// mdq_embed.cu - scaled embedding lookup and its gradient (mdq_ops.h).
#include "mdq_ops.cuh"

namespace {

using namespace mdq_ops;

constexpr int kThreads = 256;

template <typename TT, typename OT>
__global__ void __launch_bounds__(kThreads) embed_rows(const __grid_constant__ mdq_embed_desc d) {
    const int64_t n = blockIdx.x;
    const int64_t id = load_id(d.ids, d.ids_dtype == MDQ_I64, n);
    const bool in = id >= 0 && id < d.vocab;
    const TT* row = static_cast<const TT*>(d.table) + (in ? id : 0) * d.table_stride;
    OT* out = static_cast<OT*>(d.out) + n * d.dim;
    for (int64_t c = threadIdx.x; c < d.dim; c += kThreads)
        out[c] = from_f<OT>(in ? to_f(row[c]) * d.scale : 0.0f);
}

template <typename WT>
__global__ void __launch_bounds__(kThreads) embed_grad_zero(WT* grad, int64_t n) {
    const int64_t step = (int64_t)gridDim.x * kThreads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += step)
        grad[i] = from_f<WT>(0.0f);
}

// Block n owns the row of ids[n] if no earlier token has the same id; it adds
// the rows of all tokens with that id in order.
template <typename GT, typename WT>
__global__ void __launch_bounds__(kThreads) embed_grad_first(const __grid_constant__
                                                             mdq_embed_grad_desc d) {
    __shared__ int seen;
    const int64_t n = blockIdx.x;
    const bool i64 = d.ids_dtype == MDQ_I64;
    const int64_t id = load_id(d.ids, i64, n);
    if (id < 0 || id >= d.vocab || id == d.padding_idx) return;
    if (threadIdx.x == 0) seen = 0;
    __syncthreads();
    bool mine = false;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) mine |= load_id(d.ids, i64, i) == id;
    if (mine) seen = 1;
    __syncthreads();
    if (seen) return;
    const GT* g = static_cast<const GT*>(d.grad_out);
    WT* out = static_cast<WT*>(d.grad) + id * d.dim;
    for (int64_t c = threadIdx.x; c < d.dim; c += kThreads) {
        float s = 0.0f;
        for (int64_t i = n; i < d.tokens; ++i)
            if (load_id(d.ids, i64, i) == id) s += to_f(g[i * d.grad_out_stride + c]);
        s *= d.scale;
        out[c] = from_f<WT>(d.accumulate ? to_f(out[c]) + s : s);
    }
}

}  // namespace

extern "C" {

mdq_status mdq_embed(const mdq_embed_desc* d, cudaStream_t stream) {
    mdq_clear_error();
    if (d == nullptr) return mdq_fail(MDQ_ERR_INVALID_ARG, "embed: null descriptor");
    if (d->tokens < 0 || d->vocab < 1 || d->dim < 1 || d->table_stride < 0)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "embed: bad size");
    if (!float_type(d->table_dtype) || !float_type(d->out_dtype))
        return mdq_fail(MDQ_ERR_UNSUPPORTED, "embed: table and out must be MDQ_F32 or MDQ_BF16");
    if (!id_type(d->ids_dtype))
        return mdq_fail(MDQ_ERR_UNSUPPORTED, "embed: ids must be MDQ_I32 or MDQ_I64");
    if (d->tokens > INT32_MAX) return mdq_fail(MDQ_ERR_TOO_LARGE, "embed: 2^31 tokens or more");
    if (d->tokens == 0) return MDQ_OK;
    if (d->table == nullptr || d->ids == nullptr || d->out == nullptr)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "embed: null pointer");
    const unsigned grid = (unsigned)d->tokens;
    const bool tb = d->table_dtype == MDQ_BF16, ob = d->out_dtype == MDQ_BF16;
    if (tb && ob) embed_rows<__nv_bfloat16, __nv_bfloat16><<<grid, kThreads, 0, stream>>>(*d);
    else if (tb) embed_rows<__nv_bfloat16, float><<<grid, kThreads, 0, stream>>>(*d);
    else if (ob) embed_rows<float, __nv_bfloat16><<<grid, kThreads, 0, stream>>>(*d);
    else embed_rows<float, float><<<grid, kThreads, 0, stream>>>(*d);
    return launch_status("embed");
}

mdq_status mdq_embed_grad_workspace_bytes(int64_t tokens, int64_t vocab, int64_t dim,
                                          int64_t* bytes) {
    mdq_clear_error();
    if (bytes == nullptr || tokens < 0 || vocab < 1 || dim < 1)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "embed grad: bad size");
    *bytes = 0;
    return MDQ_OK;
}

mdq_status mdq_embed_grad(const mdq_embed_grad_desc* d, cudaStream_t stream) {
    mdq_clear_error();
    if (d == nullptr) return mdq_fail(MDQ_ERR_INVALID_ARG, "embed grad: null descriptor");
    if (d->tokens < 0 || d->vocab < 1 || d->dim < 1 || d->grad_out_stride < 0 ||
        d->padding_idx < -1)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "embed grad: bad size");
    if (!float_type(d->grad_out_dtype) || !float_type(d->grad_dtype))
        return mdq_fail(MDQ_ERR_UNSUPPORTED, "embed grad: types must be MDQ_F32 or MDQ_BF16");
    if (!id_type(d->ids_dtype))
        return mdq_fail(MDQ_ERR_UNSUPPORTED, "embed grad: ids must be MDQ_I32 or MDQ_I64");
    if (d->accumulate && d->grad_dtype != MDQ_F32)
        return mdq_fail(MDQ_ERR_UNSUPPORTED, "embed grad: accumulate needs an MDQ_F32 gradient");
    if (d->tokens > INT32_MAX || d->vocab > INT32_MAX - 1)
        return mdq_fail(MDQ_ERR_TOO_LARGE, "embed grad: 2^31 tokens or ids or more");
    if (d->grad == nullptr || (d->tokens > 0 && (d->ids == nullptr || d->grad_out == nullptr)))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "embed grad: null pointer");
    const bool gb = d->grad_out_dtype == MDQ_BF16, wb = d->grad_dtype == MDQ_BF16;
    if (!d->accumulate) {
        const int64_t n = d->vocab * d->dim;
        if (wb) embed_grad_zero<<<148 * 8, kThreads, 0, stream>>>((__nv_bfloat16*)d->grad, n);
        else embed_grad_zero<<<148 * 8, kThreads, 0, stream>>>((float*)d->grad, n);
    }
    if (d->tokens > 0) {
        const unsigned grid = (unsigned)d->tokens;
        if (gb && wb) embed_grad_first<__nv_bfloat16, __nv_bfloat16><<<grid, kThreads, 0, stream>>>(*d);
        else if (gb) embed_grad_first<__nv_bfloat16, float><<<grid, kThreads, 0, stream>>>(*d);
        else if (wb) embed_grad_first<float, __nv_bfloat16><<<grid, kThreads, 0, stream>>>(*d);
        else embed_grad_first<float, float><<<grid, kThreads, 0, stream>>>(*d);
    }
    return launch_status("embed grad");
}

}  // extern "C"
