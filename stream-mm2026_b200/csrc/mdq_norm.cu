// mdq_norm.cu - the norm after a block with its gate and the residual's scale,
// and the norm before the next block (mdq_ops.h).
#include "mdq_ops.cuh"

namespace {

using namespace mdq_ops;

constexpr int kThreads = 256;

// Sum over the block, given to every thread.
__device__ __forceinline__ float block_sum(float v) {
    __shared__ float red[kThreads / 32];
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) s += red[i];
    return s;
}

struct Row {
    const mdq_residual_norm_desc& d;
    int64_t r;
    bool xb, hb, pb;
    __device__ Row(const mdq_residual_norm_desc& desc, int64_t row)
        : d(desc), r(row), xb(desc.x_dtype == MDQ_BF16), hb(desc.h_dtype == MDQ_BF16),
          pb(desc.param_dtype == MDQ_BF16) {}
    __device__ float x(int64_t c) const { return load_any(d.x, xb, r * d.x_stride + c); }
    __device__ float h(int64_t c) const { return load_any(d.h, hb, r * d.h_stride + c); }
    __device__ float par(const void* p, int64_t c, float none) const {
        return p == nullptr ? none : load_any(p, pb, c);
    }
    __device__ float gate(int64_t c) const {
        return d.gate == nullptr ? 1.0f
                                 : load_any(d.gate, pb, r / (d.rows / d.gate_rows) * d.dim + c);
    }
    __device__ float y(int64_t c, float mh, float rh) const {
        return fmaf((h(c) - mh) * rh, par(d.post_weight, c, 1.0f), par(d.post_bias, c, 0.0f));
    }
    __device__ float x_new(int64_t c, float mh, float rh) const {
        if (d.h == nullptr) return x(c);
        return fmaf(gate(c), y(c, mh, rh), d.residual_scale * x(c));
    }
};

__global__ void __launch_bounds__(kThreads) norm_forward(const __grid_constant__
                                                         mdq_residual_norm_desc d) {
    const Row R(d, blockIdx.x);
    const float inv = 1.0f / (float)d.dim;
    const bool layer = d.kind == MDQ_NORM_LAYER;
    float mh = 0.0f, rh = 0.0f, mx = 0.0f, rx = 0.0f;
    if (d.h != nullptr) {
        float s = 0.0f;
        if (layer) {
            for (int64_t c = threadIdx.x; c < d.dim; c += kThreads) s += R.h(c);
            mh = block_sum(s) * inv;
        }
        s = 0.0f;
        for (int64_t c = threadIdx.x; c < d.dim; c += kThreads) {
            const float v = R.h(c) - mh;
            s = fmaf(v, v, s);
        }
        rh = 1.0f / sqrtf(block_sum(s) * inv + d.eps);
    }
    if (d.n != nullptr) {
        float s = 0.0f;
        if (layer) {
            for (int64_t c = threadIdx.x; c < d.dim; c += kThreads) s += R.x_new(c, mh, rh);
            mx = block_sum(s) * inv;
        }
        s = 0.0f;
        for (int64_t c = threadIdx.x; c < d.dim; c += kThreads) {
            const float v = R.x_new(c, mh, rh) - mx;
            s = fmaf(v, v, s);
        }
        rx = 1.0f / sqrtf(block_sum(s) * inv + d.eps);
    }
    for (int64_t c = threadIdx.x; c < d.dim; c += kThreads) {
        const float v = R.x_new(c, mh, rh);
        if (d.h != nullptr) store_any(d.x_new, R.xb, R.r * d.dim + c, v);
        if (d.n != nullptr)
            store_any(d.n, R.hb, R.r * d.dim + c,
                      fmaf((v - mx) * rx, R.par(d.pre_weight, c, 1.0f), R.par(d.pre_bias, c, 0.0f)));
    }
    if (d.stats != nullptr && threadIdx.x == 0) {
        float* s = d.stats + 4 * R.r;
        s[0] = mh; s[1] = rh; s[2] = mx; s[3] = rx;
    }
}

// What one element contributes to a row's gradients.
struct Grad {
    const mdq_residual_norm_grad_desc& g;
    const Row R;
    float mh, rh, mx, rx;
    __device__ Grad(const mdq_residual_norm_grad_desc& desc, int64_t r) : g(desc), R(desc.f, r) {
        const float* s = g.f.stats + 4 * r;
        mh = s[0]; rh = s[1]; mx = s[2]; rx = s[3];
    }
    __device__ float dn(int64_t c) const {
        return g.grad_n == nullptr ? 0.0f : load_any(g.grad_n, R.hb, R.r * g.grad_n_stride + c);
    }
    __device__ float xhat(int64_t c) const { return (R.x_new(c, mh, rh) - mx) * rx; }
    __device__ float hhat(int64_t c) const { return (R.h(c) - mh) * rh; }
    __device__ float e(int64_t c) const { return dn(c) * R.par(g.f.pre_weight, c, 1.0f); }
    // the whole gradient of x_new, given the row's mean(e * xhat) and mean(e)
    __device__ float t(int64_t c, float m1, float m0) const {
        float v = g.grad_new == nullptr
                      ? 0.0f : load_any(g.grad_new, R.xb, R.r * g.grad_new_stride + c);
        if (g.grad_n != nullptr) v += rx * (e(c) - m0 - xhat(c) * m1);
        return v;
    }
    __device__ float u(int64_t c, float m1, float m0) const {
        return t(c, m1, m0) * R.gate(c) * R.par(g.f.post_weight, c, 1.0f);
    }
};

__global__ void __launch_bounds__(kThreads) norm_backward_rows(const __grid_constant__
                                                               mdq_residual_norm_grad_desc g,
                                                               float* means) {
    const Grad G(g, blockIdx.x);
    const int64_t dim = g.f.dim;
    const float inv = 1.0f / (float)dim;
    const bool layer = g.f.kind == MDQ_NORM_LAYER;
    float m1 = 0.0f, m0 = 0.0f, u1 = 0.0f, u0 = 0.0f;
    if (g.grad_n != nullptr) {
        for (int64_t c = threadIdx.x; c < dim; c += kThreads) {
            const float e = G.e(c);
            m1 = fmaf(e, G.xhat(c), m1);
            m0 += e;
        }
        m1 = block_sum(m1) * inv;
        m0 = layer ? block_sum(m0) * inv : 0.0f;
    }
    if (g.f.h != nullptr) {
        for (int64_t c = threadIdx.x; c < dim; c += kThreads) {
            const float u = G.u(c, m1, m0);
            u1 = fmaf(u, G.hhat(c), u1);
            u0 += u;
        }
        u1 = block_sum(u1) * inv;
        u0 = layer ? block_sum(u0) * inv : 0.0f;
    }
    const float a = g.f.h != nullptr ? g.f.residual_scale : 1.0f;
    for (int64_t c = threadIdx.x; c < dim; c += kThreads) {
        const int64_t i = G.R.r * dim + c;
        store_any(g.grad_x, G.R.xb, i, a * G.t(c, m1, m0));
        if (g.f.h != nullptr)
            store_any(g.grad_h, G.R.hb, i, G.rh * (G.u(c, m1, m0) - u0 - G.hhat(c) * u1));
    }
    if (threadIdx.x == 0) {
        means[2 * G.R.r] = m1;
        means[2 * G.R.r + 1] = m0;
    }
}

// Gradients of one parameter column; `gate_row` >= 0: of that row of the gate.
__global__ void __launch_bounds__(kThreads) norm_backward_columns(const __grid_constant__
                                                                  mdq_residual_norm_grad_desc g,
                                                                  const float* means) {
    const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (c >= g.f.dim) return;
    const bool pb = g.f.param_dtype == MDQ_BF16;
    const int64_t per = g.f.rows / g.f.gate_rows;
    float w1 = 0.0f, b1 = 0.0f, w2 = 0.0f, b2 = 0.0f;
    for (int64_t k = 0; k < g.f.gate_rows; ++k) {
        float dg = 0.0f;
        for (int64_t r = k * per; r < (k + 1) * per; ++r) {
            const Grad G(g, r);
            const float dn = G.dn(c);
            if (g.grad_n != nullptr) {
                w2 = fmaf(dn, G.xhat(c), w2);
                b2 += dn;
            }
            if (g.f.h != nullptr) {
                const float t = G.t(c, means[2 * r], means[2 * r + 1]), tg = t * G.R.gate(c);
                w1 = fmaf(tg, G.hhat(c), w1);
                b1 += tg;
                dg = fmaf(t, G.R.y(c, G.mh, G.rh), dg);
            }
        }
        if (g.grad_gate != nullptr) store_any(g.grad_gate, pb, k * g.f.dim + c, dg);
    }
    if (g.grad_post_weight != nullptr) store_any(g.grad_post_weight, pb, c, w1);
    if (g.grad_post_bias != nullptr) store_any(g.grad_post_bias, pb, c, b1);
    if (g.grad_pre_weight != nullptr) store_any(g.grad_pre_weight, pb, c, w2);
    if (g.grad_pre_bias != nullptr) store_any(g.grad_pre_bias, pb, c, b2);
}

mdq_status check_norm(const mdq_residual_norm_desc& d, const char* what) {
    if (d.rows < 0 || d.dim < 1 || d.x_stride < 0 || d.h_stride < 0 || d.gate_rows < 1)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "%s: bad size", what);
    if (!float_type(d.x_dtype) || !float_type(d.h_dtype) || !float_type(d.param_dtype))
        return mdq_fail(MDQ_ERR_UNSUPPORTED, "%s: types must be MDQ_F32 or MDQ_BF16", what);
    if (d.kind != MDQ_NORM_RMS && d.kind != MDQ_NORM_LAYER)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "%s: bad kind", what);
    if (d.rows > INT32_MAX || d.dim > INT32_MAX)
        return mdq_fail(MDQ_ERR_TOO_LARGE, "%s: 2^31 rows or columns or more", what);
    if (d.gate == nullptr ? d.gate_rows != 1 : d.rows % d.gate_rows != 0)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "%s: gate_rows must divide rows", what);
    if (d.rows > 0 && d.x == nullptr) return mdq_fail(MDQ_ERR_INVALID_ARG, "%s: null pointer", what);
    if (d.h == nullptr && (d.gate != nullptr || d.post_weight != nullptr || d.post_bias != nullptr))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "%s: gate and post parameters need a block", what);
    if (d.h != nullptr && d.post_weight == nullptr)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "%s: a block needs post_weight", what);
    if (d.pre_weight == nullptr && d.pre_bias != nullptr)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "%s: pre_bias without pre_weight", what);
    if (d.h == nullptr && d.pre_weight == nullptr)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "%s: neither a block nor pre_weight", what);
    return MDQ_OK;
}

}  // namespace

extern "C" {

mdq_status mdq_residual_norm(const mdq_residual_norm_desc* d, cudaStream_t stream) {
    mdq_clear_error();
    if (d == nullptr) return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm: null descriptor");
    const mdq_status st = check_norm(*d, "residual norm");
    if (st != MDQ_OK) return st;
    if (d->rows == 0) return MDQ_OK;
    if ((d->h != nullptr && d->x_new == nullptr) || (d->pre_weight != nullptr && d->n == nullptr))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm: null pointer");
    mdq_residual_norm_desc a = *d;
    if (a.pre_weight == nullptr) a.n = nullptr;
    norm_forward<<<(unsigned)d->rows, kThreads, 0, stream>>>(a);
    return launch_status("residual norm");
}

mdq_status mdq_residual_norm_grad_workspace_bytes(int64_t rows, int64_t dim, int64_t gate_rows,
                                                  int64_t* bytes) {
    mdq_clear_error();
    if (bytes == nullptr || rows < 0 || dim < 1 || gate_rows < 1)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm grad: bad size");
    *bytes = rows * 2 * (int64_t)sizeof(float);
    return MDQ_OK;
}

mdq_status mdq_residual_norm_grad(const mdq_residual_norm_grad_desc* g, cudaStream_t stream) {
    mdq_clear_error();
    if (g == nullptr) return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm grad: null descriptor");
    mdq_status st = check_norm(g->f, "residual norm grad");
    if (st != MDQ_OK) return st;
    if (g->grad_new_stride < 0 || g->grad_n_stride < 0)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm grad: bad size");
    if (g->f.pre_weight == nullptr && g->grad_n != nullptr)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm grad: grad_n without pre_weight");
    if (g->f.rows > 0 && (g->f.stats == nullptr || g->grad_x == nullptr ||
                          (g->f.h != nullptr && g->grad_h == nullptr)))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm grad: null pointer");
    int64_t need = 0;
    st = mdq_residual_norm_grad_workspace_bytes(g->f.rows, g->f.dim, g->f.gate_rows, &need);
    if (st != MDQ_OK) return st;
    if (need > 0 && (g->workspace == nullptr || g->workspace_bytes < need))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "workspace holds %lld bytes, %lld needed",
                        (long long)g->workspace_bytes, (long long)need);
    float* means = static_cast<float*>(g->workspace);
    if (g->f.rows > 0)
        norm_backward_rows<<<(unsigned)g->f.rows, kThreads, 0, stream>>>(*g, means);
    norm_backward_columns<<<(unsigned)((g->f.dim + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
        *g, means);
    return launch_status("residual norm grad");
}

}  // extern "C"
