// mdq_norm.cu - residual norm (mdq_ops.h): its entry points, the sums over CTAs,
// and the kernels for rows that no cluster holds (the others: mdq_norm.cuh).
#include "mdq_norm.cuh"

#include <utility>

namespace {

using namespace mdq_norm;

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

// ------------------------------------------------- rows wider than a cluster

__global__ void __launch_bounds__(kThreads) norm_wide(const __grid_constant__
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

__global__ void __launch_bounds__(kThreads) norm_grad_wide(const __grid_constant__
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
__global__ void __launch_bounds__(kThreads) norm_grad_wide_columns(const __grid_constant__
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

// ------------------------------------------------------------- sums over CTAs

// Adds the CTAs' sums of 32 columns, a warp every 16th CTA, and the warps' sums
// in order; forms the parameters' gradients from them.  blockIdx.y: the norm
// before, the norm behind, and then rows of the gate whose group no team had
// whole, from the teams' sums of it.
__global__ void __launch_bounds__(512) norm_grad_sum(const __grid_constant__
                                                     mdq_residual_norm_grad_desc g,
                                                     const __grid_constant__ Partials W, int blocks,
                                                     int run, int full, int grouped) {
    __shared__ float red[2][16][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t dim = g.f.dim, c = (int64_t)blockIdx.x * 32 + lane;
    const bool pb = g.f.param_dtype == MDQ_BF16;
    // Sums of `count` pairs `step` floats apart from p on, the second of a pair at `other`.
    const auto total = [&](const float* p, int64_t count, int64_t step, int64_t other, float& s, float& b) {
        s = b = 0.0f;
        if (c < dim) {
#pragma unroll 5
            for (int64_t i = warp; i < count; i += 16) {
                s += p[i * step + c];
                if (full) b += p[i * step + other + c];
            }
        }
        __syncthreads();
        red[0][warp][lane] = s;
        red[1][warp][lane] = b;
        __syncthreads();
        s = b = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            s += red[0][k][lane];
            b += red[1][k][lane];
        }
    };
    wait_previous();
    float s, b;
    const bool post = c < dim && g.f.h != nullptr && warp == 0 && blockIdx.y > 0;
    const float w = post ? load_any(g.f.post_weight, pb, c) : 0.0f;
    const float bias = post && g.f.post_bias != nullptr ? load_any(g.f.post_bias, pb, c) : 0.0f;
    if (blockIdx.y >= 2) {
        const int64_t per = g.f.rows / g.f.gate_rows;
        for (int64_t k = blockIdx.y - 2; k < g.f.gate_rows; k += gridDim.y - 2) {
            const int64_t first = k * per / run, last = ((k + 1) * per - 1) / run;   // teams
            if (first == last) continue;
            // The group began in the first of these teams, and before the others:
            // the first's second place, then the others' first.
            total(W.edges + (first * 2 + 2) * 2 * dim, last - first, 4 * dim, dim, s, b);
            if (post) {
                const float* edge = W.edges + (first * 2 + 1) * 2 * dim;
                s += edge[c];
                if (full) b += edge[dim + c];
                store_any(g.grad_gate, pb, k * dim + c, fmaf(w, s, bias * b));
            }
        }
        return;
    }
    const int kind = blockIdx.y;   // kPre or kPost; its bias is two further
    total(W.sums + kind * dim, blocks, 4 * dim, 2 * dim, s, b);
    if (warp != 0 || c >= dim) return;
    if (kind == kPre) {
        if (g.grad_pre_weight != nullptr) store_any(g.grad_pre_weight, pb, c, s);
        if (g.grad_pre_bias != nullptr) store_any(g.grad_pre_bias, pb, c, b);
        return;
    }
    // One gate for all rows is applied here, and its gradient follows from the
    // same sums; otherwise the rows applied theirs.
    float gate = 1.0f;
    if (!grouped && g.f.gate != nullptr) {
        gate = load_any(g.f.gate, pb, c);
        if (g.grad_gate != nullptr) store_any(g.grad_gate, pb, c, fmaf(w, s, bias * b));
    }
    if (g.grad_post_weight != nullptr) store_any(g.grad_post_weight, pb, c, gate * s);
    if (g.grad_post_bias != nullptr) store_any(g.grad_post_bias, pb, c, gate * b);
}

// ------------------------------------------------------------------ planning

// Threads for `share` columns in `chunks` chunks of a thread.
int threads_for(int64_t share, int chunks) { return (int)ceil_div(share, 32 * kCols * chunks) * 32; }

// Columns a CTA takes and the CTAs of a row, with at most `chunks` chunks a
// thread; false when the row is too wide for a cluster.
bool plan_columns(int64_t dim, int chunks, int* cluster, Teams* G) {
    const int64_t most = (int64_t)kTeam * kCols * chunks;
    *cluster = 1;
    while (*cluster < kMaxCluster && dim > *cluster * most) *cluster *= 2;
    if (dim > *cluster * most) return false;
    G->share = (int)(ceil_div(ceil_div(dim, *cluster), kCols) * kCols);
    return true;
}

// Bytes of a stage whose arrays take `row_bytes` a column.
int64_t stage_of(int64_t row_bytes, int arrays, bool vec, const Teams& G, int chunks) {
    return vec ? row_bytes * G.share : row_bytes * G.threads * kCols * chunks + 48 * arrays;
}
// Teams of a CTA: as many as rows for all SMs need, 512 threads at most, and so
// many stages for each that two rows are on their way, in 200 KB with `kept` bytes
// of each team beside its stages.
bool plan_ring(int64_t rows, int64_t stage, int64_t kept, bool one, Teams* G, int* stages, size_t* smem) {
    const int64_t room = 200 * 1024;
    int64_t teams = one ? 1 : kTeam / G->threads;
    const int64_t need = ceil_div(rows, 148);
    if (teams > need) teams = need < 1 ? 1 : need;
    while (teams > 1 && (3 * stage + kept) * teams > room) --teams;
    int64_t n = (room / teams - kept) / stage;
    if (n < 2) return false;
    const int64_t run = ceil_div(rows, 148 * teams);   // more would not be used
    if (n > run + 1) n = run + 1 < 2 ? 2 : run + 1;
    if (n > kMaxStages) n = kMaxStages;
    G->teams = (int)teams;
    *stages = (int)n;
    *smem = (size_t)((n * stage + kept) * teams);
    return true;
}

struct RowsPlan {
    Teams G;
    int cluster, chunks, grid;
    int stages;        // of the kernel with a ring, 0: the other
    size_t smem;
};
// Forward: two chunks a thread for many rows above 256 columns, one for narrow
// or few (as few threads as 512 allow), four where that is not enough.
// 32768 bf16 rows of 2048 / 768 / 128 columns: 96 / 46 / 16 us with two chunks, 126 /
// 81 / 13 with one, 112 / 50 / 32 with four.
// Four chunks have their parameters loaded for every row, value by value off 16
// bytes: rather twice the CTAs then (4112 bf16 rows of 16301: 235 against 425 us, layer
// norm 361 against 584), but for fp32 rows without means and biases (6704 of 10001: 343
// against 318; with them 532 against 498).
bool plan_forward(int64_t rows, int64_t dim, int64_t row_bytes, bool vec, bool full, RowsPlan* p) {
    const bool ring = full || !vec;
    for (int most = vec || (row_bytes == 8 && !full) ? 4 : 2; most >= 1; most /= 2) {
        if (!plan_columns(dim, most, &p->cluster, &p->G)) return false;
        Teams& G = p->G;
        p->chunks = rows > 296 && G.share > 256 && most > 1 ? 2 : 1;
        while (threads_for(G.share, p->chunks) > kTeam) p->chunks *= 2;
        G.threads = threads_for(G.share, p->chunks);
        p->stages = 0;
        int64_t ctas = 1;   // of an SM: 512 threads, as their registers go
        if (!ring) {
            G.teams = p->cluster > 1 || G.threads > 64 ? 1 : 128 / G.threads;
            if (G.threads * G.teams < kTeam) ctas = kTeam / (G.threads * G.teams);
        } else if (!plan_ring(rows, stage_of(row_bytes, 2, vec, G, p->chunks), 0, p->cluster > 1, &G,
                              &p->stages, &p->smem)) {
            continue;   // a stage too large: more CTAs a row
        }
        const int64_t need = ceil_div(rows, G.teams), all = 148 * ctas / p->cluster;
        p->grid = (int)(need < all ? need : all);
        G.run = (int)ceil_div(rows, (int64_t)p->grid * G.teams);
        p->grid *= p->cluster;
        return true;
    }
    return false;
}

// The backward pass's teams, their rows, and what the workspace holds.
struct GradPlan {
    Teams G;
    int cluster, chunks;
    int stages;        // of the streaming kernel, 0: the other
    size_t smem;
    int64_t blocks;    // clusters, each with a row of sums
    int64_t bytes;
};
// Rows, sums and bytes once teams are known: one CTA an SM, as their registers go.
void plan_rows(int64_t rows, int64_t dim, int64_t gate_rows, GradPlan* p) {
    Teams& G = p->G;
    const int64_t most = 148 / p->cluster;
    p->blocks = ceil_div(rows, G.teams);
    if (p->blocks > most) p->blocks = most;
    if (p->blocks < 1) p->blocks = 1;
    G.run = (int)ceil_div(rows, p->blocks * G.teams);
    if (G.run < 1) G.run = 1;
    const int64_t edges = gate_rows > 1 ? p->blocks * G.teams * 4 * dim : 0;
    p->bytes = (p->blocks * 4 * dim + edges) * (int64_t)sizeof(float);
}
bool plan_grad(int64_t rows, int64_t dim, int64_t gate_rows, bool full, GradPlan* p) {
    // Four chunks where two sums of 16384 columns fit into shared memory.
    const bool wide = !full && gate_rows == 1;
    p->stages = 0;
    p->smem = 0;
    if (!plan_columns(dim, wide ? 4 : 2, &p->cluster, &p->G)) return false;
    Teams& G = p->G;
    p->chunks = 2;
    while (threads_for(G.share, p->chunks) > kTeam) p->chunks *= 2;
    G.threads = threads_for(G.share, p->chunks);
    G.teams = 1;
    plan_rows(rows, dim, gate_rows, p);
    return true;
}
// With rows in a ring.  Above 8192 columns the steps between more than two CTAs
// take longer than the other kernel's rows (431 against 270 us for 4096 bf16 rows of
// 16384), but not than its loads of rows off 16 bytes (497 against 1597 us for 4112
// rows of 16301).  Rows off 16 bytes of more than 32768 columns, which no cluster's
// ring takes, are left to it: calls for 16 / 512 bf16 rows of 33001, 62 / 1163 us, and
// 512 of 65535, 1319, against 561 / 2053 and 2956 by the kernels for rows wider than a
// cluster.
bool plan_stream(int64_t rows, int64_t dim, int64_t gate_rows, int64_t row_bytes, bool vec, bool full,
                 GradPlan* p) {
    p->chunks = 1;
    if (!plan_columns(dim, 1, &p->cluster, &p->G) || (vec && p->cluster > 2)) return false;
    Teams& G = p->G;
    G.threads = threads_for(G.share, 1);
    const int64_t stage = stage_of(row_bytes, 4, vec, G, 1) + 16;
    // a gate of groups: every thread's sums over its groups
    const int64_t kept = gate_rows > 1 ? (full ? 64 : 32) * G.threads : 0;
    if (!plan_ring(rows, stage, kept, p->cluster > 1, &G, &p->stages, &p->smem)) return false;
    const size_t sums = kept * G.teams + (G.teams > 1 ? (full ? 4 : 2) * G.share * sizeof(float) : 0);
    if (p->smem < sums) p->smem = sums;
    plan_rows(rows, dim, gate_rows, p);
    return true;
}

#define MDQ_NORM_PICK(FN, XT, HT)                                                                  \
    ((XT) == MDQ_F32 ? ((HT) == MDQ_F32 ? FN##_ff : FN##_fb) : ((HT) == MDQ_F32 ? FN##_bf : FN##_bb))

bool vector_rows(const mdq_residual_norm_desc& d) {
    const bool p = d.dim % kCols == 0 && aligned16(d.post_weight) && aligned16(d.post_bias) &&
                   aligned16(d.pre_weight) && aligned16(d.pre_bias) && aligned16(d.gate);
    return p && rows16(d.x, d.x_stride, d.x_dtype) &&
           (d.h == nullptr || rows16(d.h, d.h_stride, d.h_dtype));
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
    if (!aligned16(a.stats)) return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm: stats misaligned");
    RowsPlan p;
    const bool vec = vector_rows(a) && aligned16(a.x_new) && aligned16(a.n);
    const bool full = a.kind == MDQ_NORM_LAYER || a.post_bias != nullptr || a.pre_bias != nullptr;
    if (plan_forward(a.rows, a.dim, type_size(a.x_dtype) + type_size(a.h_dtype), vec, full, &p))
        return status_of(MDQ_NORM_PICK(forward, a.x_dtype, a.h_dtype)(
                             a, p.G, p.chunks, p.grid, p.cluster, p.stages, p.smem, vec, full, stream),
                         "residual norm");
    norm_wide<<<(unsigned)d->rows, kThreads, 0, stream>>>(a);
    return launch_status("residual norm");
}

mdq_status mdq_residual_norm_grad_workspace_bytes(int64_t rows, int64_t dim, int64_t gate_rows,
                                                  int64_t* bytes) {
    mdq_clear_error();
    if (bytes == nullptr || rows < 0 || dim < 1 || gate_rows < 1)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm grad: bad size");
    // Enough for either kind of norm and all types.
    *bytes = rows * 2 * (int64_t)sizeof(float);
    for (int full = 0; full < 2; ++full)
        for (int vec = 0; vec < 2; ++vec)
            for (int row_bytes = 0; row_bytes <= 16; row_bytes += row_bytes < 8 ? 8 : 4) {
                GradPlan p;
                const bool ok = row_bytes == 0
                                    ? plan_grad(rows, dim, gate_rows, full, &p)
                                    : plan_stream(rows, dim, gate_rows, row_bytes, vec, full, &p);
                if (ok && p.bytes > *bytes) *bytes = p.bytes;
            }
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
    if (!aligned16(g->workspace) || !aligned16(g->f.stats))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "residual norm grad: workspace or stats misaligned");
    if (g->f.rows == 0) {   // sums over no rows, whatever the parameters hold
        const size_t row = (size_t)(g->f.dim * type_size(g->f.param_dtype));
        const std::pair<void*, int64_t> sums[] = {
            {g->grad_post_weight, 1}, {g->grad_post_bias, 1}, {g->grad_pre_weight, 1},
            {g->grad_pre_bias, 1},    {g->grad_gate, g->f.gate_rows}};
        cudaError_t e = cudaSuccess;
        for (const auto& s : sums)
            if (s.first != nullptr && e == cudaSuccess) e = cudaMemsetAsync(s.first, 0, s.second * row, stream);
        return status_of(e, "residual norm grad");
    }
    const bool grouped = g->f.gate_rows > 1;
    const bool full = g->f.kind == MDQ_NORM_LAYER || g->f.post_bias != nullptr || g->f.pre_bias != nullptr;
    const bool vec = vector_rows(g->f) && aligned16(g->grad_x) && aligned16(g->grad_h) &&
                     (g->grad_new == nullptr || rows16(g->grad_new, g->grad_new_stride, g->f.x_dtype)) &&
                     (g->grad_n == nullptr || rows16(g->grad_n, g->grad_n_stride, g->f.h_dtype));
    const int row_bytes = 2 * (int)(type_size(g->f.x_dtype) + type_size(g->f.h_dtype));
    GradPlan p;
    const bool planned = plan_stream(g->f.rows, g->f.dim, g->f.gate_rows, row_bytes, vec, full, &p) ||
                         plan_grad(g->f.rows, g->f.dim, g->f.gate_rows, full, &p);
    const int64_t need = planned ? p.bytes : g->f.rows * 2 * (int64_t)sizeof(float);
    if (need > 0 && (g->workspace == nullptr || g->workspace_bytes < need))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "workspace holds %lld bytes, %lld needed",
                        (long long)g->workspace_bytes, (long long)need);
    if (!planned) {
        float* means = static_cast<float*>(g->workspace);
        norm_grad_wide<<<(unsigned)g->f.rows, kThreads, 0, stream>>>(*g, means);
        norm_grad_wide_columns<<<(unsigned)ceil_div(g->f.dim, kThreads), kThreads, 0, stream>>>(*g, means);
        return launch_status("residual norm grad");
    }
    Partials W;
    W.sums = static_cast<float*>(g->workspace);
    W.edges = W.sums + p.blocks * 4 * g->f.dim;
    const int grid = (int)p.blocks * p.cluster;
    st = status_of(p.stages > 0 ? MDQ_NORM_PICK(stream, g->f.x_dtype, g->f.h_dtype)(
                                      *g, p.G, W, p.stages, p.smem, grid, p.cluster, vec, full, grouped, stream)
                                : MDQ_NORM_PICK(backward, g->f.x_dtype, g->f.h_dtype)(
                                      *g, p.G, W, p.chunks, grid, p.cluster, vec, full, grouped, stream),
                   "residual norm grad");
    if (st != MDQ_OK) return st;
    const bool gates = grouped && g->grad_gate != nullptr;
    const int64_t groups = !gates ? 0 : g->f.gate_rows < 256 ? g->f.gate_rows : 256;
    const dim3 columns((unsigned)ceil_div(g->f.dim, 32), g->f.h != nullptr ? (unsigned)(2 + groups) : 1);
    const cudaError_t e = launch(norm_grad_sum, columns, 512, 0, stream, 1, true, *g, W, (int)p.blocks,
                                 p.G.run, (int)full, (int)grouped);
    return status_of(e, "residual norm grad");
}

}  // extern "C"
