// mdq_norm.cuh - the norm after a block with its gate and the residual's scale,
// and the norm before the next block: the kernels of mdq_norm_*.cu, one file for
// each pair of types (mdq_ops.h).
//
// Both passes are bound by memory: forward reads x and h and writes x_new and n,
// backward reads x, h and the two gradients and writes two.  A row is held in
// registers, 8 columns a thread, by a team of up to 512 threads; rows of more
// than 4096 columns by a cluster of CTAs that exchange their sums through
// distributed shared memory.  A team goes through rows one after another and
// loads the next while it works on the present one; parameters come from the L1
// cache at the place of use.  The backward pass keeps the parameters' gradients
// of its rows in registers and leaves one partial sum for each CTA, which a
// second kernel adds in a fixed order.
#pragma once

#include "mdq_ops.cuh"

#include <cooperative_groups.h>

namespace mdq_norm {

using namespace mdq_ops;
namespace cg = cooperative_groups;

constexpr int kTeam = 512;          // threads of a team at most
constexpr int kCols = 8;            // columns of a thread
constexpr int kMaxCluster = 8;

// How rows are given to threads.
struct Teams {
    int threads;    // of a team, a multiple of 32
    int teams;      // of a CTA (1 in a cluster)
    int share;      // columns of a CTA
    int run;        // rows of a team, consecutive (backward)
};

// The columns of a thread: 8 consecutive ones on 16-byte boundaries (VECTOR), or
// `step` apart.
template <bool VECTOR>
struct Cols {
    int first, step, end;
    __device__ __forceinline__ int at(int k) const { return first + (VECTOR ? k : k * step); }
    __device__ __forceinline__ bool has(int k) const { return VECTOR ? first < end : at(k) < end; }
};

// Eight values as they were loaded, 0 outside of the row.
template <typename T, bool VECTOR>
struct Raw;
template <>
struct Raw<__nv_bfloat16, true> {
    uint4 a = {0, 0, 0, 0};
    __device__ __forceinline__ void load(const __nv_bfloat16* row, const Cols<true>& c) {
        if (c.has(0)) a = __ldcs(reinterpret_cast<const uint4*>(row + c.first));
    }
    __device__ __forceinline__ void get(float (&v)[8]) const { Vec<__nv_bfloat16>::unpack(a, v); }
};
template <>
struct Raw<float, true> {
    float4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    __device__ __forceinline__ void load(const float* row, const Cols<true>& c) {
        if (c.has(0)) {
            a = __ldcs(reinterpret_cast<const float4*>(row + c.first));
            b = __ldcs(reinterpret_cast<const float4*>(row + c.first) + 1);
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <typename T>
struct Raw<T, false> {
    T a[8];
    __device__ __forceinline__ Raw() {
#pragma unroll
        for (int k = 0; k < 8; ++k) a[k] = from_f<T>(0.0f);
    }
    __device__ __forceinline__ void load(const T* row, const Cols<false>& c) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c.has(k)) a[k] = row[c.at(k)];
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = to_f(a[k]);
    }
};

template <typename T, bool VECTOR>
__device__ __forceinline__ void store(T* row, const Cols<VECTOR>& c, const float (&v)[8]) {
    if constexpr (!VECTOR) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c.has(k)) row[c.at(k)] = from_f<T>(v[k]);
    } else if (c.has(0)) {
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint4*>(row + c.first) = Vec<T>::pack(v);
        } else {
            reinterpret_cast<float4*>(row + c.first)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(row + c.first)[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
}

// Parameters of the thread's columns; `none` without an array.
template <bool VECTOR>
__device__ __forceinline__ void parameters(const void* p, bool bf16, const Cols<VECTOR>& c, float none,
                                           float (&v)[8]) {
    if (p == nullptr || !c.has(0)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = none;
    } else if constexpr (VECTOR) {
        if (bf16) {
            Vec<__nv_bfloat16>::unpack(
                __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + c.first)), v);
        } else {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + c.first);
            const float4 a = __ldg(q), b = __ldg(q + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c.has(k) ? load_any(p, bf16, c.at(k)) : none;
    }
}

// Warps that add up at most: those of the CTAs of a cluster, or of one CTA's teams.
constexpr int kSlots = kMaxCluster * kTeam / 32;

// Sums over a team, and over the cluster where that is larger.
struct Reducer {
    float2 (*slots)[kSlots];   // [2][CTAs x warps], from `base` on this team's
    int base, team, warp, warps, lane, parity, ctas, rank;

    template <int NV>
    __device__ __forceinline__ void sum(float (&v)[NV]) {
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] = warp_sum(v[k]);
        if (warps == 1 && ctas == 1) return;
        const float2 mine = make_float2(v[0], NV > 1 ? v[NV - 1] : 0.0f);
        float2* buf = slots[parity] + base;
        parity ^= 1;   // the other buffer is read until every thread is past the next barrier
        if (ctas == 1) {
            if (lane == 0) buf[warp] = mine;
            asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(warps * 32) : "memory");
        } else {
            cg::cluster_group cluster = cg::this_cluster();
            if (lane < ctas) cluster.map_shared_rank(buf, lane)[rank * warps + warp] = mine;
            cluster.sync();
        }
        float2 s = make_float2(0.0f, 0.0f);
        for (int i = lane; i < ctas * warps; i += 32) {
            const float2 p = buf[i];
            s.x += p.x;
            s.y += p.y;
        }
        v[0] = warp_sum(s.x);
        if (NV > 1) v[NV - 1] = warp_sum(s.y);
    }
};

// A thread's place: its team's rows and its columns.
template <bool VECTOR>
struct Place {
    Reducer R;
    Cols<VECTOR> cols;
    int t, team;
    int64_t index, count;   // of the team among all
    __device__ __forceinline__ Place(const Teams& G, int dim,
                                     float2 (*slots)[kSlots]) {
        team = threadIdx.x / G.threads;
        t = threadIdx.x - team * G.threads;
        cg::cluster_group cluster = cg::this_cluster();
        R.ctas = (int)cluster.num_blocks();
        R.rank = (int)cluster.block_rank();
        R.slots = slots;
        R.base = team * (G.threads >> 5);
        R.team = team;
        R.warp = t >> 5;
        R.warps = G.threads >> 5;
        R.lane = t & 31;
        R.parity = 0;
        const int c0 = R.rank * G.share;
        cols.end = min(dim, c0 + G.share);
        cols.first = c0 + (VECTOR ? 8 * t : t);
        cols.step = G.threads;
        index = (int64_t)(blockIdx.x / R.ctas) * G.teams + team;
        count = (int64_t)(gridDim.x / R.ctas) * G.teams;
    }
};

// Mean and 1 / deviation of a row (mean 0 without `layer`), the values with
// their mean removed in `c`; places outside of the row become 0.
template <bool VECTOR>
__device__ __forceinline__ float2 statistics(Reducer& R, const Cols<VECTOR>& cols, const float (&v)[8],
                                             float (&c)[8], bool layer, float inv, float eps) {
    float mean = 0.0f;
    if (layer) {
        float s[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < 8; ++k) s[0] += v[k];
        R.sum(s);
        mean = s[0] * inv;
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        c[k] = cols.has(k) ? v[k] - mean : 0.0f;
        q[0] = fmaf(c[k], c[k], q[0]);
    }
    R.sum(q);
    return make_float2(mean, 1.0f / sqrtf(fmaf(q[0], inv, eps)));
}

template <typename XT, typename HT, bool VECTOR>
__global__ void __launch_bounds__(kTeam, 2) norm_rows(const __grid_constant__ mdq_residual_norm_desc d,
                                                      const __grid_constant__ Teams G) {
    __shared__ float2 slots[2][kSlots];
    Place<VECTOR> P(G, (int)d.dim, slots);
    const Cols<VECTOR>& cols = P.cols;
    if (P.R.ctas > 1) cg::this_cluster().sync();   // all run before their memory is written to
    const bool layer = d.kind == MDQ_NORM_LAYER, pb = d.param_dtype == MDQ_BF16;
    const float inv = 1.0f / (float)d.dim;
    const XT* x = static_cast<const XT*>(d.x);
    const HT* h = static_cast<const HT*>(d.h);
    const int64_t per = d.rows / d.gate_rows;
    Raw<XT, VECTOR> nx;
    Raw<HT, VECTOR> nh;
    const auto fetch = [&](int64_t r) {
        nx.load(x + r * d.x_stride, cols);
        if (h != nullptr) nh.load(h + r * d.h_stride, cols);
    };
    if (P.index < d.rows) fetch(P.index);
    for (int64_t r = P.index; r < d.rows; r += P.count) {
        float v[8], c[8];
        float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const Raw<XT, VECTOR> rx = nx;
        const Raw<HT, VECTOR> rh = nh;
        if (r + P.count < d.rows) fetch(r + P.count);
        if (h != nullptr) {
            rh.get(v);
            const float2 s = statistics(P.R, cols, v, c, layer, inv, d.eps);
            st.x = s.x;
            st.y = s.y;
            float w[8];
            parameters(d.post_weight, pb, cols, 1.0f, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) c[k] *= s.y * w[k];
            if (d.post_bias != nullptr) {
                parameters(d.post_bias, pb, cols, 0.0f, w);
#pragma unroll
                for (int k = 0; k < 8; ++k) c[k] += w[k];
            }
            if (d.gate != nullptr) {
                const int64_t row = d.gate_rows == 1 ? 0 : r / per;
                parameters(static_cast<const char*>(d.gate) + row * d.dim * (pb ? 2 : 4), pb, cols, 1.0f, w);
#pragma unroll
                for (int k = 0; k < 8; ++k) c[k] *= w[k];
            }
            rx.get(v);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = fmaf(d.residual_scale, v[k], c[k]);
            store(static_cast<XT*>(d.x_new) + r * d.dim, cols, v);
        } else {
            rx.get(v);
        }
        if (d.n != nullptr) {
            const float2 s = statistics(P.R, cols, v, c, layer, inv, d.eps);
            st.z = s.x;
            st.w = s.y;
            float w[8], b[8];
            parameters(d.pre_weight, pb, cols, 1.0f, w);
            parameters(d.pre_bias, pb, cols, 0.0f, b);
#pragma unroll
            for (int k = 0; k < 8; ++k) c[k] = fmaf(c[k] * s.y, w[k], b[k]);
            store(static_cast<HT*>(d.n) + r * d.dim, cols, c);
        }
        if (d.stats != nullptr && P.t == 0 && P.R.rank == 0)
            reinterpret_cast<float4*>(d.stats)[r] = st;
    }
    if (P.R.ctas > 1) cg::this_cluster().sync();   // none ends while its memory may be written to
}

// ------------------------------------------------------------------ backward

// Sums of the rows of one CTA, [kinds][dim] each, and the gate's sums of runs
// that begin or end within a CTA's rows (GROUPED).
enum { kPre = 0, kPost = 1, kPreBias = 2, kPostBias = 3 };   // of dn xh, t hh (times the gate), dn, t

// Rows of the workspace: [block][4][dim], then (GROUPED) [team][2 edges][2][dim].
struct Partials {
    float* sums;
    float* edges;
};

// FULL: a mean is removed or a bias is there, so sums without the normalised
// value are needed as well.  GROUPED: the gate differs between rows; its sums
// leave the registers at the end of every group, weighted into the others.
template <typename XT, typename HT, bool VECTOR, bool FULL, bool GROUPED>
__global__ void __launch_bounds__(kTeam, 1) norm_grad_rows(const __grid_constant__
                                                           mdq_residual_norm_grad_desc g,
                                                           const __grid_constant__ Teams G,
                                                           const __grid_constant__ Partials W) {
    __shared__ float2 slots[2][kSlots];
    extern __shared__ float shared[];   // [2 or 4][share] where a CTA has several teams
    const mdq_residual_norm_desc& d = g.f;
    Place<VECTOR> P(G, (int)d.dim, slots);
    const Cols<VECTOR>& cols = P.cols;
    if (P.R.ctas > 1) cg::this_cluster().sync();
    const bool layer = FULL && d.kind == MDQ_NORM_LAYER, pb = d.param_dtype == MDQ_BF16;
    const float inv = 1.0f / (float)d.dim;
    const XT* x = static_cast<const XT*>(d.x);
    const HT* h = static_cast<const HT*>(d.h);
    const XT* gx = static_cast<const XT*>(g.grad_new);
    const HT* gn = static_cast<const HT*>(g.grad_n);
    const int64_t per = d.rows / d.gate_rows;
    const int64_t r0 = min(d.rows, P.index * G.run), r1 = min(d.rows, r0 + G.run);

    float pre[8] = {}, post[8] = {}, pre_b[FULL ? 8 : 1] = {}, post_b[FULL ? 8 : 1] = {};
    float all[GROUPED ? 8 : 1] = {}, all_b[GROUPED && FULL ? 8 : 1] = {};
    // fp32 rows fill the registers: they are not loaded ahead.
    constexpr bool kAhead = sizeof(XT) + sizeof(HT) <= 6;
    Raw<XT, VECTOR> nx, ngx;
    Raw<HT, VECTOR> nh, ngn;
    float4 nst = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto fetch = [&](int64_t r) {
        nx.load(x + r * d.x_stride, cols);
        if (h != nullptr) nh.load(h + r * d.h_stride, cols);
        if (gn != nullptr) ngn.load(gn + r * g.grad_n_stride, cols);
        if (gx != nullptr) ngx.load(gx + r * g.grad_new_stride, cols);
        nst = __ldg(reinterpret_cast<const float4*>(d.stats) + r);
    };
    if (kAhead && r0 < r1) fetch(r0);
    // The rows of every CTA of a cluster are the same, so all take part in its sums.
    for (int64_t r = r0; r < r1; ++r) {
        if (!kAhead) fetch(r);
        const Raw<XT, VECTOR> rx = nx, rgx = ngx;
        const Raw<HT, VECTOR> rh = nh, rgn = ngn;
        const float4 st = nst;
        if (kAhead && r + 1 < r1) fetch(r + 1);
        const void* gate = d.gate;
        if (GROUPED) gate = static_cast<const char*>(gate) + r / per * d.dim * (pb ? 2 : 4);

        float t[8], hh[8], w[8], v[8];
        if (h != nullptr) {
            rh.get(hh);
#pragma unroll
            for (int k = 0; k < 8; ++k) hh[k] = cols.has(k) ? (hh[k] - st.x) * st.y : 0.0f;
        }
        rgx.get(t);
        if (gn != nullptr) {
            // x_new and its normalised value, as the forward pass had them
            float xh[8], e[8];
            rx.get(xh);
            if (h != nullptr) {
                parameters(d.post_weight, pb, cols, 1.0f, w);
                parameters(FULL ? d.post_bias : nullptr, pb, cols, 0.0f, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = fmaf(hh[k], w[k], v[k]);
                parameters(gate, pb, cols, 1.0f, w);
#pragma unroll
                for (int k = 0; k < 8; ++k) xh[k] = fmaf(d.residual_scale, xh[k], v[k] * w[k]);
            }
            rgn.get(e);
            parameters(d.pre_weight, pb, cols, 1.0f, w);
            float s[FULL ? 2 : 1] = {};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                xh[k] = cols.has(k) ? (xh[k] - st.z) * st.w : 0.0f;
                pre[k] = fmaf(e[k], xh[k], pre[k]);
                if (FULL) pre_b[k] += e[k];
                e[k] *= w[k];
                s[0] = fmaf(e[k], xh[k], s[0]);
                if (FULL) s[FULL] += e[k];
            }
            P.R.sum(s);
            const float m1 = s[0] * inv, m0 = layer ? s[FULL] * inv : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = fmaf(st.w, e[k] - m0 - xh[k] * m1, t[k]);
        }
        if (h != nullptr) {
            parameters(gate, pb, cols, 1.0f, w);
            parameters(d.post_weight, pb, cols, 1.0f, v);
            float s[FULL ? 2 : 1] = {};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (!cols.has(k)) t[k] = 0.0f;
                post[k] = fmaf(t[k], hh[k], post[k]);
                if (FULL) post_b[k] += t[k];
                v[k] *= w[k] * t[k];   // u
                s[0] = fmaf(v[k], hh[k], s[0]);
                if (FULL) s[FULL] += v[k];
                t[k] *= d.residual_scale;
            }
            store(static_cast<XT*>(g.grad_x) + r * d.dim, cols, t);
            P.R.sum(s);
            const float u1 = s[0] * inv, u0 = layer ? s[FULL] * inv : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = st.y * (v[k] - u0 - hh[k] * u1);
            store(static_cast<HT*>(g.grad_h) + r * d.dim, cols, v);
        } else {
            store(static_cast<XT*>(g.grad_x) + r * d.dim, cols, t);
        }
        if constexpr (GROUPED) {
            if (r + 1 == r1 || (r + 1) % per == 0) {   // the group ends, or this team's part of it
                const int64_t k0 = r / per, first = k0 * per, last = first + per - 1;
                const bool whole = first >= r0 && last < r1;
                float* edge = W.edges + ((P.index * 2 + (first >= r0)) * 2) * d.dim;
                parameters(gate, pb, cols, 1.0f, w);
                float w1[8], b1[8];
                parameters(d.post_weight, pb, cols, 1.0f, w1);
                parameters(FULL ? d.post_bias : nullptr, pb, cols, 0.0f, b1);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    all[k] = fmaf(w[k], post[k], all[k]);
                    const float pb_k = FULL ? post_b[FULL ? k : 0] : 0.0f;
                    if (FULL) all_b[FULL ? k : 0] = fmaf(w[k], pb_k, all_b[FULL ? k : 0]);
                    if (cols.has(k)) {
                        if (whole) {
                            store_any(g.grad_gate, pb, k0 * d.dim + cols.at(k),
                                      fmaf(w1[k], post[k], b1[k] * pb_k));
                        } else {
                            edge[cols.at(k)] = post[k];
                            edge[d.dim + cols.at(k)] = pb_k;
                        }
                    }
                    post[k] = 0.0f;
                    if (FULL) post_b[FULL ? k : 0] = 0.0f;
                }
            }
        }
    }
    if constexpr (GROUPED) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            post[k] = all[k];
            if (FULL) post_b[FULL ? k : 0] = all_b[FULL ? k : 0];
        }
    }
    // The CTA's sums: its teams add theirs in turn.
    constexpr int kKinds = FULL ? 4 : 2;
    const int c0 = P.R.rank * G.share;
    float* out = W.sums + (int64_t)(blockIdx.x / P.R.ctas) * 4 * d.dim;
    for (int i = 0; i < G.teams; ++i) {
        if (i > 0) __syncthreads();
        if (P.team != i) continue;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (!cols.has(k)) continue;
            const float mine[4] = {pre[k], post[k], FULL ? pre_b[FULL ? k : 0] : 0.0f,
                                   FULL ? post_b[FULL ? k : 0] : 0.0f};
#pragma unroll
            for (int j = 0; j < kKinds; ++j) {
                float* s = shared + j * G.share + cols.at(k) - c0;
                const float v = i > 0 ? *s + mine[j] : mine[j];
                if (i + 1 < G.teams) *s = v;
                else out[j * d.dim + cols.at(k)] = v;
            }
        }
    }
    if (P.R.ctas > 1) cg::this_cluster().sync();
}

template <typename XT, typename HT>
cudaError_t run_forward(const mdq_residual_norm_desc& d, const Teams& G, int grid, int cluster,
                        bool vector, cudaStream_t stream) {
    const int threads = G.threads * G.teams;
    return vector ? launch(norm_rows<XT, HT, true>, dim3(grid), threads, 0, stream, cluster, false, d, G)
                  : launch(norm_rows<XT, HT, false>, dim3(grid), threads, 0, stream, cluster, false, d, G);
}

template <typename XT, typename HT, bool VECTOR>
cudaError_t run_backward(const mdq_residual_norm_grad_desc& g, const Teams& G, const Partials& W,
                         int grid, int cluster, bool full, bool grouped, cudaStream_t stream) {
    const int threads = G.threads * G.teams;
    const size_t smem = G.teams > 1 ? sizeof(float) * (full ? 4 : 2) * G.share : 0;
    typedef void (*Kernel)(const mdq_residual_norm_grad_desc, const Teams, const Partials);
    const Kernel k = full ? (grouped ? (Kernel)norm_grad_rows<XT, HT, VECTOR, true, true>
                                     : (Kernel)norm_grad_rows<XT, HT, VECTOR, true, false>)
                          : (grouped ? (Kernel)norm_grad_rows<XT, HT, VECTOR, false, true>
                                     : (Kernel)norm_grad_rows<XT, HT, VECTOR, false, false>);
    return launch(k, dim3(grid), threads, smem, stream, cluster, false, g, G, W);
}

#define MDQ_NORM_TYPES(DECL)                                                                       \
    DECL(float, float, ff) DECL(float, __nv_bfloat16, fb) DECL(__nv_bfloat16, __nv_bfloat16, bb)   \
        DECL(__nv_bfloat16, float, bf)
#define MDQ_NORM_DECLARE(XT, HT, S)                                                                \
    cudaError_t forward_##S(const mdq_residual_norm_desc&, const Teams&, int, int, bool,           \
                            cudaStream_t);                                                         \
    cudaError_t backward_##S(const mdq_residual_norm_grad_desc&, const Teams&, const Partials&,    \
                             int, int, bool, bool, bool, cudaStream_t);
MDQ_NORM_TYPES(MDQ_NORM_DECLARE)

// The kernels of one pair of types (x, h), in a file of its own.
#define MDQ_NORM_INSTANTIATE(XT, HT, S)                                                            \
    namespace mdq_norm {                                                                           \
    cudaError_t forward_##S(const mdq_residual_norm_desc& d, const Teams& G, int grid,             \
                            int cluster, bool vector, cudaStream_t stream) {                       \
        return run_forward<XT, HT>(d, G, grid, cluster, vector, stream);                           \
    }                                                                                              \
    cudaError_t backward_##S(const mdq_residual_norm_grad_desc& g, const Teams& G,                 \
                             const Partials& W, int grid, int cluster, bool vector, bool full,     \
                             bool grouped, cudaStream_t stream) {                                  \
        return vector                                                                              \
                   ? run_backward<XT, HT, true>(g, G, W, grid, cluster, full, grouped, stream)     \
                   : run_backward<XT, HT, false>(g, G, W, grid, cluster, full, grouped, stream);   \
    }                                                                                              \
    }

}  // namespace mdq_norm
