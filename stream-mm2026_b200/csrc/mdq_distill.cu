// mdq_distill.cu - distillation from a teacher's top logits: loss and gradient
// (mdq_ops.h).
#include "mdq_ops.cuh"

#include <cooperative_groups.h>
#include <math_constants.h>
#include <utility>

namespace {

using namespace mdq_ops;
namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 2^x, two ulp; results below the normal range become 0.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The largest exponent as a shift: 0 where there is none, so that exponents of
// -infinity stay -infinity.
__device__ __forceinline__ float finite_max(float h) { return h == -CUDART_INF_F ? 0.0f : h; }

// Softmax statistics: the largest exponent h = z c (rounded) and the sum of
// exp2(z c - h).  Sums are rescaled by the difference of the rounded exponents
// themselves, so that their rounding cancels.
struct Stat {
    float h, s;
};
__device__ __forceinline__ Stat merge(Stat a, Stat b) {
    const float h = fmaxf(a.h, b.h), k = finite_max(h);
    return {h, a.s * ex2(a.h - k) + b.s * ex2(b.h - k)};
}

// The teacher's entries of a row, in the block's shared memory.
struct Teacher {
    int* idx;       // [top] vocabulary index, -1 absent
    float* q;       // [top] probability
    float* lq;      // [top] its logarithm
    float* sum;     // [top] probabilities of all entries with this index; -1 if an earlier has it
    float* z;       // [top] the student's logits there (rank 0 only)
};

// ---------------------------------------------------------------- whole rows

// A row stays in the shared memory of a cluster of CTAs while its maximum, its
// sum and its gradient are formed, so the logits are read from memory once and
// the gradient is written once: the pass is bound by that traffic (two
// exponentials an element take about 0.7 of its time with bf16 logits).  Each
// CTA holds a slice of whole 16-byte units, brought by bulk copies in kStages
// parts so that the sum starts with the first; the CTAs' maxima and sums meet
// through distributed shared memory.  More CTAs a row where it does not fit in
// half an SM's shared memory, or where few rows would leave SMs idle.
constexpr int kStages = 4, kMaxCluster = 8;

struct RowShared {
    unsigned long long bar[kStages];
    Stat warp[kWarps];
    Stat cta[kMaxCluster];
    int live;
};

__device__ __forceinline__ unsigned smem_at(const void* p) {
    return (unsigned)__cvta_generic_to_shared(p);
}

// A copy of a few KB lands in microseconds; the limit (hundreds of
// milliseconds) only keeps a lost one from hanging the GPU.
__device__ __forceinline__ bool wait_copy(unsigned bar) {
    for (int i = 0; i < 1 << 22; ++i) {
        unsigned done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], 0;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(bar) : "memory");
        if (done) return true;
    }
    return false;
}

// 16 bytes of a slice that start `shift` bytes (4 words + half) behind unit u.
__device__ __forceinline__ uint4 shifted(const uint32_t* words, int at, bool half) {
    uint32_t w[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = k < 4 || half ? words[at + k] : 0u;
    if (!half) return make_uint4(w[0], w[1], w[2], w[3]);
    return make_uint4(__funnelshift_r(w[0], w[1], 16), __funnelshift_r(w[1], w[2], 16),
                      __funnelshift_r(w[2], w[3], 16), __funnelshift_r(w[3], w[4], 16));
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) distill_rows(const __grid_constant__
                                                            mdq_topk_distill_desc d,
                                                            int slice_units) {
    extern __shared__ __align__(16) char raw[];
    __shared__ RowShared S;
    constexpr int N = Vec<T>::N;   // elements of a unit
    T* slice = reinterpret_cast<T*>(raw);
    Teacher K;
    K.idx = reinterpret_cast<int*>(raw + 16 * (size_t)(slice_units + 1));
    K.q = reinterpret_cast<float*>(K.idx) + d.top;
    K.lq = K.q + d.top;
    K.sum = K.lq + d.top;
    K.z = K.sum + d.top;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
    const int64_t r = blockIdx.x / C;
    const T* z = static_cast<const T*>(d.logits) + r * d.logits_stride;
    T* out = d.grad == nullptr ? nullptr : static_cast<T*>(d.grad) + r * d.grad_stride;

    // Units of the row count from the 16-byte boundary at or before its start;
    // `lead` elements of the first precede the row.  This CTA's slice: units
    // [u0, u1), elements [e0, e1) of the row.
    const int lead = (int)(((uintptr_t)z & 15) / sizeof(T));
    const int64_t units = (lead + d.vocab + N - 1) / N;
    const int64_t u0 = min(units, (int64_t)rank * slice_units);
    const int64_t u1 = min(units, u0 + slice_units);
    const int64_t e0 = max((int64_t)0, u0 * N - lead), e1 = min(d.vocab, u1 * N - lead);
    const int n = (int)(u1 - u0);

    const float w = d.weight == nullptr ? 1.0f : d.weight[r];
    bool live = w != 0.0f;
    if (tid == 0) {
#pragma unroll
        for (int k = 0; k < kStages; ++k)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_at(&S.bar[k])) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // The others of the cluster run before their shared memory is written to.
    auto started = cluster.barrier_arrive();
    const int per = (n + kStages - 1) / kStages;   // units of a stage
    if (tid == 0 && live) {
        // Whole units inside the row by bulk copies; a unit that the row shares
        // with what lies before or behind it by elements, below.
        const int first = u0 == 0 && lead > 0 ? 1 : 0;
        const int last = u1 * N - lead > d.vocab ? n - 1 : n;
        unsigned long long policy;
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
#pragma unroll
        for (int k = 0; k < kStages; ++k) {
            const int a = max(first, k * per), b = min(last, (k + 1) * per);
            const unsigned bytes = b > a ? (unsigned)(b - a) * 16u : 0u, bar = smem_at(&S.bar[k]);
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                         : "memory");
            if (bytes > 0)
                asm volatile(
                    "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
                    " [%0], [%1], %2, [%3], %4;" ::"r"(smem_at(raw) + 16u * (unsigned)a),
                    "l"(z + (u0 + a) * N - lead), "r"(bytes), "r"(bar), "l"(policy)
                    : "memory");
        }
    }
    // The shared units' elements; -infinity outside of the row.
    if (live && n > 0) {
        if (tid < N && u0 == 0 && lead > 0)
            slice[tid] = tid >= lead && tid - lead < d.vocab ? z[tid - lead] : from_f<T>(-CUDART_INF_F);
        if (tid >= 32 && tid < 32 + N && u1 * N - lead > d.vocab && !(u0 == 0 && lead > 0 && n == 1)) {
            const int64_t e = (u1 - 1) * N - lead + tid - 32;
            slice[(n - 1) * N + tid - 32] = e < d.vocab ? z[e] : from_f<T>(-CUDART_INF_F);
        }
    }
    // The teacher's distribution, by the last warp.
    const float it = 1.0f / d.temperature, c = it * kLog2e;
    if (live && warp == (threads >> 5) - 1) {
        float tm = -CUDART_INF_F;
        for (int k = lane; k < d.top; k += 32) {
            const int64_t i = load_id(d.index, d.index_dtype == MDQ_I64, r * d.top + k);
            float t = load_any(d.teacher, d.teacher_dtype == MDQ_BF16, r * d.top + k);
            const bool in = i >= 0 && i < d.vocab;
            if (!in) t = -CUDART_INF_F;
            K.idx[k] = in ? (int)i : -1;
            K.lq[k] = t;
            if (rank == 0) K.z[k] = in ? to_f(z[i]) : 0.0f;
            tm = fmaxf(tm, t != t ? 0.0f : t);   // a NaN is an entry: the row becomes NaN
        }
        tm = warp_max(tm);
        float s = 0.0f;
        for (int k = lane; k < d.top; k += 32) {
            const float l = (K.lq[k] - tm) * it;
            K.lq[k] = l;
            s += K.q[k] = K.idx[k] < 0 ? 0.0f : expf(l);
        }
        s = warp_sum(s);
        const float ls = logf(s), is = 1.0f / s;
        for (int k = lane; k < d.top; k += 32) {
            K.q[k] *= is;
            K.lq[k] -= ls;
        }
        if (lane == 0) S.live = tm != -CUDART_INF_F;
    }
    __syncthreads();
    live = live && S.live != 0;
    // Entries that share an index: the first carries their sum.
    if (live && out != nullptr)
        for (int k = tid; k < d.top; k += threads) {
            const int i = K.idx[k];
            float sum = 0.0f;
            bool first = i >= 0;
            for (int j = 0; j < d.top; ++j)
                if (K.idx[j] == i) {
                    first = first && j >= k;
                    sum += K.q[j];
                }
            K.sum[k] = first ? sum : -1.0f;
        }

    // Maximum and sum of this thread's units, two at a time.
    Stat a = {-CUDART_INF_F, 0.0f};
    const uint4* units16 = reinterpret_cast<const uint4*>(raw);
    bool arrived = true;
    if (w != 0.0f)   // also where the teacher has nothing: the copies end in this CTA's time
        for (int k = 0; k < kStages; ++k) {
            arrived &= wait_copy(smem_at(&S.bar[k]));
            if (!live) continue;
            const int end = min(n, (k + 1) * per);
            for (int u = k * per + tid; u < end; u += 2 * threads) {
                float v[2 * N];
                Vec<T>::unpack(units16[u], *reinterpret_cast<float(*)[N]>(v));
                if (u + threads < end) {
                    Vec<T>::unpack(units16[u + threads], *reinterpret_cast<float(*)[N]>(v + N));
                } else {
#pragma unroll
                    for (int j = N; j < 2 * N; ++j) v[j] = -CUDART_INF_F;
                }
                float m = v[0];
#pragma unroll
                for (int j = 1; j < 2 * N; ++j) m = fmaxf(m, v[j]);
                const float h = fmaxf(a.h, __fmul_rn(m, c)), shift = finite_max(h);
                float s = a.s * ex2(a.h - shift);
#pragma unroll
                for (int j = 0; j < 2 * N; ++j) s += ex2(fmaf(v[j], c, -shift));
                a = {h, s};
            }
        }
    if (!arrived) a.s = CUDART_NAN_F;   // the row's results become NaN
    // All threads, all CTAs.
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        a = merge(a, {__shfl_xor_sync(0xffffffffu, a.h, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
    if (lane == 0) S.warp[warp] = a;
    cluster.barrier_wait(std::move(started));
    __syncthreads();
    if (warp == 0) {
        a = lane < threads >> 5 ? S.warp[lane] : Stat{-CUDART_INF_F, 0.0f};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            a = merge(a, {__shfl_xor_sync(0xffffffffu, a.h, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
        if (lane < C) *cluster.map_shared_rank(&S.cta[rank], lane) = a;
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
    a = S.cta[0];
    for (int k = 1; k < C; ++k) a = merge(a, S.cta[k]);
    const float shift = finite_max(a.h), scale = d.scale * w;

    if (rank == 0 && warp == 0 && d.row_loss != nullptr) {
        const float le = logf(a.s);
        float l = 0.0f;
        if (live)
            for (int k = lane; k < d.top; k += 32)
                if (K.q[k] != 0.0f) l += K.q[k] * (K.lq[k] - (fmaf(K.z[k], c, -shift) * kLn2 - le));
        l = warp_sum(l);
        if (lane == 0)
            d.row_loss[r] = live ? d.temperature * d.temperature * scale * l : 0.0f;
    }
    if (out == nullptr) return;

    const float up = d.upstream == nullptr ? 1.0f : d.upstream[r * d.upstream_stride];
    const float f = live ? up * scale * d.temperature : 0.0f, pe = live ? f / a.s : 0.0f;
    // Elements up to a 16-byte boundary of the gradient, whole units, the rest.
    const int64_t count = e1 - e0;
    if (count <= 0) return;
    T* to = out + e0;
    const int at0 = (int)(e0 - (u0 * N - lead));   // place of e0 in the slice
    const int head = (int)min(count, (int64_t)((-(uintptr_t)to & 15) / sizeof(T)));
    const int body = (int)((count - head) / N), tail = (int)(count - head) - body * N;
    const int from = at0 + head;                   // place of the first whole unit
    const auto edge = [&](int i) {
        to[i] = from_f<T>(live ? pe * ex2(fmaf(to_f(slice[at0 + i]), c, -shift)) : 0.0f);
    };
    if (tid < head) edge(tid);
    if (tid >= 32 && tid < 32 + tail) edge(head + body * N + tid - 32);
    uint4* to16 = reinterpret_cast<uint4*>(to + head);
    if (!live) {
        for (int u = tid; u < body; u += threads) __stcs(to16 + u, make_uint4(0, 0, 0, 0));
        return;
    }
    const auto unit = [&](uint4 x) {
        float v[N];
        Vec<T>::unpack(x, v);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = pe * ex2(fmaf(v[j], c, -shift));
        return Vec<T>::pack(v);
    };
    if (from % N == 0) {   // the gradient's units are the logits'
        const uint4* src = units16 + from / N;
#pragma unroll 2
        for (int u = tid; u < body; u += threads) __stcs(to16 + u, unit(src[u]));
    } else {
        const int byte = from * (int)sizeof(T);
        const uint32_t* words = reinterpret_cast<const uint32_t*>(raw) + byte / 4;
        const bool half = byte % 4 != 0;
        for (int u = tid; u < body; u += threads) __stcs(to16 + u, unit(shifted(words, 4 * u, half)));
    }
    __syncthreads();
    // The teacher's entries of this slice, over what was stored there.
    for (int k = tid; k < d.top; k += threads) {
        const int64_t i = K.idx[k];
        if (i < e0 || i >= e1 || K.sum[k] < 0.0f) continue;
        const float p = pe * ex2(fmaf(to_f(slice[at0 + (i - e0)]), c, -shift));
        out[i] = from_f<T>(p - f * K.sum[k]);
    }
}

// ----------------------------------------------------------------- long rows

// Rows that no cluster can hold: three passes over memory, one block a row.
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
__global__ void __launch_bounds__(kThreads) distill_long_rows(const __grid_constant__
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
    wait_previous();
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

template <typename T>
mdq_status run_rows(const mdq_topk_distill_desc& d, cudaStream_t stream) {
    // Bytes of shared memory beside the slice, and what a CTA may have: two CTAs
    // an SM, or one for the longest rows.
    const int64_t extra = 16 + 20 * (int64_t)d.top, half = 110 * 1024, whole = 222 * 1024;
    const int64_t units = ceil_div(d.vocab + Vec<T>::N - 1, Vec<T>::N);
    int cluster = 1;
    const auto bytes = [&] { return 16 * ceil_div(units, cluster); };
    while (cluster < kMaxCluster && bytes() + extra > half) cluster *= 2;
    if (bytes() + extra > whole) {
        distill_long_rows<T><<<(unsigned)d.rows, kThreads, 0, stream>>>(d);
        return launch_status("distill");
    }
    // Few rows: more CTAs a row while that fills idle SMs with 8 KB or more each.
    while (cluster < kMaxCluster && d.rows * cluster <= 74 && bytes() >= 16 * 1024) cluster *= 2;
    const int64_t grid = d.rows * cluster;
    if (grid > INT32_MAX) return mdq_fail(MDQ_ERR_TOO_LARGE, "distill: too many rows");
    const int threads = bytes() >= 16 * 1024 ? 512 : bytes() >= 4 * 1024 ? 256 : 128;
    return status_of(launch(distill_rows<T>, dim3((unsigned)grid), threads,
                            (size_t)(bytes() + extra), stream, cluster, false, d,
                            (int)(bytes() / 16)),
                     "distill");
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
        const mdq_status st = d->logits_dtype == MDQ_BF16 ? run_rows<__nv_bfloat16>(*d, stream)
                                                          : run_rows<float>(*d, stream);
        if (st != MDQ_OK) return st;
    }
    if (d->loss == nullptr) return MDQ_OK;
    return status_of(launch(distill_total, dim3(1), kThreads, 0, stream, 1, true,
                            static_cast<const float*>(d->row_loss), d->rows, d->loss),
                     "distill");
}
