// mdq_distill.cu - distillation from a teacher's top logits: loss and gradient
// (mdq_ops.h).
//
// Bound by memory when the logits are read once: a row stays in shared memory
// between its sum and its gradient.  Few rows are split over clusters
// (distill_cluster; 8 bf16 rows of 50257: 7.3 us), many go through persistent CTAs
// whose warps run their copies ahead (distill_stream; 16384 such rows with the
// gradient 605 us, 5.4 TB/s; 2048 fp32 rows of 32000, loss alone, 45 us, 5.8 TB/s).
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
// themselves, so that their rounding cancels.  c = log2(e) / T is rounded to fp32: a
// probability is off by about 1e-7 of itself times its exponent's distance from h.
struct Stat {
    float h, s;
};
__device__ __forceinline__ Stat merge(Stat a, Stat b) {
    const float h = fmaxf(a.h, b.h), k = finite_max(h);
    return {h, a.s * ex2(a.h - k) + b.s * ex2(b.h - k)};
}

// The teacher's entries of a row, in shared memory.
struct Teacher {
    int* idx;       // [top] vocabulary index, -1 absent
    float* q;       // [top] probability
    float* lq;      // [top] its logarithm
    float* sum;     // [top] probabilities of all entries with this index; -1 if an earlier has it
    float* z;       // [top] the student's logits there
    __device__ Teacher(char* p, int top) {
        idx = reinterpret_cast<int*>(p);
        q = reinterpret_cast<float*>(idx) + top;
        lq = q + top;
        sum = lq + top;
        z = sum + top;
    }
};
constexpr int kTeacherBytes = 20;   // of an entry

// Bits in which entries of a row mark their index, to find repeated ones.
constexpr int kMarkWords = 512;

// The entries of row r, by one warp: the teacher's distribution, the student's
// logits at the entries (with `gather`), and for each index its first entry
// with the sum of the probabilities of all that share it (with `sums`).
// Returns whether the teacher has an entry.
template <typename T>
__device__ __forceinline__ bool teacher_row(const mdq_topk_distill_desc& d, int64_t r, const T* z,
                                            const Teacher& K, bool gather, bool sums,
                                            unsigned* marks, int lane) {
    const float it = 1.0f / d.temperature;
    const bool i64 = d.index_dtype == MDQ_I64, bf16 = d.teacher_dtype == MDQ_BF16;
    const auto entry = [&](int k, int& i, float& t) {
        const int64_t v = load_id(d.index, i64, r * d.top + k);
        t = load_any(d.teacher, bf16, r * d.top + k);
        const bool in = v >= 0 && v < d.vocab;
        if (!in) t = -CUDART_INF_F;
        i = in ? (int)v : -1;
    };
    // A NaN is an entry: the row becomes NaN.
    const auto larger = [](float m, float t) { return fmaxf(m, t != t ? 0.0f : t); };
    if (d.top <= 32) {   // an entry a lane
        int i = -1;
        float t = -CUDART_INF_F, zi = 0.0f;
        if (lane < d.top) entry(lane, i, t);
        if (gather && i >= 0) zi = to_f(z[i]);
        const float tm = warp_max(larger(-CUDART_INF_F, t));
        if (tm == -CUDART_INF_F) return false;
        const float l = (t - tm) * it, e = i < 0 ? 0.0f : expf(l), s = warp_sum(e);
        const float q = e * (1.0f / s);
        float sum = q;
        const unsigned same = __match_any_sync(0xffffffffu, i);
        for (unsigned others = same & (same - 1); __any_sync(0xffffffffu, others != 0);
             others &= others - 1) {   // those behind the first, in order
            const float more = __shfl_sync(0xffffffffu, q, others != 0 ? __ffs(others) - 1 : lane);
            if (others != 0) sum += more;
        }
        if (lane < d.top) {
            K.idx[lane] = i;
            K.q[lane] = q;
            K.lq[lane] = l - logf(s);
            K.sum[lane] = i >= 0 && (same & ((1u << lane) - 1)) == 0 ? sum : -1.0f;
            K.z[lane] = zi;
        }
        return true;
    }
    float tm = -CUDART_INF_F;
    for (int k = lane; k < d.top; k += 32) {
        int i;
        float t;
        entry(k, i, t);
        K.idx[k] = i;
        K.lq[k] = t;
        tm = larger(tm, t);
    }
    tm = warp_max(tm);
    if (tm == -CUDART_INF_F) return false;
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
    if (gather) {
#pragma unroll 4
        for (int k = lane; k < d.top; k += 32) K.z[k] = K.idx[k] < 0 ? 0.0f : to_f(z[K.idx[k]]);
    }
    if (sums) {
        // Entries that find their index's bit set share it with another, or only
        // the bit: for those the whole list is looked through.
        for (int k = lane; k < kMarkWords; k += 32) marks[k] = 0;
        __syncwarp();
        for (int k0 = 0; k0 < d.top; k0 += 32) {
            const int k = k0 + lane, i = k < d.top ? K.idx[k] : -1;
            bool maybe = false;
            if (i >= 0) {
                const unsigned h = (unsigned)i * 2654435761u >> 18;   // 14 bits
                maybe = atomicOr(&marks[h >> 5], 1u << (h & 31)) >> (h & 31) & 1;
            }
            if (k < d.top) K.sum[k] = i >= 0 ? K.q[k] : -1.0f;
            __syncwarp();
            for (unsigned m = __ballot_sync(0xffffffffu, maybe); m != 0; m &= m - 1) {
                const int same = __shfl_sync(0xffffffffu, i, __ffs(m) - 1);
                float sum = 0.0f;
                int first = d.top;
                for (int j = lane; j < min(d.top, k0 + 32); j += 32)
                    if (K.idx[j] == same) {
                        first = min(first, j);
                        sum += K.q[j];
                    }
                sum = warp_sum(sum);
                first = __reduce_min_sync(0xffffffffu, first);
                for (int j = lane; j < min(d.top, k0 + 32); j += 32)
                    if (K.idx[j] == same) K.sum[j] = j == first ? sum : -1.0f;
                __syncwarp();
            }
        }
    }
    return true;
}

// 2^(v c - shift) of a unit's elements, two products an instruction.
template <int N>
__device__ __forceinline__ void exponentials(float (&v)[N], float c, float shift) {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        asm("{\n\t.reg .b64 a, b, d;\n\t"
            "mov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 d, {%3, %3};\n\t"
            "fma.rn.f32x2 a, a, b, d;\n\tmov.b64 {%0, %1}, a;\n\t}"
            : "+f"(v[j]), "+f"(v[j + 1]) : "f"(c), "f"(-shift));
        v[j] = ex2(v[j]);
        v[j + 1] = ex2(v[j + 1]);
    }
}
template <int N>
__device__ __forceinline__ float largest(const float (&v)[N]) {
    float m[N / 4];
#pragma unroll
    for (int j = 0; j < N / 4; ++j)
        m[j] = fmaxf(fmaxf(v[4 * j], v[4 * j + 1]), fmaxf(v[4 * j + 2], v[4 * j + 3]));
#pragma unroll
    for (int j = 1; j < N / 4; ++j) m[0] = fmaxf(m[0], m[j]);
    return m[0];
}
template <int N>
__device__ __forceinline__ float total(const float (&v)[N]) {
    float s[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int j = 4; j < N; ++j) s[j & 3] += v[j];
    return (s[0] + s[1]) + (s[2] + s[3]);
}
template <int N>
__device__ __forceinline__ void add_values(Stat& a, float (&v)[N], float c) {
    const float h = fmaxf(a.h, __fmul_rn(largest(v), c)), shift = finite_max(h);
    exponentials(v, c, shift);
    a = {h, fmaf(a.s, ex2(a.h - shift), total(v))};
}

// Adds units first, first + threads, ... below end, four at a time.
template <typename T>
__device__ __forceinline__ void add_units(Stat& a, const uint4* units, int first, int end,
                                          int threads, float c) {
    constexpr int N = Vec<T>::N;
    int u = first;
    for (; u + 3 * threads < end; u += 4 * threads) {
        float v[4 * N];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            Vec<T>::unpack(units[u + j * threads], *reinterpret_cast<float(*)[N]>(v + j * N));
        add_values(a, v, c);
    }
    for (; u + threads < end; u += 2 * threads) {
        float v[2 * N];
        Vec<T>::unpack(units[u], *reinterpret_cast<float(*)[N]>(v));
        Vec<T>::unpack(units[u + threads], *reinterpret_cast<float(*)[N]>(v + N));
        add_values(a, v, c);
    }
    if (u < end) {
        float v[N];
        Vec<T>::unpack(units[u], v);
        add_values(a, v, c);
    }
}

__device__ __forceinline__ Stat merge_warp(Stat a) {
    float h = a.h;
    asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(h));
    return {h, warp_sum(a.s * ex2(a.h - finite_max(h)))};
}

// The loss of a row, by one warp.
__device__ __forceinline__ float row_loss(const Teacher& K, int top, Stat a, float c, int lane) {
    const float le = logf(a.s), shift = finite_max(a.h);
    float l = 0.0f;
    for (int k = lane; k < top; k += 32)
        if (K.q[k] != 0.0f) l += K.q[k] * (K.lq[k] - (fmaf(K.z[k], c, -shift) * kLn2 - le));
    return warp_sum(l);
}

// 16 bytes of shared memory from word `at` on, or from half a word behind it.
__device__ __forceinline__ uint4 shifted(const uint32_t* words, int at, bool half) {
    uint32_t w[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = k < 4 || half ? words[at + k] : 0u;
    if (!half) return make_uint4(w[0], w[1], w[2], w[3]);
    return make_uint4(__funnelshift_r(w[0], w[1], 16), __funnelshift_r(w[1], w[2], 16),
                      __funnelshift_r(w[2], w[3], 16), __funnelshift_r(w[3], w[4], 16));
}

// The softmax's part of the gradient, pe exp2(z c - shift), of `count` elements
// that lie in `part` from element at0 on: elements up to a 16-byte boundary of
// the gradient, whole units, the rest.  Where the boundaries of the gradient
// are not those of the logits, a unit is put together from two.
template <typename T>
__device__ __forceinline__ void write_part(T* to, const char* part, int at0, int count, float pe,
                                           float c, float shift, int tid, int threads) {
    constexpr int N = Vec<T>::N;
    const int head = min(count, (int)((-(uintptr_t)to & 15) / sizeof(T)));
    const int body = (count - head) / N, tail = count - head - body * N;
    const int from = at0 + head;   // place of the first whole unit
    const T* src = reinterpret_cast<const T*>(part) + at0;
    const auto edge = [&](int i) { to[i] = from_f<T>(pe * ex2(fmaf(to_f(src[i]), c, -shift))); };
    if (tid < head) edge(tid);
    if (tid >= 16 && tid < 16 + tail) edge(head + body * N + tid - 16);
    uint4* to16 = reinterpret_cast<uint4*>(to + head);
    const auto unit = [&](uint4 x) {
        float v[N];
        Vec<T>::unpack(x, v);
        exponentials(v, c, shift);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] *= pe;
        return Vec<T>::pack(v);
    };
    if (from % N == 0) {
        const uint4* units = reinterpret_cast<const uint4*>(part) + from / N;
#pragma unroll 2
        for (int u = tid; u < body; u += threads) __stcs(to16 + u, unit(units[u]));
    } else {
        const int byte = from * (int)sizeof(T);
        const uint32_t* words = reinterpret_cast<const uint32_t*>(part) + byte / 4;
        const bool half = byte % 4 != 0;
        for (int u = tid; u < body; u += threads) __stcs(to16 + u, unit(shifted(words, 4 * u, half)));
    }
}

template <typename T>
__device__ __forceinline__ void write_zeros(T* to, int64_t count, int tid, int threads) {
    const int head = (int)min(count, (int64_t)((-(uintptr_t)to & 15) / sizeof(T)));
    const int64_t body = (count - head) / Vec<T>::N;
    const int tail = (int)(count - head - body * Vec<T>::N);
    if (tid < head) to[tid] = from_f<T>(0.0f);
    if (tid >= 16 && tid < 16 + tail) to[head + body * Vec<T>::N + tid - 16] = from_f<T>(0.0f);
    for (int64_t u = tid; u < body; u += threads)
        __stcs(reinterpret_cast<uint4*>(to + head) + u, make_uint4(0, 0, 0, 0));
}

// The 16-byte units a row of logits lies in, counted from the boundary at or
// before its start; `lead` elements of the first precede the row.
template <typename T>
struct RowUnits {
    static constexpr int N = Vec<T>::N;
    const T* z;
    int64_t vocab, units;
    int lead;
    __device__ RowUnits(const mdq_topk_distill_desc& d, int64_t r)
        : z(static_cast<const T*>(d.logits) + r * d.logits_stride), vocab(d.vocab) {
        lead = (int)(((uintptr_t)z & 15) / sizeof(T));
        units = (lead + vocab + N - 1) / N;
    }
    // First element of unit u (negative for the first), and those of a part.
    __device__ int64_t element(int64_t u) const { return u * N - lead; }
    __device__ int64_t begin(int64_t u0) const { return max((int64_t)0, element(u0)); }
    __device__ int64_t end(int64_t u1) const { return min(vocab, element(u1)); }
    // Whether the unit holds elements that are not the row's: those are not
    // copied in bulk but element by element.
    __device__ bool shared(int64_t u) const {
        return (u == 0 && lead > 0) || element(u + 1) > vocab;
    }
    // The value in place t of unit u, -infinity outside of the row.
    __device__ T value(int64_t u, int t) const {
        const int64_t e = element(u) + t;
        return e >= 0 && e < vocab ? z[e] : from_f<T>(-CUDART_INF_F);
    }
};

// ------------------------------------------------------------------ few rows

// A row stays in the shared memory of a cluster of CTAs, a slice each, so that
// few rows use many SMs.  Bulk copies bring a slice in kParts parts and the sum
// starts with the first; the CTAs' statistics meet through distributed shared
// memory.
constexpr int kParts = 4, kMaxCluster = 8;

struct RowShared {
    unsigned long long bar[kParts];
    Stat warp[kWarps];
    Stat cta[kMaxCluster];
    unsigned marks[kMarkWords];
    int live;
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) distill_cluster(const __grid_constant__
                                                               mdq_topk_distill_desc d,
                                                               int slice_units) {
    extern __shared__ __align__(16) char raw[];
    __shared__ RowShared S;
    constexpr int N = Vec<T>::N;   // elements of a unit
    T* slice = reinterpret_cast<T*>(raw);
    const Teacher K(raw + 16 * (size_t)(slice_units + 1), d.top);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
    const int64_t r = blockIdx.x / C;
    const RowUnits<T> row(d, r);
    T* out = d.grad == nullptr ? nullptr : static_cast<T*>(d.grad) + r * d.grad_stride;
    // This CTA's slice: units [u0, u1).
    const int64_t u0 = min(row.units, (int64_t)rank * slice_units);
    const int64_t u1 = min(row.units, u0 + slice_units);
    const int n = (int)(u1 - u0);

    const float w = d.weight == nullptr ? 1.0f : d.weight[r];
    bool live = w != 0.0f;
    if (tid == 0) {
#pragma unroll
        for (int k = 0; k < kParts; ++k) bar_init(&S.bar[k], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // The others of the cluster run before their shared memory is written to.
    auto started = cluster.barrier_arrive();
    const int per = (n + kParts - 1) / kParts;   // units of a part
    const bool first_shared = n > 0 && row.shared(u0), last_shared = n > 0 && row.shared(u1 - 1);
    if (tid == 0 && live) {
        const unsigned long long policy = read_once();
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            const int a = max(first_shared ? 1 : 0, k * per), b = min(last_shared ? n - 1 : n, (k + 1) * per);
            copy_in(&S.bar[k], raw + 16 * (size_t)a, row.z + row.element(u0 + a),
                    b > a ? (unsigned)(b - a) * 16u : 0u, policy);
        }
    }
    if (live && first_shared && tid < N) slice[tid] = row.value(u0, tid);
    if (live && last_shared && tid >= 32 && tid < 32 + N)
        slice[(n - 1) * N + tid - 32] = row.value(u1 - 1, tid - 32);
    const float c = 1.0f / d.temperature * kLog2e;
    if (live && warp == (threads >> 5) - 1) {   // the teacher, by the last warp
        const bool has = teacher_row(d, r, row.z, K, rank == 0, out != nullptr, S.marks, lane);
        if (lane == 0) S.live = has;
    }
    __syncthreads();
    live = live && S.live != 0;

    Stat a = {-CUDART_INF_F, 0.0f};
    const uint4* units = reinterpret_cast<const uint4*>(raw);
    bool arrived = true;
    if (w != 0.0f)   // also where the teacher has nothing: the copies end in this CTA's time
        for (int k = 0; k < kParts; ++k) {
            arrived &= bar_wait(&S.bar[k], 0);
            if (live) add_units<T>(a, units, k * per + tid, min(n, (k + 1) * per), threads, c);
        }
    if (!arrived) {   // the row's results become NaN; copies still on their way end in this CTA's time
        a.s = CUDART_NAN_F;
        for (int k = 0; k < kParts; ++k) (void)bar_wait(&S.bar[k], 0);
    }
    // All threads, all CTAs.
    a = merge_warp(a);
    if (lane == 0) S.warp[warp] = a;
    cluster.barrier_wait(std::move(started));
    __syncthreads();
    if (warp == 0) {
        a = merge_warp(lane < threads >> 5 ? S.warp[lane] : Stat{-CUDART_INF_F, 0.0f});
        if (lane < C) *cluster.map_shared_rank(&S.cta[rank], lane) = a;
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
    a = S.cta[0];
    for (int k = 1; k < C; ++k) a = merge(a, S.cta[k]);

    const float scale = d.scale * w;
    if (rank == 0 && warp == 0 && d.row_loss != nullptr) {
        const float l = live ? d.temperature * d.temperature * scale * row_loss(K, d.top, a, c, lane)
                             : 0.0f;
        if (lane == 0) d.row_loss[r] = l;
    }
    const int64_t e0 = row.begin(u0), e1 = row.end(u1);
    if (out == nullptr || e1 <= e0) return;
    if (!live) return write_zeros(out + e0, e1 - e0, tid, threads);
    const float up = d.upstream == nullptr ? 1.0f : d.upstream[r * d.upstream_stride];
    const float f = up * scale * d.temperature, pe = f / a.s, shift = finite_max(a.h);
    const int at0 = (int)(e0 - row.element(u0));   // place of e0 in the slice
    write_part(out + e0, raw, at0, (int)(e1 - e0), pe, c, shift, tid, threads);
    __syncthreads();
    // The teacher's entries of this slice, over what was stored there.
    for (int k = tid; k < d.top; k += threads) {
        const int64_t i = K.idx[k];
        if (i < e0 || i >= e1 || K.sum[k] < 0.0f) continue;
        const float p = pe * ex2(fmaf(to_f(slice[at0 + (i - e0)]), c, -shift));
        out[i] = from_f<T>(p - f * K.sum[k]);
    }
}

// ----------------------------------------------------------------- many rows

// Persistent CTAs.  Rows go to them in turn; where rows have weights, those of
// weight 0 (which cost a third of the others') go round separately, so that
// every CTA gets its share of both.  The whole 16-byte units of a row are divided among the warps; every warp brings its slice of the next rows
// in pieces through a ring of its own in shared memory and refills a piece as
// soon as it is done with it, so that copies run ahead without the warps
// waiting for one another.  They meet once a row, when their maxima and sums
// are joined.  The last `stages` pieces of a slice stay in the ring until the
// gradient has been formed from them; pieces of a slice that is longer are
// brought a second time, from L2 as a rule.  With the loss alone, pieces are
// refilled at once.  One more warp looks up the teacher's entries some rows
// ahead and forms the rows' losses behind.
struct StreamPlan {
    int warps;         // that share a row
    int each;          // 16-byte units of a warp's slice
    int piece_units;   // 16-byte units of a piece
    int stages;        // pieces of a warp's ring
    int depth;         // rows whose entries are kept
    int listed;        // places of a CTA's list of rows; 0: every gridDim-th row
};
constexpr int kMaxStages = 8, kMaxDepth = 4;

// A wait of a whole warp.
[[nodiscard]] __device__ __forceinline__ bool warp_wait(void* bar, unsigned parity) {
    return __all_sync(0xffffffffu, bar_wait(bar, parity));
}

// A place in a ring: its stage, and the phase its barriers are in.
struct Place {
    int stage = 0;
    unsigned phase = 0;
    __device__ __forceinline__ void next(int stages) {
        if (++stage == stages) {
            stage = 0;
            phase ^= 1;
        }
    }
};

struct StreamShared {
    unsigned long long full[kWarps][kMaxStages];
    unsigned long long told[kMaxDepth], heard[kMaxDepth];   // entries are there, are done with
    int live[kMaxDepth];
    Stat stat[kMaxDepth];
    Stat warp[2][kWarps];
    unsigned marks[kMarkWords];
    int part[kWarps + 1];
};

__device__ __forceinline__ float row_weight(const mdq_topk_distill_desc& d, int64_t r) {
    return d.weight == nullptr ? 1.0f : __ldg(d.weight + r);
}

// The rows of this CTA: `live` of weight other than 0, then `dead` of weight 0.
struct Rows {
    const int* list;   // nullptr: every gridDim-th
    int64_t live, dead;
    __device__ __forceinline__ int64_t at(int64_t i) const {
        return list == nullptr ? blockIdx.x + i * gridDim.x : list[i];
    }
};

// Fills the list: row r is the k-th of its kind, by the kinds of the rows before
// it, and belongs to CTA k mod gridDim.  Every CTA counts for itself: the
// weights come from L2.
__device__ __forceinline__ Rows find_rows(const mdq_topk_distill_desc& d, int places, int* list,
                                          int* part) {
    if (places == 0) {
        const int64_t b = blockIdx.x;
        return {nullptr, (d.rows - b + gridDim.x - 1) / gridDim.x, 0};
    }
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int rows = (int)d.rows, each = (rows + blockDim.x - 1) / blockDim.x;
    const int r0 = min(rows, tid * each), r1 = min(rows, r0 + each);
    int mine = 0;
#pragma unroll 4
    for (int r = r0; r < r1; ++r) mine += __ldg(d.weight + r) != 0.0f;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) part[warp] = upto;
    __syncthreads();
    int before = upto - mine, all = 0;
    for (int k = 0; k < warps; ++k) {
        if (k < warp) before += part[k];
        all += part[k];
    }
    const int G = gridDim.x, b = blockIdx.x;
    const int live = all > b ? (all - b + G - 1) / G : 0;
    const int dead = rows - all > b ? (rows - all - b + G - 1) / G : 0;
    int k = before, z = r0 - before;   // places of this thread's next rows, live and dead
    int km = k % G, zm = z % G;
    for (int r = r0; r < r1; ++r) {
        if (__ldg(d.weight + r) != 0.0f) {
            if (km == b) list[k / G] = r;
            ++k;
            if (++km == G) km = 0;
        } else {
            if (zm == b) list[live + z / G] = r;
            ++z;
            if (++zm == G) zm = 0;
        }
    }
    __syncthreads();
    return {list, live, dead};
}

// A row as the warps share it: `head` elements up to the first 16-byte
// boundary, whole units, `tail` elements; warp w has `mine` units from `from` on.
template <typename T>
struct Share {
    static constexpr unsigned N = Vec<T>::N;
    const T* z;
    int head, tail, mine, from;
    __device__ __forceinline__ Share(const mdq_topk_distill_desc& d, const T* row, int first, int each)
        : z(row) {   // first: the warp's first unit
        const unsigned vocab = (unsigned)d.vocab;
        head = (int)min(vocab, (unsigned)(-(uintptr_t)z & 15) / (unsigned)sizeof(T));
        const unsigned rest = vocab - head, units = rest / N;
        tail = (int)(rest % N);
        mine = max(0, min((int)units - first, each));
        from = head + first * (int)N;
    }
};

// The entries' warp.
template <typename T>
__device__ __forceinline__ void stream_entries(const mdq_topk_distill_desc& d, const StreamPlan& P,
                                               StreamShared& S, const Rows& R, char* info,
                                               int lane) {
    const float c = 1.0f / d.temperature * kLog2e;
    Place slots;
    // The loss of row i, whose entries are in the slot, once the others are done.  If
    // they do not come, this warp ends (theirs do after a wait for their next entries),
    // and the losses from here on are NaN.
    const auto finish = [&](int slot, int64_t i, unsigned phase) {
        const bool done = warp_wait(&S.heard[slot], phase);
        if (d.row_loss == nullptr) return done;
        if (!done) {
            for (i += lane; i < R.live; i += 32) d.row_loss[R.at(i)] = CUDART_NAN_F;
            return false;
        }
        const int64_t r = R.at(i);
        const Teacher K(info + (size_t)slot * kTeacherBytes * d.top, d.top);
        float l = 0.0f;
        if (S.live[slot])
            l = d.temperature * d.temperature * d.scale * row_weight(d, r) *
                row_loss(K, d.top, S.stat[slot], c, lane);
        if (lane == 0) d.row_loss[r] = l;
        __syncwarp();
        return true;
    };
    if (d.row_loss != nullptr)
        for (int64_t i = lane; i < R.dead; i += 32) d.row_loss[R.at(R.live + i)] = 0.0f;
    for (int64_t i = 0; i < R.live; ++i) {
        const int64_t r = R.at(i);
        const int slot = slots.stage;
        if (i >= P.depth && !finish(slot, i - P.depth, slots.phase ^ 1)) return;
        const Teacher K(info + (size_t)slot * kTeacherBytes * d.top, d.top);
        const T* z = static_cast<const T*>(d.logits) + r * d.logits_stride;
        const bool live = row_weight(d, r) != 0.0f &&
                          teacher_row(d, r, z, K, true, d.grad != nullptr, S.marks, lane);
        if (lane == 0) S.live[slot] = live;
        __syncwarp();
        if (lane == 0) bar_arrive(&S.told[slot]);
        slots.next(P.depth);
    }
    if (d.row_loss == nullptr) return;
    if (R.live < P.depth) slots = {0, 1};
    for (int64_t i = max((int64_t)0, R.live - P.depth); i < R.live; ++i, slots.next(P.depth))
        if (!finish(slots.stage, i, slots.phase ^ 1)) return;
}

template <typename T>
__global__ void __launch_bounds__(kThreads + 32, 1) distill_stream(const __grid_constant__
                                                                   mdq_topk_distill_desc d,
                                                                   const __grid_constant__ StreamPlan P) {
    extern __shared__ __align__(16) char raw[];
    __shared__ StreamShared S;
    constexpr int N = Vec<T>::N;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, W = P.warps;
    const size_t piece_bytes = 16 * (size_t)P.piece_units, ring_bytes = piece_bytes * P.stages;
    char* ring = raw + warp * ring_bytes;
    char* info = raw + W * ring_bytes + 16;
    if (tid == 0) {
        for (int k = 0; k < W; ++k)
            for (int j = 0; j < P.stages; ++j) bar_init(&S.full[k][j], 1);
        for (int k = 0; k < P.depth; ++k) {
            bar_init(&S.told[k], 1);
            bar_init(&S.heard[k], W);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const Rows R = find_rows(d, P.listed,
                             reinterpret_cast<int*>(info + (size_t)P.depth * kTeacherBytes * d.top),
                             S.part);
    if (warp == W) return stream_entries<T>(d, P, S, R, info, lane);

    const float c = 1.0f / d.temperature * kLog2e;
    const bool want = d.grad != nullptr;
    // Pieces of this warp's slice: a row has one of two numbers of units, by
    // where it starts.
    const int first = warp * P.each, full_units = (int)(d.vocab / N);
    const auto mine_of = [&](int units) { return max(0, min(units - first, P.each)); };
    const int most = mine_of(full_units);
    const int most_pieces = (most + P.piece_units - 1) / P.piece_units;
    const int less_pieces = (mine_of(full_units - 1) + P.piece_units - 1) / P.piece_units;
    const auto pieces_of = [&](int units) { return units == most ? most_pieces : less_pieces; };
    const T* logits = static_cast<const T*>(d.logits);
    const unsigned long long policy = read_once();

    // Copies: piece ik of `loads` of the row before the inext-th, to the place `to`.
    const T* iz = nullptr;
    int64_t inext = 0;
    int ik = 0, loads = 0, in = 0, iunits = 0;
    Place to;
    // A wait of this warp ran out: it waits for nothing and copies nothing from then
    // on, what it has to write becomes NaN, and through its sums all of the rows do.
    bool lost = false;
    const auto copy_next = [&] {
        if (lost) return;
        while (ik == loads) {
            if (inext == R.live) return;
            const Share<T> s(d, logits + R.at(inext) * d.logits_stride, first, P.each);
            iz = s.z + s.from;
            iunits = s.mine;
            in = pieces_of(s.mine);
            loads = in + (want && in > P.stages ? in - P.stages : 0);
            ik = 0;
            ++inext;
        }
        const int piece = ik < in ? ik : ik - in;
        const int u = piece * P.piece_units, n = min(P.piece_units, iunits - u);
        // The warp has read the piece that was here: the values went into results
        // before the __syncwarp() ahead of this call.
        if (lane == 0)
            copy_in(&S.full[warp][to.stage], ring + to.stage * piece_bytes, iz + (int64_t)u * N,
                    16u * (unsigned)n, policy);
        ++ik;
        to.next(P.stages);
    };
    for (int k = 0; k < P.stages; ++k) copy_next();

    Place at, slots;
    int parity = 0;
    if (want)   // while the first copies are on their way
        for (int64_t i = 0; i < R.dead; ++i)
            write_zeros(static_cast<T*>(d.grad) + R.at(R.live + i) * d.grad_stride, d.vocab, tid, 32 * W);
    for (int64_t i = 0; i < R.live; ++i) {
        const int64_t r = R.at(i);
        const float w = row_weight(d, r);   // used behind the sum
        T* out = want ? static_cast<T*>(d.grad) + r * d.grad_stride : nullptr;
        const Share<T> s(d, logits + r * d.logits_stride, first, P.each);
        // The elements outside of whole units, by the first warp.
        const bool edge = warp == 0 && (lane < s.head || (lane >= 16 && lane < 16 + s.tail));
        const int64_t edge_at = lane < s.head ? lane : d.vocab - s.tail + lane - 16;
        float edge_value = -CUDART_INF_F;
        if (edge) edge_value = to_f(s.z[edge_at]);

        // ---- maximum and sum
        const int n = pieces_of(s.mine), keep = want ? min(n, P.stages) : 0;
        const Place begin = at;
        Stat a = {-CUDART_INF_F, 0.0f};
        for (int k = 0; k < n && !lost; ++k, at.next(P.stages)) {
            if (!warp_wait(&S.full[warp][at.stage], at.phase)) {
                lost = true;
                break;
            }
            add_units<T>(a, reinterpret_cast<const uint4*>(ring + at.stage * piece_bytes), lane,
                         min(P.piece_units, s.mine - k * P.piece_units), 32, c);
            if (k < n - keep) {
                __syncwarp();
                copy_next();
            }
        }
        if (edge) {
            const float h = __fmul_rn(edge_value, c);
            a = merge(a, {h, ex2(fmaf(edge_value, c, -finite_max(h)))});
        }
        const int slot = slots.stage;
        if (!lost && !warp_wait(&S.told[slot], slots.phase)) lost = true;
        if (lost) a.s = CUDART_NAN_F;
        a = merge_warp(a);
        if (lane == 0) S.warp[parity][warp] = a;
        asm volatile("bar.sync 1, %0;" ::"r"(32 * W) : "memory");
        a = merge_warp(lane < W ? S.warp[parity][lane] : Stat{-CUDART_INF_F, 0.0f});
        if (tid == 0) S.stat[slot] = a;
        parity ^= 1;

        if (want) {
            // ---- gradient: the pieces in the ring, then those brought again
            const bool live = !lost && S.live[slot] != 0;
            const float up = d.upstream == nullptr ? 1.0f : __ldg(d.upstream + r * d.upstream_stride);
            const float f = up * d.scale * w * d.temperature, pe = __fdividef(f, a.s);
            const float shift = finite_max(a.h);
            // The teacher's entries of this slice (the first of them, or all).
            const Teacher K(info + (size_t)slot * kTeacherBytes * d.top, d.top);
            const int end = s.from + s.mine * N;
            const auto entry = [&](int k, int& i, float& v) {
                i = -1;
                if (!live || k >= d.top) return;
                const int at_index = K.idx[k];
                const float sum = K.sum[k];
                const bool own = (at_index >= s.from && at_index < end) ||
                                 (warp == 0 && (at_index < s.head || at_index >= (int)d.vocab - s.tail));
                if (sum < 0.0f || !own) return;
                i = at_index;
                v = pe * ex2(fmaf(K.z[k], c, -shift)) - f * sum;
            };
            int entry_at = -1;
            float entry_value = 0.0f;
            entry(lane, entry_at, entry_value);
            T* mine = out + s.from;
            const bool same = ((uintptr_t)mine & 15) == 0;   // units of both are the same
            // The first piece kept is where the slice began, or, when the slice
            // took more than the ring, where the next piece is.
            Place kept = n <= P.stages ? begin : at;
            for (int k = 0; k < n; ++k) {
                const int piece = k < keep ? n - keep + k : k - keep;
                const int stage = k < keep ? kept.stage : at.stage;
                if (k < keep)
                    kept.next(P.stages);
                else if (!lost && warp_wait(&S.full[warp][stage], at.phase))
                    at.next(P.stages);
                else
                    lost = true;
                const int u0 = piece * P.piece_units, count = min(P.piece_units, s.mine - u0);
                const char* part = ring + stage * piece_bytes;
                T* dst = mine + (int64_t)u0 * N;
                if (lost) {
                    for (int j = lane; j < count * N; j += 32) dst[j] = from_f<T>(CUDART_NAN_F);
                } else if (!live) {
                    write_zeros(dst, (int64_t)count * N, lane, 32);
                } else if (same) {
                    const uint4* units = reinterpret_cast<const uint4*>(part);
#pragma unroll 2
                    for (int u = lane; u < count; u += 32) {
                        float v[N];
                        Vec<T>::unpack(units[u], v);
                        exponentials(v, c, shift);
#pragma unroll
                        for (int j = 0; j < N; ++j) v[j] *= pe;
                        __stcs(reinterpret_cast<uint4*>(dst) + u, Vec<T>::pack(v));
                    }
                } else {
                    write_part(dst, part, 0, count * N, pe, c, shift, lane, 32);
                }
                __syncwarp();
                copy_next();
            }
            if (edge) out[edge_at] = from_f<T>(lost ? CUDART_NAN_F : live ? pe * ex2(fmaf(edge_value, c, -shift)) : 0.0f);
            __syncwarp();
            // The entries, over what was stored there.
            if (entry_at >= 0) out[entry_at] = from_f<T>(entry_value);
            for (int k = lane + 32; k < d.top; k += 32) {
                entry(k, entry_at, entry_value);
                if (entry_at >= 0) out[entry_at] = from_f<T>(entry_value);
            }
        }
        __syncwarp();
        if (lane == 0) bar_arrive(&S.heard[slot]);
        slots.next(P.depth);
    }
    if (lost)   // copies still on their way end in this CTA's time
        for (; at.stage != to.stage || at.phase != to.phase; at.next(P.stages))
            (void)bar_wait(&S.full[warp][at.stage], at.phase);
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
    const int64_t units = ceil_div(d.vocab + Vec<T>::N - 1, Vec<T>::N);
    const int64_t teacher = (int64_t)kTeacherBytes * d.top;
    // At most one row an SM: clusters, with more CTAs a row while that fills
    // idle SMs with 8 KB or more each.
    int cluster = 1;
    const auto slice = [&] { return 16 * ceil_div(units, cluster); };
    while (cluster < kMaxCluster && (slice() + 16 + teacher > 110 * 1024 ||
                                     (d.rows * cluster <= 74 && slice() >= 16 * 1024)))
        cluster *= 2;
    if (d.rows <= 148 && slice() + 16 + teacher <= 222 * 1024) {
        const int threads = slice() >= 16 * 1024 ? 512 : slice() >= 4 * 1024 ? 256 : 128;
        return status_of(launch(distill_cluster<T>, dim3((unsigned)(d.rows * cluster)), threads,
                                (size_t)(slice() + 16 + teacher), stream, cluster, false, d,
                                (int)(slice() / 16)),
                         "distill");
    }
    // Many rows.  8 warps a row and two CTAs an SM, so that one computes while
    // the other joins its warps; 16 and one CTA where a row fills more than half
    // of the shared memory; fewer warps for rows below 32 KB (4 KB a warp), and
    // as many CTAs as the registers take.
    // 16x1024 rows of 50257 bf16: 605 us (5.4 TB/s) with 8 warps; when both were built
    // 598, and 718 with 16.
    StreamPlan P;
    P.warps = 1;
    while (P.warps < 8 && 16 * units >= (int64_t)P.warps * 2 * 4096) P.warps *= 2;
    if (d.grad != nullptr && 16 * units > 104 * 1024) P.warps = 16;
    const int ctas = P.warps == 1 ? 10 : P.warps == 2 ? 7 : 16 / P.warps;
    P.depth = teacher * kMaxDepth <= 8 * 1024 / ctas ? kMaxDepth : 2;
    const int64_t grid = d.rows < 148 * ctas ? d.rows : 148 * ctas;
    // Up to 65536 rows with weights are listed (two kinds, each rounded up).
    P.listed = d.weight != nullptr && d.rows <= 65536 ? (int)(ceil_div(d.rows, grid) + 1) : 0;
    // A ring of two pieces, each a whole slice where that fits.
    P.each = (int)ceil_div(ceil_div(d.vocab, Vec<T>::N), P.warps);
    P.stages = 2;
    const int64_t beside = P.depth * teacher + 4 * (int64_t)P.listed + 16;
    int64_t room = (218 * 1024 / ctas - 4608 - beside) / P.warps / 16 / P.stages;
    if (room < 128) room = 128;   // long lists of entries beside short rows
    P.piece_units = P.each < room ? P.each : (int)room;
    const size_t smem = (size_t)(16 * P.piece_units * P.stages * P.warps + beside);
    return status_of(launch(distill_stream<T>, dim3((unsigned)grid), 32 * P.warps + 32, smem, stream,
                            1, false, d, P),
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
