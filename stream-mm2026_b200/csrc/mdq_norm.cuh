// mdq_norm.cuh - the norm after a block with its gate and the residual's scale,
// and the norm before the next block: the kernels of mdq_norm_*.cu, one file for
// each pair of types (mdq_ops.h).
//
// Both passes are bound by memory: forward reads x and h and writes x_new and n,
// backward reads x, h and the two gradients and writes two.  A row is held in
// registers, up to 32 columns a thread, by a team of up to 512 threads; rows that
// are wider by a cluster of CTAs that exchange their sums through distributed
// shared memory.  Parameters stay in registers over a team's rows, up to 16 columns
// a thread.  The backward pass keeps the parameters' gradients of a team's rows on
// the chip and leaves one partial sum for each CTA, which a second kernel adds in a
// fixed order.
//
// Measured, 16384 rows of 4096: bf16 RMS norm forward 97 us (5.5 TB/s), backward 150
// (5.4 TB/s); layer norm of an fp32 stream and bf16 blocks 172 (4.7) and 203 (6.0).
// With bf16 alone the steps of a row take longer than its bytes: 132 and 185 us.
#pragma once

#include "mdq_ops.cuh"

#include <cooperative_groups.h>
#include <math_constants.h>

namespace mdq_norm {

using namespace mdq_ops;
namespace cg = cooperative_groups;

constexpr int kTeam = 512;          // threads of a team at most
constexpr int kCols = 8;            // columns of a thread's chunk
constexpr int kMaxCluster = 8;

// How rows are given to threads.
struct Teams {
    int threads;    // of a team, a multiple of 32
    int teams;      // of a CTA (1 in a cluster)
    int share;      // columns of a CTA
    int run;        // rows of a team, consecutive
};

// The columns of one chunk of a thread: 8 consecutive ones on 16-byte boundaries
// (VECTOR), or 32 apart; a warp has 256 consecutive ones either way.
template <bool VECTOR>
struct Cols {
    int first, step, end;
    __device__ __forceinline__ int at(int k) const { return first + (VECTOR ? k : k * 32); }
    __device__ __forceinline__ bool has(int k) const { return (VECTOR ? 0 : k * 32) < end - first; }
    // The thread's chunk i.
    __device__ __forceinline__ Cols chunk(int i) const { return {first + i * step * 8, step, end}; }
};

// Eight values in pairs: products, sums and fused products of a pair are one
// instruction each, which about halves what the kernels issue.
typedef float2 F8[4];
__device__ __forceinline__ float2 mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ void fill(F8& v, float x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = both(x);
}
__device__ __forceinline__ float value(const F8& v, int k) { return k & 1 ? v[k >> 1].y : v[k >> 1].x; }
__device__ __forceinline__ void set(F8& v, int k, float x) { (k & 1 ? v[k >> 1].y : v[k >> 1].x) = x; }

__device__ __forceinline__ void unpack(uint4 w, F8& v) {
    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        v[j] = make_float2(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xffff0000u));
}

// Eight values as they were loaded, 0 outside of the row.
template <typename T, bool VECTOR>
struct Raw;
template <>
struct Raw<__nv_bfloat16, true> {
    uint4 a = {0, 0, 0, 0};
    __device__ __forceinline__ void load(const __nv_bfloat16* row, const Cols<true>& c) {
        if (c.has(0)) a = __ldcs(reinterpret_cast<const uint4*>(row + c.first));
    }
    __device__ __forceinline__ void get(F8& v) const { unpack(a, v); }
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
    __device__ __forceinline__ void get(F8& v) const {
        v[0] = make_float2(a.x, a.y);
        v[1] = make_float2(a.z, a.w);
        v[2] = make_float2(b.x, b.y);
        v[3] = make_float2(b.z, b.w);
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
    __device__ __forceinline__ void get(F8& v) const {
#pragma unroll
        for (int k = 0; k < 8; ++k) set(v, k, to_f(a[k]));
    }
};

template <typename T, bool VECTOR>
__device__ __forceinline__ void store(T* row, const Cols<VECTOR>& c, const F8& v, bool ragged = true) {
    if constexpr (!VECTOR) {
        T* to = row + c.first;
        if (!ragged) {
#pragma unroll
            for (int k = 0; k < 8; ++k) to[k * 32] = from_f<T>(value(v, k));
            return;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c.has(k)) to[k * 32] = from_f<T>(value(v, k));
    } else if (c.has(0)) {
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint4*>(row + c.first) =
                make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y),
                           pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
        } else {
            reinterpret_cast<float4*>(row + c.first)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
            reinterpret_cast<float4*>(row + c.first)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
        }
    }
}

// Zeros outside of the row, whatever was read there.
template <bool VECTOR>
__device__ __forceinline__ void within_row(F8& v, const Cols<VECTOR>& c) {
    if constexpr (VECTOR) {
        if (!c.has(0)) fill(v, 0.0f);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (!c.has(k)) set(v, k, 0.0f);
    }
}

// Parameters of a chunk: `none` without an array, 0 outside of the row.
template <bool VECTOR>
__device__ __forceinline__ void parameters(const void* p, bool bf16, const Cols<VECTOR>& c, float none,
                                           F8& v) {
    if (p == nullptr || (VECTOR && !c.has(0))) {
        fill(v, c.has(0) ? none : 0.0f);
        if constexpr (!VECTOR)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (!c.has(k)) set(v, k, 0.0f);
    } else if constexpr (VECTOR) {
        if (bf16) {
            unpack(__ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + c.first)), v);
        } else {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + c.first);
            const float4 a = __ldg(q), b = __ldg(q + 1);
            v[0] = make_float2(a.x, a.y);
            v[1] = make_float2(a.z, a.w);
            v[2] = make_float2(b.x, b.y);
            v[3] = make_float2(b.z, b.w);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) set(v, k, c.has(k) ? load_any(p, bf16, c.at(k)) : 0.0f);
    }
}
// p = gate * weight and b = gate * bias (FULL), both 0 outside of the row.
template <bool FULL, bool VECTOR>
__device__ __forceinline__ void post_parameters(const mdq_residual_norm_desc& d, const void* gate, bool pb,
                                                const Cols<VECTOR>& c, F8& p, F8& b) {
    F8 g;
    parameters(d.post_weight, pb, c, 1.0f, p);
    if (FULL) parameters(d.post_bias, pb, c, 0.0f, b);
    if (gate == nullptr) return;
    parameters(gate, pb, c, 1.0f, g);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        p[j] = mul(p[j], g[j]);
        if (FULL) b[j] = mul(b[j], g[j]);
    }
}
// The values less `mean` inside of the row; outside they are 0 and stay 0.
template <bool VECTOR>
__device__ __forceinline__ void less(F8& v, const Cols<VECTOR>& c, float mean, bool ragged) {
    if (VECTOR || !ragged) {
        const float2 m = both(!ragged || c.has(0) ? -mean : 0.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = add(v[j], m);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c.has(k)) set(v, k, value(v, k) - mean);
    }
}

// Warps that add up at most: those of the CTAs of a cluster, or of one CTA's teams.
constexpr int kSlots = kMaxCluster * kTeam / 32;

// Sums over a team, and over the cluster where that is larger.
struct Reducer {
    float* slots;     // [2][values x warps x CTAs]; this team's part begins at warp `base`
    int size;         // floats of one of the two
    int base, team, warp, warps, lane, parity, ctas, rank;

    // The sums of 2^LOG values, given to every thread.  Within a warp lanes hand
    // half of their values over in each of the first LOG steps, so that the
    // shuffles grow with the number of values and not with five times that.
    template <int LOG>
    __device__ __forceinline__ void sum(float (&v)[1 << LOG]) {
        constexpr int NV = 1 << LOG, kGroup = 32 >> LOG;
#pragma unroll
        for (int s = 0; s < LOG; ++s) {
            const bool upper = lane & 16 >> s;
#pragma unroll
            for (int j = 0; j < NV >> (s + 1); ++j) {
                float& high = v[j + (NV >> (s + 1))];
                const float keep = upper ? high : v[j], give = upper ? v[j] : high;
                v[j] = keep + __shfl_xor_sync(0xffffffffu, give, 16 >> s);
            }
        }
        float r = v[0];   // of value lane / kGroup
#pragma unroll
        for (int o = kGroup / 2; o > 0; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
        if (LOG == 0 && ctas == 1) {
            if (warps > 1) {   // 16 at most, in both halves of a warp
                float* buf = slots + parity * size + base;
                parity ^= 1;
                if (lane == 0) buf[warp] = r;
                asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(warps * 32) : "memory");
                r = (lane & 15) < warps ? buf[lane & 15] : 0.0f;
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
            }
            v[0] = r;
            return;
        }
        if (warps > 1 || ctas > 1) {
            float* buf = slots + parity * size + base * NV;
            parity ^= 1;   // the other buffer is read until every thread is past the next barrier
            const int value = lane / kGroup, sub = lane % kGroup;
            if (ctas == 1) {
                if (sub == 0) buf[warp * NV + value] = r;
                asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(warps * 32) : "memory");
            } else {
                cg::cluster_group cluster = cg::this_cluster();
                for (int k = sub; k < ctas; k += kGroup)
                    cluster.map_shared_rank(buf, k)[(rank * warps + warp) * NV + value] = r;
                cluster.sync();
            }
            r = 0.0f;
            if (ctas == 1) {   // 16 warps at most
#pragma unroll
                for (int k = 0; k < 16; k += kGroup)
                    if (k + sub < warps) r += buf[(k + sub) * NV + value];
            } else {
                for (int k = sub; k < ctas * warps; k += kGroup) r += buf[k * NV + value];
            }
#pragma unroll
            for (int o = kGroup / 2; o > 0; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = __shfl_sync(0xffffffffu, r, j * kGroup);
    }
};

// A thread's place: its team's rows and its columns.
template <bool VECTOR>
struct Place {
    Reducer R;
    Cols<VECTOR> cols;
    int t, team;
    int64_t index, count;   // of the team among all
    __device__ __forceinline__ Place(const Teams& G, int dim, float* slots, int size) {
        // From the warp's first lane: the compiler then knows that a warp is in one team.
        const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), warps = G.threads >> 5;
        team = warp / warps;
        t = (int)threadIdx.x - team * G.threads;
        cg::cluster_group cluster = cg::this_cluster();
        R.ctas = (int)cluster.num_blocks();
        R.rank = (int)cluster.block_rank();
        R.slots = slots;
        R.size = size;
        R.base = team * warps;
        R.team = team;
        R.warp = warp - team * warps;
        R.warps = warps;
        R.lane = t & 31;
        R.parity = 0;
        const int c0 = R.rank * G.share;
        cols.end = min(dim, c0 + G.share);
        cols.first = c0 + (VECTOR ? 8 * t : 8 * (t & ~31) + (t & 31));
        cols.step = G.threads;
        index = (int64_t)(blockIdx.x / R.ctas) * G.teams + team;
        count = (int64_t)(gridDim.x / R.ctas) * G.teams;
    }
};

// ---------------------------------------------------------- rows in a ring

constexpr int kMaxStages = 6;

// A chunk's eight values in shared memory, the row's first at `row`.
template <typename T, bool VECTOR>
__device__ __forceinline__ void from_shared(const T* row, int at, F8& v) {
    if constexpr (!VECTOR) {
#pragma unroll
        for (int k = 0; k < 8; ++k) set(v, k, to_f(row[at + k * 32]));
    } else if constexpr (sizeof(T) == 2) {
        unpack(*reinterpret_cast<const uint4*>(row + at), v);
    } else {
        const float4 a = reinterpret_cast<const float4*>(row + at)[0];
        const float4 b = reinterpret_cast<const float4*>(row + at)[1];
        v[0] = make_float2(a.x, a.y);
        v[1] = make_float2(a.z, a.w);
        v[2] = make_float2(b.x, b.y);
        v[3] = make_float2(b.z, b.w);
    }
}

// Bytes a stage keeps for `share` columns of T: the row's 16-byte units, two of
// which it may share with its neighbours, and for threads behind the row's end.
template <typename T, bool VECTOR>
__host__ __device__ constexpr int stage_part(int share, int lanes) {
    return VECTOR ? share * (int)sizeof(T) : (lanes * (int)sizeof(T) + 47) / 16 * 16;
}

// One array whose rows come through the ring, in shared memory: a lane of the
// team's first warp copies them, so that all arrays are copied by the same few
// instructions.
struct Feed {
    const char *next, *lo, *hi;   // the next row's columns; the array's limits
    int64_t step;                 // bytes from row to row
    int bytes, at;                // of a row's columns; their place in a stage
};
constexpr int kFeeds = 5;   // h, x, grad_n, grad_new, the statistics

// Copies f's next row into the stage and arrives at its barrier.  In bulk go whole
// 16-byte units, with what the first and last hold of the neighbours (not VECTOR);
// units that reach out of the array go value by value.
template <bool VECTOR>
__device__ __forceinline__ void feed_row(Feed& f, char* stage, void* bar, unsigned long long policy) {
    const char* from = f.next;
    f.next = from + f.step;
    char* to = stage + f.at;
    if constexpr (VECTOR) {
        expect_bytes(bar, (unsigned)f.bytes);
        copy_part(bar, to, from, (unsigned)f.bytes, policy);
    } else {
        const int shift = (int)((uintptr_t)from & 15);
        const char *a = from - shift, *b = from + f.bytes + (-(uintptr_t)(from + f.bytes) & 15);
        if (a < f.lo) a += 16;
        if (b > f.hi) b -= 16;
        if (b < a) b = a;
        to += shift;   // where `from` goes
        for (int k = 0; k < min(f.bytes, (int)(a - from)); k += 2)
            *reinterpret_cast<uint16_t*>(to + k) = *reinterpret_cast<const uint16_t*>(from + k);
        for (int k = max(0, max((int)(a - from), (int)(b - from))); k < f.bytes; k += 2)
            *reinterpret_cast<uint16_t*>(to + k) = *reinterpret_cast<const uint16_t*>(from + k);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        const unsigned bytes = (unsigned)(b - a);
        expect_bytes(bar, bytes);
        if (bytes > 0) copy_part(bar, to + (a - from), a, bytes, policy);
    }
}

// A team's ring of rows: its stages, its feeds and the place it is at.
template <bool VECTOR>
struct Ring {
    char* stage0;
    unsigned long long* full;
    Feed* feeds;
    int stages, stage_bytes, left, to, stage;
    unsigned phase;
    bool feeder, lost;
    unsigned long long policy;

    // Before the first barrier of the CTA, by every thread of the team.
    // arrays[k] with strides[k] elements of sizes[k] bytes a row; parts[k]: the place
    // of its `mine` columns in a stage; the last array is 16 bytes a row (`tail`).
    template <int N>
    __device__ __forceinline__ void open(const void* const (&arrays)[N], const int64_t (&strides)[N],
                                         const int (&sizes)[N], const int (&parts)[N + 1], bool tail,
                                         int c0, int mine, int64_t rows, int64_t r0, int64_t r1, int t,
                                         int threads) {
        int there = 0;   // arrays that are fed
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const bool whole = tail && k == N - 1;
            if (t == 0) {
                const char* p = static_cast<const char*>(arrays[k]) + (whole ? 0 : (int64_t)c0 * sizes[k]);
                const int64_t step = strides[k] * sizes[k];
                const int bytes = arrays[k] == nullptr ? 0 : whole ? 16 : mine * sizes[k];
                feeds[k] = {p + r0 * step, p, p + (rows - 1) * step + bytes, step, bytes, parts[k]};
            }
            there += arrays[k] != nullptr;
            const int words = (parts[k + 1] - parts[k]) / 4;
            if (arrays[k] == nullptr)   // its place holds zeros
                for (int i = t; i < stages * words; i += threads)
                    reinterpret_cast<unsigned*>(stage0 + i / words * stage_bytes + parts[k])[i % words] = 0;
        }
        if (t == 0)
            for (int k = 0; k < stages; ++k) bar_init(&full[k], there);
        asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
        left = (int)(r1 - r0);
        to = stage = 0;
        phase = 0;
        lost = false;
        policy = read_once();
    }
    // Behind that barrier, by the team's first warp: the next row into the next stage.
    __device__ __forceinline__ void copy_row(int t) {
        if (left == 0 || lost) return;
        if (feeder) feed_row<VECTOR>(feeds[t], stage0 + to * stage_bytes, &full[to], policy);
        --left;
        if (++to == stages) to = 0;
    }
    template <int N>
    __device__ __forceinline__ void start(int t) {
        feeder = t < N && feeds[t < N ? t : 0].bytes > 0;
        if (t < 32)
            for (int k = 0; k < stages - 1; ++k) copy_row(t);
    }
    // The present row's stage, once it is there.  After a wait that ran out (`lost`)
    // nothing is waited for or copied any more, the stage stays, and the thread's
    // values of the rows are taken as NaN: through the sums all of the rows become it.
    __device__ __forceinline__ const char* row() {
        if (!lost && !bar_wait(&full[stage], phase)) lost = true;
        return stage0 + stage * stage_bytes;
    }
    __device__ __forceinline__ void next() {
        if (!lost && ++stage == stages) {
            stage = 0;
            phase ^= 1;
        }
    }
    // Copies still on their way end before the CTA does: by the lanes that asked for
    // them, from the row that was waited for up to their last.
    __device__ __forceinline__ void close(int t) {
        if (lost && t < 32 && feeder)
            for (; stage != to; phase ^= stage == 0) {
                (void)bar_wait(&full[stage], phase);
                if (++stage == stages) stage = 0;
            }
    }
};

// (rsqrtf: 2 units in the last place, where sums of a row's terms are off by more;
// a square root and a quotient are 30 instructions that every thread repeats.)
//
// Mean and 1 / deviation of a row (mean 0 without `layer`); its values lose
// their mean.
template <int I, bool VECTOR>
__device__ __forceinline__ float2 statistics(Reducer& R, const Cols<VECTOR>& cols, F8 (&v)[I],
                                             bool layer, bool ragged, float inv, float eps) {
    float mean = 0.0f;
    if (layer) {
        float2 t = both(0.0f);
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) t = add(t, v[i][j]);
        float s[1] = {t.x + t.y};
        R.sum<0>(s);
        mean = s[0] * inv;
#pragma unroll
        for (int i = 0; i < I; ++i) less(v[i], cols.chunk(i), mean, ragged);
    }
    float2 t = both(0.0f);
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) t = fma(v[i][j], v[i][j], t);
    float q[1] = {t.x + t.y};
    R.sum<0>(q);
    return make_float2(mean, rsqrtf(fmaf(q[0], inv, eps)));
}

// RMS norm without biases, rows on 16-byte boundaries: rows go straight to
// registers, I chunks of 8 columns a thread.  With one or two, the parameters stay
// in registers over a team's rows and the next row is loaded ahead; with four (rows
// above 8192 columns) neither fits, and a row is long enough to fill the time.
// 16384 bf16 rows of 4096: 96 us (5.6 TB/s); 102 against 110 through the ring when
// both were built.
template <typename XT, typename HT, int I>
__global__ void __launch_bounds__(kTeam, 1) norm_rows(const __grid_constant__ mdq_residual_norm_desc d,
                                                      const __grid_constant__ Teams G) {
    __shared__ float slots[2 * kSlots];
    Place<true> P(G, (int)d.dim, slots, kSlots);
    const Cols<true>& cols = P.cols;
    if (P.R.ctas > 1) cg::this_cluster().sync();   // all run before their memory is written to
    const bool pb = d.param_dtype == MDQ_BF16;
    const float inv = 1.0f / (float)d.dim;
    const XT* x = static_cast<const XT*>(d.x);
    const HT* h = static_cast<const HT*>(d.h);
    const int64_t per = d.rows / d.gate_rows;
    const int64_t r0 = min(d.rows, P.index * G.run), r1 = min(d.rows, r0 + G.run);
    constexpr bool kKeep = I <= 2;
    F8 kp[kKeep ? I : 1], kw[kKeep ? I : 1], none;
    if constexpr (kKeep) {
#pragma unroll
        for (int i = 0; i < I; ++i) parameters(d.pre_weight, pb, cols.chunk(i), 1.0f, kw[i]);
    }
    Raw<XT, true> nx[I];
    Raw<HT, true> nh[I];
    const XT* xr = x + r0 * d.x_stride;
    const HT* hr = h + r0 * d.h_stride;
    const auto fetch = [&] {   // the next row
#pragma unroll
        for (int i = 0; i < I; ++i) {
            if (h != nullptr) nh[i].load(hr, cols.chunk(i));
            nx[i].load(xr, cols.chunk(i));
        }
        xr += d.x_stride;
        hr += d.h_stride;
    };
    XT* xo = static_cast<XT*>(d.x_new) + r0 * d.dim;
    HT* no = static_cast<HT*>(d.n) + r0 * d.dim;
    if (kKeep && r0 < r1) fetch();
    int64_t turn = r0;   // the row at which another row of the gate begins
    const void* gate = d.gate;
    for (int64_t r = r0; r < r1; ++r, xo += d.dim, no += d.dim) {
        if (r == turn) {
            turn = r1;
            if (d.gate_rows > 1) {
                const int64_t k = r / per;
                gate = static_cast<const char*>(d.gate) + k * d.dim * (pb ? 2 : 4);
                turn = (k + 1) * per;
            }
            if (kKeep && h != nullptr)
#pragma unroll
                for (int i = 0; i < I; ++i)
                    post_parameters<false>(d, gate, pb, cols.chunk(i), kp[kKeep ? i : 0], none);
        }
        F8 v[I];
        Raw<XT, true> rx[I];
        float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (!kKeep) fetch();
#pragma unroll
        for (int i = 0; i < I; ++i) {
            rx[i] = nx[i];
            nh[i].get(v[i]);
        }
        if (kKeep && r + 1 < r1) fetch();
        if (h != nullptr) {
            st.y = statistics<I>(P.R, cols, v, false, false, inv, d.eps).y;
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const Cols<true> c = cols.chunk(i);
                F8 p, xv;
                if constexpr (kKeep) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = kp[i][j];
                } else {
                    post_parameters<false>(d, gate, pb, c, p, none);
                }
                rx[i].get(xv);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[i][j] = fma(both(d.residual_scale), xv[j], mul(mul(v[i][j], both(st.y)), p[j]));
                store(xo, c, v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < I; ++i) rx[i].get(v[i]);
        }
        if (d.n != nullptr) {
            st.w = statistics<I>(P.R, cols, v, false, false, inv, d.eps).y;
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const Cols<true> c = cols.chunk(i);
                F8 w;
                if constexpr (kKeep) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = kw[i][j];
                } else {
                    parameters(d.pre_weight, pb, c, 1.0f, w);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = mul(mul(v[i][j], both(st.w)), w[j]);
                store(no, c, v[i]);
            }
        }
        if (d.stats != nullptr && P.t == 0 && P.R.rank == 0)
            reinterpret_cast<float4*>(d.stats)[r] = st;
    }
    if (P.R.ctas > 1) cg::this_cluster().sync();   // none ends while its memory may be written to
}

// Layer norm, biases, or rows of any alignment: a team's rows come through a ring
// of `stages` in shared memory, so that no registers hold loads.  FULL: layer norm
// or biases.  4096 bf16 rows of 8192, layer norm: 71 us (93 against 115 with rows in
// registers when both were built); 16368 rows of 1601: 61 (93 against 190).
template <typename XT, typename HT, bool VECTOR, int I, bool FULL>
__global__ void __launch_bounds__(kTeam, 1) norm_rows_ring(const __grid_constant__
                                                           mdq_residual_norm_desc d,
                                                           const __grid_constant__ Teams G, int stages) {
    __shared__ float slots[2 * kSlots];
    __shared__ unsigned long long full[kTeam / 32][kMaxStages];
    __shared__ Feed feeds[kTeam / 32][2];
    extern __shared__ __align__(16) char memory[];   // [team][stage]: h, x
    Place<VECTOR> P(G, (int)d.dim, slots, kSlots);
    const Cols<VECTOR>& cols = P.cols;
    const bool layer = FULL && d.kind == MDQ_NORM_LAYER, pb = d.param_dtype == MDQ_BF16;
    const float inv = 1.0f / (float)d.dim;
    const bool has_h = d.h != nullptr;
    const int64_t per = d.rows / d.gate_rows;
    const int64_t r0 = min(d.rows, P.index * G.run), r1 = min(d.rows, r0 + G.run);
    const int c0 = P.R.rank * G.share, mine = cols.end - c0, lanes = G.threads * 8 * I;
    const int hb = stage_part<HT, VECTOR>(G.share, lanes), xb = stage_part<XT, VECTOR>(G.share, lanes);
    const void* const arrays[2] = {d.h, d.x};
    const int64_t strides[2] = {d.h_stride, d.x_stride};
    constexpr int sizes[2] = {sizeof(HT), sizeof(XT)};
    const int parts[3] = {0, hb, hb + xb};
    Ring<VECTOR> ring;
    ring.stage0 = memory + (size_t)P.team * stages * (hb + xb);
    ring.full = full[P.team];
    ring.feeds = feeds[P.team];
    ring.stages = stages;
    ring.stage_bytes = hb + xb;
    ring.open(arrays, strides, sizes, parts, false, c0, mine, d.rows, r0, r1, P.t, G.threads);
    if (P.R.ctas > 1) cg::this_cluster().sync();   // all run before their memory is written to
    else __syncthreads();
    ring.template start<2>(P.t);

    constexpr bool kKeep = I <= 2;
    F8 kp[kKeep ? I : 1], kb[kKeep && FULL ? I : 1], kw[kKeep ? I : 1], kc[kKeep && FULL ? I : 1];
    if constexpr (kKeep) {
#pragma unroll
        for (int i = 0; i < I; ++i) {
            parameters(d.pre_weight, pb, cols.chunk(i), 1.0f, kw[i]);
            if (FULL) parameters(d.pre_bias, pb, cols.chunk(i), 0.0f, kc[FULL ? i : 0]);
        }
    }
    // Threads behind the row's end read its last values (VECTOR) or what lies
    // there, and drop them (in warps that reach there: `ragged`).
    const bool ragged = ((I - 1) * G.threads + P.R.warp * 32 + 32) * 8 > mine;
    const auto place = [&](int i) {
        const int at = cols.chunk(i).first - c0;
        return VECTOR ? min(at, mine - 8) : at;
    };
    unsigned shifts[2];   // bytes by which the rows start behind a 16-byte boundary
#pragma unroll
    for (int k = 0; k < 2; ++k)
        shifts[k] = VECTOR ? 0 : (unsigned)((uintptr_t)arrays[k] + (c0 + r0 * strides[k]) * sizes[k]) & 15;
    XT* xo = static_cast<XT*>(d.x_new) + r0 * d.dim;
    HT* no = static_cast<HT*>(d.n) + r0 * d.dim;
    int64_t turn = r0;   // the row at which another row of the gate begins
    const void* gate = d.gate;
    for (int64_t r = r0; r < r1; ++r, xo += d.dim, no += d.dim) {
        if (r == turn) {
            turn = r1;
            if (d.gate_rows > 1) {
                const int64_t k = r / per;
                gate = static_cast<const char*>(d.gate) + k * d.dim * (pb ? 2 : 4);
                turn = (k + 1) * per;
            }
            if (kKeep && has_h)
#pragma unroll
                for (int i = 0; i < I; ++i)
                    post_parameters<FULL>(d, gate, pb, cols.chunk(i), kp[kKeep ? i : 0],
                                          kb[kKeep && FULL ? i : 0]);
        }
        const char* s0 = ring.row();
        const HT* hr = reinterpret_cast<const HT*>(s0 + shifts[0]);
        const XT* xr = reinterpret_cast<const XT*>(s0 + hb + shifts[1]);
        F8 v[I];
        float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        // The first sums of a row end with every thread past the row before, whose
        // stage is free then.
        const auto refill = [&] {
            if (G.threads == 32) __syncwarp();
            if (P.R.warp == 0) ring.copy_row(P.t);
        };
        if (has_h) {
#pragma unroll
            for (int i = 0; i < I; ++i) {
                from_shared<HT, VECTOR>(hr, place(i), v[i]);
                if (ragged) within_row(v[i], cols.chunk(i));
            }
            if (ring.lost) v[0][0] = both(CUDART_NAN_F);
            const float2 s = statistics<I>(P.R, cols, v, layer, ragged, inv, d.eps);
            refill();
            st.x = s.x;
            st.y = s.y;
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const Cols<VECTOR> c = cols.chunk(i);
                F8 p, b, xv;
                if constexpr (kKeep) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        p[j] = kp[i][j];
                        b[j] = kb[FULL ? i : 0][j];
                    }
                } else {
                    post_parameters<FULL>(d, gate, pb, c, p, b);
                }
                from_shared<XT, VECTOR>(xr, place(i), xv);
                if (ragged) within_row(xv, c);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[i][j] = mul(v[i][j], both(s.y));
                    if (FULL) v[i][j] = fma(v[i][j], p[j], b[j]);
                    else v[i][j] = mul(v[i][j], p[j]);
                    v[i][j] = fma(both(d.residual_scale), xv[j], v[i][j]);
                }
                store(xo, c, v[i], ragged);
            }
        } else {
#pragma unroll
            for (int i = 0; i < I; ++i) {
                from_shared<XT, VECTOR>(xr, place(i), v[i]);
                if (ragged) within_row(v[i], cols.chunk(i));
            }
            if (ring.lost) v[0][0] = both(CUDART_NAN_F);
        }
        if (d.n != nullptr) {
            const float2 s = statistics<I>(P.R, cols, v, layer, ragged, inv, d.eps);
            if (!has_h) refill();
            st.z = s.x;
            st.w = s.y;
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const Cols<VECTOR> c = cols.chunk(i);
                F8 w, b;
                if constexpr (kKeep) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        w[j] = kw[i][j];
                        b[j] = kc[FULL ? i : 0][j];
                    }
                } else {
                    parameters(d.pre_weight, pb, c, 1.0f, w);
                    if (FULL) parameters(d.pre_bias, pb, c, 0.0f, b);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[i][j] = mul(v[i][j], both(s.y));
                    if (FULL) v[i][j] = fma(v[i][j], w[j], b[j]);
                    else v[i][j] = mul(v[i][j], w[j]);
                }
                store(no, c, v[i], ragged);
            }
        }
        if (d.stats != nullptr && P.t == 0 && P.R.rank == 0)
            reinterpret_cast<float4*>(d.stats)[r] = st;
        ring.next();
        if (!VECTOR)
#pragma unroll
            for (int k = 0; k < 2; ++k) shifts[k] = (shifts[k] + (unsigned)strides[k] * sizes[k]) & 15;
    }
    ring.close(P.t);
    if (P.R.ctas > 1) cg::this_cluster().sync();   // none ends while its memory may be written to
}

// ------------------------------------------------------------------ backward

// Sums of the rows of one CTA, [kinds][dim] each.
enum { kPre = 0, kPost = 1, kPreBias = 2, kPostBias = 3 };   // of dn xh, t hh (times the gate), dn, t

// Rows of the workspace: [block][4][dim], then (GROUPED) [team][2 edges][2][dim]:
// the gate's sums of runs that begin or end within a team's rows.
struct Partials {
    float* sums;
    float* edges;
};

// What one chunk of a row holds.
template <typename XT, typename HT, bool VECTOR>
struct GradRaw {
    Raw<XT, VECTOR> x, gx;
    Raw<HT, VECTOR> h, gn;
};

// A group's sums of t hh and t leave the registers: the gate's gradient, or the
// team's part of it, and their share of the parameters' gradients, which the thread
// has in shared memory (`keep`, `step` floats apart): as they change with groups
// only, registers for them would be taken from the rows.
template <bool VECTOR, bool FULL, int G>
__device__ __forceinline__ void end_group(const mdq_residual_norm_grad_desc& g, const void* gate, bool pb,
                                          const Cols<VECTOR>& c, int64_t k0, float* edge, F8 (&group)[G],
                                          float* keep, int step) {
    const int64_t dim = g.f.dim;
    F8 w, w1, b1;
    parameters(gate, pb, c, 1.0f, w);
    parameters(g.f.post_weight, pb, c, 1.0f, w1);
    parameters(FULL ? g.f.post_bias : nullptr, pb, c, 0.0f, b1);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (!c.has(k)) continue;
        const float sum = value(group[0], k), sum_b = value(group[G - 1], k);
        keep[k * step] = fmaf(value(w, k), sum, keep[k * step]);
        if (FULL) keep[(8 + k) * step] = fmaf(value(w, k), sum_b, keep[(8 + k) * step]);
        if (edge != nullptr) {
            edge[c.at(k)] = sum;
            edge[dim + c.at(k)] = sum_b;
        } else if (g.grad_gate != nullptr) {
            store_any(g.grad_gate, pb, k0 * dim + c.at(k), fmaf(value(w1, k), sum, value(b1, k) * sum_b));
        }
    }
    fill(group[0], 0.0f);
    fill(group[G - 1], 0.0f);
}

// The CTA's sums, its teams adding theirs in turn in `shared` ([KINDS][share]).
template <bool VECTOR, int KINDS>
__device__ __forceinline__ void end_sums(const Place<VECTOR>& P, const Teams& G, const Partials& W, int dim,
                                         float* shared, const F8 (&acc)[KINDS]) {
    const int c0 = P.R.rank * G.share;
    float* out = W.sums + (int64_t)(blockIdx.x / P.R.ctas) * 4 * dim;
    for (int i = 0; i < G.teams; ++i) {
        if (i > 0) __syncthreads();
        if (P.team != i) continue;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (!P.cols.has(k)) continue;
#pragma unroll
            for (int j = 0; j < KINDS; ++j) {
                float* q = shared + j * G.share + P.cols.at(k) - c0;
                const float v = i > 0 ? *q + value(acc[j], k) : value(acc[j], k);
                if (i + 1 < G.teams) *q = v;
                else out[(int64_t)j * dim + P.cols.at(k)] = v;
            }
        }
    }
}

// With q = g w1 hh, p = g w1 and f = dx + r2 e, the gradient u = t p of the
// normalised block has
//   sum u hh = sum f q - r2 (m0 sum q + m1 sum xh q)
// (and sum u the same with p for q), so that all sums of a row are taken in one
// step, from which m1 = mean(e xh), m0 = mean(e) and the means of u follow.
//
// FULL: a mean is removed or a bias is there, so sums without the normalised
// value are needed as well.  GROUPED: the gate differs between rows; its sums go
// out at the end of every group, weighted into the others.
//
// Rows of more than 8192 columns: two or four chunks a thread, loaded straight
// into registers; the parameters' gradients are in shared memory, each value of
// one thread.
template <typename XT, typename HT, bool VECTOR, int I, bool FULL, bool GROUPED>
__global__ void __launch_bounds__(kTeam, 1) norm_grad_rows(const __grid_constant__
                                                           mdq_residual_norm_grad_desc g,
                                                           const __grid_constant__ Teams G,
                                                           const __grid_constant__ Partials W) {
    constexpr int kLog = FULL ? 3 : 2, kKinds = FULL ? 4 : 2;
    __shared__ float slots[2 * kSlots * (1 << kLog)];
    extern __shared__ __align__(16) float shared[];   // [kinds][share]
    const mdq_residual_norm_desc& d = g.f;
    Place<VECTOR> P(G, (int)d.dim, slots, kSlots << kLog);
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
    const int c0 = P.R.rank * G.share;

    const auto place_of = [&](int kind, const Cols<VECTOR>& c, int k) {
        return shared + kind * G.share + c.at(k) - c0;
    };
    // Adds to a sum in shared memory; kinds 4 and 5 are the group's.
    const auto add_to = [&](int kind, const Cols<VECTOR>& c, const F8& v) {
        if constexpr (VECTOR) {
            if (!c.has(0)) return;
            float4* q = reinterpret_cast<float4*>(place_of(kind, c, 0));
            float4 a = q[0], b = q[1];
            a.x += v[0].x; a.y += v[0].y; a.z += v[1].x; a.w += v[1].y;
            b.x += v[2].x; b.y += v[2].y; b.z += v[3].x; b.w += v[3].y;
            q[0] = a;
            q[1] = b;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c.has(k)) *place_of(kind, c, k) += value(v, k);
        }
    };
    for (int i = threadIdx.x; i < (GROUPED ? 6 : kKinds) * G.share; i += blockDim.x) shared[i] = 0.0f;
    __syncthreads();
    GradRaw<XT, HT, VECTOR> raw[I];
    float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const XT *xr = x + r0 * d.x_stride, *gxr = gx + r0 * g.grad_new_stride;
    const HT *hr = h + r0 * d.h_stride, *gnr = gn + r0 * g.grad_n_stride;
    const float4* sr = reinterpret_cast<const float4*>(d.stats) + r0;
    const auto fetch = [&] {   // the next row
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const Cols<VECTOR> c = cols.chunk(i);
            if (h != nullptr) raw[i].h.load(hr, c);
            raw[i].x.load(xr, c);
            if (gn != nullptr) raw[i].gn.load(gnr, c);
            if (gx != nullptr) raw[i].gx.load(gxr, c);
        }
        st = __ldg(sr++);
        xr += d.x_stride;
        hr += d.h_stride;
        gxr += g.grad_new_stride;
        gnr += g.grad_n_stride;
    };
    XT* xo = static_cast<XT*>(g.grad_x) + r0 * d.dim;
    HT* ho = static_cast<HT*>(g.grad_h) + r0 * d.dim;
    // The rows of every CTA of a cluster are the same, so all take part in its sums.
    int64_t turn = r0, k0 = 0;   // the row at which another row of the gate begins; this one's
    const void* gate = d.gate;
    for (int64_t r = r0; r < r1; ++r, xo += d.dim, ho += d.dim) {
        fetch();
        if (GROUPED && r == turn) {
            k0 = r / per;
            gate = static_cast<const char*>(d.gate) + k0 * d.dim * (pb ? 2 : 4);
            turn = (k0 + 1) * per;
        }
        // hh, xh, e and p of a chunk; outside of the row e and p are 0
        const auto values = [&](int i, const Cols<VECTOR>& c, F8& hh, F8& xh, F8& e, F8& p) {
            F8 b;
            raw[i].x.get(xh);
            if (h != nullptr) {
                raw[i].h.get(hh);
                post_parameters<FULL>(d, gate, pb, c, p, b);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (FULL) hh[j] = add(hh[j], both(-st.x));
                    hh[j] = mul(hh[j], both(st.y));
                    if (FULL) xh[j] = fma(both(d.residual_scale), xh[j], b[j]);
                    else xh[j] = mul(both(d.residual_scale), xh[j]);
                    xh[j] = fma(p[j], hh[j], xh[j]);
                }
            } else {
                fill(hh, 0.0f);
                fill(p, 0.0f);
            }
            raw[i].gn.get(e);
            parameters(d.pre_weight, pb, c, 1.0f, b);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (FULL) xh[j] = add(xh[j], both(-st.z));
                xh[j] = mul(xh[j], both(st.w));
                e[j] = mul(e[j], b[j]);
            }
        };
        F8 hh, xh, e, p;
        const float rx = gn != nullptr ? st.w : 0.0f, a = h != nullptr ? d.residual_scale : 1.0f;
        float2 s2[FULL ? 8 : 3];
#pragma unroll
        for (int j = 0; j < (FULL ? 8 : 3); ++j) s2[j] = both(0.0f);
#pragma unroll
        for (int i = 0; i < I; ++i) {
            F8 dx;
            values(i, cols.chunk(i), hh, xh, e, p);
            raw[i].gx.get(dx);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 q = mul(p[j], hh[j]);
                const float2 f = fma(both(rx), e[j], dx[j]);
                s2[0] = fma(e[j], xh[j], s2[0]);
                s2[1] = fma(f, q, s2[1]);
                s2[2] = fma(xh[j], q, s2[2]);
                if constexpr (FULL) {
                    s2[3] = add(s2[3], e[j]);
                    s2[4] = add(s2[4], q);
                    s2[5] = fma(f, p[j], s2[5]);
                    s2[6] = fma(xh[j], p[j], s2[6]);
                    s2[7] = add(s2[7], p[j]);
                }
            }
        }
        float s[1 << kLog] = {};
#pragma unroll
        for (int j = 0; j < (FULL ? 8 : 3); ++j) s[j] = s2[j].x + s2[j].y;
        P.R.template sum<kLog>(s);
        const float m1 = s[0] * inv;
        float m0 = 0.0f, u0 = 0.0f, u1 = fmaf(-rx * m1, s[2], s[1]);
        if constexpr (FULL) {
            if (layer) {
                m0 = s[3] * inv;
                u1 = fmaf(-rx * m0, s[4], u1);
                u0 = fmaf(-rx * m0, s[7], fmaf(-rx * m1, s[6], s[5])) * inv;
            }
        }
        u1 *= inv;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const Cols<VECTOR> c = cols.chunk(i);
            F8 t, dn, o;
            values(i, c, hh, xh, e, p);
            raw[i].gx.get(t);
            raw[i].gn.get(dn);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 y = fma(xh[j], both(-m1), e[j]);
                if (FULL) y = add(y, both(-m0));
                t[j] = fma(both(rx), y, t[j]);
                xh[j] = mul(xh[j], dn[j]);
                o[j] = mul(both(a), t[j]);
            }
            add_to(kPre, c, xh);
            if (FULL) add_to(kPreBias, c, dn);
            store(xo, c, o);
            if (h == nullptr) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = mul(t[j], p[j]);
                if (FULL) o[j] = add(o[j], both(-u0));
                o[j] = mul(both(st.y), fma(hh[j], both(-u1), o[j]));
            }
            store(ho, c, o);
#pragma unroll
            for (int j = 0; j < 4; ++j) hh[j] = mul(hh[j], t[j]);
            add_to(GROUPED ? 4 : kPost, c, hh);
            if (FULL) add_to(GROUPED ? 5 : kPostBias, c, t);
        }
        if constexpr (GROUPED) {
            if (r + 1 == r1 || r + 1 == turn) {   // the group ends, or this team's part of it
                const int64_t first = k0 * per, last = first + per - 1;
                const bool whole = first >= r0 && last < r1;
                float* edge = W.edges + ((P.index * 2 + (first >= r0)) * 2) * d.dim;
#pragma unroll
                for (int i = 0; i < I; ++i) {
                    const Cols<VECTOR> c = cols.chunk(i);
                    F8 w, w1, b1;
                    parameters(gate, pb, c, 1.0f, w);
                    parameters(d.post_weight, pb, c, 1.0f, w1);
                    parameters(FULL ? d.post_bias : nullptr, pb, c, 0.0f, b1);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if (!c.has(k)) continue;
                        const float sum = *place_of(4, c, k), sum_b = *place_of(5, c, k);
                        *place_of(kPost, c, k) += value(w, k) * sum;
                        if (FULL) *place_of(kPostBias, c, k) += value(w, k) * sum_b;
                        *place_of(4, c, k) = *place_of(5, c, k) = 0.0f;
                        if (whole) {
                            if (g.grad_gate != nullptr)
                                store_any(g.grad_gate, pb, k0 * d.dim + c.at(k),
                                          fmaf(value(w1, k), sum, value(b1, k) * sum_b));
                        } else {
                            edge[c.at(k)] = sum;
                            edge[d.dim + c.at(k)] = sum_b;
                        }
                    }
                }
            }
        }
    }
    float* out = W.sums + (int64_t)(blockIdx.x / P.R.ctas) * 4 * d.dim;
    __syncthreads();
    const int mine = max(0, min((int)d.dim - c0, G.share));
#pragma unroll
    for (int j = 0; j < kKinds; ++j)
        for (int i = threadIdx.x; i < mine; i += blockDim.x)
            out[j * d.dim + c0 + i] = shared[j * G.share + i];
    if (P.R.ctas > 1) cg::this_cluster().sync();
}

// The same with the rows in a ring, as in the forward pass, for up to 8192
// columns: one chunk of columns a thread and one or two CTAs a row.
template <typename XT, typename HT, bool VECTOR, bool FULL, bool GROUPED>
__global__ void __launch_bounds__(kTeam, 1) norm_grad_stream(const __grid_constant__
                                                             mdq_residual_norm_grad_desc g,
                                                             const __grid_constant__ Teams G,
                                                             const __grid_constant__ Partials W,
                                                             int stages) {
    constexpr int kLog = FULL ? 3 : 2, kKinds = FULL ? 4 : 2;
    __shared__ float slots[2 * kSlots * (1 << kLog)];
    __shared__ unsigned long long full[kTeam / 32][kMaxStages];
    __shared__ Feed feeds[kTeam / 32][kFeeds];
    extern __shared__ __align__(16) char memory[];   // [team][stage]: h, x, grad_n, grad_new, stats
    const mdq_residual_norm_desc& d = g.f;
    Place<VECTOR> P(G, (int)d.dim, slots, kSlots << kLog);
    const Cols<VECTOR>& cols = P.cols;
    const bool layer = FULL && d.kind == MDQ_NORM_LAYER, pb = d.param_dtype == MDQ_BF16;
    const float inv = 1.0f / (float)d.dim;
    const int64_t per = d.rows / d.gate_rows;
    const int64_t r0 = min(d.rows, P.index * G.run), r1 = min(d.rows, r0 + G.run);
    const int c0 = P.R.rank * G.share, mine = cols.end - c0, lanes = G.threads * 8;
    const bool has_h = d.h != nullptr, has_gn = g.grad_n != nullptr;

    const int hb = stage_part<HT, VECTOR>(G.share, lanes), xb = stage_part<XT, VECTOR>(G.share, lanes);
    const int at_x = hb, at_gn = hb + xb, at_gx = 2 * hb + xb;
    const int at_st = 2 * (hb + xb), stage_bytes = at_st + 16;
    const void* const arrays[kFeeds] = {d.h, d.x, g.grad_n, g.grad_new, d.stats};
    const int64_t strides[kFeeds] = {d.h_stride, d.x_stride, g.grad_n_stride, g.grad_new_stride, 4};
    constexpr int sizes[kFeeds] = {sizeof(HT), sizeof(XT), sizeof(HT), sizeof(XT), 4};
    const int parts[kFeeds + 1] = {0, at_x, at_gn, at_gx, at_st, stage_bytes};
    Ring<VECTOR> ring;
    // GROUPED: first each thread's sums over its groups
    const int kept = GROUPED ? (FULL ? 16 : 8) * (int)sizeof(float) * blockDim.x : 0;
    float* keep = reinterpret_cast<float*>(memory) + threadIdx.x;
    if (GROUPED)
        for (int k = 0; k < (FULL ? 16 : 8); ++k) keep[k * blockDim.x] = 0.0f;
    ring.stage0 = memory + kept + (size_t)P.team * stages * stage_bytes;
    ring.full = full[P.team];
    ring.feeds = feeds[P.team];
    ring.stages = stages;
    ring.stage_bytes = stage_bytes;
    ring.open(arrays, strides, sizes, parts, true, c0, mine, d.rows, r0, r1, P.t, G.threads);
    if (P.R.ctas > 1) cg::this_cluster().sync();
    else __syncthreads();
    ring.template start<kFeeds>(P.t);

    // Threads behind the row's end read its last values (VECTOR) or what lies
    // there, and drop them (in warps that reach there: `ragged`).
    const bool ragged = (P.R.warp + 1) * 256 > mine;
    const int at = VECTOR ? min(cols.first - c0, mine - 8) : cols.first - c0;
    // Bytes by which the arrays' rows start behind a 16-byte boundary.
    unsigned shifts[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        shifts[k] = VECTOR ? 0 : (unsigned)((uintptr_t)arrays[k] + (c0 + r0 * strides[k]) * sizes[k]) & 15;
    }
    F8 acc[kKinds], group[GROUPED ? 2 : 1], kp, kb, kw;
#pragma unroll
    for (int j = 0; j < kKinds; ++j) fill(acc[j], 0.0f);
#pragma unroll
    for (int j = 0; j < (GROUPED ? 2 : 1); ++j) fill(group[j], 0.0f);
    parameters(d.pre_weight, pb, cols, 1.0f, kw);
    XT* xo = static_cast<XT*>(g.grad_x) + r0 * d.dim;
    HT* ho = static_cast<HT*>(g.grad_h) + r0 * d.dim;
    const float a = has_h ? d.residual_scale : 1.0f;
    int64_t turn = r0, k0 = 0;   // the row at which another row of the gate begins; this one's
    const void* gate = d.gate;
    // The rows of every CTA of a cluster are the same, so all take part in its sums.
    for (int64_t r = r0; r < r1; ++r, xo += d.dim, ho += d.dim) {
        if (r == turn) {
            if (GROUPED) {
                k0 = r / per;
                gate = static_cast<const char*>(d.gate) + k0 * d.dim * (pb ? 2 : 4);
            }
            fill(kp, 0.0f);
            fill(kb, 0.0f);
            if (has_h) post_parameters<FULL>(d, gate, pb, cols, kp, kb);
            turn = GROUPED ? (k0 + 1) * per : r1;
        }
        const char* s0 = ring.row();
        const float4 st = ring.lost ? make_float4(CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F)
                                    : *reinterpret_cast<const float4*>(s0 + at_st);
        F8 hh, xh, dx, dn;
        const HT* gnr = reinterpret_cast<const HT*>(s0 + at_gn + shifts[2]);
        const XT* gxr = reinterpret_cast<const XT*>(s0 + at_gx + shifts[3]);
        from_shared<XT, VECTOR>(reinterpret_cast<const XT*>(s0 + at_x + shifts[1]), at, xh);
        from_shared<HT, VECTOR>(gnr, at, dn);
        from_shared<XT, VECTOR>(gxr, at, dx);
        from_shared<HT, VECTOR>(reinterpret_cast<const HT*>(s0 + shifts[0]), at, hh);
        if (ragged) {
            within_row(xh, cols);
            within_row(dn, cols);
            within_row(dx, cols);
            within_row(hh, cols);
        }
        const float rx = has_gn ? st.w : 0.0f;
        float2 s2[FULL ? 8 : 3];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (FULL) hh[j] = add(hh[j], both(-st.x));
            hh[j] = mul(hh[j], both(st.y));
            const float2 q = mul(kp[j], hh[j]), e = mul(dn[j], kw[j]);
            if (FULL) xh[j] = fma(both(a), xh[j], add(add(kb[j], both(-st.z)), q));
            else xh[j] = fma(both(a), xh[j], q);
            xh[j] = mul(xh[j], both(st.w));
            const auto take = [&](int i, float2 x, float2 y) { s2[i] = j == 0 ? mul(x, y) : fma(x, y, s2[i]); };
            const float2 f = fma(both(rx), e, dx[j]);
            take(0, e, xh[j]);
            take(1, f, q);
            take(2, xh[j], q);
            if constexpr (FULL) {
                s2[3] = j == 0 ? e : add(s2[3], e);
                s2[4] = j == 0 ? q : add(s2[4], q);
                take(5, f, kp[j]);
                take(6, xh[j], kp[j]);
                s2[7] = j == 0 ? kp[j] : add(s2[7], kp[j]);
            }
        }
        float s[1 << kLog] = {};
#pragma unroll
        for (int j = 0; j < (FULL ? 8 : 3); ++j) s[j] = s2[j].x + s2[j].y;
        P.R.template sum<kLog>(s);
        // Every thread is past the row before (a warp alone: in step): its stage is free.
        if (G.threads == 32) __syncwarp();
        if (P.R.warp == 0) ring.copy_row(P.t);
        const float m1 = s[0] * inv;
        float m0 = 0.0f, u0 = 0.0f, u1 = fmaf(-rx * m1, s[2], s[1]);
        if constexpr (FULL) {
            if (layer) {
                m0 = s[3] * inv;
                u1 = fmaf(-rx * m0, s[4], u1);
                u0 = fmaf(-rx * m0, s[7], fmaf(-rx * m1, s[6], s[5])) * inv;
            }
        }
        u1 *= inv;
        F8 o;
        if (FULL) {   // read again: the registers were the sums'
            from_shared<HT, VECTOR>(gnr, at, dn);
            from_shared<XT, VECTOR>(gxr, at, dx);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 y = fma(dn[j], kw[j], both(-m0));
            y = fma(xh[j], both(-m1), y);
            dx[j] = fma(both(rx), y, dx[j]);   // the whole gradient of x_new
            acc[kPre][j] = fma(dn[j], xh[j], acc[kPre][j]);
            if (FULL) acc[FULL ? kPreBias : 0][j] = add(acc[FULL ? kPreBias : 0][j], dn[j]);
            o[j] = mul(both(a), dx[j]);
        }
        store(xo, cols, o, ragged);
        if (has_h) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = mul(dx[j], kp[j]);
                if (FULL) o[j] = add(o[j], both(-u0));
                o[j] = mul(both(st.y), fma(hh[j], both(-u1), o[j]));
                if constexpr (GROUPED) {
                    group[0][j] = fma(dx[j], hh[j], group[0][j]);
                    group[GROUPED ? 1 : 0][j] = add(group[GROUPED ? 1 : 0][j], dx[j]);
                } else {
                    acc[kPost][j] = fma(dx[j], hh[j], acc[kPost][j]);
                    if (FULL) acc[FULL ? kPostBias : 0][j] = add(acc[FULL ? kPostBias : 0][j], dx[j]);
                }
            }
            store(ho, cols, o, ragged);
        }
        if constexpr (GROUPED) {
            if (r + 1 == r1 || r + 1 == turn) {   // the group ends, or this team's part of it
                const int64_t first = k0 * per, last = first + per - 1;
                float* edge = nullptr;
                if (first < r0 || last >= r1) edge = W.edges + ((P.index * 2 + (first >= r0)) * 2) * d.dim;
                end_group<VECTOR, FULL>(g, gate, pb, cols, k0, edge, group, keep, blockDim.x);
            }
        }
        ring.next();
        if (!VECTOR)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                shifts[k] = (shifts[k] + (unsigned)strides[k] * sizes[k]) & 15;
    }
    ring.close(P.t);
    if constexpr (GROUPED) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            set(acc[kPost], k, keep[k * blockDim.x]);
            if (FULL) set(acc[kKinds - 1], k, keep[(8 + k) * blockDim.x]);
        }
    }
    __syncthreads();
    end_sums<VECTOR, kKinds>(P, G, W, (int)d.dim, reinterpret_cast<float*>(memory + kept), acc);
    if (P.R.ctas > 1) cg::this_cluster().sync();
}

template <typename XT, typename HT>
cudaError_t run_forward(const mdq_residual_norm_desc& d, const Teams& G, int chunks, int grid,
                        int cluster, cudaStream_t stream) {
    typedef void (*Kernel)(const mdq_residual_norm_desc, const Teams);
    const Kernel k = chunks == 1   ? (Kernel)norm_rows<XT, HT, 1>
                     : chunks == 2 ? (Kernel)norm_rows<XT, HT, 2>
                                   : (Kernel)norm_rows<XT, HT, 4>;
    return launch(k, dim3(grid), G.threads * G.teams, 0, stream, cluster, false, d, G);
}

template <typename XT, typename HT, bool VECTOR, bool FULL>
cudaError_t run_ring(const mdq_residual_norm_desc& d, const Teams& G, int chunks, int grid, int cluster,
                     int stages, size_t smem, cudaStream_t stream) {
    typedef void (*Kernel)(const mdq_residual_norm_desc, const Teams, int);
    const Kernel k = chunks == 1   ? (Kernel)norm_rows_ring<XT, HT, VECTOR, 1, FULL>
                     : chunks == 2 ? (Kernel)norm_rows_ring<XT, HT, VECTOR, 2, FULL>
                                   : (Kernel)norm_rows_ring<XT, HT, VECTOR, 4, FULL>;
    return launch<215 * 1024>(k, dim3(grid), G.threads * G.teams, smem, stream, cluster, false, d, G, stages);
}

template <typename XT, typename HT, bool VECTOR>
cudaError_t run_stream(const mdq_residual_norm_grad_desc& g, const Teams& G, const Partials& W,
                       int stages, size_t smem, int grid, int cluster, bool full, bool grouped,
                       cudaStream_t stream) {
    typedef void (*Kernel)(const mdq_residual_norm_grad_desc, const Teams, const Partials, int);
    const Kernel k = full ? (grouped ? (Kernel)norm_grad_stream<XT, HT, VECTOR, true, true>
                                     : (Kernel)norm_grad_stream<XT, HT, VECTOR, true, false>)
                          : (grouped ? (Kernel)norm_grad_stream<XT, HT, VECTOR, false, true>
                                     : (Kernel)norm_grad_stream<XT, HT, VECTOR, false, false>);
    return launch<205 * 1024>(k, dim3(grid), G.threads * G.teams, smem, stream, cluster, false, g, G, W,
                              stages);
}

template <typename XT, typename HT, bool VECTOR>
cudaError_t run_backward(const mdq_residual_norm_grad_desc& g, const Teams& G, const Partials& W,
                         int chunks, int grid, int cluster, bool full, bool grouped,
                         cudaStream_t stream) {
    const int kinds = grouped ? 6 : full ? 4 : 2;
    typedef void (*Kernel)(const mdq_residual_norm_grad_desc, const Teams, const Partials);
    const Kernel k = chunks == 2 ? (grouped ? (Kernel)norm_grad_rows<XT, HT, VECTOR, 2, true, true>
                                    : full  ? (Kernel)norm_grad_rows<XT, HT, VECTOR, 2, true, false>
                                            : (Kernel)norm_grad_rows<XT, HT, VECTOR, 2, false, false>)
                                 : (Kernel)norm_grad_rows<XT, HT, VECTOR, 4, false, false>;
    return launch<210 * 1024>(k, dim3(grid), G.threads * G.teams, sizeof(float) * kinds * G.share,
                              stream, cluster, false, g, G, W);
}

#define MDQ_NORM_TYPES(DECL)                                                                       \
    DECL(float, float, ff) DECL(float, __nv_bfloat16, fb) DECL(__nv_bfloat16, __nv_bfloat16, bb)   \
        DECL(__nv_bfloat16, float, bf)
#define MDQ_NORM_DECLARE(XT, HT, S)                                                                \
    cudaError_t forward_##S(const mdq_residual_norm_desc&, const Teams&, int, int, int, int,       \
                            size_t, bool, bool, cudaStream_t);                                     \
    cudaError_t backward_##S(const mdq_residual_norm_grad_desc&, const Teams&, const Partials&,    \
                             int, int, int, bool, bool, bool, cudaStream_t);                       \
    cudaError_t stream_##S(const mdq_residual_norm_grad_desc&, const Teams&, const Partials&, int, \
                           size_t, int, int, bool, bool, bool, cudaStream_t);
MDQ_NORM_TYPES(MDQ_NORM_DECLARE)

// The kernels of one pair of types (x, h), in a file of its own.
#define MDQ_NORM_INSTANTIATE(XT, HT, S)                                                            \
    namespace mdq_norm {                                                                           \
    cudaError_t forward_##S(const mdq_residual_norm_desc& d, const Teams& G, int chunks, int grid, \
                            int cluster, int stages, size_t smem, bool vector, bool full,          \
                            cudaStream_t stream) {                                                 \
        if (stages == 0) return run_forward<XT, HT>(d, G, chunks, grid, cluster, stream);          \
        return vector ? run_ring<XT, HT, true, true>(d, G, chunks, grid, cluster, stages, smem,    \
                                                     stream)                                       \
               : full ? run_ring<XT, HT, false, true>(d, G, chunks, grid, cluster, stages, smem,   \
                                                      stream)                                      \
                      : run_ring<XT, HT, false, false>(d, G, chunks, grid, cluster, stages, smem,  \
                                                       stream);                                    \
    }                                                                                              \
    cudaError_t backward_##S(const mdq_residual_norm_grad_desc& g, const Teams& G,                 \
                             const Partials& W, int chunks, int grid, int cluster, bool vector,    \
                             bool full, bool grouped, cudaStream_t stream) {                       \
        return vector ? run_backward<XT, HT, true>(g, G, W, chunks, grid, cluster, full, grouped,  \
                                                   stream)                                         \
                      : run_backward<XT, HT, false>(g, G, W, chunks, grid, cluster, full, grouped, \
                                                    stream);                                       \
    }                                                                                              \
    cudaError_t stream_##S(const mdq_residual_norm_grad_desc& g, const Teams& G, const Partials& W,\
                           int stages, size_t smem, int grid, int cluster, bool vector, bool full, \
                           bool grouped, cudaStream_t stream) {                                    \
        return vector ? run_stream<XT, HT, true>(g, G, W, stages, smem, grid, cluster, full,       \
                                                 grouped, stream)                                  \
                      : run_stream<XT, HT, false>(g, G, W, stages, smem, grid, cluster, full,      \
                                                  grouped, stream);                                \
    }                                                                                              \
    }

}  // namespace mdq_norm
