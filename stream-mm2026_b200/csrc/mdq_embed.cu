// mdq_embed.cu - scaled embedding lookup and its gradient (mdq_ops.h).
//
// Both are bound by memory: the lookup reads a table row and writes a row for
// every token; the gradient reads a row for every token and writes the dense
// [vocab, dim] result (or reads and writes the rows that occur).
//
// Gradient by sorted tokens, so that no floating-point atomics are needed and
// repeated calls give the same bits:
//   embed_grad_sort   sorts (id, position) pairs: clusters of up to 8 CTAs hold
//                     them in registers and shared memory and exchange them
//                     through distributed shared memory; the other CTAs of the
//                     launch meanwhile write the zeros of the dense result
//   embed_grad_sum    a team of threads adds the rows of a fixed-length chunk of
//                     the sorted list: a run of equal ids inside the chunk is
//                     complete and is written, one that crosses the chunk's
//                     edge leaves a partial sum.  Chunks of equal length keep
//                     the work even however often an id occurs.
//   embed_grad_join   adds the partial sums of the runs that cross edges
// A few tokens take one launch (embed_grad_few).
//
// Measured, bf16 rows and f32 tables, ids by word frequency: lookup of 8192 rows of
// 4096 from 32000, 22.0 us (9.2 TB/s: repeated ids come from L2), of 16384 rows of 768,
// 8.5; gradient of the latter into a dense 50257 x 768 result 23.6 (sort, under 154 MB
// of zeros at 6.5 TB/s) + 12.1 + 5.8; of the former added to a 32000 x 4096 gradient 8.5
// (sort) + 41.3 + 9.0, for 67 MB of rows and the 3264 rows of the gradient that occur,
// 53 MB read and 53 written.
#include "mdq_ops.cuh"

#include <cooperative_groups.h>
#include <utility>

namespace {

using namespace mdq_ops;
namespace cg = cooperative_groups;

// ------------------------------------------------------------------- lookup

// A warp takes up to 4 x 32 chunks of 8 columns of one row (grid.y: the slices
// of a row), or `1 << sub` lanes a narrow row.  VECTOR: chunks are 8 consecutive
// columns on 16-byte boundaries; otherwise 8 columns `lanes` apart.
constexpr int kLookupThreads = 256, kLookupIter = 4;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        Vec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(p)), v);
    } else {
        float a[4], b[4];
        Vec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(p)), a);
        Vec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(p) + 1), b);
#pragma unroll
        for (int k = 0; k < 4; ++k) { v[k] = a[k]; v[4 + k] = b[k]; }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(p) = Vec<T>::pack(v);
    } else {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
}

template <typename TT, typename OT, bool VECTOR>
__global__ void __launch_bounds__(kLookupThreads) embed_rows(const __grid_constant__
                                                             mdq_embed_desc d, int sub) {
    const int lanes = 1 << sub, lane = threadIdx.x & (lanes - 1);
    const int64_t n = (int64_t)blockIdx.x * (kLookupThreads >> sub) + (threadIdx.x >> sub);
    if (n >= d.tokens) return;
    const int64_t id = load_id(d.ids, d.ids_dtype == MDQ_I64, n);
    const bool in = id >= 0 && id < d.vocab;
    const TT* row = static_cast<const TT*>(d.table) + (in ? id : 0) * d.table_stride;
    OT* out = static_cast<OT*>(d.out) + n * d.dim;
    const int c0 = (int)blockIdx.y * kLookupIter * 8 * lanes, dim = (int)d.dim;
    if constexpr (VECTOR) {
        float v[kLookupIter][8] = {};
#pragma unroll
        for (int i = 0; i < kLookupIter; ++i) {
            const int c = c0 + (i * lanes + lane) * 8;
            if (in && c < dim) load8(row + c, v[i]);
        }
#pragma unroll
        for (int i = 0; i < kLookupIter; ++i) {
            const int c = c0 + (i * lanes + lane) * 8;
            if (c >= dim) break;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[i][k] *= d.scale;
            store8(out + c, v[i]);
        }
    } else {
        // 8 values in flight a thread; whole groups of columns without checks.
        const int end = min(dim, c0 + kLookupIter * 8 * lanes);
        for (int c = c0 + lane; c < end; c += 8 * lanes) {
            float v[8];
            if (c - lane + 8 * lanes <= end) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = in ? to_f(row[c + k * lanes]) : 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) out[c + k * lanes] = from_f<OT>(v[k] * d.scale);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = in && c + k * lanes < end ? to_f(row[c + k * lanes]) : 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (c + k * lanes < end) out[c + k * lanes] = from_f<OT>(v[k] * d.scale);
            }
        }
    }
}

// --------------------------------------------------------------------- sort

constexpr int kSortThreads = 1024, kSortWarps = 32;     // at most
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;   // radix digit
constexpr int kMaxCluster = 8;
constexpr int kSlab = kMaxCluster * kSortThreads * 16;  // tokens one cluster can sort

typedef unsigned long long Pair;   // id << 32 | position

// What the sort writes for every token that has no row (outside the
// vocabulary, or the padding id): it sorts behind all rows.
struct SortArgs {
    const void* ids;
    Pair* sorted;        // [tokens]
    int64_t tokens, vocab, padding_idx;
    int64_t slabs, fill_bytes;
    char* fill;          // zeros go here
    int32_t i64, passes, bits;
};

struct SortShared {
    unsigned count[kMaxCluster][kMaxBins];      // every CTA's digit counts
    unsigned base[kMaxBins];                    // first place of this CTA's digit
    unsigned scan[kSortWarps];
};
// Shared memory of the sort: the pairs, every warp's digit counts (then its offset
// within the CTA), and the rest.
size_t sort_shared(int threads, int ipt) {
    return sizeof(Pair) * threads * ipt + sizeof(uint16_t) * (threads / 32) * kMaxBins + sizeof(SortShared);
}

// Zeros a CTA writes: a few microseconds of an SM's share of the bandwidth, so
// that the hardware balances them over the SMs that do not sort.
constexpr int64_t kFillBytes = 256 * 1024;

__device__ __forceinline__ void fill_zeros(char* p, int64_t bytes, int thread, int threads) {
    // Edges up to 16-byte boundaries in 2-byte steps (bf16 is the smallest type).
    const int64_t head = min(bytes, (int64_t)(-(uintptr_t)p & 15));
    const int64_t body = (bytes - head) / 16, tail = bytes - head - 16 * body;
    if (thread < head / 2) reinterpret_cast<uint16_t*>(p)[thread] = 0;
    if (thread < tail / 2) reinterpret_cast<uint16_t*>(p + head + 16 * body)[thread] = 0;
    uint4* q = reinterpret_cast<uint4*>(p + head);
#pragma unroll 4
    for (int i = thread; i < (int)body; i += threads) __stcs(q + i, make_uint4(0, 0, 0, 0));
}

// Stable least-significant-digit radix sort of one slab of up to C * threads * IPT
// tokens by a cluster of C CTAs.  A warp's items are consecutive tokens, so
// (CTA, warp, item, lane) is the tokens' order and ranks taken in that order
// keep it.  Ranks within a warp come from ballots over the digit's bits and a
// per-warp histogram; counts cross CTAs through distributed shared memory, and so do the pairs
// (except after the last pass, which writes them to global memory).
template <int IPT>
__global__ void __launch_bounds__(kSortThreads) embed_grad_sort(const __grid_constant__ SortArgs a) {
    extern __shared__ __align__(16) char raw[];
    const int threads = blockDim.x, warps = threads >> 5;
    Pair* buf = reinterpret_cast<Pair*>(raw);                       // [threads * IPT]
    SortShared& S = *reinterpret_cast<SortShared*>(raw + sizeof(Pair) * threads * IPT);
    uint16_t* hist = reinterpret_cast<uint16_t*>(&S + 1);           // [warps][bins]
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int64_t slab = blockIdx.x / C;
    if (slab >= a.slabs) {   // whole clusters: the dense result's zeros, kFillBytes a CTA
        const int64_t from = (blockIdx.x - a.slabs * C) * kFillBytes;
        if (from < a.fill_bytes)
            fill_zeros(a.fill + from, min(kFillBytes, a.fill_bytes - from), threadIdx.x, threads);
        return;
    }
    // Every CTA of the cluster runs before its shared memory is written to.
    auto started = cluster.barrier_arrive();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int items = threads * IPT;
    const int64_t first = slab * kSlab;
    const int64_t left = min(a.tokens - first, (int64_t)kSlab);     // of this slab
    const int own = rank * items;                                  // this CTA's first place
    const int at = w * 32 * IPT + lane;                             // item j is at + 32 j

    Pair item[IPT];
#pragma unroll
    for (int j = 0; j < IPT; ++j) {
        const int64_t i = own + at + 32 * j;
        int64_t id = a.vocab;
        if (i < left) {
            id = load_id(a.ids, a.i64, first + i);
            if (id < 0 || id > a.vocab || id == a.padding_idx) id = a.vocab;
        }
        item[j] = (Pair)id << 32 | (unsigned)(first + i);
    }
    const int bins = 1 << a.bits;
    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = 32 + pass * a.bits;
        uint16_t* mine = hist + w * bins;
        for (int i = lane; i < bins / 2; i += 32) reinterpret_cast<unsigned*>(mine)[i] = 0;
        __syncwarp();
        uint16_t place[IPT];
#pragma unroll
        for (int j = 0; j < IPT; ++j) {
            const int digit = (int)(item[j] >> shift) & (bins - 1);
            // Lanes of the same digit, a ballot for each of its bits.
            unsigned same = 0xffffffffu;
            for (int b = 0; b < a.bits; ++b) {
                const unsigned one = __ballot_sync(0xffffffffu, digit >> b & 1);
                same &= digit >> b & 1 ? one : ~one;
            }
            const int before = __popc(same & ((1u << lane) - 1));
            const uint16_t seen = mine[digit];
            place[j] = seen + before;
            __syncwarp();
            if (before == 0) mine[digit] = seen + __popc(same);
            __syncwarp();
        }
        __syncthreads();
        // Offsets of the warps within the CTA; the CTA's counts go to every CTA.
        // (Fewer threads than digits take several each.)
        if (pass == 0) cluster.barrier_wait(std::move(started));
        for (int b = tid; b < bins; b += threads) {
            unsigned total = 0;
            for (int k0 = 0; k0 < warps; k0 += 8) {
                uint16_t c[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) c[k] = k0 + k < warps ? hist[(k0 + k) * bins + b] : 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (k0 + k < warps) hist[(k0 + k) * bins + b] = (uint16_t)total;
                    total += c[k];
                }
            }
            for (int r = 0; r < C; ++r) cluster.map_shared_rank(&S.count[rank][b], r)[0] = total;
        }
        cluster.sync();
        // First place of this CTA's digit: all smaller digits, and the digit in
        // the CTAs before.  Thread t has the digits from t * each on.
        const int each = (bins + threads - 1) / threads;
        unsigned all = 0;
        for (int b = tid * each; b < min(bins, (tid + 1) * each); ++b)
            for (int r = 0; r < C; ++r) all += S.count[r][b];
        unsigned run = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        if (lane == 31) S.scan[w] = run;
        __syncthreads();
        unsigned upto = run - all;
        {
            unsigned v = lane < w ? S.scan[lane] : 0;   // the warps before
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            upto += v;
        }
        for (int b = tid * each; b < min(bins, (tid + 1) * each); ++b) {
            unsigned before = 0, here = 0;
            for (int r = 0; r < C; ++r) {
                const unsigned c = S.count[r][b];
                if (r < rank) before += c;
                here += c;
            }
            S.base[b] = upto + before;
            upto += here;
        }
        __syncthreads();
        const bool last = pass + 1 == a.passes;
#pragma unroll
        for (int j = 0; j < IPT; ++j) {
            const int digit = (int)(item[j] >> shift) & (bins - 1);
            const unsigned to = S.base[digit] + mine[digit] + place[j];
            if (last) {
                if (to < left) a.sorted[first + to] = item[j];
            } else {
                cluster.map_shared_rank(buf, to / items)[to % items] = item[j];
            }
        }
        if (last) break;
        cluster.sync();
#pragma unroll
        for (int j = 0; j < IPT; ++j) item[j] = buf[at + 32 * j];
        // No pair of the next pass is written before its cluster.sync(), which
        // follows these reads.
    }
}

// ---------------------------------------------------------------------- sum

constexpr int kUnroll = 8;

struct SumArgs {
    const Pair* sorted;     // [tokens] of this slab
    const void* grad_out;
    void* grad;
    float* partial;         // [chunks][2][dim]: sums of runs from before, and of runs that go on
    int64_t grad_out_stride, dim, vocab;
    int32_t tokens, chunk, chunks;
    int32_t tx;             // threads of a team, each with VEC columns
    float scale;
    int32_t accumulate;
};

// Thread t of a team owns columns c0 + t VEC + k (VECTOR) or c0 + k tx + t.
template <typename GT, bool VECTOR>
struct Columns {
    static constexpr int N = Vec<GT>::N;
    int64_t first, step, dim;
    __device__ Columns(int64_t slice, int t, int tx, int64_t d)
        : first(slice * tx * N + (VECTOR ? t * N : t)), step(VECTOR ? 1 : tx), dim(d) {}
    __device__ bool any() const { return first < dim; }
    __device__ bool has(int k) const { return first + k * step < dim; }
    __device__ int64_t at(int k) const { return first + k * step; }
};

template <typename GT, bool VECTOR>
struct RawRow {   // a row's values as loaded
    uint4 v;
    __device__ void load(const GT* row, const Columns<GT, true>& c) {
        v = __ldcs(reinterpret_cast<const uint4*>(row + c.first));
    }
    __device__ void add(float (&acc)[Vec<GT>::N]) const {
        float f[Vec<GT>::N];
        Vec<GT>::unpack(v, f);
#pragma unroll
        for (int k = 0; k < Vec<GT>::N; ++k) acc[k] += f[k];
    }
};
template <typename GT>
struct RawRow<GT, false> {
    GT v[Vec<GT>::N];
    __device__ void load(const GT* row, const Columns<GT, false>& c) {
#pragma unroll
        for (int k = 0; k < Vec<GT>::N; ++k) v[k] = c.has(k) ? row[c.at(k)] : from_f<GT>(0.0f);
    }
    __device__ void add(float (&acc)[Vec<GT>::N]) const {
#pragma unroll
        for (int k = 0; k < Vec<GT>::N; ++k) acc[k] += to_f(v[k]);
    }
};

// A finished sum to its row of the gradient.
template <typename GT, typename WT, bool VECTOR>
__device__ __forceinline__ void write_row(const SumArgs& a, unsigned id,
                                          const Columns<GT, VECTOR>& c,
                                          const float (&acc)[Vec<GT>::N]) {
    constexpr int N = Vec<GT>::N;
    WT* row = static_cast<WT*>(a.grad) + (int64_t)id * a.dim;
    if constexpr (VECTOR) {
        constexpr int M = N < Vec<WT>::N ? N : Vec<WT>::N;   // values of one store
#pragma unroll
        for (int k = 0; k < N; k += M) {
            float v[M];
#pragma unroll
            for (int j = 0; j < M; ++j) v[j] = acc[k + j] * a.scale;
            WT* p = row + c.first + k;
            if constexpr (sizeof(WT) == 4) {
                // Added by the L2 cache, so that no load is waited for; every
                // element is added to once, so the order does not matter.
                // (Subnormal values count as zero there.)
                if (a.accumulate)
                    asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(v[0]),
                                 "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
                else
                    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            } else if constexpr (M == 8) {
                *reinterpret_cast<uint4*>(p) = Vec<WT>::pack(v);
            } else {
                *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (c.has(k)) {
                WT* p = row + c.at(k);
                if constexpr (sizeof(WT) == 4)
                    if (a.accumulate) {
                        atomicAdd(p, acc[k] * a.scale);   // as above
                        continue;
                    }
                *p = from_f<WT>(acc[k] * a.scale);
            }
    }
}

template <typename GT, bool VECTOR>
__device__ __forceinline__ void write_partial(float* p, const Columns<GT, VECTOR>& c,
                                              const float (&acc)[Vec<GT>::N]) {
#pragma unroll
    for (int k = 0; k < Vec<GT>::N; ++k)
        if (VECTOR || c.has(k)) p[c.at(k)] = acc[k];
}

template <typename GT, typename WT, bool VECTOR>
__global__ void __launch_bounds__(256) embed_grad_sum(const __grid_constant__ SumArgs a) {
    extern __shared__ Pair pairs[];   // of the block's chunks
    const int teams = blockDim.x / a.tx, team = threadIdx.x / a.tx, t = threadIdx.x - team * a.tx;
    const int64_t c = (int64_t)blockIdx.x * teams + team;
    const Columns<GT, VECTOR> col(blockIdx.y, t, a.tx, a.dim);
    wait_previous();
    const int block0 = (int)blockIdx.x * teams * a.chunk;
    for (int i = threadIdx.x; i < teams * a.chunk && block0 + i < a.tokens; i += blockDim.x)
        pairs[i] = a.sorted[block0 + i];
    __syncthreads();
    if (c >= a.chunks || !col.any()) return;
    const int i0 = (int)c * a.chunk, i1 = min(a.tokens, i0 + a.chunk);
    const Pair* own = pairs - block0;
    const GT* rows = static_cast<const GT*>(a.grad_out);
    float* partial = a.partial + 2 * c * a.dim;
    constexpr int N = Vec<GT>::N;
    float acc[N] = {};
    unsigned id = (unsigned)(own[i0] >> 32);
    bool before = i0 > 0 && (unsigned)(a.sorted[i0 - 1] >> 32) == id;   // the run began earlier
    for (int i = i0; i < i1; i += kUnroll) {
        Pair e[kUnroll];
        RawRow<GT, VECTOR> r[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) e[u] = own[min(i + u, i1 - 1)];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (i + u < i1 && (e[u] >> 32) < (Pair)a.vocab)
                r[u].load(rows + (int64_t)(unsigned)e[u] * a.grad_out_stride, col);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (i + u >= i1) break;
            const unsigned k = (unsigned)(e[u] >> 32);
            if (k != id) {
                if (before) write_partial(partial, col, acc);
                else write_row<GT, WT, VECTOR>(a, id, col, acc);
                before = false;
                id = k;
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] = 0.0f;
            }
            if (id >= a.vocab) return;   // the rest has no row
            r[u].add(acc);
        }
    }
    const bool after = i1 < a.tokens && (unsigned)(a.sorted[i1] >> 32) == id;
    if (before) write_partial(partial, col, acc);
    else if (after) write_partial(partial + a.dim, col, acc);
    else write_row<GT, WT, VECTOR>(a, id, col, acc);
}

// Runs that cross chunk edges: a block takes the edges at which such a run
// leaves the chunk it began in, adds that chunk's second partial and the first
// partials of the chunks it goes through, each team a contiguous part of them,
// and the teams' sums in order.
template <typename GT, typename WT, bool VECTOR>
__global__ void __launch_bounds__(1024) embed_grad_join(const __grid_constant__ SumArgs a) {
    extern __shared__ float sums[];   // [teams][tx * VEC]
    constexpr int N = Vec<GT>::N;
    const int teams = blockDim.x / a.tx, team = threadIdx.x / a.tx, t = threadIdx.x - team * a.tx;
    const Columns<GT, VECTOR> col(blockIdx.y, t, a.tx, a.dim);
    wait_previous();
    for (int b = blockIdx.x; b < a.chunks - 1; b += gridDim.x) {
        // What decides about the edge is loaded at once: the pairs on both sides of
        // it, the one before this chunk, and the first pairs of the next 32 chunks.
        const int64_t edge = (int64_t)(b + 1) * a.chunk, i0 = edge - a.chunk;
        int64_t next = (int64_t)(b + 2 + (threadIdx.x & 31)) * a.chunk;
        const auto id_at = [&](int64_t i) { return (unsigned)(a.sorted[i] >> 32); };
        const unsigned id = id_at(edge), left = id_at(edge - 1), before = i0 > 0 ? id_at(i0 - 1) : 0xffffffffu;
        unsigned ahead = next < a.tokens ? id_at(next) : 0xffffffffu;
        if (id >= a.vocab || left != id || before == id) continue;   // none crosses, or it began earlier
        // The last chunk that the run reaches, 32 chunks at a time.
        int end = b + 1;
        while (true) {
            const unsigned mask = __ballot_sync(0xffffffffu, ahead == id);
            const int more = mask == 0xffffffffu ? 32 : __ffs(~mask) - 1;
            end += more;
            if (more < 32) break;
            next += 32 * (int64_t)a.chunk;
            ahead = next < a.tokens ? id_at(next) : 0xffffffffu;
        }
        // Parts b (its second partial), b + 1, ..., end (their first).
        const int parts = end - b + 1, each = (parts + teams - 1) / teams;
        float acc[N] = {};
        if (col.any()) {
            const int p0 = team * each, p1 = min(parts, p0 + each);
            for (int p = p0; p < p1; p += 4) {
                float v[4][N];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float* q = a.partial + (2 * (int64_t)(b + p + u) + (p + u == 0)) * a.dim;
#pragma unroll
                    for (int k = 0; k < N; ++k)
                        v[u][k] = p + u < p1 && (VECTOR || col.has(k)) ? q[col.at(k)] : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int k = 0; k < N; ++k) acc[k] += v[u][k];
            }
        }
#pragma unroll
        for (int k = 0; k < N; ++k) sums[(team * N + k) * a.tx + t] = acc[k];
        __syncthreads();
        if (team == 0 && col.any()) {
            for (int y = 1; y < teams; ++y)
#pragma unroll
                for (int k = 0; k < N; ++k) acc[k] += sums[(y * N + k) * a.tx + t];
            write_row<GT, WT, VECTOR>(a, id, col, acc);
        }
        __syncthreads();
    }
}

// The sums over several slabs into their result, or added to it (rows without a
// token have sums of zero, and are not touched).
template <typename WT, bool ADD>
__global__ void __launch_bounds__(256) embed_grad_finish(const float* from, WT* to, int64_t n) {
    wait_previous();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const float v = from[i];
        if constexpr (!ADD) to[i] = from_f<WT>(v);
        else if (v != 0.0f) to[i] += v;
    }
}

// ---------------------------------------------------------------- few tokens

constexpr int kFew = 512, kFewThreads = 512, kFewRows = 1024;

// Block n < tokens owns the row of ids[n] if no earlier token has the same id:
// it adds the rows of all tokens with that id, its teams of tx threads each a
// contiguous part of them, and the teams' sums in order.  The other blocks write
// the zeros of the rows that do not occur.
template <typename GT, typename WT, bool VECTOR>
__global__ void __launch_bounds__(kFewThreads) embed_grad_few(const __grid_constant__ SumArgs a,
                                                              const void* ids, int i64,
                                                              int64_t padding_idx) {
    constexpr int N = Vec<GT>::N;
    __shared__ int64_t id[kFew];
    __shared__ union {
        uint8_t present[kFewRows];
        float sums[kFewThreads * N];
    } s;
    __shared__ int where[kFew], count;
    const int tid = threadIdx.x, n = a.tokens;
    for (int i = tid; i < n; i += kFewThreads) {
        const int64_t v = load_id(ids, i64, i);
        id[i] = v < 0 || v >= a.vocab || v == padding_idx ? -1 : v;
    }
    __syncthreads();
    if ((int)blockIdx.x < n) {
        const int64_t mine = id[blockIdx.x];
        if (mine < 0) return;
        if (tid < 32) {   // the positions with this id, in order
            int found = 0;
            for (int i = 0; i < n; i += 32) {
                const bool hit = i + tid < n && id[i + tid] == mine;
                const unsigned m = __ballot_sync(0xffffffffu, hit);
                if (hit) where[found + __popc(m & ((1u << tid) - 1))] = i + tid;
                found += __popc(m);
            }
            if (tid == 0) count = found;
        }
        __syncthreads();
        if (where[0] != (int)blockIdx.x) return;
        const GT* rows = static_cast<const GT*>(a.grad_out);
        const int teams = kFewThreads / a.tx, team = tid / a.tx, t = tid - team * a.tx;
        const int hits = count, each = (hits + teams - 1) / teams;
        const int i0 = team * each, i1 = min(hits, i0 + each);   // none for threads left over
        for (int64_t slice = 0; slice * a.tx * N < a.dim; ++slice) {
            const Columns<GT, VECTOR> col(slice, t, a.tx, a.dim);
            float acc[N] = {};
            if (col.any() && team < teams)
                for (int i = i0; i < i1; i += kUnroll) {
                    RawRow<GT, VECTOR> r[kUnroll];
#pragma unroll
                    for (int u = 0; u < kUnroll; ++u)
                        if (i + u < i1) r[u].load(rows + (int64_t)where[i + u] * a.grad_out_stride, col);
#pragma unroll
                    for (int u = 0; u < kUnroll; ++u)
                        if (i + u < i1) r[u].add(acc);
                }
            if (hits > each) {   // more than one team has a part
#pragma unroll
                for (int k = 0; k < N; ++k) s.sums[k * kFewThreads + tid] = acc[k];
                __syncthreads();
                if (team == 0)
                    for (int y = 1; y * each < hits; ++y)
#pragma unroll
                        for (int k = 0; k < N; ++k) acc[k] += s.sums[k * kFewThreads + y * a.tx + t];
                __syncthreads();
            }
            if (team == 0 && col.any()) write_row<GT, WT, VECTOR>(a, (unsigned)mine, col, acc);
        }
        return;
    }
    const int64_t blocks = gridDim.x - n, each = (a.vocab + blocks - 1) / blocks;
    const int64_t r0 = (blockIdx.x - n) * each, r1 = min(a.vocab, r0 + each);
    for (int64_t r = r0; r < r1; r += kFewRows) {
        const int64_t e = min(r1, r + kFewRows);
        for (int i = tid; i < kFewRows; i += kFewThreads) s.present[i] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kFewThreads)
            if (id[i] >= r && id[i] < e) s.present[id[i] - r] = 1;
        __syncthreads();
        for (int64_t k = r + (tid >> 5); k < e; k += kFewThreads / 32) {
            if (s.present[k - r]) continue;
            WT* row = static_cast<WT*>(a.grad) + k * a.dim;
            if constexpr (VECTOR) {
                constexpr int M = 16 / sizeof(WT);
                for (int64_t c = (tid & 31) * M; c < a.dim; c += 32 * M)
                    __stcs(reinterpret_cast<uint4*>(row + c), make_uint4(0, 0, 0, 0));
            } else {
                for (int64_t c = tid & 31; c < a.dim; c += 32) row[c] = from_f<WT>(0.0f);
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ planning

// Pairs of a chunk: about 65536 threads over all teams, 8 to 64 rows each; at most
// 32 above 2048 columns, where many threads share a row anyway, and 16 where a
// block has many teams, whose pairs it keeps in shared memory.  Sum and join of
// 16384 rows of 768 with 16 / 32 a chunk: 19.5 / 17.7 us, of 8192 rows of 4096 with
// 32 / 64: 50 / 56, of 32768 rows of 1024: 44 / 34.
int chunk_of(int64_t tokens, int64_t dim) {
    const int64_t want = tokens * ceil_div(dim, 8) / 65536, most = dim < 256 ? 16 : dim > 2048 ? 32 : 64;
    int c = 8;
    while (c < most && c < want) c *= 2;
    return c;
}

// One launch instead of three: up to kFew tokens, half as many above 1024 columns,
// where the rows of an id that occurs often take longer (one block adds them).
// Calls for bf16 rows, ids by word frequency, added to a gradient of 32000 or 50257
// rows: 8 tokens of 768, 7.1 us against 13.9; 512 of 768, 12.6 against 16 to 21; 256 of
// 4096, 10.4 against 16.2, and of one id for all 256, 43 against 17.  A dense gradient of
// 50257 rows, which is mostly zeros: 27 against 31, 35.2 against 33.5, 134 against 127.
bool few(int64_t tokens, int64_t dim) { return tokens <= (dim <= 1024 ? kFew : kFew / 2); }

struct Layout {   // of the workspace
    int64_t slabs, slab_tokens, chunk, chunks;
    int64_t partial_at, wide_at, bytes;
};

Layout layout_of(int64_t tokens, int64_t vocab, int64_t dim) {
    Layout L = {};
    if (few(tokens, dim)) return L;
    L.slabs = ceil_div(tokens, kSlab);
    L.slab_tokens = tokens < kSlab ? tokens : kSlab;
    L.chunk = chunk_of(L.slab_tokens, dim);
    L.chunks = ceil_div(L.slab_tokens, L.chunk);
    L.partial_at = ceil_div(tokens * (int64_t)sizeof(Pair), 16) * 16;
    L.wide_at = L.partial_at + ceil_div(2 * L.chunks * dim * (int64_t)sizeof(float), 16) * 16;
    // Several slabs are added in fp32 before a bf16 result is rounded, or before
    // they are added to a gradient.
    L.bytes = L.wide_at + (L.slabs > 1 ? vocab * dim * (int64_t)sizeof(float) : 0);
    return L;
}

// Threads over the columns of a row, and the slices of a row: whole warps, or a
// power of two below one.
void team_of(int64_t dim, int vec, int* tx, int64_t* slices) {
    const int64_t chunks = ceil_div(dim, vec);
    if (chunks <= 16) {
        *tx = 1;
        while (*tx < chunks) *tx *= 2;
        *slices = 1;
        return;
    }
    *slices = ceil_div(chunks, 128);
    *tx = (int)ceil_div(ceil_div(chunks, *slices), 32) * 32;
    *slices = ceil_div(chunks, *tx);
}

template <typename GT, typename WT, bool VECTOR>
mdq_status sum_slab(const SumArgs& a, int64_t slices, cudaStream_t stream) {
    const int teams = 256 / a.tx > 0 ? 256 / a.tx : 1;
    cudaError_t e = launch(embed_grad_sum<GT, WT, VECTOR>,
                           dim3((unsigned)ceil_div(a.chunks, teams), (unsigned)slices),
                           teams * a.tx, sizeof(Pair) * teams * a.chunk, stream, 1, true, a);
    if (e != cudaSuccess || a.chunks < 2) return status_of(e, "embed grad");
    // whole warps: embed_grad_join votes
    const int joiners = a.tx >= 64 ? 512 / a.tx : a.tx >= 4 ? 8 : 32 / a.tx;
    const int edges = a.chunks - 1;
    e = launch(embed_grad_join<GT, WT, VECTOR>,
               dim3((unsigned)(edges < 65536 ? edges : 65536), (unsigned)slices),
               joiners * a.tx, sizeof(float) * joiners * a.tx * Vec<GT>::N, stream, 1, true, a);
    return status_of(e, "embed grad");
}

// One combination of types: few tokens in one launch, else the sums of all slabs.
template <typename GT, typename WT, bool VECTOR>
mdq_status run_grad(const mdq_embed_grad_desc& d, SumArgs a, const Layout& L, cudaStream_t stream) {
    int64_t slices = 0;
    team_of(d.dim, Vec<GT>::N, &a.tx, &slices);
    if (few(d.tokens, d.dim)) {
        // most ids occur once, and then one team works: wider than the sums'
        if (slices > 1) a.tx = kFewThreads / 2;
        int64_t fill = 0;
        if (!d.accumulate) {
            fill = ceil_div(d.vocab, kFewThreads / 32);   // a row for each warp
            fill = fill < 148 * 4 ? fill : 148 * 4;
        }
        if (d.tokens + fill == 0) return MDQ_OK;
        return status_of(launch(embed_grad_few<GT, WT, VECTOR>, dim3((unsigned)(d.tokens + fill)),
                                kFewThreads, 0, stream, 1, false, a, d.ids,
                                (int)(d.ids_dtype == MDQ_I64), d.padding_idx),
                         "embed grad");
    }
    for (int64_t s = 0; s < L.slabs; ++s) {
        const int64_t left = d.tokens - s * kSlab;
        a.sorted = static_cast<const Pair*>(d.workspace) + s * kSlab;
        a.tokens = (int32_t)(left < kSlab ? left : kSlab);
        a.chunk = (int32_t)L.chunk;
        a.chunks = (int32_t)ceil_div(a.tokens, L.chunk);
        a.accumulate = a.accumulate || s > 0;
        const mdq_status st = sum_slab<GT, WT, VECTOR>(a, slices, stream);
        if (st != MDQ_OK) return st;
    }
    return MDQ_OK;
}

template <typename GT, typename WT>
mdq_status run_grad(const mdq_embed_grad_desc& d, const SumArgs& a, const Layout& L,
                    cudaStream_t stream) {
    // 16-byte loads of grad_out and stores of the gradient: every row of both
    // starts on 16 bytes and is a whole number of them
    const bool vec = rows16(d.grad_out, d.grad_out_stride, d.grad_out_dtype) &&
                     aligned16(a.grad) && d.dim % Vec<GT>::N == 0 && d.dim % Vec<WT>::N == 0;
    return vec ? run_grad<GT, WT, true>(d, a, L, stream) : run_grad<GT, WT, false>(d, a, L, stream);
}

template <int IPT>
mdq_status run_sort(const SortArgs& a, int cluster, int threads, cudaStream_t stream) {
    const size_t smem = sort_shared(threads, IPT);
    const int64_t grid = (a.slabs + ceil_div(ceil_div(a.fill_bytes, kFillBytes), cluster)) * cluster;
    if (grid > INT32_MAX) return mdq_fail(MDQ_ERR_TOO_LARGE, "embed grad: gradient too large");
    return status_of(launch(embed_grad_sort<IPT>, dim3((unsigned)grid), threads, smem, stream,
                            cluster, false, a),
                     "embed grad sort");
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
    if (d->dim > (int64_t)1024 * 65535 - 1024)   // slices of a row in grid.y
        return mdq_fail(MDQ_ERR_TOO_LARGE, "embed: 67106816 columns at most");
    if (d->tokens == 0) return MDQ_OK;
    if (d->table == nullptr || d->ids == nullptr || d->out == nullptr)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "embed: null pointer");
    int sub = 0;
    while (sub < 5 && (8 << sub) < d->dim) ++sub;
    const dim3 grid((unsigned)ceil_div(d->tokens, kLookupThreads >> sub),
                    (unsigned)ceil_div(d->dim, (int64_t)kLookupIter * 8 << sub));
    const bool vec = d->dim % 8 == 0 && aligned16(d->out) &&
                     rows16(d->table, d->table_stride, d->table_dtype);
    const bool tb = d->table_dtype == MDQ_BF16, ob = d->out_dtype == MDQ_BF16;
    typedef void (*Kernel)(const mdq_embed_desc, int);
    typedef __nv_bfloat16 B;
    const Kernel k =
        vec ? (tb ? (ob ? (Kernel)embed_rows<B, B, true> : (Kernel)embed_rows<B, float, true>)
                  : (ob ? (Kernel)embed_rows<float, B, true> : (Kernel)embed_rows<float, float, true>))
            : (tb ? (ob ? (Kernel)embed_rows<B, B, false> : (Kernel)embed_rows<B, float, false>)
                  : (ob ? (Kernel)embed_rows<float, B, false> : (Kernel)embed_rows<float, float, false>));
    return status_of(launch(k, grid, kLookupThreads, 0, stream, 1, false, *d, sub), "embed");
}

mdq_status mdq_embed_grad_workspace_bytes(int64_t tokens, int64_t vocab, int64_t dim,
                                          int64_t* bytes) {
    mdq_clear_error();
    if (bytes == nullptr || tokens < 0 || vocab < 1 || dim < 1)
        return mdq_fail(MDQ_ERR_INVALID_ARG, "embed grad: bad size");
    if (tokens > INT32_MAX || vocab > INT32_MAX - 1 || dim > (int64_t)512 * 65535)
        return mdq_fail(MDQ_ERR_TOO_LARGE, "embed grad: 2^31 tokens or ids, or 33553920 columns, or more");
    *bytes = layout_of(tokens, vocab, dim).bytes;
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
    int64_t need = 0;
    mdq_status st = mdq_embed_grad_workspace_bytes(d->tokens, d->vocab, d->dim, &need);
    if (st != MDQ_OK) return st;
    if (d->grad == nullptr || (d->tokens > 0 && (d->ids == nullptr || d->grad_out == nullptr)))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "embed grad: null pointer");
    if (need > 0 && (d->workspace == nullptr || d->workspace_bytes < need))
        return mdq_fail(MDQ_ERR_INVALID_ARG, "workspace holds %lld bytes, %lld needed",
                        (long long)d->workspace_bytes, (long long)need);
    if (!aligned16(d->workspace)) return mdq_fail(MDQ_ERR_INVALID_ARG, "workspace misaligned");

    const Layout L = layout_of(d->tokens, d->vocab, d->dim);
    char* ws = static_cast<char*>(d->workspace);
    const bool wide = L.slabs > 1 && (d->grad_dtype == MDQ_BF16 || d->accumulate);
    const int32_t wt = wide ? (int32_t)MDQ_F32 : d->grad_dtype;
    SumArgs a = {};
    a.grad_out = d->grad_out;
    a.grad = wide ? ws + L.wide_at : d->grad;
    a.partial = reinterpret_cast<float*>(ws + L.partial_at);
    a.grad_out_stride = d->grad_out_stride;
    a.dim = d->dim;
    a.vocab = d->vocab;
    a.tokens = (int32_t)d->tokens;
    a.scale = d->scale;
    a.accumulate = d->accumulate && !wide;
    if (L.slabs > 0) {
        SortArgs s = {};
        s.ids = d->ids;
        s.sorted = reinterpret_cast<Pair*>(ws);
        s.tokens = d->tokens;
        s.vocab = d->vocab;
        s.padding_idx = d->padding_idx;
        s.slabs = L.slabs;
        s.i64 = d->ids_dtype == MDQ_I64;
        int bits = 1;
        while (bits < 32 && (d->vocab >> bits) != 0) ++bits;   // ids up to vocab itself
        s.passes = (bits + kMaxBits - 1) / kMaxBits;
        s.bits = (bits + s.passes - 1) / s.passes;
        if (!a.accumulate) {
            s.fill = static_cast<char*>(a.grad);
            s.fill_bytes = d->vocab * d->dim * type_size(wt);
        }
        // 4 items a thread (16 beyond 32768 tokens) and 8 CTAs of as few warps as
        // that takes, 8 or more; fewer CTAs for fewer tokens.
        const int ipt = d->tokens > kMaxCluster * kSortThreads * 4 ? 16 : 4;
        int cluster = 1, threads = 256;
        while (cluster < kMaxCluster && (int64_t)cluster * threads * ipt < d->tokens) cluster *= 2;
        while (threads < kSortThreads && (int64_t)cluster * threads * ipt < d->tokens) threads *= 2;
        st = ipt == 4 ? run_sort<4>(s, cluster, threads, stream) : run_sort<16>(s, cluster, threads, stream);
        if (st != MDQ_OK) return st;
    }
    typedef __nv_bfloat16 B;
    if (d->grad_out_dtype == MDQ_BF16)
        st = wt == MDQ_BF16 ? run_grad<B, B>(*d, a, L, stream) : run_grad<B, float>(*d, a, L, stream);
    else
        st = wt == MDQ_BF16 ? run_grad<float, B>(*d, a, L, stream)
                            : run_grad<float, float>(*d, a, L, stream);
    if (st != MDQ_OK || !wide) return st;
    const float* sums = static_cast<const float*>(a.grad);
    const int64_t n = d->vocab * d->dim;
    const dim3 grid(148 * 8);
    const cudaError_t e =
        d->accumulate
            ? launch(embed_grad_finish<float, true>, grid, 256, 0, stream, 1, true, sums, static_cast<float*>(d->grad), n)
            : launch(embed_grad_finish<B, false>, grid, 256, 0, stream, 1, true, sums, static_cast<B*>(d->grad), n);
    return status_of(e, "embed grad");
}

}  // extern "C"
