// Embedding lookup with scaling and its gradient.
//   forward:  out[t] = scale * table[index[t]]
//   backward: grad[v] = scale * sum over the tokens t with index[t] = v of g[t]
// A negative index, or the padding index, stands for no row: its output is zero and it adds to no gradient. An index
// past the table reads nothing: its output is NaN and it adds to no gradient.
//
// Forward: one pass, bound by HBM (rows in, rows out). A CTA takes tiles of whole rows (or a part of a long one) in the
// widest accesses that the row length and the addresses allow. Measured on a B200 (6.56 TB/s copy): 32,768 skewed rows of
// 2048 bf16 34 us (7.9 TB/s of rows in and out; frequent ones come from L2), 2M rows of 32 floats out of 4096 52 us
// (4.4 TB/s of DRAM writes as counted; two thirds of the warps active, waiting for loads).
//
// Backward: no atomics, the same sums at every run. The tokens are sorted by index (stably: tokens of one row keep their
// order; one cluster up to 65536 tokens, sort.cu beyond), and the sorted list is cut into spans, one CTA each, and those
// into chunks, one group of lanes each, which walks its chunk with a part of the columns in registers: tokens of one row
// follow each other, so a row's sum stays in fp32 registers. Rows that cross chunks are put together in shared memory,
// rows that cross spans leave one fp32 sum per span, which a second kernel adds up. Rows without a token are found by
// binary search in the sorted list and cleared by further CTAs. Bound by HBM: g is read once, the gradient written once.
#include <atomic>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "dependent.cuh"
#include "embedding.cuh"
#include "launch.h"

namespace fgs {

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;  // accesses per thread in the lookup
constexpr uint32_t kLookupLanes = kThreads;

__device__ inline float to_float(float x) { return x; }
__device__ inline float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ inline float to_float(__half x) { return __half2float(x); }
template <typename P> __device__ inline P from_float(float x);
template <> __device__ inline float from_float<float>(float x) { return x; }
template <> __device__ inline __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ inline __half from_float<__half>(float x) { return __float2half_rn(x); }

template <int BYTES> struct Access;
template <> struct Access<16> { using type = uint4; };
template <> struct Access<8> { using type = uint2; };
template <> struct Access<4> { using type = uint32_t; };
template <> struct Access<2> { using type = uint16_t; };

// N consecutive elements of type P in one access
template <typename P, int N>
struct Pack {
    using A = typename Access<N * static_cast<int>(sizeof(P))>::type;
    union {
        A raw;
        P x[N];
    };
    __device__ Pack() {}
};

// Loads of read-only data that are issued where they stand. KEEP: they may be read again soon, by another token of the
// same row, and stay in L1; else they pass it by.
template <bool KEEP>
__device__ inline uint4 load_nc(const uint4* a) {
    uint4 r;
    if (KEEP) asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(a));
    else asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(a));
    return r;
}
template <bool KEEP>
__device__ inline uint2 load_nc(const uint2* a) {
    uint2 r;
    if (KEEP) asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(a));
    else asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(a));
    return r;
}
template <bool KEEP>
__device__ inline uint32_t load_nc(const uint32_t* a) {
    uint32_t r;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(r) : "l"(a));
    return r;
}
template <bool KEEP>
__device__ inline uint16_t load_nc(const uint16_t* a) {
    uint16_t r;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(r) : "l"(a));
    return r;
}

template <bool STREAM, typename A>
__device__ inline void store(A* to, A x) {
    if (STREAM) __stcs(to, x);
    else *to = x;
}

template <typename P, int N>
__device__ inline void scale_pack(Pack<P, N>& x, uint32_t row, float scale) {
    const float fill = row == kNoRow ? 0.0f : __int_as_float(0x7fc00000);
#pragma unroll
    for (int j = 0; j < N; j++) x.x[j] = from_float<P>(row < kBadRow ? scale * to_float(x.x[j]) : fill);
}

// Short rows: a group of `lanes` lanes takes kUnits rows, whose loads are in flight together, and walks their columns.
template <typename P, int N, typename I, bool STREAM>
__global__ void __launch_bounds__(kThreads, N * sizeof(P) >= 16 ? 6 : 5) lookup_kernel(const P* __restrict__ table, const I* __restrict__ index, P* __restrict__ out, int64_t rows,
                                                          int64_t tokens, uint32_t units, uint32_t lanes, float scale, int64_t padding) {
    using A = typename Pack<P, N>::A;
    const uint32_t lane = threadIdx.x & (lanes - 1), groups = kThreads / lanes, group = threadIdx.x / lanes;
    // the CTA's tokens are those of kUnits rounds over its groups, so that it writes one stretch of the output
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (groups * kUnits) + group;
    if constexpr (sizeof(A) < 16) {  // many accesses per row: addresses and decisions are made once per row
        const A* src[kUnits];  // the rows, at this lane's first column; the table's first row stands in for none
        float fill[kUnits];    // what an absent row is filled with
        bool live[kUnits], there[kUnits];
#pragma unroll
        for (int k = 0; k < kUnits; k++) {
            const int64_t t = t0 + k * groups;
            live[k] = t < tokens;
            const uint32_t row = live[k] ? row_of(index[t], rows, padding) : kNoRow;
            there[k] = row < kBadRow;
            fill[k] = row == kNoRow ? 0.0f : __int_as_float(0x7fc00000);
            src[k] = reinterpret_cast<const A*>(table) + (there[k] ? static_cast<uint64_t>(row) * units : 0) + lane;
        }
        A* dst = reinterpret_cast<A*>(out) + t0 * units + lane;
        const uint64_t step = static_cast<uint64_t>(groups) * units;
        for (uint32_t c = lane; c < units; c += lanes) {
            Pack<P, N> x[kUnits];
#pragma unroll
            for (int k = 0; k < kUnits; k++) {  // no load waits for a decision
                if (rows > 0) x[k].raw = load_nc<true>(src[k]);
                src[k] += lanes;
            }
#pragma unroll
            for (int k = 0; k < kUnits; k++) {
#pragma unroll
                for (int j = 0; j < N; j++) x[k].x[j] = from_float<P>(there[k] ? scale * to_float(x[k].x[j]) : fill[k]);
                if (live[k]) store<STREAM>(dst + k * step, x[k].raw);
            }
            dst += lanes;
        }
    } else {  // few: they are made at each access, and take no registers (with those of the other form 41 -> 49 us for 32768
              // rows of 4 KB; with these 60 instead of 51 us for 1M rows of 45 floats there)
        uint32_t row[kUnits];
#pragma unroll
        for (int k = 0; k < kUnits; k++) {
            const int64_t t = t0 + k * groups;
            row[k] = t < tokens ? row_of(index[t], rows, padding) : kNoRow;
        }
        for (uint32_t c = lane; c < units; c += lanes) {
            Pack<P, N> x[kUnits];
#pragma unroll
            for (int k = 0; k < kUnits; k++)  // the first row stands in for none: no load waits for a decision
                if (rows > 0) x[k].raw = load_nc<true>(reinterpret_cast<const A*>(table) + static_cast<uint64_t>(row[k] < kBadRow ? row[k] : 0u) * units + c);
#pragma unroll
            for (int k = 0; k < kUnits; k++) {
                const int64_t t = t0 + k * groups;
                if (t >= tokens) continue;
                scale_pack(x[k], row[k], scale);
                store<STREAM>(reinterpret_cast<A*>(out) + t * units + c, x[k].raw);
            }
        }
    }
}

// Long rows: a CTA takes a part (kThreads * kUnits accesses) of one row.
template <typename P, int N, typename I, bool STREAM>
__global__ void __launch_bounds__(kThreads) lookup_long_kernel(const P* __restrict__ table, const I* __restrict__ index, P* __restrict__ out, int64_t rows,
                                                               uint32_t units, float scale, int64_t padding) {
    using A = typename Pack<P, N>::A;
    const uint32_t row = row_of(index[blockIdx.x], rows, padding);
    const uint32_t first = blockIdx.y * (kThreads * kUnits) + threadIdx.x;
    const A* src = reinterpret_cast<const A*>(table) + static_cast<uint64_t>(row) * units;
    A* dst = reinterpret_cast<A*>(out) + static_cast<uint64_t>(blockIdx.x) * units;
    Pack<P, N> x[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const uint32_t u = first + k * kThreads;
        if (u < units && row < kBadRow) x[k].raw = src[u];
    }
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const uint32_t u = first + k * kThreads;
        if (u >= units) continue;
        scale_pack(x[k], row, scale);
        store<STREAM>(dst + u, x[k].raw);
    }
}

// Lanes of a group that walks rows of `units` accesses: the first power of two up to `most` that covers a row, or a smaller
// one where that leaves an eighth fewer lanes idle (45 accesses: three steps of 16 lanes, not one of 64). Wide groups read
// long stretches of a row at once: 32768 rows of 256 accesses by 32 lanes 47.7 us, by 256 lanes 41.2 us.
uint32_t lanes_for(uint64_t units, uint32_t most) {
    uint32_t best = 1;
    while (best < most && best < units) best *= 2;
    for (uint32_t l = best / 2; l >= 4; l /= 2) {
        const uint64_t with = (units + l - 1) / l * l, now = (units + best - 1) / best * best;
        if (8 * with <= 7 * now) best = l;
    }
    return best;
}

// An output larger than half the L2 is written past it: 2M rows of 32 floats take 52 instead of 68 us, and a short one
// stays there for its reader.
constexpr uint64_t kStreamBytes = 64ull << 20;

template <typename P, int N, typename I, bool STREAM>
cudaError_t launch_lookup_as(const EmbeddingArgs& a, const void* table, const void* index, void* out, cudaStream_t s) {
    const uint64_t units = static_cast<uint64_t>(a.width) / N;
    if (units > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    const P* t = static_cast<const P*>(table);
    const I* i = static_cast<const I*>(index);
    P* o = static_cast<P*>(out);
    // long rows, or rows of more than a warp's accesses that are so few that groups of lanes would leave SMs idle
    if (units >= kThreads * kUnits || (units > 32 && a.tokens < 148 * 8)) {
        const uint64_t parts = (units + kThreads * kUnits - 1) / (kThreads * kUnits);
        if (parts > 65535) return cudaErrorInvalidValue;
        lookup_long_kernel<P, N, I, STREAM><<<dim3(static_cast<unsigned>(a.tokens), static_cast<unsigned>(parts)), kThreads, 0, s>>>(
            t, i, o, a.rows, static_cast<uint32_t>(units), a.scale, a.padding);
    } else {
        const uint32_t lanes = lanes_for(units, kLookupLanes);
        const uint64_t per = static_cast<uint64_t>(kThreads / lanes) * kUnits;
        lookup_kernel<P, N, I, STREAM><<<static_cast<unsigned>((static_cast<uint64_t>(a.tokens) + per - 1) / per), kThreads, 0, s>>>(
            t, i, o, a.rows, a.tokens, static_cast<uint32_t>(units), lanes, a.scale, a.padding);
    }
    return cudaGetLastError();
}

template <typename P, int N, typename I>
cudaError_t launch_lookup(const EmbeddingArgs& a, const void* table, const void* index, void* out, cudaStream_t s) {
    const uint64_t bytes = static_cast<uint64_t>(a.tokens) * static_cast<uint64_t>(a.width) * sizeof(P);
    return bytes > kStreamBytes ? launch_lookup_as<P, N, I, true>(a, table, index, out, s) : launch_lookup_as<P, N, I, false>(a, table, index, out, s);
}

// widest access (at most 16 bytes) that divides a row and that all addresses are aligned for, in elements
int access_elements(const EmbeddingArgs& a, int size, const void* p, const void* q) {
    const uintptr_t m = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(a.width * size) | 16u;
    const int bytes = static_cast<int>(m & (~m + 1));
    return bytes / size;
}

// ---------------------------------------------------------------------------------------------------
// gradient

// Stable radix sort of up to 65536 indices in one launch: a cluster of up to 8 CTAs holds all (key, token) pairs in its
// shared memory, each CTA a run of 1024 x ITEMS positions. Per pass of at most 8 bits: every warp ranks its keys by
// ballots (a warp owns consecutive positions, so the order of equal digits is kept), the CTAs tell one another their
// digit counts, and every pair is stored straight into its place in the shared memory of the CTA that owns the place.
// Bound by latency (two cluster barriers per pass): 32,768 indices by 16 bits in 16 us, 257 in 6; as several launches over
// global memory the former took 28 us.
constexpr int kSortThreads = 1024, kSortWarps = 32, kDigits = 256, kMaxCluster = 8, kMaxItems = 8;
constexpr int kRunStride = kDigits + 1;  // spreads the warps' counts of one digit over the banks
constexpr uint32_t kClusterSortMax = kSortThreads * kMaxItems * kMaxCluster;

size_t cluster_sort_smem(int items) {
    return 2 * sizeof(uint64_t) * kSortThreads * static_cast<size_t>(items) + sizeof(uint32_t) * (kSortWarps * kRunStride + kMaxCluster * kDigits + 2 * kDigits + 16);
}

template <typename I, int ITEMS>
__global__ void __launch_bounds__(kSortThreads, 1) cluster_sort_kernel(const I* __restrict__ index, uint32_t tokens, int64_t rows, int64_t padding,
                                                                       int end_bit, uint32_t* __restrict__ keys, uint32_t* __restrict__ vals) {
    namespace cg = cooperative_groups;
    extern __shared__ uint64_t pairs[];  // two buffers of kSortThreads * ITEMS pairs, which receive in turn: key in the high word
    constexpr uint32_t kRun = kSortThreads * ITEMS;
    uint32_t* run = reinterpret_cast<uint32_t*>(pairs + 2 * kRun);  // [warp][digit]
    uint32_t* counts = run + kSortWarps * kRunStride;               // [CTA][digit]
    uint32_t* base = counts + kMaxCluster * kDigits;                // first place of this CTA's keys of each digit
    uint32_t* local = base + kDigits;                               // first place of each digit in the CTA's own order
    uint32_t* totals = local + kDigits;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), ctas = cluster.num_blocks();
    allow_dependent();  // a clearing kernel may start beside this one
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t first = rank * kRun + static_cast<uint32_t>(warp) * (32 * ITEMS) + lane;  // this thread's places: first + 32 j
    uint32_t key[ITEMS], val[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        const uint32_t p = first + 32 * j;
        val[j] = p;
        key[j] = p < tokens ? row_key(index[p], rows, padding) : 0xFFFFFFFFu;  // sorts behind all others, which came before it
    }
    const int passes = (end_bit + 7) / 8, bits = (end_bit + passes - 1) / passes;
    const uint32_t mask = (1u << bits) - 1u;
    cluster.sync();  // every CTA runs before its shared memory is written to
    for (int pass = 0; pass < passes; pass++) {
        const int shift = pass * bits;
        uint64_t* to = pairs + (pass & 1) * kRun;
        uint64_t* stage = pairs + (~pass & 1) * kRun;  // free until the next pass's pairs arrive, behind its first barrier
        for (int i = t; i < kSortWarps * kRunStride; i += kSortThreads) run[i] = 0;
        __syncthreads();
        uint32_t place[ITEMS];
        uint32_t* mine = run + warp * kRunStride;
#pragma unroll
        for (int j = 0; j < ITEMS; j++) {
            const uint32_t d = (key[j] >> shift) & mask;
            uint32_t same = 0xFFFFFFFFu;
#pragma unroll
            for (int b = 0; b < 8; b++) {  // bits above the pass's are zero in all
                const uint32_t with = __ballot_sync(0xFFFFFFFFu, (d >> b) & 1u);
                same &= with ^ (((d >> b) & 1u) - 1u);
            }
            const uint32_t before = __popc(same & ((1u << lane) - 1u));
            const uint32_t prior = mine[d];
            place[j] = prior + before;
            __syncwarp();
            if (before == 0) mine[d] = prior + __popc(same);
            __syncwarp();
        }
        __syncthreads();
        // four threads per digit: exclusive sums of its counts over the warps, and the CTA's count, told to every CTA
        {
            const int d = t >> 2, q = t & 3;
            uint32_t c[8], sum = 0;
#pragma unroll
            for (int w = 0; w < 8; w++) {
                c[w] = run[(8 * q + w) * kRunStride + d];
                sum += c[w];
            }
            uint32_t incl = sum;
            for (int o = 1; o < 4; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, incl, o, 4);
                if (q >= o) incl += y;
            }
            uint32_t at = incl - sum;
#pragma unroll
            for (int w = 0; w < 8; w++) {
                run[(8 * q + w) * kRunStride + d] = at;
                at += c[w];
            }
            const uint32_t total = __shfl_sync(0xFFFFFFFFu, incl, 3, 4);
            for (uint32_t r = q; r < ctas; r += 4) cluster.map_shared_rank(counts, r)[rank * kDigits + d] = total;
        }
        cluster.sync();
        if (t < kDigits) {
            uint32_t before = 0, all = 0;
            for (uint32_t r = 0; r < ctas; r++) {
                const uint32_t c = counts[r * kDigits + t];
                before += r < rank ? c : 0u;
                all += c;
            }
            const uint32_t own = counts[rank * kDigits + t];
            uint32_t incl = all, incl_own = own;  // inclusive sums over the warp's digits, of all CTAs and of this one
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, incl, o), z = __shfl_up_sync(0xFFFFFFFFu, incl_own, o);
                if (lane >= o) {
                    incl += y;
                    incl_own += z;
                }
            }
            if (lane == 31) {
                totals[warp] = incl;
                totals[8 + warp] = incl_own;
            }
            base[t] = before + incl - all;
            local[t] = incl_own - own;
        }
        __syncthreads();
        if (t < kDigits) {
            uint32_t before = 0, before_own = 0;
            for (int w = 0; w < warp; w++) {
                before += totals[w];
                before_own += totals[8 + w];
            }
            local[t] += before_own;
            base[t] += before - local[t];  // place of a digit's key less its place in the CTA's own order
        }
        __syncthreads();
        // into digit order within the CTA, then to the owners: neighbours go to neighbouring places (pairs stored one by
        // one straight to their places took 4.7k of a pass's 14k cycles)
#pragma unroll
        for (int j = 0; j < ITEMS; j++) {
            const uint32_t d = (key[j] >> shift) & mask;
            stage[local[d] + mine[d] + place[j]] = static_cast<uint64_t>(key[j]) << 32 | val[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; j++) {
            const uint32_t i = j * kSortThreads + t;
            const uint64_t x = stage[i];
            const uint32_t p = base[(static_cast<uint32_t>(x >> 32) >> shift) & mask] + i;
            cluster.map_shared_rank(to, p / kRun)[p % kRun] = x;
        }
        cluster.sync();
#pragma unroll
        for (int j = 0; j < ITEMS; j++) {
            const uint64_t x = to[warp * (32 * ITEMS) + 32 * j + lane];
            key[j] = static_cast<uint32_t>(x >> 32);
            val[j] = static_cast<uint32_t>(x);
        }
    }
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        const uint32_t p = first + 32 * j;
        if (p < tokens) {
            keys[p] = key[j];
            vals[p] = val[j];
        }
    }
}

template <typename I, int ITEMS>
cudaError_t launch_cluster_sort(const EmbeddingArgs& a, const void* index, int end_bit, uint32_t* keys, uint32_t* vals, cudaStream_t s) {
    const uint32_t per = kSortThreads * ITEMS;
    uint32_t ctas = 1;
    while (ctas * per < static_cast<uint32_t>(a.tokens)) ctas *= 2;
    const size_t smem = cluster_sort_smem(ITEMS);
    static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may use so much shared memory
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(cluster_sort_kernel<I, ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(ctas);
    config.blockDim = dim3(kSortThreads);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = ctas;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, cluster_sort_kernel<I, ITEMS>, static_cast<const I*>(index), static_cast<uint32_t>(a.tokens), a.rows, a.padding,
                              end_bit, keys, vals);
}

// as many CTAs as a cluster has before each takes more than 1024 indices
template <typename I>
cudaError_t cluster_sort(const EmbeddingArgs& a, const void* index, int end_bit, uint32_t* keys, uint32_t* vals, cudaStream_t s) {
    const uint32_t most = kSortThreads * kMaxCluster;
    if (a.tokens <= most) return launch_cluster_sort<I, 1>(a, index, end_bit, keys, vals, s);
    if (a.tokens <= 2 * most) return launch_cluster_sort<I, 2>(a, index, end_bit, keys, vals, s);
    if (a.tokens <= 4 * most) return launch_cluster_sort<I, 4>(a, index, end_bit, keys, vals, s);
    return launch_cluster_sort<I, 8>(a, index, end_bit, keys, vals, s);
}

// Clears a gradient (102 MB in 22 us beside the sort) on the SMs that the sort before it leaves idle: launched as its
// programmatic dependent, so it starts with the sort, and waits for the sort's end before its own.
__global__ void __launch_bounds__(kThreads) clear_kernel(uint4* __restrict__ to, uint64_t bytes) {
    const uint64_t n = bytes / 16, stride = static_cast<uint64_t>(gridDim.x) * kThreads;
    const uint64_t i0 = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x;
#pragma unroll 4
    for (uint64_t i = i0; i < n; i += stride) to[i] = make_uint4(0, 0, 0, 0);
    if (i0 < bytes % 16) reinterpret_cast<uint8_t*>(to + n)[i0] = 0;
    allow_dependent();
    wait_dependency();
}

struct SumArgs {
    const uint32_t* keys;    // sorted rows
    const uint32_t* tokens;  // their tokens
    float* head;             // [spans][width] sum within a CTA's span of the row that began before it
    float* tail;             // [spans][width] sum within the span of the row that goes on behind it
    uint32_t n, rows, units;
    uint32_t lanes, parts;   // lanes of a group (a power of two, at most 32), column parts of a row
    uint32_t chunk, span, spans;  // sorted positions of a group and of a CTA; CTAs per column part
    uint32_t zero_rows;      // rows that a clearing CTA looks at
    bool cleared;            // rows without a token are zero already
    float scale;
};

constexpr uint32_t kNone = 0xFFFFFFFFu;  // no key

template <typename P, int N>
__device__ inline void write_row(P* grad, uint64_t row, uint32_t units, uint32_t col, const float (&acc)[N], float scale) {
    Pack<P, N> x;
#pragma unroll
    for (int j = 0; j < N; j++) x.x[j] = from_float<P>(scale * acc[j]);
    reinterpret_cast<typename Pack<P, N>::A*>(grad)[row * units + col] = x.raw;
}

// N consecutive partial sums (aligned to their size, up to 16 bytes)
template <int N>
__device__ inline void load_part(const float* a, float (&x)[N]) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(x + j) = *reinterpret_cast<const float4*>(a + j);
    } else if constexpr (N == 2) {
        *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(a);
    } else {
        x[0] = a[0];
    }
}
template <int N>
__device__ inline void store_part(float* a, const float (&x)[N]) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(a + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
    } else if constexpr (N == 2) {
        *reinterpret_cast<float2*>(a) = make_float2(x[0], x[1]);
    } else {
        a[0] = x[0];
    }
}

// clears the rows without a token among `zero_rows` rows
template <typename P, int N>
__device__ inline void clear_rows(P* grad, const SumArgs& a, uint32_t cta, uint8_t* used) {
    using A = typename Pack<P, N>::A;
    const uint32_t first = cta * a.zero_rows, count = a.rows - first < a.zero_rows ? a.rows - first : a.zero_rows;
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
        const uint32_t row = first + i;
        uint32_t lo = 0, hi = a.n;  // the first position whose key is not below the row
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (a.keys[mid] < row) lo = mid + 1;
            else hi = mid;
        }
        used[i] = lo < a.n && a.keys[lo] == row;
    }
    __syncthreads();
    Pack<P, N> zero;
#pragma unroll
    for (int j = 0; j < N; j++) zero.x[j] = from_float<P>(0.0f);
    A* to = reinterpret_cast<A*>(grad) + static_cast<uint64_t>(first) * a.units;
    if (a.units >= kThreads) {
        for (uint32_t i = 0; i < count; i++) {
            if (used[i]) continue;
            for (uint32_t u = threadIdx.x; u < a.units; u += kThreads) to[static_cast<uint64_t>(i) * a.units + u] = zero.raw;
        }
    } else {
        for (uint32_t u = threadIdx.x; u < count * a.units; u += kThreads)
            if (!used[u / a.units]) to[u] = zero.raw;
    }
}

// A CTA takes a span of sorted positions and a part of the columns; its groups of lanes take a chunk of the span each.
// Bound by HBM: 32,768 rows of 1024 bf16 in 20 us (97 MB, 4.9 TB/s), 2M rows of 32 floats, gathered 128 bytes at a time, in
// 54 us (4.8 TB/s). Four accesses in flight per lane and four CTAs per SM; eight and three took 6 us longer there. Eight
// narrower accesses, and six CTAs where they have 4 bytes (700k rows of 45 floats 99 -> 92 us with six).
// Within a group a row's sum stays in registers; rows that cross chunk borders are put together in shared memory, by
// doubling along the groups that lie whole within the row.
template <typename P, int N>
__global__ void __launch_bounds__(kThreads, N * sizeof(P) == 4 ? 6 : 4) sum_kernel(const P* g, P* grad, const SumArgs a) {
    using A = typename Pack<P, N>::A;
    extern __shared__ uint32_t staged[];  // the span's keys with one more on either side, and its tokens
    __shared__ float part[kThreads * N];
    __shared__ uint8_t full[kThreads];    // group: its head row goes on in the next group
    allow_dependent();
    wait_dependency();
    const uint32_t sum_ctas = a.spans * a.parts;
    if (blockIdx.x >= sum_ctas) {
        clear_rows<P, N>(grad, a, blockIdx.x - sum_ctas, reinterpret_cast<uint8_t*>(part));
        return;
    }
    const uint32_t span = blockIdx.x / a.parts, column_part = blockIdx.x % a.parts;
    const uint32_t p0 = span * a.span, have = a.n - p0 < a.span ? a.n - p0 : a.span;
    uint32_t* keys = staged + 1;
    uint32_t* tokens = keys + a.span + 1;
    for (uint32_t i = threadIdx.x; i < have; i += kThreads) {
        keys[i] = a.keys[p0 + i];
        tokens[i] = a.tokens[p0 + i];
    }
    if (threadIdx.x == 0) {
        staged[0] = p0 > 0 ? a.keys[p0 - 1] : kNone;
        keys[have] = p0 + have < a.n ? a.keys[p0 + have] : kNone;
    }
    __syncthreads();
    const uint32_t lane = threadIdx.x % a.lanes, group = threadIdx.x / a.lanes;
    const uint32_t col = column_part * a.lanes + lane;
    const uint32_t c0 = group * a.chunk, c1 = c0 + a.chunk < have ? c0 + a.chunk : have;
    const bool live = c0 < have && col < a.units;
    const A* src = reinterpret_cast<const A*>(g) + col;
    float acc[N];  // the running row
#pragma unroll
    for (int j = 0; j < N; j++) acc[j] = part[j * kThreads + threadIdx.x] = 0.0f;  // part: the row that the group began within
    uint32_t row = a.rows;
    bool first = false, on = false;
    if (live) {
        row = keys[c0];
        first = row < a.rows && keys[static_cast<int>(c0) - 1] == row;
        bool began = first;  // the running row began before the group
        constexpr int kAhead = sizeof(Pack<P, N>) >= 16 ? 4 : 8;  // accesses in flight per lane
        for (uint32_t p = c0; p < c1 && row < a.rows; p += kAhead) {
            Pack<P, N> x[kAhead];
            uint32_t key[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) {  // loaded in any case (every token has a gradient): none waits for another
                const uint32_t q = p + k < c1 ? p + k : c1 - 1;
                key[k] = keys[q];
                x[k].raw = load_nc<false>(src + static_cast<uint64_t>(tokens[q]) * a.units);
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                if (p + k >= c1) break;
                if (key[k] != row) {  // the row ends here
                    if (began) {
#pragma unroll
                        for (int j = 0; j < N; j++) part[j * kThreads + threadIdx.x] = acc[j];
                    } else {
                        write_row<P, N>(grad, row, a.units, col, acc, a.scale);
                    }
                    began = false;
                    row = key[k];
#pragma unroll
                    for (int j = 0; j < N; j++) acc[j] = 0.0f;
                    if (row >= a.rows) break;
                }
#pragma unroll
                for (int j = 0; j < N; j++) acc[j] += to_float(x[k].x[j]);
            }
        }
        on = row < a.rows && keys[c1] == row;
        if (row < a.rows) {
            if (began) {  // one row only
#pragma unroll
                for (int j = 0; j < N; j++) part[j * kThreads + threadIdx.x] = acc[j];
            } else if (!on) {
                write_row<P, N>(grad, row, a.units, col, acc, a.scale);
            }
        }
        // from here on: first: the group has a head; through: it is all one row, which goes on; on && !through: it has a tail
        on = on && !began;
        if (lane == 0) full[group] = began && row < a.rows && keys[c1] == row;
    } else if (lane == 0) {
        full[group] = 0;
    }
    const uint32_t groups = kThreads / a.lanes;
    __syncthreads();
    bool through = full[group];
    if (__syncthreads_or(through)) {  // heads behind one another: add them up along the groups
        for (uint32_t d = 1; d < groups; d *= 2) {
            float more[N];
            bool linked = through && group + d < groups;
            if (linked) {
#pragma unroll
                for (int j = 0; j < N; j++) more[j] = part[j * kThreads + threadIdx.x + d * a.lanes];
            }
            const bool next = linked && full[group + d];
            __syncthreads();
            if (linked) {
#pragma unroll
                for (int j = 0; j < N; j++) part[j * kThreads + threadIdx.x] += more[j];
                through = next;
                if (lane == 0) full[group] = next;
            }
            __syncthreads();
        }
    }
    // full[g]: the chain of heads from group g reaches the span's end and goes on behind it
    if (!live) return;
    const uint32_t width = a.units * N;
    if (on) {  // a row that begins in this group: its sum so far, and the heads behind it
        bool leaves = group + 1 == groups || c1 == have;
        if (!leaves) {
#pragma unroll
            for (int j = 0; j < N; j++) acc[j] += part[j * kThreads + threadIdx.x + a.lanes];
            leaves = full[group + 1];
        }
        if (leaves) {
            store_part<N>(a.tail + static_cast<uint64_t>(span) * width + col * N, acc);
        } else {
            write_row<P, N>(grad, row, a.units, col, acc, a.scale);
        }
    }
    if (group == 0 && first) {
#pragma unroll
        for (int j = 0; j < N; j++) acc[j] = part[j * kThreads + threadIdx.x];
        store_part<N>(a.head + static_cast<uint64_t>(span) * width + col * N, acc);
    }
}

// Adds the spans' sums of each row that crosses span borders (about 5 us where rows cross a few spans: two round trips to
// memory). A CTA looks at one span for a row that begins in it and
// goes on; slots of `lanes` lanes take the row's spans in turn, and the slots' sums are added pairwise.
template <typename P, int N>
__global__ void __launch_bounds__(kThreads) join_kernel(P* grad, const SumArgs a) {
    __shared__ float part[kThreads * N];
    wait_dependency();
    const uint32_t span = blockIdx.x;
    const uint64_t p0 = static_cast<uint64_t>(span) * a.span, p1 = p0 + a.span;
    if (p1 >= a.n) return;
    const uint32_t row = a.keys[p1];
    if (row >= a.rows || a.keys[p1 - 1] != row || (p0 > 0 && a.keys[p0 - 1] == row)) return;
    uint32_t last = span;  // the last span with the row: those behind this one that begin with it
    for (;;) {
        const uint64_t p = (static_cast<uint64_t>(last) + 1 + threadIdx.x) * a.span;
        const int more = __syncthreads_count(p < a.n && a.keys[p] == row);
        last += static_cast<uint32_t>(more);
        if (more < kThreads) break;
    }
    const uint32_t width = a.units * N;
    const uint32_t slots = kThreads / a.lanes, slot = threadIdx.x / a.lanes;
    const uint32_t col = blockIdx.y * a.lanes + threadIdx.x % a.lanes;
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; j++) acc[j] = 0.0f;
    if (col < a.units) {
        if (slot == 0) load_part<N>(a.tail + static_cast<uint64_t>(span) * width + col * N, acc);
        constexpr int kBatch = N >= 8 ? 4 : 8;  // spans in flight
        for (uint32_t c0 = span + 1 + slot; c0 <= last; c0 += kBatch * slots) {
            float x[kBatch][N];
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                const uint32_t c = c0 + k * slots;
                load_part<N>(a.head + static_cast<uint64_t>(c <= last ? c : last) * width + col * N, x[k]);
            }
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                if (c0 + k * slots > last) break;
#pragma unroll
                for (int j = 0; j < N; j++) acc[j] += x[k][j];
            }
        }
    }
    uint32_t busy = slots;  // slots that may hold a sum
    while (busy > 1 && busy / 2 >= last - span) busy /= 2;
    if (busy > 1) {
#pragma unroll
        for (int j = 0; j < N; j++) part[j * kThreads + threadIdx.x] = acc[j];
        __syncthreads();
        for (uint32_t half = busy / 2; half > 0; half /= 2) {
            if (slot < half) {
#pragma unroll
                for (int j = 0; j < N; j++) part[j * kThreads + threadIdx.x] += part[j * kThreads + threadIdx.x + half * a.lanes];
            }
            __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < N; j++) acc[j] = part[j * kThreads + threadIdx.x];
    }
    if (slot == 0 && col < a.units) write_row<P, N>(grad, row, a.units, col, acc, a.scale);
}

constexpr uint64_t kClearBytes = 32ull << 20;

struct GradBuffers {
    uint32_t *keys_a, *keys_b, *vals_a, *vals_b;
    void* sort_temp;
    size_t sort_bytes;
    float *head, *tail;
};

int bits_of(uint64_t x) {
    int b = 0;
    while (x) {
        b++;
        x >>= 1;
    }
    return b;
}

// How the sorted tokens are cut: enough groups to give each of the 148 x 1024 threads that run at once a column, 8 to 64
// positions each, and at most 4096 positions (their keys and tokens are staged in shared memory) per CTA. (Backward of
// 32,768 rows of 1024 bf16 with twice as many groups 54.9 us, with these 52.9, with half as many 57.1.)
void cut(uint64_t tokens, uint64_t units, SumArgs* S) {
    S->lanes = lanes_for(units, 32);
    S->parts = static_cast<uint32_t>((units + S->lanes - 1) / S->lanes);
    const uint32_t groups = kThreads / S->lanes;
    const uint64_t want = tokens * units / (148ull * 1024ull);
    S->chunk = 8;
    while (S->chunk < want && S->chunk < 64 && S->chunk * 2 * groups <= 4096) S->chunk *= 2;
    S->span = S->chunk * groups;
    S->spans = static_cast<uint32_t>((tokens + S->span - 1) / S->span);
}

// access width of the rows in elements: the widest (at most 16 bytes) that divides a row
int row_elements(uint64_t width, int size) {
    int n = 16 / size;
    while (width % static_cast<uint64_t>(n)) n /= 2;
    return n;
}

size_t carve(void* ws, uint64_t tokens, uint64_t rows, uint64_t width, int size, GradBuffers* B) {
    char* base = static_cast<char*>(ws);
    size_t off = 0;
    const auto take = [&](size_t bytes) {
        off = (off + 255) & ~static_cast<size_t>(255);
        char* p = base ? base + off : nullptr;
        off += bytes;
        return p;
    };
    GradBuffers b;
    const bool small = tokens <= kClusterSortMax;
    b.keys_a = reinterpret_cast<uint32_t*>(take(4 * tokens));
    b.vals_a = reinterpret_cast<uint32_t*>(take(4 * tokens));
    b.keys_b = reinterpret_cast<uint32_t*>(take(small ? 0 : 4 * tokens));
    b.vals_b = reinterpret_cast<uint32_t*>(take(small ? 0 : 4 * tokens));
    b.sort_bytes = small ? 0 : row_sort_temp_bytes(tokens);
    b.sort_temp = take(b.sort_bytes);
    // Narrower accesses (misaligned addresses) widen the groups of lanes, so a CTA has fewer of them and there are more spans
    // as a rule: room for the most that any width makes.
    uint64_t spans = 1;
    for (int n = row_elements(width, size); n >= 1; n /= 2) {
        SumArgs S{};
        cut(tokens, width / n, &S);
        spans = S.spans > spans ? S.spans : spans;
    }
    b.head = reinterpret_cast<float*>(take(4 * spans * width));
    b.tail = reinterpret_cast<float*>(take(4 * spans * width));
    if (B) *B = b;
    return off;
}

template <typename P, int N>
cudaError_t launch_sums(const EmbeddingArgs& a, const void* g, void* grad, SumArgs S, cudaStream_t s) {
    const uint64_t units = static_cast<uint64_t>(a.width) / N;
    if (units > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    S.units = static_cast<uint32_t>(units);
    cut(static_cast<uint64_t>(a.tokens), units, &S);
    uint64_t zero_rows = 8192 / units;  // about 128 KB of a CTA's rows
    zero_rows = zero_rows < 1 ? 1 : zero_rows > kThreads ? kThreads : zero_rows;
    S.zero_rows = static_cast<uint32_t>(zero_rows);
    const uint64_t ctas = static_cast<uint64_t>(S.spans) * S.parts + (S.cleared ? 0 : (static_cast<uint64_t>(a.rows) + zero_rows - 1) / zero_rows);
    if (ctas > 0x7FFFFFFFull || S.parts > 65535) return cudaErrorInvalidValue;
    const size_t smem = sizeof(uint32_t) * (2 * static_cast<size_t>(S.span) + 2);
    const cudaError_t e = launch_dependent(sum_kernel<P, N>, dim3(static_cast<unsigned>(ctas)), kThreads, smem, s, static_cast<const P*>(g), static_cast<P*>(grad), S);
    if (e != cudaSuccess || S.spans == 1) return e;
    return launch_dependent(join_kernel<P, N>, dim3(S.spans, S.parts), kThreads, 0, s, static_cast<P*>(grad), S);
}

}  // namespace

// calls F<P, N> for the table's type and the access width in elements
#define FGS_BY_ACCESS(dtype, elements, CALL)                                                                          \
    (dtype == kDtypeF32 ? (elements >= 4 ? CALL(float, 4) : elements == 2 ? CALL(float, 2) : CALL(float, 1))         \
     : dtype == kDtypeBf16 ? (elements >= 8   ? CALL(__nv_bfloat16, 8)                                               \
                              : elements == 4 ? CALL(__nv_bfloat16, 4)                                               \
                              : elements == 2 ? CALL(__nv_bfloat16, 2)                                               \
                                              : CALL(__nv_bfloat16, 1))                                              \
                           : (elements >= 8   ? CALL(__half, 8)                                                      \
                              : elements == 4 ? CALL(__half, 4)                                                      \
                              : elements == 2 ? CALL(__half, 2)                                                      \
                                              : CALL(__half, 1)))

cudaError_t launch_embedding_lookup(const EmbeddingArgs& a, const void* table, const void* index, void* out, cudaStream_t s) {
    if (a.tokens == 0 || a.width == 0) return cudaSuccess;
    const int n = access_elements(a, a.dtype == kDtypeF32 ? 4 : 2, table, out);
#define FGS_LOOKUP(P, N) (a.wide_index ? launch_lookup<P, N, int64_t>(a, table, index, out, s) : launch_lookup<P, N, int32_t>(a, table, index, out, s))
    return FGS_BY_ACCESS(a.dtype, n, FGS_LOOKUP);
#undef FGS_LOOKUP
}

size_t embedding_workspace_bytes(int64_t tokens, int64_t rows, int64_t width) {
    size_t most = 0;  // for any type
    for (int size = 2; size <= 4; size *= 2) {
        const size_t b = carve(nullptr, static_cast<uint64_t>(tokens), static_cast<uint64_t>(rows), static_cast<uint64_t>(width), size, nullptr);
        most = b > most ? b : most;
    }
    return most;
}

cudaError_t launch_embedding_grad(const EmbeddingArgs& a, const void* index, const void* g, void* grad, void* ws, cudaStream_t s) {
    if (a.rows == 0 || a.width == 0) return cudaSuccess;
    const int size = a.dtype == kDtypeF32 ? 4 : 2;
    if (a.tokens == 0) return cudaMemsetAsync(grad, 0, static_cast<size_t>(a.rows) * static_cast<size_t>(a.width) * static_cast<size_t>(size), s);
    GradBuffers B;
    carve(ws, static_cast<uint64_t>(a.tokens), static_cast<uint64_t>(a.rows), static_cast<uint64_t>(a.width), size, &B);
    const uint32_t tokens = static_cast<uint32_t>(a.tokens);
    const int end_bit = bits_of(static_cast<uint64_t>(a.rows));
    SumArgs S{};
    cudaError_t e;
    if (tokens <= kClusterSortMax) {
        e = a.wide_index ? cluster_sort<int64_t>(a, index, end_bit, B.keys_a, B.vals_a, s) : cluster_sort<int32_t>(a, index, end_bit, B.keys_a, B.vals_a, s);
        // The sort keeps at most 8 SMs busy: the others clear a large gradient meanwhile (rows that have tokens are written
        // again, which costs less than looking for the others afterwards; a small one is not worth the launch).
        const uint64_t bytes = static_cast<uint64_t>(a.rows) * static_cast<uint64_t>(a.width) * static_cast<uint64_t>(size);
        S.cleared = bytes >= kClearBytes && reinterpret_cast<uintptr_t>(grad) % 16 == 0;
        if (e == cudaSuccess && S.cleared) e = launch_dependent(clear_kernel, dim3(148 * 8), kThreads, 0, s, static_cast<uint4*>(grad), bytes);
        if (e != cudaSuccess) return e;
        S.keys = B.keys_a;
        S.tokens = B.vals_a;
    } else {
        e = row_sort(index, a.wide_index, a.rows, a.padding, tokens, end_bit, B.keys_a, B.keys_b, B.vals_a, B.vals_b, B.sort_temp, B.sort_bytes, &S.keys,
                     &S.tokens, s);
        if (e != cudaSuccess) return e;
    }
    S.head = B.head;
    S.tail = B.tail;
    S.n = tokens;
    S.rows = static_cast<uint32_t>(a.rows);
    S.scale = a.scale;
    const int n = access_elements(a, size, g, grad);
#define FGS_SUMS(P, N) launch_sums<P, N>(a, g, grad, S, s)
    return FGS_BY_ACCESS(a.dtype, n, FGS_SUMS);
#undef FGS_SUMS
}

}  // namespace fgs
