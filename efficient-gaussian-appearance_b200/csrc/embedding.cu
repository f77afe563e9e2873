// Embedding lookup with scaling and its gradient.
//   forward:  out[t] = scale * table[index[t]]
//   backward: grad[v] = scale * sum over the tokens t with index[t] = v of g[t]
// A negative index, or the padding index, stands for no row: its output is zero and it adds to no gradient. An index
// past the table reads nothing: its output is NaN and it adds to no gradient.
//
// Forward: one pass, bound by HBM (rows in, rows out). A CTA takes tiles of whole rows (or a part of a long one) in the
// widest accesses that the row length and the addresses allow.
//
// Backward: no atomics, the same sums at every run. The tokens are sorted by index (stable radix sort, sort.cu: tokens
// of one row keep their order), the sorted list is cut into chunks of C tokens, and a group of lanes walks each chunk
// with a row's columns in registers: tokens of the same row follow each other, so their sum stays in fp32 registers. A row whose tokens
// all lie in one chunk is written there. A row that crosses chunk borders leaves a partial sum per chunk (fp32), which
// a second kernel adds up in the chunks' order. Rows without a token are set to zero by further CTAs of the first
// kernel, which read one flag byte per row. Bound by HBM: g is read once, the gradient written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "launch.h"

namespace fgs {

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;  // accesses per thread in the lookup

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

// row of an index: the row itself, kNoRow (padding) or kBadRow (past the table)
constexpr uint32_t kNoRow = 0xFFFFFFFFu, kBadRow = 0xFFFFFFFEu;
template <typename I>
__device__ inline uint32_t row_of(I index, int64_t rows, int64_t padding) {
    const int64_t i = static_cast<int64_t>(index);
    if (i < 0 || i == padding) return kNoRow;
    return i < rows ? static_cast<uint32_t>(i) : kBadRow;
}

// a CTA takes `per` tokens (rows of `units` accesses), or with per = 1 the part blockIdx.y of one row
template <typename P, int N, typename I>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const P* __restrict__ table, const I* __restrict__ index, P* __restrict__ out, int64_t rows,
                                                          int64_t tokens, uint32_t units, uint32_t per, float scale, int64_t padding) {
    using A = typename Pack<P, N>::A;
    const A* src = reinterpret_cast<const A*>(table);
    A* dst = reinterpret_cast<A*>(out);
    const uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * per;
    const uint32_t have = tokens - t0 < per ? static_cast<uint32_t>(tokens - t0) : per;
    const uint32_t n = have * units;  // at most max(units, kThreads * kUnits)
    const uint32_t first = blockIdx.y * (kThreads * kUnits) + threadIdx.x;
    Pack<P, N> x[kUnits];
    uint32_t row[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const uint32_t u = first + k * kThreads;
        row[k] = kNoRow;
        if (u >= n) continue;
        const uint32_t t = per == 1 ? 0u : u / units;
        row[k] = row_of(index[t0 + t], rows, padding);
        if (row[k] < kBadRow) x[k].raw = src[static_cast<uint64_t>(row[k]) * units + (u - t * units)];
    }
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const uint32_t u = first + k * kThreads;
        if (u >= n) continue;
        const float fill = row[k] == kNoRow ? 0.0f : __int_as_float(0x7fc00000);
#pragma unroll
        for (int j = 0; j < N; j++) x[k].x[j] = from_float<P>(row[k] < kBadRow ? scale * to_float(x[k].x[j]) : fill);
        dst[t0 * units + u] = x[k].raw;
    }
}

template <typename P, int N, typename I>
cudaError_t launch_lookup(const EmbeddingArgs& a, const void* table, const void* index, void* out, cudaStream_t s) {
    const uint64_t units = static_cast<uint64_t>(a.width) / N;
    if (units > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    const uint32_t span = kThreads * kUnits;
    const uint32_t per = units >= span ? 1u : static_cast<uint32_t>(span / units);
    const uint64_t ctas = (static_cast<uint64_t>(a.tokens) + per - 1) / per;
    const uint64_t parts = per == 1 ? (units + span - 1) / span : 1;
    if (ctas > 0x7FFFFFFFull || parts > 65535) return cudaErrorInvalidValue;
    lookup_kernel<P, N, I><<<dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(parts)), kThreads, 0, s>>>(
        static_cast<const P*>(table), static_cast<const I*>(index), static_cast<P*>(out), a.rows, a.tokens, static_cast<uint32_t>(units), per, a.scale,
        a.padding);
    return cudaGetLastError();
}

// widest access (at most 16 bytes) that divides a row and that all addresses are aligned for, in elements
int access_elements(const EmbeddingArgs& a, int size, const void* p, const void* q) {
    const uintptr_t m = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(a.width * size) | 16u;
    const int bytes = static_cast<int>(m & (~m + 1));
    return bytes / size;
}

// ---------------------------------------------------------------------------------------------------
// gradient

// sort keys (the row; `rows` for tokens that add to none), token numbers, and the flags of the rows that have a token
template <typename I>
__global__ void __launch_bounds__(kThreads) keys_kernel(const I* __restrict__ index, uint32_t tokens, int64_t rows, int64_t padding,
                                                        uint32_t* __restrict__ keys, uint32_t* __restrict__ vals, uint8_t* __restrict__ used) {
    const uint32_t t = blockIdx.x * kThreads + threadIdx.x;
    if (t >= tokens) return;
    const uint32_t r = row_of(index[t], rows, padding);
    keys[t] = r < kBadRow ? r : static_cast<uint32_t>(rows);
    vals[t] = t;
    if (r < kBadRow) used[r] = 1;
}

struct SumArgs {
    const uint32_t* keys;    // sorted rows
    const uint32_t* tokens;  // their tokens
    const uint8_t* used;
    float* head;             // [chunks][width] partial sum of the row that began in an earlier chunk
    float* tail;             // [chunks][width] partial sum of the row that goes on in the next chunk
    uint32_t n, rows, units, chunk, chunks;
    uint32_t lanes, groups;  // lanes of a group (a power of two, at most 32), column parts of a row
    uint32_t sum_ctas;
    float scale;
};

template <typename P, int N>
__device__ inline void write_row(P* grad, uint64_t row, uint32_t units, uint32_t col, const float (&acc)[N], float scale) {
    Pack<P, N> x;
#pragma unroll
    for (int j = 0; j < N; j++) x.x[j] = from_float<P>(scale * acc[j]);
    reinterpret_cast<typename Pack<P, N>::A*>(grad)[row * units + col] = x.raw;
}

// One group of `lanes` lanes per (chunk, part of the columns).
template <typename P, int N>
__global__ void __launch_bounds__(kThreads) sum_kernel(const P* __restrict__ g, P* __restrict__ grad, const SumArgs a) {
    using A = typename Pack<P, N>::A;
    if (blockIdx.x >= a.sum_ctas) {  // rows without a token
        const uint64_t total = static_cast<uint64_t>(a.rows) * a.units;
        const uint64_t stride = static_cast<uint64_t>(gridDim.x - a.sum_ctas) * kThreads;
        Pack<P, N> zero;
#pragma unroll
        for (int j = 0; j < N; j++) zero.x[j] = from_float<P>(0.0f);
        for (uint64_t u = static_cast<uint64_t>(blockIdx.x - a.sum_ctas) * kThreads + threadIdx.x; u < total; u += stride)
            if (!a.used[u / a.units]) reinterpret_cast<A*>(grad)[u] = zero.raw;
        return;
    }
    const uint64_t worker = (static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x) / a.lanes;
    const uint32_t chunk = static_cast<uint32_t>(worker / a.groups);
    const uint32_t col = static_cast<uint32_t>(worker % a.groups) * a.lanes + threadIdx.x % a.lanes;
    if (chunk >= a.chunks || col >= a.units) return;
    const uint32_t p0 = chunk * a.chunk;
    const uint32_t p1 = a.n - p0 < a.chunk ? a.n : p0 + a.chunk;
    const A* src = reinterpret_cast<const A*>(g);
    const uint32_t width = a.units * N;
    bool first = p0 > 0 && a.keys[p0 - 1] == a.keys[p0];  // the running row began in an earlier chunk
    uint32_t row = a.keys[p0];
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; j++) acc[j] = 0.0f;
    constexpr int kAhead = 8;
    for (uint32_t p = p0; p < p1 && row < a.rows; p += kAhead) {
        Pack<P, N> x[kAhead];
        uint32_t key[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            key[k] = a.rows;
            if (p + k >= p1) continue;
            key[k] = a.keys[p + k];
            if (key[k] < a.rows) x[k].raw = src[static_cast<uint64_t>(a.tokens[p + k]) * a.units + col];
        }
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            if (p + k >= p1) break;
            if (key[k] != row) {  // the row ends here
                if (first) {
#pragma unroll
                    for (int j = 0; j < N; j++) a.head[static_cast<uint64_t>(chunk) * width + col * N + j] = acc[j];
                } else {
                    write_row<P, N>(grad, row, a.units, col, acc, a.scale);
                }
                first = false;
                row = key[k];
#pragma unroll
                for (int j = 0; j < N; j++) acc[j] = 0.0f;
                if (row >= a.rows) break;
            }
#pragma unroll
            for (int j = 0; j < N; j++) acc[j] += to_float(x[k].x[j]);
        }
    }
    if (row >= a.rows) return;
    const bool on = p1 < a.n && a.keys[p1] == row;
    if (first || on) {
        float* to = first ? a.head : a.tail;
#pragma unroll
        for (int j = 0; j < N; j++) to[static_cast<uint64_t>(chunk) * width + col * N + j] = acc[j];
    } else {
        write_row<P, N>(grad, row, a.units, col, acc, a.scale);
    }
}

// Adds the partial sums of each row that crosses a chunk border: the CTA's warps look at 256 chunks for rows that begin
// in them and go on, and then sum each of those with all threads: slots of `lanes` lanes take the row's chunks in turn,
// and the slots' sums are added in order.
template <typename P, int N>
__global__ void __launch_bounds__(kThreads) join_kernel(P* __restrict__ grad, const SumArgs a) {
    __shared__ uint32_t found[32];
    __shared__ uint32_t last[32];
    __shared__ int n_found;
    __shared__ float part[kThreads * N];
    const uint32_t width = a.units * N;
    if (threadIdx.x == 0) n_found = 0;
    if (threadIdx.x < 32) {
        const uint32_t chunk = blockIdx.x * 32 + threadIdx.x;
        bool starts = false;
        uint32_t end = 0;
        if (chunk < a.chunks) {
            const uint64_t p0 = static_cast<uint64_t>(chunk) * a.chunk, p1 = p0 + a.chunk;
            if (p1 < a.n) {
                const uint32_t row = a.keys[p1 - 1];
                starts = row < a.rows && a.keys[p1] == row && !(p0 > 0 && a.keys[p0] == row && a.keys[p0 - 1] == row);
                if (starts) {  // the first position past p1 with another row
                    uint32_t lo = static_cast<uint32_t>(p1), hi = a.n;
                    while (hi - lo > 1) {
                        const uint32_t mid = lo + (hi - lo) / 2;
                        if (a.keys[mid] == row) lo = mid;
                        else hi = mid;
                    }
                    end = lo / a.chunk;
                }
            }
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, starts);
        if (starts) {
            const int at = __popc(mask & ((1u << threadIdx.x) - 1u));
            found[at] = chunk;
            last[at] = end;
        }
        if (threadIdx.x == 0) n_found = __popc(mask);
    }
    __syncthreads();
    const uint32_t slots = kThreads / a.lanes, slot = threadIdx.x / a.lanes;
    const uint32_t col = blockIdx.y * a.lanes + threadIdx.x % a.lanes;
    for (int f = 0; f < n_found; f++) {
        float acc[N];
#pragma unroll
        for (int j = 0; j < N; j++) acc[j] = 0.0f;
        if (col < a.units) {
            if (slot == 0) {
#pragma unroll
                for (int j = 0; j < N; j++) acc[j] = a.tail[static_cast<uint64_t>(found[f]) * width + col * N + j];
            }
#pragma unroll 4
            for (uint32_t c = found[f] + 1 + slot; c <= last[f]; c += slots) {
#pragma unroll
                for (int j = 0; j < N; j++) acc[j] += a.head[static_cast<uint64_t>(c) * width + col * N + j];
            }
        }
#pragma unroll
        for (int j = 0; j < N; j++) part[threadIdx.x * N + j] = acc[j];
        __syncthreads();
        for (uint32_t half = slots / 2; half > 0; half /= 2) {
            if (slot < half) {
#pragma unroll
                for (int j = 0; j < N; j++) part[threadIdx.x * N + j] += part[(threadIdx.x + half * a.lanes) * N + j];
            }
            __syncthreads();
        }
        if (slot == 0 && col < a.units) {
#pragma unroll
            for (int j = 0; j < N; j++) acc[j] = part[threadIdx.x * N + j];
            write_row<P, N>(grad, a.keys[static_cast<uint64_t>(found[f] + 1) * a.chunk], a.units, col, acc, a.scale);
        }
        __syncthreads();
    }
}

struct GradBuffers {
    uint32_t *keys_a, *keys_b, *vals_a, *vals_b;
    uint8_t* used;
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

// tokens of a chunk: enough chunks to give each of 148 x 2048 threads a column, between 8 and 256 tokens
uint32_t chunk_of(uint64_t tokens, uint64_t width) {
    const uint64_t c = tokens * ((width + 3) / 4) / (148ull * 2048ull);
    uint32_t p = 8;
    while (p < c && p < 256) p *= 2;
    return p;
}

size_t carve(void* ws, uint64_t tokens, uint64_t rows, uint64_t width, GradBuffers* B) {
    char* base = static_cast<char*>(ws);
    size_t off = 0;
    const auto take = [&](size_t bytes) {
        off = (off + 255) & ~static_cast<size_t>(255);
        char* p = base ? base + off : nullptr;
        off += bytes;
        return p;
    };
    GradBuffers b;
    b.keys_a = reinterpret_cast<uint32_t*>(take(4 * tokens));
    b.keys_b = reinterpret_cast<uint32_t*>(take(4 * tokens));
    b.vals_a = reinterpret_cast<uint32_t*>(take(4 * tokens));
    b.vals_b = reinterpret_cast<uint32_t*>(take(4 * tokens));
    b.used = reinterpret_cast<uint8_t*>(take(rows));
    b.sort_bytes = tile_sort_temp_bytes(tokens, 32, true);
    b.sort_temp = take(b.sort_bytes);
    const uint64_t chunk = chunk_of(tokens, width), chunks = (tokens + chunk - 1) / chunk;
    b.head = reinterpret_cast<float*>(take(4 * chunks * width));
    b.tail = reinterpret_cast<float*>(take(4 * chunks * width));
    if (B) *B = b;
    return off;
}

template <typename P, int N>
cudaError_t launch_sums(const EmbeddingArgs& a, const void* g, void* grad, SumArgs S, cudaStream_t s) {
    const uint64_t units = static_cast<uint64_t>(a.width) / N;
    if (units > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    S.units = static_cast<uint32_t>(units);
    S.lanes = 1;
    while (S.lanes < 32 && S.lanes < units) S.lanes *= 2;
    S.groups = static_cast<uint32_t>((units + S.lanes - 1) / S.lanes);
    const uint64_t threads = static_cast<uint64_t>(S.chunks) * S.groups * S.lanes;
    const uint64_t sum_ctas = (threads + kThreads - 1) / kThreads;
    const uint64_t cells = static_cast<uint64_t>(a.rows) * units;
    const uint64_t zero_ctas = cells / (kThreads * 8) + 1 < 148 * 8 ? cells / (kThreads * 8) + 1 : 148 * 8;
    if (sum_ctas + zero_ctas > 0x7FFFFFFFull || S.groups > 65535) return cudaErrorInvalidValue;
    S.sum_ctas = static_cast<uint32_t>(sum_ctas);
    sum_kernel<P, N><<<static_cast<unsigned>(sum_ctas + zero_ctas), kThreads, 0, s>>>(static_cast<const P*>(g), static_cast<P*>(grad), S);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    if (S.chunks > 1) {
        join_kernel<P, N><<<dim3((S.chunks + 31) / 32, S.groups), kThreads, 0, s>>>(static_cast<P*>(grad), S);
        e = cudaGetLastError();
    }
    return e;
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
    return carve(nullptr, static_cast<uint64_t>(tokens), static_cast<uint64_t>(rows), static_cast<uint64_t>(width), nullptr);
}

cudaError_t launch_embedding_grad(const EmbeddingArgs& a, const void* index, const void* g, void* grad, void* ws, cudaStream_t s) {
    if (a.rows == 0 || a.width == 0) return cudaSuccess;
    const int size = a.dtype == kDtypeF32 ? 4 : 2;
    if (a.tokens == 0) return cudaMemsetAsync(grad, 0, static_cast<size_t>(a.rows) * static_cast<size_t>(a.width) * static_cast<size_t>(size), s);
    GradBuffers B;
    carve(ws, static_cast<uint64_t>(a.tokens), static_cast<uint64_t>(a.rows), static_cast<uint64_t>(a.width), &B);
    const uint32_t tokens = static_cast<uint32_t>(a.tokens);
    cudaError_t e = cudaMemsetAsync(B.used, 0, static_cast<size_t>(a.rows), s);
    if (e != cudaSuccess) return e;
    const unsigned ctas = (tokens + kThreads - 1) / kThreads;
    if (a.wide_index) keys_kernel<<<ctas, kThreads, 0, s>>>(static_cast<const int64_t*>(index), tokens, a.rows, a.padding, B.keys_a, B.vals_a, B.used);
    else keys_kernel<<<ctas, kThreads, 0, s>>>(static_cast<const int32_t*>(index), tokens, a.rows, a.padding, B.keys_a, B.vals_a, B.used);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const void* keys = nullptr;
    const uint32_t* vals = nullptr;
    e = tile_sort(B.keys_a, B.keys_b, B.vals_a, B.vals_b, tokens, bits_of(static_cast<uint64_t>(a.rows)), true, B.sort_temp, B.sort_bytes, &keys, &vals, s);
    if (e != cudaSuccess) return e;
    SumArgs S{};
    S.keys = static_cast<const uint32_t*>(keys);
    S.tokens = vals;
    S.used = B.used;
    S.head = B.head;
    S.tail = B.tail;
    S.n = tokens;
    S.rows = static_cast<uint32_t>(a.rows);
    S.chunk = chunk_of(tokens, static_cast<uint64_t>(a.width));
    S.chunks = (tokens + S.chunk - 1) / S.chunk;
    S.scale = a.scale;
    const int n = access_elements(a, size, g, grad);
#define FGS_SUMS(P, N) launch_sums<P, N>(a, g, grad, S, s)
    return FGS_BY_ACCESS(a.dtype, n, FGS_SUMS);
#undef FGS_SUMS
}

}  // namespace fgs
