// AdamW over many tensors in one launch, with the moments in fp32 or in 8 bits, and the global gradient norm that
// clips it. Per element, with c the clip factor (1 without clipping) and t the tensor's step count:
//   g <- c g;  m <- b1 m + (1 - b1) g;  v <- b2 v + (1 - b2) g g
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// all in fp32 (products and sums rounded one by one: this file is built without contraction), p rounded once to its own type.
// Bound by HBM: every parameter, gradient and moment is read once and written once.
//
// Moments in 8 bits. 256 consecutive elements of a tensor (one warp's share) have one exponent byte E, the largest
// exponent among them. A code q != 0 stands for the float with the bits (q + 8 (E + 1) - top) << 20: three mantissa
// bits, counted down from the block's largest exponent. The first moment has a sign and seven bits (top = 127: 16
// octaves), the second eight bits (top = 255: 32 octaves, so that their ratio m / sqrt(v) has the same range). Float
// bits order like the values, so coding is integer arithmetic on them: no division, no table.
// Rounding: b2 = 0.999 changes v by far less than half a code step, so rounding to nearest would leave v where it is
// (simulated: -74 % after 1000 steps). A threshold u is added under the third mantissa bit instead, from the additive
// recurrence u = frac(i a + t b) of the element index i and the step t (a from the golden ratio; b = 1/r or 1/r^2 with
// r the plastic number, r^3 = r + 1): over the steps an element's thresholds are evenly spread, so its rounding errors
// cancel instead of adding up (simulated bias of v -0.4 %, update off by 11 % rms; independent random thresholds 24 %).
// Deterministic in (i, t). Values under the smallest code: m becomes that code or zero by its own threshold (unbiased);
// a nonzero v becomes the smallest code, never zero, since it divides. A block with an infinity or NaN has E = 255 and
// decodes to NaN throughout.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "launch.h"

namespace fgs {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBlock = kAdamwBlock;  // elements per warp and round; also the elements that share an exponent
static_assert(kBlock == 32 * 8, "eight elements per lane");
constexpr int kCtasPerSm = 4;
constexpr uint32_t kTurn = 0x9e3779b9u;  // 2^32 / golden ratio: the thresholds' step from element to element

struct Hyper {
    float lr[7], decay[7];  // lr / (1 - b1^t), 1 - lr wd
    int n_lr;
    float beta1, rest1, beta2, rest2, eps, root_rcp;  // rest = 1 - beta, root_rcp = 1 / sqrt(1 - b2^t)
    uint32_t dither_m, dither_v;
};

// the tensors of one launch, passed by value (kernel parameters may take 32764 bytes)
template <int CAP>
struct Table {
    uint32_t first[CAP + 1];  // first chunk of each tensor
    void* param[CAP];
    const void* grad[CAP];
    void* m[CAP];
    void* v[CAP];
    uint8_t* m_exp[CAP];
    uint8_t* v_exp[CAP];
    float* master[CAP];
    uint64_t n[CAP];
    uint8_t hyper[CAP];  // index into h; bit 7: every array is aligned for whole-lane accesses
    Hyper h[kMaxAdamwHypers];
    int n_tensors;
    uint32_t chunks;  // of kWarps blocks
    const double* partials;   // sums of squared gradients (nullptr: no clipping)
    int n_partials;
    double max_norm;
    float* norm_out;
};
constexpr int kFewTensors = 24, kManyTensors = 384;
static_assert(sizeof(Table<kManyTensors>) <= 32764, "kernel parameter limit");

__device__ inline float to_float(float x) { return x; }
__device__ inline float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ inline float to_float(__half x) { return __half2float(x); }
__device__ inline void from_float(float x, float& y) { y = x; }
__device__ inline void from_float(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
__device__ inline void from_float(float x, __half& y) { y = __float2half_rn(x); }

// eight consecutive elements of a lane: 32-byte accesses for fp32, 16 for the halves, 8 for codes
__device__ inline void load8(const float* a, float (&x)[8]) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                 : "l"(a));
}
__device__ inline void store8(float* a, const float (&x)[8]) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(a), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]),
                 "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
}
template <typename H>
__device__ inline void load8(const H* a, float (&x)[8]) {
    const uint4 r = *reinterpret_cast<const uint4*>(a);
    const H* h = reinterpret_cast<const H*>(&r);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = to_float(h[j]);
}
template <typename H>
__device__ inline void store8(H* a, const float (&x)[8]) {
    uint4 r;
    H* h = reinterpret_cast<H*>(&r);
#pragma unroll
    for (int j = 0; j < 8; j++) from_float(x[j], h[j]);
    *reinterpret_cast<uint4*>(a) = r;
}

// element of a block that a lane holds at j: eight consecutive ones per lane, or one of each 32
template <bool VEC>
__device__ inline uint32_t place(int lane, int j) { return VEC ? static_cast<uint32_t>(lane * 8 + j) : static_cast<uint32_t>(j * 32 + lane); }

// `left`: elements of the block that exist (kBlock with VEC)
template <bool VEC, typename P>
__device__ inline void load_block(const P* a, int lane, uint32_t left, float (&x)[8]) {
    if (VEC) {
        load8(a + lane * 8, x);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = place<VEC>(lane, j) < left ? to_float(a[place<VEC>(lane, j)]) : 0.0f;
    }
}
template <bool VEC, typename P>
__device__ inline void store_block(P* a, int lane, uint32_t left, const float (&x)[8]) {
    if (VEC) {
        store8(a + lane * 8, x);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (place<VEC>(lane, j) < left) from_float(x[j], a[place<VEC>(lane, j)]);
    }
}
template <bool VEC>
__device__ inline void load_codes(const uint8_t* a, int lane, uint32_t left, uint32_t (&q)[8]) {
    if (VEC) {
        const uint2 r = *reinterpret_cast<const uint2*>(a + lane * 8);
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = ((j < 4 ? r.x : r.y) >> (8 * (j & 3))) & 255u;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = place<VEC>(lane, j) < left ? a[place<VEC>(lane, j)] : 0u;
    }
}
template <bool VEC>
__device__ inline void store_codes(uint8_t* a, int lane, uint32_t left, const uint32_t (&q)[8]) {
    if (VEC) {
        uint2 r;
        r.x = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
        r.y = q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24;
        *reinterpret_cast<uint2*>(a + lane * 8) = r;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (place<VEC>(lane, j) < left) a[place<VEC>(lane, j)] = static_cast<uint8_t>(q[j]);
    }
}

// Square root within 2^-23 of the value, division within 2^-22: together 6 roundings of half a step on an update that
// is itself a small part of the parameter; the exact ones took half of the 8-bit step's instructions.
__device__ inline float root(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ inline float quotient(float x, float y) { return __fdividef(x, y); }

template <bool SIGNED>
__device__ inline void decode(const uint32_t (&q)[8], int exponent, float (&x)[8]) {
    constexpr int top = SIGNED ? 127 : 255;
    const int base = 8 * (exponent + 1) - top;
    if (base >= 0 && exponent != 255) {  // the usual case: every nonzero code is a normal float
        const uint32_t up = static_cast<uint32_t>(base) << 20;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t c = (q[j] & top) << 20;
            uint32_t bits = c ? c + up : 0u;
            if (SIGNED) bits |= (q[j] << 24) & 0x80000000u;
            x[j] = __uint_as_float(bits);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int c = static_cast<int>(q[j] & top);
        const int k = c + base;
        uint32_t bits = c > 0 && k > 0 ? static_cast<uint32_t>(k) << 20 : 0u;
        if (exponent == 255) bits = 0x7fc00000u;
        if (SIGNED) bits |= (q[j] & 128u) << 24;
        x[j] = __uint_as_float(bits);
    }
}

// codes of a block (all 32 lanes; elements that do not exist are zero); returns the exponent byte. `u0`: the threshold
// of element 0 of the block.
template <bool SIGNED, bool VEC>
__device__ inline uint32_t encode(const float (&x)[8], uint32_t u0, int lane, uint32_t (&q)[8]) {
    constexpr int top = SIGNED ? 127 : 255;
    uint32_t high = 0, small = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t b = __float_as_uint(x[j]) & 0x7fffffffu;
        high = b > high ? b : high;
        small = b < small ? b : small;
    }
    high = __reduce_max_sync(0xffffffffu, high) >> 23;
    const int base = 8 * (static_cast<int>(high) + 1) - top;
    const int floor = base > 0 ? base : 0;
    const uint32_t least = static_cast<uint32_t>(floor + 1) << 20;
    const uint32_t u = u0 + place<VEC>(lane, 0) * kTurn;
    if (high < 254 && small >= least) {  // the usual case: no element under the smallest code, none near the largest float
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t b = __float_as_uint(x[j]) & 0x7fffffffu;
            const uint32_t uj = u + (VEC ? j : 32 * j) * kTurn;
            q[j] = ((b + (uj >> 12)) >> 20) - static_cast<uint32_t>(base);
            if (SIGNED) q[j] |= (__float_as_uint(x[j]) >> 24) & 128u;
        }
        return high;
    }
    const int low = floor + 1 - base;                         // the smallest code in use
    const int cap = top < 0x7f7 - base ? top : 0x7f7 - base;  // no code past the largest finite float
    const float share = __uint_as_float(least) * 5.9604644775390625e-8f;  // least / 2^24
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t uj = u + (VEC ? j : 32 * j) * kTurn;
        const uint32_t b = __float_as_uint(x[j]) & 0x7fffffffu;
        int c = static_cast<int>((b + (uj >> 12)) >> 20) - base;
        if (b < least) {
            const bool keep = SIGNED ? __uint_as_float(b) > static_cast<float>(uj >> 8) * share : b > 0;
            c = keep ? low : 0;
        }
        c = c < cap ? c : cap;
        q[j] = static_cast<uint32_t>(c) & 255u;
        if (SIGNED) q[j] = (q[j] & 127u) | (x[j] < 0.0f ? 128u : 0u);
    }
    return high;
}

template <typename P, bool EIGHT, bool MASTER, bool VEC, int CAP>
__device__ inline void update_block(const Table<CAP>& T, int t, const Hyper& H, uint64_t start, uint32_t left, float clip, int lane) {
    P* param = static_cast<P*>(T.param[t]) + start;
    const P* grad = static_cast<const P*>(T.grad[t]) + start;
    float p[8], g[8], m[8], v[8];
    const uint64_t block = start / kBlock;
    load_block<VEC>(grad, lane, left, g);
    if (EIGHT) {
        uint32_t qm[8], qv[8];
        load_codes<VEC>(static_cast<const uint8_t*>(T.m[t]) + start, lane, left, qm);
        load_codes<VEC>(static_cast<const uint8_t*>(T.v[t]) + start, lane, left, qv);
        const int em = T.m_exp[t][block], ev = T.v_exp[t][block];
        decode<true>(qm, em, m);
        decode<false>(qv, ev, v);
    } else {
        load_block<VEC>(static_cast<const float*>(T.m[t]) + start, lane, left, m);
        load_block<VEC>(static_cast<const float*>(T.v[t]) + start, lane, left, v);
    }
    if (MASTER) load_block<VEC>(T.master[t] + start, lane, left, p);
    else load_block<VEC>(param, lane, left, p);
    // the moments decide the codes, so their products and sums are rounded one by one; the update is not coded
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float gc = clip * g[j];
        m[j] = H.beta1 * m[j] + H.rest1 * gc;
        v[j] = H.beta2 * v[j] + H.rest2 * gc * gc;
    }
    if (H.n_lr == 1) {
        const float lr = H.lr[0], decay = H.decay[0];
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = fmaf(-lr, quotient(m[j], fmaf(root(v[j]), H.root_rcp, H.eps)), p[j] * decay);
    } else {
        const uint32_t n_lr = static_cast<uint32_t>(H.n_lr), column = static_cast<uint32_t>(start % n_lr);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t c = (column + place<VEC>(lane, j)) % n_lr;
            p[j] = fmaf(-H.lr[c], quotient(m[j], fmaf(root(v[j]), H.root_rcp, H.eps)), p[j] * H.decay[c]);
        }
    }
    if (MASTER) store_block<VEC>(T.master[t] + start, lane, left, p);
    store_block<VEC>(param, lane, left, p);
    if (EIGHT) {
        if (!VEC) {  // places past the end take no part in the block's exponent (nor in anything else)
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (place<VEC>(lane, j) >= left) m[j] = v[j] = 0.0f;
        }
        uint32_t q[8];
        const uint32_t u = static_cast<uint32_t>(start) * kTurn;
        const uint32_t em = encode<true, VEC>(m, u + H.dither_m, lane, q);
        store_codes<VEC>(static_cast<uint8_t*>(T.m[t]) + start, lane, left, q);
        const uint32_t ev = encode<false, VEC>(v, u + H.dither_v, lane, q);
        store_codes<VEC>(static_cast<uint8_t*>(T.v[t]) + start, lane, left, q);
        if (lane == 0) {
            T.m_exp[t][block] = static_cast<uint8_t>(em);
            T.v_exp[t][block] = static_cast<uint8_t>(ev);
        }
    } else {
        store_block<VEC>(static_cast<float*>(T.m[t]) + start, lane, left, m);
        store_block<VEC>(static_cast<float*>(T.v[t]) + start, lane, left, v);
    }
}

// index of the tensor that owns `chunk`
template <typename TAB>
__device__ inline int owner(const TAB& T, uint32_t chunk) {
    int lo = 0, hi = T.n_tensors;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (T.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// first chunk of CTA `cta` when `chunks` are dealt out in runs as equal as they go
__device__ inline uint32_t share_of(uint32_t chunks, uint32_t cta, uint32_t ctas) {
    return static_cast<uint32_t>(static_cast<uint64_t>(chunks) * cta / ctas);
}

// sum of one double per thread over the CTA, the same in every thread and every run
__device__ inline double block_sum(double x, double* scratch) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) s += scratch[w];
    return s;
}

template <typename P, bool EIGHT, bool MASTER, int CAP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) adamw_kernel(const __grid_constant__ Table<CAP> T) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float clip = 1.0f;
    if (T.partials) {  // every CTA adds the partial sums in the same order: no further launch, no atomics
        __shared__ double scratch[kWarps];
        double x = 0.0;
        for (int i = threadIdx.x; i < T.n_partials; i += kThreads) x += T.partials[i];
        const double norm = sqrt(block_sum(x, scratch));
        const double c = T.max_norm / (norm + 1e-6);
        clip = c < 1.0 ? static_cast<float>(c) : norm == norm ? 1.0f : __int_as_float(0x7fc00000);
        if (blockIdx.x == 0 && threadIdx.x == 0) *T.norm_out = static_cast<float>(norm);
    }
    const uint32_t first = share_of(T.chunks, blockIdx.x, gridDim.x), end = share_of(T.chunks, blockIdx.x + 1, gridDim.x);
    if (first == end) return;
    // with clipping the norm has just walked the same shares front to back: their ends are still in L2
    const bool back = T.partials != nullptr;
    int t = owner(T, back ? end - 1 : first);
    for (uint32_t i = first; i < end; i++) {
        const uint32_t chunk = back ? first + end - 1 - i : i;
        while (chunk >= T.first[t + 1]) t++;
        while (chunk < T.first[t]) t--;
        const uint64_t n = T.n[t];
        const Hyper& H = T.h[T.hyper[t] & 127];
        const uint64_t start = (static_cast<uint64_t>(chunk - T.first[t]) * kWarps + warp) * kBlock;
        if (start >= n) continue;
        if ((T.hyper[t] & 128) && n - start >= kBlock) update_block<P, EIGHT, MASTER, true>(T, t, H, start, kBlock, clip, lane);
        else update_block<P, EIGHT, MASTER, false>(T, t, H, start, n - start < kBlock ? static_cast<uint32_t>(n - start) : kBlock, clip, lane);
    }
}

template <typename P, bool EIGHT, bool MASTER, int CAP>
cudaError_t launch_table(const Table<CAP>& T, int sms, cudaStream_t s) {
    const uint32_t cap = static_cast<uint32_t>(sms) * kCtasPerSm;
    adamw_kernel<P, EIGHT, MASTER, CAP><<<T.chunks < cap ? T.chunks : cap, kThreads, 0, s>>>(T);
    return cudaGetLastError();
}

int sm_count() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

template <int CAP>
cudaError_t launch_all(const AdamwTensors& A, const AdamwHyper* hypers, int dtype, bool eight, bool master, const AdamwClip& clip, cudaStream_t s) {
    const int sms = sm_count();
    const uintptr_t wide = dtype == kDtypeF32 ? 32 : 16;
    int i = 0;
    while (i < A.count) {
        Table<CAP> T;
        int k = 0, n_hyper = 0;
        int hyper_of[kMaxAdamwHypers];
        for (; i < A.count && k < CAP; i++) {
            if (A.n_elements[i] <= 0) continue;
            int h = 0;
            while (h < n_hyper && hyper_of[h] != A.hyper[i]) h++;
            if (h == n_hyper) {
                if (n_hyper == kMaxAdamwHypers) break;  // the rest goes into another launch
                hyper_of[n_hyper++] = A.hyper[i];
                const AdamwHyper& a = hypers[A.hyper[i]];
                Hyper& b = T.h[h];
                for (int j = 0; j < 7; j++) {
                    b.lr[j] = j < a.n_lr ? a.lr[j] : 0.0f;
                    b.decay[j] = j < a.n_lr ? a.decay[j] : 0.0f;
                }
                b.n_lr = a.n_lr;
                b.beta1 = a.beta1; b.rest1 = a.rest1; b.beta2 = a.beta2; b.rest2 = a.rest2;
                b.eps = a.eps; b.root_rcp = a.root_rcp;
                b.dither_m = a.step * 0xc13fa9a9u;
                b.dither_v = a.step * 0x91e10da5u;
            }
            T.param[k] = A.param[i];
            T.grad[k] = A.grad[i];
            T.m[k] = A.m[i];
            T.v[k] = A.v[i];
            T.m_exp[k] = eight ? A.m_exp[i] : nullptr;
            T.v_exp[k] = eight ? A.v_exp[i] : nullptr;
            T.master[k] = master ? A.master[i] : nullptr;
            T.n[k] = static_cast<uint64_t>(A.n_elements[i]);
            const uintptr_t moments = eight ? 8 : 32;
            const bool vec = aligned(A.param[i], wide) && aligned(A.grad[i], wide) && aligned(A.m[i], moments) && aligned(A.v[i], moments) &&
                             (!master || aligned(A.master[i], 32));
            T.hyper[k] = static_cast<uint8_t>(h | (vec ? 128 : 0));
            k++;
        }
        if (k == 0) return cudaSuccess;
        T.n_tensors = k;
        uint64_t chunks = 0;
        for (int j = 0; j < k; j++) {
            T.first[j] = static_cast<uint32_t>(chunks);
            const uint64_t per = static_cast<uint64_t>(kBlock) * kWarps;
            chunks += (T.n[j] + per - 1) / per;
            if (chunks > 0xFFFFFFFFull - 65536) return cudaErrorInvalidValue;
        }
        T.first[k] = T.chunks = static_cast<uint32_t>(chunks);
        T.partials = clip.partials;
        T.n_partials = clip.n_partials;
        T.max_norm = clip.max_norm;
        T.norm_out = clip.norm_out;
        cudaError_t e;
#define FGS_ADAMW(P, M) (eight ? launch_table<P, true, M, CAP>(T, sms, s) : launch_table<P, false, M, CAP>(T, sms, s))
        if (dtype == kDtypeF32) e = FGS_ADAMW(float, false);
        else if (dtype == kDtypeBf16) e = master ? FGS_ADAMW(__nv_bfloat16, true) : FGS_ADAMW(__nv_bfloat16, false);
        else e = master ? FGS_ADAMW(__half, true) : FGS_ADAMW(__half, false);
#undef FGS_ADAMW
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// ---------------------------------------------------------------------------------------------------
// sum of squared gradients: per-thread fp32 sums over 32 elements, added up in fp64; one partial sum per CTA

constexpr int kNormTensors = 1024;
constexpr uint32_t kNormChunk = kThreads * 8 * 4;

struct NormTable {
    uint32_t first[kNormTensors + 1];
    const void* grad[kNormTensors];
    uint64_t n[kNormTensors];
    uint8_t kind[kNormTensors];  // dtype; bit 7: aligned for whole-lane loads
    int n_tensors;
    uint32_t chunks;
    double* partials;
};
static_assert(sizeof(NormTable) <= 32764, "kernel parameter limit");

template <typename P>
__device__ inline float chunk_squares(const P* g, uint64_t left, bool vec) {
    float s = 0.0f;
    if (vec && left >= kNormChunk) {
        float x[4][8];
#pragma unroll
        for (int r = 0; r < 4; r++) load8(g + (r * kThreads + threadIdx.x) * 8, x[r]);
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int j = 0; j < 8; j++) s = fmaf(x[r][j], x[r][j], s);
    } else {
        const uint32_t n = left < kNormChunk ? static_cast<uint32_t>(left) : kNormChunk;
#pragma unroll 8
        for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
            const float x = to_float(g[j]);
            s = fmaf(x, x, s);
        }
    }
    return s;
}

__global__ void __launch_bounds__(kThreads, kNormPartials / 148) grad_squares_kernel(const __grid_constant__ NormTable T) {
    __shared__ double scratch[kWarps];
    double total = 0.0;
    const uint32_t first = share_of(T.chunks, blockIdx.x, gridDim.x), end = share_of(T.chunks, blockIdx.x + 1, gridDim.x);
    int t = owner(T, first);
    for (uint32_t chunk = first; chunk < end; chunk++) {
        while (chunk >= T.first[t + 1]) t++;
        const uint64_t start = static_cast<uint64_t>(chunk - T.first[t]) * kNormChunk;
        const uint64_t left = T.n[t] - start;
        const bool vec = T.kind[t] & 128;
        const int dtype = T.kind[t] & 127;
        float s;
        if (dtype == kDtypeF32) s = chunk_squares(static_cast<const float*>(T.grad[t]) + start, left, vec);
        else if (dtype == kDtypeBf16) s = chunk_squares(static_cast<const __nv_bfloat16*>(T.grad[t]) + start, left, vec);
        else s = chunk_squares(static_cast<const __half*>(T.grad[t]) + start, left, vec);
        total += s;
    }
    total = block_sum(total, scratch);
    if (threadIdx.x == 0) T.partials[blockIdx.x] = total;
}

// ---------------------------------------------------------------------------------------------------
// values of 8-bit moments

constexpr int kReadTensors = 512;
struct ReadTable {
    uint32_t first[kReadTensors + 1];
    const uint8_t* codes[kReadTensors];
    const uint8_t* exps[kReadTensors];
    void* out[kReadTensors];
    uint64_t n[kReadTensors];
    uint8_t kind[kReadTensors];  // bit 0: signed, bit 7: aligned
    int n_tensors;
    uint32_t chunks;
};
static_assert(sizeof(ReadTable) <= 32764, "kernel parameter limit");

constexpr uint32_t kReadBlocks = 4;  // blocks of a warp's run

template <typename O, bool SIGNED>
__device__ inline void read_blocks(const uint8_t* codes, const uint8_t* exps, O* out, uint64_t start, uint64_t left, bool vec, int lane) {
    if (vec && left >= kReadBlocks * kBlock) {  // 16 codes per lane and access, both accesses in flight
        uint4 r[2];
        uint32_t e[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            r[h] = *reinterpret_cast<const uint4*>(codes + start + h * 2 * kBlock + lane * 16);
            e[h] = exps[start / kBlock + 2 * h + (lane >> 4)];
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint32_t lo = k ? r[h].z : r[h].x, hi = k ? r[h].w : r[h].y;
                uint32_t q[8];
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; j++) q[j] = ((j < 4 ? lo : hi) >> (8 * (j & 3))) & 255u;
                decode<SIGNED>(q, static_cast<int>(e[h]), x);
                store8(out + start + h * 2 * kBlock + lane * 16 + 8 * k, x);
            }
        }
        return;
    }
    for (uint32_t b = 0; b < kReadBlocks && b * kBlock < left; b++) {
        const uint32_t have = left - b * kBlock < kBlock ? static_cast<uint32_t>(left - b * kBlock) : kBlock;
        uint32_t q[8];
        float x[8];
        load_codes<false>(codes + start + b * kBlock, lane, have, q);
        decode<SIGNED>(q, exps[start / kBlock + b], x);
        store_block<false>(out + start + b * kBlock, lane, have, x);
    }
}

template <typename O>
__global__ void __launch_bounds__(kThreads) read_moments_kernel(const __grid_constant__ ReadTable T) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t first = share_of(T.chunks, blockIdx.x, gridDim.x), end = share_of(T.chunks, blockIdx.x + 1, gridDim.x);
    int t = owner(T, first);
    for (uint32_t chunk = first; chunk < end; chunk++) {
        while (chunk >= T.first[t + 1]) t++;
        const uint64_t n = T.n[t];
        const uint64_t start = (static_cast<uint64_t>(chunk - T.first[t]) * kWarps + warp) * (kReadBlocks * kBlock);
        if (start >= n) continue;
        O* out = static_cast<O*>(T.out[t]);
        const bool vec = T.kind[t] & 128;
        if (T.kind[t] & 1) read_blocks<O, true>(T.codes[t], T.exps[t], out, start, n - start, vec, lane);
        else read_blocks<O, false>(T.codes[t], T.exps[t], out, start, n - start, vec, lane);
    }
}

}  // namespace

cudaError_t launch_adamw(const AdamwTensors& A, const AdamwHyper* hypers, int dtype, bool eight, bool master, const AdamwClip& clip, cudaStream_t s) {
    if (A.count <= kFewTensors) return launch_all<kFewTensors>(A, hypers, dtype, eight, master, clip, s);
    return launch_all<kManyTensors>(A, hypers, dtype, eight, master, clip, s);
}

cudaError_t launch_grad_squares(const void* const* grads, const int64_t* n_elements, const uint8_t* dtypes, int count, double* partials,
                                int* n_partials, cudaStream_t s) {
    *n_partials = 0;
    int i = 0;
    while (i < count) {
        NormTable T;
        int k = 0;
        uint64_t chunks = 0;
        for (; i < count && k < kNormTensors; i++) {
            if (n_elements[i] <= 0) continue;
            T.grad[k] = grads[i];
            T.n[k] = static_cast<uint64_t>(n_elements[i]);
            T.kind[k] = static_cast<uint8_t>(dtypes[i] | (aligned(grads[i], dtypes[i] == kDtypeF32 ? 32 : 16) ? 128 : 0));
            T.first[k] = static_cast<uint32_t>(chunks);
            chunks += (T.n[k] + kNormChunk - 1) / kNormChunk;
            if (chunks > 0xFFFFFFFFull - 65536) return cudaErrorInvalidValue;
            k++;
        }
        if (k == 0) return cudaSuccess;
        T.first[k] = T.chunks = static_cast<uint32_t>(chunks);
        T.n_tensors = k;
        T.partials = partials + *n_partials;
        const int grid = chunks < kNormPartials ? static_cast<int>(chunks) : kNormPartials;
        grad_squares_kernel<<<grid, kThreads, 0, s>>>(T);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        *n_partials += grid;
    }
    return cudaSuccess;
}

int grad_squares_launches(int count) { return (count + kNormTensors - 1) / kNormTensors; }

cudaError_t launch_read_moments(const uint8_t* const* codes, const uint8_t* const* exps, const uint8_t* is_signed, const int64_t* n_elements, int count,
                                void* const* out, int dtype, cudaStream_t s) {
    const uint32_t cap = static_cast<uint32_t>(sm_count()) * 8;
    int i = 0;
    while (i < count) {
        ReadTable T;
        int k = 0;
        uint64_t chunks = 0;
        for (; i < count && k < kReadTensors; i++) {
            if (n_elements[i] <= 0) continue;
            T.codes[k] = codes[i];
            T.exps[k] = exps[i];
            T.out[k] = out[i];
            T.n[k] = static_cast<uint64_t>(n_elements[i]);
            T.kind[k] = static_cast<uint8_t>((is_signed[i] ? 1 : 0) | (aligned(codes[i], 16) && aligned(out[i], dtype == kDtypeF32 ? 32 : 16) ? 128 : 0));
            T.first[k] = static_cast<uint32_t>(chunks);
            chunks += (T.n[k] + kReadBlocks * kBlock * kWarps - 1) / (kReadBlocks * kBlock * kWarps);
            if (chunks > 0xFFFFFFFFull - 65536) return cudaErrorInvalidValue;
            k++;
        }
        if (k == 0) return cudaSuccess;
        T.first[k] = T.chunks = static_cast<uint32_t>(chunks);
        T.n_tensors = k;
        const uint32_t grid = T.chunks < cap ? T.chunks : cap;
        if (dtype == kDtypeF32) read_moments_kernel<float><<<grid, kThreads, 0, s>>>(T);
        else read_moments_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(T);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace fgs
