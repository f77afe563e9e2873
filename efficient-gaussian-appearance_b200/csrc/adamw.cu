// AdamW over many tensors in one launch, with the moments in fp32 or in 8 bits, and the global gradient norm that
// clips it. Per element, with c the clip factor (1 without clipping) and t the tensor's step count:
//   g <- c g;  m <- b1 m + (1 - b1) g;  v <- b2 v + (1 - b2) g g
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// all in fp32 (products and sums rounded one by one: this file is built without contraction), p rounded once to its own type.
// Bound by HBM: every parameter, gradient and moment is read once and written once (28 bytes per fp32 element, 16 with
// 8-bit moments, 10 in bf16 with them). Measured on a B200 (6.56 TB/s copy): 59M fp32 elements 244 us (6.8 TB/s), with
// 8-bit moments 159 us (5.9 TB/s); 40M bf16 elements in 300 tensors with fp32 copies 171 us (6.6 TB/s), with 8-bit moments
// and no copies 99 us (4.0 TB/s: 63 instructions per element at 77 % of the issue slots; of 9.1 cycles per issue a warp waits
// 2.8 for loads, 2.0 ready but not picked, 1.3 for the half-rate pipes).
//
// Moments in 8 bits. 256 consecutive elements of a tensor (one warp's share) have one exponent byte E, the largest
// exponent among them. A code q != 0 stands for the float with the bits (q + 8 (E + 1) - top) << 20: three mantissa
// bits, counted down from the block's largest exponent. The first moment has a sign and seven bits (top = 127: 16
// octaves), the second eight bits (top = 255: 32 octaves, so that their ratio m / sqrt(v) has the same range). Float
// bits order like the values, so coding is integer arithmetic on them: no division, no table.
// Rounding: b2 = 0.999 changes v by far less than half a code step, so rounding to nearest would leave v where it is
// (tests/test_adamw.py simulates it: mean of v -71 % after 1000 steps of noisy gradients, updates off by 87 % rms). A threshold u is added under the third mantissa bit instead, from the additive
// recurrence u = frac(i a + t b) of the element index i and the step t (a from the golden ratio; b = 1/r or 1/r^2 with
// r the plastic number, r^3 = r + 1): over the steps an element's thresholds are evenly spread, so its rounding errors
// cancel instead of adding up (same simulation: -0.7 %, updates 11 %; independent random thresholds 0.2 %, 13 %). 1500 steps
// behind a drop of the gradients to a tenth, v lags by 10 % and the updates are off by 14 % (random ones 0.2 %, 24 %).
// Deterministic in (i, t). Values under the smallest code: m becomes that code or zero by its own threshold (unbiased);
// a nonzero v becomes the smallest code, never zero, since it divides. A block with an infinity or NaN has E = 255 and
// decodes to NaN throughout.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "dependent.cuh"
#include "launch.h"

namespace fgs {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBlock = kAdamwBlock;  // elements per warp and round; also the elements that share an exponent
static_assert(kBlock == 32 * 8, "eight elements per lane");
constexpr int kCtasPerSm = 4;  // 64 registers per thread
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
    uint32_t chunks;  // 32-bit moments: of kWarps blocks, one CTA's at a time; 8-bit moments: of `blocks` blocks, one warp's
    uint32_t blocks;
    const double* partials;   // sums of squared gradients (nullptr: no clipping)
    const float* factor;      // the clip factor, where it has been made from them (else nullptr)
    int n_partials;
    double max_norm;
    float* norm_out;
    bool dependent;  // launched as the programmatic dependent of the kernel before it
};
constexpr uint32_t kMaxRun = 8;  // blocks of a warp's run (at most 32: one lane each)

// whether the hardware hands out the CTAs as SMs become free (else: one resident grid, equal shares)
inline bool long_step(uint32_t chunks, uint32_t blocks, int sms) { return static_cast<uint64_t>(chunks) * blocks > static_cast<uint64_t>(sms) * 4 * kWarps * 8; }
// Tables of three sizes: a launch copies the whole table, and 28 KB of it took 3 us more of the host than 2 KB.
constexpr int kFewTensors = 24, kSomeTensors = 96, kManyTensors = 384;
static_assert(sizeof(Table<kManyTensors>) <= 32764, "kernel parameter limit");

__device__ inline float to_float(float x) { return x; }
__device__ inline float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ inline float to_float(__half x) { return __half2float(x); }
__device__ inline void from_float(float x, float& y) { y = x; }
__device__ inline void from_float(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
__device__ inline void from_float(float x, __half& y) { y = __float2half_rn(x); }

template <typename H>
__device__ inline void unpack8(const uint4& r, float (&x)[8]) {
    const H* h = reinterpret_cast<const H*>(&r);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = to_float(h[j]);
}

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
// loads issued where they stand: the compiler would otherwise put some of them behind the use of others
__device__ inline uint4 load16_rw(const void* a) {
    uint4 r;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(a));
    return r;
}
__device__ inline uint2 load8_rw(const void* a) {
    uint2 r;
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(a));
    return r;
}
__device__ inline void store32(void* a, const uint32_t (&x)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(a), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]),
                 "r"(x[6]), "r"(x[7])
                 : "memory");
}
template <typename H>
__device__ inline void load8(const H* a, float (&x)[8]) {
    unpack8<H>(*reinterpret_cast<const uint4*>(a), x);
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
// code bytes of a lane's eight elements: two packed words (VEC) or one per register
template <bool VEC>
__device__ inline void load_codes(const uint8_t* a, int lane, uint32_t left, uint32_t* q) {
    if (VEC) {
        const uint2 r = load8_rw(a + lane * 8);
        q[0] = r.x;
        q[1] = r.y;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = place<VEC>(lane, j) < left ? a[place<VEC>(lane, j)] : 0u;
    }
}
__device__ inline void store_codes(uint8_t* a, int lane, const uint32_t (&q)[2]) { *reinterpret_cast<uint2*>(a + lane * 8) = make_uint2(q[0], q[1]); }

// Square root within 2^-23 of the value, reciprocal too: with the product 5 roundings of half a step on an update that is
// itself a small part of the parameter; the exact ones took half of the 8-bit step's instructions. The reciprocal takes
// subnormals for zero: sqrt(v) is never one, and eps is not (checked on the host).
__device__ inline float root(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ inline float quotient(float x, float y) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    return x * r;
}

// value of one code of a block with any exponent
template <bool SIGNED>
__device__ inline float decode1(uint32_t code, int exponent) {
    constexpr int top = SIGNED ? 127 : 255;
    const int base = 8 * (exponent + 1) - top;
    const int c = static_cast<int>(code & top);
    const int k = c + base;
    uint32_t bits = c > 0 && k > 0 ? static_cast<uint32_t>(k) << 20 : 0u;
    if (exponent == 255) bits = 0x7fc00000u;
    if (SIGNED) bits |= (code & 128u) << 24;
    return __uint_as_float(bits);
}

// code of one element, `u` its threshold, in a block whose largest exponent is `high`
template <bool SIGNED>
__device__ inline uint32_t encode1(float x, uint32_t u, int high) {
    constexpr int top = SIGNED ? 127 : 255;
    const int base = 8 * (high + 1) - top;
    const int floor = base > 0 ? base : 0;
    const uint32_t least = static_cast<uint32_t>(floor + 1) << 20;
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    int c = static_cast<int>((b + (u >> 12)) >> 20) - base;
    if (b < least) {  // under the smallest code in use
        const float share = __uint_as_float(least) * 5.9604644775390625e-8f;  // least / 2^24
        const bool keep = SIGNED ? __uint_as_float(b) > static_cast<float>(u >> 8) * share : b > 0;
        c = keep ? floor + 1 - base : 0;
    }
    const int cap = top < 0x7f7 - base ? top : 0x7f7 - base;  // no code past the largest finite float
    c = c < cap ? c : cap;
    const uint32_t code = static_cast<uint32_t>(c) & 255u;
    return SIGNED ? (code & 127u) | (x < 0.0f ? 128u : 0u) : code;
}

// Values of two codes, as bf16 (which holds them exactly), from the halves of x: (q + base) << 4, zero for q = 0. Two
// codes per instruction, and products in the place of shifts and selections, which run at half the rate: the 8-bit step
// is mostly bound by them. For blocks with base >= 0, where every nonzero code has nonzero bits (subnormal ones at base 1 and
// 2, where no arithmetic touches them).
template <bool SIGNED>
__device__ inline uint32_t decode2(uint32_t x, uint32_t base) {
    const uint32_t q = SIGNED ? x & 0x007f007fu : x;
    // 16 in the halves with q != 0
    const uint32_t some = SIGNED ? ((q + 0x007f007fu) & 0x00800080u) >> 3 : ((q + 0x00ff00ffu) & 0x01000100u) >> 4;
    const uint32_t bits = q * 16u + some * base;
    return SIGNED ? bits + (x & 0x00800080u) * 256u : bits;
}
// the halves with the bytes 2 k and 2 k + 1 of a packed word
__device__ inline uint32_t code_pair(uint32_t word, int k) { return __byte_perm(word, 0, k ? 0x4342 : 0x4140); }

// values of one code each; the codes come as bytes of packed words (four each) or one per register (q[j] < 256)
template <bool SIGNED, bool PACKED>
__device__ inline void decode(const uint32_t* q, int exponent, float (&x)[8]) {
    constexpr int top = SIGNED ? 127 : 255;
    const int base = 8 * (exponent + 1) - top;
    if (base >= 0 && exponent != 255) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t two = decode2<SIGNED>(PACKED ? code_pair(q[j / 4], (j / 2) & 1) : q[j] | q[j + 1] << 16, static_cast<uint32_t>(base));
            x[j] = __uint_as_float(two << 16);
            x[j + 1] = __uint_as_float(two & 0xffff0000u);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = decode1<SIGNED>(PACKED ? (q[j / 4] >> (8 * (j & 3))) & 255u : q[j], exponent);
}

// packed codes of a whole block (all 32 lanes, eight consecutive elements each); returns the exponent byte. `u0`: the
// threshold of element 0 of the block.
template <bool SIGNED>
__device__ inline uint32_t encode(const float (&x)[8], uint32_t u0, int lane, uint32_t (&q)[2]) {
    constexpr int top = SIGNED ? 127 : 255;
    uint32_t b[8];  // bits of the magnitudes (the second moment has no sign; that of a NaN is cut off below)
#pragma unroll
    for (int j = 0; j < 8; j++) b[j] = SIGNED ? __float_as_uint(x[j]) & 0x7fffffffu : __float_as_uint(x[j]);
    uint32_t high = b[0] > b[1] ? b[0] : b[1], small = b[0] < b[1] ? b[0] : b[1];
#pragma unroll
    for (int j = 2; j < 8; j += 2) {
        high = __vimax3_u32(high, b[j], b[j + 1]);
        small = __vimin3_u32(small, b[j], b[j + 1]);
    }
    high = (__reduce_max_sync(0xffffffffu, high) >> 23) & 255u;
    const int base = 8 * (static_cast<int>(high) + 1) - top;
    const int floor = base > 0 ? base : 0;
    const uint32_t least = static_cast<uint32_t>(floor + 1) << 20;
    const uint32_t u = u0 + place<true>(lane, 0) * kTurn;
    if (high < 254 && small >= least) {  // the usual case: nothing under the smallest code or near the largest float
#pragma unroll
        for (int w = 0; w < 2; w++) {
            uint32_t k[4];  // the code in bits 24..31
#pragma unroll
            for (int j = 0; j < 4; j++) k[j] = (b[4 * w + j] + ((u + (4 * w + j) * kTurn) >> 12)) * 16u - (static_cast<uint32_t>(base) << 24);
            uint32_t word = __byte_perm(__byte_perm(k[0], k[1], 0x0073), __byte_perm(k[2], k[3], 0x0073), 0x5410);
            if (SIGNED) {
                const uint32_t lo = __byte_perm(__float_as_uint(x[4 * w]), __float_as_uint(x[4 * w + 1]), 0x0073);
                const uint32_t hi = __byte_perm(__float_as_uint(x[4 * w + 2]), __float_as_uint(x[4 * w + 3]), 0x0073);
                word |= __byte_perm(lo, hi, 0x5410) & 0x80808080u;
            }
            q[w] = word;
        }
        return high;
    }
    q[0] = q[1] = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) q[j / 4] |= encode1<SIGNED>(x[j], u + j * kTurn, static_cast<int>(high)) << (8 * (j & 3));
    return high;
}

// the addresses of a chunk's first elements
template <typename P>
struct Chunk {
    P* param;
    const P* grad;
    void* m;
    void* v;
    float* master;
};

// What a lane reads of one block. Halves read as a whole stay packed until they are used: converting them waits for the load.
template <typename P, bool EIGHT, bool MASTER>
struct Loaded {
    float p[8], g[8], m[8], v[8];
    uint4 packed_p, packed_g;
    uint32_t qm[2], qv[2];
};

template <typename P, bool EIGHT, bool MASTER, bool VEC>
__device__ inline void load_all(const Chunk<P>& C, uint32_t at, uint32_t left, int lane, Loaded<P, EIGHT, MASTER>& L) {
    constexpr bool packed = VEC && sizeof(P) == 2;
    if (packed) L.packed_g = load16_rw(C.grad + at + lane * 8);
    else load_block<VEC>(C.grad + at, lane, left, L.g);
    if (MASTER) load_block<VEC>(C.master + at, lane, left, L.p);
    else if (packed) L.packed_p = load16_rw(C.param + at + lane * 8);
    else load_block<VEC>(C.param + at, lane, left, L.p);
    if constexpr (EIGHT) {
        static_assert(VEC, "cut blocks of 8-bit moments: cut_block");
        load_codes<true>(static_cast<const uint8_t*>(C.m) + at, lane, left, L.qm);
        load_codes<true>(static_cast<const uint8_t*>(C.v) + at, lane, left, L.qv);
    } else {
        load_block<VEC>(static_cast<const float*>(C.m) + at, lane, left, L.m);
        load_block<VEC>(static_cast<const float*>(C.v) + at, lane, left, L.v);
    }
}

// The update of a lane's eight elements: p, m, v in L become the new ones. `start`: the block's first element within the tensor.
template <typename P, bool EIGHT, bool MASTER, bool VEC>
__device__ inline void update(const Hyper& H, uint64_t start, float clip, int lane, Loaded<P, EIGHT, MASTER>& L, uint32_t em, uint32_t ev) {
    if constexpr (VEC && sizeof(P) == 2) {
        unpack8<P>(L.packed_g, L.g);
        if (!MASTER) unpack8<P>(L.packed_p, L.p);
    }
    if constexpr (EIGHT) {
        decode<true, true>(L.qm, static_cast<int>(em), L.m);
        decode<false, true>(L.qv, static_cast<int>(ev), L.v);
    }
    // the moments decide the codes, so their products and sums are rounded one by one; the update is not coded
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float gc = clip * L.g[j];
        L.m[j] = H.beta1 * L.m[j] + H.rest1 * gc;
        L.v[j] = H.beta2 * L.v[j] + H.rest2 * gc * gc;
    }
    if (H.n_lr == 1) {
        const float lr = H.lr[0], decay = H.decay[0];
#pragma unroll
        for (int j = 0; j < 8; j++) L.p[j] = fmaf(-lr, quotient(L.m[j], fmaf(root(L.v[j]), H.root_rcp, H.eps)), L.p[j] * decay);
    } else {
        const uint32_t n_lr = static_cast<uint32_t>(H.n_lr), column = static_cast<uint32_t>(start % n_lr);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t c = (column + place<VEC>(lane, j)) % n_lr;
            L.p[j] = fmaf(-H.lr[c], quotient(L.m[j], fmaf(root(L.v[j]), H.root_rcp, H.eps)), L.p[j] * H.decay[c]);
        }
    }
}

template <typename P, bool EIGHT, bool MASTER, bool VEC>
__device__ inline void store_all(const Chunk<P>& C, const Hyper& H, uint64_t start, uint32_t at, uint32_t left, int lane, float (&p)[8], float (&m)[8],
                                 float (&v)[8], uint32_t& em, uint32_t& ev) {
    if (MASTER) store_block<VEC>(C.master + at, lane, left, p);
    store_block<VEC>(C.param + at, lane, left, p);
    if constexpr (EIGHT) {
        uint32_t q[2];
        const uint32_t u = static_cast<uint32_t>(start) * kTurn;
        em = encode<true>(m, u + H.dither_m, lane, q);
        store_codes(static_cast<uint8_t*>(C.m) + at, lane, q);
        ev = encode<false>(v, u + H.dither_v, lane, q);
        store_codes(static_cast<uint8_t*>(C.v) + at, lane, q);
    } else {
        store_block<VEC>(static_cast<float*>(C.m) + at, lane, left, m);
        store_block<VEC>(static_cast<float*>(C.v) + at, lane, left, v);
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

template <typename P, bool EIGHT, bool MASTER, typename TAB>
__device__ inline Chunk<P> chunk_at(const TAB& T, int t, uint64_t start) {
    return Chunk<P>{static_cast<P*>(T.param[t]) + start, static_cast<const P*>(T.grad[t]) + start, static_cast<char*>(T.m[t]) + start * (EIGHT ? 1 : 4),
                    static_cast<char*>(T.v[t]) + start * (EIGHT ? 1 : 4), MASTER ? T.master[t] + start : nullptr};
}

// A block that is cut or not aligned, one element of a lane after the other: rolled up, with the new moments in local
// memory, so that the whole blocks keep their registers (with both unrolled 80 registers and 117 us for 40M bf16 elements).
template <typename P, bool MASTER>
__device__ inline void cut_block(const Chunk<P>& C, const Hyper& H, uint64_t start, uint32_t at, uint32_t left, float clip, int lane, uint32_t& em,
                                 uint32_t& ev) {
    float m[8], v[8];
    uint32_t high_m = 0, high_v = 0;
#pragma unroll 1
    for (int j = 0; j < 8; j++) {
        const uint32_t i = place<false>(lane, j);
        m[j] = v[j] = 0.0f;  // places past the end take no part in the block's exponent (nor in anything else)
        if (i < left) {
            const float gc = clip * to_float(C.grad[at + i]);
            m[j] = H.beta1 * decode1<true>(static_cast<const uint8_t*>(C.m)[at + i], static_cast<int>(em)) + H.rest1 * gc;
            v[j] = H.beta2 * decode1<false>(static_cast<const uint8_t*>(C.v)[at + i], static_cast<int>(ev)) + H.rest2 * gc * gc;
            const uint32_t c = H.n_lr == 1 ? 0u : static_cast<uint32_t>((start + i) % static_cast<uint32_t>(H.n_lr));
            float p;
            if (MASTER) p = C.master[at + i];
            else p = to_float(C.param[at + i]);
            p = fmaf(-H.lr[c], quotient(m[j], fmaf(root(v[j]), H.root_rcp, H.eps)), p * H.decay[c]);
            if (MASTER) C.master[at + i] = p;
            from_float(p, C.param[at + i]);
        }
        const uint32_t bm = __float_as_uint(m[j]) & 0x7fffffffu, bv = __float_as_uint(v[j]) & 0x7fffffffu;
        high_m = bm > high_m ? bm : high_m;
        high_v = bv > high_v ? bv : high_v;
    }
    em = __reduce_max_sync(0xffffffffu, high_m) >> 23;
    ev = __reduce_max_sync(0xffffffffu, high_v) >> 23;
#pragma unroll 1
    for (int j = 0; j < 8; j++) {
        const uint32_t i = place<false>(lane, j);
        if (i >= left) break;
        const uint32_t u = (static_cast<uint32_t>(start) + i) * kTurn;
        static_cast<uint8_t*>(C.m)[at + i] = static_cast<uint8_t>(encode1<true>(m[j], u + H.dither_m, static_cast<int>(em)));
        static_cast<uint8_t*>(C.v)[at + i] = static_cast<uint8_t>(encode1<false>(v[j], u + H.dither_v, static_cast<int>(ev)));
    }
}

// A warp's run of blocks with 8-bit moments: lane b keeps the exponents of block b, read and written with one access per
// run. (One byte load and store per block, from different warps, made every read of a sector wait for the partial writes
// to it: 59M elements took 385 us, against 185 us without them.)
template <typename P, bool MASTER, int CAP>
__device__ inline void update_run(const Table<CAP>& T, uint32_t run, float clip, int lane) {
    const int t = owner(T, run);
    const Hyper& H = T.h[T.hyper[t] & 127];
    const uint64_t start = static_cast<uint64_t>(run - T.first[t]) * (T.blocks * kBlock);
    const uint64_t left = T.n[t] - start;
    const uint32_t have = left < T.blocks * kBlock ? static_cast<uint32_t>(left) : T.blocks * kBlock;  // elements
    const uint32_t blocks = (have + kBlock - 1) / kBlock;
    const Chunk<P> C = chunk_at<P, true, MASTER>(T, t, start);
    uint8_t* m_exp = T.m_exp[t] + start / kBlock;
    uint8_t* v_exp = T.v_exp[t] + start / kBlock;
    uint32_t em = 0, ev = 0;
    if (lane < blocks) {
        em = m_exp[lane];
        ev = v_exp[lane];
    }
    const bool vec = T.hyper[t] & 128;
    for (uint32_t b = 0; b < blocks; b++) {
        const uint32_t at = b * kBlock;
        uint32_t em_b = __shfl_sync(0xffffffffu, em, b), ev_b = __shfl_sync(0xffffffffu, ev, b);
        if (vec && have - at >= kBlock) {
            Loaded<P, true, MASTER> L;
            load_all<P, true, MASTER, true>(C, at, kBlock, lane, L);
            update<P, true, MASTER, true>(H, start + at, clip, lane, L, em_b, ev_b);
            store_all<P, true, MASTER, true>(C, H, start + at, at, kBlock, lane, L.p, L.m, L.v, em_b, ev_b);
        } else {
            cut_block<P, MASTER>(C, H, start + at, at, have - at < kBlock ? have - at : kBlock, clip, lane, em_b, ev_b);
        }
        if (lane == b) {
            em = em_b;
            ev = ev_b;
        }
    }
    if (lane < blocks) {
        m_exp[lane] = static_cast<uint8_t>(em);
        v_exp[lane] = static_cast<uint8_t>(ev);
    }
}

__device__ inline float clip_factor(double norm, double max_norm) {
    const double c = max_norm / (norm + 1e-6);
    return c < 1.0 ? static_cast<float>(c) : norm == norm ? 1.0f : __int_as_float(0x7fc00000);
}

// the norm and the clip factor from the partial sums, for steps of so many CTAs that not each should add them up
__global__ void __launch_bounds__(kThreads) clip_kernel(const double* partials, int n_partials, double max_norm, float* factor, float* norm_out) {
    __shared__ double scratch[kWarps];
    allow_dependent();
    wait_dependency();
    double x = 0.0;
    for (int i = threadIdx.x; i < n_partials; i += kThreads) x += partials[i];
    const double norm = sqrt(block_sum(x, scratch));
    if (threadIdx.x == 0) {
        *factor = clip_factor(norm, max_norm);
        *norm_out = static_cast<float>(norm);
    }
}

// The step. With fp32 moments a CTA's warps share chunks of 2048 elements, with 8-bit ones each warp takes a run of blocks.
// Aligned whole blocks move eight elements per lane (32-byte accesses in fp32).
template <typename P, bool EIGHT, bool MASTER, int CAP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) adamw_kernel(const __grid_constant__ Table<CAP> T) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float clip = 1.0f;
    if (T.partials) wait_dependency();
    if (T.factor) {
        clip = *T.factor;
    } else if (T.partials) {  // every CTA adds the partial sums in the same order: no further launch, no atomics
        __shared__ double scratch[kWarps];
        double x = 0.0;
        for (int i = threadIdx.x; i < T.n_partials; i += kThreads) x += T.partials[i];
        const double norm = sqrt(block_sum(x, scratch));
        clip = clip_factor(norm, T.max_norm);
        if (blockIdx.x == 0 && threadIdx.x == 0) *T.norm_out = static_cast<float>(norm);
    }
    const uint32_t first = share_of(T.chunks, blockIdx.x, gridDim.x), end = share_of(T.chunks, blockIdx.x + 1, gridDim.x);
    if (first == end) return;
    if constexpr (EIGHT) {
        for (uint32_t run = first + warp; run < end; run += kWarps) update_run<P, MASTER>(T, run, clip, lane);
    } else {
        const uint32_t at = static_cast<uint32_t>(warp) * kBlock;
        int t = owner(T, first);
        for (uint32_t chunk = first; chunk < end; chunk++) {
            while (chunk >= T.first[t + 1]) t++;
            const Hyper& H = T.h[T.hyper[t] & 127];
            const uint64_t start = static_cast<uint64_t>(chunk - T.first[t]) * (kWarps * kBlock);
            const uint64_t left = T.n[t] - start;
            const Chunk<P> C = chunk_at<P, EIGHT, MASTER>(T, t, start);
            Loaded<P, EIGHT, MASTER> L;
            uint32_t none = 0;
            if ((T.hyper[t] & 128) && left >= at + kBlock) {
                load_all<P, EIGHT, MASTER, true>(C, at, kBlock, lane, L);
                update<P, EIGHT, MASTER, true>(H, start + at, clip, lane, L, 0, 0);
                store_all<P, EIGHT, MASTER, true>(C, H, start + at, at, kBlock, lane, L.p, L.m, L.v, none, none);
            } else if (at < left) {
                const uint32_t have = left - at < kBlock ? static_cast<uint32_t>(left - at) : kBlock;
                load_all<P, EIGHT, MASTER, false>(C, at, have, lane, L);
                update<P, EIGHT, MASTER, false>(H, start + at, clip, lane, L, 0, 0);
                store_all<P, EIGHT, MASTER, false>(C, H, start + at, at, have, lane, L.p, L.m, L.v, none, none);
            }
        }
    }
}

template <typename P, bool EIGHT, bool MASTER, int CAP>
cudaError_t launch_table(const Table<CAP>& T, int sms, cudaStream_t s) {
    const uint32_t resident = static_cast<uint32_t>(sms) * kCtasPerSm;
    const uint32_t units = EIGHT ? (T.chunks + kWarps - 1) / kWarps : T.chunks;
    uint32_t grid = units < resident ? units : resident;
    // Long steps: CTAs of four chunks each, which the hardware hands out as SMs become free. Equal shares of one resident
    // grid ended at 123k to 172k cycles on different SMs (20M elements, 8-bit moments).
    if (long_step(T.chunks, T.blocks, sms)) grid = EIGHT ? units : (units + 3) / 4;
    // a clipped step overlaps the end of the norm's (or factor's) kernel, which its first instruction waits for
    if (T.dependent) return launch_dependent(adamw_kernel<P, EIGHT, MASTER, CAP>, dim3(grid), kThreads, 0, s, T);
    adamw_kernel<P, EIGHT, MASTER, CAP><<<grid, kThreads, 0, s>>>(T);
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
    bool factor_made = false;
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
        uint64_t blocks = 0;
        for (int j = 0; j < k; j++) blocks += (T.n[j] + kBlock - 1) / kBlock;
        T.blocks = kWarps;
        if (eight) {  // short steps are spread over as many warps as there are blocks
            T.blocks = 1;
            while (T.blocks < kMaxRun && blocks / T.blocks > static_cast<uint64_t>(sms) * 4 * kWarps * 4) T.blocks *= 2;
        }
        uint64_t chunks = 0;
        for (int j = 0; j < k; j++) {
            T.first[j] = static_cast<uint32_t>(chunks);
            const uint64_t per = static_cast<uint64_t>(kBlock) * T.blocks;
            chunks += (T.n[j] + per - 1) / per;
            if (chunks > 0xFFFFFFFFull - 65536) return cudaErrorInvalidValue;
        }
        T.first[k] = T.chunks = static_cast<uint32_t>(chunks);
        T.partials = clip.partials;
        T.n_partials = clip.n_partials;
        T.max_norm = clip.max_norm;
        T.norm_out = clip.norm_out;
        T.factor = nullptr;
        T.dependent = clip.partials != nullptr;
        if (clip.partials && long_step(T.chunks, T.blocks, sms)) {
            if (!factor_made) {
                const cudaError_t e = launch_dependent(clip_kernel, dim3(1), kThreads, 0, s, clip.partials, clip.n_partials, clip.max_norm, clip.factor, clip.norm_out);
                if (e != cudaSuccess) return e;
            }
            factor_made = true;
            T.factor = clip.factor;
        }
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
// Sum of squared gradients: per-thread fp32 sums over 32 elements, added up in fp64; one partial sum per CTA, added in a
// fixed order by the step (or clip_kernel). A thread whose fp32 sum overflows (gradients from 1.8e19 on, whose norm is finite)
// takes its share again in fp64. Bound by HBM: 80 MB of bf16 in 17 us (4.7 TB/s; with one load in flight per
// thread 31 us).

constexpr int kNormTensors = 1024;
constexpr uint32_t kNormChunk = kThreads * 8 * 4;

template <int CAP>
struct NormTable {
    uint32_t first[CAP + 1];
    const void* grad[CAP];
    uint64_t n[CAP];
    uint8_t kind[CAP];  // dtype; bit 7: aligned for whole-lane loads
    int n_tensors;
    uint32_t chunks;
    double* partials;
};
static_assert(sizeof(NormTable<kNormTensors>) <= 32764, "kernel parameter limit");

// 16 bytes, issued where it stands: the compiler would otherwise wait for each load before it issues the next one
__device__ inline uint4 load16(const void* a) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(a));
    return r;
}

// this thread's share of a chunk in fp64: `units` accesses of EACH elements, then single ones
template <typename P, int EACH>
__device__ __noinline__ double share_squares(const P* g, uint32_t units, uint32_t n) {
    double s = 0.0;
#pragma unroll 1
    for (uint32_t u = threadIdx.x; u < units; u += kThreads)
#pragma unroll 1
        for (int j = 0; j < EACH; j++) {
            const double y = to_float(g[u * EACH + j]);
            s = fma(y, y, s);
        }
#pragma unroll 1
    for (uint32_t j = units * EACH + threadIdx.x; j < n; j += kThreads) {
        const double y = to_float(g[j]);
        s = fma(y, y, s);
    }
    return s;
}

template <typename P>
__device__ inline double chunk_squares(const P* g, uint64_t left, bool vec) {
    constexpr int kEach = 16 / sizeof(P), kLoads = kNormChunk / kEach / kThreads;
    float s = 0.0f;
    const uint32_t n = left < kNormChunk ? static_cast<uint32_t>(left) : kNormChunk;
    const uint32_t units = vec ? n / kEach : 0;  // whole accesses
    uint4 x[kLoads];
#pragma unroll
    for (int r = 0; r < kLoads; r++) {
        const uint32_t u = r * kThreads + threadIdx.x;
        x[r] = make_uint4(0, 0, 0, 0);
        if (u < units) x[r] = load16(g + u * kEach);
    }
#pragma unroll
    for (int r = 0; r < kLoads; r++) {
        const P* y = reinterpret_cast<const P*>(&x[r]);
#pragma unroll
        for (int j = 0; j < kEach; j++) s = fmaf(to_float(y[j]), to_float(y[j]), s);
    }
    for (uint32_t j = units * kEach + threadIdx.x; j < n; j += kThreads) {
        const float y = to_float(g[j]);
        s = fmaf(y, y, s);
    }
    return s <= 3.4028234663852886e38f ? static_cast<double>(s) : share_squares<P, kEach>(g, units, n);
}

template <int CAP>
__global__ void __launch_bounds__(kThreads, 5) grad_squares_kernel(const __grid_constant__ NormTable<CAP> T) {
    __shared__ double scratch[kWarps];
    allow_dependent();
    double total = 0.0;
    const uint32_t first = share_of(T.chunks, blockIdx.x, gridDim.x), end = share_of(T.chunks, blockIdx.x + 1, gridDim.x);
    int t = owner(T, first);
    for (uint32_t chunk = first; chunk < end; chunk++) {
        while (chunk >= T.first[t + 1]) t++;
        const uint64_t start = static_cast<uint64_t>(chunk - T.first[t]) * kNormChunk;
        const uint64_t left = T.n[t] - start;
        const bool vec = T.kind[t] & 128;
        const int dtype = T.kind[t] & 127;
        double s;
        if (dtype == kDtypeF32) s = chunk_squares(static_cast<const float*>(T.grad[t]) + start, left, vec);
        else if (dtype == kDtypeBf16) s = chunk_squares(static_cast<const __nv_bfloat16*>(T.grad[t]) + start, left, vec);
        else s = chunk_squares(static_cast<const __half*>(T.grad[t]) + start, left, vec);
        total += s;
    }
    total = block_sum(total, scratch);
    if (threadIdx.x == 0) T.partials[blockIdx.x] = total;
}

// ---------------------------------------------------------------------------------------------------
// Values of 8-bit moments: one byte in, two (bf16, exact) or four out. Bound by HBM: both moments of 59M elements to bf16
// in 62 us (5.7 TB/s; with 16-byte instead of 32-byte stores 76 us).

constexpr int kReadTensors = 768;
template <int CAP>
struct ReadTable {
    uint32_t first[CAP + 1];
    const uint8_t* codes[CAP];
    const uint8_t* exps[CAP];
    void* out[CAP];
    uint64_t n[CAP];
    uint8_t kind[CAP];  // bit 0: signed, bit 7: aligned
    int n_tensors;
    uint32_t chunks;
};
static_assert(sizeof(ReadTable<kReadTensors>) <= 32764, "kernel parameter limit");

constexpr uint32_t kReadBlocks = 4;  // blocks of a warp's run

template <typename O, bool SIGNED>
__device__ inline void read_blocks(const uint8_t* codes, const uint8_t* exps, O* out, uint64_t start, uint64_t left, bool vec, int lane) {
    if (vec && left >= kReadBlocks * kBlock) {  // 16 codes per lane and access, both accesses in flight
        uint4 r[2];
        uint32_t e[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            r[h] = load16(codes + start + h * 2 * kBlock + lane * 16);
            e[h] = exps[start / kBlock + 2 * h + (lane >> 4)];
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            O* to = out + start + h * 2 * kBlock + lane * 16;
            const uint32_t q[4] = {r[h].x, r[h].y, r[h].z, r[h].w};
            const int base = 8 * (static_cast<int>(e[h]) + 1) - (SIGNED ? 127 : 255);
            if (sizeof(O) == 2 && base >= 0 && e[h] != 255) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; j++) w[j] = decode2<SIGNED>(code_pair(q[j / 2], j & 1), static_cast<uint32_t>(base));
                store32(to, w);
                continue;
            }
            float x[2][8];
            decode<SIGNED, true>(q, static_cast<int>(e[h]), x[0]);
            decode<SIGNED, true>(q + 2, static_cast<int>(e[h]), x[1]);
            store8(to, x[0]);
            store8(to + 8, x[1]);
        }
        return;
    }
    for (uint32_t b = 0; b < kReadBlocks && b * kBlock < left; b++) {
        const uint32_t have = left - b * kBlock < kBlock ? static_cast<uint32_t>(left - b * kBlock) : kBlock;
        uint32_t q[8];
        float x[8];
        load_codes<false>(codes + start + b * kBlock, lane, have, q);
        decode<SIGNED, false>(q, exps[start / kBlock + b], x);
        store_block<false>(out + start + b * kBlock, lane, have, x);
    }
}

template <typename O, int CAP>
__global__ void __launch_bounds__(kThreads) read_moments_kernel(const __grid_constant__ ReadTable<CAP> T) {
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
    if (A.count <= kSomeTensors) return launch_all<kSomeTensors>(A, hypers, dtype, eight, master, clip, s);
    return launch_all<kManyTensors>(A, hypers, dtype, eight, master, clip, s);
}

template <int CAP>
static cudaError_t grad_squares_by(const void* const* grads, const int64_t* n_elements, const uint8_t* dtypes, int count, double* partials,
                                int* n_partials, cudaStream_t s) {
    *n_partials = 0;
    int i = 0;
    while (i < count) {
        NormTable<CAP> T;
        int k = 0;
        uint64_t chunks = 0;
        for (; i < count && k < CAP; i++) {
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
        // one resident grid, or CTAs of two chunks that the hardware hands out as SMs become free
        const uint64_t resident = 148 * 5;
        const int grid = static_cast<int>(chunks < resident ? chunks : chunks < 2 * resident ? resident : chunks < 2 * kNormPartials ? chunks / 2 : kNormPartials);
        grad_squares_kernel<CAP><<<grid, kThreads, 0, s>>>(T);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        *n_partials += grid;
    }
    return cudaSuccess;
}

cudaError_t launch_grad_squares(const void* const* grads, const int64_t* n_elements, const uint8_t* dtypes, int count, double* partials,
                                int* n_partials, cudaStream_t s) {
    if (count <= kSomeTensors) return grad_squares_by<kSomeTensors>(grads, n_elements, dtypes, count, partials, n_partials, s);
    return grad_squares_by<kNormTensors>(grads, n_elements, dtypes, count, partials, n_partials, s);
}

int grad_squares_launches(int count) { return (count + kNormTensors - 1) / kNormTensors; }

template <int CAP>
static cudaError_t read_moments_by(const uint8_t* const* codes, const uint8_t* const* exps, const uint8_t* is_signed, const int64_t* n_elements, int count,
                                void* const* out, int dtype, cudaStream_t s) {
    const uint32_t cap = static_cast<uint32_t>(sm_count()) * 8;
    int i = 0;
    while (i < count) {
        ReadTable<CAP> T;
        int k = 0;
        uint64_t chunks = 0;
        for (; i < count && k < CAP; i++) {
            if (n_elements[i] <= 0) continue;
            T.codes[k] = codes[i];
            T.exps[k] = exps[i];
            T.out[k] = out[i];
            T.n[k] = static_cast<uint64_t>(n_elements[i]);
            T.kind[k] = static_cast<uint8_t>((is_signed[i] ? 1 : 0) | (aligned(codes[i], 16) && aligned(out[i], 32) ? 128 : 0));
            T.first[k] = static_cast<uint32_t>(chunks);
            chunks += (T.n[k] + kReadBlocks * kBlock * kWarps - 1) / (kReadBlocks * kBlock * kWarps);
            if (chunks > 0xFFFFFFFFull - 65536) return cudaErrorInvalidValue;
            k++;
        }
        if (k == 0) return cudaSuccess;
        T.first[k] = T.chunks = static_cast<uint32_t>(chunks);
        T.n_tensors = k;
        const uint32_t grid = T.chunks < cap ? T.chunks : cap;
        if (dtype == kDtypeF32) read_moments_kernel<float, CAP><<<grid, kThreads, 0, s>>>(T);
        else read_moments_kernel<__nv_bfloat16, CAP><<<grid, kThreads, 0, s>>>(T);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_read_moments(const uint8_t* const* codes, const uint8_t* const* exps, const uint8_t* is_signed, const int64_t* n_elements, int count,
                                void* const* out, int dtype, cudaStream_t s) {
    if (count <= kSomeTensors) return read_moments_by<kSomeTensors>(codes, exps, is_signed, n_elements, count, out, dtype, s);
    return read_moments_by<kReadTensors>(codes, exps, is_signed, n_elements, count, out, dtype, s);
}

}  // namespace fgs
