// adamw_cuda.cu -- one AdamW step over many tensors in one launch, moments held in 32 bits or in 8.
//
//   m <- b1 m + (1 - b1) g      v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A warp takes blocks of 256 consecutive elements of a tensor, eight per lane, over the tensors of the launch laid end to
// end; everything is read and written once: 28 bytes an element with fp32 parameters and moments, 16 with 8-bit moments,
// and those bytes are what bounds it, but for 8-bit moments, where the chain from a block's loads over its maximum to its codes takes longer
// (DRAM 42 %, issue slots 62 %, warps 43 %).  67 M elements: fp32 parameters with
// 32-bit moments 338 us (5.6 TB/s), with 8-bit ones 261 (4.1), bf16 238 (6.2) and 273.  Arithmetic is fp32, rounded to the
// parameter's type once, at the store.
//
// 8-bit moments.  The 256 elements of a block share an exponent `top` (one byte); an element's code keeps four bits of its
// exponent relative to that and S bits of its mantissa: S = 3 and a sign for m, S = 4 for the root of v (which is what the
// update divides by; a root needs half of v's exponent range and has no sign).  A code is a slice of the fp32 bits: value =
// float((code + ((top - 15) << S)) << (23 - S)), code 0 = zero.  Codes are rounded up or down at random so that their mean is
// the value: with b2 = 0.999 one step changes v by 0.1 %, far less than half a step of any 8-bit code (3 % here), so rounding
// to nearest would hold v where it is for good.  The random bits are a mix of (seed, tensor, step, element), so a run can be
// repeated.  Below the smallest code m goes to it or to zero in the same way; a root goes up to it, since the update divides
// by it.  `top` is taken after rounding up, so that the largest element is never cut off.  A value that is not finite makes
// its whole block not a number (top = 255).
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/cafe_b200.h"
#include "cafe_internal.h"
#include "cafe_float.cuh"

#define CAFE_ADAMW_BLOCK 256     // elements that share an exponent; a warp's piece of work
#define CAFE_ADAMW_THREADS 256

template <int NT>
struct CafeAdamwTensors {
    void* p[NT];
    const void* g[NT];
    void* m[NT];
    void* v[NT];
    uint8_t* mtop[NT];
    uint8_t* vtop[NT];
    int64_t* step[NT];
    int64_t n[NT];
    int64_t first[NT + 1];   // first block of each tensor in the launch's order
    int index[NT];           // number of the tensor in the optimizer; -1 - index: not on 16-byte boundaries
    int count;
};
struct CafeAdamwScalars {
    float lr, lr_decay, eps, b1, c1, b2, c2, log_b1, log_b2;
    uint32_t seed;
    int* ticket;
};

// A bijection of 32 bits: xorshifts by 16, 15, 16 between two odd multipliers, which Christopher Wellons found by searching for the least
// bias ("Prospecting for Hash Functions", nullprogram.com, 2018).
__device__ __forceinline__ uint32_t cafe_mix32(uint32_t x) {
    x ^= x >> 16; x *= 0x7FEB352Du; x ^= x >> 15; x *= 0x846CA68Bu; x ^= x >> 16;
    return x;
}

// A block's exponent `top` as the number that a code is counted from
template <int S> __device__ __forceinline__ uint32_t cafe_code_base(uint32_t top) { return (top - 15u) << S; }
// the exponent for a block whose largest magnitude has these bits: of the code grid's next point that is not below it
template <int S> __device__ __forceinline__ uint32_t cafe_code_top(uint32_t largest) {
    const uint32_t t = (largest + (1u << (23 - S)) - 1u) >> 23;
    return t < 16u ? 16u : t > 255u ? 255u : t;
}
// eight codes to their values
template <int S> __device__ __forceinline__ void cafe_code_values(const uint32_t* codes, uint32_t top, float* v) {
    const uint32_t base = cafe_code_base<S>(top) << (23 - S);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t x = codes[i >> 2] << (24 - 8 * (i & 3));   // the code in the highest byte (and others' below it)
        const uint32_t low = S == 3 ? (x >> 4) & 0x07f00000u : (x >> 5) & 0x07f80000u, bits = low ? low + base : 0u;
        v[i] = __uint_as_float(S == 3 ? bits | (x & 0x80000000u) : bits);
    }
    if (top == 255u) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(0x7fffffffu);
    }
}
// eight values to codes, rounded by the 16 random bits of each (S = 3 the low ones, else the high ones)
template <int S> __device__ __forceinline__ void cafe_codes(const float* v, uint32_t top, const uint32_t* rnd, uint32_t* codes) {
    const uint32_t base = cafe_code_base<S>(top) << (23 - S), least = base + (1u << (23 - S));
    uint32_t c[8], smallest = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = S == 3 ? __float_as_uint(v[i]) & 0x7fffffffu : __float_as_uint(v[i]);
        const uint32_t r = S == 3 ? (rnd[i] & 0xffffu) << 4 : (rnd[i] >> 16) << 3;
        c[i] = (bits + r - base) >> (23 - S);
        smallest = min(smallest, bits);
    }
    if (smallest < least) {   // below the smallest code: to it or to zero, or up to it
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t bits = __float_as_uint(v[i]) & 0x7fffffffu, r = rnd[i] & 0xffffu;
            const uint32_t low = S == 3 ? ((float)r * (__uint_as_float(least) * 0x1p-16f) < __uint_as_float(bits) ? 1u : 0u) : (bits ? 1u : 0u);
            if (bits < least) c[i] = low;
        }
    }
    codes[0] = codes[1] = 0u;
    if (top == 255u) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t x = S == 3 ? c[i] | ((__float_as_uint(v[i]) >> 24) & 0x80u) : c[i];
        codes[i >> 2] |= x << (8 * (i & 3));
    }
}

// Square root and reciprocal to 2^-22 of their value, for the update alone.
__device__ __forceinline__ float cafe_root_fast(float v) { float r; asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float cafe_inverse_fast(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
// The root that is kept: one step of Newton's iteration from the hardware's reciprocal root, x' = x + (v - x^2) y / 2 with x = v y,
// leaves less than 2^-24 of the value beside the last rounding.  Below the normal numbers it is zero or coarse; v that overflows
// gives a NaN, and with it its block.
__device__ __forceinline__ float cafe_root(float v) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaxf(v, 1.17549435e-38f)));
    const float x = v * y;
    return fmaf(fmaf(-x, x, v), 0.5f * y, x);
}

// eight consecutive elements, `ok` of them valid
template <typename T> __device__ __forceinline__ void cafe_load8(const T* p, int ok, bool vec, T* out) {
    if (vec && ok == 8) {
        const uint4* q = reinterpret_cast<const uint4*>(p);
        uint4* o = reinterpret_cast<uint4*>(out);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) o[i] = q[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = i < ok ? p[i] : cafe_from_float<T>(0.f);
    }
}
template <typename T> __device__ __forceinline__ void cafe_store8(T* p, int ok, bool vec, const T* in) {
    if (vec && ok == 8) {
        uint4* q = reinterpret_cast<uint4*>(p);
        const uint4* o = reinterpret_cast<const uint4*>(in);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = o[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < ok) p[i] = in[i];
    }
}
__device__ __forceinline__ void cafe_load_codes(const uint8_t* p, int ok, uint32_t* c) {   // (codes are the library's own arrays: on 8-byte boundaries)
    if (ok == 8) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        c[0] = x.x; c[1] = x.y;
    } else {
        c[0] = c[1] = 0u;
        for (int i = 0; i < ok; ++i) c[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    }
}
__device__ __forceinline__ void cafe_store_codes(uint8_t* p, int ok, const uint32_t* c) {
    if (ok == 8) *reinterpret_cast<uint2*>(p) = make_uint2(c[0], c[1]);
    else for (int i = 0; i < ok; ++i) p[i] = (uint8_t)(c[i >> 2] >> (8 * (i & 3)));
}

template <int NT>
__device__ __forceinline__ int cafe_adamw_find(const CafeAdamwTensors<NT>& P, int64_t block) {
    int lo = 0, hi = P.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (P.first[mid] <= block) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// The moments' products and sums are single roundings without contraction: a block's codes are then those of the formulas
// evaluated one operation after the other, whatever the compiler would fuse.
template <typename T, int BITS, int NT>
__global__ void __launch_bounds__(CAFE_ADAMW_THREADS, 4) k_adamw(const __grid_constant__ CafeAdamwTensors<NT> P, const CafeAdamwScalars S) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (CAFE_ADAMW_THREADS / 32);
    int t = -1;
    int64_t begin = 0, end = 0;       // the tensor's blocks
    float rate = 0.f, scale = 0.f;    // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    uint32_t key0 = 0;
    bool vec = false;
    for (int64_t blk = (int64_t)blockIdx.x * (CAFE_ADAMW_THREADS / 32) + (threadIdx.x >> 5); blk < P.first[P.count]; blk += warps) {
        const bool fresh = blk >= end;
        if (fresh) {
            t = cafe_adamw_find(P, blk);
            begin = P.first[t];
            end = P.first[t + 1];
            vec = P.index[t] >= 0;
        }
        const int64_t own = blk - begin, at = own * CAFE_ADAMW_BLOCK + lane * 8, left = P.n[t] - at;
        const int ok = left >= 8 ? 8 : left > 0 ? (int)left : 0;
        alignas(16) T p[8], g[8];
        alignas(16) float m[8], v[8];
        uint32_t cm[2], cv[2], tm = 0, tv = 0;
        T* pp = static_cast<T*>(P.p[t]) + at;
        cafe_load8(pp, ok, vec, p);
        cafe_load8(static_cast<const T*>(P.g[t]) + at, ok, vec, g);
        if constexpr (BITS == 32) {
            cafe_load8(static_cast<const float*>(P.m[t]) + at, ok, vec, m);
            cafe_load8(static_cast<const float*>(P.v[t]) + at, ok, vec, v);
        } else {
            cafe_load_codes(static_cast<const uint8_t*>(P.m[t]) + at, ok, cm);
            cafe_load_codes(static_cast<const uint8_t*>(P.v[t]) + at, ok, cv);
            tm = P.mtop[t][own];
            tv = P.vtop[t][own];
        }
        if (fresh) {
            const int64_t step = *P.step[t] + 1;
            rate = S.lr / -expm1f((float)step * S.log_b1);
            scale = rsqrtf(-expm1f((float)step * S.log_b2));
            const int index = vec ? P.index[t] : -1 - P.index[t];
            key0 = cafe_mix32(cafe_mix32(S.seed + 0x9E3779B9u * (uint32_t)(index + 1)) ^ (uint32_t)step);
        }
        if constexpr (BITS == 8) {
            cafe_code_values<3>(cm, tm, m);
            cafe_code_values<4>(cv, tv, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], v[i]);
        }
        uint32_t most_m = 0, most_v = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float gi = cafe_to_float(g[i]), pi = cafe_to_float(p[i]);
            m[i] = __fadd_rn(__fmul_rn(m[i], S.b1), __fmul_rn(gi, S.c1));
            v[i] = __fadd_rn(__fmul_rn(v[i], S.b2), __fmul_rn(__fmul_rn(gi, S.c2), gi));
            const float r = BITS == 8 ? cafe_root(v[i]) : cafe_root_fast(v[i]);
            p[i] = cafe_from_float<T>(pi - fmaf(S.lr_decay, pi, rate * m[i] * cafe_inverse_fast(fmaf(r, scale, S.eps))));
            if constexpr (BITS == 8) {
                v[i] = r;
                if (ok < 8 && i >= ok) m[i] = v[i] = 0.f;
                most_m = max(most_m, __float_as_uint(m[i]) & 0x7fffffffu);
                most_v = max(most_v, __float_as_uint(v[i]));
            }
        }
        cafe_store8(pp, ok, vec, p);
        if constexpr (BITS == 32) {
            cafe_store8(static_cast<float*>(P.m[t]) + at, ok, vec, m);
            cafe_store8(static_cast<float*>(P.v[t]) + at, ok, vec, v);
        } else {
            tm = cafe_code_top<3>(__reduce_max_sync(0xffffffffu, most_m));
            tv = cafe_code_top<4>(__reduce_max_sync(0xffffffffu, most_v));
            const uint32_t key = cafe_mix32(key0 + (uint32_t)(at >> 32));
            uint32_t rnd[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) rnd[i] = cafe_mix32((uint32_t)(at + i) ^ key);
            cafe_codes<3>(m, tm, rnd, cm);
            cafe_codes<4>(v, tv, rnd, cv);
            cafe_store_codes(static_cast<uint8_t*>(P.m[t]) + at, ok, cm);
            cafe_store_codes(static_cast<uint8_t*>(P.v[t]) + at, ok, cv);
            if (lane == 0) { P.mtop[t][own] = (uint8_t)tm; P.vtop[t][own] = (uint8_t)tv; }
        }
    }
    // the last block to finish counts the step: by then every block has read the counters
    __shared__ bool last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(S.ticket, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (last) {
        for (int t = threadIdx.x; t < P.count; t += CAFE_ADAMW_THREADS) *P.step[t] += 1;
        if (threadIdx.x == 0) *S.ticket = 0;
    }
}

// the values that 8-bit moments stand for, in bf16 (their 4 and 5 significant bits fit): out in the places of p and g
template <int NT>
__global__ void __launch_bounds__(CAFE_ADAMW_THREADS) k_adamw_moments(const __grid_constant__ CafeAdamwTensors<NT> P) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (CAFE_ADAMW_THREADS / 32);
    for (int64_t blk = (int64_t)blockIdx.x * (CAFE_ADAMW_THREADS / 32) + (threadIdx.x >> 5); blk < P.first[P.count]; blk += warps) {
        const int t = cafe_adamw_find(P, blk);
        const int64_t own = blk - P.first[t], at = own * CAFE_ADAMW_BLOCK + lane * 8, left = P.n[t] - at;
        const int ok = left >= 8 ? 8 : left > 0 ? (int)left : 0;
        const bool vec = P.index[t] >= 0;
        uint32_t cm[2], cv[2];
        cafe_load_codes(static_cast<const uint8_t*>(P.m[t]) + at, ok, cm);
        cafe_load_codes(static_cast<const uint8_t*>(P.v[t]) + at, ok, cv);
        float vm[8], vr[8];
        cafe_code_values<3>(cm, P.mtop[t][own], vm);
        cafe_code_values<4>(cv, P.vtop[t][own], vr);
        alignas(16) __nv_bfloat16 m[8], r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) { m[i] = __float2bfloat16_rn(vm[i]); r[i] = __float2bfloat16_rn(vr[i]); }
        cafe_store8(static_cast<__nv_bfloat16*>(P.p[t]) + at, ok, vec, m);
        cafe_store8(static_cast<__nv_bfloat16*>(const_cast<void*>(P.g[t])) + at, ok, vec, r);
    }
}

static bool adamw_on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// tensors [from, to) of the caller's lists as one launch's table; returns its blocks of 256 elements
template <int NT>
static int64_t adamw_table(CafeAdamwTensors<NT>* P, int from, int to, void* const* p, const void* const* g, void* const* m, void* const* v,
                           uint8_t* const* mtop, uint8_t* const* vtop, int64_t* const* step, const int64_t* n, const int* index) {
    P->count = to - from;
    P->first[0] = 0;
    for (int i = from; i < to; ++i) {
        const int k = i - from;
        P->p[k] = p[i]; P->g[k] = g[i]; P->m[k] = m[i]; P->v[k] = v[i];
        P->mtop[k] = mtop ? mtop[i] : nullptr; P->vtop[k] = vtop ? vtop[i] : nullptr;
        P->step[k] = step ? step[i] : nullptr;
        P->n[k] = n[i];
        P->first[k + 1] = P->first[k] + (n[i] + CAFE_ADAMW_BLOCK - 1) / CAFE_ADAMW_BLOCK;
        const bool vec = adamw_on16(p[i]) && adamw_on16(g[i]) && (mtop || (adamw_on16(m[i]) && adamw_on16(v[i])));
        const int ix = index ? index[i] : i;
        P->index[k] = vec ? ix : -1 - ix;
    }
    return P->first[P->count];
}
static unsigned adamw_grid(int64_t blocks, int per_sm) {
    const int64_t g = (blocks + CAFE_ADAMW_THREADS / 32 - 1) / (CAFE_ADAMW_THREADS / 32), most = 148 * (int64_t)per_sm;
    return (unsigned)(g < 1 ? 1 : g < most ? g : most);
}
template <typename T, int NT>
static void adamw_launch(int bits, const CafeAdamwTensors<NT>& P, const CafeAdamwScalars& S, int64_t blocks, cudaStream_t st) {
    const unsigned grid = adamw_grid(blocks, 4);
    if (bits == 32) k_adamw<T, 32, NT><<<grid, CAFE_ADAMW_THREADS, 0, st>>>(P, S);
    else k_adamw<T, 8, NT><<<grid, CAFE_ADAMW_THREADS, 0, st>>>(P, S);
}
// tensors per launch: what fits the 4 KB of parameters that a launch passes cheaply, or, for longer lists, 32 KB
#define CAFE_ADAMW_FEW 48
#define CAFE_ADAMW_MANY 400
static_assert(sizeof(CafeAdamwTensors<CAFE_ADAMW_FEW>) + sizeof(CafeAdamwScalars) <= 4096, "parameters of one launch");
static_assert(sizeof(CafeAdamwTensors<CAFE_ADAMW_MANY>) + sizeof(CafeAdamwScalars) <= 32764, "parameters of one launch");

static int adamw_lists_ok(int count, void* const* p, const void* const* g, void* const* m, void* const* v, const int64_t* n) {
    if (count < 0 || (count > 0 && (!p || !g || !m || !v || !n))) return 0;
    for (int i = 0; i < count; ++i)
        if (n[i] < 0 || (n[i] > 0 && (!p[i] || !g[i] || !m[i] || !v[i]))) return 0;
    return 1;
}

extern "C" {

int cafe_adamw_step(int count, void* const* p_dev, const void* const* g_dev, void* const* m_dev, void* const* v_dev, uint8_t* const* mtop_dev,
                    uint8_t* const* vtop_dev, int64_t* const* step_dev, const int64_t* numel, const int* index, int dtype, int bits,
                    double lr, double beta1, double beta2, double eps, double weight_decay, uint32_t seed, int* ticket_dev, void* stream) {
    if (!adamw_lists_ok(count, p_dev, g_dev, m_dev, v_dev, numel) || (bits != 32 && bits != 8) || dtype < CAFE_F32 || dtype > CAFE_F16) return CAFE_ERR_ARG;
    if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0)) return CAFE_ERR_ARG;
    if (count == 0) return CAFE_OK;
    if (!ticket_dev || !step_dev || (bits == 8 && (!mtop_dev || !vtop_dev))) return CAFE_ERR_ARG;
    for (int i = 0; i < count; ++i) {
        if (!step_dev[i]) return CAFE_ERR_ARG;
        if (bits == 8 && numel[i] > 0 && (!mtop_dev[i] || !vtop_dev[i] || ((uintptr_t)m_dev[i] & 7) || ((uintptr_t)v_dev[i] & 7))) return CAFE_ERR_ARG;
    }
    CafeAdamwScalars S;
    S.lr = (float)lr; S.lr_decay = (float)(lr * weight_decay); S.eps = (float)eps;
    S.b1 = (float)beta1; S.c1 = (float)(1.0 - beta1); S.b2 = (float)beta2; S.c2 = (float)(1.0 - beta2);
    S.log_b1 = (float)log(beta1); S.log_b2 = (float)log(beta2);   // (log 0 = -inf: 1 - 0^t = 1)
    S.seed = seed; S.ticket = ticket_dev;
    const cudaStream_t st = (cudaStream_t)stream;
    uint8_t* const* mt = bits == 8 ? mtop_dev : nullptr;
    uint8_t* const* vt = bits == 8 ? vtop_dev : nullptr;
    for (int from = 0; from < count;) {
        const bool few = count - from <= CAFE_ADAMW_FEW;
        const int most = few ? CAFE_ADAMW_FEW : CAFE_ADAMW_MANY, to = count - from < most ? count : from + most;
#define ADAMW_GO(NT)                                                                                                                \
    do {                                                                                                                            \
        static thread_local CafeAdamwTensors<NT> P;                                                                                 \
        const int64_t blocks = adamw_table<NT>(&P, from, to, p_dev, g_dev, m_dev, v_dev, mt, vt, step_dev, numel, index);           \
        CAFE_PROF(CAFE_P_ADAMW, st);                                                                                                \
        if (dtype == CAFE_F32) adamw_launch<float, NT>(bits, P, S, blocks, st);                                                     \
        else if (dtype == CAFE_BF16) adamw_launch<__nv_bfloat16, NT>(bits, P, S, blocks, st);                                       \
        else adamw_launch<__half, NT>(bits, P, S, blocks, st);                                                                      \
    } while (0)
        if (few) ADAMW_GO(CAFE_ADAMW_FEW); else ADAMW_GO(CAFE_ADAMW_MANY);
#undef ADAMW_GO
        from = to;
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) { cafe_internal_set_error(cudaGetErrorString(e)); return CAFE_ERR_CUDA; }
    return CAFE_OK;
}

int cafe_adamw_moments(int count, const uint8_t* const* m_dev, const uint8_t* const* mtop_dev, const uint8_t* const* r_dev,
                       const uint8_t* const* rtop_dev, const int64_t* numel, void* const* m_out_dev, void* const* r_out_dev, void* stream) {
    if (!adamw_lists_ok(count, m_out_dev, (const void* const*)r_out_dev, (void* const*)m_dev, (void* const*)r_dev, numel)) return CAFE_ERR_ARG;
    if (count > 0 && (!mtop_dev || !rtop_dev)) return CAFE_ERR_ARG;
    for (int i = 0; i < count; ++i)
        if (numel[i] > 0 && (!mtop_dev[i] || !rtop_dev[i] || ((uintptr_t)m_dev[i] & 7) || ((uintptr_t)r_dev[i] & 7))) return CAFE_ERR_ARG;
    const cudaStream_t st = (cudaStream_t)stream;
    for (int from = 0; from < count;) {
        const bool few = count - from <= CAFE_ADAMW_FEW;
        const int most = few ? CAFE_ADAMW_FEW : CAFE_ADAMW_MANY, to = count - from < most ? count : from + most;
#define MOMENTS_GO(NT)                                                                                                              \
    do {                                                                                                                            \
        static thread_local CafeAdamwTensors<NT> P;                                                                                 \
        const int64_t blocks = adamw_table<NT>(&P, from, to, m_out_dev, (const void* const*)r_out_dev, (void* const*)m_dev,         \
                                               (void* const*)r_dev, (uint8_t* const*)mtop_dev, (uint8_t* const*)rtop_dev, nullptr, numel, nullptr); \
        CAFE_PROF(CAFE_P_ADAMW, st);                                                                                                \
        k_adamw_moments<NT><<<adamw_grid(blocks, 8), CAFE_ADAMW_THREADS, 0, st>>>(P);                                               \
    } while (0)
        if (few) MOMENTS_GO(CAFE_ADAMW_FEW); else MOMENTS_GO(CAFE_ADAMW_MANY);
#undef MOMENTS_GO
        from = to;
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) { cafe_internal_set_error(cudaGetErrorString(e)); return CAFE_ERR_CUDA; }
    return CAFE_OK;
}

}  // extern "C"
