// dense.cuh -- what the kernels of the dense layers share: activations, the description of a product, its end.
#pragma once
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "../../include/cafe_b200.h"
#include "cafe_internal.h"
#include "cafe_float.cuh"
#include "tcgen05.cuh"

#define CAFE_LIN_BM 128   // rows of a block's outputs

// act(z), and its derivative.  Exponentials and reciprocals come from the hardware's functions: relative error 2^-22 + 2^-24 |x| of
// exp(x), 2^-23 of 1 / x, which is what a sum in fp32 has anyway; the exactly rounded forms tripled the instructions of an epilogue
// (65536x479x1024 with GELU and slope 574 us against 394 without).
__device__ __forceinline__ float cafe_exp(float x) { return __expf(x); }
__device__ __forceinline__ float cafe_inverse(float x) { return __fdividef(1.f, x); }
__device__ __forceinline__ float cafe_act(float z, int act, float* slope) {
    switch (act) {
        case CAFE_ACT_RELU: *slope = z > 0.f ? 1.f : 0.f; return z > 0.f ? z : (z != z ? z : 0.f);
        case CAFE_ACT_SIGMOID: case CAFE_ACT_SILU: {
            // e = exp(-|z|) never overflows; s and t = 1 - s keep their relative precision in both tails
            const float e = cafe_exp(-fabsf(z)), d = cafe_inverse(1.f + e);
            const float s = z >= 0.f ? d : e * d, t = z >= 0.f ? e * d : d;
            if (act == CAFE_ACT_SIGMOID) { *slope = s * t; return s; }
            *slope = s * (1.f + z * t);
            return z * s;
        }
        case CAFE_ACT_GELU: {
            // the normal distribution's tail below -|z|: half of exp(-z^2 / 2) times exp(y^2) erfc(y), y = |z| / sqrt(2), for which
            // a polynomial of degree 9 in t = 1 / (1 + y / 2) without constant term was fitted here (least largest relative error
            // on [0, 12]: 4.4e-8; evaluated in fp32 3.2e-7).  The derivative takes the same exponential.
            const float e = cafe_exp(-0.5f * z * z), t = cafe_inverse(1.f + 0.353553391f * fabsf(z));
            float q = -0.0593632702f;
            q = fmaf(q, t, 0.286011492f); q = fmaf(q, t, -0.490175051f); q = fmaf(q, t, 0.28147069f); q = fmaf(q, t, -0.0289692743f);
            q = fmaf(q, t, 0.203677501f); q = fmaf(q, t, 0.242853828f); q = fmaf(q, t, 0.282409568f); q = fmaf(q, t, 0.282084473f);
            const float h = 0.5f * e * (q * t), c = z > 0.f ? 1.f - h : h;
            *slope = c + z * e * 0.398942280f;
            return z * c;
        }
        default: *slope = 1.f; return z;
    }
}
// N at a time: z becomes act(z), d its derivative
template <int N> __device__ __forceinline__ void cafe_act_all(float* z, int act, float* d) {
#define CAFE_ACT_CASE(A) case A: { _Pragma("unroll") for (int q = 0; q < N; ++q) z[q] = cafe_act(z[q], A, d + q); break; }
    switch (act) {
        CAFE_ACT_CASE(CAFE_ACT_RELU)
        CAFE_ACT_CASE(CAFE_ACT_SIGMOID)
        CAFE_ACT_CASE(CAFE_ACT_GELU)
        CAFE_ACT_CASE(CAFE_ACT_SILU)
        default: {
#pragma unroll
            for (int q = 0; q < N; ++q) d[q] = 1.f;
        }
    }
#undef CAFE_ACT_CASE
}

// The derivative kept for the backward: fp32, or beside bf16 a code of 16 bits.  bf16 gradients have the exponents of fp32 (a sigmoid
// under a cross-entropy meets gy = -1 / y, so that a derivative of 1e-35 still counts), which fp16 alone has not: it is zero below
// 2^-25, where gz = -1 became 0 from z = -17.5 on.  No derivative reaches 2 (they lie in [-0.2, 1.2]), so the codes of fp16 from 2 on are free and
// hold the bf16 codes of what is below 2^-17 (at most 0x3700, added to 0x4000).  Error: 2^-11 of the value down to 2^-14, 2^-25 down to 2^-17, where
// that is 2^-8 of it, and 2^-8 of it below, down to bf16's own smallest numbers; gz's rounding to bf16 has 2^-8.
struct CafeSlope16 { uint16_t code; };
template <> __device__ __forceinline__ float cafe_to_float<CafeSlope16>(CafeSlope16 x) {
    const uint32_t m = x.code & 0x7fffu;
    const float low = __uint_as_float((x.code & 0x8000u) << 16 | (m - 0x4000u) << 16);
    return m - 0x4000u < 0x3c00u ? low : __half2float(__ushort_as_half(x.code));   // (from 0x7c00 on: not a number)
}
// two codes at once (what is below 2 in magnitude, or not a number, carries nothing from one to the other); one by one they took 14 us of
// the 254 of 16384x1024x4096 forward with GELU and residual, so 3
__device__ __forceinline__ uint32_t cafe_slope16_pair(float x, float y) {
    const __half2 high = __floats2half2_rn(x, y);
    const __nv_bfloat162 low = __floats2bfloat162_rn(x, y);
    const uint32_t small = __hlt2_mask(__habs2(high), __float2half2_rn(0x1p-17f));
    return ((reinterpret_cast<const uint32_t&>(low) + 0x40004000u) & small) | (reinterpret_cast<const uint32_t&>(high) & ~small);
}
template <> __device__ __forceinline__ CafeSlope16 cafe_from_float<CafeSlope16>(float x) { return CafeSlope16{(uint16_t)cafe_slope16_pair(x, x)}; }
// N derivatives as they are kept (out on 4 bytes)
template <int N> __device__ __forceinline__ void cafe_slopes(const float* d, float* out) {
#pragma unroll
    for (int q = 0; q < N; ++q) out[q] = d[q];
}
template <int N> __device__ __forceinline__ void cafe_slopes(const float* d, CafeSlope16* out) {
#pragma unroll
    for (int q = 0; q < N; q += 2) reinterpret_cast<uint32_t*>(out)[q / 2] = cafe_slope16_pair(d[q], d[q + 1]);
}
template <typename T> struct CafeSlopeOf { typedef float type; };
template <> struct CafeSlopeOf<__nv_bfloat16> { typedef CafeSlope16 type; };

// a load through the read-only path
template <typename T> __device__ __forceinline__ T cafe_ldg(const T* p) { return __ldg(p); }
template <> __device__ __forceinline__ CafeSlope16 cafe_ldg<CafeSlope16>(const CafeSlope16* p) { return CafeSlope16{__ldg(&p->code)}; }

struct CafeJob {
    const void *a, *as, *b;
    int64_t lda, ldas, ldb;
    int a_kc, b_kc, a_vec, as_vec, b_vec;   // k contiguous; 16-byte loads allowed
    int slope_kind, rows, cols, depth;
    int tiles_n, tiles;
    const void *bias, *res;
    int64_t ldr, ldo, lds;
    int act, out_vec, res_vec;              // 16-byte stores of four outputs (and slopes), loads of four of the residual; ..
    int out_row, slope_row, res_row;        // .. rows on 16 bytes
    void *out, *slope_out, *gb;             // gb: sums over k of A(i, k), by the blocks of the first column of tiles
};
struct CafeJobs {
    CafeJob job[2];
    int count;
};

__device__ __forceinline__ void cafe_put16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// The large sums of split operands and the others joined.  Of infinite operands the large sums alone are right: the lower parts of an
// infinity are NaN, and times a lower part that is zero it would be one too.  (An infinity times a number below 2^-133, whose upper
// part is zero, becomes NaN.)
__device__ __forceinline__ float cafe_join_sums(float large, float rest) { return fabsf(large) < INFINITY ? large + rest : large; }
// Split operands: after how many pieces of the large sums the others are taken out as well (pieces of 256 of k, so every 4096).  They
// are 2^-8 of the result, but five products feed them and the tensor cores cut every addition off (CAFE_TILES_CHUNK's comment has
// the figures).
#define CAFE_LIN_LOW 16
// fp32 for splitting: every NaN with its upper bits set (an upper part that is cut off must not become an infinity)
__device__ __forceinline__ float cafe_quiet(float x) { return x + 0.f; }

// ---- the end of a product --------------------------------------------------------------------------------------------
// A thread's N consecutive columns of a row of the block's sums to shared memory.
template <int N> __device__ __forceinline__ void cafe_sums_put(const float* acc, uint32_t at) {
#pragma unroll
    for (int c = 0; c < N; c += 4)
        cafe_put16(at + 4 * c, __float_as_uint(acc[c]), __float_as_uint(acc[c + 1]), __float_as_uint(acc[c + 2]), __float_as_uint(acc[c + 3]));
}
// Four neighbouring elements of the residual (row i, columns j ..), as they lie.
template <typename T> struct CafeQuad { alignas(4 * sizeof(T)) T v[4]; };
template <typename T>
__device__ __forceinline__ void cafe_quad_residual(const CafeJob& J, int64_t i, int64_t j, CafeQuad<T>& x) {
    const T* p = static_cast<const T*>(J.res) + i * J.ldr + j;
    const int n = (int)min((int64_t)4, J.cols - j);
    if (J.res_vec && n == 4) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(x.v) = __ldg(reinterpret_cast<const uint4*>(p));
        else *reinterpret_cast<uint2*>(x.v) = __ldg(reinterpret_cast<const uint2*>(p));
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) x.v[q] = q < n ? __ldg(p + q) : cafe_from_float<T>(0.f);
    }
}
// Four neighbouring outputs (row i, columns j ..): bias, activation, residual, rounding, stores.
template <typename T>
__device__ __forceinline__ void cafe_quad_end(const CafeJob& J, int64_t i, int64_t j, const float* v, const float* bias, const CafeQuad<T>& res) {
    typedef typename CafeSlopeOf<T>::type ST;
    const int n = (int)min((int64_t)4, J.cols - j);
    const bool vec = J.out_vec && n == 4;
    alignas(16) T o[4];
    alignas(16) ST sl[4];
    float z[4], d[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) z[q] = v[q] + bias[q];
    cafe_act_all<4>(z, J.act, d);
    if (J.res) {
#pragma unroll
        for (int q = 0; q < 4; ++q) z[q] += cafe_to_float(res.v[q]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = cafe_from_float<T>(z[q]);
    T* out = static_cast<T*>(J.out) + i * J.ldo + j;
    if (vec) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(o);
        else *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(o);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) if (q < n) out[q] = o[q];
    }
    if (J.slope_out) {
        cafe_slopes<4>(d, sl);
        ST* so = static_cast<ST*>(J.slope_out) + i * J.lds + j;
        if (vec) {
            if constexpr (sizeof(ST) == 4) *reinterpret_cast<uint4*>(so) = *reinterpret_cast<const uint4*>(sl);
            else *reinterpret_cast<uint2*>(so) = *reinterpret_cast<const uint2*>(sl);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) if (q < n) so[q] = sl[q];
        }
    }
}
template <typename T> __device__ __forceinline__ void cafe_quad_bias(const CafeJob& J, int64_t j, float* bias) {
#pragma unroll
    for (int q = 0; q < 4; ++q) bias[q] = J.bias && j + q < J.cols ? cafe_to_float(__ldg(static_cast<const T*>(J.bias) + j + q)) : 0.f;
}
// This block's share of the tile's rows (of a cluster of `splits` blocks, by rank): the blocks' sums in the order of ranks, then
// bias, activation, residual and the stores.  COLS columns at a pitch of COLS + 4 floats from `base` of every block.
template <typename T, int COLS, int SPLITS>
__device__ __forceinline__ void cafe_finish_of(const CafeJob& J, uint32_t base, int row0, int col0, int rank, int threads) {
    constexpr int pitch = COLS + 4, quads = COLS / 4;
    const int per = CAFE_LIN_BM / SPLITS;
    for (int e = threadIdx.x; e < per * quads; e += threads) {
        const int r = rank * per + e / quads, c = (e % quads) * 4;
        const int64_t i = row0 + r, j = col0 + c;
        if (i >= J.rows || j >= J.cols) continue;
        const uint32_t at = base + (uint32_t)(r * pitch + c) * 4u;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (SPLITS == 1) asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at) : "memory");
        else {
            float4 x[SPLITS];
#pragma unroll
            for (int q = 0; q < SPLITS; ++q) x[q] = cafe_cluster_load4(cafe_cluster_map(at, q));
#pragma unroll
            for (int q = 0; q < SPLITS; ++q) { v[0] += x[q].x; v[1] += x[q].y; v[2] += x[q].z; v[3] += x[q].w; }
        }
        float bias[4];
        cafe_quad_bias<T>(J, j, bias);
        CafeQuad<T> res;
        if (J.res) cafe_quad_residual<T>(J, i, j, res);
        cafe_quad_end<T>(J, i, j, v, bias, res);
    }
}
template <typename T, int COLS>
__device__ __forceinline__ void cafe_finish(const CafeJob& J, uint32_t base, int row0, int col0, int rank, int splits, int threads) {
    if (splits == 1) cafe_finish_of<T, COLS, 1>(J, base, row0, col0, rank, threads);
    else if (splits == 2) cafe_finish_of<T, COLS, 2>(J, base, row0, col0, rank, threads);
    else if (splits == 4) cafe_finish_of<T, COLS, 4>(J, base, row0, col0, rank, threads);
    else cafe_finish_of<T, COLS, 8>(J, base, row0, col0, rank, threads);
}

// a kernel's limit of shared memory, once per device (always the same value: threads that do it at the same time do no harm)
static inline cudaError_t dense_allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>* devices) {
    int d = 0;
    cudaError_t e = cudaGetDevice(&d);
    if (e != cudaSuccess || (d < 64 && (devices->load(std::memory_order_relaxed) >> d & 1))) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && d < 64) devices->fetch_or((uint64_t)1 << d, std::memory_order_relaxed);
    return e;
}

// A launch in clusters of `cluster` blocks.  EARLY: it may start while the kernel before it in the stream ends (its kernel waits:
// cafe_wait_for_earlier); for kernels of one block an SM.  Smaller blocks would crowd onto the SMs that are free first and leave
// others empty later (gW of 65536x1024x479 in 256 blocks: 476 or 669 us).
template <bool EARLY, typename... P, typename... A>
static inline cudaError_t dense_start(void (*kernel)(P...), dim3 grid, unsigned threads, int shared, int cluster, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (EARLY) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = (unsigned)cluster; at[n].val.clusterDim.y = 1; at[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    CAFE_PROF(CAFE_P_LINEAR, st);
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ---- the calls -------------------------------------------------------------------------------------------------------
struct CafeForward {
    const void *x, *w, *bias, *res;
    int64_t ldx, ldw, ldr;
    int M, N, K, act;
    void *y, *slope;
    int64_t ldy, lds;
};
struct CafeBackward {
    const void *gy, *slope, *x, *w;
    int64_t ldg, lds, ldx, ldw;
    int slope_kind, M, N, K;
    void *gx, *gw, *gb;
    int64_t ldgx, ldgw;
};
// dense_tiles.cu: large layers.  Bytes of workspace that a call would take (0: not one for it), and the calls.
int64_t cafe_tiles_forward_work(const CafeForward& f, int dtype);
int64_t cafe_tiles_backward_work(const CafeBackward& f, int dtype);
cudaError_t cafe_tiles_forward(const CafeForward& f, int dtype, const CafeJob& job, void* work, cudaStream_t st);
cudaError_t cafe_tiles_backward(const CafeBackward& f, int dtype, const CafeJob* gw, const CafeJob* gx, void* work, cudaStream_t st);
cudaError_t cafe_tiles_gave_up(int* flag);
