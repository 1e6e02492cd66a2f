// dense_cuda.cu -- the layers of the MLPs around the embedding path (dlrm_s_pytorch.py:213-251, dcn.py:410-422):
//
//   z = x W^T + b      y = act(z) + r
//   gz = gy * act'(z)  gx = gz W   gW = gz^T x   gb = sum over rows of gz   gr = gy
//
// for x [M, K], W [N, K], rows of any pitch, in fp32, bf16 or fp16 with sums in fp32.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/cafe_b200.h"
#include "cafe_internal.h"
#include "cafe_float.cuh"

// act(z), and its derivative
__device__ __forceinline__ float cafe_act(float z, int act, float* slope) {
    switch (act) {
        case CAFE_ACT_RELU: *slope = z > 0.f ? 1.f : 0.f; return z > 0.f ? z : (z != z ? z : 0.f);
        case CAFE_ACT_SIGMOID: case CAFE_ACT_SILU: {
            // e = exp(-|z|) never overflows; s and t = 1 - s keep their relative precision in both tails
            const float e = expf(-fabsf(z)), d = 1.f / (1.f + e);
            const float s = z >= 0.f ? d : e * d, t = z >= 0.f ? e * d : d;
            if (act == CAFE_ACT_SIGMOID) { *slope = s * t; return s; }
            *slope = s * (1.f + z * t);
            return z * s;
        }
        case CAFE_ACT_GELU: {
            const float c = 0.5f * erfcf(z * -0.70710678118654752f);
            *slope = c + z * expf(-0.5f * z * z) * 0.39894228040143268f;
            return z * c;
        }
        default: *slope = 1.f; return z;
    }
}

// the derivative kept for the backward: fp32 beside fp32, else fp16 (11 bits where bf16 would leave 8; it lies in [-0.2, 1.2])
template <typename T> struct CafeSlopeOf { typedef __half type; };
template <> struct CafeSlopeOf<float> { typedef float type; };

// C(i, j) = sum_k A(i, k) B(j, k); A may be multiplied by a slope of the same indices
struct CafeProduct {
    const void *a, *b, *slope;
    int64_t a_i, a_k, s_i, s_k, b_j, b_k;
    int slope_kind, rows, cols, depth;
    const void *bias, *res;
    int64_t ldr;
    int act;
    void *out, *slope_out;
    int64_t ldo, lds;
};
template <typename T>
__device__ __forceinline__ float cafe_sloped(const void* a, int64_t at, const void* slope, int64_t st, int kind) {
    const float v = cafe_to_float(static_cast<const T*>(a)[at]);
    if (kind == CAFE_SLOPE_VALUES) return v * cafe_to_float(static_cast<const typename CafeSlopeOf<T>::type*>(slope)[st]);
    if (kind == CAFE_SLOPE_OUTPUT) return cafe_to_float(static_cast<const T*>(slope)[st]) > 0.f ? v : 0.f;
    return v;
}

// a block makes 64 x 64 outputs, a thread 4 x 4 of them
#define CAFE_LIN_TILE 64
#define CAFE_LIN_DEPTH 16
template <typename T>
__global__ void __launch_bounds__(256) k_linear(const CafeProduct P) {
    __shared__ float A[CAFE_LIN_DEPTH][CAFE_LIN_TILE + 1], B[CAFE_LIN_DEPTH][CAFE_LIN_TILE + 1];
    const int64_t i0 = (int64_t)blockIdx.x * CAFE_LIN_TILE, j0 = (int64_t)blockIdx.y * CAFE_LIN_TILE;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < P.depth; k0 += CAFE_LIN_DEPTH) {
        for (int e = threadIdx.x; e < CAFE_LIN_TILE * CAFE_LIN_DEPTH; e += 256) {
            const int ka = P.a_k == 1 ? e % CAFE_LIN_DEPTH : e / CAFE_LIN_TILE, i = P.a_k == 1 ? e / CAFE_LIN_DEPTH : e % CAFE_LIN_TILE;
            const int64_t gi = i0 + i, gk = k0 + ka;
            A[ka][i] = gi < P.rows && gk < P.depth
                           ? cafe_sloped<T>(P.a, gi * P.a_i + gk * P.a_k, P.slope, gi * P.s_i + gk * P.s_k, P.slope_kind) : 0.f;
            const int kb = P.b_k == 1 ? e % CAFE_LIN_DEPTH : e / CAFE_LIN_TILE, j = P.b_k == 1 ? e / CAFE_LIN_DEPTH : e % CAFE_LIN_TILE;
            const int64_t gj = j0 + j, hk = k0 + kb;
            B[kb][j] = gj < P.cols && hk < P.depth ? cafe_to_float(static_cast<const T*>(P.b)[gj * P.b_j + hk * P.b_k]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < CAFE_LIN_DEPTH; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += A[k][ty + 16 * i] * B[k][tx + 16 * j];
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t gi = i0 + ty + 16 * i, gj = j0 + tx + 16 * j;
            if (gi >= P.rows || gj >= P.cols) continue;
            float z = acc[i][j], s;
            if (P.bias) z += cafe_to_float(static_cast<const T*>(P.bias)[gj]);
            z = cafe_act(z, P.act, &s);
            if (P.res) z += cafe_to_float(static_cast<const T*>(P.res)[gi * P.ldr + gj]);
            static_cast<T*>(P.out)[gi * P.ldo + gj] = cafe_from_float<T>(z);
            if (P.slope_out) static_cast<typename CafeSlopeOf<T>::type*>(P.slope_out)[gi * P.lds + gj] = cafe_from_float<typename CafeSlopeOf<T>::type>(s);
        }
}
template <typename T>
__global__ void __launch_bounds__(256) k_linear_bias_grad(const void* gy, int64_t ldg, const void* slope, int64_t lds, int kind, int M, int N, void* gb) {
    __shared__ float part[8][32];
    const int64_t n = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    float s = 0.f;
    if (n < N)
        for (int64_t m = threadIdx.x >> 5; m < M; m += 8) s += cafe_sloped<T>(gy, m * ldg + n, slope, m * lds + n, kind);
    part[threadIdx.x >> 5][threadIdx.x & 31] = s;
    __syncthreads();
    if (threadIdx.x < 32 && n < N) {
        for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
        static_cast<T*>(gb)[n] = cafe_from_float<T>(s);
    }
}

static int dense_done() {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) { cafe_internal_set_error(cudaGetErrorString(e)); return CAFE_ERR_CUDA; }
    return CAFE_OK;
}
template <typename T>
static void dense_product(const CafeProduct& P, cudaStream_t st) {
    if (P.rows == 0 || P.cols == 0) return;
    CAFE_PROF(CAFE_P_LINEAR, st);
    k_linear<T><<<dim3((unsigned)((P.rows + 63) / 64), (unsigned)((P.cols + 63) / 64)), 256, 0, st>>>(P);
}

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
template <typename T>
static void dense_forward(const CafeForward& f, cudaStream_t st) {
    CafeProduct P = {};
    P.a = f.x; P.a_i = f.ldx; P.a_k = 1; P.b = f.w; P.b_j = f.ldw; P.b_k = 1;
    P.rows = f.M; P.cols = f.N; P.depth = f.K;
    P.bias = f.bias; P.res = f.res; P.ldr = f.ldr; P.act = f.act; P.out = f.y; P.ldo = f.ldy; P.slope_out = f.slope; P.lds = f.lds;
    dense_product<T>(P, st);
}
template <typename T>
static void dense_backward(const CafeBackward& f, cudaStream_t st) {
    CafeProduct P = {};
    P.slope_kind = f.slope_kind; P.slope = f.slope; P.a = f.gy;
    if (f.gx) {
        P.a_i = f.ldg; P.a_k = 1; P.s_i = f.lds; P.s_k = 1; P.b = f.w; P.b_j = 1; P.b_k = f.ldw;
        P.rows = f.M; P.cols = f.K; P.depth = f.N; P.out = f.gx; P.ldo = f.ldgx;
        dense_product<T>(P, st);
    }
    if (f.gw) {
        P.a_i = 1; P.a_k = f.ldg; P.s_i = 1; P.s_k = f.lds; P.b = f.x; P.b_j = 1; P.b_k = f.ldx;
        P.rows = f.N; P.cols = f.K; P.depth = f.M; P.out = f.gw; P.ldo = f.ldgw;
        dense_product<T>(P, st);
    }
    if (f.gb && f.N > 0) {
        CAFE_PROF(CAFE_P_LINEAR, st);
        k_linear_bias_grad<T><<<(unsigned)((f.N + 31) / 32), 256, 0, st>>>(f.gy, f.ldg, f.slope, f.lds, f.slope_kind, f.M, f.N, f.gb);
    }
}
#define DENSE_TYPED(dtype, ...)                                              \
    do {                                                                     \
        if ((dtype) == CAFE_F32) { typedef float T; __VA_ARGS__; }           \
        else if ((dtype) == CAFE_BF16) { typedef __nv_bfloat16 T; __VA_ARGS__; } \
        else { typedef __half T; __VA_ARGS__; }                              \
    } while (0)

static int dense_type_ok(int dtype) { return dtype == CAFE_F32 || dtype == CAFE_BF16 || dtype == CAFE_F16; }
// (a row pitch below the row's length is right for one row only, or for a row that is read again for every row: pitch 0)
static int dense_rows_ok(const void* p, int64_t ld, int rows, int cols) { return rows == 0 || cols == 0 || (p && (rows == 1 || ld >= cols)); }
static int dense_sizes_ok(int M, int N, int K) { return M >= 0 && N >= 0 && K >= 0 && M <= CAFE_LINEAR_MAX && N <= CAFE_LINEAR_MAX && K <= CAFE_LINEAR_MAX; }

static int dense_forward_ok(const CafeForward& f) {
    if (!dense_sizes_ok(f.M, f.N, f.K) || f.act < CAFE_ACT_NONE || f.act > CAFE_ACT_SILU) return 0;
    if (f.N > 0 && f.M > 0 && (!dense_rows_ok(f.x, f.ldx, f.M, f.K) || !dense_rows_ok(f.w, f.ldw, f.N, f.K))) return 0;
    if (!dense_rows_ok(f.y, f.ldy, f.M, f.N) || (f.slope && !dense_rows_ok(f.slope, f.lds, f.M, f.N))) return 0;
    return !f.res || f.ldr == 0 || dense_rows_ok(f.res, f.ldr, f.M, f.N);
}
static int dense_backward_ok(const CafeBackward& f) {
    if (!dense_sizes_ok(f.M, f.N, f.K) || f.slope_kind < CAFE_SLOPE_NONE || f.slope_kind > CAFE_SLOPE_OUTPUT) return 0;
    if (!(f.ldg == 0 && f.gy) && !dense_rows_ok(f.gy, f.ldg, f.M, f.N)) return 0;
    if (f.slope_kind != CAFE_SLOPE_NONE && !dense_rows_ok(f.slope, f.lds, f.M, f.N)) return 0;
    if (f.gx && (!dense_rows_ok(f.gx, f.ldgx, f.M, f.K) || (f.M > 0 && !dense_rows_ok(f.w, f.ldw, f.N, f.K)))) return 0;
    if (f.gw && (!dense_rows_ok(f.gw, f.ldgw, f.N, f.K) || (f.N > 0 && !dense_rows_ok(f.x, f.ldx, f.M, f.K)))) return 0;
    return 1;
}

extern "C" {

int cafe_linear_forward(const void* x_dev, int64_t ldx, const void* w_dev, int64_t ldw, const void* bias_dev, const void* res_dev, int64_t ldr,
                        int M, int N, int K, int dtype, int act, void* y_dev, int64_t ldy, void* slope_dev, int64_t lds, void* stream) {
    const CafeForward f = {x_dev, w_dev, bias_dev, res_dev, ldx, ldw, ldr, M, N, K, act, y_dev, slope_dev, ldy, lds};
    if (!dense_type_ok(dtype) || !dense_forward_ok(f)) return CAFE_ERR_ARG;
    DENSE_TYPED(dtype, dense_forward<T>(f, (cudaStream_t)stream));
    return dense_done();
}

int cafe_linear_backward(const void* gy_dev, int64_t ldg, const void* slope_dev, int64_t lds, int slope_kind, const void* x_dev, int64_t ldx,
                         const void* w_dev, int64_t ldw, int M, int N, int K, int dtype, void* gx_dev, int64_t ldgx, void* gw_dev, int64_t ldgw,
                         void* gb_dev, void* stream) {
    const CafeBackward f = {gy_dev, slope_dev, x_dev, w_dev, ldg, lds, ldx, ldw, slope_kind, M, N, K, gx_dev, gw_dev, gb_dev, ldgx, ldgw};
    if (!dense_type_ok(dtype) || !dense_backward_ok(f)) return CAFE_ERR_ARG;
    DENSE_TYPED(dtype, dense_backward<T>(f, (cudaStream_t)stream));
    return dense_done();
}

int cafe_mlp_forward(int layers, const int* widths, int M, const void* x_dev, int64_t ldx, const void* const* w_dev, const int64_t* ldw,
                     const void* const* bias_dev, const int* acts, int dtype, void* const* y_dev, const int64_t* ldy, void* const* slope_dev,
                     void* stream) {
    if (!dense_type_ok(dtype) || layers < 1 || layers > CAFE_MLP_MAX_LAYERS || !widths || !w_dev || !ldw || !bias_dev || !acts || !y_dev || !ldy) return CAFE_ERR_ARG;
    CafeForward f[CAFE_MLP_MAX_LAYERS];
    for (int l = 0; l < layers; ++l) {
        f[l] = {l ? y_dev[l - 1] : x_dev, w_dev[l], bias_dev[l], nullptr, l ? ldy[l - 1] : ldx, ldw[l], 0, M, widths[l + 1], widths[l], acts[l],
                y_dev[l], slope_dev ? slope_dev[l] : nullptr, ldy[l], ldy[l]};
        if (!dense_forward_ok(f[l])) return CAFE_ERR_ARG;
    }
    for (int l = 0; l < layers; ++l) DENSE_TYPED(dtype, dense_forward<T>(f[l], (cudaStream_t)stream));
    return dense_done();
}

int64_t cafe_mlp_backward_work(int layers, const int* widths, int M, int dtype) {
    int64_t most = 0;
    for (int l = 1; l < layers; ++l) most = widths[l] > most ? widths[l] : most;
    return 2 * ((((most + 7) & ~(int64_t)7) * M * (dtype == CAFE_F32 ? 4 : 2) + 255) & ~(int64_t)255);
}

int cafe_mlp_backward(int layers, const int* widths, int M, const void* gy_dev, int64_t ldg, const void* x_dev, int64_t ldx,
                      const void* const* w_dev, const int64_t* ldw, const int* acts, int dtype, const void* const* y_dev, const int64_t* ldy,
                      const void* const* slope_dev, void* gx_dev, int64_t ldgx, void* const* gw_dev, void* const* gb_dev, void* work_dev,
                      int64_t work_bytes, void* stream) {
    if (!dense_type_ok(dtype) || layers < 1 || layers > CAFE_MLP_MAX_LAYERS || !widths || !w_dev || !ldw || !acts || !y_dev || !ldy || !gw_dev || !gb_dev) return CAFE_ERR_ARG;
    const int64_t need = cafe_mlp_backward_work(layers, widths, M, dtype);
    if (need > 0 && (!work_dev || work_bytes < need || ((uintptr_t)work_dev & 15))) return CAFE_ERR_ARG;
    CafeBackward f[CAFE_MLP_MAX_LAYERS];
    for (int l = layers - 1; l >= 0; --l) {
        const bool last = l == layers - 1;
        const int kind = acts[l] == CAFE_ACT_NONE ? CAFE_SLOPE_NONE : slope_dev && slope_dev[l] ? CAFE_SLOPE_VALUES : CAFE_SLOPE_OUTPUT;
        if (kind == CAFE_SLOPE_OUTPUT && acts[l] != CAFE_ACT_RELU) return CAFE_ERR_ARG;
        char* const half[2] = {(char*)work_dev, (char*)work_dev + need / 2};
        const int64_t ldn = (widths[l + 1] + 7) & ~7, ldk = (widths[l] + 7) & ~7;
        f[l] = {last ? gy_dev : half[l & 1], kind == CAFE_SLOPE_VALUES ? slope_dev[l] : y_dev[l], l ? y_dev[l - 1] : x_dev, w_dev[l],
                last ? ldg : ldn, ldy[l], l ? ldy[l - 1] : ldx, ldw[l], kind, M, widths[l + 1], widths[l],
                l ? half[(l - 1) & 1] : gx_dev, gw_dev[l], gb_dev[l], l ? ldk : ldgx, widths[l]};
        if (!dense_backward_ok(f[l])) return CAFE_ERR_ARG;
    }
    for (int l = layers - 1; l >= 0; --l) DENSE_TYPED(dtype, dense_backward<T>(f[l], (cudaStream_t)stream));
    return dense_done();
}

}  // extern "C"
