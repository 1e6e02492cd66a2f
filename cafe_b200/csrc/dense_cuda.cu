// dense_cuda.cu -- the layers of the MLPs around the embedding path (dlrm_s_pytorch.py:213-251, dcn.py:410-422):
//
//   z = x W^T + b      y = act(z) + r
//   gz = gy * act'(z)  gx = gz W   gW = gz^T x   gb = sum over rows of gz   gr = gy
//
// for x [M, K], W [N, K], rows of any pitch, in fp32, bf16 or fp16 with sums in fp32.
#include "dense.cuh"

// ---- one matrix product: C(i, j) = sum_k A(i, k) B(j, k) ---------------------------------------------------------------
// The three products of a layer differ only in which index of each operand is contiguous (y: k of both; gx: k of gz, j of W; gW:
// i of gz, j of x) and in what happens at the end, so one kernel takes them all, two at a time where a backward has two.
// A block makes 128 x BN outputs.  Eight warps load pieces of eight consecutive k (or, where i or j is contiguous, eight rows
// of k, lanes along i or j), multiply A by the slope where there is one, and store them to shared memory in the order the
// tensor cores read; one thread issues the products; eight warps take the sums out of tensor memory.  The pieces of the next
// turn are in registers before this turn's are stored.  Blocks of a cluster share the depth of one tile (1 to 8 of them: short
// of tiles, long in k) and add their sums through each other's shared memory, in the order of their ranks: no atomics, no
// memory of its own, the same bits on every run.
//
// fp32.  An operand is cut into three bf16 parts, h + m + l = x exactly (each the next 8 bits of the mantissa, cut off, not
// rounded: nothing overflows), and six of the nine products are added: hh, and hm + mh + mm + hl + lh in sums of their own.
// What is left out is below 2^-23 of a product.  The tensor cores cut sums off instead of rounding them, so hh, whose sums
// are as large as the result, is taken out and added in registers every CHUNK of k; the others are 2^-8 of it and are not.
#define CAFE_LIN_THREADS 512       // 8 warps that load, 8 that take sums out, the first of which issues the products

template <typename T> struct CafeLin {   // 16-bit types
    static constexpr int parts = 1, BK = 64, chunk = 64, type = 0;   // chunk: turns of BK between two times that sums are taken out
};
template <> struct CafeLin<__nv_bfloat16> { static constexpr int parts = 1, BK = 64, chunk = 64, type = 1; };
template <> struct CafeLin<float> { static constexpr int parts = 3, BK = 32, chunk = 8, type = 1; };
template <typename T, int BN> struct CafeLinShape {
    static constexpr int rowb = CafeLin<T>::BK * 2;
    static constexpr int a_part = CAFE_LIN_BM * rowb, b_part = BN * rowb, stage = CafeLin<T>::parts * (a_part + b_part);
    static constexpr int tile = CAFE_LIN_BM * (BN + 4) * 4;
    static constexpr int stages = 196608 / stage < 6 ? 196608 / stage : 6;
    static constexpr int bytes = (stage * stages > tile ? stage * stages : tile) + 1024;
    static constexpr int tm_cols = CafeLin<T>::parts == 3 ? 2 * BN : BN;
};

__device__ int g_dense_gave_up;   // a wait ran out (its outputs are not numbers)

// eight values along k of one row: fp32, or 16-bit values two to a register
template <typename T> struct CafePiece { uint32_t v[4]; };
template <> struct CafePiece<float> { float v[8]; };

template <typename T> __device__ __forceinline__ void cafe_piece_set(CafePiece<T>& p, int j, T x) {
    if constexpr (sizeof(T) == 4) p.v[j] = x;
    else {
        const uint32_t b = (uint32_t)reinterpret_cast<const uint16_t&>(x);
        if (j & 1) p.v[j >> 1] |= b << 16; else p.v[j >> 1] = b;
    }
}
template <typename T> __device__ __forceinline__ T cafe_piece_get(const CafePiece<T>& p, int j) {
    if constexpr (sizeof(T) == 4) return p.v[j];
    else {
        const uint16_t b = (uint16_t)(p.v[j >> 1] >> (j & 1 ? 16 : 0));
        return reinterpret_cast<const T&>(b);
    }
}
// elements (row, k .. k + 8) of an operand; nothing outside [0, rows) x [., kend) is read
template <typename T>
__device__ __forceinline__ void cafe_piece_load(CafePiece<T>& p, const void* base, int64_t ld, int kc, int vec, int row, int rows, int k, int kend) {
    const T* b = static_cast<const T*>(base);
    if (kc) {
        const T* src = b + (int64_t)row * ld + k;
        if (row < rows && vec && k + 8 <= kend) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(src));
            if constexpr (sizeof(T) == 4) {
                const uint4 y = __ldg(reinterpret_cast<const uint4*>(src) + 1);
                p.v[0] = __uint_as_float(x.x); p.v[1] = __uint_as_float(x.y); p.v[2] = __uint_as_float(x.z); p.v[3] = __uint_as_float(x.w);
                p.v[4] = __uint_as_float(y.x); p.v[5] = __uint_as_float(y.y); p.v[6] = __uint_as_float(y.z); p.v[7] = __uint_as_float(y.w);
            } else { p.v[0] = x.x; p.v[1] = x.y; p.v[2] = x.z; p.v[3] = x.w; }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) cafe_piece_set<T>(p, j, row < rows && k + j < kend ? __ldg(src + j) : cafe_from_float<T>(0.f));
        }
    } else {
        const T* src = b + (int64_t)k * ld + row;
#pragma unroll
        for (int j = 0; j < 8; ++j) cafe_piece_set<T>(p, j, row < rows && k + j < kend ? __ldg(src + (int64_t)j * ld) : cafe_from_float<T>(0.f));
    }
}
template <typename T, typename S>
__device__ __forceinline__ void cafe_piece_slope(CafePiece<T>& p, const CafePiece<S>& s) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float x = cafe_to_float(cafe_piece_get<T>(p, 2 * j)) * cafe_to_float(cafe_piece_get<S>(s, 2 * j));
        const float y = cafe_to_float(cafe_piece_get<T>(p, 2 * j + 1)) * cafe_to_float(cafe_piece_get<S>(s, 2 * j + 1));
        cafe_piece_set<T>(p, 2 * j, cafe_from_float<T>(x));
        cafe_piece_set<T>(p, 2 * j + 1, cafe_from_float<T>(y));
    }
}
template <typename T>
__device__ __forceinline__ void cafe_piece_mask(CafePiece<T>& p, const CafePiece<T>& y) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const T a = cafe_piece_get<T>(p, 2 * j), b = cafe_piece_get<T>(p, 2 * j + 1);
        cafe_piece_set<T>(p, 2 * j, cafe_to_float(cafe_piece_get<T>(y, 2 * j)) > 0.f ? a : cafe_from_float<T>(0.f));
        cafe_piece_set<T>(p, 2 * j + 1, cafe_to_float(cafe_piece_get<T>(y, 2 * j + 1)) > 0.f ? b : cafe_from_float<T>(0.f));
    }
}
// a piece to its place in the operand's part(s), `part` bytes apart
__device__ __forceinline__ void cafe_piece_store(const CafePiece<float>& p, uint32_t at, int part) {
    uint32_t h[4], m[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float x = p.v[2 * j], y = p.v[2 * j + 1];
        h[j] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
        const float xm = x - __uint_as_float(__float_as_uint(x) & 0xffff0000u), ym = y - __uint_as_float(__float_as_uint(y) & 0xffff0000u);
        m[j] = __byte_perm(__float_as_uint(xm), __float_as_uint(ym), 0x7632);
        const float xl = xm - __uint_as_float(__float_as_uint(xm) & 0xffff0000u), yl = ym - __uint_as_float(__float_as_uint(ym) & 0xffff0000u);
        l[j] = __byte_perm(__float_as_uint(xl), __float_as_uint(yl), 0x7632);
    }
    cafe_put16(at, h[0], h[1], h[2], h[3]);
    cafe_put16(at + part, m[0], m[1], m[2], m[3]);
    cafe_put16(at + 2 * part, l[0], l[1], l[2], l[3]);
}
template <typename T> __device__ __forceinline__ void cafe_piece_store(const CafePiece<T>& p, uint32_t at, int) { cafe_put16(at, p.v[0], p.v[1], p.v[2], p.v[3]); }

// One turn's pieces of this thread: `R` rows of an operand, BK deep, over 256 threads.  Piece number u: with k contiguous the
// pieces of a row follow one another (neighbouring lanes read on in the row), else the rows do.
template <typename T, int R, int BK = CafeLin<T>::BK> struct CafeTurn {
    static constexpr int per_row = BK / 8, total = R * per_row, each = (total + 255) / 256;
    CafePiece<T> p[each];
    __device__ __forceinline__ static int row_of(int u, int kc) { return kc ? u / per_row : u % R; }
    __device__ __forceinline__ static int piece_of(int u, int kc) { return kc ? u % per_row : u / R; }
    __device__ __forceinline__ void load(const void* base, int64_t ld, int kc, int vec, int row0, int rows, int k0, int kend, int tid) {
#pragma unroll
        for (int i = 0; i < each; ++i) {
            const int u = tid + i * 256;
            if (total % 256 == 0 || u < total) cafe_piece_load<T>(p[i], base, ld, kc, vec, row0 + row_of(u, kc), rows, k0 + 8 * piece_of(u, kc), kend);
        }
    }
    __device__ __forceinline__ void store(uint32_t at, int part, int kc, int tid) const {
#pragma unroll
        for (int i = 0; i < each; ++i) {
            const int u = tid + i * 256;
            if (total % 256 == 0 || u < total)
                cafe_piece_store(p[i], at + cafe_swizzle<BK * 2>(row_of(u, kc), piece_of(u, kc)), part);
        }
    }
};

template <typename T, int BN>
__global__ void __launch_bounds__(CAFE_LIN_THREADS, 1) k_linear(const __grid_constant__ CafeJobs P, int splits) {
    typedef CafeLin<T> L;
    typedef CafeLinShape<T, BN> Sh;
    typedef typename CafeSlopeOf<T>::type ST;
    extern __shared__ char sh_raw[];
    __shared__ __align__(8) uint64_t bars[2 * Sh::stages + 3];
    __shared__ uint32_t tm_at;
    __shared__ volatile int bail;
    __shared__ float bias_sum[2][CAFE_LIN_BM];
    const uint32_t base = (cafe_smem(sh_raw) + 1023u) & ~1023u;
    const uint32_t bar0 = cafe_smem(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (Sh::stages + s); };
    const uint32_t acc_full = bar0 + 8u * (2 * Sh::stages), acc_empty = acc_full + 8, all_done = acc_full + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    int tile = blockIdx.x / splits;
    const int rank = blockIdx.x - tile * splits;
    const int which = tile >= P.job[0].tiles;
    if (which) tile -= P.job[0].tiles;
    const CafeJob& J = P.job[which];
    const int tm = tile / J.tiles_n, tn = tile - tm * J.tiles_n, row0 = tm * CAFE_LIN_BM, col0 = tn * BN;
    const int turns_all = (J.depth + L::BK - 1) / L::BK, share = (turns_all + splits - 1) / splits;
    const int t0 = min(rank * share, turns_all), turns = min(share, turns_all - t0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < Sh::stages; ++s) { cafe_bar_init(full(s), 8); cafe_bar_init(empty(s), 1); }
        cafe_bar_init(acc_full, 1);
        cafe_bar_init(acc_empty, 8);
        cafe_bar_init(all_done, 1);
        cafe_fence_barrier_init();
        bail = 0;
    }
    if (warp == 8) cafe_tm_alloc(cafe_smem(&tm_at), Sh::tm_cols);
    cafe_tc_before();
    __syncthreads();
    cafe_tc_after();
    const uint32_t tmem = tm_at;

    constexpr int half_cols = BN / 2;
    float acc[half_cols];
    if (warp < 8) {
        // ---- operands into shared memory
        const int tid = threadIdx.x;
        const bool sums = J.gb && tn == 0;
        CafeTurn<T, CAFE_LIN_BM> a[2];
        CafeTurn<ST, CAFE_LIN_BM, L::BK> sl;
        CafeTurn<T, CAFE_LIN_BM> ym;
        CafeTurn<T, BN> b[2];
        float bsum = 0.f, bchunk = 0.f;
        auto load = [&](int t, int h) {
            const int k0 = (t0 + t) * L::BK;
            a[h].load(J.a, J.lda, J.a_kc, J.a_vec, row0, J.rows, k0, J.depth, tid);
            b[h].load(J.b, J.ldb, J.b_kc, J.b_vec, col0, J.cols, k0, J.depth, tid);
        };
        if (turns > 0) load(0, 0);
#pragma unroll 2
        for (int t = 0; t < turns; ++t) {
            const int h = t & 1, s = t % Sh::stages;
            const int k0 = (t0 + t) * L::BK;
            if (J.slope_kind == CAFE_SLOPE_VALUES) sl.load(J.as, J.ldas, J.a_kc, J.as_vec, row0, J.rows, k0, J.depth, tid);
            else if (J.slope_kind == CAFE_SLOPE_OUTPUT) ym.load(J.as, J.ldas, J.a_kc, J.as_vec, row0, J.rows, k0, J.depth, tid);
            if (t + 1 < turns) load(t + 1, h ^ 1);
            if (J.slope_kind == CAFE_SLOPE_VALUES) {
                if (sums) {   // (the sum takes gz before its rounding)
                    float x = 0.f;
#pragma unroll
                    for (int i = 0; i < CafeTurn<T, CAFE_LIN_BM>::each; ++i)
#pragma unroll
                        for (int j = 0; j < 8; ++j) x += cafe_to_float(cafe_piece_get<T>(a[h].p[i], j)) * cafe_to_float(cafe_piece_get<ST>(sl.p[i], j));
                    bchunk += x;
                }
#pragma unroll
                for (int i = 0; i < CafeTurn<T, CAFE_LIN_BM>::each; ++i) cafe_piece_slope<T, ST>(a[h].p[i], sl.p[i]);
            } else {
                if (J.slope_kind == CAFE_SLOPE_OUTPUT) {
#pragma unroll
                    for (int i = 0; i < CafeTurn<T, CAFE_LIN_BM>::each; ++i) cafe_piece_mask<T>(a[h].p[i], ym.p[i]);
                }
                if (sums) {
                    float x = 0.f;
#pragma unroll
                    for (int i = 0; i < CafeTurn<T, CAFE_LIN_BM>::each; ++i)
#pragma unroll
                        for (int j = 0; j < 8; ++j) x += cafe_to_float(cafe_piece_get<T>(a[h].p[i], j));
                    bchunk += x;
                }
            }
            if ((t & 31) == 31) { bsum += bchunk; bchunk = 0.f; }
            if (t >= Sh::stages && !cafe_bar_wait(empty(s), (uint32_t)(t / Sh::stages - 1) & 1u, &bail)) break;
            const uint32_t at = base + s * Sh::stage;
            a[h].store(at, Sh::a_part, J.a_kc, tid);
            b[h].store(at + L::parts * Sh::a_part, Sh::b_part, J.b_kc, tid);
            cafe_fence_async();
            __syncwarp();
            if (lane == 0) cafe_bar_arrive(full(s));
        }
        if (sums) bias_sum[tid >> 7][tid & 127] = bsum + bchunk;   // (rows contiguous: a thread's pieces are all of row tid & 127)
    } else {
        // ---- products, and sums out of tensor memory: warps 8 to 11 the left half of the columns, 12 to 15 the right, 32 rows each
        const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)((warp - 8) / 4 * half_cols);
        auto take = [&](uint32_t at, bool first) {
#pragma unroll
            for (int c = 0; c < half_cols; c += 16) {
                float v[16];
                cafe_tm_load16(at + c, v);
                cafe_tm_wait_load();
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c + i] = first ? v[i] : acc[c + i] + v[i];
            }
        };
        constexpr uint32_t instr = cafe_mma_instr(L::type, CAFE_LIN_BM, BN);
        const int chunks = (turns + L::chunk - 1) / L::chunk;
        bool fine = true;
        for (int c = 0; c < chunks && fine; ++c) {
            if (warp == 8) {
                if (lane == 0) {
                    const int end = min(turns, (c + 1) * L::chunk);
                    if (c > 0) fine = cafe_bar_wait(acc_empty, (uint32_t)(c - 1) & 1u, &bail);
                    for (int t = c * L::chunk; t < end && fine; ++t) {
                        const int s = t % Sh::stages;
                        if (!(fine = cafe_bar_wait(full(s), (uint32_t)(t / Sh::stages) & 1u, &bail))) break;
                        cafe_tc_after();
                        const uint32_t a = base + s * Sh::stage, b = a + L::parts * Sh::a_part;
#pragma unroll
                        for (int k = 0; k < L::BK / 16; ++k)
                            cafe_mma(tmem, cafe_operand<Sh::rowb>(a + 32 * k), cafe_operand<Sh::rowb>(b + 32 * k), instr, t > c * L::chunk || k > 0);
                        if (t == end - 1) cafe_mma_commit(acc_full);
                        if constexpr (L::parts == 3) {
#pragma unroll
                            for (int q = 0; q < 5; ++q) {
                                constexpr int ia[5] = {0, 1, 1, 0, 2}, ib[5] = {1, 0, 1, 2, 0};
#pragma unroll
                                for (int k = 0; k < L::BK / 16; ++k)
                                    cafe_mma(tmem + BN, cafe_operand<Sh::rowb>(a + ia[q] * Sh::a_part + 32 * k),
                                             cafe_operand<Sh::rowb>(b + ib[q] * Sh::b_part + 32 * k), instr, t > 0 || q > 0 || k > 0);
                            }
                        }
                        cafe_mma_commit(empty(s));
                    }
                    if (!fine || c == chunks - 1) cafe_mma_commit(all_done);
                }
                fine = __shfl_sync(0xffffffffu, (int)fine, 0);
            }
            if (fine) fine = cafe_bar_wait(acc_full, (uint32_t)c & 1u, &bail);
            cafe_tc_after();
            __syncwarp();
            if (__all_sync(0xffffffffu, fine)) take(from, c == 0); else fine = false;
            cafe_tc_before();
            __syncwarp();
            if (lane == 0) cafe_bar_arrive(acc_empty);
        }
        if (turns > 0) {
            // (also: nothing is still reading the operands, even where a wait has run out)
            fine = cafe_bar_wait(all_done, 0, &bail) && fine;
            cafe_tc_after();
            fine = __all_sync(0xffffffffu, fine);
            if (L::parts == 3 && fine) take(from + BN, false);
        } else {
#pragma unroll
            for (int i = 0; i < half_cols; ++i) acc[i] = 0.f;
        }
        if (!fine) {
            g_dense_gave_up = 1;
#pragma unroll
            for (int i = 0; i < half_cols; ++i) acc[i] = __uint_as_float(0x7fffffffu);
        }
        cafe_tc_before();
    }
    __syncthreads();
    cafe_tc_after();
    if (warp == 8) cafe_tm_free(tmem, Sh::tm_cols);

    // ---- the block's sums to shared memory, and what belongs at the end
    if (warp >= 8) {
        const int r = (warp & 3) * 32 + lane, c0 = (warp - 8) / 4 * half_cols;
        cafe_sums_put<L::parts == 3, half_cols>(J, acc, base + (uint32_t)(r * (BN + 4) + c0) * 4u, row0 + r, col0 + c0, t0 * L::BK,
                                                min(J.depth, (t0 + turns) * L::BK), !bail);
    }
    if (splits > 1) cafe_cluster_sync(); else __syncthreads();
    cafe_finish<T, BN>(J, base, row0, col0, rank, splits, CAFE_LIN_THREADS);
    if (J.gb && tn == 0 && rank == 0 && threadIdx.x < CAFE_LIN_BM && row0 + (int)threadIdx.x < J.rows) {
        float x = 0.f;
        for (int q = 0; q < splits; ++q) {
            const uint32_t at = cafe_smem(&bias_sum[0][threadIdx.x]), to = splits > 1 ? cafe_cluster_map(at, q) : cafe_cluster_map(at, cafe_cluster_rank());
            x += cafe_cluster_load(to) + cafe_cluster_load(to + 4 * CAFE_LIN_BM);
        }
        static_cast<T*>(J.gb)[row0 + threadIdx.x] = cafe_from_float<T>(x);
    }
    if (splits > 1) cafe_cluster_sync();   // (others may still read this block's sums)
}

static bool dense_on(const void* p, int64_t ld, int size, int bytes) { return ((uintptr_t)p % bytes) == 0 && (ld * size) % bytes == 0; }

template <typename T, int BN>
static cudaError_t dense_launch_bn(CafeJobs& P, int splits, cudaStream_t st) {
    int tiles = 0;
    for (int q = 0; q < P.count; ++q) {
        CafeJob& J = P.job[q];
        J.tiles_n = J.cols > 0 ? (J.cols + BN - 1) / BN : 1;   // (no columns: a bias gradient alone)
        J.tiles = ((J.rows + CAFE_LIN_BM - 1) / CAFE_LIN_BM) * J.tiles_n;
        tiles += J.tiles;
    }
    if (tiles == 0) return cudaSuccess;
    constexpr int bytes = CafeLinShape<T, BN>::bytes;
    cudaError_t e = cudaFuncSetAttribute(k_linear<T, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * splits));
    cfg.blockDim = dim3(CAFE_LIN_THREADS);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)splits; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CAFE_PROF(CAFE_P_LINEAR, st);
    return cudaLaunchKernelEx(&cfg, k_linear<T, BN>, (const CafeJobs&)P, splits);
}

// Width of the tiles and blocks per tile: the pair whose estimate is least.  A turn (BK of depth) of a 128, 64 and 32 wide tile
// takes about 1, 0.65 and 0.5 units, a block costs 6 units beside its turns and 1 more where sums are exchanged; blocks run
// 148 at a time, so the whole takes the longest block or all blocks' sum / 148, whichever is more.
template <typename T>
static cudaError_t dense_launch(CafeJobs& P, cudaStream_t st) {
    static const int widths[3] = {128, 64, 32};
    static const double unit[3] = {1.0, 0.65, 0.5};
    int best_n = 0, best_s = 1;
    double best = 1e300;
    for (int n = 0; n < 3; ++n)
        for (int s = 1; s <= 8; s *= 2) {
            double longest = 0, sum = 0;
            int64_t blocks = 0;
            for (int q = 0; q < P.count; ++q) {
                const CafeJob& J = P.job[q];
                const int turns = (J.depth + CafeLin<T>::BK - 1) / CafeLin<T>::BK;
                const double one = (double)((turns + s - 1) / s) * unit[n] + 6 + (s > 1 ? 1 : 0);
                const double tiles = (double)((J.rows + CAFE_LIN_BM - 1) / CAFE_LIN_BM) * (J.cols > 0 ? (J.cols + widths[n] - 1) / widths[n] : 1);
                longest = one > longest ? one : longest;
                sum += one * tiles * s;
                blocks += (int64_t)tiles * s;
            }
            const double est = sum / 148 > longest ? sum / 148 : longest;
            if (est < best * 0.999 && blocks < (1 << 30)) { best = est; best_n = n; best_s = s; }
        }
    if (best_n == 0) return dense_launch_bn<T, 128>(P, best_s, st);
    if (best_n == 1) return dense_launch_bn<T, 64>(P, best_s, st);
    return dense_launch_bn<T, 32>(P, best_s, st);
}

static int dense_done(cudaError_t e) {
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) { cafe_internal_set_error(cudaGetErrorString(e)); return CAFE_ERR_CUDA; }
    return CAFE_OK;
}

template <typename T>
static cudaError_t dense_forward(const CafeForward& f, int dtype, void* work, int64_t work_bytes, cudaStream_t st) {
    if (f.M == 0 || f.N == 0) return cudaSuccess;
    CafeJobs P = {};
    CafeJob& J = P.job[0];
    P.count = 1;
    const int size = sizeof(T);
    J.a = f.x; J.lda = f.ldx; J.a_kc = 1; J.a_vec = dense_on(f.x, f.ldx, size, 16);
    J.b = f.w; J.ldb = f.ldw; J.b_kc = 1; J.b_vec = dense_on(f.w, f.ldw, size, 16);
    J.rows = f.M; J.cols = f.N; J.depth = f.K;
    J.bias = f.bias; J.res = f.res; J.ldr = f.ldr; J.act = f.act; J.out = f.y; J.ldo = f.ldy; J.slope_out = f.slope; J.lds = f.lds;
    const int ssize = sizeof(typename CafeSlopeOf<T>::type);
    J.res_vec = f.res && dense_on(f.res, f.ldr, size, 4 * size);
    J.out_vec = dense_on(f.y, f.ldy, size, 4 * size) && (!f.slope || dense_on(f.slope, f.lds, ssize, 4 * ssize));
    const int64_t need = cafe_tiles_forward_work(f, dtype);
    if (need > 0 && work && work_bytes >= need) return cafe_tiles_forward(f, dtype, J, work, st);
    return dense_launch<T>(P, st);
}
template <typename T>
static cudaError_t dense_backward(const CafeBackward& f, int dtype, void* work, int64_t work_bytes, cudaStream_t st) {
    CafeJobs P = {};
    const int size = sizeof(T), ssize = f.slope_kind == CAFE_SLOPE_VALUES ? (int)sizeof(typename CafeSlopeOf<T>::type) : size;
    const int g_vec = dense_on(f.gy, f.ldg, size, 16), s_vec = f.slope_kind != CAFE_SLOPE_NONE && dense_on(f.slope, f.lds, ssize, 16);
    if ((f.gw && f.K > 0) || (f.gb && f.N > 0)) {
        // (without gW wanted, one column of tiles of nothing makes the bias gradient)
        CafeJob& J = P.job[P.count++];
        J.a = f.gy; J.lda = f.ldg; J.a_vec = g_vec; J.as = f.slope; J.ldas = f.lds; J.as_vec = s_vec; J.slope_kind = f.slope_kind;
        J.b = f.x; J.ldb = f.ldx;
        J.rows = f.N; J.cols = f.gw ? f.K : 0; J.depth = f.M;
        J.out = f.gw; J.ldo = f.ldgw; J.out_vec = dense_on(f.gw, f.ldgw, size, 4 * size); J.gb = f.gb;
    }
    if (f.gx && f.M > 0 && f.K > 0) {
        CafeJob& J = P.job[P.count++];
        J.a = f.gy; J.lda = f.ldg; J.a_kc = 1; J.a_vec = g_vec; J.as = f.slope; J.ldas = f.lds; J.as_vec = s_vec; J.slope_kind = f.slope_kind;
        J.b = f.w; J.ldb = f.ldw;
        J.rows = f.M; J.cols = f.K; J.depth = f.N;
        J.out = f.gx; J.ldo = f.ldgx; J.out_vec = dense_on(f.gx, f.ldgx, size, 4 * size);
    }
    const int64_t need = cafe_tiles_backward_work(f, dtype);
    if (need > 0 && work && work_bytes >= need)
        return cafe_tiles_backward(f, dtype, f.gw || f.gb ? &P.job[0] : nullptr, f.gx ? &P.job[P.count - 1] : nullptr, work, st);
    return P.count ? dense_launch<T>(P, st) : cudaSuccess;
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

// (work that is there must be on 16 bytes)
static int dense_work_ok(const void* work, int64_t bytes) { return !work || (bytes >= 0 && ((uintptr_t)work & 15) == 0); }
static int64_t dense_half(int layers, const int* widths, int M, int dtype) {
    int64_t most = 0;
    for (int l = 1; l < layers; ++l) most = widths[l] > most ? widths[l] : most;
    return (((most + 7) & ~(int64_t)7) * M * (dtype == CAFE_F32 ? 4 : 2) + 255) & ~(int64_t)255;
}
// what lies between the layers of an MLP is on 16 bytes, rows and all
static const void* const k_aligned = (const void*)256;

extern "C" {

int64_t cafe_linear_forward_work(const void* x_dev, int64_t ldx, const void* w_dev, int64_t ldw, int M, int N, int K, int dtype) {
    CafeForward f = {};
    f.x = x_dev; f.ldx = ldx; f.w = w_dev; f.ldw = ldw; f.M = M; f.N = N; f.K = K;
    return dense_type_ok(dtype) && dense_sizes_ok(M, N, K) ? cafe_tiles_forward_work(f, dtype) : 0;
}

int cafe_linear_forward(const void* x_dev, int64_t ldx, const void* w_dev, int64_t ldw, const void* bias_dev, const void* res_dev, int64_t ldr,
                        int M, int N, int K, int dtype, int act, void* y_dev, int64_t ldy, void* slope_dev, int64_t lds, void* work_dev,
                        int64_t work_bytes, void* stream) {
    const CafeForward f = {x_dev, w_dev, bias_dev, res_dev, ldx, ldw, ldr, M, N, K, act, y_dev, slope_dev, ldy, lds};
    if (!dense_type_ok(dtype) || !dense_forward_ok(f) || !dense_work_ok(work_dev, work_bytes)) return CAFE_ERR_ARG;
    cudaError_t e;
    DENSE_TYPED(dtype, e = dense_forward<T>(f, dtype, work_dev, work_bytes, (cudaStream_t)stream));
    return dense_done(e);
}

int64_t cafe_linear_backward_work(const void* gy_dev, int64_t ldg, int slope_kind, const void* x_dev, int64_t ldx, const void* w_dev, int64_t ldw,
                                  int M, int N, int K, int dtype, int want_gx, int want_gw, int want_gb) {
    CafeBackward f = {};
    f.gy = gy_dev; f.ldg = ldg; f.slope_kind = slope_kind; f.x = x_dev; f.ldx = ldx; f.w = w_dev; f.ldw = ldw; f.M = M; f.N = N; f.K = K;
    f.gx = want_gx ? (void*)k_aligned : nullptr; f.gw = want_gw ? (void*)k_aligned : nullptr; f.gb = want_gb ? (void*)k_aligned : nullptr;
    return dense_type_ok(dtype) && dense_sizes_ok(M, N, K) ? cafe_tiles_backward_work(f, dtype) : 0;
}

int cafe_linear_backward(const void* gy_dev, int64_t ldg, const void* slope_dev, int64_t lds, int slope_kind, const void* x_dev, int64_t ldx,
                         const void* w_dev, int64_t ldw, int M, int N, int K, int dtype, void* gx_dev, int64_t ldgx, void* gw_dev, int64_t ldgw,
                         void* gb_dev, void* work_dev, int64_t work_bytes, void* stream) {
    const CafeBackward f = {gy_dev, slope_dev, x_dev, w_dev, ldg, lds, ldx, ldw, slope_kind, M, N, K, gx_dev, gw_dev, gb_dev, ldgx, ldgw};
    if (!dense_type_ok(dtype) || !dense_backward_ok(f) || !dense_work_ok(work_dev, work_bytes)) return CAFE_ERR_ARG;
    cudaError_t e;
    DENSE_TYPED(dtype, e = dense_backward<T>(f, dtype, work_dev, work_bytes, (cudaStream_t)stream));
    return dense_done(e);
}

int64_t cafe_mlp_forward_work(int layers, const int* widths, int M, const void* x_dev, int64_t ldx, const void* const* w_dev, const int64_t* ldw, int dtype) {
    if (layers < 1 || layers > CAFE_MLP_MAX_LAYERS || !widths || !w_dev || !ldw) return 0;
    int64_t most = 0;
    for (int l = 0; l < layers; ++l) {
        const int64_t need = cafe_linear_forward_work(l ? k_aligned : x_dev, l ? (widths[l] + 7) & ~7 : ldx, w_dev[l], ldw[l], M, widths[l + 1], widths[l], dtype);
        most = need > most ? need : most;
    }
    return most;
}

int cafe_mlp_forward(int layers, const int* widths, int M, const void* x_dev, int64_t ldx, const void* const* w_dev, const int64_t* ldw,
                     const void* const* bias_dev, const int* acts, int dtype, void* const* y_dev, const int64_t* ldy, void* const* slope_dev,
                     void* work_dev, int64_t work_bytes, void* stream) {
    if (!dense_type_ok(dtype) || layers < 1 || layers > CAFE_MLP_MAX_LAYERS || !widths || !w_dev || !ldw || !bias_dev || !acts || !y_dev || !ldy) return CAFE_ERR_ARG;
    if (!dense_work_ok(work_dev, work_bytes)) return CAFE_ERR_ARG;
    CafeForward f[CAFE_MLP_MAX_LAYERS];
    for (int l = 0; l < layers; ++l) {
        f[l] = {l ? y_dev[l - 1] : x_dev, w_dev[l], bias_dev[l], nullptr, l ? ldy[l - 1] : ldx, ldw[l], 0, M, widths[l + 1], widths[l], acts[l],
                y_dev[l], slope_dev ? slope_dev[l] : nullptr, ldy[l], ldy[l]};
        if (!dense_forward_ok(f[l])) return CAFE_ERR_ARG;
    }
    cudaError_t e = cudaSuccess;
    for (int l = 0; l < layers && e == cudaSuccess; ++l) DENSE_TYPED(dtype, e = dense_forward<T>(f[l], dtype, work_dev, work_bytes, (cudaStream_t)stream));
    return dense_done(e);
}

int64_t cafe_mlp_backward_work(int layers, const int* widths, int M, const void* gy_dev, int64_t ldg, const void* x_dev, int64_t ldx,
                               const void* const* w_dev, const int64_t* ldw, int dtype) {
    if (!dense_type_ok(dtype) || layers < 1 || layers > CAFE_MLP_MAX_LAYERS || !widths || !w_dev || !ldw || M < 0 || M > CAFE_LINEAR_MAX) return 0;
    int64_t most = 0;
    for (int l = 0; l < layers; ++l) {
        const int64_t ldn = (widths[l + 1] + 7) & ~7, ldk = (widths[l] + 7) & ~7;
        const int64_t need = cafe_linear_backward_work(l == layers - 1 ? gy_dev : k_aligned, l == layers - 1 ? ldg : ldn, CAFE_SLOPE_VALUES,
                                                       l ? k_aligned : x_dev, l ? ldk : ldx, w_dev[l], ldw[l], M, widths[l + 1], widths[l], dtype, 1, 1, 1);
        most = need > most ? need : most;
    }
    return 2 * dense_half(layers, widths, M, dtype) + most;
}

int cafe_mlp_backward(int layers, const int* widths, int M, const void* gy_dev, int64_t ldg, const void* x_dev, int64_t ldx,
                      const void* const* w_dev, const int64_t* ldw, const int* acts, int dtype, const void* const* y_dev, const int64_t* ldy,
                      const void* const* slope_dev, void* gx_dev, int64_t ldgx, void* const* gw_dev, void* const* gb_dev, void* work_dev,
                      int64_t work_bytes, void* stream) {
    if (!dense_type_ok(dtype) || layers < 1 || layers > CAFE_MLP_MAX_LAYERS || !widths || !w_dev || !ldw || !acts || !y_dev || !ldy || !gw_dev || !gb_dev) return CAFE_ERR_ARG;
    if (M < 0 || M > CAFE_LINEAR_MAX) return CAFE_ERR_ARG;
    for (int l = 0; l <= layers; ++l) if (widths[l] < 0 || widths[l] > CAFE_LINEAR_MAX) return CAFE_ERR_ARG;
    const int64_t half_bytes = dense_half(layers, widths, M, dtype);
    if (half_bytes > 0 && (!work_dev || work_bytes < 2 * half_bytes)) return CAFE_ERR_ARG;
    if (!dense_work_ok(work_dev, work_bytes)) return CAFE_ERR_ARG;
    char* const half[2] = {(char*)work_dev, (char*)work_dev + half_bytes};
    CafeBackward f[CAFE_MLP_MAX_LAYERS];
    for (int l = layers - 1; l >= 0; --l) {
        const bool last = l == layers - 1;
        const int kind = acts[l] == CAFE_ACT_NONE ? CAFE_SLOPE_NONE : slope_dev && slope_dev[l] ? CAFE_SLOPE_VALUES : CAFE_SLOPE_OUTPUT;
        if (kind == CAFE_SLOPE_OUTPUT && acts[l] != CAFE_ACT_RELU) return CAFE_ERR_ARG;
        const int64_t ldn = (widths[l + 1] + 7) & ~7, ldk = (widths[l] + 7) & ~7;
        f[l] = {last ? gy_dev : half[l & 1], kind == CAFE_SLOPE_VALUES ? slope_dev[l] : y_dev[l], l ? y_dev[l - 1] : x_dev, w_dev[l],
                last ? ldg : ldn, ldy[l], l ? ldy[l - 1] : ldx, ldw[l], kind, M, widths[l + 1], widths[l],
                l ? half[(l - 1) & 1] : gx_dev, gw_dev[l], gb_dev[l], l ? ldk : ldgx, widths[l]};
        if (!dense_backward_ok(f[l])) return CAFE_ERR_ARG;
    }
    cudaError_t e = cudaSuccess;
    for (int l = layers - 1; l >= 0 && e == cudaSuccess; --l)
        DENSE_TYPED(dtype, e = dense_backward<T>(f[l], dtype, half[1] + half_bytes, work_bytes - 2 * half_bytes, (cudaStream_t)stream));
    return dense_done(e);
}

}  // extern "C"
