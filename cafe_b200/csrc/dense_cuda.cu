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

__device__ int g_dense_gave_up;   // 1: a wait of k_linear ran out (its outputs are not numbers)

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
// Eight elements along k from `src`, the first of them, KC: contiguous, else `ld` apart.  FULL: all eight are inside; otherwise
// `left` of them, and nothing else is read.
template <typename T, bool KC, bool FULL>
__device__ __forceinline__ void cafe_piece_load(CafePiece<T>& p, const T* src, int64_t ld, bool vec, int left) {
    if (KC && FULL && vec) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(src));
        if constexpr (sizeof(T) == 4) {
            const uint4 y = __ldg(reinterpret_cast<const uint4*>(src) + 1);
            p.v[0] = __uint_as_float(x.x); p.v[1] = __uint_as_float(x.y); p.v[2] = __uint_as_float(x.z); p.v[3] = __uint_as_float(x.w);
            p.v[4] = __uint_as_float(y.x); p.v[5] = __uint_as_float(y.y); p.v[6] = __uint_as_float(y.z); p.v[7] = __uint_as_float(y.w);
        } else { p.v[0] = x.x; p.v[1] = x.y; p.v[2] = x.z; p.v[3] = x.w; }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) cafe_piece_set<T>(p, j, FULL || j < left ? cafe_ldg(src + (KC ? (int64_t)j : j * ld)) : cafe_from_float<T>(0.f));
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
        const float x = cafe_quiet(p.v[2 * j]), y = cafe_quiet(p.v[2 * j + 1]);
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

// One turn's pieces of this thread: `R` rows of an operand, BK deep, over 256 threads.  With k contiguous the pieces of a row
// follow one another (neighbouring lanes read on in the row), else the rows do.  Rows past the last one read the last one again:
// what comes of them is not stored.
template <typename T, int R, int BK, bool KC> struct CafeTurn {
    static constexpr int per_row = BK / 8, total = R * per_row, each = (total + 255) / 256;
    CafePiece<T> p[each];
    __device__ __forceinline__ static int row_of(int u) { return KC ? u / per_row : u % R; }
    __device__ __forceinline__ static int piece_of(int u) { return KC ? u % per_row : u / R; }
    __device__ __forceinline__ static bool has(int u) { return total % 256 == 0 || u < total; }
    // base: element (row0, 0); last: rows there are from row0, less one
    template <bool FULL> __device__ __forceinline__ void load(const T* base, int64_t ld, bool vec, int last, int k0, int kend, int tid) {
#pragma unroll
        for (int i = 0; i < each; ++i) {
            const int u = tid + i * 256, k = k0 + 8 * piece_of(u), r = min(row_of(u), last);
            if (has(u)) cafe_piece_load<T, KC, FULL>(p[i], base + (KC ? r * ld + k : k * ld + r), ld, vec, kend - k);
        }
    }
    __device__ __forceinline__ void store(uint32_t at, int part, int tid) const {
#pragma unroll
        for (int i = 0; i < each; ++i) {
            const int u = tid + i * 256;
            if (has(u)) cafe_piece_store(p[i], at + cafe_swizzle<BK * 2>(row_of(u), piece_of(u)), part);
        }
    }
    __device__ __forceinline__ float sum() const {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < each; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) x += cafe_to_float(cafe_piece_get<T>(p[i], j));
        return x;
    }
};

// The loading warps' part of a block: AK and BK_: k contiguous in A and B; KIND: what A is multiplied by.
template <typename T, int BN, bool AK, bool BK_, int KIND>
__device__ __forceinline__ void cafe_produce(const CafeJob& J, uint32_t base, uint32_t full0, uint32_t empty0, volatile int* bail, int row0, int col0, int t0, int turns,
                                             float* bias_sum) {
    typedef CafeLin<T> L;
    typedef CafeLinShape<T, BN> Sh;
    typedef typename CafeSlopeOf<T>::type ST;
    const int tid = threadIdx.x, lane = tid & 31;
    const T* A = static_cast<const T*>(J.a) + (AK ? row0 * J.lda : (int64_t)row0);
    const T* B = static_cast<const T*>(J.b) + (BK_ ? col0 * J.ldb : (int64_t)col0);
    const int64_t s0 = AK ? row0 * J.ldas : (int64_t)row0;
    const int a_last = J.rows - 1 - row0, b_last = max(0, J.cols - 1 - col0);
    CafeTurn<T, CAFE_LIN_BM, L::BK, AK> a[2];
    CafeTurn<T, BN, L::BK, BK_> b[2];
    CafeTurn<ST, CAFE_LIN_BM, L::BK, AK> sl;
    CafeTurn<T, CAFE_LIN_BM, L::BK, AK> ym;
    float bsum = 0.f, bchunk = 0.f;
    const bool columns = J.cols > 0;
    auto load = [&](int t, int h) {
        const int k0 = (t0 + t) * L::BK;
        if (k0 + L::BK <= J.depth) {
            a[h].template load<true>(A, J.lda, J.a_vec, a_last, k0, J.depth, tid);
            if (columns) b[h].template load<true>(B, J.ldb, J.b_vec, b_last, k0, J.depth, tid);
        } else {
            a[h].template load<false>(A, J.lda, false, a_last, k0, J.depth, tid);
            if (columns) b[h].template load<false>(B, J.ldb, false, b_last, k0, J.depth, tid);
        }
    };
    auto load_slope = [&](int t) {
        const int k0 = (t0 + t) * L::BK;
        if constexpr (KIND == CAFE_SLOPE_VALUES) {
            if (k0 + L::BK <= J.depth) sl.template load<true>(static_cast<const ST*>(J.as) + s0, J.ldas, J.as_vec, a_last, k0, J.depth, tid);
            else sl.template load<false>(static_cast<const ST*>(J.as) + s0, J.ldas, false, a_last, k0, J.depth, tid);
        } else if constexpr (KIND == CAFE_SLOPE_OUTPUT) {
            if (k0 + L::BK <= J.depth) ym.template load<true>(static_cast<const T*>(J.as) + s0, J.ldas, J.as_vec, a_last, k0, J.depth, tid);
            else ym.template load<false>(static_cast<const T*>(J.as) + s0, J.ldas, false, a_last, k0, J.depth, tid);
        }
    };
    load(0, 0);
    load_slope(0);
#pragma unroll 2
    for (int t = 0; t < turns; ++t) {
        const int h = t & 1, s = t % Sh::stages;
        if (t + 1 < turns) load(t + 1, h ^ 1);
        if constexpr (KIND == CAFE_SLOPE_VALUES) {
            if (bias_sum) {   // (the sum takes gz before its rounding)
                float x = 0.f;
#pragma unroll
                for (int i = 0; i < a[h].each; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) x += cafe_to_float(cafe_piece_get<T>(a[h].p[i], j)) * cafe_to_float(cafe_piece_get<ST>(sl.p[i], j));
                bchunk += x;
            }
#pragma unroll
            for (int i = 0; i < a[h].each; ++i) cafe_piece_slope<T, ST>(a[h].p[i], sl.p[i]);
        } else {
            if constexpr (KIND == CAFE_SLOPE_OUTPUT) {
#pragma unroll
                for (int i = 0; i < a[h].each; ++i) cafe_piece_mask<T>(a[h].p[i], ym.p[i]);
            }
            if (bias_sum) bchunk += a[h].sum();
        }
        if (t + 1 < turns) load_slope(t + 1);
        if ((t & 31) == 31) { bsum += bchunk; bchunk = 0.f; }
        if (t >= Sh::stages && !cafe_bar_wait(empty0 + 8u * s, (uint32_t)(t / Sh::stages - 1) & 1u, bail)) break;
        const uint32_t at = base + s * Sh::stage;
        a[h].store(at, Sh::a_part, tid);
        if (columns) b[h].store(at + L::parts * Sh::a_part, Sh::b_part, tid);
        cafe_fence_async();
        __syncwarp();
        if (lane == 0) cafe_bar_arrive(full0 + 8u * s);
    }
    if (bias_sum) bias_sum[tid] = bsum + bchunk;   // (rows contiguous: a thread's pieces are all of row tid & 127)
}

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
    cafe_next_may_start();
    if (warp == 8) cafe_tm_alloc(cafe_smem(&tm_at), Sh::tm_cols);
    cafe_tc_before();
    __syncthreads();
    cafe_tc_after();
    cafe_wait_for_earlier();
    const uint32_t tmem = tm_at;

    constexpr int half_cols = BN / 2;
    float acc[half_cols];
    if (warp < 8) {
        // ---- operands into shared memory
        float* const sums = J.gb && tn == 0 ? &bias_sum[0][0] : nullptr;
#define PRODUCE(AK, BK_, KIND) cafe_produce<T, BN, AK, BK_, KIND>(J, base, full(0), empty(0), &bail, row0, col0, t0, turns, sums)
        if (turns == 0) { if (sums) sums[threadIdx.x] = 0.f; }
        else if (J.b_kc) PRODUCE(true, true, CAFE_SLOPE_NONE);
        else if (J.a_kc) {
            if (J.slope_kind == CAFE_SLOPE_VALUES) PRODUCE(true, false, CAFE_SLOPE_VALUES);
            else if (J.slope_kind == CAFE_SLOPE_OUTPUT) PRODUCE(true, false, CAFE_SLOPE_OUTPUT);
            else PRODUCE(true, false, CAFE_SLOPE_NONE);
        } else {
            if (J.slope_kind == CAFE_SLOPE_VALUES) PRODUCE(false, false, CAFE_SLOPE_VALUES);
            else if (J.slope_kind == CAFE_SLOPE_OUTPUT) PRODUCE(false, false, CAFE_SLOPE_OUTPUT);
            else PRODUCE(false, false, CAFE_SLOPE_NONE);
        }
#undef PRODUCE
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
        auto join = [&]() {   // fp32: the other sums
#pragma unroll
            for (int c = 0; c < half_cols; c += 16) {
                float v[16];
                cafe_tm_load16(from + BN + c, v);
                cafe_tm_wait_load();
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c + i] = cafe_join_sums(acc[c + i], v[i]);
            }
        };
        constexpr uint32_t instr = cafe_mma_instr(L::type, CAFE_LIN_BM, BN);
        const int chunks = (turns + L::chunk - 1) / L::chunk;
        bool fine = true;
        for (int c = 0; c < chunks && fine; ++c) {
            if (warp == 8) {
                const int end = min(turns, (c + 1) * L::chunk);
                const bool low = L::parts == 3 && (c + 1) % CAFE_LIN_LOW == 0 && c < chunks - 1;
                if (c > 0) fine = __all_sync(0xffffffffu, cafe_bar_wait(acc_empty, (uint32_t)(c - 1) & 1u, &bail));
                for (int t = c * L::chunk; t < end && fine; ++t) {
                    const int s = t % Sh::stages;
                    if (!(fine = __all_sync(0xffffffffu, cafe_bar_wait(full(s), (uint32_t)(t / Sh::stages) & 1u, &bail)))) break;
                    cafe_tc_after();
                    const uint32_t a = base + s * Sh::stage, b = a + L::parts * Sh::a_part;
                    if (cafe_elect()) {
#pragma unroll
                        for (int k = 0; k < L::BK / 16; ++k)
                            cafe_mma(tmem, cafe_operand<Sh::rowb>(a + 32 * k), cafe_operand<Sh::rowb>(b + 32 * k), instr, t > c * L::chunk || k > 0);
                        if (t == end - 1 && !low) cafe_mma_commit(acc_full);
                        if constexpr (L::parts == 3) {
#pragma unroll
                            for (int q = 0; q < 5; ++q) {
                                constexpr int ia[5] = {0, 1, 1, 0, 2}, ib[5] = {1, 0, 1, 2, 0};
#pragma unroll
                                for (int k = 0; k < L::BK / 16; ++k)
                                    cafe_mma(tmem + BN, cafe_operand<Sh::rowb>(a + ia[q] * Sh::a_part + 32 * k),
                                             cafe_operand<Sh::rowb>(b + ib[q] * Sh::b_part + 32 * k), instr, t % (L::chunk * CAFE_LIN_LOW) > 0 || q > 0 || k > 0);
                            }
                            if (t == end - 1 && low) cafe_mma_commit(acc_full);
                        }
                        cafe_mma_commit(empty(s));
                    }
                    __syncwarp();
                }
                if ((!fine || c == chunks - 1) && cafe_elect()) cafe_mma_commit(all_done);
                __syncwarp();
            }
            if (fine) fine = cafe_bar_wait(acc_full, (uint32_t)c & 1u, &bail);
            cafe_tc_after();
            __syncwarp();
            fine = __all_sync(0xffffffffu, fine);
            if (fine) take(from, c == 0);
            if (L::parts == 3 && fine && (c + 1) % CAFE_LIN_LOW == 0 && c < chunks - 1) join();
            cafe_tc_before();
            __syncwarp();
            if (lane == 0) cafe_bar_arrive(acc_empty);
        }
        if (turns > 0) {
            // (also: nothing is still reading the operands, even where a wait has run out)
            fine = cafe_bar_wait(all_done, 0, &bail) && fine;
            cafe_tc_after();
            fine = __all_sync(0xffffffffu, fine);
            if (L::parts == 3 && fine) join();
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
        cafe_sums_put<half_cols>(acc, base + (uint32_t)(r * (BN + 4) + c0) * 4u);
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
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = dense_allow_shared((const void*)k_linear<T, BN>, bytes, &allowed);
    if (e != cudaSuccess) return e;
    return dense_start<true>(k_linear<T, BN>, dim3((unsigned)(tiles * splits)), CAFE_LIN_THREADS, bytes, splits, st, P, splits);
}

// Width of the tiles and blocks per tile: the pair whose estimate is least.  A turn (BK of depth) of a 64 and a 32 wide tile takes
// about 1 and 0.75 units, a block costs 9 units beside its turns and 1 to 2 more where sums are exchanged; 148, 148,
// 132 and 120 blocks run at a time in clusters of 1, 2, 4 and 8 (what the device says), so the whole takes the longest block or,
// with more blocks than that, all blocks' sum over them.
template <typename T>
static cudaError_t dense_launch(CafeJobs& P, cudaStream_t st) {
    static const int widths[2] = {64, 32}, room[4] = {148, 148, 132, 120};
    static const double unit[2] = {1.0, 0.75}, exchange[4] = {0, 1.5, 2, 3};
    int best_n = 0, best_s = 0;
    double best = 1e300;
    for (int n = 0; n < 2; ++n)
        for (int s = 0; s < 4; ++s) {
            double longest = 0, sum = 0;
            int64_t blocks = 0;
            for (int q = 0; q < P.count; ++q) {
                const CafeJob& J = P.job[q];
                const int turns = (J.depth + CafeLin<T>::BK - 1) / CafeLin<T>::BK;
                const double one = (double)((turns + (1 << s) - 1) >> s) * unit[n] + 9 + exchange[s];
                const int64_t tiles = (int64_t)((J.rows + CAFE_LIN_BM - 1) / CAFE_LIN_BM) * (J.cols > 0 ? (J.cols + widths[n] - 1) / widths[n] : 1);
                longest = one > longest ? one : longest;
                sum += one * (double)(tiles << s);
                blocks += tiles << s;
            }
            const double all = sum / room[s], est = blocks > room[s] && all + 0.5 * longest > longest ? all + 0.5 * longest : longest;
            if (est < best * 0.999 && blocks < (1 << 30)) { best = est; best_n = n; best_s = s; }
        }
    return best_n == 0 ? dense_launch_bn<T, 64>(P, 1 << best_s, st) : dense_launch_bn<T, 32>(P, 1 << best_s, st);
}

static int dense_done(cudaError_t e) {
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) { cafe_internal_set_error(cudaGetErrorString(e)); return CAFE_ERR_CUDA; }
    return CAFE_OK;
}

// ---- a few rows against many -------------------------------------------------------------------------------------------
// y for at most 16 rows of x (one request to score), or of W (a last layer of one output): each of the many rows is read once, or
// twice where there are more than eight few, in plain fp32 multiply-adds; tiles of 128 would mostly be padding.  A block takes eight
// of the many rows at a time for every warp that has a share of k of its own: `kw` warps divide k among them, the others take
// further rows.  A lane has four k of eight many and FEW few rows at a time, so 8 + FEW loads feed 32 FEW multiply-adds; sums of a
// warp's lanes are halved and exchanged until each lane holds FEW / 4 of them (FEW >= 4), sums of the kw warps are added in their
// order through shared memory.  Bound by latency (a chain of launch, loads, exchange) until the many rows are a few MB, then by
// their bytes: 1024x1024 1 row 2.9 us, 8 rows 5.2, 16 rows 6.1 (sixteen few at a time, one block an SM: 7.5); 4096x4096, in L2, 11 us
// (6.1 TB/s), 25, 52 (73).
struct CafeFew {
    const void *few, *many, *bias, *res;
    int64_t ldf, ldm, ldr, ldo, lds;
    int nfew, nmany, depth, kw, vec, act, few_is_row;   // few_is_row: the few are rows of x, so the output is [few][many]
    void *out, *slope_out;
};
#define CAFE_FEW_MANY 8      // of the many rows at a time
#define CAFE_FEW_MOST 16
template <typename T> __device__ __forceinline__ void cafe_few_load(const T* p, bool vec, int lane, int left, float* v) {
    if (vec) {   // lane's four k: 4 lane + {0 .. 3}
        if (4 * lane + 4 <= left) {
            alignas(16) T x[4];
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(x) = __ldg(reinterpret_cast<const uint4*>(p + 4 * lane));
            else *reinterpret_cast<uint2*>(x) = __ldg(reinterpret_cast<const uint2*>(p + 4 * lane));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = cafe_to_float(x[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = 4 * lane + j < left ? cafe_to_float(__ldg(p + 4 * lane + j)) : 0.f;
        }
    } else {     // lane + {0, 32, 64, 96}
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = lane + 32 * j < left ? cafe_to_float(__ldg(p + lane + 32 * j)) : 0.f;
    }
}
template <typename T, int FEW>
__global__ void __launch_bounds__(256, FEW == 1 ? 3 : 2) k_few(const CafeFew P) {
    typedef typename CafeSlopeOf<T>::type ST;
    constexpr int N = CAFE_FEW_MANY * FEW;
    __shared__ float part[8][N];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int groups = 8 / P.kw, group = warp / P.kw, kpart = warp % P.kw;
    const int few0 = blockIdx.y * FEW, nfew = P.nfew - few0;   // (of this block; at least one)
    const int64_t per_block = (int64_t)groups * CAFE_FEW_MANY, first = blockIdx.x * per_block + group * CAFE_FEW_MANY;
    cafe_next_may_start();
    // k in steps of 128, shared out among kw warps
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    if (first < P.nmany) {
        const T* few = static_cast<const T*>(P.few) + few0 * P.ldf;
        const T* many = static_cast<const T*>(P.many) + first * P.ldm;
        const int last = (int)min((int64_t)CAFE_FEW_MANY, P.nmany - first) - 1;
        float w[CAFE_FEW_MANY][4];
        auto load_many = [&](int k) {
#pragma unroll
            for (int c = 0; c < CAFE_FEW_MANY; ++c) cafe_few_load(many + min(c, last) * P.ldm + k, P.vec, lane, P.depth - k, w[c]);
        };
        int k = kpart * 128;
        // (weights of a layer that follows one of its call were there before the call: they are fetched while that one ends)
        if (!P.few_is_row) cafe_wait_for_earlier();
        if (k < P.depth) load_many(k);
        if (P.few_is_row) cafe_wait_for_earlier();
        while (k < P.depth) {
            const int left = P.depth - k;
#pragma unroll
            for (int f = 0; f < FEW; ++f) {
                float x[4];
                cafe_few_load(few + min(f, nfew - 1) * P.ldf + k, P.vec, lane, left, x);
#pragma unroll
                for (int c = 0; c < CAFE_FEW_MANY; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[f * CAFE_FEW_MANY + c] += x[j] * w[c][j];
            }
            k += P.kw * 128;
            if (k < P.depth) load_many(k);
        }
    } else cafe_wait_for_earlier();
    // halving exchange: after it lane l holds, at acc[i], the whole sum number (l >> SH) * (N >> LG) + i
    constexpr int LG = N >= 32 ? 5 : N == 16 ? 4 : 3;   // halvings that leave something to halve
#pragma unroll
    for (int h = 0; h < LG; ++h) {
        const int half = N >> (h + 1), m = 16 >> h;
        const bool up = (lane & m) != 0;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if (i < half) {
                const float send = up ? acc[i] : acc[i + half], keep = up ? acc[i + half] : acc[i];
                acc[i] = keep + __shfl_xor_sync(0xffffffffu, send, m);
            }
        }
    }
#pragma unroll
    for (int h = LG; h < 5; ++h) acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], 16 >> h);
    if ((lane & ((32 >> LG) - 1)) == 0) {
#pragma unroll
        for (int i = 0; i < (N >> LG); ++i) part[warp][(lane >> (5 - LG)) * (N >> LG) + i] = acc[i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < groups * N; e += 256) {
        const int g = e / N, q = e % N;
        // neighbouring threads write neighbouring outputs
        const int f = P.few_is_row ? q / CAFE_FEW_MANY : q % FEW, c = P.few_is_row ? q % CAFE_FEW_MANY : q / FEW;
        const int64_t many = blockIdx.x * per_block + g * CAFE_FEW_MANY + c;
        if (f >= nfew || many >= P.nmany) continue;
        float z = 0.f;
        for (int w = 0; w < P.kw; ++w) z += part[g * P.kw + w][f * CAFE_FEW_MANY + c];
        const int64_t i = P.few_is_row ? few0 + f : many, j = P.few_is_row ? many : few0 + f;
        float d = 1.f;
        if (P.bias) z += cafe_to_float(__ldg(static_cast<const T*>(P.bias) + j));
        if (P.act != CAFE_ACT_NONE) z = cafe_act(z, P.act, &d);
        if (P.res) z += cafe_to_float(__ldg(static_cast<const T*>(P.res) + i * P.ldr + j));
        static_cast<T*>(P.out)[i * P.ldo + j] = cafe_from_float<T>(z);
        if (P.slope_out) static_cast<ST*>(P.slope_out)[i * P.lds + j] = cafe_from_float<ST>(d);
    }
}
template <typename T>
static cudaError_t dense_few(const CafeForward& f, bool follows, cudaStream_t st) {
    CafeFew P = {};
    P.few_is_row = f.M <= f.N;
    const bool r = P.few_is_row;
    P.few = r ? f.x : f.w; P.ldf = r ? f.ldx : f.ldw; P.nfew = r ? f.M : f.N;
    P.many = r ? f.w : f.x; P.ldm = r ? f.ldw : f.ldx; P.nmany = r ? f.N : f.M;
    P.depth = f.K; P.act = f.act; P.bias = f.bias; P.res = f.res; P.ldr = f.ldr;
    P.out = f.y; P.ldo = f.ldy; P.slope_out = f.slope; P.lds = f.lds;
    const int size = sizeof(T);
    P.vec = dense_on(f.x, f.ldx, size, 4 * size) && dense_on(f.w, f.ldw, size, 4 * size);
    // as many warps along k as have 128 of it, fewer where there are many rows to share out anyway
    P.kw = 1;
    while (P.kw < 8 && P.kw * 128 < f.K && (int64_t)P.nmany * P.kw < 148 * 16 * 8 * 8) P.kw *= 2;
    const int per_block = 8 / P.kw * CAFE_FEW_MANY;
    const unsigned grid = (unsigned)((P.nmany + per_block - 1) / per_block);
    auto start = [&](void (*kernel)(CafeFew), unsigned few) {
        const dim3 g(grid, (P.nfew + few - 1) / few);
        return follows ? dense_start<true>(kernel, g, 256, 0, 1, st, P) : dense_start<false>(kernel, g, 256, 0, 1, st, P);
    };
    return P.nfew <= 1 ? start(k_few<T, 1>, 1) : P.nfew <= 4 ? start(k_few<T, 4>, 4) : start(k_few<T, 8>, 8);
}

// The backward of a layer of at most 16 outputs: gx = gz W is a sum of few outer products, gW = gz^T x a few long sums, both bound
// by the bytes of x and gx, which are read and written once here, in plain fp32 multiply-adds (2048 x 256 -> 1: 36 us as tiles of 128
// that are padding, 8 and 5 by the two kernels here).  A block has 256 columns of k, a thread four of them and every other row of the block's rows; sums of
// blocks' rows go to `part` and k_few_join adds them in order.
struct CafeFewBack {
    const void *gy, *slope, *x, *w;
    int64_t ldg, lds, ldx, ldw, ldgx;
    int kind, M, N, K, rows, vec, vec_out;   // rows: of a block
    void* gx;
    float* part;                             // [row blocks][N][K + 1]: gW and, behind it, gb; or null
};
template <typename T, int FEW>
__global__ void __launch_bounds__(128) k_few_back(const CafeFewBack P) {
    typedef typename CafeSlopeOf<T>::type ST;
    __shared__ float half[FEW][64][4];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int k = blockIdx.x * 256 + tx * 4, n4 = min(4, P.K - k);
    const int m0 = blockIdx.y * P.rows, m1 = min(m0 + P.rows, P.M);
    cafe_next_may_start();
    float w[FEW][4], acc[FEW][4], gb[FEW];
#pragma unroll
    for (int n = 0; n < FEW; ++n) {
        gb[n] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[n][j] = 0.f;
            w[n][j] = P.gx && n < P.N && j < n4 ? cafe_to_float(__ldg(static_cast<const T*>(P.w) + n * P.ldw + k + j)) : 0.f;
        }
    }
#pragma unroll 4
    for (int64_t m = m0 + ty; m < m1; m += 2) {
        float g[FEW], x[4];
#pragma unroll
        for (int n = 0; n < FEW; ++n) {
            float v = n < P.N ? cafe_to_float(__ldg(static_cast<const T*>(P.gy) + m * P.ldg + n)) : 0.f;
            if (n < P.N && P.kind == CAFE_SLOPE_VALUES) v *= cafe_to_float(cafe_ldg(static_cast<const ST*>(P.slope) + m * P.lds + n));
            else if (n < P.N && P.kind == CAFE_SLOPE_OUTPUT) v = cafe_to_float(__ldg(static_cast<const T*>(P.slope) + m * P.lds + n)) > 0.f ? v : 0.f;
            g[n] = v;
            gb[n] += v;
        }
        if (P.part) {
            const T* p = static_cast<const T*>(P.x) + m * P.ldx + k;
            if (P.vec && n4 == 4) {
                alignas(16) T v[4];
                if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(p));
                else *reinterpret_cast<uint2*>(v) = __ldg(reinterpret_cast<const uint2*>(p));
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = cafe_to_float(v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = P.x && j < n4 ? cafe_to_float(__ldg(p + j)) : 0.f;
            }
#pragma unroll
            for (int n = 0; n < FEW; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[n][j] += g[n] * x[j];
        }
        if (P.gx && n4 > 0) {
            alignas(16) T o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float s = 0.f;
#pragma unroll
                for (int n = 0; n < FEW; ++n) s += g[n] * w[n][j];
                o[j] = cafe_from_float<T>(s);
            }
            T* to = static_cast<T*>(P.gx) + m * P.ldgx + k;
            if (P.vec_out && n4 == 4) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(o);
                else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(o);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) if (j < n4) to[j] = o[j];
            }
        }
    }
    if (!P.part) return;
    if (ty == 1) {
#pragma unroll
        for (int n = 0; n < FEW; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) half[n][tx][j] = acc[n][j];
    }
    __shared__ float half_gb[FEW];
    if (threadIdx.x == 64) {
#pragma unroll
        for (int n = 0; n < FEW; ++n) half_gb[n] = gb[n];
    }
    __syncthreads();
    if (ty == 0) {
#pragma unroll
        for (int n = 0; n < FEW; ++n) {
            if (n >= P.N) break;
            float* to = P.part + ((int64_t)blockIdx.y * P.N + n) * (P.K + 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) if (j < n4) to[k + j] = acc[n][j] + half[n][tx][j];
            if (threadIdx.x == 0 && blockIdx.x == 0) to[P.K] = gb[n] + half_gb[n];
        }
    }
}
// eight warps share the row blocks of 32 neighbouring sums
template <typename T>
__global__ void __launch_bounds__(256) k_few_join(const float* part, int blocks, int N, int K, void* gw, int64_t ldgw, void* gb) {
    __shared__ float sum[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t e = (int64_t)blockIdx.x * 32 + lane, all = (int64_t)N * (K + 1);
    cafe_next_may_start();
    float s = 0.f;
    if (e < all)
#pragma unroll 4
        for (int b = warp; b < blocks; b += 8) s += part[b * all + e];
    sum[warp][lane] = s;
    __syncthreads();
    if (warp || e >= all) return;
#pragma unroll
    for (int q = 1; q < 8; ++q) s += sum[q][lane];
    const int n = (int)(e / (K + 1)), k = (int)(e - (int64_t)n * (K + 1));
    if (k < K) { if (gw) static_cast<T*>(gw)[n * ldgw + k] = cafe_from_float<T>(s); }
    else if (gb) static_cast<T*>(gb)[n] = cafe_from_float<T>(s);
}
// rows of a block: blocks for every SM several times over, but at least 16 rows each
static int dense_few_rows(int M, int K) {
    const int64_t across = (K + 255) / 256, want = (148 * 8 + across - 1) / across;
    int64_t rows = (M + want - 1) / want;
    rows = rows < 16 ? 16 : rows;
    if (M > rows * 32768) rows = (M + 32767) / 32768;
    return (int)rows;
}
static int64_t dense_few_back_work(const CafeBackward& f) {
    if (f.N < 1 || f.N > CAFE_FEW_MOST || f.M < 1 || f.K < 1 || !(f.gw || f.gb)) return 0;
    const int rows = dense_few_rows(f.M, f.K);
    return (int64_t)((f.M + rows - 1) / rows) * f.N * (f.K + 1) * 4;
}
template <typename T>
static cudaError_t dense_few_back(const CafeBackward& f, void* work, cudaStream_t st) {
    CafeFewBack P = {};
    P.gy = f.gy; P.slope = f.slope; P.x = f.gw ? f.x : nullptr; P.w = f.w;
    P.ldg = f.ldg; P.lds = f.lds; P.ldx = f.ldx; P.ldw = f.ldw; P.ldgx = f.ldgx;
    P.kind = f.slope_kind; P.M = f.M; P.N = f.N; P.K = f.K; P.gx = f.gx;
    P.part = f.gw || f.gb ? (float*)work : nullptr;
    P.rows = dense_few_rows(f.M, f.K);
    const int size = sizeof(T);
    P.vec = P.x && dense_on(f.x, f.ldx, size, 4 * size);
    P.vec_out = f.gx && dense_on(f.gx, f.ldgx, size, 4 * size);
    const int blocks = (f.M + P.rows - 1) / P.rows;
    const dim3 grid((unsigned)((f.K + 255) / 256), (unsigned)blocks);
    cudaError_t e;
    if (f.N <= 1) e = dense_start<false>(k_few_back<T, 1>, grid, 128, 0, 1, st, P);
    else if (f.N <= 4) e = dense_start<false>(k_few_back<T, 4>, grid, 128, 0, 1, st, P);
    else if (f.N <= 8) e = dense_start<false>(k_few_back<T, 8>, grid, 128, 0, 1, st, P);
    else e = dense_start<false>(k_few_back<T, 16>, grid, 128, 0, 1, st, P);
    if (e != cudaSuccess || !P.part) return e;
    return dense_start<false>(k_few_join<T>, dim3((unsigned)(((int64_t)f.N * (f.K + 1) + 31) / 32)), 256, 0, 1, st, (const float*)P.part, blocks, f.N, f.K, f.gw, f.ldgw, f.gb);
}

// `follows`: the kernel before it in the stream is that of the layer before it in the same call, of as few rows
template <typename T>
static cudaError_t dense_forward(const CafeForward& f, int dtype, bool follows, void* work, int64_t work_bytes, cudaStream_t st) {
    if (f.M == 0 || f.N == 0) return cudaSuccess;
    if (f.M <= CAFE_FEW_MOST || f.N <= CAFE_FEW_MOST) return dense_few<T>(f, follows, st);
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
    J.out_row = dense_on(f.y, f.ldy, size, 16);
    J.res_row = f.res && dense_on(f.res, f.ldr, size, 16);
    J.slope_row = f.slope && dense_on(f.slope, f.lds, sizeof(typename CafeSlopeOf<T>::type), 16);
    J.out_vec = dense_on(f.y, f.ldy, size, 4 * size) && (!f.slope || dense_on(f.slope, f.lds, ssize, 4 * ssize));
    const int64_t need = cafe_tiles_forward_work(f, dtype);
    if (need > 0 && work && work_bytes >= need) return cafe_tiles_forward(f, dtype, J, work, st);
    return dense_launch<T>(P, st);
}
template <typename T>
static cudaError_t dense_backward(const CafeBackward& f, int dtype, void* work, int64_t work_bytes, cudaStream_t st) {
    if (f.N >= 1 && f.N <= CAFE_FEW_MOST && f.M >= 1 && f.K >= 1) {
        const int64_t few = dense_few_back_work(f);
        if (few == 0 || (work && work_bytes >= few)) return f.gx || few ? dense_few_back<T>(f, work, st) : cudaSuccess;
    }
    CafeJobs P = {};
    const int size = sizeof(T), ssize = f.slope_kind == CAFE_SLOPE_VALUES ? (int)sizeof(typename CafeSlopeOf<T>::type) : size;
    const int g_vec = dense_on(f.gy, f.ldg, size, 16), s_vec = f.slope_kind != CAFE_SLOPE_NONE && dense_on(f.slope, f.lds, ssize, 16);
    if ((f.gw && f.K > 0) || (f.gb && f.N > 0)) {
        // (without gW wanted, one column of tiles of nothing makes the bias gradient)
        CafeJob& J = P.job[P.count++];
        J.a = f.gy; J.lda = f.ldg; J.a_vec = g_vec; J.as = f.slope; J.ldas = f.lds; J.as_vec = s_vec; J.slope_kind = f.slope_kind;
        J.b = f.x; J.ldb = f.ldx;
        J.rows = f.N; J.cols = f.gw ? f.K : 0; J.depth = f.M;
        J.out = f.gw; J.ldo = f.ldgw; J.out_vec = dense_on(f.gw, f.ldgw, size, 4 * size); J.out_row = dense_on(f.gw, f.ldgw, size, 16); J.gb = f.gb;
    }
    if (f.gx && f.M > 0 && f.K > 0) {
        CafeJob& J = P.job[P.count++];
        J.a = f.gy; J.lda = f.ldg; J.a_kc = 1; J.a_vec = g_vec; J.as = f.slope; J.ldas = f.lds; J.as_vec = s_vec; J.slope_kind = f.slope_kind;
        J.b = f.w; J.ldb = f.ldw;
        J.rows = f.M; J.cols = f.K; J.depth = f.N;
        J.out = f.gx; J.ldo = f.ldgx; J.out_vec = dense_on(f.gx, f.ldgx, size, 4 * size); J.out_row = dense_on(f.gx, f.ldgx, size, 16);
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
    DENSE_TYPED(dtype, e = dense_forward<T>(f, dtype, false, work_dev, work_bytes, (cudaStream_t)stream));
    return dense_done(e);
}

int64_t cafe_linear_backward_work(const void* gy_dev, int64_t ldg, int slope_kind, const void* x_dev, int64_t ldx, const void* w_dev, int64_t ldw,
                                  int M, int N, int K, int dtype, int want_gx, int want_gw, int want_gb) {
    CafeBackward f = {};
    f.gy = gy_dev; f.ldg = ldg; f.slope_kind = slope_kind; f.x = x_dev; f.ldx = ldx; f.w = w_dev; f.ldw = ldw; f.M = M; f.N = N; f.K = K;
    f.gx = want_gx ? (void*)k_aligned : nullptr; f.gw = want_gw ? (void*)k_aligned : nullptr; f.gb = want_gb ? (void*)k_aligned : nullptr;
    if (!dense_type_ok(dtype) || !dense_sizes_ok(M, N, K)) return 0;
    const int64_t few = dense_few_back_work(f);
    return few ? few : cafe_tiles_backward_work(f, dtype);
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

int cafe_linear_gave_up(int* count) {
    if (!count) return CAFE_ERR_ARG;
    int mine = 0, tiles = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&mine, g_dense_gave_up, sizeof mine);
    if (e == cudaSuccess) e = cafe_tiles_gave_up(&tiles);
    *count = mine + tiles;
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
    for (int l = 0; l < layers && e == cudaSuccess; ++l) {
        const bool follows = l > 0 && M <= CAFE_FEW_MOST && widths[l] > 0;
        DENSE_TYPED(dtype, e = dense_forward<T>(f[l], dtype, follows, work_dev, work_bytes, (cudaStream_t)stream));
    }
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
    int first = gx_dev ? 0 : layers;   // the lowest layer that a gradient is wanted of: below it nothing is computed
    for (int l = layers - 1; l >= 0; --l) if (gw_dev[l] || gb_dev[l]) first = l < first ? l : first;
    for (int l = layers - 1; l >= first; --l) {
        const bool last = l == layers - 1;
        const bool plain = acts[l] == CAFE_ACT_NONE || M == 0 || widths[l + 1] == 0;   // (a layer without outputs has no slope either)
        const int kind = plain ? CAFE_SLOPE_NONE : slope_dev && slope_dev[l] ? CAFE_SLOPE_VALUES : CAFE_SLOPE_OUTPUT;
        if (kind == CAFE_SLOPE_OUTPUT && acts[l] != CAFE_ACT_RELU) return CAFE_ERR_ARG;
        const int64_t ldn = (widths[l + 1] + 7) & ~7, ldk = (widths[l] + 7) & ~7;
        f[l] = {last ? gy_dev : half[l & 1], kind == CAFE_SLOPE_VALUES ? slope_dev[l] : y_dev[l], l ? y_dev[l - 1] : x_dev, w_dev[l],
                last ? ldg : ldn, ldy[l], l ? ldy[l - 1] : ldx, ldw[l], kind, M, widths[l + 1], widths[l],
                l > first ? half[(l - 1) & 1] : l ? nullptr : gx_dev, gw_dev[l], gb_dev[l], l ? ldk : ldgx, widths[l]};
        if (!dense_backward_ok(f[l])) return CAFE_ERR_ARG;
    }
    cudaError_t e = cudaSuccess;
    for (int l = layers - 1; l >= first && e == cudaSuccess; --l)
        DENSE_TYPED(dtype, e = dense_backward<T>(f[l], dtype, half[1] + half_bytes, work_bytes - 2 * half_bytes, (cudaStream_t)stream));
    return dense_done(e);
}

}  // extern "C"
