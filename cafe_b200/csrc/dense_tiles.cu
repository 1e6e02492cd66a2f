// dense_tiles.cu -- the products of large layers: operands laid out for the copy engine first, then tiles that nothing but copies
// and matrix instructions work on.
//
// dense_cuda.cu's kernel cuts and stores its operands itself, once for every tile that reads them; its loading warps set its
// pace.  Where a product is large that work is done once: k_parts writes x, W or gz = gy * act'(z) as bf16 parts (three of fp32,
// pitch rounded up to 16 bytes; 16-bit tensors only where their rows are not on 16 bytes or a slope belongs to them, otherwise
// they are read in place), with the column sums of gz on the way, and k_tiles fetches boxes of them by cp.async.bulk.tensor
// in the order the tensor cores read, whichever index is contiguous.
//
// k_tiles: a block makes 128 x BN outputs; one thread fetches, one issues products, four warps take the sums out (and meanwhile
// add up the bias gradient).  Two blocks share an SM, so that one's end runs beside the other's products; two stages of 48 KB
// each.  Held sums leave 40 of a thread's 168 registers for the rest: 492 bytes of spill stores and 352 of loads in fp32, 172 and 112 in
// fp16; k_tiles_pair in fp32 48 and 116.  Blocks of a cluster share the depth of a tile as in dense_cuda.cu.
#include <cuda.h>

#include "dense.cuh"

#define CAFE_TILES_THREADS 192
#define CAFE_PARTS_COLS 256
// rows of a block of k_parts (a row of partial column sums each): short blocks while they are few, so that all are under way at
// once (1 M elements: 32 rows 3 us, 128 rows 8), long ones where there are enough (16384 x 4096: 128 rows save a third)
static __host__ __device__ constexpr int cafe_parts_rows(int rows, int cols) {
    return (int64_t)((rows + 127) / 128) * ((cols + CAFE_PARTS_COLS - 1) / CAFE_PARTS_COLS) >= 1024 ? 128 : 32;
}

__device__ int g_tiles_gave_up;   // 1: a wait ran out (its outputs are not numbers)
cudaError_t cafe_tiles_gave_up(int* flag) { return cudaMemcpyFromSymbol(flag, g_tiles_gave_up, sizeof *flag); }

template <typename T> struct CafeTiles {
    static constexpr int parts = 1, BK = 64, type = 0;
    typedef T part;
};
template <> struct CafeTiles<__nv_bfloat16> { static constexpr int parts = 1, BK = 64, type = 1; typedef __nv_bfloat16 part; };
template <> struct CafeTiles<float> { static constexpr int parts = 3, BK = 32, type = 1; typedef __nv_bfloat16 part; };
// fp32: turns of 32 between two times that the large sums are taken out, and the others.  The tensor cores cut an instruction's products and
// their sum off: in proportion to the depth, and towards zero.  Relative error (norms; signed, all positive operands) of a depth of 65 536
// in one go 9.4e-6, 3.6e-5; with the large sums in pieces of 256 of k and the others in one go 2.6e-6, 1.1e-5 (131 072: 4.9e-6, 2.0e-5); with
// the others in pieces of 4096 5.0e-7, 7.2e-7 (131 072: 5.8e-7, 7.5e-7; 4096: 3.0e-7, 2.1e-7), where plain fp32 has 4.6e-6, 3.7e-6.  Larger
// pieces were not measurably faster.
#define CAFE_TILES_CHUNK 8
template <typename T> static constexpr int cafe_tiles_chunk() { return CafeTiles<T>::parts == 3 ? CAFE_TILES_CHUNK : 4096 / CafeTiles<T>::BK; }
// 16 bits: a tile's sums stay in tensor memory to the end, so a block adds over its share of the depth in one go, and what is cut off
// grows with it: 6.3e-9 (bf16 5.8e-9) of a sum of positive products for each k, in cuBLAS's products as in these.  No block gets more
// than loses a fifth of what rounding the result may change (2^-11 = 4.9e-4, bf16 3.9e-3): 1.0e-4 and 7.6e-4.  Longer depths are
// shared by a cluster's blocks, and where eight are not enough (fp16 beyond 131 072) their sums are held in registers and taken out
// every 4096 of k.
template <typename T> static constexpr int cafe_tiles_depth() { return sizeof(T) == 4 ? 1 << 30 : CafeTiles<T>::type ? 1 << 17 : 1 << 14; }
#define CAFE_TILES_LOW (CAFE_TILES_CHUNK * CAFE_LIN_LOW)   // turns between two times that the other sums are

// ---- operands as parts ---------------------------------------------------------------------------------------------------
struct CafePartsJob {
    const void *src, *slope;
    int64_t ld, lds, pitch, plane;   // pitch and plane of dst in elements
    int kind, vec, slope_vec, rows, cols, blocks_x, blocks;
    void* dst;                       // null: sums only
    float* sums;                     // [row blocks][cols] sums of the rows of each block, or null
};
struct CafeParts {
    CafePartsJob job[3];
    int count;
};
template <typename T> __device__ __forceinline__ void cafe_read8(const T* p, int n, bool vec, float* v) {
    if (vec && n == 8) {
        alignas(16) T x[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(x)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = cafe_to_float(x[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < n ? cafe_to_float(cafe_ldg(p + j)) : 0.f;
    }
}
// Bound by its bytes: fp32 4 in (8 with a slope) and 6 out an element (17.8 M elements of x and W 27 us, 6.5 TB/s with what stays in L2).
template <typename T>
__global__ void __launch_bounds__(256) k_parts(const __grid_constant__ CafeParts P) {
    typedef typename CafeSlopeOf<T>::type ST;
    __shared__ float part[8][CAFE_PARTS_COLS];
    int block = blockIdx.x, q = 0;
    while (q + 1 < P.count && block >= P.job[q].blocks) block -= P.job[q++].blocks;
    const CafePartsJob& J = P.job[q];
    const int by = block / J.blocks_x, bx = block - by * J.blocks_x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col = bx * CAFE_PARTS_COLS + lane * 8, n = min(8, J.cols - col);
    float sum[8] = {};
    const int per = cafe_parts_rows(J.rows, J.cols);
    const int64_t r0 = (int64_t)by * per, r1 = min(r0 + per, (int64_t)J.rows);
    cafe_next_may_start();
    if (n > 0) {
#pragma unroll 4
        for (int64_t r = r0 + warp; r < r1; r += 8) {
            alignas(16) float v[8];
            cafe_read8(static_cast<const T*>(J.src) + r * J.ld + col, n, J.vec, v);
            if (J.kind == CAFE_SLOPE_VALUES) {
                float s[8];
                cafe_read8(static_cast<const ST*>(J.slope) + r * J.lds + col, n, J.slope_vec, s);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= s[j];
            } else if (J.kind == CAFE_SLOPE_OUTPUT) {
                float s[8];
                cafe_read8(static_cast<const T*>(J.slope) + r * J.lds + col, n, J.slope_vec, s);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = s[j] > 0.f ? v[j] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += v[j];
            if (!J.dst) continue;
            uint4* out = reinterpret_cast<uint4*>(static_cast<typename CafeTiles<T>::part*>(J.dst) + r * J.pitch + col);
            if constexpr (sizeof(T) == 2) {
                alignas(16) T o[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = cafe_from_float<T>(v[j]);
                *out = *reinterpret_cast<const uint4*>(o);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = cafe_quiet(v[j]);
#pragma unroll
                for (int p = 0; p < 3; ++p) {   // the next 8 bits of each, cut off
                    uint32_t o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        o[j] = __byte_perm(__float_as_uint(v[2 * j]), __float_as_uint(v[2 * j + 1]), 0x7632);
                        v[2 * j] -= __uint_as_float(__float_as_uint(v[2 * j]) & 0xffff0000u);
                        v[2 * j + 1] -= __uint_as_float(__float_as_uint(v[2 * j + 1]) & 0xffff0000u);
                    }
                    out[(int64_t)p * J.plane / 8] = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
        }
    }
    if (!J.sums) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) part[warp][lane * 8 + j] = sum[j];
    __syncthreads();
    const int c = bx * CAFE_PARTS_COLS + threadIdx.x;
    if (c >= J.cols) return;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += part[w][threadIdx.x];
    J.sums[(int64_t)by * J.cols + c] = s;
}

// ---- tiles ---------------------------------------------------------------------------------------------------------------
template <typename T, int BN> struct CafeTilesShape {
    typedef CafeTiles<T> L;
    static constexpr int rowb = L::BK * 2;
    static constexpr int a_part = CAFE_LIN_BM * rowb, b_part = BN * rowb, stage = L::parts * (a_part + b_part);
    static constexpr int tile = CAFE_LIN_BM * (128 + 4) * 4;
    static constexpr int stages = 98304 / stage < 6 ? 98304 / stage : 6;
    static constexpr int bytes = (stage * stages > tile ? stage * stages : tile) + 1024;
    static constexpr int tm_cols = L::parts == 3 ? 2 * BN : BN;
};
#define CAFE_TILES_ROWS (1 << 20)   // of x that these kernels take
struct CafeTilesArgs {
    CUtensorMap a, b;
    CafeJob job;
    const float* sums;   // partial column sums of A for job.gb
    int sum_rows, splits;
};

// HOLD: the sums are taken out and added in registers on the way (fp32: always; 16 bits: depths too long for tensor memory, BN = 128).
template <typename T, int BN, bool HOLD>
__global__ void __launch_bounds__(CAFE_TILES_THREADS, 2) k_tiles(const __grid_constant__ CafeTilesArgs P) {
    typedef CafeTiles<T> L;
    typedef CafeTilesShape<T, BN> Sh;
    extern __shared__ char sh_raw[];
    __shared__ __align__(8) uint64_t bars[2 * Sh::stages + 3];
    __shared__ uint32_t tm_at;
    __shared__ volatile int bail;
    const uint32_t base = (cafe_smem(sh_raw) + 1023u) & ~1023u;
    const uint32_t bar0 = cafe_smem(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (Sh::stages + s); };
    const uint32_t acc_full = bar0 + 8u * (2 * Sh::stages), acc_empty = acc_full + 8, all_done = acc_full + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const CafeJob& J = P.job;
    const int splits = P.splits, tile = blockIdx.x / splits, rank = blockIdx.x - tile * splits;
    const int tm = tile / J.tiles_n, tn = tile - tm * J.tiles_n, row0 = tm * CAFE_LIN_BM, col0 = tn * BN;
    const int turns_all = (J.depth + L::BK - 1) / L::BK, share = (turns_all + splits - 1) / splits;
    const int t0 = min(rank * share, turns_all), turns = min(share, turns_all - t0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < Sh::stages; ++s) { cafe_bar_init(full(s), 1); cafe_bar_init(empty(s), 1); }
        cafe_bar_init(acc_full, 1);
        cafe_bar_init(acc_empty, 4);
        cafe_bar_init(all_done, 1);
        cafe_fence_barrier_init();
        bail = 0;
    }
    cafe_next_may_start();
    if (warp == 1) cafe_tm_alloc(cafe_smem(&tm_at), Sh::tm_cols);
    cafe_tc_before();
    __syncthreads();
    cafe_tc_after();
    const uint32_t tmem = tm_at;

    static_assert(HOLD ? BN == 128 : L::parts == 1, "sums held by a thread");
    constexpr int taken = HOLD ? BN : 32, CHUNK = cafe_tiles_chunk<T>();
    float acc[taken];
    const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    bool fine = true;
    if (warp == 0) {
        // ---- boxes of the operands
        int t = 0, s = 0;
        uint32_t phase = 1;   // (a fresh barrier's phase before its first counts as over)
        for (int k0 = t0 * L::BK; t < turns; ++t, k0 += L::BK) {
            if (!(fine = __all_sync(0xffffffffu, cafe_bar_wait(empty(s), phase, &bail)))) break;
            const uint32_t a = base + s * Sh::stage, b = a + L::parts * Sh::a_part, bar = full(s);
            if (cafe_elect()) {
                cafe_bar_expect(bar, Sh::stage);
                if (J.a_kc) cafe_box_load(a, &P.a, k0, row0, 0, bar);
                else
#pragma unroll
                    for (int q = 0; q < CAFE_LIN_BM / 64; ++q) cafe_box_load(a + q * L::parts * L::BK * 128, &P.a, row0 + 64 * q, k0, 0, bar);
                if (J.b_kc) cafe_box_load(b, &P.b, k0, col0, 0, bar);
                else
#pragma unroll
                    for (int q = 0; q < BN / 64; ++q) cafe_box_load(b + q * L::parts * L::BK * 128, &P.b, col0 + 64 * q, k0, 0, bar);
            }
            if (++s == Sh::stages) { s = 0; phase ^= 1u; }
        }
        if (!fine)   // given up: the copies in flight end before the block does
            for (int u = max(0, t - Sh::stages); u < t; ++u)
                for (int i = 0; i < (1 << 20) && !cafe_bar_try(full(u % Sh::stages), (uint32_t)(u / Sh::stages) & 1u); ++i) {}
    } else if (warp == 1) {
        // ---- products
        const uint32_t instr = cafe_mma_instr(L::type, CAFE_LIN_BM, BN) | (J.a_kc ? 0u : 1u << 15) | (J.b_kc ? 0u : 1u << 16);
        const uint64_t da = J.a_kc ? cafe_operand<Sh::rowb>(base) : cafe_operand_mn(base, L::parts * L::BK * 128);
        const uint64_t db = J.b_kc ? cafe_operand<Sh::rowb>(base + L::parts * Sh::a_part) : cafe_operand_mn(base + L::parts * Sh::a_part, L::parts * L::BK * 128);
        // offsets in 16-byte units: from a part to the next, from 16 k to the next 16
        const uint32_t ap = (J.a_kc ? Sh::a_part : L::BK * 128) >> 4, bp = (J.b_kc ? Sh::b_part : L::BK * 128) >> 4;
        const uint32_t ak = (J.a_kc ? 32 : 2048) >> 4, bk = (J.b_kc ? 32 : 2048) >> 4;
        int s = 0, in_chunk = 0;
        uint32_t phase = 0, chunk_phase = 1;
        for (int t = 0; t < turns; ++t) {
            if (!(fine = __all_sync(0xffffffffu, cafe_bar_wait(full(s), phase, &bail)))) break;
            if (HOLD && in_chunk == 0 && t > 0) {
                if (!(fine = __all_sync(0xffffffffu, cafe_bar_wait(acc_empty, chunk_phase & 1u, &bail)))) break;
            }
            cafe_tc_after();
            const uint64_t a = da + (uint32_t)(s * Sh::stage >> 4), b = db + (uint32_t)(s * Sh::stage >> 4);
            const bool ends = in_chunk == CHUNK - 1 || t == turns - 1, low = L::parts == 3 && (t + 1) % CAFE_TILES_LOW == 0 && t < turns - 1;
            if (cafe_elect()) {
#pragma unroll
                for (int k = 0; k < L::BK / 16; ++k) cafe_mma(tmem, a + ak * k, b + bk * k, instr, in_chunk > 0 || k > 0);
                if (HOLD && ends && !low) cafe_mma_commit(acc_full);
                if constexpr (L::parts == 3) {
#pragma unroll
                    for (int q = 0; q < 5; ++q) {
                        constexpr int ia[5] = {0, 1, 1, 0, 2}, ib[5] = {1, 0, 1, 2, 0};
#pragma unroll
                        for (int k = 0; k < L::BK / 16; ++k)
                            cafe_mma(tmem + BN, a + ia[q] * ap + ak * k, b + ib[q] * bp + bk * k, instr, t % CAFE_TILES_LOW > 0 || q > 0 || k > 0);
                    }
                    if (low) cafe_mma_commit(acc_full);
                }
                cafe_mma_commit(empty(s));
            }
            ++in_chunk;
            if (HOLD && ends) { in_chunk = 0; ++chunk_phase; }
            if (++s == Sh::stages) { s = 0; phase ^= 1u; }
        }
        __syncwarp();
        if (cafe_elect()) cafe_mma_commit(all_done);
    } else {
        // ---- sums out of tensor memory, 32 rows a warp; before that the bias gradient from its partial sums
        if (P.sums && tn == 0 && rank == 0) {
            const int r = row0 + (int)threadIdx.x - 64;
            if (r < J.rows) {
                float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
                int q = 0;
                for (; q + 4 <= P.sum_rows; q += 4) {
                    s0 += __ldg(P.sums + (int64_t)q * J.rows + r);
                    s1 += __ldg(P.sums + (int64_t)(q + 1) * J.rows + r);
                    s2 += __ldg(P.sums + (int64_t)(q + 2) * J.rows + r);
                    s3 += __ldg(P.sums + (int64_t)(q + 3) * J.rows + r);
                }
                for (; q < P.sum_rows; ++q) s0 += __ldg(P.sums + (int64_t)q * J.rows + r);
                static_cast<T*>(J.gb)[r] = cafe_from_float<T>((s0 + s1) + (s2 + s3));
            }
            __syncwarp();
        }
        if constexpr (HOLD) {
            auto take = [&](uint32_t at, bool first) {
#pragma unroll
                for (int c = 0; c < BN; c += 16) {
                    float v[16];
                    cafe_tm_load16(at + c, v);
                    cafe_tm_wait_load();
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[c + i] = first ? v[i] : acc[c + i] + v[i];
                }
            };
            auto join = [&]() {   // fp32: the other sums
#pragma unroll
                for (int c = 0; c < BN; c += 16) {
                    float v[16];
                    cafe_tm_load16(from + BN + c, v);
                    cafe_tm_wait_load();
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[c + i] = cafe_join_sums(acc[c + i], v[i]);
                }
            };
            const int chunks = (turns + CHUNK - 1) / CHUNK;
            if (turns == 0) {
#pragma unroll
                for (int i = 0; i < BN; ++i) acc[i] = 0.f;
            }
            for (int c = 0; c < chunks && fine; ++c) {
                fine = cafe_bar_wait(acc_full, (uint32_t)c & 1u, &bail);
                cafe_tc_after();
                fine = __all_sync(0xffffffffu, fine);
                if (fine) take(from, c == 0);
                if (L::parts == 3 && fine && (c + 1) % CAFE_LIN_LOW == 0 && c < chunks - 1) join();
                cafe_tc_before();
                __syncwarp();
                if (lane == 0) cafe_bar_arrive(acc_empty);
            }
            fine = cafe_bar_wait(all_done, 0, &bail) && fine;
            cafe_tc_after();
            fine = __all_sync(0xffffffffu, fine);
            if (L::parts == 3 && fine && turns > 0) join();
        } else {
            fine = cafe_bar_wait(all_done, 0, &bail);
            cafe_tc_after();
            fine = __all_sync(0xffffffffu, fine);
        }
        if (!fine) g_tiles_gave_up = 1;
    }
    __syncwarp();
    // ---- 128 columns at a time: sums to shared memory (the stages are free: all products are done), then what belongs at the end
    for (int h = 0; h < BN / 128; ++h) {
        if (col0 + h * 128 >= J.cols) break;   // (the same for all blocks of the cluster)
        __syncthreads();
        if (warp >= 2) {
            const int r = (warp & 3) * 32 + lane;
            const uint32_t at = base + (uint32_t)(r * 132) * 4u;
            const bool ok = fine && !bail;
            if constexpr (HOLD) {
                if (!ok) {
#pragma unroll
                    for (int i = 0; i < BN; ++i) acc[i] = __uint_as_float(0x7fffffffu);
                }
                cafe_sums_put<BN>(acc, at);
            } else {
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    cafe_tm_load16(from + h * 128 + c, acc);
                    cafe_tm_load16(from + h * 128 + c + 16, acc + 16);
                    cafe_tm_wait_load();
                    if (!ok || turns == 0) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) acc[i] = ok ? 0.f : __uint_as_float(0x7fffffffu);
                    }
                    cafe_sums_put<32>(acc, at + 4 * c);
                }
            }
        }
        if (splits > 1) cafe_cluster_sync(); else __syncthreads();
        cafe_finish<T, 128>(J, base, row0, col0 + h * 128, rank, splits, CAFE_TILES_THREADS);
        if (splits > 1) cafe_cluster_sync();   // (others may still read this block's sums)
    }
    cafe_tc_before();
    __syncthreads();
    cafe_tc_after();
    if (warp == 1) cafe_tm_free(tmem, Sh::tm_cols);
}

// ---- tiles one after the other, by pairs of blocks --------------------------------------------------------------------------
// Where there are tiles enough: two blocks, an SM each, work on tiles of 256 x BN, tile after tile.  Each fetches its own 128 rows of
// A and half of B's, so an SM's boxes are half to three quarters of those of a block by itself, and the products no longer wait
// for them (16384x1024x1024 in fp32: 48 KB for 768 cycles of products an SM came at 29 bytes a cycle, tensor cores busy 46 %).
// Block 0 issues the products of both; the boxes of both complete on its barriers (no thread stands between a copy and the products
// that read it).
//
// fp32: eight warps have 32 rows and half of the columns each.  They take the large sums out every 256 of k and everything when a
// tile's products are done, into registers; tensor memory is then free for the next tile, whose products run while this one is
// finished.  16 bits: two sets of sums in tensor memory, two groups of four warps take turns, a lane takes sixteen sums at a time.
// Either way a lane has a row: bias, activation, residual; results go to its warp's staging rows, from which the warp writes 128
// bytes of a row at a time.  Nobody waits for another warp.
#define CAFE_PAIR_THREADS 320
#define CAFE_PAIRS 74          // pairs of blocks that run at a time
template <typename T, int BN> struct CafePairShape {
    typedef CafeTiles<T> L;
    typedef typename CafeSlopeOf<T>::type ST;
    static constexpr int rowb = L::BK * 2;
    static constexpr int a_part = CAFE_LIN_BM * rowb, b_part = BN / 2 * rowb, stage = L::parts * (a_part + b_part);
    static constexpr int cols = sizeof(T) == 2 && sizeof(ST) == 2 ? 64 : 32;                  // of a pass
    static constexpr int out_row = cols * sizeof(T), slope_row = cols * sizeof(ST);           // bytes
    static constexpr int staging = 32 * (out_row + slope_row);
    static constexpr int room = 229376 - 8 * staging, stages = room / stage < 6 ? room / stage : 6;
    static constexpr int bytes = stage * stages + 8 * staging + 1024;
    static constexpr int sets = L::parts == 3 ? 1 : 2, tm_set = L::parts == 3 ? 2 * BN : BN;
    static constexpr int takers = L::parts == 3 ? 8 : 4;                                      // warps of a block that share a tile
    static constexpr int mine = L::parts == 3 ? BN / 2 : BN;                                  // columns of a warp
};
__device__ __forceinline__ uint4 cafe_get16(uint32_t at) {
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
    return x;
}
// Staged rows of ROW bytes: 16-byte piece c of row r lies at piece c ^ r (of as many as a row has, at most eight).
template <int ROW> __device__ __forceinline__ uint32_t cafe_staged(uint32_t at, int r, int c) {
    return at + (uint32_t)(r * ROW + ((c ^ (r & (ROW >= 128 ? 7 : ROW / 16 - 1))) << 4));
}
// The warp's 32 rows of W columns between shared memory and rows of E elsewhere, `n` columns and `m` rows of them there; on the way
// out rows of `add` are added.
template <typename E, int W>
__device__ __forceinline__ void cafe_rows_out(uint32_t at, E* to, int64_t ld, bool on16, const E* add, int64_t lda, bool add16, int m, int n, int lane) {
    constexpr int ROW = W * sizeof(E), per = ROW / 16, each = 16 / sizeof(E);
    const int c = lane % per;
    const bool whole = (c + 1) * each <= n;
#pragma unroll 4
    for (int r = lane / per; r < m; r += 32 / per) {
        alignas(16) E x[each], y[each];
        if (add) {
            const E* p = add + r * lda + c * each;
            if (add16 && whole) *reinterpret_cast<uint4*>(y) = __ldg(reinterpret_cast<const uint4*>(p));
            else {
#pragma unroll
                for (int q = 0; q < each; ++q) y[q] = c * each + q < n ? cafe_ldg(p + q) : cafe_from_float<E>(0.f);
            }
        }
        *reinterpret_cast<uint4*>(x) = cafe_get16(cafe_staged<ROW>(at, r, c));
        if (add) {
#pragma unroll
            for (int q = 0; q < each; ++q) x[q] = cafe_from_float<E>(cafe_to_float(x[q]) + cafe_to_float(y[q]));
        }
        E* p = to + r * ld + c * each;
        if (on16 && whole) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(x);
        else {
#pragma unroll
            for (int q = 0; q < each; ++q) if (c * each + q < n) p[q] = x[q];
        }
    }
}
template <typename E, int W> __device__ __forceinline__ void cafe_rows_in(uint32_t at, const E* from, int64_t ld, bool on16, int m, int n, int lane) {
    constexpr int ROW = W * sizeof(E), per = ROW / 16, each = 16 / sizeof(E);
#pragma unroll 4
    for (int r = lane / per; r < m; r += 32 / per) {
        const int c = lane % per;
        const E* p = from + r * ld + c * each;
        const uint32_t to = cafe_staged<ROW>(at, r, c);
        if (on16 && (c + 1) * each <= n) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(p) : "memory");
        else {
            alignas(16) E x[each];
#pragma unroll
            for (int q = 0; q < each; ++q) x[q] = c * each + q < n ? __ldg(p + q) : cafe_from_float<E>(0.f);
            const uint4 y = *reinterpret_cast<const uint4*>(x);
            cafe_put16(to, y.x, y.y, y.z, y.w);
        }
    }
}


// the end of sixteen neighbouring sums of a row (columns j ..), the lane's own, r = lane: bias, activation, residual from the staged row, rounding, staging
template <typename T, int OUT_ROW, int SLOPE_ROW, bool RES>
__device__ __forceinline__ void cafe_row_end(const CafeJob& J, float* z, int64_t j, uint32_t out, uint32_t slopes, int r, int c) {
    typedef typename CafeSlopeOf<T>::type ST;
    constexpr int each = 16 / sizeof(T), slope_each = 16 / sizeof(ST);
    float d[16];
    if (J.bias) {   // (a lane loads one of them)
        const int64_t i = j + (r & 15);
        const float mine = i < J.cols ? cafe_to_float(__ldg(static_cast<const T*>(J.bias) + i)) : 0.f;
#pragma unroll
        for (int q = 0; q < 16; ++q) z[q] += __shfl_sync(0xffffffffu, mine, q);
    }
    cafe_act_all<16>(z, J.act, d);
#pragma unroll
    for (int p = 0; p < 16; p += each) {
        const uint32_t at = cafe_staged<OUT_ROW>(out, r, (c + p) / each);
        alignas(16) T x[each];
        if (RES && J.res) {
            *reinterpret_cast<uint4*>(x) = cafe_get16(at);
#pragma unroll
            for (int q = 0; q < each; ++q) z[p + q] += cafe_to_float(x[q]);
        }
#pragma unroll
        for (int q = 0; q < each; ++q) x[q] = cafe_from_float<T>(z[p + q]);
        const uint4 y = *reinterpret_cast<const uint4*>(x);
        cafe_put16(at, y.x, y.y, y.z, y.w);
    }
    if (J.slope_out) {
#pragma unroll
        for (int p = 0; p < 16; p += slope_each) {
            alignas(16) ST x[slope_each];
            cafe_slopes<slope_each>(d + p, x);
            const uint4 y = *reinterpret_cast<const uint4*>(x);
            cafe_put16(cafe_staged<SLOPE_ROW>(slopes, r, (c + p) / slope_each), y.x, y.y, y.z, y.w);
        }
    }
}
// 32 of a lane's sums to its staging row, and back sixteen at a time
template <int I> __device__ __forceinline__ void cafe_row_put(const float* acc, uint32_t at, int lane) {
#pragma unroll
    for (int c = 0; c < 32; c += 4)
        cafe_put16(cafe_staged<128>(at, lane, c / 4), __float_as_uint(acc[I + c]), __float_as_uint(acc[I + c + 1]), __float_as_uint(acc[I + c + 2]), __float_as_uint(acc[I + c + 3]));
}

struct CafePairArgs {
    CUtensorMap a[2], b[2];
    CafeJob job[2];      // the longer tiles first
    int count;
    const float* sums;   // [sum_rows][gb_cols]: partial sums of a bias gradient, added up on the way
    int sum_rows, gb_cols;
    void* gb;
    int share[CAFE_PAIRS + 1];
    // fp32: the first product's depth in `splits` parts, whose sums go to `partial` ([part][rows][pitch]) for k_parts_join to add
    int splits, pitch;
    float* partial;
};
// A backward's two products are one launch.  The first one's tiles (the longer) go round the pairs; the second one's are handed out
// so that all pairs end at about the same time, pair p has those from share[p] to share[p + 1]: 2048x1024x1024 takes the time of gW
// alone (backward 84 us as two launches, 70 as one).
struct CafePairTiles {
    int first, step, own, from, all;   // of the first product: first, first + step, .. `own` of them (part by part); of the second: from, from + 1, ..
    __device__ __forceinline__ CafePairTiles(const CafePairArgs& P, int pair, int pairs) {
        const int units = P.job[0].tiles * P.splits;
        first = pair; step = pairs;
        own = pair < units ? (units - pair + pairs - 1) / pairs : 0;
        from = P.share[pair];
        all = own + P.share[pair + 1] - from;
    }
    __device__ __forceinline__ int which(int n) const { return n >= own; }
    __device__ __forceinline__ int tile(const CafePairArgs& P, int n) const { return n < own ? (first + n * step) % P.job[0].tiles : from + n - own; }
    __device__ __forceinline__ int part(const CafePairArgs& P, int n) const { return n < own ? (first + n * step) / P.job[0].tiles : 0; }
    // the turns [t0, t1) of the n-th tile
    template <int BK> __device__ __forceinline__ void turns(const CafePairArgs& P, int n, int* t0, int* t1) const {
        const int all_turns = (P.job[which(n)].depth + BK - 1) / BK;
        *t0 = 0; *t1 = all_turns;
        if (n < own && P.splits > 1) {
            const int share = (all_turns + P.splits - 1) / P.splits;
            *t0 = part(P, n) * share;
            *t1 = min(all_turns, *t0 + share);
        }
    }
};
// the parts' sums of a product, added in order
__global__ void __launch_bounds__(256) k_parts_join(const float* partial, int splits, int rows, int cols, int pitch, float* out, int64_t ldo) {
    const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x, per = pitch / 4, all = (int64_t)rows * pitch;
    if (q >= rows * per) return;
    const int64_t r = q / per;
    const int c = (int)(q - r * per) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = 0; p < splits; ++p) {
        const float4 y = __ldg(reinterpret_cast<const float4*>(partial + p * all + r * pitch + c));
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) if (c + j < cols) out[r * ldo + c + j] = v[j];
}

template <typename T, int BN>
__global__ void __launch_bounds__(CAFE_PAIR_THREADS, 1) k_tiles_pair(const __grid_constant__ CafePairArgs P) {
    typedef CafeTiles<T> L;
    typedef CafePairShape<T, BN> Sh;
    typedef typename CafeSlopeOf<T>::type ST;
    extern __shared__ char sh_raw[];
    __shared__ __align__(8) uint64_t bars[2 * Sh::stages + 8];
    __shared__ uint32_t tm_at;
    __shared__ volatile int bail;
    const uint32_t base = (cafe_smem(sh_raw) + 1023u) & ~1023u;
    const uint32_t bar0 = cafe_smem(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (Sh::stages + s); };
    const uint32_t more = bar0 + 8u * (2 * Sh::stages);
    // a chunk's large sums are ready / taken (fp32); for each set of sums: all of a tile's are ready / taken
    const uint32_t chunk_full = more, chunk_taken = more + 8u;
    auto tile_full = [&](int g) { return more + 16u + 8u * g; };
    auto tile_taken = [&](int g) { return more + 32u + 8u * g; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cafe_cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const CafePairTiles list(P, pair, pairs);

    if (threadIdx.x == 0) {
        for (int s = 0; s < Sh::stages; ++s) { cafe_bar_init(full(s), 1); cafe_bar_init(empty(s), 1); }   // (full: block 0's, for the boxes of both)
        cafe_bar_init(chunk_full, 1);
        cafe_bar_init(chunk_taken, 2 * Sh::takers);
        for (int g = 0; g < 2; ++g) { cafe_bar_init(tile_full(g), 1); cafe_bar_init(tile_taken(g), 2 * Sh::takers); }
        cafe_fence_barrier_init();
        bail = 0;
    }
    cafe_next_may_start();
    if (warp == 1) cafe_tm_alloc2(cafe_smem(&tm_at), Sh::sets * Sh::tm_set);
    cafe_tc_before();
    __syncthreads();
    cafe_cluster_sync();
    cafe_tc_after();
    cafe_wait_for_earlier();
    const uint32_t tmem = tm_at;

    if (warp == 0) {
        // ---- boxes of the operands: this block's rows of A, this block's half of B's
        bool fine = true;
        int s = 0;
        uint32_t phase = 1;   // (a fresh barrier's phase before its first counts as over)
        int64_t u = 0;
        for (int n = 0; n < list.all && fine; ++n) {
            const int which = list.which(n), tile = list.tile(P, n);
            int t0, t1;
            list.turns<L::BK>(P, n, &t0, &t1);
            const CafeJob& J = P.job[which];
            const CUtensorMap *ma = &P.a[which], *mb = &P.b[which];
            const int tm = tile / J.tiles_n, row0 = tm * 256 + rank * 128, col0 = (tile - tm * J.tiles_n) * BN + rank * (BN / 2);
            const int a_kc = J.a_kc, b_kc = J.b_kc;
            for (int k0 = t0 * L::BK; k0 < t1 * L::BK; k0 += L::BK, ++u) {
                if (!(fine = __all_sync(0xffffffffu, cafe_bar_wait(empty(s), phase, &bail)))) break;
                const uint32_t a = base + s * Sh::stage, b = a + L::parts * Sh::a_part, bar = cafe_cluster_map(full(s), 0);
                if (cafe_elect()) {
                    if (rank == 0) cafe_bar_expect(full(s), 2 * Sh::stage);   // (block 1's bytes may come before: the phase waits for this arrival)
                    if (a_kc) cafe_box_load2(a, ma, k0, row0, 0, bar);
                    else
#pragma unroll
                        for (int q = 0; q < CAFE_LIN_BM / 64; ++q) cafe_box_load2(a + q * L::parts * L::BK * 128, ma, row0 + 64 * q, k0, 0, bar);
                    if (b_kc) cafe_box_load2(b, mb, k0, col0, 0, bar);
                    else
#pragma unroll
                        for (int q = 0; q < BN / 128; ++q) cafe_box_load2(b + q * L::parts * L::BK * 128, mb, col0 + 64 * q, k0, 0, bar);
                }
                if (++s == Sh::stages) { s = 0; phase ^= 1u; }
            }
        }
        if (!fine) {   // given up: the copies in flight end before the block does (block 1's complete at block 0: it waits 16 ms)
            if (rank == 0) {
                for (int64_t v = u > Sh::stages ? u - Sh::stages : 0; v < u; ++v)
                    for (int i = 0; i < (1 << 20) && !cafe_bar_try(full((int)(v % Sh::stages)), (uint32_t)(v / Sh::stages) & 1u); ++i) {}
            } else
                for (int i = 0; i < (1 << 14); ++i) __nanosleep(1000);
        }
    } else if (warp == 1 && rank == 1) {
        // (block 0 issues)
    } else if (warp == 1) {
        // ---- products
        bool fine = true;
        int s = 0, n = 0;
        uint32_t phase = 0, chunk_phase = 0;
        for (; n < list.all && fine; ++n) {
            const CafeJob& J = P.job[list.which(n)];
            int t0, t1;
            list.turns<L::BK>(P, n, &t0, &t1);
            const int turns = t1 - t0;
            const uint32_t instr = cafe_mma_instr(L::type, 256, BN) | (J.a_kc ? 0u : 1u << 15) | (J.b_kc ? 0u : 1u << 16);
            const uint64_t da = J.a_kc ? cafe_operand<Sh::rowb>(base) : cafe_operand_mn(base, L::parts * L::BK * 128);
            const uint64_t db = J.b_kc ? cafe_operand<Sh::rowb>(base + L::parts * Sh::a_part) : cafe_operand_mn(base + L::parts * Sh::a_part, L::parts * L::BK * 128);
            // offsets in 16-byte units: from a part to the next, from 16 k to the next 16
            const uint32_t ap = (J.a_kc ? Sh::a_part : L::BK * 128) >> 4, bp = (J.b_kc ? Sh::b_part : L::BK * 128) >> 4;
            const uint32_t ak = (J.a_kc ? 32 : 2048) >> 4, bk = (J.b_kc ? 32 : 2048) >> 4;
            const int g = n % Sh::sets;
            const uint32_t sums = tmem + g * Sh::tm_set;
            if (n >= Sh::sets && !(fine = __all_sync(0xffffffffu, cafe_bar_wait<true>(tile_taken(g), (uint32_t)(n / Sh::sets - 1) & 1u, &bail)))) break;
            int in_chunk = 0;
            for (int t = 0; t < turns; ++t) {
                if (!(fine = __all_sync(0xffffffffu, cafe_bar_wait(full(s), phase, &bail)))) break;
                if (L::parts == 3 && in_chunk == 0 && t > 0) {
                    if (!(fine = __all_sync(0xffffffffu, cafe_bar_wait<true>(chunk_taken, chunk_phase, &bail)))) break;
                    chunk_phase ^= 1u;
                }
                cafe_tc_after();
                const uint64_t a = da + (uint32_t)(s * Sh::stage >> 4), b = db + (uint32_t)(s * Sh::stage >> 4);
                const bool ends = in_chunk == CAFE_TILES_CHUNK - 1 && t < turns - 1, low = ends && (t + 1) % CAFE_TILES_LOW == 0;
                if (cafe_elect()) {
#pragma unroll
                    for (int k = 0; k < L::BK / 16; ++k) cafe_mma2(sums, a + ak * k, b + bk * k, instr, in_chunk > 0 || k > 0);
                    if constexpr (L::parts == 3) {
                        if (ends && !low) cafe_mma_commit2(chunk_full);
#pragma unroll
                        for (int q = 0; q < 5; ++q) {
                            constexpr int ia[5] = {0, 1, 1, 0, 2}, ib[5] = {1, 0, 1, 2, 0};
#pragma unroll
                            for (int k = 0; k < L::BK / 16; ++k)
                                cafe_mma2(sums + BN, a + ia[q] * ap + ak * k, b + ib[q] * bp + bk * k, instr, t % CAFE_TILES_LOW > 0 || q > 0 || k > 0);
                        }
                        if (low) cafe_mma_commit2(chunk_full);
                    }
                    cafe_mma_commit2(empty(s));
                }
                ++in_chunk;
                if (L::parts == 3 && in_chunk == CAFE_TILES_CHUNK) in_chunk = 0;
                if (++s == Sh::stages) { s = 0; phase ^= 1u; }
            }
            __syncwarp();
            if (cafe_elect()) cafe_mma_commit2(tile_full(g));
        }
        if (!fine)   // given up: products in flight end before the block does
            for (int i = 0; i < (1 << 20) && !cafe_bar_try<true>(tile_full(n % Sh::sets), (uint32_t)(n / Sh::sets) & 1u); ++i) {}
    } else {
        // ---- sums out of tensor memory and out of the block
        constexpr int W = Sh::cols;
        const int half = (warp - 2) >> 2, rows = (warp & 3) * 32;
        const uint32_t out = base + Sh::stages * Sh::stage + (warp - 2) * Sh::staging, slopes = out + 32 * Sh::out_row;
        const uint32_t lanes = (uint32_t)rows << 16;
        uint32_t chunk_phase = 0;
        bool fine = true;
        if (P.sums) {
            for (int c = blockIdx.x * 256 + (int)threadIdx.x - 64; c < P.gb_cols; c += gridDim.x * 256) {
                float x[4] = {0.f, 0.f, 0.f, 0.f};
                int q = 0;
                for (; q + 4 <= P.sum_rows; q += 4)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] += __ldg(P.sums + (int64_t)(q + i) * P.gb_cols + c);
                for (; q < P.sum_rows; ++q) x[0] += __ldg(P.sums + (int64_t)q * P.gb_cols + c);
                static_cast<T*>(P.gb)[c] = cafe_from_float<T>((x[0] + x[1]) + (x[2] + x[3]));
            }
            __syncwarp();
        }
        // fp32: every tile, the warp's half of the columns; 16 bits: every other tile, all of them
        for (int n = L::parts == 3 ? 0 : half; n < list.all; n += L::parts == 3 ? 1 : 2) {
            const int tile = list.tile(P, n);
            const CafeJob& J = P.job[list.which(n)];
            int t0, t1;
            list.turns<L::BK>(P, n, &t0, &t1);
            const int turns = t1 - t0;
            const int g = n % Sh::sets, tm = tile / J.tiles_n, col0 = (tile - tm * J.tiles_n) * BN + (L::parts == 3 ? half * Sh::mine : 0);
            const int64_t row0 = (int64_t)tm * 256 + rank * 128 + rows;
            const int m = (int)max((int64_t)0, min((int64_t)32, J.rows - row0)), columns = max(0, min(Sh::mine, J.cols - col0));
            const uint32_t from = tmem + g * Sh::tm_set + lanes + (L::parts == 3 ? half * Sh::mine : 0);
            const uint32_t taken = cafe_cluster_map(tile_taken(g), 0);
            if constexpr (L::parts == 3) {
                float acc[Sh::mine];
                auto take = [&](uint32_t at, bool first_sums) {
#pragma unroll
                    for (int c = 0; c < Sh::mine; c += 16) {
                        float v[16];
                        cafe_tm_load16(at + c, v);
                        cafe_tm_wait_load();
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[c + i] = first_sums ? v[i] : acc[c + i] + v[i];
                    }
                };
                auto join = [&]() {   // the other sums
#pragma unroll
                    for (int c = 0; c < Sh::mine; c += 16) {
                        float v[16];
                        cafe_tm_load16(from + BN + c, v);
                        cafe_tm_wait_load();
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[c + i] = cafe_join_sums(acc[c + i], v[i]);
                    }
                };
                const int between = turns > 0 ? (turns - 1) / CAFE_TILES_CHUNK : 0;   // chunks that do not end the tile
                for (int c = 0; c < between && fine; ++c, chunk_phase ^= 1u) {
                    fine = cafe_bar_wait<true>(chunk_full, chunk_phase, &bail);
                    cafe_tc_after();
                    fine = __all_sync(0xffffffffu, fine);
                    if (fine) take(from, c == 0);
                    if (fine && (c + 1) % CAFE_LIN_LOW == 0) join();
                    cafe_tc_before();
                    __syncwarp();
                    if (lane == 0) cafe_bar_arrive_at(cafe_cluster_map(chunk_taken, 0));
                }
                if (fine) fine = cafe_bar_wait<true>(tile_full(g), (uint32_t)(n / Sh::sets) & 1u, &bail);
                cafe_tc_after();
                fine = __all_sync(0xffffffffu, fine);
                if (fine) {
                    take(from, between == 0);
                    join();
                } else {
#pragma unroll
                    for (int i = 0; i < Sh::mine; ++i) acc[i] = __uint_as_float(0x7fffffffu);
                }
                cafe_tc_before();
                __syncwarp();
                if (lane == 0) cafe_bar_arrive_at(taken);
#pragma unroll 1
                for (int h = 0; h < columns; h += W) {
                    switch (h) {
                        case 0: cafe_row_put<0>(acc, out, lane); break;
                        case 32: cafe_row_put<32 % Sh::mine>(acc, out, lane); break;
                        case 64: cafe_row_put<64 % Sh::mine>(acc, out, lane); break;
                        default: cafe_row_put<96 % Sh::mine>(acc, out, lane); break;
                    }
#pragma unroll 1
                    for (int c = 0; c < W; c += 16) {
                        float z[16];
#pragma unroll
                        for (int q = 0; q < 16; q += 4) {
                            const uint4 x = cafe_get16(cafe_staged<128>(out, lane, (c + q) / 4));
                            z[q] = __uint_as_float(x.x); z[q + 1] = __uint_as_float(x.y); z[q + 2] = __uint_as_float(x.z); z[q + 3] = __uint_as_float(x.w);
                        }
                        cafe_row_end<T, Sh::out_row, Sh::slope_row, false>(J, z, col0 + h + c, out, slopes, lane, c);
                    }
                    __syncwarp();
                    const int here = min(W, columns - h);
                    if (P.splits > 1 && list.which(n) == 0)
                        cafe_rows_out<float, W>(out, P.partial + ((int64_t)list.part(P, n) * J.rows + row0) * P.pitch + col0 + h, P.pitch, true, nullptr, 0, false, m,
                                                min(W, P.pitch - col0 - h), lane);
                    else
                    cafe_rows_out<T, W>(out, static_cast<T*>(J.out) + row0 * J.ldo + col0 + h, J.ldo, J.out_row,
                                        J.res ? static_cast<const T*>(J.res) + row0 * J.ldr + col0 + h : nullptr, J.ldr, J.res_row, m, here, lane);
                    if (J.slope_out)
                        cafe_rows_out<ST, W>(slopes, static_cast<ST*>(J.slope_out) + row0 * J.lds + col0 + h, J.lds, J.slope_row, (const ST*)nullptr, 0, 0, m, here, lane);
                    __syncwarp();   // the staging rows are free
                }
            } else {
                // the residual's rows lie in the staging rows before the results do
                auto residual = [&](int h) {
                    if (!J.res) return;
                    cafe_rows_in<T, W>(out, static_cast<const T*>(J.res) + row0 * J.ldr + col0 + h, J.ldr, J.res_row, m, min(W, J.cols - col0 - h), lane);
                    asm volatile("cp.async.commit_group;" ::: "memory");
                };
                residual(0);
                if (fine) fine = cafe_bar_wait<true>(tile_full(g), (uint32_t)(n / Sh::sets) & 1u, &bail);
                cafe_tc_after();
                fine = __all_sync(0xffffffffu, fine);
#pragma unroll 1
                for (int h = 0; h < columns; h += W) {
                    if (J.res) asm volatile("cp.async.wait_group 0;" ::: "memory");
                    __syncwarp();
#pragma unroll 1
                    for (int c = 0; c < W; c += 16) {
                        float z[16];
                        cafe_tm_load16(from + h + c, z);
                        cafe_tm_wait_load();
                        if (!fine) {
#pragma unroll
                            for (int q = 0; q < 16; ++q) z[q] = __uint_as_float(0x7fffffffu);
                        }
                        cafe_row_end<T, Sh::out_row, Sh::slope_row, true>(J, z, col0 + h + c, out, slopes, lane, c);
                    }
                    if (h + W >= columns) {   // tensor memory has been read
                        cafe_tc_before();
                        __syncwarp();
                        if (lane == 0) cafe_bar_arrive_at(taken);
                    }
                    __syncwarp();
                    const int here = min(W, columns - h);
                    cafe_rows_out<T, W>(out, static_cast<T*>(J.out) + row0 * J.ldo + col0 + h, J.ldo, J.out_row, (const T*)nullptr, 0, 0, m, here, lane);
                    if (J.slope_out)
                        cafe_rows_out<ST, W>(slopes, static_cast<ST*>(J.slope_out) + row0 * J.lds + col0 + h, J.lds, J.slope_row, (const ST*)nullptr, 0, 0, m, here, lane);
                    __syncwarp();   // the staging rows are free
                    if (h + W < columns) residual(h + W);
                }
            }
        }
        if (!fine) g_tiles_gave_up = 1;
    }
    cafe_tc_before();
    __syncthreads();
    cafe_cluster_sync();   // all of the pair's products are done and taken
    cafe_tc_after();
    if (warp == 1) cafe_tm_free2(tmem, Sh::sets * Sh::tm_set);
    cafe_cluster_sync();
}

// ---- host ----------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled tiles_encoder() {
    static const EncodeTiled f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) p = nullptr;
        return (EncodeTiled)p;
    }();
    return f;
}

// The encoder asks for the calling thread's context, which a thread that has not called the runtime yet (the autograd engine's in its
// first backward) does not have: setting the device that is current anyway makes it.
static cudaError_t tiles_ready() {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaSetDevice(device);
    return e != cudaSuccess ? e : tiles_encoder() ? cudaSuccess : cudaErrorNotSupported;
}

// an operand as the copies see it: rows x cols (cols contiguous), `parts` planes
struct TilesOperand {
    const void* at;
    int64_t pitch, plane;
    int rows, cols;
};
// `kc`: cols is the depth
template <typename T>
static bool tiles_map(CUtensorMap* map, const TilesOperand& o, int kc, int box) {
    typedef CafeTiles<T> L;
    const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)L::parts};
    const cuuint64_t strides[2] = {(cuuint64_t)o.pitch * 2, (cuuint64_t)(L::parts == 1 ? o.pitch : o.plane) * 2};
    const cuuint32_t boxes[3] = {(cuuint32_t)(kc ? L::BK : 64), (cuuint32_t)(kc ? box : L::BK), (cuuint32_t)L::parts}, steps[3] = {1, 1, 1};
    const CUtensorMapDataType type = L::type ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUtensorMapSwizzle sw = kc && L::BK == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    return tiles_encoder()(map, type, 3, const_cast<void*>(o.at), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int BN, bool HOLD>
static cudaError_t tiles_launch_bn(CafeTilesArgs& P, const TilesOperand& a, const TilesOperand& b, cudaStream_t st) {
    // (a bias gradient alone: no columns, no depth, nothing fetched)
    if (P.job.depth > 0 && (!tiles_map<T>(&P.a, a, P.job.a_kc, CAFE_LIN_BM) || !tiles_map<T>(&P.b, b, P.job.b_kc, BN))) return cudaErrorInvalidValue;
    P.job.tiles_n = P.job.cols > 0 ? (P.job.cols + BN - 1) / BN : 1;
    P.job.tiles = ((P.job.rows + CAFE_LIN_BM - 1) / CAFE_LIN_BM) * P.job.tiles_n;
    constexpr int bytes = CafeTilesShape<T, BN>::bytes;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = dense_allow_shared((const void*)k_tiles<T, BN, HOLD>, bytes, &allowed);
    if (e != cudaSuccess) return e;
    return dense_start<false>(k_tiles<T, BN, HOLD>, dim3((unsigned)(P.job.tiles * P.splits)), CAFE_TILES_THREADS, bytes, P.splits, st, P);
}
// One product of a call: its job, its operands, and for gW where the bias gradient's partial sums are
struct TilesProduct {
    CafeJob job;
    TilesOperand a, b;
    int splits;         // parts of the depth whose sums go to `partial` first (pairs of blocks, fp32; else 1)
    float* partial;
};
struct TilesSums {
    const float* at;
    int rows, cols;
    void* gb;
};
// what a pair's tile of a product takes, in the units of the estimates below
template <typename T> static double tiles_pair_cost(const CafeJob& J, int bn, int splits) {
    return (CafeTiles<T>::parts == 3 ? 1.2 : bn == 256 ? 2.7 : 2.2) * (((J.depth + CafeTiles<T>::BK - 1) / CafeTiles<T>::BK + splits - 1) / splits) + 3;
}
// Parts of the depth of a product that has so few tiles that clusters of eight blocks each leave SMs idle (gW of a narrow layer): two
// rounds of all pairs, each part at least 32 turns and none empty.  fp32.  Backward of 47373x572x175 425 us without, 345 with;
// 30000x256x256 212, 148; 4096x352x1024 (12 tiles) 79, 73; but 65536x479x1024 (16) 892, 962.  From 13 to 20 tiles at 2048 to 65 536 rows there
// is no rule: without and with, 15 tiles (768x640) 62, 42 at 2048 and 222, 219 at 16 384; 16 (1024x512) 61, 56 and 228, 290; 20
// (1024x640) 45, 69 and 292, 283.
static int tiles_splits(int rows, int cols, int depth) {
    const int64_t tiles = (int64_t)((rows + 255) / 256) * ((cols + 127) / 128), turns = (depth + 31) / 32;
    if (tiles > 12) return 1;
    int64_t s = 2 * CAFE_PAIRS / tiles;
    if (s > turns / 32) s = turns / 32;
    while (s > 1 && ((turns + s - 1) / s) * (s - 1) >= turns) --s;
    return s > 1 ? (int)s : 1;
}
static int64_t tiles_partial_bytes(int rows, int cols, int splits) { return splits > 1 ? (((int64_t)splits * rows * ((cols + 3) & ~3) * 4 + 255) & ~(int64_t)255) : 0; }
// The second product's tiles handed out to the pairs that have the first one's in turn: the least time in which all are done (by
// bisection), and who has how many (share may be null).
static double tiles_share(int64_t tiles0, double cost0, int64_t tiles1, double cost1, int pairs, int* share) {
    double lo = 0, hi = cost0 * (double)((tiles0 + pairs - 1) / pairs) + cost1 * (double)((tiles1 + pairs - 1) / pairs);
    auto room = [&](double t, int p) {
        const double left = t - cost0 * (double)(tiles0 > p ? (tiles0 - p + pairs - 1) / pairs : 0);
        return left > 0 ? (int64_t)(left / cost1 + 1e-9) : 0;
    };
    for (int i = 0; i < 24; ++i) {
        const double t = 0.5 * (lo + hi);
        int64_t n = 0;
        for (int p = 0; p < pairs; ++p) n += room(t, p);
        if (n >= tiles1) hi = t; else lo = t;
    }
    if (share) {
        int64_t at = 0;
        for (int p = 0; p < pairs; ++p) {
            share[p] = (int)at;
            at += room(hi, p);
            at = at > tiles1 ? tiles1 : at;
        }
        share[pairs] = (int)tiles1;   // (room for all by construction)
    }
    const double first = cost0 * (double)((tiles0 + pairs - 1) / pairs);
    return hi > first ? hi : first;
}
template <typename T, int BN>
static cudaError_t tiles_launch_pair(TilesProduct* q, int count, const TilesSums& sums, cudaStream_t st) {
    CafePairArgs P = {};
    P.count = count;
    P.splits = q[0].splits; P.partial = q[0].partial; P.pitch = (q[0].job.cols + 3) & ~3;
    int tiles = 0;
    for (int i = 0; i < count; ++i) {
        CafeJob& J = q[i].job;
        if (!tiles_map<T>(&P.a[i], q[i].a, J.a_kc, CAFE_LIN_BM) || !tiles_map<T>(&P.b[i], q[i].b, J.b_kc, BN / 2)) return cudaErrorInvalidValue;
        J.tiles_n = (J.cols + BN - 1) / BN;
        J.tiles = ((J.rows + 255) / 256) * J.tiles_n;
        tiles += J.tiles * (i ? 1 : P.splits);
        P.job[i] = J;
    }
    const int pairs = tiles < CAFE_PAIRS ? tiles : CAFE_PAIRS;
    P.sums = sums.at; P.sum_rows = sums.rows; P.gb_cols = sums.cols; P.gb = sums.gb;
    if (count == 2)
        tiles_share(P.job[0].tiles * P.splits, tiles_pair_cost<T>(P.job[0], BN, P.splits), P.job[1].tiles, tiles_pair_cost<T>(P.job[1], BN, 1), pairs, P.share);
    constexpr int bytes = CafePairShape<T, BN>::bytes;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = dense_allow_shared((const void*)k_tiles_pair<T, BN>, bytes, &allowed);
    if (e != cudaSuccess) return e;
    const cudaError_t r = dense_start<true>(k_tiles_pair<T, BN>, dim3(2u * pairs), CAFE_PAIR_THREADS, bytes, 2, st, P);
    if (r != cudaSuccess || P.splits == 1) return r;
    const CafeJob& J = P.job[0];
    return dense_start<false>(k_parts_join, dim3((unsigned)(((int64_t)J.rows * P.pitch / 4 + 255) / 256)), 256, 0, 1, st, (const float*)P.partial, P.splits, J.rows,
                              J.cols, P.pitch, (float*)J.out, J.ldo);
}
// Whether the sums of a product are held in registers by k_tiles
template <typename T> static bool tiles_held(int depth) { return CafeTiles<T>::parts == 3 || depth > 8ll * cafe_tiles_depth<T>(); }
// Pairs of blocks through tile after tile, or two blocks an SM and clusters that share a tile's depth: whichever estimate is less,
// in turns of a 128 x 128 tile at the tensor cores' full rate.  A pair's turn takes 1.2 (fp32) or, 256 columns wide, 2.7 (16 bits)
// of these, a tile 3 more and a launch 14; two blocks on an SM share its tensor cores and wait for their boxes, 2.7 (fp32) or 3.3 a
// turn of 128 columns each, and cost 14 a tile, one alone 1.7 or 2.  (Measured both ways: 4096x4096x4096 bf16 pairs 105 us, clusters
// 129; 2048x1024x1024 bf16 24.6 and 22.6; 65536x479x1024 fp32 364 and 433; 2048x1024x512 fp32 40 and 36.)  296, 296, 284 and 264
// blocks run at a time in clusters of 1, 2, 4 and 8 (what the device says).
template <typename T> static double tiles_estimate_clusters(const CafeJob& J, int* splits) {
    constexpr bool split = CafeTiles<T>::parts == 3;
    const bool hold = tiles_held<T>(J.depth);
    const int bn = !split && !hold && J.cols > 128 ? 256 : 128;
    const int64_t tiles = (int64_t)((J.rows + CAFE_LIN_BM - 1) / CAFE_LIN_BM) * (J.cols > 0 ? (J.cols + bn - 1) / bn : 1);
    const int turns = (J.depth + CafeTiles<T>::BK - 1) / CafeTiles<T>::BK;
    static const int room[4] = {296, 296, 284, 264};
    double best = 1e300;
    for (int s = 0; s < 4; ++s) {
        if (!hold && ((turns + (1 << s) - 1) >> s) * (int64_t)CafeTiles<T>::BK > cafe_tiles_depth<T>()) continue;
        const int64_t blocks = tiles << s, rounds = (blocks + room[s] - 1) / room[s];
        const double est = (double)rounds * ((blocks > 148 ? split ? 2.7 : 3.3 : split ? 1.7 : 2.0) * (bn / 128) * ((turns + (1 << s) - 1) >> s) + 14 + s);
        if (est < best * 0.999) { best = est; *splits = 1 << s; }
    }
    return best;
}
template <typename T> static double tiles_estimate_pairs(const TilesProduct* q, int count, int bn) {
    double cost[2], join = 0;
    int64_t tiles[2];
    for (int i = 0; i < count; ++i) {
        const CafeJob& J = q[i].job;
        if (J.depth == 0 || J.cols == 0 || J.depth > cafe_tiles_depth<T>()) return 1e300;
        const int splits = q[i].splits;
        cost[i] = tiles_pair_cost<T>(J, bn, splits);
        tiles[i] = (int64_t)((J.rows + 255) / 256) * ((J.cols + bn - 1) / bn) * splits;
        if (splits > 1) join += 8 + 1e-6 * splits * J.rows * J.cols;
    }
    if (count == 1) return (double)((tiles[0] + CAFE_PAIRS - 1) / CAFE_PAIRS) * cost[0] + 14 + join;
    return tiles_share(tiles[0], cost[0], tiles[1], cost[1], CAFE_PAIRS, nullptr) + 14 + join;
}
template <typename T>
static cudaError_t tiles_launch_clusters(const TilesProduct& q, int splits, const TilesSums& sums, cudaStream_t st) {
    CafeTilesArgs P = {};
    P.job = q.job;
    P.splits = splits;
    P.sums = sums.at; P.sum_rows = sums.rows;
    if constexpr (CafeTiles<T>::parts == 3 || CAFE_TILES_ROWS > 8ll * cafe_tiles_depth<T>()) {   // (no others are that deep)
        if (tiles_held<T>(q.job.depth)) return tiles_launch_bn<T, 128, true>(P, q.a, q.b, st);
    }
    if constexpr (CafeTiles<T>::parts == 1) return q.job.cols > 128 ? tiles_launch_bn<T, 256, false>(P, q.a, q.b, st) : tiles_launch_bn<T, 128, false>(P, q.a, q.b, st);
    return cudaErrorNotSupported;
}
// `count` products; the partial sums, if any, belong to the first
template <typename T>
static cudaError_t tiles_launch(TilesProduct* q, int count, const TilesSums& sums, cudaStream_t st) {
    const TilesSums none = {};
    bool wide = false;
    if constexpr (CafeTiles<T>::parts == 1)
        for (int i = 0; i < count; ++i) wide |= q[i].job.cols > 128;
    const int bn = wide ? 256 : 128;
    double apart = 0, each[2];
    int splits[2];
    for (int i = 0; i < count; ++i) {
        const double c = tiles_estimate_clusters<T>(q[i].job, &splits[i]), p = tiles_estimate_pairs<T>(q + i, 1, bn);
        each[i] = p;
        apart += c < p ? c : p;
        if (c < p) each[i] = 1e300;
    }
    auto pair = [&](TilesProduct* p, int n, const TilesSums& s) {
        if constexpr (CafeTiles<T>::parts == 1) {
            if (wide) return tiles_launch_pair<T, 256>(p, n, s, st);
        }
        return tiles_launch_pair<T, 128>(p, n, s, st);
    };
    // (longer tiles first, but the parts are always the first product's)
    if (count == 2 && q[0].splits == 1 && q[1].job.depth > q[0].job.depth) {
        TilesProduct t[2] = {q[1], q[0]};
        if (tiles_estimate_pairs<T>(t, 2, bn) < apart) return pair(t, 2, sums);
    } else if (count == 2 && tiles_estimate_pairs<T>(q, 2, bn) < apart) return pair(q, 2, sums);
    for (int i = 0; i < count; ++i) {
        const cudaError_t e = each[i] < 1e300 ? pair(q + i, 1, i ? none : sums) : tiles_launch_clusters<T>(q[i], splits[i], i ? none : sums, st);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

static int64_t tiles_round(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }
static int64_t tiles_pitch(int cols) { return (cols + 7) & ~7; }
static int64_t tiles_bytes(int parts, int rows, int cols) { return tiles_round((int64_t)parts * rows * tiles_pitch(cols) * 2); }
// (one row that stands for all, pitch 0, is laid out like any other that copies cannot read)
static bool tiles_in_place(int dtype, const void* p, int64_t ld, int cols) { return dtype != CAFE_F32 && ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld >= cols; }

// an operand: in place, or laid out at *work by a job of the next k_parts launch
template <typename T>
static TilesOperand tiles_operand(CafeParts* P, char** work, int dtype, const void* src, int64_t ld, int rows, int cols, const void* slope, int64_t lds,
                                  int kind, float* sums) {
    typedef CafeTiles<T> L;
    const bool in_place = kind == CAFE_SLOPE_NONE && tiles_in_place(dtype, src, ld, cols);
    TilesOperand o = {src, ld, 0, rows, cols};
    if (in_place && !sums) return o;
    CafePartsJob& J = P->job[P->count++];
    J.src = src; J.slope = slope; J.ld = ld; J.lds = lds; J.kind = kind;
    J.vec = ((uintptr_t)src & 15) == 0 && ld * (int64_t)sizeof(T) % 16 == 0;
    const int ss = kind == CAFE_SLOPE_VALUES ? (int)sizeof(typename CafeSlopeOf<T>::type) : (int)sizeof(T);
    J.slope_vec = ((uintptr_t)slope & 15) == 0 && lds * ss % 16 == 0;
    J.rows = rows; J.cols = cols; J.sums = sums;
    J.blocks_x = (cols + CAFE_PARTS_COLS - 1) / CAFE_PARTS_COLS;
    J.blocks = J.blocks_x * ((rows + cafe_parts_rows(rows, cols) - 1) / cafe_parts_rows(rows, cols));
    J.dst = nullptr;
    if (!in_place) {
        J.dst = *work;
        J.pitch = o.pitch = tiles_pitch(cols);
        J.plane = o.plane = (int64_t)rows * J.pitch;
        o.at = *work;
        *work += tiles_bytes(L::parts, rows, cols);
    }
    return o;
}
template <typename T>
static cudaError_t tiles_parts(const CafeParts& P, cudaStream_t st) {
    int blocks = 0;
    for (int q = 0; q < P.count; ++q) blocks += P.job[q].blocks;
    if (blocks == 0) return cudaSuccess;
    return dense_start<false>(k_parts<T>, dim3((unsigned)blocks), 256, 0, 1, st, P);
}

// Which calls: products of at least so many multiply-adds (the two of a backward share what is laid out: 1777x367x511 in fp16 forward
// 28 us by this file, 21 by dense_cuda.cu's kernel, backward 45 and 50) that are no narrow strips.
#define CAFE_TILES_LEAST (1ll << 29)
#define CAFE_TILES_LEAST_BACK (1ll << 27)
static bool tiles_large(int M, int N, int K, int64_t least) {
    return (int64_t)M * N * K >= least && M >= 128 && N >= 64 && K >= 64 && M <= CAFE_TILES_ROWS && N <= 1 << 17 && K <= 1 << 17;
}

int64_t cafe_tiles_forward_work(const CafeForward& f, int dtype) {
    if (!tiles_large(f.M, f.N, f.K, CAFE_TILES_LEAST)) return 0;
    const int parts = dtype == CAFE_F32 ? 3 : 1;
    return 256 + (tiles_in_place(dtype, f.x, f.ldx, f.K) ? 0 : tiles_bytes(parts, f.M, f.K)) + (tiles_in_place(dtype, f.w, f.ldw, f.K) ? 0 : tiles_bytes(parts, f.N, f.K));
}
int64_t cafe_tiles_backward_work(const CafeBackward& f, int dtype) {
    if (!tiles_large(f.M, f.N, f.K, CAFE_TILES_LEAST_BACK) || (!f.gx && !f.gw)) return 0;
    const int parts = dtype == CAFE_F32 ? 3 : 1;
    int64_t need = 256;
    if (f.slope_kind != CAFE_SLOPE_NONE || !tiles_in_place(dtype, f.gy, f.ldg, f.N)) need += tiles_bytes(parts, f.M, f.N);
    if (f.gx && !tiles_in_place(dtype, f.w, f.ldw, f.K)) need += tiles_bytes(parts, f.N, f.K);
    if (f.gw && !tiles_in_place(dtype, f.x, f.ldx, f.K)) need += tiles_bytes(parts, f.M, f.K);
    if (f.gw && dtype == CAFE_F32) need += tiles_partial_bytes(f.N, f.K, tiles_splits(f.N, f.K, f.M));
    if (f.gb) need += tiles_round((int64_t)((f.M + cafe_parts_rows(f.M, f.N) - 1) / cafe_parts_rows(f.M, f.N)) * f.N * 4);
    return need;
}

template <typename T>
static cudaError_t tiles_forward(const CafeForward& f, int dtype, const CafeJob& job, char* work, cudaStream_t st) {
    CafeParts parts = {};
    const TilesOperand x = tiles_operand<T>(&parts, &work, dtype, f.x, f.ldx, f.M, f.K, nullptr, 0, CAFE_SLOPE_NONE, nullptr);
    const TilesOperand w = tiles_operand<T>(&parts, &work, dtype, f.w, f.ldw, f.N, f.K, nullptr, 0, CAFE_SLOPE_NONE, nullptr);
    cudaError_t e = tiles_parts<T>(parts, st);
    if (e != cudaSuccess) return e;
    TilesProduct q = {job, x, w, 1, nullptr};
    return tiles_launch<T>(&q, 1, TilesSums{}, st);
}
template <typename T>
static cudaError_t tiles_backward(const CafeBackward& f, int dtype, const CafeJob* gw, const CafeJob* gx, char* work, cudaStream_t st) {
    CafeParts parts = {};
    float* sums = nullptr;
    const int sum_rows = (f.M + cafe_parts_rows(f.M, f.N) - 1) / cafe_parts_rows(f.M, f.N);
    if (f.gb) {
        sums = (float*)work;
        work += tiles_round((int64_t)sum_rows * f.N * 4);
    }
    const TilesOperand g = tiles_operand<T>(&parts, &work, dtype, f.gy, f.ldg, f.M, f.N, f.slope, f.lds, f.slope_kind, sums);
    TilesOperand w = {}, x = {};
    if (gx) w = tiles_operand<T>(&parts, &work, dtype, f.w, f.ldw, f.N, f.K, nullptr, 0, CAFE_SLOPE_NONE, nullptr);
    if (f.gw) x = tiles_operand<T>(&parts, &work, dtype, f.x, f.ldx, f.M, f.K, nullptr, 0, CAFE_SLOPE_NONE, nullptr);
    cudaError_t e = tiles_parts<T>(parts, st);
    if (e != cudaSuccess) return e;
    TilesProduct q[2];
    int count = 0;
    if (gw) {   // (without gW wanted: no columns, no depth, the bias gradient alone)
        const int splits = f.gw && dtype == CAFE_F32 ? tiles_splits(f.N, f.K, f.M) : 1;
        q[count] = {*gw, g, x, splits, (float*)work};
        work += tiles_partial_bytes(f.N, f.K, splits);
        if (!f.gw) q[count].job.depth = 0;
        ++count;
    }
    if (gx) q[count++] = {*gx, g, w, 1, nullptr};
    return tiles_launch<T>(q, count, f.gb ? TilesSums{sums, sum_rows, f.N, f.gb} : TilesSums{}, st);
}
cudaError_t cafe_tiles_forward(const CafeForward& f, int dtype, const CafeJob& job, void* work, cudaStream_t st) {
    const cudaError_t e = tiles_ready();
    if (e != cudaSuccess) return e;
    char* const at = (char*)(((uintptr_t)work + 255) & ~(uintptr_t)255);
    return dtype == CAFE_F32 ? tiles_forward<float>(f, dtype, job, at, st)
                             : dtype == CAFE_BF16 ? tiles_forward<__nv_bfloat16>(f, dtype, job, at, st) : tiles_forward<__half>(f, dtype, job, at, st);
}
cudaError_t cafe_tiles_backward(const CafeBackward& f, int dtype, const CafeJob* gw, const CafeJob* gx, void* work, cudaStream_t st) {
    const cudaError_t e = tiles_ready();
    if (e != cudaSuccess) return e;
    char* const at = (char*)(((uintptr_t)work + 255) & ~(uintptr_t)255);
    return dtype == CAFE_F32 ? tiles_backward<float>(f, dtype, gw, gx, at, st)
                             : dtype == CAFE_BF16 ? tiles_backward<__nv_bfloat16>(f, dtype, gw, gx, at, st) : tiles_backward<__half>(f, dtype, gw, gx, at, st);
}
