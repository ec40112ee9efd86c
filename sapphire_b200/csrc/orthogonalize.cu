// Orthogonalised update of a matrix (Newton-Schulz products):
//
//   X = G / (|G|_F + eps), then `steps` times
//   A = X X^T,   B = b A + c A A,   X = a X + B X
//
// on the shorter side of G (a tall G is worked on transposed, so X is R x C with R <= C).
//
// All products run on the tensor cores with fp16 operands and fp32 accumulators.  The
// singular values of every matrix in the iteration are bounded (the host checks the
// bound for the given coefficients), so the matrices are kept as fp16 numbers scaled by
// 2^13, which cannot overflow and keeps small entries out of the subnormal range.
//
//   fp32 and fp16 input: every matrix is a sum of two fp16 parts, hi = fp16(x) and
//     lo = fp16(x - hi), 22 bits of mantissa.  A product is hi.lo + lo.hi + hi.hi, three
//     tensor-core products at the fp16 rate (a product of two TF32 parts would run at half
//     of it).  The tensor core cuts its fp32 accumulation short instead of rounding it,
//     so a chain of accumulations ends after CHUNK_KB k-blocks and the chains are added
//     in registers.  a X is added in the epilogue: inside the chains it would triple
//     their error.
//   bf16 input (both sides longer than 128): the products take the hi parts alone (11 bits; the result keeps 8), with
//     X = (a + B) hi + a lo: a stands on the diagonal of B, which saves reading hi again.
//     X has both parts because rounding X itself every step would feed the small singular
//     directions, which a step multiplies by a, with the rounding errors of the large ones.
//     Why one part: the three roundings a step (of X, A and B; each adds about as much) leave
//     the result off by 0.6e-3 to 1.2e-3 (2-norm), less than its own rounding to bf16, 1.66e-3;
//     together 1.78e-3 to 2.07e-3 where two parts, and fp32 arithmetic, give 1.66e-3.  Two parts
//     take three products: 1.02 ms instead of 0.47 for 4 x 1024 x 4096, 3.64 instead of 1.28 for
//     4096 x 4096, 157 us instead of 121 for 2 x 153 x 188.  Dropping one of the roundings alone
//     saves little of the error.  Who needs more than this has the fp32 call.
//
// Five steps take 150 us for 784 x 512 fp32, 470 to 505 us for 4 x 1024 x 4096 bf16 and 3.6 to
// 3.8 ms for 4096 x 4096 fp32, by box (1375 GFLOP in triangles, 362 to 382 TFLOP/s, three times
// that as fp16 products).
//
// A and A A are symmetric: only tiles on and above the diagonal are computed, and a tile
// above it is also stored transposed.  X X^T and A A read both operands along k; B X reads
// X in rows of k ("MN-major"), so no matrix is ever transposed in memory.
#include <cmath>
#include <type_traits>

#include "gemm_common.cuh"
#include "orthogonalize.cuh"

namespace sb200 {

using namespace gemm;

namespace {

constexpr int KB = 64;                           // fp16 elements of k per block: one 128-byte swizzle row
constexpr int MMA_K = 16;
constexpr int TILE_BYTES = 128 * KB * 2;         // 128 rows (or columns) x 64 k
constexpr int MN_CHUNK_BYTES = 64 * KB * 2;      // MN-major: 64 k rows x 64 columns
constexpr int CHUNK_KB = 2;                      // k-blocks per accumulation chain with two parts (1 in the sliced kernel)
constexpr int LONG_CHAIN_KB = 64;                // of X X^T with one part: 256 accumulations lose 2.4e-5 of a sum of positive terms
constexpr float SCALE = ORTH_SCALE, INV_SCALE = ORTH_INV_SCALE;
constexpr double LARGEST = 7.5;                  // of a singular value: 7.5 * 2^13 < 65504
constexpr int EPI_WARPS = 16;
constexpr int THREADS = 64 + EPI_WARPS * 32;
constexpr int NORM_BLOCKS = 512;                 // partial sums of squares per matrix
constexpr int ORTH_PANEL = 8;
constexpr int MAX_SLICES = 8;
constexpr int PART_LD = 132;                     // floats per row of a partial tile in shared memory

enum Product { GRAM, POLY, APPLY, LONG_GRAM };   // LONG_GRAM: X X^T in chains of LONG_CHAIN_KB (one part, pairs)

// A matrix of the iteration: [parts][batch][rows][ld] fp16, part 0 = hi, 1 = lo.
struct Split {
    f16* p;
    int64_t ld, batch_stride, part_stride;
};

struct OrthParams {
    int R, C, batch;
    int rows, cols, num_kb;                      // of the product
    int tiles_m, tiles_n, tiles;                 // per matrix
    int chunk_kb, slices;
    Split prev, out;                             // prev: added with `coef`; out: the result
    int out_parts;
    float coef, alpha, diagonal;                 // result = diagonal + coef * prev + alpha * accumulator (scaled by 2^13)
    void* final_out;                             // APPLY, last step: the caller's matrix
    int64_t final_ld, final_stride;
    int final_type, tall, final_vec;
    unsigned* status;
    unsigned long long wait_limit_ns;
    int test_stall_kb;
};

// The epilogue of the pair kernel moves blocks of 32 rows through shared memory (their
// 16-byte pieces permuted against bank conflicts): a thread owns a row of the accumulator,
// and 32 rows a warp touched with plain 16-byte accesses cost 32 cycles of the load/store
// unit each (an epilogue of 24 us where the products take 5); through shared memory the
// lanes of a row share it.  TMA would do the same, but it is what feeds the tensor core:
// blocks moved by TMA made the operand tiles late (9.6 us a tile).  Sixteen warps, because
// the work is a chain of short latencies (eight took twice as long), in a loop that is not
// unrolled over the blocks, because code that runs once a tile misses the instruction cache.
template <bool SPLIT>
struct OrthSmem {
    static constexpr int PARTS = SPLIT ? 2 : 1;
    static constexpr int STAGE = 2 * PARTS * TILE_BYTES;
    static constexpr int STAGES = SPLIT ? 3 : 5;
    static constexpr int TILES = STAGE * STAGES;
    static constexpr int BW = SPLIT ? 16 : 32;   // columns of an epilogue block
    static constexpr int EPI_PART = 32 * BW * 2; // one part of a block
    static constexpr int EPI_BUF = 2 * EPI_PART; // one per warp
    static constexpr int EPI = EPI_WARPS * EPI_BUF;
    static constexpr int BARS = ((2 * STAGES + 4) * 8 + 16 + 15) & ~15;
    static constexpr int TOTAL = TILES + EPI + BARS + 1024;
    static_assert(TOTAL <= 227 * 1024, "shared memory per CTA");
    static_assert(TILES >= 128 * PART_LD * 4 + 128 * 129 * 4, "what the sliced kernel keeps in the place of the stages");
};

// 16-byte piece c of row r of a block with `pieces` of them a row
template <int PIECES>
__device__ __forceinline__ int piece_at(int r, int c)
{
    static_assert(PIECES == 2 || PIECES == 4 || PIECES == 8, "rows of 32, 64 or 128 bytes");
    return r * PIECES + (PIECES == 8 ? c ^ (r & 7) : PIECES == 4 ? c ^ ((r >> 1) & 3) : c ^ ((r >> 2) & 1));
}

// Tile t of a matrix; symmetric products walk over the tiles with tn >= tm only.
__device__ __forceinline__ void orth_tile(int t, const OrthParams& p, bool symmetric, int& tm, int& tn)
{
    if (!symmetric) {
        tile_coords(t, p.tiles_m, p.tiles_n, ORTH_PANEL, tm, tn);
        return;
    }
    int row = 0, len = p.tiles_n;
    while (t >= len) {
        t -= len;
        ++row;
        --len;
    }
    tm = row;
    tn = row + t;
}

__device__ __forceinline__ void store_transposed(const Raw<f16, 8>& hi, const Raw<f16, 8>& lo, f16* out, const Split& m,
                                                 int parts, int row, int col, int cols)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (col + e < cols) {                    // lanes hold neighbouring rows: contiguous in the output
            f16* o = out + static_cast<int64_t>(col + e) * m.ld + row;
            *o = hi.e[e];
            if (parts == 2) o[m.part_stride] = lo.e[e];
        }
    }
}

template <typename F>
__device__ __forceinline__ void with_final_type(const OrthParams& p, int b, F f)
{
    const int64_t at = b * p.final_stride;
    if (p.final_type == SB200_F32) f(static_cast<float*>(p.final_out) + at);
    else if (p.final_type == SB200_BF16) f(static_cast<bf16*>(p.final_out) + at);
    else f(static_cast<f16*>(p.final_out) + at);
}

// One warp's block of 32 rows x BW columns of the caller's matrix, stored by rows.  v: this
// lane's row.  buf: 128 BW bytes of shared memory nobody else uses.
template <int BW, typename T>
__device__ __forceinline__ void final_block(T* out, const OrthParams& p, uint8_t* buf, int row0, int col0,
                                            const float (&v)[BW])
{
    constexpr int PER = 16 / static_cast<int>(sizeof(T));        // elements of a piece
    constexpr int PIECES = BW / PER;                             // pieces of a row
    const int lane = threadIdx.x & 31;
    T* b = reinterpret_cast<T*>(buf);
    __syncwarp();
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
        float x[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) x[e] = v[c * PER + e];
        store_f<false>(b + piece_at<PIECES>(lane, c) * PER, x);
    }
    __syncwarp();
    if (p.final_vec && col0 + BW <= p.C) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = i * (32 / PIECES) + lane / PIECES, c = lane % PIECES;
            Raw<T, PER> x;
            load_raw<false>(x, b + piece_at<PIECES>(r, c) * PER);
            if (row0 + r < p.R) store_raw<true>(out + static_cast<int64_t>(row0 + r) * p.final_ld + col0 + c * PER, x);
        }
    } else {
#pragma unroll 1
        for (int i = lane; i < 32 * BW; i += 32) {
            const int r = i / BW, c = i % BW;
            if (row0 + r < p.R && col0 + c < p.C)
                out[static_cast<int64_t>(row0 + r) * p.final_ld + col0 + c] = b[piece_at<PIECES>(r, c / PER) * PER + c % PER];
        }
    }
    __syncwarp();
}

// PAIR: a cluster of two CTAs per 256 x 256 tile (cta_group::2), clusters walk over the
// tiles.  Otherwise: a cluster of p.slices CTAs per 128 x 128 tile, each with its slice of
// the k-blocks; the partial tiles meet in shared memory, and each CTA finishes its share
// of the columns.
template <int WHAT, bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
orth_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                    const OrthParams p)
{
    using S = OrthSmem<SPLIT>;
    constexpr bool SYMMETRIC = WHAT != APPLY;
    constexpr bool B_MN = WHAT == APPLY;
    constexpr int CTAS = PAIR ? 2 : 1;
    constexpr int BM = 128 * CTAS, BN = 128 * CTAS;
    constexpr int COLS = BN / (EPI_WARPS / 4);   // accumulator columns of an epilogue warp
    constexpr int BW = S::BW, PIECES = BW / 8;
    constexpr uint32_t TMEM_COLS = 2 * BN;
    // what the epilogue adds to the product: A, and X or its low part alone (see the top)
    constexpr bool READS_HI = WHAT == POLY || (WHAT == APPLY && SPLIT);
    constexpr bool READS_LO = WHAT == APPLY || (WHAT == POLY && SPLIT);

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* epi = smem + S::TILES;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(epi + S::EPI);
    uint64_t* empty_bar = full_bar + S::STAGES;
    uint64_t* tmem_full = empty_bar + S::STAGES;
    uint64_t* tmem_empty = tmem_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_ctarank();
    const Abort ab{abort_flag, p.status, p.wait_limit_ns};

    auto wait = [&](uint64_t* bar, uint32_t parity, unsigned code) {
        if (!PAIR) return wait_bar(bar, parity, ab, code);
        return wait_bar_cluster(bar, parity, ab, code);
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&tmem_full[i], 1);
            ptx::mbar_init(&tmem_empty[i], EPI_WARPS * CTAS);
        }
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&map_a);
        ptx::prefetch_tensormap(&map_b);
    }
    if (warp == 1) {
        if (PAIR) {
            ptx::tmem_alloc_pair(tmem_slot, TMEM_COLS);
            ptx::tmem_relinquish_pair();
        } else {
            ptx::tmem_alloc(tmem_slot, TMEM_COLS);
            ptx::tmem_relinquish();
        }
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (PAIR) ptx::cluster_sync();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();

    const int group = PAIR ? 2 : p.slices;       // CTAs of the cluster
    const int unit = blockIdx.x / group;
    const int units = gridDim.x / group;
    const int total = p.tiles * p.batch;
    // this CTA's k-blocks
    const int per_slice = PAIR ? p.num_kb : (p.num_kb + p.slices - 1) / p.slices;
    const int kb_first = PAIR ? 0 : min(p.num_kb, static_cast<int>(rank) * per_slice);
    const int kb_last = PAIR ? p.num_kb : min(p.num_kb, kb_first + per_slice);
    const uint32_t pair_rank = PAIR ? rank : 0u;

    if (warp == 0) {
        // ------------------------------------------------------ TMA producer
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            int issued = 0;
            for (int t = unit; ok && t < total; t += units) {
                const int b = t / p.tiles;
                int tm, tn;
                orth_tile(t % p.tiles, p, SYMMETRIC, tm, tn);
                const int m0 = tm * BM + static_cast<int>(pair_rank) * 128;
                const int n0 = tn * BN + static_cast<int>(pair_rank) * 128;
                for (int kb = kb_first; kb < kb_last; ++kb) {
                    if (p.test_stall_kb >= 0 && issued++ >= p.test_stall_kb) {
                        ok = false;              // test hook: the other roles' waits run out
                        break;
                    }
                    if (!(ok = wait(&empty_bar[s], ph ^ 1u, FAULT_PRODUCER_WAIT))) break;
                    uint8_t* st = smem + s * S::STAGE;
                    const int k0 = kb * KB;
                    if (pair_rank == 0) ptx::mbar_arrive_expect_tx(&full_bar[s], CTAS * S::STAGE);
                    const uint32_t lead = PAIR ? ptx::map_to_cta(ptx::smem_u32(&full_bar[s]), 0) : 0u;
                    auto load = [&](uint8_t* dst, const CUtensorMap* map, int x, int y, int z) {
                        if (PAIR) ptx::tma_load_3d_pair(dst, map, lead, x, y, z);
                        else ptx::tma_load_3d(dst, map, &full_bar[s], x, y, z);
                    };
#pragma unroll
                    for (int part = 0; part < S::PARTS; ++part) {
                        const int z = part * p.batch + b;
                        uint8_t* sa = st + part * TILE_BYTES;
                        uint8_t* sb = st + (S::PARTS + part) * TILE_BYTES;
                        load(sa, &map_a, k0, m0, z);
                        if (B_MN) {
                            load(sb, &map_b, n0, k0, z);
                            load(sb + MN_CHUNK_BYTES, &map_b, n0 + 64, k0, z);
                        } else {
                            load(sb, &map_b, k0, n0, z);
                        }
                    }
                    if (++s == S::STAGES) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------- MMA issuer (a pair's leader only)
        if (lane == 0 && pair_rank == 0) {
            constexpr uint32_t idesc = ptx::make_idesc_f16(BM, BN, 0, B_MN);
            constexpr uint32_t A_STEP = MMA_K * 2, B_STEP = B_MN ? MMA_K * 128u : MMA_K * 2u;
            constexpr uint32_t B_LBO = B_MN ? MN_CHUNK_BYTES : 16u;
            int s = 0;
            uint32_t ph = 0;
            int acc = 0;
            uint32_t acc_ph = 0;
            bool ok = true;
            for (int t = unit; ok && t < total; t += units) {
                for (int kb0 = kb_first; ok && kb0 < kb_last; kb0 += p.chunk_kb) {
                    if (!(ok = wait(&tmem_empty[acc], acc_ph ^ 1u, FAULT_MMA_WAIT_TMEM))) break;
                    ptx::tc_fence_after_sync();
                    const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
                    const int kb1 = min(kb0 + p.chunk_kb, kb_last);
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (!(ok = wait(&full_bar[s], ph, FAULT_MMA_WAIT_FULL))) break;
                        ptx::tc_fence_after_sync();
                        const uint32_t sa = ptx::smem_u32(smem + s * S::STAGE);
                        const uint32_t sb = sa + S::PARTS * TILE_BYTES;
#pragma unroll
                        for (int pass = 0; pass < (SPLIT ? 3 : 1); ++pass) {
                            // hi.lo, lo.hi, hi.hi: small terms first
                            const uint32_t pa = sa + (SPLIT && pass == 1 ? TILE_BYTES : 0);
                            const uint32_t pb = sb + (SPLIT && pass == 0 ? TILE_BYTES : 0);
#pragma unroll
                            for (int k = 0; k < KB / MMA_K; ++k) {
                                const uint64_t da = ptx::make_smem_desc(pa + k * A_STEP, 16u, 1024u, ptx::LAYOUT_SW128);
                                const uint64_t db = ptx::make_smem_desc(pb + k * B_STEP, B_LBO, 1024u, ptx::LAYOUT_SW128);
                                const uint32_t more = (kb > kb0 || pass > 0 || k > 0) ? 1u : 0u;
                                if (PAIR) ptx::mma_f16_pair(d, da, db, idesc, more);
                                else ptx::mma_f16(d, da, db, idesc, more);
                            }
                        }
                        if (PAIR) ptx::mma_commit_pair(&empty_bar[s], 3);
                        else ptx::mma_commit(&empty_bar[s]);
                        if (++s == S::STAGES) {
                            s = 0;
                            ph ^= 1u;
                        }
                    }
                    if (!ok) break;
                    if (PAIR) ptx::mma_commit_pair(&tmem_full[acc], 3);
                    else ptx::mma_commit(&tmem_full[acc]);
                    acc ^= 1;
                    if (acc == 0) acc_ph ^= 1u;
                }
            }
        }
    } else {
        // ---------------------------------------------------------- epilogue
        // warp w reads TMEM lanes 32 (w % 4) .. + 31 and a quarter of the columns
        const int q = warp & 3, quarter = (warp - 2) >> 2;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(quarter * COLS);
        f16* buf = reinterpret_cast<f16*>(epi + (warp - 2) * S::EPI_BUF);
        f16* buf_lo = buf + S::EPI_PART / 2;
        // by rows: PIECES lanes share a row of a block
        const int by_row = lane / PIECES, by_col = lane % PIECES;
        int acc = 0;
        uint32_t acc_ph = 0;
        bool ok = true;
        auto release = [&]() {                   // this accumulator is read: on to the other
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) ptx::mbar_arrive_cluster(ptx::map_to_cta(ptx::smem_u32(&tmem_empty[acc]), 0));
                else ptx::mbar_arrive(&tmem_empty[acc]);
            }
            acc ^= 1;
            if (acc == 0) acc_ph ^= 1u;
        };
        for (int t = unit; ok && t < total; t += units) {
            const int b = t / p.tiles;
            int tm, tn;
            orth_tile(t % p.tiles, p, SYMMETRIC, tm, tn);
            const int row0 = tm * BM + static_cast<int>(pair_rank) * 128 + q * 32;
            const int col0 = tn * BN + quarter * COLS;
            // blocks of columns this warp has to finish; none where its rows or columns are beyond the matrix
            const int blocks = row0 < p.rows && col0 < p.cols ? min(COLS, p.cols - col0 + BW - 1) / BW : 0;
            const f16* prev = p.prev.p + b * p.prev.batch_stride + static_cast<int64_t>(row0 + by_row) * p.prev.ld + col0 + by_col * 8;
            auto fetch = [&](int i) {            // block i of it, asynchronously
#pragma unroll
                for (int it = 0; it < PIECES; ++it) {
                    const int r = it * (32 / PIECES) + by_row;
                    const int bytes = row0 + r < p.rows ? 16 : 0;        // (the pitch covers whole blocks of columns)
                    const f16* src = prev + (bytes ? static_cast<int64_t>(it * (32 / PIECES)) * p.prev.ld + i * BW : 0);
                    if (READS_HI) ptx::cp_async_16(buf + piece_at<PIECES>(r, by_col) * 8, src, bytes);
                    if (READS_LO) ptx::cp_async_16(buf_lo + piece_at<PIECES>(r, by_col) * 8, src + p.prev.part_stride, bytes);
                }
            };
            if constexpr (PAIR && (READS_HI || READS_LO)) {
                if (blocks > 0) fetch(0);        // travels while the products run
            }
            if (SPLIT || !PAIR || WHAT == LONG_GRAM) {
                // chains of accumulations are added here, rounded to nearest
                float sum[COLS];
#pragma unroll
                for (int j = 0; j < COLS; ++j) sum[j] = 0.0f;
                for (int kb0 = kb_first; kb0 < kb_last; kb0 += p.chunk_kb) {
                    if (!(ok = wait(&tmem_full[acc], acc_ph, FAULT_EPI_WAIT))) break;
                    ptx::tc_fence_after_sync();
#pragma unroll
                    for (int c = 0; c < COLS / 16; ++c) {
                        uint32_t v[16];
                        ptx::tmem_ld_32x16(lane_base + static_cast<uint32_t>(acc * BN + c * 16), v);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) sum[c * 16 + j] = __fadd_rn(sum[c * 16 + j], __uint_as_float(v[j]));
                    }
                    if (PAIR && kb0 + p.chunk_kb >= kb_last) break;
                    release();
                }
                if (!ok) break;
                if constexpr (PAIR) {
                    // the total goes back into the last accumulator, for the loop over the blocks
#pragma unroll
                    for (int c = 0; c < COLS / 16; ++c) {
                        uint32_t v[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(sum[c * 16 + j]);
                        ptx::tmem_st_32x16(lane_base + static_cast<uint32_t>(acc * BN + c * 16), v);
                    }
                    ptx::tmem_st_wait();
                } else {
                    // every role of this CTA is done with the stages (the last product has read
                    // them): the partial tile goes there
                    float* part = reinterpret_cast<float*>(smem) + (q * 32 + lane) * PART_LD + quarter * COLS;
#pragma unroll
                    for (int j = 0; j < COLS; j += 4)
                        *reinterpret_cast<float4*>(part + j) = make_float4(sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
                }
            } else {
                if (!(ok = wait(&tmem_full[acc], acc_ph, FAULT_EPI_WAIT))) break;
                ptx::tc_fence_after_sync();
            }
            if constexpr (!PAIR) continue;       // (one tile a cluster: the rest is below)
            f16* out = p.out.p + b * p.out.batch_stride;
            f16* out_rows = out + static_cast<int64_t>(row0 + by_row) * p.out.ld + col0 + by_col * 8;
            const bool mirror = SYMMETRIC && tn > tm;            // (all rows of such a tile are in the matrix)
#pragma unroll 1
            for (int i = 0; i < blocks; ++i) {
                const int col = col0 + i * BW;
                uint32_t a[BW];
                if constexpr (BW == 32) ptx::tmem_ld_32x32(lane_base + static_cast<uint32_t>(acc * BN + i * BW), a);
                else ptx::tmem_ld_32x16(lane_base + static_cast<uint32_t>(acc * BN + i * BW), a);
                if (READS_HI || READS_LO) {
                    ptx::cp_async_wait_all();
                    __syncwarp();
                }
                ptx::tmem_ld_wait();
                float v[BW];
#pragma unroll
                for (int c = 0; c < PIECES; ++c) {
                    float h[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                    Raw<f16, 8> x;
                    if (READS_LO) {
                        load_raw<false>(x, buf_lo + piece_at<PIECES>(lane, c) * 8);
                        join_f16(h, x);
                    }
                    if (READS_HI) {
                        load_raw<false>(x, buf + piece_at<PIECES>(lane, c) * 8);
                        join_f16(h, x);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float y = __uint_as_float(a[c * 8 + e]) * p.alpha;
                        v[c * 8 + e] = READS_HI || READS_LO ? fmaf(p.coef, h[e], y) : y;
                        if (WHAT == POLY && !SPLIT && row0 + lane == col + c * 8 + e) v[c * 8 + e] += p.diagonal;
                    }
                }
                if (WHAT == APPLY && p.final_out) {
#pragma unroll
                    for (int e = 0; e < BW; ++e) v[e] *= INV_SCALE;
                    with_final_type(p, b, [&](auto* o) {
                        if (p.tall) {
                            if (row0 + lane < p.R) {
#pragma unroll
                                for (int e = 0; e < BW; ++e)
                                    if (col + e < p.C)
                                        o[static_cast<int64_t>(col + e) * p.final_ld + row0 + lane] =
                                            from_f<std::remove_pointer_t<decltype(o)>>(v[e]);
                            }
                        } else {
                            final_block<BW>(o, p, reinterpret_cast<uint8_t*>(buf), row0, col, v);
                        }
                    });
                } else {
                    // in place (a lane reads and writes its own row), then out by rows
#pragma unroll
                    for (int c = 0; c < PIECES; ++c) {
                        Raw<f16, 8> hi, lo;
                        split_f16(v + c * 8, hi, lo);
                        store_raw<false>(buf + piece_at<PIECES>(lane, c) * 8, hi);
                        if (p.out_parts == 2) store_raw<false>(buf_lo + piece_at<PIECES>(lane, c) * 8, lo);
                        if (SYMMETRIC && mirror) store_transposed(hi, lo, out, p.out, p.out_parts, row0 + lane, col + c * 8, p.cols);
                    }
                    __syncwarp();
#pragma unroll
                    for (int it = 0; it < PIECES; ++it) {
                        const int r = it * (32 / PIECES) + by_row;
                        if (row0 + r < p.rows) {
                            f16* o = out_rows + static_cast<int64_t>(it * (32 / PIECES)) * p.out.ld + i * BW;
                            Raw<f16, 8> x;
                            load_raw<false>(x, buf + piece_at<PIECES>(r, by_col) * 8);
                            store_raw<false>(o, x);
                            if (p.out_parts == 2) {
                                load_raw<false>(x, buf_lo + piece_at<PIECES>(r, by_col) * 8);
                                store_raw<!SPLIT>(o + p.out.part_stride, x);
                            }
                        }
                    }
                }
                __syncwarp();
                if ((READS_HI || READS_LO) && i + 1 < blocks) fetch(i + 1);
            }
            release();
        }
    }

    if constexpr (!PAIR) {
        // The slices of a tile meet: CTA r adds its share of the rows of all of them, in slice
        // order.  A warp takes whole rows, so that what crosses between the SMs and what goes
        // to memory are runs of 512 and 256 bytes (a thread a row took 8 us for 64 KB).
        __syncthreads();
        const int share = 128 / p.slices;
        ptx::cluster_sync();
        if (warp >= 2 && *abort_flag == 0) {
            const int b = unit / p.tiles;
            int tm, tn;
            orth_tile(unit % p.tiles, p, SYMMETRIC, tm, tn);
            const int first = static_cast<int>(rank) * share;    // of this CTA's rows
            const int col = tn * BN + lane * 4;
            const bool mirror = SYMMETRIC && tn > tm;
            const bool last = WHAT == APPLY && p.final_out;
            const f16* prev = p.prev.p + b * p.prev.batch_stride + col;
            f16* out = p.out.p + b * p.out.batch_stride;
            // for results that are stored transposed: [128 columns][share rows] of fp32 behind the partial tile
            float* turned = reinterpret_cast<float*>(smem) + 128 * PART_LD;
            const int turned_ld = share + 1;
#pragma unroll 2
            for (int r = warp - 2; r < share; r += EPI_WARPS) {
                const int row = tm * BM + first + r;
                const bool in = row < p.rows && col < p.cols;
                float h[4] = {0.0f, 0.0f, 0.0f, 0.0f}, l[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (in) {                        // rows have a pitch of a multiple of 64: whole vectors fit
                    if (READS_HI) load_f<false>(h, prev + static_cast<int64_t>(row) * p.prev.ld);
                    if (READS_LO) load_f<false>(l, prev + p.prev.part_stride + static_cast<int64_t>(row) * p.prev.ld);
                }
                const uint32_t at = ptx::smem_u32(smem) + static_cast<uint32_t>(((first + r) * PART_LD + lane * 4) * 4);
                float4 x[MAX_SLICES];
#pragma unroll
                for (int s = 0; s < MAX_SLICES; ++s)
                    if (s < p.slices) x[s] = ptx::ld_cluster_f4(ptx::map_to_cta(at, s));
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < MAX_SLICES; ++s) {
                    if (s < p.slices) {          // (a slice without work wrote zeros)
                        v[0] += x[s].x; v[1] += x[s].y; v[2] += x[s].z; v[3] += x[s].w;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] *= p.alpha;
                    if (READS_HI || READS_LO) v[e] = fmaf(p.coef, h[e] + l[e], v[e]);
                    if (WHAT == POLY && !SPLIT && row == col + e) v[e] += p.diagonal;
                    if (last) v[e] *= INV_SCALE;
                }
                Raw<f16, 4> hi, lo;
                split_f16(v, hi, lo);
                if (mirror || (last && p.tall)) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) turned[(lane * 4 + e) * turned_ld + r] = v[e];
                }
                if (!in) continue;
                if (last) {
                    if (!p.tall)
                        with_final_type(p, b, [&](auto* o) {
                            o += static_cast<int64_t>(row) * p.final_ld + col;
                            if (p.final_vec && col + 4 <= p.cols) {
                                store_f<false>(o, v);
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (col + e < p.cols) o[e] = from_f<std::remove_pointer_t<decltype(o)>>(v[e]);
                            }
                        });
                    continue;
                }
                f16* o = out + static_cast<int64_t>(row) * p.out.ld + col;
                store_raw<false>(o, hi);
                if (p.out_parts == 2) store_raw<false>(o + p.out.part_stride, lo);
            }
            if (mirror || (last && p.tall)) {
                asm volatile("bar.sync 1, %0;" ::"n"(EPI_WARPS * 32) : "memory");
                for (int i = threadIdx.x - 64; i < 128 * share; i += EPI_WARPS * 32) {
                    const int c = i / share, r = i % share;
                    const int at_col = tn * BN + c, at_row = tm * BM + first + r;
                    if (at_col >= p.cols || at_row >= p.rows) continue;
                    const float x = turned[c * turned_ld + r];
                    if (last) {
                        with_final_type(p, b, [&](auto* o) {
                            o[static_cast<int64_t>(at_col) * p.final_ld + at_row] = from_f<std::remove_pointer_t<decltype(o)>>(x);
                        });
                    } else {
                        f16* o = out + static_cast<int64_t>(at_col) * p.out.ld + at_row;
                        const f16 hi = __float2half_rn(x);
                        *o = hi;
                        if (p.out_parts == 2) o[p.out.part_stride] = __float2half_rn(x - __half2float(hi));
                    }
                }
            }
        }
    }

    // common exit, also after an abort; a CTA of a cluster stays while a peer may touch its memory
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync_relaxed();
    if (warp == 1) {
        __syncwarp();
        ptx::tc_fence_after_sync();
        if (PAIR) ptx::tmem_dealloc_pair(tmem_base, TMEM_COLS);
        else ptx::tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// ------------------------------------------------------- norm and first split

// partial[matrix][block]: sums of squares.  Threads walk over accesses of VEC elements,
// eight of them in flight.  The squares of an access are added in fp32 where they stay
// well inside its range, else in fp64; the accesses are added in fp64.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
orth_norm_kernel(double* __restrict__ partial, const T* __restrict__ g, int64_t ld, int64_t stride, int64_t rows,
                 int64_t cols)
{
    constexpr int DEEP = 8;
    __shared__ double sh[8];
    const T* m = g + blockIdx.y * stride;
    const int64_t nvec = cols / VEC, total = rows * nvec;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    double s = 0.0;
    for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i0 < total; i0 += step * DEEP) {
        Raw<T, VEC> r[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
            const int64_t i = i0 + k * step;
            const int64_t row = total <= UINT32_MAX ? static_cast<uint32_t>(i) / static_cast<uint32_t>(nvec) : i / nvec;
            if (i < total) load_raw<false>(r[k], m + row * ld + (i - row * nvec) * VEC);
        }
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
            if (i0 + k * step >= total) continue;
            float most = 0.0f, sum = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float x = to_f(r[k].e[e]);
                most = fmaxf(most, fabsf(x));
                sum = fmaf(x, x, sum);
            }
            if (most == 0.0f || (most > 1e-15f && most < 1e15f)) {
                s += static_cast<double>(sum);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const double x = static_cast<double>(to_f(r[k].e[e]));
                    s = fma(x, x, s);
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 8; ++i) t += sh[i];
        partial[blockIdx.y * gridDim.x + blockIdx.x] = t;
    }
}

// X0 = G / (|G| + eps) (transposed when TALL) as scaled fp16 parts; 64 x 64 tiles, a thread
// has eight neighbouring elements of two rows.
template <typename T, bool VEC, bool TALL>
__global__ void __launch_bounds__(256)
orth_split_kernel(Split x, const double* __restrict__ partial, int parts, const T* __restrict__ g, int64_t ld,
                  int64_t stride, int64_t rows, int64_t cols, float eps)
{
    __shared__ float tile[TALL ? 64 : 1][65];
    __shared__ double squares;
    const T* m = g + blockIdx.z * stride;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 64, c0 = static_cast<int64_t>(blockIdx.x) * 64;
    const int tx = (threadIdx.x & 7) * 8, ty = threadIdx.x >> 3;
    Raw<T, 8> in[2];                             // requested before the norm is known
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int64_t r = r0 + ty + k * 32, c = c0 + tx;
        const T* src = m + r * ld + c;
        if (VEC && r < rows && c + 8 <= cols) {
            load_raw<false>(in[k], src);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) in[k].e[e] = r < rows && c + e < cols ? src[e] : from_f<T>(0.0f);
        }
    }
    if (threadIdx.x < 32) {
        double s = 0.0;
        for (int i = threadIdx.x; i < parts; i += 32) s += partial[blockIdx.z * parts + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (threadIdx.x == 0) squares = s;
    }
    __syncthreads();
    const OrthInverse inv(squares, eps);
    f16* out = x.p + blockIdx.z * x.batch_stride;
    const int64_t xr0 = TALL ? c0 : r0, xc0 = TALL ? r0 : c0, xrows = TALL ? cols : rows;
    if (TALL) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) tile[ty + k * 32][tx + e] = to_f(in[k].e[e]);
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int64_t r = xr0 + ty + k * 32;
        if (r >= xrows) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = inv(TALL ? tile[tx + e][ty + k * 32] : to_f(in[k].e[e]));
        Raw<f16, 8> hi, lo;
        split_f16(v, hi, lo);
        f16* o = out + r * x.ld + xc0 + tx;      // the pitch is a multiple of 64: the columns fit
        store_raw<false>(o, hi);
        store_raw<false>(o + x.part_stride, lo);
    }
}

// ------------------------------------------------------------------------- host

struct OrthPlan {
    int64_t R, C, batch, ldx, lda;
    bool split;
    int64_t x[2], a, b, norm, total;             // byte offsets
};

OrthPlan plan_orth(int64_t rows, int64_t cols, int64_t batch, int type)
{
    OrthPlan q{};
    q.R = rows < cols ? rows : cols;
    q.C = rows < cols ? cols : rows;
    q.batch = batch;
    if (orthogonalize_small_always(rows, cols)) {        // never read: a page, so that every call has a workspace
        q.total = 4096;
        return q;
    }
    q.ldx = (q.C + 63) / 64 * 64;
    q.lda = (q.R + 63) / 64 * 64;
    q.split = type != SB200_BF16 || q.R <= 128;  // whichever kernel a narrow matrix takes, its operands have 22 bits
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    for (int i = 0; i < 2; ++i) q.x[i] = take(2 * batch * q.R * q.ldx * 2);
    q.a = take((q.split ? 2 : 1) * batch * q.R * q.lda * 2);
    q.b = take((q.split ? 2 : 1) * batch * q.R * q.lda * 2);
    q.norm = take(batch * NORM_BLOCKS * 8);
    q.total = at + 256;                          // the base is rounded up to 256 bytes
    return q;
}

// box: 64 elements along the contiguous dimension (a row of the 128-byte swizzle) x box_rows rows
int orth_map(sb200_ctx* ctx, CUtensorMap* map, const Split& m, int64_t cols, int64_t rows, int64_t matrices, int box_rows)
{
    EncodeTiledFn enc = reinterpret_cast<EncodeTiledFn>(ctx->encode_tiled);
    if (!enc) return SB200_ERR_UNSUPPORTED;
    const TensorMapKey key{reinterpret_cast<uint64_t>(m.p), cols, rows, m.ld, matrices, m.batch_stride, box_rows, 3};
    return cached_map(ctx, map, key, [&](CUtensorMap* t) {
        cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(matrices)};
        cuuint64_t strides[2] = {static_cast<cuuint64_t>(m.ld) * 2, static_cast<cuuint64_t>(m.batch_stride) * 2};
        cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
        cuuint32_t estr[3] = {1, 1, 1};
        return enc(t, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, m.p, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
}

struct OrthMaps {
    CUtensorMap a, b;
};

template <int WHAT, bool PAIR, bool SPLIT>
int launch_product(sb200_ctx* ctx, const OrthMaps& m, OrthParams p, cudaStream_t stream)
{
    auto kern = orth_product_kernel<WHAT, PAIR, SPLIT>;
    constexpr int SMEM = OrthSmem<SPLIT>::TOTAL;
    static bool attr_done[16] = {};
    if (ctx->device >= 16 || !attr_done[ctx->device]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) return SB200_ERR_CUDA;
        if (ctx->device < 16) attr_done[ctx->device] = true;
    }
    constexpr int TILE = PAIR ? 256 : 128;
    p.tiles_m = (p.rows + TILE - 1) / TILE;
    p.tiles_n = (p.cols + TILE - 1) / TILE;
    p.tiles = WHAT == APPLY ? p.tiles_m * p.tiles_n : p.tiles_m * (p.tiles_m + 1) / 2;
    const long long total = static_cast<long long>(p.tiles) * p.batch;
    const int group = PAIR ? 2 : p.slices;
    const long long most = PAIR ? ctx->sm_count / 2 : total;     // pairs walk over the tiles
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(group * (total < most ? total : most)));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(group);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, m.a, m.b, p);
    ctx->launches += 1;
    return err == cudaSuccess && cudaGetLastError() == cudaSuccess ? SB200_OK : SB200_ERR_CUDA;
}

// Pairs or slices.  A k-block of a 256 x 256 tile on a pair of SMs takes hardly longer than
// one of a 128 x 128 tile on one SM (whose tensor core waits for shared memory: 128 bytes a
// cycle feed it and take in the tiles), so a pair does four times the work on twice the SMs;
// slices win where the tiles are too few to fill the device.  Both are estimated from
// measured parts, in us: a launch up to its first tile 2; a k-block 0.36 (pair) and 0.33,
// with two parts 0.85 and 0.65; the epilogue of a pair 2.8 and 4.5, of a cluster of s slices
// 2.2 and 5 / s.  Returns 0 for pairs, else the number of slices.
int slices_for(const sb200_ctx* ctx, int64_t rows, int64_t cols, int64_t batch, int num_kb, bool symmetric, bool split)
{
    auto tiles = [&](int64_t t) {
        const int64_t tm = (rows + t - 1) / t, tn = (cols + t - 1) / t;
        return (symmetric ? tm * (tm + 1) / 2 : tm * tn) * batch;
    };
    auto waves = [](int64_t n, int64_t at_once) { return static_cast<double>((n + at_once - 1) / at_once); };
    const int64_t sms = ctx->sm_count, t1 = tiles(128), t2 = tiles(256);
    int s = 1;
    while (s < MAX_SLICES && 2 * s <= num_kb && t1 * 2 * s <= sms) s *= 2;
    const double sliced = waves(t1 * s, sms) * (2.0 + (num_kb + s - 1) / s * (split ? 0.65 : 0.33) + 2.2 + 5.0 / s);
    const double paired = 2.0 + waves(t2, sms / 2) * num_kb * (split ? 0.85 : 0.36) + (split ? 4.5 : 2.8);
    return sliced < paired ? s : 0;
}

template <int WHAT>
int product(sb200_ctx* ctx, bool split, const OrthMaps& m, OrthParams p, cudaStream_t stream)
{
    p.slices = slices_for(ctx, p.rows, p.cols, p.batch, p.num_kb, WHAT != APPLY, split);
    // One part: X X^T runs over the longer side, up to 2^20, and its diagonal adds positive terms alone, so that
    // what the chain cuts off goes to one side: 3.0e-3 of a sum over 2^19 columns in a single chain (measured,
    // 0.8 x 2^-23 an accumulation).  The others run over the shorter side; where that is 2^16 (X in its parts
    // and copies then takes 69 GB) a chain loses 4e-4, less than the half step of its fp16 operands.
    const bool chains = WHAT == GRAM && !split && p.num_kb > LONG_CHAIN_KB;
    p.chunk_kb = split ? (p.slices == 0 ? CHUNK_KB : 1) : chains ? LONG_CHAIN_KB : p.num_kb;
    if (p.slices == 0) {
        // (a kernel apart from GRAM: with the code for the chains that one has 96 registers instead of 85,
        // and 4 x 1024 x 4096 takes 497 us instead of 495)
        if constexpr (WHAT == GRAM)
            if (chains) return launch_product<LONG_GRAM, true, false>(ctx, m, p, stream);
        return split ? launch_product<WHAT, true, true>(ctx, m, p, stream) : launch_product<WHAT, true, false>(ctx, m, p, stream);
    }
    return split ? launch_product<WHAT, false, true>(ctx, m, p, stream) : launch_product<WHAT, false, false>(ctx, m, p, stream);
}

// Largest |f(u)| over [0, top]: at its ends or where the derivative d0 + d1 u + d2 u^2 is zero.
template <typename F>
double largest(F f, double top, double d0, double d1, double d2)
{
    double m = 0.0;
    auto look = [&](double u) {
        const double v = std::fabs(f(u));
        if (!(v <= m)) m = v;                    // (not a number counts as larger)
    };
    look(0.0);
    look(top);
    double root[2] = {-1.0, -1.0};
    if (d2 != 0.0) {
        const double disc = d1 * d1 - 4.0 * d2 * d0;
        if (disc >= 0.0) {
            const double h = -0.5 * (d1 + std::copysign(std::sqrt(disc), d1));
            root[0] = h / d2;
            if (h != 0.0) root[1] = d0 / h;
        }
    } else if (d1 != 0.0) {
        root[0] = -d0 / d1;
    }
    for (double u : root)
        if (u > 0.0 && u < top) look(u);
    return m;
}

// Whether every matrix of the iteration stays inside the range of the scaled fp16 parts:
// s bounds the singular values of X, b s^2 + c s^4 is B's norm, with a in front the norm of
// what stands in its place for bf16.  One per cent is for rounding.
bool bounded(double a, double b, double c, int steps)
{
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
    double s = 1.01;
    for (int k = 0; k < steps; ++k) {
        const double top = s * s;                // in u = s^2
        const double m = largest([&](double u) { return b * u + c * u * u; }, top, b, 2.0 * c, 0.0);
        const double d = largest([&](double u) { return a + b * u + c * u * u; }, top, b, 2.0 * c, 0.0);
        if (!(top < LARGEST) || !(m < LARGEST) || !(d < LARGEST)) return false;
        s = 1.01 * largest([&](double u) { return std::sqrt(u) * (a + b * u + c * u * u); }, top, a, 3.0 * b, 5.0 * c);
    }
    return true;
}

constexpr int64_t MAX_SIDE = int64_t(1) << 20;
constexpr int MAX_STEPS = 64;

}  // namespace
}  // namespace sb200

using namespace sb200;

extern "C" int64_t sb200_orthogonalize_workspace(int64_t rows, int64_t cols, int64_t batch, int type)
{
    if (rows < 0 || cols < 0 || batch < 0 || !known_type(type) || rows > MAX_SIDE || cols > MAX_SIDE || batch > 65535) return -1;
    return plan_orth(rows, cols, batch, type).total;
}

extern "C" int sb200_orthogonalize(sb200_ctx* ctx, void* out, int64_t ldo, int64_t stride_out, const void* g, int64_t ldg,
                                   int64_t stride_g, int64_t rows, int64_t cols, int64_t batch, int steps, float a, float b,
                                   float c, float eps, int type, void* workspace, int64_t workspace_bytes, sb200_stream stream_)
{
    TraceRange trace("sb200_orthogonalize");
    if (!ctx || rows < 0 || cols < 0 || batch < 0 || ldo < cols || ldg < cols || stride_out < 0 || stride_g < 0 ||
        !known_type(type) || steps < 1 || !(eps >= 0.0f))
        return SB200_ERR_INVALID_ARG;
    if (batch > 1 && stride_out < (rows - 1) * ldo + cols) return SB200_ERR_INVALID_ARG;   // outputs would overlap
    if (rows > MAX_SIDE || cols > MAX_SIDE || batch > 65535 || steps > MAX_STEPS) return SB200_ERR_TOO_LARGE;
    if (!bounded(a, b, c, steps)) return SB200_ERR_UNSUPPORTED;
    if (rows == 0 || cols == 0 || batch == 0) return SB200_OK;
    if (!out || !g || !aligned_to(out, type_bytes(type)) || !aligned_to(g, type_bytes(type))) return SB200_ERR_INVALID_ARG;
    const OrthPlan q = plan_orth(rows, cols, batch, type);
    if (!workspace || workspace_bytes < q.total) return SB200_ERR_INVALID_ARG;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const OrthCall call{out, ldo, batch > 1 ? stride_out : 0, g, ldg, batch > 1 ? stride_g : 0, rows, cols, batch, steps, a, b, c, eps, type};
    if (orthogonalize_small_fits(ctx, call)) return launch_orthogonalize_small(ctx, call, stream);
    if (orthogonalize_small_always(rows, cols)) return SB200_ERR_CUDA;   // (the device did not grant the kernel its shared memory)
    unsigned char* ws = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
    const int tall = rows > cols;

    auto matrix = [&](int64_t at, int64_t ld) {
        Split m;
        m.p = reinterpret_cast<f16*>(ws + at);
        m.ld = ld;
        m.batch_stride = q.R * ld;
        m.part_stride = batch * q.R * ld;
        return m;
    };
    const Split X[2] = {matrix(q.x[0], q.ldx), matrix(q.x[1], q.ldx)};
    const Split A = matrix(q.a, q.lda), B = matrix(q.b, q.lda);
    double* partial = reinterpret_cast<double*>(ws + q.norm);

    const dim3 split_grid(static_cast<unsigned>((cols + 63) / 64), static_cast<unsigned>((rows + 63) / 64), static_cast<unsigned>(batch));
    auto start = [&](auto t) {
        using T = decltype(t);
        constexpr int WIDE = 16 / sizeof(T);
        const T* gp = static_cast<const T*>(g);
        const bool wide = cols % WIDE == 0 && ldg % WIDE == 0 && (batch == 1 || stride_g % WIDE == 0) && aligned_to(g, 16);
        // about 8 accesses a thread
        const int64_t accesses = rows * cols / (wide ? WIDE : 1);
        int64_t blocks = (accesses + 2047) / 2048;
        const int parts = static_cast<int>(blocks < NORM_BLOCKS ? blocks : NORM_BLOCKS);
        const dim3 norm_grid(parts, static_cast<unsigned>(batch));
        if (wide) orth_norm_kernel<T, WIDE><<<norm_grid, 256, 0, stream>>>(partial, gp, ldg, stride_g, rows, cols);
        else orth_norm_kernel<T, 1><<<norm_grid, 256, 0, stream>>>(partial, gp, ldg, stride_g, rows, cols);
        auto split = [&](auto kern) { kern<<<split_grid, 256, 0, stream>>>(X[0], partial, parts, gp, ldg, stride_g, rows, cols, eps); };
        if (tall) { if (wide) split(orth_split_kernel<T, true, true>); else split(orth_split_kernel<T, false, true>); }
        else { if (wide) split(orth_split_kernel<T, true, false>); else split(orth_split_kernel<T, false, false>); }
    };
    if (type == SB200_F32) start(float{});
    else if (type == SB200_BF16) start(bf16{});
    else start(f16{});
    ctx->launches += 2;
    if (cudaGetLastError() != cudaSuccess) return SB200_ERR_CUDA;

    const int64_t xm = 2 * batch, am = (q.split ? 2 : 1) * batch;
    CUtensorMap x_rows[2], x_cols[2], a_rows, b_rows;
    for (int i = 0; i < 2; ++i) {
        if (const int rc = orth_map(ctx, &x_rows[i], X[i], q.C, q.R, xm, 128)) return rc;
        if (const int rc = orth_map(ctx, &x_cols[i], X[i], q.C, q.R, xm, KB)) return rc;
    }
    if (const int rc = orth_map(ctx, &a_rows, A, q.R, q.R, am, 128)) return rc;
    if (const int rc = orth_map(ctx, &b_rows, B, q.R, q.R, am, 128)) return rc;

    OrthParams p{};
    p.R = static_cast<int>(q.R);
    p.C = static_cast<int>(q.C);
    p.batch = static_cast<int>(batch);
    p.status = ctx->d_status;
    p.wait_limit_ns = ctx->wait_limit_ns;
    p.test_stall_kb = ctx->test_stall_kb;
    const int kb_c = static_cast<int>((q.C + KB - 1) / KB), kb_r = static_cast<int>((q.R + KB - 1) / KB);
    for (int k = 0; k < steps; ++k) {
        const int from = k & 1, to = from ^ 1;
        // A = X X^T
        p.rows = p.cols = p.R;
        p.num_kb = kb_c;
        p.prev = p.out = A;
        p.out_parts = q.split ? 2 : 1;
        p.alpha = INV_SCALE;
        p.final_out = nullptr;
        if (const int rc = product<GRAM>(ctx, q.split, {x_rows[from], x_rows[from]}, p, stream)) return rc;
        // B = b A + c A A (+ a on the diagonal)
        p.num_kb = kb_r;
        p.out = B;
        p.coef = b;
        p.alpha = c * INV_SCALE;
        p.diagonal = a * SCALE;
        if (const int rc = product<POLY>(ctx, q.split, {a_rows, a_rows}, p, stream)) return rc;
        // X = a X + B X
        p.cols = p.C;
        p.prev = X[from];
        p.out = X[to];
        p.out_parts = 2;
        p.coef = a;
        p.alpha = INV_SCALE;
        if (k + 1 == steps) {
            p.final_out = out;
            p.final_ld = ldo;
            p.final_stride = batch > 1 ? stride_out : 0;
            p.final_type = type;
            p.tall = tall;
            p.final_vec = !tall && aligned_to(out, 16) && (ldo * type_bytes(type)) % 16 == 0 &&
                          (p.final_stride * type_bytes(type)) % 16 == 0;
        }
        if (const int rc = product<APPLY>(ctx, q.split, {b_rows, x_cols[from]}, p, stream)) return rc;
    }
    return SB200_OK;
}
