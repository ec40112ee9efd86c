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
//     in registers.
//   bf16 input: the products take the hi parts alone (11 bits; the result keeps 8).
//     X still has both parts and the a X term uses both: rounding X itself every step
//     would feed the small singular directions, which a step multiplies by a, with the
//     rounding errors of the large ones.
//
// A and A A are symmetric: only tiles on and above the diagonal are computed, and a tile
// above it is also stored transposed.  X X^T and A A read both operands along k; B X reads
// X in rows of k ("MN-major"), so no matrix is ever transposed in memory.
#include <cmath>

#include "gemm_common.cuh"
#include "typed.cuh"

namespace sb200 {

using namespace gemm;

namespace {

constexpr int KB = 64;                           // fp16 elements of k per block: one 128-byte swizzle row
constexpr int MMA_K = 16;
constexpr int TILE_BYTES = 128 * KB * 2;         // 128 rows (or columns) x 64 k
constexpr int MN_CHUNK_BYTES = 64 * KB * 2;      // MN-major: 64 k rows x 64 columns
constexpr int CHUNK_KB = 2;                      // k-blocks per accumulation chain with two parts
constexpr float SCALE = 8192.0f;                 // 2^13
constexpr float INV_SCALE = 1.0f / 8192.0f;
constexpr double LARGEST = 7.5;                  // of a singular value: 7.5 * 2^13 < 65504
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + EPI_WARPS * 32;
constexpr int NORM_BLOCKS = 256;                 // partial sums of squares per matrix
constexpr int ORTH_PANEL = 8;

enum Product { GRAM, POLY, APPLY };

// A matrix of the iteration: [parts][batch][rows][ld] fp16, part 0 = hi, 1 = lo.
struct Split {
    f16* p;
    int64_t ld, batch_stride, part_stride;
};

struct OrthParams {
    int R, C, batch;
    int rows, cols, num_kb;                      // of the product
    int tiles_m, tiles_n, tiles;                 // per matrix
    int chunk_kb;
    Split prev, out;                             // prev: added with `coef`; out: the result
    int out_parts, prev_parts;
    float coef, alpha;                           // result = coef * prev + alpha * accumulator (scaled by 2^13)
    void* final_out;                             // APPLY, last step: the caller's matrix
    int64_t final_ld, final_stride;
    int final_type, tall;
    unsigned* status;
    unsigned long long wait_limit_ns;
    int test_stall_kb;
};

template <bool SPLIT>
struct OrthSmem {
    static constexpr int PARTS = SPLIT ? 2 : 1;
    static constexpr int STAGE = 2 * PARTS * TILE_BYTES;
    static constexpr int STAGES = SPLIT ? 3 : 6;
    static constexpr int TILES = STAGE * STAGES;
    static constexpr int BARS = ((2 * STAGES + 4) * 8 + 16 + 15) & ~15;
    static constexpr int TOTAL = TILES + BARS + 1024;
    static_assert(TOTAL <= 227 * 1024, "shared memory per CTA");
};

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

template <typename T>
__device__ __forceinline__ void final_store(T* out, int64_t ld, int tall, int row, int col0, const float* v, int R, int C)
{
    if (tall) {                                  // lanes hold neighbouring rows: contiguous in the output
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (row < R && col0 + j < C) out[static_cast<int64_t>(col0 + j) * ld + row] = from_f<T>(v[j]);
        return;
    }
    if (row >= R) return;
    T* o = out + static_cast<int64_t>(row) * ld + col0;
    if (col0 + 8 <= C && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = v[j];
        store_f<false>(o, f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col0 + j < C) o[j] = from_f<T>(v[j]);
    }
}

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
    constexpr int COLS = BN / 2;                 // accumulator columns of an epilogue warp
    constexpr uint32_t TMEM_COLS = 2 * BN;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::TILES);
    uint64_t* empty_bar = full_bar + S::STAGES;
    uint64_t* tmem_full = empty_bar + S::STAGES;
    uint64_t* tmem_empty = tmem_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? ptx::cluster_ctarank() : 0u;
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

    const int unit = PAIR ? blockIdx.x >> 1 : blockIdx.x;
    const int units = PAIR ? gridDim.x >> 1 : gridDim.x;
    const int total = p.tiles * p.batch;

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
                const int m0 = tm * BM + static_cast<int>(rank) * 128;
                const int n0 = tn * BN + static_cast<int>(rank) * 128;
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    if (p.test_stall_kb >= 0 && issued++ >= p.test_stall_kb) {
                        ok = false;              // test hook: the other roles' waits run out
                        break;
                    }
                    if (!(ok = wait(&empty_bar[s], ph ^ 1u, FAULT_PRODUCER_WAIT))) break;
                    uint8_t* st = smem + s * S::STAGE;
                    const int k0 = kb * KB;
                    if (rank == 0) ptx::mbar_arrive_expect_tx(&full_bar[s], CTAS * S::STAGE);
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
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = ptx::make_idesc_f16(BM, BN, 0, B_MN);
            constexpr uint32_t A_STEP = MMA_K * 2, B_STEP = B_MN ? MMA_K * 128u : MMA_K * 2u;
            constexpr uint32_t B_LBO = B_MN ? MN_CHUNK_BYTES : 16u;
            int s = 0;
            uint32_t ph = 0;
            int acc = 0;
            uint32_t acc_ph = 0;
            bool ok = true;
            for (int t = unit; ok && t < total; t += units) {
                for (int kb0 = 0; ok && kb0 < p.num_kb; kb0 += p.chunk_kb) {
                    if (!(ok = wait(&tmem_empty[acc], acc_ph ^ 1u, FAULT_MMA_WAIT_TMEM))) break;
                    ptx::tc_fence_after_sync();
                    const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
                    const int kb1 = min(kb0 + p.chunk_kb, p.num_kb);
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
        // warp w reads TMEM lanes 32 (w % 4) .. + 31 and one half of the columns
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(half * COLS);
        int acc = 0;
        uint32_t acc_ph = 0;
        bool ok = true;
        for (int t = unit; ok && t < total; t += units) {
            const int b = t / p.tiles;
            int tm, tn;
            orth_tile(t % p.tiles, p, SYMMETRIC, tm, tn);
            const int row = tm * BM + static_cast<int>(rank) * 128 + q * 32 + lane;
            const int col0 = tn * BN + half * COLS;
            float sum[COLS];
#pragma unroll
            for (int j = 0; j < COLS; ++j) sum[j] = 0.0f;
            for (int kb0 = 0; ok && kb0 < p.num_kb; kb0 += p.chunk_kb) {
                if (!(ok = wait(&tmem_full[acc], acc_ph, FAULT_EPI_WAIT))) break;
                ptx::tc_fence_after_sync();
#pragma unroll
                for (int c = 0; c < COLS / 32; ++c) {
                    uint32_t v[32];
                    ptx::tmem_ld_32x32(lane_base + static_cast<uint32_t>(acc * BN + c * 32), v);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[c * 32 + j] = __fadd_rn(sum[c * 32 + j], __uint_as_float(v[j]));
                }
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) ptx::mbar_arrive_cluster(ptx::map_to_cta(ptx::smem_u32(&tmem_empty[acc]), 0));
                    else ptx::mbar_arrive(&tmem_empty[acc]);
                }
                acc ^= 1;
                if (acc == 0) acc_ph ^= 1u;
            }
            if (!ok) break;
            const bool row_in = row < p.rows;
            const f16* prev = p.prev.p + b * p.prev.batch_stride + static_cast<int64_t>(row) * p.prev.ld;
            f16* out = p.out.p + b * p.out.batch_stride;
#pragma unroll
            for (int j = 0; j < COLS; j += 8) {
                const int col = col0 + j;
                if (col >= p.cols) break;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = sum[j + e] * p.alpha;
                if (WHAT != GRAM && row_in) {
                    float h[8];
                    load_f<false>(h, prev + col);
                    if (p.prev_parts == 2) {
                        float l[8];
                        load_f<false>(l, prev + p.prev.part_stride + col);
#pragma unroll
                        for (int e = 0; e < 8; ++e) h[e] += l[e];
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = fmaf(p.coef, h[e], v[e]);
                }
                if (WHAT == APPLY && p.final_out) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= INV_SCALE;
                    const int64_t at = b * p.final_stride;
                    if (p.final_type == SB200_F32)
                        final_store(static_cast<float*>(p.final_out) + at, p.final_ld, p.tall, row, col, v, p.R, p.C);
                    else if (p.final_type == SB200_BF16)
                        final_store(static_cast<bf16*>(p.final_out) + at, p.final_ld, p.tall, row, col, v, p.R, p.C);
                    else
                        final_store(static_cast<f16*>(p.final_out) + at, p.final_ld, p.tall, row, col, v, p.R, p.C);
                    continue;
                }
                Raw<f16, 8> hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    hi.e[e] = __float2half_rn(v[e]);
                    lo.e[e] = __float2half_rn(v[e] - __half2float(hi.e[e]));
                }
                if (row_in) {                    // rows have a pitch of a multiple of 64: whole vectors fit
                    f16* o = out + static_cast<int64_t>(row) * p.out.ld + col;
                    store_raw<false>(o, hi);
                    if (p.out_parts == 2) store_raw<false>(o + p.out.part_stride, lo);
                }
                if (SYMMETRIC && tn > tm && row_in) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (col + e < p.cols) {
                            f16* o = out + static_cast<int64_t>(col + e) * p.out.ld + row;
                            *o = hi.e[e];
                            if (p.out_parts == 2) o[p.out.part_stride] = lo.e[e];
                        }
                    }
                }
            }
        }
    }

    // common exit, also after an abort; a CTA of a pair stays while its peer may touch its memory
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (PAIR) ptx::cluster_sync();
    if (warp == 1) {
        __syncwarp();
        ptx::tc_fence_after_sync();
        if (PAIR) ptx::tmem_dealloc_pair(tmem_base, TMEM_COLS);
        else ptx::tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// ------------------------------------------------------- norm and first split

// partial[matrix][block]: sums of squares, in fp64 (squares of fp32 numbers leave the fp32 range)
template <typename T>
__global__ void __launch_bounds__(256)
orth_norm_kernel(double* __restrict__ partial, const T* __restrict__ g, int64_t ld, int64_t stride, int64_t rows,
                 int64_t cols)
{
    __shared__ double sh[8];
    const T* m = g + blockIdx.y * stride;
    double s = 0.0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* row = m + r * ld;
        for (int64_t j = threadIdx.x; j < cols; j += blockDim.x) {
            const double x = static_cast<double>(to_f(row[j]));
            s = fma(x, x, s);
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

// X0 = G / (|G| + eps) (transposed when tall) as scaled fp16 parts; 64 x 64 tiles.
template <typename T>
__global__ void __launch_bounds__(256)
orth_split_kernel(Split x, const double* __restrict__ partial, int parts, const T* __restrict__ g, int64_t ld,
                  int64_t stride, int64_t rows, int64_t cols, int tall, float eps)
{
    __shared__ float tile[64][65];
    __shared__ float inv_sh;
    if (threadIdx.x < 32) {
        double s = 0.0;
        for (int i = threadIdx.x; i < parts; i += 32) s += partial[blockIdx.z * parts + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (threadIdx.x == 0) inv_sh = static_cast<float>(static_cast<double>(SCALE) / (sqrt(s) + static_cast<double>(eps)));
    }
    __syncthreads();
    const float inv = inv_sh;
    const T* m = g + blockIdx.z * stride;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 64, c0 = static_cast<int64_t>(blockIdx.x) * 64;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int i = ty; i < 64; i += 4) {
        const int64_t r = r0 + i, c = c0 + tx;
        tile[i][tx] = r < rows && c < cols ? to_f(m[r * ld + c]) * inv : 0.0f;
    }
    __syncthreads();
    f16* out = x.p + blockIdx.z * x.batch_stride;
    const int64_t xr0 = tall ? c0 : r0, xc0 = tall ? r0 : c0;
    const int64_t xrows = tall ? cols : rows;
    for (int i = ty; i < 64; i += 4) {
        const float v = tall ? tile[tx][i] : tile[i][tx];
        const int64_t r = xr0 + i;
        if (r < xrows) {                         // the pitch is a multiple of 64: the columns fit
            f16* o = out + r * x.ld + xc0 + tx;
            const f16 hi = __float2half_rn(v);
            o[0] = hi;
            o[x.part_stride] = __float2half_rn(v - __half2float(hi));
        }
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
    q.ldx = (q.C + 63) / 64 * 64;
    q.lda = (q.R + 63) / 64 * 64;
    q.split = type != SB200_BF16;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    for (int i = 0; i < 2; ++i) q.x[i] = take(2 * batch * q.R * q.ldx * 2);
    q.a = take((q.split ? 2 : 1) * batch * q.R * q.lda * 2);
    q.b = take((q.split ? 2 : 1) * batch * q.R * q.lda * 2);
    q.norm = take(batch * NORM_BLOCKS * 8);
    q.total = at + 256;                          // the base is rounded up to 256 bytes
    return q;
}

// box: 64 elements along the contiguous dimension x box_rows rows
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

template <int WHAT, bool PAIR, bool SPLIT>
int launch_product(sb200_ctx* ctx, const CUtensorMap& ma, const CUtensorMap& mb, OrthParams p, cudaStream_t stream)
{
    auto kern = orth_product_kernel<WHAT, PAIR, SPLIT>;
    constexpr int SMEM = OrthSmem<SPLIT>::TOTAL;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) return SB200_ERR_CUDA;
    constexpr int TILE = PAIR ? 256 : 128;
    p.tiles_m = (p.rows + TILE - 1) / TILE;
    p.tiles_n = (p.cols + TILE - 1) / TILE;
    p.tiles = WHAT == APPLY ? p.tiles_m * p.tiles_n : p.tiles_m * (p.tiles_m + 1) / 2;
    const long long total = static_cast<long long>(p.tiles) * p.batch;
    const long long most = PAIR ? ctx->sm_count / 2 : ctx->sm_count;
    const long long units = total < most ? total : most;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(PAIR ? 2 * units : units));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
    if (PAIR) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 2;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, ma, mb, p);
    ctx->launches += 1;
    return err == cudaSuccess && cudaGetLastError() == cudaSuccess ? SB200_OK : SB200_ERR_CUDA;
}

template <int WHAT>
int product(sb200_ctx* ctx, bool pair, bool split, const CUtensorMap& ma, const CUtensorMap& mb, const OrthParams& p,
            cudaStream_t stream)
{
    if (pair)
        return split ? launch_product<WHAT, true, true>(ctx, ma, mb, p, stream) : launch_product<WHAT, true, false>(ctx, ma, mb, p, stream);
    return split ? launch_product<WHAT, false, true>(ctx, ma, mb, p, stream) : launch_product<WHAT, false, false>(ctx, ma, mb, p, stream);
}

// Largest |f| of an odd or even polynomial over [0, s], by its samples: the polynomials
// are smooth, 1024 samples are within a thousandth of the maximum.
template <typename F>
double largest(F f, double s)
{
    double m = 0.0;
    for (int i = 0; i <= 1024; ++i) {
        const double v = std::fabs(f(s * i / 1024.0));
        if (!(v <= m)) m = v;
    }
    return m;
}

// Whether every matrix of the iteration stays inside the range of the scaled fp16 parts.
bool bounded(double a, double b, double c, int steps)
{
    double s = 1.01;
    for (int k = 0; k < steps; ++k) {
        const double m = largest([&](double t) { return b * t * t + c * t * t * t * t; }, s);
        if (!(s * s < LARGEST) || !(m < LARGEST)) return false;
        s = 1.01 * largest([&](double t) { return t * (a + b * t * t + c * t * t * t * t); }, s);
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
    if (!out || !g) return SB200_ERR_INVALID_ARG;
    const OrthPlan q = plan_orth(rows, cols, batch, type);
    if (!workspace || workspace_bytes < q.total) return SB200_ERR_INVALID_ARG;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
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

    const int parts = static_cast<int>(rows < NORM_BLOCKS ? rows : NORM_BLOCKS);
    const dim3 norm_grid(parts, static_cast<unsigned>(batch));
    const dim3 split_grid(static_cast<unsigned>((cols + 63) / 64), static_cast<unsigned>((rows + 63) / 64), static_cast<unsigned>(batch));
    auto start = [&](auto t) {
        using T = decltype(t);
        const T* gp = static_cast<const T*>(g);
        orth_norm_kernel<T><<<norm_grid, 256, 0, stream>>>(partial, gp, ldg, stride_g, rows, cols);
        orth_split_kernel<T><<<split_grid, 256, 0, stream>>>(X[0], partial, parts, gp, ldg, stride_g, rows, cols, tall, eps);
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
    // A pair of SMs per 256 x 256 tile when there are enough of those to fill the device
    auto pairs = [&](int64_t r, int64_t n, bool symmetric) {
        const int64_t tm = (r + 255) / 256, tn = (n + 255) / 256;
        return (symmetric ? tm * (tm + 1) / 2 : tm * tn) * batch >= ctx->sm_count / 2;
    };
    const bool pair_a = pairs(q.R, q.R, true), pair_x = pairs(q.R, q.C, false);
    for (int k = 0; k < steps; ++k) {
        const int from = k & 1, to = from ^ 1;
        // A = X X^T
        p.rows = p.cols = p.R;
        p.num_kb = kb_c;
        p.chunk_kb = q.split ? CHUNK_KB : kb_c;
        p.prev = A;
        p.prev_parts = 0;
        p.out = A;
        p.out_parts = q.split ? 2 : 1;
        p.coef = 0.0f;
        p.alpha = INV_SCALE;
        p.final_out = nullptr;
        if (const int rc = product<GRAM>(ctx, pair_a, q.split, x_rows[from], x_rows[from], p, stream)) return rc;
        // B = b A + c A A
        p.num_kb = kb_r;
        p.chunk_kb = q.split ? CHUNK_KB : kb_r;
        p.prev_parts = p.out_parts;
        p.out = B;
        p.coef = b;
        p.alpha = c * INV_SCALE;
        if (const int rc = product<POLY>(ctx, pair_a, q.split, a_rows, a_rows, p, stream)) return rc;
        // X = a X + B X
        p.cols = p.C;
        p.prev = X[from];
        p.prev_parts = 2;
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
        }
        if (const int rc = product<APPLY>(ctx, pair_x, q.split, b_rows, x_cols[from], p, stream)) return rc;
    }
    return SB200_OK;
}
