// The orthogonalised update of a matrix with a side of at most 128 (and the other of at
// most 4096) in one launch: all its steps by one cluster of 1 to 16 CTAs, X in shared
// memory all the while.  The general way (orthogonalize.cu) takes three launches a step,
// each with a pipeline to fill and results that travel through the L2: about 9 us a
// product whatever its size, when these products are less than one.
//
// X is R x C, R <= 128; CTA s holds columns [s W, (s + 1) W), W a multiple of 64 up to
// 256, as two
// fp16 parts in the layout the tensor core reads (rows of 64 columns = 128 bytes, 128-byte
// swizzle).  The same bytes serve as both operands of X X^T (rows of k) and as the right
// operand of B X (columns of n).  A step:
//   partial X X^T over the CTA's columns (tensor core)
//   its sum over the cluster: each CTA adds a share of the rows of all partials through
//     distributed shared memory, splits the sums into parts and stores them in every CTA
//   B = b A + c A A by every CTA for itself
//   X = a X + B X on the CTA's columns
// Products and parts are those of the general way with two parts, for bf16 too: the products
// are too short to gain from one.  Accumulation chains have 32 of k (64 in B X where W columns
// leave room for two accumulators only; the general way's have 64 or 128).  Five steps take 50 us for 128 x 128 fp32 (135 in
// launches), 77 for 128 x 1000, 86 for 128 x 2000, 108 for 128 x 4000.
#include <type_traits>

#include "gemm_common.cuh"
#include "orthogonalize.cuh"

namespace sb200 {

using namespace gemm;

namespace {

constexpr int SMALL_THREADS = 512, SMALL_WARPS = 16;
constexpr int SMALL_TILE = 128 * 128;            // 128 rows of 64 fp16 elements, in bytes
constexpr int SMALL_W = 256;                     // columns of a CTA at most
constexpr int SMALL_CTAS = 16;                   // beyond PORTABLE_CTAS where the device grants clusters of that size
constexpr int PORTABLE_CTAS = 8;
constexpr int SMALL_X_PART = SMALL_W / 64 * SMALL_TILE;
constexpr int SMALL_A_PART = 2 * SMALL_TILE;
constexpr int SMALL_SMEM = 2 * SMALL_X_PART + 2 * SMALL_A_PART + 256 + 1024;

struct SmallParams {
    OrthCall q;
    int R, C, W, ctas, tall;
    unsigned* status;
    unsigned long long wait_limit_ns;
    int test_stall_kb;
};

// 16-byte piece `c8` (eight columns) of row r of a matrix of 64-column tiles
__device__ __forceinline__ int small_piece(int r, int c8)
{
    return (c8 >> 3) * SMALL_TILE + r * 128 + (((c8 & 7) ^ (r & 7)) << 4);
}

template <typename T>
__global__ void __launch_bounds__(SMALL_THREADS, 1) orth_small_kernel(const SmallParams p)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* x = smem;                           // [2 parts][W / 64 tiles]
    uint8_t* am = smem + 2 * SMALL_X_PART;       // A, then B: [2 parts][2 tiles]; before that the partial X X^T in fp32
    double* norm = reinterpret_cast<double*>(am + 2 * SMALL_A_PART);     // [SMALL_WARPS]: the warps', then [0] the CTA's
    uint64_t* done = reinterpret_cast<uint64_t*>(norm + SMALL_WARPS);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = p.ctas > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const int64_t matrix = blockIdx.x / p.ctas;
    const Abort ab{abort_flag, p.status, p.wait_limit_ns};
    if (tid == 0) {
        ptx::mbar_init(done, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 0) {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();

    // ---- this CTA's columns of G, eight elements of X a piece: the norm, then the parts
    const T* g = static_cast<const T*>(p.q.g) + matrix * p.q.stride_g;
    const int c_first = rank * p.W, pieces = 128 * p.W / 8;
    constexpr int PER = 128 * SMALL_W / 8 / SMALL_THREADS;
    float v[PER][8];
    float sum = 0.0f, most = 0.0f;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = k * SMALL_THREADS + tid;
        // neighbouring lanes on neighbouring memory: along the columns of X, or its rows when G is tall
        const int r = p.tall ? i & 127 : i / (p.W / 8), c = c_first + (p.tall ? i >> 7 : i % (p.W / 8)) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = i < pieces && r < p.R && c + e < p.C;
            v[k][e] = in ? to_f(p.tall ? g[static_cast<int64_t>(c + e) * p.q.ldg + r] : g[static_cast<int64_t>(r) * p.q.ldg + c + e]) : 0.0f;
            most = fmaxf(most, fabsf(v[k][e]));
            sum = fmaf(v[k][e], v[k][e], sum);
        }
    }
    double total = static_cast<double>(sum);
    if (!(most == 0.0f || (most > 1e-15f && most < 1e15f))) {            // squares beyond the fp32 range
        total = 0.0;
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) total = fma(static_cast<double>(v[k][e]), static_cast<double>(v[k][e]), total);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) norm[warp] = total;
    __syncthreads();
    total = 0.0;
    for (int w = 0; w < SMALL_WARPS; ++w) total += norm[w];
    if (p.ctas > 1) {
        __syncthreads();
        if (tid == 0) norm[0] = total;
        ptx::cluster_sync();
        total = 0.0;
        for (int s = 0; s < p.ctas; ++s) total += ptx::ld_cluster_f64(ptx::map_to_cta(ptx::smem_u32(norm), s));
    }
    const OrthInverse inv(total, p.q.eps);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = k * SMALL_THREADS + tid;
        if (i >= pieces) continue;
        const int r = p.tall ? i & 127 : i / (p.W / 8), c8 = p.tall ? i >> 7 : i % (p.W / 8);
        Raw<f16, 8> hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] = inv(v[k][e]);
        split_f16(v[k], hi, lo);
        store_raw<false>(reinterpret_cast<f16*>(x + small_piece(r, c8)), hi);
        store_raw<false>(reinterpret_cast<f16*>(x + SMALL_X_PART + small_piece(r, c8)), lo);
    }

    uint32_t phase = 0;
    bool ok = true;
    const int q = warp & 3, group = warp >> 2, row = q * 32 + lane;      // TMEM lanes and a quarter of the columns
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(q * 32) << 16);
    // one thread issues `products`; everybody waits until they are done
    auto run = [&](auto products) {
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before_sync();
        __syncthreads();
        if (tid == 0) {
            ptx::tc_fence_after_sync();
            if (ok) products();                  // (none behind a wait that gave up)
            if (p.test_stall_kb < 0) ptx::mma_commit(done);              // (test hook: the wait below runs out)
        }
        __syncwarp();
        if (ok) ok = wait_bar(done, phase, ab, FAULT_EPI_WAIT);
        phase ^= 1u;
        ptx::tc_fence_after_sync();
    };
    const uint32_t x_at = ptx::smem_u32(x), a_at = ptx::smem_u32(am);
    // One chain of accumulations into d: `count` times 16 of k.  Small terms come first: the
    // tensor core cuts what it adds at the accumulator's last place, which matters only once
    // hi.hi has begun.  Chains have 32 of k: with 64 the result of narrow matrices (68 x 3567)
    // was off by 2.0e-6, twice as much as fp32 arithmetic.
    auto chain = [&](uint32_t d, uint32_t a_part, uint32_t a, uint32_t b, uint32_t b_part, uint32_t idesc, uint32_t b_step, uint32_t b_lbo,
                     auto count) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const uint32_t pa = a + (pass == 1 ? a_part : 0), pb = b + (pass == 0 ? b_part : 0);
#pragma unroll
            for (int k = 0; k < decltype(count)::value; ++k)
                ptx::mma_f16(d, ptx::make_smem_desc(pa + k * 32, 16u, 1024u, ptx::LAYOUT_SW128),
                             ptx::make_smem_desc(pb + k * b_step, b_lbo, 1024u, ptx::LAYOUT_SW128), idesc, pass > 0 || k > 0);
        }
    };
    auto add_chains = [&](float (&to)[32], int col, int count, int pitch) {
#pragma unroll 1
        for (int c = 0; c < count; c += 2) {     // (an even number: two loads under way)
            uint32_t u[32], v[32];
            ptx::tmem_ld_32x32(lane_base + c * pitch + col, u);
            ptx::tmem_ld_32x32(lane_base + (c + 1) * pitch + col, v);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) to[j] = __fadd_rn(__fadd_rn(to[j], __uint_as_float(u[j])), __uint_as_float(v[j]));
        }
    };
    using Two = std::integral_constant<int, 2>;
    using Four = std::integral_constant<int, 4>;
    const int k_chains = p.R > 64 ? 4 : 2;       // of the products over R

    for (int step = 0; step < p.q.steps; ++step) {
        // ---- partial X X^T, a chain per 32 columns, four at a time
        float acc[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[j] = 0.0f;
        const int chains = p.W / 32;
#pragma unroll 1
        for (int c0 = 0; c0 < chains; c0 += 4) {
            const int count = min(4, chains - c0);
            run([&]() {
                constexpr uint32_t idesc = ptx::make_idesc_f16(128, 128, 0, 0);
                for (int c = 0; c < count; ++c) {
                    const uint32_t at = x_at + ((c0 + c) >> 1) * SMALL_TILE + ((c0 + c) & 1) * 64;
                    chain(tmem + c * 128, SMALL_X_PART, at, at, SMALL_X_PART, idesc, 32, 16u, Two{});
                }
            });
            add_chains(acc, group * 32, count, 128);
        }
        if (p.ctas == 1) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                Raw<f16, 8> hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[c * 8 + e] *= ORTH_INV_SCALE;
                split_f16(acc + c * 8, hi, lo);
                store_raw<false>(reinterpret_cast<f16*>(am + small_piece(row, group * 4 + c)), hi);
                store_raw<false>(reinterpret_cast<f16*>(am + SMALL_A_PART + small_piece(row, group * 4 + c)), lo);
            }
        } else {
            // [128 rows][32 pieces of four], a row's pieces permuted by its number
#pragma unroll
            for (int c = 0; c < 8; ++c)
                *reinterpret_cast<float4*>(am + row * 512 + (((group * 8 + c) ^ (row & 31)) << 4)) =
                    make_float4(acc[c * 4], acc[c * 4 + 1], acc[c * 4 + 2], acc[c * 4 + 3]);
            ptx::cluster_sync();
            // this CTA's rows: a warp takes whole ones, four columns a lane
            const int share = 128 / p.ctas;      // 64 to 8 rows: 4 a warp at most
            Raw<f16, 4> hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k * SMALL_WARPS + warp >= share) break;
                const int r = rank * share + k * SMALL_WARPS + warp;
                const uint32_t at = a_at + static_cast<uint32_t>(r * 512 + ((lane ^ (r & 31)) << 4));
                float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
                for (int s0 = 0; s0 < p.ctas; s0 += 8) {         // eight loads under way
                    float4 part[8];
#pragma unroll
                    for (int s = 0; s < 8; ++s)
                        if (s0 + s < p.ctas) part[s] = ptx::ld_cluster_f4(ptx::map_to_cta(at, s0 + s));
#pragma unroll
                    for (int s = 0; s < 8; ++s)
                        if (s0 + s < p.ctas) { t[0] += part[s].x; t[1] += part[s].y; t[2] += part[s].z; t[3] += part[s].w; }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] *= ORTH_INV_SCALE;
                split_f16(t, hi[k], lo[k]);
            }
            ptx::cluster_sync();                 // the partials are read: A may take their place
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k * SMALL_WARPS + warp >= share) break;
                const int r = rank * share + k * SMALL_WARPS + warp;
                const uint32_t at = a_at + static_cast<uint32_t>(small_piece(r, lane >> 1) + (lane & 1) * 8);
                for (int s = 0; s < p.ctas; ++s) {
                    const uint32_t to = ptx::map_to_cta(at, s);
                    ptx::st_cluster_b64(to, *reinterpret_cast<const uint2*>(hi[k].e));
                    ptx::st_cluster_b64(to + SMALL_A_PART, *reinterpret_cast<const uint2*>(lo[k].e));
                }
            }
            ptx::cluster_sync();
        }

        // ---- B = b A + c A A in A's place
        run([&]() {
            constexpr uint32_t idesc = ptx::make_idesc_f16(128, 128, 0, 0);
            for (int c = 0; c < k_chains; ++c) {
                const uint32_t at = a_at + (c >> 1) * SMALL_TILE + (c & 1) * 64;
                chain(tmem + c * 128, SMALL_A_PART, at, at, SMALL_A_PART, idesc, 32, 16u, Two{});
            }
        });
        {
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[j] = 0.0f;
            add_chains(acc, group * 32, k_chains, 128);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                f16* at = reinterpret_cast<f16*>(am + small_piece(row, group * 4 + c));
                float h[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                Raw<f16, 8> hi, lo;
                load_raw<false>(lo, at + SMALL_A_PART / 2);
                join_f16(h, lo);
                load_raw<false>(hi, at);
                join_f16(h, hi);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = fmaf(p.q.b, h[e], acc[c * 8 + e] * (p.q.c * ORTH_INV_SCALE));
                split_f16(h, hi, lo);
                store_raw<false>(at, hi);
                store_raw<false>(at + SMALL_A_PART / 2, lo);
            }
        }

        // ---- X = a X + B X on this CTA's columns
        // (where W columns leave room for two accumulators only, chains of 64 rows)
        const int merged = k_chains * p.W > 512 ? 2 : 1, x_chains = k_chains / merged;
        run([&]() {
            const uint32_t idesc = ptx::make_idesc_f16(128, p.W, 0, 1);
            for (int c = 0; c < x_chains; ++c) {
                const int first = c * merged;    // in units of 32 rows
                const uint32_t a = a_at + (first >> 1) * SMALL_TILE + (first & 1) * 64, b = x_at + first * 32 * 128;
                if (merged == 2) chain(tmem + c * p.W, SMALL_A_PART, a, b, SMALL_X_PART, idesc, 16 * 128, SMALL_TILE, Four{});
                else chain(tmem + c * p.W, SMALL_A_PART, a, b, SMALL_X_PART, idesc, 16 * 128, SMALL_TILE, Two{});
            }
        });
        const bool last = step + 1 == p.q.steps;
        const int width = p.W / 4;               // columns of this warp
#pragma unroll 1
        for (int j = 0; j < width; j += 16) {
            float y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = 0.0f;
#pragma unroll 1
            for (int c = 0; c < x_chains; c += 2) {
                uint32_t u[16], v[16];
                ptx::tmem_ld_32x16(lane_base + c * p.W + group * width + j, u);
                ptx::tmem_ld_32x16(lane_base + (c + 1) * p.W + group * width + j, v);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = __fadd_rn(__fadd_rn(y[e], __uint_as_float(u[e])), __uint_as_float(v[e]));
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                f16* at = reinterpret_cast<f16*>(x + small_piece(row, (group * width + j) / 8 + c));
                float h[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                Raw<f16, 8> hi, lo;
                load_raw<false>(lo, at + SMALL_X_PART / 2);
                join_f16(h, lo);
                load_raw<false>(hi, at);
                join_f16(h, hi);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = fmaf(p.q.a, h[e], y[c * 8 + e] * ORTH_INV_SCALE);
                if (!last) {
                    split_f16(h, hi, lo);
                    store_raw<false>(at, hi);
                    store_raw<false>(at + SMALL_X_PART / 2, lo);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[c * 8 + e] = h[e] * ORTH_INV_SCALE;
                }
            }
            if (last) {
                T* out = static_cast<T*>(p.q.out) + matrix * p.q.stride_out;
                const int col = c_first + group * width + j;
                if (p.tall) {                    // lanes hold neighbouring rows: contiguous in the output
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (row < p.R && col + e < p.C) out[static_cast<int64_t>(col + e) * p.q.ldo + row] = from_f<T>(y[e]);
                } else {
                    // through B's place, which is free: out by rows of 16 columns, two rows an access
                    float* mine = reinterpret_cast<float*>(am) + warp * 32 * 17;
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 16; ++e) mine[lane * 17 + e] = y[e];
                    __syncwarp();
#pragma unroll 4
                    for (int r = lane >> 4; r < 32; r += 2) {
                        const int c = col + (lane & 15);
                        if (q * 32 + r < p.R && c < p.C) out[static_cast<int64_t>(q * 32 + r) * p.q.ldo + c] = from_f<T>(mine[r * 17 + (lane & 15)]);
                    }
                }
            }
        }
    }

    ptx::tc_fence_before_sync();
    __syncthreads();
    if (p.ctas > 1) ptx::cluster_sync_relaxed();         // a peer may still store into this CTA's A
    if (warp == 0) {
        __syncwarp();
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem, 512);
    }
}

template <typename T>
cudaLaunchConfig_t small_config(cudaLaunchAttribute (&attr)[2], int64_t batch, int ctas, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(batch * ctas));
    cfg.blockDim = dim3(SMALL_THREADS);
    cfg.dynamicSmemBytes = SMALL_SMEM;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cfg;
}

// The largest cluster this kernel can have on the context's device: SMALL_CTAS, PORTABLE_CTAS, or 0 (asked once).
template <typename T>
int largest_cluster(const sb200_ctx* ctx)
{
    static int known[16] = {};                   // + 1
    if (ctx->device < 16 && known[ctx->device]) return known[ctx->device] - 1;
    auto kern = orth_small_kernel<T>;
    int most = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMALL_SMEM) == cudaSuccess) {
        most = PORTABLE_CTAS;
        cudaLaunchAttribute attr[2];
        cudaLaunchConfig_t cfg = small_config<T>(attr, 1, SMALL_CTAS, nullptr);
        cfg.numAttrs = 1;
        int fit = 0;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
            cudaOccupancyMaxActiveClusters(&fit, kern, &cfg) == cudaSuccess && fit > 0)
            most = SMALL_CTAS;
        cudaGetLastError();
    }
    if (ctx->device < 16 && most > 0) known[ctx->device] = most + 1;     // (a refusal is asked about again)
    return most;
}

// f(T{}) for an element type of the ABI
template <typename F>
int with_small_type(int type, F f)
{
    return type == SB200_F32 ? f(float{}) : type == SB200_F16 ? f(f16{}) : f(bf16{});
}

}  // namespace

bool orthogonalize_small_always(int64_t rows, int64_t cols)
{
    const int64_t r = rows < cols ? rows : cols, c = rows < cols ? cols : rows;
    return r <= 128 && c <= SMALL_W * PORTABLE_CTAS;
}

bool orthogonalize_small_fits(const sb200_ctx* ctx, const OrthCall& q)
{
    const int64_t r = q.rows < q.cols ? q.rows : q.cols, c = q.rows < q.cols ? q.cols : q.rows;
    if (r > 128 || c > SMALL_W * SMALL_CTAS) return false;
    return with_small_type(q.type, [&](auto t) -> int {
        const int most = largest_cluster<decltype(t)>(ctx);
        return c <= static_cast<int64_t>(SMALL_W) * most;
    });
}

int launch_orthogonalize_small(sb200_ctx* ctx, const OrthCall& q, cudaStream_t stream)
{
    return with_small_type(q.type, [&](auto t) -> int {
        using T = decltype(t);
        SmallParams p{};
        p.q = q;
        p.tall = q.rows > q.cols;
        p.R = static_cast<int>(p.tall ? q.cols : q.rows);
        p.C = static_cast<int>(p.tall ? q.rows : q.cols);
        // The sum over the cluster costs about 4 us a step, 256 columns a CTA instead of 128 about
        // as much: one CTA up to 256 columns, then as many as give each 128.
        p.ctas = 1;
        if (p.C > SMALL_W)
            while (p.ctas < largest_cluster<T>(ctx) && p.ctas * 128 < p.C) p.ctas *= 2;
        p.W = ((p.C + p.ctas - 1) / p.ctas + 63) / 64 * 64;
        p.status = ctx->d_status;
        p.wait_limit_ns = ctx->wait_limit_ns;
        p.test_stall_kb = ctx->test_stall_kb;
        cudaLaunchAttribute attr[2];
        const cudaLaunchConfig_t cfg = small_config<T>(attr, q.batch, p.ctas, stream);
        const cudaError_t err = cudaLaunchKernelEx(&cfg, orth_small_kernel<T>, p);
        ctx->launches += 1;
        return err == cudaSuccess && cudaGetLastError() == cudaSuccess ? SB200_OK : SB200_ERR_CUDA;
    });
}

}  // namespace sb200
