// Layer norm over the last dimension, forward and backward.
//
//   mean = sum_j x_j / n          rstd = (sum_j (x_j - mean)^2 / n + eps)^-1/2
//   h_j = (x_j - mean) rstd       y_j = h_j w_j + b_j
//   g_j = dy_j w_j                dx_j = rstd (g_j - sum_k g_k / n - h_j sum_k g_k h_k / n)
//   dw_j = sum_rows dy_j h_j      db_j = sum_rows dy_j
//
// Memory bound: the forward pass has to read x and write y, the backward pass to read
// x and dy and write dx.  A row is read once, held in the registers of the threads that
// share it (a group of 1 to 32 lanes, or a block of up to 512 threads, 16 elements a
// thread), and its sums are taken over those registers, so the variance is the mean of
// squared differences from the mean, not a difference of large sums.  All sums are
// fp32.  The blocks walk over rows; in the backward pass every thread therefore keeps
// the column sums of its own columns in registers over all the rows its block sees,
// writes one partial sum a block, and a second kernel adds the partials in block order:
// no atomics, the same bits run to run.
#include "typed.cuh"

namespace sb200 {
namespace {

constexpr int EPT = 16;                 // elements of a row per thread
constexpr int MAX_THREADS = 512;        // threads per row at most
constexpr int REGISTER_COLS = EPT * MAX_THREADS;
constexpr int GROUP_BLOCK = 256;        // block size when a row belongs to a warp or less

// Sum over the threads that share a row.  WARP: the `lanes` (power of two) neighbouring
// lanes; otherwise the block, through one barrier: callers alternate between two
// buffers, so that a buffer is written again only after a later barrier.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, int lanes, float* buf)
{
    if constexpr (WARP) {
        for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    } else {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
        __syncthreads();
        float s = 0.0f;
        for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) s += buf[i];
        return s;
    }
}

template <typename W, int VEC>
__device__ __forceinline__ void load_weight(float (&f)[VEC], const W* w, int64_t col, float none)
{
    if (w) {
        load_f<false>(f, w + col);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = none;
    }
}

// `lanes` threads per row (blockDim.x of them when WARP is false).
template <typename T, typename W, int VEC, bool WARP>
__global__ void __launch_bounds__(MAX_THREADS)
ln_forward_kernel(T* y, int64_t ldy, float* __restrict__ mean_out, float* __restrict__ rstd_out, const T* x,
                  int64_t ldx, const W* __restrict__ w, const W* __restrict__ b, int64_t rows, int cols, float eps,
                  int lanes)
{
    constexpr int NV = EPT / VEC;
    __shared__ float buf[2][MAX_THREADS / 32];
    const int lane = WARP ? (threadIdx.x & (lanes - 1)) : threadIdx.x;
    const int64_t group = WARP ? (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / lanes : blockIdx.x;
    const int64_t groups = WARP ? static_cast<int64_t>(gridDim.x) * blockDim.x / lanes : gridDim.x;
    const int nvec = cols / VEC;
    const float inv_n = 1.0f / static_cast<float>(cols);
    // every lane of a warp makes the same number of trips: the shuffles name all of them
    const int64_t first = WARP ? group - (threadIdx.x & 31) / lanes : group;
    for (int64_t r0 = first; r0 < rows; r0 += groups) {
        const int64_t r = r0 + (group - first);
        const bool mine = r < rows;
        Raw<T, VEC> raw[NV];
        const T* xr = x + r * ldx;
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int v = s * lanes + lane;
            if (mine && v < nvec) load_raw<true>(raw[s], xr + static_cast<int64_t>(v) * VEC);
        }
        float f[EPT], sum = 0.0f;
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const bool in = mine && s * lanes + lane < nvec;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                f[s * VEC + i] = in ? to_f(raw[s].e[i]) : 0.0f;
                sum += f[s * VEC + i];
            }
        }
        const float mean = row_sum<WARP>(sum, lanes, buf[0]) * inv_n;
        float sq = 0.0f;
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const bool in = s * lanes + lane < nvec;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                f[s * VEC + i] -= mean;
                if (in) sq = fmaf(f[s * VEC + i], f[s * VEC + i], sq);
            }
        }
        const float var = row_sum<WARP>(sq, lanes, buf[1]) * inv_n;
        const float rstd = 1.0f / sqrtf(var + eps);
        if (mine && lane == 0) {
            if (mean_out) mean_out[r] = mean;
            if (rstd_out) rstd_out[r] = rstd;
        }
        T* yr = y + r * ldy;
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int v = s * lanes + lane;
            if (!mine || v >= nvec) continue;
            float wf[VEC], bf[VEC], o[VEC];
            load_weight(wf, w, static_cast<int64_t>(v) * VEC, 1.0f);
            load_weight(bf, b, static_cast<int64_t>(v) * VEC, 0.0f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = fmaf(f[s * VEC + i] * rstd, wf[i], bf[i]);
            store_f<true>(yr + static_cast<int64_t>(v) * VEC, o);
        }
    }
}

// Rows too long for registers: three passes over the row, which the caches hold.
template <typename T, typename W>
__global__ void __launch_bounds__(MAX_THREADS)
ln_forward_long_kernel(T* y, int64_t ldy, float* __restrict__ mean_out, float* __restrict__ rstd_out, const T* x,
                       int64_t ldx, const W* __restrict__ w, const W* __restrict__ b, int64_t rows, int64_t cols,
                       float eps)
{
    __shared__ float buf[2][MAX_THREADS / 32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        float sum = 0.0f;
        for (int64_t j = threadIdx.x; j < cols; j += blockDim.x) sum += to_f(xr[j]);
        const float mean = row_sum<false>(sum, 0, buf[0]) / static_cast<float>(cols);
        float sq = 0.0f;
        for (int64_t j = threadIdx.x; j < cols; j += blockDim.x) {
            const float d = to_f(xr[j]) - mean;
            sq = fmaf(d, d, sq);
        }
        const float rstd = 1.0f / sqrtf(row_sum<false>(sq, 0, buf[1]) / static_cast<float>(cols) + eps);
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[r] = mean;
            if (rstd_out) rstd_out[r] = rstd;
        }
        T* yr = y + r * ldy;
        for (int64_t j = threadIdx.x; j < cols; j += blockDim.x)
            yr[j] = from_f<T>(fmaf((to_f(xr[j]) - mean) * rstd, w ? to_f(w[j]) : 1.0f, b ? to_f(b[j]) : 0.0f));
    }
}

// ---------------------------------------------------------------- backward pass

// partial: [2][gridDim.x][cols] column sums of this block's rows (dweight, then dbias), or null.
// Dynamic shared memory (WARP, partial != null): 2 * cols floats.
template <typename T, typename W, int VEC, bool WARP>
__global__ void __launch_bounds__(MAX_THREADS)
ln_backward_kernel(T* dx, int64_t lddx, float* __restrict__ partial, const T* dy, int64_t lddy, const T* x,
                   int64_t ldx, const W* __restrict__ w, const float* __restrict__ mean_in,
                   const float* __restrict__ rstd_in, int64_t rows, int cols, int accumulate, int lanes)
{
    constexpr int NV = EPT / VEC;
    __shared__ float buf[4][MAX_THREADS / 32];
    extern __shared__ float cols_sum[];
    const int lane = WARP ? (threadIdx.x & (lanes - 1)) : threadIdx.x;
    const int64_t group = WARP ? (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / lanes : blockIdx.x;
    const int64_t groups = WARP ? static_cast<int64_t>(gridDim.x) * blockDim.x / lanes : gridDim.x;
    const int nvec = cols / VEC;
    const float inv_n = 1.0f / static_cast<float>(cols);
    float dw[EPT], db[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) dw[i] = db[i] = 0.0f;
    const int64_t first = WARP ? group - (threadIdx.x & 31) / lanes : group;
    int flip = 0;
    for (int64_t r0 = first; r0 < rows; r0 += groups, flip ^= 2) {
        const int64_t r = r0 + (group - first);
        const bool mine = r < rows;
        Raw<T, VEC> rx[NV], ry[NV];
        const T* xr = x + r * ldx;
        const T* yr = dy + r * lddy;
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int v = s * lanes + lane;
            if (mine && v < nvec) {
                load_raw<true>(rx[s], xr + static_cast<int64_t>(v) * VEC);
                load_raw<true>(ry[s], yr + static_cast<int64_t>(v) * VEC);
            }
        }
        const float mean = mine ? mean_in[r] : 0.0f, rstd = mine ? rstd_in[r] : 0.0f;
        float h[EPT], g[EPT], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int v = s * lanes + lane;
            if (mine && v < nvec) {
                float wf[VEC];
                load_weight(wf, w, static_cast<int64_t>(v) * VEC, 1.0f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const int k = s * VEC + i;
                    const float d = to_f(ry[s].e[i]);
                    h[k] = (to_f(rx[s].e[i]) - mean) * rstd;
                    dw[k] = fmaf(d, h[k], dw[k]);
                    db[k] += d;
                    g[k] = d * wf[i];
                    s1 += g[k];
                    s2 = fmaf(g[k], h[k], s2);
                }
            }
        }
        const float m1 = row_sum<WARP>(s1, lanes, buf[flip]) * inv_n;
        const float m2 = row_sum<WARP>(s2, lanes, buf[flip + 1]) * inv_n;
        if (dx) {
            T* dr = dx + r * lddx;
#pragma unroll
            for (int s = 0; s < NV; ++s) {
                const int v = s * lanes + lane;
                if (!mine || v >= nvec) continue;
                float o[VEC];
                if (accumulate) {
                    load_f<true>(o, dr + static_cast<int64_t>(v) * VEC);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) o[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const int k = s * VEC + i;
                    o[i] += rstd * (g[k] - m1 - h[k] * m2);
                }
                store_f<true>(dr + static_cast<int64_t>(v) * VEC, o);
            }
        }
    }
    if (!partial) return;
    float* pw = partial + static_cast<int64_t>(blockIdx.x) * cols;
    float* pb = pw + static_cast<int64_t>(gridDim.x) * cols;
    if (!WARP) {
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int v = s * lanes + lane;
            if (v >= nvec) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                pw[v * VEC + i] = dw[s * VEC + i];
                pb[v * VEC + i] = db[s * VEC + i];
            }
        }
        return;
    }
    // the groups of the block one after another, in order
    for (int j = threadIdx.x; j < 2 * cols; j += blockDim.x) cols_sum[j] = 0.0f;
    const int my_group = threadIdx.x / lanes;
    for (int gi = 0; gi < static_cast<int>(blockDim.x) / lanes; ++gi) {
        __syncthreads();
        if (gi != my_group) continue;
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int v = s * lanes + lane;
            if (v >= nvec) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                cols_sum[v * VEC + i] += dw[s * VEC + i];
                cols_sum[cols + v * VEC + i] += db[s * VEC + i];
            }
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < cols; j += blockDim.x) {
        pw[j] = cols_sum[j];
        pb[j] = cols_sum[cols + j];
    }
}

// Rows too long for registers: dx with two passes over the row, column sums separately.
template <typename T, typename W>
__global__ void __launch_bounds__(MAX_THREADS)
ln_backward_long_kernel(T* dx, int64_t lddx, const T* dy, int64_t lddy, const T* x, int64_t ldx,
                        const W* __restrict__ w, const float* __restrict__ mean_in,
                        const float* __restrict__ rstd_in, int64_t rows, int64_t cols, int accumulate)
{
    __shared__ float buf[4][MAX_THREADS / 32];
    int flip = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, flip ^= 2) {
        const T* xr = x + r * ldx;
        const T* yr = dy + r * lddy;
        const float mean = mean_in[r], rstd = rstd_in[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t j = threadIdx.x; j < cols; j += blockDim.x) {
            const float g = to_f(yr[j]) * (w ? to_f(w[j]) : 1.0f);
            s1 += g;
            s2 = fmaf(g, (to_f(xr[j]) - mean) * rstd, s2);
        }
        const float m1 = row_sum<false>(s1, 0, buf[flip]) / static_cast<float>(cols);
        const float m2 = row_sum<false>(s2, 0, buf[flip + 1]) / static_cast<float>(cols);
        T* dr = dx + r * lddx;
        for (int64_t j = threadIdx.x; j < cols; j += blockDim.x) {
            const float g = to_f(yr[j]) * (w ? to_f(w[j]) : 1.0f);
            const float h = (to_f(xr[j]) - mean) * rstd;
            const float o = rstd * (g - m1 - h * m2);
            dr[j] = from_f<T>(accumulate ? to_f(dr[j]) + o : o);
        }
    }
}

// Partial column sums of a slice of rows, one thread a column: the layout of ln_backward_kernel's partial.
template <typename T>
__global__ void __launch_bounds__(256)
ln_backward_long_cols_kernel(float* __restrict__ partial, const T* __restrict__ dy, int64_t lddy,
                             const T* __restrict__ x, int64_t ldx, const float* __restrict__ mean_in,
                             const float* __restrict__ rstd_in, int64_t rows, int64_t cols)
{
    const int64_t j = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (j >= cols) return;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    float dw = 0.0f, db = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const float d = to_f(dy[r * lddy + j]);
        dw = fmaf(d, (to_f(x[r * ldx + j]) - mean_in[r]) * rstd_in[r], dw);
        db += d;
    }
    partial[blockIdx.y * cols + j] = dw;
    partial[(gridDim.y + blockIdx.y) * cols + j] = db;
}

// out[j] (+)= sum over `parts` partials, in order within each of 32 slices, then slice by slice.
template <typename W>
__global__ void __launch_bounds__(1024)
ln_reduce_kernel(W* __restrict__ dweight, W* __restrict__ dbias, const float* __restrict__ partial, int parts,
                 int64_t cols, int accumulate)
{
    __shared__ float sh[32][33];
    W* out = blockIdx.y ? dbias : dweight;
    if (!out) return;
    const float* src = partial + static_cast<int64_t>(blockIdx.y) * parts * cols;
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    const int per = (parts + 31) / 32;
    float s = 0.0f;
    if (j < cols) {
        const int end = min(parts, (slice + 1) * per);
#pragma unroll 4
        for (int p = slice * per; p < end; ++p) s += src[p * cols + j];
    }
    sh[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && j < cols) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += sh[i][lane];
        out[j] = from_f<W>(accumulate ? to_f(out[j]) + t : t);
    }
}

// ------------------------------------------------------------------------- host

struct Shape {
    int64_t rows, cols;
    bool vec;           // 16-byte accesses are allowed
    bool is_long;
    int lanes, block;   // threads per row, threads per block
    int64_t grid;       // blocks: enough to fill the device, no more than there is work
};

int power_of_two_at_least(int64_t n)
{
    int p = 1;
    while (p < n) p <<= 1;
    return p;
}

Shape shape_of(int sm_count, int64_t rows, int64_t cols, int vec_elems, bool vec)
{
    Shape s{};
    s.rows = rows;
    s.cols = cols;
    s.vec = vec;
    s.is_long = cols > REGISTER_COLS;
    const int64_t nvec = vec ? cols / vec_elems : cols;
    const int64_t slots = vec ? EPT / vec_elems : EPT;
    const int64_t threads = (nvec + slots - 1) / slots;
    if (s.is_long) {
        s.lanes = s.block = MAX_THREADS;
    } else if (threads <= 32) {
        s.lanes = power_of_two_at_least(threads);
        s.block = GROUP_BLOCK;
    } else {
        s.lanes = s.block = static_cast<int>((threads + 31) / 32 * 32);
    }
    const int64_t per_block = s.block / s.lanes;
    const int64_t want = (rows + per_block - 1) / per_block;
    const int64_t fill = static_cast<int64_t>(sm_count) * (1024 / s.block);
    s.grid = want < fill ? want : fill;
    return s;
}

int check_types(int type, int weight_type)
{
    if (!known_type(type) || !known_type(weight_type)) return SB200_ERR_INVALID_ARG;
    if (weight_type != SB200_F32 && weight_type != type) return SB200_ERR_UNSUPPORTED;
    return SB200_OK;
}

// f(T{}, W{}) for the element types named by the ABI's codes
template <typename F>
int with_types(int type, int weight_type, F f)
{
    if (type == SB200_F32) return f(float{}, float{});
    if (type == SB200_BF16) return weight_type == SB200_F32 ? f(bf16{}, float{}) : f(bf16{}, bf16{});
    return weight_type == SB200_F32 ? f(f16{}, float{}) : f(f16{}, f16{});
}

// The number of partial column sums of the backward pass depends on the device and the
// shape alone, not on alignment: both kernels of a row length get the same count.
int64_t backward_parts(int sm_count, int64_t rows, int64_t cols)
{
    if (cols > REGISTER_COLS) {
        const int64_t tiles = (cols + 255) / 256;
        int64_t slices = (8ll * sm_count + tiles - 1) / tiles;
        if (slices > rows) slices = rows;
        return slices < 1 ? 1 : slices;
    }
    // one block per SM at least; two when there are many rows
    return 2ll * sm_count < rows ? 2ll * sm_count : (rows < 1 ? 1 : rows);
}

}  // namespace
}  // namespace sb200

using namespace sb200;

extern "C" int sb200_layer_norm(sb200_ctx* ctx, void* y, int64_t ldy, float* mean, float* rstd, const void* x,
                                int64_t ldx, const void* weight, const void* bias, int64_t rows, int64_t cols,
                                float eps, int type, int weight_type, sb200_stream stream_)
{
    TraceRange trace("sb200_layer_norm");
    if (!ctx || rows < 0 || cols < 1 || ldx < cols || ldy < cols || !(eps >= 0.0f)) return SB200_ERR_INVALID_ARG;
    if (const int rc = check_types(type, weight_type)) return rc;
    if (rows == 0) return SB200_OK;
    if (!x || !y) return SB200_ERR_INVALID_ARG;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    return with_types(type, weight_type, [&](auto t, auto wt) {
        using T = decltype(t);
        using W = decltype(wt);
        constexpr int VEC = 16 / sizeof(T);
        const bool vec = cols % VEC == 0 && ldx % VEC == 0 && ldy % VEC == 0 && aligned_to(x, 16) && aligned_to(y, 16) &&
                         aligned_to(weight, 16) && aligned_to(bias, 16);
        const Shape s = shape_of(ctx->sm_count, rows, cols, VEC, vec);
        const unsigned grid = static_cast<unsigned>(s.grid);
        T* yp = static_cast<T*>(y);
        const T* xp = static_cast<const T*>(x);
        const W* wp = static_cast<const W*>(weight);
        const W* bp = static_cast<const W*>(bias);
        const int n = static_cast<int>(s.is_long ? 0 : cols);
        if (s.is_long)
            ln_forward_long_kernel<T, W><<<grid, s.block, 0, stream>>>(yp, ldy, mean, rstd, xp, ldx, wp, bp, rows, cols, eps);
        else if (s.lanes <= 32 && vec)
            ln_forward_kernel<T, W, VEC, true><<<grid, s.block, 0, stream>>>(yp, ldy, mean, rstd, xp, ldx, wp, bp, rows, n, eps, s.lanes);
        else if (s.lanes <= 32)
            ln_forward_kernel<T, W, 1, true><<<grid, s.block, 0, stream>>>(yp, ldy, mean, rstd, xp, ldx, wp, bp, rows, n, eps, s.lanes);
        else if (vec)
            ln_forward_kernel<T, W, VEC, false><<<grid, s.block, 0, stream>>>(yp, ldy, mean, rstd, xp, ldx, wp, bp, rows, n, eps, s.lanes);
        else
            ln_forward_kernel<T, W, 1, false><<<grid, s.block, 0, stream>>>(yp, ldy, mean, rstd, xp, ldx, wp, bp, rows, n, eps, s.lanes);
        ctx->launches += 1;
        return cudaGetLastError() == cudaSuccess ? SB200_OK : SB200_ERR_CUDA;
    });
}

extern "C" int64_t sb200_layer_norm_backward_workspace(const sb200_ctx* ctx, int64_t rows, int64_t cols)
{
    if (!ctx || rows < 0 || cols < 1) return -1;
    return backward_parts(ctx->sm_count, rows, cols) * cols * 2 * static_cast<int64_t>(sizeof(float));
}

extern "C" int sb200_layer_norm_backward(sb200_ctx* ctx, void* dx, int64_t lddx, void* dweight, void* dbias,
                                         const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight,
                                         const float* mean, const float* rstd, int64_t rows, int64_t cols, int type,
                                         int weight_type, int accumulate_dx, int accumulate_weight, void* workspace,
                                         int64_t workspace_bytes, sb200_stream stream_)
{
    TraceRange trace("sb200_layer_norm_backward");
    if (!ctx || rows < 0 || cols < 1 || ldx < cols || lddy < cols || (dx && lddx < cols)) return SB200_ERR_INVALID_ARG;
    if (const int rc = check_types(type, weight_type)) return rc;
    if (rows > 0 && (!x || !dy || !mean || !rstd)) return SB200_ERR_INVALID_ARG;
    const bool sums = dweight || dbias;
    if (sums && (!workspace || !aligned_to(workspace, 16) ||
                 workspace_bytes < sb200_layer_norm_backward_workspace(ctx, rows, cols)))
        return SB200_ERR_INVALID_ARG;
    if (!sums && (!dx || rows == 0)) return SB200_OK;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    float* partial = sums ? static_cast<float*>(workspace) : nullptr;
    return with_types(type, weight_type, [&](auto t, auto wt) {
        using T = decltype(t);
        using W = decltype(wt);
        constexpr int VEC = 16 / sizeof(T);
        T* dxp = static_cast<T*>(dx);
        const T* yp = static_cast<const T*>(dy);
        const T* xp = static_cast<const T*>(x);
        const W* wp = static_cast<const W*>(weight);
        int parts = 0;
        if (rows > 0) {
            const bool vec = cols % VEC == 0 && ldx % VEC == 0 && lddy % VEC == 0 && aligned_to(x, 16) &&
                             aligned_to(dy, 16) && aligned_to(weight, 16) &&
                             (!dx || (lddx % VEC == 0 && aligned_to(dx, 16)));
            const Shape s = shape_of(ctx->sm_count, rows, cols, VEC, vec);
            const int64_t most = backward_parts(ctx->sm_count, rows, cols);
            if (s.is_long) {
                // the column sums first: dx may overwrite dy
                if (sums) {
                    parts = static_cast<int>(most);
                    const dim3 grid(static_cast<unsigned>((cols + 255) / 256), static_cast<unsigned>(parts));
                    ln_backward_long_cols_kernel<T><<<grid, 256, 0, stream>>>(partial, yp, lddy, xp, ldx, mean, rstd, rows, cols);
                    ctx->launches += 1;
                }
                if (dx) {
                    ln_backward_long_kernel<T, W><<<static_cast<unsigned>(s.grid), s.block, 0, stream>>>(
                        dxp, lddx, yp, lddy, xp, ldx, wp, mean, rstd, rows, cols, accumulate_dx);
                    ctx->launches += 1;
                }
            } else {
                const int64_t want = s.grid < most ? s.grid : most;
                parts = static_cast<int>(want);
                const unsigned grid = static_cast<unsigned>(want);
                const int n = static_cast<int>(cols);
                const size_t smem = s.lanes <= 32 && sums ? static_cast<size_t>(2 * cols) * sizeof(float) : 0;
                if (s.lanes <= 32 && vec)
                    ln_backward_kernel<T, W, VEC, true><<<grid, s.block, smem, stream>>>(dxp, lddx, partial, yp, lddy, xp, ldx, wp, mean, rstd, rows, n, accumulate_dx, s.lanes);
                else if (s.lanes <= 32)
                    ln_backward_kernel<T, W, 1, true><<<grid, s.block, smem, stream>>>(dxp, lddx, partial, yp, lddy, xp, ldx, wp, mean, rstd, rows, n, accumulate_dx, s.lanes);
                else if (vec)
                    ln_backward_kernel<T, W, VEC, false><<<grid, s.block, 0, stream>>>(dxp, lddx, partial, yp, lddy, xp, ldx, wp, mean, rstd, rows, n, accumulate_dx, s.lanes);
                else
                    ln_backward_kernel<T, W, 1, false><<<grid, s.block, 0, stream>>>(dxp, lddx, partial, yp, lddy, xp, ldx, wp, mean, rstd, rows, n, accumulate_dx, s.lanes);
                ctx->launches += 1;
            }
        }
        if (sums) {
            const dim3 grid(static_cast<unsigned>((cols + 31) / 32), 2);
            ln_reduce_kernel<W><<<grid, 1024, 0, stream>>>(static_cast<W*>(dweight), static_cast<W*>(dbias), partial, parts, cols, accumulate_weight);
            ctx->launches += 1;
        }
        return cudaGetLastError() == cudaSuccess ? SB200_OK : SB200_ERR_CUDA;
    });
}
