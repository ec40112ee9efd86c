// Layer norm over the last dimension, forward and backward.
//
//   mean = sum_j x_j / n          rstd = (sum_j (x_j - mean)^2 / n + eps)^-1/2
//   h_j = (x_j - mean) rstd       y_j = h_j w_j + b_j
//   g_j = dy_j w_j                dx_j = rstd (g_j - sum_k g_k / n - h_j sum_k g_k h_k / n)
//   dw_j = sum_rows dy_j h_j      db_j = sum_rows dy_j
//
// Memory bound: the forward pass has to read x and write y, the backward pass to read
// x and dy and write dx.  A row is read once, held in the registers of the threads that
// share it (a group of 1 to 32 lanes, or a block of up to 512 threads; 16 elements a
// thread, in the forward pass 32 where rows have more than 512), and its sums are taken over those registers, so the variance is the mean of
// squared differences from a mean, not a difference of large sums.  All sums are fp32.
// The blocks walk over rows; each thread keeps its columns' weights in registers and has
// its pieces of the next rows on the way into shared memory (its own slots, so nothing
// but the thread itself waits for them): the memory system always has several rows a
// block to work on, which one row at a time in registers does not give it (65536 x 4096
// bf16 forward: 291 us, so 180 to 193 or 5.6 to 6.0 TB/s; 32768 x 4096 fp32 backward: 238 to
// 251 us, 6.4 to 6.8 TB/s).  In the backward pass every thread keeps the column sums of its
// columns in registers over all the rows its block sees, writes one partial sum a block,
// and a second kernel adds the partials in block order: no atomics, the same bits run to
// run.  Rows that 16-byte accesses do not fit take 4-byte ones.  Odd rows of 16-bit elements
// take 16-byte ones all the same where all arrays' rows start at the same distance from a
// boundary: the grid makes steps of 8 rows, so that the distance is a thread's own and its
// columns stay (16384 x 4095 bf16: forward 225 -> 128 us, backward 474 -> 169), else 2-byte ones.
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "ptx.cuh"
#include "typed.cuh"

namespace sb200 {
namespace {

constexpr int EPT = 16;                 // elements of a row per thread (backward pass)
constexpr int MAX_THREADS = 512;        // threads per row at most
constexpr int MAX_WARPS = MAX_THREADS / 32;
constexpr int REGISTER_COLS = EPT * MAX_THREADS;
constexpr int GROUP_BLOCK = 256;        // block size when a row belongs to a warp or less

// A thread's pieces of the coming rows of one array, in shared memory: STAGES rows of E
// elements, piece s of stage k at [(k * NV + s) * blockDim + thread].  2-byte accesses have
// no asynchronous form: those pieces are read when the row is due.
template <typename T, int VEC, int E>
struct Pieces {
    static constexpr int NV = E / VEC, BYTES = VEC * static_cast<int>(sizeof(T));
    static constexpr bool ASYNC = BYTES >= 4;
    static_assert(BYTES == 2 || BYTES == 4 || BYTES == 16, "access width");
    static constexpr int STAGES = !ASYNC ? 1 : sizeof(T) == 4 ? 3 : 4, AHEAD = STAGES - 1;
    static constexpr int SMEM = ASYNC ? STAGES * E * static_cast<int>(sizeof(T)) : 0;      // per thread

    Raw<T, VEC> next[ASYNC ? 1 : NV];
    unsigned char* base;

    // The pieces of a row that starts `shift` elements behind a 16-byte boundary (SHIFT): piece v
    // holds elements v VEC - shift and the following ones.  What lies before the row comes
    // along in the first piece (clean() makes it zero), except where that is not of the array.
    __device__ void request_shifted(const T* row, bool in, bool at_start, int stage, int lane, int lanes, int nvec, int cols, int shift)
    {
        if (!in) return;
        if constexpr (BYTES == 16) {
#pragma unroll 4
            for (int s = 0; s < NV; ++s) {
                const int v = s * lanes + lane;
                if (v >= nvec) break;
                const int at = v * VEC - shift, end = cols - at < VEC ? cols - at : VEC;
                if (at < 0 && at_start) {
                    T* to = reinterpret_cast<T*>(slot(stage, s));
                    for (int i = -at; i < VEC; ++i) to[i] = i < end ? row[at + i] : from_f<T>(0.0f);
                } else {
                    ptx::cp_async_16(slot(stage, s), row + at, end * static_cast<int>(sizeof(T)));
                }
            }
        }
    }
    __device__ void clean(int stage, int lane, int shift)
    {
        if (lane == 0)
            for (int i = 0; i < shift; ++i) reinterpret_cast<T*>(slot(stage, 0))[i] = from_f<T>(0.0f);
    }

    // pieces beyond the row are zero and stay so
    __device__ void init(unsigned char* smem, int lane, int lanes, int nvec)
    {
        base = smem + threadIdx.x * BYTES;
        Raw<T, VEC> zero;
#pragma unroll
        for (int i = 0; i < VEC; ++i) zero.e[i] = from_f<T>(0.0f);
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            if constexpr (ASYNC) {
                for (int k = 0; k < STAGES; ++k)
                    if (s * lanes + lane >= nvec) store_raw<false>(reinterpret_cast<T*>(slot(k, s)), zero);
            } else {
                next[s] = zero;
            }
        }
    }
    __device__ unsigned char* slot(int stage, int s) const { return base + (stage * NV + s) * static_cast<int>(blockDim.x) * BYTES; }

    // the pieces of the row at `row` (in: whether there is one) into a stage
    __device__ void request(const T* row, bool in, int stage, int lane, int lanes, int nvec)
    {
        if (!in) return;
        row += static_cast<int64_t>(lane) * VEC;
        if constexpr (ASYNC) {
#pragma unroll 4
            for (int s = 0; s < NV; ++s) {
                if (s * lanes + lane >= nvec) break;
                if constexpr (BYTES == 16) ptx::cp_async_16(slot(stage, s), row, 16);
                else ptx::cp_async_4(slot(stage, s), row);
                row += lanes * VEC;
            }
        } else {
#pragma unroll
            for (int s = 0; s < NV; ++s)
                if (s * lanes + lane < nvec) load_raw<true>(next[s], row + s * lanes * VEC);
        }
    }
    __device__ void get(Raw<T, VEC>& r, int stage, int s) const
    {
        if constexpr (ASYNC) load_raw<false>(r, reinterpret_cast<const T*>(slot(stage, s)));
        else r = next[s];
    }
};

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

// Elements from a 16-byte boundary to the start of row r.
template <typename T>
__device__ __forceinline__ int row_shift(const T* x, int64_t ldx, int64_t r)
{
    return static_cast<int>((reinterpret_cast<uintptr_t>(x) / sizeof(T) + static_cast<uintptr_t>(r * ldx)) % (16 / sizeof(T)));
}

__device__ __forceinline__ float lanes_sum(float v, int lanes)
{
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// E elements of this thread's pieces as pairs: pair j holds elements 2 j and 2 j + 1, of
// two pieces when a piece is one element.
template <int VEC, int E, typename P, typename T>
__device__ __forceinline__ void get_pairs(float2 (&f)[E / 2], const P& pieces, int stage)
{
#pragma unroll
    for (int s = 0; s < P::NV; s += VEC == 1 ? 2 : 1) {
        Raw<T, VEC> a;
        pieces.get(a, stage, s);
        if constexpr (VEC == 1) {
            Raw<T, VEC> b;
            pieces.get(b, stage, s + 1);
            f[s / 2] = make_float2(to_f(a.e[0]), to_f(b.e[0]));
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i += 2) f[(s * VEC + i) / 2] = pair_f(a.e + i);
        }
    }
}

// This thread's weights, in the same order; `none` where there are none.
template <int VEC, int E, bool SHIFT, typename W>
__device__ __forceinline__ void get_weights(float2 (&f)[E / 2], const W* w, float none, int lane, int lanes, int nvec, int cols,
                                            int shift)
{
    float* one = reinterpret_cast<float*>(f);
#pragma unroll
    for (int s = 0; s < E / VEC; ++s) {
        float a[VEC];
        const int v = s * lanes + lane;
#pragma unroll
        for (int i = 0; i < VEC; ++i) a[i] = none;
        if constexpr (SHIFT) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int j = v * VEC - shift + i;
                if (w && j >= 0 && j < cols) a[i] = to_f(w[j]);
            }
        } else {
            if (w && v < nvec) load_f<false>(a, w + static_cast<int64_t>(v) * VEC);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) one[s * VEC + i] = a[i];
    }
}

// Which of this thread's elements are in the row.
template <int VEC, int E>
__device__ __forceinline__ uint32_t valid_elements(int lane, int lanes, int cols, int shift)
{
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int j = (e / VEC * lanes + lane) * VEC - shift + e % VEC;
        if (j >= 0 && j < cols) bits |= 1u << e;
    }
    return bits;
}

// Elements that are not in the row become x.
template <int E>
__device__ __forceinline__ void fill_invalid(float2 (&f)[E / 2], uint32_t valid, float x)
{
    if (valid == (E == 32 ? 0xffffffffu : (1u << (E & 31)) - 1u)) return;
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
        if (!((valid >> (2 * j)) & 1u)) f[j].x = x;
        if (!((valid >> (2 * j + 1)) & 1u)) f[j].y = x;
    }
}

// The pairs back into pieces of a row.
template <int VEC, int E, bool SHIFT, typename T>
__device__ __forceinline__ void put_pairs(T* row, const float2 (&f)[E / 2], int lane, int lanes, int nvec, uint32_t valid, int shift)
{
    row += static_cast<int64_t>(lane) * VEC - (SHIFT ? shift : 0);
#pragma unroll
    for (int s = 0; s < E / VEC; ++s) {
        if constexpr (SHIFT) {
            const uint32_t bits = (valid >> (s * VEC)) & ((1u << VEC) - 1u);
            Raw<T, VEC> r;
#pragma unroll
            for (int i = 0; i < VEC; i += 2) set_pair(r.e + i, f[(s * VEC + i) / 2]);
            if (bits == (1u << VEC) - 1u) {
                store_raw<true>(row + s * lanes * VEC, r);
            } else if (bits) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if ((bits >> i) & 1u) row[s * lanes * VEC + i] = r.e[i];
            }
        } else if (s * lanes + lane < nvec) {
            Raw<T, VEC> r;
            if constexpr (VEC == 1) {
                r.e[0] = from_f<T>(s & 1 ? f[s / 2].y : f[s / 2].x);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i += 2) set_pair(r.e + i, f[(s * VEC + i) / 2]);
            }
            store_raw<true>(row + s * lanes * VEC, r);
        }
    }
}

// `lanes` threads per row (blockDim.x of them when WARP is false), E elements each: what a
// row costs a thread beside its elements (two sums over the warp, one over the block) is as
// much as 16 elements, so rows of more than a warp get 32; pairs of elements share an
// instruction.  What bounds it is the instructions, not the memory, when rows are of 16 bits.
// SHIFT: rows that start anywhere, the same distance behind a 16-byte boundary in x and y.
// The distance is that of every row a thread sees: the grid makes steps of whole periods.
template <typename T, typename W, int VEC, int E, bool WARP, bool SHIFT>
__global__ void __maxnreg__(E == 32 || VEC == 1 || SHIFT ? 128 : 80)
ln_forward_kernel(T* y, int64_t ldy, float* __restrict__ mean_out, float* __restrict__ rstd_out, const T* x,
                  int64_t ldx, const W* __restrict__ w, const W* __restrict__ b, int64_t rows, int cols, float eps,
                  int lanes)
{
    using P = Pieces<T, VEC, E>;
    constexpr int NV = P::NV, AHEAD = P::AHEAD;
    extern __shared__ __align__(16) unsigned char smem[];
    // a warp's sum and sum of squared differences from its own mean; two buffers, so that
    // one barrier a row is enough: a buffer is written again behind the other one's barrier
    __shared__ float2 part[2][MAX_WARPS], count[MAX_WARPS];      // count: elements of a warp, and 1 / that
    const int lane = WARP ? (threadIdx.x & (lanes - 1)) : threadIdx.x;
    const int64_t group = WARP ? (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / lanes : blockIdx.x;
    const int64_t groups = WARP ? static_cast<int64_t>(gridDim.x) * blockDim.x / lanes : gridDim.x;
    const int shift = SHIFT ? row_shift(x, ldx, group) : 0, nvec = SHIFT ? (cols + shift + VEC - 1) / VEC : cols / VEC;
    const uint32_t valid = SHIFT ? valid_elements<VEC, E>(lane, lanes, cols, shift) : 0;
    const float inv_n = 1.0f / static_cast<float>(cols);
    // elements in this thread's warp (or group)
    int mine = SHIFT ? __popc(valid) : 0;
#pragma unroll
    for (int s = 0; s < NV; ++s)
        if (!SHIFT) mine += s * lanes + lane < nvec ? VEC : 0;
    const float warp_n = lanes_sum(static_cast<float>(mine), WARP ? lanes : 32);
    const float warp_inv = warp_n > 0.0f ? 1.0f / warp_n : 0.0f;
    if (!WARP && (threadIdx.x & 31) == 0) count[threadIdx.x >> 5] = make_float2(warp_n, warp_inv);   // (read behind a barrier)

    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    P px;
    px.init(smem, lane, lanes, nvec);
    // every lane of a warp makes the same number of trips: the shuffles name all of them
    const int64_t first = WARP ? group - (threadIdx.x & 31) / lanes : group;
    const int64_t off = group - first;
    auto request = [&](int64_t r, int stage) {
        if constexpr (SHIFT) px.request_shifted(x + r * ldx, r < rows, r * ldx < shift, stage, lane, lanes, nvec, cols, shift);
        else px.request(x + r * ldx, r < rows, stage, lane, lanes, nvec);
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
        const int64_t r = first + k * groups + off;
        request(r, k);
        if (P::ASYNC) ptx::cp_async_commit();
    }
    float2 wf[E / 2], bf[E / 2];
    get_weights<VEC, E, SHIFT>(wf, w, 1.0f, lane, lanes, nvec, cols, shift);
    get_weights<VEC, E, SHIFT>(bf, b, 0.0f, lane, lanes, nvec, cols, shift);
    int stage = 0, flip = 0;
    for (int64_t r0 = first; r0 < rows; r0 += groups) {
        const int64_t r = r0 + off;
        const bool has = r < rows;
        if constexpr (P::ASYNC) ptx::cp_async_wait<AHEAD - 1>();
        else request(r, 0);
        if constexpr (SHIFT) px.clean(stage, lane, shift);
        float2 f[E / 2];
        get_pairs<VEC, E, P, T>(f, px, stage);
        if constexpr (P::ASYNC) {
            request(r + AHEAD * groups, (stage + AHEAD) % P::STAGES);
            ptx::cp_async_commit();
            stage = stage + 1 == P::STAGES ? 0 : stage + 1;
        }
        float2 s2 = f[0];
#pragma unroll
        for (int j = 1; j < E / 2; ++j) s2 = add2(s2, f[j]);
        const float sum = lanes_sum(s2.x + s2.y, WARP ? lanes : 32);
        const float near = sum * warp_inv;               // the mean over this warp's elements
        float2 q2 = both(0.0f);
        if constexpr (SHIFT) fill_invalid<E>(f, valid, near);    // beyond the row: no difference
#pragma unroll
        for (int s = 0; s < NV; s += VEC == 1 ? 2 : 1) {
            const bool in = SHIFT || s * lanes + lane < nvec;
            if constexpr (VEC == 1) {
                float2 g = f[s / 2];                     // beyond the row: no difference
                if (!in) g.x = near;
                if ((s + 1) * lanes + lane >= nvec) g.y = near;
                const float2 d = add2(g, both(-near));
                q2 = fma2(d, d, q2);
            } else if (in) {
#pragma unroll
                for (int i = 0; i < VEC; i += 2) {
                    const float2 d = add2(f[(s * VEC + i) / 2], both(-near));
                    q2 = fma2(d, d, q2);
                }
            }
        }
        float sq = lanes_sum(q2.x + q2.y, WARP ? lanes : 32);
        float mean = near;
        if (!WARP) {
            // the squares from the common mean: those from the warp's own, and its distance
            float2* p = part[flip];
            flip ^= 1;
            if ((threadIdx.x & 31) == 0) p[threadIdx.x >> 5] = make_float2(sum, sq);
            __syncthreads();
            const int i = threadIdx.x & (MAX_WARPS - 1);
            const bool in = i < static_cast<int>(blockDim.x >> 5);
            const float2 q = in ? p[i] : make_float2(0.0f, 0.0f), n = in ? count[i] : make_float2(0.0f, 0.0f);
            mean = lanes_sum(q.x, MAX_WARPS) * inv_n;
            const float d = fmaf(q.x, n.y, -mean);
            sq = lanes_sum(fmaf(n.x * d, d, q.y), MAX_WARPS);
        }
        const float rstd = rsqrtf(fmaf(sq, inv_n, eps));
        if (!has) continue;
        if (lane == 0) {
            if (mean_out) mean_out[r] = mean;
            if (rstd_out) rstd_out[r] = rstd;
        }
#pragma unroll
        for (int j = 0; j < E / 2; ++j) f[j] = fma2(mul2(add2(f[j], both(-mean)), both(rstd)), wf[j], bf[j]);
        put_pairs<VEC, E, SHIFT>(y + r * ldy, f, lane, lanes, nvec, valid, shift);
    }
}

// Sum over a block (rows too long for registers); `buf` is one of two used in turn.
__device__ __forceinline__ float2 block_sum(float2 v, float2* buf)
{
    v.x = lanes_sum(v.x, 32);
    v.y = lanes_sum(v.y, 32);
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    float2 s = make_float2(0.0f, 0.0f);
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) { s.x += buf[i].x; s.y += buf[i].y; }
    return s;
}

// Rows too long for registers: three passes over the row, which the caches hold.
template <typename T, typename W, int VEC>
__global__ void __launch_bounds__(MAX_THREADS)
ln_forward_long_kernel(T* y, int64_t ldy, float* __restrict__ mean_out, float* __restrict__ rstd_out, const T* x,
                       int64_t ldx, const W* __restrict__ w, const W* __restrict__ b, int64_t rows, int64_t cols,
                       float eps)
{
    __shared__ float2 buf[2][MAX_WARPS];
    const int64_t nvec = cols / VEC;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        float sum = 0.0f;
#pragma unroll 4
        for (int64_t v = threadIdx.x; v < nvec; v += blockDim.x) {
            float f[VEC];
            load_f<false>(f, xr + v * VEC);
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum += f[i];
        }
        const float mean = block_sum(make_float2(sum, 0.0f), buf[0]).x / static_cast<float>(cols);
        float sq = 0.0f;
#pragma unroll 4
        for (int64_t v = threadIdx.x; v < nvec; v += blockDim.x) {
            float f[VEC];
            load_f<false>(f, xr + v * VEC);
#pragma unroll
            for (int i = 0; i < VEC; ++i) sq = fmaf(f[i] - mean, f[i] - mean, sq);
        }
        const float rstd = rsqrtf(block_sum(make_float2(sq, 0.0f), buf[1]).x / static_cast<float>(cols) + eps);
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[r] = mean;
            if (rstd_out) rstd_out[r] = rstd;
        }
        T* yr = y + r * ldy;
#pragma unroll 2
        for (int64_t v = threadIdx.x; v < nvec; v += blockDim.x) {
            float f[VEC], wf[VEC], bf[VEC];
            load_f<true>(f, xr + v * VEC);
            load_weight(wf, w, v * VEC, 1.0f);
            load_weight(bf, b, v * VEC, 0.0f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = fmaf((f[i] - mean) * rstd, wf[i], bf[i]);
            store_f<true>(yr + v * VEC, f);
        }
    }
}

// ---------------------------------------------------------------- backward pass

// partial: [2][gridDim.x][cols] column sums of this block's rows (dweight, then dbias), or null.
// Dynamic shared memory: the pieces of x and dy, and later (WARP, partial != null) 2 * cols floats.
template <typename T, typename W, int VEC, bool WARP, bool SHIFT>
__global__ void __launch_bounds__(MAX_THREADS)
ln_backward_kernel(T* dx, int64_t lddx, float* __restrict__ partial, const T* dy, int64_t lddy, const T* x,
                   int64_t ldx, const W* __restrict__ w, const float* __restrict__ mean_in,
                   const float* __restrict__ rstd_in, int64_t rows, int cols, int accumulate, int lanes)
{
    using P = Pieces<T, VEC, EPT>;
    constexpr int NV = P::NV, AHEAD = P::AHEAD;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float2 part[2][MAX_WARPS];                // two buffers, one barrier a row
    const int lane = WARP ? (threadIdx.x & (lanes - 1)) : threadIdx.x;
    const int64_t group = WARP ? (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / lanes : blockIdx.x;
    const int64_t groups = WARP ? static_cast<int64_t>(gridDim.x) * blockDim.x / lanes : gridDim.x;
    const int shift = SHIFT ? row_shift(x, ldx, group) : 0, nvec = SHIFT ? (cols + shift + VEC - 1) / VEC : cols / VEC;
    const uint32_t valid = valid_elements<VEC, EPT>(lane, lanes, cols, shift);
    const float inv_n = 1.0f / static_cast<float>(cols);
    P px, py;
    px.init(smem, lane, lanes, nvec);
    py.init(smem + blockDim.x * P::SMEM, lane, lanes, nvec);
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int64_t first = WARP ? group - (threadIdx.x & 31) / lanes : group;
    const int64_t off = group - first;
    auto request = [&](int64_t r, int stage) {
        if constexpr (SHIFT) {
            px.request_shifted(x + r * ldx, r < rows, r * ldx < shift, stage, lane, lanes, nvec, cols, shift);
            py.request_shifted(dy + r * lddy, r < rows, r * lddy < shift, stage, lane, lanes, nvec, cols, shift);
        } else {
            px.request(x + r * ldx, r < rows, stage, lane, lanes, nvec);
            py.request(dy + r * lddy, r < rows, stage, lane, lanes, nvec);
        }
        if (P::ASYNC) ptx::cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) request(first + k * groups + off, k);
    float2 dw2[EPT / 2], db2[EPT / 2], wf[EPT / 2];
#pragma unroll
    for (int j = 0; j < EPT / 2; ++j) dw2[j] = db2[j] = both(0.0f);
    get_weights<VEC, EPT, SHIFT>(wf, w, 1.0f, lane, lanes, nvec, cols, shift);
    float mean_next = first + off < rows ? mean_in[first + off] : 0.0f;
    float rstd_next = first + off < rows ? rstd_in[first + off] : 0.0f;
    int stage = 0, flip = 0;
    for (int64_t r0 = first; r0 < rows; r0 += groups) {
        const int64_t r = r0 + off;
        const bool has = r < rows;
        const float mean = mean_next, rstd = rstd_next;
        if constexpr (P::ASYNC) ptx::cp_async_wait<AHEAD - 1>();
        else request(r, 0);
        if constexpr (SHIFT) {
            px.clean(stage, lane, shift);
            py.clean(stage, lane, shift);
        }
        float2 h[EPT / 2], d[EPT / 2], a1 = both(0.0f), a2 = both(0.0f);
        if (!WARP || has) {
            get_pairs<VEC, EPT, P, T>(h, px, stage);
            get_pairs<VEC, EPT, P, T>(d, py, stage);
            // beyond the row dy is zero, and so is all that is added up: h must be finite there, and
            // (0 - mean) rstd need not be where the row itself is (a constant one of large numbers)
            fill_invalid<EPT>(h, valid, mean);
#pragma unroll
            for (int j = 0; j < EPT / 2; ++j) {
                h[j] = mul2(add2(h[j], both(-mean)), both(rstd));
                dw2[j] = fma2(d[j], h[j], dw2[j]);
                db2[j] = add2(db2[j], d[j]);
                d[j] = mul2(d[j], wf[j]);                // from here on dy * weight
                a1 = add2(a1, d[j]);
                a2 = fma2(d[j], h[j], a2);
            }
        }
        if (r + groups < rows) {
            mean_next = mean_in[r + groups];
            rstd_next = rstd_in[r + groups];
        }
        if constexpr (P::ASYNC) {
            request(r + AHEAD * groups, (stage + AHEAD) % P::STAGES);
            stage = stage + 1 == P::STAGES ? 0 : stage + 1;
        }
        float s1 = lanes_sum(a1.x + a1.y, WARP ? lanes : 32);
        float s2 = lanes_sum(a2.x + a2.y, WARP ? lanes : 32);
        if (!WARP) {
            float2* p = part[flip];
            flip ^= 1;
            if ((threadIdx.x & 31) == 0) p[threadIdx.x >> 5] = make_float2(s1, s2);
            __syncthreads();
            const int i = threadIdx.x & (MAX_WARPS - 1);
            const float2 q = i < static_cast<int>(blockDim.x >> 5) ? p[i] : make_float2(0.0f, 0.0f);
            s1 = lanes_sum(q.x, MAX_WARPS);
            s2 = lanes_sum(q.y, MAX_WARPS);
        }
        if (dx && has) {
            const float m1 = s1 * inv_n, m2 = s2 * inv_n;
            T* dr = dx + r * lddx;
#pragma unroll
            for (int j = 0; j < EPT / 2; ++j) d[j] = mul2(fma2(h[j], both(-m2), add2(d[j], both(-m1))), both(rstd));
            if (accumulate) {
#pragma unroll
                for (int s = 0; s < NV; ++s) {
                    if (s * lanes + lane >= nvec) continue;
                    const T* from = dr + static_cast<int64_t>(s * lanes + lane) * VEC - shift;
                    const uint32_t bits = (valid >> (s * VEC)) & ((1u << VEC) - 1u);
                    float o[VEC];
                    if (!SHIFT || bits == (1u << VEC) - 1u) {
                        load_f<true>(o, from);
                    } else {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) o[i] = (bits >> i) & 1u ? to_f(from[i]) : 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        float2& t = d[(s * VEC + i) / 2];
                        if ((s * VEC + i) & 1) t.y += o[i]; else t.x += o[i];
                    }
                }
            }
            put_pairs<VEC, EPT, SHIFT>(dr, d, lane, lanes, nvec, valid, shift);
        }
    }
    if (!partial) return;
    const float* dw = reinterpret_cast<const float*>(dw2);
    const float* db = reinterpret_cast<const float*>(db2);
    float* pw = partial + static_cast<int64_t>(blockIdx.x) * cols;
    float* pb = pw + static_cast<int64_t>(gridDim.x) * cols;
    if (!WARP) {
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int v = s * lanes + lane;
            if (v >= nvec) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (SHIFT && !((valid >> (s * VEC + i)) & 1u)) continue;
                pw[v * VEC - shift + i] = dw[s * VEC + i];
                pb[v * VEC - shift + i] = db[s * VEC + i];
            }
        }
        return;
    }
    // the groups of the block one after another, in order; the pieces' place is free
    float* cols_sum = reinterpret_cast<float*>(smem);
    __syncthreads();
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
                if (SHIFT && !((valid >> (s * VEC + i)) & 1u)) continue;
                cols_sum[v * VEC - shift + i] += dw[s * VEC + i];
                cols_sum[cols + v * VEC - shift + i] += db[s * VEC + i];
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
template <typename T, typename W, int VEC>
__global__ void __launch_bounds__(MAX_THREADS)
ln_backward_long_kernel(T* dx, int64_t lddx, const T* dy, int64_t lddy, const T* x, int64_t ldx,
                        const W* __restrict__ w, const float* __restrict__ mean_in,
                        const float* __restrict__ rstd_in, int64_t rows, int64_t cols, int accumulate)
{
    __shared__ float2 buf[2][MAX_WARPS];
    const int64_t nvec = cols / VEC;
    int flip = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, flip ^= 1) {
        const T* xr = x + r * ldx;
        const T* yr = dy + r * lddy;
        const float mean = mean_in[r], rstd = rstd_in[r];
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll 2
        for (int64_t v = threadIdx.x; v < nvec; v += blockDim.x) {
            float f[VEC], g[VEC], wf[VEC];
            load_f<false>(f, xr + v * VEC);
            load_f<false>(g, yr + v * VEC);
            load_weight(wf, w, v * VEC, 1.0f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                g[i] *= wf[i];
                s.x += g[i];
                s.y = fmaf(g[i], (f[i] - mean) * rstd, s.y);
            }
        }
        s = block_sum(s, buf[flip]);
        const float m1 = s.x / static_cast<float>(cols), m2 = s.y / static_cast<float>(cols);
        T* dr = dx + r * lddx;
#pragma unroll 2
        for (int64_t v = threadIdx.x; v < nvec; v += blockDim.x) {
            float f[VEC], g[VEC], wf[VEC], o[VEC];
            load_f<false>(f, xr + v * VEC);
            load_f<false>(g, yr + v * VEC);
            load_weight(wf, w, v * VEC, 1.0f);
            if (accumulate) {
                load_f<false>(o, dr + v * VEC);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] += rstd * (g[i] * wf[i] - m1 - (f[i] - mean) * rstd * m2);
            store_f<true>(dr + v * VEC, o);
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
#pragma unroll 8
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
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
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

int power_of_two_at_least(int64_t n)
{
    int p = 1;
    while (p < n) p <<= 1;
    return p;
}

struct Shape {
    int lanes, block;   // threads per row, threads per block
    int64_t blocks;     // that the rows give work to
};

Shape shape_of(int64_t rows, int64_t cols, int vec, int ept)
{
    Shape s{};
    const int64_t threads = (cols / vec + ept / vec - 1) / (ept / vec);
    if (threads <= 32) {
        s.lanes = power_of_two_at_least(threads);
        s.block = GROUP_BLOCK;
    } else {
        s.lanes = s.block = threads > MAX_THREADS ? MAX_THREADS : static_cast<int>((threads + 31) / 32 * 32);
    }
    const int64_t per_block = s.block / s.lanes;
    s.blocks = (rows + per_block - 1) / per_block;
    return s;
}

// A kernel as a type: what is remembered about it is remembered per kernel, not per signature.
template <auto K>
struct Kernel {
    static constexpr auto run = K;
};

// How many blocks of this size the device holds at once (asked once per kernel, size and device).
template <auto K>
int64_t resident_blocks(const sb200_ctx* ctx, Kernel<K>, int block, int smem)
{
    constexpr int DEVICES = 16;
    static int per_sm[DEVICES][MAX_WARPS + 1] = {};
    int ask = 0;
    int& n = ctx->device < DEVICES ? per_sm[ctx->device][block / 32] : ask;
    if (n == 0) {
        // the limit for every block size: one size must not take back what another was granted
        int got = 0;
        cudaFuncAttributes attr;
        if (cudaFuncGetAttributes(&attr, K) != cudaSuccess) return 0;
        const int most = 227 * 1024 - static_cast<int>(attr.sharedSizeBytes);
        if (smem > most || cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) return 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&got, K, block, smem) != cudaSuccess) return 0;
        n = got;
    }
    return static_cast<int64_t>(n) * ctx->sm_count;
}

// The widest access (elements) that fits all rows and the weights: 16, 4 or the element's own bytes.
template <typename T, typename W>
int access_width(int64_t cols, const void* w, const void* b, std::initializer_list<std::pair<const void*, int64_t>> arrays)
{
    for (int bytes : {16, 4}) {
        const int vec = bytes / static_cast<int>(sizeof(T));
        const size_t weights = vec * sizeof(W) < 16 ? vec * sizeof(W) : 16;
        bool ok = cols % vec == 0 && aligned_to(w, weights) && aligned_to(b, weights);
        for (const auto& a : arrays) ok = ok && a.second % vec == 0 && aligned_to(a.first, bytes);
        if (ok) return vec;
    }
    return 1;
}

template <int N>
using Int = std::integral_constant<int, N>;

// Whether the rows of all arrays start at the same distance from a 16-byte boundary, row by row.
template <typename T>
bool same_shift(std::initializer_list<std::pair<const void*, int64_t>> arrays)
{
    const auto& a = *arrays.begin();
    for (const auto& b : arrays)
        if ((reinterpret_cast<uintptr_t>(a.first) - reinterpret_cast<uintptr_t>(b.first)) % 16 != 0 ||
            (a.second - b.second) % static_cast<int64_t>(16 / sizeof(T)) != 0)
            return false;
    return true;
}

// Elements of the pieces that a row may touch, whatever its shift.
int64_t shifted_span(int64_t cols, int vec) { return (cols + 2 * vec - 2) / vec * vec; }

// Blocks for rows with a shift: every thread's steps are whole periods of it, at most 8 rows.
int64_t whole_periods(int64_t blocks, int64_t wanted) { return blocks < wanted ? blocks / 8 * 8 : wanted; }

// f(Int<vec>{}) for an access width of access_width()
template <typename T, typename F>
int with_width(int vec, F f)
{
    if (vec == 16 / static_cast<int>(sizeof(T))) return f(Int<16 / static_cast<int>(sizeof(T))>{});
    if constexpr (sizeof(T) == 2) {
        if (vec == 2) return f(Int<2>{});
    }
    return f(Int<1>{});
}

// Beyond any memory; within them no size and no grid's extent overflows (ln_reduce_kernel has a
// block for 32 columns).
constexpr int64_t MAX_ROWS = int64_t(1) << 40;
constexpr int64_t MAX_COLS = int64_t(1) << 35;

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
    if (rows > MAX_ROWS || cols > MAX_COLS) return SB200_ERR_TOO_LARGE;
    if (rows == 0) return SB200_OK;
    if (!x || !y || !aligned_to(x, type_bytes(type)) || !aligned_to(y, type_bytes(type)) || !aligned_to(weight, type_bytes(weight_type)) ||
        !aligned_to(bias, type_bytes(weight_type)) || !aligned_to(mean, 4) || !aligned_to(rstd, 4))
        return SB200_ERR_INVALID_ARG;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    return with_types(type, weight_type, [&](auto t, auto wt) -> int {
        using T = decltype(t);
        using W = decltype(wt);
        const int width = access_width<T, W>(cols, weight, bias, {{x, ldx}, {y, ldy}});
        if constexpr (sizeof(T) == 2) {
            // odd rows (4-byte accesses, where they fit, are better: 16384 x 4094 bf16 71 us, 137 in this way)
            constexpr int FULL = 16 / static_cast<int>(sizeof(T));
            const int64_t span = shifted_span(cols, FULL);
            if (width == 1 && same_shift<T>({{x, ldx}, {y, ldy}}) && span <= 32 * MAX_THREADS) {
                auto launch = [&](auto kern, auto e) -> int {
                    const Shape s = shape_of(rows, span, FULL, decltype(e)::value);
                    const int smem = s.block * Pieces<T, FULL, decltype(e)::value>::SMEM;
                    const int64_t most = resident_blocks(ctx, kern, s.block, smem);
                    if (most < 8) return SB200_ERR_CUDA;
                    return launch_after(ctx, kern.run, static_cast<unsigned>(whole_periods(most, s.blocks)), s.block, smem, stream, static_cast<T*>(y),
                                        ldy, mean, rstd, static_cast<const T*>(x), ldx, static_cast<const W*>(weight), static_cast<const W*>(bias),
                                        rows, static_cast<int>(cols), eps, s.lanes);
                };
                // 16 elements a thread as far as they go (the masks of 32 do not fit the registers: 4095 columns 139 us, 128 with 16)
                if (span <= 16 * 32) return launch(Kernel<ln_forward_kernel<T, W, FULL, 16, true, true>>{}, Int<16>{});
                if (span <= 16 * MAX_THREADS) return launch(Kernel<ln_forward_kernel<T, W, FULL, 16, false, true>>{}, Int<16>{});
                return launch(Kernel<ln_forward_kernel<T, W, FULL, 32, false, true>>{}, Int<32>{});
            }
        }
        return with_width<T>(width, [&](auto v) -> int {
            constexpr int VEC = decltype(v)::value;
            // 32 elements a thread for rows of more than 512 columns, so that a warp holds 1024;
            // 16 where 2-byte accesses hold every element in a register of its own
            constexpr bool WIDE = VEC * sizeof(T) >= 4;
            constexpr int MANY = WIDE ? 32 : 16;
            const bool many = WIDE && cols > 16 * 32;
            const Shape s = shape_of(rows, cols, VEC, many ? MANY : 16);
            auto launch = [&](auto kern, int smem, auto... last) -> int {
                const int64_t most = resident_blocks(ctx, kern, s.block, smem);
                if (most < 1) return SB200_ERR_CUDA;
                return launch_after(ctx, kern.run, static_cast<unsigned>(s.blocks < most ? s.blocks : most), s.block, smem, stream, static_cast<T*>(y), ldy, mean,
                                    rstd, static_cast<const T*>(x), ldx, static_cast<const W*>(weight), static_cast<const W*>(bias), rows,
                                    last...);
            };
            if (cols > MANY * MAX_THREADS) return launch(Kernel<ln_forward_long_kernel<T, W, VEC>>{}, 0, cols, eps);
            const int n = static_cast<int>(cols);
            if (many) {
                const int smem = s.block * Pieces<T, VEC, MANY>::SMEM;
                if (s.lanes <= 32) return launch(Kernel<ln_forward_kernel<T, W, VEC, MANY, true, false>>{}, smem, n, eps, s.lanes);
                return launch(Kernel<ln_forward_kernel<T, W, VEC, MANY, false, false>>{}, smem, n, eps, s.lanes);
            }
            const int smem = s.block * Pieces<T, VEC, 16>::SMEM;
            if (s.lanes <= 32) return launch(Kernel<ln_forward_kernel<T, W, VEC, 16, true, false>>{}, smem, n, eps, s.lanes);
            if constexpr (WIDE) return SB200_ERR_INVALID_ARG;    // (not reached: such rows have 32 elements a thread)
            else return launch(Kernel<ln_forward_kernel<T, W, VEC, 16, false, false>>{}, smem, n, eps, s.lanes);
        });
    });
}

extern "C" int64_t sb200_layer_norm_backward_workspace(const sb200_ctx* ctx, int64_t rows, int64_t cols)
{
    if (!ctx || rows < 0 || cols < 1 || rows > MAX_ROWS || cols > MAX_COLS) return -1;
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
    if (rows > MAX_ROWS || cols > MAX_COLS) return SB200_ERR_TOO_LARGE;
    if (rows > 0 && (!x || !dy || !mean || !rstd)) return SB200_ERR_INVALID_ARG;
    for (const void* at : {static_cast<const void*>(x), dy, static_cast<const void*>(dx)})
        if (!aligned_to(at, type_bytes(type))) return SB200_ERR_INVALID_ARG;
    for (const void* at : {weight, static_cast<const void*>(dweight), static_cast<const void*>(dbias)})
        if (!aligned_to(at, type_bytes(weight_type))) return SB200_ERR_INVALID_ARG;
    if (!aligned_to(mean, 4) || !aligned_to(rstd, 4)) return SB200_ERR_INVALID_ARG;
    const bool sums = dweight || dbias;
    if (sums && (!workspace || !aligned_to(workspace, 16) ||
                 workspace_bytes < sb200_layer_norm_backward_workspace(ctx, rows, cols)))
        return SB200_ERR_INVALID_ARG;
    if (!sums && (!dx || rows == 0)) return SB200_OK;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    float* partial = sums ? static_cast<float*>(workspace) : nullptr;
    return with_types(type, weight_type, [&](auto t, auto wt) -> int {
        using T = decltype(t);
        using W = decltype(wt);
        T* dxp = static_cast<T*>(dx);
        const T* yp = static_cast<const T*>(dy);
        const T* xp = static_cast<const T*>(x);
        const W* wp = static_cast<const W*>(weight);
        int parts = 0;
        if (rows > 0) {
            const int width = dx ? access_width<T, W>(cols, weight, nullptr, {{x, ldx}, {dy, lddy}, {dx, lddx}})
                                 : access_width<T, W>(cols, weight, nullptr, {{x, ldx}, {dy, lddy}});
            const int64_t bound = backward_parts(ctx->sm_count, rows, cols);
            constexpr int FULL = 16 / static_cast<int>(sizeof(T));
            const int64_t span = shifted_span(cols, FULL);
            const std::pair<const void*, int64_t> out{dx ? dx : x, dx ? lddx : ldx};
            const bool shifted = width == 1 && span <= REGISTER_COLS && same_shift<T>({{x, ldx}, {dy, lddy}, out});
            const int n = static_cast<int>(cols);
            auto launch = [&](auto kern, auto v, auto shift) -> int {
                constexpr int VEC = decltype(v)::value;
                constexpr bool SHIFT = decltype(shift)::value;
                const Shape s = shape_of(rows, SHIFT ? span : cols, VEC, EPT);
                int smem = 2 * s.block * Pieces<T, VEC, EPT>::SMEM;
                if (s.lanes <= 32 && smem < 2 * 32 * EPT * 4) smem = 2 * 32 * EPT * 4;      // column sums of such rows
                const int64_t most = resident_blocks(ctx, kern, s.block, smem);
                if (most < 8) return SB200_ERR_CUDA;
                const int64_t grid = most < bound ? most : bound;
                parts = static_cast<int>(SHIFT ? whole_periods(grid, s.blocks) : s.blocks < grid ? s.blocks : grid);
                return launch_after(ctx, kern.run, static_cast<unsigned>(parts), s.block, smem, stream, dxp, lddx, partial, yp, lddy, xp, ldx, wp, mean, rstd,
                                    rows, n, accumulate_dx, s.lanes);
            };
            auto any = [&]() -> int {
                if constexpr (sizeof(T) == 2) {
                    if (shifted)
                        return shape_of(rows, span, FULL, EPT).lanes <= 32
                                   ? launch(Kernel<ln_backward_kernel<T, W, FULL, true, true>>{}, Int<FULL>{}, std::true_type{})
                                   : launch(Kernel<ln_backward_kernel<T, W, FULL, false, true>>{}, Int<FULL>{}, std::true_type{});
                }
                return with_width<T>(width, [&](auto v) -> int {
                    constexpr int VEC = decltype(v)::value;
                    const Shape s = shape_of(rows, cols, VEC, EPT);
                    if (cols > REGISTER_COLS) {
                        // the column sums first: dx may overwrite dy
                        if (sums) {
                            parts = static_cast<int>(bound);
                            const dim3 grid(static_cast<unsigned>((cols + 255) / 256), static_cast<unsigned>(parts));
                            ln_backward_long_cols_kernel<T><<<grid, 256, 0, stream>>>(partial, yp, lddy, xp, ldx, mean, rstd, rows, cols);
                            ctx->launches += 1;
                        }
                        if (dx) {
                            Kernel<ln_backward_long_kernel<T, W, VEC>> kern;
                            const int64_t most = resident_blocks(ctx, kern, s.block, 0);
                            if (most < 1) return SB200_ERR_CUDA;
                            kern.run<<<static_cast<unsigned>(s.blocks < most ? s.blocks : most), s.block, 0, stream>>>(
                                dxp, lddx, yp, lddy, xp, ldx, wp, mean, rstd, rows, cols, accumulate_dx);
                            ctx->launches += 1;
                        }
                        return SB200_OK;
                    }
                    return s.lanes <= 32 ? launch(Kernel<ln_backward_kernel<T, W, VEC, true, false>>{}, v, std::false_type{})
                                         : launch(Kernel<ln_backward_kernel<T, W, VEC, false, false>>{}, v, std::false_type{});
                });
            };
            if (const int rc = any()) return rc;
        }
        if (sums) {
            const dim3 grid(static_cast<unsigned>((cols + 31) / 32), 2);
            if (const int rc = launch_after(ctx, ln_reduce_kernel<W>, grid, 1024, 0, stream, static_cast<W*>(dweight), static_cast<W*>(dbias),
                                            partial, parts, cols, accumulate_weight)) return rc;
        }
        return static_cast<int>(cudaGetLastError() == cudaSuccess ? SB200_OK : SB200_ERR_CUDA);
    });
}
