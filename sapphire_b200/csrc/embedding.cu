// Embedding lookup and its gradient.
//
//   out[t, :]    = scale * table[ids[t], :]                       (zero where ids[t] < 0)
//   dtable[v, :] = scale * sum over t with ids[t] == v of dout[t, :]
//
// Both are bound by memory: the lookup reads the rows that are named and writes one row
// a token; the gradient reads one row a token and writes the whole table (or, when it
// accumulates, reads and writes the rows that are named).
//
// The gradient needs the tokens of one vocabulary row together and in a fixed order, so
// that the sum is the same run to run.  The token positions are sorted by vocabulary row
// with a stable radix sort (9 bits a pass: two passes up to 262143 rows); the sorted list
// is cut into pieces of equal length, whatever rows they hold, so that a frequent token
// does not make one block slow; a block adds up the runs of its piece, stores the runs
// that lie inside it and leaves the sums of a run that crosses into a neighbour to a
// second kernel that adds them in order.
#include <type_traits>

#include "typed.cuh"

namespace sb200 {
namespace {

constexpr int LOOKUP_THREADS = 256;
constexpr int LOOKUP_ROWS = 4;           // tokens a thread has in flight

__device__ __forceinline__ void report_range(unsigned* status) { atomicCAS(status, 0u, static_cast<unsigned>(FAULT_TOKEN_RANGE)); }

// `lanes` (power of two) threads per token, VEC elements an access.
template <typename TT, typename TA, typename I, int VEC>
__global__ void __launch_bounds__(LOOKUP_THREADS)
lookup_kernel(TA* __restrict__ out, int64_t ldo, const TT* __restrict__ table, int64_t ldt,
              const I* __restrict__ ids, int64_t n, int64_t vocab, int nvec, float scale, int lanes,
              unsigned* status)
{
    const int lane = threadIdx.x & (lanes - 1);
    const int per_block = LOOKUP_THREADS / lanes;
    const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * per_block) * LOOKUP_ROWS + threadIdx.x / lanes;
    int64_t id[LOOKUP_ROWS];
#pragma unroll
    for (int k = 0; k < LOOKUP_ROWS; ++k) {
        const int64_t t = t0 + static_cast<int64_t>(k) * per_block;
        id[k] = t < n ? static_cast<int64_t>(ids[t]) : -1;
        if (id[k] >= vocab) {
            if (lane == 0) report_range(status);
            id[k] = -1;
        }
    }
    for (int v = lane; v < nvec; v += lanes) {
        Raw<TT, VEC> r[LOOKUP_ROWS];
#pragma unroll
        for (int k = 0; k < LOOKUP_ROWS; ++k)
            if (id[k] >= 0) load_raw<false>(r[k], table + id[k] * ldt + static_cast<int64_t>(v) * VEC);
#pragma unroll
        for (int k = 0; k < LOOKUP_ROWS; ++k) {
            const int64_t t = t0 + static_cast<int64_t>(k) * per_block;
            if (t >= n) continue;
            float f[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = id[k] >= 0 ? to_f(r[k].e[i]) * scale : 0.0f;
            store_f<true>(out + t * ldo + static_cast<int64_t>(v) * VEC, f);
        }
    }
}

// ------------------------------------------------------------------------- sort

constexpr int DIGIT_BITS = 9;
constexpr int DIGITS = 1 << DIGIT_BITS;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_ROUNDS = 2;                               // items a thread per tile
constexpr int SORT_TILE = SORT_THREADS * SORT_ROUNDS;
constexpr int SORT_BLOCKS = 64;                              // at most: every block reads all counts

// The sort key of a token: its vocabulary row, or `vocab` (last) for padding.
template <typename I>
__device__ __forceinline__ uint32_t key_of(I id, int64_t vocab, unsigned* status)
{
    const int64_t v = static_cast<int64_t>(id);
    if (v >= vocab) report_range(status);
    return static_cast<uint32_t>(v < 0 || v >= vocab ? vocab : v);
}

// counts[block][digit] of this block's slice.  FIRST: keys come from ids; marks the rows that occur.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS)
sort_count_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ touched, const I* __restrict__ ids,
                  const uint32_t* __restrict__ keys, int64_t n, int64_t per_block, int64_t vocab, int shift,
                  unsigned* status)
{
    __shared__ uint32_t hist[DIGITS];
    for (int d = threadIdx.x; d < DIGITS; d += SORT_THREADS) hist[d] = 0;
    __syncthreads();
    const int64_t i0 = blockIdx.x * per_block, i1 = min(n, i0 + per_block);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += SORT_THREADS) {
        uint32_t key;
        if constexpr (FIRST) {
            key = key_of(ids[i], vocab, status);
            if (touched && key < vocab) atomicOr(&touched[key >> 5], 1u << (key & 31));
        } else {
            key = keys[i];
        }
        atomicAdd(&hist[(key >> shift) & (DIGITS - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < DIGITS; d += SORT_THREADS) counts[blockIdx.x * DIGITS + d] = hist[d];
}

// Stable scatter of this block's slice by one digit.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS)
sort_scatter_kernel(uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out,
                    const uint32_t* __restrict__ counts, const I* __restrict__ ids,
                    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int64_t n,
                    int64_t per_block, int64_t vocab, int shift, unsigned* status)
{
    __shared__ uint32_t offset[DIGITS];                      // where this block's next item of a digit goes
    __shared__ unsigned short ahead[SORT_WARPS][DIGITS];     // items of a digit in the warps before, this tile
    __shared__ uint32_t scan[SORT_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = gridDim.x;

    // first place of a digit: all items of smaller digits, then the blocks before this one
    uint32_t total = 0, before = 0;
    if (threadIdx.x < DIGITS) {
        for (int b = 0; b < blocks; ++b) {
            const uint32_t c = counts[b * DIGITS + threadIdx.x];
            total += c;
            if (b < static_cast<int>(blockIdx.x)) before += c;
        }
    }
    uint32_t incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    if (threadIdx.x < DIGITS) {
        uint32_t base = 0;
        for (int w = 0; w < warp; ++w) base += scan[w];
        offset[threadIdx.x] = base + incl - total + before;
    }

    const int64_t i0 = blockIdx.x * per_block, i1 = min(n, i0 + per_block);
    for (int64_t tile = i0; tile < i1; tile += SORT_TILE) {
        __syncthreads();                                     // offsets of the tile before are final
        for (int d = threadIdx.x; d < SORT_WARPS * DIGITS; d += SORT_THREADS)
            (&ahead[0][0])[d] = 0;
        __syncthreads();
        uint32_t key[SORT_ROUNDS], from[SORT_ROUNDS], digit[SORT_ROUNDS], rank[SORT_ROUNDS];
#pragma unroll
        for (int k = 0; k < SORT_ROUNDS; ++k) {
            const int64_t i = tile + warp * (32 * SORT_ROUNDS) + k * 32 + lane;
            const bool in = i < i1;
            key[k] = from[k] = 0;
            if (in) {
                if constexpr (FIRST) {
                    key[k] = key_of(ids[i], vocab, status);
                    from[k] = static_cast<uint32_t>(i);
                } else {
                    key[k] = keys[i];
                    from[k] = pos[i];
                }
            }
            digit[k] = in ? (key[k] >> shift) & (DIGITS - 1) : static_cast<uint32_t>(DIGITS);
            const unsigned same = __match_any_sync(0xffffffffu, digit[k]);
            const unsigned lower = same & ((1u << lane) - 1u);
            rank[k] = __popc(lower);
            if (in) rank[k] += ahead[warp][digit[k]];
            __syncwarp();
            if (in && lower == 0) ahead[warp][digit[k]] += static_cast<unsigned short>(__popc(same));
            __syncwarp();
        }
        __syncthreads();
        uint32_t in_tile = 0;
        if (threadIdx.x < DIGITS) {
#pragma unroll 8
            for (int w = 0; w < SORT_WARPS; ++w) {
                const uint32_t c = ahead[w][threadIdx.x];
                ahead[w][threadIdx.x] = static_cast<unsigned short>(in_tile);
                in_tile += c;
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < SORT_ROUNDS; ++k) {
            if (digit[k] < DIGITS) {
                const uint32_t to = offset[digit[k]] + ahead[warp][digit[k]] + rank[k];
                keys_out[to] = key[k];
                pos_out[to] = from[k];
            }
        }
        __syncthreads();
        if (threadIdx.x < DIGITS) offset[threadIdx.x] += in_tile;
    }
}

// --------------------------------------------------------------------- gradient

constexpr int GRAD_THREADS = 256;
constexpr int GRAD_UNROLL = 8;           // token rows a thread has in flight
constexpr int MAX_PIECE = 1024;          // sorted tokens per block at most

// Zeroes the rows no token names; one warp a row.
template <typename TT, int VEC>
__global__ void __launch_bounds__(256)
zero_rows_kernel(TT* __restrict__ dtable, int64_t ldt, const uint32_t* __restrict__ touched, int64_t vocab,
                 int64_t nvec)
{
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
    Raw<TT, VEC> zero;
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero.e[i] = from_f<TT>(0.0f);
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); v < vocab; v += warps) {
        if ((touched[v >> 5] >> (v & 31)) & 1u) continue;
        TT* row = dtable + v * ldt;
        for (int64_t k = threadIdx.x & 31; k < nvec; k += 32) store_raw<true>(row + k * VEC, zero);
    }
}

template <typename TT, int VEC>
__device__ __forceinline__ void write_row(TT* p, const float (&sum)[VEC], float scale, int accumulate)
{
    float o[VEC];
    if (accumulate) {
        load_f<false>(o, p);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = fmaf(sum[i], scale, o[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = sum[i] * scale;
    }
    store_f<true>(p, o);
}

// Block (piece, column tile).  edge: [pieces][2][nvec * VEC] sums of the runs that cross a
// piece's ends: [0] of the run that came in from the piece before (whether or not it also
// goes on), [1] of a run that starts here and goes on.
template <typename TT, typename TA, int VEC>
__global__ void __launch_bounds__(GRAD_THREADS)
grad_pieces_kernel(TT* __restrict__ dtable, int64_t ldt, float* __restrict__ edge, const TA* __restrict__ dout,
                   int64_t ldo, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int64_t n,
                   int piece, int64_t vocab, int64_t nvec, float scale, int accumulate)
{
    __shared__ uint32_t skey[MAX_PIECE + 2], spos[MAX_PIECE];
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * piece;
    const int count = static_cast<int>(min(static_cast<int64_t>(piece), n - i0));
    // skey[0] and skey[count + 1]: the neighbours' keys, or a key that no row has
    for (int i = threadIdx.x; i < count + 2; i += blockDim.x) {
        const int64_t at = i0 + i - 1;
        skey[i] = at >= 0 && at < n ? keys[at] : 0xffffffffu;
    }
    for (int i = threadIdx.x; i < count; i += blockDim.x) spos[i] = pos[i0 + i];
    __syncthreads();
    const int64_t v = static_cast<int64_t>(blockIdx.y) * blockDim.x + threadIdx.x;
    if (v >= nvec) return;
    const TA* src = dout + v * VEC;
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
    bool came_in = skey[0] == skey[1];
    for (int b = 0; b < count; b += GRAD_UNROLL) {
        Raw<TA, VEC> r[GRAD_UNROLL];
#pragma unroll
        for (int k = 0; k < GRAD_UNROLL; ++k)
            if (b + k < count && skey[b + k + 1] < vocab) load_raw<true>(r[k], src + static_cast<int64_t>(spos[b + k]) * ldo);
#pragma unroll
        for (int k = 0; k < GRAD_UNROLL; ++k) {
            if (b + k >= count) break;
            const uint32_t key = skey[b + k + 1];
            if (key >= vocab) break;                         // padding sorts last
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] += to_f(r[k].e[i]);
            if (skey[b + k + 2] == key && b + k + 1 < count) continue;
            const bool goes_on = skey[b + k + 2] == key;
            if (came_in || goes_on) {
                float* e = edge + ((static_cast<int64_t>(blockIdx.x) * 2 + (came_in ? 0 : 1)) * nvec + v) * VEC;
#pragma unroll
                for (int i = 0; i < VEC; ++i) e[i] = sum[i];
            } else {
                write_row<TT, VEC>(dtable + static_cast<int64_t>(key) * ldt + v * VEC, sum, scale, accumulate);
            }
            came_in = false;
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
        }
    }
}

// Block (piece, column tile): if a run starts in this piece and goes on, adds its parts.
// blockDim.x = lanes * slices; a slice adds neighbouring pieces, the slices are added in order.
template <typename TT, int VEC>
__global__ void __launch_bounds__(GRAD_THREADS)
grad_join_kernel(TT* __restrict__ dtable, int64_t ldt, const float* __restrict__ edge,
                 const uint32_t* __restrict__ keys, int64_t n, int piece, int64_t vocab, int64_t nvec, float scale,
                 int accumulate, int lanes)
{
    __shared__ float part[GRAD_THREADS * VEC];
    const int64_t p = blockIdx.x, i0 = p * piece, i1 = i0 + piece;
    if (i1 >= n) return;                                     // the last piece hands nothing on
    const uint32_t key = keys[i1 - 1];
    if (key >= vocab || keys[i1] != key) return;
    if (i0 > 0 && keys[i0] == key && keys[i0 - 1] == key) return;      // it started further ahead
    // last piece whose first key is this one
    int64_t lo = p + 1, hi = (n - 1) / piece;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) / 2;
        if (keys[mid * piece] == key) lo = mid; else hi = mid - 1;
    }
    const int64_t parts = lo - p + 1;                        // this piece's [1], then [0] of p + 1 .. lo
    const int lane = threadIdx.x % lanes, slice = threadIdx.x / lanes, slices = blockDim.x / lanes;
    const int64_t v = static_cast<int64_t>(blockIdx.y) * lanes + lane;
    const int64_t per = (parts + slices - 1) / slices;
    const int64_t q0 = slice * per, q1 = min(parts, q0 + per);
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
    if (v < nvec) {
#pragma unroll 4
        for (int64_t q = q0; q < q1; ++q) {
            const float* e = edge + (((p + q) * 2 + (q == 0 ? 1 : 0)) * nvec + v) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] += e[i];
        }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) part[threadIdx.x * VEC + i] = sum[i];
    __syncthreads();
    if (slice != 0 || v >= nvec) return;
    for (int s = 1; s < slices; ++s)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] += part[(s * lanes + lane) * VEC + i];
    write_row<TT, VEC>(dtable + static_cast<int64_t>(key) * ldt + v * VEC, sum, scale, accumulate);
}

// ------------------------------------------------------------------------- host

constexpr int64_t MAX_TOKENS = int64_t(1) << 30;
constexpr int64_t MAX_VOCAB = (int64_t(1) << 31) - 2;
constexpr int64_t MAX_COLS = int64_t(1) << 20;           // column tiles are a grid's y extent

int check_types(int table_type, int type, int index_bits)
{
    if (!known_type(table_type) || !known_type(type) || (index_bits != 32 && index_bits != 64))
        return SB200_ERR_INVALID_ARG;
    // equal, or one side in fp32
    return table_type == type || table_type == SB200_F32 || type == SB200_F32 ? SB200_OK : SB200_ERR_UNSUPPORTED;
}

template <typename F>
int with_types(int table_type, int type, F f)
{
    if (table_type == SB200_F32)
        return type == SB200_F32 ? f(float{}, float{}) : type == SB200_BF16 ? f(float{}, bf16{}) : f(float{}, f16{});
    if (table_type == SB200_BF16) return type == SB200_F32 ? f(bf16{}, float{}) : f(bf16{}, bf16{});
    return type == SB200_F32 ? f(f16{}, float{}) : f(f16{}, f16{});
}

// 16 bytes of the narrower of the two types
template <typename TT, typename TA>
constexpr int wide() { return 16 / (sizeof(TT) < sizeof(TA) ? sizeof(TT) : sizeof(TA)); }

template <typename TT, typename TA>
bool can_vector(const void* table, int64_t ldt, const void* act, int64_t lda, int64_t cols)
{
    constexpr int VEC = wide<TT, TA>();
    return cols % VEC == 0 && (ldt * static_cast<int64_t>(sizeof(TT))) % 16 == 0 &&
           (lda * static_cast<int64_t>(sizeof(TA))) % 16 == 0 && aligned_to(table, 16) && aligned_to(act, 16);
}

int power_of_two(int64_t n, int most)
{
    int p = 1;
    while (p < n && p < most) p <<= 1;
    return p;
}

struct GradPlan {
    int64_t blocks, per_block;           // of the sort
    int passes;
    int piece;
    int64_t pieces;
    // byte offsets into the workspace
    int64_t counts, touched, keys[2], pos[2], edge, total;
};

GradPlan plan_grad(int sm_count, int64_t n, int64_t vocab, int64_t cols)
{
    GradPlan g{};
    const int64_t tiles = n > 0 ? (n + SORT_TILE - 1) / SORT_TILE : 1;
    const int64_t tiles_per_block = (tiles + SORT_BLOCKS - 1) / SORT_BLOCKS;
    g.per_block = tiles_per_block * SORT_TILE;
    g.blocks = (n + g.per_block - 1) / g.per_block;
    int bits = 0;
    while (bits < 32 && (vocab >> bits) != 0) ++bits;        // keys 0 .. vocab
    g.passes = (bits + DIGIT_BITS - 1) / DIGIT_BITS;
    // pieces: enough blocks to keep every SM busy (about 16 of GRAD_THREADS threads, a
    // thread holding at least 4 columns), no fewer than 8 tokens each
    const int64_t tiles_n = (cols + 4 * GRAD_THREADS - 1) / (4 * GRAD_THREADS);
    int64_t piece = n * tiles_n / (16ll * sm_count);
    if (piece < GRAD_UNROLL) piece = GRAD_UNROLL;
    if (piece > 32) piece = 32;
    if (n / piece > 8192) piece = n / 8192;                  // long lists: bounds the edge sums
    if (piece > MAX_PIECE) piece = MAX_PIECE;
    g.piece = static_cast<int>(piece);
    g.pieces = (n + piece - 1) / piece;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    g.counts = take(g.blocks * DIGITS * 4);
    g.touched = take((vocab + 31) / 32 * 4);
    for (int i = 0; i < 2; ++i) { g.keys[i] = take(n * 4); g.pos[i] = take(n * 4); }
    g.edge = take(g.pieces * 2 * cols * 4);
    g.total = at;
    return g;
}

template <typename I>
void sort_tokens(sb200_ctx* ctx, const GradPlan& g, unsigned char* ws, const I* ids, int64_t n, int64_t vocab,
                 uint32_t* touched, const uint32_t** keys, const uint32_t** pos, cudaStream_t stream)
{
    auto u32 = [&](int64_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
    uint32_t* counts = u32(g.counts);
    const unsigned grid = static_cast<unsigned>(g.blocks);
    const uint32_t *kin = nullptr, *pin = nullptr;
    for (int pass = 0; pass < g.passes; ++pass) {
        const int shift = pass * DIGIT_BITS;
        uint32_t *kout = u32(g.keys[pass & 1]), *pout = u32(g.pos[pass & 1]);
        if (pass == 0) {
            sort_count_kernel<I, true><<<grid, SORT_THREADS, 0, stream>>>(counts, touched, ids, nullptr, n, g.per_block, vocab, shift, ctx->d_status);
            sort_scatter_kernel<I, true><<<grid, SORT_THREADS, 0, stream>>>(kout, pout, counts, ids, nullptr, nullptr, n, g.per_block, vocab, shift, ctx->d_status);
        } else {
            sort_count_kernel<I, false><<<grid, SORT_THREADS, 0, stream>>>(counts, nullptr, nullptr, kin, n, g.per_block, vocab, shift, ctx->d_status);
            sort_scatter_kernel<I, false><<<grid, SORT_THREADS, 0, stream>>>(kout, pout, counts, nullptr, kin, pin, n, g.per_block, vocab, shift, ctx->d_status);
        }
        ctx->launches += 2;
        kin = kout;
        pin = pout;
    }
    *keys = kin;
    *pos = pin;
}

template <typename TT, typename TA, int VEC>
void launch_grad(sb200_ctx* ctx, const GradPlan& g, TT* dtable, int64_t ldt, float* edge, const TA* dout, int64_t ldo,
                 const uint32_t* keys, const uint32_t* pos, const uint32_t* touched, int64_t n, int64_t vocab,
                 int64_t cols, float scale, int accumulate, cudaStream_t stream)
{
    const int64_t nvec = cols / VEC;
    if (!accumulate) {
        int64_t grid = (vocab + 7) / 8;
        if (grid > 16ll * ctx->sm_count) grid = 16ll * ctx->sm_count;
        zero_rows_kernel<TT, VEC><<<static_cast<unsigned>(grid), 256, 0, stream>>>(dtable, ldt, touched, vocab, nvec);
        ctx->launches += 1;
    }
    if (n == 0) return;
    const int threads = power_of_two(nvec, GRAD_THREADS) < 32 ? 32 : power_of_two(nvec, GRAD_THREADS);
    const dim3 grid(static_cast<unsigned>(g.pieces), static_cast<unsigned>((nvec + threads - 1) / threads));
    grad_pieces_kernel<TT, TA, VEC><<<grid, threads, 0, stream>>>(dtable, ldt, edge, dout, ldo, keys, pos, n, g.piece, vocab, nvec, scale, accumulate);
    // few columns a block and many slices: a run of many pieces is added by slices at the same time
    const int lanes = threads < 32 ? threads : 32;
    const dim3 join(static_cast<unsigned>(g.pieces), static_cast<unsigned>((nvec + lanes - 1) / lanes));
    grad_join_kernel<TT, VEC><<<join, GRAD_THREADS, 0, stream>>>(dtable, ldt, edge, keys, n, g.piece, vocab, nvec, scale, accumulate, lanes);
    ctx->launches += 2;
}

}  // namespace
}  // namespace sb200

using namespace sb200;

extern "C" int sb200_embedding(sb200_ctx* ctx, void* out, int64_t ldo, const void* table, int64_t ldt, const void* ids,
                               int index_bits, int64_t n, int64_t vocab, int64_t cols, float scale, int table_type,
                               int type, sb200_stream stream_)
{
    TraceRange trace("sb200_embedding");
    if (!ctx || n < 0 || vocab < 0 || cols < 0 || ldo < cols || ldt < cols) return SB200_ERR_INVALID_ARG;
    if (const int rc = check_types(table_type, type, index_bits)) return rc;
    if (n > MAX_TOKENS || vocab > MAX_VOCAB || cols > MAX_COLS) return SB200_ERR_TOO_LARGE;
    if (n == 0 || cols == 0) return SB200_OK;
    if (!out || !ids || (vocab > 0 && !table) || !aligned_to(ids, index_bits / 8)) return SB200_ERR_INVALID_ARG;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    return with_types(table_type, type, [&](auto tt, auto ta) {
        using TT = decltype(tt);
        using TA = decltype(ta);
        constexpr int WIDE = wide<TT, TA>();
        const bool vec = can_vector<TT, TA>(table, ldt, out, ldo, cols);
        const int64_t nvec = vec ? cols / WIDE : cols;
        const int lanes = power_of_two(nvec, LOOKUP_THREADS);
        const int64_t per_block = static_cast<int64_t>(LOOKUP_THREADS / lanes) * LOOKUP_ROWS;
        const unsigned grid = static_cast<unsigned>((n + per_block - 1) / per_block);
        auto go = [&](auto id, auto v) {
            using I = decltype(id);
            lookup_kernel<TT, TA, I, decltype(v)::value><<<grid, LOOKUP_THREADS, 0, stream>>>(
                static_cast<TA*>(out), ldo, static_cast<const TT*>(table), ldt, static_cast<const I*>(ids), n, vocab,
                static_cast<int>(nvec), scale, lanes, ctx->d_status);
        };
        using One = std::integral_constant<int, 1>;
        using Wide = std::integral_constant<int, WIDE>;
        if (index_bits == 64) { if (vec) go(int64_t{}, Wide{}); else go(int64_t{}, One{}); }
        else { if (vec) go(int32_t{}, Wide{}); else go(int32_t{}, One{}); }
        ctx->launches += 1;
        return cudaGetLastError() == cudaSuccess ? SB200_OK : SB200_ERR_CUDA;
    });
}

extern "C" int64_t sb200_embedding_backward_workspace(const sb200_ctx* ctx, int64_t n, int64_t vocab, int64_t cols)
{
    if (!ctx || n < 0 || vocab < 0 || cols < 0 || n > MAX_TOKENS || vocab > MAX_VOCAB || cols > MAX_COLS) return -1;
    return plan_grad(ctx->sm_count, n, vocab, cols).total;
}

extern "C" int sb200_embedding_backward(sb200_ctx* ctx, void* dtable, int64_t ldt, const void* dout, int64_t ldo,
                                        const void* ids, int index_bits, int64_t n, int64_t vocab, int64_t cols,
                                        float scale, int table_type, int type, int accumulate, void* workspace,
                                        int64_t workspace_bytes, sb200_stream stream_)
{
    TraceRange trace("sb200_embedding_backward");
    if (!ctx || n < 0 || vocab < 0 || cols < 0 || ldo < cols || ldt < cols) return SB200_ERR_INVALID_ARG;
    if (const int rc = check_types(table_type, type, index_bits)) return rc;
    if (n > MAX_TOKENS || vocab > MAX_VOCAB || cols > MAX_COLS) return SB200_ERR_TOO_LARGE;
    if (vocab == 0 || cols == 0 || (n == 0 && accumulate)) return SB200_OK;
    if (!dtable || (n > 0 && (!dout || !ids || !aligned_to(ids, index_bits / 8)))) return SB200_ERR_INVALID_ARG;
    const GradPlan g = plan_grad(ctx->sm_count, n, vocab, cols);
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < g.total) return SB200_ERR_INVALID_ARG;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    uint32_t* touched = nullptr;
    if (!accumulate) {
        touched = reinterpret_cast<uint32_t*>(ws + g.touched);
        if (cudaMemsetAsync(touched, 0, static_cast<size_t>((vocab + 31) / 32 * 4), stream) != cudaSuccess) return SB200_ERR_CUDA;
    }
    const uint32_t *keys = nullptr, *pos = nullptr;
    if (n > 0) {
        if (index_bits == 64)
            sort_tokens(ctx, g, ws, static_cast<const int64_t*>(ids), n, vocab, touched, &keys, &pos, stream);
        else
            sort_tokens(ctx, g, ws, static_cast<const int32_t*>(ids), n, vocab, touched, &keys, &pos, stream);
    }
    float* edge = reinterpret_cast<float*>(ws + g.edge);
    return with_types(table_type, type, [&](auto tt, auto ta) {
        using TT = decltype(tt);
        using TA = decltype(ta);
        TT* dt = static_cast<TT*>(dtable);
        const TA* dy = static_cast<const TA*>(dout);
        if (can_vector<TT, TA>(dtable, ldt, dout, ldo, cols))
            launch_grad<TT, TA, wide<TT, TA>()>(ctx, g, dt, ldt, edge, dy, ldo, keys, pos, touched, n, vocab, cols, scale, accumulate, stream);
        else
            launch_grad<TT, TA, 1>(ctx, g, dt, ldt, edge, dy, ldo, keys, pos, touched, n, vocab, cols, scale, accumulate, stream);
        return cudaGetLastError() == cudaSuccess ? SB200_OK : SB200_ERR_CUDA;
    });
}
