// Embedding lookup and its gradient.
//
//   out[t, :]    = scale * table[ids[t], :]                       (zero where ids[t] < 0)
//   dtable[v, :] = scale * sum over t with ids[t] == v of dout[t, :]
//
// Both are bound by memory: the lookup reads the rows that are named and writes one row
// a token; the gradient reads one row a token and writes the whole table (or, when it
// accumulates, reads and writes the rows that are named).  65536 tokens x 4096 bf16: lookup
// 125 us (5.4 TB/s), gradient into an fp32 table 304 us (5.2 TB/s), added to it 229 us.
//
// The gradient needs the tokens of one vocabulary row together and in a fixed order, so
// that the sum is the same run to run.  The token positions are sorted by vocabulary row
// with a stable radix sort (9 bits a pass: two passes up to 262143 rows): up to 16384
// tokens by one block in shared memory, while the other SMs fill the table with zeros;
// more by up to 64 blocks, two launches a pass, which also mark the rows that occur, so
// that only the others are filled.  The sorted list is cut into pieces of equal length,
// whatever rows they hold, so that a frequent token does not make one block slow; a block
// adds up the runs that start in its piece, up to a piece's length beyond its end.  Runs
// longer than a piece leave a partial sum in every piece they touch, and a second kernel
// adds those in order; it works through a list of these runs (one block a piece, most of
// them with nothing to join, took 99 us where the sums took 129).
#include <type_traits>

#include "ptx.cuh"
#include "typed.cuh"

namespace sb200 {
namespace {

constexpr int LOOKUP_THREADS = 256;
constexpr int LOOKUP_LANES = 64;         // threads a token at most

// Every thread that meets such a number writes the same value.
__device__ __forceinline__ void report_range(unsigned* token_range) { *token_range = 1u; }

// `lanes` (power of two) threads per token, VEC elements an access.  What counts is how many
// accesses a thread has under way: eight of one row where rows are long enough (65536 x
// 4096 bf16: 125 us; two of each of four rows, 145), else one of each of ROWS rows.  The
// result is stored as usual, not as a stream: it is read next (and 7 us faster).
template <typename TT, typename TA, typename I, int VEC, int ROWS>
__global__ void __launch_bounds__(LOOKUP_THREADS)
lookup_kernel(TA* __restrict__ out, int64_t ldo, const TT* __restrict__ table, int64_t ldt,
              const I* __restrict__ ids, int64_t n, int64_t vocab, int nvec, float scale, int lanes,
              unsigned* token_range)
{
    const int lane = threadIdx.x & (lanes - 1);
    const int per_block = LOOKUP_THREADS / lanes;
    const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * per_block) * ROWS + threadIdx.x / lanes;
    int64_t id[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        const int64_t t = t0 + static_cast<int64_t>(k) * per_block;
        id[k] = t < n ? static_cast<int64_t>(ids[t]) : -1;
        if (id[k] >= vocab) {
            if (lane == 0) report_range(token_range);
            id[k] = -1;
        }
    }
#pragma unroll (ROWS == 1 ? 8 : 1)
    for (int v = lane; v < nvec; v += lanes) {
        Raw<TT, VEC> r[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k)
            if (id[k] >= 0) load_raw<false>(r[k], table + id[k] * ldt + static_cast<int64_t>(v) * VEC);
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const int64_t t = t0 + static_cast<int64_t>(k) * per_block;
            if (t >= n) continue;
            float f[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = id[k] >= 0 ? to_f(r[k].e[i]) * scale : 0.0f;
            store_f<false>(out + t * ldo + static_cast<int64_t>(v) * VEC, f);
        }
    }
}

// ------------------------------------------------------------------------- sort

constexpr int DIGIT_BITS = 9;
constexpr int DIGITS = 1 << DIGIT_BITS;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_ROUNDS = 1;                               // items a thread per tile
constexpr int SORT_TILE = SORT_THREADS * SORT_ROUNDS;
constexpr int SORT_BLOCKS = 64;                              // at most: every block reads all counts

// The sort key of a token: its vocabulary row, or `vocab` (last) for padding.
template <typename I>
__device__ __forceinline__ uint32_t key_of(I id, int64_t vocab, unsigned* token_range)
{
    const int64_t v = static_cast<int64_t>(id);
    if (v >= vocab) report_range(token_range);
    return static_cast<uint32_t>(v < 0 || v >= vocab ? vocab : v);
}

// counts[block][digit] of this block's slice.  FIRST: keys come from ids; marks the rows that occur.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS)
sort_count_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ touched, const I* __restrict__ ids,
                  const uint32_t* __restrict__ keys, int64_t n, int64_t per_block, int64_t vocab, int shift,
                  unsigned* token_range)
{
    __shared__ uint32_t hist[DIGITS];
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    for (int d = threadIdx.x; d < DIGITS; d += SORT_THREADS) hist[d] = 0;
    __syncthreads();
    const int64_t i0 = blockIdx.x * per_block, i1 = min(n, i0 + per_block);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += SORT_THREADS) {
        uint32_t key;
        if constexpr (FIRST) {
            key = key_of(ids[i], vocab, token_range);
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
                    int64_t per_block, int64_t vocab, int shift, unsigned* token_range)
{
    __shared__ uint32_t offset[DIGITS];                      // where this block's next item of a digit goes
    __shared__ unsigned short ahead[SORT_WARPS][DIGITS];     // items of a digit in the warps before, this tile
    __shared__ uint32_t scan[SORT_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = gridDim.x;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();

    // first place of a digit: all items of smaller digits, then the blocks before this one
    uint32_t total = 0, before = 0;
    if (threadIdx.x < DIGITS) {
#pragma unroll 16
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
                    key[k] = key_of(ids[i], vocab, token_range);
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

// ------------------------------------------------------------- sort by one block

constexpr int SMALL_ROUNDS = 16;                             // items a thread at most
constexpr int SMALL_TOKENS = SORT_THREADS * SMALL_ROUNDS;
constexpr int SMALL_SMEM = SMALL_TOKENS * 6 + SORT_WARPS * DIGITS * 2 + DIGITS * 4 + SORT_WARPS * 4;

// Fills rows [v0, v1) with zeros, those marked in `touched` (if any) left out; `lanes` (power
// of two) threads a row.  A word of marks serves 32 rows.
template <typename TT, int VEC>
__device__ __forceinline__ void zero_rows(TT* dtable, int64_t ldt, int64_t nvec, int64_t v0, int64_t v1,
                                          const uint32_t* touched)
{
    Raw<TT, VEC> zero;
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero.e[i] = from_f<TT>(0.0f);
    int lanes = 1;
    while (lanes < nvec && lanes < static_cast<int>(blockDim.x)) lanes <<= 1;
    const int lane = threadIdx.x & (lanes - 1), rows = blockDim.x / lanes;
    uint32_t marks = 0;
    int64_t marks_of = -1;
    for (int64_t v = v0 + threadIdx.x / lanes; v < v1; v += rows) {
        if (touched && (v >> 5) != marks_of) {
            marks_of = v >> 5;
            marks = touched[marks_of];
        }
        if ((marks >> (v & 31)) & 1u) continue;
        TT* row = dtable + v * ldt;
#pragma unroll 4
        for (int64_t k = lane; k < nvec; k += lanes) store_raw<true>(row + k * VEC, zero);
    }
}

// Block 0 sorts n <= SMALL_TOKENS tokens; the others fill dtable (null: none of them) with zeros.
// A whole pass in shared memory: an item's place is (items of smaller digits) + (items of its
// digit in the warps before) + (its rank in its warp).
template <typename I, typename TT, int VEC>
__global__ void __launch_bounds__(SORT_THREADS)
sort_small_kernel(uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out, uint32_t* __restrict__ long_runs,
                  const I* __restrict__ ids, int n, int64_t vocab, int passes, TT* __restrict__ dtable, int64_t ldt,
                  int64_t nvec, unsigned* token_range)
{
    ptx::griddep_launch_dependents();
    if (blockIdx.x > 0) {
        // neighbouring rows to a block, so that its stores are neighbours
        const int64_t per = (vocab + gridDim.x - 2) / (gridDim.x - 1), v0 = (blockIdx.x - 1) * per;
        zero_rows<TT, VEC>(dtable, ldt, nvec, v0, min(vocab, v0 + per), nullptr);
        return;
    }
    extern __shared__ __align__(16) unsigned char smem[];
    uint32_t* skey = reinterpret_cast<uint32_t*>(smem);
    uint32_t* offset = skey + SMALL_TOKENS;
    uint32_t* scan = offset + DIGITS;
    unsigned short* ahead = reinterpret_cast<unsigned short*>(scan + SORT_WARPS);      // [SORT_WARPS][DIGITS]
    unsigned short* spos = ahead + SORT_WARPS * DIGITS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rounds = (n + SORT_THREADS - 1) / SORT_THREADS;
    const int i0 = warp * rounds * 32 + lane;
    if (threadIdx.x == 0) *long_runs = 0;
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * DIGIT_BITS;
        for (int d = threadIdx.x; d < SORT_WARPS * DIGITS / 2; d += SORT_THREADS) reinterpret_cast<uint32_t*>(ahead)[d] = 0;
        __syncthreads();
        uint32_t key[SMALL_ROUNDS], where[SMALL_ROUNDS];     // where: rank in the warp << 16 | position in ids
#pragma unroll
        for (int k = 0; k < SMALL_ROUNDS; ++k) {
            const int i = i0 + k * 32;
            key[k] = where[k] = 0;
            if (k < rounds && i < n) {
                key[k] = pass == 0 ? key_of(ids[i], vocab, token_range) : skey[i];
                where[k] = pass == 0 ? i : spos[i];
            }
        }
#pragma unroll
        for (int k = 0; k < SMALL_ROUNDS; ++k) {
            if (k >= rounds) break;
            const bool in = i0 + k * 32 < n;
            const uint32_t digit = in ? (key[k] >> shift) & (DIGITS - 1) : static_cast<uint32_t>(DIGITS);
            const unsigned same = __match_any_sync(0xffffffffu, digit);
            const unsigned lower = same & ((1u << lane) - 1u);
            unsigned short* mine = ahead + warp * DIGITS + digit;
            if (in) where[k] |= static_cast<uint32_t>(__popc(lower) + *mine) << 16;
            __syncwarp();
            if (in && lower == 0) *mine += static_cast<unsigned short>(__popc(same));
            __syncwarp();
        }
        __syncthreads();
        uint32_t total = 0;
        if (threadIdx.x < DIGITS) {
#pragma unroll 8
            for (int w = 0; w < SORT_WARPS; ++w) {
                const uint32_t c = ahead[w * DIGITS + threadIdx.x];
                ahead[w * DIGITS + threadIdx.x] = static_cast<unsigned short>(total);
                total += c;
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
            offset[threadIdx.x] = base + incl - total;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < SMALL_ROUNDS; ++k) {
            if (k < rounds && i0 + k * 32 < n) {
                const uint32_t digit = (key[k] >> shift) & (DIGITS - 1);
                const uint32_t to = offset[digit] + ahead[warp * DIGITS + digit] + (where[k] >> 16);
                skey[to] = key[k];
                spos[to] = static_cast<unsigned short>(where[k]);
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += SORT_THREADS) {
        keys_out[i] = skey[i];
        pos_out[i] = spos[i];
    }
}

// --------------------------------------------------------------------- gradient

constexpr int GRAD_THREADS = 256;
constexpr int GRAD_UNROLL = 8;           // token rows a thread has in flight
constexpr int MAX_PIECE = 1024;          // sorted tokens per piece at most
constexpr int64_t ZERO_UNIT = 64 * 1024; // bytes of the table a block fills, about
constexpr int64_t ZERO_ROWS = 256;       // and rows at most

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

struct GradArgs {
    const uint32_t *keys, *pos;
    float* edge;                 // [pieces][2][cols]: see the kernel
    uint32_t* long_runs;         // count, then from word 2 the pieces in which long runs start, and their rows
    const uint32_t* touched;     // rows that occur (null: nothing is filled with zeros)
    int64_t n, vocab, nvec, ldt, ldo;
    int64_t units, zero_units, zero_rows;        // pieces (`groups` a block) x column tiles; blocks that fill zero_rows rows each
    int64_t pieces;
    int piece, groups, tiles, accumulate;
    float scale;
};

// Blocks that add up a piece's share of one column tile, and blocks that fill rows with
// zeros, in proportion.  edge: sums of long runs (more tokens than a piece): [0] of a run
// that came in from the piece before, whether or not it goes on; [1] of one that starts here.
// Four blocks of 256 threads an SM (64 registers), six where an access is short: with three
// it is a tenth slower.
// ONE: one piece a block (compiled apart: known places of the window are worth a tenth).
template <typename TT, typename TA, int VEC, bool ONE>
__global__ void __launch_bounds__(GRAD_THREADS, VEC < 4 ? 6 : VEC == 8 && sizeof(TA) == 4 ? 2 : 4)
grad_pieces_kernel(TT* __restrict__ dtable, const TA* __restrict__ dout, const GradArgs a)
{
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    int64_t unit = blockIdx.x;
    if (a.zero_units > 0) {
        const int64_t all = a.units + a.zero_units;
        const int64_t z = unit * a.zero_units / all, after = (unit + 1) * a.zero_units / all;
        if (after > z) {
            zero_rows<TT, VEC>(dtable, a.ldt, a.nvec, z * a.zero_rows, min(a.vocab, (z + 1) * a.zero_rows), a.touched);
            return;
        }
        unit -= z;
    }
    // Narrow tables: several pieces to a block, a group of lanes each.
    extern __shared__ uint32_t windows[];        // per group: keys of [i0 - piece - 1, i1 + piece], positions of [i0, i1 + piece)
    __shared__ int ends[GRAD_THREADS / 32][4];   // where the runs at the piece's ends begin and end, relative to i0
    const int piece = a.piece, groups = ONE ? 1 : a.groups, lanes = ONE ? blockDim.x : blockDim.x / groups;
    const int group = ONE ? 0 : threadIdx.x / lanes, lane = ONE ? threadIdx.x : threadIdx.x % lanes;
    const int64_t p = unit / a.tiles * groups + group, i0 = p * piece;
    const int count = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(piece), a.n - i0)));
    uint32_t* window = windows + group * (5 * piece + 2);
    const uint32_t* key = window + piece + 1;                // key[i]: of sorted token i0 + i
    uint32_t* spos = window + 3 * piece + 2;
    int& first_from = ends[group][0];
    int& first_to = ends[group][1];
    int& last_from = ends[group][2];
    int& last_to = ends[group][3];
    for (int i = lane; i < 3 * piece + 2; i += lanes) {
        const int64_t at = i0 + i - piece - 1;
        window[i] = at >= 0 && at < a.n ? a.keys[at] : 0xffffffffu;      // no row's key
    }
    for (int i = lane; i < 2 * piece; i += lanes) spos[i] = i0 + i < a.n ? a.pos[i0 + i] : 0;
    if (lane == 0) {
        first_from = last_from = -piece;
        first_to = last_to = count + piece;
    }
    __syncthreads();
    const uint32_t k_first = key[0], k_last = key[count > 0 ? count - 1 : 0];
    for (int i = lane - piece; i < count + piece; i += lanes) {
        const uint32_t k = key[i];
        if (i < 0 && k != k_first) atomicMax(&first_from, i + 1);
        if (i >= 0 && k != k_first) atomicMin(&first_to, i);
        if (i < count && k != k_last) atomicMax(&last_from, i + 1);
        if (i >= count && k != k_last) atomicMin(&last_to, i);
    }
    __syncthreads();
    if (count == 0) return;                      // a group behind the last piece
    // a run that came in: a short one is its first piece's, of a long one this piece has a part
    const bool came_in = key[-1] == k_first;
    const bool first_long = came_in && first_to - first_from > piece;
    const int begin = came_in && !first_long ? first_to : 0;
    // a run that starts here and goes on: a short one to its end, of a long one the part here
    const bool goes_on = key[count] == k_last && last_from >= 0;
    const bool last_long = goes_on && last_to - last_from > piece;
    const int end = goes_on && !last_long ? last_to : count;
    const int tile = static_cast<int>(unit % a.tiles);
    if (lane == 0 && tile == 0 && last_long && k_last < a.vocab)
        reinterpret_cast<uint2*>(a.long_runs)[1 + atomicAdd(a.long_runs, 1u)] = make_uint2(static_cast<uint32_t>(p), k_last);
    const int64_t v = static_cast<int64_t>(tile) * lanes + lane;
    if (v >= a.nvec) return;
    const TA* src = dout + v * VEC;
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
    bool first = first_long;
    for (int b = begin; b < end; b += GRAD_UNROLL) {
        Raw<TA, VEC> r[GRAD_UNROLL];
#pragma unroll
        for (int k = 0; k < GRAD_UNROLL; ++k)
            if (b + k < end && key[b + k] < a.vocab) load_raw<true>(r[k], src + static_cast<int64_t>(spos[b + k]) * a.ldo);
#pragma unroll
        for (int k = 0; k < GRAD_UNROLL; ++k) {
            const int i = b + k;
            if (i >= end) break;
            const uint32_t row = key[i];
            if (row >= a.vocab) break;                       // padding sorts last
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[e] += to_f(r[k].e[e]);
            if (i + 1 < end && key[i + 1] == row) continue;
            const bool cut = last_long && i + 1 == end;
            if (first || cut) {
                float* to = a.edge + ((p * 2 + (first ? 0 : 1)) * a.nvec + v) * VEC;
#pragma unroll
                for (int e = 0; e < VEC; ++e) to[e] = sum[e];
            } else {
                write_row<TT, VEC>(dtable + static_cast<int64_t>(row) * a.ldt + v * VEC, sum, a.scale, a.accumulate);
            }
            first = false;
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[e] = 0.0f;
        }
    }
}

// Adds the parts of the long runs: a block takes one run and one column tile at a time.
// blockDim.x = lanes * slices; a slice adds neighbouring pieces, the slices are added in order.
template <typename TT, int VEC>
__global__ void __launch_bounds__(GRAD_THREADS)
grad_join_kernel(TT* __restrict__ dtable, const GradArgs a, int lanes, int col_tiles)
{
    ptx::griddep_wait();
    __shared__ float part[GRAD_THREADS * VEC];
    const int64_t runs = *a.long_runs;
    const int lane = threadIdx.x % lanes, slice = threadIdx.x / lanes, slices = blockDim.x / lanes;
    for (int64_t job = blockIdx.x; job < runs * col_tiles; job += gridDim.x) {
        const uint2 run = reinterpret_cast<const uint2*>(a.long_runs)[1 + job / col_tiles];
        const int64_t p = run.x, v = job % col_tiles * lanes + lane;
        const uint32_t key = run.y;
        // pieces behind p that begin with this row, a block's width at a time
        int64_t parts = 1;                                   // this piece's [1], then [0] of the next ones
        for (;;) {
            const int64_t q = p + parts + threadIdx.x;
            const int same = __syncthreads_count(q < a.pieces && a.keys[q * a.piece] == key);
            parts += same;
            if (same < static_cast<int>(blockDim.x)) break;
        }
        const int64_t per = (parts + slices - 1) / slices;
        const int64_t q0 = slice * per, q1 = min(parts, q0 + per);
        float sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
        if (v < a.nvec) {
#pragma unroll 4
            for (int64_t q = q0; q < q1; ++q) {
                const float* e = a.edge + (((p + q) * 2 + (q == 0 ? 1 : 0)) * a.nvec + v) * VEC;
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum[i] += e[i];
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) part[threadIdx.x * VEC + i] = sum[i];
        __syncthreads();
        if (slice != 0 || v >= a.nvec) continue;
        for (int s = 1; s < slices; ++s)
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] += part[(s * lanes + lane) * VEC + i];
        write_row<TT, VEC>(dtable + static_cast<int64_t>(key) * a.ldt + v * VEC, sum, a.scale, a.accumulate);
    }
}

// ------------------------------------------------------------------------- host

constexpr int64_t MAX_TOKENS = int64_t(1) << 30;
constexpr int64_t MAX_VOCAB = (int64_t(1) << 31) - 2;
constexpr int64_t MAX_COLS = int64_t(1) << 20;           // pieces of a row are counted in 32 bits

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

template <int N>
using Int = std::integral_constant<int, N>;

// f(Int<elements per access>{}): 16 bytes of the narrower type where all rows allow it, two
// elements where one side has 16 bits, else one element.
template <typename TT, typename TA, typename F>
int with_width(const void* table, int64_t ldt, const void* act, int64_t lda, int64_t cols, F f)
{
    constexpr int NARROW = sizeof(TT) < sizeof(TA) ? sizeof(TT) : sizeof(TA);
    auto fits = [&](int vec) {
        const size_t bt = vec * sizeof(TT) < 16 ? vec * sizeof(TT) : 16, ba = vec * sizeof(TA) < 16 ? vec * sizeof(TA) : 16;
        return cols % vec == 0 && (ldt * static_cast<int64_t>(sizeof(TT))) % bt == 0 &&
               (lda * static_cast<int64_t>(sizeof(TA))) % ba == 0 && aligned_to(table, bt) && aligned_to(act, ba);
    };
    if (fits(16 / NARROW)) return f(Int<16 / NARROW>{});
    if constexpr (NARROW == 2) {
        if (fits(2)) return f(Int<2>{});
    }
    return f(Int<1>{});
}

int power_of_two(int64_t n, int most)
{
    int p = 1;
    while (p < n && p < most) p <<= 1;
    return p;
}

struct GradPlan {
    bool small;                          // sorted by one block
    int64_t blocks, per_block;           // of the sort otherwise
    int passes;
    int piece;
    int64_t pieces;
    // byte offsets into the workspace
    int64_t counts, long_runs, touched, keys[2], pos[2], edge, total;
};

GradPlan plan_grad(int sm_count, int64_t n, int64_t vocab, int64_t cols)
{
    GradPlan g{};
    g.small = n <= SMALL_TOKENS;
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
    if (piece > 64) piece = 64;
    if (n / piece > 8192) piece = n / 8192;                  // long lists: bounds the partial sums
    if (piece > MAX_PIECE) piece = MAX_PIECE;
    g.piece = static_cast<int>(piece);
    g.pieces = (n + piece - 1) / piece;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    g.long_runs = take((g.pieces + 1) * 8);                  // cleared together with the next
    g.touched = take((vocab + 31) / 32 * 4);
    g.counts = take(g.blocks * DIGITS * 4);
    for (int i = 0; i < 2; ++i) { g.keys[i] = take(n * 4); g.pos[i] = take(n * 4); }
    g.edge = take(g.pieces * 2 * cols * 4);
    g.total = at;
    return g;
}

// More than SMALL_TOKENS: two launches a pass.  *buffer: which (0 or 1) holds the result.
template <typename I>
int sort_large(sb200_ctx* ctx, const GradPlan& g, unsigned char* ws, const I* ids, int64_t n, int64_t vocab,
               uint32_t* touched, int* buffer, cudaStream_t stream)
{
    auto u32 = [&](int64_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
    uint32_t* counts = u32(g.counts);
    for (int pass = 0; pass < g.passes; ++pass) {
        const int shift = pass * DIGIT_BITS, to = pass & 1;
        uint32_t *kout = u32(g.keys[to]), *pout = u32(g.pos[to]);
        const uint32_t *kin = u32(g.keys[to ^ 1]), *pin = u32(g.pos[to ^ 1]);
        int rc = launch_after(ctx, pass == 0 ? sort_count_kernel<I, true> : sort_count_kernel<I, false>, static_cast<unsigned>(g.blocks), SORT_THREADS, 0, stream,
                              counts, touched, ids, kin, n, g.per_block, vocab, shift, ctx->d_status + TOKEN_RANGE_WORD);
        if (!rc)
            rc = launch_after(ctx, pass == 0 ? sort_scatter_kernel<I, true> : sort_scatter_kernel<I, false>, static_cast<unsigned>(g.blocks), SORT_THREADS, 0,
                              stream, kout, pout, counts, ids, kin, pin, n, g.per_block, vocab, shift, ctx->d_status + TOKEN_RANGE_WORD);
        if (rc) return rc;
    }
    *buffer = (g.passes - 1) & 1;
    return SB200_OK;
}

template <typename I, typename TT, typename TA, int VEC>
int launch_grad(sb200_ctx* ctx, const GradPlan& g, unsigned char* ws, TT* dtable, int64_t ldt, const TA* dout, int64_t ldo,
                const I* ids, int64_t n, int64_t vocab, int64_t cols, float scale, int accumulate, cudaStream_t stream)
{
    auto u32 = [&](int64_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
    const int64_t nvec = cols / VEC;
    uint32_t* touched = nullptr;
    int buffer = 0;
    if (g.small) {
        auto kern = sort_small_kernel<I, TT, VEC>;
        static bool attr_done[16] = {};
        if (ctx->device >= 16 || !attr_done[ctx->device]) {
            if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMALL_SMEM) != cudaSuccess) return SB200_ERR_CUDA;
            if (ctx->device < 16) attr_done[ctx->device] = true;
        }
        int64_t fill = accumulate ? 0 : vocab < ctx->sm_count ? vocab : ctx->sm_count - 1;
        kern<<<static_cast<unsigned>(1 + fill), SORT_THREADS, SMALL_SMEM, stream>>>(
            u32(g.keys[0]), u32(g.pos[0]), u32(g.long_runs), ids, static_cast<int>(n), vocab, g.passes, dtable, ldt, nvec, ctx->d_status + TOKEN_RANGE_WORD);
        ctx->launches += 1;
        if (cudaGetLastError() != cudaSuccess) return SB200_ERR_CUDA;
        if (n == 0) return SB200_OK;
    } else {
        const int64_t clear = accumulate ? 4 : g.touched + (vocab + 31) / 32 * 4 - g.long_runs;
        if (cudaMemsetAsync(ws + g.long_runs, 0, static_cast<size_t>(clear), stream) != cudaSuccess) return SB200_ERR_CUDA;
        if (!accumulate) touched = u32(g.touched);
        if (const int rc = sort_large(ctx, g, ws, ids, n, vocab, touched, &buffer, stream)) return rc;
    }
    GradArgs a{};
    a.keys = u32(g.keys[buffer]);
    a.pos = u32(g.pos[buffer]);
    a.edge = reinterpret_cast<float*>(ws + g.edge);
    a.long_runs = u32(g.long_runs);
    a.touched = touched;
    a.n = n; a.vocab = vocab; a.nvec = nvec; a.ldt = ldt; a.ldo = ldo;
    // a block of 64 to 256 threads per piece; for narrow tables a group of 32 lanes (the windows
    // of a block's groups stay within 40 KB)
    const int threads = nvec > 32 ? power_of_two(nvec, GRAD_THREADS) : GRAD_THREADS;
    a.groups = nvec > 32 ? 1 : GRAD_THREADS / 32;
    while (a.groups > 1 && a.groups * (5 * g.piece + 2) * 4 > 40 * 1024) a.groups /= 2;
    const int lanes_each = threads / a.groups;
    a.pieces = g.pieces;
    a.tiles = static_cast<int>((nvec + lanes_each - 1) / lanes_each);
    a.units = (g.pieces + a.groups - 1) / a.groups * a.tiles;
    if (touched) {
        const int64_t row = cols * static_cast<int64_t>(sizeof(TT));
        a.zero_rows = row * ZERO_ROWS < ZERO_UNIT ? ZERO_ROWS : row < ZERO_UNIT ? ZERO_UNIT / row : 1;
        a.zero_units = (vocab + a.zero_rows - 1) / a.zero_rows;
    }
    a.piece = g.piece;
    a.accumulate = accumulate;
    a.scale = scale;
    if (a.units + a.zero_units > INT32_MAX) return SB200_ERR_TOO_LARGE;
    if (const int rc = launch_after(ctx, a.groups == 1 ? grad_pieces_kernel<TT, TA, VEC, true> : grad_pieces_kernel<TT, TA, VEC, false>, static_cast<unsigned>(a.units + a.zero_units), threads,
                                    static_cast<size_t>(a.groups) * (5 * g.piece + 2) * 4, stream, dtable, dout, a)) return rc;
    // few columns a block and many slices: a run of many pieces is added by slices at the same time
    const int lanes = 32, col_tiles = static_cast<int>((nvec + lanes - 1) / lanes);
    const int64_t jobs = g.pieces * col_tiles, most = 8ll * ctx->sm_count;
    return launch_after(ctx, grad_join_kernel<TT, VEC>, static_cast<unsigned>(jobs < most ? jobs : most), GRAD_THREADS, 0, stream, dtable, a, lanes, col_tiles);
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
    if (!out || !ids || (vocab > 0 && !table) || !aligned_to(ids, index_bits / 8) || !aligned_to(out, type_bytes(type)) ||
        !aligned_to(table, type_bytes(table_type)))
        return SB200_ERR_INVALID_ARG;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    return with_types(table_type, type, [&](auto tt, auto ta) -> int {
        using TT = decltype(tt);
        using TA = decltype(ta);
        return with_width<TT, TA>(table, ldt, out, ldo, cols, [&](auto v) -> int {
            constexpr int VEC = decltype(v)::value;
            const int64_t nvec = cols / VEC;
            const int lanes = power_of_two(nvec, LOOKUP_LANES);
            auto go = [&](auto id, auto r) {
                using I = decltype(id);
                constexpr int ROWS = decltype(r)::value;
                const int64_t per_block = static_cast<int64_t>(LOOKUP_THREADS / lanes) * ROWS;
                const unsigned grid = static_cast<unsigned>((n + per_block - 1) / per_block);
                lookup_kernel<TT, TA, I, VEC, ROWS><<<grid, LOOKUP_THREADS, 0, stream>>>(
                    static_cast<TA*>(out), ldo, static_cast<const TT*>(table), ldt, static_cast<const I*>(ids), n, vocab,
                    static_cast<int>(nvec), scale, lanes, ctx->d_status + TOKEN_RANGE_WORD);
            };
            auto rows = [&](auto id) {
                if (nvec > LOOKUP_LANES) go(id, Int<1>{});
                else go(id, Int<4>{});
            };
            if (index_bits == 64) rows(int64_t{});
            else rows(int32_t{});
            ctx->launches += 1;
            return cudaGetLastError() == cudaSuccess ? SB200_OK : SB200_ERR_CUDA;
        });
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
    if (!dtable || !aligned_to(dtable, type_bytes(table_type)) || !aligned_to(dout, type_bytes(type)) ||
        (n > 0 && (!dout || !ids || !aligned_to(ids, index_bits / 8))))
        return SB200_ERR_INVALID_ARG;
    const GradPlan g = plan_grad(ctx->sm_count, n, vocab, cols);
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < g.total) return SB200_ERR_INVALID_ARG;
    DeviceGuard dev(ctx->device);
    if (!dev.ok) return SB200_ERR_CUDA;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    return with_types(table_type, type, [&](auto tt, auto ta) -> int {
        using TT = decltype(tt);
        using TA = decltype(ta);
        TT* dt = static_cast<TT*>(dtable);
        const TA* dy = static_cast<const TA*>(dout);
        return with_width<TT, TA>(dtable, ldt, dout, ldo, cols, [&](auto v) -> int {
            constexpr int VEC = decltype(v)::value;
            if (index_bits == 64)
                return launch_grad<int64_t, TT, TA, VEC>(ctx, g, ws, dt, ldt, dy, ldo, static_cast<const int64_t*>(ids), n, vocab, cols, scale, accumulate, stream);
            return launch_grad<int32_t, TT, TA, VEC>(ctx, g, ws, dt, ldt, dy, ldo, static_cast<const int32_t*>(ids), n, vocab, cols, scale, accumulate, stream);
        });
    });
}
