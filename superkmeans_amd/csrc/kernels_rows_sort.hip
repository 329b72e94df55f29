// Rows sorted by a key: the places of routed choices in the order of their groups, and the gradient of a table whose rows
// were looked up, by tokens sorted by id.
//
// Both need a stable order, so that nothing depends on which workgroup came first: a choice's slot is the number of
// choices before it in the order (group, place), and a table row's gradient adds its tokens in that order.  There are
// no floating-point atomics.
//
// One pass of the sort over `bins` digit values is three launches.  A wavefront owns a tile of consecutive elements and
// walks it 64 at a time: lanes with equal digits find each other with one ballot per digit bit, a counter per digit in LDS
// carries the tile's count from round to round, and every element's rank in its tile is stored.  Then one wavefront per
// digit scans its row of tile counts, and the last launch adds the three numbers that make up an element's place.
// Against a sort by 8-bit digits this needs one pass for up to 2,048 groups and two for tables of up to 4 million rows.
#include "rows_common.h"

namespace skm {
namespace {

constexpr int MAX_DIGIT_BITS = 11;
constexpr uint32_t MAX_BINS = 1u << MAX_DIGIT_BITS;

// Where an element's key comes from: table ids or choices as the caller has them (anything outside [0, limit) becomes
// limit), or the keys that the pass before left.
struct KeySource {
    const void* at;
    int type;        // SKM_U32 or SKM_I64
    uint32_t limit;
    __device__ __forceinline__ uint32_t operator()(const size_t i) const {
        const uint64_t id = type == SKM_I64 ? reinterpret_cast<const uint64_t*>(at)[i] : (uint64_t) reinterpret_cast<const uint32_t*>(at)[i];
        return id < limit ? (uint32_t) id : limit;
    }
};

// Lanes of the wavefront whose digit equals this lane's (lanes that are not `in` match nobody).
__device__ __forceinline__ unsigned long long equal_lanes(const bool in, const uint32_t digit, const int bits) {
    unsigned long long match = __ballot(in);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long vote = __ballot(in && ((digit >> b) & 1u));
        match &= ((digit >> b) & 1u) ? vote : ~vote;
    }
    return match;
}
__device__ __forceinline__ unsigned long long lanes_below(const uint32_t lane) { return (1ull << lane) - 1ull; }

__device__ __forceinline__ uint32_t wave_inclusive_sum(uint32_t v, const uint32_t lane) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t t = __shfl_up(v, off);
        if (lane >= (uint32_t) off) v += t;
    }
    return v;
}

// First launch of a pass, one wavefront per tile.
__global__ __launch_bounds__(64) void tile_ranks_kernel(
    const KeySource source, const size_t n, const int shift, const uint32_t mask, const int bits, const uint32_t bins,
    const uint32_t rounds, const uint32_t n_tiles, uint16_t* __restrict__ ranks, uint32_t* __restrict__ counts
) {
    extern __shared__ uint32_t count[];
    const uint32_t lane = threadIdx.x;
    for (uint32_t b = lane; b < bins; b += 64) count[b] = 0;
    __syncthreads();
    const size_t first = (size_t) blockIdx.x * rounds * 64;
    for (uint32_t r = 0; r < rounds; ++r) {
        const size_t i = first + (size_t) r * 64 + lane;
        const bool in = i < n;
        const uint32_t digit = in ? (source(i) >> shift) & mask : 0;
        const unsigned long long match = equal_lanes(in, digit, bits);
        const uint32_t below = (uint32_t) __popcll(match & lanes_below(lane));
        const uint32_t before = in ? count[digit] : 0;
        __syncthreads();  // one wavefront: orders the reads before the writes
        if (in) {
            ranks[i] = (uint16_t) (before + below);
            if (below == 0) count[digit] = before + (uint32_t) __popcll(match);
        }
        __syncthreads();
    }
    for (uint32_t b = lane; b < bins; b += 64) counts[(size_t) b * n_tiles + blockIdx.x] = count[b];
}

// Second launch: one wavefront per digit turns its row of tile counts into the counts of the tiles before, and leaves the
// digit's total.
__global__ __launch_bounds__(64) void tile_counts_scan_kernel(
    uint32_t* __restrict__ counts, const uint32_t n_tiles, uint32_t* __restrict__ totals
) {
    const uint32_t lane = threadIdx.x;
    uint32_t* row = counts + (size_t) blockIdx.x * n_tiles;
    uint32_t carry = 0;
    for (uint32_t t0 = 0; t0 < n_tiles; t0 += 64 * 4) {
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t t = t0 + j * 64 + lane;
            v[j] = t < n_tiles ? row[t] : 0;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t t = t0 + j * 64 + lane;
            const uint32_t incl = wave_inclusive_sum(v[j], lane);
            if (t < n_tiles) row[t] = carry + incl - v[j];
            carry += __shfl(incl, 63);
        }
    }
    if (lane == 0) totals[blockIdx.x] = carry;
}

// Exclusive sums of `bins` totals into base[] (LDS), by a workgroup of 256.
__device__ __forceinline__ void scan_totals(const uint32_t* totals, const uint32_t bins, uint32_t* base, uint32_t* wave_sum) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t each = (bins + 255) / 256, from = min(tid * each, bins), to = min(from + each, bins);
    uint32_t mine = 0;
    for (uint32_t b = from; b < to; ++b) mine += totals[b];
    const uint32_t incl = wave_inclusive_sum(mine, lane);
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    uint32_t running = incl - mine;
    for (uint32_t w = 0; w < wave; ++w) running += wave_sum[w];
    for (uint32_t b = from; b < to; ++b) {
        base[b] = running;
        running += totals[b];
    }
    __syncthreads();
}

constexpr int PLACE_PER_THREAD = 4;

// Third launch: every element's place.  A radix pass moves its key and its index there; the only pass of a route writes
// the slots, the order and the offsets instead (bin `bins - 1` then holds the dropped choices).
template <bool ROUTE>
__global__ __launch_bounds__(256) void place_kernel(
    const KeySource source, const size_t n, const int shift, const uint32_t mask, const uint32_t bins, const uint32_t tile,
    const uint32_t n_tiles, const uint16_t* __restrict__ ranks, const uint32_t* __restrict__ counts,
    const uint32_t* __restrict__ totals, const uint32_t* __restrict__ index_in, uint32_t* __restrict__ keys_out,
    uint32_t* __restrict__ index_out, uint32_t* __restrict__ slots, uint32_t* __restrict__ order, uint32_t* __restrict__ offsets
) {
    __shared__ uint32_t base[MAX_BINS];
    __shared__ uint32_t wave_sum[4];
    scan_totals(totals, bins, base, wave_sum);
    if (ROUTE && blockIdx.x == 0)
        for (uint32_t b = threadIdx.x; b < bins; b += 256) offsets[b] = base[b];
#pragma unroll
    for (int j = 0; j < PLACE_PER_THREAD; ++j) {
        const size_t i = ((size_t) blockIdx.x * PLACE_PER_THREAD + j) * 256 + threadIdx.x;
        if (i >= n) continue;
        const uint32_t key = source(i), digit = (key >> shift) & mask;
        const uint32_t place = base[digit] + counts[(size_t) digit * n_tiles + (uint32_t) (i / tile)] + ranks[i];
        if (ROUTE) {
            const bool kept = key < source.limit;
            slots[i] = kept ? place : SKM_NO_ROW;
            if (order) order[place] = kept ? (uint32_t) i : SKM_NO_ROW;
        } else {
            keys_out[place] = key;
            index_out[place] = index_in ? index_in[i] : (uint32_t) i;
        }
    }
}

// offsets[c] = first position of the sorted keys whose key is at least c, for c in [0, limit]: a binary search per c, which
// takes the same time however the keys are spread.
__global__ __launch_bounds__(256) void key_bounds_kernel(
    const uint32_t* __restrict__ keys, const uint32_t n, const uint32_t limit, uint32_t* __restrict__ offsets
) {
    const uint64_t c = (uint64_t) blockIdx.x * 256 + threadIdx.x;
    if (c > limit) return;
    uint32_t low = 0, high = n;
    while (low < high) {
        const uint32_t mid = low + (high - low) / 2;
        if (keys[mid] < c) low = mid + 1;
        else high = mid;
    }
    offsets[c] = low;
}

// Slots and order of a route that took several passes.
__global__ __launch_bounds__(256) void route_places_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ index, const size_t n, const uint32_t groups,
    uint32_t* __restrict__ slots, uint32_t* __restrict__ order
) {
    const size_t p = (size_t) blockIdx.x * 256 + threadIdx.x;
    if (p >= n) return;
    const bool kept = keys[p] < groups;
    slots[index[p]] = kept ? (uint32_t) p : SKM_NO_ROW;
    if (order) order[p] = kept ? index[p] : SKM_NO_ROW;
}

// A whole route in one workgroup of 16 wavefronts, each with a contiguous share of the choices and counters of its own:
// a decoding step's few thousand choices cost one launch instead of three.
constexpr uint32_t ONE_LAUNCH_BINS = 1024, ONE_LAUNCH_ROUNDS = 8;
constexpr size_t ONE_LAUNCH_CHOICES = (size_t) 1024 * ONE_LAUNCH_ROUNDS;

template <int ROUNDS>
__global__ __launch_bounds__(1024) void route_one_launch_kernel(
    const uint32_t* __restrict__ choices, const uint32_t n, const uint32_t groups, const int bits, uint32_t* __restrict__ slots,
    uint32_t* __restrict__ order, uint32_t* __restrict__ offsets
) {
    extern __shared__ uint16_t count16[];  // [16][groups + 1]; no count passes ONE_LAUNCH_CHOICES
    __shared__ uint32_t wave_sum[16];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = groups + 1;
    for (uint32_t b = tid; b < 16 * bins; b += 1024) count16[b] = 0;
    __syncthreads();
    uint16_t* mine = count16 + wave * bins;
    const uint32_t first = wave * ROUNDS * 64;
    uint32_t key[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = first + r * 64 + lane;
        key[r] = i < n ? choices[i] : 0;
        key[r] = key[r] < groups ? key[r] : groups;
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool in = first + r * 64 + lane < n;
        const unsigned long long match = equal_lanes(in, key[r], bits);
        const uint32_t below = (uint32_t) __popcll(match & lanes_below(lane));
        const uint32_t before = in ? mine[key[r]] : 0;
        rank[r] = before + below;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // a wavefront's LDS accesses stay in this order
        if (in && below == 0) mine[key[r]] = (uint16_t) (before + __popcll(match));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    // thread b: the counts of bin b in the wavefronts before, then the bins before
    uint32_t total = 0;
    if (tid < bins)
        for (int w = 0; w < 16; ++w) {
            const uint32_t c = count16[w * bins + tid];
            count16[w * bins + tid] = (uint16_t) total;
            total += c;
        }
    const uint32_t incl = wave_inclusive_sum(total, lane);
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    uint32_t base = incl - total;
    for (uint32_t w = 0; w < wave; ++w) base += wave_sum[w];
    if (tid < bins) {
        offsets[tid] = base;
        for (int w = 0; w < 16; ++w) count16[w * bins + tid] += (uint16_t) base;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = first + r * 64 + lane;
        if (i >= n) continue;
        const uint32_t place = mine[key[r]] + rank[r];
        const bool kept = key[r] < groups;
        slots[i] = kept ? place : SKM_NO_ROW;
        if (order) order[place] = kept ? i : SKM_NO_ROW;
    }
}

int bits_for(const uint64_t bins) {
    int bits = 1;
    while ((uint64_t(1) << bits) < bins) ++bits;
    return bits;
}

size_t aligned(const size_t bytes) { return (bytes + 255) / 256 * 256; }

// Plan of a sort of n keys in [0, limit]: passes of equal digit widths, and where its arrays lie in the scratch.
struct SortPlan {
    size_t n;
    uint32_t limit;
    int passes, bits_per_pass;
    uint32_t bins, rounds, tile, n_tiles;
    size_t at_ranks, at_counts, at_totals, at_keys[2], at_index[2], bytes;

    SortPlan(const size_t n_, const size_t limit_, const bool one_pass_moves_nothing) : n(n_), limit((uint32_t) limit_) {
        const int bits = bits_for((uint64_t) limit + 1);
        passes = (bits + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
        bits_per_pass = (bits + passes - 1) / passes;
        bins = passes == 1 ? limit + 1 : 1u << bits_per_pass;
        // a short tile spreads few keys over many wavefronts; with many keys a tile has at least as many elements as
        // there are digit values, so that the counts take no more memory than the keys
        rounds = n <= (size_t(1) << 20) ? 8 : std::max<uint32_t>(8, bins / 64);
        tile = rounds * 64;
        n_tiles = (uint32_t) ((n + tile - 1) / tile);
        size_t at = 0;
        const auto take = [&](const size_t bytes) {
            const size_t here = at;
            at += aligned(bytes);
            return here;
        };
        at_ranks = take(n * 2);
        at_counts = take((size_t) bins * n_tiles * 4);
        at_totals = take((size_t) bins * 4);
        const bool moves = passes > 1 || !one_pass_moves_nothing;
        for (int b = 0; b < 2; ++b) {
            at_keys[b] = moves && (b == 0 || passes > 1) ? take(n * 4) : 0;
            at_index[b] = moves && (b == 0 || passes > 1) ? take(n * 4) : 0;
        }
        bytes = at;
    }
    int last() const { return (passes - 1) & 1; }  // which pair of arrays holds the result
};

struct RouteOut {
    uint32_t *slots, *order, *offsets;
};

// Queues the passes of a sort; `route`: the single pass writes these instead of sorted keys.
int launch_sort(skm_ctx* ctx, const SortPlan& p, const KeySource& first, char* scratch, const RouteOut* route) {
    uint16_t* ranks = (uint16_t*) (scratch + p.at_ranks);
    uint32_t* counts = (uint32_t*) (scratch + p.at_counts);
    uint32_t* totals = (uint32_t*) (scratch + p.at_totals);
    const unsigned place_blocks = (unsigned) ((p.n + 256 * PLACE_PER_THREAD - 1) / (256 * PLACE_PER_THREAD));
    KeySource source = first;
    const uint32_t* index_in = nullptr;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.bits_per_pass;
        const uint32_t mask = p.passes == 1 ? 0xffffffffu : p.bins - 1;
        tile_ranks_kernel<<<p.n_tiles, 64, p.bins * 4, ctx->stream>>>(source, p.n, shift, mask, bits_for(p.bins), p.bins, p.rounds,
                                                                     p.n_tiles, ranks, counts);
        SKM_TRY(check_hip(hipGetLastError(), "tile_ranks_kernel launch"));
        tile_counts_scan_kernel<<<p.bins, 64, 0, ctx->stream>>>(counts, p.n_tiles, totals);
        SKM_TRY(check_hip(hipGetLastError(), "tile_counts_scan_kernel launch"));
        uint32_t* keys_out = (uint32_t*) (scratch + p.at_keys[pass & 1]);
        uint32_t* index_out = (uint32_t*) (scratch + p.at_index[pass & 1]);
        if (route)
            place_kernel<true><<<place_blocks, 256, 0, ctx->stream>>>(source, p.n, shift, mask, p.bins, p.tile, p.n_tiles, ranks, counts,
                                                                      totals, nullptr, nullptr, nullptr, route->slots, route->order,
                                                                      route->offsets);
        else
            place_kernel<false><<<place_blocks, 256, 0, ctx->stream>>>(source, p.n, shift, mask, p.bins, p.tile, p.n_tiles, ranks, counts,
                                                                       totals, index_in, keys_out, index_out, nullptr, nullptr, nullptr);
        SKM_TRY(check_hip(hipGetLastError(), "place_kernel launch"));
        source = KeySource{keys_out, SKM_U32, p.limit};
        index_in = index_out;
    }
    return SKM_OK;
}

// ---------------------------------------------------------------------------------------------
// Gradient of a lookup
// ---------------------------------------------------------------------------------------------

constexpr int GRAD_AHEAD = 4;  // token rows requested before the first is added

// Adds the grad rows of the tokens at [j0, j1) of `index` (sorted order) to sum; `at`: the lane's vector in the row.
template <class T, int E>
__device__ __forceinline__ void add_tokens(const T* __restrict__ grad, const size_t stride, const uint32_t* __restrict__ index,
                                           const uint32_t j0, const uint32_t j1, const uint32_t at, vec_of<float, E>& sum) {
    for (uint32_t j = j0; j < j1; j += GRAD_AHEAD) {
        vec_of<T, E> v[GRAD_AHEAD];
#pragma unroll
        for (int q = 0; q < GRAD_AHEAD; ++q) {
            const uint32_t i = index[min(j + q, j1 - 1)];
            v[q] = load_vec<T, E>(grad + (size_t) i * stride + (size_t) at * E);
        }
#pragma unroll
        for (int q = 0; q < GRAD_AHEAD; ++q)
            if (j + q < j1) sum += widen<E>(v[q]);
    }
}

template <class O, int E>
__device__ __forceinline__ void put_sum(O* to, const vec_of<float, E> sum, const float scale, const bool accumulate) {
    vec_of<float, E> r = sum * scale;
    if (accumulate) r += widen<E>(load_vec<O, E>(to));
    store_vec<O, E>(to, narrow<O, E>(r));
}

// Table rows of at most `most` tokens: a sum each, or zeros where there are none (nothing when accumulating).
template <class T, class O, int E>
__global__ __launch_bounds__(ROWS_THREADS) void lookup_grad_rows_kernel(
    const T* __restrict__ grad, const size_t grad_stride, const uint32_t* __restrict__ index, const uint32_t* __restrict__ offsets,
    const size_t rows, const uint32_t most, const float scale, O* __restrict__ out, const size_t out_stride, const int accumulate,
    const RowSplit s
) {
    const uint32_t lane = threadIdx.x & 63, in_row = lane & (s.lanes - 1), row_of_wave = lane / s.lanes;
    const uint64_t step = (uint64_t) gridDim.x * (ROWS_THREADS / 64);
    for (uint64_t u = (uint64_t) blockIdx.x * (ROWS_THREADS / 64) + (threadIdx.x >> 6); u < s.units; u += step) {
        const size_t row = (size_t) (u / s.pieces) * (64 / s.lanes) + row_of_wave;
        const uint32_t at = (uint32_t) (u % s.pieces) * s.lanes + in_row;
        if (row >= rows || at >= s.vectors) continue;
        const uint32_t j0 = offsets[row], j1 = offsets[row + 1];
        if (j1 - j0 > most || (accumulate && j0 == j1)) continue;
        vec_of<float, E> sum = {};
        add_tokens<T, E>(grad, grad_stride, index, j0, j1, at, sum);
        put_sum<O, E>(out + row * out_stride + (size_t) at * E, sum, scale, accumulate);
    }
}

// Rows of more tokens than that: the sorted tokens are cut into chunks of `most`.  A chunk leaves at most two sums: of the
// row that its first token belongs to (slot 0) and of another one that its last token belongs to (slot 1), as far
// as they are such long rows.
template <class T, int E>
__global__ __launch_bounds__(ROWS_THREADS) void lookup_grad_chunks_kernel(
    const T* __restrict__ grad, const size_t grad_stride, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ index,
    const uint32_t* __restrict__ offsets, const uint32_t n, const uint32_t rows, const uint32_t most, float* __restrict__ parts,
    const uint32_t vectors, const uint32_t pieces, const uint32_t chunks
) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t u = (uint64_t) blockIdx.x * (ROWS_THREADS / 64) + (threadIdx.x >> 6);
    if (u >= (uint64_t) chunks * pieces) return;
    const uint32_t c = (uint32_t) (u / pieces), at = (uint32_t) (u % pieces) * 64 + lane;
    if (at >= vectors) return;
    const uint32_t from = c * most, to = (uint32_t) min((uint64_t) n, (uint64_t) from + most);
    const uint32_t head = keys[from], tail = keys[to - 1];
    float* part = parts + (size_t) c * 2 * vectors * E + (size_t) at * E;
    if (head < rows && offsets[head + 1] - offsets[head] > most) {
        vec_of<float, E> sum = {};
        add_tokens<T, E>(grad, grad_stride, index, from, min(to, offsets[head + 1]), at, sum);
        store_vec<float, E>(part, sum);
    }
    if (tail < rows && offsets[tail] > from && offsets[tail + 1] - offsets[tail] > most) {
        vec_of<float, E> sum = {};
        add_tokens<T, E>(grad, grad_stride, index, offsets[tail], to, at, sum);
        store_vec<float, E>(part + (size_t) vectors * E, sum);
    }
}

// The long row that begins in a chunk (a row of more than `most` tokens covers the end of the chunk it begins in, so
// there is at most one): its chunks' sums added up in order.
template <class O, int E>
__global__ __launch_bounds__(ROWS_THREADS) void lookup_grad_join_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ offsets, const uint32_t n, const uint32_t rows, const uint32_t most,
    const float* __restrict__ parts, const float scale, O* __restrict__ out, const size_t out_stride, const int accumulate,
    const uint32_t vectors, const uint32_t pieces, const uint32_t chunks
) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t u = (uint64_t) blockIdx.x * (ROWS_THREADS / 64) + (threadIdx.x >> 6);
    if (u >= (uint64_t) chunks * pieces) return;
    const uint32_t c = (uint32_t) (u / pieces), at = (uint32_t) (u % pieces) * 64 + lane;
    if (at >= vectors) return;
    const uint32_t from = c * most, to = (uint32_t) min((uint64_t) n, (uint64_t) from + most);
    const uint32_t row = keys[to - 1];
    if (row >= rows || offsets[row] < from || offsets[row + 1] - offsets[row] <= most) return;
    const uint32_t last = (offsets[row + 1] - 1) / most;
    const size_t chunk = (size_t) 2 * vectors * E;
    const float* part = parts + (size_t) at * E;
    vec_of<float, E> sum = load_vec<float, E>(part + c * chunk + (offsets[row] == from ? 0 : (size_t) vectors * E));
    for (uint32_t i = c + 1; i <= last; ++i) sum += load_vec<float, E>(part + i * chunk);
    put_sum<O, E>(out + (size_t) row * out_stride + (size_t) at * E, sum, scale, accumulate);
}

// Few tokens: no sort.  The first token of every id looks through the others for the same id and adds them in order; the
// table was set to zeros before (unless accumulating).
constexpr size_t FEW_TOKENS = 2048;

template <class T, class O, int E>
__global__ __launch_bounds__(ROWS_THREADS) void lookup_grad_few_kernel(
    const T* __restrict__ grad, const size_t grad_stride, const KeySource source, const uint32_t n, const float scale,
    O* __restrict__ out, const size_t out_stride, const int accumulate, const uint32_t vectors, const uint32_t pieces
) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t u = blockIdx.x * (ROWS_THREADS / 64) + (threadIdx.x >> 6);
    if (u >= n * pieces) return;
    const uint32_t t = u / pieces, at = (u % pieces) * 64 + lane;
    const uint32_t id = source(t);
    if (id == source.limit) return;
    bool earlier = false;
    for (uint32_t s = lane; s < t; s += 64) earlier |= source(s) == id;
    if (__ballot(earlier)) return;
    vec_of<float, E> sum = {};
    for (uint32_t s0 = t / 64 * 64; s0 < n; s0 += 64) {
        const uint32_t s = s0 + lane;
        unsigned long long same = __ballot(s >= t && s < n && source(s) == id);
        while (same) {
            const uint32_t i = s0 + (uint32_t) __builtin_ctzll(same);
            same &= same - 1;
            if (at < vectors) sum += widen<E>(load_vec<T, E>(grad + (size_t) i * grad_stride + (size_t) at * E));
        }
    }
    if (at < vectors) put_sum<O, E>(out + (size_t) id * out_stride + (size_t) at * E, sum, scale, accumulate);
}

template <class O, int E>
__global__ __launch_bounds__(ROWS_THREADS) void zero_rows_kernel(O* __restrict__ out, const size_t rows, const size_t stride, const RowSplit s) {
    const uint32_t lane = threadIdx.x & 63, in_row = lane & (s.lanes - 1), row_of_wave = lane / s.lanes;
    const uint64_t step = (uint64_t) gridDim.x * (ROWS_THREADS / 64);
    for (uint64_t u = (uint64_t) blockIdx.x * (ROWS_THREADS / 64) + (threadIdx.x >> 6); u < s.units; u += step) {
        const size_t row = (size_t) (u / s.pieces) * (64 / s.lanes) + row_of_wave;
        const uint32_t at = (uint32_t) (u % s.pieces) * s.lanes + in_row;
        if (row < rows && at < s.vectors) store_vec<O, E>(out + row * stride + (size_t) at * E, vec_of<O, E>{});
    }
}

// Scratch of the sorted path: the sort, the rows' offsets, the chunks' sums.
struct GradPlan {
    SortPlan sort;
    uint32_t most, chunks;
    size_t at_offsets, at_parts, bytes;
    GradPlan(const size_t n, const size_t rows, const size_t d) : sort(n, rows, false) {
        most = n <= 32768 ? 64 : 256;
        chunks = (uint32_t) ((n + most - 1) / most);
        at_offsets = sort.bytes;
        at_parts = at_offsets + aligned((rows + 1) * 4);
        bytes = at_parts + aligned((size_t) chunks * 2 * d * 4);
    }
};

} // namespace
} // namespace skm

using namespace skm;

extern "C" {

int skm_route_scratch(size_t n, size_t choices, size_t groups, size_t* out_bytes) {
    SKM_REQUIRE(out_bytes, "null output");
    SKM_REQUIRE(groups > 0 && groups <= SKM_ROUTE_MAX_GROUPS, "groups out of range");
    SKM_REQUIRE(choices > 0 && choices <= SKM_ROUTE_MAX_CHOICES, "choices out of range");
    SKM_REQUIRE(n <= SKM_ROUTE_MAX_PLACES / choices, "n * choices out of range");
    const size_t places = n * choices;
    *out_bytes = places == 0 || (places <= ONE_LAUNCH_CHOICES && groups < ONE_LAUNCH_BINS) ? 0 : SortPlan(places, groups, true).bytes;
    return SKM_OK;
}

int skm_route(skm_ctx* ctx, const uint32_t* d_choices, size_t n, size_t choices, size_t groups, uint32_t* d_slots,
              uint32_t* d_order, uint32_t* d_offsets, void* d_scratch, size_t scratch_bytes) {
    SKM_REQUIRE(ctx, "null context");
    size_t need = 0;
    SKM_TRY(skm_route_scratch(n, choices, groups, &need));
    SKM_REQUIRE(d_offsets && (n == 0 || (d_choices && d_slots)), "null pointer");
    SKM_REQUIRE((address(d_choices) | address(d_slots) | address(d_order) | address(d_offsets)) % 4 == 0,
                "pointers must be aligned to their elements");
    const size_t places = n * choices;
    SKM_REQUIRE(!overlap(d_choices, places * 4, d_slots, places * 4) && !overlap(d_choices, places * 4, d_order, places * 4),
                "slots and order must not overlap the choices");
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/route");
    if (places == 0) return skm_fill_u32(ctx, d_offsets, 0, groups + 1);
    if (places <= ONE_LAUNCH_CHOICES && groups < ONE_LAUNCH_BINS) {
        const size_t lds = 16 * (groups + 1) * sizeof(uint16_t);
        const int bits = bits_for(groups + 1);
        const auto launch = [&](auto rounds) {
            route_one_launch_kernel<decltype(rounds)::value><<<1, 1024, lds, ctx->stream>>>(
                d_choices, (uint32_t) places, (uint32_t) groups, bits, d_slots, d_order, d_offsets);
            return check_hip(hipGetLastError(), "route_one_launch_kernel launch");
        };
        if (places <= 1024) return launch(std::integral_constant<int, 1>{});
        if (places <= 1024 * 3) return launch(std::integral_constant<int, 3>{});
        return launch(std::integral_constant<int, ONE_LAUNCH_ROUNDS>{});
    }
    const SortPlan plan(places, groups, true);
    void* scratch = nullptr;
    SKM_TRY(call_scratch(ctx, __func__, d_scratch, scratch_bytes, plan.bytes, &scratch));
    const KeySource source{d_choices, SKM_U32, (uint32_t) groups};
    const RouteOut out{d_slots, d_order, d_offsets};
    if (plan.passes == 1) return launch_sort(ctx, plan, source, (char*) scratch, &out);
    SKM_TRY(launch_sort(ctx, plan, source, (char*) scratch, nullptr));
    const uint32_t* keys = (const uint32_t*) ((char*) scratch + plan.at_keys[plan.last()]);
    const uint32_t* index = (const uint32_t*) ((char*) scratch + plan.at_index[plan.last()]);
    key_bounds_kernel<<<(unsigned) (groups / 256 + 1), 256, 0, ctx->stream>>>(keys, (uint32_t) places, (uint32_t) groups, d_offsets);
    SKM_TRY(check_hip(hipGetLastError(), "key_bounds_kernel launch"));
    route_places_kernel<<<(unsigned) ((places + 255) / 256), 256, 0, ctx->stream>>>(keys, index, places, (uint32_t) groups, d_slots, d_order);
    return check_hip(hipGetLastError(), "route_places_kernel launch");
}

int skm_lookup_rows_grad_scratch(size_t n, size_t rows, size_t d, size_t* out_bytes) {
    SKM_REQUIRE(out_bytes, "null output");
    SKM_REQUIRE(d > 0 && d <= SKM_ROW_MAX_D, "d out of range");
    SKM_REQUIRE(rows < SKM_NO_ROW && n <= SKM_ROUTE_MAX_PLACES, "rows or n out of range");
    *out_bytes = n <= FEW_TOKENS || rows == 0 ? 0 : GradPlan(n, rows, d).bytes;
    return SKM_OK;
}

int skm_lookup_rows_grad(skm_ctx* ctx, const void* d_grad, int type, size_t grad_stride, const void* d_ids, int ids_type, size_t n,
                         size_t rows, size_t d, float scale, void* d_out, int out_type, size_t out_stride, int accumulate,
                         void* d_scratch, size_t scratch_bytes) {
    SKM_REQUIRE(ctx, "null context");
    SKM_REQUIRE(is_value_type(type), "type must be SKM_F32, SKM_F16 or SKM_BF16");
    SKM_REQUIRE(out_type == type || out_type == SKM_F32, "out_type must be the gradient's type or SKM_F32");
    SKM_REQUIRE(ids_type == SKM_U32 || ids_type == SKM_I64, "ids_type must be SKM_U32 or SKM_I64");
    size_t need = 0;
    SKM_TRY(skm_lookup_rows_grad_scratch(n, rows, d, &need));
    SKM_REQUIRE(grad_stride >= d && out_stride >= d, "strides must be at least d");
    if (rows == 0 || (n == 0 && accumulate)) return SKM_OK;
    SKM_REQUIRE(d_out && (n == 0 || (d_grad && d_ids)), "null pointer");
    const size_t size = type_size(type), out_size = type_size(out_type);
    SKM_REQUIRE(address(d_ids) % (ids_type == SKM_I64 ? 8 : 4) == 0 && address(d_grad) % size == 0 && address(d_out) % out_size == 0,
                "pointers must be aligned to their elements");
    SKM_REQUIRE(!overlap(d_grad, span(n, grad_stride, d, size), d_out, span(rows, out_stride, d, out_size)), "out overlaps the gradient");
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/lookup_grad");
    // elements per lane: what the gradient's alignment gives in one load and the table's in stores of at most 16 bytes
    const size_t in_width = common_width({address(d_grad), grad_stride * size, d * size});
    const size_t out_width = common_width({address(d_out), out_stride * out_size, d * out_size});
    size_t per_lane = in_width / size;
    if (out_width < 16) per_lane = std::min(per_lane, out_width / out_size);
    const KeySource source{d_ids, ids_type, (uint32_t) rows};
    const auto run = [&](auto sample, auto out_sample) {
        using T = decltype(sample);
        using O = decltype(out_sample);
        return for_width<T>(per_lane * size, [&](auto elements) {
            constexpr int E = decltype(elements)::value;
            const uint32_t vectors = (uint32_t) (d / E), pieces = (vectors + 63) / 64;
            const RowSplit s = split_rows(rows, vectors, 1);
            O* out = (O*) d_out;
            if (n <= FEW_TOKENS) {
                if (!accumulate) {
                    zero_rows_kernel<O, E><<<row_blocks(s), ROWS_THREADS, 0, ctx->stream>>>(out, rows, out_stride, s);
                    SKM_TRY(check_hip(hipGetLastError(), "zero_rows_kernel launch"));
                }
                if (n == 0) return (int) SKM_OK;
                const unsigned blocks = (unsigned) ((n * pieces + ROWS_THREADS / 64 - 1) / (ROWS_THREADS / 64));
                lookup_grad_few_kernel<T, O, E><<<blocks, ROWS_THREADS, 0, ctx->stream>>>(
                    (const T*) d_grad, grad_stride, source, (uint32_t) n, scale, out, out_stride, accumulate, vectors, pieces);
                return check_hip(hipGetLastError(), "lookup_grad_few_kernel launch");
            }
            const GradPlan plan(n, rows, d);
            void* at = nullptr;
            SKM_TRY(call_scratch(ctx, "skm_lookup_rows_grad", d_scratch, scratch_bytes, plan.bytes, &at));
            char* scratch = (char*) at;
            SKM_TRY(launch_sort(ctx, plan.sort, source, scratch, nullptr));
            const uint32_t* keys = (const uint32_t*) (scratch + plan.sort.at_keys[plan.sort.last()]);
            const uint32_t* index = (const uint32_t*) (scratch + plan.sort.at_index[plan.sort.last()]);
            uint32_t* offsets = (uint32_t*) (scratch + plan.at_offsets);
            float* parts = (float*) (scratch + plan.at_parts);
            key_bounds_kernel<<<(unsigned) (rows / 256 + 1), 256, 0, ctx->stream>>>(keys, (uint32_t) n, (uint32_t) rows, offsets);
            SKM_TRY(check_hip(hipGetLastError(), "key_bounds_kernel launch"));
            lookup_grad_rows_kernel<T, O, E><<<row_blocks(s), ROWS_THREADS, 0, ctx->stream>>>(
                (const T*) d_grad, grad_stride, index, offsets, rows, plan.most, scale, out, out_stride, accumulate, s);
            SKM_TRY(check_hip(hipGetLastError(), "lookup_grad_rows_kernel launch"));
            const uint64_t units = (uint64_t) plan.chunks * pieces;
            const unsigned blocks = (unsigned) ((units + ROWS_THREADS / 64 - 1) / (ROWS_THREADS / 64));
            lookup_grad_chunks_kernel<T, E><<<blocks, ROWS_THREADS, 0, ctx->stream>>>(
                (const T*) d_grad, grad_stride, keys, index, offsets, (uint32_t) n, (uint32_t) rows, plan.most, parts, vectors, pieces,
                plan.chunks);
            SKM_TRY(check_hip(hipGetLastError(), "lookup_grad_chunks_kernel launch"));
            lookup_grad_join_kernel<O, E><<<blocks, ROWS_THREADS, 0, ctx->stream>>>(
                keys, offsets, (uint32_t) n, (uint32_t) rows, plan.most, parts, scale, out, out_stride, accumulate, vectors, pieces,
                plan.chunks);
            return check_hip(hipGetLastError(), "lookup_grad_join_kernel launch");
        });
    };
    return for_type(type, [&](auto sample) {
        if (out_type == type) return run(sample, sample);
        return run(sample, float{});
    });
}

} // extern "C"
