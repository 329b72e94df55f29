// Rows sorted by a key: the places of routed choices in the order of their groups, and the gradient of a table whose rows
// were looked up, by tokens sorted by id.
//
// Both need a stable order, so that nothing depends on which workgroup came first: a choice's slot is the number of
// choices before it in the order (group, place), and a table row's gradient adds its tokens in that order.  There are
// no floating-point atomics.
//
// One pass of the sort over `bins` digit values is two launches.  A workgroup of 16 wavefronts owns a tile of consecutive
// elements and every wavefront a contiguous share of it, which it walks 64 at a time: lanes with equal digits find each other
// with one ballot per digit bit, and a counter per digit and wavefront in LDS carries the count from round to round.  That
// gives every element's rank in its tile, and the tile its counts.  The second launch adds up the counts of the tiles
// before (every workgroup reads the whole table, which is small; with many tiles a launch in between scans it) and moves
// the elements: 5 + 7 us for 65,536 keys of 9 bits, bound by latencies.  Up to 8,192 choices are one tile, and one launch: 512 of
// 64 groups 3.7 us.  With 10-bit digits a route takes one pass for up to 1,023 groups and a table of up to a million rows two.
#include "rows_common.h"

namespace skm {
namespace {

constexpr int MAX_DIGIT_BITS = 10;
constexpr uint32_t MAX_BINS = 1u << MAX_DIGIT_BITS;  // a thread of a workgroup each
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int MAX_ROUNDS = 8;
constexpr uint32_t TILES_WITHOUT_SCAN = 128;

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

// Exclusive sum over the threads of a workgroup; ends on a barrier.
__device__ __forceinline__ uint32_t block_exclusive_sum(const uint32_t v, uint32_t* wave_sum) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t incl = wave_inclusive_sum(v, lane);
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    uint32_t base = incl - v;
    for (uint32_t w = 0; w < wave; ++w) base += wave_sum[w];
    __syncthreads();
    return base;
}

// Where a pass puts its elements: a radix pass their keys and indices, the only pass of a route the slots, the order
// and the offsets (bin `bins - 1` then holds the dropped choices).
struct Places {
    const uint32_t* index_in;  // null: an element's index is its position
    uint32_t *keys, *index;
    uint32_t *slots, *order, *offsets;
    template <bool ROUTE>
    __device__ __forceinline__ void put(const size_t i, const uint32_t key, const uint32_t limit, const uint32_t place) const {
        if (ROUTE) {
            const bool kept = key < limit;
            slots[i] = kept ? place : SKM_NO_ROW;
            if (order) order[place] = kept ? (uint32_t) i : SKM_NO_ROW;
        } else {
            keys[place] = key;
            index[place] = index_in ? index_in[i] : (uint32_t) i;
        }
    }
};

// First launch of a pass: ranks in the tile and the tile's counts.  ONLY: the tile is all there is, and a route is done
// with it.
template <int ROUNDS, bool ONLY>
__global__ __launch_bounds__(SORT_THREADS) void tile_ranks_kernel(
    const KeySource source, const size_t n, const int shift, const uint32_t mask, const int bits, const uint32_t bins,
    uint16_t* __restrict__ ranks, uint32_t* __restrict__ counts, const Places places
) {
    extern __shared__ uint16_t count[];  // [SORT_WAVES][bins]; a tile has at most 8,192 elements
    __shared__ uint32_t wave_sum[SORT_WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (uint32_t b = tid; b < SORT_WAVES * bins; b += SORT_THREADS) count[b] = 0;
    const size_t first = (size_t) blockIdx.x * (SORT_THREADS * ROUNDS) + wave * (ROUNDS * 64) + lane;
    uint32_t key[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) key[r] = first + r * 64 < n ? source(first + r * 64) : 0;
    __syncthreads();
    uint16_t* mine = count + wave * bins;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool in = first + r * 64 < n;
        const uint32_t digit = (key[r] >> shift) & mask;
        const unsigned long long match = equal_lanes(in, digit, bits);
        const uint32_t below = (uint32_t) __popcll(match & lanes_below(lane));
        const uint32_t before = in ? mine[digit] : 0;
        rank[r] = before + below;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // a wavefront's LDS accesses stay in this order
        if (in && below == 0) mine[digit] = (uint16_t) (before + __popcll(match));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    // thread b: the counts of digit b in the wavefronts before
    uint32_t total = 0;
    if (tid < bins)
        for (int w = 0; w < SORT_WAVES; ++w) {
            const uint32_t c = count[w * bins + tid];
            count[w * bins + tid] = (uint16_t) total;
            total += c;
        }
    if (ONLY) {
        const uint32_t base = block_exclusive_sum(total, wave_sum);
        if (tid < bins) {
            places.offsets[tid] = base;
            for (int w = 0; w < SORT_WAVES; ++w) count[w * bins + tid] += (uint16_t) base;
        }
    } else if (tid < bins) {
        counts[(size_t) blockIdx.x * bins + tid] = total;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const size_t i = first + r * 64;
        if (i >= n) continue;
        const uint32_t at = mine[(key[r] >> shift) & mask] + rank[r];
        if (ONLY) places.put<true>(i, key[r], source.limit, at);
        else ranks[i] = (uint16_t) at;
    }
}

// With many tiles: a wavefront per digit turns the tiles' counts into the counts of the tiles before, and leaves the total.
__global__ __launch_bounds__(64) void tile_counts_scan_kernel(
    uint32_t* __restrict__ counts, const uint32_t bins, const uint32_t n_tiles, uint32_t* __restrict__ totals
) {
    const uint32_t lane = threadIdx.x;
    uint32_t carry = 0;
    for (uint32_t t0 = 0; t0 < n_tiles; t0 += 64 * 4) {
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t t = t0 + j * 64 + lane;
            v[j] = t < n_tiles ? counts[(size_t) t * bins + blockIdx.x] : 0;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t t = t0 + j * 64 + lane;
            const uint32_t incl = wave_inclusive_sum(v[j], lane);
            if (t < n_tiles) counts[(size_t) t * bins + blockIdx.x] = carry + incl - v[j];
            carry += __shfl(incl, 63);
        }
    }
    if (lane == 0) totals[blockIdx.x] = carry;
}

// Last launch: the elements of a tile to their places.  SCANNED: the counts are those of the tiles before already.
template <bool ROUTE, bool SCANNED>
__global__ __launch_bounds__(SORT_THREADS) void place_kernel(
    const KeySource source, const size_t n, const int shift, const uint32_t mask, const uint32_t bins, const uint32_t rounds,
    const uint32_t n_tiles, const uint16_t* __restrict__ ranks, const uint32_t* __restrict__ counts,
    const uint32_t* __restrict__ totals, const Places places
) {
    __shared__ uint32_t base[MAX_BINS];
    __shared__ uint32_t wave_sum[SORT_WAVES];
    const uint32_t tid = threadIdx.x, tile = blockIdx.x;
    uint32_t before = 0, total = 0;
    if (tid < bins) {
        if (SCANNED) {
            before = counts[(size_t) tile * bins + tid];
            total = totals[tid];
        } else {
#pragma unroll 8
            for (uint32_t t = 0; t < n_tiles; ++t) {
                const uint32_t c = counts[(size_t) t * bins + tid];
                total += c;
                before += t < tile ? c : 0;
            }
        }
    }
    const uint32_t start = block_exclusive_sum(total, wave_sum);
    if (tid < bins) {
        base[tid] = start + before;
        if (ROUTE && tile == 0) places.offsets[tid] = start;
    }
    __syncthreads();
    for (uint32_t r = 0; r < rounds; ++r) {
        const size_t i = ((size_t) tile * rounds + r) * SORT_THREADS + tid;
        if (i >= n) return;
        const uint32_t key = source(i);
        places.put<ROUTE>(i, key, source.limit, base[(key >> shift) & mask] + ranks[i]);
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
    uint32_t bins, rounds, n_tiles;
    size_t at_ranks, at_counts, at_totals, at_keys[2], at_index[2], bytes;

    SortPlan(const size_t n_, const size_t limit_, const bool route) : n(n_), limit((uint32_t) limit_) {
        const int bits = bits_for((uint64_t) limit + 1);
        passes = (bits + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
        bits_per_pass = (bits + passes - 1) / passes;
        bins = passes == 1 ? limit + 1 : 1u << bits_per_pass;
        // short tiles spread few keys over many compute units; more than 32 tiles bring nothing
        rounds = 1;
        while (rounds < MAX_ROUNDS && (size_t) SORT_THREADS * rounds * 32 < n) rounds *= 2;
        const bool only = route && passes == 1 && n <= (size_t) SORT_THREADS * MAX_ROUNDS;
        if (only)
            while ((size_t) SORT_THREADS * rounds < n) rounds *= 2;
        const uint32_t tile = SORT_THREADS * rounds;
        n_tiles = (uint32_t) ((n + tile - 1) / tile);
        size_t at = 0;
        const auto take = [&](const size_t bytes) {
            const size_t here = at;
            at += aligned(bytes);
            return here;
        };
        at_ranks = at_counts = at_totals = 0;
        if (!only) {
            at_ranks = take(n * 2);
            at_counts = take((size_t) bins * n_tiles * 4);
            at_totals = take((size_t) bins * 4);
        }
        const bool moves = passes > 1 || !route;
        for (int b = 0; b < 2; ++b) {
            at_keys[b] = moves && (b == 0 || passes > 1) ? take(n * 4) : 0;
            at_index[b] = moves && (b == 0 || passes > 1) ? take(n * 4) : 0;
        }
        bytes = at;
    }
    int last() const { return (passes - 1) & 1; }  // which pair of arrays holds the result
};

// Queues the passes of a sort; `route`: the single pass writes these instead of sorted keys.
int launch_sort(skm_ctx* ctx, const SortPlan& p, const KeySource& first, char* scratch, const Places* route) {
    uint16_t* ranks = (uint16_t*) (scratch + p.at_ranks);
    uint32_t* counts = (uint32_t*) (scratch + p.at_counts);
    uint32_t* totals = (uint32_t*) (scratch + p.at_totals);
    KeySource source = first;
    Places to{};
    const size_t lds = (size_t) SORT_WAVES * p.bins * sizeof(uint16_t);
    const int bits = bits_for(p.bins);
    const bool scanned = p.n_tiles > TILES_WITHOUT_SCAN;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.bits_per_pass;
        const uint32_t mask = p.passes == 1 ? 0xffffffffu : p.bins - 1;
        if (route) {
            to = *route;
        } else {
            to.index_in = to.index;
            to.keys = (uint32_t*) (scratch + p.at_keys[pass & 1]);
            to.index = (uint32_t*) (scratch + p.at_index[pass & 1]);
        }
        const bool only = route && p.n_tiles == 1 && p.at_totals == 0;
        const auto rank = [&](auto rounds) {
            constexpr int R = decltype(rounds)::value;
            if (only) tile_ranks_kernel<R, true><<<1, SORT_THREADS, lds, ctx->stream>>>(source, p.n, shift, mask, bits, p.bins, ranks, counts, to);
            else tile_ranks_kernel<R, false><<<p.n_tiles, SORT_THREADS, lds, ctx->stream>>>(source, p.n, shift, mask, bits, p.bins, ranks, counts, to);
            return check_hip(hipGetLastError(), "tile_ranks_kernel launch");
        };
        SKM_TRY(p.rounds == 1 ? rank(std::integral_constant<int, 1>{}) : p.rounds == 2 ? rank(std::integral_constant<int, 2>{})
                : p.rounds == 4 ? rank(std::integral_constant<int, 4>{}) : rank(std::integral_constant<int, 8>{}));
        if (only) return SKM_OK;
        if (scanned) {
            tile_counts_scan_kernel<<<p.bins, 64, 0, ctx->stream>>>(counts, p.bins, p.n_tiles, totals);
            SKM_TRY(check_hip(hipGetLastError(), "tile_counts_scan_kernel launch"));
        }
        const auto place = [&](auto kernel) {
            kernel<<<p.n_tiles, SORT_THREADS, 0, ctx->stream>>>(source, p.n, shift, mask, p.bins, p.rounds, p.n_tiles, ranks, counts, totals, to);
            return check_hip(hipGetLastError(), "place_kernel launch");
        };
        if (route) SKM_TRY(scanned ? place(place_kernel<true, true>) : place(place_kernel<true, false>));
        else SKM_TRY(scanned ? place(place_kernel<false, true>) : place(place_kernel<false, false>));
        source = KeySource{to.keys, SKM_U32, p.limit};
    }
    return SKM_OK;
}

// ---------------------------------------------------------------------------------------------
// Gradient of a lookup
// ---------------------------------------------------------------------------------------------

template <class O, int E>
__device__ __forceinline__ void put_sum(O* to, const vec_of<float, E> sum, const float scale, const bool accumulate) {
    vec_of<float, E> r = sum * scale;
    if (accumulate) r += widen<E>(load_vec<O, E>(to));
    store_vec_once<O, E>(to, narrow<O, E>(r));
}

struct GradArgs {
    const void* grad;
    size_t grad_stride;
    void* out;
    size_t out_stride;
    float scale;
    bool accumulate;
    uint32_t n, rows, d, vectors, last, pieces;  // vectors per row, the last one's column; pieces of 64 vectors
    // sorted tokens: their keys and positions, in chunks of `chunk`, and the chunks' sums of rows that go past them
    const uint32_t *keys, *index;
    uint32_t chunk, chunks;
    float* parts;
};

// The sorted tokens are cut into chunks, so that however the ids are spread every wavefront adds up the same number of tokens,
// GRAD_AHEAD of them on their way before the first is added.  A row whose tokens are all in a chunk is stored; of the
// rows that began before the chunk or go on after it, at most two, the sum of this chunk's tokens goes to `parts`: slot 0 if
// the row holds the chunk's first token, else slot 1.  Rows of few vectors share a wavefront: `lanes` lanes to a chunk.
constexpr int GRAD_AHEAD = 8, GRAD_VECTORS = 2;  // vectors a lane holds of a row

template <class T, class O, int E>
__device__ __forceinline__ void grad_of_chunk(const GradArgs& g, const RowSplit& s, const uint64_t unit) {
    const T* grad = reinterpret_cast<const T*>(g.grad);
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t c = unit / s.pieces * (64 / s.lanes) + lane / s.lanes;
    if (c >= g.chunks) return;
    const uint32_t first = (uint32_t) (unit % s.pieces) * s.lanes * GRAD_VECTORS + (lane & (s.lanes - 1));
    const uint32_t from = (uint32_t) c * g.chunk, to = (uint32_t) min((uint64_t) g.n, (uint64_t) from + g.chunk);
    uint32_t row = g.keys[from];
    if (row >= g.rows) return;  // nobody's tokens are at the end
    const bool goes_on = to < g.n && g.keys[to] == g.keys[to - 1];
    bool whole = from == 0 || g.keys[from - 1] != row;  // the row began in this chunk
    int slot = 0;
    vec_of<float, E> sum[GRAD_VECTORS] = {};
    const auto put = [&](const bool ends) {
#pragma unroll
        for (int i = 0; i < GRAD_VECTORS; ++i) {
            const uint32_t at = first + i * s.lanes;
            if (at < g.vectors) {
                if (whole && ends) put_sum<O, E>(reinterpret_cast<O*>(g.out) + (size_t) row * g.out_stride + column<E>(at, g.last), sum[i], g.scale, g.accumulate);
                else store_vec<float, E>(g.parts + ((size_t) c * 2 + slot) * g.d + column<E>(at, g.last), sum[i]);
            }
            sum[i] = vec_of<float, E>{};
        }
        whole = true;
        slot = 1;
    };
    for (uint32_t j = from; j < to; j += GRAD_AHEAD) {
        vec_of<T, E> v[GRAD_AHEAD][GRAD_VECTORS];
        uint32_t key[GRAD_AHEAD], token[GRAD_AHEAD];
#pragma unroll
        for (int q = 0; q < GRAD_AHEAD; ++q) {
            key[q] = g.keys[min(j + q, to - 1)];
            token[q] = g.index[min(j + q, to - 1)];
        }
#pragma unroll
        for (int q = 0; q < GRAD_AHEAD; ++q)
#pragma unroll
            for (int i = 0; i < GRAD_VECTORS; ++i)  // past the row's end its last vector, which is not used: no conditions on loads
                v[q][i] = load_vec<T, E>(grad + (size_t) token[q] * g.grad_stride + column<E>(min(first + i * s.lanes, g.vectors - 1), g.last));
#pragma unroll
        for (int q = 0; q < GRAD_AHEAD; ++q) {
            if (j + q >= to) break;
            if (key[q] != row) {
                put(true);
                row = key[q];
                if (row >= g.rows) return;
            }
#pragma unroll
            for (int i = 0; i < GRAD_VECTORS; ++i) sum[i] += widen<E>(v[q][i]);
        }
    }
    put(!goes_on);
}

// Zeros for the rows without a token: a lane each finds whether its row has one (a binary search in the sorted keys), then the
// wavefront stores the rows that have none one after the other.
constexpr uint32_t FILL_ROWS = 16;

template <class O, int E>
__device__ __forceinline__ void fill_rows(const GradArgs& g, const uint32_t unit) {
    const uint32_t lane = threadIdx.x & 63, row = unit * FILL_ROWS + lane;
    bool empty = false;
    if (lane < FILL_ROWS && row < g.rows) {
        uint32_t low = 0, high = g.n;
        while (low < high) {
            const uint32_t mid = low + (high - low) / 2;
            if (g.keys[mid] < row) low = mid + 1;
            else high = mid;
        }
        empty = low == g.n || g.keys[low] != row;
    }
    for (unsigned long long left = __ballot(empty); left; left &= left - 1) {
        O* out = reinterpret_cast<O*>(g.out) + (size_t) (unit * FILL_ROWS + (uint32_t) __builtin_ctzll(left)) * g.out_stride;
        for (uint32_t at = lane; at < g.vectors; at += 64) store_vec_once<O, E>(out + column<E>(at, g.last), vec_of<O, E>{});
    }
}

// One launch for both: the chunks, whose wavefronts wait for memory, under the fill.  Bound by memory: 65,536 tokens of 1,536
// 16-bit elements into 65,536 rows of fp32, 0.6 GB, in 119 us, 5.1 TB/s.
template <class T, class O, int E>
__global__ __launch_bounds__(ROWS_THREADS) void lookup_grad_kernel(const GradArgs g, const RowSplit s, const uint32_t chunk_blocks, const uint32_t first_block) {
    const uint32_t wave = threadIdx.x >> 6, block = first_block + blockIdx.x;
    if (block < chunk_blocks) {
        const uint64_t unit = (uint64_t) block * (ROWS_THREADS / 64) + wave;
        if (unit < s.units) grad_of_chunk<T, O, E>(g, s, unit);
    } else {
        const uint64_t unit = (uint64_t) (block - chunk_blocks) * (ROWS_THREADS / 64) + wave;
        if (unit * FILL_ROWS < g.rows) fill_rows<O, E>(g, (uint32_t) unit);
    }
}

// The row that begins in chunk c and goes on after it, and how many chunks have a sum of it (0: there is none).  All lanes
// of a wavefront ask for the same chunk.
struct Crossing {
    uint32_t row, parts;
    bool at_start;  // it begins with the chunk: the sum is in slot 0, else in slot 1
};
__device__ __forceinline__ Crossing crossing_row(const GradArgs& g, const uint32_t c) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t from = (uint64_t) c * g.chunk, to = from + g.chunk;
    Crossing x{0, 0, false};
    if (to >= g.n) return x;
    const uint32_t before = g.keys[from > 0 ? from - 1 : 0], head = g.keys[from], tail = g.keys[to - 1], next = g.keys[to];
    x.row = tail;
    x.at_start = head == tail;
    if (tail >= g.rows || next != tail || (x.at_start && from > 0 && before == tail)) return x;
    x.parts = 1;
    for (uint32_t d0 = c + 1;; d0 += 64) {  // the following chunks whose first token is the row's
        const uint64_t first = (uint64_t) (d0 + lane) * g.chunk;
        const unsigned long long other = ~__ballot(first < g.n && g.keys[first < g.n ? first : 0] == x.row);
        x.parts += other ? (uint32_t) __builtin_ctzll(other) : 64;
        if (other) return x;
    }
}

// Adds up the chunks' sums of the rows that go past a chunk.  A row of at most JOIN_ALONE sums takes one wavefront (the first
// `alone_blocks` workgroups), a longer one a workgroup, whose wavefronts take contiguous shares, added in order: such rows
// begin at least JOIN_ALONE chunks apart, so a workgroup looks for the one of JOIN_ALONE chunks.
constexpr uint32_t JOIN_ALONE = 16;
constexpr int JOIN_THREADS = 512;

template <class O, int E>
__global__ __launch_bounds__(JOIN_THREADS) void lookup_grad_join_kernel(const GradArgs g, const uint32_t alone_blocks, const uint32_t first_block) {
    constexpr int WAVES = JOIN_THREADS / 64;
    __shared__ vec_of<float, E> share[WAVES][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, block = first_block + blockIdx.x;
    const size_t stride = (size_t) 2 * g.d;
    uint32_t c, piece;
    Crossing x;
    const bool alone = block < alone_blocks;
    if (alone) {
        const uint64_t unit = (uint64_t) block * WAVES + wave;
        if (unit >= (uint64_t) g.chunks * g.pieces) return;
        c = (uint32_t) (unit / g.pieces), piece = (uint32_t) (unit % g.pieces);
        x = crossing_row(g, c);
        if (x.parts == 0 || x.parts > JOIN_ALONE) return;
    } else {
        const uint32_t unit = block - alone_blocks, c0 = unit / g.pieces * JOIN_ALONE;
        piece = unit % g.pieces;
        // lane i < JOIN_ALONE: does a row begin in chunk c0 + i that holds the first token of the JOIN_ALONE chunks after it
        const uint64_t from = (uint64_t) (c0 + lane) * g.chunk, far = from + (uint64_t) JOIN_ALONE * g.chunk;
        bool here = lane < JOIN_ALONE && far < g.n;
        if (here) {
            const uint32_t row = g.keys[far];
            here = row < g.rows && g.keys[from + g.chunk - 1] == row && !(from > 0 && g.keys[from - 1] == row && g.keys[from] == row);
        }
        const unsigned long long which = __ballot(here);
        if (!which) return;
        c = c0 + (uint32_t) __builtin_ctzll(which);
        x = crossing_row(g, c);
    }
    const uint32_t at = piece * 64 + lane;
    const uint32_t each = alone ? x.parts : (x.parts + WAVES - 1) / WAVES;
    const uint32_t p0 = alone ? 0 : min(wave * each, x.parts), p1 = min(p0 + each, x.parts);
    vec_of<float, E> sum = {};
    if (at < g.vectors) {
        const float* part = g.parts + c * stride + column<E>(at, g.last);
#pragma unroll 8
        for (uint32_t p = p0; p < p1; ++p) sum += load_vec<float, E>(part + p * stride + (p == 0 && !x.at_start ? stride / 2 : 0));
    }
    if (!alone) {
        share[wave][lane] = sum;
        __syncthreads();
        for (int w = 1; w < WAVES && wave == 0; ++w) sum += share[w][lane];
    }
    if ((alone || wave == 0) && at < g.vectors)
        put_sum<O, E>(reinterpret_cast<O*>(g.out) + (size_t) x.row * g.out_stride + column<E>(at, g.last), sum, g.scale, g.accumulate);
}

// Few tokens: one launch and no sort, 8 us for 1,021 tokens of 3 KiB into 4,096 rows (the sorted path takes six launches).  A
// workgroup owns a piece of every `step`-th row, reads all ids, and lists the tokens of its rows in order
// (every wavefront those of a contiguous share).  Then its wavefronts take the rows one by one, and together those of
// many tokens, each wavefront the tokens of its share.
constexpr size_t FEW_TOKENS = 2048;
constexpr int FEW_THREADS = 512, FEW_AHEAD = 4;
constexpr uint32_t FEW_ROWS = 64;  // of a workgroup, at most
constexpr uint32_t FEW_MOST = 8;   // tokens of a row that one wavefront adds up
// A row's tokens are a chain here: with many on every row the sort is faster (2,048 tokens on one row: 71 us here, 16 sorted).
inline bool few_tokens(const size_t n, const size_t rows) { return n <= FEW_TOKENS && (n <= 256 || n <= 32 * rows); }
template <int E>
constexpr int FEW_VECTORS = E >= 8 ? 2 : 4;  // vectors a lane holds of a row, at most

template <class T, class O, int E, int V>  // V: vectors a lane holds of a row
__global__ __launch_bounds__(FEW_THREADS) void lookup_grad_few_kernel(const GradArgs g, const KeySource source, const uint32_t step, const uint32_t first_block) {
    constexpr int WAVES = FEW_THREADS / 64, SHARE = FEW_TOKENS / WAVES;
    __shared__ uint32_t listed[WAVES][SHARE];  // number of the row, token
    __shared__ uint32_t many[WAVES], of_row[FEW_ROWS];
    __shared__ vec_of<float, E> share[WAVES][V][64];
    const T* grad = reinterpret_cast<const T*>(g.grad);
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t block = first_block + blockIdx.x, mine = (g.rows - 1 - block) / step + 1;  // rows block, + step, ...
    if (threadIdx.x < FEW_ROWS) of_row[threadIdx.x] = 0;
    uint32_t id[SHARE / 64];
#pragma unroll
    for (int q = 0; q < SHARE / 64; ++q) {
        const uint32_t t = wave * SHARE + q * 64 + lane;
        id[q] = t < g.n ? source(t) : source.limit;
    }
    __syncthreads();
    uint32_t count = 0;
#pragma unroll
    for (int q = 0; q < SHARE / 64; ++q) {
        const uint32_t r = id[q] / step;
        const bool here = id[q] < source.limit && id[q] - r * step == block;
        const unsigned long long who = __ballot(here);
        if (here) {
            listed[wave][count + (uint32_t) __popcll(who & lanes_below(lane))] = r << 16 | (wave * SHARE + q * 64 + lane);
            atomicAdd(&of_row[r], 1u);
        }
        count += (uint32_t) __popcll(who);
    }
    if (lane == 0) many[wave] = count;
    __syncthreads();
    // adds the tokens of row r in the w-th share; `at`: the lane's first vector, the others 64 apart
    const auto add_share = [&](const uint32_t w, const uint32_t r, const uint32_t at, vec_of<float, E> (&sum)[V]) {
        for (uint32_t k0 = 0; k0 < many[w]; k0 += 64) {
            const uint32_t entry = k0 + lane < many[w] ? listed[w][k0 + lane] : 0xffffffffu;
            unsigned long long same = __ballot(entry >> 16 == r);
            while (same) {
                // past the row's end its last vector, which is not used: conditions of lanes would keep the loads from being
                // on their way together
                vec_of<T, E> v[FEW_AHEAD][V];
                const int taken = min(__popcll(same), FEW_AHEAD);
#pragma unroll
                for (int q = 0; q < FEW_AHEAD; ++q)
                    if (q < taken) {
                        const uint32_t t = __builtin_amdgcn_readlane(entry, (uint32_t) __builtin_ctzll(same)) & 0xffffu;
                        same &= same - 1;
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            v[q][i] = load_vec<T, E>(grad + (size_t) t * g.grad_stride + column<E>(min(at + i * 64, g.vectors - 1), g.last));
                    }
#pragma unroll
                for (int q = 0; q < FEW_AHEAD; ++q)
                    if (q < taken)
#pragma unroll
                        for (int i = 0; i < V; ++i) sum[i] += widen<E>(v[q][i]);
            }
        }
    };
    const auto put = [&](const uint32_t r, const uint32_t at, const vec_of<float, E> (&sum)[V], const float scale) {
        O* out = reinterpret_cast<O*>(g.out) + (size_t) (r * step + block) * g.out_stride;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (at + i * 64 < g.vectors) put_sum<O, E>(out + column<E>(at + i * 64, g.last), sum[i], scale, g.accumulate);
    };
    const uint32_t at = blockIdx.y * (64 * V) + lane;  // the workgroup's piece of the rows
    for (uint32_t r = wave; r < mine; r += WAVES) {
        const uint32_t tokens = of_row[r];
        if (tokens > FEW_MOST || (g.accumulate && tokens == 0)) continue;
        vec_of<float, E> sum[V] = {};
        if (tokens)
            for (uint32_t w = 0; w < WAVES; ++w) add_share(w, r, at, sum);
        put(r, at, sum, tokens ? g.scale : 1.0f);  // zeros whatever the scale
    }
    for (uint32_t r = 0; r < mine; ++r) {
        if (of_row[r] <= FEW_MOST) continue;
        vec_of<float, E> sum[V] = {};
        add_share(wave, r, at, sum);
#pragma unroll
        for (int i = 0; i < V; ++i) share[wave][i][lane] = sum[i];
        __syncthreads();
        if (wave == 0) {
            for (int w = 1; w < WAVES; ++w)
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += share[w][i][lane];
            put(r, at, sum, g.scale);
        }
        __syncthreads();
    }
}

// Scratch of the sorted path: the sort and the chunks' sums.
struct GradPlan {
    SortPlan sort;
    uint32_t chunk, chunks;
    size_t at_parts, bytes;
    GradPlan(const size_t n, const size_t rows, const size_t d) : sort(n, rows, false) {
        // The additions of a chunk, and of a row's chunks, are chains: short chunks give more wavefronts and more sums to join
        // (the whole call for 65,536 tokens of text: chunks of 16 160 us, of 32 168), longer ones for more tokens keep the joins
        // short where many are on one row (500,000 tokens on 4 rows: 32 247 us, 64 170, 128 149; a million of text: 32 173, 64
        // 163, 128 185).
        chunk = n <= (size_t(1) << 17) ? 16 : n <= (size_t(1) << 20) ? 64 : 256;
        chunks = (uint32_t) ((n + chunk - 1) / chunk);
        at_parts = sort.bytes;
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
    *out_bytes = places == 0 ? 0 : SortPlan(places, groups, true).bytes;
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
    const Argument from{"the choices", vector_memory(d_choices, places, 4)}, slots{"slots", vector_memory(d_slots, places, 4)};
    const Argument order{"order", vector_memory(d_order, places, 4)}, offsets{"offsets", vector_memory(d_offsets, groups + 1, 4)};
    SKM_TRY(check_apart(__func__, slots, {from, order, offsets}));
    SKM_TRY(check_apart(__func__, order, {from, offsets}));
    SKM_TRY(check_apart(__func__, offsets, {from}));
    SKM_TRY(check_apart(__func__, {"scratch", vector_memory(d_scratch, need, 1)}, {from, slots, order, offsets}));
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/route");
    if (places == 0) return skm_fill_u32(ctx, d_offsets, 0, groups + 1);
    const SortPlan plan(places, groups, true);
    void* scratch = nullptr;
    SKM_TRY(call_scratch(ctx, __func__, d_scratch, scratch_bytes, plan.bytes, &scratch));
    const KeySource source{d_choices, SKM_U32, (uint32_t) groups};
    const Places places_out{nullptr, nullptr, nullptr, d_slots, d_order, d_offsets};
    if (plan.passes == 1) return launch_sort(ctx, plan, source, (char*) scratch, &places_out);
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
    *out_bytes = few_tokens(n, rows) || rows == 0 ? 0 : GradPlan(n, rows, d).bytes;
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
    const Argument grad{"grad", matrix_memory(d_grad, n, grad_stride, d, size)};
    const Argument ids{"the ids", vector_memory(d_ids, n, ids_type == SKM_I64 ? 8 : 4)};
    const Argument out{"out", matrix_memory(d_out, rows, out_stride, d, out_size)};
    SKM_TRY(check_apart(__func__, out, {grad, ids}));
    SKM_TRY(check_apart(__func__, {"scratch", vector_memory(d_scratch, need, 1)}, {grad, ids, out}));
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/lookup_grad");
    // an accumulated vector must not be added twice
    const size_t per_lane = vector_elements(size, out_size, d, accumulate != 0);
    const KeySource source{d_ids, ids_type, (uint32_t) rows};
    const auto run = [&](auto sample, auto out_sample) {
        using T = decltype(sample);
        using O = decltype(out_sample);
        return for_elements<std::conditional_t<(sizeof(O) > sizeof(T)), O, T>>(per_lane, [&](auto elements) {
            constexpr int E = decltype(elements)::value;
            GradArgs g{};
            g.grad = d_grad;
            g.grad_stride = grad_stride;
            g.out = d_out;
            g.out_stride = out_stride;
            g.scale = scale;
            g.accumulate = accumulate != 0;
            g.n = (uint32_t) n;
            g.rows = (uint32_t) rows;
            g.d = (uint32_t) d;
            g.vectors = (uint32_t) ((d + E - 1) / E);
            g.last = (uint32_t) (d - E);
            g.pieces = (g.vectors + 63) / 64;
            if (few_tokens(n, rows)) {
                // a workgroup per row up to 1,024, then a few rows each: reading the ids costs a workgroup about as much as two rows
                const uint32_t step = (uint32_t) std::max<size_t>(std::min<size_t>(rows, 1024), (rows + FEW_ROWS - 1) / FEW_ROWS);
                const auto launch = [&](auto held) {
                    constexpr int V = decltype(held)::value;
                    const uint32_t pieces = (g.vectors + 64 * V - 1) / (64 * V);
                    return launch_in_parts(step, [&](const uint32_t first, const unsigned blocks) {
                        lookup_grad_few_kernel<T, O, E, V><<<dim3(blocks, pieces), FEW_THREADS, 0, ctx->stream>>>(g, source, step, first);
                        return check_hip(hipGetLastError(), "lookup_grad_few_kernel launch");
                    });
                };
                if (g.vectors <= 64) return launch(std::integral_constant<int, 1>{});
                if (g.vectors <= 128) return launch(std::integral_constant<int, 2>{});
                if (FEW_VECTORS<E> > 2 && g.vectors <= 192) return launch(std::integral_constant<int, FEW_VECTORS<E> - 1>{});
                return launch(std::integral_constant<int, FEW_VECTORS<E>>{});
            }
            const GradPlan plan(n, rows, d);
            g.chunk = plan.chunk;
            g.chunks = plan.chunks;
            const RowSplit s = split_rows(plan.chunks, d, E, GRAD_VECTORS);
            constexpr uint64_t PER_BLOCK = ROWS_THREADS / 64;
            const uint64_t chunk_blocks = (s.units + PER_BLOCK - 1) / PER_BLOCK;
            const uint64_t fill_units = accumulate ? 0 : (rows + FILL_ROWS - 1) / FILL_ROWS;
            const uint64_t blocks = chunk_blocks + (fill_units + PER_BLOCK - 1) / PER_BLOCK;
            if (blocks > 0x7fffffffULL || (uint64_t) g.chunks * g.pieces > 0x7fffffffULL)
                return set_error(SKM_ERR_INVALID, "skm_lookup_rows_grad: more than 2^31 workgroups");
            void* at = nullptr;
            SKM_TRY(call_scratch(ctx, "skm_lookup_rows_grad", d_scratch, scratch_bytes, plan.bytes, &at));
            char* scratch = (char*) at;
            SKM_TRY(launch_sort(ctx, plan.sort, source, scratch, nullptr));
            g.keys = (const uint32_t*) (scratch + plan.sort.at_keys[plan.sort.last()]);
            g.index = (const uint32_t*) (scratch + plan.sort.at_index[plan.sort.last()]);
            g.parts = (float*) (scratch + plan.at_parts);
            SKM_TRY(launch_in_parts(blocks, [&](const uint32_t first_block, const unsigned count) {
                lookup_grad_kernel<T, O, E><<<count, ROWS_THREADS, 0, ctx->stream>>>(g, s, (uint32_t) chunk_blocks, first_block);
                return check_hip(hipGetLastError(), "lookup_grad_kernel launch");
            }));
            constexpr uint64_t JOINS = JOIN_THREADS / 64;
            const uint32_t alone_blocks = (uint32_t) (((uint64_t) g.chunks * g.pieces + JOINS - 1) / JOINS);
            const uint32_t long_blocks = (g.chunks + JOIN_ALONE - 1) / JOIN_ALONE * g.pieces;
            return launch_in_parts((uint64_t) alone_blocks + long_blocks, [&](const uint32_t first_block, const unsigned count) {
                lookup_grad_join_kernel<O, E><<<count, JOIN_THREADS, 0, ctx->stream>>>(g, alone_blocks, first_block);
                return check_hip(hipGetLastError(), "lookup_grad_join_kernel launch");
            });
        });
    };
    return for_type(type, [&](auto sample) {
        if (out_type == type) return run(sample, sample);
        return run(sample, float{});
    });
}

} // extern "C"
