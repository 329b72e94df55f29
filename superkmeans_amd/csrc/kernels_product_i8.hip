// Rows quantised to 8 bits with one scale each, and products of such rows: over one matrix of weights, or over a matrix per
// group of consecutive rows.
//
//   scale[t] = max|x[t]| / 127,  q[t][k] = rint(127 x[t][k] / max|x[t]|)
//   out[m][n] = (sum_k a[m][k] b[n][k]) * a_scale[m] * b_scale[n] + bias[n]
//
// The sum is exact: 8-bit products in 32-bit integers, which hold SKM_PRODUCT_MAX_K of them.
#include "rows_common.h"

namespace skm {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------------------------
// Quantisation
// ---------------------------------------------------------------------------------------------

// The whole numbers nearest to 127 x / most, ties to even, as bytes.  The fp32 product of x and the rounded 127 / most is at most
// 127 * (2^-23 + 2^-48) < 1.52e-5 off, so that the choice between two numbers can only be wrong that near to the border between
// them; there the quotient is taken in fp64, where 127 x is exact and a quotient of two fp32 numbers cannot round onto a border.
// Adding 1.5 * 2^23 rounds an fp32 number of that size to a whole one, whose last byte is the step.
template <int E>
__device__ __forceinline__ vec_of<int8_t, E> nearest_steps(const vec_of<float, E> x, const float most, const float inverse) {
    uint32_t step[E];
    bool border = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float t = x[e] * inverse, shifted = t + 12582912.0f;
        border |= !(fabsf(t - (shifted - 12582912.0f)) < 0.49998f);
        step[e] = __float_as_uint(shifted);
    }
    if (border)
#pragma unroll
        for (int e = 0; e < E; ++e) step[e] = (uint32_t) (int) rint((double) x[e] * 127.0 / (double) most);
    if constexpr (E % 4 == 0) {
        vec_of<uint32_t, E / 4> words;
#pragma unroll
        for (int w = 0; w < E / 4; ++w) {
            const uint32_t low = __builtin_amdgcn_perm(step[4 * w + 1], step[4 * w], 0x0c0c0400u);
            const uint32_t high = __builtin_amdgcn_perm(step[4 * w + 3], step[4 * w + 2], 0x0c0c0400u);
            words[w] = __builtin_amdgcn_perm(high, low, 0x05040100u);
        }
        return __builtin_bit_cast(vec_of<int8_t, E>, words);
    } else {
        vec_of<int8_t, E> r;
#pragma unroll
        for (int e = 0; e < E; ++e) r[e] = (int8_t) step[e];
        return r;
    }
}

// Largest magnitudes, element by element, as the numbers' bits without the sign: ordered like the numbers, infinities and NaN
// above all.
template <class T, int E>
using bits_of = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t> __attribute__((ext_vector_type(E)));

// WAVES wavefronts to a row.  A row of up to 64 WAVES HELD vectors is read once and held in registers; of a longer one what is
// past that is read twice.  Bound by memory for 32-bit rows (4,096 of 8,192 elements 29 us, 5.8 TB/s), by memory and the dozen
// instructions per element about equally for 16-bit ones (8,192 of 4,096 24 us, 4.2 TB/s).
constexpr int QUANTIZE_THREADS = 256;

template <class T, int E, int WAVES, int HELD>
__global__ __launch_bounds__(QUANTIZE_THREADS) void quantize_rows_kernel(
    const T* __restrict__ x, const size_t n, const uint32_t vectors, const uint32_t last, const size_t x_stride, int8_t* __restrict__ q,
    const size_t q_stride, float* __restrict__ scales
) {
    constexpr int ROWS = QUANTIZE_THREADS / 64 / WAVES, LANES = 64 * WAVES;  // ROWS per workgroup
    __shared__ uint32_t wave_most[QUANTIZE_THREADS / 64];
    const uint32_t in_row = threadIdx.x % LANES;
    const size_t turns = (n + ROWS - 1) / ROWS;  // the same for every thread, which all meet at the barriers
    for (size_t turn = blockIdx.x; turn < turns; turn += gridDim.x) {
        const size_t t = turn * ROWS + threadIdx.x / LANES;
        const T* row = x + t * x_stride;
        const uint32_t mine = t < n ? vectors : 0;
        bits_of<T, E> largest = 0;
        const auto look = [&](const vec_of<T, E> v) {
            largest = __builtin_elementwise_max(largest, __builtin_bit_cast(bits_of<T, E>, v) & (bits_of<T, E>) (sizeof(T) == 2 ? 0x7fff : 0x7fffffff));
        };
        vec_of<T, E> held[HELD];
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (in_row + i * LANES < mine) held[i] = load_vec<T, E>(row + column<E>(in_row + i * LANES, last));
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (in_row + i * LANES < mine) look(held[i]);
        for (uint32_t at = in_row + HELD * LANES; at < mine; at += LANES) look(load_vec<T, E>(row + column<E>(at, last)));
        auto one = largest[0];
#pragma unroll
        for (int e = 1; e < E; ++e) one = one > largest[e] ? one : largest[e];
        uint32_t most = __float_as_uint((float) __builtin_bit_cast(T, one));
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) most = max(most, (uint32_t) __shfl_xor(most, off));
        if (WAVES > 1) {
            __syncthreads();  // the row before has been looked at
            if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = most;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) most = max(most, wave_most[threadIdx.x / LANES * WAVES + w]);
        }
        const bool usable = most != 0 && most < 0x7f800000u;
        const float m = __uint_as_float(most);
        const float inverse = m > 1e-30f ? 127.0f / m : __builtin_nanf("");  // NaN sends every element through fp64
        if (in_row == 0 && t < n) scales[t] = most < 0x7f800000u ? m / 127.0f : __builtin_nanf("");
        const auto put = [&](const uint32_t at, const vec_of<T, E> v) {
            const vec_of<int8_t, E> r = usable ? nearest_steps<E>(widen<E>(v), m, inverse) : vec_of<int8_t, E>{};
            store_vec<int8_t, E>(q + t * q_stride + column<E>(at, last), r);
        };
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (in_row + i * LANES < mine) put(in_row + i * LANES, held[i]);
        for (uint32_t at = in_row + HELD * LANES; at < mine; at += LANES) put(at, load_vec<T, E>(row + column<E>(at, last)));
    }
}

// ---------------------------------------------------------------------------------------------
// Product
// ---------------------------------------------------------------------------------------------

struct ProductArgs {
    const int8_t* a;
    const float* a_scale;
    const int8_t* b;
    const float* b_scale;
    const float* bias;
    const uint32_t* offsets;  // null: one group of all rows
    void* out;
    size_t a_stride, b_stride, b_group_stride, out_stride;
    uint32_t m, n, k, groups;
};

// Rows [first, end) of one group.
struct RowTile {
    uint32_t group, first, end;
};

// The tile of `tm` rows with the given number; first >= end where there is none.  Group g has the numbers from
// offsets[g] / tm + g on: as many as its rows can need, whatever the other groups hold, so that the group of a number is found by
// a search and the numbers of all groups end at m / tm + groups.  Every wavefront of a workgroup looks by itself, at 64 groups
// at a time.  Offsets are clamped to the rows there are.
__device__ __forceinline__ RowTile find_rows(const ProductArgs& p, const uint32_t tm, const uint32_t number) {
    if (!p.offsets) {
        const uint32_t first = number * tm;
        return {0, min(first, p.m), min(p.m, first + tm)};
    }
    const uint32_t lane = threadIdx.x & 63;
    uint32_t low = 0, many = p.groups;  // the group is one of `many` from `low` on
    for (;;) {
        const uint32_t step = (many + 63) / 64, g = low + lane * step;
        const bool begun = lane * step < many && min(p.offsets[g], p.m) / tm + g <= number;
        const unsigned long long before = __ballot(begun);
        if (!before) return {0, 0, 0};
        const uint32_t at = 63 - (uint32_t) __builtin_clzll(before);
        low += at * step;
        many = min(step, many - at * step);
        if (step == 1) break;
    }
    const uint32_t from = min(p.offsets[low], p.m), to = min(p.offsets[low + 1], p.m);
    const uint64_t first = (uint64_t) from + (uint64_t) (number - from / tm - low) * tm;
    if (first >= to) return {0, 0, 0};
    return {low, (uint32_t) first, (uint32_t) min((uint64_t) to, first + tm)};
}

// 16 bytes of a row, at any address: the load instruction takes them unaligned too, only the compiler has to be told.
__device__ __forceinline__ intx4 load16(const int8_t* p) {
    intx4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
// The 16 bytes from column k on of a row of `columns` >= 16, zeros past its end: where fewer are left, the last 16 of the row,
// shifted.
__device__ __forceinline__ intx4 load16_end(const int8_t* row, const int k, const int columns) {
    const int left = columns - k;
    const int8_t* from = row + (left >= 16 ? k : columns - 16);
    unsigned long long half[2];
    __builtin_memcpy(half, from, 16);
    int drop = left >= 16 ? 0 : 16 - left;  // bytes that are before column k
    if (drop >= 8) {
        half[0] = half[1];
        half[1] = 0;
        drop -= 8;
    }
    drop = min(drop, 7);
    half[0] = half[0] >> (8 * drop) | (half[1] << 1) << (63 - 8 * drop);
    half[1] >>= 8 * drop;
    if (left <= 0) half[0] = half[1] = 0;
    intx4 v;
    __builtin_memcpy(&v, half, 16);
    return v;
}
// The same for a row of any length.
__device__ __forceinline__ intx4 load16_short(const int8_t* row, const int k, const int columns) {
    unsigned long long half[2] = {0, 0};
#pragma unroll 1
    for (int i = 0; i < 16 && k + i < columns; ++i) half[i >> 3] |= (unsigned long long) (uint8_t) row[k + i] << (8 * (i & 7));
    intx4 v;
    __builtin_memcpy(&v, half, 16);
    return v;
}

// ---- few rows: the weights go from memory to the registers, once ----
//
// A workgroup owns 16 RT rows and 16 NB columns of the result; its wavefronts share the columns of the operands, and
// their 32-bit sums are added through LDS (exact, so the split does not show).  With a row or a few per matrix every
// byte of the weights is read once and used at once, so nothing is gained by LDS; what counts is how many bytes are on their
// way: each wavefront requests AHEAD steps of 64 columns before it uses the first.  Bound by memory: 64 matrices of 2,048 x 1,024
// on 512 rows take 30 us, 4.6 TB/s; one row through 4,096 x 4,096 5.7 us, 3 TB/s, where the launch and one latency are most of it.
template <class O, int RT, int NB, int WAVES, int AHEAD>
__global__ __launch_bounds__(WAVES * 64) void product_few_rows_kernel(const ProductArgs p, const uint32_t tiles_n, const uint32_t first_block) {
    constexpr int TM = 16 * RT, TN = 16 * NB;
    __shared__ int part[WAVES][TM][TN + 4];
    const uint32_t block = first_block + blockIdx.x;
    const RowTile rows = find_rows(p, TM, block / tiles_n);
    if (rows.first >= rows.end) return;
    const uint32_t n0 = block % tiles_n * TN;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // lane l holds row l % 16 of a block and 16 columns from 16 (l / 16) on
    const int8_t *a[RT], *b[NB];
#pragma unroll
    for (int i = 0; i < RT; ++i) a[i] = p.a + (size_t) min(rows.first + i * 16 + (lane & 15), rows.end - 1) * p.a_stride + (lane >> 4) * 16;
#pragma unroll
    for (int j = 0; j < NB; ++j)
        b[j] = p.b + rows.group * p.b_group_stride + (size_t) min(n0 + j * 16 + (lane & 15), p.n - 1) * p.b_stride + (lane >> 4) * 16;
    intx4 acc[NB][RT] = {};
    const uint32_t steps = (p.k + 63) / 64, each = (steps + WAVES - 1) / WAVES;
    const uint32_t from = min(wave * each, steps), to = min(from + each, steps), full = min(to, p.k / 64);
    const auto multiply = [&](const intx4 (&x)[RT], const intx4 (&w)[NB]) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], x[i], acc[j][i], 0, 0, 0);
    };
    uint32_t s = from;
    intx4 x[AHEAD][RT], w[AHEAD][NB];
    const auto request = [&](const int q, const uint32_t step) {
#pragma unroll
        for (int j = 0; j < NB; ++j) w[q][j] = load16(b[j] + (size_t) step * 64);
#pragma unroll
        for (int i = 0; i < RT; ++i) x[q][i] = load16(a[i] + (size_t) step * 64);
    };
#pragma unroll
    for (int q = 0; q < AHEAD; ++q)
        if (s + q < full) request(q, s + q);
    for (; s + 2 * AHEAD <= full; s += AHEAD)
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            multiply(x[q], w[q]);
            request(q, s + AHEAD + q);
        }
    // up to 2 AHEAD - 1 steps are left, the first AHEAD of them requested
#pragma unroll
    for (int q = 0; q < AHEAD; ++q)
        if (s + q < full) {
            multiply(x[q], w[q]);
            if (s + AHEAD + q < full) request(q, s + AHEAD + q);
        }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q)
        if (s + AHEAD + q < full) multiply(x[q], w[q]);
    if (from < to && full < to) {  // the columns' end
        const int skip = (lane >> 4) * 16, k = (int) (full * 64) + skip;
        if (p.k >= 16) {
#pragma unroll
            for (int j = 0; j < NB; ++j) w[0][j] = load16_end(b[j] - skip, k, (int) p.k);
#pragma unroll
            for (int i = 0; i < RT; ++i) x[0][i] = load16_end(a[i] - skip, k, (int) p.k);
        } else {
#pragma unroll
            for (int j = 0; j < NB; ++j) w[0][j] = load16_short(b[j] - skip, k, (int) p.k);
#pragma unroll
            for (int i = 0; i < RT; ++i) x[0][i] = load16_short(a[i] - skip, k, (int) p.k);
        }
        multiply(x[0], w[0]);
    }
    // block (j, i): lane l holds the columns 4 (l / 16) .. + 3 of the result's row l % 16
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < RT; ++i)
            *reinterpret_cast<intx4*>(&part[wave][i * 16 + (lane & 15)][j * 16 + (lane >> 4) * 4]) = acc[j][i];
    __syncthreads();
    const float* b_scale = p.b_scale + (size_t) rows.group * p.n;
    const float* bias = p.bias ? p.bias + (size_t) rows.group * p.n : nullptr;
    for (uint32_t e = threadIdx.x; e < TM * TN; e += WAVES * 64) {
        const uint32_t r = e / TN, c = e % TN, m = rows.first + r, n = n0 + c;
        if (m >= rows.end || n >= p.n) continue;
        int sum = 0;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) sum += part[v][r][c];
        const float value = (float) sum * p.a_scale[m] * b_scale[n] + (bias ? bias[n] : 0.0f);
        reinterpret_cast<O*>(p.out)[(size_t) m * p.out_stride + n] = (O) value;
    }
}

// ---- many rows: tiles through LDS ----
//
// 2 x WN wavefronts, each FM x FN blocks of 32 x 32, so a tile is 64 FM x 32 WN FN.  A stage is 128 columns (a cache line) of
// both operands; two stages are in LDS and a third is on its way in registers.
// The largest tile is 256 x 256 by eight wavefronts of 128 x 64.  Four of 128 x 128 read a third less LDS and hold 512 registers,
// one wavefront to a SIMD: whatever it waits for, the matrix unit waits for too (8,192 x 8,192 x 4,096: 263 us against 253, and
// 230 against 191 on zeros, where power does not limit the clock).  Two per SIMD fill each other's waits.
// What bounds it: 253 us are 2.17 PFLOP/s of 8-bit operations, 43 % of the matrix units' peak at 2.4 GHz.  By the counters the
// units are busy in 55 % of the cycles, and there are 1.9 GHz of them: the clock falls with the bits that change in the
// operands.  Memory is not it (0.4 GB past the L2; with every stage reading the same columns 3 % less time).
// Chunks of 16 bytes are stored at position chunk ^ (row / 2 % 8) of their row: two rows fill the banks once, so the 16 rows
// that are read at a time have to differ in the pair, not in the row (row % 8 there: 2 % more time).
constexpr int STAGE_K = 128;

template <int FM, int FN, int WN>
constexpr size_t tiles_lds_bytes() {
    return (size_t) 2 * (64 * FM + 32 * WN * FN) * STAGE_K;
}

// Number of a workgroup to tile: workgroups whose number is equal mod 8 run on the same die and share its L2, where 32 of them
// at a time take a block of `super_m` x 32 / super_m neighbouring tiles.  The blocks that do not go round the eight dies (from
// number `even` on) are dealt out tile by tile, so that no die has a block more than another.
struct TileMap {
    uint32_t super_m, super_n, across, tiles_n, even;
    __device__ __forceinline__ bool operator()(const uint32_t number, uint32_t& tile_m, uint32_t& tile_n) const {
        uint32_t super = number >> 5, within = number & 31;
        if (number < even) {
            super = (number >> 8) * 8 + (number & 7);
            within = (number >> 3) & 31;
        }
        tile_m = super / across * super_m + within % super_m;
        tile_n = super % across * super_n + within / super_m;
        return tile_n < tiles_n;
    }
};

template <class O, int FM, int FN, int WN>
__global__ __launch_bounds__(128 * WN, 2) void product_tiles_kernel(const ProductArgs p, const TileMap map, const uint32_t first_block) {
    constexpr int TM = 64 * FM, TN = 32 * WN * FN, ROWS = 16 * WN, NLA = TM / ROWS, NLB = TN / ROWS;  // ROWS of a load by all threads
    constexpr uint32_t STAGE = (TM + TN) * STAGE_K;
    extern __shared__ __align__(16) int8_t lds[];  // [2][TM + TN][STAGE_K]
    uint32_t tile_m, tile_n;
    if (!map(first_block + blockIdx.x, tile_m, tile_n)) return;
    const RowTile rows = find_rows(p, TM, tile_m);
    if (rows.first >= rows.end) return;
    const uint32_t n0 = tile_n * TN;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t wm = wave / WN * FM * 32, wn = wave % WN * FN * 32;

    // memory to registers: a thread takes 16 bytes of every ROWS-th row; rows past the end repeat the last one and are not stored
    const uint32_t ld_row = tid >> 3, ld_chunk = tid & 7;
    const int8_t* a_base = p.a + (size_t) rows.first * p.a_stride;
    const int8_t* b_base = p.b + rows.group * p.b_group_stride + (size_t) n0 * p.b_stride;
    uint32_t a_at[NLA], b_at[NLB];
#pragma unroll
    for (int i = 0; i < NLA; ++i) a_at[i] = min(ld_row + ROWS * i, rows.end - 1 - rows.first) * (uint32_t) p.a_stride + ld_chunk * 16;
#pragma unroll
    for (int i = 0; i < NLB; ++i) b_at[i] = min(ld_row + ROWS * i, p.n - 1 - n0) * (uint32_t) p.b_stride + ld_chunk * 16;
    intx4 ra[NLA], rb[NLB];
    const uint32_t stages = (p.k + STAGE_K - 1) / STAGE_K, full = p.k / STAGE_K;
    const auto request = [&](const uint32_t s) {
        const int8_t *as = a_base + (size_t) s * STAGE_K, *bs = b_base + (size_t) s * STAGE_K;
#pragma unroll
        for (int i = 0; i < NLA; ++i) ra[i] = load16(as + a_at[i]);
#pragma unroll
        for (int i = 0; i < NLB; ++i) rb[i] = load16(bs + b_at[i]);
    };
    const auto request_last = [&](const uint32_t s) {  // a stage that the rows end in
        const int k = (int) (s * STAGE_K + ld_chunk * 16);
#pragma unroll
        for (int i = 0; i < NLA; ++i) ra[i] = load16_end(a_base + (a_at[i] - ld_chunk * 16), k, (int) p.k);
#pragma unroll
        for (int i = 0; i < NLB; ++i) rb[i] = load16_end(b_base + (b_at[i] - ld_chunk * 16), k, (int) p.k);
    };
    const auto request_any = [&](const uint32_t s) {
        if (s < full) request(s);
        else request_last(s);
    };
    const uint32_t st = ld_row * STAGE_K + ((ld_chunk ^ ((ld_row >> 1) & 7)) << 4);
    const auto publish = [&](const uint32_t buffer) {
        int8_t* to = lds + buffer * STAGE + st;
#pragma unroll
        for (int i = 0; i < NLA; ++i) *reinterpret_cast<intx4*>(to + i * ROWS * STAGE_K) = ra[i];
#pragma unroll
        for (int i = 0; i < NLB; ++i) *reinterpret_cast<intx4*>(to + (TM + i * ROWS) * STAGE_K) = rb[i];
    };
    // registers of a block: lane l holds row l % 32 and 16 columns from 16 (l / 32) on
    const uint32_t fr = (lane & 31) * STAGE_K;
    intx4 fa[2][FM], fb[2][FN];
    const auto fetch = [&](const uint32_t buffer, const int slice, const int to) {
        const int8_t* at = lds + buffer * STAGE + fr + (((2 * slice + (lane >> 5)) ^ ((lane >> 1) & 7)) << 4);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[to][j] = *reinterpret_cast<const intx4*>(at + (TM + wn + j * 32) * STAGE_K);
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[to][i] = *reinterpret_cast<const intx4*>(at + (wm + i * 32) * STAGE_K);
    };
    intx16 acc[FM][FN] = {};
    const auto multiply = [&](const int of) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[of][j], fa[of][i], acc[i][j], 0, 0, 0);
    };

    // One stage: while a slice is multiplied the next one is read; the barrier sits before the last slice's products, when every
    // read of the stage has returned, and the next stage's first slice is read under them.
    const auto stage = [&](const uint32_t s, auto hot) {  // hot: stages s + 1 and s + 2 exist and are whole
        constexpr bool HOT = decltype(hot)::value;
        const uint32_t cur = s & 1;
        if (HOT || s + 1 < stages) publish(cur ^ 1);  // its last readers passed the barrier of stage s - 1
        if (HOT) request(s + 2);
        else if (s + 2 < stages) request_any(s + 2);
        fetch(cur, 1, 1);
        multiply(0);
        __builtin_amdgcn_sched_barrier(0);
        fetch(cur, 2, 0);
        multiply(1);
        __builtin_amdgcn_sched_barrier(0);
        fetch(cur, 3, 1);
        multiply(0);
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        if (HOT || s + 1 < stages) fetch(cur ^ 1, 0, 0);
        multiply(1);
        __builtin_amdgcn_sched_barrier(0);
    };
    request_any(0);
    publish(0);
    if (stages > 1) request_any(1);
    __syncthreads();
    fetch(0, 0, 0);
    uint32_t s = 0;
    for (; s + 2 < full; ++s) stage(s, std::true_type{});
#pragma unroll 1
    for (; s < stages; ++s) stage(s, std::false_type{});

    // Results, 32 rows at a time through LDS (each wavefront in a part of its own), so that rows are stored 16 bytes per lane.
    // Element r of block (i, j): row l % 32, column 8 (r / 4) + 4 (l / 32) + r % 4.
    constexpr int E = 16 / sizeof(O), COLUMNS = FN * 32, LD = COLUMNS + E;
    static_assert((size_t) 2 * WN * 32 * LD * sizeof(O) + 2 * TN * sizeof(float) <= (size_t) 2 * STAGE, "results go through the stages' LDS");
    __syncthreads();
    O* staged = reinterpret_cast<O*>(lds) + wave * 32 * LD;
    float* b_scale = reinterpret_cast<float*>(lds + (size_t) 2 * WN * 32 * LD * sizeof(O));
    float* bias = b_scale + TN;
    if (tid < TN) {
        const size_t n = (size_t) rows.group * p.n + min(n0 + tid, p.n - 1);
        b_scale[tid] = p.b_scale[n];
        bias[tid] = p.bias ? p.bias[n] : 0.0f;
    }
    __syncthreads();
    O* out = reinterpret_cast<O*>(p.out);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const uint32_t m0 = rows.first + wm + i * 32;
        const float a_scale = p.a_scale[min(m0 + (lane & 31), rows.end - 1)];
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t c = j * 32 + 8 * r + 4 * (lane >> 5);
                const vec_of<float, 4> scale = *reinterpret_cast<const vec_of<float, 4>*>(&b_scale[wn + c]);
                const vec_of<float, 4> shift = *reinterpret_cast<const vec_of<float, 4>*>(&bias[wn + c]);
                vec_of<float, 4> v;
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = (float) acc[i][j][4 * r + q] * a_scale * scale[q] + shift[q];
                *reinterpret_cast<vec_of<O, 4>*>(&staged[(lane & 31) * LD + c]) = narrow<O, 4>(v);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int q = 0; q < 32 * COLUMNS / (64 * E); ++q) {
            const uint32_t r = (q * 64 + lane) / (COLUMNS / E), c = (q * 64 + lane) % (COLUMNS / E) * E;
            const uint32_t m = m0 + r, n = n0 + wn + c;
            if (m >= rows.end || n >= p.n) continue;
            const vec_of<O, E> v = *reinterpret_cast<const vec_of<O, E>*>(&staged[r * LD + c]);
            O* to = out + (size_t) m * p.out_stride + n;
            if (n + E <= p.n) store_vec_once<O, E>(to, v);
            else
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (n + e < p.n) to[e] = v[e];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <class O, int RT, int NB, int WAVES, int AHEAD>
int launch_few_rows(skm_ctx* ctx, const ProductArgs& p) {
    const uint32_t tiles_n = (p.n + 16 * NB - 1) / (16 * NB);
    const uint64_t blocks = ((uint64_t) (p.m + 16 * RT - 1) / (16 * RT) + (p.offsets ? p.groups : 0)) * tiles_n;
    if (blocks > 0x7fffffffULL) return set_error(SKM_ERR_INVALID, "skm_product_i8: more than 2^31 tiles");
    return launch_in_parts(blocks, [&](const uint32_t first, const unsigned count) {
        product_few_rows_kernel<O, RT, NB, WAVES, AHEAD><<<count, WAVES * 64, 0, ctx->stream>>>(p, tiles_n, first);
        return check_hip(hipGetLastError(), "product_few_rows_kernel launch");
    });
}

template <class O, int FM, int FN, int WN>
int launch_tiles(skm_ctx* ctx, const ProductArgs& p) {
    constexpr size_t lds = tiles_lds_bytes<FM, FN, WN>();
    constexpr uint32_t TN = 32 * WN * FN;
    const uint32_t tiles_n = (p.n + TN - 1) / TN;
    const uint64_t tiles_m = (uint64_t) (p.m + 64 * FM - 1) / (64 * FM) + (p.offsets ? p.groups : 0);
    uint32_t super_n = 1;
    while (super_n < 8 && super_n < tiles_n) super_n *= 2;
    const uint32_t super_m = 32 / super_n, across = (tiles_n + super_n - 1) / super_n;
    const uint64_t supers = (tiles_m + super_m - 1) / super_m * across, blocks = supers * 32;
    if (blocks > 0x7fffffffULL) return set_error(SKM_ERR_INVALID, "skm_product_i8: more than 2^31 tiles");
    const TileMap map{super_m, super_n, across, tiles_n, (uint32_t) (supers / 8 * 256)};
    const auto launch = [&](auto kernel) {
        SKM_TRY(check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int) lds),
                          "hipFuncSetAttribute(MaxDynamicSharedMemorySize)"));
        return launch_in_parts(blocks, [&](const uint32_t first, const unsigned count) {  // parts begin at multiples of 8: dies stay
            kernel<<<count, 128 * WN, lds, ctx->stream>>>(p, map, first);
            return check_hip(hipGetLastError(), "product_tiles_kernel launch");
        });
    };
    return launch(product_tiles_kernel<O, FM, FN, WN>);
}

// The kernel for a call: the largest tile that still gives every compute unit a workgroup (the largest one already where three
// quarters get one).  A larger tile reads each operand fewer times, and loses more than that where it leaves compute units
// without one (us, bf16 results, the chosen one in brackets):
//     rows x n x k         256 x 256  128 x 256  128 x 128  128 x 64  64 x 64   few rows: 32 x 64  32 x 32  32 x 16  16 x 16
//     8192 x 8192 x 4096     [258]       292        320       380
//     3000 x 4096 x 4096      [55]        67         63        77        89
//     2048 x 4096 x 4096       49        [38]        43        51
//     1024 x 4096 x 4096                  30        [24]       28        32
//      512 x 4096 x 4096                  29         21       [19]       19                  50
//      256 x 4096 x 4096                             20        17       [15]                 26
//      128 x 4096 x 4096                                       17        14                 [14]       17
//       64 x 4096 x 4096                                                                     14       [10]       12
//       64 x 1024 x 4096                                                                               10         8       [7]
//       16 x 4096 x 4096                                                                                9         7       [8]
// Over groups the host knows the rows of a group on average only, and every group's last tile is part empty.  There 64 x 64
// tiles pay from 9 rows on (64 groups, n 2048, k 1024: 16 rows each 29 us against 35 us with the few rows' best tile, 8 rows
// each 29 us with 16 x 64 of those), 128 rows to a tile from 49 on (64 rows each 36 against 40 us), 256 from 129 on
// (512 rows each 125 us with either; 8 groups of 4,096, n 4096, k 1536: 267 against 278 us).
template <class O>
int launch_product(skm_ctx* ctx, const ProductArgs& p) {
    constexpr uint64_t WANTED = 256;
    const bool grouped = p.offsets != nullptr;
    const uint64_t rows = ((uint64_t) p.m + p.groups - 1) / p.groups;  // of a group, on average
    const auto tiles = [&](const uint64_t tm, const uint64_t tn) { return p.groups * ((rows + tm - 1) / tm) * ((p.n + tn - 1) / tn); };
    // what the tiles' loads assume: 16 columns at least, a tile's offsets in 32 bits
    if (p.k >= 16 && p.a_stride < (1u << 23) && p.b_stride < (1u << 23)) {
        const uint64_t many = grouped ? 48 : 64;
        if (rows > 128 && tiles(256, 256) >= WANTED * 3 / 4) return launch_tiles<O, 4, 2, 4>(ctx, p);
        if (rows > many && tiles(128, 256) >= WANTED) return launch_tiles<O, 2, 2, 4>(ctx, p);
        if (rows > many && tiles(128, 128) >= WANTED) return launch_tiles<O, 2, 1, 4>(ctx, p);
        if (rows > many && tiles(128, 64) >= WANTED) return launch_tiles<O, 2, 1, 2>(ctx, p);
        if (rows > (grouped ? 8 : 32) && tiles(64, 64) >= WANTED) return launch_tiles<O, 1, 1, 2>(ctx, p);
    }
    if (rows > 16 && tiles(32, 64) >= WANTED) return launch_few_rows<O, 2, 4, 8, 2>(ctx, p);
    if (rows > 16 && tiles(32, 32) >= WANTED) return launch_few_rows<O, 2, 2, 8, 4>(ctx, p);
    if (rows > 16) return launch_few_rows<O, 2, 1, 8, 4>(ctx, p);
    if (grouped && tiles(16, 64) >= 4 * WANTED) return launch_few_rows<O, 1, 4, 4, 4>(ctx, p);
    if (grouped) return launch_few_rows<O, 2, 2, 4, 4>(ctx, p);
    return launch_few_rows<O, 1, 1, 8, 8>(ctx, p);
}

} // namespace
} // namespace skm

using namespace skm;

extern "C" {

int skm_quantize_rows(skm_ctx* ctx, const void* d_x, int type, size_t n, size_t d, size_t x_stride, int8_t* d_q, size_t q_stride,
                      float* d_scales) {
    SKM_REQUIRE(ctx, "null context");
    SKM_REQUIRE(is_value_type(type), "type must be SKM_F32, SKM_F16 or SKM_BF16");
    SKM_REQUIRE(d > 0 && d <= SKM_ROW_MAX_D, "d out of range");
    SKM_REQUIRE(x_stride >= d && q_stride >= d, "strides must be at least d");
    SKM_REQUIRE(n < SKM_NO_ROW, "n must fit in 32 bits");
    if (n == 0) return SKM_OK;
    SKM_REQUIRE(d_x && d_q && d_scales, "null pointer");
    const size_t size = type_size(type);
    SKM_REQUIRE(address(d_x) % size == 0 && address(d_scales) % 4 == 0, "pointers must be aligned to their elements");
    const Argument x{"x", matrix_memory(d_x, n, x_stride, d, size)}, q{"q", matrix_memory(d_q, n, q_stride, d, 1)};
    SKM_TRY(check_apart(__func__, q, {x}));
    SKM_TRY(check_apart(__func__, {"scales", vector_memory(d_scales, n, 4)}, {x, q}));
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/quantize");
    return for_type(type, [&](auto sample) {
        using T = decltype(sample);
        return for_elements<T>(vector_elements(size, 1, d), [&](auto elements) {
            constexpr int E = decltype(elements)::value;
            const uint32_t vectors = (uint32_t) ((d + E - 1) / E);
            const auto launch = [&](auto waves, auto held) {
                constexpr int WAVES = decltype(waves)::value, HELD = decltype(held)::value, ROWS = QUANTIZE_THREADS / 64 / WAVES;
                const unsigned blocks = (unsigned) std::min<uint64_t>((n + ROWS - 1) / ROWS, ROWS_MAX_BLOCKS);
                quantize_rows_kernel<T, E, WAVES, HELD><<<blocks, QUANTIZE_THREADS, 0, ctx->stream>>>((const T*) d_x, n, vectors, (uint32_t) (d - E), x_stride,
                                                                                                      d_q, q_stride, d_scales);
                return check_hip(hipGetLastError(), "quantize_rows_kernel launch");
            };
            if (vectors <= 256) return launch(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
            if (vectors <= 512) return launch(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
            return launch(std::integral_constant<int, 4>{}, std::integral_constant<int, 8>{});
        });
    });
}

int skm_product_i8(skm_ctx* ctx, const int8_t* d_a, size_t m, size_t a_stride, const float* d_a_scale, const int8_t* d_b, size_t n,
                   size_t k, size_t b_stride, const float* d_b_scale, const float* d_bias, size_t groups, size_t b_group_stride,
                   const uint32_t* d_offsets, void* d_out, int out_type, size_t out_stride) {
    SKM_REQUIRE(ctx, "null context");
    SKM_REQUIRE(is_value_type(out_type), "out_type must be SKM_F32, SKM_F16 or SKM_BF16");
    SKM_REQUIRE(n > 0 && n <= SKM_ROW_MAX_D, "n out of range");
    SKM_REQUIRE(k > 0 && k <= SKM_PRODUCT_MAX_K, "k out of range");
    SKM_REQUIRE(m <= SKM_PRODUCT_MAX_M, "m out of range");
    SKM_REQUIRE(a_stride >= k && b_stride >= k && out_stride >= n, "strides must be at least the row length");
    SKM_REQUIRE(b_stride < (size_t(1) << 40) && (!d_offsets || b_group_stride < (size_t(1) << 46)), "strides out of range");
    if (d_offsets) {
        SKM_REQUIRE(groups > 0 && groups <= SKM_PRODUCT_MAX_GROUPS, "groups out of range");
        SKM_REQUIRE(groups == 1 || b_group_stride >= (n - 1) * b_stride + k, "b_group_stride must be at least a group's matrix");
    }
    if (m == 0) return SKM_OK;
    SKM_REQUIRE(d_a && d_a_scale && d_b && d_b_scale && d_out, "null pointer");
    const size_t out_size = type_size(out_type);
    SKM_REQUIRE((address(d_a_scale) | address(d_b_scale) | address(d_bias) | address(d_offsets)) % 4 == 0 && address(d_out) % out_size == 0,
                "pointers must be aligned to their elements");
    const size_t matrices = d_offsets ? groups : 1;
    // of several matrices the whole range
    const Memory b = matrices == 1 ? matrix_memory(d_b, n, b_stride, k, 1)
                                   : matrix_memory(d_b, 1, (matrices - 1) * b_group_stride + (n - 1) * b_stride + k,
                                                   (matrices - 1) * b_group_stride + (n - 1) * b_stride + k, 1);
    SKM_TRY(check_apart(__func__, {"out", matrix_memory(d_out, m, out_stride, n, out_size)},
                        {{"a", matrix_memory(d_a, m, a_stride, k, 1)}, {"a_scale", vector_memory(d_a_scale, m, 4)}, {"b", b},
                         {"b_scale", vector_memory(d_b_scale, matrices * n, 4)}, {"the bias", vector_memory(d_bias, matrices * n, 4)},
                         {"the offsets", vector_memory(d_offsets, d_offsets ? groups + 1 : 0, 4)}}));
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/product");
    const ProductArgs p{d_a, d_a_scale, d_b, d_b_scale, d_bias, d_offsets, d_out, a_stride, b_stride, d_offsets ? b_group_stride : 0,
                        out_stride, (uint32_t) m, (uint32_t) n, (uint32_t) k, d_offsets ? (uint32_t) groups : 1};
    return for_type(out_type, [&](auto sample) {
        using O = decltype(sample);
        return launch_product<O>(ctx, p);
    });
}

} // extern "C"
