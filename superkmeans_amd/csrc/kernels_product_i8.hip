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

// The whole number nearest to 127 x / most, ties to even.  The fp32 product is at most 2 units of its last place off
// (3e-5 at 127), so that the choice between two numbers can only be wrong next to the border between them; there the
// quotient is taken in fp64, where 127 x is exact and a quotient of two fp32 numbers cannot round onto a border.
__device__ __forceinline__ int nearest_step(const float x, const float most, const float inverse) {
    const float t = x * inverse;
    const float r = rintf(t);
    if (fabsf(t - r) < 0.4999f) return (int) r;
    return (int) rint((double) x * 127.0 / (double) most);
}

constexpr int QUANTIZE_THREADS = 256;

template <class T, int E>
__global__ __launch_bounds__(QUANTIZE_THREADS) void quantize_rows_kernel(
    const T* __restrict__ x, const size_t n, const uint32_t vectors, const size_t x_stride, int8_t* __restrict__ q,
    const size_t q_stride, float* __restrict__ scales
) {
    __shared__ uint32_t wave_most[QUANTIZE_THREADS / 64];
    for (size_t t = blockIdx.x; t < n; t += gridDim.x) {
        const T* row = x + t * x_stride;
        uint32_t most = 0;  // bits of the largest magnitude: ordered like the numbers, infinities and NaN above all
        for (uint32_t at = threadIdx.x; at < vectors; at += QUANTIZE_THREADS) {
            const vec_of<float, E> v = widen<E>(load_vec<T, E>(row + (size_t) at * E));
#pragma unroll
            for (int e = 0; e < E; ++e) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) most = max(most, (uint32_t) __shfl_xor(most, off));
        if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < QUANTIZE_THREADS / 64; ++w) most = max(most, wave_most[w]);
        __syncthreads();
        const bool usable = most != 0 && most < 0x7f800000u;
        const float m = __uint_as_float(most);
        const float inverse = m > 1e-30f ? 127.0f / m : __builtin_nanf("");  // NaN sends every element through fp64
        if (threadIdx.x == 0) scales[t] = most < 0x7f800000u ? m / 127.0f : __builtin_nanf("");
        for (uint32_t at = threadIdx.x; at < vectors; at += QUANTIZE_THREADS) {
            const vec_of<float, E> v = widen<E>(load_vec<T, E>(row + (size_t) at * E));
            vec_of<int8_t, E> r = {};
            if (usable)
#pragma unroll
                for (int e = 0; e < E; ++e) r[e] = (int8_t) nearest_step(v[e], m, inverse);
            *reinterpret_cast<vec_of<int8_t, E>*>(q + t * q_stride + (size_t) at * E) = r;
        }
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

// The tile of `tm` rows with the given number, counted through the groups; first == end where there is none.  Offsets are
// clamped to the rows there are.  Every wavefront of a workgroup finds it by itself, 64 groups at a time.
__device__ __forceinline__ RowTile find_rows(const ProductArgs& p, const uint32_t tm, uint32_t number) {
    if (!p.offsets) {
        const uint32_t first = number * tm;
        return {0, min(first, p.m), min(p.m, first + tm)};
    }
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t g0 = 0; g0 < p.groups; g0 += 64) {
        const uint32_t g = g0 + lane;
        uint32_t from = 0, to = 0;
        if (g < p.groups) {
            from = min(p.offsets[g], p.m);
            to = max(from, min(p.offsets[g + 1], p.m));
        }
        const uint32_t tiles = (to - from + tm - 1) / tm;
        uint32_t incl = tiles;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t t = __shfl_up(incl, off);
            if (lane >= (uint32_t) off) incl += t;
        }
        const unsigned long long past = __ballot(incl > number);
        if (past) {
            const int at = __builtin_ctzll(past);
            const uint32_t before = __shfl(incl - tiles, at);
            const uint32_t first = __shfl(from, at) + (number - before) * tm;
            return {g0 + at, first, min((uint32_t) __shfl(to, at), first + tm)};
        }
        number -= __shfl(incl, 63);
    }
    return {0, 0, 0};
}

// 16 columns of a row from column k on, zeros past the last one.  W: the bytes that pointers and strides are aligned to.
template <int W>
__device__ __forceinline__ intx4 load_columns(const int8_t* row, const uint32_t k, const uint32_t columns) {
    if constexpr (W == 16) {
        if (k + 16 <= columns) return *reinterpret_cast<const intx4*>(row + k);
    }
    intx4 v = {};
    if constexpr (W >= 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (k + 4 * i + 4 <= columns) v[i] = *reinterpret_cast<const int*>(row + k + 4 * i);
            else
                for (uint32_t j = 0; j < 4; ++j)
                    if (k + 4 * i + j < columns) v[i] |= (int) (uint8_t) row[k + 4 * i + j] << (8 * j);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (k + 4 * i + j < columns) v[i] |= (int) (uint8_t) row[k + 4 * i + j] << (8 * j);
    }
    return v;
}

template <class O>
__device__ __forceinline__ void put(void* out, const size_t at, const float v) {
    reinterpret_cast<O*>(out)[at] = (O) v;
}

// 128 x 128 tiles, four wavefronts of 64 x 64 in 32 x 32 blocks, 64 columns of both operands at a time in LDS.
constexpr int TILE = 128, TILE_K = 64, TILE_STRIDE = TILE_K + 16;  // 16 bytes of padding: rows start in different banks

template <class O, int W>
__global__ __launch_bounds__(256) void product_tile_kernel(const ProductArgs p, const uint32_t tiles_n) {
    __shared__ __align__(16) int8_t As[TILE * TILE_STRIDE];
    __shared__ __align__(16) int8_t Bs[TILE * TILE_STRIDE];
    const RowTile rows = find_rows(p, TILE, blockIdx.x / tiles_n);
    if (rows.first >= rows.end) return;
    const uint32_t n0 = blockIdx.x % tiles_n * TILE;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    const int8_t* b = p.b + (size_t) rows.group * p.b_group_stride;
    intx16 acc[2][2] = {};
    for (uint32_t k0 = 0; k0 < p.k; k0 += TILE_K) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t r = (tid >> 2) + i * 64, c = (tid & 3) * 16;
            const uint32_t row_a = min(rows.first + r, rows.end - 1), row_b = min(n0 + r, p.n - 1);  // repeated rows are not stored
            *reinterpret_cast<intx4*>(&As[r * TILE_STRIDE + c]) = load_columns<W>(p.a + (size_t) row_a * p.a_stride, k0 + c, p.k);
            *reinterpret_cast<intx4*>(&Bs[r * TILE_STRIDE + c]) = load_columns<W>(b + (size_t) row_b * p.b_stride, k0 + c, p.k);
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < TILE_K; kk += 32) {
            intx4 fa[2], fb[2];
            const uint32_t c = kk + (lane >> 5) * 16;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = *reinterpret_cast<const intx4*>(&As[(wm + i * 32 + (lane & 31)) * TILE_STRIDE + c]);
                fb[i] = *reinterpret_cast<const intx4*>(&Bs[(wn + i * 32 + (lane & 31)) * TILE_STRIDE + c]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t n = n0 + wn + j * 32 + (lane & 31);
        if (n >= p.n) continue;
        const float b_scale = p.b_scale[(size_t) rows.group * p.n + n];
        const float bias = p.bias ? p.bias[(size_t) rows.group * p.n + n] : 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t m = rows.first + wm + i * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                if (m < rows.end) put<O>(p.out, (size_t) m * p.out_stride + n, (float) acc[i][j][r] * p.a_scale[m] * b_scale + bias);
            }
    }
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
    SKM_REQUIRE(!overlap(d_x, span(n, x_stride, d, size), d_q, span(n, q_stride, d, 1)), "q overlaps x");
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/quantize");
    const size_t in_width = common_width({address(d_x), x_stride * size, d * size});
    const size_t per_lane = std::min(in_width / size, common_width({address(d_q), q_stride, d}));
    return for_type(type, [&](auto sample) {
        using T = decltype(sample);
        return for_width<T>(per_lane * size, [&](auto elements) {
            constexpr int E = decltype(elements)::value;
            const unsigned blocks = (unsigned) std::min<uint64_t>(n, ROWS_MAX_BLOCKS);
            quantize_rows_kernel<T, E><<<blocks, QUANTIZE_THREADS, 0, ctx->stream>>>((const T*) d_x, n, (uint32_t) (d / E), x_stride, d_q,
                                                                                     q_stride, d_scales);
            return check_hip(hipGetLastError(), "quantize_rows_kernel launch");
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
    if (d_offsets) {
        SKM_REQUIRE(groups > 0 && groups <= SKM_PRODUCT_MAX_GROUPS, "groups out of range");
        SKM_REQUIRE(groups == 1 || b_group_stride >= (n - 1) * b_stride + k, "b_group_stride must be at least a group's matrix");
    }
    if (m == 0) return SKM_OK;
    SKM_REQUIRE(d_a && d_a_scale && d_b && d_b_scale && d_out, "null pointer");
    const size_t out_size = type_size(out_type);
    SKM_REQUIRE((address(d_a_scale) | address(d_b_scale) | address(d_bias) | address(d_offsets)) % 4 == 0 && address(d_out) % out_size == 0,
                "pointers must be aligned to their elements");
    const size_t out_bytes = span(m, out_stride, n, out_size);
    SKM_REQUIRE(!overlap(d_a, span(m, a_stride, k, 1), d_out, out_bytes), "out overlaps a");
    SKM_REQUIRE(!overlap(d_b, (d_offsets ? (groups - 1) * b_group_stride : 0) + span(n, b_stride, k, 1), d_out, out_bytes), "out overlaps b");
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/product");
    const ProductArgs p{d_a, d_a_scale, d_b, d_b_scale, d_bias, d_offsets, d_out, a_stride, b_stride, d_offsets ? b_group_stride : 0,
                        out_stride, (uint32_t) m, (uint32_t) n, (uint32_t) k, d_offsets ? (uint32_t) groups : 1};
    const size_t width = common_width({address(d_a), address(d_b), a_stride, b_stride, p.b_group_stride});
    return for_type(out_type, [&](auto sample) {
        using O = decltype(sample);
        const uint32_t tiles_n = (uint32_t) ((n + TILE - 1) / TILE);
        const uint64_t tiles_m = (m + TILE - 1) / TILE + (d_offsets ? groups : 0);
        SKM_REQUIRE(tiles_m * tiles_n <= 0x7fffffffULL, "too many tiles for one launch");
        const unsigned blocks = (unsigned) (tiles_m * tiles_n);
        if (width == 16) product_tile_kernel<O, 16><<<blocks, 256, 0, ctx->stream>>>(p, tiles_n);
        else if (width >= 4) product_tile_kernel<O, 4><<<blocks, 256, 0, ctx->stream>>>(p, tiles_n);
        else product_tile_kernel<O, 1><<<blocks, 256, 0, ctx->stream>>>(p, tiles_n);
        return check_hip(hipGetLastError(), "product_tile_kernel launch");
    });
}

} // extern "C"
