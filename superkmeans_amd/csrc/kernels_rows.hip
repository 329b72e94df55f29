// Rows of a table looked up by id, rows sent to their groups and brought back with weights, and the gradients of the
// latter.  All of it moves rows: the bytes of the rows bound every kernel here, and the arithmetic is a product and a sum
// per element.
#include "rows_common.h"

namespace skm {

int call_scratch(skm_ctx* ctx, const char* who, void* given, const size_t given_bytes, const size_t need, void** out) {
    if (need == 0) {
        *out = nullptr;
        return SKM_OK;
    }
    if (given) {
        if (given_bytes < need)
            return set_error(SKM_ERR_INVALID, "%s: %zu bytes of scratch given, %zu needed", who, given_bytes, need);
        if (address(given) % 16) return set_error(SKM_ERR_INVALID, "%s: scratch must be 16-byte aligned", who);
        *out = given;
        return SKM_OK;
    }
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    SKM_HIP_TRY(hipStreamIsCapturing(ctx->stream, &status));
    if (status != hipStreamCaptureStatusNone)
        return set_error(SKM_ERR_INVALID, "%s: a captured call brings its own scratch", who);
    if (need > ctx->workspace_limit)
        return set_error(SKM_ERR_INVALID, "%s: %zu bytes of scratch needed, the workspace limit is %zu", who, need,
                         ctx->workspace_limit);
    return workspace(ctx, skm_ctx::WS_ROWS, need, out);
}

namespace {

constexpr int UNROLL = 4;  // vectors a lane requests before it uses the first

// id of position i, or a number at or past every table size where there is none
__device__ __forceinline__ uint64_t id_at(const void* ids, const int ids_type, const size_t i) {
    return ids_type == SKM_I64 ? reinterpret_cast<const uint64_t*>(ids)[i] : (uint64_t) reinterpret_cast<const uint32_t*>(ids)[i];
}

// out[t] = scale * table[id_t], a row of zeros where the id is no row.  A wavefront takes TOKENS rows at a time and requests all
// their ids, then UNROLL vectors per lane of all the rows, before it stores the first: with one row at a time the wavefronts
// that a compute unit holds do not have enough bytes on their way (a million rows of 4 KiB: one row at a time 790 us, four 782,
// eight 783).  Bound by the stores: those 4.1 GB in 783 us are 5.2 TB/s, next to 1.5 GB of table rows
// that miss the compute dies' L2.
template <class T, int E, int TOKENS>
__global__ __launch_bounds__(ROWS_THREADS) void lookup_rows_kernel(
    const T* __restrict__ table, const size_t rows, const size_t table_stride, const void* __restrict__ ids, const int ids_type,
    const size_t n, const float scale, T* __restrict__ out, const size_t out_stride, const RowSplit s
) {
    const uint32_t lane = threadIdx.x & 63, in_row = lane & (s.lanes - 1), row_of_wave = lane / s.lanes, rows_of_wave = 64 / s.lanes;
    const uint64_t step = (uint64_t) gridDim.x * (ROWS_THREADS / 64);
    for (uint64_t u = (uint64_t) blockIdx.x * (ROWS_THREADS / 64) + (threadIdx.x >> 6); u < s.units; u += step) {
        const size_t t = (size_t) (u / s.pieces) * (TOKENS * rows_of_wave) + row_of_wave;
        const uint32_t first = (uint32_t) (u % s.pieces) * s.lanes * UNROLL + in_row;
        uint64_t id[TOKENS];
#pragma unroll
        for (int q = 0; q < TOKENS; ++q) id[q] = t + q * rows_of_wave < n ? id_at(ids, ids_type, t + q * rows_of_wave) : rows;
        vec_of<T, E> v[TOKENS][UNROLL];
#pragma unroll
        for (int q = 0; q < TOKENS; ++q)
#pragma unroll
            for (int i = 0; i < UNROLL; ++i) {
                const uint32_t at = first + i * s.lanes;
                if (at < s.vectors && id[q] < rows) v[q][i] = load_vec<T, E>(table + id[q] * table_stride + column<E>(at, s.last));
                else v[q][i] = vec_of<T, E>{};
            }
#pragma unroll
        for (int q = 0; q < TOKENS; ++q) {
            if (t + q * rows_of_wave >= n) break;
#pragma unroll
            for (int i = 0; i < UNROLL; ++i) {
                const uint32_t at = first + i * s.lanes;
                if (at < s.vectors) {
                    const vec_of<T, E> r = scale == 1.0f || id[q] >= rows ? v[q][i] : narrow<T, E>(widen<E>(v[q][i]) * scale);
                    store_vec_once<T, E>(out + (t + q * rows_of_wave) * out_stride + column<E>(at, s.last), r);
                }
            }
        }
    }
}

// out[slot[t][j]] = x[t] for every choice j that has a slot: the row is read once and stored once per choice.  Bound by memory:
// 32,768 rows of 8 KiB to 2 groups each, 0.8 GB, in 134 us, 6.0 TB/s.
template <class T, int E>
__global__ __launch_bounds__(ROWS_THREADS) void dispatch_rows_kernel(
    const T* __restrict__ x, const size_t x_stride, const size_t n, const uint32_t* __restrict__ slots, const uint32_t choices,
    const size_t out_rows, T* __restrict__ out, const size_t out_stride, const RowSplit s
) {
    const uint32_t lane = threadIdx.x & 63, in_row = lane & (s.lanes - 1), row_of_wave = lane / s.lanes;
    const uint64_t step = (uint64_t) gridDim.x * (ROWS_THREADS / 64);
    for (uint64_t u = (uint64_t) blockIdx.x * (ROWS_THREADS / 64) + (threadIdx.x >> 6); u < s.units; u += step) {
        const size_t t = (size_t) (u / s.pieces) * (64 / s.lanes) + row_of_wave;
        if (t >= n) continue;
        const uint32_t first = (uint32_t) (u % s.pieces) * s.lanes * UNROLL + in_row;
        vec_of<T, E> v[UNROLL];
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const uint32_t at = first + i * s.lanes;
            if (at < s.vectors) v[i] = load_vec_once<T, E>(x + t * x_stride + column<E>(at, s.last));
        }
        for (uint32_t j = 0; j < choices; ++j) {
            const uint32_t slot = slots[t * choices + j];
            if (slot >= out_rows) continue;
#pragma unroll
            for (int i = 0; i < UNROLL; ++i) {
                const uint32_t at = first + i * s.lanes;
                if (at < s.vectors) store_vec_once<T, E>(out + (size_t) slot * out_stride + column<E>(at, s.last), v[i]);
            }
        }
    }
}

__device__ __forceinline__ float weight_at(const void* weights, const int type, const size_t i) {
    if (type == SKM_F32) return reinterpret_cast<const float*>(weights)[i];
    if (type == SKM_F16) return (float) reinterpret_cast<const _Float16*>(weights)[i];
    return (float) reinterpret_cast<const __bf16*>(weights)[i];
}
__device__ __forceinline__ void put_weight(void* weights, const int type, const size_t i, const float v) {
    if (type == SKM_F32) reinterpret_cast<float*>(weights)[i] = v;
    else if (type == SKM_F16) reinterpret_cast<_Float16*>(weights)[i] = (_Float16) v;
    else reinterpret_cast<__bf16*>(weights)[i] = (__bf16) v;
}

constexpr int COMBINE_UNROLL = 4;  // vectors per lane
constexpr int COMBINE_AHEAD = 2;   // choices whose rows are requested together

// out[t] = sum_j w[t][j] * rows[slot[t][j]], j ascending, in fp32.  A lane has COMBINE_AHEAD x COMBINE_UNROLL vectors on their
// way.  Bound by memory: 16,384 sums over 8 rows of 3 KiB, 0.45 GB, in 75 us, 6.0 TB/s.
template <class T, int E>
__global__ __launch_bounds__(ROWS_THREADS) void combine_rows_kernel(
    const T* __restrict__ rows, const size_t n_rows, const size_t rows_stride, const uint32_t* __restrict__ slots, const size_t n,
    const uint32_t choices, const void* __restrict__ weights, const int weights_type, T* __restrict__ out, const size_t out_stride,
    const RowSplit s
) {
    const uint32_t lane = threadIdx.x & 63, in_row = lane & (s.lanes - 1), row_of_wave = lane / s.lanes;
    const uint64_t step = (uint64_t) gridDim.x * (ROWS_THREADS / 64);
    for (uint64_t u = (uint64_t) blockIdx.x * (ROWS_THREADS / 64) + (threadIdx.x >> 6); u < s.units; u += step) {
        const size_t t = (size_t) (u / s.pieces) * (64 / s.lanes) + row_of_wave;
        if (t >= n) continue;
        const uint32_t first = (uint32_t) (u % s.pieces) * s.lanes * COMBINE_UNROLL + in_row;
        vec_of<float, E> sum[COMBINE_UNROLL] = {};
        for (uint32_t j0 = 0; j0 < choices; j0 += COMBINE_AHEAD) {
            vec_of<T, E> v[COMBINE_AHEAD][COMBINE_UNROLL];
            uint32_t slot[COMBINE_AHEAD];
            float w[COMBINE_AHEAD];
#pragma unroll
            for (int j = 0; j < COMBINE_AHEAD; ++j) {
                slot[j] = j0 + j < choices ? slots[t * choices + j0 + j] : SKM_NO_ROW;
                w[j] = 1.0f;
                if (weights && slot[j] < n_rows) w[j] = weight_at(weights, weights_type, t * choices + j0 + j);
            }
#pragma unroll
            for (int j = 0; j < COMBINE_AHEAD; ++j)
#pragma unroll
                for (int i = 0; i < COMBINE_UNROLL; ++i) {
                    const uint32_t at = first + i * s.lanes;
                    if (slot[j] < n_rows && at < s.vectors)
                        v[j][i] = load_vec_once<T, E>(rows + (size_t) slot[j] * rows_stride + column<E>(at, s.last));
                }
#pragma unroll
            for (int j = 0; j < COMBINE_AHEAD; ++j)
                if (slot[j] < n_rows)
#pragma unroll
                    for (int i = 0; i < COMBINE_UNROLL; ++i) sum[i] += w[j] * widen<E>(v[j][i]);
        }
#pragma unroll
        for (int i = 0; i < COMBINE_UNROLL; ++i) {
            const uint32_t at = first + i * s.lanes;
            if (at < s.vectors) store_vec_once<T, E>(out + t * out_stride + column<E>(at, s.last), narrow<T, E>(sum[i]));
        }
    }
}

// grad_rows[slot[t][j]] = w[t][j] * grad[t] and grad_w[t][j] = <grad[t], rows[slot[t][j]]>: one walk over the token's row
// for each GRAD_CHOICES choices, WAVES wavefronts per token.  Bound by memory: 10,007 tokens of 4,000 bytes and 4 choices,
// 0.36 GB, in 68 us, 5.3 TB/s (85 us with one wavefront per token, which has a token's vectors in four turns).
template <int WAVES>
constexpr int GRAD_THREADS = WAVES > 4 ? WAVES * 64 : ROWS_THREADS;

template <class T, int E, int WAVES, int GRAD_CHOICES>
__global__ __launch_bounds__(GRAD_THREADS<WAVES>) void combine_rows_grad_kernel(
    const T* __restrict__ grad, const size_t n, const uint32_t vectors, const uint32_t last, const size_t grad_stride, const T* __restrict__ rows,
    const size_t n_rows, const size_t rows_stride, const uint32_t* __restrict__ slots, const uint32_t choices,
    const void* __restrict__ weights, const int weights_type, T* __restrict__ grad_rows, const size_t grad_rows_stride,
    void* __restrict__ grad_weights
) {
    constexpr int TOKENS = GRAD_THREADS<WAVES> / 64 / WAVES;  // tokens per workgroup
    __shared__ float part[GRAD_THREADS<WAVES> / 64][GRAD_CHOICES];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t in_row = threadIdx.x % (64 * WAVES);
    // every thread of a workgroup takes the same number of turns, so that all of them meet at the barriers
    const size_t turns = (n + TOKENS - 1) / TOKENS;
    for (size_t turn = blockIdx.x; turn < turns; turn += gridDim.x) {
        const size_t t = turn * TOKENS + wave / WAVES;
        for (uint32_t j0 = 0; j0 < choices; j0 += GRAD_CHOICES) {
            float dot[GRAD_CHOICES] = {};
            if (t < n) {
                uint32_t slot[GRAD_CHOICES];
                float w[GRAD_CHOICES];
#pragma unroll
                for (int j = 0; j < GRAD_CHOICES; ++j) {
                    slot[j] = j0 + j < choices ? slots[t * choices + j0 + j] : SKM_NO_ROW;
                    w[j] = 1.0f;
                    if (weights && slot[j] < n_rows) w[j] = weight_at(weights, weights_type, t * choices + j0 + j);
                }
                for (uint32_t at = in_row; at < vectors; at += 64 * WAVES) {
                    const uint32_t c = column<E>(at, last);
                    const int repeated = (int) (at * E - c);  // elements that the vector before has too
                    const vec_of<float, E> g = widen<E>(load_vec<T, E>(grad + t * grad_stride + c));
                    vec_of<T, E> y[GRAD_CHOICES];
                    if (grad_weights) {
#pragma unroll
                        for (int j = 0; j < GRAD_CHOICES; ++j)
                            if (slot[j] < n_rows) y[j] = load_vec_once<T, E>(rows + (size_t) slot[j] * rows_stride + c);
                    }
#pragma unroll
                    for (int j = 0; j < GRAD_CHOICES; ++j) {
                        if (slot[j] >= n_rows) continue;
                        if (grad_weights) {
                            const vec_of<float, E> p = g * widen<E>(y[j]);
                            float sum = 0.0f;
#pragma unroll
                            for (int e = 0; e < E; ++e) sum += e >= repeated ? p[e] : 0.0f;
                            dot[j] += sum;
                        }
                        if (grad_rows)
                            store_vec_once<T, E>(grad_rows + (size_t) slot[j] * grad_rows_stride + c, narrow<T, E>(g * w[j]));
                    }
                }
            }
            if (grad_weights) {
#pragma unroll
                for (int j = 0; j < GRAD_CHOICES; ++j)
#pragma unroll
                    for (int off = 32; off > 0; off >>= 1) dot[j] += __shfl_xor(dot[j], off);
                if (WAVES == 1) {
                    if (t < n && lane == 0)
#pragma unroll
                        for (int j = 0; j < GRAD_CHOICES; ++j)
                            if (j0 + j < choices) put_weight(grad_weights, weights_type, t * choices + j0 + j, dot[j]);
                } else {
                    __syncthreads();  // the sums of the turn before have been read
                    if (lane == 0)
#pragma unroll
                        for (int j = 0; j < GRAD_CHOICES; ++j) part[wave][j] = dot[j];
                    __syncthreads();
                    if (t < n && in_row < GRAD_CHOICES && j0 + in_row < choices) {
                        float sum = 0.0f;
                        for (int i = 0; i < WAVES; ++i) sum += part[wave / WAVES * WAVES + i][in_row];
                        put_weight(grad_weights, weights_type, t * choices + j0 + in_row, sum);
                    }
                }
            }
        }
    }
}

} // namespace
} // namespace skm

using namespace skm;

extern "C" {

int skm_lookup_rows(skm_ctx* ctx, const void* d_table, int type, size_t rows, size_t d, size_t table_stride, const void* d_ids,
                    int ids_type, size_t n, float scale, void* d_out, size_t out_stride) {
    SKM_REQUIRE(ctx, "null context");
    SKM_REQUIRE(is_value_type(type), "type must be SKM_F32, SKM_F16 or SKM_BF16");
    SKM_REQUIRE(ids_type == SKM_U32 || ids_type == SKM_I64, "ids_type must be SKM_U32 or SKM_I64");
    SKM_REQUIRE(d > 0 && d <= SKM_ROW_MAX_D, "d out of range");
    SKM_REQUIRE(table_stride >= d && out_stride >= d, "strides must be at least d");
    SKM_REQUIRE(rows < SKM_NO_ROW && n < SKM_NO_ROW, "rows and n must fit in 32 bits");
    if (n == 0) return SKM_OK;
    SKM_REQUIRE(d_ids && d_out && (d_table || rows == 0), "null pointer");
    const size_t size = type_size(type);
    SKM_REQUIRE(address(d_ids) % (ids_type == SKM_I64 ? 8 : 4) == 0 && address(d_table) % size == 0 && address(d_out) % size == 0,
                "pointers must be aligned to their elements");
    SKM_TRY(check_apart(__func__, {"out", matrix_memory(d_out, n, out_stride, d, size)},
                        {{"the table", matrix_memory(d_table, rows, table_stride, d, size)},
                         {"the ids", vector_memory(d_ids, n, ids_type == SKM_I64 ? 8 : 4)}}));
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/lookup");
    return for_type(type, [&](auto sample) {
        using T = decltype(sample);
        return for_elements<T>(vector_elements(size, size, d), [&](auto elements) {
            constexpr int E = decltype(elements)::value;
            const auto launch = [&](auto tokens) {
                constexpr int TOKENS = decltype(tokens)::value;
                const RowSplit s = split_rows((n + TOKENS - 1) / TOKENS, d, E, UNROLL);
                lookup_rows_kernel<T, E, TOKENS><<<row_blocks(s), ROWS_THREADS, 0, ctx->stream>>>(
                    (const T*) d_table, rows, table_stride, d_ids, ids_type, n, scale, (T*) d_out, out_stride, s);
                return check_hip(hipGetLastError(), "lookup_rows_kernel launch");
            };
            // several rows to a wavefront once there are wavefronts for the whole chip all the same (32 on each compute unit)
            if (split_rows(n, d, E, UNROLL).units >= 4 * 8192) return launch(std::integral_constant<int, 4>{});
            return launch(std::integral_constant<int, 1>{});
        });
    });
}

int skm_dispatch_rows(skm_ctx* ctx, const void* d_x, int type, size_t n, size_t d, size_t x_stride, const uint32_t* d_slots,
                      size_t choices, void* d_out, size_t out_rows, size_t out_stride) {
    SKM_REQUIRE(ctx, "null context");
    SKM_REQUIRE(is_value_type(type), "type must be SKM_F32, SKM_F16 or SKM_BF16");
    SKM_REQUIRE(d > 0 && d <= SKM_ROW_MAX_D, "d out of range");
    SKM_REQUIRE(x_stride >= d && out_stride >= d, "strides must be at least d");
    SKM_REQUIRE(n < SKM_NO_ROW && out_rows < SKM_NO_ROW, "row counts must fit in 32 bits");
    SKM_REQUIRE(choices > 0 && choices <= SKM_ROUTE_MAX_CHOICES, "choices out of range");
    if (n == 0 || out_rows == 0) return SKM_OK;
    SKM_REQUIRE(d_x && d_slots && d_out, "null pointer");
    const size_t size = type_size(type);
    SKM_REQUIRE(address(d_slots) % 4 == 0 && address(d_x) % size == 0 && address(d_out) % size == 0,
                "pointers must be aligned to their elements");
    SKM_TRY(check_apart(__func__, {"out", matrix_memory(d_out, out_rows, out_stride, d, size)},
                        {{"x", matrix_memory(d_x, n, x_stride, d, size)}, {"the slots", vector_memory(d_slots, n * choices, 4)}}));
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/dispatch");
    return for_type(type, [&](auto sample) {
        using T = decltype(sample);
        return for_elements<T>(vector_elements(size, size, d), [&](auto elements) {
            constexpr int E = decltype(elements)::value;
            const RowSplit s = split_rows(n, d, E, UNROLL);
            dispatch_rows_kernel<T, E><<<row_blocks(s), ROWS_THREADS, 0, ctx->stream>>>(
                (const T*) d_x, x_stride, n, d_slots, (uint32_t) choices, out_rows, (T*) d_out, out_stride, s);
            return check_hip(hipGetLastError(), "dispatch_rows_kernel launch");
        });
    });
}

int skm_combine_rows(skm_ctx* ctx, const void* d_rows, int type, size_t n_rows, size_t d, size_t rows_stride,
                     const uint32_t* d_slots, size_t n, size_t choices, const void* d_weights, int weights_type, void* d_out,
                     size_t out_stride) {
    SKM_REQUIRE(ctx, "null context");
    SKM_REQUIRE(is_value_type(type), "type must be SKM_F32, SKM_F16 or SKM_BF16");
    SKM_REQUIRE(!d_weights || is_value_type(weights_type), "weights_type must be SKM_F32, SKM_F16 or SKM_BF16");
    SKM_REQUIRE(d > 0 && d <= SKM_ROW_MAX_D, "d out of range");
    SKM_REQUIRE(rows_stride >= d && out_stride >= d, "strides must be at least d");
    SKM_REQUIRE(n < SKM_NO_ROW && n_rows < SKM_NO_ROW, "row counts must fit in 32 bits");
    SKM_REQUIRE(choices > 0 && choices <= SKM_ROUTE_MAX_CHOICES, "choices out of range");
    if (n == 0) return SKM_OK;
    SKM_REQUIRE((d_rows || n_rows == 0) && d_slots && d_out, "null pointer");
    const size_t size = type_size(type);
    SKM_REQUIRE(address(d_slots) % 4 == 0 && address(d_rows) % size == 0 && address(d_out) % size == 0 &&
                (!d_weights || address(d_weights) % type_size(weights_type) == 0), "pointers must be aligned to their elements");
    SKM_TRY(check_apart(__func__, {"out", matrix_memory(d_out, n, out_stride, d, size)},
                        {{"the rows", matrix_memory(d_rows, n_rows, rows_stride, d, size)}, {"the slots", vector_memory(d_slots, n * choices, 4)},
                         {"the weights", vector_memory(d_weights, n * choices, type_size(weights_type))}}));
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/combine");
    return for_type(type, [&](auto sample) {
        using T = decltype(sample);
        return for_elements<T>(vector_elements(size, size, d), [&](auto elements) {
            constexpr int E = decltype(elements)::value;
            const RowSplit s = split_rows(n, d, E, COMBINE_UNROLL);
            combine_rows_kernel<T, E><<<row_blocks(s), ROWS_THREADS, 0, ctx->stream>>>(
                (const T*) d_rows, n_rows, rows_stride, d_slots, n, (uint32_t) choices, d_weights, weights_type, (T*) d_out,
                out_stride, s);
            return check_hip(hipGetLastError(), "combine_rows_kernel launch");
        });
    });
}

int skm_combine_rows_grad(skm_ctx* ctx, const void* d_grad, int type, size_t n, size_t d, size_t grad_stride, const void* d_rows,
                          size_t n_rows, size_t rows_stride, const uint32_t* d_slots, size_t choices, const void* d_weights,
                          int weights_type, void* d_grad_rows, size_t grad_rows_stride, void* d_grad_weights) {
    SKM_REQUIRE(ctx, "null context");
    SKM_REQUIRE(is_value_type(type), "type must be SKM_F32, SKM_F16 or SKM_BF16");
    SKM_REQUIRE((!d_weights && !d_grad_weights) || is_value_type(weights_type), "weights_type must be SKM_F32, SKM_F16 or SKM_BF16");
    SKM_REQUIRE(d > 0 && d <= SKM_ROW_MAX_D, "d out of range");
    SKM_REQUIRE(grad_stride >= d && (!d_grad_weights || rows_stride >= d) && (!d_grad_rows || grad_rows_stride >= d),
                "strides must be at least d");
    SKM_REQUIRE(n < SKM_NO_ROW && n_rows < SKM_NO_ROW, "row counts must fit in 32 bits");
    SKM_REQUIRE(choices > 0 && choices <= SKM_ROUTE_MAX_CHOICES, "choices out of range");
    if (n == 0) return SKM_OK;
    SKM_REQUIRE(d_grad_rows || d_grad_weights, "no output asked for");
    SKM_REQUIRE(d_grad && d_slots && (d_rows || !d_grad_weights || n_rows == 0), "null pointer");
    const size_t size = type_size(type), weight_size = type_size(weights_type);
    SKM_REQUIRE(address(d_slots) % 4 == 0 && address(d_grad) % size == 0 && address(d_rows) % size == 0 &&
                address(d_grad_rows) % size == 0 && (!d_weights || address(d_weights) % weight_size == 0) &&
                (!d_grad_weights || address(d_grad_weights) % weight_size == 0), "pointers must be aligned to their elements");
    const Argument grad_rows{"grad_rows", matrix_memory(d_grad_rows, d_grad_rows ? n_rows : 0, grad_rows_stride, d, size)};
    const Argument grad_weights{"grad_weights", vector_memory(d_grad_weights, n * choices, weight_size)};
    const Argument grad{"grad", matrix_memory(d_grad, n, grad_stride, d, size)}, slots{"the slots", vector_memory(d_slots, n * choices, 4)};
    const Argument weights{"the weights", vector_memory(d_weights, n * choices, weight_size)};
    const Argument rows{"the rows", matrix_memory(d_rows, d_grad_weights ? n_rows : 0, rows_stride, d, size)};  // else not read
    SKM_TRY(check_apart(__func__, grad_rows, {grad, slots, weights, rows, grad_weights}));
    SKM_TRY(check_apart(__func__, grad_weights, {grad, slots, weights, rows}));
    OnDevice on(ctx);
    ScopedStage st(ctx, "rows/combine_grad");
    return for_type(type, [&](auto sample) {
        using T = decltype(sample);
        return for_elements<T>(vector_elements(size, size, d), [&](auto elements) {
            constexpr int E = decltype(elements)::value;
            const uint32_t vectors = (uint32_t) ((d + E - 1) / E);
            const auto launch = [&](auto waves, auto together) {
                constexpr int WAVES = decltype(waves)::value;
                constexpr size_t TOKENS = GRAD_THREADS<WAVES> / 64 / WAVES;
                const size_t turns = (n + TOKENS - 1) / TOKENS;
                const unsigned blocks = (unsigned) std::min<uint64_t>(ROWS_MAX_BLOCKS, turns);
                combine_rows_grad_kernel<T, E, WAVES, decltype(together)::value><<<blocks, GRAD_THREADS<WAVES>, 0, ctx->stream>>>(
                    (const T*) d_grad, n, vectors, (uint32_t) (d - E), grad_stride, (const T*) d_rows, n_rows, rows_stride, d_slots, (uint32_t) choices,
                    d_weights, weights_type, (T*) d_grad_rows, grad_rows_stride, d_grad_weights);
                return check_hip(hipGetLastError(), "combine_rows_grad_kernel launch");
            };
            const auto launch_waves = [&](auto waves) {
                if (choices <= 2) return launch(waves, std::integral_constant<int, 2>{});
                if (choices <= 4) return launch(waves, std::integral_constant<int, 4>{});
                return launch(waves, std::integral_constant<int, 8>{});
            };
            // few long rows: what a call takes is one walk over a row (9 rows of 3,968 over 6 choices 17 us with 4 wavefronts, 13 with
            // 16; 300 rows of 4,096 over 8 choices 23 and 26)
            if (vectors > 256 && n <= 64) return launch_waves(std::integral_constant<int, 16>{});
            if (vectors > 64) return launch_waves(std::integral_constant<int, 4>{});
            return launch_waves(std::integral_constant<int, 1>{});
        });
    });
}

} // extern "C"
