// What the operators on rows of typed device tensors share: element types, vectors of them, the split of rows over
// wavefronts, and the checks of their entry points.
#pragma once

#include "skm_internal.h"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace skm {

template <class T, int N>
using vec_of = T __attribute__((ext_vector_type(N)));

// Sums are held in fp32; a result is rounded once, to nearest even, when it is stored.
template <int N, class T>
__device__ __forceinline__ vec_of<float, N> widen(const vec_of<T, N> v) {
    return __builtin_convertvector(v, vec_of<float, N>);
}
template <class T, int N>
__device__ __forceinline__ vec_of<T, N> narrow(const vec_of<float, N> v) {
    return __builtin_convertvector(v, vec_of<T, N>);
}

// Vectors of up to 16 bytes at any element: the memory instructions take them unaligned too, only the compiler has to be told.
// (Against narrower aligned accesses, 16,384 rows of 1,001 16-bit elements are quantised in 15 us instead of 26.)
template <class T, int N>
using loose_vec __attribute__((aligned(sizeof(T)))) = vec_of<T, N>;

// Results that are wider than their inputs take two stores.
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const vec_of<T, N> v) {
    if constexpr (sizeof(T) * N <= 16) {
        *reinterpret_cast<loose_vec<T, N>*>(p) = v;
    } else {
        constexpr int H = N / 2;
        vec_of<T, H> lo, hi;
#pragma unroll
        for (int i = 0; i < H; ++i) lo[i] = v[i], hi[i] = v[H + i];
        store_vec<T, H>(p, lo);
        store_vec<T, H>(p + H, hi);
    }
}
// Loads and stores of what a kernel touches once: they leave more of the memory's rate to the rest (a million rows of 4 KiB
// looked up 901 -> 790 us, 16,384 rows added up over 8 rows each 89 -> 77 us).
template <class T, int N>
__device__ __forceinline__ void store_vec_once(T* p, const vec_of<T, N> v) {
    if constexpr (sizeof(T) * N <= 16) {
        __builtin_nontemporal_store(v, reinterpret_cast<loose_vec<T, N>*>(p));
    } else {
        constexpr int H = N / 2;
        vec_of<T, H> lo, hi;
#pragma unroll
        for (int i = 0; i < H; ++i) lo[i] = v[i], hi[i] = v[H + i];
        store_vec_once<T, H>(p, lo);
        store_vec_once<T, H>(p + H, hi);
    }
}
template <class T, int N>
__device__ __forceinline__ vec_of<T, N> load_vec_once(const T* p) {
    static_assert(sizeof(T) * N <= 16, "one load");
    return __builtin_nontemporal_load(reinterpret_cast<const loose_vec<T, N>*>(p));
}
template <class T, int N>
__device__ __forceinline__ vec_of<T, N> load_vec(const T* p) {
    if constexpr (sizeof(T) * N <= 16) {
        return *reinterpret_cast<const loose_vec<T, N>*>(p);
    } else {
        constexpr int H = N / 2;
        const vec_of<T, H> lo = load_vec<T, H>(p), hi = load_vec<T, H>(p + H);
        vec_of<T, N> v;
#pragma unroll
        for (int i = 0; i < H; ++i) v[i] = lo[i], v[H + i] = hi[i];
        return v;
    }
}

inline size_t type_size(const int type) { return type == SKM_F32 ? 4 : 2; }
inline bool is_value_type(const int type) { return type == SKM_F32 || type == SKM_F16 || type == SKM_BF16; }

inline size_t address(const void* p) { return reinterpret_cast<size_t>(p); }

// The memory of an argument: `rows` pieces of `width` bytes, `pitch` bytes from one to the next (no less than the width).
struct Memory {
    size_t at, rows, pitch, width;
    size_t length() const { return rows ? (rows - 1) * pitch + width : 0; }
};
inline Memory matrix_memory(const void* p, const size_t rows, const size_t stride, const size_t d, const size_t size) {
    if (!p || rows == 0) return {0, 0, 0, 0};
    size_t last;
    // a distance that no address space has: all of it
    if (__builtin_mul_overflow(stride, size, &last) || __builtin_mul_overflow(rows, last, &last) || last > SIZE_MAX - address(p))
        return {0, 1, SIZE_MAX, SIZE_MAX};
    if (stride == d) return {address(p), 1, rows * d * size, rows * d * size};
    return {address(p), rows, stride * size, d * size};
}
inline Memory vector_memory(const void* p, const size_t n, const size_t size) { return matrix_memory(p, n, 1, 1, size); }

// Whether the ranges of two arguments meet, from the first byte to the last: where both have rows of one pitch, as views of
// columns of one buffer do, whether their rows meet.
inline bool meet(const Memory& a, const Memory& b) {
    if (a.rows == 0 || b.rows == 0) return false;
    if (a.at >= b.at + b.length() || b.at >= a.at + a.length()) return false;
    if (a.pitch != b.pitch) return true;
    const size_t past = b.at >= a.at ? (b.at - a.at) % a.pitch : (a.pitch - (a.at - b.at) % a.pitch) % a.pitch;
    return past < a.width || past + b.width > a.pitch;
}

struct Argument {
    const char* name;
    Memory memory;
};
// SKM_ERR_INVALID where an output shares memory with an argument that is read, or with another output.
inline int check_apart(const char* who, const Argument& out, const std::initializer_list<Argument> others) {
    for (const Argument& other : others)
        if (meet(out.memory, other.memory)) return set_error(SKM_ERR_INVALID, "%s: %s overlaps %s", who, out.name, other.name);
    return SKM_OK;
}

// The calling thread's device is the context's while an entry point launches, and what it was afterwards (the default
// stream, which a context may be made on, belongs to the current device).
class OnDevice {
  public:
    explicit OnDevice(const skm_ctx* ctx) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = ctx->device;
        if (before_ != ctx->device) switched_ = hipSetDevice(ctx->device) == hipSuccess;
    }
    ~OnDevice() {
        if (switched_) (void) hipSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;

  private:
    int before_ = 0;
    bool switched_ = false;
};

// Scratch of a call: the caller's block, or the context's workspace where none is given.  The workspace may grow, which
// allocates and waits, and two graphs captured on one context would share it: under capture the caller brings the block.
int call_scratch(skm_ctx* ctx, const char* who, void* given, size_t given_bytes, size_t need, void** out);

// Elements of a vector for rows of d: as many as 16 bytes of the wider type hold, fewer for rows that are shorter than that.
// `whole`: vectors must not overlap.
inline size_t vector_elements(const size_t size, const size_t other_size, const size_t d, const bool whole = false) {
    size_t e = 16 / std::max(size, other_size);
    while (whole ? d % e != 0 : d < e) e /= 2;
    return e;
}

// How rows are handed out.  A wavefront takes `lanes` lanes per row (a power of two) and so 64 / lanes rows at a time; a
// row of more than lanes * UNROLL vectors is cut into pieces that different wavefronts take.  Where the vector's elements do not
// divide the row, its last vector begins earlier and repeats elements of the one before: what is stored twice is the same.
struct RowSplit {
    uint32_t vectors;  // vectors per row
    uint32_t last;     // column of the last one
    uint32_t lanes;
    uint32_t pieces;   // pieces per row
    uint64_t units;    // wavefronts' worth of work: groups of 64 / lanes rows times pieces
};
// Column of the at-th vector.
template <int E>
__device__ __forceinline__ uint32_t column(const uint32_t at, const uint32_t last) {
    return min(at * E, last);
}
inline RowSplit split_rows(const size_t n, const size_t d, const size_t elements, const uint32_t unroll) {
    RowSplit s;
    const size_t vectors = (d + elements - 1) / elements;
    s.vectors = (uint32_t) vectors;
    s.last = (uint32_t) (d - elements);
    s.lanes = 1;
    while (s.lanes < 64 && (size_t) s.lanes * unroll < vectors) s.lanes *= 2;
    const size_t per_piece = (size_t) s.lanes * unroll;
    s.pieces = (uint32_t) ((vectors + per_piece - 1) / per_piece);
    const size_t rows_per_wave = 64 / s.lanes;
    s.units = (uint64_t) ((n + rows_per_wave - 1) / rows_per_wave) * s.pieces;
    return s;
}
constexpr int ROWS_THREADS = 256;
constexpr uint64_t ROWS_MAX_BLOCKS = uint64_t(1) << 22;  // of a launch; beyond that a wavefront takes several units
inline unsigned row_blocks(const RowSplit& s) {
    const uint64_t per_block = ROWS_THREADS / 64;
    return (unsigned) std::max<uint64_t>(1, std::min(ROWS_MAX_BLOCKS, (s.units + per_block - 1) / per_block));
}

// A launch has fewer than 2^32 threads in a dimension, so more workgroups than ROWS_MAX_BLOCKS go in several launches: calls
// launch(number of the first workgroup, workgroups).  Blocks fit in 32 bits.
template <class F>
int launch_in_parts(const uint64_t blocks, F&& launch) {
    for (uint64_t first = 0; first < blocks; first += ROWS_MAX_BLOCKS)
        SKM_TRY(launch((uint32_t) first, (unsigned) std::min(ROWS_MAX_BLOCKS, blocks - first)));
    return SKM_OK;
}

// Calls f with a value of the element type, and with the elements of a vector, that a call asks for.
template <class F>
int for_type(const int type, F&& f) {
    if (type == SKM_F32) return f(float{});
    if (type == SKM_F16) return f(_Float16{});
    return f(__bf16{});
}
template <class T, class F>
int for_elements(const size_t elements, F&& f) {
    if constexpr (sizeof(T) == 2)
        if (elements == 8) return f(std::integral_constant<int, 8>{});
    if (elements == 4) return f(std::integral_constant<int, 4>{});
    if (elements == 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

} // namespace skm
