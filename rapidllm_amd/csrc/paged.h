// paged.h -- what the kernels over a paged KV cache share (paged.hip, tree_attn.hip).
#pragma once

#include "internal.h"

namespace rl {

// The row types of the paged operators, and the cache type each goes with.
struct RowF32 {
    using T = float;
    using C = _Float16;
};
struct RowF16 {
    using T = _Float16;
    using C = _Float16;
};
struct RowBF16 {
    using T = __bf16;
    using C = __bf16;
};

template <class T>
struct Vec4 {
    typedef T type __attribute__((ext_vector_type(4)));
};
template <class T>
__device__ inline f32x4 load4(const T* p) {
    const auto v = *reinterpret_cast<const typename Vec4<T>::type*>(p);
    return f32x4{static_cast<float>(v[0]), static_cast<float>(v[1]), static_cast<float>(v[2]), static_cast<float>(v[3])};
}
// rounds to nearest even
template <class T>
__device__ inline void store4(T* p, f32x4 v) {
    typename Vec4<T>::type o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = static_cast<T>(v[i]);
    *reinterpret_cast<typename Vec4<T>::type*>(p) = o;
}

constexpr int64_t kMaxPositions = 1 << 30;  // of a table's row: sums of two stay in 32 bits

// A sequence of a step: rows r0 .. r0 + n - 1, context ctx.  Whatever the arrays hold, the rows
// stay within 0 .. rows and the positions within the table's capacity.
struct SeqSpan {
    int r0, n, ctx;
};
__device__ inline SeqSpan seq_span(const int* row_start, const int* ctx_lens, int b, int rows, int64_t capacity) {
    SeqSpan s;
    s.r0 = min(max(row_start[b], 0), rows);
    s.n = static_cast<int>(min(static_cast<int64_t>(min(max(row_start[b + 1], s.r0), rows) - s.r0), capacity));
    s.ctx = static_cast<int>(min(static_cast<int64_t>(max(ctx_lens[b], 0)), capacity - s.n));
    return s;
}

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Arguments that every paged operator checks: the cache's description and the row type.
inline void check_cache(const RlPagedCache* c, int layer, const char* what) {
    const std::string w(what);
    RL_REQUIRE(c && c->k && c->v, RL_ERR_RANGE, w + ": null cache");
    RL_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, RL_ERR_UNSUPPORTED,
               w + ": head_dim must be 64, 128 or 256");
    RL_REQUIRE(c->dtype == RL_Q_F16 || c->dtype == RL_Q_BF16, RL_ERR_UNSUPPORTED, w + ": the cache must be F16 or BF16");
    RL_REQUIRE(c->page_size >= 1 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0, RL_ERR_UNSUPPORTED,
               w + ": page_size must be a power of two up to 4096");
    RL_REQUIRE(c->n_pages >= 1 && c->n_kv >= 1 && c->n_kv <= 1024 && c->n_layers >= 1, RL_ERR_RANGE,
               w + ": bad cache sizes");
    RL_REQUIRE(layer >= 0 && layer < c->n_layers, RL_ERR_RANGE, w + ": no such layer");
    const int64_t dense = static_cast<int64_t>(c->n_pages) * c->n_kv * c->page_size * c->head_dim;
    RL_REQUIRE(c->n_layers == 1 || c->layer_stride >= dense, RL_ERR_RANGE, w + ": layers overlap");
    RL_REQUIRE(c->layer_stride % 8 == 0 && aligned(c->k, 16) && aligned(c->v, 16), RL_ERR_RANGE,
               w + ": cache must be 16-byte aligned");
}
inline void check_rows_type(const RlPagedCache* c, int dtype, const char* what) {
    RL_REQUIRE(dtype == c->dtype || (dtype == RL_Q_F32 && c->dtype == RL_Q_F16), RL_ERR_UNSUPPORTED,
               std::string(what) + ": rows must be F32 over an F16 cache, or of the cache's type");
}
inline size_t type_bytes(int dtype) { return dtype == RL_Q_F32 ? 4 : 2; }
inline void check_strided(const void* p, int64_t row, int64_t head, int dtype, const char* what) {
    RL_REQUIRE(aligned(p, 4 * type_bytes(dtype)) && row % 4 == 0 && head % 4 == 0, RL_ERR_RANGE,
               std::string(what) + ": rows and heads must start at multiples of four elements");
}

}  // namespace rl
