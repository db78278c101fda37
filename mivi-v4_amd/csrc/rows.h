// What the operators over rows of f32, f16 or bf16 tensors share ([rows]
// [heads][dim], the last dimension contiguous, strides in elements): host
// checks, and loads and stores of 8 elements at any element's address.
#pragma once

#include "common.h"

namespace mivi {

// --------------------------------------------------------------- host side
inline size_t type_bytes(int32_t t) {
    return t == MIVI_GGML_F32 ? 4 : t == MIVI_GGML_F16 || t == MIVI_GGML_BF16 ? 2 : 0;
}

// Elements from the first to the last of rows x heads x dim, or SIZE_MAX.
inline size_t span(size_t rows, size_t row_stride, size_t heads, size_t head_stride, size_t dim) {
    size_t a, b, c;
    if (__builtin_mul_overflow(rows - 1, row_stride, &a) || __builtin_mul_overflow(heads - 1, head_stride, &b) ||
        __builtin_add_overflow(a, b, &c) || __builtin_add_overflow(c, dim, &c) || c > (size_t)INT64_MAX / 8)
        return SIZE_MAX;
    return c;
}

inline int32_t check_tensor(const char* what, const void* p, size_t len, int32_t type, size_t rows, size_t row_stride,
                            size_t heads, size_t head_stride, size_t dim, bool written) {
    const size_t need = span(rows, row_stride, heads, head_stride, dim);
    if (need == SIZE_MAX) return err_overflow();
    if (len < need) return err_buffer_too_small(need, len);
    if (!p) return set_error(MIVI_ERR_INVALID_ARGUMENT, "null %s", what);
    if ((uintptr_t)p % type_bytes(type)) return set_error(MIVI_ERR_INVALID_ARGUMENT, "%s not aligned to its type", what);
    // rows and heads that are written must not overlap each other
    if (written && heads > 1 && head_stride < dim)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "%s: head stride %zu < head_dim %zu", what, head_stride, dim);
    if (written && rows > 1) {
        const bool rows_outer = row_stride >= (heads - 1) * head_stride + dim;
        const bool heads_outer = heads > 1 && row_stride >= dim && head_stride >= (rows - 1) * row_stride + dim;
        if (!rows_outer && !heads_outer)
            return set_error(MIVI_ERR_INVALID_ARGUMENT, "%s: rows of stride %zu overlap", what, row_stride);
    }
    return MIVI_OK;
}

// A tensor that is written over the one it is made from lies as that one does.
inline int32_t check_in_place(const char* what, const void* out, size_t out_row, size_t out_head, const void* in,
                              size_t in_row, size_t in_head, size_t rows, size_t heads) {
    if (out != in || !out) return MIVI_OK;
    if ((rows > 1 && out_row != in_row) || (heads > 1 && out_head != in_head))
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "%s in place has other strides", what);
    return MIVI_OK;
}

// A plain array of `need` elements of `elem` bytes.
inline int32_t check_array(const char* what, const void* p, size_t len, size_t need, size_t elem) {
    if (len < need) return err_buffer_too_small(need, len);
    if (need && !p) return set_error(MIVI_ERR_INVALID_ARGUMENT, "null %s", what);
    if ((uintptr_t)p % elem) return set_error(MIVI_ERR_INVALID_ARGUMENT, "%s not aligned to its type", what);
    return MIVI_OK;
}

// A launch counts the threads of a dimension in 32 bits.
inline bool grid_fits(size_t groups, size_t threads) { return groups <= UINT32_MAX / threads; }

}  // namespace mivi

// ------------------------------------------------------------- device side
// 16 and 8 bytes at any address: one load or store instruction on gfx950,
// whatever the alignment.
typedef uint32_t u32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));

template <int T>
constexpr int kElem = T == MIVI_GGML_F32 ? 4 : 2;

template <int T>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
    if constexpr (T == MIVI_GGML_F32) return ((const float*)p)[i];
    else if constexpr (T == MIVI_GGML_F16) return half_bits_to_f32(((const uint16_t*)p)[i]);
    else return bf16_bits_to_f32(((const uint16_t*)p)[i]);
}

template <int T>
__device__ __forceinline__ uint32_t elem_bits(float v) {
    if constexpr (T == MIVI_GGML_F16) return f32_to_half_bits(v);
    else return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v);
}

template <int T>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float v) {
    if constexpr (T == MIVI_GGML_F32) ((float*)p)[i] = v;
    else ((uint16_t*)p)[i] = (uint16_t)elem_bits<T>(v);
}

// n of 8 elements from element i on; the others are 0.
template <int T>
__device__ __forceinline__ void load_row8(const void* p, int64_t i, int n, float (&x)[8]) {
    if (n >= 8) {
        const uint8_t* at = (const uint8_t*)p + i * kElem<T>;
        const u32x4_a1 a = *(const u32x4_a1*)at;
        if constexpr (T == MIVI_GGML_F32) {
            const u32x4_a1 b = *(const u32x4_a1*)(at + 16);
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = __uint_as_float(a[e]), x[4 + e] = __uint_as_float(b[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t h = a[e / 2] >> (e % 2 * 16);
                x[e] = T == MIVI_GGML_F16 ? half_bits_to_f32(h) : bf16_bits_to_f32(h);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = e < n ? load_elem<T>(p, i + e) : 0.f;
    }
}

// n of 8 values to element i on.
template <int T>
__device__ __forceinline__ void store_row8(void* p, int64_t i, int n, const float (&x)[8]) {
    if (n >= 8) {
        uint8_t* at = (uint8_t*)p + i * kElem<T>;
        if constexpr (T == MIVI_GGML_F32) {
            u32x4_a1 a, b;
#pragma unroll
            for (int e = 0; e < 4; e++) a[e] = __float_as_uint(x[e]), b[e] = __float_as_uint(x[4 + e]);
            *(u32x4_a1*)at = a;
            *(u32x4_a1*)(at + 16) = b;
        } else {
            u32x4_a1 a;
#pragma unroll
            for (int e = 0; e < 4; e++) a[e] = elem_bits<T>(x[2 * e]) | elem_bits<T>(x[2 * e + 1]) << 16;
            *(u32x4_a1*)at = a;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n) store_elem<T>(p, i + e, x[e]);
    }
}
