// Root-mean-square norm of rows, with the residual's addition before it, into
// the rows' type or into 8-bit codes with scales.
//
//   s = x + r,   f = (mean s^2 + eps)^(-1/2),   out = s f w
//   8 bits: in a group with A = max |s w|, code = rint(127 s w / A) (ties to
//   even), scale = A f / 127.
//
// A code does not depend on f: A f / 127 is taken out of (s f w) / (A f / 127)
// by hand, so codes follow from the inputs alone, whatever order f's sum was
// taken in. They are formed in 64 bits (the card's vector rate for them is that
// of 32 bits), where s w is exact or next to it, and only a quotient within
// 1e-9 of a half is divided out, which decides every tie.
//
// Squares are summed in 64 bits: no finite row overflows.
//
// One pass: a row's elements stay in registers between the sum and the store,
// 8 a chunk, E chunks a thread; rows longer than 32768 (16384 for 8 bits, whose
// 64-bit products take twice the registers) are read twice.
#include <algorithm>

#include "rows.h"

using namespace mivi;

namespace {

struct NormArgs {
    const void *x, *r;  // r: null without a residual
    void *ro, *out;     // ro: null where the sum is not kept
    const float* w;
    int8_t* codes;
    float* scales;
    int64_t x_row, x_head, r_row, r_head, ro_row, ro_head, o_row, o_head;
    double eps, inv_dim;
    uint32_t n_rows, heads;  // n_rows: rows times heads
    int dim, group;          // group: a row's dimensions where it has one scale
    int lanes, waves;        // of a row: waves, or (waves 0) lanes of one, a power of two
};

// ------------------------------------------------- 64-bit reductions of lanes
template <bool MAX>
__device__ __forceinline__ double op2(double a, double b) { return MAX ? fmax(a, b) : a + b; }

__device__ __forceinline__ double join2(float lo, float hi) {
    return __hiloint2double((int)__float_as_uint(hi), (int)__float_as_uint(lo));
}

template <bool MAX, int O>
__device__ __forceinline__ double fold(double v) {
    const float lo = __uint_as_float((uint32_t)__double2loint(v)), hi = __uint_as_float((uint32_t)__double2hiint(v));
    if constexpr (O >= 16) {
        float l0, l1, h0, h1;
        if constexpr (O == 16) swap16(lo, l0, l1), swap16(hi, h0, h1);
        else swap32(lo, l0, l1), swap32(hi, h0, h1);
        return op2<MAX>(join2(l0, h0), join2(l1, h1));
    } else if constexpr (O == 4) {
        return op2<MAX>(v, join2(xor4_mov(lo), xor4_mov(hi)));
    } else {
        constexpr int ctrl = O == 8 ? 0x128 : O == 2 ? 0x4E : 0xB1;
        return op2<MAX>(v, join2(dpp_mov<ctrl>(lo), dpp_mov<ctrl>(hi)));
    }
}

// Over groups of `lanes` neighbouring lanes, a power of two, in all of them.
template <bool MAX>
__device__ __forceinline__ double fold_lanes(double v, int lanes) {
    if (lanes > 1) v = fold<MAX, 1>(v);
    if (lanes > 2) v = fold<MAX, 2>(v);
    if (lanes > 4) v = fold<MAX, 4>(v);
    if (lanes > 8) v = fold<MAX, 8>(v);
    if (lanes > 16) v = fold<MAX, 16>(v);
    if (lanes > 32) v = fold<MAX, 32>(v);
    return v;
}

// Over the workgroup: its waves' sums through `part`.
template <bool MAX>
__device__ __forceinline__ double fold_row(double v, const NormArgs& a, double* part) {
    v = fold_lanes<MAX>(v, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < a.waves; i++) v = op2<MAX>(v, part[i]);
    return v;
}

// The instructions' 1 / sqrt x and 1 / x (2^-24) with a Newton step: 2^-46, in six
// instructions where the library's take forty to eighty.
__device__ __forceinline__ double inv_sqrt(double m) {
    const double y = __builtin_amdgcn_rsq(m);
    return m > 1.7976931348623157e308 ? 0.0 : y * fma(-0.5 * m, y * y, 1.5);
}
__device__ __forceinline__ double inverse(double x) {
    const double y = __builtin_amdgcn_rcp(x);
    return fma(fma(-x, y, 1.0), y, y);
}

// --------------------------------------------------------------- the kernels
// s of n elements (up to 8) from i on; where `keep`, written to ro too.
template <int T, class F>
__device__ __forceinline__ void load_sum(const NormArgs& a, int64_t xo, int64_t ro, int64_t i, int n, F (&s)[8]) {
    float x[8];
    load_row8<T>(a.x, xo + i, n, x);
    if (a.r) {
        float r[8];
        load_row8<T>(a.r, ro + i, n, r);
#pragma unroll
        for (int e = 0; e < 8; e++) s[e] = (F)x[e] + (F)r[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) s[e] = x[e];
    }
}

template <int T, class F>
__device__ __forceinline__ void keep_sum(const NormArgs& a, int64_t off, int n, const F (&s)[8]) {
    if (!a.ro) return;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = (float)s[e];
    store_row8<T>(a.ro, off, n, y);
}

__device__ __forceinline__ double largest(double m, const double (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) m = fmax(m, v[e] != v[e] ? (double)__builtin_inff() : fabs(v[e]));
    return m;
}

// Codes of 8 values of a group whose largest magnitude is top; nothing that
// stands for a value where top or the row's sum is not finite.
__device__ __forceinline__ void store_codes(int8_t* at, int n, const double (&v)[8], double top, bool ok) {
    const double inv = top > 0 ? 127 * inverse(top) : 0.0;
    int c[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const double q = v[e] * inv;
        double k = rint(q);
        if (fabs(fabs(q - k) - 0.5) < 1e-9) k = rint(127 * v[e] / top);
        c[e] = ok ? (int)k : 0;
    }
    if (n >= 8) {
        u32x2_a1 w;
#pragma unroll
        for (int h = 0; h < 2; h++)
            w[h] = (uint32_t)(c[4 * h] & 0xFF) | (uint32_t)(c[4 * h + 1] & 0xFF) << 8 |
                   (uint32_t)(c[4 * h + 2] & 0xFF) << 16 | (uint32_t)c[4 * h + 3] << 24;
        *(u32x2_a1*)at = w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n) at[e] = (int8_t)c[e];
    }
}

// E chunks of 8 elements a thread, held between the sum and the store; E = 0:
// any number, read again. HBM bounds it: 16384 bf16 rows of 8192 with the residual
// and its sum 184 us, 5.8 TB/s (a copy reaches 5.1); 2048 f32 rows of 2048 into 8
// bits 13.2 us, 4.5 TB/s, vector instructions half of the cycles; eight such rows
// 4.2, a chain of two loads, sum, largest value and store.
template <int T, int E, bool Q8>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs a) {
    typedef typename std::conditional<Q8, double, float>::type F;
    constexpr bool HOLD = E > 0;
    __shared__ double part[2][16];
    const int tid = threadIdx.x;
    const int t = tid, dim = a.dim;
    const uint32_t row = blockIdx.x, r0 = row / a.heads, h0 = row - r0 * a.heads;
    const int64_t xo = r0 * a.x_row + h0 * a.x_head, rr = r0 * a.r_row + h0 * a.r_head;
    const int64_t ko = r0 * a.ro_row + h0 * a.ro_head, oo = r0 * a.o_row + h0 * a.o_head;
    const int tpr = 64 * a.waves;
    const int steps = HOLD ? E : (a.dim + 8 * tpr - 1) / (8 * tpr);

    F s[HOLD ? E : 1][8];
    float w[HOLD ? E : 1][8];
    double sum = 0, top = 0;
#pragma unroll
    for (int e = 0; e < (HOLD ? E : 1); e++) {
        if constexpr (HOLD) {
            const int i = (t + e * tpr) * 8, n = dim - i;
            if (n > 0) {
                load_sum<T>(a, xo, rr, i, n, s[e]);
                load_row8<MIVI_GGML_F32>(a.w, i, n, w[e]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) s[e][j] = 0, w[e][j] = 0.f;
            }
        }
    }
    for (int e = 0; e < steps; e++) {
        F(&v)[8] = s[HOLD ? e : 0];
        const int i = (t + e * tpr) * 8, n = dim - i;
        if constexpr (!HOLD) {
            if (n <= 0) continue;
            load_sum<T>(a, xo, rr, i, n, v);
            if (Q8) load_row8<MIVI_GGML_F32>(a.w, i, n, w[0]);
        } else if (n > 0) {
            keep_sum<T>(a, ko + i, n, v);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) sum = fma((double)v[j], (double)v[j], sum);
        if constexpr (Q8) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] *= w[HOLD ? e : 0][j];
            if (a.group == a.dim) top = largest(top, v);
        }
    }
    sum = fold_row<false>(sum, a, part[0]);
    const double f = inv_sqrt(fma(sum, a.inv_dim, a.eps));
    const bool ok = sum <= 1.7976931348623157e308;
    if constexpr (Q8) {
        if (a.group == a.dim) top = fold_row<true>(top, a, part[1]);
    }
    const float f32 = (float)f;
    const int ng = Q8 ? a.dim / a.group : 0;
    for (int e = 0; e < steps; e++) {
        F(&v)[8] = s[HOLD ? e : 0];
        const int i = (t + e * tpr) * 8, n = dim - i;
        if constexpr (!HOLD) {
            if (n > 0) {
                load_sum<T>(a, xo, rr, i, n, v);
                load_row8<MIVI_GGML_F32>(a.w, i, n, w[0]);
                keep_sum<T>(a, ko + i, n, v);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = 0, w[0][j] = 0.f;
            }
            if constexpr (Q8) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] *= w[0][j];
            }
        }
        if constexpr (Q8) {
            if (a.group != a.dim) top = fold_lanes<true>(largest(0, v), a.group / 8);
            const bool fine = ok && top <= 1.7976931348623157e308;
            if (n > 0) {
                store_codes(a.codes + (int64_t)row * a.dim + i, n, v, top, fine);
                if (i % a.group == 0)
                    a.scales[(int64_t)row * ng + i / a.group] = fine ? (float)(top * f * (1.0 / 127)) : __builtin_nanf("");
            }
        } else if (n > 0) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = v[j] * f32 * w[HOLD ? e : 0][j];
            store_row8<T>(a.out, oo + i, n, y);
        }
    }
}

// Rows of up to 512 elements, 8 a lane: R rows for every group of lanes, all
// their loads first. 131168 fp16 rows of 64: 8.9 us, 3.8 TB/s, vector instructions
// 62 % of the cycles (one row a group 9.6).
template <int T, int R, bool Q8>
__global__ __launch_bounds__(256) void norm_short_kernel(NormArgs a) {
    typedef typename std::conditional<Q8, double, float>::type F;
    const int t = threadIdx.x & (a.lanes - 1), i = t * 8;
    const uint32_t groups = gridDim.x * 256 / a.lanes, first = (blockIdx.x * 256 + threadIdx.x) / a.lanes;
    F s[R][8];
    int n[R];
    int64_t ko[R], oo[R];
#pragma unroll
    for (int e = 0; e < R; e++) {
        const uint32_t row = first + e * groups;
        const bool live = row < a.n_rows;  // lanes behind the last row take part with no elements
        const uint32_t r = live ? row / a.heads : 0, h = live ? row - r * a.heads : 0;
        n[e] = live ? a.dim - i : 0;
        ko[e] = r * a.ro_row + h * a.ro_head + i, oo[e] = r * a.o_row + h * a.o_head + i;
        load_sum<T>(a, r * a.x_row + h * a.x_head, r * a.r_row + h * a.r_head, i, n[e], s[e]);
    }
    float w[8];
    load_row8<MIVI_GGML_F32>(a.w, i, a.dim - i, w);
#pragma unroll
    for (int e = 0; e < R; e++) {
        if (n[e] > 0) keep_sum<T>(a, ko[e], n[e], s[e]);
        double sum = 0, top = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) sum = fma((double)s[e][j], (double)s[e][j], sum);
        sum = fold_lanes<false>(sum, a.lanes);
        const double f = inv_sqrt(fma(sum, a.inv_dim, a.eps));
        if constexpr (Q8) {
#pragma unroll
            for (int j = 0; j < 8; j++) s[e][j] *= w[j];
            top = fold_lanes<true>(largest(0, s[e]), a.group == a.dim ? a.lanes : a.group / 8);
            const bool fine = sum <= 1.7976931348623157e308 && top <= 1.7976931348623157e308;
            if (n[e] > 0) {
                const int64_t row = first + e * groups;
                store_codes(a.codes + row * a.dim + i, n[e], s[e], top, fine);
                if (i % a.group == 0)
                    a.scales[row * (a.dim / a.group) + i / a.group] =
                        fine ? (float)(top * f * (1.0 / 127)) : __builtin_nanf("");
            }
        } else if (n[e] > 0) {
            const float f32 = (float)f;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = s[e][j] * f32 * w[j];
            store_row8<T>(a.out, oo[e], n[e], y);
        }
    }
}

template <int T, bool Q8>
void launch_norm(const NormArgs& a, int e, unsigned grid, unsigned threads, hipStream_t s) {
    if (a.waves == 0) {
        if (e == 1) norm_short_kernel<T, 1, Q8><<<grid, threads, 0, s>>>(a);
        else norm_short_kernel<T, 4, Q8><<<grid, threads, 0, s>>>(a);
        return;
    }
    switch (e) {
        case 1: norm_kernel<T, 1, Q8><<<grid, threads, 0, s>>>(a); break;
        case 2: norm_kernel<T, 2, Q8><<<grid, threads, 0, s>>>(a); break;
        case 4:
            if constexpr (!Q8) {
                norm_kernel<T, 4, Q8><<<grid, threads, 0, s>>>(a);
                break;
            }
        default: norm_kernel<T, 0, Q8><<<grid, threads, 0, s>>>(a); break;
    }
}

// Lays the rows out and launches: rows of up to 512 elements on the fewest
// lanes that take 8 each, four rows a group where that leaves 8 waves a CU;
// longer ones on as many waves as take E chunks a thread.
int32_t run_norm(NormArgs a, int32_t type, bool q8, size_t rows, size_t heads, size_t dim, hipStream_t s) {
    const size_t n_rows = rows * heads, chunks = (dim + 7) / 8;
    size_t grid, threads = 256;
    int e = 1;
    a.n_rows = (uint32_t)n_rows, a.heads = (uint32_t)heads, a.dim = (int)dim;
    a.inv_dim = 1.0 / (double)dim;
    a.lanes = 64, a.waves = 0;
    if (chunks <= 64) {
        a.lanes = 1;
        while ((size_t)a.lanes < chunks) a.lanes *= 2;
        if (n_rows * a.lanes >= 4 * 8 * 64 * (size_t)num_cus()) e = 4;
        grid = (n_rows * a.lanes + 256 * e - 1) / (256 * e);
    } else {
        e = chunks <= 1024 ? 1 : chunks <= 2048 ? 2 : chunks <= 4096 && !q8 ? 4 : 0;
        a.waves = (int)std::min<size_t>(16, e ? ((chunks + e - 1) / e + 63) / 64 : 16);
        grid = n_rows, threads = 64 * a.waves;
    }
    if (!grid_fits(grid, threads)) return err_overflow();
    clear_error();
#define NORM(T) (q8 ? launch_norm<T, true>(a, e, (unsigned)grid, (unsigned)threads, s) \
                    : launch_norm<T, false>(a, e, (unsigned)grid, (unsigned)threads, s))
    if (type == MIVI_GGML_F32) NORM(MIVI_GGML_F32);
    else if (type == MIVI_GGML_F16) NORM(MIVI_GGML_F16);
    else NORM(MIVI_GGML_BF16);
#undef NORM
    MIVI_HIP_CHECK(hipGetLastError());
    return MIVI_OK;
}

// What both entry points check: sizes, x, the residual and its sum, the weights.
int32_t check_norm(NormArgs* a, int32_t type, size_t rows, size_t heads, size_t dim, const float* weight,
                   size_t weight_len, float eps) {
    if (!type_bytes(type)) return err_unsupported(type);
    size_t all;
    if (dim == 0 || heads == 0)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "%zu heads of %zu dimensions", heads, dim);
    if (dim > (size_t)INT32_MAX / 2 || __builtin_mul_overflow(rows, heads, &all) || all > (size_t)INT32_MAX)
        return err_overflow();
    if (!(eps >= 1e-30f && eps <= 3.402823466e38f))
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "eps %g (1e-30 or more)", (double)eps);
    const int32_t rc = check_array("weight", weight, weight_len, dim, 4);
    if (rc) return rc;
    *a = {};
    a->w = weight, a->eps = (double)eps;
    return MIVI_OK;
}

}  // namespace

extern "C" int32_t mivi_hip_rms_norm(int32_t type, void* out, size_t out_len, size_t out_row_stride,
                                     size_t out_head_stride, const void* x, size_t x_len, size_t x_row_stride,
                                     size_t x_head_stride, const void* residual, size_t residual_len,
                                     size_t residual_row_stride, size_t residual_head_stride, void* sum,
                                     size_t sum_len, size_t sum_row_stride, size_t sum_head_stride,
                                     const float* weight, size_t weight_len, float eps, size_t rows, size_t heads,
                                     size_t dim, void* stream) {
    NormArgs a;
    int32_t rc = check_norm(&a, type, rows, heads, dim, weight, weight_len, eps);
    if (rc) return rc;
    if (rows == 0) return clear_error();
    if ((rc = check_tensor("x", x, x_len, type, rows, x_row_stride, heads, x_head_stride, dim, false)) ||
        (rc = check_tensor("out", out, out_len, type, rows, out_row_stride, heads, out_head_stride, dim, true)) ||
        (residual && (rc = check_tensor("residual", residual, residual_len, type, rows, residual_row_stride, heads,
                                        residual_head_stride, dim, false))) ||
        (sum && (rc = check_tensor("sum", sum, sum_len, type, rows, sum_row_stride, heads, sum_head_stride, dim, true))))
        return rc;
    for (const void* w : {(const void*)out, (const void*)sum}) {
        const size_t wr = w == out ? out_row_stride : sum_row_stride, wh = w == out ? out_head_stride : sum_head_stride;
        if ((rc = check_in_place("x", w, wr, wh, x, x_row_stride, x_head_stride, rows, heads)) ||
            (rc = check_in_place("residual", w, wr, wh, residual, residual_row_stride, residual_head_stride, rows, heads)))
            return rc;
    }
    if (out == sum) return set_error(MIVI_ERR_INVALID_ARGUMENT, "out and sum are one tensor");
    a.x = x, a.x_row = (int64_t)x_row_stride, a.x_head = (int64_t)x_head_stride;
    a.r = residual, a.r_row = (int64_t)residual_row_stride, a.r_head = (int64_t)residual_head_stride;
    a.ro = sum, a.ro_row = (int64_t)sum_row_stride, a.ro_head = (int64_t)sum_head_stride;
    a.out = out, a.o_row = (int64_t)out_row_stride, a.o_head = (int64_t)out_head_stride;
    return run_norm(a, type, false, rows, heads, dim, (hipStream_t)stream);
}

extern "C" int32_t mivi_hip_rms_norm_q8(int32_t type, uint8_t* codes, size_t codes_len, float* scales,
                                        size_t scales_len, size_t group, const void* x, size_t x_len,
                                        size_t x_row_stride, const void* residual, size_t residual_len,
                                        size_t residual_row_stride, void* sum, size_t sum_len,
                                        size_t sum_row_stride, const float* weight, size_t weight_len, float eps,
                                        size_t rows, size_t dim, void* stream) {
    NormArgs a;
    int32_t rc = check_norm(&a, type, rows, 1, dim, weight, weight_len, eps);
    if (rc) return rc;
    if (group != 0 && group != 32 && group != 64 && group != 128 && group != 256 && group != 512)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "groups of %zu (32, 64, 128, 256, 512, or 0 for whole rows)", group);
    if (group && dim % group) return err_misaligned(dim, group);
    if (rows == 0) return clear_error();
    size_t all;
    if (__builtin_mul_overflow(rows, dim, &all) || all > (size_t)INT64_MAX / 8) return err_overflow();
    if ((rc = check_array("codes", codes, codes_len, all, 1)) ||
        (rc = check_array("scales", scales, scales_len, group ? all / group : rows, 4)) ||
        (rc = check_tensor("x", x, x_len, type, rows, x_row_stride, 1, 0, dim, false)) ||
        (residual && (rc = check_tensor("residual", residual, residual_len, type, rows, residual_row_stride, 1, 0, dim,
                                        false))) ||
        (sum && (rc = check_tensor("sum", sum, sum_len, type, rows, sum_row_stride, 1, 0, dim, true))))
        return rc;
    if ((rc = check_in_place("x", sum, sum_row_stride, 0, x, x_row_stride, 0, rows, 1)) ||
        (rc = check_in_place("residual", sum, sum_row_stride, 0, residual, residual_row_stride, 0, rows, 1)))
        return rc;
    a.x = x, a.x_row = (int64_t)x_row_stride;
    a.r = residual, a.r_row = (int64_t)residual_row_stride;
    a.ro = sum, a.ro_row = (int64_t)sum_row_stride;
    a.codes = (int8_t*)codes, a.scales = scales, a.group = (int)(group ? group : dim);
    return run_norm(a, type, true, rows, 1, dim, (hipStream_t)stream);
}
