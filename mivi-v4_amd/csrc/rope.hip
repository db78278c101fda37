// Rotary positions: pairs (a, b) of a head's first rot dimensions turned by
// position times frequency,
//   a' = m (a cos t - b sin t),  b' = m (b cos t + a sin t),
// pairs (2 i, 2 i + 1) or (i, i + rot / 2); the dimensions behind them copied.
//
// Angles are taken in 64 bits and reduced to an eighth of a turn there: at
// position 10^6 a 32-bit product is off by 0.03 radians. The sine and cosine of
// what is left are Taylor polynomials in 32 bits (largest omitted term 2e-9).
//
// A wave has one row, so its position is found once (a search of `starts` by
// all lanes at once), and a lane 8 pairs of one head after another, so its
// angles are formed once for all of them. HBM bounds it: 35 K bf16 rows of 40 heads
// of 128, 96 of them turned, 191 us, 4.7 TB/s (301 with angles for every eight
// heads); eight rows of 40 heads of 64 take 4.6, three loads in a chain.
#include <math.h>

#include <algorithm>

#include "rows.h"

using namespace mivi;

namespace {

struct RopeArgs {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head;
    const double* freqs;
    const int32_t *positions, *starts, *lens;
    float scale;
    int rows, heads, kv, hd, rot, n_seq;
    int units, tail;    // 8-pair units of a head; units of 16 dimensions that are copied
    int per, parts;     // heads a wave takes at once; waves of a row
    int copy_q, copy_k; // whether the dimensions behind rot are copied
};

// Sequence of the wave's row, or -1: the last s with starts[s] <= row, if row is
// before starts[s + 1]. 64 boundaries a step.
__device__ __forceinline__ int wave_seq(const int32_t* starts, int n_seq, int row) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = n_seq;  // the sequence is in lo .. lo + n - 1
    while (n > 1) {
        const int step = (n + 63) / 64, at = lo + lane * step;
        // boundaries do not decrease: the lanes whose part starts at or before the row
        const uint64_t b = __ballot(lane * step < n && starts[min(at, n_seq)] <= row);
        const int c = max((int)__popcll(b) - 1, 0);
        n = min(step, n - c * step);
        lo += c * step;
    }
    return starts[lo] <= row && row < starts[lo + 1] ? lo : -1;
}

// Cosine and sine of t turns.
__device__ __forceinline__ void turn(double t, float* c, float* s) {
    const double k = rint(4 * t);
    const float x = (float)((t - 0.25 * k) * 6.283185307179586);  // at most pi / 4
    const float y = x * x;
    float sn = fmaf(y, 2.7557319e-6f, -1.9841270e-4f);
    sn = fmaf(y, sn, 8.3333333e-3f);
    sn = fmaf(y, sn, -0.16666667f);
    sn = fmaf(x * y, sn, x);
    float cs = fmaf(y, -2.7557319e-7f, 2.4801587e-5f);
    cs = fmaf(y, cs, -1.3888889e-3f);
    cs = fmaf(y, cs, 4.1666667e-2f);
    cs = fmaf(y, cs, -0.5f);
    cs = fmaf(y, cs, 1.0f);
    const int quarter = (int)(k - 4 * floor(0.25 * k));
    const bool odd = quarter & 1;
    const float a = odd ? sn : cs, b = odd ? cs : sn;
    *c = quarter == 1 || quarter == 2 ? -a : a;
    *s = quarter >= 2 ? -b : b;
}

template <int T, bool HALF>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    const int lane = threadIdx.x & 63;
    const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = (int)(wave / (uint32_t)a.parts), part = (int)(wave % (uint32_t)a.parts);
    if (row >= a.rows) return;
    int pos;
    if (a.positions) {
        pos = a.positions[row];
    } else {
        const int s = wave_seq(a.starts, a.n_seq, row);
        if (s < 0) return;
        pos = (int)((int64_t)a.lens[s] - a.starts[s + 1] + row);
    }
    const int per_head = a.units + a.tail, slot = lane / per_head, u = lane % per_head;
    if (slot >= a.per) return;
    const int half = a.rot / 2, n = min(8, half - u * 8);  // pairs of this lane's unit
    const bool turns = u < a.units;
    float c[8], s[8];
    if (turns) {
        const double turns_a_position = 0.15915494309189535 * pos;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            turn(turns_a_position * (e < n ? a.freqs[u * 8 + e] : 0.0), &c[e], &s[e]);
            c[e] *= a.scale, s[e] *= a.scale;
        }
    }
    // two runs of 8 elements a head: its firsts and seconds, or 16 neighbours with
    // the pairs side by side; of the dimensions behind rot 16 neighbours too
    const int i0 = turns ? HALF ? u * 8 : u * 16 : a.rot + (u - a.units) * 16;
    const int i1 = turns && HALF ? half + u * 8 : i0 + 8;
    const int n0 = turns ? HALF ? n : 2 * n : a.hd - i0, n1 = turns && HALF ? n : n0 - 8;
    const int all = a.heads + a.kv, step = a.parts * a.per;
    const auto at = [&](int h, const void** x, int64_t* xi, void** o, int64_t* oi) {
        const bool is_q = h < a.heads;
        const int hh = is_q ? h : h - a.heads;
        *x = is_q ? a.q : a.k, *o = is_q ? a.q_out : a.k_out;
        *xi = (int64_t)row * (is_q ? a.q_row : a.k_row) + hh * (is_q ? a.q_head : a.k_head);
        *oi = (int64_t)row * (is_q ? a.qo_row : a.ko_row) + hh * (is_q ? a.qo_head : a.ko_head);
        return h < all && (turns || (is_q ? a.copy_q : a.copy_k));
    };
    // two heads' loads before their stores
    for (int h = part * a.per + slot; h < all; h += 2 * step) {
        float v[2][2][8];
        void* o[2];
        int64_t oi[2];
        bool live[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const void* x;
            int64_t xi;
            live[j] = at(h + j * step, &x, &xi, &o[j], &oi[j]);
            if (live[j]) {
                load_row8<T>(x, xi + i0, n0, v[j][0]);
                load_row8<T>(x, xi + i1, n1, v[j][1]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (!live[j]) continue;
            if (turns) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float& p = HALF ? v[j][0][e] : v[j][e / 4][e % 4 * 2];
                    float& q = HALF ? v[j][1][e] : v[j][e / 4][e % 4 * 2 + 1];
                    const float y = fmaf(p, c[e], -(q * s[e]));
                    q = fmaf(q, c[e], p * s[e]);
                    p = y;
                }
            }
            store_row8<T>(o[j], oi[j] + i0, n0, v[j][0]);
            store_row8<T>(o[j], oi[j] + i1, n1, v[j][1]);
        }
    }
}

}  // namespace

extern "C" int32_t mivi_hip_rope(int32_t type, void* q_out, size_t q_out_len, size_t q_out_row_stride,
                                 size_t q_out_head_stride, const void* q, size_t q_len, size_t q_row_stride,
                                 size_t q_head_stride, size_t n_heads, void* k_out, size_t k_out_len,
                                 size_t k_out_row_stride, size_t k_out_head_stride, const void* k, size_t k_len,
                                 size_t k_row_stride, size_t k_head_stride, size_t n_kv_heads, size_t rows,
                                 size_t head_dim, size_t rot_dim, int32_t half_pairs, const void* freqs,
                                 size_t freqs_len, float scale, const int32_t* positions, size_t positions_len,
                                 const int32_t* starts, const int32_t* lens, size_t n_seq, void* stream) {
    if (!type_bytes(type)) return err_unsupported(type);
    if (n_heads + n_kv_heads == 0 || n_heads > 65535 || n_kv_heads > 65535)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "%zu heads and %zu kv heads", n_heads, n_kv_heads);
    if (head_dim == 0 || head_dim > 512)  // a head's units are lanes of one wave
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "heads of %zu dimensions (1 to 512)", head_dim);
    if (rot_dim % 2) return err_misaligned(rot_dim, 2);
    if (rot_dim == 0 || rot_dim > head_dim)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "%zu of %zu dimensions turned", rot_dim, head_dim);
    if (rows > (size_t)INT32_MAX || n_seq > (size_t)INT32_MAX - 4096) return err_overflow();
    int32_t rc = check_array("freqs", freqs, freqs_len, rot_dim / 2, 8);
    if (rc) return rc;
    if (positions ? starts || lens : !starts || (n_seq && !lens))
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "either positions, or starts and lens");
    if (positions && (rc = check_array("positions", positions, positions_len, rows, 4))) return rc;
    if ((uintptr_t)starts % 4 || (uintptr_t)lens % 4)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "starts or lens not 4-byte aligned");
    if (rows == 0 || (!positions && n_seq == 0)) return clear_error();
    if ((n_heads &&
         ((rc = check_tensor("q", q, q_len, type, rows, q_row_stride, n_heads, q_head_stride, head_dim, false)) ||
          (rc = check_tensor("q_out", q_out, q_out_len, type, rows, q_out_row_stride, n_heads, q_out_head_stride,
                             head_dim, true)))) ||
        (n_kv_heads &&
         ((rc = check_tensor("k", k, k_len, type, rows, k_row_stride, n_kv_heads, k_head_stride, head_dim, false)) ||
          (rc = check_tensor("k_out", k_out, k_out_len, type, rows, k_out_row_stride, n_kv_heads, k_out_head_stride,
                             head_dim, true)))))
        return rc;
    if ((rc = check_in_place("q", q_out, q_out_row_stride, q_out_head_stride, q, q_row_stride, q_head_stride, rows,
                             n_heads)) ||
        (rc = check_in_place("k", k_out, k_out_row_stride, k_out_head_stride, k, k_row_stride, k_head_stride, rows,
                             n_kv_heads)))
        return rc;
    if (n_heads && n_kv_heads && q_out == k_out)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "q_out and k_out are one tensor");
    RopeArgs a = {};
    a.q = q, a.k = k, a.q_out = q_out, a.k_out = k_out;
    a.q_row = (int64_t)q_row_stride, a.q_head = (int64_t)q_head_stride;
    a.k_row = (int64_t)k_row_stride, a.k_head = (int64_t)k_head_stride;
    a.qo_row = (int64_t)q_out_row_stride, a.qo_head = (int64_t)q_out_head_stride;
    a.ko_row = (int64_t)k_out_row_stride, a.ko_head = (int64_t)k_out_head_stride;
    a.freqs = (const double*)freqs, a.positions = positions, a.starts = starts, a.lens = lens, a.scale = scale;
    a.rows = (int)rows, a.heads = (int)n_heads, a.kv = (int)n_kv_heads, a.hd = (int)head_dim, a.rot = (int)rot_dim;
    a.n_seq = (int)n_seq;
    a.copy_q = q_out != q, a.copy_k = k_out != k;
    a.units = (int)((rot_dim / 2 + 7) / 8);
    a.tail = a.copy_q || a.copy_k ? (int)((head_dim - rot_dim + 15) / 16) : 0;
    a.per = 64 / (a.units + a.tail);
    // waves of a row: one for each time that its heads fill one, fewer where rows
    // alone are 16 a CU, so that angles serve several heads
    const size_t passes = (n_heads + n_kv_heads + a.per - 1) / a.per;
    a.parts = (int)std::min(passes, std::max<size_t>(1, 16 * (size_t)num_cus() / rows));
    size_t waves;
    if (__builtin_mul_overflow(rows, (size_t)a.parts, &waves) || !grid_fits((waves + 3) / 4, 256)) return err_overflow();
    clear_error();
    const unsigned grid = (unsigned)((waves + 3) / 4);
    hipStream_t s = (hipStream_t)stream;
#define ROPE(T)                                                      \
    if (half_pairs) rope_kernel<T, true><<<grid, 256, 0, s>>>(a);    \
    else rope_kernel<T, false><<<grid, 256, 0, s>>>(a)
    if (type == MIVI_GGML_F32) { ROPE(MIVI_GGML_F32); }
    else if (type == MIVI_GGML_F16) { ROPE(MIVI_GGML_F16); }
    else { ROPE(MIVI_GGML_BF16); }
#undef ROPE
    MIVI_HIP_CHECK(hipGetLastError());
    return MIVI_OK;
}

extern "C" int32_t mivi_hip_rope_frequencies(int32_t kind, float base, float factor, size_t context, size_t rot_dim,
                                             void* freqs, size_t freqs_len) {
    if (kind < MIVI_ROPE_PLAIN || kind > MIVI_ROPE_MODEL)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "no frequencies of kind %d", kind);
    if (!(base > 1.f && base <= 3.402823466e38f))
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "base %g (more than 1)", (double)base);
    if (!(factor > 0.f && factor <= 3.402823466e38f))
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "factor %g (more than 0)", (double)factor);
    if ((kind == MIVI_ROPE_YARN || kind == MIVI_ROPE_MODEL) && context == 0)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "no trained context");
    if (rot_dim == 0 || rot_dim % 2) return err_misaligned(rot_dim, 2);
    const int32_t rc = check_array("freqs", freqs, freqs_len, rot_dim / 2, 8);
    if (rc) return rc;
    clear_error();
    const double turn = 6.283185307179586, d = (double)rot_dim, f = factor > 1.f ? (double)factor : 1.0;
    double b = (double)base;
    if (kind == MIVI_ROPE_BASE && rot_dim > 2) b *= pow(f, d / (d - 2));
    // the pair that turns n times over the trained context
    const auto pair = [&](double n) { return d * log((double)context / (n * turn)) / (2 * log(b)); };
    for (size_t i = 0; i < rot_dim / 2; i++) {
        const double plain = pow(b, -(double)(2 * i) / d);
        double far = 0;  // how much of it is divided
        if (kind == MIVI_ROPE_LINEAR) {
            far = 1;
        } else if (kind == MIVI_ROPE_YARN) {
            const double lo = std::max(floor(pair(32)), 0.0), hi = std::min(ceil(pair(1)), d - 1);
            far = ((double)i - lo) / std::max(hi - lo, 1e-3);
        } else if (kind == MIVI_ROPE_MODEL) {
            const double lo = (double)context / 32, hi = (double)context;
            far = (turn / plain - lo) / (hi - lo);
        }
        far = std::min(std::max(far, 0.0), 1.0);
        ((double*)freqs)[i] = plain * (1 - far) + plain / f * far;
    }
    return MIVI_OK;
}
