// Products with 4-bit weights that have a scale (and a zero) for each group of
// columns of a row: out[b][n] = sum_k x[b][k] (c[n][k] - z) s, z = 8 without
// zeros; x in f32, f16 or bf16, or as 8-bit codes with scales.
//
// On the matrix cores, whatever the batch: c - z is a small integer and enters
// them exactly, as fp16 (x in fp16), bf16 (x in bf16; x in f32 as three bf16
// parts, 24 bits, that take three columns of the product) or int8 (8-bit x),
// 32 columns a product; a group's sum is multiplied by its scale in f32 (8-bit
// x: an exact integer by the product of both scales). Scaling the weights first
// would round every one of them.
//
// Packed layout (mivi_hip_w4_pack), tiles of 16 rows, steps of 128 columns,
// padded with codes and scales of 0:
//   codes   [tile][step][lane 64][16 bytes]: lane r + 16 q holds of row r the
//           columns 32 j + 8 q .. + 7 of the step in dword j, column 2 p at
//           nibble p and 2 p + 1 at nibble 4 + p: the operand of product j, one
//           contiguous KB a wave;
//   scales  [tile][step][q][unit][4] of rows 4 q .. + 3 (16 bits): those that
//           lane r + 16 q multiplies its results by. A unit is a group of 32 or
//           64 columns, or the step where groups have 128 or more;
//   zeros   [tile][step][row][unit] bytes, where there are zeros.
//
// A workgroup has 8 waves: wk of them share a tile's steps, 8 / wk tiles. x goes
// through LDS in operand order, [32 columns][q][column of the product].
#include <algorithm>

#include "rows.h"

using namespace mivi;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32_a1 __attribute__((aligned(1)));

constexpr int kWaves = 8;
constexpr int kStep = 128;   // columns of a step
constexpr int kRing = 4;     // steps of a wave in flight
constexpr size_t kLds = 64 * 1024;

enum XKind { X_F16, X_BF16, X_F32, X_I8 };
constexpr int parts_of(int x) { return x == X_F32 ? 3 : 1; }

struct W4Args {
    const uint8_t *codes, *scales, *zeros;  // planes of the packed weights; zeros: or null
    const void* x;
    const float* x_scales;
    void* out;
    int64_t x_row, out_row;
    int rows, cols, batch, tiles, steps;
    int block;      // inputs of a workgroup
    int wk;         // waves of a tile
    int phase;      // steps of x in LDS: all, or a multiple of wk times kRing
    int w_units;    // units of a step that have a scale of their own
    int x_shift, x_groups;  // 8-bit x: log2 of a scale's columns, scales of a row; -1, 1: a row has one
    int bf16_scales, out_type;
};

__device__ __forceinline__ float scale_f32(uint32_t bits, bool bf16) {
    return bf16 ? bf16_bits_to_f32(bits) : half_bits_to_f32(bits);
}

// Eight weights c - z of a dword, in the order of the columns.
__device__ __forceinline__ half8 weights_f16(uint32_t w, uint32_t z) {
    // a nibble in the low bits of 1024 is 1024 + c, in the next four 1024 + 16 c
    const half2v lo = __builtin_bit_cast(half2v, 0x64006400u | z << 16 | z);                 // 1024 + z
    const half2v hi = __builtin_bit_cast(half2v, 0xD400D400u | z << 20 | z << 4);            // -(64 + z)
    const half2v sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    union { half8 v; half2v h[4]; } r;
    const uint32_t w8 = w >> 8;
    r.h[0] = __builtin_bit_cast(half2v, (w & 0x000F000Fu) | 0x64006400u) - lo;
    r.h[1] = __builtin_elementwise_fma(__builtin_bit_cast(half2v, (w & 0x00F000F0u) | 0x64006400u), sixteenth, hi);
    r.h[2] = __builtin_bit_cast(half2v, (w8 & 0x000F000Fu) | 0x64006400u) - lo;
    r.h[3] = __builtin_elementwise_fma(__builtin_bit_cast(half2v, (w8 & 0x00F000F0u) | 0x64006400u), sixteenth, hi);
    return r.v;
}
__device__ __forceinline__ bf16x8 weights_bf16(uint32_t w, float z) {
    const uint32_t even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;
    union { bf16x8 v; uint32_t u[4]; } r;
#pragma unroll
    for (int p = 0; p < 4; p++) {  // integers up to 15: the upper halves of the floats are exact
        const uint32_t pairs = p % 2 ? odd : even;  // columns 2 p and 2 p + 1: bytes p / 2 and 2 + p / 2
        const uint32_t a = __float_as_uint(ubyte_f32(pairs, p / 2) - z);
        const uint32_t b = __float_as_uint(ubyte_f32(pairs, 2 + p / 2) - z);
        r.u[p] = __builtin_amdgcn_perm(b, a, 0x07060302);
    }
    return r.v;
}
// In the order 0 4 1 5 2 6 3 7 of the columns, in which x is laid out too.
__device__ __forceinline__ long weights_i8(uint32_t w, uint32_t zzzz) {
    const uint32_t even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;
    // bytes 128 + c - z borrow nothing from each other
    const uint32_t a = ((even | 0x80808080u) - zzzz) ^ 0x80808080u, b = ((odd | 0x80808080u) - zzzz) ^ 0x80808080u;
    return (long)((uint64_t)b << 32 | a);
}

// x of `count` inputs and the phase's columns to LDS.
template <int X, int U>
__device__ __forceinline__ void stage(const W4Args& a, uint8_t* lds, int b0, int count, int cols_x, int k0, int kn) {
    const int n8 = kn / 8;
    if constexpr (X == X_I8) {  // and the scales of a step's sums, behind the codes
        if (a.x_shift >= 0) {
            float* xs = (float*)(lds + a.phase * 16 * cols_x * 8);
            const int n = kn / kStep * U;
            for (int i = threadIdx.x; i < count * n; i += kWaves * 64) {
                const int b = i / n, u = i % n, k = min(k0 + u * (kStep / U), a.cols - 1);
                xs[u * cols_x + b] = a.x_scales[(int64_t)(b0 + b) * a.x_groups + (k >> a.x_shift)];
            }
        }
    }
    for (int i = threadIdx.x; i < count * n8; i += kWaves * 64) {
        const int b = i / n8, c = i % n8, k = k0 + c * 8;
        const int64_t at = (int64_t)(b0 + b) * a.x_row + k;
        const bool in = k < a.cols;
        if constexpr (X == X_I8) {
            u32x2 v = {0, 0};
            if (in) v = *(const u32x2_a1*)((const int8_t*)a.x + at);
            *(u32x2*)(lds + ((int64_t)c * cols_x + b) * 8) =
                u32x2{__builtin_amdgcn_perm(v.y, v.x, 0x05010400), __builtin_amdgcn_perm(v.y, v.x, 0x07030602)};
        } else if constexpr (X == X_F32) {
            float v[8];
            load_row8<MIVI_GGML_F32>(a.x, at, in ? 8 : 0, v);
            bf16x8 p[3];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                __bf16 p0, p1, p2;
                split_bf16(v[e], p0, p1, p2);
                p[0][e] = p0, p[1][e] = p1, p[2][e] = p2;
            }
#pragma unroll
            for (int j = 0; j < 3; j++) *(bf16x8*)(lds + ((int64_t)c * cols_x + 3 * b + j) * 16) = p[j];
        } else {
            u32x4 v = {0, 0, 0, 0};
            if (in) v = *(const u32x4_a1*)((const uint16_t*)a.x + at);
            *(u32x4*)(lds + ((int64_t)c * cols_x + b) * 16) = v;
        }
    }
}

// U: sums of a step that are scaled by themselves; NT: tiles of 16 columns.
template <int X, int U, int NT>
__global__ __launch_bounds__(kWaves * 64) void w4_kernel(W4Args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int XB = X == X_I8 ? 8 : 16, PARTS = parts_of(X), PER = 4 / U;
    typedef typename std::conditional<X == X_I8, i32x4, f32x4>::type D;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wk = wave % a.wk, wm = wave / a.wk;
    const int wms = kWaves / a.wk, tile = blockIdx.x * wms + wm;
    const bool live = tile < a.tiles;
    const int b0 = blockIdx.y * a.block, count = min(a.block, a.batch - b0), cols_x = count * PARTS;
    int col[NT];  // columns behind the last repeat it: their results are not used
#pragma unroll
    for (int n = 0; n < NT; n++) col[n] = min(16 * n + r, cols_x - 1);
    const float* xs = (const float*)(lds + a.phase * 16 * cols_x * 8);
    const int64_t first = (int64_t)(live ? tile : 0) * a.steps;
    const int mine = live ? max(0, (a.steps - wk + a.wk - 1) / a.wk) : 0;  // steps of this wave

    u32x4 codes[kRing];
    u32x2 sc[kRing][U];
    uint32_t zc[kRing][U];
    const auto fetch = [&](int slot, int i) {
        const int64_t st = first + wk + i * a.wk;
        codes[slot] = *(const u32x4*)(a.codes + st * 1024 + lane * 16);
        const uint8_t* s = a.scales + (st * 4 + q) * a.w_units * 8;
#pragma unroll
        for (int u = 0; u < U; u++) sc[slot][u] = *(const u32x2*)(s + u * a.w_units / U * 8);
        const uint8_t* z = a.zeros + (st * 16 + r) * a.w_units;
#pragma unroll
        for (int u = 0; u < U; u++) zc[slot][u] = a.zeros ? z[u * a.w_units / U] & 15 : 8;
    };
    f32x4 acc[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) acc[n] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int p = 0; p < kRing; p++)
        if (p < mine) fetch(p, p);

    const auto compute = [&](int slot, int local) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            D d[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) d[n] = D{0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < PER; p++) {
                const int j = u * PER + p;
                const uint8_t* xl = lds + (local * 16 + j * 4 + q) * cols_x * XB;
                const uint32_t w = codes[slot][j], z = zc[slot][u];
                if constexpr (X == X_F16) {
                    const half8 wv = weights_f16(w, z);
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        d[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wv, *(const half8*)(xl + col[n] * XB), d[n], 0, 0, 0);
                } else if constexpr (X == X_I8) {
                    const long wv = weights_i8(w, z * 0x01010101u);
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        d[n] = __builtin_amdgcn_mfma_i32_16x16x32_i8(wv, *(const long*)(xl + col[n] * XB), d[n], 0, 0, 0);
                } else {
                    const bf16x8 wv = weights_bf16(w, (float)z);
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        d[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, *(const bf16x8*)(xl + col[n] * XB), d[n], 0, 0, 0);
                }
            }
            const u32x2 s = sc[slot][u];
            const float f[4] = {scale_f32(s.x & 0xFFFF, a.bf16_scales), scale_f32(s.x >> 16, a.bf16_scales),
                                scale_f32(s.y & 0xFFFF, a.bf16_scales), scale_f32(s.y >> 16, a.bf16_scales)};
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float m = 1.f;
                if constexpr (X == X_I8) {
                    if (a.x_shift >= 0) m = xs[(local * U + u) * cols_x + col[n]];
                }
#pragma unroll
                for (int i = 0; i < 4; i++) acc[n][i] = fmaf((float)d[n][i], X == X_I8 ? f[i] * m : f[i], acc[n][i]);
            }
        }
    };

    const int per_phase = a.phase / a.wk;
    for (int ph = 0; ph * a.phase < a.steps; ph++) {
        if (ph) __syncthreads();
        stage<X, U>(a, lds, b0, count, cols_x, ph * a.phase * kStep, min(a.phase, a.steps - ph * a.phase) * kStep);
        __syncthreads();
        const int end = min(mine, (ph + 1) * per_phase);
        for (int i = ph * per_phase; i < end; i += kRing) {
#pragma unroll
            for (int p = 0; p < kRing; p++) {
                if (i + p < end) {
                    compute(p, wk + (i + p) * a.wk - ph * a.phase);
                    if (i + p + kRing < mine) fetch(p, i + p + kRing);
                }
            }
        }
    }

    // join the waves of a tile and the parts of an input
    __syncthreads();
    float* red = (float*)lds;
#pragma unroll
    for (int n = 0; n < NT; n++) *(f32x4*)(red + ((wave * NT + n) * 16 + r) * 16 + q * 4) = acc[n];
    __syncthreads();
    for (int i = tid; i < wms * count * 16; i += kWaves * 64) {
        const int m = i & 15, b = (i >> 4) % count, w = (i >> 4) / count;
        const int row = (blockIdx.x * wms + w) * 16 + m;
        if (row >= a.rows) continue;
        float v = 0;
        for (int p = PARTS - 1; p >= 0; p--)
            for (int k = 0; k < a.wk; k++) v += red[((w * a.wk + k) * NT * 16 + b * PARTS + p) * 16 + m];
        if constexpr (X == X_I8) {
            if (a.x_shift < 0) v *= a.x_scales[b0 + b];
        }
        const int64_t o = (int64_t)(b0 + b) * a.out_row + row;
        if (a.out_type == MIVI_GGML_F32) store_elem<MIVI_GGML_F32>(a.out, o, v);
        else if (a.out_type == MIVI_GGML_F16) store_elem<MIVI_GGML_F16>(a.out, o, v);
        else store_elem<MIVI_GGML_BF16>(a.out, o, v);
    }
}

// ------------------------------------------------------------------ packing
__global__ __launch_bounds__(256) void w4_pack_codes_kernel(const uint8_t* codes, uint8_t* dst, int rows, int cols,
                                                            int steps, int64_t cells) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // a lane's 16 bytes
    if (i >= cells * 64) return;
    const int lane = i & 63, r = lane & 15, q = lane >> 4;
    const int64_t tile = (i >> 6) / steps, step = (i >> 6) % steps;
    const int64_t row = tile * 16 + r;
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int k = (int)step * kStep + 32 * j + 8 * q;
        uint32_t w = 0;
        if (row < rows && k < cols) w = *(const u32_a1*)(codes + row * (cols / 2) + k / 2);
        uint32_t o = 0;
#pragma unroll
        for (int p = 0; p < 4; p++) o |= (w >> (8 * p) & 15) << (4 * p) | (w >> (8 * p + 4) & 15) << (16 + 4 * p);
        v[j] = o;
    }
    *(u32x4*)(dst + i * 16) = v;
}

__global__ __launch_bounds__(256) void w4_pack_scales_kernel(const uint16_t* scales, const uint8_t* zeros,
                                                             uint16_t* s_dst, uint8_t* z_dst, int rows, int cols,
                                                             int group, int steps, int units, int64_t cells) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // a row's unit
    if (i >= cells * 16 * units) return;
    const int u = (int)(i % units), r = (int)(i / units % 16);
    const int64_t cell = i / units / 16, row = cell / steps * 16 + r;
    const int k = (int)(cell % steps) * kStep + u * (kStep / units);
    const bool in = row < rows && k < cols;
    const int64_t at = row * (cols / group) + k / group;
    s_dst[((cell * 4 + r / 4) * units + u) * 4 + r % 4] = in ? scales[at] : 0;
    if (zeros) z_dst[i] = in ? zeros[at] & 15 : 0;
}

// --------------------------------------------------------------- host side
struct Packed {
    size_t tiles, steps, units, codes, scales, zeros;  // the planes' bytes
    size_t bytes() const { return codes + scales + zeros; }
};

// Sizes of packed weights, or an error.
int32_t packed_of(size_t rows, size_t cols, size_t group, bool zeros, Packed* p) {
    if (rows == 0 || cols == 0) return set_error(MIVI_ERR_INVALID_ARGUMENT, "%zu x %zu weights", rows, cols);
    if (cols % 32) return err_misaligned(cols, 32);
    if (group != 32 && group != 64 && group != cols && (group == 0 || group % kStep))
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "groups of %zu (32, 64, a multiple of 128 or the whole row)", group);
    if (cols % group) return err_misaligned(cols, group);
    if (rows > (size_t)INT32_MAX - 15 || cols > (size_t)INT32_MAX / 8) return err_overflow();
    p->tiles = (rows + 15) / 16, p->steps = (cols + kStep - 1) / kStep;
    p->units = group == 32 ? 4 : group == 64 ? 2 : 1;
    size_t cells, all;
    if (__builtin_mul_overflow(p->tiles, p->steps, &cells) || __builtin_mul_overflow(cells, (size_t)2048, &all) ||
        all > (size_t)INT64_MAX / 8)
        return err_overflow();
    p->codes = cells * 1024, p->scales = cells * 32 * p->units, p->zeros = zeros ? cells * 16 * p->units : 0;
    return MIVI_OK;
}

template <int X, int U, int NT>
void launch_w4(const W4Args& a, dim3 grid, size_t lds, hipStream_t s) {
    w4_kernel<X, U, NT><<<grid, kWaves * 64, lds, s>>>(a);
}
template <int X, int U>
void launch_w4(const W4Args& a, int nt, dim3 grid, size_t lds, hipStream_t s) {
    if (nt == 1) launch_w4<X, U, 1>(a, grid, lds, s);
    else if (nt == 2) launch_w4<X, U, 2>(a, grid, lds, s);
    else launch_w4<X, U, 4>(a, grid, lds, s);
}
template <int X>
void launch_w4(const W4Args& a, int units, int nt, dim3 grid, size_t lds, hipStream_t s) {
    if (units == 1) launch_w4<X, 1>(a, nt, grid, lds, s);
    else if (units == 2) launch_w4<X, 2>(a, nt, grid, lds, s);
    else launch_w4<X, 4>(a, nt, grid, lds, s);
}

// The part that both products share: x is laid out in `a` already.
int32_t run_w4(W4Args a, int x, int32_t type, void* out, size_t out_len, size_t out_row_stride, const uint8_t* packed,
               size_t packed_len, int32_t scale_type, bool zeros, size_t batch, size_t rows, size_t cols, size_t group,
               int x_units, hipStream_t s) {
    Packed p;
    int32_t rc = packed_of(rows, cols, group, zeros, &p);
    if (rc) return rc;
    if (scale_type != MIVI_GGML_F16 && scale_type != MIVI_GGML_BF16) return err_unsupported(scale_type);
    if (batch > (size_t)INT32_MAX) return err_overflow();
    if ((rc = check_array("packed", packed, packed_len, p.bytes(), 1)) ||
        (batch && (rc = check_tensor("out", out, out_len, type, batch, out_row_stride, 1, 0, rows, true))))
        return rc;
    if ((uintptr_t)packed % 16) return set_error(MIVI_ERR_INVALID_ARGUMENT, "packed not 16-byte aligned");
    if (batch == 0) return clear_error();
    const int parts = parts_of(x), xb = x == X_I8 ? 8 : 16;
    const size_t all = batch * parts;
    const int nt = all <= 16 ? 1 : all <= 32 ? 2 : 4;
    const size_t block = std::min<size_t>(batch, 16 * nt / parts), blocks = (batch + block - 1) / block;
    const int units = std::max((int)p.units, x_units);
    const size_t step_bytes = block * parts * (16 * xb + (x == X_I8 ? 4 * units : 0));
    // waves of a tile: as many as keep 16 a CU busy, and as x's columns allow
    a.wk = 8;
    while (a.wk > 1 && p.tiles * a.wk > 16 * (size_t)num_cus()) a.wk /= 2;
    size_t phase = (p.steps + a.wk - 1) / a.wk * a.wk;
    if (phase * step_bytes > kLds) {
        while (a.wk > 1 && a.wk * kRing * step_bytes > kLds) a.wk /= 2;
        phase = kLds / (a.wk * kRing * step_bytes) * a.wk * kRing;
    }
    a.phase = (int)phase;
    const size_t wms = kWaves / a.wk, grid_x = (p.tiles + wms - 1) / wms;
    const size_t lds = std::max<size_t>(a.phase * step_bytes, (size_t)kWaves * nt * 1024);
    if (!grid_fits(grid_x, kWaves * 64) || blocks > 65535) return err_overflow();
    clear_error();
    a.codes = packed, a.scales = packed + p.codes, a.zeros = zeros ? packed + p.codes + p.scales : nullptr;
    a.out = out, a.out_row = (int64_t)out_row_stride, a.out_type = type;
    a.rows = (int)rows, a.cols = (int)cols, a.batch = (int)batch;
    a.tiles = (int)p.tiles, a.steps = (int)p.steps, a.block = (int)block;
    a.w_units = (int)p.units, a.bf16_scales = scale_type == MIVI_GGML_BF16;
    const dim3 grid((unsigned)grid_x, (unsigned)blocks);
    switch (x) {
        case X_F16: launch_w4<X_F16>(a, units, nt, grid, lds, s); break;
        case X_BF16: launch_w4<X_BF16>(a, units, nt, grid, lds, s); break;
        case X_F32: launch_w4<X_F32>(a, units, nt, grid, lds, s); break;
        default: launch_w4<X_I8>(a, units, nt, grid, lds, s); break;
    }
    MIVI_HIP_CHECK(hipGetLastError());
    return MIVI_OK;
}

}  // namespace

extern "C" size_t mivi_hip_w4_packed_size(size_t rows, size_t cols, size_t group, int32_t has_zeros) {
    Packed p;
    if (packed_of(rows, cols, group, has_zeros != 0, &p)) return 0;
    return p.bytes();
}

extern "C" int32_t mivi_hip_w4_pack(const uint8_t* codes, size_t codes_len, int32_t scale_type, const void* scales,
                                    size_t scales_len, const uint8_t* zeros, size_t zeros_len, uint8_t* packed,
                                    size_t packed_len, size_t rows, size_t cols, size_t group, void* stream) {
    Packed p;
    int32_t rc = packed_of(rows, cols, group, zeros != nullptr, &p);
    if (rc) return rc;
    if (scale_type != MIVI_GGML_F16 && scale_type != MIVI_GGML_BF16) return err_unsupported(scale_type);
    if ((rc = check_array("codes", codes, codes_len, rows * (cols / 2), 1)) ||
        (rc = check_array("scales", scales, scales_len, rows * (cols / group), 2)) ||
        (zeros && (rc = check_array("zeros", zeros, zeros_len, rows * (cols / group), 1))) ||
        (rc = check_array("packed", packed, packed_len, p.bytes(), 1)))
        return rc;
    if ((uintptr_t)packed % 16) return set_error(MIVI_ERR_INVALID_ARGUMENT, "packed not 16-byte aligned");
    const size_t cells = p.tiles * p.steps, grid = (cells * 64 + 255) / 256;
    if (!grid_fits(grid, 256)) return err_overflow();
    clear_error();
    hipStream_t s = (hipStream_t)stream;
    w4_pack_codes_kernel<<<(unsigned)grid, 256, 0, s>>>(codes, packed, (int)rows, (int)cols, (int)p.steps,
                                                        (int64_t)cells);
    MIVI_HIP_CHECK(hipGetLastError());
    w4_pack_scales_kernel<<<(unsigned)((cells * 16 * p.units + 255) / 256), 256, 0, s>>>(
        (const uint16_t*)scales, zeros, (uint16_t*)(packed + p.codes), packed + p.codes + p.scales, (int)rows,
        (int)cols, (int)group, (int)p.steps, (int)p.units, (int64_t)cells);
    MIVI_HIP_CHECK(hipGetLastError());
    return MIVI_OK;
}

extern "C" int32_t mivi_hip_w4_matmul_rows(int32_t type, void* out, size_t out_len, size_t out_row_stride,
                                           const uint8_t* packed, size_t packed_len, int32_t scale_type,
                                           int32_t has_zeros, const void* x, size_t x_len, size_t x_row_stride,
                                           size_t batch, size_t rows, size_t cols, size_t group, void* stream) {
    if (!type_bytes(type)) return err_unsupported(type);
    int32_t rc;
    if (batch && (rc = check_tensor("x", x, x_len, type, batch, x_row_stride, 1, 0, cols, false))) return rc;
    W4Args a = {};
    a.x = x, a.x_row = (int64_t)x_row_stride;
    return run_w4(a, type == MIVI_GGML_F32 ? X_F32 : type == MIVI_GGML_F16 ? X_F16 : X_BF16, type, out, out_len,
                  out_row_stride, packed, packed_len, scale_type, has_zeros != 0, batch, rows, cols, group, 1,
                  (hipStream_t)stream);
}

extern "C" int32_t mivi_hip_w4_matmul_rows_q8(int32_t type, void* out, size_t out_len, size_t out_row_stride,
                                              const uint8_t* packed, size_t packed_len, int32_t scale_type,
                                              int32_t has_zeros, const uint8_t* codes, size_t codes_len,
                                              const float* scales, size_t scales_len, size_t x_group, size_t batch,
                                              size_t rows, size_t cols, size_t group, void* stream) {
    if (!type_bytes(type)) return err_unsupported(type);
    if (x_group != 0 && x_group != 32 && x_group != 64 && x_group != 128 && x_group != 256 && x_group != 512)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "groups of %zu (32, 64, 128, 256, 512, or 0 for whole rows)", x_group);
    if (x_group && cols % x_group) return err_misaligned(cols, x_group);
    size_t all;
    if (__builtin_mul_overflow(batch, cols, &all) || all > (size_t)INT64_MAX / 8) return err_overflow();
    int32_t rc;
    if ((rc = check_array("codes", codes, codes_len, all, 1)) ||
        (rc = check_array("scales", scales, scales_len, x_group ? all / x_group : batch, 4)))
        return rc;
    W4Args a = {};
    a.x = codes, a.x_row = (int64_t)cols;
    a.x_scales = scales, a.x_groups = (int)(x_group ? cols / x_group : 1);
    a.x_shift = x_group ? __builtin_ctzll(x_group) : -1;
    return run_w4(a, X_I8, type, out, out_len, out_row_stride, packed, packed_len, scale_type, has_zeros != 0, batch,
                  rows, cols, group, x_group == 32 ? 4 : x_group == 64 ? 2 : 1, (hipStream_t)stream);
}
