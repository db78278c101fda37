// Products with 4-bit weights that have a scale (and a zero) for each group of
// columns of a row: out[b][n] = sum_k x[b][k] (c[n][k] - z) s, z = 8 without
// zeros; x in f32, f16 or bf16, or as 8-bit codes with scales.
//
// On the matrix cores, whatever the batch: c - z is a small integer and enters
// them exactly, as fp16 (x in fp16, and in f32 as two fp16 parts, which take two
// columns of the product), bf16 or int8 (8-bit x), 32 columns a product; a group's
// sum is multiplied by its scale in f32 (8-bit x: an exact integer by the weights'
// scale, then by the input's). Scaling the weights first would round every one of them.
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
// A workgroup has 8 or 16 waves: wk of them share a tile's steps. x goes through
// LDS in operand order.
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
constexpr int kRing = 3;     // steps of a wave in flight (w4_rows_kernel)
constexpr size_t kLds = 128 * 1024, kLdsFew = 156 * 1024;
// inputs of a launch: in blocks of 8, the smallest, 2^15 of the 65535 that a grid's
// second dimension may have
constexpr size_t kMostInputs = (size_t)1 << 18;

enum XKind { X_F16, X_BF16, X_F32, X_I8 };
constexpr int parts_of(int x) { return x == X_F32 ? 2 : 1; }  // columns of the product that an input takes
// pieces of x a thread of w4_rows_kernel stages at most
constexpr int items_of(int x, int waves) { return (waves == 8 ? 8 : 5) / parts_of(x); }

struct W4Args {
    const uint8_t *codes, *scales, *zeros;  // planes of the packed weights (zeros: the codes where there are none)
    const void* x;
    const float* x_scales;
    void* out;
    int64_t x_row, out_row;
    int rows, cols, batch, tiles, steps;
    int block;      // inputs of a workgroup
    int wk;         // waves of a tile
    int x_shift, x_groups;  // 8-bit x: log2 of a scale's columns, scales of a row; -1, 1: a row has one
    int bf16_scales, has_zeros, out_type;
};

// A scale's four rows of a unit, as the factors of a lane's four results.
__device__ __forceinline__ void scales_f32(u32x2 s, bool bf16, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t bits = s[i / 2] >> (i % 2 * 16);
        const float a = half_bits_to_f32(bits), b = bf16_bits_to_f32(bits);
        f[i] = bf16 ? b : a;
    }
}

// (w & mask) | bits in one instruction, which takes one scalar and no literal: the
// compiler makes two of it, with literals.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(bits));
    return r;
}

// Eight weights c - z of a dword, in the order of the columns.
__device__ __forceinline__ half8 weights_f16(uint32_t w, uint32_t z) {
    // a nibble in the low bits of 1024 is 1024 + c, in the next four 1024 + 16 c
    const half2v lo = __builtin_bit_cast(half2v, 0x64006400u | z << 16 | z);                 // 1024 + z
    const half2v hi = __builtin_bit_cast(half2v, 0xD400D400u | z << 20 | z << 4);            // -(64 + z)
    const half2v sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    union { half8 v; half2v h[4]; } r;
    const uint32_t w8 = w >> 8, k = 0x64006400u;
    r.h[0] = __builtin_bit_cast(half2v, and_or(w, 0x000F000Fu, k)) - lo;
    r.h[1] = __builtin_elementwise_fma(__builtin_bit_cast(half2v, and_or(w, 0x00F000F0u, k)), sixteenth, hi);
    r.h[2] = __builtin_bit_cast(half2v, and_or(w8, 0x000F000Fu, k)) - lo;
    r.h[3] = __builtin_elementwise_fma(__builtin_bit_cast(half2v, and_or(w8, 0x00F000F0u, k)), sixteenth, hi);
    return r.v;
}
// Byte K of w as a float; the compiler takes a nibble out first, two instructions.
template <int K>
__device__ __forceinline__ float byte_f32(uint32_t w) {
    float f;
    if constexpr (K == 0) asm("v_cvt_f32_ubyte0 %0, %1" : "=v"(f) : "v"(w));
    else if constexpr (K == 1) asm("v_cvt_f32_ubyte1 %0, %1" : "=v"(f) : "v"(w));
    else if constexpr (K == 2) asm("v_cvt_f32_ubyte2 %0, %1" : "=v"(f) : "v"(w));
    else asm("v_cvt_f32_ubyte3 %0, %1" : "=v"(f) : "v"(w));
    return f;
}
__device__ __forceinline__ bf16x8 weights_bf16(uint32_t w, float z) {
    const uint32_t even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;
    union { bf16x8 v; uint32_t u[4]; } r;
    // columns 2 p and 2 p + 1 are bytes p / 2 and 2 + p / 2 of even or odd;
    // integers up to 15: the upper halves of the floats are exact
    const auto pair = [&](float a, float b) {
        return __builtin_amdgcn_perm(__float_as_uint(b - z), __float_as_uint(a - z), 0x07060302);
    };
    r.u[0] = pair(byte_f32<0>(even), byte_f32<2>(even));
    r.u[1] = pair(byte_f32<0>(odd), byte_f32<2>(odd));
    r.u[2] = pair(byte_f32<1>(even), byte_f32<3>(even));
    r.u[3] = pair(byte_f32<1>(odd), byte_f32<3>(odd));
    return r.v;
}
// In the order 0 4 1 5 2 6 3 7 of the columns, in which x is laid out too.
__device__ __forceinline__ long weights_i8(uint32_t w, uint32_t zzzz) {
    const uint32_t even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;
    // bytes 128 + c - z borrow nothing from each other
    const uint32_t a = ((even | 0x80808080u) - zzzz) ^ 0x80808080u, b = ((odd | 0x80808080u) - zzzz) ^ 0x80808080u;
    return (long)((uint64_t)b << 32 | a);
}

// What a lane holds of a step: a row's codes, the scales of its results' rows,
// and zeros: where ROW of its own row (a byte a unit), else of those of its
// results (bytes [row 4 q + i][unit]).
template <int W, bool ROW>
struct Step {
    u32x4 codes;
    u32x2 scales[W];
    uint32_t zeros[ROW ? 1 : W];
};

// Loads without a branch: of weights without zeros the codes stand in for them.
template <int W, bool ROW>
__device__ __forceinline__ void fetch(const W4Args& a, int64_t st, int lane, Step<W, ROW>* o) {
    o->codes = *(const u32x4*)(a.codes + st * 1024 + lane * 16);
    const int q = lane >> 4;
    const uint8_t* s = a.scales + st * (32 * W) + q * (8 * W);
    if constexpr (W == 1) {
        o->scales[0] = *(const u32x2*)s;
    } else {
#pragma unroll
        for (int u = 0; u < W; u += 2) {
            const u32x4 v = *(const u32x4*)(s + u * 8);
            o->scales[u] = u32x2{v.x, v.y}, o->scales[u + 1] = u32x2{v.z, v.w};
        }
    }
    const uint8_t* z = a.zeros + st * (16 * W);
    if constexpr (ROW) {
        const int r = lane & 15;
        uint32_t v;
        if constexpr (W == 4) v = ((const uint32_t*)z)[r];
        else if constexpr (W == 2) v = ((const uint16_t*)z)[r];
        else v = z[r];
        o->zeros[0] = a.has_zeros ? v : 0x08080808u;
    } else {
#pragma unroll
        for (int u = 0; u < W; u++) {
            const uint32_t v = ((const uint32_t*)(z + q * (4 * W)))[u];
            o->zeros[u] = a.has_zeros ? v : 0x08080808u;
        }
    }
}

// An operand of x: 8 columns of one input, 16 bytes or 8.
template <int X>
struct Operand { u32x4 v; };
template <>
struct Operand<X_I8> { u32x2 v; };

// A dword's weights as an operand, and a product of 16 rows and 16 columns, 32
// deep.
template <int X>
struct Weights8 {
    u32x4 v;
    __device__ __forceinline__ Weights8(uint32_t w, uint32_t z) {
        if constexpr (X == X_F16) v = __builtin_bit_cast(u32x4, weights_f16(w, z));
        else v = __builtin_bit_cast(u32x4, weights_bf16(w, (float)z));
    }
    __device__ __forceinline__ f32x4 times(const Operand<X>& x, f32x4 d) const {
        if constexpr (X == X_F16)
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, v), __builtin_bit_cast(half8, x.v), d, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, x.v), d, 0, 0, 0);
    }
};
template <>
struct Weights8<X_I8> {
    long v;
    __device__ __forceinline__ Weights8(uint32_t w, uint32_t z) { v = weights_i8(w, z * 0x01010101u); }
    __device__ __forceinline__ i32x4 times(const Operand<X_I8>& x, i32x4 d) const {
        return __builtin_amdgcn_mfma_i32_16x16x32_i8(v, __builtin_bit_cast(long, x.v), d, 0, 0, 0);
    }
};

// x as it lies in memory: 8 columns from k on of input b, or the last 8 where
// there are none (then `blank` makes zeros of them).
template <int X>
struct Raw { u32x4 v[X == X_F32 ? 2 : 1]; };
template <>
struct Raw<X_I8> { u32x2 v[1]; };

template <int X>
constexpr int kXBytes = X == X_I8 ? 1 : X == X_F32 ? 4 : 2;
template <int X>
__device__ __forceinline__ const uint8_t* x_at(const W4Args& a, int b, int k) {
    return (const uint8_t*)a.x + ((int64_t)b * a.x_row + k) * kXBytes<X>;
}
template <int X>
__device__ __forceinline__ Raw<X> load_x(const uint8_t* p) {
    Raw<X> r;
    if constexpr (X == X_I8) {
        r.v[0] = *(const u32x2_a1*)p;
    } else {
        r.v[0] = *(const u32x4_a1*)p;
        if constexpr (X == X_F32) r.v[1] = *(const u32x4_a1*)(p + 16);
    }
    return r;
}
template <int X>
__device__ __forceinline__ Raw<X> load_x(const W4Args& a, int b, int k) {
    return load_x<X>(x_at<X>(a, b, min(k, a.cols - 8)));
}
template <int X>
__device__ __forceinline__ void blank(Raw<X>* r, bool in) {
#pragma unroll
    for (int i = 0; i < (X == X_F32 ? 2 : 1); i++)
#pragma unroll
        for (int j = 0; j < (X == X_I8 ? 2 : 4); j++) r->v[i][j] = in ? r->v[i][j] : 0u;
}

// It as an operand (f16, bf16 and 8-bit x).
template <int X>
__device__ __forceinline__ void operand(const Raw<X>& r, Operand<X>* o) {
    if constexpr (X == X_I8) {
        o->v = u32x2{__builtin_amdgcn_perm(r.v[0].y, r.v[0].x, 0x05010400),
                       __builtin_amdgcn_perm(r.v[0].y, r.v[0].x, 0x07030602)};
    } else {
        o->v = r.v[0];
    }
}

// The scale of 8-bit input b's unit u of a step.
template <int U>
__device__ __forceinline__ float x_scale(const W4Args& a, int b, int step, int u) {
    const int k = min(step * kStep + u * (kStep / U), a.cols - 1);
    return a.x_scales[(int64_t)b * a.x_groups + (k >> a.x_shift)];
}

// Joins the waves of a tile and the parts of an input, and stores the tiles of a
// workgroup from first_tile on: red holds [wave][column][16 rows].
template <int X, int PARTS, int WAVES>
__device__ __forceinline__ void store_tiles(const W4Args& a, const float* red, int first_tile, int b0, int count,
                                            int columns) {
    const int wms = WAVES / a.wk, sh = 31 - __clz(wms);  // tiles, a power of two
    for (int i = threadIdx.x; i < count * wms * 16; i += WAVES * 64) {
        const int m = i & 15, t = i >> 4 & (wms - 1), b = i >> 4 >> sh;
        const int row = (first_tile + t) * 16 + m;
        if (row >= a.rows) continue;
        float v = 0;
#pragma unroll
        for (int p = PARTS - 1; p >= 0; p--)
            for (int k = 0; k < a.wk; k++) v += red[((t * a.wk + k) * columns + b * PARTS + p) * 16 + m];
        if constexpr (X == X_I8) {
            if (a.x_shift < 0) v *= a.x_scales[b0 + b];
        }
        const int64_t o = (int64_t)(b0 + b) * a.out_row + row;
        if (a.out_type == MIVI_GGML_F32) store_elem<MIVI_GGML_F32>(a.out, o, v);
        else if (a.out_type == MIVI_GGML_F16) store_elem<MIVI_GGML_F16>(a.out, o, v);
        else store_elem<MIVI_GGML_BF16>(a.out, o, v);
    }
}

// --------------------------------------------------------------- few inputs
// Up to 16 columns of the product. x lies whole in LDS, in operand order, and
// tiles stream past it. f16 inputs stay as they are; bf16 and f32 ones are held
// in fp16, each step's 128 columns multiplied by the power of two that takes
// their largest to 2^14 .. 2^15 (bf16 ones to no less than 2^-39 of that largest;
// f32 ones in two parts: scaled_operands). Against 8-bit x the weights enter as
// codes and z sum x comes off their sums, all whole numbers. (With codes as the fp16
// numbers c 2^-24, masks alone, one input takes up to 4 % less, but sums have 17
// bits: the matrix cores align products by their operands' exponents as if all were
// normal numbers.)
//
// HBM and vector instructions bound it: one fp16 input over 65535 x 2048 in groups
// of 64 with zeros 16.2 us, 4.5 TB/s, the vector pipe 57 % of the cycles; eight 8-bit
// ones over 28672 x 8192 26.5 us, 4.6 TB/s, 41 %; one f32 input over 8192 x 2048 5.9, a
// chain of x's load, its conversion, four steps and the join.
constexpr int kFewRing = 4;  // steps of a wave in flight

struct FewArgs {
    W4Args w;
    int n;                         // steps of a wave
    int pitch, sums, red;          // bytes of LDS: of 8 columns; before x's sums and factors; before the results
};

// Largest magnitude's bits over 16 lanes; sums over 16, 8 or 4.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    const auto f = [](uint32_t x) { return __uint_as_float(x); };
    const auto u = [](float x) { return __float_as_uint(x); };
    v = max(v, u(dpp_mov<0xB1>(f(v))));
    v = max(v, u(dpp_mov<0x4E>(f(v))));
    v = max(v, u(xor4_mov(f(v))));
    return max(v, u(dpp_mov<0x128>(f(v))));
}
template <int U>
__device__ __forceinline__ float unit_sum(float v) {
    v += dpp_mov<0xB1>(v);
    v += dpp_mov<0x4E>(v);
    if (U <= 2) v += xor4_mov(v);
    if (U <= 1) v += dpp_mov<0x128>(v);
    return v;
}

// 8 columns of a bf16 or f32 input as fp16 operands, and what the step's results
// are to be multiplied by. 16 lanes have a step. The first part of an f32 input
// leaves at most 2^3; 2^12 times that, the second has its own 11 bits whatever the
// input's size next to the step's largest (with one factor for both, an input 2^-24
// of the largest kept 15 bits of 24). Both together are off by 2^-23 of the input (a
// third part would take half as many columns again, and the sums' roundings add
// more), or by the 2^-37 that a subnormal second part leaves: 2^-51 of the largest.
template <int X>
__device__ __forceinline__ void scaled_operands(const Raw<X>& r, Operand<X_F16> (&o)[parts_of(X)],
                                                float (&factor)[parts_of(X)]) {
    float v[8];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if constexpr (X == X_F32) v[e] = __uint_as_float(r.v[e / 4][e % 4]);
        else v[e] = bf16_bits_to_f32(r.v[0][e / 2] >> (e % 2 * 16));
        top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    }
    // biased exponents: 2^(14 - e) for a largest value of 2^e, 2^126 at most
    const int ex = min(127 + 14 - ((int)(max16(top) >> 23) - 127), 253);
    const float up = __uint_as_float((uint32_t)ex << 23);
    factor[0] = __uint_as_float((uint32_t)(254 - ex) << 23);
    if constexpr (X == X_F32) factor[1] = factor[0] * 0x1p-12f;
    half8 h[parts_of(X)];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float y = v[e] * up;
        h[0][e] = (_Float16)y;
        // what an infinity leaves is nothing
        if constexpr (X == X_F32)
            h[1][e] = (_Float16)(__builtin_fabsf(y) == __builtin_inff() ? 0.f : (y - (float)h[0][e]) * 0x1p12f);
    }
#pragma unroll
    for (int p = 0; p < parts_of(X); p++) o[p].v = __builtin_bit_cast(u32x4, h[p]);
}

template <int X, int U, int W, bool SB, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 4) void w4_few_kernel(FewArgs g) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr bool I8 = X == X_I8;
    constexpr int PARTS = parts_of(X), PER = 4 / U, XB = I8 ? 8 : 16;
    typedef typename std::conditional<I8, i32x4, f32x4>::type D;
    const W4Args& a = g.w;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wk = wave % a.wk, wm = wave / a.wk;
    const int wms = WAVES / a.wk, stride = gridDim.x * wms, cols_x = a.batch * PARTS, col = min(r, cols_x - 1);
    int* sums = (int*)(lds + g.sums);                               // of -x where it has 8 bits: [step][unit][column]
    float* factors = (float*)sums + (I8 ? a.steps * U * cols_x : 0);  // the same, of others [step][column]

    Step<W, !I8> w[kFewRing];
    int tile = blockIdx.x * wms + wm, next_tile = tile, next = 0;  // of the next fetch
    const auto refill = [&](int slot) {
        // behind the last step and tile those are loaded again
        fetch<W, !I8>(a, (int64_t)min(next_tile, a.tiles - 1) * a.steps + min(wk + next * a.wk, a.steps - 1), lane, &w[slot]);
        if (++next == g.n) next = 0, next_tile += stride;
    };
#pragma unroll
    for (int p = 0; p < kFewRing; p++) refill(p);

    // x to LDS, four pieces of 8 columns of a thread's on their way at once
    const int n8 = a.steps * 16, items = a.batch * n8;
    for (int base = 0; base < items; base += 4 * WAVES * 64) {
        Raw<X> raw[4];
        int at[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = min(base + e * WAVES * 64 + tid, items - 1), b = i / n8, c = i - b * n8;
            at[e] = base + e * WAVES * 64 + tid < items ? c << 4 | b : -1;
            raw[e] = load_x<X>(a, b, c * 8);
            blank<X>(&raw[e], c * 8 < a.cols);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (base + e * WAVES * 64 >= items) break;
            const int c = at[e] >> 4, b = at[e] & 15;
            uint8_t* to = lds + c * g.pitch + b * PARTS * XB;
            if constexpr (I8) {
                const int unit = (c >> 4) * U + (c & 15) / (16 / U);
                const bool head = at[e] >= 0 && (c & (16 / U - 1)) == 0;
                Operand<X> o;
                operand<X>(raw[e], &o);
                int s = __builtin_amdgcn_sdot4((int)o.v.x, 0x01010101, 0, false);
                s = __builtin_amdgcn_sdot4((int)o.v.y, 0x01010101, s, false);
                const float sum = unit_sum<U>((float)s);  // whole numbers far below 2^24
                if (at[e] >= 0) *(Operand<X>*)to = o;
                if (head) {
                    sums[unit * cols_x + b] = -(int)sum;
                    factors[unit * cols_x + b] = a.x_shift < 0 ? 1.f : x_scale<U>(a, b, c >> 4, unit & (U - 1));
                }
            } else {
                Operand<X_F16> o[PARTS];
                float factor[PARTS];
                if constexpr (X == X_F16) o[0].v = raw[e].v[0];
                else scaled_operands<X>(raw[e], o, factor);
#pragma unroll
                for (int p = 0; p < PARTS; p++) {
                    if (at[e] >= 0) *(Operand<X_F16>*)(to + p * XB) = o[p];
                    if (X != X_F16 && at[e] >= 0 && (c & 15) == 0) factors[(c >> 4) * cols_x + b * PARTS + p] = factor[p];
                }
            }
        }
    }
    __syncthreads();

    f32x4 acc = {0, 0, 0, 0};
    int s = 0, it = 0, t0 = blockIdx.x * wms;
    const auto compute = [&](const Step<W, !I8>& c, int step) {
        const uint8_t* xl = lds + (step * 16 + q) * g.pitch + col * XB;
        const int at = step * U * cols_x + col;
        Operand<I8 ? X_I8 : X_F16> x[4];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = *(const Operand<I8 ? X_I8 : X_F16>*)(xl + j * 4 * g.pitch);
        int sum[U];
        float m[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if constexpr (I8) sum[u] = sums[at + u * cols_x], m[u] = factors[at + u * cols_x];
            else if (u == 0) m[u] = X == X_F16 ? 1.f : factors[step * cols_x + col];
        }
        constexpr int per_w = U / W;
        D d[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            d[u] = D{0, 0, 0, 0};
#pragma unroll
            for (int j = u * PER; j < (u + 1) * PER; j++) {
                if constexpr (I8) {
                    const uint32_t even = c.codes[j] & 0x0F0F0F0Fu, odd = c.codes[j] >> 4 & 0x0F0F0F0Fu;
                    d[u] = __builtin_amdgcn_mfma_i32_16x16x32_i8((long)((uint64_t)odd << 32 | even),
                                                                 __builtin_bit_cast(long, x[j].v), d[u], 0, 0, 0);
                } else {
                    const Weights8<X_F16> wv(c.codes[j], c.zeros[0] >> (8 * (u / per_w)) & 15);
                    d[u] = wv.times(x[j], d[u]);
                }
            }
        }
        f32x4 part = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < U; u++) {
            float f[4];
            scales_f32(c.scales[u / per_w], SB, f);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (I8) {
                    const int byte = i * W + u / per_w, z = (int)(c.zeros[byte / 4] >> (byte % 4 * 8) & 0xFF);
                    // (a product of 24 bits and the sum in one instruction)
                    // and the input's scale last: the scales' product alone may be no
                    // normal number, or none at all where the sum is 0
                    acc[i] = fmaf((float)(d[u][i] + __mul24(z, sum[u])) * f[i], m[u], acc[i]);
                } else if constexpr (X == X_F16) {
                    acc[i] = fmaf(d[u][i], f[i], acc[i]);
                } else {
                    part[i] = fmaf(d[u][i], f[i], part[i]);
                }
            }
        }
        if constexpr (!I8 && X != X_F16) {
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = fmaf(part[i], m[0], acc[i]);
        }
    };
    while (t0 < a.tiles) {
#pragma unroll
        for (int p = 0; p < kFewRing; p++) {
            if (t0 >= a.tiles) break;
            const int step = wk + s * a.wk;
            if (tile < a.tiles && step < a.steps) compute(w[p], step);
            refill(p);
            if (++s == g.n) {
                float* red = (float*)(lds + g.red) + it * (WAVES * 256);
                *(f32x4*)(red + (wave * 16 + r) * 16 + q * 4) = acc;
                __syncthreads();
                store_tiles<X, PARTS, WAVES>(a, red, t0, 0, a.batch, 16);
                acc = f32x4{0, 0, 0, 0};
                s = 0, it ^= 1, t0 += stride, tile += stride;
            }
        }
    }
}

// Bytes of LDS for 8 columns of x: 16-byte slots, or 8-byte ones with an odd number
// of tiles' worth, so that neighbouring rows are in different banks.
constexpr int rows_pitch(bool i8, int nt) { return i8 ? (nt | 1) * 128 : nt * 256; }

// Whether w4_rows_kernel has a form of 16 waves for nt tiles of columns: where 128
// registers hold it.
constexpr bool rows_of_16(int x, int units, int nt) {
    return nt >= 2 && nt <= 5 && (x != X_I8 || units * nt <= 6) && (x != X_F32 || units == 1 || nt < 5);
}

// And one of 8 tiles of columns, by 256 registers.
constexpr bool rows_of_8(int x, int units) { return x != X_I8 || units < 4; }

// More inputs, or deeper rows: NT tiles of 16 columns; x goes through LDS, wk
// steps of it at a time, 8 columns of all inputs after another, loaded into
// registers a phase ahead. 8 waves have two buffers and one barrier a phase; 16
// have one buffer and two barriers, but four waves a SIMD, whose loads from LDS,
// products and sums overlap better. 80 bf16 inputs over 14336 x 4096 in groups of 32
// with zeros: 28.1 us, 334 TFLOP/s; the vector pipe (conversion, a scale for every
// product's results) 58 % of the cycles, the matrix cores 15 %, LDS 27 %.
template <int X, int U, int W, int NT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void w4_rows_kernel(W4Args a) {
    static_assert(WAVES == 8 ? NT < 8 || rows_of_8(X, U) : rows_of_16(X, U, NT), "a form that no plan takes");
    constexpr int BUFFERS = WAVES == 8 ? 2 : 1, RING = WAVES == 8 ? kRing : 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr bool I8 = X == X_I8, SCALED = X == X_F32;
    constexpr int XB = I8 ? 8 : 16, PARTS = parts_of(X), PER = 4 / U;
    constexpr int ITEMS = items_of(X, WAVES);
    typedef typename std::conditional<X == X_I8, i32x4, f32x4>::type D;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wk = wave % a.wk, wm = wave / a.wk;
    const int wms = WAVES / a.wk, tile = blockIdx.x * wms + wm;
    const bool live = tile < a.tiles;
    const int b0 = blockIdx.y * a.block, count = min(a.block, a.batch - b0), cols_x = count * PARTS;
    // An operand of 8 columns of x and column c of the product is at slot c ^ (its
    // place of 16 in the step): a wave's stores, one c, and its loads, 16 c at each of
    // four places, both take every bank in turn. (80 inputs with the slots in order and
    // 16 bytes over a row: 43 % of the LDS's cycles were conflicts.) Slots behind the
    // last column hold anything: their results are not used.
    constexpr int pitch = rows_pitch(I8, NT);
    int slot[4];
#pragma unroll
    for (int j = 0; j < 4; j++) slot[j] = (r ^ q ^ 4 * j) * XB + j * 4 * pitch;
    const int xs_at = a.wk * 16 * pitch;  // behind x its scales (8-bit x) or factors (f32)
    const int buffer = (xs_at + a.wk * cols_x * 4 * (I8 ? U : SCALED ? 1 : 0) + 15) / 16 * 16;
    // a thread stages 8 columns of every (threads / pieces of an input)-th input
    const int n8 = a.wk * 16, c8 = tid & (n8 - 1), bx = tid / n8, b_step = WAVES * 64 / n8;
    const int phases = (a.steps + a.wk - 1) / a.wk;
    const int64_t first = (int64_t)(live ? tile : 0) * a.steps;

    const int full = a.cols / (a.wk * kStep);  // phases with no columns behind the last
    const uint8_t* xp[ITEMS];
#pragma unroll
    for (int e = 0; e < ITEMS; e++) xp[e] = x_at<X>(a, b0 + min(bx + e * b_step, count - 1), 0);
    Raw<X> raw[ITEMS];
    float xs_raw[2];  // 8-bit x: scales of (inputs x units): count wk <= 4 ITEMS WAVES and U <= 4, so two a thread do
    const int nu = a.wk * U;
    const auto load = [&](int ph) {
        if constexpr (X == X_I8) {
            if (a.x_shift >= 0) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int i = tid + e * WAVES * 64, u = i & (nu - 1);
                    xs_raw[e] = x_scale<U>(a, b0 + min(i / nu, count - 1), ph * a.wk + u / U, u % U);
                }
            }
        }
        const int64_t at = (int64_t)min(ph * a.wk * kStep + c8 * 8, a.cols - 8) * kXBytes<X>;
#pragma unroll
        for (int e = 0; e < ITEMS; e++)
            if (e * b_step < count) raw[e] = load_x<X>(xp[e] + at);
    };
    const auto store = [&](int ph) {
        uint8_t* to = lds + (BUFFERS == 2 ? (ph & 1) * buffer : 0);
#pragma unroll
        for (int e = 0; e < ITEMS; e++) {
            const int b = bx + e * b_step;
            if (b < count) {
                if (ph >= full) blank<X>(&raw[e], (ph * a.wk * 16 + c8) * 8 < a.cols);
                if constexpr (SCALED) {
                    Operand<X_F16> o[PARTS];
                    float factor[PARTS];
                    scaled_operands<X>(raw[e], o, factor);
#pragma unroll
                    for (int p = 0; p < PARTS; p++) {
                        *(Operand<X_F16>*)(to + c8 * pitch + ((b * PARTS + p) ^ (c8 & 15)) * XB) = o[p];
                        if ((c8 & 15) == 0) ((float*)(to + xs_at))[(c8 >> 4) * cols_x + b * PARTS + p] = factor[p];
                    }
                } else {
                    Operand<X> o;
                    operand<X>(raw[e], &o);
                    *(Operand<X>*)(to + c8 * pitch + (b ^ (c8 & 15)) * XB) = o;
                }
            }
        }
        if constexpr (X == X_I8) {
            if (a.x_shift >= 0) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int i = tid + e * WAVES * 64, b = i / nu;
                    if (b < count) ((float*)(to + xs_at))[(i & (nu - 1)) * cols_x + b] = xs_raw[e];
                }
            }
        }
    };

    f32x4 acc[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) acc[n] = f32x4{0, 0, 0, 0};
    Step<W, true> w[RING];
    load(0);
    const auto refill = [&](int slot, int ph) {  // behind the last step it is loaded again
        fetch<W, true>(a, first + min(wk + ph * a.wk, a.steps - 1), lane, &w[slot]);
    };
#pragma unroll
    for (int p = 0; p < RING; p++) refill(p, p);
    store(0);

    for (int base = 0; base < phases; base += RING) {
#pragma unroll
        for (int p = 0; p < RING; p++) {
            const int ph = base + p;
            if (ph >= phases) break;
            __syncthreads();  // this phase's x is there, the phase before is read
            if (ph + 1 < phases) load(ph + 1);
            if (live && wk + ph * a.wk < a.steps) {
                const Step<W, true>& c = w[p];
                const uint8_t* xl = lds + (BUFFERS == 2 ? (ph & 1) * buffer : 0) + (wk * 16 + q) * pitch;
                const float* xs = (const float*)(lds + (BUFFERS == 2 ? (ph & 1) * buffer : 0) + xs_at) + wk * (I8 ? U : 1) * cols_x;
                f32x4 part[SCALED ? NT : 1];
#pragma unroll
                for (int n = 0; n < (SCALED ? NT : 1); n++) part[n] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < U; u++) {
                    D d[NT];
#pragma unroll
                    for (int n = 0; n < NT; n++) d[n] = D{0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < PER; k++) {
                        const int j = u * PER + k;
                        const Weights8<SCALED ? X_F16 : X> wv(c.codes[j], c.zeros[0] >> (8 * (u / (U / W))) & 15);
#pragma unroll
                        for (int n = 0; n < NT; n++)
                            d[n] = wv.times(*(const Operand<SCALED ? X_F16 : X>*)(xl + slot[j] + 16 * n * XB), d[n]);
                    }
                    float f[4];
                    scales_f32(c.scales[u / (U / W)], a.bf16_scales, f);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float m = 1.f;
                        if constexpr (X == X_I8) {
                            if (a.x_shift >= 0) m = xs[u * cols_x + min(16 * n + r, cols_x - 1)];
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if constexpr (SCALED) part[n][i] = fmaf(d[n][i], f[i], part[n][i]);
                            else if constexpr (I8) acc[n][i] = fmaf((float)d[n][i] * f[i], m, acc[n][i]);
                            else acc[n][i] = fmaf(d[n][i], f[i], acc[n][i]);
                        }
                    }
                }
                if constexpr (SCALED) {
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const float m = xs[min(16 * n + r, cols_x - 1)];
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[n][i] = fmaf(part[n][i], m, acc[n][i]);
                    }
                }
            }
            refill(p, ph + RING);
            if (BUFFERS == 1) __syncthreads();  // this phase's x is read
            if (ph + 1 < phases) store(ph + 1);
        }
    }
    __syncthreads();
    float* red = (float*)lds;
#pragma unroll
    for (int n = 0; n < NT; n++) *(f32x4*)(red + ((wave * NT + n) * 16 + r) * 16 + q * 4) = acc[n];
    __syncthreads();
    store_tiles<X, PARTS, WAVES>(a, red, blockIdx.x * wms, b0, count, 16 * NT);
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
    // (rows: the 16 tiles of a workgroup may reach 255 behind the last)
    if (rows > (size_t)INT32_MAX - 1023 || cols > (size_t)INT32_MAX / 8) return err_overflow();
    p->tiles = (rows + 15) / 16, p->steps = (cols + kStep - 1) / kStep;
    p->units = group == 32 ? 4 : group == 64 ? 2 : 1;
    size_t cells, all;
    if (__builtin_mul_overflow(p->tiles, p->steps, &cells) || __builtin_mul_overflow(cells, (size_t)2048, &all) ||
        all > (size_t)INT64_MAX / 8)
        return err_overflow();
    p->codes = cells * 1024, p->scales = cells * 32 * p->units, p->zeros = zeros ? cells * 16 * p->units : 0;
    return MIVI_OK;
}

// How a product is laid out: w4_few_kernel, or w4_rows_kernel with nt tiles of
// columns.
struct W4Plan {
    bool few;
    int nt, waves;
    dim3 grid;
    size_t lds;
    FewArgs g;
};

template <int X, int U, int W>
void launch_rows(const W4Args& a, const W4Plan& p, hipStream_t s) {
#define ROWS(N)                                                                                     \
    if constexpr (rows_of_16(X, U, N))                                                              \
        if (p.waves == 16) {                                                                        \
            w4_rows_kernel<X, U, W, N, 16><<<p.grid, 1024, p.lds, s>>>(a);                          \
            break;                                                                                  \
        }                                                                                           \
    w4_rows_kernel<X, U, W, N, 8><<<p.grid, 512, p.lds, s>>>(a)
    switch (p.nt) {
        case 1: ROWS(1); break;
        case 2: ROWS(2); break;
        case 3: ROWS(3); break;
        case 4: ROWS(4); break;
        case 5: ROWS(5); break;
        default:
            if constexpr (rows_of_8(X, U)) {
                ROWS(8);
            }
            break;
    }
#undef ROWS
}
template <int X, int U, int W>
void launch_w4(const W4Args& a, W4Plan& p, hipStream_t s) {
    if (!p.few) return launch_rows<X, U, W>(a, p, s);
    p.g.w = a;
#define FEW(SB)                                                                                 \
    if (p.waves == 8) w4_few_kernel<X, U, W, SB, 8><<<p.grid, 512, p.lds, s>>>(p.g);            \
    else w4_few_kernel<X, U, W, SB, 16><<<p.grid, 1024, p.lds, s>>>(p.g)
    if (a.bf16_scales) { FEW(true); }
    else { FEW(false); }
#undef FEW
}
// u: sums of a step that are scaled by themselves, w: those that the weights'
// groups ask for (fewer where 8-bit inputs have the finer scales)
template <int X>
void launch_w4(const W4Args& a, int u, int w, W4Plan& p, hipStream_t s) {
    if (u == w) {
        if (u == 1) launch_w4<X, 1, 1>(a, p, s);
        else if (u == 2) launch_w4<X, 2, 2>(a, p, s);
        else launch_w4<X, 4, 4>(a, p, s);
    } else if constexpr (X == X_I8) {
        if (u == 2) launch_w4<X, 2, 1>(a, p, s);
        else if (w == 1) launch_w4<X, 4, 1>(a, p, s);
        else launch_w4<X, 4, 2>(a, p, s);
    }
}

W4Plan w4_plan(W4Args* a, int x, int units, size_t batch, size_t tiles, size_t steps) {
    W4Plan p = {};
    const size_t cus = (size_t)num_cus();
    {
        const size_t columns = batch * parts_of(x), xb = x == X_I8 ? 8 : 16;
        // columns of a multiple of 64 bytes would store to the same banks
        const size_t pitch = columns * xb + (columns * xb % 64 ? 0 : 16);
        const size_t x_bytes = steps * 16 * pitch, sums = steps * columns * 4 * (x == X_I8 ? 2 * units : 1);
        const size_t red = (x_bytes + sums + 15) / 16 * 16;
        // 16 waves a CU: two workgroups of 8, or one of 16 where x fills LDS
        p.waves = red + 2 * 8 * 1024 <= kLdsFew / 2 ? 8 : 16;
        p.lds = red + 2 * p.waves * 1024;
        if (columns <= 16 && steps <= 65536 && p.lds <= kLdsFew) {
            p.few = true;
            a->wk = 1;
            // waves of a tile, as many as keep 16 a CU busy: at least a ring's steps
            // each, half of one where that leaves CUs without work
            while (a->wk < kWaves && tiles * a->wk < 16 * cus &&
                   steps >= (size_t)a->wk * (tiles * a->wk < 8 * cus ? kFewRing : 2 * kFewRing))
                a->wk *= 2;
            p.g.n = (int)((steps + a->wk - 1) / a->wk);
            p.g.pitch = (int)pitch, p.g.sums = (int)x_bytes, p.g.red = (int)red;
            // workgroups as many as fit the card, with as many tiles each
            const size_t groups = (tiles * a->wk + p.waves - 1) / p.waves, fit = cus * (16 / p.waves);
            const size_t rounds = (groups + fit - 1) / fit;
            p.grid = dim3((unsigned)((groups + rounds - 1) / rounds));
            a->block = (int)batch;
            return p;
        }
    }
    const size_t parts = parts_of(x);
    // Blocks of inputs, waves of a workgroup and of a tile by an estimate. A phase
    // of 8 waves takes 1.2 us and 0.06 a tile of columns where a CU has one workgroup
    // (staging, products and the barrier in turn), 0.35 and 0.2 where two share it;
    // of 16 waves, which have twice the steps, 1.35 and 0.28. Measured, the first of each
    // the estimate's choice: 80 bf16 inputs, 14336 x 4096, groups of 32: one block and 16
    // waves 29.7 us, 8 waves 34.8, two blocks 38 and 48; 4096 x 14336, groups of 128: two
    // blocks and 16 waves 33.0, 8 waves 41, one block 66 and 85; 512 inputs, 14336 x 4096:
    // blocks of 128 and 8 waves 116, of 64 and 16 waves 114, of 74 and 16 waves 126; 80 f32
    // ones: two blocks and 16 waves 45, 8 waves 54, four blocks 54 and more. (8-bit inputs
    // take less than a phase is thought to: 80 over 8192 x 2048 two blocks of 8 waves 17.5,
    // of 16 11.4; 512 over 14336 x 4096 blocks of 128 135, of 64 and 16 waves 109.)
    double best = 0;
    for (const int nt : {1, 2, 3, 4, 5, 8}) {
        if (nt == 8 && !rows_of_8(x, units)) break;
        const size_t most = 16 * nt / parts, blocks = (batch + most - 1) / most, block = (batch + blocks - 1) / blocks;
        if (best > 0 && (block * parts + 15) / 16 * 2 <= (size_t)nt) break;  // the batch has no more columns
        const size_t step_bytes =
            16 * rows_pitch(x == X_I8, nt) + 4 * block * (x == X_I8 ? units : x == X_F32 ? parts : 0);
        for (int form = 0; form < 9; form++) {
            const int waves = form < 4 ? 8 : 16, wk = form < 4 ? 1 << form : 1 << (form - 4);
            if (waves == 16 && !rows_of_16(x, units, nt)) break;
            const size_t items = (block * wk * 16 + waves * 64 - 1) / (waves * 64);
            const size_t buffers = (waves == 8 ? 2 : 1) * ((wk * step_bytes + 15) / 16 * 16);
            if ((wk > 1 || waves == 16) && (buffers > kLds || items > (size_t)items_of(x, waves))) continue;
            const size_t lds = std::max<size_t>(buffers, (size_t)waves * nt * 1024), phases = (steps + wk - 1) / wk;
            const size_t fit = waves == 8 && nt <= 3 && lds <= 80 * 1024 ? 2 : 1, grid_x = (tiles * wk + waves - 1) / waves;
            const size_t of_cu = (grid_x * blocks + cus - 1) / cus;
            const double staging = x == X_F32 ? (waves == 8 ? 0.35 : 0.7) * (double)items : 0;  // the conversion
            const double alone = (waves == 8 ? 1.2 + 0.06 * nt : 1.35 + 0.28 * nt) + staging, shared = 0.35 + 0.2 * nt + staging;
            const double us = (double)phases * ((double)(of_cu / fit) * std::max(alone, (double)fit * shared) +
                                                (of_cu % fit ? alone : 0.0));
            if (best == 0 || us < best) {
                best = us;
                p.nt = nt, p.lds = lds, p.waves = waves, a->wk = wk, a->block = (int)block;
                p.grid = dim3((unsigned)std::min<size_t>(grid_x, UINT32_MAX), (unsigned)blocks);
            }
        }
    }
    return p;
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
    const int units = std::max((int)p.units, x_units);
    a.codes = packed, a.scales = packed + p.codes, a.zeros = zeros ? packed + p.codes + p.scales : packed;
    a.has_zeros = zeros;
    a.out_row = (int64_t)out_row_stride, a.out_type = type;
    a.rows = (int)rows, a.cols = (int)cols;
    a.tiles = (int)p.tiles, a.steps = (int)p.steps;
    a.bf16_scales = scale_type == MIVI_GGML_BF16;
    // launches of `most` inputs, and one of those behind the last of them
    const size_t most = std::min(batch, kMostInputs), left = batch % most;
    W4Args args[2] = {a, a};
    W4Plan plans[2];
    for (int i = 0; i < (left ? 2 : 1); i++) {
        args[i].batch = (int)(i ? left : most);
        plans[i] = w4_plan(&args[i], x, units, args[i].batch, p.tiles, p.steps);
        if (!grid_fits(plans[i].grid.x, 1024)) return err_overflow();
    }
    const size_t x_bytes = x == X_I8 ? 1 : type_bytes(type);
    for (size_t b = 0; b < batch; b += most) {
        W4Args& l = args[batch - b < most];
        W4Plan& plan = plans[batch - b < most];
        l.x = (const uint8_t*)a.x + b * (size_t)a.x_row * x_bytes;
        if (x == X_I8) l.x_scales = a.x_scales + b * (size_t)a.x_groups;
        l.out = (uint8_t*)out + b * out_row_stride * type_bytes(type);
        switch (x) {
            case X_F16: launch_w4<X_F16>(l, units, (int)p.units, plan, s); break;
            case X_BF16: launch_w4<X_BF16>(l, units, (int)p.units, plan, s); break;
            case X_F32: launch_w4<X_F32>(l, units, (int)p.units, plan, s); break;
            default: launch_w4<X_I8>(l, units, (int)p.units, plan, s); break;
        }
        MIVI_HIP_CHECK(hipGetLastError());
    }
    return clear_error();
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
