// A paged key/value cache held in 4 bits: rows quantised into it, read back
// from it, and attention over it. (The reference's 4-bit caches,
// crates/mivi-kv/src/cache.rs:5-15, rotate rows and use code books; this one
// holds plain block-scaled integers, which enter the matrix cores exactly.)
//
// Values. Blocks of 32 dimensions of one token and head: a scale d and 32
// codes c in 0..15 standing for (c - 8) d. With m the block's value of largest
// magnitude (the positive one of a tie), d = -m / 8 rounded to 8 significant
// bits (bf16) and then to fp16, and c - 8 = rint(x / d) limited to -8..7: m
// itself is the code 0. NaN is held as 0, values past 21760 as 21760, so every
// held value is finite; and as d has 8 significant bits and |c - 8| is 8 or at
// most 3 bits wide, (c - 8) d has at most 11 and is an fp16 number exactly.
// The attention below therefore multiplies the held values themselves, in
// fp16 operands, and rounds neither K nor V.
//
// Layout. A page holds page_tokens tokens (a multiple of 32) of every kv head,
// head by head; a head's tokens lie in groups of 32, 36 hd bytes each:
//   K codes   16 hd bytes, block b and lane l = (token mod 16) + 16 quarter at
//             q4_at(b, l): 8 bytes, one dword a half of the group, holding the
//             8 dimensions 8 quarter .. + 7 of the block, dimension 2 i at bit
//             4 i and 2 i + 1 at bit 16 + 4 i;
//   V codes   16 hd bytes, block b and lane l = n + 16 quarter (n = dimension
//             mod 16, quarter of the tokens 4 quarter .. + 3 and 16 + those):
//             8 bytes, one a token (in the order 0 2 1 3 within a dword), the
//             low nibble dimension n of the block, the high one n + 16;
//   K scales  fp16 [token mod 16][half of the group][block];
//   V scales  fp16 [block][quarter][8 tokens].
// These are the operands of v_mfma_f32_16x16x32_f16: 32 dimensions of K, a
// block, are one product of the scores K q (A = K, rows tokens), whose results
// (lane: query row l mod 16, tokens 4 quarter + i of each half) are the B
// operand of V p as they stand, and lane l loads both codes in 16-byte pieces.
// No byte is shared by two tokens, so rows of one group may be written by
// different waves.
//
// Batches. Rows are ragged: rows starts[s] .. starts[s + 1] - 1 belong to
// sequence s and are its last positions, lens[s] - n .. lens[s] - 1.
#include <algorithm>

#include "common.h"

using namespace mivi;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x4_a8 __attribute__((ext_vector_type(4), aligned(8)));

constexpr int kGroup = 32;         // tokens of a group
constexpr float kMaxScale = 2720;  // 170 * 2^4 (8 significant bits): 24 times it is an fp16 number
constexpr float kMaxValue = 8 * kMaxScale;

// What the three entry points share: the cache and the batch over it.
struct Q4Batch {
    uint8_t* cache;
    const int32_t* pages;   // page ids, row s of page_stride for sequence s
    const int32_t* starts;  // [n_seq + 1]
    const int32_t* lens;    // [n_seq]
    int64_t page_stride, n_pages, page_bytes;
    int n_seq, n_kv, hd, gpp;  // gpp: groups of a page
    int cap;                   // positions that the table covers
};

// A group's byte of block b, lane l: two blocks side by side where there are
// two, so that a lane's 16 bytes are one load.
__host__ __device__ constexpr int q4_at(int nb, int b, int lane) {
    return b / 2 < nb / 2 ? b / 2 * 1024 + lane * 16 + b % 2 * 8 : b / 2 * 1024 + lane * 8;
}

// Sequence of row r, or -1: the last s with starts[s] <= r, if r is before
// starts[s + 1].
__device__ __forceinline__ int seq_of(const Q4Batch& a, int r) {
    int lo = 0, hi = a.n_seq;  // starts[lo] <= r < starts[hi] where there is such a pair
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid] <= r) lo = mid;
        else hi = mid;
    }
    return a.starts[lo] <= r && r < a.starts[lo + 1] ? lo : -1;
}

// Address of the group of sequence s and kv head h at group index g, or null
// where the table has no page of the cache there.
__device__ __forceinline__ uint8_t* group_ptr(const Q4Batch& a, int s, int h, int g) {
    const int pi = g / a.gpp;
    const int page = a.pages[(int64_t)s * a.page_stride + pi];
    if (page < 0 || page >= a.n_pages) return nullptr;
    return a.cache + (int64_t)page * a.page_bytes + ((int64_t)h * a.gpp + (g - pi * a.gpp)) * (36 * a.hd);
}

// Position of row r of sequence s and whether the table covers it.
__device__ __forceinline__ bool row_pos(const Q4Batch& a, int s, int r, int* pos) {
    const int64_t p = (int64_t)a.lens[s] - a.starts[s + 1] + r;
    *pos = (int)p;
    return p >= 0 && p < a.cap;
}

// --------------------------------------------------------- element types
template <int T>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
    if constexpr (T == MIVI_GGML_F32) return ((const float*)p)[i];
    else if constexpr (T == MIVI_GGML_F16) return half_bits_to_f32(((const uint16_t*)p)[i]);
    else return bf16_bits_to_f32(((const uint16_t*)p)[i]);
}

template <int T>
__device__ __forceinline__ uint32_t half_type_bits(float v) {
    if constexpr (T == MIVI_GGML_F16) return f32_to_half_bits(v);
    else return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v);
}

// 8 values from element i on; `wide`: the address is 16-byte aligned.
template <int T>
__device__ __forceinline__ void load8(const void* p, int64_t i, bool wide, float (&x)[8]) {
    if (!wide) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = load_elem<T>(p, i + e);
    } else if constexpr (T == MIVI_GGML_F32) {
        const f32x4 a = *(const f32x4*)((const float*)p + i), b = *(const f32x4*)((const float*)p + i + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = a[e], x[e + 4] = b[e];
    } else {
        const u32x4 w = *(const u32x4*)((const uint16_t*)p + i);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[2 * e] = T == MIVI_GGML_F16 ? half_bits_to_f32(w[e]) : bf16_bits_to_f32(w[e]);
            x[2 * e + 1] = T == MIVI_GGML_F16 ? half_bits_to_f32(w[e] >> 16) : bf16_bits_to_f32(w[e] >> 16);
        }
    }
}

// N (4 or 8) values to element i on; `wide`: the address is aligned to the
// N values' bytes, 16 at most.
template <int T, int N>
__device__ __forceinline__ void store_n(void* p, int64_t i, bool wide, const float (&x)[N]) {
    if constexpr (T == MIVI_GGML_F32) {
        if (wide) {
#pragma unroll
            for (int e = 0; e < N; e += 4) *(f32x4*)((float*)p + i + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) ((float*)p)[i + e] = x[e];
        }
    } else {
        uint32_t w[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; e++) w[e] = half_type_bits<T>(x[2 * e]) | half_type_bits<T>(x[2 * e + 1]) << 16;
        uint16_t* o = (uint16_t*)p + i;
        if (wide) {
            if constexpr (N == 8) *(u32x4*)o = u32x4{w[0], w[1], w[2], w[3]};
            else *(u32x2*)o = u32x2{w[0], w[1]};
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) o[e] = (uint16_t)(w[e / 2] >> (e % 2 * 16));
        }
    }
}

// --------------------------------------------------------------- append
// Value i of a quad of lanes' neighbour (quad_perm).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}

// The codes of 8 values of a block whose other 24 the quad's lanes hold, each
// 0..15, and the block's scale as fp16 bits.
__device__ __forceinline__ uint32_t quantise8(const float (&in)[8], int (&code)[8]) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = in[e] == in[e] ? fminf(fmaxf(in[e], -kMaxValue), kMaxValue) : 0.f;
    }
    float hi = x[0], lo = x[0];
#pragma unroll
    for (int e = 1; e < 8; e++) hi = fmaxf(hi, x[e]), lo = fminf(lo, x[e]);
    hi = fmaxf(hi, dpp_mov<0xB1>(hi));
    hi = fmaxf(hi, dpp_mov<0x4E>(hi));
    lo = fminf(lo, dpp_mov<0xB1>(lo));
    lo = fminf(lo, dpp_mov<0x4E>(lo));
    const float m = hi >= -lo ? hi : lo;
    const float y = fminf(fmaxf(m * -0.125f, -kMaxScale), kMaxScale);
    const uint32_t dh = f32_to_half_bits((float)(__bf16)y);
    const float d = half_bits_to_f32(dh);
    // rint(x / d): the estimate from the reciprocal is at most one off, and the
    // remainder x - n d says which way (one fma: exact enough that its sign
    // against +- d / 2 is right, d / 2 being representable); ties to even
    const float r = d != 0.f ? 1.0f / d : 0.f, half = 0.5f * fabsf(d);
    const float step = d < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float n = rintf(x[e] * r);
        const float rem = fmaf(-n, d, x[e]);
        const float ar = fabsf(rem);
        if (ar > half || (ar == half && ((int)n & 1))) n += rem > 0.f ? step : -step;
        n = d != 0.f ? fminf(fmaxf(n, -8.f), 7.f) : 0.f;
        code[e] = (int)n + 8;
    }
    return dh;
}

// One lane 8 dimensions (a block's quarter) of one row and head, K or V
// (blockIdx.y); lanes of a quad one block.
template <int T>
__global__ void __launch_bounds__(256) kv_q4_append_kernel(Q4Batch a, const void* k, const void* v, int64_t k_row,
                                                           int64_t k_head, int64_t v_row, int64_t v_head, int rows,
                                                           int wide_k, int wide_v) {
    const int hd = a.hd, nb = hd / 32, per = a.n_kv * nb * 4;
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row64 = idx / per;
    if (row64 >= rows) return;  // a quad leaves as a whole: per is a multiple of 4
    const int row = (int)row64, rest = (int)(idx - row64 * per);
    const int c = rest & 3, b = (rest >> 2) % nb, h = (rest >> 2) / nb;
    const int s = seq_of(a, row);
    int pos;
    if (s < 0 || !row_pos(a, s, row, &pos)) return;
    uint8_t* g = group_ptr(a, s, h, pos / kGroup);
    if (!g) return;
    const bool is_v = blockIdx.y != 0;
    const int t = pos % kGroup;
    float x[8];
    int code[8];
    load8<T>(is_v ? v : k, (int64_t)row * (is_v ? v_row : k_row) + h * (is_v ? v_head : k_head) + b * 32 + c * 8,
             is_v ? wide_v : wide_k, x);
    const uint32_t d = quantise8(x, code);
    if (!is_v) {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) w |= (uint32_t)code[e] << (4 * (e / 2) + 16 * (e % 2));
        *(uint32_t*)(g + q4_at(nb, b, t % 16 + 16 * c) + t / 16 * 4) = w;
        if (c == 0) *(uint16_t*)(g + 32 * hd + 2 * (t % 16 * 2 * nb + t / 16 * nb + b)) = (uint16_t)d;
    } else {
        // lanes 0 and 1 hold dimensions 0..15 of the block, lanes 2 and 3 the
        // ones 16 further: a lane stores four of the eight pairs it can form
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) w |= (uint32_t)code[e] << (4 * e);
        const uint32_t o = dpp_u32<0x4E>(w);  // lane ^ 2
        const uint32_t lo = c < 2 ? w : o, hi = c < 2 ? o : w;
        const int byte = 16 * hd + t / 16 * 4 + ((t & 1) * 2 | (t >> 1 & 1));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = (c >> 1) * 4 + i, n = (c & 1) * 8 + e;
            g[byte + q4_at(nb, b, n + 16 * (t % 16 / 4))] = (uint8_t)((lo >> (4 * e) & 15) | (hi >> (4 * e) & 15) << 4);
        }
        if (c == 0)
            *(uint16_t*)(g + 34 * hd + 2 * (b * 32 + t % 16 / 4 * 8 + t / 16 * 4 + t % 4)) = (uint16_t)d;
    }
}

// ----------------------------------------------------------------- read
template <int T>
__global__ void __launch_bounds__(256) kv_q4_read_kernel(Q4Batch a, void* k, void* v, int64_t k_row, int64_t k_head,
                                                         int64_t v_row, int64_t v_head, int rows, int wide_k,
                                                         int wide_v) {
    const int hd = a.hd, nb = hd / 32, per = a.n_kv * nb * 4;
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row64 = idx / per;
    if (row64 >= rows) return;
    const int row = (int)row64, rest = (int)(idx - row64 * per);
    const int c = rest & 3, b = (rest >> 2) % nb, h = (rest >> 2) / nb;
    const int s = seq_of(a, row);
    if (s < 0) return;
    const bool is_v = blockIdx.y != 0;
    int pos;
    const uint8_t* g = row_pos(a, s, row, &pos) ? group_ptr(a, s, h, pos / kGroup) : nullptr;
    float x[8] = {};
    if (g) {
        const int t = pos % kGroup;
        if (!is_v) {
            const uint32_t w = *(const uint32_t*)(g + q4_at(nb, b, t % 16 + 16 * c) + t / 16 * 4);
            const float d = half_bits_to_f32(*(const uint16_t*)(g + 32 * hd + 2 * (t % 16 * 2 * nb + t / 16 * nb + b)));
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = (float)((int)(w >> (4 * (e / 2) + 16 * (e % 2)) & 15) - 8) * d;
        } else {
            const int byte = 16 * hd + t / 16 * 4 + ((t & 1) * 2 | (t >> 1 & 1));
            const float d = half_bits_to_f32(
                *(const uint16_t*)(g + 34 * hd + 2 * (b * 32 + t % 16 / 4 * 8 + t / 16 * 4 + t % 4)));
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t w = g[byte + q4_at(nb, b, (c & 1) * 8 + e + 16 * (t % 16 / 4))];
                x[e] = (float)((int)(w >> (c / 2 * 4) & 15) - 8) * d;
            }
        }
    }
    store_n<T, 8>(is_v ? v : k, (int64_t)row * (is_v ? v_row : k_row) + h * (is_v ? v_head : k_head) + b * 32 + c * 8,
                  is_v ? wide_v : wide_k, x);
}

// ------------------------------------------------------------ attention
struct Q4Attn {
    Q4Batch b;
    const void* q;
    void* out;
    int64_t q_row, q_head, o_row, o_head;
    int type, wide_q, wide_o;
    int n_heads, gq;      // gq: query heads of a kv head
    int rows, max_rows, tiles;  // row tiles of 16 (row, query head) pairs a sequence and kv head
    int nsplit, window;
    float scale;
    float* part_acc;      // [rows * n_heads][nsplit][hd]
    float* part_ml;       // [rows * n_heads][nsplit][2]
};

// Codes of one dword as four fp16 pairs 16 + c: nibbles (0, 4), (1, 5), (2, 6),
// (3, 7) into the top mantissa bits of 16.0.
__device__ __forceinline__ half2v pair16(uint32_t w, int i) {
    const uint32_t x = i == 0 ? w << 6 : i == 1 ? w << 2 : i == 2 ? w >> 2 : w >> 6;
    return __builtin_bit_cast(half2v, (x & 0x03C003C0u) | 0x4C004C00u);
}
// (16 + c) d - 24 d = (c - 8) d, exact; dm = -24 d (10 significant bits, exact)
__device__ __forceinline__ half2v held(half2v x, half2v d, half2v dm) { return __builtin_elementwise_fma(x, d, dm); }

__device__ __forceinline__ float load_q(const Q4Attn& a, int64_t i) {
    return a.type == MIVI_GGML_F32   ? load_elem<MIVI_GGML_F32>(a.q, i)
           : a.type == MIVI_GGML_F16 ? load_elem<MIVI_GGML_F16>(a.q, i)
                                     : load_elem<MIVI_GGML_BF16>(a.q, i);
}
__device__ __forceinline__ void load_q8(const Q4Attn& a, int64_t i, float (&x)[8]) {
    if (a.type == MIVI_GGML_F32) load8<MIVI_GGML_F32>(a.q, i, a.wide_q, x);
    else if (a.type == MIVI_GGML_F16) load8<MIVI_GGML_F16>(a.q, i, a.wide_q, x);
    else load8<MIVI_GGML_BF16>(a.q, i, a.wide_q, x);
}
__device__ __forceinline__ void store_o4(const Q4Attn& a, int64_t i, const float (&x)[4]) {
    if (a.type == MIVI_GGML_F32) store_n<MIVI_GGML_F32, 4>(a.out, i, a.wide_o, x);
    else if (a.type == MIVI_GGML_F16) store_n<MIVI_GGML_F16, 4>(a.out, i, a.wide_o, x);
    else store_n<MIVI_GGML_BF16, 4>(a.out, i, a.wide_o, x);
}

// value of the quarters of a lane's query row (lanes l mod 16 + 16 j), joined
__device__ __forceinline__ float quarters_max(float v) {
    float x, y;
    swap16(v, x, y);
    v = fmaxf(x, y);
    swap32(v, x, y);
    return fmaxf(x, y);
}
__device__ __forceinline__ float quarters_sum(float v) {
    float x, y;
    swap16(v, x, y);
    v = x + y;
    swap32(v, x, y);
    return x + y;
}

// The largest finite exponent normalisation of a query row: the power of two
// that puts its largest magnitude into [2^14, 2^15), so that fp16 holds 11 bits
// of every value down to 2^-28 of the largest (23 bits with the second plane).
// A row with an infinity or NaN, or of zeros, stays as it is.
__device__ __forceinline__ int row_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    if (u == 0 || u >= 0x7F800000u) return 0;
    return 14 - ilogbf(amax);
}

// A group's codes and scales as lane l loads them.
template <int NB>
struct Q4Raw {
    uint32_t k[2 * NB], v[2 * NB], ks[NB], vs[4 * NB];
};
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {  // 4-byte aligned
    if constexpr (N >= 4) {
        const u32x4_a4 x = *(const u32x4_a4*)p;
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = x[i];
        load_words<N - 4>(p + 16, w + 4);
    } else if constexpr (N >= 2) {
        const u32x2_a4 x = *(const u32x2_a4*)p;
        w[0] = x[0], w[1] = x[1];
        load_words<N - 2>(p + 8, w + 2);
    } else if constexpr (N == 1) {
        w[0] = *(const uint32_t*)p;
    }
}
template <int NB>
__device__ __forceinline__ void load_codes(const uint8_t* p, int lane, uint32_t (&w)[2 * NB]) {
#pragma unroll
    for (int i = 0; i < NB / 2; i++) {
        const u32x4 x = *(const u32x4*)(p + i * 1024 + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) w[4 * i + j] = x[j];
    }
    if constexpr (NB % 2) {
        const u32x2 x = *(const u32x2*)(p + NB / 2 * 1024 + lane * 8);
        w[2 * NB - 2] = x[0], w[2 * NB - 1] = x[1];
    }
}
template <int NB>
__device__ __forceinline__ void load_group(const uint8_t* g, int lane, Q4Raw<NB>& r) {
    constexpr int hd = 32 * NB;
    load_codes<NB>(g, lane, r.k);
    load_words<NB>(g + 32 * hd + lane % 16 * 4 * NB, r.ks);
    load_codes<NB>(g + 16 * hd, lane, r.v);
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const u32x4 x = *(const u32x4*)(g + 34 * hd + (b * 4 + lane / 16) * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) r.vs[4 * b + j] = x[j];
    }
}

__device__ __forceinline__ half2v as_half2(uint32_t w) { return __builtin_bit_cast(half2v, w); }
__device__ __forceinline__ half8 join8(half2v a, half2v b, half2v c, half2v d) {
    return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

constexpr float kPShift = 15;  // weights are held times 2^15: fp16 reaches 2^-39 of the largest

// Row tiles of 16 (row, query head) pairs f = i gq + head of one sequence and
// kv head over a share of its groups; wave w of the four takes every fourth
// group. One pass with the running maximum and sum of the softmax; P is the
// planes of the query rows and of the weights (2 for f32 values: each plane an
// fp16 operand, 22 bits in all; 1 for fp16 and bf16 values, whose queries fp16
// holds exactly and whose outputs have no more bits than the weights).
template <int NB, int P>
__global__ void __launch_bounds__(256) kv_q4_attn_kernel(Q4Attn a) {
    constexpr int hd = 32 * NB;
    __shared__ float red_ml[4][16][2];
    __shared__ float red_acc[4][16][hd + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quarter = lane >> 4;
    int64_t id = blockIdx.x;
    const int split = (int)(id % a.nsplit);
    id /= a.nsplit;
    const int tile = (int)(id % a.tiles);
    id /= a.tiles;
    const int h = (int)(id % a.b.n_kv), s = (int)(id / a.b.n_kv);
    const int start = a.b.starts[s], count = a.b.starts[s + 1] - start;
    if (start < 0 || start >= a.rows) return;
    const int64_t pairs = (int64_t)min(min(count, a.max_rows), a.rows - start) * a.gq;
    const int64_t f0 = (int64_t)tile * 16;
    if (f0 >= pairs) return;
    const int len = a.b.lens[s];
    // positions lo .. hi - 1 are seen by this lane's row; those of the tile's
    // first and last row bound all others
    const int64_t first_pos = (int64_t)len - count;
    auto see_hi = [&](int64_t i) { return (int)min<int64_t>(max<int64_t>(first_pos + i + 1, 0), a.b.cap); };
    auto see_lo = [&](int64_t i) {
        return a.window ? (int)min<int64_t>(max<int64_t>(first_pos + i + 1 - a.window, 0), a.b.cap) : 0;
    };
    const int64_t f = f0 + col;
    const bool active = f < pairs;
    const int64_t row_i = (active ? f : pairs - 1) / a.gq;
    const int head = h * a.gq + (int)((active ? f : pairs - 1) - row_i * a.gq);
    const int lo = see_lo(row_i), hi = see_hi(row_i);
    const int64_t i_first = f0 / a.gq, i_last = (min<int64_t>(f0 + 15, pairs - 1)) / a.gq;
    const int lo_all = see_lo(i_last), hi_all = see_hi(i_first);  // seen by every row: lo_all .. hi_all - 1
    const int valid = min(max(len, 0), a.b.cap);
    const int g_lo = see_lo(i_first) / kGroup, g_hi = (see_hi(i_last) + kGroup - 1) / kGroup;
    const int per = (max(g_hi - g_lo, 0) + a.nsplit - 1) / a.nsplit;
    const int g_begin = g_lo + split * per, g_end = min(g_begin + per, g_hi);

    // the query row as B operands: block b, dimensions 8 quarter .. + 7
    half8 q[P][NB];
    float sc;
    {
        float x[NB][8];
        float amax = 0.f;
        const int64_t base = (int64_t)(start + row_i) * a.q_row + head * a.q_head + quarter * 8;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            load_q8(a, base + b * 32, x[b]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float m = fabsf(x[b][e]);
                amax = m == m ? fmaxf(amax, m) : __builtin_inff();
            }
        }
        amax = quarters_max(amax);
        const int ex = row_exponent(amax);
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = ldexpf(x[b][e], ex);
                const _Float16 top = (_Float16)y;
                q[0][b][e] = top;
                if constexpr (P == 2) q[1][b][e] = (_Float16)(y - (float)top);
            }
        }
        sc = ldexpf(a.scale * 1.44269504088896340736f, -ex);
    }

    float m_run = -__builtin_inff(), l_run = 0.f;
    f32x4 acc[2 * NB];
#pragma unroll
    for (int j = 0; j < 2 * NB; j++) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int g = g_begin + wave; g < g_end; g += 4) {
        const uint8_t* gp = group_ptr(a.b, s, h, g);
        if (!gp) continue;  // no page there: not seen
        Q4Raw<NB> r;
        load_group<NB>(gp, lane, r);
        // scores: rows tokens, columns query rows
        f32x4 st[2];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            st[half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int si = half * NB + b;
                const _Float16 ds = __builtin_bit_cast(half2v, r.ks[si / 2])[si % 2];
                const half2v d = {ds, ds}, dm = d * (_Float16)-24;
                const uint32_t w = r.k[2 * b + half];
                const half8 kk = join8(held(pair16(w, 0), d, dm), held(pair16(w, 1), d, dm),
                                       held(pair16(w, 2), d, dm), held(pair16(w, 3), d, dm));
#pragma unroll
                for (int p = 0; p < P; p++)
                    st[half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q[p][b], st[half], 0, 0, 0);
            }
        }
        const int t0 = g * kGroup;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = st[i / 4][i % 4] * sc;
        if (t0 < lo_all || t0 + kGroup > hi_all) {  // some row sees only a part
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int t = t0 + i / 4 * 16 + quarter * 4 + i % 4;
                x[i] = t >= lo && t < hi ? x[i] : -__builtin_inff();
            }
            // what is behind the sequence's end is anything: no scale may be NaN
            if (t0 + kGroup > valid) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int t = t0 + j / 2 * 16 + quarter * 4 + j % 2 * 2;
                    const uint32_t keep = (t < valid ? 0xFFFFu : 0u) | (t + 1 < valid ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int b = 0; b < NB; b++) r.vs[4 * b + j] &= keep;
                }
            }
        }
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < 8; i++) mx = fmaxf(mx, x[i]);
        mx = quarters_max(mx);
        if (__any(mx > m_run)) {
            const float m_new = fmaxf(m_run, mx);
            const float m_ref = m_new == -__builtin_inff() ? 0.f : m_new;
            const float f_old = exp2f(m_run - m_ref);
            m_run = m_new;
            l_run *= f_old;
#pragma unroll
            for (int j = 0; j < 2 * NB; j++) acc[j] *= f_old;
        }
        const float m_ref = (m_run == -__builtin_inff() ? 0.f : m_run) - kPShift;
        half8 pw[P];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float w = exp2f(x[i] - m_ref);
            l_run += w;
            const _Float16 top = (_Float16)w;
            pw[0][i] = top;
            if constexpr (P == 2) pw[1][i] = (_Float16)(w - (float)top);
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            half2v d[4], dm[4];
#pragma unroll
            for (int j = 0; j < 4; j++) d[j] = as_half2(r.vs[4 * b + j]), dm[j] = d[j] * (_Float16)-24;
#pragma unroll
            for (int z = 0; z < 2; z++) {
                const uint32_t w0 = r.v[2 * b], w1 = r.v[2 * b + 1];
                const half8 vv = join8(held(pair16(w0, z), d[0], dm[0]), held(pair16(w0, z + 2), d[1], dm[1]),
                                       held(pair16(w1, z), d[2], dm[2]), held(pair16(w1, z + 2), d[3], dm[3]));
#pragma unroll
                for (int p = 0; p < P; p++)
                    acc[2 * b + z] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, pw[p], acc[2 * b + z], 0, 0, 0);
            }
        }
    }
    l_run = quarters_sum(l_run);

    // join the four waves
    if (quarter == 0) red_ml[wave][col][0] = m_run, red_ml[wave][col][1] = l_run;
#pragma unroll
    for (int j = 0; j < 2 * NB; j++) *(f32x4*)&red_acc[wave][col][j * 16 + quarter * 4] = acc[j];
    __syncthreads();
    constexpr int kQuads = hd / 4;
    for (int u = threadIdx.x; u < 16 * kQuads; u += 256) {
        const int c = u / kQuads, d4 = u % kQuads * 4;
        const int64_t fc = f0 + c;
        if (fc >= pairs) continue;
        float m = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < 4; w++) m = fmaxf(m, red_ml[w][c][0]);
        const float m_ref = m == -__builtin_inff() ? 0.f : m;
        float l = 0.f, o[4] = {};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float e = exp2f(red_ml[w][c][0] - m_ref);
            l += e * red_ml[w][c][1];
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = fmaf(e, red_acc[w][c][d4 + i], o[i]);
        }
        const int64_t i = fc / a.gq;
        const int hh = h * a.gq + (int)(fc - i * a.gq);
        if (a.nsplit == 1) {
            const float inv = l == 0.f ? 0.f : 1.0f / l;  // a row that sees nothing is zero
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] *= inv;
            store_o4(a, (int64_t)(start + i) * a.o_row + hh * a.o_head + d4, o);
        } else {
            const int64_t p = ((int64_t)(start + i) * a.n_heads + hh) * a.nsplit + split;
            *(f32x4*)(a.part_acc + p * hd + d4) = f32x4{o[0], o[1], o[2], o[3]};
            if (d4 == 0) a.part_ml[2 * p] = m, a.part_ml[2 * p + 1] = l;
        }
    }
}

// The shares of a (row, head) joined: a quarter wave of hd / 4 lanes each.
__global__ void __launch_bounds__(256) kv_q4_join_kernel(Q4Attn a, int rows) {
    const int hd = a.b.hd, quads = hd / 4;
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t pr = u / quads;
    const int d4 = (int)(u - pr * quads) * 4;
    if (pr >= (int64_t)rows * a.n_heads) return;
    const int row = (int)(pr / a.n_heads), head = (int)(pr - (int64_t)row * a.n_heads);
    const int s = seq_of(a.b, row);
    if (s < 0 || row - a.b.starts[s] >= a.max_rows) return;
    const float* ml = a.part_ml + pr * a.nsplit * 2;
    const float* pa = a.part_acc + pr * a.nsplit * hd + d4;
    float m = -__builtin_inff();  // never NaN: a NaN score is in the sums alone
    for (int i = 0; i < a.nsplit; i++) m = fmaxf(m, ml[2 * i]);
    const float m_ref = m == -__builtin_inff() ? 0.f : m;
    float l = 0.f, o[4] = {};
    for (int i = 0; i < a.nsplit; i++) {
        const float e = exp2f(ml[2 * i] - m_ref);
        l += e * ml[2 * i + 1];
        const f32x4 x = *(const f32x4*)(pa + (int64_t)i * hd);
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = fmaf(e, x[j], o[j]);
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] *= inv;
    store_o4(a, (int64_t)row * a.o_row + head * a.o_head + d4, o);
}

// ----------------------------------------------------------- host checks
constexpr size_t kMaxPageTokens = 1024;

bool head_dim_ok(size_t hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 192 || hd == 256; }

size_t type_bytes(int32_t t) { return t == MIVI_GGML_F32 ? 4 : t == MIVI_GGML_F16 || t == MIVI_GGML_BF16 ? 2 : 0; }

// Elements from the first to the last of rows x heads x hd, or SIZE_MAX.
size_t span(size_t rows, size_t row_stride, size_t heads, size_t head_stride, size_t hd) {
    size_t a, b, c;
    if (__builtin_mul_overflow(rows - 1, row_stride, &a) || __builtin_mul_overflow(heads - 1, head_stride, &b) ||
        __builtin_add_overflow(a, b, &c) || __builtin_add_overflow(c, hd, &c) || c > (size_t)INT64_MAX / 8)
        return SIZE_MAX;
    return c;
}

int32_t check_tensor(const char* what, const void* p, size_t len, int32_t type, size_t rows, size_t row_stride,
                     size_t heads, size_t head_stride, size_t hd, bool written) {
    const size_t need = span(rows, row_stride, heads, head_stride, hd);
    if (need == SIZE_MAX) return err_overflow();
    if (len < need) return err_buffer_too_small(need, len);
    if (!p) return set_error(MIVI_ERR_INVALID_ARGUMENT, "null %s", what);
    if ((uintptr_t)p % type_bytes(type)) return set_error(MIVI_ERR_INVALID_ARGUMENT, "%s not aligned to its type", what);
    // rows and heads that are written must not overlap each other
    if (written && heads > 1 && head_stride < hd)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "%s: head stride %zu < head_dim %zu", what, head_stride, hd);
    if (written && rows > 1) {
        const bool rows_outer = row_stride >= (heads - 1) * head_stride + hd;
        const bool heads_outer = heads > 1 && row_stride >= hd && head_stride >= (rows - 1) * row_stride + hd;
        if (!rows_outer && !heads_outer)
            return set_error(MIVI_ERR_INVALID_ARGUMENT, "%s: rows of stride %zu overlap", what, row_stride);
    }
    return MIVI_OK;
}

// Vector access: pointer and strides multiples of `bytes`.
int wide_ok(const void* p, size_t row_stride, size_t head_stride, size_t elem, size_t bytes) {
    return (uintptr_t)p % bytes == 0 && row_stride * elem % bytes == 0 && head_stride * elem % bytes == 0;
}

int32_t check_geometry(size_t n_kv, size_t hd, size_t page_tokens) {
    if (hd % 32) return err_misaligned(hd, 32);
    if (!head_dim_ok(hd))
        return set_error(MIVI_ERR_UNSUPPORTED, "head_dim %zu: a 4-bit cache has 32, 64, 96, 128, 192 or 256", hd);
    if (page_tokens % kGroup) return err_misaligned(page_tokens, kGroup);
    if (page_tokens == 0 || page_tokens > kMaxPageTokens)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "page of %zu tokens (32 to %zu)", page_tokens, kMaxPageTokens);
    if (n_kv == 0 || n_kv > 65535) return set_error(MIVI_ERR_INVALID_ARGUMENT, "%zu kv heads", n_kv);
    return MIVI_OK;
}

int32_t make_batch(Q4Batch* b, const uint8_t* cache, size_t cache_len, size_t n_kv, size_t hd, size_t page_tokens,
                   const int32_t* pages, size_t pages_stride, size_t pages_per_seq, size_t n_seq,
                   const int32_t* starts, const int32_t* lens, size_t rows) {
    int32_t rc = check_geometry(n_kv, hd, page_tokens);
    if (rc) return rc;
    const size_t page_bytes = mivi_hip_kv_q4_page_bytes(n_kv, hd, page_tokens);
    const size_t n_pages = cache_len / page_bytes;
    if (n_pages == 0) return err_buffer_too_small(page_bytes, cache_len);
    if (n_pages > (size_t)INT32_MAX) return err_overflow();
    size_t cap, table;
    if (n_seq > (size_t)INT32_MAX || rows > (size_t)INT32_MAX || pages_per_seq > (size_t)INT32_MAX ||
        __builtin_mul_overflow(pages_per_seq, page_tokens, &cap) || cap > (size_t)INT32_MAX - 2 * kGroup ||
        __builtin_mul_overflow(n_seq, pages_stride, &table) || table > (size_t)INT64_MAX / 8)
        return err_overflow();
    if (n_seq > 1 && pages_stride < pages_per_seq)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "pages_stride %zu < pages_per_seq %zu", pages_stride, pages_per_seq);
    if (!cache || (pages_per_seq && !pages) || !starts || !lens)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "null argument");
    if ((uintptr_t)cache % 16) return set_error(MIVI_ERR_INVALID_ARGUMENT, "cache not 16-byte aligned");
    if ((uintptr_t)pages % 4 || (uintptr_t)starts % 4 || (uintptr_t)lens % 4)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "table, starts or lens not 4-byte aligned");
    *b = Q4Batch{(uint8_t*)cache, pages,     starts,        lens,    (int64_t)pages_stride, (int64_t)n_pages,
                 (int64_t)page_bytes, (int)n_seq, (int)n_kv, (int)hd, (int)(page_tokens / kGroup), (int)cap};
    return MIVI_OK;
}

// Shares of a sequence's groups: enough workgroups for the card where rows and
// heads make few.
int split_count(size_t n_seq, size_t max_rows, size_t gq, size_t n_kv, size_t cap) {
    const size_t tiles = (max_rows * gq + 15) / 16;
    const size_t wgs = std::max<size_t>(1, n_seq * n_kv * tiles);
    const size_t groups = (cap + kGroup - 1) / kGroup;
    const size_t want = (4 * (size_t)num_cus() + wgs - 1) / wgs;
    return (int)std::max<size_t>(1, std::min<size_t>({want, (groups + 3) / 4, 64}));
}

template <int NB>
void launch_attn(const Q4Attn& a, unsigned grid, int planes, hipStream_t s) {
    if (planes == 2) kv_q4_attn_kernel<NB, 2><<<grid, 256, 0, s>>>(a);
    else kv_q4_attn_kernel<NB, 1><<<grid, 256, 0, s>>>(a);
}

}  // namespace

extern "C" size_t mivi_hip_kv_q4_page_bytes(size_t n_kv_heads, size_t head_dim, size_t page_tokens) {
    if (check_geometry(n_kv_heads, head_dim, page_tokens)) return 0;
    return n_kv_heads * (page_tokens / kGroup) * 36 * head_dim;
}

extern "C" int32_t mivi_hip_kv_q4_append(uint8_t* cache, size_t cache_len, size_t n_kv_heads, size_t head_dim,
                                         size_t page_tokens, const int32_t* pages, size_t pages_stride,
                                         size_t pages_per_seq, size_t n_seq, const int32_t* starts,
                                         const int32_t* lens, int32_t type, const void* k, size_t k_len,
                                         size_t k_row_stride, size_t k_head_stride, const void* v, size_t v_len,
                                         size_t v_row_stride, size_t v_head_stride, size_t rows, void* stream) {
    if (!type_bytes(type)) return err_unsupported(type);
    Q4Batch b;
    int32_t rc = make_batch(&b, cache, cache_len, n_kv_heads, head_dim, page_tokens, pages, pages_stride,
                            pages_per_seq, n_seq, starts, lens, rows);
    if (rc) return rc;
    if (rows == 0 || n_seq == 0) return clear_error();
    if ((rc = check_tensor("k", k, k_len, type, rows, k_row_stride, n_kv_heads, k_head_stride, head_dim, false)) ||
        (rc = check_tensor("v", v, v_len, type, rows, v_row_stride, n_kv_heads, v_head_stride, head_dim, false)))
        return rc;
    const size_t blocks = (rows * n_kv_heads * (head_dim / 8) + 255) / 256;
    if (blocks > (size_t)INT32_MAX) return err_overflow();
    clear_error();
    const size_t e = type_bytes(type);
    const int wk = wide_ok(k, k_row_stride, k_head_stride, e, 16), wv = wide_ok(v, v_row_stride, v_head_stride, e, 16);
    const dim3 grid((unsigned)blocks, 2);
    hipStream_t s = (hipStream_t)stream;
#define APPEND(T)                                                                                                   \
    kv_q4_append_kernel<T><<<grid, 256, 0, s>>>(b, k, v, (int64_t)k_row_stride, (int64_t)k_head_stride,             \
                                                (int64_t)v_row_stride, (int64_t)v_head_stride, (int)rows, wk, wv)
    if (type == MIVI_GGML_F32) APPEND(MIVI_GGML_F32);
    else if (type == MIVI_GGML_F16) APPEND(MIVI_GGML_F16);
    else APPEND(MIVI_GGML_BF16);
#undef APPEND
    MIVI_HIP_CHECK(hipGetLastError());
    return MIVI_OK;
}

extern "C" int32_t mivi_hip_kv_q4_read(const uint8_t* cache, size_t cache_len, size_t n_kv_heads, size_t head_dim,
                                       size_t page_tokens, const int32_t* pages, size_t pages_stride,
                                       size_t pages_per_seq, size_t n_seq, const int32_t* starts, const int32_t* lens,
                                       int32_t type, void* k, size_t k_len, size_t k_row_stride, size_t k_head_stride,
                                       void* v, size_t v_len, size_t v_row_stride, size_t v_head_stride, size_t rows,
                                       void* stream) {
    if (!type_bytes(type)) return err_unsupported(type);
    Q4Batch b;
    int32_t rc = make_batch(&b, cache, cache_len, n_kv_heads, head_dim, page_tokens, pages, pages_stride,
                            pages_per_seq, n_seq, starts, lens, rows);
    if (rc) return rc;
    if (rows == 0 || n_seq == 0) return clear_error();
    if ((rc = check_tensor("k", k, k_len, type, rows, k_row_stride, n_kv_heads, k_head_stride, head_dim, true)) ||
        (rc = check_tensor("v", v, v_len, type, rows, v_row_stride, n_kv_heads, v_head_stride, head_dim, true)))
        return rc;
    const size_t blocks = (rows * n_kv_heads * (head_dim / 8) + 255) / 256;
    if (blocks > (size_t)INT32_MAX) return err_overflow();
    clear_error();
    const size_t e = type_bytes(type);
    const int wk = wide_ok(k, k_row_stride, k_head_stride, e, 16), wv = wide_ok(v, v_row_stride, v_head_stride, e, 16);
    const dim3 grid((unsigned)blocks, 2);
    hipStream_t s = (hipStream_t)stream;
#define READ(T)                                                                                                   \
    kv_q4_read_kernel<T><<<grid, 256, 0, s>>>(b, k, v, (int64_t)k_row_stride, (int64_t)k_head_stride,             \
                                              (int64_t)v_row_stride, (int64_t)v_head_stride, (int)rows, wk, wv)
    if (type == MIVI_GGML_F32) READ(MIVI_GGML_F32);
    else if (type == MIVI_GGML_F16) READ(MIVI_GGML_F16);
    else READ(MIVI_GGML_BF16);
#undef READ
    MIVI_HIP_CHECK(hipGetLastError());
    return MIVI_OK;
}

extern "C" size_t mivi_hip_kv_q4_attention_workspace(size_t n_seq, size_t rows, size_t max_rows, size_t n_heads,
                                                     size_t n_kv_heads, size_t head_dim, size_t max_tokens) {
    if (n_kv_heads == 0 || n_heads == 0 || n_heads % n_kv_heads || rows == 0 || n_seq == 0) return 0;
    max_rows = std::min(max_rows, rows);
    const int ns = split_count(n_seq, max_rows, n_heads / n_kv_heads, n_kv_heads, max_tokens);
    return ns == 1 ? 0 : rows * n_heads * ns * (head_dim + 2) * sizeof(float);
}

extern "C" int32_t mivi_hip_kv_q4_attention(
    int32_t type, void* out, size_t out_len, size_t out_row_stride, size_t out_head_stride, const void* q, size_t q_len,
    size_t q_row_stride, size_t q_head_stride, size_t rows, size_t max_rows, size_t n_heads, float scale,
    size_t window, const uint8_t* cache, size_t cache_len, size_t n_kv_heads, size_t head_dim, size_t page_tokens,
    const int32_t* pages, size_t pages_stride, size_t pages_per_seq, size_t n_seq, const int32_t* starts,
    const int32_t* lens, void* workspace, size_t workspace_bytes, void* stream) {
    if (!type_bytes(type)) return err_unsupported(type);
    Q4Attn a = {};
    int32_t rc = make_batch(&a.b, cache, cache_len, n_kv_heads, head_dim, page_tokens, pages, pages_stride,
                            pages_per_seq, n_seq, starts, lens, rows);
    if (rc) return rc;
    if (n_heads == 0 || n_heads % n_kv_heads || n_heads > 65535)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "%zu heads over %zu kv heads", n_heads, n_kv_heads);
    if (rows == 0 || n_seq == 0 || max_rows == 0) return clear_error();
    if ((rc = check_tensor("q", q, q_len, type, rows, q_row_stride, n_heads, q_head_stride, head_dim, false)) ||
        (rc = check_tensor("out", out, out_len, type, rows, out_row_stride, n_heads, out_head_stride, head_dim, true)))
        return rc;
    max_rows = std::min(max_rows, rows);
    const size_t gq = n_heads / n_kv_heads;
    size_t cap = pages_per_seq * page_tokens;
    const size_t need = mivi_hip_kv_q4_attention_workspace(n_seq, rows, max_rows, n_heads, n_kv_heads, head_dim, cap);
    if (workspace_bytes < need) return err_buffer_too_small(need, workspace_bytes);
    if (need && !workspace) return set_error(MIVI_ERR_INVALID_ARGUMENT, "null workspace");
    if (need && (uintptr_t)workspace % 16)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "workspace not 16-byte aligned");
    const int ns = split_count(n_seq, max_rows, gq, n_kv_heads, cap);
    const size_t tiles = (max_rows * gq + 15) / 16;
    const size_t grid = tiles * n_seq * n_kv_heads * ns;
    const size_t join = (rows * n_heads * (head_dim / 4) + 255) / 256;
    if (grid > (size_t)INT32_MAX || join > (size_t)INT32_MAX) return err_overflow();
    clear_error();
    a.q = q, a.out = out;
    a.q_row = (int64_t)q_row_stride, a.q_head = (int64_t)q_head_stride;
    a.o_row = (int64_t)out_row_stride, a.o_head = (int64_t)out_head_stride;
    a.type = type;
    const size_t e = type_bytes(type);
    a.wide_q = wide_ok(q, q_row_stride, q_head_stride, e, 16);
    a.wide_o = wide_ok(out, out_row_stride, out_head_stride, e, 4 * e);
    a.n_heads = (int)n_heads, a.gq = (int)gq;
    a.rows = (int)rows, a.max_rows = (int)max_rows, a.tiles = (int)tiles;
    a.nsplit = ns;
    a.window = (int)std::min<size_t>(window, (size_t)INT32_MAX);
    a.scale = scale;
    a.part_acc = (float*)workspace;
    a.part_ml = a.part_acc + rows * n_heads * ns * head_dim;
    hipStream_t s = (hipStream_t)stream;
    const int planes = type == MIVI_GGML_F32 ? 2 : 1;
    switch (head_dim / 32) {
        case 1: launch_attn<1>(a, (unsigned)grid, planes, s); break;
        case 2: launch_attn<2>(a, (unsigned)grid, planes, s); break;
        case 3: launch_attn<3>(a, (unsigned)grid, planes, s); break;
        case 4: launch_attn<4>(a, (unsigned)grid, planes, s); break;
        case 6: launch_attn<6>(a, (unsigned)grid, planes, s); break;
        default: launch_attn<8>(a, (unsigned)grid, planes, s); break;
    }
    MIVI_HIP_CHECK(hipGetLastError());
    if (ns > 1) {
        kv_q4_join_kernel<<<(unsigned)join, 256, 0, s>>>(a, (int)rows);
        MIVI_HIP_CHECK(hipGetLastError());
    }
    return MIVI_OK;
}
