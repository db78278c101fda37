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
#include <type_traits>

#include "common.h"

using namespace mivi;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));

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
    uint32_t gpp_inv;          // floor(2^32 / gpp) + 1, 0 for gpp 1
    int cap;                   // positions that the table covers
};

// A group's byte of block b, lane l: two blocks side by side where there are
// two, so that a lane's 16 bytes are one load.
__host__ __device__ constexpr int q4_at(int nb, int b, int lane) {
    return b / 2 < nb / 2 ? b / 2 * 1024 + lane * 16 + b % 2 * 8 : b / 2 * 1024 + lane * 8;
}

// Page of group g of a sequence, g / gpp: exact for gpp <= 32 and g < 2^27.
__device__ __forceinline__ int page_index(const Q4Batch& a, int g) {
    return a.gpp_inv ? (int)__umulhi((uint32_t)g, a.gpp_inv) : g;
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
    const int pi = page_index(a, g);
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
__device__ __forceinline__ uint32_t half_type_bits(float v) {
    if constexpr (T == MIVI_GGML_F16) return f32_to_half_bits(v);
    else return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v);
}

// 8 values from element i on, as they lie; `wide`: the address is 16-byte aligned.
template <int T>
constexpr int kWords8 = T == MIVI_GGML_F32 ? 8 : 4;
template <int T>
__device__ __forceinline__ void load8_words(const void* p, int64_t i, bool wide, uint32_t (&w)[kWords8<T>]) {
    const uint8_t* at = (const uint8_t*)p + i * (T == MIVI_GGML_F32 ? 4 : 2);
    if (wide) {
#pragma unroll
        for (int e = 0; e < kWords8<T>; e += 4) {
            const u32x4 x = *(const u32x4*)(at + 4 * e);
#pragma unroll
            for (int j = 0; j < 4; j++) w[e + j] = x[j];
        }
    } else {
#pragma unroll
        for (int e = 0; e < kWords8<T>; e++)
            w[e] = T == MIVI_GGML_F32 ? ((const uint32_t*)at)[e]
                                      : ((const uint16_t*)at)[2 * e] | (uint32_t)((const uint16_t*)at)[2 * e + 1] << 16;
    }
}
template <int T>
__device__ __forceinline__ void words_to_f32(const uint32_t (&w)[kWords8<T>], float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if constexpr (T == MIVI_GGML_F32) x[e] = __uint_as_float(w[e]);
        else if constexpr (T == MIVI_GGML_F16) x[e] = half_bits_to_f32(w[e / 2] >> (e % 2 * 16));
        else x[e] = bf16_bits_to_f32(w[e / 2] >> (e % 2 * 16));
    }
}

template <int T>
__device__ __forceinline__ void load8(const void* p, int64_t i, bool wide, float (&x)[8]) {
    uint32_t w[kWords8<T>];
    load8_words<T>(p, i, wide, w);
    words_to_f32<T>(w, x);
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
// Largest over the four lanes l mod 16 + 16 j.
__device__ __forceinline__ float quarters_max(float v) {
    float x, y;
    swap16(v, x, y);
    v = fmaxf(x, y);
    swap32(v, x, y);
    return fmaxf(x, y);
}

// Value i of a quad of lanes' neighbour (quad_perm).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}

// Largest over the four lanes of a block: a quad, or the quarters l mod 16 + 16 j.
template <bool QUAD>
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
    if constexpr (QUAD) {
        v = max(v, dpp_u32<0xB1>(v));
        return max(v, dpp_u32<0x4E>(v));
    } else {
        const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(a[0], a[1]);
        const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return max(b[0], b[1]);
    }
}

// Codes of 8 values of a block whose other 24 three more lanes hold, and the
// block's scale as fp16 bits. The codes come as one dword of nibbles: value e at
// nibble e (V), or 2 i at nibble i and 2 i + 1 at nibble 4 + i (K).
//
// Magnitudes are compared as integers: of the bit patterns the largest signed
// one is the largest positive value, the largest unsigned one the negative value
// of largest magnitude, and a NaN or a value past the limit shows in either, so
// that only blocks with one pay for the limits.
//
// c - 8 = rint(x / d), ties to even: t = x / d by the reciprocal and one
// correction is exact wherever x / d is an fp32 number, so at every tie, and a
// sum with 1.5 * 2^23 rounds it. For fp16 and bf16 values nothing else lies so
// near a tie that t could round to it (x / d is no nearer to a half than 2^-15,
// d having 8 bits and x 11). An fp32 x may: there the remainder x - n d, exact in
// one fma, decides.
template <int T, bool QUAD>
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], bool v_order, uint32_t* scale) {
    uint32_t pos = 0, neg = 0;
    const uint32_t most = __float_as_uint(kMaxValue);
    auto extent = [&] {
        int p = 0;
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            p = max(p, max((int)__float_as_uint(x[e]), (int)__float_as_uint(x[e + 1])));
            n = max(n, max(__float_as_uint(x[e]), __float_as_uint(x[e + 1])));
        }
        pos = block_max<QUAD>((uint32_t)p);
        n = block_max<QUAD>(n);
        neg = n & 0x80000000u ? n & 0x7FFFFFFFu : 0u;
    };
    extent();
    if (__any(max(pos, neg) > most)) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -kMaxValue), kMaxValue) : 0.f;
        extent();
    }
    const float m = pos >= neg ? __uint_as_float(pos) : -__uint_as_float(neg);
    const uint32_t dh = f32_to_half_bits((float)(__bf16)(m * -0.125f));
    *scale = dh;
    const float d = half_bits_to_f32(dh), r = d != 0.f ? __builtin_amdgcn_rcpf(d) : 0.f;
    constexpr uint32_t kZero = 0x4B400008u;  // bits of 1.5 * 2^23 + 8: the code is the low nibble
    const float half_d = d != 0.f ? 0.5f * fabsf(d) : __builtin_inff();
    uint32_t u[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float t = x[e] * r, q = fmaf(fmaf(-t, d, x[e]), r, t);
        const float sum = q + __uint_as_float(kZero);
        u[e] = __float_as_uint(sum);
        if constexpr (T == MIVI_GGML_F32) {
            const float n = sum - __uint_as_float(kZero);
            const float rem = fmaf(-n, d, x[e]);
            // past the half, or on it at an odd code: the code beside it
            const float edge = __uint_as_float(__float_as_uint(half_d) - (u[e] & 1));
            const int way = (int)(__float_as_uint(rem) ^ __float_as_uint(d)) >> 31 | 1;
            if (fabsf(rem) > edge) u[e] += way;
        }
        u[e] = min(max(u[e], kZero - 8), kZero + 7);
    }
    // nibbles from the top: each step 16 times the last, the constants out at the end
    uint32_t w = 0;
    if (v_order) {
#pragma unroll
        for (int i = 7; i >= 0; i--) w = (w << 4) + u[i];
    } else {
#pragma unroll
        for (int i = 7; i >= 0; i--) w = (w << 4) + u[i < 4 ? 2 * i : 2 * i - 7];
    }
    return w - (kZero - 8) * 0x11111111u;
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
    uint32_t d;
    load8<T>(is_v ? v : k, (int64_t)row * (is_v ? v_row : k_row) + h * (is_v ? v_head : k_head) + b * 32 + c * 8,
             is_v ? wide_v : wide_k, x);
    const uint32_t w = quantise8<T, true>(x, is_v, &d);
    if (!is_v) {
        *(uint32_t*)(g + q4_at(nb, b, t % 16 + 16 * c) + t / 16 * 4) = w;
        if (c == 0) *(uint16_t*)(g + 32 * hd + 2 * (t % 16 * 2 * nb + t / 16 * nb + b)) = (uint16_t)d;
    } else {
        // lanes 0 and 1 hold dimensions 0..15 of the block, lanes 2 and 3 the
        // ones 16 further: a lane stores four of the eight pairs it can form
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

// ------------------------------------------------------ codes to values
// Codes of one dword as four fp16 pairs 16 + c: nibbles (0, 4), (1, 5), (2, 6),
// (3, 7) into the top mantissa bits of 16.0. The constants are held in
// registers that the compiler does not see through: as literals they cost two
// instructions (and, or) in place of one.
struct Q4Bits {
    uint32_t mask = 0x03C003C0u, sixteen = 0x4C004C00u;
    __device__ __forceinline__ Q4Bits() {
        asm("" : "+s"(mask));
        asm("" : "+v"(sixteen));
    }
    __device__ __forceinline__ half2v pair(uint32_t w, int i) const {
        const uint32_t x = i == 0 ? w << 6 : i == 1 ? w << 2 : i == 2 ? w >> 2 : w >> 6;
        return __builtin_bit_cast(half2v, (x & mask) | sixteen);
    }
};
// (16 + c) d - 24 d = (c - 8) d, exact; dm = -24 d (10 significant bits, exact)
__device__ __forceinline__ half2v held(half2v x, half2v d, half2v dm) { return __builtin_elementwise_fma(x, d, dm); }

__device__ __forceinline__ half2v as_half2(uint32_t w) { return __builtin_bit_cast(half2v, w); }
__device__ __forceinline__ half8 join8(half2v a, half2v b, half2v c, half2v d) {
    return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// K codes of a token's eight dimensions: the A operand of its block.
__device__ __forceinline__ half8 held_k(const Q4Bits& q, uint32_t w, _Float16 ds) {
    const half2v d = {ds, ds}, dm = d * (_Float16)-24;
    return join8(held(q.pair(w, 0), d, dm), held(q.pair(w, 1), d, dm), held(q.pair(w, 2), d, dm),
                 held(q.pair(w, 3), d, dm));
}
// V codes of eight tokens: the A operands of the block's two halves of 16
// dimensions; sc: the tokens' four scale pairs.
__device__ __forceinline__ void held_v(const Q4Bits& q, uint32_t w0, uint32_t w1, const uint32_t* sc, half8 (&v)[2]) {
    half2v d[4], dm[4];
#pragma unroll
    for (int j = 0; j < 4; j++) d[j] = as_half2(sc[j]), dm[j] = d[j] * (_Float16)-24;
#pragma unroll
    for (int z = 0; z < 2; z++)
        v[z] = join8(held(q.pair(w0, z), d[0], dm[0]), held(q.pair(w0, z + 2), d[1], dm[1]),
                     held(q.pair(w1, z), d[2], dm[2]), held(q.pair(w1, z + 2), d[3], dm[3]));
}

// A group's codes and scales as lane l loads them: K or V codes of all blocks,
// the K scales of token l mod 16 in both halves, the V scales of the quarter.
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
template <int NB, int B0 = 0, int B1 = NB>  // blocks B0 .. B1 - 1, B0 even
__device__ __forceinline__ void load_codes(const uint8_t* p, int lane, uint32_t* w) {
#pragma unroll
    for (int b = B0; b < B1; b += 2) {
        if (b + 1 < NB) {
            const u32x4 x = __builtin_nontemporal_load((const u32x4*)(p + b / 2 * 1024 + lane * 16));
#pragma unroll
            for (int j = 0; j < 4; j++) w[2 * (b - B0) + j] = x[j];
        } else {
            const u32x2 x = *(const u32x2*)(p + b / 2 * 1024 + lane * 8);
            w[2 * (b - B0)] = x[0], w[2 * (b - B0) + 1] = x[1];
        }
    }
}
template <int NB>
__device__ __forceinline__ void load_k(const uint8_t* g, int lane, uint32_t (&k)[2 * NB], uint32_t (&ks)[NB]) {
    load_codes<NB>(g, lane, k);
    load_words<NB>(g + 1024 * NB + lane % 16 * 4 * NB, ks);
}
template <int NB, int B0 = 0, int B1 = NB>
__device__ __forceinline__ void load_v(const uint8_t* g, int lane, uint32_t* v, uint32_t* vs) {
    load_codes<NB, B0, B1>(g + 512 * NB, lane, v);
#pragma unroll
    for (int b = B0; b < B1; b++) {
        const u32x4 x = *(const u32x4*)(g + 1088 * NB + (b * 4 + lane / 16) * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) vs[4 * (b - B0) + j] = x[j];
    }
}
template <int NB>
__device__ __forceinline__ _Float16 k_scale(const uint32_t (&ks)[NB], int half, int b) {
    const int i = half * NB + b;
    return as_half2(ks[i / 2])[i % 2];
}

// ------------------------------------------------- whole groups at a time
// Rows that are many: a workgroup takes one group of one sequence, its waves (of
// all workgroups that share the group) one head's K or V after another, the next
// one's loads issued before the present one is worked on. Sequence s has the
// groups' units from U(s) = starts[s] / 32 + 2 s on: its n rows touch at most
// (n - 2) / 32 + 2 groups, and U(s + 1) - U(s) is no less, so no sum over the
// sequences is needed to place them.
//
// 24 bf16 prompts of up to 701 rows, 8 heads of 128 (52 MB in, 15 out): written
// in 21.8 us, 17 vector instructions an element and 64 lanes, read in 15.0; 8
// values a lane wherever they lie took 48 and 36. 8 x 32768 rows of 8 heads of 64
// to fp16 (688 MB): 141 us, 4.9 TB/s, 94 % of a copy's rate.
struct Q4Unit {
    int s, g;      // sequence and group
    bool there;    // whether the table has a page of the cache there
    int64_t off;   // of the group of head 0
    int64_t row0;  // row of the group's token 0
    int t0, t1;    // tokens of the group that are rows of the call
};

// Last s with key(s) <= u (key does not decrease): 64 sequences a look.
template <class Key>
__device__ __forceinline__ int wave_search(int n, int lane, int u, Key key) {
    int lo = 0;
    while (n > 1) {
        const int step = (n + 63) / 64;
        const int64_t i = (int64_t)lane * step;
        const int count = __popcll(__ballot(i < n && key(lo + (int)i) <= u));
        if (count == 0) return lo;
        lo += (count - 1) * step;
        n = min(step, n - (count - 1) * step);
    }
    return lo;
}

__device__ __forceinline__ bool unit_of(const Q4Batch& a, int u, int rows, int lane, Q4Unit* o) {
    const int s = __builtin_amdgcn_readfirstlane(
        wave_search(a.n_seq, lane, u, [&](int i) { return (a.starts[i] >> 5) + 2 * i; }));
    const int start = a.starts[s];
    const int local = u - ((start >> 5) + 2 * s);
    const int64_t count = min<int64_t>((int64_t)a.starts[s + 1] - start, (int64_t)rows - start);
    if (start < 0 || count <= 0 || local < 0) return false;
    const int64_t p0 = (int64_t)a.lens[s] - ((int64_t)a.starts[s + 1] - start);  // position of the first row
    const int64_t g = (p0 >> 5) + local, base = g * kGroup;
    if (base >= p0 + count) return false;
    o->row0 = start + (base - p0);
    o->t0 = (int)max<int64_t>(p0 - base, 0);
    o->t1 = (int)min<int64_t>(p0 + count - base, kGroup);
    o->there = base >= 0 && base < a.cap;
    o->off = 0;
    if (o->there) {
        const int pi = page_index(a, (int)g), page = a.pages[(int64_t)s * a.page_stride + pi];
        o->there = page >= 0 && page < a.n_pages;
        o->off = (int64_t)page * a.page_bytes + ((int)g - pi * a.gpp) * (36 * a.hd);
    }
    return true;
}

// A wave's LDS is its own: its writes before its reads, in the compiler's order
// too.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A group's V codes in LDS: 16 bytes more a quarter of the tokens, so that the
// quarters are in different banks. (Dimensions n and n + 8 of a pair of blocks
// are not, at 128 bytes: a byte store takes two turns, 39 to 48 % of the LDS's
// cycles from 64 dimensions on, which are 4 % of the kernel's.) Pair of blocks i at
// 1088 i, an odd last block alone behind them; lane n + 16 quarter of it at
// n * size + quarter * (16 size + 16) with 16 or 8 bytes a lane.
constexpr int kImage = 4 * 1088;  // bytes of the largest (8 blocks)

template <int T>
__global__ void __launch_bounds__(256) kv_q4_append_groups_kernel(Q4Batch a, const void* k, const void* v,
                                                                  int64_t k_row, int64_t k_head, int64_t v_row,
                                                                  int64_t v_head, int rows, int wide_k, int wide_v) {
    __shared__ __attribute__((aligned(16))) uint8_t image[4][kImage];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Q4Unit u;
    if (!unit_of(a, blockIdx.x, rows, lane, &u) || !u.there) return;
    const bool is_v = wave & 1;
    const int hd = a.hd, nb = hd / 32, t16 = lane & 15, c = lane >> 4;
    const void* x = is_v ? v : k;
    const int64_t rs = is_v ? v_row : k_row, hs = is_v ? v_head : k_head;
    const int wide = is_v ? wide_v : wide_k, step = gridDim.y * 2;
    const int64_t base = (u.row0 + t16) * rs + c * 8;
    const bool in[2] = {t16 >= u.t0 && t16 < u.t1, t16 + 16 >= u.t0 && t16 + 16 < u.t1};
    const bool whole = u.t1 - u.t0 == kGroup;
    uint8_t* img = image[wave];
    auto work = [&](auto kind) {
        constexpr bool kIsV = decltype(kind)::value;
        uint32_t next[4][kWords8<T>];  // [block of the pair][half]
        auto fetch = [&](int h, int b) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int e = 0; e < kWords8<T>; e++) next[i][e] = 0;
                if (in[i % 2] && b + i / 2 < nb) load8_words<T>(x, base + h * hs + i % 2 * 16 * rs + (b + i / 2) * 32, wide, next[i]);
            }
        };
        const int h0 = blockIdx.y * 2 + (wave >> 1);
        if (h0 < a.n_kv) fetch(h0, 0);
        for (int h = h0; h < a.n_kv; h += step) {
            uint8_t* g = a.cache + u.off + (int64_t)h * a.gpp * (36 * hd);
            for (int b = 0; b < nb; b += 2) {
                const bool two = b + 1 < nb;
                float val[4][8];
#pragma unroll
                for (int i = 0; i < 4; i++) words_to_f32<T>(next[i], val[i]);
                if (b + 2 < nb) fetch(h, b + 2);
                else if (h + step < a.n_kv) fetch(h + step, 0);
                uint32_t w[4], d[4];
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = quantise8<T, false>(val[i], kIsV, &d[i]);
                const int off = q4_at(nb, b, lane);  // of the lane's dwords: [block][half]
                if (!kIsV) {
                    if (whole) {
                        if (two) *(u32x4*)(g + off) = u32x4{w[0], w[1], w[2], w[3]};
                        else *(u32x2*)(g + off) = u32x2{w[0], w[1]};
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (in[i % 2] && (i < 2 || two)) *(uint32_t*)(g + off + 4 * i) = w[i];
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (c == 0 && in[i % 2] && (i < 2 || two))
                            *(uint16_t*)(g + 32 * hd + 2 * (t16 * 2 * nb + i % 2 * nb + b + i / 2)) = (uint16_t)d[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (i >= 2 && !two) break;
                        // lanes of quarters 0 and 1 hold dimensions 0..15 of the
                        // block, 2 and 3 the ones 16 further: with the lane 32 away a
                        // lane forms four of the eight pairs: n = n0 + j
                        const auto other = __builtin_amdgcn_permlane32_swap(w[i], w[i], false, false);
                        const uint32_t lo = other[0] >> (c >> 1) * 16, hi = other[1] >> (c >> 1) * 16;
                        const uint32_t even = (lo & 0x0F0Fu) | (hi & 0x0F0Fu) << 4;        // j = 0, 2
                        const uint32_t odd = (lo >> 4 & 0x0F0Fu) | (hi & 0xF0F0u);         // j = 1, 3
                        const int n0 = (c & 1) * 8 + (c >> 1) * 4, size = two ? 16 : 8;
                        const int byte = i / 2 * 8 + i % 2 * 4 + ((t16 & 1) * 2 | (t16 >> 1 & 1));
                        auto put = [&](uint8_t* at) {
                            at[0] = (uint8_t)even, at[2 * size] = (uint8_t)(even >> 8);
                            at[size] = (uint8_t)odd, at[3 * size] = (uint8_t)(odd >> 8);
                        };
                        if (whole) put(img + b / 2 * 1088 + n0 * size + t16 / 4 * (16 * size + 16) + byte);
                        else if (in[i % 2]) put(g + 16 * hd + b / 2 * 1024 + (n0 + t16 / 4 * 16) * size + byte);
                        if (c == 0 && in[i % 2])
                            *(uint16_t*)(g + 34 * hd + 2 * ((b + i / 2) * 32 + t16 / 4 * 8 + i % 2 * 4 + t16 % 4)) = (uint16_t)d[i];
                    }
                }
            }
            if (kIsV && whole) {
                wave_sync();
                for (int i = 0; i < nb / 2; i++)
                    *(u32x4*)(g + 16 * hd + i * 1024 + lane * 16) =
                        *(const u32x4*)(img + i * 1088 + lane % 16 * 16 + lane / 16 * 272);
                if (nb % 2)
                    *(u32x2*)(g + 16 * hd + nb / 2 * 1024 + lane * 8) =
                        *(const u32x2*)(img + nb / 2 * 1088 + lane % 16 * 8 + lane / 16 * 144);
                wave_sync();
            }
        }
    };
    if (is_v) work(std::true_type{});
    else work(std::false_type{});
}

// 8 fp16 values (4 dwords) as values of type T to element i on. LINES: the wave
// stores whole rows, around the caches; pieces of 64 bytes (K) go through L2,
// which joins them (8 x 32768 rows of 64 to fp16: 142 us; all around the caches
// 167, all through them 157).
template <int T, bool LINES>
__device__ __forceinline__ void store8_half(void* p, int64_t i, bool wide, u32x4 w) {
    if (T == MIVI_GGML_F16 && wide) {
        if (LINES) __builtin_nontemporal_store(w, (u32x4*)((uint16_t*)p + i));
        else *(u32x4*)((uint16_t*)p + i) = w;
        return;
    }
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = half_bits_to_f32(w[e / 2] >> (e % 2 * 16));
    store_n<T, 8>(p, i, wide, x);
}

// The held values are fp16 numbers: they are formed as the attention forms them
// and widened. K comes out in rows; V goes through LDS, a row of hd values and 8
// bytes more a token: the quarters of the tokens, which are stored together, are
// in different banks. Reading back, 8 of 16 bytes a lane at a time, is without
// conflicts where 16 lanes hold two tokens (64 dimensions: their rows' 8 bytes
// interleave); elsewhere conflicts are 18 to 24 % of the LDS's cycles, 2 to 4 %
// of the kernel's.
template <int T, int NB>
__global__ void __launch_bounds__(256) kv_q4_read_groups_kernel(Q4Batch a, void* k, void* v, int64_t k_row,
                                                                int64_t k_head, int64_t v_row, int64_t v_head,
                                                                int rows, int wide_k, int wide_v) {
    constexpr int hd = 32 * NB, kRow = hd + 4;
    __shared__ __attribute__((aligned(16))) _Float16 tile[2][32 * kRow];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Q4Unit u;
    if (!unit_of(a, blockIdx.x, rows, lane, &u)) return;
    const bool is_v = wave & 1;
    const int t16 = lane & 15, c = lane >> 4, step = gridDim.y * 2, h0 = blockIdx.y * 2 + (wave >> 1);
    const Q4Bits bits;
    const uint8_t* g0 = a.cache + u.off;
    const int64_t hs = (int64_t)a.gpp * (36 * hd);
    uint32_t w[2 * NB], sc[4 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) w[i] = 0;
#pragma unroll
    for (int i = 0; i < 4 * NB; i++) sc[i] = 0;  // no page: zeros
    if (!is_v) {
        uint32_t(&ks)[NB] = *(uint32_t(*)[NB]) sc;
        const int64_t base = (u.row0 + t16) * k_row + c * 8;
        const bool in[2] = {t16 >= u.t0 && t16 < u.t1, t16 + 16 >= u.t0 && t16 + 16 < u.t1};
        if (u.there && h0 < a.n_kv) load_k<NB>(g0 + h0 * hs, lane, w, ks);
        for (int h = h0; h < a.n_kv; h += step) {
            u32x4 out[2 * NB];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int half = 0; half < 2; half++)
                    out[2 * b + half] = __builtin_bit_cast(u32x4, held_k(bits, w[2 * b + half], k_scale<NB>(ks, half, b)));
            if (u.there && h + step < a.n_kv) load_k<NB>(g0 + (h + step) * hs, lane, w, ks);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int half = 0; half < 2; half++)
                    if (in[half]) store8_half<T, false>(k, base + h * k_head + half * 16 * k_row + b * 32, wide_k, out[2 * b + half]);
        }
    } else {
        _Float16* own = tile[wave >> 1];
        if (u.there && h0 < a.n_kv) load_v<NB>(g0 + h0 * hs, lane, w, sc);
        for (int h = h0; h < a.n_kv; h += step) {
            // lane: dimension t16 of each half block, tokens 4 c + i of each half group
            _Float16* at = own + 4 * c * kRow + t16;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                half8 vv[2];
                held_v(bits, w[2 * b], w[2 * b + 1], &sc[4 * b], vv);
#pragma unroll
                for (int z = 0; z < 2; z++)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        at[(i / 4 * 16 + i % 4) * kRow + b * 32 + z * 16] = vv[z][i];
            }
            if (u.there && h + step < a.n_kv) load_v<NB>(g0 + (h + step) * hs, lane, w, sc);
            wave_sync();
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) {
                const int piece = i * 64 + lane, t = piece / (4 * NB), d = piece % (4 * NB) * 8;
                const u32x2 lo = *(const u32x2*)(own + t * kRow + d), hi = *(const u32x2*)(own + t * kRow + d + 4);
                if (t >= u.t0 && t < u.t1)
                    store8_half<T, true>(v, (u.row0 + t) * v_row + h * v_head + d, wide_v, u32x4{lo[0], lo[1], hi[0], hi[1]});
            }
            wave_sync();
        }
    }
}

// ------------------------------------------------------------ attention
struct Q4Attn {
    Q4Batch b;
    const void* q;
    void* out;
    int64_t q_row, q_head, o_row, o_head;
    int type, wide_q, wide_o;
    int n_heads, gq;            // gq: query heads of a kv head
    int rows, max_rows, tiles;  // row tiles of tile_pairs (row, query head) pairs a sequence and kv head
    int tile_pairs;
    int nsplit;                 // parts of a pair that the workspace has room for
    int chunk;                  // groups of a share of a tile; 0: even shares
    int share_min;              // even shares: groups of the smallest
    int window;
    float scale;
    float* part_acc;            // [rows * n_heads][nsplit][hd]
    float* part_ml;             // [rows * n_heads][nsplit][2]
};

// Row of a pair.
__device__ __forceinline__ int row_of(const Q4Attn& a, int f) { return (int)((uint32_t)f / (uint32_t)a.gq); }

// A query row's blocks, 8 values each at i + 32 b: every load before any use.
template <int NB>
__device__ __forceinline__ void load_row(const Q4Attn& a, int64_t i, float (&x)[NB][8]) {
    if (!a.wide_q) {
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if (a.type == MIVI_GGML_F32) load8<MIVI_GGML_F32>(a.q, i + 32 * b, false, x[b]);
            else if (a.type == MIVI_GGML_F16) load8<MIVI_GGML_F16>(a.q, i + 32 * b, false, x[b]);
            else load8<MIVI_GGML_BF16>(a.q, i + 32 * b, false, x[b]);
        }
    } else if (a.type == MIVI_GGML_F32) {
        f32x4 w[NB][2];
#pragma unroll
        for (int b = 0; b < NB; b++)
            w[b][0] = *(const f32x4*)((const float*)a.q + i + 32 * b), w[b][1] = *(const f32x4*)((const float*)a.q + i + 32 * b + 4);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[b][e] = w[b][e / 4][e % 4];
    } else {
        u32x4 w[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) w[b] = *(const u32x4*)((const uint16_t*)a.q + i + 32 * b);
        const bool f16 = a.type == MIVI_GGML_F16;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t u = w[b][e / 2] >> (e % 2 * 16);
                x[b][e] = f16 ? half_bits_to_f32(u) : bf16_bits_to_f32(u);
            }
    }
}
__device__ __forceinline__ void store_o4(const Q4Attn& a, int64_t i, const float (&x)[4]) {
    if (a.type == MIVI_GGML_F32) store_n<MIVI_GGML_F32, 4>(a.out, i, a.wide_o, x);
    else if (a.type == MIVI_GGML_F16) store_n<MIVI_GGML_F16, 4>(a.out, i, a.wide_o, x);
    else store_n<MIVI_GGML_BF16, 4>(a.out, i, a.wide_o, x);
}

// The power of two that puts a query row's largest magnitude into
// [2^14, 2^15), so that fp16 holds 11 bits of every value down to 2^-28 of the
// largest (22 bits with the second plane). A row with an infinity or NaN, or
// of zeros, stays as it is.
__device__ __forceinline__ int row_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    if (u == 0 || u >= 0x7F800000u) return 0;
    return 14 - ilogbf(amax);
}

// What a sequence's rows see: positions lo(i) .. hi(i) - 1 for row i.
struct Q4Seen {
    int first;  // position of row 0
    int cap, window;
    __device__ __forceinline__ int hi(int i) const { return min(max(first + i + 1, 0), cap); }
    __device__ __forceinline__ int lo(int i) const { return window ? min(max(max(first + i + 1, 0) - window, 0), cap) : 0; }
};

// Groups g_lo .. g_hi - 1 hold what rows i0 .. i1 see.
__device__ __forceinline__ void tile_groups(const Q4Seen& see, int i0, int i1, int* g_lo, int* g_hi) {
    *g_lo = see.lo(i0) / kGroup;
    *g_hi = (see.hi(i1) + kGroup - 1) / kGroup;
}

// A V scale pair j (of 4) of the lane's quarter in a group at t0, without the
// tokens before `from` and from `valid` on: what lies before the first row's
// window or behind the last row is anything, and 0 * NaN is NaN.
__device__ __forceinline__ uint32_t keep_mask(int t0, int quarter, int j, int from, int valid) {
    const int t = t0 + j / 2 * 16 + quarter * 4 + j % 2 * 2;
    return (t >= from && t < valid ? 0xFFFFu : 0u) | (t + 1 >= from && t + 1 < valid ? 0xFFFF0000u : 0u);
}

// A weight is 2^(y - m), y = st sc as an fp32 number. A row's reference m moves
// only when some y is more than kReach above it, and then lies kPShift below the
// largest: no weight passes 2^15, and fp16 resolves 2^-36 of the largest. From
// kFar on m is the largest y itself: kPShift less would round, by 16 at 2^27, and
// weights of infinity or of zero alone would come of it. For the same reason the
// exponent is formed from y, as m was, in two roundings: in one fma the product's
// own rounding, 8 at 2^27, would stand between them. (The second instruction is
// 1 to 2 % of a prompt's time, nothing of a single token's.)
constexpr float kPShift = 11, kReach = 15, kFar = 1 << 20;
constexpr float kUnseen = -3.402823466e38f;  // m of a row that has seen nothing

// 16 (row, query head) pairs as the columns of the products; lane l works on
// column l mod 16. PQ, PW: fp16 planes of the queries and of the weights.
template <int NB, int PQ, int PW>
struct Q4Tile {
    half8 q[PQ][NB];     // B operands: block b, dimensions 8 quarter .. + 7
    float sc;            // a raw score times sc is the exponent to base 2
    float m;             // reference exponent
    f32x4 acc[2 * NB];   // sums of w V: dimensions 16 j + 4 quarter + i
    f32x4 l;             // sums of w, the same in all four
    int lo, hi;          // positions seen

    __device__ __forceinline__ void init(const Q4Attn& a, const Q4Seen& see, int row0, int h, int f, int pairs,
                                         int quarter) {
        const int fc = min(f, pairs - 1);  // columns past the last pair repeat it; they are not stored
        const int i = row_of(a, fc), head = h * a.gq + (fc - i * a.gq);
        lo = see.lo(i), hi = see.hi(i);
        float x[NB][8], amax = 0.f;
        const int64_t base = (int64_t)(row0 + i) * a.q_row + head * a.q_head + quarter * 8;
        const float sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f;
        load_row<NB>(a, base, x);
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = fabsf(x[b][e]);
                amax = v == v ? fmaxf(amax, v) : __builtin_inff();
            }
        }
        amax = quarters_max(amax);
        const int ex = row_exponent(amax);
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = ldexpf(x[b][e], ex) * sign;
                const _Float16 top = (_Float16)y;
                q[0][b][e] = top;
                if constexpr (PQ == 2) q[1][b][e] = (_Float16)(y - (float)top);
            }
        }
        // positive, so that the largest score has the largest exponent and a
        // hidden one's -inf stays that; no more than 2^89, so that no exponent is
        // infinite (raw scores are below 2^38: 256 products of 2^15 and 21760).
        // Raw scores that differ do so by 2^-48 at least, fp16's smallest step
        // squared: past 2^89 the largest has all the weight either way. The scale
        // is brought into range first: log2(e) times it may have no number.
        sc = ldexpf(fabsf(a.scale), -ex) * 1.44269504088896340736f;
        sc = fminf(fmaxf(sc, 1.17549435e-38f), 0x1p89f);
        m = kUnseen;
        l = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 2 * NB; j++) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // The scores of a group (tokens 4 quarter + i of each half) to weights, the
    // B operands of the sums. The maximum over the quarters is formed only when
    // some lane has a score so much larger than its row's reference.
    __device__ __forceinline__ void weigh(const f32x4 (&st)[2], half8 (&w)[PW]) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = st[i / 4][i % 4] * sc;
        float mx = y[0];
#pragma unroll
        for (int i = 1; i < 8; i++) mx = fmaxf(mx, y[i]);
        if (__any(mx - m > kReach)) {  // m + kReach would round
            const float most = quarters_max(mx), m_new = fmaxf(m, most - (fabsf(most) < kFar ? kPShift : 0.f));
            const float f = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= f;
#pragma unroll
            for (int j = 0; j < 2 * NB; j++) acc[j] *= f;
        }
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const f32x2 x = {__builtin_amdgcn_exp2f(y[i] - m), __builtin_amdgcn_exp2f(y[i + 1] - m)};
            const half2v top = __builtin_convertvector(x, half2v);
            w[0][i] = top.x, w[0][i + 1] = top.y;
            if constexpr (PW == 2) {  // x - top, exact, in one instruction each
                const f32x2 rest = {fmaf((float)top.x, -1.f, x.x), fmaf((float)top.y, -1.f, x.y)};
                const half2v low = __builtin_convertvector(rest, half2v);
                w[1][i] = low.x, w[1][i + 1] = low.y;
            }
        }
    }

    // Scores that the row does not see.
    __device__ __forceinline__ void hide(f32x4 (&st)[2], int t0, int quarter) const {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int t = t0 + i / 4 * 16 + quarter * 4 + i % 4;
            st[i / 4][i % 4] = t >= lo && t < hi ? st[i / 4][i % 4] : -__builtin_inff();
        }
    }
};

__device__ __forceinline__ f32x4 mfma16(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ half8 ones8() {
    const _Float16 o = 1;
    return half8{o, o, o, o, o, o, o, o};
}

// What a workgroup knows of its sequence's rows.
struct Q4Rows {
    int start, pairs;
    int from, valid;  // positions that may be seen by a row
    Q4Seen see;
};
__device__ __forceinline__ bool rows_of(const Q4Attn& a, int s, Q4Rows* r) {
    const int start = a.b.starts[s], len = a.b.lens[s];
    const int64_t count = (int64_t)a.b.starts[s + 1] - start;
    r->start = start;
    const int n = start < 0 || start >= a.rows ? 0 : (int)min<int64_t>(count, min(a.max_rows, a.rows - start));
    r->pairs = n * a.gq;  // rows times heads fits 31 bits
    r->see = Q4Seen{(int)max<int64_t>(len - count, INT32_MIN), a.b.cap, a.window};
    r->from = r->see.lo(0), r->valid = r->see.hi(n - 1);
    return r->pairs > 0;
}

// Values d4 .. d4 + 3 of a pair's sums o over the weights' sum l: the output
// (part < 0), or one part of it.
__device__ __forceinline__ void store_pair(const Q4Attn& a, const Q4Rows& r, int h, int f, int part, int d4,
                                           float m, float l, float (&o)[4]) {
    const int i = row_of(a, f), head = h * a.gq + (f - i * a.gq);
    if (part < 0) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;  // a row that sees nothing is zero
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] *= inv;
        store_o4(a, (int64_t)(r.start + i) * a.o_row + head * a.o_head + d4, o);
    } else {
        const int64_t p = ((int64_t)(r.start + i) * a.n_heads + head) * a.nsplit + part;
        *(f32x4*)(a.part_acc + p * a.b.hd + d4) = f32x4{o[0], o[1], o[2], o[3]};
        if (d4 == 0) a.part_ml[2 * p] = m, a.part_ml[2 * p + 1] = l;
    }
}

// A sequence's groups of one head: the page id of a group (loaded well before
// its address is wanted), then the address, null where that is no page of the
// cache. Groups from `end` on have the last one's id and no address.
struct Q4Groups {
    const uint8_t* base;
    const int32_t* table;
    int end;
    __device__ __forceinline__ Q4Groups(const Q4Attn& a, int s, int h, int g_end)
        : base(a.b.cache + (int64_t)h * a.b.gpp * (36 * a.b.hd)), table(a.b.pages + (int64_t)s * a.b.page_stride),
          end(g_end) {}
    __device__ __forceinline__ int id(const Q4Attn& a, int g) const { return table[page_index(a.b, min(g, end - 1))]; }
    __device__ __forceinline__ const uint8_t* at(const Q4Attn& a, int g, int id) const {
        const int64_t off = (int64_t)id * a.b.page_bytes + (g - page_index(a.b, g) * a.b.gpp) * (36 * a.b.hd);
        return g < end && (uint32_t)id < (uint32_t)a.b.n_pages ? base + off : nullptr;
    }
};

// A workgroup's place: a head and sequence, a tile of its pairs, a range of the
// groups that the tile sees, and where its sums go (store_pair).
struct Q4Place {
    Q4Rows r;
    int h, s, part, g_begin, g_end;
    int f0;  // first pair of the tile
};

// Shares of `chunk` groups of a tile; false if this one has no work.
__device__ __forceinline__ bool place_of(const Q4Attn& a, int split, int tile, int head_seq, Q4Place* p) {
    p->part = a.nsplit == 1 ? -1 : split;
    p->h = head_seq % a.b.n_kv, p->s = head_seq / a.b.n_kv;
    p->f0 = tile * a.tile_pairs;
    if (!rows_of(a, p->s, &p->r) || p->f0 >= p->r.pairs) return false;
    int g_lo, g_hi;
    tile_groups(p->r.see, row_of(a, p->f0), row_of(a, min(p->f0 + a.tile_pairs, p->r.pairs) - 1), &g_lo, &g_hi);
    p->g_begin = g_lo + split * a.chunk, p->g_end = min(p->g_begin + a.chunk, g_hi);
    return split == 0 || p->g_begin < p->g_end;  // the join does not read an empty share but the first
}

// Even shares, where a sequence's pairs are one tile: the groups of all
// sequences and heads in one row, sequence by sequence and head by head, cut at
// every `size` and between heads. Each piece is one workgroup's, so that no
// workgroup has more than `size` whatever the lengths. The head that starts at
// x, with i heads before it, has the workgroups from x / size + i on (the next
// one's first is past its last). Every wave forms the cut by itself, 64
// sequences a look. (All positions fit 31 bits: the plan takes other shares
// where they might not.)
struct Q4Cut {
    int total;   // groups of all sequences and heads
    int size;    // of a share
    int lo, n;   // this lane's sequence of the first 64: its first group, its groups
    int before;  // groups of a head of the sequences before it
};
__device__ __forceinline__ int udiv(int a, int b) { return (int)((uint32_t)a / (uint32_t)b); }
__device__ __forceinline__ void seq_groups(const Q4Attn& a, int s, int* lo, int* n) {
    Q4Rows r;
    *lo = *n = 0;
    if (s >= a.b.n_seq || !rows_of(a, s, &r)) return;
    int hi;
    tile_groups(r.see, 0, row_of(a, r.pairs - 1), lo, &hi);
    *n = max(hi - *lo, 0);
}
__device__ __forceinline__ int wave_before(int v, int lane) {  // sum of the lanes before
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    return x - v;
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

__device__ __forceinline__ Q4Cut cut_of(const Q4Attn& a, int lane, int shares) {
    Q4Cut c;
    seq_groups(a, lane, &c.lo, &c.n);
    c.before = wave_before(c.n, lane);
    c.total = lane_value(c.before + c.n, 63);
    int most = c.n;
    for (int base = 64; base < a.b.n_seq; base += 64) {
        int lo, n;
        seq_groups(a, base + lane, &lo, &n);
        c.total += lane_value(wave_before(n, lane) + n, 63);
        most = max(most, n);
    }
    c.total *= a.b.n_kv;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
    most = __builtin_amdgcn_readfirstlane(most);
    // no pair has more parts than the workspace has room for: n groups lie in
    // at most (n - 1) / size + 2 shares
    const int even = udiv(c.total + shares - 1, shares), least = udiv(most + a.nsplit - 2, max(a.nsplit - 1, 1));
    c.size = udiv(max(max(even, least), a.share_min) + a.share_min - 1, a.share_min) * a.share_min;
    return c;
}

// The piece of workgroup u; false if it has none.
__device__ __forceinline__ bool piece_of(const Q4Attn& a, int lane, int shares, int u, Q4Place* p) {
    const Q4Cut c = cut_of(a, lane, shares);
    const int kv = a.b.n_kv;
    int base = 0, lo = c.lo, n = c.n, before = c.before, run = 0;  // run: groups before sequence `base`
    for (;;) {  // the 64 sequences that hold it
        const int next = run + lane_value(before + n, 63);
        if (base + 64 >= a.b.n_seq || udiv(next * kv, c.size) + (base + 64) * kv > u) break;
        run = next;
        base += 64;
        seq_groups(a, base + lane, &lo, &n);
        before = wave_before(n, lane);
    }
    const uint64_t at =
        __ballot(base + lane < a.b.n_seq && udiv((run + before) * kv, c.size) + (base + lane) * kv <= u);
    const int l = at ? 63 - __clzll(at) : 0;
    lo = lane_value(lo, l), n = lane_value(n, l);
    const int x0 = (run + lane_value(before, l)) * kv;
    int h = 0;  // the last head whose first workgroup is u or before
    for (int h0 = 0; h0 < kv; h0 += 64) {
        const int hh = h0 + lane;
        const uint64_t m = __ballot(hh < kv && udiv(x0 + hh * n, c.size) + (base + l) * kv + hh <= u);
        if (m) h = h0 + 63 - __clzll(m);
    }
    const int x = x0 + h * n, first = udiv(x, c.size), last = udiv(x + max(n, 1) - 1, c.size);
    const int part = u - (first + (base + l) * kv + h);
    if (n == 0 || part < 0 || part > last - first || !rows_of(a, base + l, &p->r)) return false;
    p->s = base + l, p->h = h, p->f0 = 0;
    p->part = first == last ? -1 : part;
    p->g_begin = lo + max((first + part) * c.size - x, 0);
    p->g_end = lo + min((first + part + 1) * c.size - x, n);
    return true;
}

// A workgroup's place by even shares (chunk 0), or by shares of a tile: heads and
// sequences next to each other, so that a head's workgroups are on one XCD (and
// its L2) where the heads are a multiple of 8; the last tiles, which see most,
// first.
__device__ __forceinline__ bool head_place(const Q4Attn& a, int lane, int shares, Q4Place* p) {
    if (a.chunk == 0) return piece_of(a, lane, shares, blockIdx.x, p);
    const int heads = a.b.n_kv * a.b.n_seq, id = blockIdx.x / heads;
    return place_of(a, id % a.nsplit, a.tiles - 1 - id / a.nsplit, blockIdx.x % heads, p);
}

// Up to 16 pairs of a sequence and kv head: a workgroup takes a range of their
// groups, each of its four waves every fourth one straight from memory to
// operands, and joins the waves at the end. One pass with the running maximum
// and sum of the softmax. Planes: two hold 22 bits of a value, one 11. Queries
// of 16 bits need one (bf16 has 8 bits, and past 2^-28 of a row's largest what
// fp16 lacks is 2^-39 of that). Weights rounded to 11 bits put an error of about
// 2^-12 of sum w |v| / sqrt(tokens) on an output: beside an fp16 output's own
// rounding that is 1.1 to 1.5 times its rms error, so fp16 takes two (64 ragged
// sequences of up to 8192, 8 heads of 128: 76 -> 84 us, prompts of 32768 2.26 ->
// 2.88 ms; the rms error is then the rounding's); beside a bf16 output's it is 1 %
// at most, so bf16 takes one.
//
// K of the next group is on its way during the sums, V during the scores, and
// page ids two groups ahead of that.
//
// Bound: about 210 (hd 64, two planes) to 300 (hd 128, one) vector instructions
// a group, half of them codes to values, 76 and 62 % of the cycles. 8 sequences of
// 32768 tokens, 8 heads of 64, f32: 40 us, 151 MB, 3.8 TB/s (the loads alone took
// 28 us of 41). 64 ragged sequences of up to 8192, 8 heads of 128, bf16:
// 69 us, 297 MB, 4.3 TB/s. No faster: the next group's scores formed beside this
// one's sums (46 us where the kernel took 42), five waves a SIMD (45), four groups'
// scores in sets of four columns (fewer exponentials, two waves a SIMD: 41).
//
// Waves a SIMD that the registers are held to: 17 nb words of codes, scales and
// sums and 4 nb a plane of queries beside about 40 others; 4 where the weights
// have a plane more (64 ragged fp16 sequences, 8 heads of 128: three waves 84 us,
// four with spills 88).
constexpr int step_waves(int nb, int pq, int pw) {
    const int words = nb * (17 + 4 * pq) + 4 * (pw - pq);
    return words <= 84 ? 4 : words <= 102 ? 3 : 2;
}
template <int NB, int PQ, int PW>
__global__ void __launch_bounds__(256, step_waves(NB, PQ, PW)) kv_q4_step_kernel(Q4Attn a, int shares) {
    constexpr int hd = 32 * NB, NW = 4;
    __shared__ float red_ml[NW][16][2];
    __shared__ float red_acc[NW][16][hd + 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quarter = lane >> 4;
    Q4Place pl;
    if (!head_place(a, lane, shares, &pl)) return;
    const Q4Rows& r = pl.r;
    const int lo_all = r.see.lo(row_of(a, r.pairs - 1)), hi_all = r.see.hi(0);  // seen by every row: lo_all .. hi_all - 1
    const Q4Groups groups(a, pl.s, pl.h, pl.g_end);
    const Q4Bits bits;
    Q4Tile<NB, PQ, PW> t;
    uint32_t k[2 * NB], ks[NB], v[2 * NB], vs[4 * NB];
    int g = pl.g_begin + wave;
    const uint8_t *gp = nullptr, *next = nullptr;
    int id = -1;  // page id of the group after next
    if (g < pl.g_end) {
        const int id0 = groups.id(a, g), id1 = groups.id(a, g + NW);
        id = groups.id(a, g + 2 * NW);
        gp = groups.at(a, g, id0), next = groups.at(a, g + NW, id1);
        // loads go somewhere in any case: a group that is not there is read as
        // the cache's first, and hidden
        load_k<NB>(gp ? gp : a.b.cache, lane, k, ks);
        load_v<NB>(gp ? gp : a.b.cache, lane, v, vs);
    }
    t.init(a, r.see, r.start, pl.h, col, r.pairs, quarter);

    for (; g < pl.g_end; g += NW) {
        const uint8_t* from = next ? next : a.b.cache;
        const uint8_t* after = groups.at(a, g + 2 * NW, id);
        id = groups.id(a, g + 3 * NW);
        // scores: rows tokens, columns query rows
        f32x4 st[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const half8 kk = held_k(bits, k[2 * b + half], k_scale<NB>(ks, half, b));
#pragma unroll
                for (int p = 0; p < PQ; p++) st[half] = mfma16(kk, t.q[p][b], st[half]);
            }
        }
        load_k<NB>(from, lane, k, ks);
        const int t0 = g * kGroup;
        if (!gp || t0 < lo_all || t0 + kGroup > hi_all) {  // some row sees only a part
            t.hide(st, gp ? t0 : -1 - kGroup, quarter);
            const int valid = gp ? r.valid : 0;
            if (t0 < r.from || t0 + kGroup > valid) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t keep = keep_mask(t0, quarter, j, r.from, valid);
#pragma unroll
                    for (int b = 0; b < NB; b++) vs[4 * b + j] &= keep;
                }
            }
        }
        half8 w[PW];
        t.weigh(st, w);
#pragma unroll
        for (int p = 0; p < PW; p++) t.l = mfma16(ones8(), w[p], t.l);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            half8 vv[2];
            held_v(bits, v[2 * b], v[2 * b + 1], &vs[4 * b], vv);
#pragma unroll
            for (int z = 0; z < 2; z++) {
#pragma unroll
                for (int p = 0; p < PW; p++) t.acc[2 * b + z] = mfma16(vv[z], w[p], t.acc[2 * b + z]);
            }
        }
        load_v<NB>(from, lane, v, vs);
        gp = next, next = after;
    }

    // join the waves
    constexpr int kQuads = hd / 4;
    if (quarter == 0) red_ml[wave][col][0] = t.m, red_ml[wave][col][1] = t.l[0];
#pragma unroll
    for (int j = 0; j < 2 * NB; j++) *(f32x4*)&red_acc[wave][col][j * 16 + quarter * 4] = t.acc[j];
    __syncthreads();
    for (int u = threadIdx.x; u < 16 * kQuads; u += 256) {
        const int f = u / kQuads, d4 = u % kQuads * 4;
        if (f >= r.pairs) continue;
        float m = kUnseen;  // never NaN: a NaN score is in the sums alone
#pragma unroll
        for (int w = 0; w < NW; w++) m = fmaxf(m, red_ml[w][f][0]);
        float l = 0.f, o[4] = {};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float e = __builtin_amdgcn_exp2f(red_ml[w][f][0] - m);
            l = fmaf(e, red_ml[w][f][1], l);
            const f32x4 x = *(const f32x4*)&red_acc[w][f][d4];
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = fmaf(e, x[i], o[i]);
        }
        store_pair(a, r, pl.h, f, pl.part, d4, m, l, o);
    }
}

// Many pairs: a workgroup's NW waves take 16 NT pairs each and share the held
// values of TG groups at a time, converted once into LDS in operand order (one
// 16-byte piece a lane, read and written without bank conflicts). Two buffers:
// one is worked on while the next groups are converted into the other, and the
// two steps after are on their way from memory. Each wave converts K or V of
// some blocks of one group.
//
// Bound: vector instructions and matrix instructions of a SIMD in turn. 2 x 2048
// bf16 rows at 32768 tokens, 32 / 8 heads of 128 (NT 2, NW 8): 2.25 ms, 894
// TFLOP/s, matrix pipe busy 39 %, vector pipe 45; with four waves a conversion 12 %
// more. 2048 f32 rows at 4096, heads of 64: 132 us, the planes doubling both
// products. 16 x 5 bf16 rows at up to 12000 tokens, 4 heads of 128 (NT 1): 34 us,
// the chain of barrier, scores, weights and sums of one tile a wave.
template <int NB, int PQ, int PW, int NT, int NW, int TG>
__global__ void __launch_bounds__(64 * NW) kv_q4_rows_kernel(Q4Attn a, int shares) {
    constexpr int kPer = NW / 2 / TG;                             // waves of a group, K or V
    constexpr int kBlocks = ((NB + 1) / 2 + kPer - 1) / kPer * 2;  // blocks of one of them, an even number
    constexpr int kHave = kBlocks < NB ? kBlocks : NB;
    __shared__ half8 kf[2][TG][2 * NB][64], vf[2][TG][2 * NB][64];
    __shared__ int have[2][TG];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quarter = lane >> 4;
    Q4Place pl;
    if (!head_place(a, lane, shares, &pl)) return;
    const Q4Bits bits;
    const Q4Rows& r = pl.r;
    const int f_wave = pl.f0 + wave * (16 * NT);
    const bool active = f_wave < r.pairs;
    const int i_first = row_of(a, f_wave), i_last = row_of(a, min(f_wave + 16 * NT, r.pairs) - 1);
    int lo_any = 0, hi_any = 0, lo_all = 0, hi_all = 0;  // seen by any, by every row of the wave
    if (active) {
        lo_any = r.see.lo(i_first), hi_any = r.see.hi(i_last);
        lo_all = r.see.lo(i_last), hi_all = r.see.hi(i_first);
    }
    const Q4Groups groups(a, pl.s, pl.h, pl.g_end);
    const bool is_v = wave & 1;
    const int part = (wave >> 1) % kPer, mine = (wave >> 1) / kPer;  // blocks from kBlocks part on of group `mine`

    // two steps' words on their way: codes, and the V scales of the blocks or
    // the K scales of all blocks
    uint32_t c[2][2 * kBlocks], sc[2][4 * kHave > NB ? 4 * kHave : NB];
    const uint8_t* gp[2] = {nullptr, nullptr};
    int page = -1;  // page id of this wave's group of the next fetch
    // f(first block, number of blocks), constants, of this wave's part
    auto with_blocks = [&](auto f) {
#pragma unroll
        for (int p = 0; p < kPer; p++) {
            if (p != part) continue;
            if (p == 0) f(std::integral_constant<int, 0>{}, std::integral_constant<int, kHave>{});
            if constexpr (kPer > 1 && kBlocks < NB) {
                if (p == 1) f(std::integral_constant<int, kBlocks>{}, std::integral_constant<int, (NB < 2 * kBlocks ? NB : 2 * kBlocks) - kBlocks>{});
            }
            if constexpr (kPer > 2 && 2 * kBlocks < NB) {
                if (p == 2) f(std::integral_constant<int, 2 * kBlocks>{}, std::integral_constant<int, (NB < 3 * kBlocks ? NB : 3 * kBlocks) - 2 * kBlocks>{});
            }
            if constexpr (kPer > 3 && 3 * kBlocks < NB) {
                if (p == 3) f(std::integral_constant<int, 3 * kBlocks>{}, std::integral_constant<int, NB - 3 * kBlocks>{});
            }
        }
    };
    auto fetch = [&](int g, auto slot) {  // this wave's share of the step at g, and the page id for the one after
        constexpr int i = decltype(slot)::value;
        gp[i] = groups.at(a, g + mine, page);
        page = groups.id(a, g + mine + TG);
        if (!gp[i]) return;
        with_blocks([&](auto first, auto count) {
            constexpr int b = decltype(first)::value, n = decltype(count)::value;
            if (is_v) {
                load_v<NB, b, b + n>(gp[i], lane, c[i], sc[i]);
            } else {
                load_words<NB>(gp[i] + 1024 * NB + lane % 16 * 4 * NB, sc[i]);
                load_codes<NB, b, b + n>(gp[i], lane, c[i]);
            }
        });
    };
    auto convert = [&](int g, auto slot) {  // into the buffer of the slot's number
        constexpr int i = decltype(slot)::value;
        if (is_v && part == 0 && lane == 0) have[i][mine] = gp[i] != nullptr;
        if (!gp[i]) return;
        with_blocks([&](auto first, auto count) {
            constexpr int b = decltype(first)::value, n = decltype(count)::value;
            if (is_v) {
                const int t0 = (g + mine) * kGroup;
                if (t0 < r.from || t0 + kGroup > r.valid) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t keep = keep_mask(t0, quarter, j, r.from, r.valid);
#pragma unroll
                        for (int e = 0; e < n; e++) sc[i][4 * e + j] &= keep;
                    }
                }
#pragma unroll
                for (int e = 0; e < n; e++) {
                    half8 vv[2];
                    held_v(bits, c[i][2 * e], c[i][2 * e + 1], &sc[i][4 * e], vv);
                    vf[i][mine][2 * (b + e)][lane] = vv[0];
                    vf[i][mine][2 * (b + e) + 1][lane] = vv[1];
                }
            } else {
#pragma unroll
                for (int e = 0; e < n; e++) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const int si = half * NB + b + e;
                        kf[i][mine][si][lane] = held_k(bits, c[i][2 * e + half], as_half2(sc[i][si / 2])[si % 2]);
                    }
                }
            }
        });
    };

    constexpr std::integral_constant<int, 0> s0{};
    constexpr std::integral_constant<int, 1> s1{};
    const int g_begin = pl.g_begin, g_end = pl.g_end;
    if (g_begin < g_end) {
        page = groups.id(a, g_begin + mine);
        fetch(g_begin, s0);
        fetch(g_begin + TG, s1);
    }
    Q4Tile<NB, PQ, PW> t[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) t[n].init(a, r.see, r.start, pl.h, f_wave + 16 * n + col, r.pairs, quarter);
    if (g_begin < g_end) {
        convert(g_begin, s0);
        fetch(g_begin + 2 * TG, s0);
    }
    __syncthreads();
    // one step: the next one's groups into the other buffer, the loads of the
    // one two further, then the scores and sums of this one's
    auto step = [&](int g, auto slot, auto other) {
        constexpr int buf = decltype(slot)::value;
        if (g + TG < g_end) {
            convert(g + TG, other);
            fetch(g + 3 * TG, other);
        }
#pragma unroll
        for (int gg = 0; gg < TG; gg++) {
            const int t0 = (g + gg) * kGroup;
            // nothing there, or nothing that a row of this wave sees
            if (!__builtin_amdgcn_readfirstlane(have[buf][gg]) || t0 >= hi_any || t0 + kGroup <= lo_any) continue;
            f32x4 st[NT][2];
#pragma unroll
            for (int half = 0; half < 2; half++) {
#pragma unroll
                for (int n = 0; n < NT; n++) st[n][half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const half8 k = kf[buf][gg][half * NB + b][lane];
#pragma unroll
                    for (int n = 0; n < NT; n++) {
#pragma unroll
                        for (int p = 0; p < PQ; p++) st[n][half] = mfma16(k, t[n].q[p][b], st[n][half]);
                    }
                }
            }
            if (t0 < lo_all || t0 + kGroup > hi_all) {
#pragma unroll
                for (int n = 0; n < NT; n++) t[n].hide(st[n], t0, quarter);
            }
            half8 w[NT][PW];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                t[n].weigh(st[n], w[n]);
#pragma unroll
                for (int p = 0; p < PW; p++) t[n].l = mfma16(ones8(), w[n][p], t[n].l);
            }
#pragma unroll
            for (int j = 0; j < 2 * NB; j++) {
                const half8 v = vf[buf][gg][j][lane];
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int p = 0; p < PW; p++) t[n].acc[j] = mfma16(v, w[n][p], t[n].acc[j]);
                }
            }
        }
        __syncthreads();
    };
    for (int g = g_begin; g < g_end; g += 2 * TG) {
        step(g, s0, s1);
        if (g + TG < g_end) step(g + TG, s1, s0);
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int f = f_wave + 16 * n + col;
        if (f >= r.pairs) continue;
#pragma unroll
        for (int j = 0; j < 2 * NB; j++) {
            float o[4] = {t[n].acc[j][0], t[n].acc[j][1], t[n].acc[j][2], t[n].acc[j][3]};
            store_pair(a, r, pl.h, f, pl.part, j * 16 + quarter * 4, t[n].m, t[n].l[0], o);
        }
    }
}

// wave_max without LDS traffic, as xsum_all64.
__device__ __forceinline__ float xmax_all64(float v) {
    float a, b;
    swap32(v, a, b);
    v = fmaxf(a, b);
    swap16(v, a, b);
    v = fmaxf(a, b);
    v = fmaxf(v, dpp_mov<0x128>(v));
    v = fmaxf(v, xor4_mov(v));
    v = fmaxf(v, dpp_mov<0x4E>(v));
    return fmaxf(v, dpp_mov<0xB1>(v));
}

// The parts of a (row, head) joined by one wave: lane i weighs part i (there
// are at most 64), then the lanes take four values each of 256 / hd parts at a
// time. `shares`: workgroups of the even shares.
constexpr int kMaxSplit = 64;
__global__ void __launch_bounds__(256) kv_q4_join_kernel(Q4Attn a, int shares) {
    const int hd = a.b.hd, lane = threadIdx.x & 63;
    const int64_t pr = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (pr >= (int64_t)a.rows * a.n_heads) return;
    const int row = udiv((int)pr, a.n_heads), head = (int)pr - row * a.n_heads;  // rows times heads fits 31 bits
    const int s = __builtin_amdgcn_readfirstlane(wave_search(a.b.n_seq, lane, row, [&](int i) { return a.b.starts[i]; }));
    const int i = row - a.b.starts[s];
    Q4Rows r;
    if (i < 0 || row >= a.b.starts[s + 1] || !rows_of(a, s, &r)) return;
    const int f = i * a.gq + head - udiv(head, a.gq) * a.gq;
    if (f >= r.pairs) return;
    int n;
    if (a.chunk == 0) {
        const Q4Cut c = cut_of(a, lane, shares);
        int base = 0, lo, groups = c.n, before = c.before, run = 0;
        for (; s >= base + 64; base += 64) {
            run += lane_value(before + groups, 63);
            seq_groups(a, base + 64 + lane, &lo, &groups);
            before = wave_before(groups, lane);
        }
        const int own = s - base;
        const int x = (run + lane_value(before, own)) * a.b.n_kv + udiv(head, a.gq) * lane_value(groups, own);
        groups = lane_value(groups, own);
        n = groups == 0 ? 0 : udiv(x + groups - 1, c.size) - udiv(x, c.size) + 1;
        if (n == 1) return;  // stored already
    } else {
        const int f0 = f - f % a.tile_pairs;
        int g_lo, g_hi;
        tile_groups(r.see, row_of(a, f0), row_of(a, min(f0 + a.tile_pairs, r.pairs) - 1), &g_lo, &g_hi);
        n = min((max(g_hi - g_lo, 0) + a.chunk - 1) / a.chunk, a.nsplit);
    }
    const int quads = hd / 4, per = 64 / quads;  // hd 96 and 192: lanes past the last quad repeat one
    const int d4 = lane % quads * 4, first = min(lane / quads, per - 1);
    const float* pa = a.part_acc + pr * a.nsplit * hd + d4;
    const float* ml = a.part_ml + pr * a.nsplit * 2;
    // all loads of up to 8 per parts, before any use
    f32x4 x[8];
    auto fetch = [&](int j) {
#pragma unroll
        for (int c = 0; c < 8; c++) x[c] = *(const f32x4*)(pa + (int64_t)min(j + c * per + first, n - 1) * hd);
    };
    float m_i = kUnseen, l_i = 0.f;
    if (n) {
        if (lane < n) m_i = ml[2 * lane], l_i = ml[2 * lane + 1];
        fetch(0);
    }
    float o[4] = {};
    const float m = xmax_all64(m_i);
    const float e_i = __builtin_amdgcn_exp2f(m_i - m);  // used up to part n
    const float l = xsum_all64(e_i * l_i);
    for (int j = 0; j < n; j += 8 * per) {
        if (j) fetch(j);
#pragma unroll
        for (int c = 0; c < 8; c++) {
            const int k = j + c * per + first;
            const float e = __shfl(e_i, min(k, 63), 64);
#pragma unroll
            for (int d = 0; d < 4; d++) o[d] = fmaf(k < n ? e : 0.f, x[c][d], o[d]);
        }
    }
    // sum over the parts' lanes
    for (int c = 0; c < 4; c++) {
        float v = o[c];
        for (int k = 1; k < per; k++) v += __shfl(o[c], min(lane + k * quads, 63), 64);
        o[c] = v;
    }
    if (lane >= quads) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < 4; c++) o[c] *= inv;
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

// A launch counts the threads of a dimension in 32 bits.
bool grid_fits(size_t groups, size_t threads) { return groups <= UINT32_MAX / threads; }

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
    if (!cache || !starts || (n_seq && (!lens || (pages_per_seq && !pages))))
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "null argument");
    if ((uintptr_t)cache % 16) return set_error(MIVI_ERR_INVALID_ARGUMENT, "cache not 16-byte aligned");
    if ((uintptr_t)pages % 4 || (uintptr_t)starts % 4 || (uintptr_t)lens % 4)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "table, starts or lens not 4-byte aligned");
    *b = Q4Batch{(uint8_t*)cache, pages,     starts,        lens,    (int64_t)pages_stride, (int64_t)n_pages,
                 (int64_t)page_bytes, (int)n_seq, (int)n_kv, (int)hd, (int)(page_tokens / kGroup),
                 0, (int)cap};
    if (b->gpp > 1) b->gpp_inv = (uint32_t)((1ull << 32) / b->gpp + 1);
    return MIVI_OK;
}

// Grid of the kernels that take whole groups: units times as many workgroups a
// unit as fill the card (each wave at least one head's K or V); none (x = 0)
// where the call has fewer than 8 rows a sequence: those go 8 values a lane. (64
// sequences, 8 bf16 heads of 128, written and read back by groups and 8 values a
// lane: 4 rows each 12.5 and 9.1 us, 8 rows 12.9 and 10.8, 16 rows 14.0 and 14.3,
// 32 rows 14.3 and 19.3.)
dim3 group_grid(size_t rows, size_t n_seq, size_t n_kv) {
    if (rows < 8 * n_seq) return dim3(0, 0);
    const size_t units = rows / kGroup + 2 * n_seq, most = (n_kv + 1) / 2;
    const size_t want = (8 * (size_t)num_cus() + units - 1) / units;
    return dim3((unsigned)units, (unsigned)std::min(most, want));
}

template <int T, class... Args>
void launch_read_groups(size_t nb, dim3 grid, hipStream_t s, Args... args) {
    switch (nb) {
        case 1: kv_q4_read_groups_kernel<T, 1><<<grid, 256, 0, s>>>(args...); break;
        case 2: kv_q4_read_groups_kernel<T, 2><<<grid, 256, 0, s>>>(args...); break;
        case 3: kv_q4_read_groups_kernel<T, 3><<<grid, 256, 0, s>>>(args...); break;
        case 4: kv_q4_read_groups_kernel<T, 4><<<grid, 256, 0, s>>>(args...); break;
        case 6: kv_q4_read_groups_kernel<T, 6><<<grid, 256, 0, s>>>(args...); break;
        default: kv_q4_read_groups_kernel<T, 8><<<grid, 256, 0, s>>>(args...); break;
    }
}

// How an attention call is laid out.
struct Q4Plan {
    // kv_q4_step_kernel; kv_q4_rows_kernel of 64 pairs a workgroup (four waves
    // of 16), of 128 (eight of 16, four of 32), of 256 (eight of 32)
    enum { kStep, kFew, kSome, kMid, kMany } form;
    size_t tile_pairs, tiles, chunk, nsplit, shares, share_min, grid;
    size_t threads() const { return form == kSome || form == kMany ? 512 : 256; }
};

Q4Plan attn_plan(size_t n_seq, size_t max_rows, size_t gq, size_t n_kv, size_t hd, int planes, size_t cap,
                 size_t window) {
    Q4Plan p = {};
    const size_t pairs = max_rows * gq, cus = (size_t)num_cus();
    size_t heads;
    if (__builtin_mul_overflow(n_seq, n_kv, &heads)) heads = SIZE_MAX;
    // By registers: two tiles a wave and two or three workgroups a CU up to 96
    // dimensions, one tile a wave past 128; at 128 the 256 pairs that share a
    // conversion need two workgroups a CU's worth of tiles to end evenly (8 kv
    // heads, 2 x 2048 bf16 rows at 32768: 2260 us, with 128 pairs 2590; 2048 rows
    // of one prompt from its start 88 and 70), and two planes of queries do not
    // fit one tile a wave twice on a CU (2 x 700 f32 rows at 32768: 1370 and
    // 1720). 65 to 128 pairs as two tiles of 64: 8 x 25 f32 rows at 4096, heads
    // of 128, 59.6 us, as one of 128 114 (bf16 49.9 and 71.5, f32 heads of 64
    // 40.5 and 50.9).
    p.form = pairs <= 16    ? Q4Plan::kStep
             : pairs <= 128 ? Q4Plan::kFew
             : hd > 128     ? Q4Plan::kSome
             : hd <= 96     ? Q4Plan::kMid
             : planes == 2 || heads >= 2 * cus || heads * ((pairs + 255) / 256) >= 2 * cus ? Q4Plan::kMany
                                                                                          : Q4Plan::kSome;
    p.tile_pairs = p.form == Q4Plan::kStep ? 16 : p.form == Q4Plan::kFew ? 64 : p.form == Q4Plan::kMany ? 256 : 128;
    p.tiles = (pairs + p.tile_pairs - 1) / p.tile_pairs;
    // groups that a tile can see
    size_t tokens = cap;
    if (window) tokens = std::min(cap, std::min(window, cap) + p.tile_pairs / gq + 1 + 2 * kGroup);
    const size_t groups = std::max<size_t>(1, (tokens + kGroup - 1) / kGroup);
    size_t all, wgs;
    if (__builtin_mul_overflow(heads, groups, &all)) all = SIZE_MAX;
    // One part a head, which needs no second kernel, where it is short: 8 groups
    // a wave, 4 of more than 128 dimensions, 8 groups in all of more rows. (In one
    // part and in shares with a join, captured: one token, 8 heads of 64, f32, at
    // 1024 tokens 9.0 and 11.2 us, at 2048 13.6 and 11.3; 64 sequences at 1024 15.5
    // and 26.4; 4 sequences of 4 bf16 heads of 256 at 512 12.2 and 14.1, at 1024
    // 17.4 and 14.5; 16 rows at 256 10.2 and 13.9, at 512 15.3 and 13.9.)
    if (p.tiles == 1 && groups <= (p.form == Q4Plan::kStep ? hd <= 128 ? 32 : 16 : 8)) {
        p.chunk = groups, p.nsplit = 1, p.grid = heads;
        return p;
    }
    if (p.tiles == 1 && all <= (size_t)INT32_MAX / 2) {
        // even shares: four workgroups a CU, each at least one step of every wave
        p.share_min = 4;
        p.shares = std::min(cus * 4, (all + p.share_min - 1) / p.share_min);
        p.nsplit = std::min<size_t>({(size_t)kMaxSplit, p.shares / n_kv + 2, groups / p.share_min + 2});
        p.grid = p.shares + heads;
        return p;
    }
    // Tiles by themselves, their groups in shares where that fills the card
    // better: the rounds that the workgroups take, one to three a CU, times a
    // share's groups at about 1.1 us, against the join's 10 us and its traffic,
    // twice the parts at 4 TB/s.
    if (__builtin_mul_overflow(heads, p.tiles, &wgs)) wgs = SIZE_MAX;
    const size_t slots = cus * (p.form == Q4Plan::kFew ? 3 : p.form == Q4Plan::kMid ? 2 : 1);
    double best = 0;
    for (size_t ns = 1; ns <= (size_t)kMaxSplit && (ns == 1 || wgs < 4 * slots); ns++) {
        const size_t chunk = ((groups + ns - 1) / ns + 3) / 4 * 4, n = (groups + chunk - 1) / chunk;
        const size_t rounds = wgs == SIZE_MAX ? 1 : (wgs * n + slots - 1) / slots;
        const double parts = (double)n_seq * max_rows * gq * n_kv * n * (hd + 2) * 4;
        const double us = (double)rounds * chunk * 1.1 + (n > 1 ? 10 + 2 * parts / 4e6 : 0);
        if (ns == 1 || us < best) best = us, p.chunk = chunk, p.nsplit = n;
    }
    if (__builtin_mul_overflow(wgs, p.nsplit, &p.grid)) p.grid = SIZE_MAX;
    return p;
}

template <int NB, int PQ, int PW>
void launch_attn(const Q4Attn& a, const Q4Plan& p, hipStream_t s) {
    const unsigned grid = (unsigned)p.grid;
    const int shares = (int)p.shares;
    if (p.form == Q4Plan::kStep) {
        kv_q4_step_kernel<NB, PQ, PW><<<grid, 256, 0, s>>>(a, shares);
    } else if (p.form == Q4Plan::kFew) {
        // two groups a step at 64 dimensions (16 x 5 bf16 rows at up to 12000
        // tokens, 4 heads: 35.4 -> 32.0 us); at 128 their LDS halves the workgroups
        // of a CU (42.4 -> 51.2)
        kv_q4_rows_kernel<NB, PQ, PW, 1, 4, NB <= 2 ? 2 : 1><<<grid, 256, 0, s>>>(a, shares);
    } else if constexpr (NB <= 3) {
        kv_q4_rows_kernel<NB, PQ, PW, 2, 4, 2><<<grid, 256, 0, s>>>(a, shares);
    } else if constexpr (NB == 4) {
        if constexpr (PQ == 1) {
            if (p.form == Q4Plan::kSome) {
                kv_q4_rows_kernel<NB, PQ, PW, 1, 8, 1><<<grid, 512, 0, s>>>(a, shares);
                return;
            }
        }
        kv_q4_rows_kernel<NB, PQ, PW, 2, 8, 2><<<grid, 512, 0, s>>>(a, shares);
    } else {
        kv_q4_rows_kernel<NB, PQ, PW, 1, 8, 1><<<grid, 512, 0, s>>>(a, shares);
    }
}
template <int NB>
void launch_attn(const Q4Attn& a, const Q4Plan& p, hipStream_t s) {
    if (a.type == MIVI_GGML_F32) launch_attn<NB, 2, 2>(a, p, s);
    else if (a.type == MIVI_GGML_F16) launch_attn<NB, 1, 2>(a, p, s);
    else launch_attn<NB, 1, 1>(a, p, s);
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
    const dim3 grid = group_grid(rows, n_seq, n_kv_heads);
    if (!grid_fits(grid.x ? grid.x : blocks, 256)) return err_overflow();
    clear_error();
    const size_t e = type_bytes(type);
    const int wk = wide_ok(k, k_row_stride, k_head_stride, e, 16), wv = wide_ok(v, v_row_stride, v_head_stride, e, 16);
    hipStream_t s = (hipStream_t)stream;
#define APPEND(T)                                                                                                    \
    if (grid.x)                                                                                                      \
        kv_q4_append_groups_kernel<T><<<grid, 256, 0, s>>>(b, k, v, (int64_t)k_row_stride, (int64_t)k_head_stride,   \
                                                           (int64_t)v_row_stride, (int64_t)v_head_stride, (int)rows, \
                                                           wk, wv);                                                  \
    else                                                                                                             \
        kv_q4_append_kernel<T><<<dim3((unsigned)blocks, 2), 256, 0, s>>>(                                            \
            b, k, v, (int64_t)k_row_stride, (int64_t)k_head_stride, (int64_t)v_row_stride, (int64_t)v_head_stride,   \
            (int)rows, wk, wv)
    if (type == MIVI_GGML_F32) { APPEND(MIVI_GGML_F32); }
    else if (type == MIVI_GGML_F16) { APPEND(MIVI_GGML_F16); }
    else { APPEND(MIVI_GGML_BF16); }
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
    const dim3 grid = group_grid(rows, n_seq, n_kv_heads);
    if (!grid_fits(grid.x ? grid.x : blocks, 256)) return err_overflow();
    clear_error();
    const size_t e = type_bytes(type);
    const int wk = wide_ok(k, k_row_stride, k_head_stride, e, 16), wv = wide_ok(v, v_row_stride, v_head_stride, e, 16);
    hipStream_t s = (hipStream_t)stream;
#define READ(T)                                                                                                      \
    if (grid.x)                                                                                                      \
        launch_read_groups<T>(head_dim / 32, grid, s, b, k, v, (int64_t)k_row_stride, (int64_t)k_head_stride,        \
                              (int64_t)v_row_stride, (int64_t)v_head_stride, (int)rows, wk, wv);                     \
    else                                                                                                             \
        kv_q4_read_kernel<T><<<dim3((unsigned)blocks, 2), 256, 0, s>>>(                                              \
            b, k, v, (int64_t)k_row_stride, (int64_t)k_head_stride, (int64_t)v_row_stride, (int64_t)v_head_stride,   \
            (int)rows, wk, wv)
    if (type == MIVI_GGML_F32) { READ(MIVI_GGML_F32); }
    else if (type == MIVI_GGML_F16) { READ(MIVI_GGML_F16); }
    else { READ(MIVI_GGML_BF16); }
#undef READ
    MIVI_HIP_CHECK(hipGetLastError());
    return MIVI_OK;
}

extern "C" size_t mivi_hip_kv_q4_attention_workspace(size_t n_seq, size_t rows, size_t max_rows, size_t n_heads,
                                                     size_t n_kv_heads, size_t head_dim, size_t max_tokens,
                                                     size_t window) {
    if (n_kv_heads == 0 || n_heads == 0 || n_heads % n_kv_heads || rows == 0 || n_seq == 0 || max_rows == 0) return 0;
    // no call has these: their products could wrap round
    if (n_heads > 65535 || !head_dim_ok(head_dim) || std::max({n_seq, rows, max_tokens}) > (size_t)INT32_MAX) return 0;
    size_t parts = 1;
    for (int planes = 1; planes <= 2; planes++)
        parts = std::max(parts, attn_plan(n_seq, std::min(max_rows, rows), n_heads / n_kv_heads, n_kv_heads, head_dim,
                                          planes, max_tokens, window).nsplit);
    return parts == 1 ? 0 : rows * n_heads * parts * (head_dim + 2) * sizeof(float);
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
    if (!(scale >= -3.402823466e38f && scale <= 3.402823466e38f))
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "scale %g is not finite", (double)scale);
    if (rows == 0 || n_seq == 0 || max_rows == 0) return clear_error();
    if ((rc = check_tensor("q", q, q_len, type, rows, q_row_stride, n_heads, q_head_stride, head_dim, false)) ||
        (rc = check_tensor("out", out, out_len, type, rows, out_row_stride, n_heads, out_head_stride, head_dim, true)))
        return rc;
    max_rows = std::min(max_rows, rows);
    const size_t gq = n_heads / n_kv_heads, cap = pages_per_seq * page_tokens;
    const int planes = type == MIVI_GGML_F32 ? 2 : 1;
    const Q4Plan p = attn_plan(n_seq, max_rows, gq, n_kv_heads, head_dim, planes, cap, window);
    const size_t need =
        mivi_hip_kv_q4_attention_workspace(n_seq, rows, max_rows, n_heads, n_kv_heads, head_dim, cap, window);
    if (workspace_bytes < need) return err_buffer_too_small(need, workspace_bytes);
    if (need && !workspace) return set_error(MIVI_ERR_INVALID_ARGUMENT, "null workspace");
    if (need && (uintptr_t)workspace % 16)
        return set_error(MIVI_ERR_INVALID_ARGUMENT, "workspace not 16-byte aligned");
    const size_t join_grid = (rows * n_heads + 3) / 4;  // a wave a row and head
    if (!grid_fits(p.grid, p.threads()) || rows * n_heads > (size_t)INT32_MAX - 4096 ||
        (p.nsplit > 1 && !grid_fits(join_grid, 256)))
        return err_overflow();
    clear_error();
    a.q = q, a.out = out;
    a.q_row = (int64_t)q_row_stride, a.q_head = (int64_t)q_head_stride;
    a.o_row = (int64_t)out_row_stride, a.o_head = (int64_t)out_head_stride;
    a.type = type;
    const size_t e = type_bytes(type);
    a.wide_q = wide_ok(q, q_row_stride, q_head_stride, e, 16);
    a.wide_o = wide_ok(out, out_row_stride, out_head_stride, e, 4 * e);
    a.n_heads = (int)n_heads, a.gq = (int)gq;
    a.rows = (int)rows, a.max_rows = (int)max_rows;
    a.tiles = (int)p.tiles, a.tile_pairs = (int)p.tile_pairs;
    a.nsplit = (int)p.nsplit, a.chunk = (int)p.chunk, a.share_min = (int)p.share_min;
    a.window = (int)std::min<size_t>(window, (size_t)INT32_MAX);
    a.scale = scale;
    a.part_acc = (float*)workspace;
    a.part_ml = a.part_acc + rows * n_heads * p.nsplit * head_dim;
    hipStream_t s = (hipStream_t)stream;
    switch (head_dim / 32) {
        case 1: launch_attn<1>(a, p, s); break;
        case 2: launch_attn<2>(a, p, s); break;
        case 3: launch_attn<3>(a, p, s); break;
        case 4: launch_attn<4>(a, p, s); break;
        case 6: launch_attn<6>(a, p, s); break;
        default: launch_attn<8>(a, p, s); break;
    }
    MIVI_HIP_CHECK(hipGetLastError());
    if (p.nsplit > 1) {
        kv_q4_join_kernel<<<(unsigned)join_grid, 256, 0, s>>>(a, (int)p.shares);
        MIVI_HIP_CHECK(hipGetLastError());
    }
    return MIVI_OK;
}
