// Verification of drafted tokens against the target's probabilities.
//
// Row i of a sequence's n rows but the last holds the target's probabilities p
// and the draft's q of the place where token t was drafted; it is accepted if
// u q(t) < p(t) there and in every row before it. The next token is drawn from
// the first row that is not: from max(p - q, 0), or from p in the last row
// (nothing was drafted there) and where nothing is left; it is the first index
// whose cumulative sum passes pick times the whole. A token so found has the
// target's distribution, whatever q is.
//
// u q < p is decided exactly: the product of two f32 numbers is a 64-bit one.
// Differences and sums are 64-bit too, in one fixed order.
//
// A sequence reads one row of each distribution, cut into chunks of 4096 over
// the card: every chunk's workgroup finds the row itself (a few loads, where a
// kernel of its own would cost a launch) and sums its chunk; a second kernel,
// one workgroup a sequence, finds the chunk and the index in it. 64 sequences of
// 128256: 17.2 us, 3.8 TB/s behind a chain of three loads, and 6.9, chains of loads
// and scans; one sequence of 65536: 5.0 and 5.8.
#include <algorithm>

#include "rows.h"

using namespace mivi;

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;                    // probabilities a thread
constexpr int kChunk = kThreads * kPer;

struct VerifyArgs {
    const float *target, *draft;  // draft: null where every drafted token was certain
    int64_t t_row, d_row;
    const int32_t *drafted, *starts;
    const float *accept, *pick;
    int32_t *tokens, *counts;
    double2* parts;   // [n_seq][chunks]: what is left of a chunk, and its p
    int32_t* found;   // [n_seq]: accepted tokens
    int rows, n, chunks;
};

// A probability: what is negative, infinite or NaN counts as none.
__device__ __forceinline__ double chance(float v) { return v > 0.f && v <= 3.40282347e38f ? (double)v : 0.0; }

// Rows [lo, hi) of sequence s, within the call's.
__device__ __forceinline__ void seq_rows(const VerifyArgs& a, int s, int* lo, int* hi) {
    *lo = max(a.starts[s], 0);
    *hi = min(a.starts[s + 1], a.rows);
}

__device__ __forceinline__ bool accepted(const VerifyArgs& a, int r) {
    const int t = a.drafted[r];
    if (t < 0 || t >= a.n) return false;
    const double p = chance(a.target[r * a.t_row + t]);
    const double q = a.draft ? chance(a.draft[r * a.d_row + t]) : 1.0;
    return (double)a.accept[r] * q < p;
}

// 16 values of p and of what is left from index i on, of row r.
__device__ __forceinline__ void load16(const VerifyArgs& a, int r, bool last, int i, double (&left)[kPer],
                                       double (&p)[kPer]) {
    const int t = last || a.draft ? -1 : a.drafted[r];
#pragma unroll
    for (int h = 0; h < kPer; h += 8) {
        float x[8], y[8];
        load_row8<MIVI_GGML_F32>(a.target, r * a.t_row + i + h, a.n - i - h, x);
        if (!last && a.draft) load_row8<MIVI_GGML_F32>(a.draft, r * a.d_row + i + h, a.n - i - h, y);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[h + e] = chance(x[e]);
            const double q = last ? 0.0 : a.draft ? chance(y[e]) : i + h + e == t ? 1.0 : 0.0;
            left[h + e] = fmax(p[h + e] - q, 0.0);
        }
    }
}

__device__ __forceinline__ double shfl_up(double v, int o) { return __shfl_up(v, o, 64); }

// Sums before this thread (exclusive), and in *all of the workgroup.
__device__ __forceinline__ double scan(double v, double* sh, double* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double inc = v;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const double w = shfl_up(inc, o);
        if (lane >= o) inc += w;
    }
    if (lane == 63) sh[wave] = inc;
    __syncthreads();
    double before = 0;
    for (int i = 0; i < wave; i++) before += sh[i];
    *all = sh[0] + sh[1] + sh[2] + sh[3];
    __syncthreads();
    // the lane before's inclusive sum: an exclusive one without cancellation
    const double up = shfl_up(inc, 1);
    return before + (lane ? up : 0.0);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// The first thread (from `base` on) that passes into at, the last with any mass
// into behind.
__device__ __forceinline__ void mark(bool passes, bool some, int base, int* at, int* behind) {
    const uint64_t a = __ballot(passes), b = __ballot(some);
    const int wave = base + (threadIdx.x & ~63);
    if ((threadIdx.x & 63) == 0) {
        if (a) atomicMin(at, wave + (int)__ffsll((unsigned long long)a) - 1);
        if (b) atomicMax(behind, wave + 63 - (int)__clzll((long long)b));
    }
}

__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
    __shared__ int first;
    __shared__ double sh[2][kThreads / 64];
    const int s = blockIdx.y, tid = threadIdx.x;
    int lo, hi;
    seq_rows(a, s, &lo, &hi);
    if (hi <= lo) return;
    // the first row that is not accepted
    int row = hi - 1;
    if (tid == 0) first = row;
    __syncthreads();
    for (int64_t b = lo; b < hi - 1; b += kThreads) {
        const int64_t r = b + tid;
        if (r < hi - 1 && !accepted(a, (int)r)) atomicMin(&first, (int)r);
        __syncthreads();
        row = first;
        __syncthreads();  // read by all before the next rows' threads write it
        if (row < hi - 1) break;
    }
    if (blockIdx.x == 0 && tid == 0) a.found[s] = row - lo;
    double left[kPer], p[kPer], l = 0, m = 0;
    const int64_t i = (int64_t)blockIdx.x * kChunk + tid * kPer;
    if (i < a.n) {
        load16(a, row, row == hi - 1, (int)i, left, p);
#pragma unroll
        for (int e = 0; e < kPer; e++) l += left[e], m += p[e];
    }
    l = wave_sum64(l), m = wave_sum64(m);
    if ((tid & 63) == 0) sh[0][tid >> 6] = l, sh[1][tid >> 6] = m;
    __syncthreads();
    if (tid == 0)
        a.parts[(int64_t)s * a.chunks + blockIdx.x] =
            double2{sh[0][0] + sh[0][1] + sh[0][2] + sh[0][3], sh[1][0] + sh[1][1] + sh[1][2] + sh[1][3]};
}

// The chunk whose cumulative sum passes u times the whole, then the index in
// it. Sums of the two kernels may differ in the last bits: where none passes,
// it is the last with any mass.
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
    __shared__ double sh[kThreads / 64];
    __shared__ int at, behind, found;
    __shared__ double before;
    const int s = blockIdx.x, tid = threadIdx.x;
    int lo, hi;
    seq_rows(a, s, &lo, &hi);
    if (hi <= lo) {
        if (tid == 0) a.counts[s] = 0;
        return;
    }
    const int count = a.found[s], row = lo + count;
    const bool last = row == hi - 1;
    const double2* parts = a.parts + (int64_t)s * a.chunks;
    // the whole, with the first chunks' sums in hand
    const double2 mine = tid < a.chunks ? parts[tid] : double2{0, 0};
    double l = mine.x, whole;
    for (int64_t c = tid + kThreads; c < a.chunks; c += kThreads) l += parts[c].x;
    const double first = scan(l, sh, &whole);
    const bool one = a.chunks <= kThreads;
    const bool from_p = whole == 0;  // nothing is left of the row
    if (from_p) {
        double m = mine.y;
        for (int64_t c = tid + kThreads; c < a.chunks; c += kThreads) m += parts[c].y;
        scan(m, sh, &whole);
    }
    int token = -1;
    if (whole > 0) {
        const double goal = (double)a.pick[s] * whole;
        if (tid == 0) at = INT32_MAX, behind = -1;
        __syncthreads();
        double base = 0;
        for (int64_t b = 0; b < a.chunks; b += kThreads) {
            const int64_t c = b + tid;
            double v = b == 0 ? (from_p ? mine.y : mine.x) : 0.0;
            if (b && c < a.chunks) v = from_p ? parts[c].y : parts[c].x;
            double all = 0;
            const double ex = one && !from_p ? first : base + scan(v, sh, &all);
            mark(v > 0 && ex + v > goal, v > 0, (int)b, &at, &behind);
            __syncthreads();
            if (at == (int)c) before = ex;
            base += all;
            if (at != INT32_MAX) break;
        }
        __syncthreads();
        const bool passed = at != INT32_MAX;
        const int chunk = passed ? at : behind;
        const double rest = passed ? goal - before : whole;
        __syncthreads();
        if (tid == 0) at = INT32_MAX, behind = -1;
        const int64_t i = (int64_t)chunk * kChunk + tid * kPer;
        double left[kPer], p[kPer], v = 0;
        if (i < a.n) {
            load16(a, row, last, (int)i, left, p);
#pragma unroll
            for (int e = 0; e < kPer; e++) {
                if (from_p) left[e] = p[e];
                v += left[e];
            }
        }
        double all;
        const double ex = scan(v, sh, &all);
        mark(v > 0 && ex + v > rest, v > 0, 0, &at, &behind);
        __syncthreads();
        if (tid == (at != INT32_MAX ? at : behind)) {  // its sum passes: the same sums pass in it
            double sum = 0;
            int hit = -1, some = 0;
#pragma unroll
            for (int e = 0; e < kPer; e++) {
                sum += left[e];
                if (left[e] > 0) {
                    some = e;
                    if (hit < 0 && ex + sum > rest) hit = e;
                }
            }
            found = (int)i + (hit >= 0 ? hit : some);
        }
        __syncthreads();
        token = found;
    }
    if (tid == 0) a.counts[s] = count;
    for (int64_t r = (int64_t)lo + tid; r < hi; r += kThreads)
        a.tokens[r] = r < row ? a.drafted[r] : r == row ? token : -1;
}

size_t chunks_of(size_t n) { return (n + kChunk - 1) / kChunk; }

}  // namespace

extern "C" size_t mivi_hip_verify_rows_workspace(size_t n, size_t n_seq) {
    if (n > (size_t)INT32_MAX || n_seq > 65535) return 0;
    return n_seq * (chunks_of(n) * sizeof(double2) + sizeof(int32_t));
}

extern "C" int32_t mivi_hip_verify_rows(int32_t* tokens, size_t tokens_len, int32_t* counts, size_t counts_len,
                                        const float* target, size_t target_len, size_t target_row_stride,
                                        const float* draft, size_t draft_len, size_t draft_row_stride,
                                        const int32_t* drafted, size_t drafted_len, const float* accept,
                                        size_t accept_len, const float* pick, size_t pick_len, const int32_t* starts,
                                        size_t n_seq, size_t rows, size_t n, void* workspace, size_t workspace_bytes,
                                        void* stream) {
    if (n == 0) return set_error(MIVI_ERR_INVALID_ARGUMENT, "no probabilities in a row");
    if (n > (size_t)INT32_MAX - kChunk || rows > (size_t)INT32_MAX - kThreads || n_seq > 65535) return err_overflow();
    if (n_seq == 0) return clear_error();
    int32_t rc;
    if ((rc = check_array("counts", counts, counts_len, n_seq, 4)) ||
        (rc = check_array("pick", pick, pick_len, n_seq, 4)) ||
        (rc = check_array("tokens", tokens, tokens_len, rows, 4)) ||
        (rc = check_array("drafted", drafted, drafted_len, rows, 4)) ||
        (rc = check_array("accept", accept, accept_len, rows, 4)) ||
        (rc = check_array("starts", starts, n_seq + 1, n_seq + 1, 4)))
        return rc;
    if (rows && ((rc = check_tensor("target", target, target_len, MIVI_GGML_F32, rows, target_row_stride, 1, 0, n, false)) ||
                 (draft && (rc = check_tensor("draft", draft, draft_len, MIVI_GGML_F32, rows, draft_row_stride, 1, 0, n,
                                              false)))))
        return rc;
    const size_t need = mivi_hip_verify_rows_workspace(n, n_seq);
    if (workspace_bytes < need) return err_buffer_too_small(need, workspace_bytes);
    if (!workspace) return set_error(MIVI_ERR_INVALID_ARGUMENT, "null workspace");
    if ((uintptr_t)workspace % 16) return set_error(MIVI_ERR_INVALID_ARGUMENT, "workspace not 16-byte aligned");
    const size_t chunks = chunks_of(n);
    if (!grid_fits(chunks, kThreads) || chunks * n_seq > UINT32_MAX / kThreads) return err_overflow();
    clear_error();
    VerifyArgs a = {};
    a.target = target, a.draft = draft, a.t_row = (int64_t)target_row_stride, a.d_row = (int64_t)draft_row_stride;
    a.drafted = drafted, a.starts = starts, a.accept = accept, a.pick = pick;
    a.tokens = tokens, a.counts = counts;
    a.parts = (double2*)workspace, a.found = (int32_t*)(a.parts + n_seq * chunks);
    a.rows = (int)rows, a.n = (int)n, a.chunks = (int)chunks;
    hipStream_t s = (hipStream_t)stream;
    verify_sums_kernel<<<dim3((unsigned)chunks, (unsigned)n_seq), kThreads, 0, s>>>(a);
    MIVI_HIP_CHECK(hipGetLastError());
    verify_pick_kernel<<<(unsigned)n_seq, kThreads, 0, s>>>(a);
    MIVI_HIP_CHECK(hipGetLastError());
    return MIVI_OK;
}
