// Log probabilities of given tokens, the entropy and the largest alternatives
// of each row of logits, in one pass over them:
//   m = max x, S = sum e^(x - m), T = sum e^(x - m) (m - x)
//   logprob[t] = (x_t - m) - log S,  entropy = log S + T / S
// (every term of T is at least 0: no cancellation), alternatives by (value,
// lowest index), NaN never among them.
//
// chunk_kernel: a workgroup holds CHUNK logits of a row in registers, so the
// maximum, the sums and the alternatives take one read. The alternatives: of
// the 256 threads' maxima the k-th largest, tau, is at most the k-th largest
// value, and only the at most k threads not below it hold larger ones: the
// values above tau, and as many equal to it as are missing (lowest indices),
// go to LDS as 64-bit keys (value, ~index) and are ranked by counting.
// merge_kernel: a workgroup a row joins the chunks.
//
// Bound: the logits' bytes, once, for many rows; for few the two launches'
// chains of reductions. Measured on MI355X: 512 rows of 128256 logits, top 5,
// 47 to 50 us (263 MB: 6.0 TB/s in chunk_kernel's 44 us; a read kernel 7.05), top 20
// / 33 / 64 53 / 55 / 63 us (k keys of each of 16 chunks written, read and ranked by
// comparing all pairs, so the square of k); one row, top 20, 11.8 us, top 64 13.8; 37
// rows of 32003 of which a mask leaves 50, top 8, 12 us; without alternatives 44,
// 6.2 and 6.7 us.
#include "decoder_math.hpp"
#include "mimg_device.hpp"
#include "mimg_kernels.hpp"

namespace mimg {
namespace lp {

typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int VEC = 8;                // float4s a thread
constexpr int CHUNK = 256 * 4 * VEC;  // logits a workgroup
constexpr int KMAX = 64;

// Orders floats as unsigned integers (no negative zero: x + 0); 0 for NaN.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x == x ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

struct Part {
    float m, s, t, pad;
};

struct Args {
    const float* x;
    int64_t ld;
    int n, rows, chunks, top;
    const int32_t* targets;
    float *logprob, *entropy;
    int32_t* top_ids;
    float* top_lp;
    Part* part;      // [rows][chunks]
    uint64_t* keys;  // [rows][chunks][top], largest first, 0 past the last
};

// Keys cand[0..c) in LDS: the `top` largest, in order, into out (0 past c). Eight
// are read at a time; cand has room for seven more than c.
__device__ __forceinline__ void ranked(uint64_t* cand, int c, int top, uint64_t* out) {
    if (threadIdx.x < 7) cand[c + threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < c; i += 256) {
        const uint64_t k = cand[i];
        int r = 0;
        for (int j = 0; j < c; j += 8) {
            uint64_t o[8];
#pragma unroll
            for (int b = 0; b < 8; b++) o[b] = cand[j + b];
#pragma unroll
            for (int b = 0; b < 8; b++) r += o[b] > k ? 1 : 0;
        }
        if (r < top) out[r] = k;
    }
    for (int i = c + (int)threadIdx.x; i < top; i += 256) out[i] = 0;
}

__global__ __launch_bounds__(256) void chunk_kernel(Args A) {
    __shared__ float red[3][4];
    __shared__ uint32_t tmax[256];
    __shared__ uint64_t cand[KMAX * 4 * VEC + KMAX + 7];
    __shared__ int cnt[2][4];
    __shared__ uint32_t tau_s;
    __shared__ int ncand;
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    const int row = blockIdx.x / (unsigned)A.chunks, chunk = blockIdx.x - row * A.chunks;
    const float* xr = A.x + (int64_t)row * A.ld;
    const int i0 = chunk * CHUNK + 4 * tid;
    float x[4 * VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const int i = i0 + 1024 * j;
        if (i + 4 <= A.n) {
            const f32x4a4 v = __builtin_nontemporal_load((const f32x4a4*)(xr + i));
#pragma unroll
            for (int b = 0; b < 4; b++) x[4 * j + b] = v[b];
        } else {
#pragma unroll
            for (int b = 0; b < 4; b++) x[4 * j + b] = i + b < A.n ? xr[i + b] : -__builtin_inff();
        }
    }
    float mx = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < 4 * VEC; j++) mx = fmaxf(mx, x[j]);
    const float wm = wave_max_f32(mx);
    if (l == 0) red[0][w] = wm;
    if (tid == 0) ncand = 0;
    // the thread's largest value as a number; 0 where it holds no logit
    tmax[tid] = i0 < A.n ? order_of(mx) : 0u;
    __syncthreads();
    const float m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float mm = m == -__builtin_inff() ? 0.f : m;
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int j = 0; j < 4 * VEC; j++) {
        const float d = x[j] - mm, e = __builtin_amdgcn_exp2f(d * 1.44269504f);
        s += e;
        t = __builtin_fmaf(e, -fmaxf(d, -1.0e4f), t);  // (e is 0 there; never 0 * inf)
    }
    s = wave_sum_f32(s);
    t = wave_sum_f32(t);
    if (l == 0) {
        red[1][w] = s;
        red[2][w] = t;
    }
    if (A.top > 0 && w == 0) {
        // tau: the k-th largest of the threads' maxima, bit by bit, or as soon as
        // k of them are not below it
        const uint32_t a = tmax[l], b = tmax[64 + l], c = tmax[128 + l], d = tmax[192 + l];
        uint32_t tau = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t y = tau | 1u << bit;
            const int n = __popcll(__ballot(a >= y)) + __popcll(__ballot(b >= y)) + __popcll(__ballot(c >= y)) +
                          __popcll(__ballot(d >= y));
            if (n >= A.top) tau = y;
            if (n == A.top) break;
        }
        if (l == 0) tau_s = tau;
    }
    __syncthreads();
    if (tid == 0) {
        Part p;
        p.m = m;
        p.s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
        p.t = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
        p.pad = 0.f;
        A.part[(int64_t)row * A.chunks + chunk] = p;
    }
    if (A.top == 0) return;
    // below -inf: fewer than k threads hold a logit, all of theirs are taken
    const uint32_t tau = tau_s;
    const bool all = tau < 0x007FFFFFu;
    const float tf = all ? -__builtin_inff() : value_of(tau);
    // Those above tau, by the wave: counted, then stored (of 64 values mostly none).
    if (__any(mx > tf)) {
        int n = 0;
#pragma unroll
        for (int j = 0; j < 4 * VEC; j++) n += __popcll(__ballot(x[j] > tf));
        int at = 0;
        if (l == 0) at = atomicAdd(&ncand, n);
        at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
        for (int j = 0; j < 4 * VEC; j++) {
            const unsigned long long has = __ballot(x[j] > tf);
            if (has == 0) continue;
            if (x[j] > tf)
                cand[at + __popcll(has & ((1ull << l) - 1))] =
                    (uint64_t)order_of(x[j]) << 32 | (uint32_t)~(uint32_t)(i0 + 1024 * (j >> 2) + (j & 3));
            at += __popcll(has);
        }
    }
    __syncthreads();
    // Then those equal to tau of the lowest indices, 1024 j + 4 thread + b, step
    // by step until there are k (mostly one step: they are one, or a mask's).
    int c = ncand;
    uint32_t same = 0;
    if (c < A.top && mx >= tf)
#pragma unroll
        for (int j = 0; j < 4 * VEC; j++) same |= x[j] == tf && i0 + 1024 * (j >> 2) + (j & 3) < A.n ? 1u << j : 0u;
    for (int j = 0; j < VEC && c < A.top; j++) {
        const uint32_t four = (same >> (4 * j)) & 15u;
        int n = 0, at = 0;
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const unsigned long long has = __ballot((four >> b) & 1);
            n += __popcll(has);
            at += __popcll(has & ((1ull << l) - 1));
        }
        if (l == 0) cnt[j & 1][w] = n;
        __syncthreads();
        at += c;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int v = cnt[j & 1][i];
            at += i < w ? v : 0;
            c += v;
        }
#pragma unroll
        for (int b = 0; b < 4; b++)
            if (((four >> b) & 1) && at < A.top) cand[at++] = (uint64_t)order_of(tf) << 32 | (uint32_t)~(uint32_t)(i0 + 1024 * j + b);
    }
    c = min(c, max(A.top, ncand));
    ranked(cand, c, A.top, A.keys + ((int64_t)row * A.chunks + chunk) * A.top);
}

constexpr int MAX_CHUNKS = 256;

// Keys of a row that merge_kernel ranks as they are (of more it first drops what
// a bound excludes: 320 keys 8.7 us as they are, 5.5 with the bound), and that
// it reads ahead.
constexpr int AS_THEY_ARE = 128, HELD = 1024;

__global__ __launch_bounds__(256) void merge_kernel(Args A) {
    __shared__ float red[3][4];
    __shared__ uint64_t cand[(KMAX - 1) * KMAX + 1 + 7];
    __shared__ uint64_t held[HELD];
    __shared__ uint64_t heads[MAX_CHUNKS];
    __shared__ uint64_t best[KMAX];
    __shared__ uint64_t bound_s;
    __shared__ int ncand;
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, row = blockIdx.x;
    const Part* part = A.part + (int64_t)row * A.chunks;
    const uint64_t* keys = A.keys + (int64_t)row * A.chunks * A.top;
    const int nkeys = A.chunks * A.top;
    const bool small = nkeys <= AS_THEY_ARE, ahead = nkeys <= HELD;
    // all that is read, on its way at once
    Part p = {-__builtin_inff(), 0.f, 0.f, 0.f};
    if (tid < A.chunks) p = part[tid];
    uint64_t mine[HELD / 256];
    if (ahead) {
#pragma unroll
        for (int j = 0; j < HELD / 256; j++) mine[j] = tid + 256 * j < nkeys ? keys[tid + 256 * j] : 0;
    }
    float xt = 0.f;
    bool given = false;
    if (tid == 0 && A.logprob) {
        const int id = A.targets[row];
        given = id >= 0 && id < A.n;
        if (given) xt = A.x[(int64_t)row * A.ld + id];
    }
    const float wm = wave_max_f32(p.m);
    if (l == 0) red[0][w] = wm;
    if (tid < KMAX) best[tid] = 0;  // what stays 0 has no key
    if (tid == 0) {
        ncand = 0;
        bound_s = ~0ull;
    }
    if (ahead) {
#pragma unroll
        for (int j = 0; j < HELD / 256; j++)
            if (tid + 256 * j < nkeys) (small ? cand : held)[tid + 256 * j] = mine[j];
    }
    __syncthreads();
    const float m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    // a chunk's sums at the row's maximum: e^(x-m) = e^(x-p.m) f, m - x = (p.m - x) + away
    const float away = p.m == -__builtin_inff() ? 0.f : m - p.m;
    const float f = __builtin_amdgcn_exp2f(-away * 1.44269504f);
    const float s1 = wave_sum_f32(f * p.s);
    const float t1 = wave_sum_f32(f > 0.f || f != f ? f * __builtin_fmaf(away, p.s, p.t) : 0.f);
    if (l == 0) {
        red[1][w] = s1;
        red[2][w] = t1;
    }
    // A bound that at least k keys reach: of each chunk's r-th key the least, r =
    // ceil(k / chunks), or with k chunks and more the k-th largest first key.
    const int r = (A.top + A.chunks - 1) / A.chunks;
    if (!small && tid < A.chunks) heads[tid] = ahead ? held[tid * A.top + r - 1] : keys[tid * A.top + r - 1];
    __syncthreads();
    const float s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const float t = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
    const float log_s = logf(s);
    if (tid == 0) {
        if (A.entropy) A.entropy[row] = log_s + t / s;
        if (A.logprob) A.logprob[row] = given ? (xt - m) - log_s : 0.f;
    }
    if (A.top == 0) return;
    if (!small) {
        if (A.chunks < A.top) {
            if (tid < A.chunks) atomicMin((unsigned long long*)&bound_s, (unsigned long long)heads[tid]);
        } else if (tid < A.chunks) {
            const uint64_t k = heads[tid];
            int above = 0;
            for (int j = 0; j < A.chunks; j++) above += heads[j] > k ? 1 : 0;
            // (first keys are distinct but for the zeros of chunks without any)
            if (above < A.top) atomicMin((unsigned long long*)&bound_s, (unsigned long long)k);
        }
        __syncthreads();
        const uint64_t bound = bound_s;
        for (int i = tid; i < nkeys; i += 256) {
            const uint64_t k = ahead ? held[i] : keys[i];
            if (k != 0 && k >= bound) cand[atomicAdd(&ncand, 1)] = k;
        }
        __syncthreads();
    }
    ranked(cand, small ? nkeys : ncand, A.top, best);
    __syncthreads();
    if (tid < A.top) {
        const uint64_t k = best[tid];
        const int64_t at = (int64_t)row * A.top + tid;
        if (A.top_ids) A.top_ids[at] = k ? (int32_t)~(uint32_t)k : -1;
        if (A.top_lp) A.top_lp[at] = k ? (value_of((uint32_t)(k >> 32)) - m) - log_s : __builtin_nanf("");
    }
}

}  // namespace lp

int logprobs_max_n() { return lp::CHUNK * lp::MAX_CHUNKS; }

uint64_t logprobs_ws_bytes(int64_t rows, int64_t n, int top) {
    const uint64_t parts = (uint64_t)rows * (uint64_t)((n + lp::CHUNK - 1) / lp::CHUNK);
    return parts * (sizeof(lp::Part) + 8 * (uint64_t)top);
}

hipError_t launch_logprobs(const float* x, int64_t rows, int64_t n, int64_t ld, const int32_t* targets, int top,
                           float* logprob, float* entropy, int32_t* top_ids, float* top_lp, void* ws, hipStream_t s) {
    lp::Args A{};
    A.x = x;
    A.ld = ld;
    A.n = (int)n;
    A.rows = (int)rows;
    A.chunks = (int)((n + lp::CHUNK - 1) / lp::CHUNK);
    A.top = top;
    A.targets = targets;
    A.logprob = logprob;
    A.entropy = entropy;
    A.top_ids = top_ids;
    A.top_lp = top_lp;
    A.part = (lp::Part*)ws;
    A.keys = (uint64_t*)(A.part + (int64_t)rows * A.chunks);
    hipLaunchKernelGGL(lp::chunk_kernel, dim3((unsigned)(rows * A.chunks)), dim3(256), 0, s, A);
    hipLaunchKernelGGL(lp::merge_kernel, dim3((unsigned)rows), dim3(256), 0, s, A);
    return hipGetLastError();
}

}  // namespace mimg
