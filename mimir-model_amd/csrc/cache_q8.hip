// Stores into the 8-bit key-value cache (cache_q8.hpp) and reads back from it.
//
// A store of T rows touches some blocks; the new scale of a block and kv head
// is s = max(s_old, amax / 127) over the finite new values (s_old = 0 where
// the block's first entry is among the rows: the block begins anew), and an
// entry is rint(x / s), ties to even, of the exact quotient. Where s grew, the
// entries that stay are requantized, rint(q * s_old / s).
//
// A workgroup per (row or a few, kv head, keys or values) looks through the
// rows' indices; that of a block's first row takes all of the block's rows (of
// two with one index the last), the others end at once, mostly on their left
// neighbour's index. So a block is written by one workgroup and the result
// does not depend on order.
//
// Bound: 8 d bytes read and 2 d written a row and kv head; at the usual sizes
// the chain from the index to the rows, the maximum and the bytes. Measured on
// MI355X, 8 kv heads of 128 dims: 1 row 4.2 us, 64 rows of 64 sequences 5.3, a
// prompt of 512 rows 7.9, of 2048 11 (21 MB: 1.9 TB/s), of 4000 19, 16384 90, 65535
// 1000: each block's workgroups look through the whole index, a third of the
// time at 4 x 1000 rows of 64 dims (15.6 us, of which 4.6) and most of it from 16384
// rows on. One workgroup for several heads looks once: 16384 rows by a third less,
// but 2048 by a quarter more, so each head looks for itself. With rope (32 query
// heads): 1 row 4.8 us, 64 rows of 64 sequences 6.4, prompts of 512 / 2048 / 4000 rows
// 13 / 30 / 50: a 64-bit sine and cosine for each pair of a row, once in each kv
// head's keys and once in q's.
#include "cache_q8.hpp"
#include "mimg_device.hpp"
#include "decoder_math.hpp"
#include "mimg_kernels.hpp"

namespace mimg {
namespace {

typedef float f32x2a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

struct StoreArgs {
    float* q;  // rotated in place (ROPE)
    const float *k, *v;
    const int64_t *index, *pos;
    const double* inv_freq;
    int T, H, Hkv, d, rotary, interleaved;
    int each, runs;  // rows a workgroup looks at; runs of 32 rows, a workgroup of each run in turn
    int groups;  // of workgroups that store, one for each kv head's keys and values; behind them those that turn q
    int qw;      // of which there are qw a row
    int64_t C, nb;
    uint8_t* cache;
};

// Dims a and b of pair i of a head, and whether rope.v1 turns it.
struct Pair {
    int a, b;
    bool rot;
};
__device__ __forceinline__ Pair pair_of(int i, int rotary, int interleaved) {
    const int h2 = rotary / 2;
    if (interleaved) return {2 * i, 2 * i + 1, i < h2};
    if (i < h2) return {i, i + h2, true};
    return {rotary + 2 * (i - h2), rotary + 2 * (i - h2) + 1, false};
}
// Cosine and sine of a pair's angle, in 64 bits, rounded.
__device__ __forceinline__ float2 turn_of(int64_t pos, double inv_freq) {
    double c, s;
    sincos((double)pos * inv_freq, &s, &c);
    return make_float2((float)c, (float)s);
}
__device__ __forceinline__ void turn(float& xa, float& xb, float2 cs) {
    const float x1 = xa, x2 = xb;
    xa = x1 * cs.x - x2 * cs.y;
    xb = x2 * cs.x + x1 * cs.y;
}

__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// rint(x / s) + 128, ties to even, of the exact quotient, for |x / s| < 128:
// r is x times s's float32 reciprocal, within 2^-15 of the quotient (three
// roundings of 2^-24, |r| < 128), so with f = floor(r) the quotient rounds to f
// or f + 1, and the sign of x - (f + 1/2) s says which: a fused multiply-add's
// sign is exact (x and s are whole multiples of 2^-149).
__device__ __forceinline__ uint32_t q8_round(float f, float sign) {
    const float h = f + 0.5f;
    const float n = sign > 0.f ? f + 1.f : (sign < 0.f ? f : __builtin_rintf(h));
    return (uint32_t)((int)fminf(fmaxf(n, -127.f), 127.f) + 128);
}
__device__ __forceinline__ uint32_t q8_new(float x, float inv, float s) {
    const float f = __builtin_floorf(x * inv);
    return q8_round(f, __builtin_fmaf(-(f + 0.5f), s, x));
}
// The same for x = q * was, an integer times the old scale. (f + 1/2) s = p + e;
// near p the difference q * was - p is exact (32-bit products, above 2^-25 of
// them), farther off its sign is plain.
__device__ __forceinline__ uint32_t q8_again(float q, float was, float ratio, float s) {
    const float f = __builtin_floorf(q * ratio), h = f + 0.5f;
    const float p = h * s, e = __builtin_fmaf(h, s, -p);
    return q8_round(f, __builtin_fmaf(q, was, -p) - e);
}

template <int DP, bool ROPE>
__global__ __launch_bounds__(256) void store_q8_kernel(StoreArgs A) {
    constexpr int NP = DP / 16;  // pairs of dims that a thread holds
    constexpr int HALF = Q8C_BLOCK * DP, WORDS = (HALF / 16 + 255) / 256;
    __shared__ __align__(16) uint8_t image[HALF];
    __shared__ int rows[Q8C_BLOCK];
    __shared__ int2 list[Q8C_BLOCK];  // the entries to store and their rows
    __shared__ float part[4];
    __shared__ uint32_t newbad;
    __shared__ int earlier;
    const int tid = threadIdx.x;
    int np = A.d / 2;
    if constexpr (ROPE) {
        if ((int)blockIdx.y >= A.groups) {  // the workgroups behind the stores' turn q
            // a thread keeps to one pair, so one 64-bit sine and cosine serve its heads
            const int u = ((int)blockIdx.y - A.groups) * (int)gridDim.x + (int)blockIdx.x, t = u / A.qw;
            if (t >= A.T) return;
            const int per = 256 / np, sub = tid / np, i = tid - sub * np;
            const Pair p = pair_of(i, A.rotary, A.interleaved);
            if (sub >= per || !p.rot) return;
            const float2 cs = turn_of(A.pos[t], A.inv_freq[i]);
            for (int h = (u - t * A.qw) * per + sub; h < A.H; h += A.qw * per) {
                float* r = A.q + ((int64_t)t * A.H + h) * A.d;
                float xa = r[p.a], xb = r[p.b];
                turn(xa, xb, cs);
                r[p.a] = xa;
                r[p.b] = xb;
            }
            return;
        }
    }
    const int hk = blockIdx.x >> 1, half = blockIdx.x & 1, g = blockIdx.y;
    const int t0 = A.runs > 1 ? g % A.runs * 32 + g / A.runs * A.each : g * A.each;
    const int64_t first = tid < A.T ? A.index[tid] : -1;
    // Lane j: row t0 + j and the one before it. The rows that may be a block's
    // first (outside the cache: not stored).
    const int tl = t0 + (tid & 63);
    const bool look_at = tl < A.T && (tid & 63) < A.each;
    const int64_t mine = look_at ? A.index[tl] : -1, left = look_at && tl > 0 ? A.index[tl - 1] : -1;
    const bool inside = mine >= 0 && mine < A.C;
    unsigned long long todo = __ballot(inside && !(left >= 0 && left < A.C && (left >> 5) == (mine >> 5)));
    for (; todo; todo &= todo - 1) {
        const int j0 = __builtin_ctzll(todo), t = t0 + j0;
        const int64_t at = __shfl(mine, j0), blk = at >> 5;
        // (an index outside the cache may lie in its last, partial block)
        auto in_block = [&](int64_t i) { return i >= 0 && i < A.C && (i >> 5) == blk; };
        uint8_t* dst = A.cache + q8c_record(A.nb, hk, blk, DP) + half * HALF;
        Q8Meta* mp = (Q8Meta*)(A.cache + q8c_meta(A.nb, A.Hkv, hk, blk, DP));
        // what is held, on its way unless this row begins the block anew
        u32x4 held[WORDS];
        float was = 0.f;
        uint32_t wasbad = 0;
        if ((at & 31) != 0) {
#pragma unroll
            for (int i = 0; i < WORDS; i++)
                if (tid + 256 * i < HALF / 16) held[i] = ((const u32x4*)dst)[tid + 256 * i];
            was = half ? mp->vs : mp->ks;
            wasbad = half ? mp->vbad : mp->kbad;
        }
        __syncthreads();  // (the last block is done)
        if (tid < Q8C_BLOCK) rows[tid] = -1;
        if (tid == 0) {
            newbad = 0;
            earlier = 0;
        }
        __syncthreads();
        auto look = [&](int i, int64_t x) {
            if (!in_block(x)) return;
            if (i < t) earlier = 1;
            else atomicMax(&rows[x & (Q8C_BLOCK - 1)], i);
        };
        if (tid < A.T) look(tid, first);
        for (int i = tid + 256; i < A.T; i += 8 * 256) {
            int64_t x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = i + 256 * j < A.T ? A.index[i + 256 * j] : -1;
#pragma unroll
            for (int j = 0; j < 8; j++) look(i + 256 * j, x[j]);
        }
        __syncthreads();
        if (earlier) continue;
        const bool used = (tid & 63) < Q8C_BLOCK && rows[tid & 31] >= 0;
        const uint32_t stored = (uint32_t)__ballot(used);
        if (tid < 64 && used) list[__popc(stored & ((1u << tid) - 1))] = make_int2(tid, rows[tid]);
        __syncthreads();
        const bool fresh = stored & 1;
        asm volatile("" : "+s"(np));  // (the items' places are not kept in registers over the blocks)
        const int items = __popc(stored) * np;
        uint32_t inv_np = ((1u << 20) + np - 1) / np;  // items / np: at most 4096 items
        float xs[2 * NP];
        float amax = 0.f;
        // (all loads on their way before the first is used)
#pragma unroll
        for (int j = 0; j < NP; j++) {
            const int it = tid + 256 * j;
            xs[2 * j] = xs[2 * j + 1] = 0.f;
            if (it < items) {
                const int u = (int)(((uint32_t)it * inv_np) >> 20), i = it - u * np;
                const int64_t row = ((int64_t)list[u].y * A.Hkv + hk) * A.d;
                if (ROPE && half == 0) {
                    const Pair p = pair_of(i, A.rotary, A.interleaved);
                    xs[2 * j] = A.k[row + p.a];
                    xs[2 * j + 1] = A.k[row + p.b];
                } else {
                    const f32x2a4 v = *(const f32x2a4*)((half ? A.v : A.k) + row + 2 * i);
                    xs[2 * j] = v.x;
                    xs[2 * j + 1] = v.y;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NP; j++) {
            const int it = tid + 256 * j;
            if (it >= items) continue;
            float &xa = xs[2 * j], &xb = xs[2 * j + 1];
            if (ROPE && half == 0) {
                // (unrolled, so that the pairs' sines overlap: a loop of one copy into LDS
                // takes a third longer for 64 rows of 8 heads of 128 dims)
                const int u = (int)(((uint32_t)it * inv_np) >> 20), i = it - u * np;
                if (pair_of(i, A.rotary, A.interleaved).rot) turn(xa, xb, turn_of(A.pos[list[u].y], A.inv_freq[i]));
            }
            if (!(finite_bits(xa) && finite_bits(xb))) {
                atomicOr(&newbad, 1u << list[(uint32_t)it * inv_np >> 20].x);
                xa = finite_bits(xa) ? xa : 0.f;
                xb = finite_bits(xb) ? xb : 0.f;
            }
            amax = fmaxf(amax, fmaxf(__builtin_fabsf(xa), __builtin_fabsf(xb)));
        }
        amax = wave_max_f32(amax);
        if ((tid & 63) == 0) part[tid >> 6] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
        if (fresh) was = 0.f;
        const float need = amax > 0.f ? fmaxf(amax / 127.f, Q8C_FLOOR) : 0.f, s = fmaxf(was, need);
        const float inv = s > 0.f ? 1.f / s : 0.f;
        const bool whole = fresh || need > was;  // the other entries change too
        if (whole) {
            const float ratio = was * inv;
#pragma unroll
            for (int i = 0; i < WORDS; i++) {
                if (tid + 256 * i >= HALF / 16) break;
                u32x4 w4 = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
                if (!fresh && was > 0.f) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint32_t r = 0;
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            const float qv = (float)((held[i][j] >> (8 * b)) & 255u) - 128.f;
                            r |= q8_again(qv, was, ratio, s) << (8 * b);
                        }
                        w4[j] = r;
                    }
                }
                ((u32x4*)image)[tid + 256 * i] = w4;
            }
            __syncthreads();
        }
        asm volatile("" : "+s"(inv_np));
        // an item's two bytes into the image, or straight into the record
        auto put = [&](uint8_t* to, int j) {
            const int it = tid + 256 * j;
            if (it >= items) return;
            const int u = (int)(((uint32_t)it * inv_np) >> 20), i = it - u * np, e = list[u].x;
            const Pair p = ROPE && half == 0 ? pair_of(i, A.rotary, A.interleaved) : Pair{2 * i, 2 * i + 1, false};
            to[half ? q8c_vbyte(e, p.a) : q8c_kbyte(e, p.a, DP)] = (uint8_t)q8_new(xs[2 * j], inv, s);
            to[half ? q8c_vbyte(e, p.b) : q8c_kbyte(e, p.b, DP)] = (uint8_t)q8_new(xs[2 * j + 1], inv, s);
        };
        if (whole) {
#pragma unroll
            for (int j = 0; j < NP; j++) put(image, j);
        } else {
#pragma unroll
            for (int j = 0; j < NP; j++) put(dst, j);
        }
        if (whole) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WORDS; i++)
                if (tid + 256 * i < HALF / 16) ((u32x4*)dst)[tid + 256 * i] = ((const u32x4*)image)[tid + 256 * i];
        }
        if (tid == 0) {
            const uint32_t bad = (fresh ? 0u : wasbad & ~stored) | newbad;
            if (half) {
                mp->vs = s;
                mp->vbad = bad;
            } else {
                mp->ks = s;
                mp->kbad = bad;
            }
        }
    }
}

// Entries index[t] as float32 rows [T, Hkv, d]: value * scale; zeros outside
// the cache, NaN where the entry held a value that is not finite. Four dims a
// thread.
__global__ __launch_bounds__(256) void load_q8_kernel(const uint8_t* __restrict__ cache, const int64_t* __restrict__ index,
                                                      int64_t quads, int Hkv, int d, int64_t C, int64_t nb,
                                                      float* __restrict__ k, float* __restrict__ v) {
    const int dp = q8c_dp(d), d4 = d / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < quads; i += (int64_t)gridDim.x * 256) {
        const int64_t th = i / d4;
        const int dd = (int)(i - th * d4) * 4, hk = (int)(th % Hkv);
        const int64_t at = index[th / Hkv];
        f32x4a4 ko = {0.f, 0.f, 0.f, 0.f}, vo = ko;
        if (at >= 0 && at < C) {
            const int64_t blk = at >> 5;
            const int e = (int)(at & 31);
            const Q8Meta m = *(const Q8Meta*)(cache + q8c_meta(nb, Hkv, hk, blk, dp));
            const uint8_t* rec = cache + q8c_record(nb, hk, blk, dp);
            const uint32_t kw = *(const uint32_t*)(rec + q8c_kbyte(e, dd, dp));
            const uint8_t* vp = rec + Q8C_BLOCK * dp;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                ko[j] = (float)((int)((kw >> (8 * j)) & 255u) - 128) * m.ks;
                vo[j] = (float)((int)vp[q8c_vbyte(e, dd + j)] - 128) * m.vs;
                if (((m.kbad | m.vbad) >> e) & 1) ko[j] = vo[j] = __builtin_nanf("");
            }
        }
        *(f32x4a4*)(k + i * 4) = ko;
        *(f32x4a4*)(v + i * 4) = vo;
    }
}

template <bool ROPE>
hipError_t launch_store(StoreArgs a, hipStream_t s) {
    // A decode batch's rows are a block each and want a workgroup each; of a
    // prompt's, one in 32 begins a block. The workgroups of every 32nd row come
    // one after another in the grid (then those of the rows behind these), so
    // that a prompt's, which all have such a row or all the one at the same
    // place, are spread over the compute units, and the rest end in their
    // shadow: 10.6 us for a prompt of 2048 rows of 8 heads of 128 dims, in the
    // rows' order 17.7. Rows a workgroup, 1 / 2 / 8 / 32: prompts of 512 rows 8.0, 7.8,
    // 7.7, 7.7 us, 1024 11.2, 8.5, 8.4, 8.4, 2048 20, 14, 10.6, 10.5, 4000 38, 27, 19.4,
    // 19.3; decode batches of 128 rows 7.9, 7.7, 16, 55, 512 25, 23, 26, 76, 2048 87, 80,
    // 80, 101. 64 decode rows 5.1 us one by one in their order (as a prompt's the
    // same, a prompt of 65 rows 7.4 and 7.0), by twos 6.4.
    a.each = a.T <= 64 ? 1 : (a.T <= 1024 ? 2 : (a.T <= 2048 ? 8 : 32));
    a.runs = a.T <= 64 ? 1 : (a.T + 31) / 32;
    a.groups = a.T <= 64 ? a.T : a.runs * (32 / a.each);
    const int parts = 2 * a.Hkv;
    const int rounds = (a.H + 256 / (a.d / 2) - 1) / (256 / (a.d / 2));  // heads a thread turns alone in its row
    a.qw = a.T > 64 ? 1 : (rounds < 256 ? rounds : 256);
    const dim3 grid((unsigned)parts, (unsigned)(a.groups + (ROPE ? (a.T * a.qw + parts - 1) / parts : 0)));
    switch (q8c_dp(a.d)) {
    case 64: hipLaunchKernelGGL((store_q8_kernel<64, ROPE>), grid, dim3(256), 0, s, a); break;
    case 128: hipLaunchKernelGGL((store_q8_kernel<128, ROPE>), grid, dim3(256), 0, s, a); break;
    case 192: hipLaunchKernelGGL((store_q8_kernel<192, ROPE>), grid, dim3(256), 0, s, a); break;
    case 256: hipLaunchKernelGGL((store_q8_kernel<256, ROPE>), grid, dim3(256), 0, s, a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_store_q8(const float* k, const float* v, const int64_t* index, int T, int Hkv, int d, int64_t C,
                              void* cache, hipStream_t s) {
    StoreArgs a{};
    a.k = k;
    a.v = v;
    a.index = index;
    a.T = T;
    a.Hkv = Hkv;
    a.d = d;
    a.C = C;
    a.nb = q8c_blocks(C);
    a.cache = (uint8_t*)cache;
    return launch_store<false>(a, s);
}

hipError_t launch_rope_kv_q8(float* q, const float* k, const float* v, const int64_t* pos, const int64_t* index,
                             const double* inv_freq, int T, int H, int Hkv, int d, int rotary, int interleaved,
                             int64_t C, void* cache, hipStream_t s) {
    StoreArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.index = index;
    a.pos = pos;
    a.inv_freq = inv_freq;
    a.T = T;
    a.H = H;
    a.Hkv = Hkv;
    a.d = d;
    a.rotary = rotary;
    a.interleaved = interleaved;
    a.C = C;
    a.nb = q8c_blocks(C);
    a.cache = (uint8_t*)cache;
    return launch_store<true>(a, s);
}

hipError_t launch_kv_load_q8(const void* cache, const int64_t* index, int T, int Hkv, int d, int64_t C, float* k, float* v,
                             hipStream_t s) {
    const int64_t quads = (int64_t)T * Hkv * (d / 4), wgs = (quads + 255) / 256;
    hipLaunchKernelGGL(load_q8_kernel, dim3((unsigned)(wgs < 65536 ? wgs : 65536)), dim3(256), 0, s, (const uint8_t*)cache,
                       index, quads, Hkv, d, C, q8c_blocks(C), k, v);
    return hipGetLastError();
}

}  // namespace mimg
