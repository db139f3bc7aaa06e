// Stores into the 8-bit key-value cache (cache_q8.hpp) and reads back from it.
//
// A store of T rows touches some blocks; the new scale of a block and kv head
// is s = max(s_old, amax / 127) over the finite new values (s_old = 0 where
// the block's first entry is among the rows: the block begins anew), and an
// entry is rint(x / s), ties to even, decided in 64 bits. Where s grew, the
// entries that stay are requantized, rint(q * s_old / s).
//
// A workgroup per (row, kv head) looks through the rows' indices; that of a
// block's first row takes all of the block's rows (of two with one index the
// last), the others end at once, mostly on their left neighbour's index. So a
// block is written by one workgroup and the result does not depend on order.
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
__device__ __forceinline__ void turn(float& xa, float& xb, int64_t pos, double inv_freq) {
    const double ang = (double)pos * inv_freq;
    const float c = (float)cos(ang), sn = (float)sin(ang), x1 = xa, x2 = xb;
    xa = x1 * c - x2 * sn;
    xb = x2 * c + x1 * sn;
}

__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// rint(x / s) + 128 for |x / s| <= 127 but for the scale's rounding; s = 0: zero.
__device__ __forceinline__ uint32_t q8_byte(double x, double s) {
    const double r = s > 0.0 ? __builtin_rint(x / s) : 0.0;
    return (uint32_t)((int)fmin(fmax(r, -127.0), 127.0) + 128);
}

template <int DP, bool ROPE>
__global__ __launch_bounds__(256) void store_q8_kernel(StoreArgs A) {
    constexpr int NP = DP / 16;  // pairs of a row that one of its eight threads holds
    constexpr int HALF = Q8C_BLOCK * DP;
    __shared__ __align__(16) uint8_t image[HALF];
    __shared__ int rows[Q8C_BLOCK];
    __shared__ float part[2][4];
    __shared__ uint32_t newbad;
    __shared__ int earlier;
    const int t = blockIdx.x, hk = blockIdx.y, tid = threadIdx.x;
    if constexpr (ROPE) {
        if (hk >= A.Hkv) {  // the workgroups behind the kv heads' turn q
            const int n = A.H * (A.d / 2);
            for (int j = (hk - A.Hkv) * 256 + tid; j < n; j += ((int)gridDim.y - A.Hkv) * 256) {
                const int h = j / (A.d / 2);
                const Pair p = pair_of(j - h * (A.d / 2), A.rotary, A.interleaved);
                if (!p.rot) continue;
                float* r = A.q + ((int64_t)t * A.H + h) * A.d;
                float xa = r[p.a], xb = r[p.b];
                turn(xa, xb, A.pos[t], A.inv_freq[A.interleaved ? p.a / 2 : p.a]);
                r[p.a] = xa;
                r[p.b] = xb;
            }
            return;
        }
    }
    const int64_t at = A.index[t];
    if (at < 0 || at >= A.C) return;  // outside the cache: not stored
    const int64_t blk = at >> 5;
    // (an index outside the cache may lie in its last, partial block)
    auto in_block = [&](int64_t i) { return i >= 0 && i < A.C && (i >> 5) == blk; };
    if (t > 0 && in_block(A.index[t - 1])) return;
    if (tid < Q8C_BLOCK) rows[tid] = -1;
    if (tid == 0) {
        newbad = 0;
        earlier = 0;
    }
    __syncthreads();
    for (int i = tid; i < A.T; i += 256) {
        const int64_t x = A.index[i];
        if (!in_block(x)) continue;
        if (i < t) earlier = 1;
        else atomicMax(&rows[x & (Q8C_BLOCK - 1)], i);
    }
    __syncthreads();
    if (earlier) return;

    // eight threads an entry: thread c holds its pairs c, c + 8, ...
    const int e = tid >> 3, c = tid & 7, row = rows[e], np = A.d / 2;
    const bool fresh = rows[0] >= 0;
    float kx[2 * NP], vx[2 * NP];
    float kmax = 0.f, vmax = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < NP; j++) {
        const int i = c + 8 * j;
        kx[2 * j] = kx[2 * j + 1] = vx[2 * j] = vx[2 * j + 1] = 0.f;
        if (row < 0 || i >= np) continue;
        const float* kr = A.k + ((int64_t)row * A.Hkv + hk) * A.d;
        const f32x2a4 v = *(const f32x2a4*)(A.v + ((int64_t)row * A.Hkv + hk) * A.d + 2 * i);
        float ka, kb;
        if constexpr (ROPE) {
            const Pair p = pair_of(i, A.rotary, A.interleaved);
            ka = kr[p.a];
            kb = kr[p.b];
            if (p.rot) turn(ka, kb, A.pos[row], A.inv_freq[i]);
        } else {
            ka = kr[2 * i];
            kb = kr[2 * i + 1];
        }
        bad |= !(finite_bits(ka) && finite_bits(kb) && finite_bits(v.x) && finite_bits(v.y));
        kx[2 * j] = finite_bits(ka) ? ka : 0.f;
        kx[2 * j + 1] = finite_bits(kb) ? kb : 0.f;
        vx[2 * j] = finite_bits(v.x) ? v.x : 0.f;
        vx[2 * j + 1] = finite_bits(v.y) ? v.y : 0.f;
        kmax = fmaxf(kmax, fmaxf(__builtin_fabsf(kx[2 * j]), __builtin_fabsf(kx[2 * j + 1])));
        vmax = fmaxf(vmax, fmaxf(__builtin_fabsf(vx[2 * j]), __builtin_fabsf(vx[2 * j + 1])));
    }
    if (bad) atomicOr(&newbad, 1u << e);
    kmax = wave_max_f32(kmax);
    vmax = wave_max_f32(vmax);
    if ((tid & 63) == 0) {
        part[0][tid >> 6] = kmax;
        part[1][tid >> 6] = vmax;
    }
    __syncthreads();
    const int dp = DP;
    Q8Meta* mp = (Q8Meta*)(A.cache + q8c_meta(A.nb, A.Hkv, hk, blk, dp));
    const Q8Meta old = *mp;
    uint32_t stored = 0;
    for (int i = 0; i < Q8C_BLOCK; i++) stored |= rows[i] >= 0 ? 1u << i : 0u;
    Q8Meta now;
    now.bad = (fresh ? 0u : old.bad & ~stored) | newbad;
    now.zero = 0;
    uint8_t* rec = A.cache + q8c_record(A.nb, hk, blk, dp);
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const float* pm = part[half];
        const float amax = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]));
        const float was = fresh ? 0.f : (half ? old.vs : old.ks);
        const float need = amax > 0.f ? fmaxf(amax / 127.f, Q8C_FLOOR) : 0.f;
        const float s = fmaxf(was, need);
        (half ? now.vs : now.ks) = s;
        uint8_t* dst = rec + half * HALF;
        const bool whole = fresh || need > was;  // the other entries change too
        if (whole) {
            for (int i = tid; i < HALF / 16; i += 256) {
                u32x4 w = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
                if (!fresh) {
                    w = ((const u32x4*)dst)[i];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint32_t r = 0;
                        for (int b = 0; b < 4; b++) {
                            const int qv = (int)((w[j] >> (8 * b)) & 255u) - 128;
                            r |= q8_byte((double)qv * (double)was, (double)s) << (8 * b);
                        }
                        w[j] = r;
                    }
                }
                ((u32x4*)image)[i] = w;
            }
            __syncthreads();
        }
        uint8_t* to = whole ? image : dst;
        if (row >= 0) {
#pragma unroll
            for (int j = 0; j < NP; j++) {
                const int i = c + 8 * j;
                if (i >= np) continue;
                Pair p = {2 * i, 2 * i + 1, false};
                if (ROPE && half == 0) p = pair_of(i, A.rotary, A.interleaved);
                const float xa = half ? vx[2 * j] : kx[2 * j], xb = half ? vx[2 * j + 1] : kx[2 * j + 1];
                to[half ? q8c_vbyte(e, p.a) : q8c_kbyte(e, p.a, dp)] = (uint8_t)q8_byte((double)xa, (double)s);
                to[half ? q8c_vbyte(e, p.b) : q8c_kbyte(e, p.b, dp)] = (uint8_t)q8_byte((double)xb, (double)s);
            }
        }
        if (whole) {
            __syncthreads();
            for (int i = tid; i < HALF / 16; i += 256) ((u32x4*)dst)[i] = ((const u32x4*)image)[i];
            __syncthreads();
        }
    }
    if (tid == 0) *mp = now;
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
                if ((m.bad >> e) & 1) ko[j] = vo[j] = __builtin_nanf("");
            }
        }
        *(f32x4a4*)(k + i * 4) = ko;
        *(f32x4a4*)(v + i * 4) = vo;
    }
}

template <bool ROPE>
hipError_t launch_store(const StoreArgs& a, hipStream_t s) {
    // q: a few hundred pairs a workgroup (each takes a 64-bit sine and cosine)
    const int qw = ROPE ? (a.H * (a.d / 2) + 255) / 256 : 0;
    const dim3 grid((unsigned)a.T, (unsigned)(a.Hkv + qw));
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
