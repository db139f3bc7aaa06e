// Attention over the 8-bit key-value cache (cache_q8.hpp), to float32
// accuracy: out = sum_j p_j v_j / sum_j p_j, p_j = exp(q.k_j / sqrt(d) - m),
// over the entries that a query sees, in one pass with a running maximum.
//
// Both products run on v_mfma_f32_16x16x32_f16. The cached integers are exact
// in f16. What multiplies them is split into two f16 parts, hi = f16(x),
// lo = f16(x - hi), 22 bits together: a query row is first scaled by a power
// of two to a largest value in [2^14, 2^15), a weight is at most 2^15. So a
// product is two instructions with a float32 sum, as near as float32
// products are, at several times their rate.
//
// The scores are taken transposed, S^T = K Q^T: 16 columns are (token, query
// head) pairs of one kv head, and a lane ends with eight keys' scores of one
// column. Those are the lane's own operand of O^T = V^T P^T (the cache holds
// the values in that key order), so no weight moves between lanes.
//
// A block's value scale goes into the exponent: w_j = p_j * vs. The running
// maximum M is that of w (log2), the sum adds w_j / vs, and O = sum w_j * int
// needs no scaling by block. M moves only when a column's new maximum passes
// it by 2^7 (weights are taken 2^8 up, so they stay below 2^15): the rescaling
// of O is rare, and no maximum crosses lanes otherwise.
#include "cache_q8.hpp"
#include "decoder_math.hpp"
#include "mimg_device.hpp"
#include "mimg_kernels.hpp"

namespace mimg {
namespace aq {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr float M_NONE = -3.0e38f;  // a column's M before its first key
constexpr int COLS = 16;            // (token, head) pairs of a tile

struct Args {
    const float* q;  // [T][H][d]
    const uint8_t* cache;
    const int64_t *kend, *kstart;
    int T, H, Hkv, G, d;
    int64_t C, maxk, nb;
    float* out;      // [T][H][d]
    float* part;     // [splits][T * H][DP] sums, then [splits][T * H] of {M, l}
    int splits, cpt;  // cpt: columns a tile takes
};

__device__ __forceinline__ int wave_min_i32(int v) {
    v = min(v, lane_xor<32>(v));
    v = min(v, lane_xor<16>(v));
    v = min(v, lane_xor<8>(v));
    v = min(v, lane_xor<4>(v));
    v = min(v, lane_xor<2>(v));
    v = min(v, lane_xor<1>(v));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i32(int v) { return -wave_min_i32(-v); }

// Eight cache bytes as f16: 0x6400 | byte is 1024 + value + 128.
__device__ __forceinline__ v8h widen(uint32_t a, uint32_t b) {
    const v2h off = {(_Float16)1152.f, (_Float16)1152.f};
    const v2h w0 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - off;
    const v2h w1 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - off;
    const v2h w2 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - off;
    const v2h w3 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - off;
    return v8h{w0.x, w0.y, w1.x, w1.y, w2.x, w2.y, w3.x, w3.y};
}
__device__ __forceinline__ v4f mfma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The blocks that the columns of a tile see, as disjoint rising ranges.
struct Ranges {
    int2 iv[COLS];
    int n, total;
};
// By one wave; each lane gives the blocks [sb, eb) of a column (eb = 0: none).
__device__ __forceinline__ void join_ranges(int sb, int eb, Ranges& r) {
    int done = 0, n = 0, total = 0;
    for (;;) {
        const int s = wave_min_i32(eb > done ? max(sb, done) : 0x7fffffff);
        if (s == 0x7fffffff) break;
        int e = s;
        for (;;) {
            const int e2 = wave_max_i32(sb <= e && eb > e ? eb : e);
            if (e2 == e) break;
            e = e2;
        }
        if ((threadIdx.x & 63) == 0) r.iv[n] = make_int2(s, e);
        n++;
        total += e - s;
        done = e;
    }
    if ((threadIdx.x & 63) == 0) {
        r.n = n;
        r.total = total;
    }
}

// A column's query, its two parts as operands and the factor of its scores
// (log2, without the block's key scale; NaN where q is not finite).
template <int DP>
struct Query {
    v8h hi[DP / 32], lo[DP / 32];
    float scale;
};
template <int DP>
__device__ __forceinline__ void load_query(Query<DP>& Q, const float* row, int d, int g) {
    float amax = 0.f;
    bool fin = true;
    float x[DP / 32][8];
#pragma unroll
    for (int s = 0; s < DP / 32; s++) {
        const int d0 = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
        f32x4a4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
        if (d0 < d) {  // d is a multiple of 8
            a = *(const f32x4a4*)(row + d0);
            b = *(const f32x4a4*)(row + d0 + 4);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[s][j] = j < 4 ? a[j & 3] : b[j & 3];
            fin &= (__float_as_uint(x[s][j]) & 0x7f800000u) != 0x7f800000u;
            amax = fmaxf(amax, __builtin_fabsf(x[s][j]));
        }
    }
    amax = fmaxf(amax, lane_xor_f32<16>(amax));
    amax = fmaxf(amax, lane_xor_f32<32>(amax));
    int f = fin ? 1 : 0;
    f &= lane_xor<16>(f);
    f &= lane_xor<32>(f);
    // amax * 2^e in [2^14, 2^15)
    const int e = amax > 0.f && f ? 15 - __builtin_amdgcn_frexp_expf(amax) : 0;
    const float k = (float)(1.4426950408889634 / sqrt((double)d));
    Q.scale = f ? __builtin_ldexpf(k, -e) : __builtin_nanf("");
#pragma unroll
    for (int s = 0; s < DP / 32; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float v = f ? __builtin_ldexpf(x[s][j], e) : 0.f;
            const _Float16 h = (_Float16)v;
            Q.hi[s][j] = h;
            Q.lo[s][j] = (_Float16)(v - (float)h);
        }
}

// A column's running state: O^T tiles (dims 16 i + 4 g .. +3), M (the same in
// the four lanes of a column), l (each lane's own keys).
template <int DP>
struct State {
    v4f o[DP / 16];
    float M, l;
};

// The eight weights of a lane from its scores (key 16 kt + 4 g + i of block
// blk), M moved where needed, and the operands of the second product.
struct Weights {
    v8h hi, lo;
};
template <int DP>
__device__ __forceinline__ Weights weigh(v4f s0, v4f s1, const Q8Meta& m, float scale, int blk, int g, int k0, int n,
                                         bool all_seen, State<DP>& S) {
    const float vs = m.vs > 0.f ? m.vs : Q8C_FLOOR;
    const float lv = __builtin_amdgcn_logf(vs), cs = scale * m.ks;
    float iv = __builtin_amdgcn_rcpf(vs);
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = (j < 4 ? s0[j & 3] : s1[j & 3]) * cs;
    if (!all_seen || m.bad) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int e = 16 * (j >> 2) + 4 * g + (j & 3);
            if ((m.bad >> e) & 1) y[j] = __builtin_nanf("");
            if ((unsigned)(Q8C_BLOCK * blk + e - k0) >= (unsigned)n) y[j] = -__builtin_inff();
        }
    }
    float mx = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
    mx += lv;
    if (__any(mx > S.M + 7.f)) {
        float cm = fmaxf(mx, lane_xor_f32<16>(mx));
        cm = fmaxf(cm, lane_xor_f32<32>(cm));
        const float M = fmaxf(S.M, cm), a = exp2_hw(0.5f * (S.M - M));
        S.M = M;
        S.l = S.l * a * a;
#pragma unroll
        for (int i = 0; i < DP / 16; i++) S.o[i] *= a * a;
    }
    float base = lv - S.M + 8.f;
    // Where a lane's w are all below 2^-60 of the largest (a block of zeros or
    // nearly beside large values) they count in the sum alone, as p: with the
    // scale in them they could pass float32's range.
    const bool deep = mx < S.M - 60.f;
    if (__any(deep)) {
        base = deep ? 8.f - S.M : base;
        iv = deep ? 1.f : iv;
    }
    Weights w;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float p = exp2_hw(y[j] + base);
        sum += p;
        const _Float16 h = (_Float16)p;
        w.hi[j] = h;
        w.lo[j] = (_Float16)(p - (float)h);
    }
    S.l = __builtin_fmaf(sum, iv, S.l);
    if (!(m.vs > 0.f) || __any(deep)) {  // a block of zeros, whatever its integers
        const bool none = deep || !(m.vs > 0.f);
        w.hi = none ? v8h{} : w.hi;
        w.lo = none ? v8h{} : w.lo;
    }
    return w;
}

// Few columns: a workgroup per (tile of 16 columns, kv head, split of the
// keys); its four waves take blocks in turn, straight from memory, each with
// a state of its own, joined at the end.
template <int DP>
__global__ __launch_bounds__(256) void few_kernel(Args A) {
    __shared__ Ranges R;
    __shared__ float ml[4][2][COLS];
    __shared__ __align__(16) float os[2][COLS][DP];
    const int tid = threadIdx.x, l = tid & 63, g = l >> 4, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % (unsigned)A.Hkv, c0 = (blockIdx.x / (unsigned)A.Hkv) * A.cpt;
    const int ncol = min(A.cpt, A.T * A.G - c0), col = l & 15;
    const int c = c0 + min(col, ncol - 1), t = c / A.G;
    const int head = t * A.H + hk * A.G + (c - t * A.G);
    const AttRange r = att_range(A.kend, A.kstart, t, A.C, A.maxk);
    const int k0 = (int)r.k0, n = (int)r.n;
    if (w == 0) join_ranges(k0 >> 5, n > 0 ? (k0 + n + 31) >> 5 : 0, R);
    Query<DP> Q;
    load_query<DP>(Q, A.q + (int64_t)head * A.d, A.d, g);
    __syncthreads();
    const int total = R.total, per = max((total + A.splits - 1) / A.splits, 4);
    const int p0 = (int)blockIdx.y * per, p1 = min(total, p0 + per);
    State<DP> S;
#pragma unroll
    for (int i = 0; i < DP / 16; i++) S.o[i] = v4f{0.f, 0.f, 0.f, 0.f};
    S.M = M_NONE;
    S.l = 0.f;
    int i = 0, below = 0;  // blocks of the ranges before range i
    for (int p = p0 + w; p < p1; p += 4) {
        int2 iv = R.iv[i];
        while (p - below >= iv.y - iv.x) {
            below += iv.y - iv.x;
            iv = R.iv[++i];
        }
        const int blk = __builtin_amdgcn_readfirstlane(iv.x + p - below);
        const u32x4* rec = (const u32x4*)(A.cache + q8c_record(A.nb, hk, blk, DP)) + l;
        const Q8Meta m = *(const Q8Meta*)(A.cache + q8c_meta(A.nb, A.Hkv, hk, blk, DP));
        v4f s[2];
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
            s[kt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < DP / 64; x++) {
                const u32x4 u = rec[(kt * (DP / 64) + x) * 64];
                const v8h a = widen(u.x, u.y), b = widen(u.z, u.w);
                s[kt] = mfma(a, Q.lo[2 * x], s[kt]);
                s[kt] = mfma(b, Q.lo[2 * x + 1], s[kt]);
                s[kt] = mfma(a, Q.hi[2 * x], s[kt]);
                s[kt] = mfma(b, Q.hi[2 * x + 1], s[kt]);
            }
        }
        const bool all_seen = __all(k0 <= Q8C_BLOCK * blk && k0 + n >= Q8C_BLOCK * (blk + 1));
        const Weights W = weigh<DP>(s[0], s[1], m, Q.scale, blk, g, k0, n, all_seen, S);
#pragma unroll
        for (int x = 0; x < DP / 32; x++) {
            const u32x4 u = rec[(DP / 32 + x) * 64];
            const v8h a = widen(u.x, u.y), b = widen(u.z, u.w);
            S.o[2 * x] = mfma(a, W.lo, S.o[2 * x]);
            S.o[2 * x + 1] = mfma(b, W.lo, S.o[2 * x + 1]);
            S.o[2 * x] = mfma(a, W.hi, S.o[2 * x]);
            S.o[2 * x + 1] = mfma(b, W.hi, S.o[2 * x + 1]);
        }
    }
    // join: every wave's O to the largest M, then waves 2, 3 into 0, 1 and 1 into 0
    S.l += lane_xor_f32<16>(S.l);
    S.l += lane_xor_f32<32>(S.l);
    if (l < COLS) {
        ml[w][0][l] = S.M;
        ml[w][1][l] = S.l;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(ml[0][0][col], ml[1][0][col]), fmaxf(ml[2][0][col], ml[3][0][col]));
    float L = 0.f;
#pragma unroll
    for (int x = 0; x < 4; x++) {  // (in two factors: l may be large where M is small)
        const float f = exp2_hw(0.5f * (ml[x][0][col] - M));
        L += ml[x][1][col] * f * f;
    }
    const float a = exp2_hw(S.M - M);
#pragma unroll
    for (int x = 0; x < DP / 16; x++) S.o[x] *= a;
#pragma unroll
    for (int step = 2; step >= 1; step >>= 1) {
        if (w >= step && w < 2 * step)
#pragma unroll
            for (int x = 0; x < DP / 16; x++) *(v4f*)&os[w - step][col][16 * x + 4 * g] = S.o[x];
        __syncthreads();
        if (w < step)
#pragma unroll
            for (int x = 0; x < DP / 16; x++) S.o[x] += *(const v4f*)&os[w][col][16 * x + 4 * g];
        __syncthreads();
    }
    if (w != 0 || col >= ncol) return;
    if (A.splits > 1) {
        const int64_t rows = (int64_t)A.T * A.H, at = (int64_t)blockIdx.y * rows + head;
        float2* pml = (float2*)(A.part + (int64_t)A.splits * rows * DP);
        const bool none = p0 >= p1 || n == 0;
        if (g == 0) pml[at] = make_float2(none ? -__builtin_inff() : M, L);
        if (none) return;
#pragma unroll
        for (int x = 0; x < DP / 16; x++) *(v4f*)(A.part + at * DP + 16 * x + 4 * g) = S.o[x];
        return;
    }
    // a row that sees no key gives zeros, one whose weights are all zero NaN
    const float inv = n == 0 ? 0.f : (L > 0.f ? 1.f / L : __builtin_nanf(""));
#pragma unroll
    for (int x = 0; x < DP / 16; x++) {
        const int d0 = 16 * x + 4 * g;
        if (d0 < A.d) *(f32x4a4*)(A.out + (int64_t)head * A.d + d0) = n == 0 ? v4f{0.f, 0.f, 0.f, 0.f} : S.o[x] * inv;
    }
}

// The splits of a row joined: a wave per (token, head).
template <int DP>
__global__ __launch_bounds__(256) void join_kernel(Args A) {
    const int64_t rows = (int64_t)A.T * A.H, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int l = threadIdx.x & 63;
    if (row >= rows) return;
    const float2* pml = (const float2*)(A.part + (int64_t)A.splits * rows * DP);
    const float2 x = l < A.splits ? pml[l * rows + row] : make_float2(-__builtin_inff(), 0.f);  // at most 64 splits
    const float M = wave_max_f32(x.x);
    const float wl = x.x == -__builtin_inff() ? 0.f : exp2_hw(x.x - M);
    const float wh = exp2_hw(0.5f * (x.x - M));
    const float L = wave_sum_f32(x.x == -__builtin_inff() ? 0.f : x.y * wh * wh);
    const unsigned long long used = __ballot(x.x != -__builtin_inff());
    float o[DP / 64];
#pragma unroll
    for (int j = 0; j < DP / 64; j++) o[j] = 0.f;
    for (unsigned long long m = used; m; m &= m - 1) {
        const int s = __builtin_ctzll(m);
        const float f = __shfl(wl, s);
        const float* p = A.part + ((int64_t)s * rows + row) * DP + l;
#pragma unroll
        for (int j = 0; j < DP / 64; j++) o[j] = __builtin_fmaf(f, p[64 * j], o[j]);
    }
    const float inv = L > 0.f ? 1.f / L : __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < DP / 64; j++)
        if (64 * j + l < A.d) A.out[row * A.d + 64 * j + l] = used ? o[j] * inv : 0.f;
}

// How a call is cut: columns a tile and splits of the keys.
struct Cut {
    int cpt, tiles, splits;
};
Cut cut(int64_t T, int H, int Hkv, int64_t maxk) {
    const int64_t G = H / Hkv, cols = T * G;
    Cut c;
    // few tokens: a tile per token, each with its own range of keys (a decode
    // batch's sequences have none in common)
    c.cpt = G <= COLS && T < 64 ? (int)G : COLS;
    c.tiles = (int)((cols + c.cpt - 1) / c.cpt);
    const int64_t wgs = (int64_t)c.tiles * Hkv, blocks = (maxk + Q8C_BLOCK - 1) / Q8C_BLOCK;
    int64_t s = (1024 + wgs - 1) / wgs;
    if (s > blocks / 8) s = blocks / 8;
    c.splits = (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
    return c;
}

template <int DP>
hipError_t launch(Args A, const Cut& c, hipStream_t s) {
    A.cpt = c.cpt;
    A.splits = c.splits;
    hipLaunchKernelGGL(few_kernel<DP>, dim3((unsigned)(c.tiles * A.Hkv), (unsigned)c.splits), dim3(256), 0, s, A);
    if (c.splits > 1)
        hipLaunchKernelGGL(join_kernel<DP>, dim3((unsigned)(((int64_t)A.T * A.H + 3) / 4)), dim3(256), 0, s, A);
    return hipGetLastError();
}

}  // namespace aq

uint64_t attention_q8_ws_bytes(int64_t T, int H, int Hkv, int d, int64_t maxk) {
    const aq::Cut c = aq::cut(T, H, Hkv, maxk);
    return c.splits > 1 ? (uint64_t)c.splits * (uint64_t)T * (uint64_t)H * (q8c_dp(d) + 2) * 4 : 0;
}

hipError_t launch_attention_q8(const float* q, const void* cache, const int64_t* kend, const int64_t* kstart, int T, int H,
                               int Hkv, int d, int64_t C, int64_t maxk, float* out, float* ws, hipStream_t s) {
    aq::Args A{};
    A.q = q;
    A.cache = (const uint8_t*)cache;
    A.kend = kend;
    A.kstart = kstart;
    A.T = T;
    A.H = H;
    A.Hkv = Hkv;
    A.G = H / Hkv;
    A.d = d;
    A.C = C;
    A.maxk = maxk;
    A.nb = q8c_blocks(C);
    A.out = out;
    A.part = ws;
    const aq::Cut c = aq::cut(T, H, Hkv, maxk);
    switch (q8c_dp(d)) {
    case 64: return aq::launch<64>(A, c, s);
    case 128: return aq::launch<128>(A, c, s);
    case 192: return aq::launch<192>(A, c, s);
    case 256: return aq::launch<256>(A, c, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mimg
