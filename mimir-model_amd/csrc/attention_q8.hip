// Attention over the 8-bit key-value cache (cache_q8.hpp), to float32
// accuracy: out = sum_j p_j v_j / sum_j p_j, p_j = exp(q.k_j / sqrt(d) - m),
// over the entries that a query sees, in one pass with a running maximum.
//
// Both products run on v_mfma_f32_16x16x32_f16. The cached integers are exact
// in f16. What multiplies them is split into two f16 parts, hi = f16(x),
// lo = f16(x - hi), 22 bits together: a query row is first scaled by a power
// of two to a largest value in [2^14, 2^15), a weight is at most 2^15. A
// weight's lo is held 2^11 times up, its values 2^11 times down, so that small
// weights keep their bits (Weights, below). So a product is two instructions
// with a float32 sum, as near as float32 products are, at several times their
// rate.
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
//
// Bound: few rows (few_kernel) by the cache's bytes, read once for the query
// heads of a kv head; many rows of one sequence (many_kernel) by the matrix
// cores, 8 d flops a (query, key) pair with the two parts, 1240 to 1296 TFLOP/s
// in a large f16 product. Measured on MI355X, 32 heads, 8 kv heads, d = 128:
//   64 sequences of 2048 keys   41 us, 233 MB: 5.7 TB/s (a read kernel 7.05)
//   1 sequence of 131072 keys   49 us, 269 MB; 4.6 of them join_kernel
//   8 sequences of 2048 keys    10.8 us and join_kernel's 3.1: mostly the way
//                               from the launch to the first weight
//   2048 rows behind 6100 keys  406 to 419 us, 478 GFLOP: 1.14 to 1.18 PFLOP/s
// d = 64, one row of 181 keys 5.4 us. The two parts cost the decode rows nothing
// that shows (the matrix cores are at work 7 us of the 41, under the loads) and a
// prompt twice its products; with one part the outputs' error would be 2^-11, not
// float32's.
#include <algorithm>
#include <cmath>
#include <type_traits>

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

// In the present group of instructions: n times a product and then v vector ones.
template <int N, int V>
__device__ __forceinline__ void alternate() {
#pragma unroll
    for (int i = 0; i < N; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, V, 0);
    }
}

constexpr float M_NONE = -3.0e38f;  // a column's M before its first key
constexpr int COLS = 16;            // (token, head) pairs of a tile
// In place of a split's sum: the row is written (split 0); no more splits.
constexpr float DONE = -1.f, STOP = -2.f;

struct Args {
    const float* q;  // [T][H][d]
    const uint8_t* cache;
    const int64_t *kend, *kstart;
    int T, H, Hkv, G, d;
    float factor;    // log2(e) / sqrt(d)
    int64_t C, maxk, nb;
    float* out;      // [T][H][d]
    float* part;     // [splits][T * H][DP] sums, then [splits][T * H] of {M, l}
    int splits;      // of the keys, places in the workspace
    int few_splits;  // those that few_kernel cuts a token's keys into
    int many_splits; // and many_kernel a tile's
    int fours;       // see splits_of()
    int tpt, fan;    // tokens a tile of many_kernel; groups of workgroups of few_kernel that share one
    int group, inv;  // tokens whose columns fit a tile of 16; 256 / G, rounded up: c / G = c * inv / 256
    int least;       // blocks that a token sees at least, or many_kernel takes none
};

// Eight cache bytes as f16: 0x6400 | byte is 1024 + value + 128.
__device__ __forceinline__ v8h widen(uint32_t a, uint32_t b) {
    const v2h off = {(_Float16)1152.f, (_Float16)1152.f};
    const v2h w0 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - off;
    const v2h w1 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - off;
    const v2h w2 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - off;
    const v2h w3 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - off;
    return v8h{w0.x, w0.y, w1.x, w1.y, w2.x, w2.y, w3.x, w3.y};
}
// Values for the low parts of the weights, which are held LOW times up (below):
// times 1 / LOW, exact.
constexpr float LOW = 0x1p11f;
__device__ __forceinline__ v8h lowered(v8h v) {
    const _Float16 f = (_Float16)(1.f / LOW);
    return v * v8h{f, f, f, f, f, f, f, f};
}
__device__ __forceinline__ v4f mfma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// att_range for a token of the whole wave: its ends by scalar loads (nothing
// writes them while these kernels run).
__device__ __forceinline__ AttRange range_of(const Args& A, int t) {
    typedef const __attribute__((address_space(4))) int64_t* Constant;
    int64_t end = *(Constant)(uintptr_t)(A.kend + t), start = A.kstart ? *(Constant)(uintptr_t)(A.kstart + t) : 0;
    return att_range(&end, &start, 0, A.C, A.maxk);
}

// A block's scales in scalar registers, by scalar loads: the cache does not
// change while these kernels run, and blk is uniform. (In vector registers they
// cost many_kernel its last ones: 43 spilled, 34 us became 52 at 128 rows.)
struct Scales {
    float ks, vs;
    uint32_t bad;
};
__device__ __forceinline__ Scales scales_of(const Q8Meta* meta, int blk) {
    typedef const __attribute__((address_space(4))) u32x4* Constant;
    const u32x4 v = *(Constant)(uintptr_t)(meta + blk);
    return {__uint_as_float(v.x), __uint_as_float(v.y), v.z | v.w};
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Step s of a lane's query row: dims 64 (s / 2) + 16 g + 8 (s % 2) .. +7, the
// key operand's order.
struct Eight {
    float x[8];
};
__device__ __forceinline__ Eight query_step(const float* row, int d, int s, int g) {
    const int d0 = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
    f32x4a4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    if (d0 < d) {  // d is a multiple of 8
        a = *(const f32x4a4*)(row + d0);
        b = *(const f32x4a4*)(row + d0 + 4);
    }
    return Eight{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
// A row in two parts, scaled to a largest value in [2^14, 2^15) (NaN where it is
// not finite): returns the exponent that takes this back.
template <int DP>
__device__ __forceinline__ int row_exponent(const Eight* x, bool& finite) {
    float amax = 0.f;
    int f = 1;
#pragma unroll
    for (int s = 0; s < DP / 32; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            f &= (__float_as_uint(x[s].x[j]) & 0x7f800000u) != 0x7f800000u ? 1 : 0;
            amax = fmaxf(amax, __builtin_fabsf(x[s].x[j]));
        }
    amax = fmaxf(amax, lane_xor_f32<16>(amax));
    amax = fmaxf(amax, lane_xor_f32<32>(amax));
    f &= lane_xor<16>(f);
    f &= lane_xor<32>(f);
    finite = f;
    return amax > 0.f && f ? __builtin_amdgcn_frexp_expf(amax) - 15 : 0;
}
__device__ __forceinline__ void two_parts(const Eight& x, int exponent, bool finite, v8h& hi, v8h& lo) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float v = finite ? __builtin_ldexpf(x.x[j], -exponent) : __builtin_nanf("");
        const _Float16 h = (_Float16)v;
        hi[j] = h;
        lo[j] = (_Float16)(v - (float)h);
    }
}

// A column's running state: O^T tiles (dims 16 i + 4 g .. +3), M (the same in
// the four lanes of a column), l (each lane's own keys).
template <int DP>
struct State {
    v4f o[DP / 16];
    float M, l;
};

// A block's value scale for the exponents: log2 in whole steps and the rest in
// [0, 1), so that it costs no bits beside M, however far from one the scale is
// (as one number 1.6e-6 of an output where scales are near 2^-90 or 2^64, so 5e-7;
// 2048 rows behind 6100 keys 416 us as one, so 419); reciprocal (of a block of
// zeros the floor's; its weights are left out below).
struct Scale {
    float whole8, rest, iv;  // (weights are taken 2^8 up)
    __device__ __forceinline__ float log2() const { return whole8 - 8.f + rest; }
    // Of the exponents, with M taken off.
    __device__ __forceinline__ float offset(float M) const { return (whole8 - M) + rest; }
};
__device__ __forceinline__ Scale value_scale(const Scales& m) {
    const float vs = m.vs > 0.f ? m.vs : Q8C_FLOOR;
    const uint32_t b = __float_as_uint(vs);  // (a normal number)
    return {(float)((int)(b >> 23) - (127 - 8)), __builtin_amdgcn_logf(__uint_as_float((b & 0x7fffffu) | 0x3f800000u)), __builtin_amdgcn_rcpf(vs)};
}
// The factor of a row's scores of a block: the block's, log2(e) / sqrt(d) times
// its key scale, with the row's exponent (which alone may pass float32's range).
// At least float32's smallest normal number, so that -inf times it is -inf.
__device__ __forceinline__ float key_scale(float block, int exponent) {
    return __builtin_amdgcn_fmed3f(__builtin_ldexpf(block, exponent), 1.17549435e-38f, 3.40282347e38f);
}
// (In a chain: v_max3_f32 takes products as they come, v_max_f32 wants each
// made canonical first, one instruction more.)
__device__ __forceinline__ float largest(v4f s0, v4f s1) {
    const float a = fmaxf(fmaxf(s0.x, s0.y), s0.z), b = fmaxf(fmaxf(a, s0.w), s1.x), c = fmaxf(fmaxf(b, s1.y), s1.z);
    return fmaxf(c, s1.w);
}
// Whether a lane's scores need no more than their weights: the largest exponent
// is at most 15 (M is near enough), and not so small, -52, that the scale in it
// could matter. (NaN: no.)
__device__ __forceinline__ bool near_enough(float top, float cs, float base) {
    return __builtin_fabsf(__builtin_fmaf(top, cs, base) + 18.5f) <= 33.5f;
}

// What a block may need before its weights, in lanes or as a whole: entries
// that a column does not see (-inf) or that are not finite (NaN), M moved, and
// weights left out. Returns the exponents' offset; may change the scores and
// their factor.
template <int DP>
__device__ __forceinline__ float correct(v4f& s0, v4f& s1, const Scales& m, float& cs, Scale v, int blk, int g, int k0, int n,
                                         State<DP>& S) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float& x = j < 4 ? ((float*)&s0)[j] : ((float*)&s1)[j - 4];
        const int e = 16 * (j >> 2) + 4 * g + (j & 3);
        if ((m.bad >> e) & 1) x = __builtin_nanf("");
        if ((unsigned)(Q8C_BLOCK * blk + e - k0) >= (unsigned)n) x = -__builtin_inff();
    }
    const float lv = v.log2(), mx = largest(s0, s1) * cs + lv;
    if (__any(mx - S.M > 7.f)) {
        float cm = fmaxf(mx, lane_xor_f32<16>(mx));
        cm = fmaxf(cm, lane_xor_f32<32>(cm));
        const float M = fmaxf(S.M, cm), a = exp2_hw(0.5f * (S.M - M));
        S.M = M;
        S.l = S.l * a * a;  // (in two factors: l may be large where M is small)
#pragma unroll
        for (int i = 0; i < DP / 16; i++) S.o[i] *= a * a;
    }
    const bool zeros = !(m.vs > 0.f), below = mx < S.M - 60.f, out = zeros || below;
    float base = v.offset(S.M), pbase = 8.f - S.M;
    // Where M is 2^20 or more its own rounding shows beside the fused product's,
    // which has none: by 2^28 a column's largest exponent would be far from 8. The
    // products are rounded as they are in M there, and become the exponents.
    const bool far = __builtin_fabsf(S.M) >= 0x1p20f;
    if (__any(far)) {
        if (far) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s0[j] = (s0[j] * cs + lv) - S.M + 8.f;
                s1[j] = (s1[j] * cs + lv) - S.M + 8.f;
            }
            cs = 1.f;
            base = 0.f;
            pbase = -lv;
        }
    }
    // A block of zeros, and lanes whose w are all below 2^-60 of the largest,
    // count in the sum alone, as p: with the scale in them they could pass
    // float32's range (p beside w: at most 2^8 * 2^96, where the block's floor set M).
    if (!__any(out)) return base;
    if (out) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) sum += exp2_hw(__builtin_fmaf(j < 4 ? s0[j & 3] : s1[j & 3], cs, below ? pbase : base));
        S.l = __builtin_fmaf(sum, below ? 1.f : v.iv, S.l);
        base = -__builtin_inff();
    }
    return base;
}

// The eight weights of a lane in two parts, each rounded to nearest: h =
// f16(y), and what is left of y, LOW times up, so that it does not end where
// h does, at 2^-24. The largest y of a column is 2^8 or more, so the error is at
// most 2^-22 of a weight or 2^-44 of the largest, whichever is more, and does
// not lean to a side. Behind a first key 10 nats above the next largest, its
// value zero, outputs over 2000 and 100000 keys are 1.6e-6 and 3.2e-6 of sum p |v| off,
// behind one of 18 nats 7e-5 over 2000; with both parts in one scale, rounded
// towards zero, 1.5e-4, 2.1e-4 and 0.16. It costs 40 vector instructions of
// many_kernel's 215 a block: 2048 rows behind 6100 keys 414 us against 392.
struct Weights {
    uint32_t hi[4], lo[4];
    __device__ __forceinline__ v8h h() const { return __builtin_bit_cast(v8h, (u32x4){hi[0], hi[1], hi[2], hi[3]}); }
    __device__ __forceinline__ v8h r() const { return __builtin_bit_cast(v8h, (u32x4){lo[0], lo[1], lo[2], lo[3]}); }
};
// Those of one key tile: two words of each part; their sum.
__device__ __forceinline__ float weigh_tile(v4f s, float cs, float base, uint32_t* hi, uint32_t* lo) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = exp2_hw(__builtin_fmaf(s[j], cs, base));
#pragma unroll
    for (int j = 0; j < 2; j++) {
        hi[j] = __builtin_bit_cast(uint32_t, v2h{(_Float16)y[2 * j], (_Float16)y[2 * j + 1]});
        asm("" : "+v"(hi[j]));  // (one conversion for both, not once more for each half)
        const v2h h = __builtin_bit_cast(v2h, hi[j]);
        const v2h r = {(_Float16)__builtin_fmaf((float)h.x, -LOW, y[2 * j] * LOW),
                       (_Float16)__builtin_fmaf((float)h.y, -LOW, y[2 * j + 1] * LOW)};
        lo[j] = __builtin_bit_cast(uint32_t, r);
    }
    return (y[0] + y[1]) + (y[2] + y[3]);
}

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

constexpr int MAX_COLS = 128;  // columns of a tile of many_kernel, and so tokens

// The blocks that a workgroup's columns see, as disjoint rising ranges.
struct Ranges {
    int2 iv[MAX_COLS];
    int2 kn[MAX_COLS];  // each column's first key and number of keys
    int total;
};
// The blocks [s0, e0) and [s1, e1) of the tokens l and 64 + l of a tile (e = 0:
// none).
struct Spans {
    int s0, e0, s1, e1;
};
__device__ __forceinline__ int2 span_of(const Args& A, int t) {
    const AttRange r = att_range(A.kend, A.kstart, t, A.C, A.maxk);
    return r.n > 0 ? make_int2((int)(r.k0 >> 5), (int)((r.k0 + r.n + 31) >> 5)) : make_int2(0, 0);
}
// Those of the tokens from t0 up to a tile's number.
__device__ __forceinline__ Spans spans_of(const Args& A, int t0) {
    const int l = threadIdx.x & 63, t = t0 + l, last = min(A.T, t0 + A.tpt);
    const int2 a = t < last ? span_of(A, t) : make_int2(0, 0), b = t + 64 < last ? span_of(A, t + 64) : make_int2(0, 0);
    return {a.x, a.y, b.x, b.y};
}
// Whether many_kernel takes a tile: its tokens see the same blocks (a prompt),
// not each its own (a decode batch). many_kernel reads a block once for the
// tile, at 3.6 ns (128 columns of 128 dims, all compute units busy; on smaller
// grids twice that and more), few_kernel once for each token and 16 heads, at
// 0.8 ns from the caches: taken where the tokens' blocks are the tile's times its
// columns / 16. A last tile with few tokens goes as the last full number of tokens
// does, not to few_kernel, whose splits are for all tokens (130 rows of 32 heads
// behind 8000 keys, two in the last tile: 67 us, else 140). many_kernel takes no
// tile unless a token of it, or the call's last, sees `least` blocks. By a whole
// wave.
__device__ __forceinline__ bool takes_many(const Args& A, int t0, int cols) {
    const Spans p = spans_of(A, max(min(t0, A.T - A.tpt), 0));
    const int span = wave_max_i32(max(p.e0, p.e1)) - wave_min_i32(min(p.e0 ? p.s0 : 0x7fffffff, p.e1 ? p.s1 : 0x7fffffff));
    // (128 spans of 2^25 blocks pass an int; both kernels round the sum alike)
    const float sum = wave_sum_f32((float)(p.e0 - p.s0) + (float)(p.e1 - p.s1)) * (float)((A.G + COLS - 1) / COLS);
    const int2 end = span_of(A, A.T - 1);  // (a prompt's longest: its tiles go one way)
    const int most = max(wave_max_i32(max(p.e0 - p.s0, p.e1 - p.s1)), end.y - end.x);
    return sum > 0.f && most >= A.least && sum >= (float)(cols / 16) * (float)span;
}
// By one wave.
__device__ __forceinline__ void join_ranges(const Spans& p, Ranges& r) {
    const int s0 = p.s0, e0 = p.e0, s1 = p.s1, e1 = p.e1;
    int done = 0, n = 0, total = 0;
    for (;;) {
        const int s = wave_min_i32(min(e0 > done ? max(s0, done) : 0x7fffffff, e1 > done ? max(s1, done) : 0x7fffffff));
        if (s == 0x7fffffff) break;
        int e = s;
        for (;;) {
            const int e2 = wave_max_i32(max(s0 <= e && e0 > e ? e0 : e, s1 <= e && e1 > e ? e1 : e));
            if (e2 == e) break;
            e = e2;
        }
        if ((threadIdx.x & 63) == 0) r.iv[n] = make_int2(s, e);
        n++;
        total += e - s;
        done = e;
    }
    if ((threadIdx.x & 63) == 0) r.total = total;
}

template <int DP>
constexpr int MANY_COLS = DP <= 128 ? MAX_COLS : MAX_COLS / 2;

// Few rows: a workgroup per (token, kv head, split of the keys) and up to 16
// query heads. Its NW waves take the token's blocks in turn, straight from
// memory, each with a state of its own, joined at the end. A wave has its next
// block's keys in flight while it works on one, and the values during the
// score product (the values a block ahead as well, or both two blocks: 64 x
// 2048 keys 45 and 49 us against 40, with registers for four and three waves a
// SIMD where this has four; two are there). The query's parts lie in LDS (for
// the registers).
//
// GROUP (keys that are split, at most 8 query heads a kv head): the tokens whose
// heads fill the 16 columns, where three quarters of what they see is shared (a
// short prompt, a draft), are taken together, and the group's workgroups, one a
// token else, are further splits.
//
// BESIDE many_kernel: a workgroup takes every fan-th group of a tile that is not
// many_kernel's. (In one instance this loop cost every call its registers and
// nearly half a microsecond before the first load.)
constexpr int NW = 4;
template <int DP>
struct FewLds {
    union {
        v8h q[2][DP / 32][64];
        float o[NW][COLS][DP + 4];  // rows four banks apart
    };
    float ml[NW][2][COLS];
    int keys[COLS];  // that a column sees (a group's)
};
// The splits that so many blocks are worth, of n: of eight blocks, with `fours`
// (few workgroups) of four up to 16 of them; none up to 8 blocks. In a cache of
// 8192 keys, d = 64 / 128: 200 keys 7.1 / 8.5 us whole, 7.5 / 8.4 in two; 500 in
// four 7.5 / 8.4, in two 8.3 / 9.5; 2000 in 16 7.7 / 8.6, in eight 8.3 / 9.5. But 24
// rows of 16 heads behind 2000 keys in fours 12.5 us, in eights 11.2.
__host__ __device__ __forceinline__ int splits_of(int64_t n, int64_t blocks, bool fours) {
    const int64_t eight = (blocks + 7) / 8, four = (blocks + 3) / 4;
    const int64_t s = !fours || eight > 16 ? eight : (four < 16 ? four : 16);
    return blocks <= 8 ? 1 : (int)(n < s ? n : s);
}
template <int DP, bool BESIDE, bool GROUP>
__global__ __launch_bounds__(64 * NW, DP <= 128 ? 3 : 1) void few_kernel(Args A) {
    __shared__ FewLds<DP> S_;
    const int tid = threadIdx.x, l = tid & 63, g = l >> 4, col = l & 15, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // (divisions only where there is something to divide: a dozen of them are
    // most of a microsecond before the first load)
    const int sub = GROUP || A.G > COLS ? (int)blockIdx.x / A.Hkv : 0, hk = (int)blockIdx.x - sub * A.Hkv;
    const int g0 = GROUP ? 0 : sub * COLS, P = GROUP ? A.group : 1;  // (GROUP: sub is the workgroup's place)
    int t0 = (int)blockIdx.y * P, last = min(A.T, t0 + P);
    if constexpr (BESIDE) {
        const int unit = blockIdx.y, tile = unit / A.fan;
        if (takes_many(A, tile * A.tpt, MANY_COLS<DP>)) return;
        last = min(A.T, (tile + 1) * A.tpt);
        t0 = tile * A.tpt + (unit - tile * A.fan) * P;
        if (t0 >= last) return;
    }
    do {
    // The workgroup's columns: heads of a token, or of the group's tokens.
    const int t = t0 + (GROUP ? sub : 0);
    const AttRange own = range_of(A, min(t, A.T - 1));
    int head0 = t * A.H + hk * A.G + g0, step = 0, ncol = min(COLS, A.G - g0);
    int split = blockIdx.z;
    int k0 = (int)own.k0, n = (int)own.n;  // the keys that the lane's column sees
    int from = k0, to = k0 + n;            // and those that all columns see
    int b0 = k0 >> 5, total = n > 0 ? ((k0 + n + 31) >> 5) - b0 : 0;
    int nsplit = splits_of(A.few_splits, total, A.fours);
    bool packed = false;
    if constexpr (GROUP) {
        const int tc = (col * A.inv) >> 8, tn = min(P, last - t0);
        const AttRange r = att_range(A.kend, A.kstart, t0 + min(tc, tn - 1), A.C, A.maxk);
        const int rn = (int)r.n;
        int lo = rn > 0 ? (int)r.k0 : 0x7fffffff, hi = rn > 0 ? (int)r.k0 + rn : 0;
        int sum = rn > 0 && tc < tn && col == tc * A.G ? rn : 0;
        auto row16 = [&](auto f) {
            f(std::integral_constant<int, 1>{});
            f(std::integral_constant<int, 2>{});
            f(std::integral_constant<int, 4>{});
            f(std::integral_constant<int, 8>{});
        };
        row16([&](auto m) {
            lo = min(lo, lane_xor<m.value>(lo));
            hi = max(hi, lane_xor<m.value>(hi));
            sum += lane_xor<m.value>(sum);
        });
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
        sum = __builtin_amdgcn_readfirstlane(sum);
        packed = tn > 1 && hi > lo && (float)sum >= 0.75f * (float)tn * (float)(hi - lo);
        if (packed) {
            k0 = (int)r.k0;
            n = rn;
            from = k0;
            to = rn > 0 ? k0 + rn : 0;
            row16([&](auto m) {
                from = max(from, lane_xor<m.value>(from));
                to = min(to, lane_xor<m.value>(to));
            });
            from = __builtin_amdgcn_readfirstlane(from);
            to = __builtin_amdgcn_readfirstlane(to);
            b0 = lo >> 5;
            total = ((hi + 31) >> 5) - b0;
            head0 = t0 * A.H + hk * A.G;
            step = A.H - A.G;
            ncol = tn * A.G;
            nsplit = splits_of(min(A.few_splits * P, A.splits), total, false);
            split = split * P + sub;
            if (w == 0 && l < COLS) S_.keys[l] = n;
        } else if (sub >= tn) {
            split = nsplit;  // (nothing for this one)
        }
    }
    b0 = __builtin_amdgcn_readfirstlane(b0);
    total = __builtin_amdgcn_readfirstlane(total);
    if (split < nsplit) {
    const int mycol = min(col, ncol - 1);
    Eight x[DP / 32];
    const float* row = A.q + (int64_t)(head0 + mycol + (GROUP ? ((mycol * A.inv) >> 8) * step : 0)) * A.d;
#pragma unroll
    for (int s = 0; s < DP / 32; s++) x[s] = query_step(row, A.d, s, g);
    const int per = nsplit > 1 ? max((total + nsplit - 1) / nsplit, NW) : max(total, NW);
    int b = b0 + split * per + w;
    const int b1 = min(b0 + total, b0 + (split + 1) * per);
    const u32x4* rec = (const u32x4*)A.cache + l;
    constexpr int64_t REC = 2 * Q8C_BLOCK * DP / 16;
    const int64_t first = (int64_t)hk * A.nb;
    const Q8Meta* meta = (const Q8Meta*)(A.cache + q8c_meta(A.nb, A.Hkv, hk, 0, DP));
    u32x4 kb[DP / 32], vb[DP / 32];
    Scales m;
    auto fetch_k = [&](int blk) {
        const u32x4* p = rec + (first + blk) * REC;
#pragma unroll
        for (int i = 0; i < DP / 32; i++) kb[i] = __builtin_nontemporal_load(p + 64 * i);
        m = scales_of(meta, blk);
    };
    if (b < b1) fetch_k(b);
    bool finite;
    const int exponent = row_exponent<DP>(x, finite);
#pragma unroll
    for (int s = 0; s < DP / 32; s++)
        if (s % NW == w) two_parts(x[s], exponent, finite, S_.q[0][s][l], S_.q[1][s][l]);
    __syncthreads();
    State<DP> S;
#pragma unroll
    for (int i = 0; i < DP / 16; i++) S.o[i] = v4f{0.f, 0.f, 0.f, 0.f};
    S.M = M_NONE;
    S.l = 0.f;
    while (b < b1) {
        {
            const u32x4* p = rec + (first + b) * REC + 64 * (DP / 32);
#pragma unroll
            for (int i = 0; i < DP / 32; i++) vb[i] = __builtin_nontemporal_load(p + 64 * i);
        }
        v4f s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < DP / 64; i++)
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const u32x4 u = kb[kt * (DP / 64) + i];
                const v8h ka = widen(u.x, u.y), kc = widen(u.z, u.w);
                s[kt] = mfma(ka, S_.q[1][2 * i][l], s[kt]);
                s[kt] = mfma(kc, S_.q[1][2 * i + 1][l], s[kt]);
                s[kt] = mfma(ka, S_.q[0][2 * i][l], s[kt]);
                s[kt] = mfma(kc, S_.q[0][2 * i + 1][l], s[kt]);
            }
        const Scales mb = m;
        const int blk = b;
        b += NW;
        if (b < b1) fetch_k(b);
        const bool all_seen = from <= Q8C_BLOCK * blk && to >= Q8C_BLOCK * (blk + 1);
        const Scale v = value_scale(mb);
        float cs = key_scale(A.factor * mb.ks, exponent);
        float base = v.offset(S.M);
        if (!all_seen || mb.bad || !(mb.vs > 0.f) || __builtin_amdgcn_ballot_w64(near_enough(largest(s[0], s[1]), cs, base)) != ~0ull)
            base = correct<DP>(s[0], s[1], mb, cs, v, blk, g, k0, n, S);
        Weights W;
        const float sum = weigh_tile(s[0], cs, base, W.hi, W.lo) + weigh_tile(s[1], cs, base, W.hi + 2, W.lo + 2);
        S.l = __builtin_fmaf(sum, v.iv, S.l);
#pragma unroll
        for (int i = 0; i < DP / 32; i++) {
            __builtin_amdgcn_sched_barrier(0);
            const v8h va = widen(vb[i].x, vb[i].y), vc = widen(vb[i].z, vb[i].w);
            S.o[2 * i] = mfma(va, W.h(), S.o[2 * i]);
            S.o[2 * i + 1] = mfma(vc, W.h(), S.o[2 * i + 1]);
            S.o[2 * i] = mfma(lowered(va), W.r(), S.o[2 * i]);
            S.o[2 * i + 1] = mfma(lowered(vc), W.r(), S.o[2 * i + 1]);
        }
    }
    // join the waves' states
    S.l += lane_xor_f32<16>(S.l);
    S.l += lane_xor_f32<32>(S.l);
    if (l < COLS) {
        S_.ml[w][0][l] = S.M;
        S_.ml[w][1][l] = S.l;
    }
    __syncthreads();  // (every wave has read its query for the last time)
    if (col < ncol)
#pragma unroll
        for (int i = 0; i < DP / 16; i++) *(v4f*)&S_.o[w][col][16 * i + 4 * g] = S.o[i];
    __syncthreads();
    const int64_t rows = (int64_t)A.T * A.H;
    for (int i = tid; i < ncol * (DP / 4); i += 64 * NW) {
        const int c = i / (DP / 4), d4 = (i - c * (DP / 4)) * 4;
        float M = S_.ml[0][0][c];
#pragma unroll
        for (int j = 1; j < NW; j++) M = fmaxf(M, S_.ml[j][0][c]);
        float L = 0.f;
        v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NW; j++) {  // (in two factors: l may be large where M is small)
            const float f = exp2_hw(0.5f * (S_.ml[j][0][c] - M));
            L += S_.ml[j][1][c] * f * f;
            o += *(const v4f*)&S_.o[j][c][d4] * (f * f);
        }
        const int64_t head = head0 + c + (GROUP ? ((c * A.inv) >> 8) * step : 0);
        const bool none = split * per >= total || (GROUP && packed && S_.keys[c] <= 0);
        float2* ml = (float2*)(A.part + (int64_t)A.splits * rows * DP);
        if (nsplit > 1) {
            const int64_t at = (int64_t)split * rows + head;
            if (d4 == 0) ml[at] = make_float2(none ? -__builtin_inff() : M, L);
            if (!none) *(v4f*)(A.part + at * DP + d4) = o;
            if (d4 == 0 && split == 0 && A.splits > nsplit) ml[nsplit * rows + head] = make_float2(0.f, STOP);
        } else {
            if (d4 == 0 && A.splits > 1) ml[head] = make_float2(0.f, DONE);
            // a row that sees no key gives zeros, one whose weights are all zero NaN
            if (d4 < A.d)
                *(f32x4a4*)(A.out + head * A.d + d4) = none ? v4f{0.f, 0.f, 0.f, 0.f} : o * (L > 0.f ? 1.f / L : __builtin_nanf(""));
        }
    }
    }
    if constexpr (BESIDE) __syncthreads();  // (the last group's sums are read)
    } while (BESIDE && (t0 += A.fan * P) < last);
}

// Many rows: a workgroup per (tile of whole tokens, at most 64 NCT columns, kv
// head, split of the keys), 16 NCT columns a wave. A block's record is widened
// once for the four waves into LDS, in operand order, and an operand read from
// there serves 2 NCT products. Three buffers, one barrier a block: while a
// block is worked on, the next one's scores are taken, the one after it is
// written, and the one after that is in flight. (d = 64: three waves a SIMD,
// 2048 rows behind 8000 keys 349 us; two 361.)
template <int DP, int NCT>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : 2) void many_kernel(Args A) {
    constexpr int WC = 16 * NCT, PIECES = DP / 64;  // columns a wave; 16-byte pieces of a record a thread
    __shared__ v8h buf[3][DP / 8][64];
    __shared__ Ranges R;
    const int tid = threadIdx.x, l = tid & 63, g = l >> 4, col = l & 15, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % (unsigned)A.Hkv;
    // The last columns (the most keys of a prompt) first, but every other 256
    // workgroups rising: a CU's two share it, and get as many keys in all as
    // another's two.
    const int tiles = gridDim.x / (unsigned)A.Hkv, turn = max(256 / A.Hkv, 1), ti = blockIdx.x / (unsigned)A.Hkv;
    const int r0 = ti / turn * turn, tile = (ti / turn) & 1 ? r0 + min(turn, tiles - r0) - 1 - (ti - r0) : ti;
    const int t0 = (tiles - 1 - tile) * A.tpt, cols = min(A.tpt, A.T - t0) * A.G;
    if (!takes_many(A, t0, MANY_COLS<DP>)) return;
    if (w == 0) join_ranges(spans_of(A, t0), R);
    int exponent[NCT];
    v8h qhi[NCT][DP / 32], qlo[NCT][DP / 32];
    State<DP> S[NCT];
    int from = 0, to = 0x7fffffff;  // keys that all of the wave's columns see
#pragma unroll
    for (int ct = 0; ct < NCT; ct++) {
        const int c = min(WC * w + 16 * ct + col, cols - 1), t = t0 + c / A.G, head = t * A.H + hk * A.G + c % A.G;
        const AttRange r = att_range(A.kend, A.kstart, t, A.C, A.maxk);
        if (g == 0) R.kn[WC * w + 16 * ct + col] = make_int2((int)r.k0, (int)r.n);
        from = max(from, (int)r.k0);
        to = min(to, r.n > 0 ? (int)(r.k0 + r.n) : 0);
        Eight x[DP / 32];
#pragma unroll
        for (int s = 0; s < DP / 32; s++) x[s] = query_step(A.q + (int64_t)head * A.d, A.d, s, g);
        bool finite;
        exponent[ct] = row_exponent<DP>(x, finite);
#pragma unroll
        for (int s = 0; s < DP / 32; s++) two_parts(x[s], exponent[ct], finite, qhi[ct][s], qlo[ct][s]);
#pragma unroll
        for (int i = 0; i < DP / 16; i++) S[ct].o[i] = v4f{0.f, 0.f, 0.f, 0.f};
        S[ct].M = M_NONE;
        S[ct].l = 0.f;
    }
    from = wave_max_i32(from);
    to = wave_min_i32(to);
    __syncthreads();
    const int total = R.total, per = max((total + A.many_splits - 1) / A.many_splits, 8);
    const int p0 = (int)blockIdx.y * per, p1 = min(total, p0 + per);
    // The block of position p (rising): ranges [.., end) lie `shift` above theirs.
    int i = -1, end = 0, shift = 0;
    auto block_at = [&](int p) {
        while (p >= end) {
            const int2 iv = R.iv[++i];
            shift = __builtin_amdgcn_readfirstlane(iv.x) - end;
            end += __builtin_amdgcn_readfirstlane(iv.y) - __builtin_amdgcn_readfirstlane(iv.x);
        }
        return p + shift;
    };
    const Q8Meta* meta = (const Q8Meta*)(A.cache + q8c_meta(A.nb, A.Hkv, hk, 0, DP));
    u32x4 raw[PIECES];
    auto fetch = [&](u32x4 (&r)[PIECES], int blk) {
        const u32x4* p = (const u32x4*)(A.cache + q8c_record(A.nb, hk, blk, DP)) + tid;
#pragma unroll
        for (int j = 0; j < PIECES; j++) r[j] = p[256 * j];
    };
    // Half h of the thread's pieces: 0 .. DP / 32 - 1.
    auto put = [&](v8h (*b)[64], const u32x4 (&q)[PIECES], int h) {
        const u32x4 r = q[h >> 1];
        b[2 * (w + 4 * (h >> 1)) + (h & 1)][l] = h & 1 ? widen(r.z, r.w) : widen(r.x, r.y);
    };
    constexpr int NS = DP / 32;  // steps of a score product, and pairs of dim tiles
    int here = 0, next = 0, after = 0;  // blocks of positions p, p + 1 (in LDS), p + 2 (in flight)
    Scales mh{}, mn{};
    v4f sa[NCT][2], sb[NCT][2];
    float top[NCT];  // the largest of a lane's scores
    if (p0 < p1) {
        u32x4 raw0[PIECES], raw1[PIECES];
        here = next = after = block_at(p0);
        fetch(raw0, here);
        if (p0 + 1 < p1) next = after = block_at(p0 + 1);
        fetch(raw1, next);
        if (p0 + 2 < p1) after = block_at(p0 + 2);
        fetch(raw, after);
#pragma unroll
        for (int h = 0; h < NS; h++) put(buf[0], raw0, h);
#pragma unroll
        for (int h = 0; h < NS; h++) put(buf[1], raw1, h);
        mh = scales_of(meta, here);
        mn = scales_of(meta, next);
    }
    __syncthreads();
    if (p0 < p1) {
#pragma unroll
        for (int ct = 0; ct < NCT; ct++) sa[ct][0] = sa[ct][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NS; x++)
#pragma unroll
            for (int ct = 0; ct < NCT; ct++)
#pragma unroll
                for (int kt = 0; kt < 2; kt++) {
                    sa[ct][kt] = mfma(buf[0][kt * NS + x][l], qlo[ct][x], sa[ct][kt]);
                    sa[ct][kt] = mfma(buf[0][kt * NS + x][l], qhi[ct][x], sa[ct][kt]);
                }
#pragma unroll
        for (int ct = 0; ct < NCT; ct++) top[ct] = largest(sa[ct][0], sa[ct][1]);
    }
    int bi = 0;
    // One block: its weights beside the next block's score product, then the
    // second product beside the record after that (past the last block: what
    // the buffers hold, unused). In groups of 4 NCT products, a dozen or two
    // vector instructions between them: a wave's matrix and vector
    // instructions overlap when they alternate, those of two waves hardly do.
    // Operands are read from LDS a group ahead.
    auto step = [&](int p, v4f (&s)[NCT][2], v4f (&sn)[NCT][2]) {
        const int b1 = bi == 2 ? 0 : bi + 1, b2 = b1 == 2 ? 0 : b1 + 1;
        v8h (*kb)[64] = buf[b1], (*vb)[64] = buf[bi] + DP / 16, (*pb)[64] = buf[b2];
        v8h k0 = kb[0][l], k1 = kb[NS][l];
        const Scales m = mh;
        const Scale v = value_scale(m);
        const float block = A.factor * m.ks;
        float cs[NCT], base[NCT];
        bool fine = true;
#pragma unroll
        for (int ct = 0; ct < NCT; ct++) {
            cs[ct] = key_scale(block, exponent[ct]);
            base[ct] = v.offset(S[ct].M);
            fine &= near_enough(top[ct], cs[ct], base[ct]);
        }
        if (!(Q8C_BLOCK * here >= from && Q8C_BLOCK * (here + 1) <= to && m.bad == 0 && m.vs > 0.f && __builtin_amdgcn_ballot_w64(fine) == ~0ull)) {
#pragma unroll
            for (int ct = 0; ct < NCT; ct++) {
                const int2 k = R.kn[WC * w + 16 * ct + col];
                base[ct] = correct<DP>(s[ct][0], s[ct][1], m, cs[ct], v, here, g, k.x, k.y, S[ct]);
            }
        }
        here = next;
        next = after;
        mh = mn;
        mn = scales_of(meta, next);
        Weights W[NCT];
        float sum[NCT][2];
        v8h v0, v1;
#pragma unroll
        for (int ct = 0; ct < NCT; ct++) sn[ct][0] = sn[ct][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NS; x++) {
            __builtin_amdgcn_sched_barrier(0);
            v8h n0, n1;
            if (x + 1 < NS) {
                n0 = kb[x + 1][l];
                n1 = kb[NS + x + 1][l];
            } else {
                v0 = vb[0][l];
                v1 = vb[1][l];
            }
#pragma unroll
            for (int j = x * 2 * NCT / NS; j < (x + 1) * 2 * NCT / NS; j++)
                sum[j >> 1][j & 1] = weigh_tile(s[j >> 1][j & 1], cs[j >> 1], base[j >> 1], W[j >> 1].hi + 2 * (j & 1),
                                                W[j >> 1].lo + 2 * (j & 1));
#pragma unroll
            for (int ct = 0; ct < NCT; ct++) {
                sn[ct][0] = mfma(k0, qlo[ct][x], sn[ct][0]);
                sn[ct][1] = mfma(k1, qlo[ct][x], sn[ct][1]);
            }
#pragma unroll
            for (int ct = 0; ct < NCT; ct++) {
                sn[ct][0] = mfma(k0, qhi[ct][x], sn[ct][0]);
                sn[ct][1] = mfma(k1, qhi[ct][x], sn[ct][1]);
            }
            alternate<4 * NCT, 3>();
            k0 = n0;
            k1 = n1;
        }
#pragma unroll
        for (int ct = 0; ct < NCT; ct++) {
            S[ct].l = __builtin_fmaf(sum[ct][0] + sum[ct][1], v.iv, S[ct].l);
            asm volatile("" : "+v"(S[ct].l));  // (the sums among the products above)
        }
#pragma unroll
        for (int x = 0; x < NS; x++) {
            __builtin_amdgcn_sched_barrier(0);
            v8h n0, n1;
            if (x + 1 < NS) {
                n0 = vb[2 * x + 2][l];
                n1 = vb[2 * x + 3][l];
            }
            put(pb, raw, x);
            if (x == NS - 1)
#pragma unroll
                for (int ct = 0; ct < NCT; ct++) {
                    top[ct] = largest(sn[ct][0], sn[ct][1]);
                    asm volatile("" : "+v"(top[ct]));  // (here, not behind the products)
                }
#pragma unroll
            for (int ct = 0; ct < NCT; ct++) {
                S[ct].o[2 * x] = mfma(v0, W[ct].h(), S[ct].o[2 * x]);
                S[ct].o[2 * x + 1] = mfma(v1, W[ct].h(), S[ct].o[2 * x + 1]);
            }
            v0 = lowered(v0);  // (here by each wave: a second copy in LDS 424 us for 414, d = 64 390 for 340)
            v1 = lowered(v1);
#pragma unroll
            for (int ct = 0; ct < NCT; ct++) {
                S[ct].o[2 * x] = mfma(v0, W[ct].r(), S[ct].o[2 * x]);
                S[ct].o[2 * x + 1] = mfma(v1, W[ct].r(), S[ct].o[2 * x + 1]);
            }
            alternate<4 * NCT, DP <= 64 ? 1 : 2>();
            v0 = n0;
            v1 = n1;
        }
        __builtin_amdgcn_sched_barrier(0);
        if (p + 3 < p1) after = block_at(p + 3);
        fetch(raw, after);
        bi = b1;
        __syncthreads();
    };
    for (int p = p0; p < p1; p += 2) {
        step(p, sa, sb);
        if (p + 1 < p1) step(p + 1, sb, sa);
    }
    const int64_t rows = (int64_t)A.T * A.H;
#pragma unroll
    for (int ct = 0; ct < NCT; ct++) {
        float L = S[ct].l + lane_xor_f32<16>(S[ct].l);
        L += lane_xor_f32<32>(L);
        const int c = WC * w + 16 * ct + col, head = (t0 + c / A.G) * A.H + hk * A.G + c % A.G;
        if (c >= cols) continue;
        const bool none = p0 >= p1 || R.kn[WC * w + 16 * ct + col].y <= 0;
        if (A.splits > 1) {
            const int64_t at = (int64_t)blockIdx.y * rows + head;
            if (g == 0) {
                float2* ml = (float2*)(A.part + (int64_t)A.splits * rows * DP);
                ml[at] = make_float2(none ? -__builtin_inff() : S[ct].M, L);
                if (blockIdx.y == 0 && A.splits > A.many_splits) ml[A.many_splits * rows + head] = make_float2(0.f, STOP);
            }
            if (none) continue;
#pragma unroll
            for (int x = 0; x < DP / 16; x++) *(v4f*)(A.part + at * DP + 16 * x + 4 * g) = S[ct].o[x];
        } else {
            const float inv = L > 0.f ? 1.f / L : __builtin_nanf("");
#pragma unroll
            for (int x = 0; x < DP / 16; x++) {
                const int d0 = 16 * x + 4 * g;
                if (d0 < A.d) *(f32x4a4*)(A.out + (int64_t)head * A.d + d0) = none ? v4f{0.f, 0.f, 0.f, 0.f} : S[ct].o[x] * inv;
            }
        }
    }
}

// The splits of a row joined, DP / 4 threads a row and split. WIDE: a workgroup
// per row, 1024 / DP of its splits at a time; else 1024 / DP rows a workgroup.
template <int DP, bool WIDE>
__global__ __launch_bounds__(256) void join_kernel(Args A) {
    constexpr int LANES = DP / 4, GROUPS = 256 / LANES;
    __shared__ __align__(16) float os[WIDE ? GROUPS : 1][DP];
    const int64_t rows = (int64_t)A.T * A.H;
    const int tid = threadIdx.x, u = tid / LANES, d4 = (tid - u * LANES) * 4;
    const int64_t row = WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * GROUPS + u;
    const float2* pml = (const float2*)(A.part + (int64_t)A.splits * rows * DP);
    v4f o = {0.f, 0.f, 0.f, 0.f};
    float M = -__builtin_inff(), L = 0.f;
    if constexpr (WIDE) {
        const int l = tid & 63;
        const float2 x = l < A.splits ? pml[l * rows + row] : make_float2(-__builtin_inff(), 0.f);  // at most 64 splits
        if (__shfl(x.y, 0) == DONE) return;
        const unsigned long long stop = __ballot(x.y == STOP);
        const int splits = stop ? __builtin_ctzll(stop) : A.splits;
        const bool none = l >= splits || x.x == -__builtin_inff();
        M = wave_max_f32(none ? -__builtin_inff() : x.x);
        const float wh = none ? 0.f : exp2_hw(0.5f * (x.x - M));
        L = wave_sum_f32(none ? 0.f : x.y * wh * wh);
        // N loads a thread on their way together, without a branch between them, which
        // would make each wait (64 splits 4.6 us, with it 5.4; past the last split
        // one is read again, and what a split that holds nothing has is not used).
        auto add = [&](auto count) {
            constexpr int N = decltype(count)::value;
            v4f v[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int s = min(i * GROUPS + u, splits - 1);
                v[i] = *(const v4f*)(A.part + ((int64_t)s * rows + row) * DP + d4);
            }
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int s = i * GROUPS + u;
                const float f = __shfl(wh, s & 63);
                if (s < splits && f != 0.f) o += v[i] * (f * f);
            }
        };
        if (splits <= GROUPS) add(std::integral_constant<int, 1>{});
        else if (splits <= 2 * GROUPS) add(std::integral_constant<int, 2>{});
        else if (splits <= 4 * GROUPS) add(std::integral_constant<int, 4>{});
        else add(std::integral_constant<int, (64 + GROUPS - 1) / GROUPS>{});
        if (u < GROUPS) *(v4f*)&os[u][d4] = o;
        __syncthreads();
        if (u != 0) return;
#pragma unroll
        for (int j = 1; j < GROUPS; j++) o += *(const v4f*)&os[j][d4];
    } else {
        if (u >= GROUPS || row >= rows) return;
        // in batches of eight splits, all loads of one on their way together
        int splits = A.splits;
        for (int s0 = 0; s0 < splits; s0 += 8) {
            float2 x[8];
            v4f v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = s0 + j < A.splits ? pml[(s0 + j) * rows + row] : make_float2(-__builtin_inff(), 0.f);
            if (s0 == 0 && x[0].y == DONE) return;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (x[j].y == STOP) splits = min(splits, s0 + j);
                if (s0 + j >= splits) x[j] = make_float2(-__builtin_inff(), 0.f);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int s = min(s0 + j, A.splits - 1);
                v[j] = *(const v4f*)(A.part + ((int64_t)s * rows + row) * DP + d4);
            }
            float m = M;
#pragma unroll
            for (int j = 0; j < 8; j++) m = fmaxf(m, x[j].x);
            if (m == -__builtin_inff()) continue;
            const float a = M == -__builtin_inff() ? 0.f : exp2_hw(0.5f * (M - m));
            M = m;
            L = L * a * a;
            o *= a * a;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (x[j].x == -__builtin_inff()) continue;  // (what was read of it means nothing)
                const float wh = exp2_hw(0.5f * (x[j].x - M));
                L += x[j].y * wh * wh;
                o += v[j] * (wh * wh);
            }
        }
    }
    const float inv = M == -__builtin_inff() ? 0.f : (L > 0.f ? 1.f / L : __builtin_nanf(""));
    if (d4 < A.d) *(f32x4a4*)(A.out + row * A.d + d4) = M == -__builtin_inff() ? v4f{0.f, 0.f, 0.f, 0.f} : o * inv;
}

// How a call is cut.
struct Cut {
    bool many, fours;
    int tpt, fan, least, group;
    int64_t units, subs, many_wgs;
    int splits, few_splits, many_splits;
};
// The rules' constants, each with both sides as measured (MI355X, 32 heads, 8 kv
// heads, us, d = 64 / 128 where two are given).

// Up to these blocks of max_keys nothing is split: 8 sequences of 300 / 500 keys of
// 128 dims 8.0 / 9.0, with splits and join_kernel 10.3 / 10.6.
constexpr int64_t WHOLE_BLOCKS = 16;
// few_kernel's workgroups that splits are to give, two for each compute unit.
constexpr int64_t FEW_WGS = 512;
// Rows (times kv heads and 16s of query heads) from which few_kernel splits by
// eights of blocks, not by fours: see splits_of().
constexpr int64_t FOURS_ROWS = 16;
// Prompts are many_kernel's, a decode batch of as many sequences few_kernel's:
// the ranges, on the device, tell them apart, so both are launched, and each
// leaves the other's tiles. That costs a decode batch 5 to 9 us (64 sequences of 2000
// keys of 128 dims 40 in a cache of theirs, 48 where max_keys is 4096 and more; 256
// 82 and 87 / 155 and 164), so it is done from so many tokens and row-blocks
// (rows as above times blocks of max_keys) on.
constexpr int64_t MANY_TOKENS = 64, MANY_ROW_BLOCKS = 1 << 16;
// A prompt's rows cost few_kernel their number times the blocks, many_kernel a
// start of some 20 us: from as many row-blocks that the rows see on (on the device;
// the host knows max_keys) it takes them. few_kernel and many_kernel: 64 rows behind
// 2000 keys 21 and 24 / 31 and 33, behind 4000 34 and 28 / 52 and 34; 128 behind 1000
// 21 and 25 / 32 and 33, behind 2000 34 and 28 / 52 and 35; 256 behind none 12 and
// 19 / 19 and 25, behind 1000 37 and 29 / 58 and 38. From 512 tokens on that many are
// seen in any case.
constexpr int64_t LEAST_ROW_BLOCKS = 40000, LEAST_TOKENS = 512;
// Rows a workgroup of few_kernel beside many_kernel takes, by dims up to 64 and more:
// as many as give so many workgroups. 256 sequences of 2000 keys one by one / by twos
// / by fours 90, 87 and 102 / 168, 177 and 165.
constexpr int64_t BESIDE_WGS_64 = 1024, BESIDE_WGS = 512;
// many_kernel's splits: the least work of the fullest compute unit, its
// workgroups times their blocks, each with a start worth so many blocks; one
// alone on a unit has 3 / 5 of the rate of two (past 192 dims all of it). 384 rows
// behind 8000 keys of 128 dims, 96 workgroups: 147 in 6 splits, 118 in 5, 134 in 4;
// 1280 rows, 320: 450 whole, 385 in 2, 343 in 3 and 4; behind none 66, 66 and 75 in 3.
constexpr int64_t START_BLOCKS = 16;
// Rows up to which join_kernel takes a workgroup a row, and with more than so many
// splits: 256 rows (8 behind 8000 keys, 64 splits) 16 for the call, the other way
// 25; 2048 (64 behind 30000) 81 and 88; 4096 (128 behind 8000, 16) 57 and 59; but
// 8192 (256 behind 8000, 8) 88 and 86.
constexpr int WIDE_ROWS = 1024, WIDE_SPLITS = 8, WIDE_ROWS_SPLIT = 4096;

Cut cut(int64_t T, int H, int Hkv, int d, int64_t maxk) {
    const int64_t G = H / Hkv, subs = (G + COLS - 1) / COLS, blocks = (maxk + Q8C_BLOCK - 1) / Q8C_BLOCK;
    const int64_t cols = d <= 128 ? MAX_COLS : MAX_COLS / 2, rows = T * Hkv * subs;
    Cut c{};
    c.least = T < LEAST_TOKENS ? (int)(LEAST_ROW_BLOCKS / rows) : 0;
    c.many = T >= MANY_TOKENS && G <= cols && blocks >= c.least && rows * blocks >= MANY_ROW_BLOCKS;
    if (c.many) c.tpt = (int)(cols / G);
    c.fours = rows <= FOURS_ROWS;
    c.few_splits = (int)std::min<int64_t>((FEW_WGS - 1 + rows) / rows, blocks <= WHOLE_BLOCKS ? 1 : splits_of(64, blocks, c.fours));
    // Rows that split their keys may be of one sequence each, or a short prompt's:
    // the device packs the latter's tokens into a tile's columns, and their
    // workgroups share the keys (16 / 32 rows behind 8000 keys, d = 128, 33 and 55 us
    // apart, 19 and 25 so; without splits it gains nothing: 48 rows behind none 6.5
    // apart, 8.8 so).
    c.group = c.few_splits > 1 && G <= COLS / 2 ? (int)std::min<int64_t>(COLS / G, T) : 1;
    if (!c.many) c.tpt = c.group;
    const int64_t tiles = (T + c.tpt - 1) / c.tpt, groups = (c.tpt + c.group - 1) / c.group;
    c.many_wgs = tiles * Hkv;
    c.fan = 1;
    if (c.many) {
        const int64_t each = std::max<int64_t>(rows / (d <= 64 ? BESIDE_WGS_64 : BESIDE_WGS), 1);
        c.fan = (int)((groups + each - 1) / each);
    }
    c.units = tiles * c.fan;
    c.subs = subs;
    c.many_splits = 1;
    const int64_t most = blocks <= WHOLE_BLOCKS ? 1 : std::min<int64_t>(blocks / 8, 64);
    for (int64_t s = 1, best = INT64_MAX; c.many && s <= most; s++) {
        const int64_t n = (c.many_wgs * s + 255) / 256;
        const int64_t cost = n * ((blocks + s - 1) / s + START_BLOCKS) * (n == 1 && d <= 192 ? 5 : 3);
        if (cost < best) {
            best = cost;
            c.many_splits = (int)s;
        }
    }
    c.splits = c.few_splits > 1 ? std::min(c.few_splits * c.group, 64) : 1;
    if (c.many_splits > c.splits) c.splits = c.many_splits;
    return c;
}

template <int DP>
hipError_t launch(Args A, const Cut& c, hipStream_t s) {
    A.splits = c.splits;
    A.few_splits = c.few_splits;
    A.many_splits = c.many_splits;
    A.fours = c.fours;
    A.group = c.group;
    A.inv = (256 + A.G - 1) / A.G;
    A.tpt = c.tpt;
    A.fan = c.fan;
    A.least = c.least;
    const dim3 few((unsigned)(A.Hkv * c.subs * c.group), (unsigned)c.units, (unsigned)c.few_splits);
    if (c.many && c.group > 1) hipLaunchKernelGGL((few_kernel<DP, true, true>), few, dim3(64 * NW), 0, s, A);
    else if (c.many) hipLaunchKernelGGL((few_kernel<DP, true, false>), few, dim3(64 * NW), 0, s, A);
    else if (c.group > 1) hipLaunchKernelGGL((few_kernel<DP, false, true>), few, dim3(64 * NW), 0, s, A);
    else hipLaunchKernelGGL((few_kernel<DP, false, false>), few, dim3(64 * NW), 0, s, A);
    if (c.many)
        hipLaunchKernelGGL((many_kernel<DP, MANY_COLS<DP> / 64>), dim3((unsigned)c.many_wgs, (unsigned)c.many_splits), dim3(256), 0, s, A);
    const int rows = A.T * A.H, groups = 1024 / DP;
    if (c.splits > 1 && (rows <= WIDE_ROWS || (c.splits > WIDE_SPLITS && rows <= WIDE_ROWS_SPLIT)))
        hipLaunchKernelGGL((join_kernel<DP, true>), dim3((unsigned)rows), dim3(256), 0, s, A);
    else if (c.splits > 1)
        hipLaunchKernelGGL((join_kernel<DP, false>), dim3((unsigned)((rows + groups - 1) / groups)), dim3(256), 0, s, A);
    return hipGetLastError();
}

}  // namespace aq

uint64_t attention_q8_ws_bytes(int64_t T, int H, int Hkv, int d, int64_t maxk) {
    const aq::Cut c = aq::cut(T, H, Hkv, d, maxk);
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
    A.factor = (float)(1.4426950408889634 / std::sqrt((double)d));
    A.C = C;
    A.maxk = maxk;
    A.nb = q8c_blocks(C);
    A.out = out;
    A.part = ws;
    const aq::Cut c = aq::cut(T, H, Hkv, d, maxk);
    switch (q8c_dp(d)) {
    case 64: return aq::launch<64>(A, c, s);
    case 128: return aq::launch<128>(A, c, s);
    case 192: return aq::launch<192>(A, c, s);
    case 256: return aq::launch<256>(A, c, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mimg
