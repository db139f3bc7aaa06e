// The products of a mixture of experts: block-quantized weights of many
// experts [experts][N][K] x 8-bit activations, each (token, choice) pair with
// its expert's matrix, in the order of a plan (experts.hpp).
//
// Numerics. Per (weight row, activation row) and block the exact int32 sums of
// the other 8-bit products, then one float chain in block order:
//   Q4_K  S = sum_k sc_s(k) q_k y_k, M = sum_s m_s xs_s,
//         tot = fma(f32(S), d*dx, tot), off = fma(f32(M), dmin*dx, off)
//   Q6_K  S = sum_k sc_s(k) (q_k - 32) y_k, tot = fma(f32(S), d*dx, tot)
//   Q8_0  (blocks of 32) S = sum_k q_k y_k, tot = fma(f32(S), d*dx, tot)
// so a pair's row is bit for bit what its expert's matrix alone gives with
// dequant_matmul_a8.v2 (block 256), and for Q8_0 what the tiled product with
// blocks of 32 gives, whatever else the call holds.
//
// Layout. A workgroup of four waves takes BM = 32, 64 or (Q6_K) 96 pairs of one
// expert against 128 weight rows (32 a wave), or with swiglu against 64 rows of
// gate and the same 64 of up. The integer products are v_mfma_i32_32x32x32_i8:
// the activations are the row operand, the weights the column operand (lane l
// holds weight row l % 32), so a lane needs one block scale. A wave's raw blocks
// lie in an LDS slot of its own (read into registers, then overwritten by the
// next block's copies; Q4_K by whole lines of 128 bytes, two a row), the pairs'
// int8 rows (16-byte chunks XOR-swizzled by row) and scales in two shared stages;
// all of it by global_load_lds, one barrier a block. sc*q of Q4_K is split in
// two int8 planes, sc = 8 sh + sl, its mins are one v_mfma_f32_32x32x16_f16 over
// xs = 64 hi + lo (every operand and partial sum an integer that f16 and f32 hold
// exactly), as in gemm_q4k.hip; sc*(q - 32) of Q6_K is 256 hi + lo.
//
// Which workgroup has which tile is decided on the device: the grid is as
// large as any choice of that many pairs could need, a wave adds up the
// experts' tiles from the plan, and what is past the last tile ends. The tiles
// are in order by expert, weight rows, pairs, dealt to the XCDs in eight runs, so
// that the tiles that share weights meet in one L2.
//
// Bounds (calls one after another, with their quantizer). Few pairs an expert: the
// weights' way into LDS. 64 tokens, two of 8 experts, 4096 x 14336 Q4_K gate and up
// 121 to 133 us: 537 MB at 4.0 to 4.4 TB/s, where the copies alone take 108 to 117 us
// and the instructions alone 100; 181 tokens, four of 60, 2048 x 1408 Q8_0 85 us: 373
// MB at 4.4 TB/s. Many: vector instructions beside the matrix cores. 2048 tokens,
// two of 8: gate and up 1375 us, 0.70 POP/s of products and 1.4 of the planes' (the
// matrix cores at work 42 % of the cycles, vector instructions 66 %; a library
// product of 8192^3 on the same card 1.95), down 4096 x 14336 Q6_K 740 us for the tiles
// alone, 0.65 and 1.3 POP/s (38 and 66 %, conflicts of the LDS 20 %). Q8_0 has one
// plane, but a float step every 32 weights: gate and up 1880 us (23 and 60 %).
//
// Rows of x the quantizer refused and weight rows with a non-finite block
// scale take the float32 path (f32path.hpp) at the end.
#include <algorithm>
#include <type_traits>

#include "decoder_math.hpp"
#include "experts.hpp"
#include "f32path.hpp"
#include "mimg_device.hpp"
#include "mimg_kernels.hpp"

namespace mimg {
namespace xp {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v32f __attribute__((ext_vector_type(32)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

struct Mat {
    const uint8_t* W;     // [experts * N] rows
    const uint8_t* wref;  // [experts * N]
};

struct Args {
    Mat mat[2];           // the matrix, or gate and up
    float* y;             // [pairs][N]
    const int32_t* plan;
    int64_t rb, K;
    int64_t wbytes;       // bytes of a matrix of all experts
    int64_t wg0;          // workgroups of the launches before this one
    int N, nb, experts, pairs;  // nb: blocks (of 256; of 32 for Q8_0) of a row
    int rowdiv;           // a pair's activation row is pair / rowdiv
    ActPtrs act;
    const uint8_t* parts; // Q4_K: the sums of 32 as f16 parts, 32 bytes a block
    const float* x;       // f32 activations (fallback)
};

// AL (Q8_0): rows, and with them groups, start 4-byte aligned (K a multiple of
// 64), as the copies need it.
template <uint32_t DT, int MT_, bool AL_ = false, int RW_ = 32>
struct Cfg {
    static constexpr int RW = RW_;  // weight rows of a wave
    static constexpr bool AL = AL_;
    static constexpr int MT = MT_, T = 256, BM = 32 * MT;
    static constexpr bool K32 = DT == DT_Q8_0;
    // A row's group of 256 weights: the 16-byte chunks of its slot. Q6_K and
    // Q8_0 groups are 2-byte aligned: copied from the 16-byte boundary below
    // them, the chunks that cover them and one more where that spreads the
    // rows' dwords over the banks (60 and 76 dwords a row); aligned Q8_0 groups
    // are 17 whole chunks (68 dwords).
    static constexpr int GROUP = DT == DT_Q4_K ? Q4K_BYTES : DT == DT_Q6_K ? Q6K_BYTES : 8 * Q80_BYTES;
    static constexpr int WCH = DT == DT_Q4_K ? 9 : DT == DT_Q6_K ? 15 : AL ? 17 : 19;
    static constexpr int OCC = AL && MT == 1 ? 3 : 2;  // workgroups a compute unit holds
    static constexpr int WSLOT = 16 * WCH;
    // Q4_K: a row's bytes in whole lines of 128, two of them in the slot: a
    // block (144 bytes, from a multiple of 16 on) lies in two lines, and when it
    // is in registers at least one of them is free for the next. Block by
    // block every line that two blocks share would be fetched twice. The
    // chunks of a line are XOR-swizzled by row.
    static constexpr bool LINES = DT == DT_Q4_K;
    static constexpr int WDMA = LINES ? RW / 8 : (RW * WCH + 63) / 64;  // copies of a group, or of a line
    static constexpr int WWAVE = RW * (LINES ? 256 : WSLOT);
    static constexpr int WBYTES = 4 * WWAVE;
    static constexpr int ADMA = BM * 16 / T;
    static constexpr int ABYTES = BM * 256;
    static constexpr int XBYTES = DT == DT_Q4_K ? 32 * BM : 0;     // a row's sums in f16 parts
    static constexpr int DBYTES = K32 ? BM * 32 : (BM + 63) / 64 * 256;  // 8 scales a row, or one
    static constexpr int BUF = ABYTES + XBYTES + DBYTES;
    static constexpr int SMEM = WBYTES + 2 * BUF;
    static_assert(ADMA * T == BM * 16 && BM <= (DT == DT_Q4_K ? 64 : 128) && 2 * 64 * BM * 4 <= SMEM, "tile shape");
    static_assert(OCC * (SMEM + 8 * BM + 256) <= 160 * 1024, "workgroups a compute unit");
};

// s_waitcnt with vmcnt <= N (N < 64), the other counters unconstrained.
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xC07F); }

// A workgroup's tile: expert e, its pairs' first place in the order, how many
// of them the tile has, and the tile of weight rows.
struct Tile {
    int e, f0, m, nt;
};

// Inclusive sums over the wave: within rows of 16 lanes (shifts by 1, 2, 4, 8),
// then each row's last lane into the rows behind it.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return v;
}

template <int PER>
__device__ __forceinline__ bool find_tile_of(const Args& A, int ntn, int BM, Tile& r) {
    const int lane = threadIdx.x & 63;
    int f[PER], cnt[PER], upto[PER], total = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = 64 * i + lane, c = min(e, A.experts - 1);
        const int a = A.plan[c], b = A.plan[c + 1];
        f[i] = min(max(a, 0), A.pairs);
        cnt[i] = e < A.experts ? min(max(b, f[i]), A.pairs) - f[i] : 0;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        int s = (cnt[i] + BM - 1) / BM;
        s = wave_scan(s);
        upto[i] = total + s;
        total = __builtin_amdgcn_readlane(upto[i], 63);
    }
    const int64_t all = (int64_t)total * ntn, per = (all + 7) / 8;
    const int64_t wg = A.wg0 + blockIdx.x, idx = (wg & 7) * per + (wg >> 3);
    if ((wg >> 3) >= per || idx >= all) return false;
    const int u = (int)(idx / ntn);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const uint64_t past = __ballot(upto[i] > u);
        if (past == 0) continue;
        const int l = __ffsll((unsigned long long)past) - 1;
        const int n = __builtin_amdgcn_readlane(cnt[i], l), tiles = (n + BM - 1) / BM;
        const int first = __builtin_amdgcn_readlane(upto[i], l) - tiles;
        const int in = (int)(idx - (int64_t)first * ntn), mc = in % tiles;
        r.e = 64 * i + l;
        r.nt = in / tiles;
        r.f0 = __builtin_amdgcn_readlane(f[i], l) + mc * BM;
        r.m = min(n - mc * BM, BM);
        return true;
    }
    return false;
}
__device__ __forceinline__ bool find_tile(const Args& A, int ntn, int BM, Tile& r) {
    if (A.experts <= 64) return find_tile_of<1>(A, ntn, BM, r);
    if (A.experts <= 128) return find_tile_of<2>(A, ntn, BM, r);
    return find_tile_of<8>(A, ntn, BM, r);
}

// The copies of a thread: group 0's sources; group b adds a constant step.
template <uint32_t DT, class C>
struct Copies {
    // Weights: offsets from a base that the wave shares, 16-byte aligned.
    const uint8_t* wbase;
    uint32_t w[C::WDMA];
    int64_t wroom;  // bytes from the base to the last 16 that a copy may read
    const uint8_t *a[C::ADMA], *s;
    const uint8_t* d8[C::K32 ? C::DBYTES / 1024 : 1];
    uint32_t wave;
    __device__ __forceinline__ void init_weights(const Args& A, const Mat& M, int64_t row0, int n0) {
        const int t = threadIdx.x, l = t & 63;
        wave = __builtin_amdgcn_readfirstlane(t >> 6);
        const uint8_t* p = M.W + (row0 + min(n0, A.N - 1)) * A.rb;  // (a wave past the last row: that row)
        wbase = C::AL ? p : (const uint8_t*)__builtin_align_down(p, 16);
        const uint32_t mis = (uint32_t)(p - wbase);
        wroom = M.W + A.wbytes + WEIGHT_PAD - 16 - wbase;
#pragma unroll
        for (int i = 0; i < C::WDMA; i++) {
            const int c = min(64 * i + l, C::RW * C::WCH - 1);
            const int r = C::LINES ? 8 * i + (l >> 3) : c / C::WCH, j = C::LINES ? (l & 7) ^ ((r >> 1) & 7) : c - C::WCH * r;
            const uint32_t o = mis + (uint32_t)max(min(r, A.N - 1 - n0), 0) * (uint32_t)A.rb;
            // (Q6_K: rounded down for each block)
            w[i] = (C::AL || DT == DT_Q6_K ? o : o & ~15u) + 16 * j;
        }
    }
    __device__ __forceinline__ void init_rows(const Args& A, const int* rows) {
        const int t = threadIdx.x, l = t & 63;
#pragma unroll
        for (int i = 0; i < C::ADMA; i++) {
            const int c = C::T * i + t, r = c >> 4, k = c & 15;
            a[i] = (const uint8_t*)A.act.q + (int64_t)rows[r] * A.K + 16 * (k ^ (r & 15));
        }
        // (waves 0 and 1: scales of 64 rows each; 2 and 3: Q4_K's sums of 32)
        if (DT == DT_Q4_K && wave >= 2) {
            s = A.parts + (int64_t)rows[min(32 * (int)(wave - 2) + (l >> 1), C::BM - 1)] * (A.K / 8) + 16 * (l & 1);
        } else {
            s = (const uint8_t*)(A.act.d32 + (int64_t)rows[min(wave == 1 ? 64 + l : l, C::BM - 1)] * (A.K / 32));
        }
        if constexpr (C::K32) {
#pragma unroll
            for (int i = 0; i < C::DBYTES / 1024; i++) {
                const int c = C::T * i + t;
                d8[i] = (const uint8_t*)(A.act.d32 + (int64_t)rows[c >> 3] * (A.K / 32) + (c & 7));
            }
        }
    }
    // (LINES: line b instead of group b, the last one's end perhaps behind
    // the row, at most 112 bytes behind the buffer's last)
    __device__ __forceinline__ void line(int b, uint32_t lds) const {
#pragma unroll
        for (int i = 0; i < C::WDMA; i++)
            lds_copy16_at(wbase + 128 * (int64_t)b, w[i], lds + C::WWAVE * wave + C::RW * 128 * (b & 1) + 1024 * i);
    }
    // The last line that block b needs.
    static __device__ __forceinline__ int lines_to(int b) { return (9 * b + 8) >> 3; }
    __device__ __forceinline__ void weights(int b, uint32_t lds) const {
        if constexpr (C::LINES) {
            for (int i = b > 0 ? lines_to(b - 1) + 1 : 0; i <= lines_to(b); i++) line(i, lds);
            return;
        }
        const int l = threadIdx.x & 63;
        const uint8_t* base = wbase + (DT == DT_Q6_K ? 0 : (int64_t)b * C::GROUP);
        const int64_t room = wroom - (base - wbase);
        // A slot has more chunks than its group (Q6_K, Q8_0): those of the
        // last rows may not lie in the buffer, nor those of a last group of
        // fewer blocks.
        const uint32_t last = (uint32_t)min(room, (int64_t)0xFFFFFFF0) & ~15u;
#pragma unroll
        for (int i = 0; i < C::WDMA; i++) {
            uint32_t o = w[i];
            if constexpr (DT == DT_Q6_K) o = (o + (uint32_t)b * C::GROUP) & ~15u;
            if constexpr (DT != DT_Q4_K) o = min(o, last);
            if (64 * i + 64 <= C::RW * C::WCH || l < C::RW * C::WCH - 64 * i) lds_copy16_at(base, o, lds + C::WWAVE * wave + 1024 * i);
        }
    }
    __device__ __forceinline__ void activations(int b, uint32_t lds) const {
#pragma unroll
        for (int i = 0; i < C::ADMA; i++) lds_copy16(a[i] + 256 * (int64_t)b, lds + 1024 * wave + 16 * C::T * i);
        if constexpr (C::K32) {
#pragma unroll
            for (int i = 0; i < C::DBYTES / 1024; i++)
                lds_copy4(d8[i] + 32 * (int64_t)b, lds + C::ABYTES + 256 * wave + 4 * C::T * i);
        } else {
            if (DT == DT_Q4_K && wave >= 2 && 32 * (wave - 2) < C::BM) lds_copy16(s + 32 * (int64_t)b, lds + C::ABYTES + 1024 * (wave - 2));
            if (64 * wave < C::BM) lds_copy4(s + 32 * (int64_t)b, lds + C::ABYTES + C::XBYTES + 256 * wave);
        }
    }
};

// 16 bytes at an LDS address that is 2-byte aligned: five aligned dwords and
// a byte realignment.
__device__ __forceinline__ u32x4 lds_read16_a2(const uint8_t* p) {
    const uint32_t sh = (uint32_t)((uintptr_t)p & 3);
    const uint32_t* w = (const uint32_t*)__builtin_align_down(p, 4);
    const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3], w4 = w[4];
    return u32x4{__builtin_amdgcn_alignbyte(w1, w0, sh), __builtin_amdgcn_alignbyte(w2, w1, sh),
                 __builtin_amdgcn_alignbyte(w3, w2, sh), __builtin_amdgcn_alignbyte(w4, w3, sh)};
}
__device__ __forceinline__ uint32_t lds_read2_a2(const uint8_t* p) {
    const uint32_t w = *(const uint32_t*)__builtin_align_down(p, 4);
    return ((uintptr_t)p & 2) ? w >> 16 : w & 0xFFFFu;
}

// A lane's part of its weight row's group: the raw bytes in registers, from
// which the operands of a k step of 32 are built (lanes g = 0 and 1 of a row
// hold its elements 16 g .. 16 g + 15).
template <uint32_t DT, bool AL = false>
struct Group;

template <>
struct Group<DT_Q4_K> {
    u32x4 q[4];
    Q4KScales s;
    float d, dmin;
    // From the lines' slot: row is the lane's row in it with its swizzle.
    // Chunk c of the row (16 bytes) is at row ^ place(c).
    static __device__ __forceinline__ uint32_t place(int c) { return (uint32_t)(((c & 8) << 9) | ((c & 7) << 4)); }
    __device__ __forceinline__ void read(const uint8_t* slot, uint32_t row, int b, int g) {
        const u32x4 h = *(const u32x4*)(slot + (row ^ place(9 * b)));
        d = f16_to_f32(h.x & 0xFFFFu);
        dmin = f16_to_f32(h.x >> 16);
        s = q4k_scales(h.y, h.z, h.w);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint32_t p0 = place(9 * b + 1 + 2 * c), p1 = place(9 * b + 2 + 2 * c);
            q[c] = *(const u32x4*)(slot + (row ^ (g ? p1 : p0)));
        }
    }
    __device__ __forceinline__ void planes(int ks, int, v4i& H, v4i& L) const {
        const uint32_t sc = byte_of(s.sc, ks);
        const short sh = (short)(sc >> 3), sl = (short)(sc & 7);
        const s16x2 shp = {sh, sh}, slp = {sl, sl};
        const u32x4 qd = q[ks >> 1];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const s16x2 nib = as_s16x2((qd[k] >> (4 * (ks & 1))) & 0x0F0F0F0Fu);
            H[k] = (int)as_u32(nib * shp);
            L[k] = (int)as_u32(nib * slp);
        }
    }
    // The mins as the column operand of the f16 product: 64 m_s (g = 0), m_s (g = 1).
    __device__ __forceinline__ v8h mins(int g) const {
        const uint32_t mw[2] = {(uint32_t)s.m, (uint32_t)(s.m >> 32)};
        const h2 mul = g ? h2{(_Float16)1.0f, (_Float16)1.0f} : h2{(_Float16)64.0f, (_Float16)64.0f};
        const h2 c1024 = {(_Float16)1024.0f, (_Float16)1024.0f};
        v8h r;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t u = __builtin_amdgcn_perm(0u, mw[j >> 1], (j & 1) ? 0x0C030C02u : 0x0C010C00u);
            const h2 f = (__builtin_bit_cast(h2, u | 0x64006400u) - c1024) * mul;
            r[2 * j] = f.x;
            r[2 * j + 1] = f.y;
        }
        return r;
    }
};

template <>
struct Group<DT_Q6_K> {
    u32x4 ql[4], qh[2], sc;
    float d;
    __device__ __forceinline__ void read(const uint8_t* wr, int g) {
#pragma unroll
        for (int i = 0; i < 4; i++) ql[i] = lds_read16_a2(wr + 64 * (i >> 1) + 32 * (i & 1) + 16 * g);
#pragma unroll
        for (int h = 0; h < 2; h++) qh[h] = lds_read16_a2(wr + 128 + 32 * h + 16 * g);
        sc = lds_read16_a2(wr + 192);
        d = f16_to_f32(lds_read2_a2(wr + 208));
    }
    __device__ __forceinline__ void planes(int ks, int g, v4i& H, v4i& L) const {
        const int h = ks >> 2, p = ks & 3;
        const u32x4 lo = ql[2 * h + (p & 1)], hi = qh[h];
        // scale 8 h + 2 p + g, and w + 128 = scale q - 32 scale + 128 in 16 bits
        const uint32_t sw = sc[2 * h + (p >> 1)] >> (16 * (p & 1));
        const int s = (int)(int8_t)(uint8_t)(g ? sw >> 8 : sw);
        const short cu = (short)(128 - 32 * s);
        const s16x2 s2 = {(short)s, (short)s}, c2 = {cu, cu};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t q6 = (((p >> 1) ? (lo[k] >> 4) : lo[k]) & 0x0F0F0F0Fu) | (((hi[k] >> (2 * p)) & 0x03030303u) << 4);
            const uint32_t ue = as_u32(as_s16x2(__builtin_amdgcn_perm(0u, q6, 0x0C020C00u)) * s2 + c2);
            const uint32_t uo = as_u32(as_s16x2(__builtin_amdgcn_perm(0u, q6, 0x0C030C01u)) * s2 + c2);
            H[k] = (int)__builtin_amdgcn_perm(uo, ue, 0x07030501u);
            L[k] = (int)(__builtin_amdgcn_perm(uo, ue, 0x06020400u) ^ 0x80808080u);
        }
    }
};

template <bool AL>
struct Group<DT_Q8_0, AL> {
    // A block's 16 bytes of the lane as the five aligned dwords that hold them
    // (four where they are aligned).
    u32x4 w[8];
    uint32_t w4[8], sh;  // the first block's misalignment; the next one's is the other
    float d[8];
    __device__ __forceinline__ void read(const uint8_t* wr, int g) {
        sh = AL ? 2 : ((uint32_t)(uintptr_t)wr + 2) & 2;
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
            const uint8_t* p = wr + Q80_BYTES * ks;
            const uint32_t* q = (const uint32_t*)(AL ? p + (ks & 1 ? 2 : 0) + 16 * g : __builtin_align_down(p + 2 + 16 * g, 4));
            w[ks] = u32x4{q[0], q[1], q[2], q[3]};
            w4[ks] = AL && (ks & 1) ? 0 : q[4];
            d[ks] = f16_to_f32(AL ? (ks & 1 ? *(const uint32_t*)(p - 2) >> 16 : *(const uint32_t*)p & 0xFFFFu) : lds_read2_a2(p));
        }
    }
    __device__ __forceinline__ v4i block(int ks) const {
        if (AL && (ks & 1)) return __builtin_bit_cast(v4i, w[ks]);
        const uint32_t s = ks & 1 ? 2 - sh : sh;
        return v4i{(int)__builtin_amdgcn_alignbyte(w[ks].y, w[ks].x, s), (int)__builtin_amdgcn_alignbyte(w[ks].z, w[ks].y, s),
                   (int)__builtin_amdgcn_alignbyte(w[ks].w, w[ks].z, s), (int)__builtin_amdgcn_alignbyte(w4[ks], w[ks].w, s)};
    }
};

template <uint32_t DT, class C, bool SW>
__global__ __launch_bounds__(C::T, C::OCC) void tile_kernel(Args A) {
    constexpr int MT = C::MT, BM = C::BM, BN = SW ? 64 : 128;
    __shared__ __align__(16) uint8_t smem[C::SMEM];  // weights, then two activation stages
    __shared__ int rows[BM], outs[(BM + 63) / 64 * 64], flags[1];
    const int t = threadIdx.x, l = t & 63, wave = t >> 6;
    const int a = l & 31, g = l >> 5;
    Tile tile;
    if (!find_tile(A, (A.N + BN - 1) / BN, BM, tile)) return;
    const int n0 = tile.nt * BN, wn0 = n0 + 32 * (SW ? wave & 1 : wave);  // this wave's first weight row
    const int64_t row0 = (int64_t)tile.e * A.N;
    // (by value through a scalar: the copies take their base from it)
    const bool second = SW && __builtin_amdgcn_readfirstlane(wave) >= 2;
    const Mat M = {second ? A.mat[1].W : A.mat[0].W, second ? A.mat[1].wref : A.mat[0].wref};

    Copies<DT, C> cp;
    cp.init_weights(A, M, row0, __builtin_amdgcn_readfirstlane(wn0));
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem);
    // The tile's pairs, behind them the weights (which need the tile alone):
    // the first ones have landed when at most the weights' copies are left.
    // (Past the tile's pairs the last one again, whose results are not written.)
    if (64 * cp.wave < BM) lds_copy4(A.plan + plan_layout(A.pairs, A.experts).order + tile.f0 + min(t, tile.m - 1), outs + 64 * cp.wave);
    cp.weights(0, lds0);
    if (64 * cp.wave < BM) wait_vmcnt<C::WDMA>();
    if (t == 0) flags[0] = 0;
    lds_barrier();
    if (t < BM) {
        const int pair = min(max(outs[t], 0), A.pairs - 1);
        outs[t] = pair;
        rows[t] = pair / A.rowdiv;
    }
    lds_barrier();
    cp.init_rows(A, rows);
    cp.activations(0, lds0 + C::WBYTES);
    {
        int f = 0;
        if (l < 32) f |= wn0 + l < A.N && M.wref[row0 + wn0 + l] != 0;
        if (t < tile.m) f |= A.act.ok[rows[t]] == 0;
        if (f) flags[0] = 1;
    }
    float tot[MT][16], off[DT == DT_Q4_K ? MT : 1][16];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            tot[i][r] = 0.f;
            if (DT == DT_Q4_K) off[i][r] = 0.f;
        }
    const int asw = (a & 15) ^ g;  // chunk 2 ks + g of row a: slot 2 ks ^ asw
    // the lane's group in its slot (Q6_K, Q8_0: from the boundary below it)
    const uint32_t wmis = DT == DT_Q4_K ? 0 : (uint32_t)(uintptr_t)(M.W + (row0 + min(wn0 + a, A.N - 1)) * A.rb);
    const int ng = C::K32 ? (A.nb + 7) / 8 : A.nb;
    // The row's groups, for the first 32 L pairs and R results of a lane (the
    // pairs below 2 R of 32). Half the float step where a tile of 32 has at most 16
    // pairs: 64 tokens, eight of 64 experts, gate and up 2048 x 1024 44.0 -> 42.6 us,
    // 8 tokens 29.4 -> 29.0, 37 tokens, four of 60, down Q8_0 50.5 -> 49.3; a quarter
    // for 8 gives nothing more. Half of all: of tiles of 64 an expert's last
    // one is often half empty (512 tokens, gate and up of eight of 64 experts 2048 x
    // 1024 84.6 -> 81.5 us, of two of 8 4096 x 14336 402 -> 393, 2048 tokens 1280 ->
    // 1273; tiles of 96 have no registers left for a second form, 772 -> 796).
    auto groups = [&](auto live, auto results) __attribute__((always_inline)) {
        constexpr int L = decltype(live)::value, R = decltype(results)::value;
        for (int b = 0; b < ng; b++) {
            wait_vmcnt<0>();
            lds_barrier();  // group b's copies have landed, group b - 1's activations are read
            const uint8_t* buf = smem + C::WBYTES + (b & 1) * C::BUF;
            const uint8_t* al = buf + a * 256;
            Group<DT, C::AL> grp;
            if constexpr (C::LINES) {
                grp.read(smem + C::WWAVE * cp.wave, (uint32_t)(128 * a + 16 * ((a >> 1) & 7)), b, g);
            } else {
                grp.read(smem + C::WWAVE * cp.wave + a * C::WSLOT + (C::AL ? 0 : (wmis + (uint32_t)b * C::GROUP) & 15u), g);
            }
            if (b + 1 < ng) {
                cp.activations(b + 1, lds0 + C::WBYTES + ((b + 1) & 1) * C::BUF);
                wait_lgkm0();  // the wave's weight slot is read
                cp.weights(b + 1, lds0);
            }
            v16i acc[2][L];
            if constexpr (!C::K32) {
                v4i av[L];
#pragma unroll
                for (int i = 0; i < L; i++) av[i] = *(const v4i*)(al + i * 8192 + 16 * asw);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int ks = 0; ks < 8; ks++) {
                    v4i pH, pL, nx[L];
                    grp.planes(ks, g, pH, pL);
#pragma unroll
                    for (int i = 0; i < L; i++)
                        if (ks < 7) nx[i] = *(const v4i*)(al + i * 8192 + 16 * ((2 * ks + 2) ^ asw));
                    const v16i z = {};
#pragma unroll
                    for (int i = 0; i < L; i++) {
                        acc[0][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[i], pH, ks ? acc[0][i] : z, 0, 0, 0);
                        acc[1][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[i], pL, ks ? acc[1][i] : z, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < L; i++) av[i] = nx[i];
                }
                // The products at raised priority, the float step in what they
                // leave of the vector unit (2048 tokens 2 % faster than the other
                // way round, and that faster than neither).
                __builtin_amdgcn_s_setprio(0);
                const float* dl = (const float*)(buf + C::ABYTES + C::XBYTES);
                v8h bm;
                if constexpr (DT == DT_Q4_K) bm = grp.mins(g);
                v32f dd6;
#pragma unroll
                for (int i = 0; i < L; i++) {
                    if constexpr (DT == DT_Q4_K) {
                        // d*dx and dmin*dx of the tile as outer products (lanes
                        // g = 0 hold d, g = 1 dmin)
                        const v32f z = {};
                        const v32f dd = __builtin_amdgcn_mfma_f32_32x32x1f32(dl[32 * i + a], g ? grp.dmin : grp.d, z, 0, 0, 0);
                        // 64 hi + lo against 64 m and m
                        const v8h v = *(const v8h*)(buf + C::ABYTES + 32 * (32 * i + a) + 16 * g);
                        v16f Mm = {};
                        Mm = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, bm, Mm, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < R; r++) {
                            const int S = (acc[0][i][r] << 3) + acc[1][i][r];
                            tot[i][r] = __builtin_fmaf((float)S, dd[r], tot[i][r]);
                            off[i][r] = __builtin_fmaf(Mm[r], dd[16 + r], off[i][r]);
                        }
                    } else if constexpr (DT == DT_Q6_K) {
                        // d*dx of two tiles of pairs as one outer product (lanes
                        // g = 0 hold the even one's dx; 2048 tokens 793 -> 772 us)
                        if (i % 2 == 0) {
                            const v32f z = {};
                            dd6 = __builtin_amdgcn_mfma_f32_32x32x1f32(dl[32 * min(i + g, L - 1) + a], grp.d, z, 0, 0, 0);
                        }
#pragma unroll
                        for (int r = 0; r < R; r++) {
                            const int S = (acc[0][i][r] << 8) + acc[1][i][r];
                            tot[i][r] = __builtin_fmaf((float)S, dd6[16 * (i % 2) + r], tot[i][r]);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                // d*dx of two blocks (lanes g = 0 the even one's, g = 1 the odd
                // one's) as one outer product.
                const float* dl = (const float*)(buf + C::ABYTES);
                const int nk = min(8, A.nb - 8 * b);
#pragma unroll
                for (int ks = 0; ks < 8; ks += 2) {
                    if (ks < nk) {
                        const v4i w0 = grp.block(ks), w1 = grp.block(ks + 1);
                        const float dw = g ? grp.d[ks + 1] : grp.d[ks];
                        const v16i z = {};
                        const v32f zf = {};
#pragma unroll
                        for (int i = 0; i < L; i++) {
                            acc[0][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(*(const v4i*)(al + i * 8192 + 16 * ((2 * ks) ^ asw)), w0, z, 0, 0, 0);
                            acc[1][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(*(const v4i*)(al + i * 8192 + 16 * ((2 * ks + 2) ^ asw)), w1, z, 0, 0, 0);
                            const v32f dd = __builtin_amdgcn_mfma_f32_32x32x1f32(dl[8 * (32 * i + a) + ks + g], dw, zf, 0, 0, 0);
#pragma unroll
                            for (int r = 0; r < R; r++) tot[i][r] = __builtin_fmaf((float)acc[0][i][r], dd[r], tot[i][r]);
                            if (ks + 1 < nk) {
#pragma unroll
                                for (int r = 0; r < R; r++) tot[i][r] = __builtin_fmaf((float)acc[1][i][r], dd[16 + r], tot[i][r]);
                            }
                        }
                    }
                }
            }
        }
    };
    if (MT == 2 && tile.m <= 32) groups(std::integral_constant<int, 1>(), std::integral_constant<int, 16>());
    else if (MT == 1 && tile.m <= 16) groups(std::integral_constant<int, 1>(), std::integral_constant<int, 8>());
    else groups(std::integral_constant<int, MT>(), std::integral_constant<int, 16>());

    // Result i of a lane: weight row wn0 + a, pair 8 (i / 4) + 4 g + i % 4.
    const int n = wn0 + a;
    const int refused = flags[0];
    auto result = [&](int i, int r) { return DT == DT_Q4_K ? tot[i][r] - off[DT == DT_Q4_K ? i : 0][r] : tot[i][r]; };
    if constexpr (SW) {
        // gate and up meet in LDS: ex[matrix][pair][row of the tile]
        float* ex = (float*)smem;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                ex[((wave >> 1) * BM + 32 * i + 8 * (r >> 2) + 4 * g + (r & 3)) * 64 + 32 * (wave & 1) + a] = result(i, r);
        __syncthreads();
        if (refused) {
            for (int p = t >> 3; p < 2 * BM * 64; p += C::T / 8) {
                const int c = p & 63, m = (p >> 6) % BM, k = p / (64 * BM);
                const Mat& Mk = A.mat[k];
                if (n0 + c >= A.N || m >= tile.m) continue;
                const int64_t w = row0 + n0 + c;
                if (Mk.wref[w] == 0 && A.act.ok[rows[m]] != 0) continue;
                const float v = f32dot_g8<DT>(Mk.W + w * A.rb, A.x + (int64_t)rows[m] * A.K, A.K, true);
                if ((t & 7) == 0) ex[p] = v;
            }
            __syncthreads();
        }
        for (int p = t; p < 64 * tile.m; p += C::T) {
            const int c = p & 63, m = p >> 6;
            if (n0 + c < A.N) A.y[(int64_t)outs[m] * A.N + n0 + c] = silu_mul_vec(ex[p], ex[BM * 64 + p]);
        }
    } else {
        if (n < A.N && !(refused && M.wref[row0 + n] != 0)) {
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int m = 32 * i + 8 * (r >> 2) + 4 * g + (r & 3);
                    if (m >= tile.m || (refused && A.act.ok[rows[m]] == 0)) continue;
                    A.y[(int64_t)outs[m] * A.N + n] = result(i, r);
                }
        }
        if (!refused) return;
        for (int p = t >> 3; p < BN * tile.m; p += C::T / 8) {
            const int c = p % BN, m = p / BN;
            const int64_t w = row0 + n0 + c;
            if (n0 + c >= A.N || (M.wref[w] == 0 && A.act.ok[rows[m]] != 0)) continue;
            const float v = f32dot_g8<DT>(M.W + w * A.rb, A.x + (int64_t)rows[m] * A.K, A.K, true);
            if ((t & 7) == 0) A.y[(int64_t)outs[m] * A.N + n0 + c] = v;
        }
    }
}

// The same products with 16 weight rows a wave, on v_mfma_i32_16x16x64_i8 (Q8_0,
// whose blocks have a sum each, on 16x16x32), and 32
// pairs: half the unpacking a wave and twice the waves, where tiles of 32 rows a
// wave leave SIMDs without one. Lane l holds weight row a = l % 16 and of a k step
// of 64 the elements 16 g .. 16 g + 15, g = l / 16; of a 16 x 16 result the pairs
// 4 g .. 4 g + 3.
template <uint32_t DT>
struct ThinGroup;

template <>
struct ThinGroup<DT_Q4_K> {
    u32x4 q[4];
    uint64_t sc, m;  // sc: from the lane's sub-block of a pair on
    float d, dmin;
    static __device__ __forceinline__ uint32_t place(int c) { return (uint32_t)(((c & 8) << 8) | ((c & 7) << 4)); }
    __device__ __forceinline__ void read(const uint8_t* slot, uint32_t row, int b, int g) {
        const u32x4 h = *(const u32x4*)(slot + (row ^ place(9 * b)));
        d = f16_to_f32(h.x & 0xFFFFu);
        dmin = f16_to_f32(h.x >> 16);
        const Q4KScales s = q4k_scales(h.y, h.z, h.w);
        sc = s.sc >> (8 * (g >> 1));
        m = s.m;
        const int sh = 4 * (g >> 1);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint32_t p0 = place(9 * b + 1 + 2 * c), p1 = place(9 * b + 2 + 2 * c);
            const u32x4 v = *(const u32x4*)(slot + (row ^ ((g & 1) ? p1 : p0)));
            q[c] = u32x4{v.x >> sh & 0x0F0F0F0Fu, v.y >> sh & 0x0F0F0F0Fu, v.z >> sh & 0x0F0F0F0Fu, v.w >> sh & 0x0F0F0F0Fu};
        }
    }
    __device__ __forceinline__ void planes(int ks, int, v4i& H, v4i& L) const {
        const uint32_t s = byte_of(sc, 2 * ks);
        const short sh = (short)(s >> 3), sl = (short)(s & 7);
        const s16x2 shp = {sh, sh}, slp = {sl, sl};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            H[k] = (int)as_u32(as_s16x2(q[ks][k]) * shp);
            L[k] = (int)as_u32(as_s16x2(q[ks][k]) * slp);
        }
    }
};

template <>
struct ThinGroup<DT_Q6_K> {
    u32x4 ql[2], qh[2], sc;
    float d;
    __device__ __forceinline__ void read(const uint8_t* wr, int g) {
        const int sh = 2 * (g >> 1);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            ql[h] = lds_read16_a2(wr + 64 * h + 16 * g);
            const u32x4 v = lds_read16_a2(wr + 128 + 32 * h + 16 * (g & 1));
            qh[h] = u32x4{v.x >> sh, v.y >> sh, v.z >> sh, v.w >> sh};
        }
        sc = lds_read16_a2(wr + 192);
        d = f16_to_f32(lds_read2_a2(wr + 208));
    }
    // (as Group's, quarter 2 (ks % 2) + g / 2 of half ks / 2, scale 4 ks + g)
    __device__ __forceinline__ void planes(int ks, int g, v4i& H, v4i& L) const {
        const u32x4 lo = ql[ks >> 1], hi = qh[ks >> 1];
        const int s = (int)(int8_t)(uint8_t)(sc[ks] >> (8 * g));
        const short cu = (short)(128 - 32 * s);
        const s16x2 s2 = {(short)s, (short)s}, c2 = {cu, cu};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t q6 = ((lo[k] >> (4 * (ks & 1))) & 0x0F0F0F0Fu) | (((hi[k] >> (4 * (ks & 1))) & 0x03030303u) << 4);
            const uint32_t ue = as_u32(as_s16x2(__builtin_amdgcn_perm(0u, q6, 0x0C020C00u)) * s2 + c2);
            const uint32_t uo = as_u32(as_s16x2(__builtin_amdgcn_perm(0u, q6, 0x0C030C01u)) * s2 + c2);
            H[k] = (int)__builtin_amdgcn_perm(uo, ue, 0x07030501u);
            L[k] = (int)(__builtin_amdgcn_perm(uo, ue, 0x06020400u) ^ 0x80808080u);
        }
    }
};

// (AL: see Cfg) Blocks of 32 on v_mfma_i32_16x16x32_i8: of each block the lane
// holds the elements 8 g .. 8 g + 7.
template <bool AL>
struct ThinGroupQ8 {
    uint32_t w[8][3], sh;  // a block's 8 bytes in the dwords that hold them
    float d[2];            // scales of the blocks 4 i + g
    __device__ __forceinline__ void read(const uint8_t* wr, int g) {
        sh = AL ? 2 : ((uint32_t)(uintptr_t)wr + 2) & 2;
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
            const uint8_t* p = wr + Q80_BYTES * ks + 2 + 8 * g;
            const uint32_t* q = (const uint32_t*)(AL ? p - (ks & 1 ? 0 : 2) : __builtin_align_down(p, 4));
            w[ks][0] = q[0];
            w[ks][1] = q[1];
            w[ks][2] = AL && (ks & 1) ? 0 : q[2];
        }
#pragma unroll
        for (int i = 0; i < 2; i++) d[i] = f16_to_f32(lds_read2_a2(wr + Q80_BYTES * (4 * i + g)));
    }
    __device__ __forceinline__ long block(int ks) const {
        const uint32_t s = ks & 1 ? 2 - sh : sh;
        const uint32_t lo = AL && (ks & 1) ? w[ks][0] : __builtin_amdgcn_alignbyte(w[ks][1], w[ks][0], s);
        const uint32_t hi = AL && (ks & 1) ? w[ks][1] : __builtin_amdgcn_alignbyte(w[ks][2], w[ks][1], s);
        return (long)((uint64_t)hi << 32 | lo);
    }
};

template <uint32_t DT, bool AL = false>
__global__ __launch_bounds__(256, 4) void thin_kernel(Args A) {
    using C = Cfg<DT, 1, AL, 16>;
    constexpr int BM = 32, BN = 64;
    __shared__ __align__(16) uint8_t smem[C::SMEM];
    __shared__ int rows[BM], outs[64], flags[1];
    const int t = threadIdx.x, l = t & 63, wave = t >> 6;
    const int a = l & 15, g = l >> 4;
    Tile tile;
    if (!find_tile(A, (A.N + BN - 1) / BN, BM, tile)) return;
    const int n0 = tile.nt * BN, wn0 = n0 + 16 * wave;
    const int64_t row0 = (int64_t)tile.e * A.N;
    const Mat M = A.mat[0];
    Copies<DT, C> cp;
    cp.init_weights(A, M, row0, __builtin_amdgcn_readfirstlane(wn0));
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem);
    if (cp.wave == 0) lds_copy4(A.plan + plan_layout(A.pairs, A.experts).order + tile.f0 + min(t, tile.m - 1), outs);
    cp.weights(0, lds0);
    if (cp.wave == 0) wait_vmcnt<C::WDMA>();
    if (t == 0) flags[0] = 0;
    lds_barrier();
    if (t < BM) {
        const int pair = min(max(outs[t], 0), A.pairs - 1);
        outs[t] = pair;
        rows[t] = pair / A.rowdiv;
    }
    lds_barrier();
    cp.init_rows(A, rows);
    cp.activations(0, lds0 + C::WBYTES);
    {
        int f = 0;
        if (l < 16) f |= wn0 + l < A.N && M.wref[row0 + wn0 + l] != 0;
        if (t < tile.m) f |= A.act.ok[rows[t]] == 0;
        if (f) flags[0] = 1;
    }
    float tot[2][4] = {}, off[2][4] = {};
    const uint32_t wmis = DT == DT_Q4_K ? 0 : (uint32_t)(uintptr_t)(M.W + (row0 + min(wn0 + a, A.N - 1)) * A.rb);
    const int ng = C::K32 ? (A.nb + 7) / 8 : A.nb;
    for (int b = 0; b < ng; b++) {
        wait_vmcnt<0>();
        lds_barrier();
        const uint8_t* buf = smem + C::WBYTES + (b & 1) * C::BUF;
        std::conditional_t<C::K32, ThinGroupQ8<AL>, ThinGroup<DT>> grp;
        if constexpr (C::LINES) grp.read(smem + C::WWAVE * cp.wave, (uint32_t)(128 * a + 16 * ((a >> 1) & 7)), b, g);
        else grp.read(smem + C::WWAVE * cp.wave + a * C::WSLOT + (AL ? 0 : (wmis + (uint32_t)b * C::GROUP) & 15u), g);
        if (b + 1 < ng) {
            cp.activations(b + 1, lds0 + C::WBYTES + ((b + 1) & 1) * C::BUF);
            wait_lgkm0();
            cp.weights(b + 1, lds0);
        }
        if constexpr (C::K32) {
            // d*dx of four blocks at a time as outer products (lanes g hold
            // block 4 q + g's scales)
            const float* dl = (const float*)(buf + C::ABYTES);
            const int nk = min(8, A.nb - 8 * b);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (16 * i >= tile.m) break;
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const v16f zf = {};
                    const v16f dd = __builtin_amdgcn_mfma_f32_16x16x1f32(dl[8 * (16 * i + a) + 4 * q + g], grp.d[q], zf, 0, 0, 0);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int ks = 4 * q + k;
                        if (ks < nk) {
                            const long av = *(const long*)(buf + (16 * i + a) * 256 + 16 * ((2 * ks + (g >> 1)) ^ a) + 8 * (g & 1));
                            const v4i z = {};
                            const v4i S = __builtin_amdgcn_mfma_i32_16x16x32_i8(av, grp.block(ks), z, 0, 0, 0);
#pragma unroll
                            for (int r = 0; r < 4; r++) tot[i][r] = __builtin_fmaf((float)S[r], dd[4 * k + r], tot[i][r]);
                        }
                    }
                }
            }
        } else {
            // Q6_K: the second half of the pairs only where there are any (16
            // tokens of 60 experts and the like 3 to 5 % faster; Q4_K loses 2 % with
            // more pairs than that and gains 3 % below).
            auto products = [&](auto live) __attribute__((always_inline)) {
                constexpr int I = decltype(live)::value;
                v4i acc[2][I];
#pragma unroll
                for (int ks = 0; ks < 4; ks++) {
                    v4i pH, pL;
                    grp.planes(ks, g, pH, pL);
                    const v4i z = {};
#pragma unroll
                    for (int i = 0; i < I; i++) {
                        const v4i av = *(const v4i*)(buf + (16 * i + a) * 256 + 16 * ((4 * ks + g) ^ a));
                        acc[0][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av, pH, ks ? acc[0][i] : z, 0, 0, 0);
                        acc[1][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av, pL, ks ? acc[1][i] : z, 0, 0, 0);
                    }
                }
                const float* dl = (const float*)(buf + C::ABYTES + C::XBYTES);
#pragma unroll
                for (int i = 0; i < I; i++) {
                    const float4 dx = *(const float4*)(dl + 16 * i + 4 * g);
                    const float dv[4] = {dx.x, dx.y, dx.z, dx.w};
                    if constexpr (DT == DT_Q4_K) {
                        // (k 16 .. 31 of the mins' product are zeros: lanes g = 2, 3)
                        v8h bm = {};
                        if (g < 2) {
                            Group<DT_Q4_K> full;
                            full.s.m = grp.m;
                            bm = full.mins(g);
                        }
                        const v8h v = *(const v8h*)(buf + C::ABYTES + 32 * (16 * i + a) + 16 * (g & 1));
                        v4f Mm = {};
                        Mm = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, bm, Mm, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int S = (acc[0][i][r] << 3) + acc[1][i][r];
                            tot[i][r] = __builtin_fmaf((float)S, grp.d * dv[r], tot[i][r]);
                            off[i][r] = __builtin_fmaf(Mm[r], grp.dmin * dv[r], off[i][r]);
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int S = (acc[0][i][r] << 8) + acc[1][i][r];
                            tot[i][r] = __builtin_fmaf((float)S, grp.d * dv[r], tot[i][r]);
                        }
                    }
                }
            };
            if (DT == DT_Q6_K && tile.m <= 16) products(std::integral_constant<int, 1>());
            else products(std::integral_constant<int, 2>());
        }
    }
    const int n = wn0 + a, refused = flags[0];
    if (n < A.N && !(refused && M.wref[row0 + n] != 0)) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int m = 16 * i + 4 * g + r;
                if (m >= tile.m || (refused && A.act.ok[rows[m]] == 0)) continue;
                A.y[(int64_t)outs[m] * A.N + n] = DT == DT_Q4_K ? tot[i][r] - off[i][r] : tot[i][r];
            }
    }
    if (!refused) return;
    for (int p = t >> 3; p < BN * tile.m; p += C::T / 8) {
        const int c = p % BN, m = p / BN;
        const int64_t w = row0 + n0 + c;
        if (n0 + c >= A.N || (M.wref[w] == 0 && A.act.ok[rows[m]] != 0)) continue;
        const float v = f32dot_g8<DT>(M.W + w * A.rb, A.x + (int64_t)rows[m] * A.K, A.K, true);
        if ((t & 7) == 0) A.y[(int64_t)outs[m] * A.N + n0 + c] = v;
    }
}

// The most tiles of BM pairs that any choice of that many could need: whole
// ones, and one partly filled for each expert.
static int64_t max_tiles(const Args& A, int BM) {
    const int64_t some = A.pairs < A.experts ? A.pairs : A.experts;
    return (A.pairs + some * (BM - 1)) / BM;
}

// A workgroup for every tile of BM pairs and BN weight rows, in launches of 2^31
// threads (a grid has less than 2^32): 512 experts of a pair each reach the second
// one at 2^20 rows of 64 a tile.
static hipError_t launch_grid(void (*kernel)(Args), Args A, int BM, int BN, hipStream_t stream) {
    constexpr int64_t MOST = 1 << 23;
    const int64_t wgs = (max_tiles(A, BM) * ((A.N + BN - 1) / BN) + 7) / 8 * 8;
    for (A.wg0 = 0; A.wg0 < wgs; A.wg0 += MOST) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(wgs - A.wg0, MOST)), dim3(256), 0, stream, A);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <uint32_t DT, int MT, bool SW, bool AL = false>
static hipError_t launch(const Args& A, hipStream_t stream) {
    using C = Cfg<DT, MT, AL>;
    static_assert(C::T == 256, "threads of a workgroup");
    return launch_grid(tile_kernel<DT, C, SW>, A, C::BM, SW ? 64 : 128, stream);
}

template <uint32_t DT, bool AL = false>
static hipError_t launch_thin(const Args& A, hipStream_t stream) {
    return launch_grid(thin_kernel<DT, AL>, A, 32, 64, stream);
}
// Where they are taken, us of tiles of 32 / of 16 rows a wave (down, 8 experts,
// two a token): Q6_K 8192 -> 2048, 8 tokens 67.3 / 46.7, 64 69.3 / 50.6, 14336 -> 4096,
// 8 tokens 113 / 109, 128 tokens 175 / 152, 160 tokens (672 tiles of 32) 180 / 185; 16
// experts, 8192 -> 4096, 64 tokens (616) 115 / 123; short rows, 64 experts, 1024 -> 2048
// 44.2 / 41.8, 60 experts, 1536 51.5 / 48.3. Q4_K 8192 -> 2048, 64 tokens 46.1 / 41.7,
// 14336 -> 4096, 8 tokens 72.6 / 75.6. Q8_0 60 experts, four a token, 1408 -> 2048,
// 37 tokens 49.9 / 45.4, 181 57.9 / 56.3, 1440 -> 2048 54.3 / 45.6; two of 8, 14336 ->
// 4096, 64 tokens 150 / 137. Weights of two groups in LDS: 1 to 3 % slower. Gate and
// up this way: Q8_0 2048 x 1408 1 to 3 % faster, 4096 x 14336 and Q4_K 7 to 15 % slower.
static bool thin(uint32_t dt, const Args& A) {
    if (A.pairs >= 48 * (int64_t)A.experts) return false;
    const int64_t wgs = max_tiles(A, 32) * ((A.N + 127) / 128);
    return dt == DT_Q6_K ? wgs <= 512 || A.nb <= 8 : dt == DT_Q8_0 || wgs <= 192;
}

template <uint32_t DT, bool SW>
static hipError_t launch_dt(const Args& A, hipStream_t stream) {
    if constexpr (!SW)
        if (thin(DT, A)) {
            if constexpr (DT == DT_Q8_0)
                if (A.rb % 4 == 0 && (uintptr_t)A.mat[0].W % 4 == 0) return launch_thin<DT, true>(A, stream);
            return launch_thin<DT>(A, stream);
        }
    // 64 pairs a workgroup where the experts have as many on average, of Q6_K
    // where they have 48, and 96 from that on (us a call in tiles of 32 / 64 / 96:
    // down 2048 x 1024, 64 experts, 32 pairs each 57.8 / 60.6 / -, 48 70.7 / 69.6 /
    // -, 64 - / 79.1 / 84.1, 128 - / 123.4 / 124.9, 256 - / 212 / 200; 4096 x 14336,
    // 8 experts, 48 206 / 192 / -, 64 - / 207 / 219, 128 - / 341 / 267. Q4_K gate
    // and up 2048 x 1024, 48 71 / 75, 56 78 / 79; 4096 x 14336, 48 211 / 206.)
    const int64_t E = A.experts;
    if constexpr (DT == DT_Q6_K) {
        if (A.pairs >= 96 * E) return launch<DT, 3, SW>(A, stream);
        return A.pairs >= 48 * E ? launch<DT, 2, SW>(A, stream) : launch<DT, 1, SW>(A, stream);
    }
    if constexpr (DT == DT_Q8_0)
        if (A.rb % 4 == 0 && (uintptr_t)A.mat[0].W % 4 == 0 && (uintptr_t)A.mat[1].W % 4 == 0)
            return A.pairs >= 64 * E ? launch<DT, 2, SW, true>(A, stream) : launch<DT, 1, SW, true>(A, stream);
    return A.pairs >= 64 * E ? launch<DT, 2, SW>(A, stream) : launch<DT, 1, SW>(A, stream);
}

}  // namespace xp

// Few pairs each run their expert's matrices by themselves (gemv_kquant.hip), an
// expert that two of them share twice. Measured on MI355X, us a call with
// quantizing and sum, alone / in tiles: gate and up (Q4_K), 4096 x 14336, 8
// experts, 2 / 4 / 8 / 16 pairs 29 / 49 / 88 / 160 against 39 / 66 / 98 / 105;
// 2048 x 1024, 64 experts, 8 / 16 / 32 pairs 11.2 / 16.1 / 26.5 against 15.6 /
// 18.2 / 23.5; Q8_0 (experts_q8.hip) 4096 x 7168, 8 experts, 8 pairs 89 against
// 82, 2048 x 1408, 60 experts, 8 / 16 / 32 pairs 17.1 / 26.5 / 42 against 22.9 /
// 31.5 / 37.7.
// Of many more experts (Q4_K): 2048 x 768, 128 experts, 24 / 32 / 64 pairs 17.8 /
// 22.1 / 34.5 against 19.7 / 21.0 / 28.2; 4096 x 1536, 128 experts, 32 pairs 42
// against 49 (Q6_K 69 against 81), 256 experts, 48 / 56 / 64 pairs 68 / 73 / 85 against
// 81 / 85 / 97 (the bound of 48 leaves that gain; other sizes are not measured above
// it); Q8_0 2048 x 1408, 160 experts, 24 pairs 36.7 against 33.9. Q6_K below K = 4096:
// 2048 x 768, 128 experts, 24 / 32 / 64 pairs 27.2 / 33.0 / 56.3 against 26.7 / 31.1 / 44.6,
// 2048 x 1024, 64 experts, 8 / 16 / 32 pairs 14.8 / 24.6 / 40.1 against 21.1 / 23.6 / 31.9. The
// step at K = 4096 lies between the two widths measured on either side (Q4_K, 32
// pairs of 128 experts: 1024 x 1024 24.3 against 16.3, 3584 x 1536 42.6 against 48.8, 4096 x 1536
// 44.4 against 52.5).
static bool few_pairs_swiglu(const DevWeight& w, int pairs, int experts) {
    if (pairs <= (w.dt == DT_Q8_0 ? 4 : 8) || (pairs <= 16 && experts >= 2 * pairs)) return true;
    return w.dt != DT_Q8_0 && experts >= 4 * pairs && pairs <= (w.k >= 4096 ? 48 : 24);
}
// down with the sum in its launch, alone / in tiles: 14336 -> 4096, 8 experts, 2 /
// 4 / 8 / 12 / 16 pairs Q6_K 28 / 45 / 75 / 102 / 131 against 70 / 72 / 88 / 98 / 105, 12 /
// 16 pairs Q4_K 66 / 83 against 70 / 72, 8 pairs Q8_0 91 against 83; 1024 -> 2048
// Q4_K, 64 experts, 8 / 16 / 32 / 64 pairs 8.8 / 10.1 / 13.0 / 19.6 against 15.1 /
// 16.5 / 19.3 / 24.5; 60 experts, 32 / 48 pairs, 1536 -> 2048 Q6_K 27.2 / 35.6 against
// 26.7 / 32.0; 1408 -> 2048 Q8_0, 16 / 32 / 48 / 64 pairs 18.3 / 28.4 / 37.0 / 44.3 against
// 19.8 / 29.7 / 34.0 / 37.4. 128 experts, 72 / 96 / 128 pairs: 768 -> 2048 Q4_K 20.7 /
// 24.6 / 28.8 against 28.8 / 31.6 / 34.2, 1536 -> 4096 52 / 66 / 84 against 60 / 69 / 79;
// 32 / 40 / 64 / 96 pairs: 768 -> 2048 Q6_K 17.4 / 20.4 / 27.4 / 37.1 against 22.0 / 24.8 / 29.5 /
// 35.5, 40 / 64 pairs 1536 -> 4096 54.0 / 79.0 against 54.8 / 75.9, 48 / 64 / 96 pairs 1408 ->
// 2048 Q8_0 38.7 / 48.0 / 64.6 against 39.6 / 45.1 / 54.7.
static bool few_pairs_combine(uint32_t dt, int pairs, int experts) {
    if (pairs <= (dt == DT_Q8_0 ? 4 : 8)) return true;
    if (dt == DT_Q4_K) return pairs <= 128 && experts >= pairs;
    return pairs <= 32 ? 2 * experts >= 3 * pairs : pairs <= 64 && experts >= 2 * pairs;
}

// (rows of an expert are counted in 32 bits, with a tile's past the last one)
bool experts_ok(const DevWeight& w, int experts) {
    const bool k256 = w.dt == DT_Q4_K || w.dt == DT_Q6_K;
    return (k256 || w.dt == DT_Q8_0) && w.k % (k256 ? 256 : 32) == 0 && (uintptr_t)w.data % (w.dt == DT_Q4_K ? 16 : 2) == 0 &&
           w.n <= (1ll << 31) - 1 && w.n / experts <= (1ll << 30) && w.row_bytes < (1 << 26);
}

// The tiles' products of ws[0], or swiglu of those of ws[0] and ws[1].
static hipError_t launch_tiles(const DevWeight* const* ws, int nmat, int experts, const ActPtrs& a, void* parts, const float* x,
                               int64_t T, int top, bool per_pair, const int32_t* plan, float* y, hipStream_t stream) {
    const DevWeight& w = *ws[0];
    const int64_t rows = per_pair ? T * top : T;
    const hipError_t e = launch_experts_quantize(w.dt, x, rows, w.k, a, parts, stream);
    if (e != hipSuccess) return e;
    xp::Args A;
    A.parts = (const uint8_t*)parts;
    for (int i = 0; i < 2; i++) {
        const DevWeight& m = *ws[i < nmat ? i : 0];
        A.mat[i].W = m.data;
        A.mat[i].wref = m.wref;
    }
    A.y = y;
    A.plan = plan;
    A.rb = w.row_bytes;
    A.K = w.k;
    A.wbytes = w.n * w.row_bytes;
    A.N = (int)(w.n / experts);
    A.nb = (int)(w.k / (w.dt == DT_Q8_0 ? 32 : 256));
    A.experts = experts;
    A.pairs = (int)(T * top);
    A.rowdiv = per_pair ? 1 : top;
    A.act = a;
    A.x = x;
    if (nmat == 2) {
        if (w.dt == DT_Q4_K) return xp::launch_dt<DT_Q4_K, true>(A, stream);
        if (w.dt == DT_Q6_K) return xp::launch_dt<DT_Q6_K, true>(A, stream);
        return xp::launch_dt<DT_Q8_0, true>(A, stream);
    }
    if (w.dt == DT_Q4_K) return xp::launch_dt<DT_Q4_K, false>(A, stream);
    if (w.dt == DT_Q6_K) return xp::launch_dt<DT_Q6_K, false>(A, stream);
    return xp::launch_dt<DT_Q8_0, false>(A, stream);
}

hipError_t launch_experts_swiglu(const DevWeight& gate, const DevWeight& up, int experts, const ActPtrs& a, void* parts,
                                 const float* x, int64_t T, int top, const int32_t* plan, float* h, hipStream_t stream) {
    const int pairs = (int)(T * top);
    if (few_pairs_swiglu(gate, pairs, experts) && gemv_experts_swiglu_ok(gate, experts, pairs)) {
        const hipError_t e = launch_quantize_act(x, T, gate.k, 256, a, stream);
        if (e != hipSuccess) return e;
        return launch_gemv_experts_swiglu(gate, up, experts, a, x, T, top, plan + plan_layout(pairs, experts).expert, h, stream);
    }
    if (few_pairs_swiglu(gate, pairs, experts) && gemv_experts_q8_ok(gate, experts, 2, pairs)) {
        const hipError_t e = launch_quantize_act(x, T, gate.k, 32, a, stream);
        if (e != hipSuccess) return e;
        return launch_gemv_experts_q8_swiglu(gate, up, experts, a, x, T, top, plan + plan_layout(pairs, experts).expert, h, stream);
    }
    const DevWeight* ws[2] = {&gate, &up};
    return launch_tiles(ws, 2, experts, a, parts, x, T, top, false, plan, h, stream);
}

hipError_t launch_experts_combine(const DevWeight& w, int experts, const ActPtrs& a, void* parts, const float* h,
                                  const float* weights, int64_t T, int top, const int32_t* plan, float* product, float* y,
                                  hipStream_t stream) {
    const int pairs = (int)(T * top);
    const int32_t* expert = plan + plan_layout(pairs, experts).expert;
    if (few_pairs_combine(w.dt, pairs, experts) && gemv_experts_sum_ok(w, experts, T, top)) {
        const hipError_t e = launch_quantize_act(h, pairs, w.k, 256, a, stream);
        return e != hipSuccess ? e : launch_gemv_experts_sum(w, experts, a, h, weights, T, top, expert, y, stream);
    }
    if (few_pairs_combine(w.dt, pairs, experts) && gemv_experts_q8_ok(w, experts, top, T)) {
        const hipError_t e = launch_quantize_act(h, pairs, w.k, 32, a, stream);
        return e != hipSuccess ? e : launch_gemv_experts_q8_sum(w, experts, a, h, weights, T, top, expert, y, stream);
    }
    const DevWeight* ws[1] = {&w};
    const hipError_t e = launch_tiles(ws, 1, experts, a, parts, h, T, top, true, plan, product, stream);
    return e != hipSuccess ? e : launch_experts_sum(product, weights, expert, T, top, w.n / experts, y, stream);
}

}  // namespace mimg
