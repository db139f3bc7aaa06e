// Q8_0 experts where a call has few (token, choice) pairs: gate, up and swiglu of
// a pair, or the weighted sum of a token's down products, in one launch.
//
// Numerics: per (weight row, activation row) and block of 32 the exact int32 S =
// sum q y, then serially in block order tot = fma(f32(S), d*dx, tot): bit for bit
// the tiles' product (experts.hip), whatever the call holds.
//
// A workgroup takes four rows of each of its sets of weights (gate and up of a
// pair's expert, or the matrices of a token's experts). A wave reads 32 blocks
// of a row at a time, 1088 consecutive bytes, a lane 16 quants of a block
// (2-byte aligned: the five dwords that hold them), the four rows' loads in
// flight together with the activations they share. The block sums and scale
// products go to a table in LDS, over which one lane a row runs the chain.
// Bound: HBM for large experts, the latency of that chain of steps for small
// ones. In tiles, whose rows of 32 pairs are mostly empty here, a workgroup
// reads its rows group after group. One token, us a call alone / in tiles: gate
// and up 2048 x 1408 of four choices 11.0 / 21.3, 4096 x 7168 of two 30.8 / 40.2;
// down 2048 x 1408 9.7 / 15.6, 4096 x 14336 33 / 70.
#include "decoder_math.hpp"
#include "experts.hpp"
#include "f32path.hpp"
#include "mimg_device.hpp"
#include "mimg_kernels.hpp"

namespace mimg {
namespace xq {

constexpr int ROWS = 4;  // of a set

struct Args {
    const uint8_t *W[2], *wref[2];  // the matrices of all experts (two: gate and up)
    int64_t rb, K;
    int N, nb, top, experts;        // nb: blocks of a row
    const int8_t* q;
    const float* d32;
    const int32_t* ok;
    const float* x;
    const int32_t* expert;          // of each pair
    const float* weights;           // of each pair (the sum)
    float* y;                       // h [pairs][N], or y [T][N]
};

template <bool SW>
__global__ __launch_bounds__(256) void gemv_kernel(Args A) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int chosen[EXPERTS_MAX_TOP];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int sets = SW ? 2 : A.top, R = ROWS * sets, row0 = (int)blockIdx.x * ROWS;
    // the first pair (SW: the only one) and the activation row of set 0
    const int64_t p0 = SW ? (int64_t)blockIdx.y : (int64_t)blockIdx.y * A.top, act0 = SW ? p0 / A.top : p0;
    uint2* table = (uint2*)smem;                                // [R][nb]: S, d*dx
    int* refused = (int*)(smem + (size_t)R * A.nb * 8);         // [R]
    float* yr = (float*)(refused + R);                          // [R]
    if (t < sets) chosen[t] = plan_expert(A.expert, SW ? p0 : p0 + t, A.experts);
    __syncthreads();
    if (SW && chosen[0] < 0) return;
    auto matrix_row = [&](int s, int r) {  // row r of set s, in the matrices of all experts
        return (int64_t)max(chosen[s], 0) * A.N + min(row0 + r, A.N - 1);
    };
    auto act_row = [&](int s) { return SW ? act0 : act0 + s; };
    int flag = 0;
    if (t < R) flag = A.wref[SW ? t / ROWS : 0][matrix_row(t / ROWS, t % ROWS)] != 0 || A.ok[act_row(t / ROWS)] == 0;
    const int runs = (A.nb + 31) / 32;
    for (int i = wave; i < sets * runs; i += 4) {
        const int s = i / runs, b = 32 * (i - s * runs) + (lane >> 1), half = lane & 1, bc = min(b, A.nb - 1);
        const int64_t act = act_row(s);
        const u32x4 y = *(const u32x4*)(A.q + act * A.K + 32 * bc + 16 * half);
        const float dx = A.d32[act * (A.K / 32) + bc];
        const uint8_t* W = A.W[SW ? s : 0] + (int64_t)bc * Q80_BYTES;
        u32x4a4 v[ROWS];
        uint32_t v4[ROWS], d[ROWS], sh[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            const uint8_t* p = W + matrix_row(s, r) * A.rb;
            const uint8_t* w = p + 2 + 16 * half;
            const uint32_t* a = (const uint32_t*)__builtin_align_down(w, 4);
            sh[r] = (uint32_t)(uintptr_t)w & 3;
            v[r] = *(const u32x4a4*)a;
            v4[r] = a[4];
            d[r] = load_u16(p);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            int S = sdot4(__builtin_amdgcn_alignbyte(v[r].y, v[r].x, sh[r]), y.x, 0);
            S = sdot4(__builtin_amdgcn_alignbyte(v[r].z, v[r].y, sh[r]), y.y, S);
            S = sdot4(__builtin_amdgcn_alignbyte(v[r].w, v[r].z, sh[r]), y.z, S);
            S = sdot4(__builtin_amdgcn_alignbyte(v4[r], v[r].w, sh[r]), y.w, S);
            S += lane_xor<1>(S);
            if (half == 0 && b < A.nb) table[(s * ROWS + r) * A.nb + b] = make_uint2((uint32_t)S, __float_as_uint(f16_to_f32(d[r]) * dx));
        }
    }
    if (t < R) refused[t] = flag;
    __syncthreads();
    if (t < R && !flag) {
        const uint2* row = table + t * A.nb;
        float tot = 0.f;
        int b = 0;
        for (; b + 8 <= A.nb; b += 8) {  // (the reads of eight steps ahead of their chain)
            uint2 v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = row[b + k];
#pragma unroll
            for (int k = 0; k < 8; k++) tot = __builtin_fmaf((float)(int)v[k].x, __uint_as_float(v[k].y), tot);
        }
        for (; b < A.nb; b++) tot = __builtin_fmaf((float)(int)row[b].x, __uint_as_float(row[b].y), tot);
        yr[t] = tot;
    }
    for (int r = t >> 3; r < R; r += 32) {  // refused rows: the float32 path, eight lanes each
        if (!refused[r]) continue;
        const int s = r / ROWS;
        const float v = f32dot_g8<DT_Q8_0>(A.W[SW ? s : 0] + matrix_row(s, r % ROWS) * A.rb, A.x + act_row(s) * A.K, A.K, true);
        if ((t & 7) == 0) yr[r] = v;
    }
    __syncthreads();
    if (t >= ROWS || row0 + t >= A.N) return;
    float out = 0.f;
    if constexpr (SW) {
        out = silu_mul_vec(yr[t], yr[ROWS + t]);
    } else {
        for (int j = 0; j < sets; j++)
            if (chosen[j] >= 0) out = __builtin_fmaf(A.weights[p0 + j], yr[j * ROWS + t], out);
    }
    A.y[(int64_t)blockIdx.y * A.N + row0 + t] = out;
}

static size_t lds_bytes(int sets, int64_t nb) { return (size_t)ROWS * sets * (nb * 8 + 8); }

static Args args(const DevWeight& w, int experts, const ActPtrs& a, const float* x, int top, const int32_t* expert) {
    Args A{};
    A.W[0] = A.W[1] = w.data;
    A.wref[0] = A.wref[1] = w.wref;
    A.rb = w.row_bytes;
    A.K = w.k;
    A.N = (int)(w.n / experts);
    A.nb = (int)(w.k / 32);
    A.top = top;
    A.experts = experts;
    A.q = a.q;
    A.d32 = a.d32;
    A.ok = a.ok;
    A.x = x;
    A.expert = expert;
    return A;
}

}  // namespace xq

// (the table within 60 KB of LDS)
bool gemv_experts_q8_ok(const DevWeight& w, int experts, int sets, int64_t groups) {
    static_assert(xq::ROWS == 4, "rows of a workgroup");
    return w.dt == DT_Q8_0 && xq::lds_bytes(sets, w.k / 32) <= 60 * 1024 && experts_gemv_grid(w.n / experts, groups);
}

hipError_t launch_gemv_experts_q8_swiglu(const DevWeight& gate, const DevWeight& up, int experts, const ActPtrs& a, const float* x,
                                         int64_t T, int top, const int32_t* expert, float* h, hipStream_t stream) {
    xq::Args A = xq::args(gate, experts, a, x, top, expert);
    A.W[1] = up.data;
    A.wref[1] = up.wref;
    A.y = h;
    hipLaunchKernelGGL(xq::gemv_kernel<true>, dim3((unsigned)((A.N + xq::ROWS - 1) / xq::ROWS), (unsigned)(T * top)), dim3(256),
                       xq::lds_bytes(2, A.nb), stream, A);
    return hipGetLastError();
}

hipError_t launch_gemv_experts_q8_sum(const DevWeight& w, int experts, const ActPtrs& a, const float* x, const float* weights,
                                      int64_t T, int top, const int32_t* expert, float* y, hipStream_t stream) {
    xq::Args A = xq::args(w, experts, a, x, top, expert);
    A.weights = weights;
    A.y = y;
    hipLaunchKernelGGL(xq::gemv_kernel<false>, dim3((unsigned)((A.N + xq::ROWS - 1) / xq::ROWS), (unsigned)T), dim3(256),
                       xq::lds_bytes(top, A.nb), stream, A);
    return hipGetLastError();
}

}  // namespace mimg
