// The router of a mixture of experts, the plan of its choices, and the sum of
// a token's experts.
//
//   logit[t, e] = sum_k x[t, k] r[e, k]
//   ids[t]      = the `top` largest logits, falling, equal ones by the lowest
//                 index, NaN behind all others
//   weight[t,j] = exp(logit[ids_j] - m) / sum exp(logit - m), m the largest,
//                 the sum over all experts or over the chosen ones
//
// Which experts are chosen is a step function of the logits: with sums rounded
// to float32 a token whose experts are nearly alike would go to another one
// whenever the order of the sum changes (with the batch, say). Products of two
// float32 are exact in float64 and their sum is kept there, on
// v_mfma_f64_16x16x4: 2 T E K operations, where reading x and r takes about
// as long (2048 tokens, 128 experts, K = 4096).
#include "decoder_math.hpp"
#include "experts.hpp"
#include "mimg_device.hpp"
#include "mimg_kernels.hpp"

namespace mimg {
namespace xr {

typedef double v4d __attribute__((ext_vector_type(4)));

// 16 tokens x 16 experts a workgroup; its waves take every WAVES-th run of 16
// k, four MFMAs each: lane l holds row l % 16 and, of a run, the elements
// 4 (l / 16) .. + 3, so that a load is a float4 and MFMA i takes the i-th of
// each lane. The number of waves is the same for every call, so a logit's sum
// has one order.
constexpr int WAVES = 8;

__global__ __launch_bounds__(64 * WAVES) void logits_kernel(const float* __restrict__ x, const float* __restrict__ r,
                                                            int64_t T, int64_t K, int E, double* __restrict__ out) {
    __shared__ double part[WAVES][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, a = lane & 15, g = lane >> 4;
    const int64_t t0 = (int64_t)blockIdx.x * 16;
    const int e0 = (int)blockIdx.y * 16;
    const float* xr = x + min(t0 + a, T - 1) * K;
    const float* rr = r + (int64_t)min(e0 + a, E - 1) * K;
    v4d acc = {0.0, 0.0, 0.0, 0.0};
    const int64_t runs = (K + 15) / 16;
    constexpr int U = 4;  // runs whose loads are in flight together
    for (int64_t c0 = wave; c0 < runs; c0 += U * WAVES) {
        float4 xv[U], rv[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t k = min(16 * (c0 + (int64_t)u * WAVES) + 4 * g, K - 4);
            xv[u] = *(const float4*)(xr + k);
            rv[u] = *(const float4*)(rr + k);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            // (past the row's end: zeros, which add nothing but to a sum of a
            // zero; whole runs past it are left out)
            const int64_t c = c0 + (int64_t)u * WAVES;
            if (c >= runs) break;
            const bool in = 16 * c + 4 * g < K;
            const float xe[4] = {xv[u].x, xv[u].y, xv[u].z, xv[u].w}, re[4] = {rv[u].x, rv[u].y, rv[u].z, rv[u].w};
#pragma unroll
            for (int i = 0; i < 4; i++)
                acc = __builtin_amdgcn_mfma_f64_16x16x4f64(in ? (double)xe[i] : 0.0, in ? (double)re[i] : 0.0, acc, 0, 0, 0);
        }
    }
    // result lane l, register i: token 4 i + l / 16, expert l % 16
#pragma unroll
    for (int i = 0; i < 4; i++) part[wave][(4 * i + g) * 16 + a] = acc[i];
    __syncthreads();
    const int o = threadIdx.x;
    if (o >= 256) return;
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) s += part[w][o];
    const int64_t t = t0 + o / 16;
    const int e = e0 + o % 16;
    if (t < T && e < E) out[t * E + e] = s;
}

// A double as an integer of the same order; NaN below all numbers, `taken`
// below that.
constexpr int64_t KEY_TAKEN = INT64_MIN, KEY_NAN = INT64_MIN + 1;
__device__ __forceinline__ int64_t order_key(double v) {
    if (!(v == v)) return KEY_NAN;
    const int64_t b = __double_as_longlong(v + 0.0);
    return b < 0 ? b ^ INT64_MAX : b;
}
__device__ __forceinline__ int64_t wave_max_i64(int64_t v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const int64_t o = __shfl_xor((long long)v, m);
        v = o > v ? o : v;
    }
    return v;
}
__device__ __forceinline__ int wave_min_i32(int v) {
    v = min(v, __shfl_xor(v, 32));
    v = min(v, lane_xor<16>(v));
    v = min(v, lane_xor<8>(v));
    v = min(v, lane_xor<4>(v));
    v = min(v, lane_xor<2>(v));
    return min(v, lane_xor<1>(v));
}

// One token's choices by one wave: lane l holds the logits of the experts l,
// l + 64, ...
template <int PER>
__device__ __forceinline__ void select(const double* logits, int E, int top, int normalize, int32_t* ids, float* weights) {
    const int lane = threadIdx.x & 63;
    double v[PER];
    int64_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 64 * i;
        v[i] = e < E ? logits[e] : 0.0;
        key[i] = e < E ? order_key(v[i]) : KEY_TAKEN;
    }
    double m = 0.0, mine = 0.0;  // the largest; the value of choice `lane`
    int id = 0;
    for (int j = 0; j < top; j++) {
        int64_t b = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < PER; i++)
            if (key[i] > b) b = key[i], at = i;
        const int64_t best = wave_max_i64(b);
        const int e = wave_min_i32(b == best ? lane + 64 * at : INT32_MAX);
        double mv = 0.0;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 64 * i == e) key[i] = KEY_TAKEN, mv = v[i];
        const double bv = __shfl(mv, e & 63);
        if (j == 0) m = bv;
        if (lane == j) mine = bv, id = e;
    }
    double sum = 0.0;
    if (normalize) {
        sum = lane < top ? exp(mine - m) : 0.0;
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 64 * i < E) sum += exp(v[i] - m);
    }
    sum = wave_sum_f64(sum);
    if (lane < top) {
        ids[lane] = id;
        weights[lane] = (float)(exp(mine - m) / sum);
    }
}
__device__ __forceinline__ void select_any(const double* logits, int E, int top, int normalize, int32_t* ids, float* weights) {
    if (E <= 64) select<1>(logits, E, top, normalize, ids, weights);
    else if (E <= 128) select<2>(logits, E, top, normalize, ids, weights);
    else if (E <= 256) select<4>(logits, E, top, normalize, ids, weights);
    else select<8>(logits, E, top, normalize, ids, weights);
}

__global__ __launch_bounds__(256) void select_kernel(const double* __restrict__ logits, int64_t T, int E, int top,
                                                     int normalize, int32_t* __restrict__ ids, float* __restrict__ weights) {
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t < T) select_any(logits + t * E, E, top, normalize, ids + t * top, weights + t * top);
}

// The plan: workgroup e of E + 1 counts the pairs of the experts below e, which
// is first[e], and writes its own pairs in order behind it; the last one those
// without an expert. Every workgroup reads all ids (64 KB at 16384 pairs), and
// a wave takes a run of them as 64 at a time, so that a place is a count of
// set bits: no counter in memory, no order of arrival.
constexpr int PLAN_T = 1024;

__device__ __forceinline__ int expert_of(int id, int E) { return id >= 0 && id < E ? id : E; }

__global__ __launch_bounds__(PLAN_T) void plan_kernel(const int32_t* __restrict__ ids, int P, int E, int32_t* __restrict__ plan) {
    constexpr int W = PLAN_T / 64;
    __shared__ int below[W], equal[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = (int)blockIdx.x;
    const PlanLayout l = plan_layout(P, E);
    const int run = (P + PLAN_T - 1) / PLAN_T * 64;  // pairs of a wave, whole 64s
    const int p0 = min(wave * run, P), p1 = min(p0 + run, P);
    int nb = 0, ne = 0;
    for (int p = p0; p < p1; p += 64) {
        const int id = p + lane < p1 ? expert_of(ids[p + lane], E) : INT32_MAX;
        nb += __popcll(__ballot(id < e));
        ne += __popcll(__ballot(id == e));
    }
    if (lane == 0) below[wave] = nb, equal[wave] = ne;
    __syncthreads();
    int at = 0;
    for (int w = 0; w < W; w++) at += below[w];
    if (threadIdx.x == 0) plan[e] = at;  // e = E: the pairs that have one
    for (int w = 0; w < wave; w++) at += equal[w];
    if (ne == 0) return;
    int32_t *order = plan + l.order, *expert = plan + l.expert;
    for (int p = p0; p < p1; p += 64) {
        const int id = p + lane < p1 ? expert_of(ids[p + lane], E) : INT32_MAX;
        const uint64_t b = __ballot(id == e);
        if (id == e) {
            order[at + __popcll(b & ((1ull << lane) - 1))] = p + lane;
            expert[p + lane] = e < E ? e : -1;
        }
        at += __popcll(b);
    }
}

// y[t] = sum_j weights[t, j] part[t, j] over the pairs that have an expert, in
// the order of the choices: one fma each.
template <int V>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ part, const float* __restrict__ weights,
                                                      const int32_t* __restrict__ expert, int top, int64_t N,
                                                      float* __restrict__ y) {
    const int64_t t = blockIdx.x, n = ((int64_t)blockIdx.y * 256 + threadIdx.x) * V;
    if (n >= N) return;
    float s[V];
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = 0.f;
    for (int j = 0; j < top; j++) {
        const int64_t p = t * top + j;
        if (expert[p] < 0) continue;
        const float w = weights[p];
        float v[V];
        if constexpr (V == 4) {
            const float4 q = *(const float4*)(part + p * N + n);
            v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
        } else {
            v[0] = part[p * N + n];
        }
#pragma unroll
        for (int i = 0; i < V; i++) s[i] = __builtin_fmaf(w, v[i], s[i]);
    }
    if constexpr (V == 4) *(float4*)(y + t * N + n) = float4{s[0], s[1], s[2], s[3]};
    else y[t * N + n] = s[0];
}

}  // namespace xr

hipError_t launch_experts_plan(const int32_t* ids, int64_t T, int top, int experts, int32_t* plan, hipStream_t s) {
    hipLaunchKernelGGL(xr::plan_kernel, dim3((unsigned)(experts + 1)), dim3(xr::PLAN_T), 0, s, ids, (int)(T * top), experts, plan);
    return hipGetLastError();
}

hipError_t launch_experts_route(const float* x, const float* router, int64_t T, int64_t K, int experts, int top, int normalize,
                                int32_t* ids, float* weights, int32_t* plan, double* logits, hipStream_t s) {
    hipLaunchKernelGGL(xr::logits_kernel, dim3((unsigned)((T + 15) / 16), (unsigned)((experts + 15) / 16)),
                       dim3(64 * xr::WAVES), 0, s, x, router, T, K, experts, logits);
    hipLaunchKernelGGL(xr::select_kernel, dim3((unsigned)((T + 3) / 4)), dim3(256), 0, s, logits, T, experts, top, normalize,
                       ids, weights);
    if (plan) return launch_experts_plan(ids, T, top, experts, plan, s);
    return hipGetLastError();
}

hipError_t launch_experts_sum(const float* part, const float* weights, const int32_t* expert, int64_t T, int top, int64_t N,
                              float* y, hipStream_t s) {
    if (N % 4 == 0)
        hipLaunchKernelGGL(xr::combine_kernel<4>, dim3((unsigned)T, (unsigned)((N / 4 + 255) / 256)), dim3(256), 0, s, part,
                           weights, expert, top, N, y);
    else
        hipLaunchKernelGGL(xr::combine_kernel<1>, dim3((unsigned)T, (unsigned)((N + 255) / 256)), dim3(256), 0, s, part,
                           weights, expert, top, N, y);
    return hipGetLastError();
}

}  // namespace mimg
