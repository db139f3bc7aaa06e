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
// v_mfma_f64_16x16x4: 2 T E K operations (2048 tokens of 128 experts, K = 4096: 32
// us at the 66 TFLOP/s that a float64 product of 8192^3 reaches, x and r are read
// in 5; the logits take 42 to 43, choices 5 and plan 5). There the matrix cores are
// at work 59 % of the cycles and vector instructions 14 %: two waves a SIMD, waiting
// for loads a quarter of their time. Few tokens are
// bound by launches (181 of 60 experts, K = 2048: 5.1, 3.5 and 3.0 us).
#include "decoder_math.hpp"
#include "experts.hpp"
#include "mimg_device.hpp"
#include "mimg_kernels.hpp"
#include "qa_chunk.hpp"

namespace mimg {
namespace xr {

typedef double v4d __attribute__((ext_vector_type(4)));

// A workgroup takes 16 MT tokens x 16 MT experts and every Z-th part of K; its
// waves take every WAVES-th run of 16 k of that part, four MFMAs each and tile:
// lane l holds row l % 16 and, of a run, the elements 4 (l / 16) .. + 3, so that
// a load is a float4 and MFMA i takes the i-th of each lane. The waves' sums
// meet in LDS, those of the Z parts in the next kernel.
constexpr int WAVES = 8;

// WHOLE: K is a multiple of 16 (no lane past a row's end in the last run).
template <int MT, bool WHOLE>
__global__ __launch_bounds__(64 * WAVES) void logits_kernel(const float* __restrict__ x, const float* __restrict__ r,
                                                            int64_t T, int64_t K, int E, double* __restrict__ out) {
    constexpr int N = 16 * MT, U = 4 / MT;  // runs whose loads are in flight together
    __shared__ double part[WAVES][N * N];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, a = lane & 15, g = lane >> 4;
    const int64_t t0 = (int64_t)blockIdx.x * N;
    const int e0 = (int)blockIdx.y * N, Z = (int)gridDim.z, z = (int)blockIdx.z;
    const float *xr[MT], *rr[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        xr[i] = x + min(t0 + 16 * i + a, T - 1) * K;
        rr[i] = r + (int64_t)min(e0 + 16 * i + a, E - 1) * K;
    }
    v4d acc[MT][MT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = v4d{0.0, 0.0, 0.0, 0.0};
    const int64_t all = (K + 15) / 16, part_runs = (all + Z - 1) / Z, runs = min(all, (z + 1) * part_runs);
    float4 xv[2][U][MT], rv[2][U][MT];
    auto load = [&](int64_t c0, int s) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t k = min(16 * (c0 + (int64_t)u * WAVES) + 4 * g, K - 4);
#pragma unroll
            for (int i = 0; i < MT; i++) {
                xv[s][u][i] = *(const float4*)(xr[i] + k);
                rv[s][u][i] = *(const float4*)(rr[i] + k);
            }
        }
    };
    // (whole runs past the end are left out, what is past it inside the last
    // run counts as zeros)
    auto multiply = [&](int64_t c0, int s) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t c = c0 + (int64_t)u * WAVES;
            if (c >= runs) break;
            const bool in = WHOLE || 16 * c + 4 * g < K;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                double xd[MT], rd[MT];
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const float xe[4] = {xv[s][u][i].x, xv[s][u][i].y, xv[s][u][i].z, xv[s][u][i].w};
                    const float re[4] = {rv[s][u][i].x, rv[s][u][i].y, rv[s][u][i].z, rv[s][u][i].w};
                    xd[i] = in ? (double)xe[q] : 0.0;
                    rd[i] = in ? (double)re[q] : 0.0;
                }
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int j = 0; j < MT; j++) acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(xd[i], rd[j], acc[i][j], 0, 0, 0);
            }
        }
    };
    constexpr int64_t STEP = U * WAVES;
    int64_t c0 = z * part_runs + wave;
    if constexpr (MT == 1) {  // (a wave has few runs)
        for (; c0 < runs; c0 += STEP) {
            load(c0, 0);
            multiply(c0, 0);
        }
    } else {  // the next runs' loads in flight under this one's products: 52 -> 46 us
        load(c0, 0);
        for (; c0 < runs; c0 += 2 * STEP) {
            load(c0 + STEP, 1);
            multiply(c0, 0);
            load(c0 + 2 * STEP, 0);
            multiply(c0 + STEP, 1);
        }
    }
    // result lane l, register q of a tile: token 4 q + l / 16, expert l % 16
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) part[wave][(16 * i + 4 * q + g) * N + 16 * j + a] = acc[i][j][q];
    __syncthreads();
    for (int o = threadIdx.x; o < N * N; o += 64 * WAVES) {
        double s = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) s += part[w][o];
        const int64_t t = t0 + o / N;
        const int e = e0 + o % N;
        if (t < T && e < E) out[((int64_t)z * T + t) * E + e] = s;
    }
}

// A double as an integer of the same order; NaN below all numbers, `taken`
// below that.
constexpr int64_t KEY_TAKEN = INT64_MIN, KEY_NAN = INT64_MIN + 1;
__device__ __forceinline__ int64_t order_key(double v) {
    if (!(v == v)) return KEY_NAN;
    const int64_t b = __double_as_longlong(v + 0.0);
    return b < 0 ? b ^ INT64_MAX : b;
}
// The wave's largest value, in every lane: within rows of 16 lanes (shifts by 1,
// 2, 4, 8), each row's last lane into the rows behind it, the last lane to all.
__device__ __forceinline__ int wave_max_last(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xF, 0xF, false));  // row_shr:1
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));  // row_bcast:15 into rows 1 and 3
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xC, 0xF, false));  // row_bcast:31 into rows 2 and 3
    return __builtin_amdgcn_readlane(v, 63);
}

// One token's choices by one wave (a choice by ballots and maxima of 32 bits: eight
// of 64 experts 2.9 us less than by maxima of 64 bits through all lanes): lane l holds the logits of the experts l,
// l + 64, ..., each the sum of Z parts `stride` apart. Lane j < top returns
// choice j.
template <int PER>
__device__ __forceinline__ int select(const double* logits, int Z, int64_t stride, int E, int top, int normalize, int32_t* ids,
                                      float* weights) {
    const int lane = threadIdx.x & 63;
    double v[PER];
    int64_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = 0.0;
    constexpr int ZU = PER <= 2 ? 8 : 2;  // parts whose loads are in flight together
    for (int z = 0; z < Z; z += ZU) {
        double p[ZU][PER];
#pragma unroll
        for (int u = 0; u < ZU; u++)
#pragma unroll
            for (int i = 0; i < PER; i++) p[u][i] = logits[min(z + u, Z - 1) * stride + min(lane + 64 * i, E - 1)];
#pragma unroll
        for (int u = 0; u < ZU; u++)
#pragma unroll
            for (int i = 0; i < PER; i++) v[i] += z + u < Z ? p[u][i] : 0.0;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) key[i] = lane + 64 * i < E ? order_key(v[i]) : KEY_TAKEN;
    double m = 0.0, mine = 0.0;  // the largest; the value of choice `lane`
    int id = 0;
    for (int j = 0; j < top; j++) {
        int64_t b = key[0];
        int at = 0;
        double bv = v[0];
#pragma unroll
        for (int i = 1; i < PER; i++)
            if (key[i] > b) b = key[i], at = i, bv = v[i];
        // the keys' upper halves, and their lower ones where lanes share it (as
        // signed numbers of the same order)
        const int hi = (int)(b >> 32), lo = (int)((uint32_t)b ^ 0x80000000u), best = wave_max_last(hi);
        uint64_t in = __ballot(hi == best);
        if (in & (in - 1)) {
            const int bl = wave_max_last(hi == best ? lo : INT32_MIN);
            in = __ballot(hi == best && lo == bl);
        }
        // of equal ones the lowest index
        uint64_t first = in;
        int slot = 0;
        if constexpr (PER > 1) {
#pragma unroll
            for (int i = PER - 1; i >= 0; i--) {
                const uint64_t here = __ballot(at == i) & in;
                if (here) first = here, slot = i;
            }
        }
        const int l = __ffsll((unsigned long long)first) - 1;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane == l && slot == i) key[i] = KEY_TAKEN;
        const int64_t bits = __double_as_longlong(bv);
        const int bh = __builtin_amdgcn_readlane((int)(bits >> 32), l), bl = __builtin_amdgcn_readlane((int)bits, l);
        bv = __longlong_as_double((int64_t)((uint64_t)(uint32_t)bh << 32 | (uint32_t)bl));
        if (j == 0) m = bv;
        if (lane == j) mine = bv, id = 64 * slot + l;
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
    return id;
}
__device__ __forceinline__ int select_any(const double* logits, int Z, int64_t stride, int E, int top, int normalize, int32_t* ids,
                                          float* weights) {
    if (E <= 64) return select<1>(logits, Z, stride, E, top, normalize, ids, weights);
    if (E <= 128) return select<2>(logits, Z, stride, E, top, normalize, ids, weights);
    if (E <= 256) return select<4>(logits, Z, stride, E, top, normalize, ids, weights);
    return select<8>(logits, Z, stride, E, top, normalize, ids, weights);
}

__global__ __launch_bounds__(256) void select_kernel(const double* __restrict__ logits, int Z, int64_t T, int E, int top,
                                                     int normalize, int32_t* __restrict__ ids, float* __restrict__ weights) {
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t < T) select_any(logits + t * E, Z, T * E, E, top, normalize, ids + t * top, weights + t * top);
}

// The plan of the choices in LDS (P <= SMALL_PAIRS), by a workgroup of 16 waves.
constexpr int SMALL_PAIRS = 512;
template <int N>  // P <= 64 N
__device__ __forceinline__ void plan_held(const int* chosen, int P, int E, int32_t* __restrict__ plan) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const PlanLayout l = plan_layout(P, E);
    for (int p = threadIdx.x; p < P; p += 1024) plan[l.expert + p] = chosen[p];
    int id[N];
#pragma unroll
    for (int i = 0; i < N; i++) id[i] = 64 * i + lane < P ? chosen[64 * i + lane] : INT32_MAX;
    for (int e = wave; e <= E; e += 16) {
        int at = 0;
#pragma unroll
        for (int i = 0; i < N; i++) at += 64 * i < P ? __popcll(__ballot(id[i] < e)) : 0;
        if (lane == 0) plan[e] = at;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (64 * i >= P) break;
            const uint64_t b = __ballot(id[i] == e);
            if (id[i] == e) plan[l.order + at + __popcll(b & ((1ull << lane) - 1))] = 64 * i + lane;
            at += __popcll(b);
        }
    }
}

__device__ __forceinline__ void plan_small(const int* chosen, int P, int E, int32_t* __restrict__ plan) {
    if (P <= 64) return plan_held<1>(chosen, P, E, plan);
    plan_held<SMALL_PAIRS / 64>(chosen, P, E, plan);
}

// One to four tokens and a small router: logits, choices and plan in one launch
// of one workgroup, a wave a part of an expert's row at a time, all tokens
// against it. One compute unit reads and multiplies slower than many, so only
// up to 2^15 products (us in a graph, one launch / two: K = 4096, 8 experts, 1
// token 5.9 / 6.6, called one by one 3 less, 2 tokens 7.4 / 6.9, 4 tokens 9.7 / 6.9;
// 1 token, 16 experts 8.1 / 6.7; K = 1024, 32 experts 6.8 / 6.5; K = 2048, 64 experts
// 14.5 / 7.4).
constexpr int ONE_T = 4, ONE_PARTS = 512;
constexpr int64_t ONE_PRODUCTS = 1 << 15;

__global__ __launch_bounds__(1024) void route_one_kernel(const float* __restrict__ x, const float* __restrict__ r, int T, int64_t K,
                                                         int E, int parts, int top, int normalize, int32_t* __restrict__ ids,
                                                         float* __restrict__ weights, int32_t* __restrict__ plan) {
    __shared__ double sums[ONE_T * ONE_PARTS];  // [part][token][expert]
    __shared__ int chosen[ONE_T * EXPERTS_MAX_TOP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, P = T * top;
    const int64_t run = ((K + parts - 1) / parts + 3) / 4 * 4;
    for (int j = wave; j < E * parts; j += 16) {
        const int e = j / parts, p = j - e * parts;
        const int64_t k0 = p * run, k1 = min(k0 + run, K);
        const float* rr = r + (int64_t)e * K;
        double acc[ONE_T] = {0.0, 0.0, 0.0, 0.0};
        constexpr int U = 4;  // float4 of a lane in flight together, and of each token
        for (int64_t k = k0 + 4 * lane; k - 4 * lane < k1; k += 256 * U) {
            float4 rv[U];
#pragma unroll
            for (int u = 0; u < U; u++) rv[u] = *(const float4*)(rr + min(k + 256 * u, K - 4));
#pragma unroll
            for (int t = 0; t < ONE_T; t++) {
                if (t >= T) break;
                float4 xv[U];
#pragma unroll
                for (int u = 0; u < U; u++) xv[u] = *(const float4*)(x + t * K + min(k + 256 * u, K - 4));
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (k + 256 * u >= k1) continue;
                    acc[t] = __builtin_fma((double)rv[u].x, (double)xv[u].x, acc[t]);
                    acc[t] = __builtin_fma((double)rv[u].y, (double)xv[u].y, acc[t]);
                    acc[t] = __builtin_fma((double)rv[u].z, (double)xv[u].z, acc[t]);
                    acc[t] = __builtin_fma((double)rv[u].w, (double)xv[u].w, acc[t]);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < ONE_T; t++) {
            if (t >= T) break;
            const double s = wave_sum_f64(acc[t]);
            if (lane == 0) sums[(p * T + t) * E + e] = s;
        }
    }
    __syncthreads();
    for (int t = wave; t < T; t += 16) {
        const int id = select_any(sums + t * E, parts, (int64_t)T * E, E, top, normalize, ids + t * top, weights + t * top);
        if (lane < top) chosen[t * top + lane] = id;
    }
    if (plan == nullptr) return;
    __syncthreads();
    plan_small(chosen, P, E, plan);
}

// Few tokens and a small router: choices and plan by one workgroup, a wave a token
// (us in a graph, so / in a launch each: K = 4096, 8 experts, 8 tokens 7.3 / 9.0, 16
// tokens 8.5 / 9.2, with two tokens a wave 32 tokens 11.4 / 9.4; 64 experts, 8 tokens
// 8.9 / 9.8, 16 tokens 11.6 / 10.1; K = 2048, 128 experts, 8 tokens 12.2 / 10.8).
constexpr int SMALL_T = 16, SMALL_LOGITS = 512;

__global__ __launch_bounds__(1024) void select_plan_kernel(const double* __restrict__ logits, int Z, int T, int E, int top,
                                                           int normalize, int32_t* __restrict__ ids, float* __restrict__ weights,
                                                           int32_t* __restrict__ plan) {
    __shared__ int chosen[SMALL_PAIRS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, P = T * top;
    for (int t = wave; t < T; t += 16) {
        const int id = select_any(logits + (int64_t)t * E, Z, (int64_t)T * E, E, top, normalize, ids + t * top, weights + t * top);
        if (lane < top) chosen[t * top + lane] = id;
    }
    __syncthreads();
    plan_small(chosen, P, E, plan);
}

// The plan: workgroup e of E + 1 counts the pairs of the experts below e, which
// is first[e], and writes its own pairs in order behind it; the last one those
// without an expert. Every workgroup reads all ids (64 KB at 16384 pairs), and
// a wave takes a run of them as 64 at a time, so that a place is a count of
// set bits: no counter in memory, no order of arrival.
constexpr int PLAN_T = 1024;

__device__ __forceinline__ int expert_of(int id, int E) { return id >= 0 && id < E ? id : E; }

// HOLD: the ids of a wave's run stay in registers between the two passes
// (P <= HOLD * PLAN_T), 0: they are read again, eight in flight together. (Read
// one by one 16384 pairs of 128 experts took 8.9 us, so 4.8.)
template <int HOLD>
__global__ __launch_bounds__(PLAN_T) void plan_kernel(const int32_t* __restrict__ ids, int P, int E, int32_t* __restrict__ plan) {
    constexpr int W = PLAN_T / 64, U = HOLD ? HOLD : 8;
    __shared__ int below[W], equal[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = (int)blockIdx.x;
    const PlanLayout l = plan_layout(P, E);
    const int n = (P + PLAN_T - 1) / PLAN_T;  // 64s of pairs of a wave
    const int p0 = min(wave * n * 64, P), p1 = min(p0 + n * 64, P);
    int id[U] = {};
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; u++) id[u] = ids[min(p0 + 64 * (i0 + u) + lane, P - 1)];
#pragma unroll
        for (int u = 0; u < U; u++) id[u] = p0 + 64 * (i0 + u) + lane < p1 ? expert_of(id[u], E) : INT32_MAX;
    };
    int nb = 0, ne = 0;
    for (int i = 0; i < n; i += U) {
        load(i);
#pragma unroll
        for (int u = 0; u < U; u++) {
            nb += __popcll(__ballot(id[u] < e));
            ne += __popcll(__ballot(id[u] == e));
        }
    }
    if (lane == 0) below[wave] = nb, equal[wave] = ne;
    __syncthreads();
    int at = 0;
#pragma unroll
    for (int w = 0; w < W; w++) at += below[w];
    if (threadIdx.x == 0) plan[e] = at;  // e = E: the pairs that have one
    for (int p = e * PLAN_T + (int)threadIdx.x; p < P; p += (E + 1) * PLAN_T) {  // pairs' experts: a share of them all
        const int x = expert_of(ids[p], E);
        plan[l.expert + p] = x < E ? x : -1;
    }
    for (int w = 0; w < wave; w++) at += equal[w];
    if (ne == 0) return;
    for (int i = 0; i < n; i += U) {
        if constexpr (HOLD == 0) load(i);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t b = __ballot(id[u] == e);
            if (id[u] == e) plan[l.order + at + __popcll(b & ((1ull << lane) - 1))] = p0 + 64 * (i + u) + lane;
            at += __popcll(b);
        }
    }
}

// The quantizer of the tiles' activations: a row by one workgroup, CPW chunks
// of 256 a wave with their loads in flight together, only what the tiles read
// (q, scales, Q4_K's sums in the form of its f16 operand, ok): 4096 rows of
// 14336 take 74 to 78 us (3.9 TB/s; Q4_K 85), 84 with every array of the other
// products where this took 74.
template <int BLOCK, int OUT, int CPW>
__global__ __launch_bounds__(1024) void quantize_kernel(const float* __restrict__ x, int64_t K, ActPtrs a, _Float16* parts) {
    const int64_t row = blockIdx.x, nch = (K + 255) / 256;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, nwaves = blockDim.x >> 6;
    const float* xr = x + row * K;
    bool bad = false;
    for (int64_t c0 = wave; c0 < nch; c0 += (int64_t)nwaves * CPW) {
        float4 v[CPW];
#pragma unroll
        for (int i = 0; i < CPW; i++) v[i] = *(const float4*)(xr + min(min(c0 + nwaves * i, nch - 1) * 256 + 4 * lane, K - 4));
#pragma unroll
        for (int i = 0; i < CPW; i++) {
            const int64_t c = c0 + nwaves * i;
            if (c >= nch) break;  // uniform within the wave
            bad |= qa_chunk<BLOCK, OUT>(v[i], row, c * 256 + 4 * lane, K, a, lane, parts);
        }
    }
    __shared__ int wflag[16];
    const bool any_bad = wg_any(bad, wflag, nwaves);
    if (threadIdx.x == 0) a.ok[row] = any_bad ? 0 : 1;
}

// y[t] = sum_j weights[t, j] part[t, j] over the pairs that have an expert, in
// the order of the choices: one fma each.
template <int V>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ part, const float* __restrict__ weights,
                                                      const int32_t* __restrict__ expert, int top, int64_t N,
                                                      float* __restrict__ y) {
    const int64_t t = blockIdx.x, n = (((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * 256 + threadIdx.x) * V;
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
    const int P = (int)(T * top);
    const dim3 grid((unsigned)(experts + 1)), block(xr::PLAN_T);
    if (P <= 4 * xr::PLAN_T) hipLaunchKernelGGL(xr::plan_kernel<4>, grid, block, 0, s, ids, P, experts, plan);
    else if (P <= 16 * xr::PLAN_T) hipLaunchKernelGGL(xr::plan_kernel<16>, grid, block, 0, s, ids, P, experts, plan);
    else hipLaunchKernelGGL(xr::plan_kernel<0>, grid, block, 0, s, ids, P, experts, plan);
    return hipGetLastError();
}

namespace xr {
// 32 x 32 tiles, which read x and r half as often from the L2, where they
// give at least 128 workgroups; 16 x 16 below. Parts of K so that a compute unit
// has one workgroup, of the small tiles one or two (us in a graph with one / two:
// K = 4096, 8 experts, 2048 tokens 23.6 / 19.2, 1024 13.9 / 13.0, 512 11.1 / 11.2;
// K = 2048, 128 experts, 181 tokens 15.2 / 14.6; of the large ones 60 experts, 2048
// tokens 24.2 / 26.0).
struct Shape {
    int n, parts;
};
static Shape route_shape(int64_t T, int experts) {
    const int64_t t32 = (T + 31) / 32 * ((experts + 31) / 32), t16 = (T + 15) / 16 * ((experts + 15) / 16);
    Shape r{t32 >= 128 ? 32 : 16, 1};
    for (const int64_t tiles = r.n == 32 ? t32 : t16; r.parts < 16 && tiles * r.parts * 2 <= (r.n == 32 ? 256 : 512);) r.parts *= 2;
    return r;
}
}  // namespace xr

// More tokens never need less: parts beyond one are of at most 512 small or 256
// large tiles, 2^18 sums.
uint64_t experts_route_ws_bytes(int64_t T, int experts) {
    const int64_t n = T * experts, parted = 16 * n < (1 << 18) ? 16 * n : 1 << 18;
    return 8 * (uint64_t)(n > parted ? n : parted);
}

hipError_t launch_experts_route(const float* x, const float* router, int64_t T, int64_t K, int experts, int top, int normalize,
                                int32_t* ids, float* weights, int32_t* plan, double* logits, hipStream_t s) {
    if (T <= xr::ONE_T && T * experts * K <= xr::ONE_PRODUCTS && T * top <= xr::SMALL_PAIRS) {
        // parts of K that keep 16 waves at work
        int parts = 1;
        while (experts * parts < 16 && K / parts >= 512) parts *= 2;
        hipLaunchKernelGGL(xr::route_one_kernel, dim3(1), dim3(1024), 0, s, x, router, (int)T, K, experts, parts, top, normalize, ids,
                           weights, plan);
        return hipGetLastError();
    }
    const xr::Shape r = xr::route_shape(T, experts);
    const dim3 grid((unsigned)((T + r.n - 1) / r.n), (unsigned)((experts + r.n - 1) / r.n), (unsigned)r.parts), block(64 * xr::WAVES);
    if (r.n == 16) hipLaunchKernelGGL((xr::logits_kernel<1, false>), grid, block, 0, s, x, router, T, K, experts, logits);
    else if (K % 16) hipLaunchKernelGGL((xr::logits_kernel<2, false>), grid, block, 0, s, x, router, T, K, experts, logits);
    else hipLaunchKernelGGL((xr::logits_kernel<2, true>), grid, block, 0, s, x, router, T, K, experts, logits);
    if (plan && T <= xr::SMALL_T && T * experts <= xr::SMALL_LOGITS && T * top <= xr::SMALL_PAIRS) {
        hipLaunchKernelGGL(xr::select_plan_kernel, dim3(1), dim3(1024), 0, s, logits, r.parts, (int)T, experts, top, normalize, ids,
                           weights, plan);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(xr::select_kernel, dim3((unsigned)((T + 3) / 4)), dim3(256), 0, s, logits, r.parts, T, experts, top, normalize,
                       ids, weights);
    if (plan) return launch_experts_plan(ids, T, top, experts, plan, s);
    return hipGetLastError();
}

namespace xr {
template <int BLOCK, int OUT>
static void launch_quantize(const float* x, int64_t rows, int64_t K, const ActPtrs& a, _Float16* parts, hipStream_t s) {
    const int64_t chunks = (K + 255) / 256;
    int waves = (int)(chunks < 16 ? chunks : 16);
    while (waves > 1 && rows * 64 * waves >= (1ll << 32)) waves /= 2;  // (a launch has less than 2^32 threads)
    const int64_t cpw = (chunks + waves - 1) / waves;
    const dim3 grid((unsigned)rows), block(64 * waves);
    if (cpw == 1) hipLaunchKernelGGL((quantize_kernel<BLOCK, OUT, 1>), grid, block, 0, s, x, K, a, parts);
    else if (cpw == 2) hipLaunchKernelGGL((quantize_kernel<BLOCK, OUT, 2>), grid, block, 0, s, x, K, a, parts);
    else hipLaunchKernelGGL((quantize_kernel<BLOCK, OUT, 4>), grid, block, 0, s, x, K, a, parts);
}
}  // namespace xr

hipError_t launch_experts_quantize(uint32_t dt, const float* x, int64_t rows, int64_t K, const ActPtrs& a, void* parts, hipStream_t s) {
    if (dt == DT_Q4_K) xr::launch_quantize<256, QA_TILE_MINS>(x, rows, K, a, (_Float16*)parts, s);
    else if (dt == DT_Q6_K) xr::launch_quantize<256, QA_TILE>(x, rows, K, a, nullptr, s);
    else xr::launch_quantize<32, QA_TILE>(x, rows, K, a, nullptr, s);
    return hipGetLastError();
}

hipError_t launch_experts_sum(const float* part, const float* weights, const int32_t* expert, int64_t T, int top, int64_t N,
                              float* y, hipStream_t s) {
    // (a grid has at most 65535 workgroups in y, and less than 2^32 threads)
    const int64_t wgs = ((N % 4 ? N : N / 4) + 255) / 256, layers = (wgs + 65534) / 65535;
    const int64_t most = ((1ll << 24) - 1) / ((wgs + layers - 1) / layers * layers);  // tokens of a launch
    for (int64_t t = 0; t < T; t += most) {
        const dim3 grid((unsigned)(T - t < most ? T - t : most), (unsigned)((wgs + layers - 1) / layers), (unsigned)layers);
        const float *p = part + t * top * N, *w = weights + t * top;
        if (N % 4 == 0) hipLaunchKernelGGL(xr::combine_kernel<4>, grid, dim3(256), 0, s, p, w, expert + t * top, top, N, y + t * N);
        else hipLaunchKernelGGL(xr::combine_kernel<1>, grid, dim3(256), 0, s, p, w, expert + t * top, top, N, y + t * N);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace mimg
