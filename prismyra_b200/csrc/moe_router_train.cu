// Training the router: per-expert counts with the balance and z losses of a batch's logits, and the logits' gradient.
//
// Over the n live rows (valid, and not masked to -inf throughout) with p = softmax(logits), f_e the share of the n*k
// picks that went to expert e and lse the log-sum-exp:
//   counts_e = picks of e,  prob_e = mean p_e,  loss = E sum_e f_e prob_e,  z = mean lse^2
//   d logit_e = p_e (c_e - sum_j p_j c_j) + p_e 2 dz lse / n + [e = id_i] w_i (dw_i - sum_j w_j dw_j),
//   c_e = dloss E counts_e / (k n^2)
// where w are the renormalised top-k weights: w = softmax of the picked logits, so their gradient stays inside the k.
// Both are one pass over the logits, bound by memory where rows are many: 131072 x 256 fp32, a tenth of it padding, takes the
// losses 28 us (126 MB, 4.5 TB/s; 141 warp instructions a row, during which none of its logits are on their way) and a finishing
// launch of 2 us, the gradient 47 us (5.7 TB/s).
// 128 x 128 bf16: 4.4 us, in one CTA; 1000 x 128: the gradient 3.7 us.
//
// A warp holds a row: lane l owns columns 128 i + 4 l + {0..3} (one 16-byte load of fp32, 8 of bf16) where rows start
// on such a boundary, else columns 32 j + l. It keeps kRowsInFlight rows in registers to cover the memory latency, and
// a lane adds its columns' probabilities over all its warp's rows in registers, so the column sums cost no traffic.
// Sums go in a fixed order (rows in a lane, warps in a CTA, CTAs in the finishing launch); only
// the integer counts use atomics.
// p = 2^(x log2 e - m) / s with m = fl(max log2 e): what m is rounded by cancels in p, and lse = ln 2 (m + log2 s) has it
// back. ex2.approx and lg2.approx are good to 2^-22, rcp.approx to 2^-23; the exponent is off by half a unit of itself.
#include <math_constants.h>

#include "lora_dev.cuh"
#include "moe_internal.h"
#include "prismyra_moe.h"

namespace pm {
namespace {

constexpr int kRowsInFlight = 4;
constexpr int kBalanceThreads = 1024;  // one CTA to an SM: its columns' sums meet in shared memory
constexpr int kGradThreads = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A NaN wins, so that it shows.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float warp_max(float v) {
    float y;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
    return y;
}
template <int LANES = 32>
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The columns a lane owns: q-th (q < 4 NV) of lane l.
template <bool VEC>
__device__ __forceinline__ int column_of(int q, int lane) {
    return VEC ? (q >> 2) * 128 + lane * 4 + (q & 3) : q * 32 + lane;
}

template <typename TL>
__device__ __forceinline__ float widen(TL v);
template <>
__device__ __forceinline__ float widen(float v) { return v; }
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename TL>
__device__ __forceinline__ TL narrow(float v);
template <>
__device__ __forceinline__ float narrow(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }

template <typename TL, int NV, bool VEC>
__device__ __forceinline__ void load_row(const TL* row, int E, int lane, float (&v)[4 * NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (VEC) {
            const int c = i * 128 + lane * 4;
            if (c < E) {  // E % 4 == 0
                if constexpr (sizeof(TL) == 4) {
                    const float4 f = __ldcs(reinterpret_cast<const float4*>(row + c));
                    v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
                } else {
                    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(row + c));
                    v[4 * i] = __uint_as_float(u.x << 16), v[4 * i + 1] = __uint_as_float(u.x & 0xffff0000u);
                    v[4 * i + 2] = __uint_as_float(u.y << 16), v[4 * i + 3] = __uint_as_float(u.y & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * i + j] = -CUDART_INF_F;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = (4 * i + j) * 32 + lane;
                v[4 * i + j] = c < E ? widen<TL>(row[c]) : -CUDART_INF_F;
            }
        }
    }
}

// Four rows' values summed over the warp at once: lane l returns the sum of v[l / 8]. Ten shuffles and adds fewer than one
// row at a time; x + y = y + x, so every row gets the same tree.
__device__ __forceinline__ float warp_sum4(const float (&v)[kRowsInFlight], int lane) {
    const bool h = lane & 16, q = lane & 8;
    const float a = (h ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, h ? v[0] : v[2], 16);
    const float b = (h ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, h ? v[1] : v[3], 16);
    float s = (q ? b : a) + __shfl_xor_sync(0xffffffffu, q ? a : b, 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// The rows from t0 on that count: bit u for row t0 + u.
__device__ __forceinline__ uint32_t wanted_rows(const uint8_t* valid, long t0, long T, int lane) {
    const bool want = lane < kRowsInFlight && t0 + lane < T && (valid == nullptr || valid[t0 + lane] != 0);
    return __ballot_sync(0xffffffffu, want);
}

template <typename TL, int NV, bool VEC>
__device__ __forceinline__ void load_rows(const TL* logits, long t0, int E, int lane, uint32_t want,
                                          float (&v)[kRowsInFlight][4 * NV]) {
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
        if ((want >> u) & 1u)
            load_row<TL, NV, VEC>(logits + t0 * E + u * E, E, lane, v[u]);
        else
#pragma unroll
            for (int q = 0; q < 4 * NV; ++q) v[u][q] = -CUDART_INF_F;
    }
}

// v: the rows' logits, replaced by multiples of their probabilities: p = v * scale. Lane l returns row l / 8's scale and
// log-sum-exp (0 where the row is -inf throughout) and whether it is live.
template <int NV>
__device__ __forceinline__ bool rows_softmax(float (&v)[kRowsInFlight][4 * NV], int lane, float* scale, float* lse) {
    float m[kRowsInFlight], s[kRowsInFlight], far = 0.0f;
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
        m[u] = v[u][0];
#pragma unroll
        for (int q = 1; q < 4 * NV; ++q) m[u] = max_nan(m[u], v[u][q]);
        m[u] = warp_max(m[u]);
    }
    const int own = lane >> 3;
    const float mo = own < 2 ? (own == 0 ? m[0] : m[1]) : (own == 2 ? m[2] : m[3]);
    const bool live = !(mo == -CUDART_INF_F);
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
        m[u] = m[u] == -CUDART_INF_F ? 0.0f : m[u];  // a row of -inf becomes 0
        far = fmaxf(far, fabsf(m[u]));
    }
    float start = mo * kLog2e * kLn2;
    if (far > 1e5f) {
        // the rounding of m log2 e, common to a row, would pass 2^0.01 and in the end overflow (as in a row masked with the
        // type's lowest value): the maximum is taken off first
#pragma unroll
        for (int u = 0; u < kRowsInFlight; ++u) {
#pragma unroll
            for (int q = 0; q < 4 * NV; ++q) v[u][q] -= m[u];
            m[u] = 0.0f;
        }
        start = mo;
    }
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
        const float base = m[u] * kLog2e;
        s[u] = 0.0f;
#pragma unroll
        for (int q = 0; q < 4 * NV; ++q) {
            v[u][q] = ex2(fmaf(v[u][q], kLog2e, -base));
            s[u] += v[u][q];
        }
    }
    const float sum = warp_sum4(s, lane);
    *scale = live ? rcp(sum) : 0.0f;
    *lse = live ? fmaf(lg2(sum), kLn2, start) : 0.0f;
    return live;
}

// Where the results go.
struct BalanceOut {
    float* loss;
    float* z_loss;
    float* prob;
    int32_t* counts;
    int32_t* tokens;
};

// Rows are dealt to warps in runs of kRowsInFlight. ONE: the only CTA, which writes the results; else each CTA leaves a
// partial: column sums and counts, the sum of lse^2 and the live rows.
template <typename TL, int NV, bool VEC, bool ONE>
__global__ void __launch_bounds__(kBalanceThreads)
    balance_kernel(const TL* __restrict__ logits, const int32_t* __restrict__ ids, const uint8_t* __restrict__ valid,
                   int T, int E, int k, float* __restrict__ psum, float* __restrict__ zsum, int32_t* __restrict__ cnt,
                   int32_t* __restrict__ tok, BalanceOut out) {
    constexpr int kWarps = kBalanceThreads / 32;
    __shared__ float sp[kWarps][128 * NV];
    __shared__ int32_t sc[128 * NV];
    __shared__ float sz[kWarps];
    __shared__ int32_t sn[kWarps];
    __shared__ double red[8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (int e = tid; e < E; e += kBalanceThreads) sc[e] = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    float acc[4 * NV];
#pragma unroll
    for (int q = 0; q < 4 * NV; ++q) acc[q] = 0.0f;
    float z = 0.0f;  // of the rows at place lane / 8 of their run
    int n = 0;
    const uint32_t inv_k = 65536u / k + 1u;  // j / k = j inv_k >> 16 for the j < 64 of a run
    const long step = (long)gridDim.x * kWarps * kRowsInFlight;
    long t0 = ((long)blockIdx.x * kWarps + warp) * kRowsInFlight;
    uint32_t want = wanted_rows(valid, t0, T, lane);
    while (t0 < T) {
        float v[kRowsInFlight][4 * NV];
        load_rows<TL, NV, VEC>(logits, t0, E, lane, want, v);
        const int m = (int)min((long)kRowsInFlight, T - t0) * k;
        int id[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) id[h] = h * 32 + lane < m ? __ldcs(ids + t0 * k + h * 32 + lane) : -1;
        t0 += step;
        want = wanted_rows(valid, t0, T, lane);  // of the next run, while this one's logits arrive
        float scale, lse;
        const uint32_t live = __ballot_sync(0xffffffffu, rows_softmax<NV>(v, lane, &scale, &lse));  // a byte per row
        z = fmaf(lse, lse, z);
#pragma unroll
        for (int u = 0; u < kRowsInFlight; ++u) {
            const float f = __shfl_sync(0xffffffffu, scale, u * 8);
#pragma unroll
            for (int q = 0; q < 4 * NV; ++q) acc[q] = fmaf(v[u][q], f, acc[q]);
        }
        n += __popc(live & 0x01010101u);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if ((unsigned)id[h] < (unsigned)E && ((live >> ((h * 32 + lane) * inv_k >> 16) * 8) & 1u))
                atomicAdd(&sc[id[h]], 1);
    }
#pragma unroll
    for (int q = 0; q < 4 * NV; ++q) sp[warp][column_of<VEC>(q, lane)] = acc[q];
    z += __shfl_xor_sync(0xffffffffu, z, 8);
    z += __shfl_xor_sync(0xffffffffu, z, 16);
    if (lane == 0) {
        sz[warp] = z;
        sn[warp] = n;
    }
    __syncthreads();
    float s = 0.0f, zs = 0.0f;
    int ns = 0;
    if (tid < E)
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += sp[w][tid];
    if (tid == 0 || ONE)
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            zs += sz[w];
            ns += sn[w];
        }
    if (!ONE) {
        if (tid < E) {
            psum[(size_t)blockIdx.x * E + tid] = s;
            cnt[(size_t)blockIdx.x * E + tid] = sc[tid];
        }
        if (tid == 0) zsum[blockIdx.x] = zs, tok[blockIdx.x] = ns;
        return;
    }
    const double inv = 1.0 / (double)max(ns, 1);
    if (tid < 256) {
        double part = 0.0;
        if (tid < E) {
            const double p = (double)s * inv;
            out.prob[tid] = (float)p;
            out.counts[tid] = sc[tid];
            part = (double)sc[tid] * p;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        if (lane == 0) red[warp] = part;
    }
    __syncthreads();
    if (tid == 0) {
        double t = 0.0;
        for (int w = 0; w < 8; ++w) t += red[w];
        *out.loss = (float)((double)E / k * t * inv);
        *out.z_loss = (float)((double)zs * inv);
        *out.tokens = ns;
    }
}

// The G partials added up, in double and in order, by one cluster: each of eight CTAs has 32 columns, each of its 16 warps
// every 16th partial; the CTAs' shares of the loss meet in the first one's shared memory.
constexpr int kFinishCtas = 8;
constexpr int kFinishThreads = 512;
__global__ void __launch_bounds__(kFinishThreads) balance_finish_kernel(const float* psum, const float* zsum,
                                                                        const int32_t* cnt, const int32_t* tok, int G,
                                                                        int E, int k, BalanceOut out) {
    constexpr int kWarps = kFinishThreads / 32;
    __shared__ double sp[kWarps][32];
    __shared__ int32_t sc[kWarps][32];
    __shared__ int32_t sn;
    __shared__ double sz;
    __shared__ float4 recv[kFinishCtas];  // a CTA's share, two halves of a double
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)blockIdx.x;
    cluster_arrive();
    pdl_wait();
    pdl_trigger();
    const int e = rank * 32 + lane;
    double p = 0.0;
    int c = 0;
    if (e < E)
#pragma unroll 10
        for (int g = warp; g < G; g += kWarps) {
            p += (double)psum[(size_t)g * E + e];
            c += cnt[(size_t)g * E + e];
        }
    sp[warp][lane] = p;
    sc[warp][lane] = c;
    if (warp == kWarps - 1) {
        double z = 0.0;
        int n = 0;
        for (int g = lane; g < G; g += 32) {
            z += (double)zsum[g];
            n += tok[g];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            z += __shfl_xor_sync(0xffffffffu, z, o);
            n += __shfl_xor_sync(0xffffffffu, n, o);
        }
        if (lane == 0) sn = n, sz = z;
    }
    __syncthreads();
    cluster_wait();  // all CTAs run
    const double inv = 1.0 / (double)max(sn, 1);
    if (warp == 0) {
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            p += sp[w][lane];
            c += sc[w][lane];
        }
        p *= inv;
        if (e < E) {
            out.prob[e] = (float)p;
            out.counts[e] = c;
        }
        double part = (double)c * p;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        if (lane == 0)
            st_cluster(cluster_addr(smem_u32(&recv[rank]), 0), __int_as_float(__double2hiint(part)),
                       __int_as_float(__double2loint(part)), 0.0f, 0.0f);
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (rank == 0 && tid == 0) {
        double t = 0.0;
        for (int q = 0; q < kFinishCtas; ++q) t += __hiloint2double(__float_as_int(recv[q].x), __float_as_int(recv[q].y));
        *out.loss = (float)((double)E / k * t * inv);
        *out.z_loss = (float)(sz * inv);
        *out.tokens = sn;
    }
}

struct GradArgs {
    const int32_t* ids;
    const float* w;   // with dw: the top-k weights and their gradient, or null
    const float* dw;
    const int32_t* counts;  // with tokens: the balance pass's, or null (no loss terms)
    const int32_t* tokens;
    const uint8_t* valid;
    float d_loss, d_z;
    const float* d_loss_dev;  // factors in device memory, or null
    const float* d_z_dev;
    int T, E, k;
};

// A warp takes kRowsInFlight rows at a time. Of their top-k terms lane u kp + j has pick j of row u (kp: k rounded up to a power of
// two; with kp = 16 the rows take two passes) and puts its term into the row's columns in shared memory, from where the row's
// lanes add them as they store.
template <typename TL, int NV, bool VEC>
__global__ void __launch_bounds__(kGradThreads, 3)
    router_grad_kernel(const TL* logits, const GradArgs g, TL* dlogits) {  // dlogits may be logits
    constexpr int kWarps = kGradThreads / 32;
    __shared__ __align__(16) float pick[kWarps][kRowsInFlight][128 * NV];  // zero between runs of rows
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int E = g.E, k = g.k;
    for (int e = lane; e < kRowsInFlight * 128 * NV; e += 32) pick[warp][0][e] = 0.0f;
    __syncwarp();
    pdl_wait();
    pdl_trigger();
    float c[4 * NV], dz = 0.0f;
#pragma unroll
    for (int q = 0; q < 4 * NV; ++q) c[q] = 0.0f;
    if (g.counts != nullptr) {
        const float n = fmaxf((float)*g.tokens, 1.0f);
        const float dl = g.d_loss * (g.d_loss_dev != nullptr ? *g.d_loss_dev : 1.0f) * (float)E / ((float)k * n * n);
        dz = g.d_z * (g.d_z_dev != nullptr ? *g.d_z_dev : 1.0f) * 2.0f / n;
#pragma unroll
        for (int q = 0; q < 4 * NV; ++q) {
            const int e = column_of<VEC>(q, lane);
            if (e < E) c[q] = dl * (float)g.counts[e];
        }
    }
    const int shift_k = k <= 1 ? 0 : 32 - __clz(k - 1), kp = 1 << shift_k;
    const int rows_pass = min(kRowsInFlight, 32 >> shift_k);  // rows whose picks the lanes hold at once
    const long step = (long)gridDim.x * kWarps * kRowsInFlight;
    long next = ((long)blockIdx.x * kWarps + warp) * kRowsInFlight;
    uint32_t want = wanted_rows(g.valid, next, g.T, lane);
    while (next < g.T) {
        const long t0 = next;
        float v[kRowsInFlight][4 * NV];
        load_rows<TL, NV, VEC>(logits, t0, E, lane, want, v);
        const int u_pick = lane >> shift_k, j_pick = lane & (kp - 1);
        int id = -1;
        float w = 0.0f, dw = 0.0f;
        auto load_pick = [&](int u0) {
            const long t = t0 + u0 + u_pick;
            id = -1;
            w = dw = 0.0f;
            if (g.w != nullptr && u_pick < rows_pass && j_pick < k && t < g.T) {
                id = g.ids[t * k + j_pick];
                w = g.w[t * k + j_pick];
                dw = g.dw[t * k + j_pick];
            }
        };
        load_pick(0);
        next += step;
        want = wanted_rows(g.valid, next, g.T, lane);  // of the next run, while this one's logits arrive
        float scale, lse, dot[kRowsInFlight];
        const uint32_t live = __ballot_sync(0xffffffffu, rows_softmax<NV>(v, lane, &scale, &lse));  // a byte per row
#pragma unroll
        for (int u = 0; u < kRowsInFlight; ++u) {
            const float f = __shfl_sync(0xffffffffu, scale, u * 8);
            dot[u] = 0.0f;
#pragma unroll
            for (int q = 0; q < 4 * NV; ++q) {
                v[u][q] *= f;
                dot[u] = fmaf(v[u][q], c[q], dot[u]);
            }
        }
        const float shift = fmaf(dz, lse, -warp_sum4(dot, lane));
#pragma unroll
        for (int u = 0; u < kRowsInFlight; ++u) {
            const float f = __shfl_sync(0xffffffffu, shift, u * 8);
#pragma unroll
            for (int q = 0; q < 4 * NV; ++q) v[u][q] *= c[q] + f;
        }
        int marks[2] = {-1, -1};  // columns this lane has put something into, per pass
        if (g.w != nullptr) {
            for (int pass = 0; pass * rows_pass < kRowsInFlight; ++pass) {
                if (pass > 0) load_pick(rows_pass);
                const int u = pass * rows_pass + u_pick;
                if (u_pick >= rows_pass || (unsigned)id >= (unsigned)E || !((live >> (u * 8)) & 1u)) id = -1;
                const float product = id >= 0 ? w * dw : 0.0f;
                float sum = product;
                for (int o = kp >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const float term = w * (dw - sum);
                const int key = id >= 0 ? u * 128 * NV + id : -1 - lane;
                const uint32_t peers = __match_any_sync(0xffffffffu, key);
                float* at = &pick[warp][0][0];
                if (__all_sync(0xffffffffu, (peers & (peers - 1u)) == 0u)) {
                    if (id >= 0) at[key] = term;
                } else {  // an expert picked twice: in order
                    for (int j = 0; j < kp; ++j) {
                        if (j_pick == j && id >= 0) at[key] += term;
                        __syncwarp();
                    }
                }
                marks[pass & 1] = id >= 0 ? key : -1;
            }
            __syncwarp();
        }
#pragma unroll
        for (int u = 0; u < kRowsInFlight; ++u) {
            const long t = t0 + u;
            if (t >= g.T) break;
            TL* row = dlogits + t * E;
            const float* pk = pick[warp][u];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (VEC) {
                    const int col = i * 128 + lane * 4;
                    if (col >= E) continue;
                    if (g.w != nullptr) {
                        const float4 f = *reinterpret_cast<const float4*>(pk + col);
                        v[u][4 * i] += f.x, v[u][4 * i + 1] += f.y, v[u][4 * i + 2] += f.z, v[u][4 * i + 3] += f.w;
                    }
                    if constexpr (sizeof(TL) == 4) {
                        __stcs(reinterpret_cast<float4*>(row + col),
                               make_float4(v[u][4 * i], v[u][4 * i + 1], v[u][4 * i + 2], v[u][4 * i + 3]));
                    } else {
                        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[u][4 * i], v[u][4 * i + 1]);
                        const __nv_bfloat162 hi = __floats2bfloat162_rn(v[u][4 * i + 2], v[u][4 * i + 3]);
                        uint2 o;
                        o.x = *reinterpret_cast<const uint32_t*>(&lo);
                        o.y = *reinterpret_cast<const uint32_t*>(&hi);
                        __stcs(reinterpret_cast<uint2*>(row + col), o);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int col = (4 * i + j) * 32 + lane;
                        if (col < E) row[col] = narrow<TL>(v[u][4 * i + j] + (g.w != nullptr ? pk[col] : 0.0f));
                    }
                }
            }
        }
        if (g.w != nullptr) {
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (marks[h] >= 0) pick[warp][0][marks[h]] = 0.0f;
            __syncwarp();
        }
    }
}

// Rows can be read (and written) in pieces of four columns.
bool whole_pieces(const void* a, const void* b, int E, int elem) {
    return E % 4 == 0 && (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % (4 * elem) == 0;
}

// Rows up to which one CTA does the whole balance pass in one launch: it holds 128 rows at a time.
constexpr int kBalanceOneCta = 256;

template <typename TL, int NV, bool VEC>
cudaError_t balance_typed(const void* logits, const int32_t* ids, const uint8_t* valid, int T, int E, int k,
                          const BalanceOut& out, void* ws, int G, cudaStream_t s) {
    const TL* lg = static_cast<const TL*>(logits);
    if (T <= kBalanceOneCta)
        return launch_pdl(balance_kernel<TL, NV, VEC, true>, dim3(1), dim3(kBalanceThreads), 0, s, lg, ids, valid, T, E, k,
                          nullptr, nullptr, nullptr, nullptr, out);
    float* psum = static_cast<float*>(ws);
    float* zsum = psum + (size_t)G * E;
    int32_t* cnt = reinterpret_cast<int32_t*>(zsum + G);
    int32_t* tok = cnt + (size_t)G * E;
    PM_TRY(launch_pdl(balance_kernel<TL, NV, VEC, false>, dim3(G), dim3(kBalanceThreads), 0, s, lg, ids, valid, T, E, k,
                      psum, zsum, cnt, tok, out));
    return launch_cluster(balance_finish_kernel, dim3(kFinishCtas), dim3(kFinishThreads), kFinishCtas, 0, s,
                          (const float*)psum, (const float*)zsum, (const int32_t*)cnt, (const int32_t*)tok, G, E, k, out);
}

template <typename TL, int NV, bool VEC>
cudaError_t grad_typed(const void* logits, const GradArgs& g, void* dlogits, int sms, cudaStream_t s) {
    const int blocks = (int)std::min<long>(((long)g.T + kGradThreads / 32 * kRowsInFlight - 1) /
                                               (kGradThreads / 32 * kRowsInFlight), (long)sms * 3);
    return launch_pdl(router_grad_kernel<TL, NV, VEC>, dim3(blocks), dim3(kGradThreads), 0, s,
                      static_cast<const TL*>(logits), g, static_cast<TL*>(dlogits));
}

// CTAs of the balance pass, each of which leaves a partial.
int balance_parts(int T, int sms) {
    if (T <= kBalanceOneCta) return 1;
    constexpr int rows = kBalanceThreads / 32 * kRowsInFlight;
    return (int)std::min<long>(((long)T + rows - 1) / rows, sms);
}

}  // namespace
}  // namespace pm

using namespace pm;

extern "C" {

size_t pm_moe_router_balance_workspace_bytes(int T, int E) {
    if (T < 0 || E <= 0 || E > kMaxExperts || T <= kBalanceOneCta) return 0;
    return (size_t)balance_parts(T, kMaxSms) * (E + 1) * 8;
}

int pm_moe_router_balance(const void* logits, int logits_f32, const int32_t* topk_ids, const uint8_t* valid, int T, int E,
                          int k, float* loss, float* z_loss, float* prob, int32_t* counts, int32_t* tokens,
                          void* workspace, size_t workspace_bytes, pm_stream_t stream) {
    if (T < 0 || E <= 0 || k <= 0) return PM_ERR_INVALID;
    if (E > kMaxExperts || k > kMaxTopK || k > E) return PM_ERR_SHAPE;
    const bool alone = T <= kBalanceOneCta;  // one CTA, which leaves no partial sums
    if (!loss || !z_loss || !prob || !counts || !tokens || (!alone && !workspace) || (T > 0 && (!logits || !topk_ids)))
        return PM_ERR_INVALID;
    if (!alone && (reinterpret_cast<uintptr_t>(workspace) & 15u)) return PM_ERR_ALIGN;
    if (workspace_bytes < pm_moe_router_balance_workspace_bytes(T, E)) return PM_ERR_WORKSPACE;
    int sms = 0;
    const int st = device_sms(&sms);
    if (st != PM_OK) return st;
    const BalanceOut out{loss, z_loss, prob, counts, tokens};
    const int G = balance_parts(T, std::min(sms, kMaxSms));
    const bool vec = whole_pieces(logits, logits, E, logits_f32 ? 4 : 2);
    cudaStream_t s = (cudaStream_t)stream;
#define PM_BALANCE(TL, NV, VEC) balance_typed<TL, NV, VEC>(logits, topk_ids, valid, T, E, k, out, workspace, G, s)
#define PM_BALANCE_E(TL) \
    (E <= 128 ? (vec ? PM_BALANCE(TL, 1, true) : PM_BALANCE(TL, 1, false)) : (vec ? PM_BALANCE(TL, 2, true) : PM_BALANCE(TL, 2, false)))
    const cudaError_t e = logits_f32 ? PM_BALANCE_E(float) : PM_BALANCE_E(__nv_bfloat16);
#undef PM_BALANCE_E
#undef PM_BALANCE
    return e == cudaSuccess ? PM_OK : PM_ERR_CUDA;
}

int pm_moe_router_grad(const void* logits, int logits_f32, const int32_t* topk_ids, const float* topk_w,
                       const float* d_topk_w, const int32_t* counts, const int32_t* tokens, const uint8_t* valid, int T,
                       int E, int k, float d_loss, const float* d_loss_dev, float d_z, const float* d_z_dev, void* dlogits,
                       pm_stream_t stream) {
    if (T < 0 || E <= 0 || k <= 0) return PM_ERR_INVALID;
    if (E > kMaxExperts || k > kMaxTopK || k > E) return PM_ERR_SHAPE;
    if ((topk_w == nullptr) != (d_topk_w == nullptr) || (counts == nullptr) != (tokens == nullptr)) return PM_ERR_INVALID;
    if (T == 0) return PM_OK;
    if (!logits || !dlogits || (topk_w != nullptr && !topk_ids)) return PM_ERR_INVALID;
    int sms = 0;
    const int st = device_sms(&sms);
    if (st != PM_OK) return st;
    const GradArgs g{topk_ids, topk_w, d_topk_w, counts, tokens, valid, d_loss, d_z, d_loss_dev, d_z_dev, T, E, k};
    const bool vec = whole_pieces(logits, dlogits, E, logits_f32 ? 4 : 2);
    cudaStream_t s = (cudaStream_t)stream;
#define PM_GRAD(TL, NV, VEC) grad_typed<TL, NV, VEC>(logits, g, dlogits, sms, s)
#define PM_GRAD_E(TL) \
    (E <= 128 ? (vec ? PM_GRAD(TL, 1, true) : PM_GRAD(TL, 1, false)) : (vec ? PM_GRAD(TL, 2, true) : PM_GRAD(TL, 2, false)))
    const cudaError_t e = logits_f32 ? PM_GRAD_E(float) : PM_GRAD_E(__nv_bfloat16);
#undef PM_GRAD_E
#undef PM_GRAD
    return e == cudaSuccess ? PM_OK : PM_ERR_CUDA;
}

}  // extern "C"
