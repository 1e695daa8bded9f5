// Low-rank adapters of many requests beside a shared projection, and their gradients: entry points, the kernel for few
// rows and the row plan of the tiled kernels (moe_lora_tiles.cu).
//
//   h[t] = s_n A_n x[t]  (R values),  out[t] = base[t] + B_n h[t],  n = adapter[t]
//   d[t] = s_n B_n^T dy[t],  dx[t] = base[t] + A_n^T d[t],  dA_n = sum_t d[t] x[t]^T,  dB_n = sum_t dy[t] h[t]^T
// A row whose adapter is outside [0, N) has no term: out = base, dx = base, nothing for dA and dB.
#include <string.h>

#include <atomic>

#include "moe_lora.h"
#include "prismyra_moe.h"
#include "lora_dev.cuh"

namespace pm {
namespace {

// ------------------------------------------------------------------------------------------- the fused kernel
// A cluster of CTAs per group of up to 16 rows of one adapter. Each warp multiplies the group's rows with its 32-column
// pieces of A straight from global memory (mma.sync m16n8k16: what costs here is the operands' way in, and these need no
// staging), the warps' sums meet in every CTA's shared memory, and each warp then makes its 32-column pieces of the result.
// One launch, two trips to memory (weights and base of the first piece are asked for before the sums meet), one cluster
// barrier; many groups at a time keep the memory busy. Bound by latency: replayed, one row 2048 -> 4096 of rank 16 4.1 us, 48
// rows of 64 adapters 5.7 us (6 MB), 731 rows of rank 8 8.6 us with the plan; where many adapters have a few rows each by how
// well its CTAs' waits overlap: 512 rows of 512 adapters of rank 16 28 us (48 MB), 4096 of 1024 61 us (180 MB).
//
// Groups come from the rows' adapters themselves up to kLoraFewRows rows (PLANNED false): a cluster per row, of which the
// first of every 16 rows of one adapter works for all of them and the others leave at once. Above that the plan lists them.
//
// Operand order: a lane's 16 bytes are 8 neighbouring values of the contraction, which the MMA takes as positions
// {2c, 2c+1, 2c+8, 2c+9} of two steps; both operands are read so, and the sum does not care. In the second product the
// MMA's column j of tile i is column 8 (j / 2) + 2 i + j % 2 of the piece, so that a lane ends up with 8 neighbours.
//
// It runs on the plan's groups where rows x ranks are few, in all or on average for a loaded adapter: every group reads its
// adapter's weights, and the tiled kernels read them once for 128 rows but work on 128 however few there are. Which adapters have
// rows the host cannot know, so the rule weighs both ends: rows spread over all adapters / all of one (or 64: the same within a
// few us). This against the tiled kernels, us replayed, 2048 -> 2048 (rows, rank, adapters):
//   in all         1000 x 64 of 4 15.8 and 17.3; 4096 x 16 of 64 21 / 19 and 28 / -; 5120 x 16 of 4 38 and 32
//   256 for each   4096 x 64 of 1024 143 / 43 and 243 / 31; 16384 x 16 of 1024 87 / 67 and 202 / 52
//   512 for each   2048 x 64 of 256 47 / 22 and 74 / 25; 4096 x 64 of 512 86 / 42 and 130 / 29; 2048 x 128 of 512 171 / 44 and
//                  232 / 31; 16384 x 32 of 1024 123 / 84 and 212 / 54; 8192 x 64 of 1024 151 / 78 and 249 / 39
//   640            5120 x 64 of 512 88 / 55 and 131 / 31
//   1024           4096 x 64 of 256 65 / 41 and 73 / 29; 8192 x 64 of 512 108 / 76 and 133 / 37; 16384 x 64 of 1024 207 / 135 and
//                  254 / 57; 65536 x 16 of 1024 256 / 217 and 284 / 169; 8192 x 16 of 128 37 / 34 and 41 / 33
// Up to 512 neither choice loses more than the other where it is the wrong one; beyond, this kernel loses up to 2.4 times on rows
// of few adapters, and the tiled ones at most 1.5 on spread rows.
constexpr long kFusedRowRanks = 65536;
constexpr long kFusedRowRanksEach = 512;
bool lora_fused(int T, int R, int N) { return (long)T * R <= std::max(kFusedRowRanks, kFusedRowRanksEach * N); }
constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewGroup = kLoraGroupRows;

struct FewArgs {
    const bf16* x;
    long ldx;
    const bf16* a;
    const bf16* b;
    const int32_t* adapter;
    const float* scale;
    const bf16* base;
    long ldbase;
    bf16* out;
    long ldout;
    int T, K, O, R, N;
    const int32_t* ngroups;  // the plan, where there is one
    const int2* groups;
    const int32_t* rows;
};

template <int NT, int CTAS>  // tiles of 8 ranks, CTAs of a cluster
constexpr size_t few_smem() {
    constexpr int r = 8 * NT, rp = NT == 1 ? 16 : 8 * NT;
    return sizeof(float) * kFewGroup * r * (kFewWarps + CTAS) + 2 * kFewGroup * (rp + 8) * 2;
}

template <int NT, bool PLANNED, int CTAS>
__global__ void __launch_bounds__(kFewThreads) lora_fused_kernel(const FewArgs g) {
    constexpr int kR = 8 * NT;                   // ranks a lane's tiles cover; g.R of them exist
    constexpr int kRp = NT == 1 ? 16 : 8 * NT;
    constexpr int kChunks = kRp / 16;
    constexpr int kLdh = kRp + 8;                // bf16 from one hidden row to the next: rows on different banks
    constexpr int kM = kFewGroup;
    extern __shared__ __align__(16) uint8_t few_raw[];
    float* red = reinterpret_cast<float*>(few_raw);      // [warps][kM][kR]
    float* recv = red + kFewWarps * kM * kR;             // [CTAs][kM][kR]
    bf16* hs = reinterpret_cast<bf16*>(recv + CTAS * kM * kR);  // [2][kM][kLdh]: halves
    __shared__ int members[kM];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)(blockIdx.x % CTAS), group = (int)(blockIdx.x / CTAS);
    const int gr = lane >> 2, c = lane & 3;
    int n, row[2];  // rows gr and gr + 8 of the group, -1: none
    if (PLANNED) {
        // rows without an adapter, dealt out to all warps; their adapters and base were there before the plan's launch
        if (g.base != g.out) {
            const long warps = (long)gridDim.x * kFewWarps;
            for (long t0 = (long)blockIdx.x * kFewWarps + warp; t0 < g.T; t0 += warps * 32) {
                const long tl = t0 + lane * warps;
                uint32_t none = __ballot_sync(0xffffffffu, tl < g.T && (unsigned)__ldcg(g.adapter + tl) >= (unsigned)g.N);
                while (none != 0) {
                    copy_row(g.base, g.ldbase, g.out, g.ldout, t0 + (__ffs(none) - 1) * warps, g.O, lane, 32);
                    none &= none - 1;
                }
            }
        }
        pdl_wait();
        pdl_trigger();
        if (group >= *g.ngroups) return;
        cluster_arrive();
        const int2 mine = g.groups[group];
        n = mine.y >> 8;
#pragma unroll
        for (int i = 0; i < 2; ++i) row[i] = i * 8 + gr < (mine.y & 255) ? g.rows[mine.x + i * 8 + gr] : -1;
    } else {
        pdl_wait();
        pdl_trigger();
        // which rows: every warp looks at all (at most 128) adapters
        int id[kLoraFewRows / 32];
#pragma unroll
        for (int w = 0; w < kLoraFewRows / 32; ++w) id[w] = w * 32 + lane < g.T ? g.adapter[w * 32 + lane] : -1;
        n = g.adapter[group];
        if ((unsigned)n >= (unsigned)g.N) {
            if (g.base != g.out)
                copy_row(g.base, g.ldbase, g.out, g.ldout, group, g.O, rank * kFewThreads + tid, CTAS * kFewThreads);
            return;
        }
        int before = 0, order[kLoraFewRows / 32], all = 0;
#pragma unroll
        for (int w = 0; w < kLoraFewRows / 32; ++w) {
            const uint32_t m = __ballot_sync(0xffffffffu, id[w] == n);
            order[w] = all + __popc(m & ((1u << lane) - 1u));
            const int left = group - w * 32;
            before += left >= 32 ? __popc(m) : left > 0 ? __popc(m & ((1u << left) - 1u)) : 0;
            all += __popc(m);
        }
        if (before % kM != 0) return;  // another row's cluster works for this one
        cluster_arrive();
        const int count = min(kM, all - before);
        if (warp == 0) {
#pragma unroll
            for (int w = 0; w < kLoraFewRows / 32; ++w)
                if (id[w] == n && order[w] >= before && order[w] < before + count) members[order[w] - before] = w * 32 + lane;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) row[i] = gr + 8 * i < count ? members[gr + 8 * i] : -1;
    }
    const int gw = rank * kFewWarps + warp;
    constexpr int kAllWarps = CTAS * kFewWarps;
    const uint4 zero = make_uint4(0, 0, 0, 0);

    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    const bf16* a = g.a + (long)n * g.R * g.K;
    for (int s = gw; s * 32 < g.K; s += kAllWarps) {
        const int k = s * 32 + c * 8;
        const bool in = k < g.K;
        uint4 x[2], w[NT];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            x[i] = in && row[i] >= 0 ? *reinterpret_cast<const uint4*>(g.x + (long)row[i] * g.ldx + k) : zero;
#pragma unroll
        for (int j = 0; j < NT; ++j)
            w[j] = in && j * 8 < g.R ? *reinterpret_cast<const uint4*>(a + (long)(j * 8 + gr) * g.K + k) : zero;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            mma16816(acc[j], x[0].x, x[1].x, x[0].y, x[1].y, w[j].x, w[j].y);
            mma16816(acc[j], x[0].z, x[1].z, x[0].w, x[1].w, w[j].z, w[j].w);
        }
    }
    // this warp's first piece of the result: its weights and base, on their way while the sums meet
    const bf16* b = g.b + (long)n * g.O * g.R;
    uint2 wb[4][kChunks];
    uint4 y[2];
    auto ask = [&](int u) {
        const int o = u * 32 + (gr >> 1) * 8 + (gr & 1);
        const bool in = u * 32 + (gr >> 1) * 8 < g.O;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < kChunks; ++q)
                wb[i][q] = in && q * 16 + c * 4 < g.R
                               ? *reinterpret_cast<const uint2*>(b + (long)(o + 2 * i) * g.R + q * 16 + c * 4)
                               : make_uint2(0, 0);
        const int col = u * 32 + c * 8;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            y[i] = g.base != nullptr && col < g.O && row[i] >= 0
                       ? *reinterpret_cast<const uint4*>(g.base + (long)row[i] * g.ldbase + col)
                       : zero;
    };
    int u = gw;
    if (u * 32 < g.O) ask(u);

#pragma unroll
    for (int j = 0; j < NT; ++j) {
        float* at = red + (warp * kM + gr) * kR + j * 8 + c * 2;
        *reinterpret_cast<float2*>(at) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(at + 8 * kR) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    cluster_wait();  // all CTAs of the cluster run
    for (int i = tid; i < kM * kR / 4; i += kFewThreads) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float4 p = *reinterpret_cast<const float4*>(red + w * kM * kR + i * 4);
            v.x += p.x, v.y += p.y, v.z += p.z, v.w += p.w;
        }
        const uint32_t at = smem_u32(recv + rank * kM * kR + i * 4);
#pragma unroll
        for (int q = 0; q < CTAS; ++q) st_cluster(cluster_addr(at, q), v.x, v.y, v.z, v.w);
    }
    cluster_arrive();
    cluster_wait();
    const float sc = g.scale != nullptr ? g.scale[n] : 1.0f;
    for (int i = tid; i < kM * kRp; i += kFewThreads) {
        const int r = i % kRp, m = i / kRp;
        float v = 0.0f;
        if (r < g.R) {  // the padding of the rank stays 0 whatever the rows hold; rows that are none go nowhere
#pragma unroll
            for (int q = 0; q < CTAS; ++q) v += recv[(q * kM + m) * kR + r];
            v *= sc;
        }
        split2(v, hs + m * kLdh + r, hs + (kM + m) * kLdh + r);
    }
    __syncthreads();

    for (; u * 32 < g.O; u += kAllWarps) {
        const int col = u * 32 + c * 8;
        float d[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[i][e] = 0.0f;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int q = 0; q < kChunks; ++q) {
                const bf16* at = hs + (half * kM + gr) * kLdh + q * 16 + c * 4;
                const uint2 h0 = *reinterpret_cast<const uint2*>(at), h1 = *reinterpret_cast<const uint2*>(at + 8 * kLdh);
#pragma unroll
                for (int i = 0; i < 4; ++i) mma16816(d[i], h0.x, h1.x, h0.y, h1.y, wb[i][q].x, wb[i][q].y);
            }
        if (any_not_finite(d)) {  // once more (here: a call would cost registers, of which four CTAs to an SM have 64 a thread)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!any_not_finite(d[i])) continue;  // a tile at a time
                float high[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int q = 0; q < kChunks; ++q) {
                    const bf16* at = hs + gr * kLdh + q * 16 + c * 4;
                    const uint2 h0 = *reinterpret_cast<const uint2*>(at), h1 = *reinterpret_cast<const uint2*>(at + 8 * kLdh);
                    mma16816(high, h0.x, h1.x, h0.y, h1.y, wb[i][q].x, wb[i][q].y);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) d[i][e] = both_halves(d[i][e], high[e]);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint4 o = y[h];
            o.x = add_bf16x2(o.x, d[0][2 * h], d[0][2 * h + 1]);
            o.y = add_bf16x2(o.y, d[1][2 * h], d[1][2 * h + 1]);
            o.z = add_bf16x2(o.z, d[2][2 * h], d[2][2 * h + 1]);
            o.w = add_bf16x2(o.w, d[3][2 * h], d[3][2 * h + 1]);
            if (col < g.O && row[h] >= 0) *reinterpret_cast<uint4*>(g.out + (long)row[h] * g.ldout + col) = o;
        }
        if ((u + kAllWarps) * 32 < g.O) ask(u + kAllWarps);
    }
}

template <int NT, bool PLANNED, int CTAS>
cudaError_t launch_fused_as(const FewArgs& g, int groups, cudaStream_t s) {
    constexpr size_t smem = few_smem<NT, CTAS>();
    if (smem > (48 << 10)) {
        static std::atomic<bool> configured[64];
        PM_TRY(raise_smem((const void*)lora_fused_kernel<NT, PLANNED, CTAS>, smem, configured));
    }
    return launch_cluster(lora_fused_kernel<NT, PLANNED, CTAS>, dim3((unsigned)groups * CTAS), dim3(kFewThreads), CTAS, smem,
                          s, g);
}

template <bool PLANNED, int CTAS>
cudaError_t launch_fused(const FewArgs& g, int groups, cudaStream_t s) {
    if (g.R <= 8) return launch_fused_as<1, PLANNED, CTAS>(g, groups, s);
    if (g.R <= 16) return launch_fused_as<2, PLANNED, CTAS>(g, groups, s);
    if (g.R <= 32) return launch_fused_as<4, PLANNED, CTAS>(g, groups, s);
    if (g.R <= 64) return launch_fused_as<8, PLANNED, CTAS>(g, groups, s);
    return launch_fused_as<16, PLANNED, CTAS>(g, groups, s);
}

// On the plan's groups: eight CTAs for each where every CTA has an SM of its own, four where all can be there at a time, else
// two (us replayed with eight, four and two): 11 groups of rank 128, 4096 -> 4096 18.1, 23.1, 34.6; 22 of rank 64 13.1, 12.2,
// 15.0; 66 of rank 32 16.8, 11.4, 12.1; 136 of rank 16 12.9, 10.0, 11.1; 272 18.0, 15.4, 14.7; 1062 56, 44, 43.
cudaError_t launch_groups(const FewArgs& g, int sms, cudaStream_t s) {
    const int groups = lora_max_groups(g.T, g.N);
    const int resident = g.R <= 16 ? 4 : g.R <= 32 ? 3 : g.R <= 64 ? 2 : 1;  // CTAs of an SM, by their registers
    if (groups * 8 <= sms) return launch_fused<true, 8>(g, groups, s);
    return groups * 4 <= sms * resident ? launch_fused<true, 4>(g, groups, s) : launch_fused<true, 2>(g, groups, s);
}

// ------------------------------------------------------------------------------------------- the row plan
// A stable counting sort of the rows by adapter, every adapter's rows starting a block of their own. Each warp has a run of
// rows that it counts and, once all counts are known (a thread sums an adapter's over the warps; a warp for each took 12 us
// more at 1000 adapters), places in order (equal adapters in a warp find each other with match, about 1 us where all 32
// differ). One CTA up to kPlanOneCta rows; above, one cluster of eight, which exchange their counts
// through shared memory. Bound by latency; after the wait for its predecessor, one CTA against eight: 731 rows 2.4 and
// 2.8 us, 2048 2.7 and 2.9, 5120 3.7 and 2.8, 16384 7.2 and 3.5; 4096 rows of 64 adapters in any order 8.8 and 6.3.
constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanCtas = 8;
constexpr int kPlanOneCta = 2048;
constexpr int kPlanAhead = 4;  // ids a lane has in flight, and keeps between counting and placing where they are all

template <int CTAS>
size_t plan_smem(int N) {
    return sizeof(int32_t) * ((size_t)kPlanWarps * (N | 1) + (size_t)N * (CTAS + 4));
}

template <int CTAS>
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const int32_t* ids, int T, int N, const LoraPlan p) {
    extern __shared__ int32_t plan_raw[];
    const int pitch = N | 1;                  // an adapter's counters of all warps lie on different banks
    int32_t* mine = plan_raw;                 // [warps][pitch] a warp's rows per adapter, then where its next one goes
    int32_t* all = mine + kPlanWarps * pitch; // [CTAs][N] a CTA's rows per adapter
    int32_t* total = all + CTAS * N;          // [N] rows
    int32_t* block = total + N;               // [N] first block
    int32_t* start = block + N;               // [N] slot of this CTA's first row
    int32_t* group = start + N;               // [N] first group
    __shared__ int sums[3][kPlanWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)blockIdx.x;
    for (int i = tid; i < kPlanWarps * pitch; i += kPlanThreads) mine[i] = 0;
    if (CTAS > 1) cluster_arrive();
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    const long per = (((long)T + CTAS * kPlanWarps - 1) / (CTAS * kPlanWarps) + 31) / 32 * 32;
    const int gw = rank * kPlanWarps + warp;
    const long lo = min((long)T, gw * per), hi = min((long)T, lo + per);
    int32_t* wm = mine + warp * pitch;
    int v[kPlanAhead];
    auto load = [&](long t0) {
#pragma unroll
        for (int q = 0; q < kPlanAhead; ++q) {
            const long t = t0 + q * 32 + lane;
            v[q] = t < hi ? ids[t] : -1;
        }
    };
    for (long t0 = lo; t0 < hi; t0 += 32 * kPlanAhead) {
        load(t0);
#pragma unroll
        for (int q = 0; q < kPlanAhead; ++q)
            if ((unsigned)v[q] < (unsigned)N) atomicAdd(&wm[v[q]], 1);
    }
    __syncthreads();
    if (CTAS > 1) cluster_wait();  // every CTA runs: its shared memory may be written
    // an adapter's counts over the 32 warps, a thread for each adapter
    if (tid < N) {
        int own[kPlanWarps], s = 0;
#pragma unroll
        for (int w = 0; w < kPlanWarps; ++w) own[w] = mine[w * pitch + tid];
#pragma unroll
        for (int w = 0; w < kPlanWarps; ++w) {
            mine[w * pitch + tid] = s;
            s += own[w];
        }
        if (CTAS == 1) {
            all[tid] = s;
        } else {
#pragma unroll
            for (int q = 0; q < CTAS; ++q)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(smem_u32(all + rank * N + tid), q)), "r"(s)
                             : "memory");
        }
    }
    if (CTAS == 1) __syncthreads();
    if (CTAS > 1) {
        cluster_arrive();
        cluster_wait();
    }
    // prefix sums over the adapters of their blocks and units, a thread per adapter
    int c = 0, before = 0;
    if (tid < N) {
#pragma unroll
        for (int q = 0; q < CTAS; ++q) {
            if (q == rank) before = c;
            c += all[q * N + tid];
        }
        total[tid] = c;
    }
    const int blocks = (c + kLoraTile - 1) / kLoraTile;
    const int units = c > 0 ? (c + kLoraStepRows - 1) / kLoraStepRows + kLoraTileUnits : 0;
    const int groups = (c + kLoraGroupRows - 1) / kLoraGroupRows;
    int pb = blocks, pu = units, pg = groups;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int ub = __shfl_up_sync(0xffffffffu, pb, o), uu = __shfl_up_sync(0xffffffffu, pu, o),
                  ug = __shfl_up_sync(0xffffffffu, pg, o);
        if (lane >= o) pb += ub, pu += uu, pg += ug;
    }
    if (lane == 31) sums[0][warp] = pb, sums[1][warp] = pu, sums[2][warp] = pg;
    __syncthreads();
    int wb = sums[0][lane], wu = sums[1][lane], wg = sums[2][lane];  // of warp `lane` (32 warps)
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int ub = __shfl_up_sync(0xffffffffu, wb, o), uu = __shfl_up_sync(0xffffffffu, wu, o),
                  ug = __shfl_up_sync(0xffffffffu, wg, o);
        if (lane >= o) wb += ub, wu += uu, wg += ug;
    }
    const int allb = __shfl_sync(0xffffffffu, wb, 31), allu = __shfl_sync(0xffffffffu, wu, 31),
              allg = __shfl_sync(0xffffffffu, wg, 31);
    pb += __shfl_sync(0xffffffffu, wb - sums[0][lane], warp) - blocks;
    pu += __shfl_sync(0xffffffffu, wu - sums[1][lane], warp) - units;
    pg += __shfl_sync(0xffffffffu, wg - sums[2][lane], warp) - groups;
    if (tid < N) {
        block[tid] = pb;
        group[tid] = pg;
        start[tid] = pb * kLoraTile + before;
        if (rank == 0) p.first[tid] = p.grouped ? pg : pb, p.units[tid] = p.grouped ? c : pu;
    }
    if (rank == 0 && tid == 0) {
        p.first[N] = allb;
        p.units[N] = allu;
        *p.nblocks = allb;
        *p.ngroups = allg;
    }
    if (rank == 0 && tid < 4) p.status[tid] = 0;
    __syncthreads();
    for (long t0 = lo; t0 < hi; t0 += 32 * kPlanAhead) {
        if (per > 32 * kPlanAhead) load(t0);  // else they are still here
#pragma unroll
        for (int q = 0; q < kPlanAhead; ++q) {  // 32 rows in order
            if (t0 + q * 32 >= hi) break;
            const int n = v[q];
            const bool ok = (unsigned)n < (unsigned)N;
            const uint32_t peers = __match_any_sync(0xffffffffu, ok ? n : -1 - lane);
            const int before = __popc(peers & ((1u << lane) - 1u));
            int at = 0;
            if (ok) at = wm[n];
            __syncwarp();  // all of an adapter's lanes have read its counter before the first of them moves it on
            if (ok && before == 0) wm[n] = at + __popc(peers);
            if (ok) p.rows[start[n] + at + before] = (int32_t)(t0 + q * 32 + lane);
            __syncwarp();
        }
    }
    // each adapter's groups, or its blocks and the slots behind its last row: a share of all threads for each, of 32 and more
    // where they write whole blocks
    const int mate = rank * kPlanThreads + tid, threads = CTAS * kPlanThreads;
    if (p.grouped) {
        const int share = threads / N;
        const int n = mate / share;
        if (n >= N) return;
        for (int i = mate % share, rows = total[n]; i * kLoraGroupRows < rows; i += share)
            p.groups[group[n] + i] =
                make_int2(block[n] * kLoraTile + i * kLoraGroupRows, n << 8 | min(kLoraGroupRows, rows - i * kLoraGroupRows));
        return;
    }
    const int share = max(threads / N, 32);
    for (int n = mate / share; n < N; n += threads / share) {
        const int rows = total[n], b0 = block[n], nb = (rows + kLoraTile - 1) / kLoraTile;
        for (int i = mate % share; i < nb; i += share) p.adapter[b0 + i] = n;
        for (int i = rows + mate % share; i < nb * kLoraTile; i += share) p.rows[b0 * kLoraTile + i] = -1;
    }
}

// ------------------------------------------------------------------------------------------- entry points
bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A matrix of rows: 16-byte aligned, and so is each row.
bool rows_ok(const void* p, int64_t ld, int T, int width, bool written) {
    return a16(p) && ld % 8 == 0 && (T <= 1 || ld >= width || (ld >= 0 && !written));
}

// A result on top of base has base's row distance, and no result is on top of u or v.
bool apart(const void* out, int64_t ldout, const void* base, int64_t ldbase, int T, const void* u, const void* v) {
    return out != u && out != v && (out != base || ldout == ldbase || T <= 1);
}

int check_lora(int T, int K, int O, int R, int N) {
    if (T < 0 || K <= 0 || O <= 0 || R <= 0 || N <= 0) return PM_ERR_INVALID;
    if (K % 8 || O % 8 || R % 8 || R > kLoraMaxRank || N > kLoraMaxAdapters || T > kLoraMaxRows || K > kLoraMaxWidth ||
        O > kLoraMaxWidth)
        return PM_ERR_SHAPE;
    return PM_OK;
}

// The plan and what the tiled kernels need, carved from `base` (null: sizes only).
struct Carved {
    LoraPlan plan;
    bf16 *h, *d;
    float* partial;
    void* frags;
    size_t bytes;
};
Carved carve(void* base, int T, int N, int R, bool grad) {
    uint8_t* p = static_cast<uint8_t*>(base);
    size_t off = 0;
    auto take = [&](size_t n) {
        uint8_t* at = p == nullptr ? nullptr : p + off;
        off = (off + n + 255) / 256 * 256;
        return at;
    };
    const size_t blocks = lora_max_blocks(T, N), hidden = blocks * kLoraTile * 2 * lora_rp(R) * sizeof(bf16);
    Carved c;
    c.plan.status = (int32_t*)take(16);  // the workspace's first word, as pm_moe_read_status reads it
    c.plan.grouped = grad ? lora_grad_is_grouped(T, R, N) : lora_fused(T, R, N);
    c.plan.nblocks = (int32_t*)take(4);
    c.plan.ngroups = (int32_t*)take(4);
    c.plan.groups = c.plan.grouped ? (int2*)take((size_t)lora_max_groups(T, N) * sizeof(int2)) : nullptr;
    c.plan.units = (int32_t*)take(((size_t)N + 1) * 4);
    c.plan.first = (int32_t*)take(((size_t)N + 1) * 4);
    c.plan.adapter = (int32_t*)take(blocks * 4);
    c.plan.rows = (int32_t*)take(blocks * kLoraTile * 4);
    c.h = c.plan.grouped ? nullptr : (bf16*)take(hidden);
    c.frags = grad && c.plan.grouped ? take(lora_frag_bytes(T, N)) : nullptr;
    c.d = grad && !c.plan.grouped ? (bf16*)take(hidden) : nullptr;
    c.partial = grad && !c.plan.grouped ? (float*)take(lora_partial_bytes(R)) : nullptr;
    c.bytes = off;
    return c;
}

int status_of(cudaError_t e) { return e == cudaSuccess ? PM_OK : PM_ERR_CUDA; }

}  // namespace

cudaError_t raise_smem(const void* kernel, size_t bytes, std::atomic<bool>* configured) {
    int dev = 0;
    PM_TRY(cudaGetDevice(&dev));
    if (dev < 64 && configured[dev].load(std::memory_order_acquire)) return cudaSuccess;
    PM_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (dev < 64) configured[dev].store(true, std::memory_order_release);
    return cudaSuccess;
}

cudaError_t launch_lora_plan(const int32_t* adapter, int T, int N, const LoraPlan& p, cudaStream_t s) {
    static std::atomic<bool> configured[2][64];
    if (T <= kPlanOneCta) {
        PM_TRY(raise_smem((const void*)lora_plan_kernel<1>, plan_smem<1>(kLoraMaxAdapters), configured[0]));
        return launch_pdl(lora_plan_kernel<1>, dim3(1), dim3(kPlanThreads), plan_smem<1>(N), s, adapter, T, N, p);
    }
    PM_TRY(raise_smem((const void*)lora_plan_kernel<kPlanCtas>, plan_smem<kPlanCtas>(kLoraMaxAdapters), configured[1]));
    return launch_cluster(lora_plan_kernel<kPlanCtas>, dim3(kPlanCtas), dim3(kPlanThreads), kPlanCtas,
                          plan_smem<kPlanCtas>(N), s, adapter, T, N, p);
}

}  // namespace pm

using namespace pm;

extern "C" {

size_t pm_lora_workspace_bytes(int T, int K, int O, int R, int N, int grad) {
    if (check_lora(T, K, O, R, N) != PM_OK) return 0;
    if (grad ? lora_grad_is_few(T, R, N) : T <= kLoraFewRows) return 0;
    return carve(nullptr, T, N, R, grad != 0).bytes;
}

int pm_lora(const void* x, int64_t ldx, const void* a, const void* b, const int32_t* adapter, const float* scale,
            const void* base, int64_t ldbase, void* out, int64_t ldout, int T, int K, int O, int R, int N, void* workspace,
            size_t workspace_bytes, pm_stream_t stream) {
    int st = check_lora(T, K, O, R, N);
    if (st != PM_OK) return st;
    if (T == 0) return PM_OK;
    if (!x || !a || !b || !adapter || !out || (T > kLoraFewRows && !workspace)) return PM_ERR_INVALID;
    if (!a16(a) || !a16(b) || !rows_ok(x, ldx, T, K, false) || !rows_ok(out, ldout, T, O, true) ||
        (base && !rows_ok(base, ldbase, T, O, false)) || (T > kLoraFewRows && !a16(workspace)))
        return PM_ERR_ALIGN;
    if (workspace_bytes < pm_lora_workspace_bytes(T, K, O, R, N, 0)) return PM_ERR_WORKSPACE;
    if (!apart(out, ldout, base, ldbase, T, x, x)) return PM_ERR_INVALID;
    int sms = 0;
    if ((st = device_sms(&sms)) != PM_OK) return st;
    cudaStream_t s = (cudaStream_t)stream;
    if (T <= kLoraFewRows) {
        const FewArgs f{(const bf16*)x, ldx, (const bf16*)a, (const bf16*)b, adapter, scale, (const bf16*)base, ldbase,
                        (bf16*)out, ldout, T, K, O, R, N, nullptr, nullptr, nullptr};
        return status_of(launch_fused<false, 8>(f, T, s));
    }
    const LoraShape g{T, K, O, R, N};
    const Carved w = carve(workspace, T, N, R, false);
    cudaError_t e = launch_lora_plan(adapter, T, N, w.plan, s);
    if (w.plan.grouped) {
        const FewArgs f{(const bf16*)x, ldx, (const bf16*)a, (const bf16*)b, adapter, scale, (const bf16*)base, ldbase,
                        (bf16*)out, ldout, T, K, O, R, N, w.plan.ngroups, w.plan.groups, w.plan.rows};
        if (e == cudaSuccess) e = launch_groups(f, sms, s);
        return status_of(e);
    }
    const LoraDown down{(const bf16*)x, ldx, (const bf16*)a, K, true, w.h};
    if (e == cudaSuccess) e = launch_lora_down(&down, 1, scale, w.plan, g, sms, s);
    const LoraUp up{w.h, (const bf16*)b, O, false, (const bf16*)base, ldbase, (bf16*)out, ldout, nullptr};
    if (e == cudaSuccess) e = launch_lora_up(up, adapter, w.plan, g, sms, s);
    return status_of(e);
}

int pm_lora_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* a, const void* b,
                 const int32_t* adapter, const float* scale, const void* base, int64_t ldbase, void* dx, int64_t lddx,
                 void* da, void* db, int T, int K, int O, int R, int N, void* workspace, size_t workspace_bytes,
                 pm_stream_t stream) {
    int st = check_lora(T, K, O, R, N);
    if (st != PM_OK) return st;
    const bool few = lora_grad_is_few(T, R, N);
    if (!da || !db || (!few && !workspace) || (T > 0 && (!dy || !x || !a || !b || !adapter || !dx))) return PM_ERR_INVALID;
    if (!a16(a) || !a16(b) || !a16(da) || !a16(db) || (!few && !a16(workspace))) return PM_ERR_ALIGN;
    if (T > 0 && (!rows_ok(dy, lddy, T, O, false) || !rows_ok(x, ldx, T, K, false) || !rows_ok(dx, lddx, T, K, true) ||
                  (base && !rows_ok(base, ldbase, T, K, false))))
        return PM_ERR_ALIGN;
    if (workspace_bytes < pm_lora_workspace_bytes(T, K, O, R, N, 1)) return PM_ERR_WORKSPACE;
    if (T > 0 && !apart(dx, lddx, base, ldbase, T, x, dy)) return PM_ERR_INVALID;
    int sms = 0;
    if ((st = device_sms(&sms)) != PM_OK) return st;
    cudaStream_t s = (cudaStream_t)stream;
    const LoraShape g{T, K, O, R, N};
    if (T == 0) {
        cudaError_t e = cudaMemsetAsync(da, 0, (size_t)N * R * K * 2, s);
        if (e == cudaSuccess) e = cudaMemsetAsync(db, 0, (size_t)N * R * O * 2, s);
        if (e == cudaSuccess && !few) e = cudaMemsetAsync(workspace, 0, 16, s);  // the status
        return status_of(e);
    }
    const LoraGradFew f{(const bf16*)dy, (const bf16*)x, (const bf16*)a, (const bf16*)b, lddy, ldx, adapter, scale,
                        (const bf16*)base, ldbase, (bf16*)dx, lddx, (bf16*)da, (bf16*)db};
    if (few) return status_of(launch_lora_grad_few(f, g, sms, s));
    const Carved w = carve(workspace, T, N, R, true);
    cudaError_t e = launch_lora_plan(adapter, T, N, w.plan, s);
    if (w.plan.grouped) {
        if (e == cudaSuccess) e = launch_lora_grad_groups(f, g, w.plan, w.frags, sms, s);
        return status_of(e);
    }
    LoraDown down[2] = {{(const bf16*)x, ldx, (const bf16*)a, K, true, w.h},
                        {(const bf16*)dy, lddy, (const bf16*)b, O, false, w.d}};
    if (O > K) std::swap(down[0], down[1]);  // the longer CTAs start first
    if (e == cudaSuccess) e = launch_lora_down(down, 2, scale, w.plan, g, sms, s);
    // the weights' gradients next: they read x and dy again, which the L2 cache still has in part
    const LoraOuter outer{(const bf16*)x, (const bf16*)dy, ldx, lddy, w.h, w.d, (bf16*)da, (bf16*)db, w.partial};
    if (e == cudaSuccess) e = launch_lora_outer(outer, w.plan, g, sms, s);
    const LoraUp up{w.d, (const bf16*)a, K, true, (const bf16*)base, ldbase, (bf16*)dx, lddx, &outer};
    if (e == cudaSuccess) e = launch_lora_up(up, adapter, w.plan, g, sms, s);
    return status_of(e);
}

}  // extern "C"
