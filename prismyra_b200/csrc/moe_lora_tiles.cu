// The tiled adapter kernels: rows sorted by adapter (moe_lora.cu's plan) in blocks of 128, products on tcgen05.
//
//   down   h = scale * (x a^T): a block's rows are the MMA's 128-row operand. Where there are few blocks a cluster of CTAs
//          shares one, each with a part of the width, and the sums meet in shared memory. (Left in global memory for the
//          last CTA to add up they took 5 us longer at 5120 rows; the weights as the 128-row operand and 32 rows of x as
//          columns needed no sharing but was slower too: an MMA takes its 128 rows' time however few columns it has.)
//          The R values of a row are kept as two bf16 halves (hi + lo, 16 significant bits)
//   up     out = base + h b^T: the halves' products with the same weights, accumulated in fp32
//   outer  da, db = sum over an adapter's rows: the rows are the MMA's contraction, both operands "MN-major"
// Rows are gathered with 16-byte cp.async into the 128-byte-swizzled layout that TMA would write (row r, 16-byte piece c
// at r * 128 + ((c ^ (r & 7)) << 4)), so any order of adapters costs the same; weights and hidden rows come by TMA
// through three-dimensional maps, whose bounds keep one adapter's tile off its neighbour's weights.
//
// Programmatic launches: every CTA of these kernels waits for its predecessor (pdl_wait) before it lets its successor
// start (pdl_trigger), so what the launch before the predecessor wrote is complete when a kernel starts and may be read
// before its own wait: outer and up read the plan and their inputs so, and up after outer the hidden rows too (it does not
// depend on outer, and takes its SMs over as they become free). Such reads pass L1 by (ld.cg, cp.async.cg, TMA). Every CTA
// waits before it ends all the same, which keeps completion transitive.
#include <string.h>

#include <atomic>

#include "lora_dev.cuh"
#include "moe_lora.h"

namespace pm {
namespace {

// Shared-memory operand descriptors (desc_kmajor_sw128 in ptx.cuh) in halves: the upper word is the same for all operands
// here, and the lower one moves with the address, so a step costs the issuing thread one 32-bit add per operand. K-major:
// rows of 128 bytes of the contraction. MN-major: the contraction index is the row of 128 bytes (64 values of the other
// index), 8-row atoms of 1024 bytes, further 64-value blocks block_bytes apart (leading byte offset).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t kmajor(uint32_t smem_addr) { return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t mnmajor(uint32_t smem_addr, uint32_t block_bytes) {
    return ((smem_addr & 0x3FFFFu) >> 4) | ((block_bytes >> 4) << 16);
}
__device__ __forceinline__ void mma_desc(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "n"(kDescHi)
        : "memory");
}
constexpr uint32_t kMajorA = 1u << 15, kMajorB = 1u << 16;  // instruction descriptor: operand is MN-major

__device__ __forceinline__ uint32_t tmem_cols(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512; }

__device__ __forceinline__ int align1024(uint32_t a) { return (int)((1024u - (a & 1023u)) & 1023u); }

// Where part i of G of a line of n starts.
__device__ __forceinline__ unsigned part_start(unsigned n, unsigned i, unsigned G) { return n / G * i + min(i, n % G); }

// ------------------------------------------------------------------------------------------- down
// Warps 0-3 copy the block's rows in and signal each stage themselves, warp 5 brings the weights, warp 4 multiplies: 64 columns
// a step, about 400 cycles of the issuing thread, 16 KB of rows. Long batches wait for the rows, at 3.9 to 4.1 TB/s, short of what
// this memory gives (the up kernel reads and writes 5.3 TB/s): 26 us for 100 MB (8192 rows, widths 2048 and 4096; 16 us where x
// comes from L2), 33 us for 134 MB. Neither the weights nor the MMAs hold it up; that the CTAs are unlike in bytes and one or two to
// an SM, and that a step takes 128 bytes of rows 4 to 8 KB apart, are likely and not measured apart. Where rows are few, latency: 12
// us at 5120 rows of 2048, R = 64, 10 MB of weights and 21 MB of rows.
constexpr int kDownMaxStages = 12;
constexpr int kDownThreads = 192;    // warps 0-3: rows in, sums out; warp 4: MMA; warp 5: weights by TMA
constexpr int kDownXBytes = kLoraTile * 128;  // 64 columns of the width per stage

struct DownPart {
    const bf16* src;
    long ld;
    int width;
    int by_rank;
    bf16* out;
};
struct DownArgs {
    DownPart part[2];
    const float* scale;
    const int32_t* nblocks;
    const int32_t* adapter;
    const int32_t* rows;
    int* err;
    int R;
    int wbytes;  // shared memory of one stage's weights
    int stages;
};
struct DownTail {
    uint64_t full[kDownMaxStages];
    uint64_t empty[kDownMaxStages];
    uint64_t done;
    uint32_t tmem_base;
    int abort;
    uint32_t have[4];  // which of the block's rows there are
};

inline int down_wbytes(int R, bool by_rank) { return by_rank ? lora_rp(R) * 128 : (lora_rp(R) + 63) / 64 * 8192; }
// As many stages as leave room for `resident` CTAs on an SM.
inline int down_stages(int wbytes, int resident) {
    return std::min(kDownMaxStages, (resident == 1 ? 208 << 10 : 108 << 10) / (kDownXBytes + wbytes));
}
// A cluster's sums, 128 rows of Rp + 4 fp32, take the ring's place.
inline size_t down_smem(int R, int wbytes, int stages) {
    return 1024 + std::max((size_t)stages * (kDownXBytes + wbytes), (size_t)kLoraTile * (lora_rp(R) + 4) * 4) + sizeof(DownTail);
}

__global__ void __launch_bounds__(kDownThreads)
    lora_down_kernel(const __grid_constant__ CUtensorMap tm_w0, const __grid_constant__ CUtensorMap tm_w1, const DownArgs g) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + align1024(smem_u32(smem_raw));
    const uint32_t sbase = smem_u32(smem);
    const int stage_bytes = kDownXBytes + g.wbytes, stages = g.stages;
    const int Rp = lora_rp(g.R);
    const int ldr = Rp + 4;  // floats from one received row to the next: 16-byte pieces of 8 rows on different banks
    float* recv = reinterpret_cast<float*>(smem);  // [splits][128 / splits][ldr], once the ring has been read
    DownTail* tail = reinterpret_cast<DownTail*>(smem + max(stages * stage_bytes, kLoraTile * ldr * 4));
    volatile int* abort = &tail->abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t splits, rank;
    asm("mov.u32 %0, %cluster_nctaid.x;" : "=r"(splits));
    asm("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
    const int block = (int)(blockIdx.x / splits);
    const DownPart part = blockIdx.y == 0 ? g.part[0] : g.part[1];
    const CUtensorMap* tm_w = blockIdx.y == 0 ? &tm_w0 : &tm_w1;
    const uint32_t cols = tmem_cols(Rp);

    if (tid == 0) {
        for (int st = 0; st < stages; ++st) {
            mbar_init(smem_u32(&tail->full[st]), 128 + 1);  // copying threads, TMA
            mbar_init(smem_u32(&tail->empty[st]), 1);
        }
        mbar_init(smem_u32(&tail->done), 1);
        tail->abort = 0;
        fence_barrier_init();
        fence_proxy_async_smem();
        prefetch_tensormap(tm_w);
    }
    if (warp == 4) {
        tmem_alloc(smem_u32(&tail->tmem_base), cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tail->tmem_base;
    const int all = (part.width + 63) / 64;
    const int lo = (int)part_start(all, rank, splits), steps = (int)part_start(all, rank + 1, splits) - lo;
    pdl_wait();
    pdl_trigger();
    // asked for together; without meaning (but within the plan) where the block is none
    const int c = tid & 7, r0 = (tid >> 3) & 15;  // piece, and first of eight rows 16 apart, of the copies
    int row[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) row[i] = g.rows[block * kLoraTile + r0 + 16 * i];
    const int own = warp < 4 ? g.rows[block * kLoraTile + tid] : -1;
    const int n = g.adapter[block];
    const bool live = block < *g.nblocks;  // the same for the whole cluster

    if (live) {
        const float sc = g.scale != nullptr ? g.scale[n] : 1.0f;
        if (warp < 4) {
            const bf16* p[8];
            uint32_t ok = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = part.src + (row[i] < 0 ? 0L : (long)row[i] * part.ld) + lo * 64 + c * 8;
                ok |= (row[i] < 0 ? 0u : 1u) << i;
            }
            const uint32_t dst = sbase + r0 * 128 + ((c ^ (r0 & 7)) << 4);  // r0 + 16 i has the same low bits
            const uint32_t h = __ballot_sync(0xffffffffu, own >= 0);
            if (lane == 0) tail->have[warp] = h;
            int st = 0;
            uint32_t phase = 1;
            for (int s = 0; s < steps; ++s) {
                if (s >= stages) mbar_wait(smem_u32(&tail->empty[st]), phase, abort);
                const bool in = (lo + s) * 64 + c * 8 < part.width;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool v = in && ((ok >> i) & 1u);
                    cp_async16(dst + st * stage_bytes + i * 2048, v ? p[i] + s * 64 : part.src, v);
                }
                cp_async_arrive(smem_u32(&tail->full[st]));
                if (++st == stages) { st = 0; phase ^= 1u; }
            }
            cp_async_commit();
            cp_async_wait<0>();
        } else if (warp == 5) {
            if (lane == 0) {
                const int boxes = (Rp + 63) / 64;
                const uint32_t bytes = part.by_rank ? Rp * 128 : boxes * 8192;
                int st = 0;
                uint32_t phase = 1;
                for (int s = 0; s < steps; ++s) {
                    if (s >= stages && !mbar_wait(smem_u32(&tail->empty[st]), phase, abort)) break;
                    const uint32_t w = sbase + st * stage_bytes + kDownXBytes, fb = smem_u32(&tail->full[st]);
                    const int col = (lo + s) * 64;
                    mbar_arrive_expect_tx(fb, bytes);
                    if (part.by_rank)
                        tma_load_3d(w, tm_w, fb, col, 0, n);
                    else
                        for (int q = 0; q < boxes; ++q) tma_load_3d(w + q * 8192, tm_w, fb, q * 64, col, n);
                    if (++st == stages) { st = 0; phase ^= 1u; }
                }
            }
        } else if (lane == 0) {
            const uint32_t idesc = idesc_f32acc(1, 1, kLoraTile, Rp) | (part.by_rank ? 0u : kMajorB);
            const uint32_t wstep = part.by_rank ? 2 : 128;  // 16 of the width: 32 bytes, or 16 rows of 128
            const uint32_t dx0 = kmajor(sbase);
            const uint32_t dw0 = part.by_rank ? kmajor(sbase + kDownXBytes) : mnmajor(sbase + kDownXBytes, 8192);
            int st = 0;
            uint32_t phase = 0;
            for (int s = 0; s < steps; ++s) {
                if (!mbar_wait(smem_u32(&tail->full[st]), phase, abort)) break;
                fence_proxy_async_smem();  // the copied rows, for the tensor core
                tc_fence_after();
                const uint32_t dx = dx0 + st * (stage_bytes >> 4), dw = dw0 + st * (stage_bytes >> 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) mma_desc(tmem, dx + 2 * j, dw + wstep * j, idesc, s > 0 || j > 0);
                mma_commit(smem_u32(&tail->empty[st]));
                if (++st == stages) { st = 0; phase ^= 1u; }
            }
            mma_commit(smem_u32(&tail->done));
        }
        __syncwarp();
        mbar_wait(smem_u32(&tail->done), 0, abort);
        tc_fence_after();
        bf16* out = part.out + (long)block * kLoraTile * 2 * Rp;
        const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
        if (splits == 1) {
            if (warp < 4) {  // a thread per row
                for (int q = 0; q < Rp; q += 16) {
                    uint32_t r[16];
                    tmem_ld16(mine + q, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        float v[8];  // not the padding: 0, whatever the row or the weights hold
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = own >= 0 && q + e < g.R ? __uint_as_float(r[e + k]) * sc : 0.0f;
                        uint4 hi, lw;
                        split8(v, &hi, &lw);
                        *reinterpret_cast<uint4*>(out + (long)tid * 2 * Rp + q + e) = hi;
                        *reinterpret_cast<uint4*>(out + (long)tid * 2 * Rp + Rp + q + e) = lw;
                    }
                }
                tc_fence_before();
            }
        } else {
            // all products done in the whole cluster: the rings may be written
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            // sums out: the row of this thread, over its part of the width, to the CTA that adds that row up
            const int per = kLoraTile / (int)splits;
            if (warp < 4) {
                const uint32_t dst = cluster_addr(smem_u32(recv + ((int)rank * per + tid % per) * ldr), (uint32_t)(tid / per));
                for (int q = 0; q < Rp; q += 32) {  // the columns past Rp of the last 32 are allocated, and not sent
                    uint32_t r[32];
                    tmem_ld32(mine + q, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        if (q + i < Rp)  // a narrow part may have no steps for this CTA
                            st_cluster(dst + (q + i) * 4, steps > 0 ? __uint_as_float(r[i]) : 0.0f,
                                       steps > 0 ? __uint_as_float(r[i + 1]) : 0.0f, steps > 0 ? __uint_as_float(r[i + 2]) : 0.0f,
                                       steps > 0 ? __uint_as_float(r[i + 3]) : 0.0f);
                }
                tc_fence_before();
            }
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            // the rows this CTA adds up, the splits in order, 8 columns a thread at a time
            const int groups = Rp / 8;
            const uint32_t inv = 65536u / groups + 1u;  // i / groups = i inv >> 16 for i < 2048
            for (int i = tid; i < per * groups; i += kDownThreads) {
                const int r = (int)(i * inv >> 16), q = (i - r * groups) * 8, at = (int)rank * per + r;
                const bool keep = q < g.R && ((tail->have[at >> 5] >> (at & 31)) & 1u);
                float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                for (int s = 0; s < (int)splits; ++s) {
                    const float4 a = *reinterpret_cast<const float4*>(recv + (s * per + r) * ldr + q);
                    const float4 b = *reinterpret_cast<const float4*>(recv + (s * per + r) * ldr + q + 4);
                    v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
                    v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = keep ? v[k] * sc : 0.0f;
                uint4 hi, lw;
                split8(v, &hi, &lw);
                *reinterpret_cast<uint4*>(out + (long)at * 2 * Rp + q) = hi;
                *reinterpret_cast<uint4*>(out + (long)at * 2 * Rp + Rp + q) = lw;
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        tmem_dealloc(tmem, cols);
    }
    if (tid == 0 && tail->abort) atomicExch(g.err, 1);
}

// ------------------------------------------------------------------------------------------- outer
// Tiles of 256 columns x R ranks, 64 rows a step: both operands have the row (the contraction) as their row in shared memory,
// so x and dy are read as they lie. hi and lo are neighbours in a hidden row, one MMA of 2 Rp columns makes both sums.
// Bound by what comes into an SM: 48 KB a step at R = 64, of which 16 KB are hidden rows from L2; 100 MB of x and dy in
// 12.7 us (8192 rows, R = 16, mostly from L2), 134 MB in 23.5 us (16384 rows, R = 64).
constexpr int kOuterThreads = 320;  // warps 0-3: rows in; 4-7: results out; 8: MMA; 9: TMA
constexpr int kOuterXBytes = kLoraStepRows * kLoraCols * 2;

struct OuterArgs {
    const bf16 *x, *dy;
    long ldx, lddy;
    bf16 *da, *db;
    float* partial;  // [CTAs][2][Rp][kLoraCols]
    const int32_t* units;
    const int32_t* first;
    const int32_t* rows;
    int* err;
    int K, O, R, N;
    int tiles_a, tiles_b;
    int stages, gbytes;
};
constexpr int kOuterMaxStages = 4;
struct OuterTail {
    uint64_t full[kOuterMaxStages];
    uint64_t empty[kOuterMaxStages];
    uint64_t afull[2];
    uint64_t aempty[2];
    uint32_t tmem_base;
    int abort;
};
inline int outer_gbytes(int R) { return (2 * lora_rp(R) + 63) / 64 * 8192; }
inline int outer_stages(int R) { return lora_rp(R) <= 64 ? 4 : 3; }
inline size_t outer_smem(int R, int N) {
    return 1024 + (size_t)outer_stages(R) * (kOuterXBytes + outer_gbytes(R)) + sizeof(OuterTail) + ((size_t)N + 1) * 8;
}

// The work is a line of units: adapter by adapter, its column tiles (da's, then db's), a tile's rows 64 at a time and then
// kLoraTileUnits for writing it (without these, adapters of a few rows made some CTAs take 10 us longer than the rest at
// 16384 rows and 16 adapters). It is cut into as many equal parts as there are CTAs (units at most). A tile that one CTA does
// whole is written by it; otherwise each leaves a partial sum, and the up kernel's spare warps add them in order.
struct Walk {
    const int32_t* units;  // [N + 1]
    int N, tiles;
    unsigned left;         // units of this CTA's part from here on
    int n, tile, total, at;  // the tile's steps, and where in it (past its steps: in the writing)
    int step, len;         // the segment: steps [step, step + len) of the tile's total
    __device__ __forceinline__ void start(unsigned s) {
        int a = 0, b = N;  // the adapter with units[n] * tiles <= s < units[n + 1] * tiles
        while (b - a > 1) {
            const int m = (a + b) >> 1;
            if ((unsigned)units[m] * tiles <= s)
                a = m;
            else
                b = m;
        }
        n = a;
        const unsigned each = units[a + 1] - units[a], local = s - (unsigned)units[a] * tiles;
        total = (int)each - kLoraTileUnits;
        tile = (int)(local / each);
        at = (int)(local % each);
    }
    // The next segment of this CTA, or false. Until the next call n and tile are its.
    __device__ __forceinline__ bool next() {
        while (left > 0) {
            if (at < total) {
                step = at;
                len = (int)min((unsigned)(total - at), left);
                at += len;
                left -= len;
                return true;
            }
            const unsigned skip = min((unsigned)(total + kLoraTileUnits - at), left);
            at += (int)skip;
            left -= skip;
            if (at < total + kLoraTileUnits) break;
            at = 0;
            if (++tile < tiles) continue;
            tile = 0;
            do ++n;
            while (n < N && units[n + 1] == units[n]);
            if (n < N) total = units[n + 1] - units[n] - kLoraTileUnits;
        }
        return false;
    }
};

// Ranks r0 .. r0 + 7 of one column's sums, to da [R][K] or db [O][R].
__device__ __forceinline__ void store_ranks(const OuterArgs& g, bool is_a, int n, int col, int r0, const float (&v)[8]) {
    if (is_a) {
        if (col >= g.K) return;
        bf16* p = g.da + ((long)n * g.R + r0) * g.K + col;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[(long)i * g.K] = __float2bfloat16_rn(v[i]);
    } else {
        if (col >= g.O) return;
        uint4 o;
        __nv_bfloat162* b = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4*>(g.db + ((long)n * g.O + col) * g.R + r0) = o;
    }
}

__global__ void __launch_bounds__(kOuterThreads, 1)
    lora_outer_kernel(const __grid_constant__ CUtensorMap tm_h, const __grid_constant__ CUtensorMap tm_d, const OuterArgs g) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + align1024(smem_u32(smem_raw));
    const uint32_t sbase = smem_u32(smem);
    const int stage_bytes = kOuterXBytes + g.gbytes;
    OuterTail* tail = reinterpret_cast<OuterTail*>(smem + g.stages * stage_bytes);
    int32_t* units = reinterpret_cast<int32_t*>(tail + 1);  // [N + 1]
    int32_t* first = units + g.N + 1;                       // [N + 1]
    volatile int* abort = &tail->abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int Rp = lora_rp(g.R);
    const int bufs = Rp <= 64 ? 2 : 1;          // accumulators of two 128-column halves x 2 Rp columns each
    const uint32_t cols = tmem_cols(bufs * 4 * Rp);

    for (int i = tid; i <= g.N; i += kOuterThreads) {
        units[i] = __ldcg(g.units + i);
        first[i] = __ldcg(g.first + i);
    }
    if (tid == 0) {
        for (int st = 0; st < kOuterMaxStages; ++st) {
            mbar_init(smem_u32(&tail->full[st]), 128 + 1);  // copying threads, TMA
            mbar_init(smem_u32(&tail->empty[st]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&tail->afull[b]), 1);
            mbar_init(smem_u32(&tail->aempty[b]), 4);
        }
        tail->abort = 0;
        fence_barrier_init();
        fence_proxy_async_smem();
        prefetch_tensormap(&tm_h);
        prefetch_tensormap(&tm_d);
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(&tail->tmem_base), cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tail->tmem_base;
    const int tiles = g.tiles_a + g.tiles_b;
    const unsigned total = (unsigned)units[g.N] * tiles, parts = max(1u, min(gridDim.x, total));
    Walk walk{units, g.N, tiles, 0u, 0, 0, 0, 0, 0, 0};
    if (blockIdx.x < parts && total > 0) {
        const unsigned s0 = part_start(total, blockIdx.x, parts);
        walk.left = part_start(total, blockIdx.x + 1, parts) - s0;
        walk.start(s0);
    }

    if (warp < 4) {
        // rows in: a step's 64 rows x 256 columns as four 64-column blocks of [64][128 bytes]; this thread: piece c of
        // rows r0, r0 + 16, r0 + 32, r0 + 48 in each block. The rows' numbers are asked for a step ahead.
        const int c = tid & 7, r0 = tid >> 3;
        const uint32_t dst = sbase + r0 * 128 + ((c ^ (r0 & 7)) << 4);
        int st = 0;
        uint32_t phase = 1;
        int row[4];
        bool have = walk.next();
        int q = 0;  // of the segment
        auto ask = [&]() {
            const int32_t* p = g.rows + (long)first[walk.n] * kLoraTile + (walk.step + q) * kLoraStepRows + r0;
#pragma unroll
            for (int k = 0; k < 4; ++k) row[k] = __ldcg(p + 16 * k);
        };
        if (have) ask();
        for (int i = 0; have; ++i) {
            const bool is_a = walk.tile < g.tiles_a;
            const bf16* src = is_a ? g.x : g.dy;
            const long ld = is_a ? g.ldx : g.lddy;
            const int width = is_a ? g.K : g.O, col0 = (is_a ? walk.tile : walk.tile - g.tiles_a) * kLoraCols + c * 8;
            const bf16* p[4];
            uint32_t ok = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                p[k] = src + (row[k] < 0 ? 0L : (long)row[k] * ld) + col0;
                ok |= (row[k] < 0 ? 0u : 1u) << k;
            }
            if (++q == walk.len) {
                have = walk.next();
                q = 0;
            }
            if (have) ask();
            if (i >= g.stages) mbar_wait(smem_u32(&tail->empty[st]), phase, abort);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const bool in = ((ok >> k) & 1u) && col0 + b * 64 < width;
                    cp_async16(dst + st * stage_bytes + b * 8192 + k * 2048, in ? p[k] + b * 64 : src, in);
                }
            cp_async_arrive(smem_u32(&tail->full[st]));
            if (++st == g.stages) { st = 0; phase ^= 1u; }
        }
        cp_async_commit();
        cp_async_wait<0>();
    } else if (warp == 9) {
        if (lane == 0) {
            const int boxes = g.gbytes / 8192;
            int st = 0;
            uint32_t phase = 1;
            pdl_wait();  // the hidden rows
            pdl_trigger();
            fence_proxy_async_global();  // they were written with plain stores
            bool ok = true;
            for (int i = 0; ok && walk.next();) {
                const CUtensorMap* tm = walk.tile < g.tiles_a ? &tm_d : &tm_h;
                int slot = first[walk.n] * kLoraTile + walk.step * kLoraStepRows;
                for (int q = 0; q < walk.len; ++q, ++i, slot += kLoraStepRows) {
                    if (i >= g.stages && !mbar_wait(smem_u32(&tail->empty[st]), phase, abort)) { ok = false; break; }
                    const uint32_t fb = smem_u32(&tail->full[st]);
                    mbar_arrive_expect_tx(fb, g.gbytes);
                    for (int b = 0; b < boxes; ++b)
                        tma_load_2d(sbase + st * stage_bytes + kOuterXBytes + b * 8192, tm, fb, b * 64, slot);
                    if (++st == g.stages) { st = 0; phase ^= 1u; }
                }
            }
        }
    } else if (warp == 8) {
        if (lane == 0) {
            const uint32_t idesc = idesc_f32acc(1, 1, 128, 2 * Rp) | kMajorA | kMajorB;
            const uint32_t dx0 = mnmajor(sbase, 8192), dg0 = mnmajor(sbase + kOuterXBytes, 8192);
            int seg = 0, st = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (; ok && walk.next(); ++seg) {
                const int len = walk.len;
                const int buf = seg % bufs, use = seg / bufs;
                if (use > 0 && !mbar_wait(smem_u32(&tail->aempty[buf]), (use - 1) & 1, abort)) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * 4 * Rp;
                for (int q = 0; q < len; ++q) {
                    if (!mbar_wait(smem_u32(&tail->full[st]), phase, abort)) { ok = false; break; }
                    fence_proxy_async_smem();  // the copied rows, for the tensor core
                    tc_fence_after();
                    const uint32_t dx = dx0 + st * (stage_bytes >> 4), dg = dg0 + st * (stage_bytes >> 4);
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int j = 0; j < kLoraStepRows / 16; ++j)  // 16 rows: 16 x 128 bytes
                            mma_desc(d + half * 2 * Rp, dx + half * 1024 + j * 128, dg + j * 128, idesc, q > 0 || j > 0);
                    mma_commit(smem_u32(&tail->empty[st]));
                    if (++st == g.stages) { st = 0; phase ^= 1u; }
                }
                mma_commit(smem_u32(&tail->afull[buf]));
            }
        }
    } else {
        const int w = warp & 3;
        // adapters without rows: zeros, before the first sums are there
        for (int n = 0; n < g.N; ++n) {
            if (units[n + 1] != units[n]) continue;
            uint4* pa = reinterpret_cast<uint4*>(g.da + (long)n * g.R * g.K);
            uint4* pb = reinterpret_cast<uint4*>(g.db + (long)n * g.R * g.O);
            const long step = (long)gridDim.x * 128, from = (long)blockIdx.x * 128 + (tid & 127);
            for (long i = from; i < (long)g.R * g.K / 8; i += step) pa[i] = make_uint4(0, 0, 0, 0);
            for (long i = from; i < (long)g.R * g.O / 8; i += step) pb[i] = make_uint4(0, 0, 0, 0);
        }
        int seg = 0;
        for (; walk.next(); ++seg) {
            const int slot = seg == 0 ? 0 : 1;
            const bool is_a = walk.tile < g.tiles_a, whole = walk.len == walk.total;
            const int n = walk.n, tile = is_a ? walk.tile : walk.tile - g.tiles_a;
            const int buf = seg % bufs, use = seg / bufs;
            if (!mbar_wait(smem_u32(&tail->afull[buf]), use & 1, abort)) break;
            tc_fence_after();
            float* part = g.partial + ((long)blockIdx.x * 2 + slot) * Rp * kLoraCols;
            for (int half = 0; half < 2; ++half) {
                const int c = half * 128 + w * 32 + lane;
                const uint32_t t = tmem + ((uint32_t)(w * 32) << 16) + buf * 4 * Rp + half * 2 * Rp;
                for (int q = 0; q < Rp; q += 16) {
                    uint32_t a[16], b[16];
                    tmem_ld16(t + q, a);
                    tmem_ld16(t + Rp + q, b);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        if (q + e >= g.R) break;
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            v[k] = both_halves(__uint_as_float(a[e + k]) + __uint_as_float(b[e + k]), __uint_as_float(a[e + k]));
                        if (whole) {
                            store_ranks(g, is_a, n, tile * kLoraCols + c, q + e, v);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) part[(long)(q + e + k) * kLoraCols + c] = v[k];
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&tail->aempty[buf]));
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, cols);
    }
    if (tid == 0 && tail->abort) atomicExch(g.err, 1);
}

// Adds up the partial sums of the tiles that CTAs of lora_outer_kernel shared. A tile is found by the first boundary between
// two CTAs' parts that lies among its steps; four warps of the W (this one is w; W is even) take a boundary, 64 columns and
// 8 ranks at a time.
__device__ void sum_shared_tiles(const OuterArgs& g, const int32_t* units, int ctas, int w, int W, int lane) {
    const int tiles = g.tiles_a + g.tiles_b, Rp = lora_rp(g.R), per = g.R / 8 * (kLoraCols / 64);
    const unsigned total = (unsigned)units[g.N] * tiles, G = min((unsigned)ctas, total);
    const int P = W >= 4 ? 4 : 1, crews = W / P;  // warps to a boundary, boundaries at a time: at least one
    if (w >= crews * P) return;
    for (unsigned b = 1 + w / P; b < G; b += crews) {
        const unsigned s = part_start(total, b, G), before = part_start(total, b - 1, G);
        Walk at{units, g.N, tiles, 0u, 0, 0, 0, 0, 0, 0};
        at.start(s);
        const unsigned start = s - at.at, end = start + at.total;
        if (at.at == 0 || s >= end || before > start) continue;
        unsigned last = b;  // the CTA that did the tile's last steps
        while (last + 1 < G && part_start(total, last + 1, G) < end) ++last;
        // CTA b - 1 began with this tile if its part starts here or in the tile before's writing; the others all did
        const int slot = start - before <= (unsigned)kLoraTileUnits ? 0 : 1;
        const bool is_a = at.tile < g.tiles_a;
        const int col0 = (is_a ? at.tile : at.tile - g.tiles_a) * kLoraCols;
        for (int item = w % P; item < per; item += P) {
            const int r = item / (kLoraCols / 64) * 8, c = item % (kLoraCols / 64) * 64 + lane * 2;
            const float* p = g.partial + ((long)((b - 1) * 2 + slot) * Rp + r) * kLoraCols + c;
            float2 t[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = __ldcg(reinterpret_cast<const float2*>(p + (long)k * kLoraCols));
            p = g.partial + ((long)b * 2 * Rp + r) * kLoraCols + c;
            for (unsigned i = b; i <= last; ++i, p += 2L * Rp * kLoraCols)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float2 f = __ldcg(reinterpret_cast<const float2*>(p + (long)k * kLoraCols));
                    t[k].x += f.x, t[k].y += f.y;
                }
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = t[k].x;
            store_ranks(g, is_a, at.n, col0 + c, r, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = t[k].y;
            store_ranks(g, is_a, at.n, col0 + c + 1, r, v);
        }
    }
}

// ------------------------------------------------------------------------------------------- up
// 128 rows x 64 columns a unit, every CTA a run of units, two CTAs to an SM: the products of a unit go into one of two
// accumulators while the result warps add the other to base, which they fetched two units ahead, and store whole 64-byte
// pieces of rows. Bound by memory: 84 MB in 18.5 us (5120 rows of 4096: 4.5 TB/s), 134 MB in 25.5 us (16384 of 2048: 5.3 TB/s), of
// which looking for results that are not finite takes 0.7.
constexpr int kUpCols = 64;       // columns of a unit
constexpr int kUpStages = 3;
constexpr int kUpThreads = 384;   // warps 0-7: base in, results out; 8: MMA; 9: TMA; 10, 11: rows without an adapter, shared
                                  // gradient tiles

// A warp's 32 x 32 results in its stage of shared memory (a row per lane, 16-byte pieces as the kernel lays them), once more where
// they are not finite and their column's weights hold an infinity: h this lane's row of high halves, base its row (null: 0), first
// the warp's first column. by_rank: w is [R][width], else [width][R]. The hidden rows are there: their products are.
__device__ __noinline__ void again(uint8_t* stage, const bf16* h, const bf16* w, int by_rank, int R, int width, int first,
                                   const bf16* base) {
    const int lane = threadIdx.x & 31;
    auto weights = [&](int j, int r, uint32_t (&v)[8]) {  // column j's ranks r .. r + 7, as the upper halves of fp32
        if (by_rank) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = (uint32_t)__bfloat16_as_ushort(w[(long)(r + k) * width + first + j]) << 16;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(w + (long)(first + j) * R + r);
            v[0] = u.x << 16, v[1] = u.x & 0xffff0000u, v[2] = u.y << 16, v[3] = u.y & 0xffff0000u;
            v[4] = u.z << 16, v[5] = u.z & 0xffff0000u, v[6] = u.w << 16, v[7] = u.w & 0xffff0000u;
        }
    };
    uint32_t v[8];
    bool inf = false;
    if (first + lane < width)
        for (int r = 0; r < R; r += 8) {
            weights(lane, r, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) inf |= (v[k] & 0x7fffffffu) == 0x7f800000u;
        }
    for (uint32_t todo = __ballot_sync(0xffffffffu, inf); todo != 0; todo &= todo - 1) {
        const int j = __ffs(todo) - 1;
        float s = 0.0f;
        for (int r = 0; r < R; r += 8) {
            const uint4 u = __ldcg(reinterpret_cast<const uint4*>(h + r));
            const uint32_t g[4] = {u.x, u.y, u.z, u.w};
            weights(j, r, v);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                s = fmaf(__uint_as_float(k & 1 ? g[k >> 1] & 0xffff0000u : g[k >> 1] << 16), __uint_as_float(v[k]), s);
        }
        if (base != nullptr) s += __bfloat162float(__ldcg(base + first + j));
        bf16* o = reinterpret_cast<bf16*>(stage + lane * 64 + (((j >> 3) ^ ((lane >> 1) & 3)) << 4)) + (j & 7);
        if (!finite(__bfloat162float(*o))) *o = __float2bfloat16_rn(s);
    }
}

struct UpArgs {
    const bf16* h;
    const bf16* w;
    const bf16* base;
    long ldbase;
    bf16* out;
    long ldout;
    const int32_t* row_adapter;  // of every row: those without one are copied
    const int32_t* nblocks;
    const int32_t* adapter;
    const int32_t* rows;
    int* err;
    int T, N, R, width, by_rank;
    int hbytes, wbytes;
    int sum_ctas;    // AFTER_OUTER: lora_outer_kernel's CTAs, whose partial sums are to be added up
    OuterArgs sums;
};
struct UpTail {
    uint64_t hfull, hempty;
    uint64_t wfull[kUpStages];
    uint64_t wempty[kUpStages];
    uint64_t afull[2];
    uint64_t aempty[2];
    uint32_t tmem_base;
    int abort;
};
inline int up_hbytes(int R) { return (2 * lora_rp(R) + 63) / 64 * 16384; }
inline int up_wbytes(int R) { return std::max(lora_rp(R) * 128, (lora_rp(R) + 63) / 64 * 8192); }
inline size_t up_smem(int R, int N, bool sums) {
    return 1024 + (size_t)up_hbytes(R) + (size_t)kUpStages * (up_wbytes(R) + 16384) + sizeof(UpTail) + (sums ? ((size_t)N + 1) * 4 : 0);
}

// AFTER_OUTER: the launch before is lora_outer_kernel. The hidden rows were complete before that let this kernel start, and
// its shared tiles are added up here.
template <bool AFTER_OUTER>
__global__ void __launch_bounds__(kUpThreads, 2)
    lora_up_kernel(const __grid_constant__ CUtensorMap tm_h, const __grid_constant__ CUtensorMap tm_w, const UpArgs g) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + align1024(smem_u32(smem_raw));
    const uint32_t sbase = smem_u32(smem);
    const uint32_t wring = sbase + g.hbytes, yring = wring + kUpStages * g.wbytes;
    UpTail* tail = reinterpret_cast<UpTail*>(smem + g.hbytes + kUpStages * (g.wbytes + 16384));
    volatile int* abort = &tail->abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int Rp = lora_rp(g.R);

    if (tid == 0) {
        mbar_init(smem_u32(&tail->hfull), 1);
        mbar_init(smem_u32(&tail->hempty), 1);
        for (int st = 0; st < kUpStages; ++st) {
            mbar_init(smem_u32(&tail->wfull[st]), 1);
            mbar_init(smem_u32(&tail->wempty[st]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&tail->afull[b]), 1);
            mbar_init(smem_u32(&tail->aempty[b]), 8);
        }
        tail->abort = 0;
        fence_barrier_init();
        fence_proxy_async_smem();
        prefetch_tensormap(&tm_h);
        prefetch_tensormap(&tm_w);
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(&tail->tmem_base), 2 * kUpCols);
        tmem_relinquish();
    }
    // this CTA's units: a run of the (block, column tile) pairs, blocks outermost
    const unsigned tiles = (g.width + kUpCols - 1) / kUpCols, units = (unsigned)__ldcg(g.nblocks) * tiles;
    const unsigned u0 = part_start(units, blockIdx.x, gridDim.x);
    const int count = (int)(part_start(units, blockIdx.x + 1, gridDim.x) - u0);
    const int block0 = (int)(u0 / tiles), tile0 = (int)(u0 % tiles);
    auto next_tile = [tiles](int& block, int& tile) {
        if (++tile == (int)tiles) tile = 0, ++block;
    };
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tail->tmem_base;

    if (warp == 9) {
        if (lane == 0) {
            const int boxes = (Rp + 63) / 64;
            int wblock = block0, wtile = tile0, wn = count > 0 ? __ldcg(g.adapter + block0) : 0, wst = 0;
            uint32_t wphase = 1;
            auto load_w = [&](int i) {
                if (i >= kUpStages && !mbar_wait(smem_u32(&tail->wempty[wst]), wphase, abort)) return;
                const uint32_t w = wring + wst * g.wbytes, fb = smem_u32(&tail->wfull[wst]);
                if (g.by_rank) {
                    mbar_arrive_expect_tx(fb, Rp * 128);
                    tma_load_3d(w, &tm_w, fb, wtile * kUpCols, 0, wn);
                } else {
                    mbar_arrive_expect_tx(fb, boxes * 8192);
                    for (int q = 0; q < boxes; ++q) tma_load_3d(w + q * 8192, &tm_w, fb, q * 64, wtile * kUpCols, wn);
                }
                const int before = wblock;
                next_tile(wblock, wtile);
                if (wblock != before && i + 1 < count) wn = __ldcg(g.adapter + wblock);
                if (++wst == kUpStages) { wst = 0; wphase ^= 1u; }
            };
            for (int i = 0; i < min(count, kUpStages); ++i) load_w(i);
            if (!AFTER_OUTER) {
                pdl_wait();  // the hidden rows
                pdl_trigger();
            }
            fence_proxy_async_global();  // they were written with plain stores
            int hblock = -1, hloads = 0, block = block0, tile = tile0;
            for (int i = 0; i < count; ++i, next_tile(block, tile)) {
                if (block != hblock) {
                    if (hloads > 0 && !mbar_wait(smem_u32(&tail->hempty), (hloads - 1) & 1, abort)) break;
                    const uint32_t fb = smem_u32(&tail->hfull);
                    mbar_arrive_expect_tx(fb, g.hbytes);
                    for (int q = 0; q * 16384 < g.hbytes; ++q) tma_load_2d(sbase + q * 16384, &tm_h, fb, q * 64, block * kLoraTile);
                    hblock = block;
                    ++hloads;
                }
                if (i + kUpStages < count) load_w(i + kUpStages);
            }
        }
    } else if (warp == 8) {
        if (lane == 0) {
            const uint32_t idesc = idesc_f32acc(1, 1, kLoraTile, kUpCols) | (g.by_rank ? kMajorB : 0u);
            const uint32_t dh0 = kmajor(sbase), dw0 = g.by_rank ? mnmajor(wring, 8192) : kmajor(wring);
            int hblock = -1, hloads = 0, block = block0, tile = tile0, st = 0;
            uint32_t phase = 0;
            for (int i = 0; i < count; ++i, next_tile(block, tile)) {
                const int buf = i & 1;
                if (block != hblock) {
                    if (!mbar_wait(smem_u32(&tail->hfull), hloads & 1, abort)) break;
                    hblock = block;
                    ++hloads;
                }
                if (!mbar_wait(smem_u32(&tail->wfull[st]), phase, abort)) break;
                if (i >= 2 && !mbar_wait(smem_u32(&tail->aempty[buf]), ((i >> 1) - 1) & 1, abort)) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * kUpCols, dw = dw0 + st * (g.wbytes >> 4);
                bool more = false;
                for (int half = 0; half < 2; ++half)
                    for (int j = 0; j < Rp / 16; ++j) {
                        const int hc = half * Rp + 16 * j;  // column of the hidden row
                        mma_desc(d, dh0 + (hc >> 6) * 1024 + ((hc & 63) >> 3), dw + (g.by_rank ? j * 128 : (j >> 2) * 512 + 2 * (j & 3)),
                                 idesc, more);
                        more = true;
                    }
                mma_commit(smem_u32(&tail->wempty[st]));
                if (i + 1 < count && tile + 1 == (int)tiles) mma_commit(smem_u32(&tail->hempty));
                mma_commit(smem_u32(&tail->afull[buf]));
                if (++st == kUpStages) { st = 0; phase ^= 1u; }
            }
        }
    } else if (warp >= 10) {
        // rows without an adapter: copied (or zeroed), dealt out one by one, since such rows come in runs
        const int spare = (int)blockIdx.x * 2 + warp - 10, spares = (int)gridDim.x * 2;
        if (g.base != g.out)
            for (long t0 = spare; t0 < g.T; t0 += spares * 32L) {
                const long tl = t0 + lane * (long)spares;
                const int n = tl < g.T ? __ldcg(g.row_adapter + tl) : 0;
                uint32_t none = __ballot_sync(0xffffffffu, (unsigned)n >= (unsigned)g.N);
                while (none != 0) {
                    copy_row(g.base, g.ldbase, g.out, g.ldout, t0 + (__ffs(none) - 1) * (long)spares, g.width, lane, 32);
                    none &= none - 1;
                }
            }
        if (AFTER_OUTER) {
            int32_t* units = reinterpret_cast<int32_t*>(tail + 1);  // [N + 1]
            for (int i = (warp - 10) * 32 + lane; i <= g.N; i += 64) units[i] = __ldcg(g.sums.units + i);
            named_bar_sync(1, 64);
            pdl_wait();  // the partial sums
            pdl_trigger();
            sum_shared_tiles(g.sums, units, g.sum_ctas, spare, spares, lane);
        }
    } else {
        // a warp works on 32 rows (its quarter of TMEM) and 32 columns; its pieces of base, 32 rows of 64 bytes, travel
        // kUpStages - 1 units ahead. Piece c of row r is at r * 64 + ((c ^ (r / 2 & 3)) << 4): a thread's own row and the
        // copies' four lanes to a row both touch all banks evenly.
        const int quarter = warp & 3, half = warp >> 2;
        uint8_t* ys = smem + (yring - sbase) + warp * 2048;  // + stage * 16384
        const uint32_t ya = yring + warp * 2048;
        const int c = lane & 3, sub = lane >> 2;  // piece, and first of four rows 8 apart, of the copies
        const int mycol = half * 32 + c * 8;      // of this lane's copies within the unit
        const bf16* from[4];                      // of these rows in the block last fetched for
        uint32_t have = 0;
        int pblock = -1, fblock = block0, ftile = tile0, fetched = 0, fst = 0;
        auto fetch = [&]() {
            if (fblock != pblock) {
                pblock = fblock;
                have = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = __ldcg(g.rows + fblock * kLoraTile + quarter * 32 + q * 8 + sub);
                    from[q] = g.base + (row < 0 ? 0L : (long)row * g.ldbase) + mycol;
                    have |= (row < 0 ? 0u : 1u) << q;
                }
            }
            const int col = ftile * kUpCols;
            const bool in = col + mycol < g.width;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = q * 8 + sub;
                const bool ok = in && ((have >> q) & 1u);
                cp_async16(ya + fst * 16384 + r * 64 + ((c ^ ((r >> 1) & 3)) << 4), ok ? from[q] + col : g.base, ok);
            }
            ++fetched;
            if (++fst == kUpStages) fst = 0;
            next_tile(fblock, ftile);
        };
        for (int k = 0; k < kUpStages - 1; ++k) {
            if (g.base != nullptr && fetched < count) fetch();
            cp_async_commit();
        }
        bf16* to[4];
        uint32_t there = 0;
        int tblock = -1, block = block0, tile = tile0, st = 0;
        for (int i = 0; i < count; ++i, next_tile(block, tile)) {
            const int buf = i & 1;
            if (block != tblock) {
                tblock = block;
                there = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = __ldcg(g.rows + block * kLoraTile + quarter * 32 + q * 8 + sub);
                    to[q] = g.out + (row < 0 ? 0L : (long)row * g.ldout) + mycol;
                    there |= (row < 0 ? 0u : 1u) << q;
                }
            }
            if (g.base != nullptr && fetched < count) fetch();
            cp_async_commit();
            cp_async_wait<kUpStages - 1>();
            __syncwarp();
            if (!mbar_wait(smem_u32(&tail->afull[buf]), (i >> 1) & 1, abort)) break;
            tc_fence_after();
            uint8_t* at = ys + st * 16384;
            uint32_t r[32];
            tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + buf * kUpCols + half * 32, r);
            uint4 y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                y[q] = g.base != nullptr ? *reinterpret_cast<const uint4*>(at + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4))
                                         : make_uint4(0, 0, 0, 0);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&tail->aempty[buf]));
            Unusual unusual;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                y[q].x = add_bf16x2(y[q].x, __uint_as_float(r[q * 8]), __uint_as_float(r[q * 8 + 1]));
                y[q].y = add_bf16x2(y[q].y, __uint_as_float(r[q * 8 + 2]), __uint_as_float(r[q * 8 + 3]));
                y[q].z = add_bf16x2(y[q].z, __uint_as_float(r[q * 8 + 4]), __uint_as_float(r[q * 8 + 5]));
                y[q].w = add_bf16x2(y[q].w, __uint_as_float(r[q * 8 + 6]), __uint_as_float(r[q * 8 + 7]));
                *reinterpret_cast<uint4*>(at + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = y[q];
                unusual.see(y[q]);
            }
            if (unusual.any()) {
                const int slot = block * kLoraTile + quarter * 32 + lane, row = __ldcg(g.rows + slot);
                again(at, g.h + (long)slot * 2 * Rp, g.w + (long)__ldcg(g.adapter + block) * g.R * g.width, g.by_rank, g.R,
                      g.width, tile * kUpCols + half * 32, row < 0 || g.base == nullptr ? nullptr : g.base + (long)row * g.ldbase);
            }
            __syncwarp();
            const int col = tile * kUpCols;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int rr = q * 8 + sub;
                y[q] = *reinterpret_cast<const uint4*>(at + rr * 64 + ((c ^ ((rr >> 1) & 3)) << 4));
            }
            if (col + mycol < g.width) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if ((there >> q) & 1u) *reinterpret_cast<uint4*>(to[q] + col) = y[q];
            }
            __syncwarp();  // read out before the stage is filled again
            if (++st == kUpStages) st = 0;
        }
        cp_async_wait<0>();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * kUpCols);
    }
    if (tid == 0 && tail->abort) atomicExch(g.err, 1);
    pdl_wait();
}

// ------------------------------------------------------------------------------------------- launches
bool encode_weights(CUtensorMap* map, const bf16* w, int N, int rows, int cols, int box_rows) {
    return encode_tmap_3d_bf16(map, w, cols, rows, N, 64, box_rows);
}

bool encode_hidden(CUtensorMap* map, const bf16* h, long slots, int Rp, int box_rows) {
    return encode_tmap_2d(map, h, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 2 * Rp, slots, (uint64_t)Rp * 4, 64, box_rows);
}

}  // namespace

size_t lora_partial_bytes(int R) { return (size_t)kMaxSms * 2 * lora_rp(R) * kLoraCols * 4; }

cudaError_t launch_lora_down(const LoraDown* parts, int count, const float* scale, const LoraPlan& p, const LoraShape& g,
                             int sms, cudaStream_t s) {
    static std::atomic<bool> configured[64];
    PM_TRY(raise_smem((const void*)lora_down_kernel, 213 << 10, configured));
    CUtensorMap tm[2];
    DownArgs a;
    memset(&a, 0, sizeof(a));
    int steps = 0;
    for (int i = 0; i < count; ++i) {
        const LoraDown& d = parts[i];
        if (!(d.by_rank ? encode_weights(&tm[i], d.w, g.N, g.R, d.width, lora_rp(g.R))
                        : encode_weights(&tm[i], d.w, g.N, d.width, g.R, 64)))
            return cudaErrorInvalidValue;
        a.part[i] = DownPart{d.src, d.ld, d.width, d.by_rank ? 1 : 0, d.out};
        a.wbytes = std::max(a.wbytes, down_wbytes(g.R, d.by_rank));
        steps = std::max(steps, cdiv(d.width, 64));
    }
    if (count == 1) tm[1] = tm[0];
    a.scale = scale;
    a.nblocks = p.nblocks;
    a.adapter = p.adapter;
    a.rows = p.rows;
    a.err = p.status;
    a.R = g.R;
    const int blocks = lora_max_blocks(g.T, g.N);
    // CTAs per block: up to four while that makes no more than two to an SM and leaves each eight steps. Replayed calls in us
    // with one, two and four: 1000 x 2048 -> 4096 of rank 64 22.5, 20.0, 18.0; 2500 x 4096 -> 4096 of rank 32 36.6, 29.2,
    // 24.6; gradients of 333 rows of rank 16 here 24.0, 20.7, 18.6; 4096 x 512 (eight steps) 18.5, 19.8, -; eight instead of
    // four: 17.1, 24.3, 17.8, but 28.2 against 24.6 at 2048 rows of rank 128.
    int splits = 1;
    while (splits < 4 && (long)blocks * splits * 2 * count <= 2L * sms && steps >= splits * 16) splits *= 2;
    a.stages = down_stages(a.wbytes, blocks * splits * count <= sms ? 1 : 2);
    return launch_cluster(lora_down_kernel, dim3(blocks * splits, count), dim3(kDownThreads), splits,
                          down_smem(g.R, a.wbytes, a.stages), s, tm[0], tm[1], a);
}

static OuterArgs outer_args(const LoraOuter& o, const LoraPlan& p, const LoraShape& g) {
    OuterArgs a;
    memset(&a, 0, sizeof(a));
    a.x = o.x;
    a.dy = o.dy;
    a.ldx = o.ldx;
    a.lddy = o.lddy;
    a.da = o.da;
    a.db = o.db;
    a.partial = o.partial;
    a.units = p.units;
    a.first = p.first;
    a.rows = p.rows;
    a.err = p.status;
    a.K = g.K;
    a.O = g.O;
    a.R = g.R;
    a.N = g.N;
    a.tiles_a = cdiv(g.K, kLoraCols);
    a.tiles_b = cdiv(g.O, kLoraCols);
    a.stages = outer_stages(g.R);
    a.gbytes = outer_gbytes(g.R);
    return a;
}

cudaError_t launch_lora_outer(const LoraOuter& o, const LoraPlan& p, const LoraShape& g, int sms, cudaStream_t s) {
    static std::atomic<bool> configured[64];
    PM_TRY(raise_smem((const void*)lora_outer_kernel, std::max(outer_smem(64, kLoraMaxAdapters), outer_smem(kLoraMaxRank, kLoraMaxAdapters)), configured));
    const int blocks = lora_max_blocks(g.T, g.N), Rp = lora_rp(g.R);
    const OuterArgs a = outer_args(o, p, g);
    CUtensorMap th, td;
    if (!encode_hidden(&th, o.h, (long)blocks * kLoraTile, Rp, kLoraStepRows) ||
        !encode_hidden(&td, o.d, (long)blocks * kLoraTile, Rp, kLoraStepRows))
        return cudaErrorInvalidValue;
    return launch_pdl(lora_outer_kernel, dim3(std::min(sms, kMaxSms)), dim3(kOuterThreads), outer_smem(g.R, g.N), s, th, td, a);
}

cudaError_t launch_lora_up(const LoraUp& u, const int32_t* adapter, const LoraPlan& p, const LoraShape& g, int sms,
                           cudaStream_t s) {
    static std::atomic<bool> configured[2][64];
    const bool after = u.sums != nullptr;
    auto kernel = after ? lora_up_kernel<true> : lora_up_kernel<false>;
    PM_TRY(raise_smem((const void*)kernel, up_smem(kLoraMaxRank, kLoraMaxAdapters, after), configured[after]));
    const int blocks = lora_max_blocks(g.T, g.N), Rp = lora_rp(g.R);
    CUtensorMap th, tw;
    if (!encode_hidden(&th, u.h, (long)blocks * kLoraTile, Rp, kLoraTile) ||
        !(u.by_rank ? encode_weights(&tw, u.w, g.N, g.R, u.width, Rp) : encode_weights(&tw, u.w, g.N, u.width, g.R, 64)))
        return cudaErrorInvalidValue;
    UpArgs a;
    memset(&a, 0, sizeof(a));
    a.h = u.h;
    a.w = u.w;
    a.base = u.base;
    a.ldbase = u.ldbase;
    a.out = u.out;
    a.ldout = u.ldout;
    a.row_adapter = adapter;
    a.nblocks = p.nblocks;
    a.adapter = p.adapter;
    a.rows = p.rows;
    a.err = p.status;
    a.T = g.T;
    a.N = g.N;
    a.R = g.R;
    a.width = u.width;
    a.by_rank = u.by_rank ? 1 : 0;
    if (after) {
        a.sum_ctas = std::min(sms, kMaxSms);
        a.sums = outer_args(*u.sums, p, g);
    }
    a.hbytes = up_hbytes(g.R);
    a.wbytes = up_wbytes(g.R);
    const size_t smem = up_smem(g.R, g.N, after);
    const int resident = smem <= 113 * 1024 ? 2 : 1;
    const long units = (long)blocks * cdiv(u.width, kUpCols);
    return launch_pdl(kernel, dim3((unsigned)std::min<long>(units, (long)sms * resident)), dim3(kUpThreads),
                      smem, s, th, tw, a);
}

}  // namespace pm
