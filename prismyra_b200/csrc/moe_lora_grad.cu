// The adapters' gradients for few rows.
//
//   d[t] = s_n B_n^T dy[t],  h[t] = s_n A_n x[t],  dx[t] = base[t] + A_n^T d[t],  dA_n = sum_t d[t] x[t]^T,
//   dB_n = sum_t dy[t] h[t]^T
//
// Two products onto the rank make d and h, 16 rows at a time; they are kept as two bf16 halves (hi + lo, 16 significant bits).
// Then 64 columns at a time of dx, dA and dB are a warp's. All products are mma.sync m16n8k16 on operands straight from global
// memory: few rows make this latency, not arithmetic.
//
//   one launch     a cluster of CTAs per adapter finds the adapter's rows itself; the partial sums of d and h, and then their
//                  halves, go through the cluster's shared memory
//   three launches the row plan, a CTA per 16 rows for d and one for h, then all column blocks of all adapters: no cluster's
//                  SMs have to do an adapter of many rows
//
// Operand order. Where the contraction lies along a row of memory a lane's 16 bytes are 8 neighbouring values of it, taken as
// positions {2c, 2c+1, 2c+8, 2c+9} of two steps. Where it runs across rows (rows of x and dy for dA and dB, ranks of A for dx)
// a lane reads 8 columns of the four rows at those positions and pairs up neighbouring rows: value i of its 8 columns is
// column gr of the MMA's tile i, so that a lane's results are again 8 neighbours.
#include <atomic>

#include "lora_dev.cuh"
#include "moe_lora.h"

namespace pm {
namespace {

// One launch up to these rows x ranks (with up to kLoraGradFewRows rows; half of them where adapters are more than
// kGradFewAdapters, since the one that has all rows then has two CTAs), three up to these rows of rank 16, in all or on average
// for an adapter, the tiled kernels above. 2048 -> 2048, us replayed, one launch / three / tiled (rows, rank, adapters):
//   16 x 16 of 1 7.1, 10, 16; 64 x 16 of 4 9.0, 11, 17; 128 x 16 of 1 15.5, 11, 17
//   128 x 16 of 64 spread 12, 14, 36, all of one adapter 41, 16, 28
//   512 x 16 of 4 32, 14.7, 21; of 64 spread 12 to 17, 17, 38, all of one 48 to 143, 31, 29
//   800 x 16 of 4 -, 16.8, 22; of 64 spread -, 18, 39, all of one -, 43, 32
//   1200 x 16 of 1 -, 25, 26; 2000 x 16 of 4 -, 31, 27
//   1000 x 16 of 1000 -, 134, 317; 2048 x 16 of 512 spread -, 93, 206, all of one -, 131, 119, of 16 -, 51, 113
//   4096 x 16 of 1024 spread -, 180, 373, all of one -, 292, 219, of 16 -, 100, 221; 1000 x 16 of 256 45, 58 and 29 on groups, 110,
//   70 and 64 tiled: which adapters have rows the host cannot know, and the groups lose least where they are the wrong choice
//   32 x 64 of 4 14.8, -, 19; 128 x 64 of 8 22, 25, 20; 1000 x 64 of 16 -, 49, 33: the warps' MMAs take 16 rows at a time, at a
//   fraction of the tensor core's rate
constexpr int kGradFewRowRanks = 2048;
constexpr int kGradFewAdapters = 32;
constexpr int kGradGroupedRows = 800;
constexpr int kGradGroupedEach = 4;
// Threads of a CTA by its tiles of 8 ranks: what 64 Ki registers allow.
template <int NT>
__host__ __device__ constexpr int grad_threads() { return NT <= 4 ? 512 : 256; }

struct GradFewArgs : LoraGradFew {
    int T, K, O, R, N;
    int tiles;  // of 16 rows, that one adapter can have
};

// Warps that share the sums of one tile of 16 rows in a CTA, where there are tiles of them for `warps`.
__device__ __forceinline__ int grad_subs(int tiles, int warps) {
    return tiles * 8 <= warps ? 4 : tiles * 4 <= warps ? 2 : 1;
}
template <int NT>  // tiles of 8 ranks
__host__ __device__ constexpr int grad_ld() { return (NT == 1 ? 16 : 8 * NT) + 8; }  // rows of halves on different banks
template <int NT>
constexpr size_t grad_smem(int tiles) {
    return sizeof(float) * (size_t)std::max(tiles, grad_threads<NT>() / 64) * 32 * 8 * NT +
           2 * 4 * (size_t)tiles * 16 * grad_ld<NT>() + sizeof(int) * (size_t)tiles * 16;
}

__device__ __forceinline__ void ldmatrix_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t lower(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t upper(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
// Two bf16: those of `stored` that are finite, else those of `other`.
__device__ __forceinline__ uint32_t keep_finite(uint32_t stored, uint32_t other) {
    const uint32_t m = ((stored & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((stored & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
    return (other & m) | (stored & ~m);
}
// Value i of 8 columns, of two neighbouring rows.
__device__ __forceinline__ void pair_rows(const uint4& p, const uint4& q, uint32_t (&out)[8]) {
    out[0] = lower(p.x, q.x), out[1] = upper(p.x, q.x), out[2] = lower(p.y, q.y), out[3] = upper(p.y, q.y);
    out[4] = lower(p.z, q.z), out[5] = upper(p.z, q.z), out[6] = lower(p.w, q.w), out[7] = upper(p.w, q.w);
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    uint4 o;
    __nv_bfloat162* b = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    return o;
}
// NT neighbouring bf16, NT = 1, 2, 4 or 8.
template <int NT>
struct Ranks {
    uint32_t w[(NT + 1) / 2];
    __device__ __forceinline__ void load(const bf16* p, bool in) {
        if constexpr (NT == 1) {
            w[0] = in ? *reinterpret_cast<const uint16_t*>(p) : 0u;
        } else if constexpr (NT == 2) {
            w[0] = in ? *reinterpret_cast<const uint32_t*>(p) : 0u;
        } else if constexpr (NT == 4) {
            const uint2 v = in ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
            w[0] = v.x, w[1] = v.y;
        } else {
            const uint4 v = in ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        }
    }
};
template <int NT>
__device__ __forceinline__ uint32_t pair_ranks(const Ranks<NT>& p, const Ranks<NT>& q, int j) {
    return j & 1 ? upper(p.w[j >> 1], q.w[j >> 1]) : lower(p.w[j >> 1], q.w[j >> 1]);
}

// Sums of d (is_h false) or h of 16 rows over a part of the width: pieces `part`, `part` + step, .. of 32 columns. Rows t0 (this
// lane's gr of the 16) and t1 (gr + 8), -1: none. Column i of the MMA's tile j is rank NT i + j.
template <int NT>
__device__ __forceinline__ void sums16(const GradFewArgs& g, const bf16* a, const bf16* b, bool is_h, int t0, int t1, int part,
                                       int step, float (&acc)[NT][4]) {
    constexpr int kAhead = NT <= 2 ? 4 : 2;  // pieces a warp has on their way
    const int lane = threadIdx.x & 31, gr = lane >> 2, c = lane & 3;
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    const int width = is_h ? g.K : g.O;
    const bf16* p0 = is_h ? g.x + (t0 < 0 ? 0L : t0 * g.ldx) : g.dy + (t0 < 0 ? 0L : t0 * g.lddy);
    const bf16* p1 = is_h ? g.x + (t1 < 0 ? 0L : t1 * g.ldx) : g.dy + (t1 < 0 ? 0L : t1 * g.lddy);
    for (int s = part; s * 32 < width; s += kAhead * step) {
        uint4 v0[kAhead], v1[kAhead];
#pragma unroll
        for (int p = 0; p < kAhead; ++p) {
            const int k = (s + p * step) * 32 + c * 8;
            v0[p] = k < width && t0 >= 0 ? *reinterpret_cast<const uint4*>(p0 + k) : zero;
            v1[p] = k < width && t1 >= 0 ? *reinterpret_cast<const uint4*>(p1 + k) : zero;
        }
        if (is_h) {
            uint4 w[kAhead][NT];
#pragma unroll
            for (int p = 0; p < kAhead; ++p) {
                const int k = (s + p * step) * 32 + c * 8;
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    w[p][j] = k < width && gr * NT + j < g.R
                                  ? *reinterpret_cast<const uint4*>(a + (long)(gr * NT + j) * g.K + k)
                                  : zero;
            }
#pragma unroll
            for (int p = 0; p < kAhead; ++p)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    mma16816(acc[j], v0[p].x, v1[p].x, v0[p].y, v1[p].y, w[p][j].x, w[p][j].y);
                    mma16816(acc[j], v0[p].z, v1[p].z, v0[p].w, v1[p].w, w[p][j].z, w[p][j].w);
                }
        } else {
            Ranks<NT> w[kAhead][8];  // ranks gr NT .. of 8 columns
#pragma unroll
            for (int p = 0; p < kAhead; ++p) {
                const int k = (s + p * step) * 32 + c * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    w[p][e].load(b + (long)(k + e) * g.R + gr * NT, k < width && gr * NT < g.R);
            }
#pragma unroll
            for (int p = 0; p < kAhead; ++p)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    mma16816(acc[j], v0[p].x, v1[p].x, v0[p].y, v1[p].y, pair_ranks(w[p][0], w[p][1], j),
                             pair_ranks(w[p][2], w[p][3], j));
                    mma16816(acc[j], v0[p].z, v1[p].z, v0[p].w, v1[p].w, pair_ranks(w[p][4], w[p][5], j),
                             pair_ranks(w[p][6], w[p][7], j));
                }
        }
    }
}

// This lane's sums of row gr + 8 h: ranks 2 c NT .. 2 (c + 1) NT - 1.
template <int NT>
__device__ __forceinline__ void lane_ranks(const float (&acc)[NT][4], int h, float (&f)[2 * NT]) {
#pragma unroll
    for (int j = 0; j < NT; ++j) f[j] = acc[j][2 * h], f[NT + j] = acc[j][2 * h + 1];
}

// 64 columns of A as the right operand of dx: [step of 16 ranks][first, second half of its positions][tile of columns].
template <int NT>
struct RankRows {
    static constexpr int kSteps = NT == 1 ? 1 : NT / 2;
    uint32_t w[kSteps][2][8];
    __device__ __forceinline__ void load(const bf16* a, int R, int K, int block) {
        const int lane = threadIdx.x & 31, gr = lane >> 2, c = lane & 3, col = block * 64 + gr * 8;
#pragma unroll
        for (int q = 0; q < kSteps; ++q) {
            uint4 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = q * 16 + 2 * c + (e & 1) + (e >> 1) * 8;
                v[e] = r < R && col < K ? __ldcg(reinterpret_cast<const uint4*>(a + (long)r * K + col))
                                        : make_uint4(0, 0, 0, 0);
            }
            pair_rows(v[0], v[1], w[q][0]);
            pair_rows(v[2], v[3], w[q][1]);
        }
    }
};

// 64 columns of dx for 16 rows, t[0] and t[1] this lane's (-1: none). load asks for base; finish takes d's halves from
// frag(half, step).
struct RowsOfDx {
    int t[2];
    uint4 y[2][2];
    __device__ __forceinline__ void load(const GradFewArgs& g, int block) {
        const int c = threadIdx.x & 3;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int o = block * 64 + (2 * c + e) * 8;
                y[h][e] = g.base != nullptr && t[h] >= 0 && o < g.K
                              ? __ldcg(reinterpret_cast<const uint4*>(g.base + (long)t[h] * g.ldbase + o))
                              : make_uint4(0, 0, 0, 0);
            }
    }
    template <int NT, class Frag>
    __device__ __forceinline__ void finish(const GradFewArgs& g, int block, const RankRows<NT>& a, Frag frag) {
        const int c = threadIdx.x & 3;
        float d[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[i][e] = 0.0f;
#pragma unroll
        for (int hl = 0; hl < 2; ++hl)
#pragma unroll
            for (int q = 0; q < RankRows<NT>::kSteps; ++q) {
                const uint4 f = frag(hl, q);
#pragma unroll
                for (int i = 0; i < 8; ++i) mma16816(d[i], f.x, f.y, f.z, f.w, a.w[q][0][i], a.w[q][1][i]);
            }
        if (any_not_finite(d)) {  // once more
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (!any_not_finite(d[i])) continue;  // a tile at a time: registers of one
                float high[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int q = 0; q < RankRows<NT>::kSteps; ++q) {
                    const uint4 f = frag(0, q);
                    mma16816(high, f.x, f.y, f.z, f.w, a.w[q][0][i], a.w[q][1][i]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) d[i][e] = both_halves(d[i][e], high[e]);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int o = block * 64 + (2 * c + e) * 8, k = 2 * h + e;
                uint4 r = y[h][e];
                r.x = add_bf16x2(r.x, d[0][k], d[1][k]);
                r.y = add_bf16x2(r.y, d[2][k], d[3][k]);
                r.z = add_bf16x2(r.z, d[4][k], d[5][k]);
                r.w = add_bf16x2(r.w, d[6][k], d[7][k]);
                if (t[h] >= 0 && o < g.K) *reinterpret_cast<uint4*>(g.dx + (long)t[h] * g.lddx + o) = r;
            }
    }
};

struct WeightSide {
    const bf16* src;  // x or dy
    long ld;
    bf16* out;        // the adapter's dA [R][width] or dB [width][R]
    int width, R;
    bool is_a;
};
// 64 columns of dA or dB, summed over tiles from, from + step, .. of 16 rows: row(i) is the adapter's row i or -1,
// frag(tile, half, step) the halves of d or h with their rows as the contraction. GLOBAL: both come from global memory, and are
// asked for ahead like the rows themselves (one tile; with four the warps' registers left one CTA an SM: 333 rows 13.5 us, not
// 11.8).
// acc, dA: [steps of 16 ranks][8 tiles of columns]; dB: [steps of 16 ranks][4 tiles of 16 columns][2 tiles of 8 ranks].
// HIGH: of the high halves alone, after a store of sums of both that were not all finite; those that were stay.
template <int NT, bool GLOBAL>
struct WeightBlock {
    static constexpr int kSteps = NT == 1 ? 1 : NT / 2;
    float acc[kSteps * 8][4];
    template <bool HIGH, class Row, class Frag>
    __device__ __forceinline__ void sum(const WeightSide& s, int block, int from, int step, int tiles, Row row, Frag frag) {
        const int lane = threadIdx.x & 31, gr = lane >> 2, c = lane & 3;
        const int width = s.width, col = block * 64 + gr * 8;
        const bf16* src = s.src;
        const long ld = s.ld;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        int id[4];
        uint4 v[4], f[2][kSteps];
        auto number = [&](int tile) {
#pragma unroll
            for (int e = 0; e < 4; ++e) id[e] = tile < tiles ? row(tile * 16 + 2 * c + (e & 1) + (e >> 1) * 8) : -1;
        };
        auto ask = [&](int tile) {
            if (!GLOBAL) number(tile);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = id[e] >= 0 && col < width ? *reinterpret_cast<const uint4*>(src + (long)id[e] * ld + col) : zero;
            if (!GLOBAL) return;
#pragma unroll
            for (int hl = 0; hl < (HIGH ? 1 : 2); ++hl)
#pragma unroll
                for (int q = 0; q < kSteps; ++q) f[hl][q] = tile < tiles ? frag(tile, hl, q) : zero;
            number(tile + step);
        };
        if (GLOBAL) number(from);
        ask(from);
#pragma unroll
        for (int i = 0; i < kSteps * 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
        for (int tile = from; tile < tiles; tile += step) {
            uint32_t lo[8], hi[8];
            pair_rows(v[0], v[1], lo);
            pair_rows(v[2], v[3], hi);
            if (!GLOBAL) ask(tile + step);
#pragma unroll
            for (int hl = 0; hl < (HIGH ? 1 : 2); ++hl)
#pragma unroll
                for (int q = 0; q < kSteps; ++q) {
                    const uint4 r = GLOBAL ? f[hl][q] : frag(tile, hl, q);
                    if (s.is_a) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) mma16816(acc[q * 8 + i], r.x, r.y, r.z, r.w, lo[i], hi[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float(&d)[4] = acc[q * 8 + i * 2], (&e)[4] = acc[q * 8 + i * 2 + 1];
                            mma16816(d, lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1], r.x, r.z);
                            if (NT > 1) mma16816(e, lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1], r.y, r.w);
                        }
                    }
                }
            if (GLOBAL) ask(tile + step);
        }
    }
    template <bool HIGH>
    __device__ __forceinline__ void store(const WeightSide& s, int block) const {
        const int lane = threadIdx.x & 31, gr = lane >> 2, c = lane & 3;
        if (s.is_a) {
#pragma unroll
            for (int q = 0; q < kSteps; ++q)
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // rank gr or gr + 8, columns 2c or 2c + 1 of the tiles
                    const int r = q * 16 + (k >> 1) * 8 + gr, o = block * 64 + (2 * c + (k & 1)) * 8;
                    float f[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = acc[q * 8 + i][k];
                    if (r < s.R && o < s.width) {
                        uint4* p = reinterpret_cast<uint4*>(s.out + (long)r * s.width + o);
                        uint4 v = pack8(f);
                        if (HIGH) {
                            const uint4 was = *p;
                            v = make_uint4(keep_finite(was.x, v.x), keep_finite(was.y, v.y), keep_finite(was.z, v.z),
                                           keep_finite(was.w, v.w));
                        }
                        *p = v;
                    }
                }
        } else if (block * 64 + gr * 8 < s.width) {
            bf16* db = s.out + (long)(block * 64 + gr * 8) * s.R;
#pragma unroll
            for (int q = 0; q < kSteps; ++q)
#pragma unroll
                for (int i = 0; i < 8; ++i) {  // tile i / 2 of 16 columns, of its rank tile i % 2
                    const int r = q * 16 + (i & 1) * 8 + 2 * c;
                    if (r < s.R) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t* p = reinterpret_cast<uint32_t*>(db + ((i >> 1) * 2 + h) * s.R + r);
                            const __nv_bfloat162 two = __floats2bfloat162_rn(acc[q * 8 + i][2 * h], acc[q * 8 + i][2 * h + 1]);
                            uint32_t v = *reinterpret_cast<const uint32_t*>(&two);
                            if (HIGH) v = keep_finite(*p, v);
                            *p = v;
                        }
                    }
                }
        }
    }
    // What is not finite once more.
    template <class Row, class Frag>
    static __device__ __noinline__ void again(const bf16* src, long ld, bf16* out, int width, int R, bool is_a, int block,
                                              int tiles, Row row, Frag frag) {
        const WeightSide s{src, ld, out, width, R, is_a};
        WeightBlock w;
        w.template sum<true>(s, block, 0, 1, tiles, row, frag);
        w.template store<true>(s, block);
    }
};

// A 16 x 16 tile of halves at `at`, its rows kLd apart: as they lie (the left operand of dx), and with the rows as the
// contraction.
template <int LD>
__device__ __forceinline__ uint4 frag_rows(const bf16* at) {
    const int lane = threadIdx.x & 31;
    const bf16* p = at + (lane >> 2) * LD + 2 * (lane & 3);
    return make_uint4(*reinterpret_cast<const uint32_t*>(p), *reinterpret_cast<const uint32_t*>(p + 8 * LD),
                      *reinterpret_cast<const uint32_t*>(p + 8), *reinterpret_cast<const uint32_t*>(p + 8 * LD + 8));
}
template <int LD>
__device__ __forceinline__ uint4 frag_trans(const bf16* at) {
    const int lane = threadIdx.x & 31;  // an 8 x 8 matrix's rows: rows 0 or 8 on of the tile, ranks 0 or 8 on
    uint32_t r[4];
    ldmatrix_trans(smem_u32(at + ((lane & 7) + (lane >> 4) * 8) * LD + (lane >> 3 & 1) * 8), r);
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// ------------------------------------------------------------------------------------------- one launch
template <int NT, int CTAS>
__global__ void __launch_bounds__(grad_threads<NT>()) lora_grad_few_kernel(const GradFewArgs g) {
    constexpr int kThreads = grad_threads<NT>(), kWarps = kThreads / 32;
    constexpr int kR = 8 * NT;                  // ranks of the tiles; g.R of them exist
    constexpr int kRp = NT == 1 ? 16 : 8 * NT;
    constexpr int kLd = grad_ld<NT>();
    constexpr int kVectors = 32 / CTAS;         // of a tile's 16 rows of d and of h, those that a CTA adds up
    extern __shared__ __align__(16) uint8_t grad_raw[];
    __shared__ int found[kWarps];
    float* recv = reinterpret_cast<float*>(grad_raw);                         // [tiles][kVectors][slots][kR]
    bf16* halves = reinterpret_cast<bf16*>(recv + max(g.tiles, kWarps / 2) * 32 * kR);  // [d, h][hi, lo][16 tiles][kLd]
    int* list = reinterpret_cast<int*>(halves + 4 * g.tiles * 16 * kLd);      // rows, -1: none
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, c = lane & 3;
    const int rank = (int)(blockIdx.x % CTAS), n = (int)(blockIdx.x / CTAS);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    pdl_wait();
    pdl_trigger();

    // the adapter's rows, in order, a thread for each row; rows without one are dealt out to all CTAs
    static_assert(kLoraGradFewRows <= kThreads, "every row has a thread");
    const int id = tid < g.T ? g.adapter[tid] : 0;
    const uint32_t eq = __ballot_sync(0xffffffffu, tid < g.T && id == n);
    if (lane == 0) found[warp] = __popc(eq);
    __syncthreads();
    int at = __popc(eq & ((1u << lane) - 1u)), count = 0;
#pragma unroll
    for (int w = 0; w < kLoraGradFewRows / 32; ++w) {
        if (w < warp) at += found[w];
        count += found[w];
    }
    const int tiles = (count + 15) / 16;
    if ((eq >> lane) & 1u) list[at] = tid;
    if (g.base != g.dx) {
        uint32_t none = __ballot_sync(0xffffffffu, (unsigned)id >= (unsigned)g.N && tid % gridDim.x == blockIdx.x);
        for (; none != 0; none &= none - 1)
            copy_row(g.base, g.ldbase, g.dx, g.lddx, warp * 32 + __ffs(none) - 1, g.K, lane, 32);
    }
    bf16* da = g.da + (long)n * g.R * g.K;
    bf16* db = g.db + (long)n * g.R * g.O;
    if (count == 0) {  // the whole cluster
        for (long i = rank * kThreads + tid; i < (long)g.R * g.K / 8; i += CTAS * kThreads)
            reinterpret_cast<uint4*>(da)[i] = zero;
        for (long i = rank * kThreads + tid; i < (long)g.R * g.O / 8; i += CTAS * kThreads)
            reinterpret_cast<uint4*>(db)[i] = zero;
        return;
    }
    if (tid < tiles * 16 - count) list[count + tid] = -1;
    if (NT == 1)  // ranks 8 to 15 of the halves
        for (int i = tid; i < 4 * tiles * 16; i += kThreads) *reinterpret_cast<uint4*>(halves + i * kLd + 8) = zero;
    __syncthreads();
    cluster_arrive();

    // d and h: 16 rows and a part of the width per item; column i of the MMA's tile j is rank NT i + j
    const bf16* a = g.a + (long)n * g.R * g.K;
    const bf16* b = g.b + (long)n * g.O * g.R;
    const int subs = grad_subs(tiles, kWarps), slots = CTAS * subs;
    bool waited = false;
    for (int it = warp; it < 2 * tiles * subs; it += kWarps) {
        const bool is_h = it < tiles * subs;
        const int tile = it / subs % tiles, part = rank * subs + it % subs;
        const int t0 = list[tile * 16 + gr], t1 = list[tile * 16 + 8 + gr];
        float acc[NT][4];
        sums16<NT>(g, a, b, is_h, t0, t1, part, slots, acc);
        if (!waited) cluster_wait();  // all CTAs of the cluster run
        waited = true;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int v = (is_h ? 16 : 0) + h * 8 + gr;
            const uint32_t dst = cluster_addr(smem_u32(recv + ((tile * kVectors + v % kVectors) * slots + part) * kR),
                                              (uint32_t)(v / kVectors));
            float f[2 * NT];
            lane_ranks<NT>(acc, h, f);
            if constexpr (NT == 1) {
                st_cluster(dst + c * 8, __float_as_uint(f[0]), __float_as_uint(f[1]));
            } else {
#pragma unroll
                for (int j = 0; j < 2 * NT; j += 4) st_cluster(dst + (2 * c * NT + j) * 4, f[j], f[j + 1], f[j + 2], f[j + 3]);
            }
        }
    }
    if (!waited) cluster_wait();
    cluster_arrive();
    cluster_wait();

    // the sums of this CTA's vectors, four ranks a thread, to all
    const float sc = g.scale != nullptr ? g.scale[n] : 1.0f;
    for (int i = tid; i < tiles * kVectors * (kR / 4); i += kThreads) {
        const int q = i % (kR / 4) * 4, v = i / (kR / 4), tile = v / kVectors, owned = rank * kVectors + v % kVectors;
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < slots; ++k) {
            const float4 p = *reinterpret_cast<const float4*>(recv + (v * slots + k) * kR + q);
            s.x += p.x, s.y += p.y, s.z += p.z, s.w += p.w;
        }
        const int row = tile * 16 + (owned & 15);
        const bool keep = q < g.R && list[row] >= 0;  // the padding is 0 whatever the rows hold
        bf16 hi[4], lo[4];
        split2(keep ? s.x * sc : 0.0f, hi, lo);
        split2(keep ? s.y * sc : 0.0f, hi + 1, lo + 1);
        split2(keep ? s.z * sc : 0.0f, hi + 2, lo + 2);
        split2(keep ? s.w * sc : 0.0f, hi + 3, lo + 3);
        auto two = [](bf16 u, bf16 w) { return (uint32_t)__bfloat16_as_ushort(u) | (uint32_t)__bfloat16_as_ushort(w) << 16; };
        const uint32_t to = smem_u32(halves + ((owned >> 4) * 2 * tiles * 16 + row) * kLd + q);
#pragma unroll
        for (int k = 0; k < CTAS; ++k) {
            st_cluster(cluster_addr(to, k), two(hi[0], hi[1]), two(hi[2], hi[3]));
            st_cluster(cluster_addr(to + tiles * 16 * kLd * 2, k), two(lo[0], lo[1]), two(lo[2], lo[3]));
        }
    }
    cluster_arrive();
    cluster_wait();

    // 64 columns of dA, dB or dx per item: dA and dB first, dx in as many parts of the rows as there are warps left for
    const int half = tiles * 16 * kLd, kb = (g.K + 63) / 64, ob = (g.O + 63) / 64;
    const bf16 *dh = halves, *hh = halves + 2 * half;  // [hi, lo][16 tiles][kLd]
    const int parts = max(1, min(tiles, (CTAS * kWarps - kb - ob) / kb));
    for (int it = rank * kWarps + warp; it < kb + ob + parts * kb; it += CTAS * kWarps) {
        if (it < kb + ob) {
            const bool is_a = it < kb;
            const int block = is_a ? it : it - kb;
            const bf16* from = is_a ? dh : hh;
            WeightBlock<NT, false> w;
            const WeightSide s{is_a ? g.x : g.dy, is_a ? g.ldx : g.lddy, is_a ? da : db, is_a ? g.K : g.O, g.R, is_a};
            auto row = [&](int i) { return list[i]; };
            auto frag = [&](int tile, int hl, int q) { return frag_trans<kLd>(from + hl * half + tile * 16 * kLd + q * 16); };
            w.template sum<false>(s, block, 0, 1, tiles, row, frag);
            w.template store<false>(s, block);
            if (any_not_finite(w.acc)) {  // once more
                w.template sum<true>(s, block, 0, 1, tiles, row, frag);
                w.template store<true>(s, block);
            }
        } else {
            const int block = (it - kb - ob) % kb;
            RankRows<NT> w;
            w.load(a, g.R, g.K, block);
            for (int tile = (it - kb - ob) / kb; tile < tiles; tile += parts) {
                RowsOfDx r;
                r.t[0] = list[tile * 16 + gr], r.t[1] = list[tile * 16 + 8 + gr];
                r.load(g, block);
                r.finish<NT>(g, block, w, [dh, half, tile](int hl, int q) {
                    return frag_rows<kLd>(dh + hl * half + tile * 16 * kLd + q * 16);
                });
            }
        }
    }
}

// ------------------------------------------------------------------------------------------- three launches
// d and h of the plan's groups, 16 rows each, as the fragments that the last launch's MMAs take: [group][d with its rows as the
// contraction, d as its rows lie, h with its rows as the contraction][hi, lo][step of 16 ranks][lane].
constexpr int kGroupThreads = 256;
constexpr int kGroupWarps = kGroupThreads / 32;
template <int NT>
__global__ void __launch_bounds__(kGroupThreads) lora_grad_hidden_kernel(const GradFewArgs g, const LoraPlan plan, uint4* frags) {
    constexpr int kThreads = kGroupThreads, kWarps = kGroupWarps;
    constexpr int kR = 8 * NT, kLd = grad_ld<NT>(), kSteps = NT == 1 ? 1 : NT / 2;
    extern __shared__ __align__(16) uint8_t grad_raw[];
    float* red = reinterpret_cast<float*>(grad_raw);                       // [warps][16][kR]
    bf16* halves = reinterpret_cast<bf16*>(red + kWarps * 16 * kR);        // [hi, lo][16][kLd]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, c = lane & 3;
    const int group = (int)(blockIdx.x >> 1);
    const bool is_h = blockIdx.x & 1;
    if (NT == 1 && tid < 32) *reinterpret_cast<uint4*>(halves + tid * kLd + 8) = make_uint4(0, 0, 0, 0);
    pdl_wait();
    pdl_trigger();
    if (group >= *plan.ngroups) return;
    const int2 e = plan.groups[group];
    const int n = e.y >> 8, count = e.y & 255;
    const int t0 = gr < count ? plan.rows[e.x + gr] : -1, t1 = gr + 8 < count ? plan.rows[e.x + gr + 8] : -1;
    float acc[NT][4];
    sums16<NT>(g, g.a + (long)n * g.R * g.K, g.b + (long)n * g.O * g.R, is_h, t0, t1, warp, kWarps, acc);
    const float sc = g.scale != nullptr ? g.scale[n] : 1.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float f[2 * NT];
        lane_ranks<NT>(acc, h, f);
#pragma unroll
        for (int j = 0; j < NT; ++j)
            *reinterpret_cast<float2*>(red + (warp * 16 + h * 8 + gr) * kR + 2 * c * NT + 2 * j) =
                make_float2(f[2 * j], f[2 * j + 1]);
    }
    __syncthreads();
    for (int i = tid; i < 16 * kR; i += kThreads) {
        const int row = i / kR, r = i % kR;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += red[(w * 16 + row) * kR + r];
        split2(row < count && r < g.R ? v * sc : 0.0f, halves + row * kLd + r, halves + (16 + row) * kLd + r);
    }
    __syncthreads();
    uint4* out = frags + (long)group * 6 * kSteps * 32 + lane;
    for (int i = warp; i < 2 * kSteps; i += kWarps) {  // half and step
        const bf16* at = halves + i / kSteps * 16 * kLd + i % kSteps * 16;
        out[((is_h ? 4 : 0) * kSteps + i) * 32] = frag_trans<kLd>(at);
        if (!is_h) out[(2 * kSteps + i) * 32] = frag_rows<kLd>(at);
    }
}

// All column blocks: CTAs for dA and dB first, then for dx. SPLIT warps of a CTA share a block of dA or dB, each with every
// SPLIT-th 16 rows, and add up through shared memory.
template <int NT, int SPLIT>
__global__ void __launch_bounds__(kGroupThreads, 2) lora_grad_finish_kernel(const GradFewArgs g, const LoraPlan plan,
                                                                           const uint4* frags, int weight_ctas) {
    constexpr int kSteps = NT == 1 ? 1 : NT / 2, kAcc = kSteps * 8;
    constexpr int kBlocks = kGroupWarps / SPLIT;
    extern __shared__ __align__(16) uint8_t grad_raw[];
    float4* red = reinterpret_cast<float4*>(grad_raw);  // [blocks][SPLIT - 1][kAcc][32]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2;
    const int kb = (g.K + 63) / 64, ob = (g.O + 63) / 64;
    if (g.base != g.dx) {  // rows without an adapter, dealt out to all warps; adapters and base were there before the plan
        const long warps = (long)gridDim.x * kGroupWarps;
        for (long t = (long)blockIdx.x * kGroupWarps + warp; t < g.T; t += warps)
            if ((unsigned)__ldcg(g.adapter + t) >= (unsigned)g.N) copy_row(g.base, g.ldbase, g.dx, g.lddx, t, g.K, lane, 32);
    }
    if ((int)blockIdx.x < weight_ctas) {
        const int per = (kb + ob + kBlocks - 1) / kBlocks;
        const int n = (int)blockIdx.x / per, it = (int)blockIdx.x % per * kBlocks + warp / SPLIT, part = warp % SPLIT;
        const bool live = it < kb + ob, is_a = it < kb;
        const int block = is_a ? it : it - kb;
        const int first = __ldcg(plan.first + n), rows = __ldcg(plan.units + n), tiles = live ? (rows + 15) / 16 : 0;
        const int32_t* at = plan.rows + (rows > 0 ? __ldcg(&plan.groups[first].x) : 0);
        pdl_wait();
        pdl_trigger();
        const uint4* f = frags + ((long)first * 6 + (is_a ? 0 : 4)) * kSteps * 32 + lane;
        WeightBlock<NT, true> w;
        auto row = [at, rows](int i) { return i < rows ? __ldcg(at + i) : -1; };
        auto frag = [f](int tile, int hl, int q) { return __ldcg(f + ((long)tile * 6 * kSteps + hl * kSteps + q) * 32); };
        const WeightSide s{is_a ? g.x : g.dy, is_a ? g.ldx : g.lddy, (is_a ? g.da : g.db) + (long)n * g.R * (is_a ? g.K : g.O),
                           is_a ? g.K : g.O, g.R, is_a};
        w.template sum<false>(s, block, part, SPLIT, tiles, row, frag);
        if (SPLIT > 1) {
            float4* mine = red + warp / SPLIT * (SPLIT - 1) * kAcc * 32 + lane;
            if (part > 0) {
#pragma unroll
                for (int i = 0; i < kAcc; ++i)
                    mine[((part - 1) * kAcc + i) * 32] = make_float4(w.acc[i][0], w.acc[i][1], w.acc[i][2], w.acc[i][3]);
            }
            __syncthreads();
            if (part > 0) return;
            for (int p = 0; p < SPLIT - 1; ++p)
#pragma unroll
                for (int i = 0; i < kAcc; ++i) {
                    const float4 v = mine[(p * kAcc + i) * 32];
                    w.acc[i][0] += v.x, w.acc[i][1] += v.y, w.acc[i][2] += v.z, w.acc[i][3] += v.w;
                }
        }
        if (!live) return;
        w.template store<false>(s, block);
        if (any_not_finite(w.acc)) w.again(s.src, s.ld, s.out, s.width, s.R, is_a, block, tiles, row, frag);
        return;
    }
    const int per = (kb + kGroupWarps - 1) / kGroupWarps;
    const int group = ((int)blockIdx.x - weight_ctas) / per, block = ((int)blockIdx.x - weight_ctas) % per * kGroupWarps + warp;
    const bool live = group < __ldcg(plan.ngroups) && block < kb;
    RankRows<NT> w;
    RowsOfDx r;
    if (live) {
        const int2 e = __ldcg(&plan.groups[group]);
        r.t[0] = gr < (e.y & 255) ? __ldcg(plan.rows + e.x + gr) : -1;
        r.t[1] = gr + 8 < (e.y & 255) ? __ldcg(plan.rows + e.x + gr + 8) : -1;
        w.load(g.a + (long)(e.y >> 8) * g.R * g.K, g.R, g.K, block);
        r.load(g, block);
    }
    pdl_wait();
    pdl_trigger();
    if (!live) return;
    const uint4* f = frags + ((long)group * 6 + 2) * kSteps * 32 + lane;
    r.finish<NT>(g, block, w, [f](int hl, int q) { return __ldcg(f + (hl * kSteps + q) * 32); });
}

template <int NT, int SPLIT>
cudaError_t launch_finish(const GradFewArgs& g, const LoraPlan& plan, const uint4* frags, int groups, cudaStream_t s) {
    constexpr int kBlocks = kGroupWarps / SPLIT;
    constexpr size_t smem = (size_t)kBlocks * (SPLIT - 1) * (NT == 1 ? 8 : NT * 4) * 32 * sizeof(float4);
    const int kb = (g.K + 63) / 64, ob = (g.O + 63) / 64;
    const int weights = g.N * ((kb + ob + kBlocks - 1) / kBlocks), rows = groups * ((kb + kGroupWarps - 1) / kGroupWarps);
    static_assert(smem <= (48 << 10), "within the limit that needs no asking");
    return launch_pdl(lora_grad_finish_kernel<NT, SPLIT>, dim3((unsigned)(weights + rows)), dim3(kGroupThreads), smem, s, g, plan,
                      frags, weights);
}

template <int NT>
cudaError_t launch_groups(const GradFewArgs& g, const LoraPlan& plan, uint4* frags, int sms, cudaStream_t s) {
    constexpr size_t smem = sizeof(float) * kGroupWarps * 16 * 8 * NT + 2 * 2 * 16 * grad_ld<NT>();
    const int groups = lora_max_groups(g.T, g.N);
    static_assert(smem <= (48 << 10), "within the limit that needs no asking");
    PM_TRY(launch_pdl(lora_grad_hidden_kernel<NT>, dim3((unsigned)groups * 2), dim3(kGroupThreads), smem, s, g, plan, frags));
    // sharing where column blocks of all adapters are few: 512 rows of one of 64 adapters 24 us with four warps to a block, 31 us
    // with one, but 27 and 17 where the 64 have them all
    const int blocks = (g.K + 63) / 64 + (g.O + 63) / 64;
    return (long)g.N * blocks <= 8L * sms ? launch_finish<NT, 4>(g, plan, frags, groups, s)
                                          : launch_finish<NT, 1>(g, plan, frags, groups, s);
}

template <int NT, int CTAS>
cudaError_t launch_as(const GradFewArgs& g, cudaStream_t s) {
    constexpr int kRows = kGradFewRowRanks / (NT == 1 ? 8 : NT * 4 + 8);  // ranks from there on have these tiles
    constexpr size_t most = grad_smem<NT>((std::min(kRows, kLoraGradFewRows) + 15) / 16);
    static std::atomic<bool> configured[64];
    PM_TRY(raise_smem((const void*)lora_grad_few_kernel<NT, CTAS>, most, configured));
    return launch_cluster(lora_grad_few_kernel<NT, CTAS>, dim3((unsigned)g.N * CTAS), dim3(grad_threads<NT>()), CTAS,
                          grad_smem<NT>(g.tiles), s, g);
}

template <int CTAS>
cudaError_t launch_ranks(const GradFewArgs& g, cudaStream_t s) {
    if (g.R <= 8) return launch_as<1, CTAS>(g, s);
    if (g.R <= 16) return launch_as<2, CTAS>(g, s);
    if (g.R <= 32) return launch_as<4, CTAS>(g, s);
    return launch_as<8, CTAS>(g, s);
}

}  // namespace

bool lora_grad_is_few(int T, int R, int N) {
    return R <= 64 && T <= (N <= kGradFewAdapters ? kLoraGradFewRows : kLoraGradFewRows / 2) && T * R <= kGradFewRowRanks;
}
bool lora_grad_is_grouped(int T, int R, int N) { return T <= std::max(kGradGroupedRows, kGradGroupedEach * N) && R <= 16; }

cudaError_t launch_lora_grad_few(const LoraGradFew& f, const LoraShape& h, int sms, cudaStream_t s) {
    const GradFewArgs g{f, h.T, h.K, h.O, h.R, h.N, (h.T + 15) / 16};
    // as many CTAs for each adapter as can be there together (100 rows of 64 adapters with eight, four and two: 26, 16, 12 us; 64
    // rows of 4: 9.4, 12.6, 17); a part of the GPU takes one or two clusters of eight SMs, so not sms / 8 of them
    if (h.N * 10 <= sms) return launch_ranks<8>(g, s);
    return h.N * 4 <= sms ? launch_ranks<4>(g, s) : launch_ranks<2>(g, s);
}

size_t lora_frag_bytes(int T, int N) { return (size_t)lora_max_groups(T, N) * 6 * 32 * sizeof(uint4); }

cudaError_t launch_lora_grad_groups(const LoraGradFew& f, const LoraShape& h, const LoraPlan& p, void* frags, int sms,
                                    cudaStream_t s) {
    const GradFewArgs g{f, h.T, h.K, h.O, h.R, h.N, 0};
    return h.R <= 8 ? launch_groups<1>(g, p, (uint4*)frags, sms, s) : launch_groups<2>(g, p, (uint4*)frags, sms, s);
}

}  // namespace pm
