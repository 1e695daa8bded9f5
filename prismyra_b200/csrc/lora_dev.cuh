// Device helpers of the adapter kernels: 16-byte asynchronous copies, cluster shared memory, and the two-halves form of the
// values between the two products.
#pragma once

#include "ptx.cuh"

namespace pm {

// 16 bytes (zeros unless valid); the 256 bytes around them go to L2 (a row's next columns are wanted soon).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Arrive (once for this thread) on an mbarrier when every cp.async it has issued so far has completed. Whoever waits on the
// barrier sees the copies; before the tensor core reads them it has to pass a proxy fence, which the waiting thread issues
// (in the copying threads the same fence would hold up the copies still in flight: 1000 cycles a step).
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_addr(uint32_t smem, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float a, float b, float c, float d) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d)
                 : "memory");
}

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t a, uint32_t b) {
    asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
// The warp's 16 x 16 by 16 x 8 product, for rows too few for the tensor core's 128.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A value as the sum of two bf16: hi rounded to nearest (to zero where that would overflow), lo what is left: together 16
// significant bits. A value that is not finite stays whole in hi.
__device__ __forceinline__ void split2(float v, __nv_bfloat16* hi, __nv_bfloat16* lo) {
    __nv_bfloat16 h = __float2bfloat16_rn(v);
    if (__hisinf(h) != 0) h = __float2bfloat16_rz(v);
    const float f = __bfloat162float(h);
    *hi = h;
    *lo = fabsf(f) <= 3.4e38f ? __float2bfloat16_rn(v - f) : __float2bfloat16_rn(0.0f);
}

// An infinite operand times a low half is NaN (a half of 0) or infinite of the other sign. So where the sum over both halves is
// not finite, the high halves' alone is the result: a high half has its value's sign, and is 0 only where the value is (or
// below 2^-134). The kernels look at what they have made and, where something is not finite, make it once more.
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }
__device__ __forceinline__ float both_halves(float both, float high) { return finite(both) ? both : high; }
// Whether one of a warp's sums is not finite.
__device__ __forceinline__ bool any_not_finite(const float (&v)[4]) {
    const float z = fmaf(v[0], 0.0f, v[1] * 0.0f) + fmaf(v[2], 0.0f, v[3] * 0.0f);
    return __any_sync(0xffffffffu, !(z == 0.0f)) != 0;
}
template <int M>
__device__ __forceinline__ bool any_not_finite(const float (&v)[M][4]) {
    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = fmaf(v[i][e], 0.0f, z[e]);
    return any_not_finite(z);
}
// The same for results, pairs of bf16, collected one by one.
struct Unusual {
    __nv_bfloat162 z[2];
    __device__ __forceinline__ Unusual() : z{__nv_bfloat162(0.0f, 0.0f), __nv_bfloat162(0.0f, 0.0f)} {}
    __device__ __forceinline__ void see(uint32_t pair, int i) {
        z[i] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&pair), __nv_bfloat162(0.0f, 0.0f), z[i]);
    }
    __device__ __forceinline__ void see(const uint4& v) { see(v.x, 0), see(v.y, 1), see(v.z, 0), see(v.w, 1); }
    __device__ __forceinline__ bool any() const {
        const __nv_bfloat162 s = __hadd2(z[0], z[1]);
        return __any_sync(0xffffffffu, (*reinterpret_cast<const uint32_t*>(&s) & 0x7fff7fffu) != 0u) != 0;
    }
};

// Eight values as their halves.
__device__ __forceinline__ void split8(const float (&v)[8], uint4* hi, uint4* lo) {
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(hi);
    __nv_bfloat162* l = reinterpret_cast<__nv_bfloat162*>(lo);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        split2(v[2 * i], &h[i].x, &l[i].x);
        split2(v[2 * i + 1], &h[i].y, &l[i].y);
    }
}

// Row t of a result that is base (zeros where there is none), by `step` threads: `from` is this one's place. Eight pieces are
// read before the first is written: base and out may be the same memory for all that the compiler knows.
__device__ __forceinline__ void copy_row(const __nv_bfloat16* base, long ldbase, __nv_bfloat16* out, long ldout, long t,
                                         int width, int from, int step) {
    for (int col = from * 8; col < width; col += step * 64) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = base != nullptr && col + i * step * 8 < width
                       ? __ldcg(reinterpret_cast<const uint4*>(base + t * ldbase + col + i * step * 8))
                       : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i * step * 8 < width) *reinterpret_cast<uint4*>(out + t * ldout + col + i * step * 8) = v[i];
    }
}

// Two bf16 plus two fp32, rounded once each.
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t y, float a, float b) {
    const __nv_bfloat162 o = __floats2bfloat162_rn(__uint_as_float(y << 16) + a, __uint_as_float(y & 0xffff0000u) + b);
    return *reinterpret_cast<const uint32_t*>(&o);
}

}  // namespace pm
