// kq_attn.cuh -- what the two attention kernels share: the geometry of a
// request, the split of the work over the grid, and the join of split rows.
//
// A request with n new tokens of L in all is n * G packed rows for each of its
// kv heads (row r is token r / G, query head h * G + r % G), so the query heads
// that share a kv head read its keys once.  Row r sees the keys
// [limit - window, limit), limit = L - n + r / G + 1.
#pragma once
#include <math.h>

#include "kq_ptx.cuh"
#include "kq_serve.cuh"

namespace kq {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Request {
    int q0, n, len;
};

// Request b of the call; b == B stands for the padding tokens behind the last
// one (no keys: their rows are written as empty).  Lengths that contradict the
// buffers are cut to them and reported.  Where offsets descend (descends) requests share
// tokens, and may be more work than the host's bound of it: the kernels then write every
// row as empty (write_empty) and take no request.
__device__ __forceinline__ Request load_request(const AttnArgs &a, int b, bool &bad) {
    Request r;
    const int c0 = a.cu[b], c1 = b < a.B ? a.cu[b + 1] : a.T;
    const int s = b < a.B ? a.seq[b] : 0;
    r.q0 = min(max(c0, 0), a.T);
    const int e = min(max(c1, r.q0), a.T);
    r.n = e - r.q0;
    r.len = min(max(s, 0), a.max_len);
    bad |= r.q0 != c0 || e != c1 || r.len != s;
    return r;
}
__device__ __forceinline__ bool descends(const AttnArgs &a, int b) { return b < a.B && a.cu[b + 1] < a.cu[b]; }

// All rows of the call as rows without keys, by the whole grid.
__device__ __forceinline__ void write_empty(const AttnArgs &a) {
    const int64_t rows = (int64_t)a.T * a.Hq, first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = first; i < rows * (a.D / 8); i += step) reinterpret_cast<uint4 *>(a.out)[i] = make_uint4(0, 0, 0, 0);
    if (a.lse)
        for (int64_t i = first; i < rows; i += step) a.lse[i] = -INFINITY;
}

// Keys [lo, hi) that the rows of tokens [t0, t1) of a request can see.
__device__ __forceinline__ void key_range(const AttnArgs &a, const Request &r, int t0, int t1, int &lo, int &hi) {
    hi = a.causal ? max(0, r.len - r.n + t1) : r.len;
    lo = a.window ? max(0, r.len - r.n + t0 + 1 - a.window) : 0;
    lo = min(lo, hi);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Capped scores in units of log2: out * tanh(u), u = x * in.  Up to |u| = CAP_NEAR the tanh
// is an odd polynomial u (k0 + u^2 (k1 + u^2 (k2 + u^2 k3))), fitted by exchange of the
// extrema (largest relative error 1.5e-7): there 1 - 2 / (1 + e^2u) cancels, and the score
// would err by 2^-22 of the cap however small it is (a cap of 1e5 on scores of a few units:
// probabilities 1.4 % off).  Beyond, 1 - 2 / (1 + e^2u) is good to some 2^-21 of itself (the
// hardware's tanh to 2^-11 only).
constexpr float CAP_NEAR = 0.4f;
constexpr float CAP_K0 = 0.9999998807907104f, CAP_K1 = -0.33331361413002014f, CAP_K2 = 0.13270977139472961f,
                CAP_K3 = -0.04755360260605812f;
struct Cap {
    float in, lin, out;  // lin = in * out, by itself: `in` may be too small for f32, `out` too large
};
__host__ __device__ __forceinline__ Cap make_cap(float scale, float softcap) {
    // (an `in` above 1e30 belongs to a cap so small that every capped score is 0)
    return Cap{fminf(scale / softcap, 1e30f), scale * LOG2E, softcap * LOG2E};
}
__device__ __forceinline__ float cap_near(float x, const Cap &c) {
    const float u = x * c.in, v = u * u;
    return x * c.lin * fmaf(v, fmaf(v, fmaf(v, CAP_K3, CAP_K2), CAP_K1), CAP_K0);
}
__device__ __forceinline__ float soft_cap(float x, const Cap &c) {
    const float u = x * c.in;
    if (fabsf(u) <= CAP_NEAR) return cap_near(x, c);
    return c.out * (1.0f - __fdividef(2.0f, 1.0f + ex2(u * (2.0f * LOG2E))));
}

// Inclusive scan of a count a thread over the block, the total, and whether any thread has
// `flag` set: then the counts are of no use, and a warp's sum of all ones, which no count
// comes near, says so (a reducing barrier took 0.3 us more of a single token's 7.2).
// U is 32 bits wide wherever the host can bound the total (a 64-bit scan takes twice the
// shuffles, and a 64-bit division some 400 clocks, each of them on the path of a single token).
template <int N, class U> __device__ __forceinline__ U block_scan(U mine, U *s_warp, U &total, bool &flag) {
    static_assert(N % 32 == 0 && N <= 1024, "whole warps");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    U v = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const U u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (__any_sync(0xffffffffu, flag)) v = ~(U)0;
    if (lane == 31) s_warp[warp] = v;
    __syncthreads();
    U w = lane < N / 32 ? s_warp[lane] : 0;
    flag = __any_sync(0xffffffffu, w == ~(U)0);
#pragma unroll
    for (int o = 1; o < N / 32; o <<= 1) {
        const U u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += u;
    }
    total = __shfl_sync(0xffffffffu, w, N / 32 - 1);
    const U below = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    return v + (warp ? below : 0);
}

// The same for two counts at once.
template <int N, class U> __device__ __forceinline__ void block_scan2(U &v, U &x, U *s_warp, U &total_v, U &total_x, bool &flag) {
    static_assert(N % 32 == 0 && N <= 1024, "whole warps");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const U a = __shfl_up_sync(0xffffffffu, v, o), b = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) v += a, x += b;
    }
    if (__any_sync(0xffffffffu, flag)) v = ~(U)0;
    if (lane == 31) s_warp[warp] = v, s_warp[32 + warp] = x;
    __syncthreads();
    U w = lane < N / 32 ? s_warp[lane] : 0, y = lane < N / 32 ? s_warp[32 + lane] : 0;
    flag = __any_sync(0xffffffffu, w == ~(U)0);
#pragma unroll
    for (int o = 1; o < N / 32; o <<= 1) {
        const U a = __shfl_up_sync(0xffffffffu, w, o), b = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) w += a, y += b;
    }
    total_v = __shfl_sync(0xffffffffu, w, N / 32 - 1), total_x = __shfl_sync(0xffffffffu, y, N / 32 - 1);
    const U below_v = __shfl_sync(0xffffffffu, w, max(warp - 1, 0)), below_x = __shfl_sync(0xffffffffu, y, max(warp - 1, 0));
    if (warp) v += below_v, x += below_x;
}

// Unit u of `total` belongs to block ((u + 1) * grid - 1) / total, when block c
// takes the units [c * total / grid, (c + 1) * total / grid).
template <class U> __device__ __forceinline__ U unit_begin(U total, int c, int grid) { return total * (U)c / (U)grid; }
template <class U> __device__ __forceinline__ int unit_block(U total, U u, int grid) { return (int)(((u + 1) * (U)grid - 1) / total); }
// Whether unit counts up to `most` may be 32 bits wide (their products with the grid too).
inline bool units_fit32(int64_t most, int grid) { return most >= 0 && most < (int64_t)(0xffffffffu / (unsigned)grid) - 1; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool full) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <bool F16> __device__ __forceinline__ uint32_t pack_half(float x, float y) {
    uint32_t v;
    if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(y), "f"(x));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(y), "f"(x));
    return v;
}

}  // namespace kq
