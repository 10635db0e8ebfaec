// kq_serve.cu -- the small operators of a serving step around the projections:
// the plan of the paged batch, rotary embedding with the cache write, and the
// routing of tokens to experts.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kq_serve.cuh"

namespace kq {
namespace {

// Sums of counts stop at PLAN_CAP instead of wrapping, so contradictory lengths
// still give ascending scans and every search stays inside its array.
__device__ __forceinline__ int sat_add(int x, int y) { return min(x + y, PLAN_CAP); }

__device__ __forceinline__ int warp_incl_scan(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = sat_add(v, u);
    }
    return v;
}

// --------------------------------------------------------------------------
// paged plan
//
// Request b holds ceil(ctx / page) pages and needs ceil((ctx + new) / page); the
// missing ones are handed out from the free list in request order, so an
// exclusive scan of the needs gives each request its first free entry, as a
// scan of the new-token counts gives its first token.  Both scans are small
// (a few KB of lengths), so every block does them whole in shared memory and
// then takes its share of the tokens and of the new table entries, each found
// by a binary search in the scanned arrays: one launch, nothing between blocks.
// A table entry that this step writes is never read by it (tokens on a new
// page take its id from the free list), so the blocks need no order.
// Bound: launch and latency, two dependent rounds of loads and the scan: 64
// requests of one token 3.9 us, 1000 requests and 44,000 tokens 5.6 us, of which
// the launch itself is some 2.3.
constexpr int PLAN_T = 1024;

__device__ __forceinline__ int upper_bound(const int *a, int n, int v) {  // entries <= v
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PLAN_T) plan_kernel(const PlanArgs a) {
    extern __shared__ int s_plan[];  // token_end[B], need_end[B]
    int *s_tok = s_plan, *s_need = s_plan + a.B;
    __shared__ int s_wt[32], s_wn[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int base_t = 0, base_n = 0, bad = 0;  // contradictory lengths (every block sees them) before missing pages
    for (int b0 = 0; b0 < a.B; b0 += PLAN_T) {
        const int b = b0 + tid;
        int n = 0, need = 0;
        if (b < a.B) {
            int ctx = a.ctx[b];
            n = a.qlen[b];
            if (ctx < 0 || n < 0 || n > a.T || (int64_t)ctx + n > 0x7fffffff) bad = ERR_LENGTHS, ctx = 0, n = 0;
            need = min((int)(((int64_t)ctx + n + a.page - 1) / a.page - ((int64_t)ctx + a.page - 1) / a.page), PLAN_CAP);
            if (blockIdx.x == 0) a.seq[b] = ctx + n;
        }
        const int it = warp_incl_scan(n, lane), in = warp_incl_scan(need, lane);
        if (lane == 31) s_wt[warp] = it, s_wn[warp] = in;
        __syncthreads();
        if (warp == 0) {
            const int st = warp_incl_scan(s_wt[lane], lane), sn = warp_incl_scan(s_wn[lane], lane);
            s_wt[lane] = st, s_wn[lane] = sn;
        }
        __syncthreads();
        if (b < a.B) {
            s_tok[b] = sat_add(base_t, sat_add(it, warp ? s_wt[warp - 1] : 0));
            s_need[b] = sat_add(base_n, sat_add(in, warp ? s_wn[warp - 1] : 0));
            if (blockIdx.x == 0) {
                a.cu[b + 1] = s_tok[b];
                if (b == 0) a.cu[0] = 0;
            }
        }
        base_t = sat_add(base_t, s_wt[31]), base_n = sat_add(base_n, s_wn[31]);
        __syncthreads();
    }
    const int stride = gridDim.x * PLAN_T, first = blockIdx.x * PLAN_T + tid;
    if (first == 0) {
        a.used[0] = base_n;
        if (a.B == 0) a.cu[0] = 0;
    }
    bad = __syncthreads_or(bad || base_t > a.T) ? ERR_LENGTHS : 0;
    for (int e = first; e < base_n; e += stride) {  // new table entries
        const int b = upper_bound(s_need, a.B, e);
        const int col = (int)(((int64_t)a.ctx[b] + a.page - 1) / a.page) + e - (b ? s_need[b - 1] : 0);
        if (!bad && (e >= a.n_free || col >= a.table_width)) bad = ERR_PAGES;
        if (col < a.table_width) a.table[b * a.table_stride + col] = e < a.n_free ? a.free_pages[e] : -1;
    }
    for (int t = first; t < a.T; t += stride) {  // tokens; those past the last request are padding
        int64_t slot = -1;
        int pos = 0;
        if (t < base_t) {
            const int b = upper_bound(s_tok, a.B, t), ctx = a.ctx[b];
            pos = ctx + t - (b ? s_tok[b - 1] : 0);
            const int held = (int)(((int64_t)ctx + a.page - 1) / a.page), col = pos / a.page;
            int id = -1;
            if (col < held) {
                if (col < a.table_width) id = a.table[b * a.table_stride + col];
            } else {
                const int e = (b ? s_need[b - 1] : 0) + col - held;
                if (e < a.n_free && col < a.table_width) id = a.free_pages[e];
            }
            if (id >= 0) slot = (int64_t)id * a.page + (pos - col * a.page);
            else if (!bad) bad = ERR_PAGES;
        }
        a.slots[t] = slot;
        a.pos[t] = pos;
    }
    if (bad) atomicCAS(a.err, 0, bad);
}

// --------------------------------------------------------------------------
// rotary embedding + cache write

template <bool F16> struct Half;
template <> struct Half<true> {
    static __device__ __forceinline__ float2 up(uint32_t v) { return __half22float2(*reinterpret_cast<__half2 *>(&v)); }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&h);
    }
};
template <> struct Half<false> {
    static __device__ __forceinline__ float2 up(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&h);
    }
};

// One task is two 16-byte vectors of a head: a half-split rotation pairs value
// i with i + rot/2, so the task takes the same eight values of both halves; an
// interleaved one pairs neighbours, so it takes sixteen values in a row; past
// `rot`, and for v, it copies sixteen values.  A thread keeps its place in the
// head, and with it its eight angles, for all of its heads of a token; all of
// its loads are issued before the first is used, and what hangs on position and
// slot (angles, the cache row) is looked up behind them.
// Out of (a, b) come a cos - b sin and b cos + a sin, in f32 and rounded once.
// Bound: HBM.  8192 tokens of 32 + 8 + 8 heads of 128: 206 MB in 37.0 us, 5.55 TB/s
// (85 % of a plain copy's rate, of which 2.3 us are the launch); one token 2.3 us.
constexpr int ROPE_T = 128, ROPE_U = 4;

template <bool F16>
__global__ void __launch_bounds__(ROPE_T) rope_kernel(const RopeArgs a) {
    const int nc = a.D >> 4, per = ROPE_T / nc;  // tasks a head, heads a pass
    const int c = threadIdx.x % nc, h0 = threadIdx.x / nc;
    if (h0 >= per) return;
    const int heads = a.Hq + 2 * a.Hk;
    const int64_t t = blockIdx.x;
    const bool turn = c < (a.rot >> 4);
    const int half = a.rot >> 1;
    const int e0 = turn ? (a.interleaved ? c * 16 : c * 8) : c * 16, e1 = turn && !a.interleaved ? half + c * 8 : e0 + 8;
    int pos = a.pos[t];
    int64_t slot = a.slots[t];
    bool bad = false;
    float cs[8], sn[8];
    int64_t cache_row = 0;
    const uint16_t *q = reinterpret_cast<const uint16_t *>(a.q) + t * a.q_ts, *k = reinterpret_cast<const uint16_t *>(a.k) + t * a.k_ts,
                   *v = reinterpret_cast<const uint16_t *>(a.v) + t * a.v_ts;
    const int step = per * gridDim.y;
    const int first = blockIdx.y * per + h0;
    for (int hb = first; hb < heads; hb += step * ROPE_U) {
        uint4 x0[ROPE_U], x1[ROPE_U];
#pragma unroll
        for (int u = 0; u < ROPE_U; u++) {
            const int h = hb + u * step;
            if (h < heads) {
                const uint16_t *src = h < a.Hq ? q + h * a.q_hs : h < a.Hq + a.Hk ? k + (h - a.Hq) * a.k_hs : v + (h - a.Hq - a.Hk) * a.v_hs;
                const int o1 = h < a.Hq + a.Hk ? e1 : c * 16 + 8, o0 = h < a.Hq + a.Hk ? e0 : c * 16;
                x0[u] = *reinterpret_cast<const uint4 *>(src + o0);
                x1[u] = *reinterpret_cast<const uint4 *>(src + o1);
            }
        }
        if (hb == first) {  // what hangs on position and slot, behind loads that do not
            if (pos < 0 || pos >= a.n_pos) bad = true, pos = pos < 0 ? 0 : a.n_pos - 1;
            if (slot >= a.n_slots) bad = true, slot = -1;
            if (turn) {
                const float4 *pc = reinterpret_cast<const float4 *>(a.cos + (int64_t)pos * half + c * 8);
                const float4 *ps = reinterpret_cast<const float4 *>(a.sin + (int64_t)pos * half + c * 8);
                *reinterpret_cast<float4 *>(cs) = pc[0], *reinterpret_cast<float4 *>(cs + 4) = pc[1];
                *reinterpret_cast<float4 *>(sn) = ps[0], *reinterpret_cast<float4 *>(sn + 4) = ps[1];
            }
            // (a 64-bit division takes some 400 clocks)
            if (slot >> 32) cache_row = slot < 0 ? 0 : (slot / a.page) * a.page_stride + (slot % a.page) * a.row_stride;
            else cache_row = ((uint32_t)slot / (uint32_t)a.page) * a.page_stride + ((uint32_t)slot % (uint32_t)a.page) * a.row_stride;
        }
#pragma unroll
        for (int u = 0; u < ROPE_U; u++) {
            const int h = hb + u * step;
            if (h >= heads) continue;
            const bool is_v = h >= a.Hq + a.Hk;
            if (turn && !is_v) {
                uint32_t w[8] = {x0[u].x, x0[u].y, x0[u].z, x0[u].w, x1[u].x, x1[u].y, x1[u].z, x1[u].w};
                if (a.interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float2 p = Half<F16>::up(w[i]);
                        w[i] = Half<F16>::down(p.x * cs[i] - p.y * sn[i], p.y * cs[i] + p.x * sn[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float2 p = Half<F16>::up(w[i]), r = Half<F16>::up(w[4 + i]);
                        w[i] = Half<F16>::down(p.x * cs[2 * i] - r.x * sn[2 * i], p.y * cs[2 * i + 1] - r.y * sn[2 * i + 1]);
                        w[4 + i] = Half<F16>::down(r.x * cs[2 * i] + p.x * sn[2 * i], r.y * cs[2 * i + 1] + p.y * sn[2 * i + 1]);
                    }
                }
                x0[u] = make_uint4(w[0], w[1], w[2], w[3]);
                x1[u] = make_uint4(w[4], w[5], w[6], w[7]);
            }
            uint16_t *dst;
            if (h < a.Hq) dst = reinterpret_cast<uint16_t *>(a.q_out) + (t * a.Hq + h) * a.D;
            else if (slot < 0) continue;
            else if (!is_v) dst = reinterpret_cast<uint16_t *>(a.kc) + cache_row + (h - a.Hq) * a.head_stride;
            else dst = reinterpret_cast<uint16_t *>(a.vc) + cache_row + (h - a.Hq - a.Hk) * a.head_stride;
            *reinterpret_cast<uint4 *>(dst + (is_v ? c * 16 : e0)) = x0[u];
            *reinterpret_cast<uint4 *>(dst + (is_v ? c * 16 + 8 : e1)) = x1[u];
        }
    }
    if (bad) atomicCAS(a.err, 0, ERR_INDEX);
}

// --------------------------------------------------------------------------
// routing
//
// One warp a token; lane l holds the experts l, l + 32, ...  Scores are exact
// functions of the logits in f32 (expf and a rounded division, the softmax's
// sum in f64 and rounded once), so a choice never hangs on the order of a sum.
// A float compares as the unsigned number of its ordered bits, so the best of
// the warp is one redux.max and its lowest index one redux.min; a lane's own keys
// are sorted first, so a round looks at one of each lane, and the scores wait in
// shared memory for the chosen.  Bound: instructions (some 900 a warp with 256
// experts in 8 groups), at 16 blocks an SM so that 8192 tokens are one wave:
// 13.0 us; 64 tokens 4.7 us, one token of 128 experts 2.7 us, of which the launch
// is 2.3 and the chain load, scores, k rounds the rest.

// Experts of closed groups come behind those of open ones, also behind what a bias of -inf
// rules out there (0: no expert, or one that is chosen already).
constexpr uint32_t CLOSED = 1u;
__device__ __forceinline__ uint32_t ordered(float f) {  // NaN below every number
    const uint32_t b = __float_as_uint(f + 0.0f);
    if (f != f) return CLOSED + 1u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T, int PER>
__device__ __forceinline__ void load_logits(float (&p)[PER], const RouteArgs &a, int64_t t, int lane) {
    const T *x = reinterpret_cast<const T *>(a.logits) + t * a.stride;
    T v[PER];
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (lane + 32 * i < a.E) v[i] = x[lane + 32 * i];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const float f = lane + 32 * i < a.E ? (float)v[i] : -INFINITY;
        p[i] = f != f ? -INFINITY : fminf(f, 3.402823466e38f);  // NaN: a masked expert; +inf: the largest number
    }
}

constexpr int ROUTE_W = 4;  // tokens a block

template <int PER>
__global__ void __launch_bounds__(ROUTE_W * 32, PER <= 8 ? 16 : 1) route_kernel(const RouteArgs a) {
    extern __shared__ float s_route[];  // scores [ROUTE_W][E]; with groups also what the choice goes by, [ROUTE_W][E]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t = (int64_t)blockIdx.x * ROUTE_W + warp;
    if (t >= a.T) return;
    constexpr uint32_t FULL = 0xffffffffu;
    float p[PER];
    uint32_t key[PER];
    float mx = -INFINITY;
    if (a.dtype == F32) load_logits<float>(p, a, t, lane);
    else if (a.dtype == BF16) load_logits<__nv_bfloat16>(p, a, t, lane);
    else load_logits<__half>(p, a, t, lane);
#pragma unroll
    for (int i = 0; i < PER; i++) mx = fmaxf(mx, p[i]);
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < PER; i++) p[i] = __frcp_rn(1.0f + expf(-p[i]));
    } else {
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
        if (mx == -INFINITY) mx = 0.f;  // every expert masked: all scores 0
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            p[i] = expf(p[i] - mx);
            s += (double)p[i];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
        const float sf = (float)s;
#pragma unroll
        for (int i = 0; i < PER; i++) p[i] = sf > 0.f ? __fdiv_rn(p[i], sf) : 0.f;
    }
    float *score = s_route + warp * a.E;
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (lane + 32 * i < a.E) score[lane + 32 * i] = p[i];
    if (a.groups > 1) {
        float *kb = score + ROUTE_W * a.E;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane + 32 * i;
            if (e < a.E) kb[e] = a.bias ? p[i] + a.bias[e] : p[i];
        }
        __syncwarp();
        // 2^m lanes a group scan its scores for the two best
        const int size = a.E / a.groups, shift = (size & (size - 1)) ? -1 : 31 - __clz(size);
        int lg = 32;
        while (lg * a.groups > 32) lg >>= 1;
        const int g = lane / lg, sub = lane & (lg - 1);
        float b1 = -INFINITY, b2 = -INFINITY;
        if (g < a.groups)
            for (int e = sub; e < size; e += lg) {
                const float v = kb[g * size + e];
                if (v > b1) b2 = b1, b1 = v;
                else if (v > b2) b2 = v;
            }
        for (int o = lg >> 1; o; o >>= 1) {
            const float o1 = __shfl_xor_sync(FULL, b1, o), o2 = __shfl_xor_sync(FULL, b2, o);
            b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
            b1 = fmaxf(b1, o1);
        }
        const uint32_t mine = ordered(b1 + b2);
        int rank = 0;
        for (int o = 0; o < a.groups; o++) {
            const uint32_t other = __shfl_sync(FULL, mine, o * lg);
            rank += other > mine || (other == mine && o < g);
        }
        const uint32_t kept = __ballot_sync(FULL, g < a.groups && rank < a.top_groups);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane + 32 * i;
            key[i] = e >= a.E ? 0u : (kept >> ((shift >= 0 ? e >> shift : e / size) * lg)) & 1u ? ordered(kb[e]) : CLOSED;
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane + 32 * i;
            key[i] = e >= a.E ? 0u : ordered(a.bias ? p[i] + a.bias[e] : p[i]);
        }
    }
    // The lane's keys in descending order, ties to the lower index (an insertion sort of
    // the registers: a strict comparison keeps equal keys in place), so that a round of
    // the selection only looks at the lanes' first ones.
    uint32_t at[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) at[i] = i;
    if (PER <= 8) {
#pragma unroll
        for (int i = 1; i < PER; i++)
#pragma unroll
            for (int j = i; j > 0; j--) {
                const bool swap = key[j] > key[j - 1];
                const uint32_t hk = swap ? key[j] : key[j - 1], lk = swap ? key[j - 1] : key[j];
                const uint32_t ha = swap ? at[j] : at[j - 1], la = swap ? at[j - 1] : at[j];
                key[j - 1] = hk, key[j] = lk, at[j - 1] = ha, at[j] = la;
            }
    }
    int my_e = 0;
    for (int c = 0; c < a.k; c++) {
        uint32_t best = key[0], e0 = lane + 32 * at[0];
        if (PER > 8) {
#pragma unroll
            for (int i = 1; i < PER; i++)
                if (key[i] > best) best = key[i], e0 = lane + 32 * i;
        }
        const uint32_t top = __reduce_max_sync(FULL, best);
        const uint32_t e = __reduce_min_sync(FULL, best == top ? e0 : 0xffffffffu);
        if (lane == c) my_e = (int)e;
        if (PER <= 8) {
            if (e0 == e) {  // the owner's next key moves up
#pragma unroll
                for (int i = 0; i + 1 < PER; i++) key[i] = key[i + 1], at[i] = at[i + 1];
                key[PER - 1] = 0u;
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (lane + 32 * i == (int)e) key[i] = 0u;
        }
    }
    __syncwarp();
    float my_w = lane < a.k ? score[my_e] : 0.f, tot = my_w;
#pragma unroll
    for (int o = 16; o; o >>= 1) tot += __shfl_xor_sync(FULL, tot, o);
    if (lane < a.k) {
        if (a.norm) my_w = tot > 0.f ? my_w / tot : 0.f;
        a.idx[t * a.k + lane] = my_e;
        a.weights[t * a.k + lane] = my_w * a.scale;
    }
}

}  // namespace

cudaError_t launch_paged_plan(const PlanArgs &a, cudaStream_t st) {
    const int most = a.T > a.B ? a.T : a.B;
    int grid = (most + PLAN_T - 1) / PLAN_T;
    grid = grid < 1 ? 1 : grid > num_sms() ? num_sms() : grid;
    const size_t smem = (size_t)(a.B > 0 ? a.B : 1) * 2 * sizeof(int);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    plan_kernel<<<grid, PLAN_T, smem, st>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_rope_kv_write(const RopeArgs &a, cudaStream_t st) {
    if (a.T == 0) return cudaSuccess;
    // a token's heads go to several blocks only when there are too few tokens
    // to fill the GPU: at one token each block then takes one head a thread
    const int per = ROPE_T / (a.D >> 4), heads = a.Hq + 2 * a.Hk;
    int split = (4 * num_sms() + a.T - 1) / a.T;
    const int most = (heads + per - 1) / per;
    split = split < 1 ? 1 : split > most ? most : split;
    const dim3 grid(a.T, split);
    if (a.dtype == F16) rope_kernel<true><<<grid, ROPE_T, 0, st>>>(a);
    else rope_kernel<false><<<grid, ROPE_T, 0, st>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_moe_route(const RouteArgs &a, cudaStream_t st) {
    if (a.T == 0) return cudaSuccess;
    const int grid = (a.T + ROUTE_W - 1) / ROUTE_W, per = (a.E + 31) / 32;
    const size_t smem = (size_t)ROUTE_W * a.E * sizeof(float) * (a.groups > 1 ? 2 : 1);
    if (per <= 1) route_kernel<1><<<grid, ROUTE_W * 32, smem, st>>>(a);
    else if (per <= 2) route_kernel<2><<<grid, ROUTE_W * 32, smem, st>>>(a);
    else if (per <= 4) route_kernel<4><<<grid, ROUTE_W * 32, smem, st>>>(a);
    else if (per <= 8) route_kernel<8><<<grid, ROUTE_W * 32, smem, st>>>(a);
    else if (per <= 16) route_kernel<16><<<grid, ROUTE_W * 32, smem, st>>>(a);
    else route_kernel<32><<<grid, ROUTE_W * 32, smem, st>>>(a);
    return cudaGetLastError();
}

}  // namespace kq
