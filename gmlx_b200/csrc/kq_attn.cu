// kq_attn.cu -- attention of few new tokens over a paged cache (decode): at most
// 16 packed rows a tile, so the work is reading keys and values once.
//
// The units of work, 64 keys of one (row tile, kv head) each, stand in one line
// over all requests, and every block takes an equal run of them, so ragged
// lengths load the GPU evenly and a single long request uses all of it.  A warp
// works alone on 16 keys of each unit: its own ring of cp.async stages, its own
// running maximum, sum and output rows (m16n8k16 products in registers), and no
// barrier until its block's run of a row tile ends.  Then the four warps join in
// shared memory; a row tile that several blocks share goes through f32 partial
// rows in the workspace, which the last block to arrive joins in block order
// (so the bits do not depend on the order of arrival).
//
// With m the running maximum of a row's scores s_j = scale q.k_j, it keeps
// l = sum e^(s_j - m) and o = sum e^(s_j - m) v_j; a larger maximum m' scales both
// by e^(m - m'), two parts (m, l, o) join the same way, and the row is o / l with
// lse = m + log l.
// Bound: reading the cache.  64 requests on contexts of up to 16384 (8 kv heads of
// 128, pages of 16): 1.97 GB in 298-306 us, 6.4-6.6 TB/s, the rate of a plain copy
// (head dim 64 5.4, 256 6.2 TB/s).  One
// token at a context of 999 is latency: 7.1 us, of which launch, lengths, table and
// the first keys are a chain of four round trips to memory, the join one more.
// Above 16 rows the products would bound it (16.8 ms for 4096 tokens on 32768,
// against 2.0 on the tensor cores).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kq_attn.cuh"

namespace kq {
namespace {

constexpr int NW = 4, KW = 16, KT = NW * KW;  // warps, keys a warp's step, keys a unit
constexpr int ROWS = 16;
constexpr int CTAS = 2;  // blocks an SM (of head dim 256 only one fits, 128 KB each: the second half of the grid follows)

template <int D> struct RL {
    static constexpr int STAGES = D >= 256 ? 2 : D >= 128 ? 3 : 6;
    static constexpr int STAGE = 2 * KW * D * 2;  // keys, then values
    static constexpr int WARP = STAGES * STAGE;
    static constexpr int RING = NW * WARP;
    static constexpr int JOIN = NW * ROWS * (D + 2) * 4;
    static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

// Partial rows of one block's share of a row tile: m, l, then the unnormalised
// output rows.  Two slots a block: 0 for a tile that began in an earlier block,
// 1 for one that goes on in the next.
__host__ __device__ constexpr int part_floats(int D) { return ROWS * (D + 2); }

// Units of one (row tile, kv head) of a request, the same for all of its row
// tiles; a request without keys still has one, which writes its empty rows.
__device__ __forceinline__ int tile_units(const AttnArgs &a, const Request &r, int &lo_tile) {
    int lo, hi;
    key_range(a, r, 0, r.n, lo, hi);
    lo_tile = lo / KT;
    return max(1, (hi + KT - 1) / KT - lo_tile);
}
template <class U> __device__ __forceinline__ U request_units(const AttnArgs &a, const Request &r) {
    const int64_t rows = (int64_t)r.n * a.G;
    if (rows == 0 || rows > a.max_rows || rows < a.min_rows) return 0;
    int lt;
    return (U)((rows + ROWS - 1) / ROWS) * (U)a.Hk * (U)tile_units(a, r, lt);
}
// token of a packed row (G divides without a division where it can)
__device__ __forceinline__ int row_token(const AttnArgs &a, int r) { return a.g_shift >= 0 ? r >> a.g_shift : r / a.G; }

template <bool F16, int D, bool CAP, class U>
__global__ void __launch_bounds__(NW * 32, CTAS) rows_kernel(const __grid_constant__ AttnArgs a) {
    using L = RL<D>;
    constexpr int CH = D / 8;  // 16-byte chunks of a row
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ U s_warp[NW], s_before;
    __shared__ int s_b, s_last;
    __shared__ Request s_rq;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    bool bad = false, bad_page = false, unordered = false;

    // units of each thread's run of requests (b == B: the padding tokens)
    const int nb = a.B + 1, per = (nb + NW * 32 - 1) / (NW * 32);
    U mine = 0;
    Request rq;
    for (int i = 0; i < per; i++) {
        const int b = tid * per + i;
        if (b < nb) mine += request_units<U>(a, rq = load_request(a, b, bad)), unordered |= descends(a, b);
    }
    U total;
    const U upto = block_scan<NW * 32, U>(mine, s_warp, total, unordered);
    if (blockIdx.x == 0 && bad) atomicCAS(a.err, 0, ERR_LENGTHS);
    if (unordered) return write_empty(a);
    // at most one block a unit, so that the blocks of a row tile are neighbours
    const int grid = (int)min((U)gridDim.x, total);
    if ((int)blockIdx.x >= grid) return;
    const U ub = unit_begin<U>(total, blockIdx.x, grid), ue = unit_begin<U>(total, blockIdx.x + 1, grid);

    // the request that holds unit ub
    if (upto - mine <= ub && ub < upto) {
        U before = upto - mine;
        int b = tid * per;
        if (per > 1)
            for (;; b++) {
                rq = load_request(a, b, bad);
                const U n = request_units<U>(a, rq);
                if (ub < before + n || b == a.B) break;
                before += n;
            }
        s_b = b, s_before = before, s_rq = rq;
    }
    __syncthreads();
    int b = s_b;
    U before = s_before;  // units before request b
    rq = s_rq;

    const uint32_t ring = smem_u32(smem) + warp * L::WARP;
    const uint16_t *kc = reinterpret_cast<const uint16_t *>(a.kc), *vc = reinterpret_cast<const uint16_t *>(a.vc);
    const int gr = lane >> 2, gc = lane & 3;
    const float sl2 = a.scale * LOG2E;
    const Cap cap = make_cap(a.scale, a.softcap);

    for (U u = ub; u < ue;) {
        U units = request_units<U>(a, rq);
        while (u >= before + units && b < a.B) {
            before += units;
            rq = load_request(a, ++b, bad);
            units = request_units<U>(a, rq);
        }
        int lo_tile;
        const int tiles = tile_units(a, rq, lo_tile);
        const U item = (u - before) / (U)tiles;
        const U u0 = before + item * (U)tiles;  // first unit of this row tile
        const int rt = (int)(item / (U)a.Hk), h = (int)(item - (U)rt * (U)a.Hk);
        const int k0 = (int)(u - u0), k1 = (int)min((U)tiles, ue - u0);
        u = u0 + k1;
        const int nrows = min(ROWS, rq.n * a.G - rt * ROWS);
        const int t0 = row_token(a, rt * ROWS), t1 = row_token(a, rt * ROWS + nrows - 1) + 1;
        int lo, hi;
        key_range(a, rq, t0, t1, lo, hi);

        // this thread's rows, their key limits, and the query fragments
        int lim[2], low[2];
        uint32_t qf[D / 16][4];
        const uint16_t *qp[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = rt * ROWS + gr + 8 * i, tok = row_token(a, r);
            const bool live = gr + 8 * i < nrows;
            lim[i] = !live ? 0 : a.causal ? rq.len - rq.n + tok + 1 : rq.len;
            low[i] = a.window ? lim[i] - a.window : 0;
            qp[i] = live ? reinterpret_cast<const uint16_t *>(a.q) + (rq.q0 + tok) * a.q_ts + (int64_t)(h * a.G + r - tok * a.G) * a.q_hs
                         : nullptr;
        }
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                qf[kk][i] = qp[i & 1] ? *reinterpret_cast<const uint32_t *>(qp[i & 1] + kk * 16 + (i >> 1) * 8 + gc * 2) : 0u;

        float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < D / 8; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[j][i] = 0.f;

        const int32_t *bt = a.table + (int64_t)min(b, a.B - 1) * a.table_stride;
        auto key_of = [&](int kt) { return (lo_tile + kt) * KT + warp * KW + (lane & (KW - 1)); };
        auto page_col = [&](int key) { return a.page_shift >= 0 ? key >> a.page_shift : key / a.page; };
        int next_page = 0;
        auto fetch_page = [&](int kt) {
            const int key = key_of(kt);
            next_page = kt < k1 && key >= lo && key < hi ? bt[page_col(key)] : 0;
        };
        auto issue = [&](int kt) {  // one step's keys and values; those outside [lo, hi) arrive as zeros
            if (kt < k1) {
                const int key = key_of(kt);
                int64_t off = -1;
                if (key >= lo && key < hi) {
                    if ((unsigned)next_page < (unsigned)a.n_pages)
                        off = next_page * a.page_stride + (key - page_col(key) * a.page) * a.row_stride + h * a.head_stride;
                    else bad_page = true;
                }
                const uint32_t dst = ring + (kt % L::STAGES) * L::STAGE;
                fetch_page(kt + 1);
#pragma unroll
                for (int i = 0; i < KW * CH / 32; i++) {
                    const int idx = lane + 32 * i, r = idx / CH, c = idx % CH;
                    const int64_t s = __shfl_sync(0xffffffffu, off, r);
                    const uint32_t d = dst + r * (D * 2) + ((c ^ (r & 7)) << 4);
                    cp_async16(d, kc + (s < 0 ? 0 : s + c * 8), s >= 0);
                    cp_async16(d + KW * D * 2, vc + (s < 0 ? 0 : s + c * 8), s >= 0);
                }
            }
            cp_async_commit();
        };
        fetch_page(k0);
#pragma unroll
        for (int s = 0; s < L::STAGES - 1; s++) issue(k0 + s);

        for (int kt = k0; kt < k1; kt++) {
            cp_async_wait<L::STAGES - 2>();
            __syncwarp();
            issue(kt + L::STAGES - 1);
            const uint32_t ks = ring + (kt % L::STAGES) * L::STAGE, vs = ks + KW * D * 2;
            float s[2][4] = {};
            {
                const int r = (lane & 7) + ((lane >> 4) << 3), cb = (lane >> 3) & 1;
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++) {
                    uint32_t kf[4];
                    ldsm4(kf, ks + r * (D * 2) + (((kk * 2 + cb) ^ (r & 7)) << 4));
                    mma16816<F16>(s[0], qf[kk], kf[0], kf[1], s[0]);
                    mma16816<F16>(s[1], qf[kk], kf[2], kf[3], s[1]);
                }
            }
            if (CAP) {
                float far = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) far = fmaxf(far, fabsf(s[i >> 2][i & 3] * cap.in));
                if (__all_sync(0xffffffffu, far <= CAP_NEAR))  // as good as always
#pragma unroll
                    for (int i = 0; i < 8; i++) s[i >> 2][i & 3] = cap_near(s[i >> 2][i & 3], cap);
                else
#pragma unroll
                    for (int i = 0; i < 8; i++) s[i >> 2][i & 3] = soft_cap(s[i >> 2][i & 3], cap);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) s[i >> 2][i & 3] *= sl2;
            }
            const int base = (lo_tile + kt) * KT + warp * KW + gc * 2;
            float mx[2] = {m[0], m[1]};
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int key = base + j * 8 + (i & 1), row = i >> 1;
                    s[j][i] = key < lim[row] && key >= low[row] ? s[j][i] : -INFINITY;
                    mx[row] = fmaxf(mx[row], s[j][i]);
                }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            }
            if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float f = m[i] == -INFINITY ? 0.f : ex2(m[i] - mx[i]);
                    m[i] = mx[i];
                    l[i] *= f;
#pragma unroll
                    for (int j = 0; j < D / 8; j++) o[j][2 * i] *= f, o[j][2 * i + 1] *= f;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float ref = m[i >> 1];
                    s[j][i] = ex2(s[j][i] - (ref == -INFINITY ? 0.f : ref));
                    l[i >> 1] += s[j][i];
                }
            // the probabilities go to the product in the value's type (8 or 11
            // bits, as the values themselves have); their sum stays in f32
            const uint32_t pf[4] = {pack_half<F16>(s[0][0], s[0][1]), pack_half<F16>(s[0][2], s[0][3]),
                                    pack_half<F16>(s[1][0], s[1][1]), pack_half<F16>(s[1][2], s[1][3])};
            {
                const int r = lane & 15, cb = lane >> 4;
#pragma unroll
                for (int j = 0; j < D / 16; j++) {
                    uint32_t vf[4];
                    ldsm4t(vf, vs + r * (D * 2) + (((j * 2 + cb) ^ (r & 7)) << 4));
                    mma16816<F16>(o[2 * j], pf, vf[0], vf[1], o[2 * j]);
                    mma16816<F16>(o[2 * j + 1], pf, vf[2], vf[3], o[2 * j + 1]);
                }
            }
            __syncwarp();
        }
        cp_async_wait<0>();
#pragma unroll
        for (int i = 0; i < 2; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }

        // join the warps: rows of (m, l) and of outputs, one set a warp
        float *sm = reinterpret_cast<float *>(smem), *so = sm + NW * ROWS * 2;
        __syncthreads();  // the rings are drained
        if (gc == 0)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                sm[(warp * ROWS + gr + 8 * i) * 2] = m[i];
                sm[(warp * ROWS + gr + 8 * i) * 2 + 1] = l[i];
            }
#pragma unroll
        for (int j = 0; j < D / 8; j++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (gr + 8 * i < nrows)
                    *reinterpret_cast<float2 *>(so + (warp * ROWS + gr + 8 * i) * D + j * 8 + gc * 2) =
                        make_float2(o[j][2 * i], o[j][2 * i + 1]);
        __syncthreads();

        const int first = unit_block<U>(total, u0, grid), last = unit_block<U>(total, u0 + tiles - 1, grid);
        const bool split = first != last;
        float *part = a.part + (int64_t)(blockIdx.x * 2 + (k0 == 0 ? 1 : 0)) * part_floats(D);
        auto store = [&](int row, int d, float4 v, float mr, float lr) {
            const int r = rt * ROWS + row;
            const float inv = lr == 0.f ? 0.f : 1.0f / lr;  // (0: no key; a NaN stays one)
            const int tok = row_token(a, r);
            const int64_t orow = (int64_t)(rq.q0 + tok) * a.Hq + h * a.G + r - tok * a.G;
            uint2 w = make_uint2(pack_half<F16>(v.x * inv, v.y * inv), pack_half<F16>(v.z * inv, v.w * inv));
            *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.out) + orow * D + d) = w;
            if (d == 0 && a.lse) a.lse[orow] = lr == 0.f ? -INFINITY : mr * LN2 + logf(lr);
        };
        for (int idx = tid; idx < nrows * (D / 4); idx += NW * 32) {
            const int row = idx / (D / 4), d = idx % (D / 4) * 4;
            float mr = -INFINITY, lr = 0.f;
#pragma unroll
            for (int w = 0; w < NW; w++) mr = fmaxf(mr, sm[(w * ROWS + row) * 2]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float mw = sm[(w * ROWS + row) * 2], f = mw == -INFINITY ? 0.f : ex2(mw - mr);
                const float4 v = *reinterpret_cast<const float4 *>(so + (w * ROWS + row) * D + d);
                lr += f * sm[(w * ROWS + row) * 2 + 1];
                acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
            }
            if (!split) store(row, d, acc, mr, lr);
            else {
                *reinterpret_cast<float4 *>(part + ROWS * 2 + row * D + d) = acc;
                if (d == 0) part[row * 2] = mr, part[row * 2 + 1] = lr;
            }
        }
        if (split) {
            __syncthreads();
            if (tid == 0) {  // releases the block's rows (ordered before it by the barrier), and acquires the others'
                int n;
                asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(n) : "l"(a.cnt + first) : "memory");
                s_last = n == last - first;
                if (s_last) a.cnt[first] = 0;
            }
            __syncthreads();
            if (s_last) {
                constexpr int BATCH = 8;  // parts whose loads are under way together
                for (int idx = tid; idx < nrows * (D / 4); idx += NW * 32) {
                    const int row = idx / (D / 4), d = idx % (D / 4) * 4;
                    float mr = -INFINITY, lr = 0.f;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int c0 = first; c0 <= last; c0 += BATCH) {
                        float2 ml[BATCH];
                        float4 v[BATCH];
#pragma unroll
                        for (int i = 0; i < BATCH; i++) {
                            const int c = min(c0 + i, last);
                            const float *p = a.part + (int64_t)(c * 2 + (c == first ? 1 : 0)) * part_floats(D);
                            ml[i] = __ldcg(reinterpret_cast<const float2 *>(p + row * 2));
                            v[i] = __ldcg(reinterpret_cast<const float4 *>(p + ROWS * 2 + row * D + d));
                            if (c0 + i > last) ml[i].x = -INFINITY;
                        }
                        float mn = mr;
#pragma unroll
                        for (int i = 0; i < BATCH; i++) mn = fmaxf(mn, ml[i].x);
                        const float fo = mr == -INFINITY ? 0.f : ex2(mr - mn);
                        lr *= fo, acc.x *= fo, acc.y *= fo, acc.z *= fo, acc.w *= fo;
#pragma unroll
                        for (int i = 0; i < BATCH; i++) {
                            const float f = ml[i].x == -INFINITY ? 0.f : ex2(ml[i].x - mn);
                            lr += f * ml[i].y;
                            acc.x += f * v[i].x, acc.y += f * v[i].y, acc.z += f * v[i].z, acc.w += f * v[i].w;
                        }
                        mr = mn;
                    }
                    store(row, d, acc, mr, lr);
                }
            }
        }
        __syncthreads();  // the joined rows are read before the next tile's keys arrive
    }
    if (bad_page) atomicCAS(a.err, 0, ERR_INDEX);
}

template <bool F16, int D, bool CAP, class U> cudaError_t launch_as(const AttnArgs &a, cudaStream_t st) {
    const int smem = RL<D>::SMEM;
    const cudaError_t e = cudaFuncSetAttribute(rows_kernel<F16, D, CAP, U>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    rows_kernel<F16, D, CAP, U><<<CTAS * num_sms(), NW * 32, smem, st>>>(a);
    return cudaGetLastError();
}

template <bool F16, int D, bool CAP> cudaError_t launch_cap(const AttnArgs &a, cudaStream_t st) {
    // row tiles (one more a request than whole ones) x heads x the most units of one
    const double most = ((double)a.T * a.G / ROWS + a.B + 1) * a.Hk * ((double)a.max_len / KT + 2);
    if (most < 1e15 && units_fit32((int64_t)most, CTAS * num_sms())) return launch_as<F16, D, CAP, uint32_t>(a, st);
    return launch_as<F16, D, CAP, int64_t>(a, st);
}

template <bool F16, int D> cudaError_t launch(const AttnArgs &a, cudaStream_t st) {
    return a.softcap > 0.f ? launch_cap<F16, D, true>(a, st) : launch_cap<F16, D, false>(a, st);
}

}  // namespace

size_t attn_part_bytes(int D) { return (size_t)2 * CTAS * num_sms() * part_floats(D) * sizeof(float); }

cudaError_t launch_attn_rows(const AttnArgs &a, int dtype, cudaStream_t st) {
    if (a.T == 0) return cudaSuccess;
    const bool f16 = dtype == F16;
    switch (a.D) {
        case 64: return f16 ? launch<true, 64>(a, st) : launch<false, 64>(a, st);
        case 128: return f16 ? launch<true, 128>(a, st) : launch<false, 128>(a, st);
        case 256: return f16 ? launch<true, 256>(a, st) : launch<false, 256>(a, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kq
