// kq_attn_sm100.cu -- attention of a chunk of new tokens over a paged cache on
// the 5th-generation tensor cores (tcgen05, accumulators in TMEM).
//
// A tile is 128 packed rows of one request and kv head (tokens x the query heads
// that share the kv head); scores S = Q K^T go to TMEM, eight warps of sixteen rows
// turn them into probabilities P = e^(S - ref), P goes back to TMEM over S and feeds
// O += P V, which stays in TMEM.  Rows are O / l at the end, l their sums of P in f32; `ref` is
// any number that keeps P in range (see the softmax), so it seldom changes.  P is
// rounded to the values' type, as the tensor core takes it.
//
// What bounds it: the products (a 128 x 128 x 16 step takes 64 clocks, and so does
// one of half its width) and as much time in exponentials (16 a clock and
// SM).  One tile's scores, softmax and product are a chain, so a block works on two
// tiles (head dim 64, 128; S of 128 keys each): the tensor core has the one while
// the other's softmax runs.  At 256 O takes half of TMEM, so there is one tile, and
// two S buffers of 64 keys.
//
// Blocks are persistent, one an SM.  The units of work (128 keys of one pair of
// tiles) stand in one line over all requests and every block takes an equal run
// of them, a pair's fixed cost (queries, first scores, results: some 8000 clocks, two
// units' time) counted in, or the block with the shortest pairs would be the last by
// far (a prompt of 2400 tokens 123 instead of 69 us); what a run cuts off goes
// through f32 partial rows in the workspace, which a second small launch joins in
// block order.  When there is a block for every pair and the longest pair takes
// little longer than an equal run (a short prompt), blocks take whole pairs instead.
//
// Warps 0-7 and 8-15: softmax of tile 0 and 1, and their results; warps 16 and 19:
// TMA of queries and keys, and of values (a page's rows of one head and 64 values
// a box; boxes that no row sees are read out of bounds, which fills zeros; two
// warps, since a 16-token page makes 16 boxes a tile at some 50 clocks each); warp
// 16 also walks the block's run of units and hands its shares of tile pairs to the
// others through slots in shared memory.  Warps 17 and 18 issue the products of
// tile 0 and 1: the queue to the tensor core is short and a thread's waits and
// commits take some 500 clocks a step, which the other warp's products cover.
//
// 4096 tokens on 32768 cached ones (32 heads over 8, dim 128): 2.05 ms over ten calls,
// 1.14 PFLOP/s, and 2.4 over thousands, at the power cap (1000 W, 1.44 GHz); 1024 on 8192
// at head dim 64, 128, 256: 125, 138, 279 us; a prompt of 512 tokens 18.9 us, of 2400
// tokens 67 us.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <string.h>

#include "kq_attn.cuh"

namespace kq {
namespace {

constexpr int TM = 128, KT = 128;  // rows a tile, keys a unit
constexpr int SOFT_WARPS = 16, K_WARP = 16, MMA_WARP = 17, V_WARP = 19, THREADS = 640;  // MMA_WARP + t: tile t
// 512 x 104 + 128 x 64 = 640 x 96 registers, what the launch holds
constexpr int SOFT_REGS = 104, OTHER_REGS = 64;
static_assert(SOFT_WARPS * 32 * SOFT_REGS + (THREADS - SOFT_WARPS * 32) * OTHER_REGS <= THREADS * 96, "register split");

template <int D> struct TL {
    static constexpr int NT = D <= 128 ? 2 : 1;
    static constexpr int KS = D <= 128 ? 128 : 64, NS = 2 / NT;  // keys of an S buffer, buffers of a tile
    static constexpr int Q_BYTES = TM * D * 2, KV_BYTES = KS * D * 2;
    static constexpr int NB = (232448 - 1792 - NT * Q_BYTES) / KV_BYTES > 6 ? 6 : (232448 - 1792 - NT * Q_BYTES) / KV_BYTES;
    static constexpr int OFF_KV = NT * Q_BYTES, OFF_BAR = OFF_KV + NB * KV_BYTES;
    static constexpr int OFF_SEG = OFF_BAR + 512;
    static constexpr int SMEM = OFF_SEG + 256 + 1024;  // slots of 64 bytes
    static constexpr int S_COL = 0, O_COL = 256;  // S buffers, then O
    // keys and values have a ring each (so that each producer sees every phase of its slots);
    // scores run NS buffers ahead
    static constexpr int NK = (NB + 1) / 2, NV = NB - NK;
    static_assert(NK >= NS + 1 && NV >= 2, "rings");
    static constexpr int PART = TM * (D + 2);        // floats of a tile's partial rows
};

struct TileArgs {
    AttnArgs a;
    int box_shift;   // log2 of a page box's rows
    int tile_tok;    // tokens a tile: 128 / G
    uint32_t q_tx;   // bytes of a tile's queries
    // capped scores, and their polynomial's coefficients as one of x (in pairs) up to |x| = cap_most
    Cap cap;
    float cap_most;
    uint64_t cap_k[4];
};

// What the join needs of a pair that block `i` begins and others end; last == i: none;
// last < 0: no request was computed, since offsets descend.
struct Split {
    int last, q0, n, tok0, h;
};
constexpr int SPLIT_FLOATS = 8 * 256;  // room for one a block in front of the partial rows
// What a pair costs besides its units, in units: queries, first reference, results.  With 1, 2, 3:
// a mixed f16 batch of 24 requests 199, 186, 193 us, a prompt of 2400 tokens 80, 69, 70 (head
// dims 64 and 128; not swept at 256).
constexpr int PAIR_COST = 2;
constexpr int JOIN_COST = 2;           // what a cut costs, in units: rows written, and the join's launch (an estimate, not swept)

__device__ __forceinline__ uint64_t gtimer() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// Bounded wait (2 s): on expiry the error is recorded, the block's abort flag
// stops all further issue, and every loop runs out.
__device__ __forceinline__ bool wait_b(uint64_t *bar, uint32_t par, volatile int *abort, int *err, int code) {
    uint64_t t0 = 0;
    for (uint32_t i = 1;; i++) {
        if (mbar_try_wait(bar, par)) return true;
        if ((i & 1023) == 0) {
            if (*abort) return false;
            const uint64_t now = gtimer();
            if (t0 == 0) t0 = now;
            if (now - t0 > 2000000000ull) {
                *abort = 1;
                atomicCAS(err, 0, code);
                return false;
            }
        }
    }
}

__device__ __forceinline__ void tma_4d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_3d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

// Shared-memory descriptors, SWIZZLE_128B, 8-row groups 1024 B apart.  The value
// fill is read along its rows' values (MN-major): its 64-value column blocks are
// KS * 128 B apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
template <int KS> __device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(KS * 128 / 16) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
template <bool F16> __device__ __forceinline__ constexpr uint32_t idesc(int n, bool b_mn) {
    const uint32_t fmt = F16 ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
}
// One lane issues, by predicate and not by a branch: the warp stays converged, so
// descriptors and addresses are computed once in uniform registers, where these
// instructions take them (under a branch each operand had to be moved there, and
// an 8-step product took 90 clocks a step beside the softmax warps instead of 64).
__device__ __forceinline__ void mma_ss(bool lead, uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
                 " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(acc),
                 "r"((uint32_t)lead)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(bool lead, uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
                 " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(acc),
                 "r"((uint32_t)lead)
                 : "memory");
}
__device__ __forceinline__ void commit(bool lead, uint64_t *bar) {
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
                 " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
                 "r"((uint32_t)lead)
                 : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define KQ_R16(r) \
    "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), \
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
#define KQ_U16(r) \
    "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), \
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
#define KQ_LIST16 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}"

// 16 lanes of tensor memory in the layout of a warp's matrix fragments: thread 4g + q
// has of each 8 f32 columns the columns 2q, 2q + 1 of lanes g (r[4i], r[4i + 1]) and
// g + 8 (r[4i + 2], r[4i + 3]); of each 4 columns of packed pairs the column q of the
// two lanes.  A row's values so stay in one warp, in four threads.  Registers hold
// what was read after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld_c32(uint32_t addr, uint32_t *r) {  // 32 columns
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 " KQ_LIST16 ", [%16];" : KQ_R16(r) : "r"(addr));
}
__device__ __forceinline__ void tmem_st_c32(uint32_t addr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%16], " KQ_LIST16 ";" ::KQ_U16(r), "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st_pairs32(uint32_t addr, const uint32_t *r) {  // 32 columns of packed pairs
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%16], " KQ_LIST16 ";" ::KQ_U16(r), "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// orders every use of r behind the wait before it
__device__ __forceinline__ void pin(uint32_t &r) { asm volatile("" : "+r"(r)); }

// Of a thread's 8 keys 0, 1, 8, 9, ..., 25 (counted from its first): those below n.
__device__ __forceinline__ uint32_t keys_below(int n) {
    n = min(max(n, 0), 32);
    return (1u << (n / 8 * 2 + min(n & 7, 2))) - 1;
}

// w[g] of thread q of a quad <-> w[q] of thread g
__device__ __forceinline__ void quad_transpose(uint32_t w[4], int lane) {
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            if (g & o) continue;
            const uint32_t give = up ? w[g] : w[g | o], got = __shfl_xor_sync(0xffffffffu, give, o);
            if (up) w[g] = got;
            else w[g | o] = got;
        }
    }
}

// Arithmetic on pairs of f32 in a 64-bit register.
__device__ __forceinline__ uint64_t pack2u(uint32_t x, uint32_t y) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(x), "r"(y));
    return v;
}
__device__ __forceinline__ uint64_t pack2f(float x, float y) { return pack2u(__float_as_uint(x), __float_as_uint(y)); }
__device__ __forceinline__ void unpack2f(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(x), "l"(y), "l"(z));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
__device__ __forceinline__ float max3f(uint32_t x, uint32_t y, uint32_t z) {
    float v;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(__uint_as_float(x)), "f"(__uint_as_float(y)), "f"(__uint_as_float(z)));
    return v;
}

// The larger of m and a row's values in a fragment of 32 columns.
__device__ __forceinline__ float largest(float m, const uint32_t *x, int row) {
#pragma unroll
    for (int k = 0; k < 16; k += 4) m = max3f(__float_as_uint(m), x[k + 2 * row], x[k + 2 * row + 1]);
    return m;
}

// 2^x of a pair, on the SFU.  (A share of the pairs on the FMA pipe, by a polynomial, was
// measured: with 0, 1, 2, 3 of 8 pairs 4096 tokens on 32768 cached took 2.19, 2.20, 2.26
// and 2.4 ms -- the issue slots are as scarce as the SFU's.)
__device__ __forceinline__ uint64_t exp2_2(uint64_t x) {
    float u, v;
    unpack2f(x, u, v);
    return pack2f(ex2(u), ex2(v));
}

// Capped scores (soft_cap).  While all of a warp's are in the polynomial's range (scores
// well within the cap: as good as always) its coefficients k hold `in` and `out` too:
// x (k0 + x^2 (k1 + x^2 (k2 + x^2 k3))).
__device__ __forceinline__ void cap_scores(uint32_t *x, const TileArgs &p) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) m = fmaxf(m, fmaxf(fabsf(__uint_as_float(x[i])), fabsf(__uint_as_float(x[i + 1]))));
    if (__all_sync(0xffffffffu, m <= p.cap_most)) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const uint64_t u = pack2u(x[i], x[i + 1]), v = mul2(u, u);
            const uint64_t y = mul2(u, fma2(v, fma2(v, fma2(v, p.cap_k[3], p.cap_k[2]), p.cap_k[1]), p.cap_k[0]));
            float a, b;
            unpack2f(y, a, b);
            x[i] = __float_as_uint(a), x[i + 1] = __float_as_uint(b);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = __float_as_uint(soft_cap(__uint_as_float(x[i]), p.cap));
    }
}

// One block's share of a pair of tiles.
struct Seg {  // 64 bytes
    int q0, n, len;        // the request
    int b, h, tok0;        // first token of the pair
    int lo, hi;            // keys its rows see
    int lo_tile, tiles;    // key tiles of the pair
    int k0, k1;            // this block's share of them
    int c[2];              // S buffers of each tile of rows in the share
    int split, last;       // whether blocks share the pair; the last of them (known to the first)
};

template <int D> struct Walk {
    static constexpr int NT = TL<D>::NT;
    const TileArgs &p;
    bool whole;  // a pair is one unit
    uint32_t ub, u, ue, before;
    Request rq;
    int b, qt;  // request, pair
    bool bad;

    __device__ __forceinline__ static int pair_units(const TileArgs &p, const Request &r, int qt, int &lo, int &hi) {
        const int t0 = qt * NT * p.tile_tok, t1 = min(r.n, t0 + NT * p.tile_tok);
        key_range(p.a, r, t0, t1, lo, hi);
        return max(1, (hi + KT - 1) / KT - lo / KT);
    }
    __device__ __forceinline__ static int pairs(const TileArgs &p, const Request &r) {
        const int64_t rows = (int64_t)r.n * p.a.G;
        if (rows == 0 || rows > p.a.max_rows || rows < p.a.min_rows) return 0;
        return (r.n + NT * p.tile_tok - 1) / (NT * p.tile_tok);
    }
    // units and pairs of a request (of its pairs first, first + step, ...); `most`: the longest pair so far
    __device__ __forceinline__ static uint32_t request_units(const TileArgs &p, const Request &r, int first, int step, uint32_t &items, int &most) {
        const int n = pairs(p, r);
        uint32_t s = 0, k = 0;
        int lo, hi;
        for (int i = first; i < n; i += step, k++) {
            const int t = pair_units(p, r, i, lo, hi);
            s += t + PAIR_COST;
            most = max(most, t);
        }
        items += k * p.a.Hk;
        return s * p.a.Hk;
    }

    __device__ __forceinline__ Walk(const TileArgs &p, bool whole, uint32_t ub, uint32_t ue, int b0, uint32_t before0)
        : p(p), whole(whole), ub(ub), u(ub), ue(ue), before(before0), b(b0), qt(0), bad(false) {
        if (u < ue) rq = load_request(p.a, b, bad);
    }
    __device__ __forceinline__ bool next(Seg &s, uint32_t total, int grid) {
        if (u >= ue) return false;
        const int lane = threadIdx.x & 31;
        for (;;) {  // the pair that holds unit u, 32 pairs at a time
            const int n = pairs(p, rq);
            if (qt < n) {
                int l, e;
                const uint32_t cost = qt + lane < n ? (whole ? 1 : pair_units(p, rq, qt + lane, l, e) + PAIR_COST) * p.a.Hk : 0;
                uint32_t upto = cost;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, u - before < upto);
                if (hit) {
                    const int j = __ffs(hit) - 1;
                    before += __shfl_sync(0xffffffffu, upto - cost, j);
                    qt += j;
                    break;
                }
                before += __shfl_sync(0xffffffffu, upto, 31);
                qt += 32;
            } else {
                qt = 0;
                if (++b > p.a.B) return false;  // (lengths that changed while they were read)
                rq = load_request(p.a, b, bad);
            }
        }
        int lo, hi;
        const int t = pair_units(p, rq, qt, lo, hi), tv = whole ? 1 : t + PAIR_COST;
        s.q0 = rq.q0, s.n = rq.n, s.len = rq.len, s.b = b, s.lo = lo, s.hi = hi;
        s.h = (int)((u - before) / (uint32_t)tv);
        const uint32_t u0 = before + (uint32_t)s.h * tv, v0 = u - u0, v1 = min((uint32_t)tv, ue - u0);
        u = u0 + v1;
        // The first PAIR_COST units of a pair are its fixed cost: a cut among them falls before
        // the pair, any other before the key tile that stands there.
        s.k0 = whole ? 0 : max(0, (int)v0 - PAIR_COST), s.k1 = whole ? t : max(0, (int)v1 - PAIR_COST);
        if (s.k1 == 0) return false;  // (and u == ue)
        s.split = s.k0 > 0 || s.k1 < t;
        s.last = s.k0 == 0 && s.k1 < t ? unit_block<uint64_t>(total, u0 + tv - 1, grid) : 0;
        s.tok0 = qt * NT * p.tile_tok;
        s.lo_tile = lo / KT;
        s.tiles = (hi + KT - 1) / KT - s.lo_tile;
        if (hi <= lo) s.tiles = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int t0 = s.tok0 + i * p.tile_tok, t1 = min(rq.n, t0 + p.tile_tok);
            int l, e;
            key_range(p.a, rq, t0, t1, l, e);
            constexpr int KS = TL<D>::KS;
            const int own = i < NT && t0 < rq.n && e > l ? (e + KS - 1) / KS - s.lo_tile * (KT / KS) : 0;
            s.c[i] = max(0, min(min(s.k1, s.tiles) * (KT / KS), own) - s.k0 * (KT / KS));
        }
        return true;
    }
};

// Reader's side of the slots: a warp takes the next share and gives it back.
constexpr int SLOTS = 4;
struct Shares {
    uint64_t *full, *empty;
    const Seg *slots;
    volatile int *abort;
    int *err;
    uint32_t i;
    __device__ __forceinline__ const Seg *take() {  // null: no more
        if (!wait_b(&full[i % SLOTS], (i / SLOTS) & 1, abort, err, 39)) return nullptr;
        const Seg *s = slots + i % SLOTS;
        return s->n > 0 ? s : nullptr;
    }
    __device__ __forceinline__ void give(int lane) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[i % SLOTS]);
        i++;
    }
};

// Partial rows of a tile that block `blk` cut -- its last pair when it begins the
// pair, else its first: m [128], l [128], unnormalised f32 rows [128][D].
template <int D> __device__ __forceinline__ float *part_of(float *base, int blk, bool begins, int t) {
    return base + SPLIT_FLOATS + (int64_t)((blk * 2 + (begins ? 1 : 0)) * TL<D>::NT + t) * TL<D>::PART;
}

template <bool F16, int D, bool CAP>
__global__ void __launch_bounds__(THREADS, 1)
    tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TileArgs p) {
    using L = TL<D>;
    constexpr int NT = L::NT, NB = L::NB, KS = L::KS, NS = L::NS;
    const AttnArgs &a = p.a;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (an offset, so that it is known to be shared memory)
    uint64_t *kv_full = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR), *kv_empty = kv_full + NB;
    uint64_t *q_full = kv_empty + NB, *q_empty = q_full + 1, *v_fix = q_empty + 1;
    uint64_t *s_full = v_fix + 1, *p_full = s_full + 2;  // [buffer]
    uint64_t *o_full = p_full + 2, *drained = o_full + 2, *turn = drained + 2;  // [tile] (o_full, two buffers: [buffer])
    uint64_t *seg_full = turn + 2, *seg_empty = seg_full + SLOTS;
    Seg *segs = reinterpret_cast<Seg *>(smem + L::OFF_SEG);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(seg_empty + SLOTS);
    volatile int *s_abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;  // warp: known uniform

    if (tid == 0) {
        for (int i = 0; i < NB; i++) mbar_init(&kv_full[i], 1), mbar_init(&kv_empty[i], NT);
        mbar_init(q_full, 1), mbar_init(q_empty, NT), mbar_init(v_fix, 1);
        for (int i = 0; i < 2; i++) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 8), mbar_init(&o_full[i], 1), mbar_init(&drained[i], 1), mbar_init(&turn[i], 1);
        for (int i = 0; i < SLOTS; i++) mbar_init(&seg_full[i], 1), mbar_init(&seg_empty[i], 1 + 9 * NT);
        *s_abort = 0;
        fence_mbar_init();
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (warp == K_WARP && lane < 3) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &tm_q : lane == 1 ? &tm_k : &tm_v) : "memory");
    // units of each thread's run of requests (b == B: the padding tokens)
    bool bad = false, unordered = false;
    const int nb = a.B + 1, per = (nb + THREADS - 1) / THREADS;
    const bool wide = nb <= THREADS / 32;  // few requests: a warp each, a lane a pair
    uint32_t mine = 0, items = 0;
    int most = 0;
    for (int i = 0; i < per && !unordered; i++) {  // (up to a descent the tokens are distinct, and their pairs few)
        const int b = wide ? warp : tid * per + i;
        if (b < nb) mine += Walk<D>::request_units(p, load_request(a, b, bad), wide ? lane : 0, wide ? 32 : 1, items, most), unordered = descends(a, b);
    }
    if (wide) {
        mine = __reduce_add_sync(0xffffffffu, mine), items = __reduce_add_sync(0xffffffffu, items);
        if (lane) mine = items = 0;
    }
    Split *splits = reinterpret_cast<Split *>(a.part);
    if (tid == 0) splits[blockIdx.x].last = blockIdx.x;
    if (blockIdx.x == 0 && bad) atomicCAS(a.err, 0, ERR_LENGTHS);
    uint32_t *s_warp = reinterpret_cast<uint32_t *>(smem);  // before the first copy arrives there
    int *s_most = reinterpret_cast<int *>(s_warp + 64);
    uint32_t *s_start = s_warp + 96;
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) s_most[warp] = most;
    uint32_t total, pairs, upto = mine, items_upto = items;
    block_scan2<THREADS, uint32_t>(upto, items_upto, s_warp, total, pairs, unordered);
    if (unordered) {  // (the join writes the rows: here that code costs registers, 1.4 of a short prompt's 19 us)
        if (tid == 0) splits[blockIdx.x].last = -1;
        tc_before();
        __syncthreads();
        tc_after();
        if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(*tmem_slot));
        return;
    }
    most = __reduce_max_sync(0xffffffffu, lane < THREADS / 32 ? s_most[lane] : 0);
    const bool whole = pairs <= gridDim.x && most <= (int)((total - PAIR_COST * pairs + gridDim.x - 1) / gridDim.x) + JOIN_COST;
    if (whole) total = pairs, upto = items_upto, mine = items;
    const int grid = (int)min(gridDim.x, total);  // at most one block a unit: a pair's blocks are neighbours
    const bool work = (int)blockIdx.x < grid;
    const uint32_t ub = work ? (uint32_t)unit_begin<uint64_t>(total, blockIdx.x, grid) : 0;
    const uint32_t ue = work ? (uint32_t)unit_begin<uint64_t>(total, blockIdx.x + 1, grid) : 0;
    if (work && upto - mine <= ub && ub < upto) s_start[0] = tid, s_start[1] = upto - mine;
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *tmem_slot;
    const int run = work ? (int)s_start[0] : 0, first_b = wide ? run >> 5 : run * per;
    const uint32_t run_before = work ? s_start[1] : 0;
    __syncthreads();
    // rows of a tile that no query fills: zeros, so that their scores ask for nothing
    for (int i = tid; i < NT * (D / 64) * TM * 8 && p.tile_tok * a.G < TM; i += THREADS)
        if ((i >> 3) % TM >= p.tile_tok * a.G) *reinterpret_cast<uint4 *>(smem + i * 16) = make_uint4(0, 0, 0, 0);
    fence_async_shared();
    __syncthreads();

    Shares shares{seg_full, seg_empty, segs, s_abort, a.err, 0};
    if (warp >= SOFT_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        if (warp == K_WARP || warp == V_WARP) {
            // box r of a tile: keys [r << shift, (r + 1) << shift) of one page, for each
            // 64 values of the head; the pages of the next tile are looked up while
            // this one waits for its place in the ring
            const int kv = warp == V_WARP, shift = p.box_shift, nrow = KS >> shift;
            const CUtensorMap *map = kv ? &tm_v : &tm_k;
            bool bad_page = false;
            const uint32_t ring = kv ? L::NV : L::NK, slot0 = kv ? L::NK : 0;
            uint32_t fill = 0, items = 0, fixes = 0;
            Walk<D> walk(p, whole, ub, kv ? ub : ue, first_b, run_before);
            auto hand_out = [&]() -> const Seg * {  // the next share, for everyone
                Seg next;
                if (!walk.next(next, total, grid)) next.n = 0;
                if (!wait_b(&seg_empty[shares.i % SLOTS], ((shares.i / SLOTS) & 1) ^ 1, s_abort, a.err, 40)) return nullptr;
                Seg *s = segs + shares.i % SLOTS;
                if (lane == 0) {
                    *s = next;
                    mbar_arrive(&seg_full[shares.i % SLOTS]);
                }
                __syncwarp();
                shares.i++;
                return next.n > 0 ? s : nullptr;
            };
            // (the key warp gives nothing back: a slot is only written again by itself)
            for (const Seg *sp; (sp = kv ? shares.take() : hand_out()) != nullptr; kv ? shares.give(lane) : (void)0) {
                const int n = max(sp->c[0], sp->c[1]), h = sp->h, lo = sp->lo, hi = sp->hi, key00 = (sp->lo_tile + sp->k0) * KT;
                if (n == 0) continue;
                const int32_t *bt = a.table + (int64_t)sp->b * a.table_stride;
                int page[4], off[4];
                auto look_up = [&](int j) {  // (only loads: the ids are looked at when they are used)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int r = lane + 32 * q, key = key00 + j * KS + (r << shift);
                        page[q] = -1, off[q] = -1;
                        if (r < nrow && key < hi && key + (1 << shift) > lo) {
                            const int col = a.page_shift >= 0 ? key >> a.page_shift : key / a.page;
                            page[q] = bt[col];
                            off[q] = key - col * a.page;
                        }
                    }
                };
                look_up(0);
                if (!kv) {
                    wait_b(q_empty, (items & 1) ^ 1, s_abort, a.err, 31);
                    items++;
                    if (lane == 0) {
                        const int live = sp->c[NT - 1] > 0 ? NT : 1;
                        mbar_arrive_expect_tx(q_full, live * p.q_tx);
                        if (!*s_abort)
                            for (int t = 0; t < live; t++)
#pragma unroll
                                for (int d = 0; d < D / 64; d++)
                                    tma_3d(smem + t * L::Q_BYTES + d * TM * 128, &tm_q, d * 64, h * a.G, sp->q0 + sp->tok0 + t * p.tile_tok, q_full);
                    }
                }
                for (int j = 0; j < n; j++, fill++) {
                    const int slot = slot0 + fill % ring;
                    uint8_t *dst = smem + L::OFF_KV + slot * L::KV_BYTES;
                    const bool ok = wait_b(&kv_empty[slot], ((fill / ring) & 1) ^ 1, s_abort, a.err, 32);
                    // a page's rows that no row sees may hold anything, and 0 * NaN is NaN:
                    // such values are cleared here before the tensor core sees them
                    const int tile0 = key00 + j * KS;
                    const bool fix = kv && (tile0 < lo || tile0 + KS > hi);
                    uint64_t *full = fix ? v_fix : &kv_full[slot];
                    if (lane == 0) mbar_arrive_expect_tx(full, L::KV_BYTES);
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int r = lane + 32 * q;
                        const bool seen = off[q] >= 0, own = (unsigned)page[q] < (unsigned)a.n_pages;
                        bad_page |= seen && !own;
                        if (r < nrow && ok)
#pragma unroll
                            for (int d = 0; d < D / 64; d++)  // page n_pages is out of bounds: zeros
                                tma_4d(dst + d * KS * 128 + (r << shift) * 128, map, d * 64, max(off[q], 0), h, seen && own ? page[q] : a.n_pages, full);
                    }
                    if (fix) {
                        wait_b(v_fix, fixes++ & 1, s_abort, a.err, 34);
                        for (int i = lane; i < KS * 8; i += 32) {
                            const int key = tile0 + (i >> 3);
                            if (key >= lo && key < hi) continue;
#pragma unroll
                            for (int d = 0; d < D / 64; d++)
                                *reinterpret_cast<uint4 *>(dst + d * KS * 128 + i * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&kv_full[slot]);
                    }
                    if (j + 1 < n) look_up(j + 1);
                }
            }
            if (bad_page) atomicCAS(a.err, 0, ERR_INDEX);
            if (*s_abort)  // nothing consumes what is still in flight: let it land before the block ends
                for (uint32_t f = fill > ring ? fill - ring : 0; f < fill; f++)
                    mbar_wait(&kv_full[slot0 + f % ring], (f / ring) & 1, 1u << 20);
            if (*s_abort && !kv && items) mbar_wait(q_full, (items - 1) & 1, 1u << 20);
            if (*s_abort && kv && fixes) mbar_wait(v_fix, (fixes - 1) & 1, 1u << 20);
        } else if (warp < MMA_WARP + NT) {
            constexpr uint32_t id_s = idesc<F16>(KS, false), id_o = idesc<F16>(D, true);
            const int t = warp - MMA_WARP;
            const uint64_t dq = desc_k(smem_u32(smem + t * L::Q_BYTES)), dk0 = desc_k(smem_u32(smem + L::OFF_KV));
            const uint64_t dv0 = desc_mn<KS>(smem_u32(smem + L::OFF_KV));
            const uint32_t d_s = tmem + L::S_COL + t * KS, d_o = tmem + L::O_COL + t * D;
            const bool lead = lane == 0;
            bool ok = true;
            uint32_t items = 0, pp = 0;               // pp: a parity bit for each buffer's p_full
            uint32_t kf = 0, kp = 0, vf = L::NK, vp = 0;  // the next slots of keys and of values, and their parities
            // The tiles take turns at the tensor core.  Left alone it would mix their steps, both
            // tiles would finish together, and so would their softmaxes: tensor core and SFU
            // would work one after the other, not side by side.
            uint32_t turns = 0;
            auto my_turn = [&] {
                if (NT == 2) ok = wait_b(&turn[t], (turns++ & 1) ^ (t == 0), s_abort, a.err, 33) && ok;
            };
            auto your_turn = [&] {
                if (NT == 2 && lead) mbar_arrive(&turn[t ^ 1]);
                __syncwarp();
            };
            auto step_k = [&] {
                if (++kf == L::NK) kf = 0, kp ^= 1;
            };
            auto step_v = [&] {
                if (++vf == NB) vf = L::NK, vp ^= 1;
            };
            for (const Seg *sp; (sp = shares.take()) != nullptr; shares.give(lane)) {
                const int c = __shfl_sync(0xffffffffu, sp->c[t], 0), n = __shfl_sync(0xffffffffu, max(sp->c[0], sp->c[1]), 0);
                if (n == 0) continue;
                ok = wait_b(q_full, items & 1, s_abort, a.err, 33) && ok;
                items++;
                // Scores S = Q K^T run NS steps ahead of the product that frees their buffer.
                // The commit behind them tells the softmax that they are there, and that the
                // products before them are done.  The last product has a barrier of its own:
                // the next share's first scores need nothing from the softmax, and could run
                // past a phase that a slow warp still waits for.
                // A tile that has no use for a fill waits for it all the same before giving it
                // back, or it could give it back twice while the other tile still reads it.
                auto keys = [&] { ok = wait_b(&kv_full[kf], kp, s_abort, a.err, 34) && ok; };
                auto scores = [&](int i) {
                    if (i < c) {
                        const uint64_t dk = dk0 + kf * (L::KV_BYTES / 16);
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++)
                            mma_ss(lead && ok, d_s + (i % NS) * KS, dq + (kk >> 2) * (TM * 8) + (kk & 3) * 2,
                                   dk + (kk >> 2) * (KS * 8) + (kk & 3) * 2, id_s, kk ? 1u : 0u);
                    }
                };
                auto behind = [&](int i) {
                    commit(lead, &kv_empty[kf]);
                    step_k();
                    if (i == n - 1) commit(lead, q_empty);
                };
                for (int i = 0; i < NS && i < n; i++) {
                    keys();
                    my_turn();
                    scores(i);
                    if (i < c) commit(lead, &s_full[t * NS + i]);
                    your_turn();
                    behind(i);
                }
                for (int i = 0; i < n; i++) {
                    const int b = i % NS;
                    ok = wait_b(&kv_full[vf], vp, s_abort, a.err, 34) && ok;
                    const uint64_t dv = dv0 + vf * (L::KV_BYTES / 16);
                    if (i < c) {
                        ok = wait_b(&p_full[t * NS + b], (pp >> b) & 1, s_abort, a.err, 35) && ok;
                        pp ^= 1u << b;
                    }
                    if (i + NS < n) keys();
                    my_turn();
                    tc_after();
                    if (i < c) {  // O += P V
#pragma unroll
                        for (int kk = 0; kk < KS / 16; kk++)
                            mma_ts(lead && ok, d_o, d_s + b * KS + kk * 8, dv + kk * 128, id_o, i > 0 || kk ? 1u : 0u);
                        if (NS > 1 || i == c - 1) commit(lead, &o_full[t + (NS > 1 ? b : 0)]);
                    }
                    if (i + NS < n) {
                        scores(i + NS);
                        if (i + NS < c) commit(lead, &s_full[t * NS + b]);
                    }
                    your_turn();
                    if (i + NS < n) behind(i + NS);
                    commit(lead, &kv_empty[vf]);
                    step_v();
                }
            }
            // no arrival is on its way to shared memory when the block ends
            commit(lead, &drained[t]);
            wait_b(&drained[t], 0, s_abort, a.err, 37);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFT_REGS));
        // softmax of 16 rows of tile t: this thread has 2 of each 8 keys of rows[0], rows[1]
        const int t = warp >> 3, q2 = (lane & 3) * 2;
        const int row0 = (warp & 3) * 32 + (warp >> 2 & 1) * 16 + (lane >> 2);  // and row0 + 8
        const uint32_t lanes = (uint32_t)((warp & 3) * 32 + (warp >> 2 & 1) * 16) << 16;
        const uint32_t o_addr = tmem + lanes + L::O_COL + t * D;
        const float sl2 = CAP ? 1.0f : a.scale * LOG2E;
        const uint64_t sl2_2 = pack2f(sl2, sl2);
        const float ref0 = F16 ? -fminf(6.f / sl2, 1e30f) : 0.f;  // f16 starts with probabilities of 2^6 times exp(score)
        uint32_t sp_bits = 0;            // a parity bit for each of the tile's s_full
        // Products are told of by o_full: with one buffer the share's last one; with two each
        // on its buffer's barrier, waited for before that buffer's next P is handed over (a
        // wait by parity must never fall two phases behind).
        uint32_t o_bits = 0;
        auto wait_o = [&](int b) {
            wait_b(&o_full[t + b], (o_bits >> b) & 1, s_abort, a.err, 38);
            o_bits ^= 1u << b;
            __syncwarp();
            tc_after();
        };
        // token of this thread's rows, from the tile's first
        const int rt0 = row0 / a.G, rt1 = (row0 + 8) / a.G;
        for (const Seg *sp; t < NT && (sp = shares.take()) != nullptr; shares.give(lane)) {
            const volatile Seg &s = *sp;
            // (what only masks and the end need is read again from the slot there)
            auto tile_tok0 = [&] { return s.tok0 + t * p.tile_tok; };
            auto tile_end = [&] { return min(s.n, tile_tok0() + p.tile_tok); };
            // keys that every row of the tile sees: buffers [i_lo, i_hi) need no mask
            const int first_key = (s.lo_tile + s.k0) * KT;
            const int all_hi = a.causal ? s.len - s.n + 1 + tile_tok0() : s.len, all_lo = a.window ? s.len - s.n + tile_end() - a.window : 0;
            const int i_hi = (all_hi - first_key) >= 0 ? (all_hi - first_key) / KS : 0, i_lo = all_lo > first_key ? (all_lo - first_key + KS - 1) / KS : 0;
            float ref[2] = {ref0, ref0}, l[2] = {0.f, 0.f};
            int seen = 0;       // bit r: row r has seen keys
            bool unset = true;  // some row of the warp may have seen none
            int told = 0;  // products of this share waited for
            const int c = s.c[t];
            for (int i = 0; i < c; i++) {
                const uint32_t s_addr = tmem + lanes + L::S_COL + (t * NS + i % NS) * KS;
                wait_b(&s_full[t * NS + i % NS], (sp_bits >> (i % NS)) & 1, s_abort, a.err, 36);
                sp_bits ^= 1u << (i % NS);
                __syncwarp();  // tensor memory is read by whole warps
                tc_after();
                if (NS > 1 && i >= NS && told < i - 1) wait_o(i % NS), told++;  // product i - 2: this S is behind it
                uint32_t x[16], pk[KS / 4];  // (as few live registers as will do: a spill here costs a third of the speed)
                const bool masked = i >= i_hi || i < i_lo;
                uint32_t vis[2];  // the keys that this thread's rows see, 8 bits for each 32 columns
                if (masked) {
                    const int key0 = (s.lo_tile + s.k0) * KT + i * KS + q2, end = tile_end() - 1, t0 = tile_tok0(), past = s.len - s.n + 1;
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const int lim = (a.causal ? past + min(t0 + (r ? rt1 : rt0), end) : s.len) - key0;
                        vis[r] = 0;
#pragma unroll
                        for (int g = 0; g < KS; g += 32)
                            vis[r] |= (keys_below(lim - g) & ~keys_below(a.window ? lim - a.window - g : 0)) << (g / 4);
                    }
                }
                auto load = [&](int g) {  // 32 columns
                    tmem_ld_c32(s_addr + g, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; k++) pin(x[k]);
                    if (CAP) cap_scores(x, p);
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < 16; k++)  // (bit e of a row: the e-th of this thread's 8 keys)
                            x[k] = vis[k >> 1 & 1] >> (g / 4 + k / 4 * 2 + (k & 1)) & 1 ? x[k] : 0xff800000u;
                    }
                };
                // P, O and l are kept relative to `ref`, and a softmax does not care which
                // as long as nothing over- or underflows, since P and f32 are floating-point:
                // bf16 bears sums of 2^-40 to 2^60; f16 of up to 2^15 a thread, and its small
                // values are only exact to 2^-25, so the row's largest must not be below 1 (nor
                // is it when 64 or 128 keys sum to as much).  So scores are taken as they are
                // (in f16 times 2^6, halfway, which rows of few keys bear too) until a sum asks
                // for a new reference: the maximum so far.  Then they are taken again.
                float sum[2];
                for (;;) {
                    uint64_t base2[2], l2[2] = {0, 0};
#pragma unroll
                    for (int r = 0; r < 2; r++) base2[r] = pack2f(-ref[r] * sl2, -ref[r] * sl2);
#pragma unroll
                    for (int g = 0; g < KS; g += 32) {
                        load(g);
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const int r = k & 1;
                            const uint64_t y = exp2_2(fma2(pack2u(x[2 * k], x[2 * k + 1]), sl2_2, base2[r]));
                            l2[r] = add2(l2[r], y);
                            float p0, p1;
                            unpack2f(y, p0, p1);
                            pk[g / 4 + k] = pack_half<F16>(p0, p1);  // rounded to the values' type for the product
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        float la, lb;
                        unpack2f(l2[r], la, lb);
                        sum[r] = la + lb;
                    }
                    bool again = fmaxf(sum[0], sum[1]) > (F16 ? 0x1p15f : 0x1p60f);
                    if (unset)
#pragma unroll
                        for (int r = 0; r < 2; r++) {  // the row's sum, by its four threads
                            float whole = sum[r] + __shfl_xor_sync(0xffffffffu, sum[r], 1);
                            whole += __shfl_xor_sync(0xffffffffu, whole, 2);
                            again |= !(seen >> r & 1) && whole < (F16 ? (float)KS : 0x1p-40f);
                        }
                    if (!__any_sync(0xffffffffu, again)) {
                        if (unset) unset = false, seen = 3;
                        break;
                    }
                    float to[2] = {seen & 1 ? ref[0] : -INFINITY, seen & 2 ? ref[1] : -INFINITY};
#pragma unroll 1
                    for (int g = 0; g < KS; g += 32) {
                        load(g);
                        to[0] = largest(to[0], x, 0), to[1] = largest(to[1], x, 1);
                    }
                    bool on = false;
                    float k[2];
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        to[r] = fmaxf(to[r], __shfl_xor_sync(0xffffffffu, to[r], 1));
                        to[r] = fmaxf(to[r], __shfl_xor_sync(0xffffffffu, to[r], 2));
                        const bool set = seen >> r & 1, first = !set && to[r] > -INFINITY;
                        on |= first || (set && to[r] > ref[r]);
                        k[r] = set && to[r] > ref[r] ? ex2((ref[r] - to[r]) * sl2) : 1.0f;  // (unset: l and O are 0)
                        if (first || set) ref[r] = to[r], seen |= 1 << r;
                        l[r] *= k[r];
                    }
                    // no way on: every row has its maximum for reference (rows without a key so
                    // far, or scores that overflow f32)
                    if (!__any_sync(0xffffffffu, on)) break;
                    if (i > 0) {
                        if (NS > 1 && told < i) wait_o((i - 1) % NS), told++;  // the last product (NS 1: this S is behind it)
#pragma unroll 1
                        for (int d = 0; d < D; d += 32) {
                            uint32_t o[16];
                            tmem_ld_c32(o_addr + d, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                pin(o[e]);
                                o[e] = __float_as_uint(__uint_as_float(o[e]) * k[e >> 1 & 1]);
                            }
                            tmem_st_c32(o_addr + d, o);
                        }
                    }
                }
#pragma unroll
                for (int g = 0; g < KS / 4; g += 16) tmem_st_pairs32(s_addr + g * 2, pk + g);
                l[0] += sum[0], l[1] += sum[1];
                tmem_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t * NS + i % NS]);
            }
            if (NS == 1 && c > 0) wait_o(0);
            for (; NS > 1 && told < c; told++) wait_o(told % NS);
            // ---- the tile's rows, or this block's part of them
            const int tok0 = tile_tok0(), live_tok = tile_end();
            if (tok0 >= s.n) continue;
            bool live[2];
#pragma unroll
            for (int r = 0; r < 2; r++) live[r] = row0 + 8 * r < p.tile_tok * a.G && tok0 + (r ? rt1 : rt0) < live_tok;
            const bool split = s.split;
            float inv[2];
            int64_t orow[2];
            float *part = part_of<D>(a.part, blockIdx.x, s.k0 == 0, t);
            if (split && tid == 0 && s.k0 == 0) splits[blockIdx.x] = Split{s.last, s.q0, s.n, s.tok0, s.h};
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int row = row0 + 8 * r;
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
                inv[r] = l[r] == 0.f ? 0.f : 1.0f / l[r];  // (0: no key; a NaN stays one)
                orow[r] = (int64_t)(s.q0 + tok0 + (r ? rt1 : rt0)) * a.Hq + s.h * a.G + row - (r ? rt1 : rt0) * a.G;
                const float ml = ref[r] * sl2;  // log2 units
                if (q2 == 0) {
                    if (split) part[row] = l[r] == 0.f ? -INFINITY : ml, part[TM + row] = l[r];
                    else if (live[r] && a.lse) a.lse[orow[r]] = l[r] == 0.f ? -INFINITY : ml * LN2 + logf(l[r]);
                }
            }
            if (split && c == 0) continue;
#pragma unroll 1
            for (int d = 0; d < D; d += 64) {
                uint32_t o[32];
                __syncwarp();
                if (c > 0) {
                    tmem_ld_c32(o_addr + d, o);
                    tmem_ld_c32(o_addr + d + 32, o + 16);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    pin(o[e]);
                    if (c == 0) o[e] = 0u;
                }
                if (split) {  // f32 rows behind m and l
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                        if (live[e >> 1 & 1])
                            *reinterpret_cast<uint2 *>(part + 2 * TM + (row0 + (e >> 1 & 1) * 8) * D + d + e / 4 * 8 + q2) = make_uint2(o[e], o[e + 1]);
                } else {
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const int r = v & 1, half = v >> 1;
                        uint32_t w[4];
#pragma unroll
                        for (int g = 0; g < 4; g++)
                            w[g] = pack_half<F16>(__uint_as_float(o[half * 16 + g * 4 + r * 2]) * inv[r], __uint_as_float(o[half * 16 + g * 4 + r * 2 + 1]) * inv[r]);
                        quad_transpose(w, lane);  // the quad's thread q: the 8 columns of group q
                        if (live[r])
                            *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(a.out) + orow[r] * D + d + half * 32 + q2 * 4) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// Joins the pair that block blockIdx.x of the tiles began and others ended: a share of
// its rows (blockIdx.y), 16 threads a row.  Few blocks, since most have nothing to do.
constexpr int JOIN_ROWS = 64, JOIN_T = 512;
template <bool F16, int D> __global__ void __launch_bounds__(JOIN_T) join_kernel(const __grid_constant__ TileArgs p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const AttnArgs &a = p.a;
    const int first = blockIdx.x, sub = threadIdx.x & 15;
    const Split s = reinterpret_cast<const Split *>(a.part)[first];
    if (s.last == first) return;
    if (s.last < 0) return write_empty(a);
    const int t = blockIdx.y * JOIN_ROWS / TM;
    for (int i = threadIdx.x >> 4; i < JOIN_ROWS; i += JOIN_T / 16) {
        const int row = blockIdx.y * JOIN_ROWS % TM + i, rt = row / a.G, tok = s.tok0 + t * p.tile_tok + rt;
        if (row >= p.tile_tok * a.G || tok >= min(s.n, s.tok0 + (t + 1) * p.tile_tok)) return;
        float m = -INFINITY, l = 0.f;
#pragma unroll 4
        for (int b = first; b <= s.last; b++) m = fmaxf(m, part_of<D>(a.part, b, b == first, t)[row]);
        float4 acc[D / 64];
#pragma unroll
        for (int k = 0; k < D / 64; k++) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int b = first; b <= s.last; b++) {
            const float *q = part_of<D>(a.part, b, b == first, t);
            const float mb = q[row], w = mb == -INFINITY ? 0.f : ex2(mb - m);
            l += w * q[TM + row];
#pragma unroll
            for (int k = 0; k < D / 64; k++) {
                const float4 v = reinterpret_cast<const float4 *>(q + 2 * TM + row * D)[sub + k * 16];
                if (w != 0.f) acc[k].x += w * v.x, acc[k].y += w * v.y, acc[k].z += w * v.z, acc[k].w += w * v.w;
            }
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        const int64_t orow = (int64_t)(s.q0 + tok) * a.Hq + s.h * a.G + row - rt * a.G;
#pragma unroll
        for (int k = 0; k < D / 64; k++)
            *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.out) + orow * D + (sub + k * 16) * 4) =
                make_uint2(pack_half<F16>(acc[k].x * inv, acc[k].y * inv), pack_half<F16>(acc[k].z * inv, acc[k].w * inv));
        if (sub == 0 && a.lse) a.lse[orow] = l == 0.f ? -INFINITY : m * LN2 + logf(l);
    }
}

// the driver's entry by name: the library itself must load on machines without a driver
decltype(&cuTensorMapEncodeTiled) encode_fn() {
    static decltype(&cuTensorMapEncodeTiled) fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<decltype(fn)>(p);
    }
    return fn;
}

bool encode(CUtensorMap *m, bool f16, int rank, const void *base, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
    const auto fn = encode_fn();
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    return fn && fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void *>(base),
                                  dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool F16, int D, bool CAP> cudaError_t launch(const AttnArgs &a, cudaStream_t st, bool &taken) {
    using L = TL<D>;
    TileArgs p;
    p.a = a;
    int shift = 0;  // the largest power of two that divides both a page and a fill
    while ((1 << shift) < L::KS && a.page % (2 << shift) == 0) shift++;
    p.box_shift = shift;
    p.tile_tok = TM / a.G;
    p.q_tx = (uint32_t)(p.tile_tok * a.G * D * 2);
    if (CAP) {
        p.cap = make_cap(a.scale, a.softcap);
        // The powers of `in` among the coefficients may leave f32's range where the scores are
        // kept to where their terms do not count: below 3e-6 those of u^4 and u^6 (1e-9 at
        // u = 0.01), below 1e-18 that of u^2 too (3e-9 at 1e-4; x^2 must stay finite).
        // A cap of 1e4, 1024 tokens on 8192 cached: 183 us, 325 by soft_cap alone.
        const float near = p.cap.in >= 3e-6f ? CAP_NEAR : p.cap.in >= 1e-18f ? 0.01f : 1e-4f;
        p.cap_most = p.cap.in <= 1e4f ? fminf(near / p.cap.in, 1e18f) : -1.f;
        const double c[4] = {CAP_K0, CAP_K1, CAP_K2, CAP_K3};
        double f = p.cap.lin;
        for (int i = 0; i < 4; i++, f *= (double)p.cap.in * p.cap.in) {
            const float k = (float)(c[i] * f);
            uint32_t bits;
            memcpy(&bits, &k, 4);
            p.cap_k[i] = (uint64_t)bits << 32 | bits;
        }
    }
    CUtensorMap mq, mk, mv;
    // A dimension of one entry has no stride of its own; one of several entries at the same
    // place (an expanded tensor), or at descending ones, is no map: the register tiles take
    // any stride.
    bool strides = true;
    auto bytes = [&](int64_t s, int64_t extent) {
        strides &= s > 0 || extent == 1;
        return (cuuint64_t)(s > 0 ? s * 2 : 16);
    };
    const cuuint64_t qd[3] = {(cuuint64_t)D, (cuuint64_t)a.Hq, (cuuint64_t)a.T};
    const cuuint64_t qs[2] = {bytes(a.q_hs, a.Hq), bytes(a.q_ts, a.T)};
    const cuuint32_t qb[3] = {64, (cuuint32_t)a.G, (cuuint32_t)p.tile_tok};
    const cuuint64_t cd[4] = {(cuuint64_t)D, (cuuint64_t)a.page, (cuuint64_t)a.Hk, (cuuint64_t)a.n_pages};
    const cuuint64_t cs[3] = {bytes(a.row_stride, a.page), bytes(a.head_stride, a.Hk), bytes(a.page_stride, a.n_pages)};
    const cuuint32_t cb[4] = {64, 1u << shift, 1, 1};
    // pairs (one more a request than whole ones) x heads x the most units of one and its fixed cost
    const double most = ((double)a.T / (L::NT * p.tile_tok) + a.B + 1) * a.Hk * ((double)a.max_len / KT + 2 + PAIR_COST);
    taken = strides && most < 4e9 && encode(&mq, F16, 3, a.q, qd, qs, qb) && encode(&mk, F16, 4, a.kc, cd, cs, cb) && encode(&mv, F16, 4, a.vc, cd, cs, cb);
    if (!taken) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(tiles_kernel<F16, D, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
    if (e != cudaSuccess) return e;
    tiles_kernel<F16, D, CAP><<<num_sms(), THREADS, L::SMEM, st>>>(mq, mk, mv, p);
    // the join's launch overlaps the tiles' end
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(num_sms(), L::NT * TM / JOIN_ROWS);
    cfg.blockDim = dim3(JOIN_T);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<F16, D>, p);
}

template <bool F16, int D> cudaError_t launch_cap(const AttnArgs &a, cudaStream_t st, bool &taken) {
    return a.softcap > 0.f ? launch<F16, D, true>(a, st, taken) : launch<F16, D, false>(a, st, taken);
}

}  // namespace

size_t attn_tiles_part_bytes(int D) {
    return ((size_t)num_sms() * 2 * (D <= 128 ? 2 : 1) * TM * (D + 2) + SPLIT_FLOATS) * sizeof(float);
}

cudaError_t launch_attn_tiles(const AttnArgs &a, int dtype, cudaStream_t st, bool &taken) {
    taken = false;
    if (a.G > TM) return cudaSuccess;
    const bool f16 = dtype == F16;
    switch (a.D) {
        case 64: return f16 ? launch_cap<true, 64>(a, st, taken) : launch_cap<false, 64>(a, st, taken);
        case 128: return f16 ? launch_cap<true, 128>(a, st, taken) : launch_cap<false, 128>(a, st, taken);
        case 256: return f16 ? launch_cap<true, 256>(a, st, taken) : launch_cap<false, 256>(a, st, taken);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kq
