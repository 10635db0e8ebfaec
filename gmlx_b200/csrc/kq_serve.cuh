// kq_serve.cuh -- arguments and launchers of the serving-step operators: the
// paged plan, rotary embedding with the cache write, attention over a paged
// cache, and expert routing.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "kq_internal.cuh"

namespace kq {

// Error-word codes of these operators (the other kernels use 1..19): the
// lengths on the device contradict the sizes the host passed / no page left for
// a new token / a position, slot or page id outside its table or cache.
constexpr int ERR_LENGTHS = 20, ERR_PAGES = 21, ERR_INDEX = 22;

struct PlanArgs {
    const int32_t *ctx, *qlen;
    int B;
    int32_t *table;
    int64_t table_stride;
    int table_width;
    const int32_t *free_pages;
    int n_free, page, T;
    int32_t *cu, *seq;
    int64_t *slots;
    int32_t *pos, *used;
    int *err;
};
constexpr int PLAN_MAX_B = 8192, PLAN_CAP = (1 << 30) - 1;
cudaError_t launch_paged_plan(const PlanArgs &a, cudaStream_t st);

struct RopeArgs {
    const void *q, *k, *v;  // [T][heads][D], strides in elements
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
    int dtype, T, Hq, Hk, D, rot, interleaved;
    const float *cos, *sin;  // [n_pos][rot / 2]
    int n_pos;
    const int32_t *pos;
    const int64_t *slots;
    void *q_out;  // [T][Hq][D]
    void *kc, *vc;
    int64_t page_stride, row_stride, head_stride;
    int page;
    int64_t n_slots;
    int *err;
};
cudaError_t launch_rope_kv_write(const RopeArgs &a, cudaStream_t st);

struct RouteArgs {
    const void *logits;
    int dtype;
    int64_t stride;
    int T, E, k, sigmoid;
    const float *bias;
    int groups, top_groups, norm;
    float scale;
    int32_t *idx;
    float *weights;
};
constexpr int ROUTE_MAX_E = 1024, ROUTE_MAX_K = 32, ROUTE_MAX_GROUPS = 32;
cudaError_t launch_moe_route(const RouteArgs &a, cudaStream_t st);

struct AttnArgs {
    const void *q;  // [T][Hq][D]
    int64_t q_ts, q_hs;
    const void *kc, *vc;
    int64_t page_stride, row_stride, head_stride;
    int page, page_shift;  // page_shift: log2(page), or -1
    int n_pages;
    const int32_t *table;
    int64_t table_stride;
    int max_len;  // table width * page, at most 2^31 - 1
    const int32_t *seq, *cu;
    int B, T, Hq, Hk, G, D, g_shift;  // g_shift: log2(G), or -1
    float scale, softcap;  // softcap 0: none
    int causal, window;    // window 0: none
    void *out;             // [T][Hq][D]
    float *lse;            // [T][Hq] or null
    float *part;           // partial results of split rows
    int *cnt;              // counters, zero on entry and left zero
    int *err;
    int max_rows;  // requests with more packed rows (tokens x G) are another launch's
    int min_rows;  // requests with fewer too
};
// Bytes of `part` the launches need for this head dimension.
size_t attn_part_bytes(int D);
size_t attn_tiles_part_bytes(int D);
// Few rows (kq_attn.cu): requests of any size, fast up to ROWS_MAX packed rows.
constexpr int ROWS_MAX = 16;
cudaError_t launch_attn_rows(const AttnArgs &a, int dtype, cudaStream_t st);
// Chunks (kq_attn_sm100.cu).  taken = false, nothing launched: a layout that
// the tensor maps cannot describe (expanded tensors among them), or more than 128
// query heads a kv head.
cudaError_t launch_attn_tiles(const AttnArgs &a, int dtype, cudaStream_t st, bool &taken);

}  // namespace kq
