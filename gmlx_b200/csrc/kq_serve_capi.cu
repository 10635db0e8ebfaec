// kq_serve_capi.cu -- C entry points of the serving-step operators: arguments
// are checked here, before any launch, and answered with a KQ_ERR_* code and
// the thread's message (as kq_capi.cu does for the projections).
#include <stdarg.h>
#include <stdio.h>

#include "../../include/kq_cuda.h"
#include "kq_serve.cuh"

using namespace kq;

namespace {

int fail(int code, const char *fmt, ...) {
    char msg[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    set_last_error(msg);
    return code;
}

int done(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return KQ_OK;
    return fail(KQ_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int need_workspace(const void *ws, size_t have, size_t need, const char *what) {
    if (!ws || have < need) return fail(KQ_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, have, need);
    return KQ_OK;
}

constexpr int64_t MOST = PLAN_CAP;  // tokens, lengths and pages are counted in 32 bits on the device

bool aligned(const void *p, int64_t s0, int64_t s1) { return !((uintptr_t)p % 16 || s0 % 8 || s1 % 8); }

int check_cache(const kq_paged_cache *c, const char *what) {
    if (!c || !c->k || !c->v) return fail(KQ_ERR_SHAPE, "%s: null cache", what);
    if (c->dtype != KQ_F16 && c->dtype != KQ_BF16) return fail(KQ_ERR_DTYPE, "%s: the cache must be f16 or bf16 (got dtype %d)", what, c->dtype);
    if (c->pages < 1 || c->pages > MOST || c->page_size < 1 || c->page_size > MOST || c->kv_heads < 1 || c->kv_heads > 65535)
        return fail(KQ_ERR_SHAPE, "%s: a cache of %lld pages of %lld tokens and %lld heads", what, (long long)c->pages,
                    (long long)c->page_size, (long long)c->kv_heads);
    if (!aligned(c->k, c->page_stride, c->row_stride) || !aligned(c->v, c->head_stride, 0))
        return fail(KQ_ERR_ALIGN, "%s: cache bases must be 16-byte aligned and strides multiples of 8", what);
    return KQ_OK;
}

// workspace of the attention: error word and the shared counter region in front
// (the layout of every call of this library), partial rows behind
constexpr size_t PART_OFF = 256 + 1024 * 1024;

}  // namespace

extern "C" {

int kq_paged_plan(const int32_t *context_lens, const int32_t *query_lens, int64_t batch, int32_t *block_tables,
                  int64_t table_stride, int64_t table_width, const int32_t *free_pages, int64_t n_free,
                  int64_t page_size, int64_t n_tokens, int32_t *cu_seqlens, int32_t *seq_lens, int64_t *slots,
                  int32_t *positions, int32_t *pages_used, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "paged_plan";
    set_last_error("");
    if (batch < 0 || batch > PLAN_MAX_B) return fail(KQ_ERR_SHAPE, "%s: batch %lld outside 0..%d", what, (long long)batch, PLAN_MAX_B);
    if (page_size < 1 || page_size > MOST) return fail(KQ_ERR_SHAPE, "%s: page size %lld", what, (long long)page_size);
    if (n_tokens < 0 || n_tokens > MOST || n_free < 0 || n_free > MOST || table_width < 0 || table_width > MOST || table_stride < table_width)
        return fail(KQ_ERR_SHAPE, "%s: %lld tokens, %lld free pages, tables of %lld entries at stride %lld", what,
                    (long long)n_tokens, (long long)n_free, (long long)table_width, (long long)table_stride);
    if (int rc = need_workspace(workspace, workspace_bytes, 256, what)) return rc;
    PlanArgs a{context_lens, query_lens, (int)batch, block_tables, table_stride, (int)table_width, free_pages,
               (int)n_free, (int)page_size, (int)n_tokens, cu_seqlens, seq_lens, slots, positions, pages_used,
               (int *)workspace};
    return done(launch_paged_plan(a, (cudaStream_t)stream), what);
}

int kq_rope_kv_write(const kq_paged_cache *cache, const void *q, int64_t q_token_stride, int64_t q_head_stride,
                     const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v,
                     int64_t v_token_stride, int64_t v_head_stride, int64_t tokens, int64_t heads, const float *cos,
                     const float *sin, int64_t n_positions, int rot, int interleaved, const int32_t *positions,
                     const int64_t *slots, void *q_out, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "rope_kv_write";
    set_last_error("");
    if (int rc = check_cache(cache, what)) return rc;
    const int64_t d = cache->dim;
    if (d < 16 || d > 1024 || d % 16) return fail(KQ_ERR_SHAPE, "%s: head dim %lld is not a multiple of 16 up to 1024", what, (long long)d);
    if (rot < 0 || rot > d || rot % 16) return fail(KQ_ERR_SHAPE, "%s: %d rotary values are not a multiple of 16 up to the head dim %lld", what, rot, (long long)d);
    if (tokens < 0 || tokens > MOST || heads < 0 || heads > 65535) return fail(KQ_ERR_SHAPE, "%s: %lld tokens of %lld heads", what, (long long)tokens, (long long)heads);
    if (n_positions < 1 || n_positions > MOST) return fail(KQ_ERR_SHAPE, "%s: a table of %lld positions", what, (long long)n_positions);
    if (!aligned(q, q_token_stride, q_head_stride) || !aligned(k, k_token_stride, k_head_stride) ||
        !aligned(v, v_token_stride, v_head_stride) || !aligned(q_out, 0, 0) || !aligned(cos, 0, 0) || !aligned(sin, 0, 0))
        return fail(KQ_ERR_ALIGN, "%s: bases must be 16-byte aligned and strides multiples of 8", what);
    if (int rc = need_workspace(workspace, workspace_bytes, 256, what)) return rc;
    RopeArgs a{};
    a.q = q, a.k = k, a.v = v;
    a.q_ts = q_token_stride, a.q_hs = q_head_stride, a.k_ts = k_token_stride, a.k_hs = k_head_stride;
    a.v_ts = v_token_stride, a.v_hs = v_head_stride;
    a.dtype = cache->dtype, a.T = (int)tokens, a.Hq = (int)heads, a.Hk = (int)cache->kv_heads, a.D = (int)d;
    a.rot = rot, a.interleaved = interleaved != 0;
    a.cos = cos, a.sin = sin, a.n_pos = (int)n_positions, a.pos = positions, a.slots = slots, a.q_out = q_out;
    a.kc = cache->k, a.vc = cache->v;
    a.page_stride = cache->page_stride, a.row_stride = cache->row_stride, a.head_stride = cache->head_stride;
    a.page = (int)cache->page_size, a.n_slots = cache->pages * cache->page_size;
    a.err = (int *)workspace;
    return done(launch_rope_kv_write(a, (cudaStream_t)stream), what);
}

size_t kq_paged_attention_workspace_size(int64_t dim) {
    if (dim < 1 || dim > 256) return PART_OFF;
    const size_t rows = attn_part_bytes((int)dim), tiles = attn_tiles_part_bytes((int)dim);
    return PART_OFF + (rows > tiles ? rows : tiles);
}

int kq_paged_attention(const kq_paged_cache *cache, const void *q, int64_t q_token_stride, int64_t q_head_stride,
                       int64_t tokens, int64_t heads, const int32_t *block_tables, int64_t table_stride,
                       int64_t table_width, const int32_t *seq_lens, const int32_t *cu_seqlens, int64_t batch,
                       int64_t max_query_len, float scale, int causal, int64_t window, float softcap, void *out,
                       float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "paged_attention";
    set_last_error("");
    if (int rc = check_cache(cache, what)) return rc;
    const int64_t d = cache->dim, hk = cache->kv_heads;
    if (d != 64 && d != 128 && d != 256) return fail(KQ_ERR_SHAPE, "%s: head dim %lld is not 64, 128 or 256", what, (long long)d);
    if (heads < 1 || heads > 65535 || heads % hk) return fail(KQ_ERR_SHAPE, "%s: %lld query heads are not a multiple of %lld kv heads", what, (long long)heads, (long long)hk);
    if (tokens < 0 || tokens > MOST / heads || batch < 0 || batch > MOST - 1 || table_width < 0 || table_width > MOST ||
        table_stride < table_width || max_query_len < 0)
        return fail(KQ_ERR_SHAPE, "%s: %lld tokens, %lld requests, tables of %lld entries at stride %lld", what,
                    (long long)tokens, (long long)batch, (long long)table_width, (long long)table_stride);
    if (window < 0 || (window && !causal)) return fail(KQ_ERR_SHAPE, "%s: a window of %lld keys (>= 0, and causal only)", what, (long long)window);
    if (!(softcap >= 0.f) || !(softcap < INFINITY) || !(scale > 0.f && scale < INFINITY))
        return fail(KQ_ERR_SHAPE, "%s: scale %g (positive), softcap %g (>= 0)", what, (double)scale, (double)softcap);
    if (!aligned(q, q_token_stride, q_head_stride) || !aligned(out, 0, 0))
        return fail(KQ_ERR_ALIGN, "%s: bases must be 16-byte aligned and strides multiples of 8", what);
    if (int rc = need_workspace(workspace, workspace_bytes, kq_paged_attention_workspace_size(d), what)) return rc;
    AttnArgs a{};
    a.q = q, a.q_ts = q_token_stride, a.q_hs = q_head_stride;
    a.kc = cache->k, a.vc = cache->v;
    a.page_stride = cache->page_stride, a.row_stride = cache->row_stride, a.head_stride = cache->head_stride;
    a.page = (int)cache->page_size, a.n_pages = (int)cache->pages, a.page_shift = -1;
    a.g_shift = -1;
    for (int s = 0; s < 31; s++) {
        if (a.page == 1 << s) a.page_shift = s;
        if (heads / hk == 1 << s) a.g_shift = s;
    }
    a.table = block_tables, a.table_stride = table_stride;
    const int64_t max_len = table_width * cache->page_size;
    a.max_len = (int)(max_len < MOST ? max_len : MOST);
    a.seq = seq_lens, a.cu = cu_seqlens, a.B = (int)batch, a.T = (int)tokens;
    a.Hq = (int)heads, a.Hk = (int)hk, a.G = (int)(heads / hk), a.D = (int)d;
    a.scale = scale, a.softcap = softcap, a.causal = causal != 0;
    a.window = (int)(window < MOST ? window : 0);  // wider than any request: none
    a.out = out, a.lse = lse;
    a.err = (int *)workspace, a.cnt = (int *)((char *)workspace + 256), a.part = (float *)((char *)workspace + PART_OFF);
    a.min_rows = 0, a.max_rows = 0x7fffffff;
    if (tokens == 0) return KQ_OK;
    // Up to ROWS_MAX packed rows a request is bound by reading its keys, and the
    // register tiles do that; longer ones go to the tensor-core tiles.  A batch may
    // hold both, so each launch then takes its kind of request, told apart by the
    // lengths on the device; a single request needs the tiles alone.
    if (max_query_len * a.G > ROWS_MAX) {
        bool taken = false;
        if (batch > 1) a.min_rows = ROWS_MAX + 1;
        if (int rc = done(launch_attn_tiles(a, cache->dtype, (cudaStream_t)stream, taken), what)) return rc;
        if (taken && batch <= 1) return KQ_OK;
        if (taken) a.max_rows = ROWS_MAX;
        a.min_rows = 0;
    }
    return done(launch_attn_rows(a, cache->dtype, (cudaStream_t)stream), what);
}

int kq_moe_route(const void *logits, int dtype, int64_t t, int64_t e, int64_t row_stride, int k, int scoring,
                 const float *bias, int n_groups, int topk_groups, int norm_topk_prob, float scale, int32_t *idx,
                 float *weights, void *stream) {
    const char *what = "moe_route";
    set_last_error("");
    if (dtype != KQ_F32 && dtype != KQ_F16 && dtype != KQ_BF16) return fail(KQ_ERR_DTYPE, "%s: logits must be f32, f16 or bf16 (got dtype %d)", what, dtype);
    if (e < 1 || e > ROUTE_MAX_E) return fail(KQ_ERR_SHAPE, "%s: expert count %lld outside 1..%d", what, (long long)e, ROUTE_MAX_E);
    if (n_groups < 1 || n_groups > ROUTE_MAX_GROUPS || e % n_groups || (n_groups > 1 && e / n_groups < 2))
        return fail(KQ_ERR_SHAPE, "%s: %d groups of %lld experts (1..%d equal groups of two or more)", what, n_groups, (long long)e, ROUTE_MAX_GROUPS);
    if (topk_groups < 1 || topk_groups > n_groups) return fail(KQ_ERR_SHAPE, "%s: %d open groups of %d", what, topk_groups, n_groups);
    if (k < 1 || k > ROUTE_MAX_K || k > e / n_groups * topk_groups)
        return fail(KQ_ERR_SHAPE, "%s: k=%d outside 1..min(%d, experts of the open groups)", what, k, ROUTE_MAX_K);
    if (scoring != KQ_SCORE_SOFTMAX && scoring != KQ_SCORE_SIGMOID) return fail(KQ_ERR_SHAPE, "%s: scoring %d", what, scoring);
    if (t < 0 || t > MOST || row_stride < 0) return fail(KQ_ERR_SHAPE, "%s: %lld tokens at stride %lld", what, (long long)t, (long long)row_stride);
    if (!(scale == scale) || scale == INFINITY || scale == -INFINITY) return fail(KQ_ERR_SHAPE, "%s: scale %g", what, (double)scale);
    RouteArgs a{logits, dtype, row_stride, (int)t, (int)e, k, scoring == KQ_SCORE_SIGMOID, bias, n_groups, topk_groups,
                norm_topk_prob != 0, scale, idx, weights};
    return done(launch_moe_route(a, (cudaStream_t)stream), what);
}

}  // extern "C"
