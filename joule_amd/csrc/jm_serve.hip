// Entry points of the serving operators: the 4-bit KV cache (jm_kvq4.hip), paged KV
// caches (jm_paged.hip) and sampling (jm_sample.hip).
#include <cmath>

#include "jm_store.h"

using jm::aligned;
using jm::fail;

namespace {

constexpr int HD = 128;

// Threads of a launch.
constexpr long long MAX_THREADS = UINT32_MAX;

// Rows of a cache: cache rows and tiles of them are counted in 32 bits, up to a
// block's step past the last.
constexpr int Q4_MAX_T = INT32_MAX - 1023;

// KV heads of a paged cache, so that a page's rows are counted in 32 bits, and the bytes
// between pages.
constexpr int PAGED_MAX_KV = 1024;
constexpr uint64_t PAGED_MAX_STRIDE = 1ull << 40;

int check_group(int group) {
    if (group != 32 && group != 64) return fail(JM_ERR_SHAPE, "group must be 64 or 32, got %d", group);
    return 0;
}

// The cache and the call's tokens as the kernels take them.
int q4_args(const jm_kv_q4* c, const int32_t* start, const int32_t* cu, int N, jm::Q4KvArgs* a) {
    if (!c) return fail(JM_ERR_ARG, "cache is NULL");
    if (int rc = check_group(c->group)) return rc;
    if (c->n_seq < 0 || c->maxT <= 0 || c->n_kv <= 0)
        return fail(JM_ERR_SHAPE, "n_seq=%d must be >= 0, maxT=%d and n_kv=%d positive", c->n_seq, c->maxT, c->n_kv);
    if (N < 0) return fail(JM_ERR_ARG, "N must be >= 0");
    if (!cu && N != c->n_seq) return fail(JM_ERR_SHAPE, "without cu there is one token a sequence: N=%d, n_seq=%d", N, c->n_seq);
    // rows are written and read by 16 threads each, a wave 4 tokens of a head
    if (((long long)N + 3) / 4 * c->n_kv * 64 > MAX_THREADS - 256)
        return fail(JM_ERR_SHAPE, "N=%d tokens of %d KV heads are more than one launch takes", N, c->n_kv);
    const int64_t bytes = jm_kv_q4_bytes(c->maxT, c->n_kv, c->group);
    if (bytes < 0) return (int)bytes;
    if (N == 0 || c->n_seq == 0) return 0;
    if (!c->k || !c->v || !start) return fail(JM_ERR_ARG, "the cache's k and v and start must be non-NULL");
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->seq_stride % 16)
        return fail(JM_ERR_ARG, "the cache's planes must be 16-byte aligned (seq_stride a multiple of 16)");
    if (c->n_seq > 1 && c->seq_stride < (uint64_t)bytes)
        return fail(JM_ERR_SHAPE, "seq_stride %llu is below a plane's %lld bytes", (unsigned long long)c->seq_stride, (long long)bytes);
    if (!aligned(start, 4) || (cu && !aligned(cu, 4))) return fail(JM_ERR_ARG, "start and cu must be 4-byte aligned");
    a->k = c->k; a->v = c->v; a->seq_stride = c->seq_stride;
    a->n_seq = c->n_seq; a->maxT = c->maxT; a->KH = c->n_kv; a->group = c->group;
    a->R = jm::q4_plane_rows(c->maxT);
    a->start = start; a->cu = cu; a->N = N;
    return 0;
}

// A tensor of 128-value rows: dtype, alignment to 4 elements, strides.
int rows_tensor(const char* name, const void* p, int dtype, int64_t ts, int64_t hs) {
    if (dtype != JM_DTYPE_F32 && dtype != JM_DTYPE_BF16) return fail(JM_ERR_ARG, "dtype must be JM_DTYPE_F32 or JM_DTYPE_BF16");
    if (!p) return fail(JM_ERR_ARG, "%s must be non-NULL", name);
    if (!aligned(p, dtype == JM_DTYPE_F32 ? 16 : 8)) return fail(JM_ERR_ARG, "%s must be aligned to 4 elements", name);
    if (ts % 4 || hs % 4) return fail(JM_ERR_ARG, "%s: the strides %lld and %lld must be multiples of 4", name, (long long)ts, (long long)hs);
    return 0;
}

// launch_kernels(workspace of `bytes`, NULL for 0) on st, the workspace held until they
// are enqueued.
template <class F>
int with_workspace(hipStream_t st, size_t bytes, const char* what, F launch_kernels) {
    jm::PluginWs ws;
    if (bytes)
        if (int rc = jm::plugin_ws(st, bytes, &ws)) return rc;
    const hipError_t e = launch_kernels((float*)ws.p);
    const hipError_t f = ws.async ? hipFreeAsync(ws.p, st) : hipSuccess;
    if (e != hipSuccess) return jm::hip_fail(e, what);
    if (f != hipSuccess) return jm::hip_fail(f, "hipFreeAsync");
    return 0;
}

// The paged cache and the call's tokens as the kernels take them (a->N stays 0 where
// there is nothing to do).
int paged_args(const jm_kv_paged* c, const int32_t* start, const int32_t* cu, int N, jm::PagedArgs* a) {
    if (!c) return fail(JM_ERR_ARG, "cache is NULL");
    if (c->dtype != JM_DTYPE_F32 && c->dtype != JM_DTYPE_BF16)
        return fail(JM_ERR_ARG, "the pages' dtype must be JM_DTYPE_F32 or JM_DTYPE_BF16");
    if (c->page < 16 || c->page > 1024 || (c->page & (c->page - 1)))
        return fail(JM_ERR_SHAPE, "page must be a power of two from 16 to 1024, got %d", c->page);
    if (c->n_seq < 0 || c->n_pages <= 0 || c->maxT <= 0 || c->n_kv <= 0)
        return fail(JM_ERR_SHAPE, "n_seq=%d must be >= 0, n_pages=%d, maxT=%d and n_kv=%d positive", c->n_seq, c->n_pages,
                    c->maxT, c->n_kv);
    if (c->maxT > Q4_MAX_T) return fail(JM_ERR_SHAPE, "maxT=%d is too large", c->maxT);
    if (c->n_kv > PAGED_MAX_KV) return fail(JM_ERR_SHAPE, "n_kv must be at most %d, got %d", PAGED_MAX_KV, c->n_kv);
    if (N < 0) return fail(JM_ERR_ARG, "N must be >= 0");
    if (!cu && N != c->n_seq) return fail(JM_ERR_SHAPE, "without cu there is one token a sequence: N=%d, n_seq=%d", N, c->n_seq);
    const uint64_t bytes = (uint64_t)c->n_kv * c->page * HD * (c->dtype == JM_DTYPE_F32 ? 4 : 2);
    if (c->n_pages > 1 && c->page_stride < bytes)
        return fail(JM_ERR_SHAPE, "page_stride %llu is below a page's %llu bytes", (unsigned long long)c->page_stride,
                    (unsigned long long)bytes);
    if (c->page_stride % 16 || c->page_stride > PAGED_MAX_STRIDE)
        return fail(JM_ERR_ARG, "page_stride must be a multiple of 16, and at most %llu", (unsigned long long)PAGED_MAX_STRIDE);
    const int entries = (c->maxT - 1) / c->page + 1;
    if (c->n_seq > 1 && c->table_stride < entries)
        return fail(JM_ERR_SHAPE, "table_stride %lld is below a sequence's %d pages", (long long)c->table_stride, entries);
    if (N == 0 || c->n_seq == 0) return 0;
    if (!c->k || !c->v || !c->table || !start) return fail(JM_ERR_ARG, "the cache's k, v and table and start must be non-NULL");
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return fail(JM_ERR_ARG, "the cache's k and v must be 16-byte aligned");
    if (!aligned(c->table, 4) || !aligned(start, 4) || (cu && !aligned(cu, 4)))
        return fail(JM_ERR_ARG, "the table, start and cu must be 4-byte aligned");
    a->k = c->k; a->v = c->v; a->page_stride = c->page_stride;
    a->table = c->table; a->table_stride = c->table_stride;
    a->n_pages = c->n_pages; a->lp = __builtin_ctz((unsigned)c->page); a->f32 = c->dtype == JM_DTYPE_F32;
    a->n_seq = c->n_seq; a->maxT = c->maxT; a->KH = c->n_kv;
    a->start = start; a->cu = cu; a->N = N;
    return 0;
}

}  // namespace

extern "C" {

int64_t jm_kv_q4_bytes(int maxT, int n_kv, int group) {
    if (maxT <= 0 || n_kv <= 0) return fail(JM_ERR_SHAPE, "maxT=%d and n_kv=%d must be positive", maxT, n_kv);
    if (maxT > Q4_MAX_T) return fail(JM_ERR_SHAPE, "maxT=%d is too large", maxT);
    if (int rc = check_group(group)) return rc;
    return (int64_t)jm::q4_plane_rows(maxT) * n_kv * (HD / 2 + 2 * HD / group);
}

int jm_kv_q4_write(const jm_kv_q4* c, const int32_t* start, const int32_t* cu, int N, const void* k, int64_t k_token,
                   int64_t k_head, const void* v, int64_t v_token, int64_t v_head, int dtype, void* stream) {
    jm::Q4KvArgs a{};
    if (int rc = q4_args(c, start, cu, N, &a)) return rc;
    if (a.N == 0) return 0;
    if (int rc = rows_tensor("k", k, dtype, k_token, k_head)) return rc;
    if (int rc = rows_tensor("v", v, dtype, v_token, v_head)) return rc;
    JM_HIP(jm::launch_q4_write(a, k, v, dtype == JM_DTYPE_BF16, {k_token, k_head, v_token, v_head}, (hipStream_t)stream),
           "4-bit cache write launch");
    return 0;
}

int jm_kv_q4_read(const jm_kv_q4* c, const int32_t* start, const int32_t* cu, int N, void* k, void* v, int dtype,
                  void* stream) {
    jm::Q4KvArgs a{};
    if (int rc = q4_args(c, start, cu, N, &a)) return rc;
    if (a.N == 0) return 0;
    if (int rc = rows_tensor("k", k, dtype, 0, 0)) return rc;
    if (int rc = rows_tensor("v", v, dtype, 0, 0)) return rc;
    JM_HIP(jm::launch_q4_read(a, k, v, dtype == JM_DTYPE_BF16, (hipStream_t)stream), "4-bit cache read launch");
    return 0;
}

int jm_kv_q4_attn(const jm_kv_q4* c, const int32_t* start, const int32_t* cu, int N, const void* q, int64_t q_token,
                  int64_t q_head, int n_heads, float scale, int dtype, void* out, void* stream) {
    jm::Q4KvArgs a{};
    if (int rc = q4_args(c, start, cu, N, &a)) return rc;
    const int qpk = n_heads > 0 && n_heads % c->n_kv == 0 ? n_heads / c->n_kv : 0;
    if (qpk != 1 && qpk != 2 && qpk != 4 && qpk != 8)
        return fail(JM_ERR_SHAPE, "n_heads / n_kv must be 1, 2, 4 or 8 (got %d / %d)", n_heads, c->n_kv);
    // (the kernels take it times log2(e))
    if (!std::isfinite(scale * 1.4426950408889634f)) return fail(JM_ERR_ARG, "scale must be finite, and below 2.3e38 in magnitude");
    if (a.N == 0) return 0;
    if (int rc = rows_tensor("q", q, dtype, q_token, q_head)) return rc;
    if (int rc = rows_tensor("out", out, dtype, 0, 0)) return rc;
    hipStream_t st = (hipStream_t)stream;
    const jm::Q4AttnPlan p = jm::q4_attn_plan(a, n_heads, dtype == JM_DTYPE_BF16, false);
    // (ranges are for few units, so that the kernel that joins them has fewer threads)
    const long long threads = (long long)c->n_kv * p.units * p.S * (p.rg ? 512 : 256);
    if (threads > MAX_THREADS) return fail(JM_ERR_SHAPE, "attention of N=%d tokens and %d KV heads is more than one launch takes", N, c->n_kv);
    return with_workspace(st, (p.o_floats + p.ml_floats) * 4, "4-bit attention launch", [&](float* part) {
        return jm::launch_q4_attn(a, p, q, dtype == JM_DTYPE_BF16, q_token, q_head, n_heads, scale, out, part, part + p.o_floats, st);
    });
}

int jm_kv_paged_append(const jm_kv_paged* c, const int32_t* start, const int32_t* cu, int N, const jm_kv_rows* r,
                       void* stream) {
    jm::PagedArgs a{};
    if (int rc = paged_args(c, start, cu, N, &a)) return rc;
    if (!r) return fail(JM_ERR_ARG, "rows is NULL");
    if (r->q && (r->n_heads <= 0 || r->n_heads > 16 * c->n_kv))
        return fail(JM_ERR_SHAPE, "n_heads=%d must be from 1 to 16 times n_kv=%d", r->n_heads, c->n_kv);
    if (!r->cos != !r->sin) return fail(JM_ERR_ARG, "cos and sin come together");
    if (!std::isfinite(r->eps) || r->eps < 0.0f) return fail(JM_ERR_ARG, "eps must be finite and >= 0");
    if (!aligned(r->cos, 16) || !aligned(r->sin, 16) || !aligned(r->q_norm, 16) || !aligned(r->k_norm, 16))
        return fail(JM_ERR_ARG, "cos, sin and the norm weights must be 16-byte aligned");
    // (16 lanes a head, heads rounded up to blocks)
    const int heads = (r->q ? r->n_heads : 0) + 2 * c->n_kv;
    if (((long long)heads + 15) / 16 * 256 * N > MAX_THREADS)
        return fail(JM_ERR_SHAPE, "N=%d tokens of %d heads are more than one launch takes", N, heads);
    if (a.N == 0) return 0;
    if (int rc = rows_tensor("k", r->k, r->dtype, r->k_token, r->k_head)) return rc;
    if (int rc = rows_tensor("v", r->v, r->dtype, r->v_token, r->v_head)) return rc;
    if (r->q) {
        if (int rc = rows_tensor("q", r->q, r->dtype, r->q_token, r->q_head)) return rc;
        if (int rc = rows_tensor("q_out", r->q_out, r->dtype, 0, 0)) return rc;
    }
    jm::PagedRows p{};
    p.x[0] = r->q; p.x[1] = r->k; p.x[2] = r->v;
    p.ts[0] = r->q_token; p.ts[1] = r->k_token; p.ts[2] = r->v_token;
    p.hs[0] = r->q_head; p.hs[1] = r->k_head; p.hs[2] = r->v_head;
    p.H = r->q ? r->n_heads : 0; p.bf = r->dtype == JM_DTYPE_BF16; p.q_out = r->q_out;
    p.cos = r->cos; p.sin = r->sin; p.w[0] = r->q_norm; p.w[1] = r->k_norm; p.eps = r->eps;
    JM_HIP(jm::launch_paged_append(a, p, (hipStream_t)stream), "paged append launch");
    return 0;
}

int jm_kv_paged_attn(const jm_kv_paged* c, const int32_t* start, const int32_t* cu, int N, const void* q, int64_t q_token,
                     int64_t q_head, int n_heads, float scale, int max_rows, int dtype, void* out, void* stream) {
    jm::PagedArgs a{};
    if (int rc = paged_args(c, start, cu, N, &a)) return rc;
    if (n_heads <= 0 || n_heads % c->n_kv || n_heads / c->n_kv > 16)
        return fail(JM_ERR_SHAPE, "n_heads / n_kv must be a whole number from 1 to 16 (got %d / %d)", n_heads, c->n_kv);
    // (the kernels take it times log2(e))
    if (!std::isfinite(scale * 1.4426950408889634f)) return fail(JM_ERR_ARG, "scale must be finite, and below 2.3e38 in magnitude");
    if (max_rows < 0) return fail(JM_ERR_ARG, "max_rows must be >= 0");
    if (a.N == 0) return 0;
    if (int rc = rows_tensor("q", q, dtype, q_token, q_head)) return rc;
    if (int rc = rows_tensor("out", out, dtype, 0, 0)) return rc;
    hipStream_t st = (hipStream_t)stream;
    const jm::PagedPlan p = jm::paged_plan(a, n_heads, dtype == JM_DTYPE_BF16, max_rows ? max_rows : c->maxT);
    // (the kernel that joins ranges: up to 256 threads a query row)
    if ((long long)c->n_kv * p.units * p.S * 512 > MAX_THREADS || (p.S > 1 && (long long)p.units * p.tp * n_heads * 256 > MAX_THREADS))
        return fail(JM_ERR_SHAPE, "attention of N=%d tokens and %d heads is more than one launch takes", N, n_heads);
    return with_workspace(st, (p.o_floats + p.ml_floats) * 4, "paged attention launch", [&](float* part) {
        return jm::launch_paged_attn(a, p, q, dtype == JM_DTYPE_BF16, q_token, q_head, n_heads, scale, out, part, part + p.o_floats, st);
    });
}

int jm_sample(const void* logits, int dtype, int64_t ld, int B, int V, const jm_sampling* how, const float* u,
              int32_t* out_tok, float* out_p, void* stream) {
    if (dtype != JM_DTYPE_F32 && dtype != JM_DTYPE_BF16) return fail(JM_ERR_ARG, "dtype must be JM_DTYPE_F32 or JM_DTYPE_BF16");
    if (B < 0) return fail(JM_ERR_ARG, "B must be >= 0");
    if (V <= 0 || V > JM_SAMPLE_MAX_V) return fail(JM_ERR_SHAPE, "V must be in [1, %d] (got %d)", JM_SAMPLE_MAX_V, V);
    if (ld < V) return fail(JM_ERR_SHAPE, "rows %lld elements apart cannot hold V=%d", (long long)ld, V);
    if (!how) return fail(JM_ERR_ARG, "the sampling settings are NULL");
    if (std::isnan(how->temperature) || std::isnan(how->top_p) || std::isnan(how->min_p))
        return fail(JM_ERR_ARG, "temperature, top_p and min_p must not be NaN");
    if (B == 0) return 0;
    if (!logits || !u || !out_tok) return fail(JM_ERR_ARG, "logits, u and out_tok must be non-NULL");
    if (!aligned(logits, dtype == JM_DTYPE_F32 ? 4 : 2)) return fail(JM_ERR_ARG, "logits must be aligned to an element");
    if (!aligned(u, 4) || !aligned(out_tok, 4) || !aligned(out_p, 4) || !aligned(how->temperature_b, 4) ||
        !aligned(how->top_k_b, 4) || !aligned(how->top_p_b, 4) || !aligned(how->min_p_b, 4))
        return fail(JM_ERR_ARG, "u, the outputs and the rows' settings must be 4-byte aligned");
    jm::SampleArgs a{};
    a.logits = logits; a.bf = dtype == JM_DTYPE_BF16; a.ld = ld; a.B = B; a.V = V;
    a.temperature = how->temperature; a.top_k = how->top_k; a.top_p = how->top_p; a.min_p = how->min_p;
    a.temperature_b = how->temperature_b; a.top_k_b = how->top_k_b; a.top_p_b = how->top_p_b; a.min_p_b = how->min_p_b;
    a.u = u; a.out_tok = out_tok; a.out_p = out_p;
    hipStream_t st = (hipStream_t)stream;
    jm::PluginWs ws;
    if (int rc = jm::plugin_ws(st, jm::sample_ws_bytes(B, V), &ws)) return rc;
    const hipError_t e = jm::launch_sample(a, ws.p, st);
    const hipError_t f = ws.async ? hipFreeAsync(ws.p, st) : hipSuccess;
    if (e != hipSuccess) return jm::hip_fail(e, "sampling launch");
    if (f != hipSuccess) return jm::hip_fail(f, "hipFreeAsync");
    return 0;
}

}  // extern "C"
