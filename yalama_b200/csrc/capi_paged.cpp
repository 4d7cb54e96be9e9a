// Kernel-level C ABI entry points (include/yalama_b200.h) of a step of several requests on a paged K/V cache:
// argument checks, the attention's workspace, and the launches. Every check comes before any device work; what lies
// in the step's device arrays is checked by the kernels (paged.cuh).
#include "capi_common.h"

#include <cstdio>

using namespace ylm;

static_assert(YLM_STEP_BAD_REQUEST == 1 && YLM_STEP_BAD_PAGE == 2 && YLM_STEP_BAD_PARENT == 4 &&
                  YLM_STEP_BAD_POSITION == 8 && YLM_STEP_TIMEOUT == 16,
              "the bits of paged.cuh");

namespace {

// Whether some of n rows of wa halves at a, sa halves apart, share memory with some of n rows of wb at b.
bool rows_overlap(const void *a, int64_t sa, int64_t wa, const void *b, int64_t sb, int64_t wb, int64_t n)
{
    if (n <= 0 || wa <= 0 || wb <= 0)
        return false;
    using Wide = __int128; // a stride can be anything
    const Wide x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    if (x >= y + 2 * ((Wide)(n - 1) * sb + wb) || y >= x + 2 * ((Wide)(n - 1) * sa + wa))
        return false;
    if (sa != sb || n == 1)
        return true; // (rows of other strides inside one another: none that can be told apart simply)
    const Wide pitch = 2 * (Wide)sa, d = ((y - x) % pitch + pitch) % pitch; // columns of the same rows
    return d < 2 * wa || d + 2 * wb > pitch;
}

// Null when the cache and the step can be used, else what is wrong with them.
const char *step_fault(const ylm_paged_cache *c, const ylm_paged_step *st)
{
    if (!c || !c->k || !c->v)
        return "null cache buffer";
    if (!aligned(c->k, 16) || !aligned(c->v, 16))
        return "cache pages must be 16-byte aligned";
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
        return "a page must be 16, 32, 64 or 128 tokens";
    if (c->n_pages <= 0 || c->hkv <= 0 || c->hkv > 65535)
        return "cache needs 1 page at least and 1..65535 KV heads";
    const int64_t layer = (int64_t)c->n_pages * c->hkv * c->page * YLM_HEAD_DIM;
    if (rows_overlap(c->k, layer, layer, c->v, layer, layer, 1))
        return "keys and values must not overlap";
    if (!st)
        return "null step";
    if (st->n_seq < 0 || st->n_seq > 65535 || st->rows < 0 || st->max_rows < 0)
        return "a step has 0..65535 requests, and rows and max_rows of 0 at least";
    if (st->n_seq == 0)
        return nullptr;
    if (!st->row_start || !st->length || !st->page_table)
        return "null step buffer";
    if (!aligned(st->row_start, 4) || !aligned(st->length, 4) || !aligned(st->page_table, 4) ||
        !aligned(st->parent, 4) || !aligned(st->fault, 4))
        return "the step's buffers must be 4-byte aligned";
    // 2^30 slots of one request: slot arithmetic keeps to 32 bits
    if (st->table_ld <= 0 || (int64_t)st->table_ld * c->page > 1 << 30)
        return "a request's table needs 1 page at least and 2^30 slots at most";
    if (st->parent && st->max_rows > YLM_TREE_ROWS)
        return "a tree has at most 128 rows a request";
    return nullptr;
}

PagedCache to_kernel(const ylm_paged_cache &c)
{
    PagedCache k;
    k.k = static_cast<__half *>(c.k);
    k.v = static_cast<__half *>(c.v);
    k.n_pages = c.n_pages;
    k.page = c.page;
    k.page_shift = c.page == 16 ? 4 : c.page == 32 ? 5 : c.page == 64 ? 6 : 7;
    k.hkv = c.hkv;
    return k;
}

PagedStep to_kernel(const ylm_paged_step &st)
{
    PagedStep k;
    k.row_start = st.row_start;
    k.length = st.length;
    k.table = st.page_table;
    k.parent = st.parent;
    k.fault = st.fault;
    k.n_seq = st.n_seq;
    k.table_ld = st.table_ld;
    k.rows = st.rows;
    k.max_rows = st.max_rows < st.rows ? st.max_rows : st.rows;
    return k;
}

bool bad_rows(const void *p, int64_t stride, int64_t heads)
{
    return stride < heads * YLM_HEAD_DIM || stride % 8 || !p || !aligned(p, 16);
}

const char *heads_fault(const ylm_paged_cache *c, int32_t hq)
{
    if (hq <= 0 || hq % c->hkv || hq / c->hkv > 128)
        return "query heads must be a multiple of the KV heads, at most 128 to one";
    return nullptr;
}

} // namespace

extern "C" {

int ylm_k_paged_append(const ylm_paged_cache *cache, const ylm_paged_step *step, const void *q, int64_t q_stride,
                       const void *k, int64_t k_stride, const void *v, int64_t v_stride, int32_t hq,
                       const void *q_norm, const void *k_norm, float eps, const void *rope_cos, const void *rope_sin,
                       int32_t max_pos, void *q_out, int64_t q_out_stride, void *stream)
{
    if (const char *f = step_fault(cache, step))
        return refuse(YLM_INVALID_ARG, f);
    if (hq < 0 || hq > 65535)
        return refuse(YLM_INVALID_ARG, "needs 0..65535 query heads");
    if (!rope_cos != !rope_sin || (rope_cos && max_pos <= 0))
        return refuse(YLM_INVALID_ARG, "the rotation needs both tables and max_pos > 0");
    if (!aligned(q_norm, 16) || !aligned(k_norm, 16) || !aligned(rope_cos, 16) || !aligned(rope_sin, 16))
        return refuse(YLM_INVALID_ARG, "norm weights and tables must be 16-byte aligned");
    if (step->n_seq == 0 || step->rows == 0)
        return done(cudaSuccess);
    if (bad_rows(k, k_stride, cache->hkv) || bad_rows(v, v_stride, cache->hkv) ||
        (hq && (bad_rows(q, q_stride, hq) || bad_rows(q_out, q_out_stride, hq))))
        return refuse(YLM_INVALID_ARG,
                      "rows must be 16-byte aligned, their strides multiples of 8 halves that hold the heads");
    // a row's blocks read and write their own heads, at any time before or after another row's
    const int64_t wq = (int64_t)hq * YLM_HEAD_DIM, wk = (int64_t)cache->hkv * YLM_HEAD_DIM;
    if (((q_out != q || q_out_stride != q_stride) && rows_overlap(q_out, q_out_stride, wq, q, q_stride, wq, step->rows)) ||
        rows_overlap(q_out, q_out_stride, wq, k, k_stride, wk, step->rows) ||
        rows_overlap(q_out, q_out_stride, wq, v, v_stride, wk, step->rows))
        return refuse(YLM_INVALID_ARG, "q_out must be q with its stride, or not overlap q, k and v");
    const int sms = device_sms();
    if (!sms || prepare_device() != cudaSuccess)
        return no_device();
    PagedAppendArgs a;
    a.c = to_kernel(*cache);
    a.st = to_kernel(*step);
    a.q = static_cast<const __half *>(q);
    a.k = static_cast<const __half *>(k);
    a.v = static_cast<const __half *>(v);
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.hq = hq;
    a.q_norm = static_cast<const __half *>(q_norm);
    a.k_norm = static_cast<const __half *>(k_norm);
    a.eps = eps;
    a.rope_cos = static_cast<const __half *>(rope_cos);
    a.rope_sin = static_cast<const __half *>(rope_sin);
    a.max_pos = max_pos;
    a.q_out = static_cast<__half *>(q_out);
    a.q_out_stride = q_out_stride;
    return done(paged_append_launch(a, sms, static_cast<cudaStream_t>(stream)));
}

int ylm_k_paged_attention_workspace(const ylm_paged_cache *cache, const ylm_paged_step *step, int32_t hq, size_t *bytes)
{
    if (!bytes)
        return refuse(YLM_INVALID_ARG, "null bytes");
    if (const char *f = step_fault(cache, step))
        return refuse(YLM_INVALID_ARG, f);
    if (const char *f = heads_fault(cache, hq))
        return refuse(YLM_INVALID_ARG, f);
    const int sms = device_sms();
    if (!sms)
        return no_device();
    PagedAttnArgs a = {};
    a.c = to_kernel(*cache);
    a.st = to_kernel(*step);
    a.st.max_rows = step->max_rows; // whatever `rows` a step of it will have
    a.hq = hq;
    *bytes = paged_attn_workspace(a, sms);
    return done(cudaSuccess);
}

int ylm_k_paged_attention(const ylm_paged_cache *cache, const ylm_paged_step *step, const void *q, int64_t q_stride,
                          int32_t hq, void *out, int64_t out_stride, void *workspace, size_t workspace_bytes,
                          void *stream)
{
    if (const char *f = step_fault(cache, step))
        return refuse(YLM_INVALID_ARG, f);
    if (const char *f = heads_fault(cache, hq))
        return refuse(YLM_INVALID_ARG, f);
    if (step->n_seq == 0 || step->rows == 0)
        return done(cudaSuccess);
    if (bad_rows(q, q_stride, hq) || bad_rows(out, out_stride, hq))
        return refuse(YLM_INVALID_ARG,
                      "rows must be 16-byte aligned, their strides multiples of 8 halves that hold the heads");
    const int64_t wq = (int64_t)hq * YLM_HEAD_DIM;
    if (rows_overlap(out, out_stride, wq, q, q_stride, wq, step->rows))
        return refuse(YLM_INVALID_ARG, "out must not overlap q");
    if (workspace && !aligned(workspace, 16))
        return refuse(YLM_INVALID_ARG, "workspace must be 16-byte aligned");
    const int sms = device_sms();
    if (!sms || prepare_device() != cudaSuccess)
        return no_device();
    PagedAttnArgs a;
    a.c = to_kernel(*cache);
    a.st = to_kernel(*step);
    a.q = static_cast<const __half *>(q);
    a.q_stride = q_stride;
    a.hq = hq;
    a.out = static_cast<__half *>(out);
    a.out_stride = out_stride;
    const size_t need = paged_attn_workspace(a, sms);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    void *ws = workspace;
    if (workspace)
    {
        if (workspace_bytes < need)
        {
            char msg[96];
            snprintf(msg, sizeof(msg), "workspace of %zu bytes, %zu needed", workspace_bytes, need);
            return refuse(YLM_INVALID_ARG, msg);
        }
    }
    else if (need)
    {
        const cudaError_t e = cudaMallocAsync(&ws, need, s);
        if (e != cudaSuccess)
            return done(e);
    }
    cudaError_t e = paged_attn_launch(a, ws, sms, s);
    if (ws && !workspace)
    {
        const cudaError_t f = cudaFreeAsync(ws, s);
        e = e != cudaSuccess ? e : f;
    }
    return done(e);
}

int ylm_k_paged_accept(const ylm_paged_cache *cache, const ylm_paged_step *step, const int64_t *tokens,
                       const int64_t *picks, int32_t layers, int64_t layer_stride, int32_t *accepted,
                       int32_t *n_accepted, int64_t *next_token, int32_t *new_length, void *stream)
{
    if (const char *f = step_fault(cache, step))
        return refuse(YLM_INVALID_ARG, f);
    const int64_t layer = (int64_t)cache->n_pages * cache->hkv * cache->page * YLM_HEAD_DIM;
    if (layers < 0 || (layers > 1 && (layer_stride < layer || layer_stride % 8)) ||
        rows_overlap(cache->k, layer_stride, layer, cache->v, layer_stride, layer, layers > 1 ? layers : 1))
        return refuse(YLM_INVALID_ARG, "layers must not overlap, and their stride be a multiple of 8 halves");
    if (step->n_seq == 0)
        return done(cudaSuccess);
    if ((step->rows && (!tokens || !picks)) || !aligned(tokens, 8) || !aligned(picks, 8))
        return refuse(YLM_INVALID_ARG, "tokens and picks must be 8-byte aligned");
    if ((step->max_rows && !accepted) || !n_accepted || !next_token || !new_length || !aligned(accepted, 4) ||
        !aligned(n_accepted, 4) || !aligned(next_token, 8) || !aligned(new_length, 4))
        return refuse(YLM_INVALID_ARG, "null or misaligned output");
    const PagedStep st = to_kernel(*step);
    // every block of a request reads the step while the first one writes the results
    const size_t n = st.n_seq;
    const struct
    {
        const void *p;
        size_t n;
    } in[] = {{st.row_start, (n + 1) * 4},
              {st.length, n * 4},
              {st.table, n * st.table_ld * 4},
              {st.parent, st.parent ? (size_t)st.rows * 4 : 0},
              {tokens, (size_t)st.rows * 8},
              {picks, (size_t)st.rows * 8}},
      out[] = {{accepted, n * step->max_rows * 4}, {n_accepted, n * 4}, {next_token, n * 8}, {new_length, n * 4}};
    for (const auto &o : out)
        for (const auto &i : in)
            if (overlap(o.p, o.n, i.p, i.n))
                return refuse(YLM_INVALID_ARG, "the results must not overlap the step, the tokens or the picks");
    for (size_t i = 0; i < 4; i++)
        for (size_t j = i + 1; j < 4; j++)
            if (overlap(out[i].p, out[i].n, out[j].p, out[j].n))
                return refuse(YLM_INVALID_ARG, "the results must not overlap one another");
    const int sms = device_sms();
    if (!sms || prepare_device() != cudaSuccess)
        return no_device();
    PagedAcceptArgs a;
    a.c = to_kernel(*cache);
    a.st = st;
    a.tokens = tokens;
    a.picks = picks;
    a.layers = layers;
    a.layer_stride = layer_stride;
    a.accepted = accepted;
    a.accepted_ld = step->max_rows;
    a.n_accepted = n_accepted;
    a.next_token = next_token;
    a.new_length = new_length;
    return done(paged_accept_launch(a, sms, static_cast<cudaStream_t>(stream)));
}

} // extern "C"
