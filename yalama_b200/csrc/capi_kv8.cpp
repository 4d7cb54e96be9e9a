// Kernel-level C ABI entry points (include/yalama_b200.h) of the 8-bit K/V
// cache and of the log probabilities: argument checks, the attention's
// workspace, and the launches. Every check comes before any device work; the
// reason of a refusal is the calling thread's ylm_last_error().
#include "../../include/yalama_b200.h"
#include "ylm_kernels.h"

#include <cuda_runtime.h>
#include <cstdio>

using namespace ylm;

namespace {

int refuse(int status, const char *why)
{
    set_last_error(why);
    return status;
}

int done(cudaError_t e)
{
    if (e == cudaSuccess)
    {
        set_last_error("");
        return YLM_OK;
    }
    // the runtime keeps a failed call's error until it is asked for, and a later launch of this library would
    // take it for its own
    cudaGetLastError();
    set_last_error(cudaGetErrorString(e));
    return YLM_CUDA_ERROR;
}

int no_device()
{
    cudaGetLastError();
    return refuse(YLM_CUDA_ERROR, "device set-up failed");
}

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Null when the cache can be used, else what is wrong with it.
const char *cache_fault(const ylm_kv8_cache *c)
{
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale)
        return "null cache buffer";
    if (c->format != YLM_KV8_E4M3 && c->format != YLM_KV8_INT8)
        return "unknown cache format";
    if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
        return "cache block must be 16, 32, 64 or 128 tokens";
    // 2^30 slots of one head are 256 GiB of codes: no device holds more, and slot arithmetic keeps to 32 bits
    if (c->cap <= 0 || c->cap > 1 << 30 || c->hkv <= 0 || c->hkv > 65535)
        return "cache needs 1..2^30 slots and 1..65535 KV heads";
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return "cache codes must be 16-byte aligned and scales 4-byte aligned";
    return nullptr;
}

Kv8Cache to_kernel(const ylm_kv8_cache &c)
{
    Kv8Cache k;
    k.k = static_cast<uint8_t *>(c.k);
    k.v = static_cast<uint8_t *>(c.v);
    k.k_scale = c.k_scale;
    k.v_scale = c.v_scale;
    k.format = c.format == YLM_KV8_E4M3 ? 0 : 1;
    k.block = c.block;
    k.cap = c.cap;
    k.hkv = c.hkv;
    return k;
}

size_t code_bytes(const ylm_kv8_cache &c) { return (size_t)c.hkv * c.cap * YLM_HEAD_DIM; }
size_t scale_bytes(const ylm_kv8_cache &c)
{
    return (size_t)c.hkv * (((size_t)c.cap + c.block - 1) / c.block) * sizeof(float);
}

bool overlap(const void *a, size_t na, const void *b, size_t nb)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

int sm_count()
{
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 0;
    return n;
}

const char *attention_fault(const ylm_kv8_cache *c, int32_t hq, int32_t t, int32_t n)
{
    if (const char *f = cache_fault(c))
        return f;
    if (hq <= 0 || hq % c->hkv || hq / c->hkv > 128)
        return "query heads must be a multiple of the KV heads, at most 128 to one";
    if (t < 0 || n < t || n > c->cap)
        return "needs 0 <= t <= n <= cap";
    return nullptr;
}

} // namespace

extern "C" {

int ylm_k_kv8_store(const ylm_kv8_cache *cache, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                    int32_t t, int32_t slot, void *stream)
{
    if (const char *f = cache_fault(cache))
        return refuse(YLM_INVALID_ARG, f);
    if (t < 0 || slot < 0 || slot > cache->cap || t > cache->cap - slot)
        return refuse(YLM_INVALID_ARG, "slots [slot, slot + t) must lie in the cache");
    if (t == 0)
        return done(cudaSuccess);
    const int64_t row = (int64_t)cache->hkv * YLM_HEAD_DIM;
    if (!k || !v || !aligned(k, 16) || !aligned(v, 16))
        return refuse(YLM_INVALID_ARG, "k and v must be 16-byte aligned");
    if (k_stride < row || v_stride < row || k_stride % 8 || v_stride % 8)
        return refuse(YLM_INVALID_ARG, "token strides must be multiples of 8 halves and hold hkv x 128");
    if (prepare_device() != cudaSuccess)
        return no_device();
    return done(kv8_store_launch(to_kernel(*cache), static_cast<const __half *>(k), static_cast<const __half *>(v),
                                 k_stride, v_stride, t, slot, static_cast<cudaStream_t>(stream)));
}

int ylm_k_kv8_attention_workspace(const ylm_kv8_cache *cache, int32_t hq, int32_t t, int32_t n, int32_t with_acc,
                                  size_t *bytes)
{
    if (!bytes)
        return refuse(YLM_INVALID_ARG, "null bytes");
    if (const char *f = attention_fault(cache, hq, t, n))
        return refuse(YLM_INVALID_ARG, f);
    const int sms = sm_count();
    if (!sms)
        return no_device();
    *bytes = kv8_attn_workspace(cache->hkv, hq, t, n, with_acc != 0, sms);
    return done(cudaSuccess);
}

int ylm_k_kv8_attention(const ylm_kv8_cache *cache, const void *q, int64_t q_stride, int32_t hq, int32_t t, int32_t n,
                        const uint32_t *mask_bits, float *acc, void *out, int64_t out_stride, void *workspace,
                        size_t workspace_bytes, void *stream)
{
    if (const char *f = attention_fault(cache, hq, t, n))
        return refuse(YLM_INVALID_ARG, f);
    if (t == 0)
        return done(cudaSuccess);
    const int64_t row = (int64_t)hq * YLM_HEAD_DIM;
    if (!q || !out || !aligned(q, 16) || !aligned(out, 16))
        return refuse(YLM_INVALID_ARG, "q and out must be 16-byte aligned");
    if (q_stride < row || out_stride < row || q_stride % 8 || out_stride % 8)
        return refuse(YLM_INVALID_ARG, "token strides must be multiples of 8 halves and hold hq x 128");
    if (!aligned(mask_bits, 4) || !aligned(acc, 4))
        return refuse(YLM_INVALID_ARG, "mask_bits and acc must be 4-byte aligned");
    if (workspace && !aligned(workspace, 16))
        return refuse(YLM_INVALID_ARG, "workspace must be 16-byte aligned");
    const int sms = sm_count();
    if (!sms || prepare_device() != cudaSuccess)
        return no_device();
    const size_t need = kv8_attn_workspace(cache->hkv, hq, t, n, acc != nullptr, sms);
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
    Kv8AttnArgs a;
    a.c = to_kernel(*cache);
    a.q = static_cast<const __half *>(q);
    a.q_stride = q_stride;
    a.hq = hq;
    a.t = t;
    a.n = n;
    a.mask = mask_bits;
    a.acc = acc;
    a.out = static_cast<__half *>(out);
    a.out_stride = out_stride;
    cudaError_t e = kv8_attn_launch(a, ws, sms, s);
    if (ws && !workspace)
    {
        const cudaError_t f = cudaFreeAsync(ws, s);
        e = e != cudaSuccess ? e : f;
    }
    return done(e);
}

int ylm_k_kv8_evict(const ylm_kv8_cache *src, const ylm_kv8_cache *dst, const float *acc_src, float *acc_dst,
                    int32_t n, int32_t n_keep, int32_t n_sink, int32_t n_recent, int32_t *kept, void *stream)
{
    if (const char *f = cache_fault(src))
        return refuse(YLM_INVALID_ARG, f);
    if (const char *f = cache_fault(dst))
        return refuse(YLM_INVALID_ARG, f);
    if (src->format != dst->format || src->block != dst->block || src->hkv != dst->hkv)
        return refuse(YLM_INVALID_ARG, "the caches must have the same format, block and KV heads");
    if (n < 0 || n > src->cap || n_keep < 0 || n_keep > n || n_keep > dst->cap)
        return refuse(YLM_INVALID_ARG, "needs n_keep <= n <= the source's cap and n_keep <= the destination's cap");
    if (n_sink < 0 || n_recent < 0 || (int64_t)n_sink + n_recent > n_keep)
        return refuse(YLM_INVALID_ARG, "needs n_sink + n_recent <= n_keep");
    if (!acc_src || !acc_dst || (n_keep && !kept) || !aligned(acc_src, 4) || !aligned(acc_dst, 4) || !aligned(kept, 4))
        return refuse(YLM_INVALID_ARG, "acc and kept must be 4-byte aligned");
    const size_t acc_s = (size_t)src->hkv * src->cap * sizeof(float), acc_d = (size_t)dst->hkv * dst->cap * sizeof(float);
    const size_t cs = code_bytes(*src), ss = scale_bytes(*src), cd = code_bytes(*dst), sd = scale_bytes(*dst);
    const struct
    {
        const void *p;
        size_t n;
    } from[] = {{src->k, cs}, {src->v, cs}, {src->k_scale, ss}, {src->v_scale, ss}, {acc_src, acc_s}},
      to[] = {{dst->k, cd},
              {dst->v, cd},
              {dst->k_scale, sd},
              {dst->v_scale, sd},
              {acc_dst, acc_d},
              {kept, (size_t)src->hkv * n_keep * sizeof(int32_t)}};
    for (const auto &f : from)
        for (const auto &t : to)
            if (overlap(f.p, f.n, t.p, t.n))
                return refuse(YLM_INVALID_ARG, "the destination must not overlap the source");
    for (size_t i = 0; i < 6; i++)
        for (size_t j = i + 1; j < 6; j++)
            if (overlap(to[i].p, to[i].n, to[j].p, to[j].n))
                return refuse(YLM_INVALID_ARG, "the destination's buffers must not overlap");
    if (prepare_device() != cudaSuccess)
        return no_device();
    Kv8EvictArgs a;
    a.src = to_kernel(*src);
    a.dst = to_kernel(*dst);
    a.acc_src = acc_src;
    a.acc_dst = acc_dst;
    a.n = n;
    a.n_keep = n_keep;
    a.n_sink = n_sink;
    a.n_recent = n_recent;
    a.kept = kept;
    return done(kv8_evict_launch(a, static_cast<cudaStream_t>(stream)));
}

int ylm_k_logprobs(const void *logits, int64_t ld, int32_t rows, int64_t vocab, const int64_t *ids,
                   const uint32_t *mask_bits, int32_t n_top, float *logprob, float *entropy, int64_t *top_ids,
                   float *top_logprobs, void *stream)
{
    if (rows < 0 || vocab <= 0 || vocab > 1 << 30 || ld < vocab)
        return refuse(YLM_INVALID_ARG, "needs rows >= 0, 1 <= vocab <= 2^30 and ld >= vocab");
    if (n_top < 0 || n_top > 64)
        return refuse(YLM_INVALID_ARG, "n_top must be 0..64");
    if ((logprob && !ids) || (n_top && (!top_ids || !top_logprobs)))
        return refuse(YLM_INVALID_ARG, "logprob needs ids, and n_top > 0 needs top_ids and top_logprobs");
    if (!logprob && !entropy && !n_top)
        return refuse(YLM_INVALID_ARG, "no output asked for");
    if (!aligned(logits, 2) || !aligned(ids, 8) || !aligned(mask_bits, 4) || !aligned(logprob, 4) ||
        !aligned(entropy, 4) || (n_top && (!aligned(top_ids, 8) || !aligned(top_logprobs, 4))))
        return refuse(YLM_INVALID_ARG, "misaligned buffer");
    if (rows == 0)
        return done(cudaSuccess);
    if (!logits)
        return refuse(YLM_INVALID_ARG, "null logits");
    const int sms = sm_count();
    if (!sms || prepare_device() != cudaSuccess)
        return no_device();
    LogprobArgs a;
    a.logits = static_cast<const __half *>(logits);
    a.ld = ld;
    a.rows = rows;
    a.vocab = vocab;
    a.ids = ids;
    a.mask_bits = mask_bits;
    a.n_top = n_top;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    return done(logprobs_launch(a, sms, static_cast<cudaStream_t>(stream)));
}

} // extern "C"
