// The 8-bit K/V cache: storing rows and evicting slots (attention over it:
// kv8_attention.cu; formats and the power-of-two scales: kv8.cuh).
#include "kv8.cuh"

namespace ylm {

constexpr int KST_THREADS = 256;

// One CTA per (cache block, KV head, K or V). Thread (r, c) = (tid / 16, tid % 16)
// holds dimensions [8c, 8c + 8) of tokens 16p + r of the block, so the block's
// new rows are read once (16 bytes a thread), stay in registers while the
// block-wide maximum gives the scale, and leave as 8-byte codes.
//   s_new = max(scale_of(max |x| of the new rows), s_old if older tokens share the block)
// Infinities count as +-65504; NaN takes no part in the maximum.
template <int FMT, int P>
__global__ void __launch_bounds__(KST_THREADS)
    kv8_store_kernel(Kv8Cache cache, const __half *k, const __half *v, int64_t k_stride, int64_t v_stride, int t,
                     int slot)
{
    constexpr int BLOCK = 16 * P;
    __shared__ float red[KST_THREADS / 32];
    const bool is_v = blockIdx.z != 0;
    const int g = blockIdx.y, b = slot / BLOCK + blockIdx.x;
    const int tid = threadIdx.x, r = tid >> 4, c = tid & 15;
    const int lo = b * BLOCK;
    const int64_t end = (int64_t)slot + t;
    const __half *src = (is_v ? v : k) + (size_t)g * YLM_HEAD_DIM + c * 8;
    const int64_t stride = is_v ? v_stride : k_stride;
    uint8_t *codes = (is_v ? cache.v : cache.k) + ((size_t)g * cache.cap + lo) * YLM_HEAD_DIM + c * 8;
    float *scale = (is_v ? cache.v_scale : cache.k_scale) + (size_t)g * ((cache.cap + BLOCK - 1) / BLOCK) + b;

    uint4 x[P];
    float amax = 0.f;
#pragma unroll
    for (int p = 0; p < P; p++)
    {
        const int64_t j = (int64_t)lo + p * 16 + r;
        x[p] = make_uint4(0, 0, 0, 0);
        if (j >= slot && j < end)
            x[p] = *reinterpret_cast<const uint4 *>(src + (j - slot) * stride);
        float f[8];
        unpack8(x[p], f);
#pragma unroll
        for (int i = 0; i < 8; i++)
            amax = fmaxf(amax, fabsf(f[i]));
    }
    const float old = lo < slot ? *scale : 0.f;
    amax = warp_max(amax);
    if ((tid & 31) == 0)
        red[tid >> 5] = amax;
    __syncthreads(); // the scale has been read, too
    amax = red[0];
#pragma unroll
    for (int w = 1; w < KST_THREADS / 32; w++)
        amax = fmaxf(amax, red[w]);
    const float now = fmaxf(kv8_scale_of<FMT>(fminf(amax, 65504.f)), old);
    const float inv = now > 0.f ? 1.f / now : 1.f;
    if (tid == 0)
        *scale = now;
#pragma unroll
    for (int p = 0; p < P; p++)
    {
        const int64_t j = (int64_t)lo + p * 16 + r;
        uint8_t *dst = codes + (size_t)(p * 16 + r) * YLM_HEAD_DIM;
        if (j >= slot && j < end)
        {
            float f[8];
            unpack8(x[p], f);
#pragma unroll
            for (int i = 0; i < 8; i++)
                f[i] = (fabsf(f[i]) > 65504.f ? copysignf(65504.f, f[i]) : f[i]) * inv;
            uint2 o;
            o.x = kv8_encode2<FMT>(f[0], f[1]) | (kv8_encode2<FMT>(f[2], f[3]) << 16);
            o.y = kv8_encode2<FMT>(f[4], f[5]) | (kv8_encode2<FMT>(f[6], f[7]) << 16);
            *reinterpret_cast<uint2 *>(dst) = o;
        }
        else if (j < slot && old != now)
        {
            uint2 o = *reinterpret_cast<const uint2 *>(dst);
            o.x = kv8_rescale4<FMT>(o.x, old * inv);
            o.y = kv8_rescale4<FMT>(o.y, old * inv);
            *reinterpret_cast<uint2 *>(dst) = o;
        }
    }
}

template <int FMT>
static cudaError_t store_fmt(const Kv8Cache &c, const __half *k, const __half *v, int64_t ks, int64_t vs, int t,
                             int slot, cudaStream_t s)
{
    const int blocks = (int)(((int64_t)slot + t - 1) / c.block) - slot / c.block + 1;
    const dim3 grid((unsigned)blocks, (unsigned)c.hkv, 2);
    switch (c.block)
    {
    case 16:
        kv8_store_kernel<FMT, 1><<<grid, KST_THREADS, 0, s>>>(c, k, v, ks, vs, t, slot);
        break;
    case 32:
        kv8_store_kernel<FMT, 2><<<grid, KST_THREADS, 0, s>>>(c, k, v, ks, vs, t, slot);
        break;
    case 64:
        kv8_store_kernel<FMT, 4><<<grid, KST_THREADS, 0, s>>>(c, k, v, ks, vs, t, slot);
        break;
    case 128:
        kv8_store_kernel<FMT, 8><<<grid, KST_THREADS, 0, s>>>(c, k, v, ks, vs, t, slot);
        break;
    default:
        return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t kv8_store_launch(const Kv8Cache &c, const __half *k, const __half *v, int64_t k_stride, int64_t v_stride,
                             int t, int slot, cudaStream_t s)
{
    if (t <= 0)
        return cudaSuccess;
    return c.format == KV8_E4M3 ? store_fmt<KV8_E4M3>(c, k, v, k_stride, v_stride, t, slot, s)
                                : store_fmt<KV8_INT8>(c, k, v, k_stride, v_stride, t, slot, s);
}

// ------------------------------------------------------------------ eviction
// The kept slots of one KV head: the first n_sink, the last n_recent, and of the
// others those of the largest accumulated weight, ties to the lower slot.
// A slot's key is 0xFFFFFFFF where it is protected, else the weight's bits in
// an order-preserving form (NaN, as the smallest, and -0 as +0).
__device__ __forceinline__ uint32_t evict_key(const float *acc, int i, int n_sink, int first_recent)
{
    if (i < n_sink || i >= first_recent)
        return 0xFFFFFFFFu;
    const float a = acc[i];
    if (a != a)
        return 0u;
    const uint32_t u = __float_as_uint(a + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int KEV_THREADS = 1024;

// One CTA per KV head: the key of the n_keep-th slot by four 8-bit radix steps
// (the histogram of a digit over the keys that share the digits found so
// far), then the kept slots in ascending order by block scans.
__global__ void __launch_bounds__(KEV_THREADS) kv8_select_kernel(Kv8EvictArgs a)
{
    __shared__ int hist[256];
    __shared__ uint32_t sel_prefix;
    __shared__ int sel_need, wsum[2][KEV_THREADS / 32];
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *acc = a.acc_src + (size_t)g * a.src.cap;
    float *acc_dst = a.acc_dst + (size_t)g * a.dst.cap;
    const int recent = a.n - a.n_recent;
    uint32_t prefix = 0;
    int need = a.n_keep; // of the keys equal to the prefix (so far), how many are kept
    for (int shift = 24; shift >= 0 && a.n_keep > 0; shift -= 8)
    {
        if (tid < 256)
            hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < a.n; i += KEV_THREADS)
        {
            const uint32_t key = evict_key(acc, i, a.n_sink, recent);
            if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
                atomicAdd(&hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0)
        {
            int b = 255;
            while (b > 0 && need > hist[b])
                need -= hist[b--];
            sel_prefix = prefix | ((uint32_t)b << shift);
            sel_need = need;
        }
        __syncthreads();
        prefix = sel_prefix;
        need = sel_need;
    }
    // kept: key > prefix, and the first `need` of key == prefix
    int base_gt = 0, base_eq = 0;
    for (int i0 = 0; i0 < a.n && a.n_keep > 0; i0 += KEV_THREADS)
    {
        const int i = i0 + tid;
        uint32_t key = 0;
        bool gt = false, eq = false;
        if (i < a.n)
        {
            key = evict_key(acc, i, a.n_sink, recent);
            gt = key > prefix;
            eq = key == prefix;
        }
        const uint32_t mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
        if (lane == 0)
        {
            wsum[0][warp] = __popc(mg);
            wsum[1][warp] = __popc(me);
        }
        __syncthreads();
        int pg = base_gt, pe = base_eq;
        for (int w = 0; w < KEV_THREADS / 32; w++)
        {
            if (w < warp)
            {
                pg += wsum[0][w];
                pe += wsum[1][w];
            }
            base_gt += wsum[0][w];
            base_eq += wsum[1][w];
        }
        __syncthreads();
        const uint32_t below = (1u << lane) - 1u;
        pg += __popc(mg & below);
        pe += __popc(me & below);
        if (gt || (eq && pe < need))
        {
            const int at = pg + min(pe, need);
            a.kept[(size_t)g * a.n_keep + at] = i;
            acc_dst[at] = acc[i];
        }
    }
    for (int i = a.n_keep + tid; i < a.dst.cap; i += KEV_THREADS)
        acc_dst[i] = 0.f;
}

// One CTA per (destination block, KV head, K or V): the block's scale is the
// largest of its tokens' old scales, and a token whose old block had a smaller
// one is rescaled to it. Eight threads move a token's 128 codes.
template <int FMT> __global__ void __launch_bounds__(256) kv8_move_kernel(Kv8EvictArgs a)
{
    __shared__ int from[128];
    __shared__ float old[128];
    __shared__ float top;
    const bool is_v = blockIdx.z != 0;
    const int g = blockIdx.y, b = blockIdx.x, tid = threadIdx.x;
    const int block = a.src.block, lo = b * block, m = min(block, a.n_keep - lo);
    const int src_blocks = (a.src.cap + block - 1) / block, dst_blocks = (a.dst.cap + block - 1) / block;
    const float *src_scale = (is_v ? a.src.v_scale : a.src.k_scale) + (size_t)g * src_blocks;
    const uint8_t *src = (is_v ? a.src.v : a.src.k) + (size_t)g * a.src.cap * YLM_HEAD_DIM;
    uint8_t *dst = (is_v ? a.dst.v : a.dst.k) + ((size_t)g * a.dst.cap + lo) * YLM_HEAD_DIM;
    if (tid < m)
    {
        from[tid] = a.kept[(size_t)g * a.n_keep + lo + tid];
        old[tid] = src_scale[from[tid] / block];
    }
    __syncthreads();
    if (tid < 32)
    {
        float s = 0.f;
        for (int i = tid; i < m; i += 32)
            s = fmaxf(s, old[i]);
        s = warp_max(s);
        if (tid == 0)
        {
            top = s;
            ((is_v ? a.dst.v_scale : a.dst.k_scale) + (size_t)g * dst_blocks)[b] = s;
        }
    }
    __syncthreads();
    const float inv = top > 0.f ? 1.f / top : 1.f;
    for (int e = tid; e < m * 8; e += 256)
    {
        const int i = e >> 3, c = e & 7;
        uint4 x = *reinterpret_cast<const uint4 *>(src + (size_t)from[i] * YLM_HEAD_DIM + c * 16);
        if (old[i] != top)
        {
            const float ratio = old[i] * inv;
            x.x = kv8_rescale4<FMT>(x.x, ratio);
            x.y = kv8_rescale4<FMT>(x.y, ratio);
            x.z = kv8_rescale4<FMT>(x.z, ratio);
            x.w = kv8_rescale4<FMT>(x.w, ratio);
        }
        *reinterpret_cast<uint4 *>(dst + (size_t)i * YLM_HEAD_DIM + c * 16) = x;
    }
}

cudaError_t kv8_evict_launch(const Kv8EvictArgs &a, cudaStream_t s)
{
    kv8_select_kernel<<<(unsigned)a.src.hkv, KEV_THREADS, 0, s>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || a.n_keep == 0)
        return e;
    const dim3 grid((unsigned)((a.n_keep + a.src.block - 1) / a.src.block), (unsigned)a.src.hkv, 2);
    if (a.src.format == KV8_E4M3)
        kv8_move_kernel<KV8_E4M3><<<grid, 256, 0, s>>>(a);
    else
        kv8_move_kernel<KV8_INT8><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}

} // namespace ylm
