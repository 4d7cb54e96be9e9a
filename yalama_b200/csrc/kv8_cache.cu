// The 8-bit K/V cache: storing rows and evicting slots (attention over it:
// kv8_attention.cu; formats and the power-of-two scales: kv8.cuh).
#include "kv8.cuh"
#include <cooperative_groups.h>

namespace ylm {

constexpr int KST_THREADS = 256;

// One CTA per (cache block, KV head, K or V). Thread (r, c) = (tid / 16, tid % 16)
// holds dimensions [8c, 8c + 8) of tokens 16p + r of the block, so the block's
// new rows are read once (16 bytes a thread), stay in registers while the
// block-wide maximum gives the scale, and leave as 8-byte codes.
//   s_new = max(scale_of(max |x| of the new rows), s_old if older tokens share the block)
// Infinities count as +-65504; NaN takes no part in the maximum.
// Measured (B200, 8 KV heads): one token 1.5 us, the launch; 2048 tokens 3.3 us = 3.9 TB/s of rows in and codes
// out, launch and one round of loads; the rows are read once and no other pass exists.
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

template <int FMT, int P>
static cudaError_t store_launch(const Kv8Cache &c, const __half *k, const __half *v, int64_t ks, int64_t vs, int t,
                                int slot, cudaStream_t s)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((int64_t)slot + t - 1) / c.block - slot / c.block + 1), (unsigned)c.hkv, 2);
    cfg.blockDim = dim3(KST_THREADS);
    cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, kv8_store_kernel<FMT, P>, c, k, v, ks, vs, t, slot);
}

template <int FMT>
static cudaError_t store_fmt(const Kv8Cache &c, const __half *k, const __half *v, int64_t ks, int64_t vs, int t,
                             int slot, cudaStream_t s)
{
    switch (c.block)
    {
    case 16:
        return store_launch<FMT, 1>(c, k, v, ks, vs, t, slot, s);
    case 32:
        return store_launch<FMT, 2>(c, k, v, ks, vs, t, slot, s);
    case 64:
        return store_launch<FMT, 4>(c, k, v, ks, vs, t, slot, s);
    case 128:
        return store_launch<FMT, 8>(c, k, v, ks, vs, t, slot, s);
    default:
        return cudaErrorInvalidValue;
    }
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
// The kept slots of one KV head: the first n_sink, the last n_recent (both
// protected: their weights are not looked at), and of the others those of the largest
// accumulated weight, ties to the lower slot. A weight's key is its bits in an
// order-preserving form (NaN, as the smallest, and -0 as +0).
__device__ __forceinline__ uint32_t evict_key(float a)
{
    if (a != a)
        return 0u;
    const uint32_t u = __float_as_uint(a + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int KEV_THREADS = 1024;
constexpr int KEV_WARPS = KEV_THREADS / 32;
constexpr int KEV_BINS = 2048;  // a radix step finds 11 bits of the key (the last one 10)
constexpr int KEV_MAXC = 8;     // CTAs of a cluster (the portable size)
// Slots up to which one CTA selects alone: the cluster's barriers cost more than they divide.
// One against eight CTAs a head, us for the eviction of half the slots (8 heads): 2100 slots 9.2 / 11.5,
// 6000 slots 12.4 / 12.7, 8000 slots 15.0 / 13.9, 20000 slots 31.7 / 23.8.
constexpr int KEV_ALONE = 6144;

// Exclusive scan over the CTA in thread order; *total gets the sum. The sums fit 32 bits.
__device__ __forceinline__ int kev_scan(int v, int *warp_sums, int *total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        x += lane >= o ? y : 0;
    }
    __syncthreads();
    if (lane == 31)
        warp_sums[warp] = x;
    __syncthreads();
    int s = warp_sums[lane]; // KEV_WARPS == 32: every warp scans the warps' sums
    const int own = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const int y = __shfl_up_sync(0xffffffffu, s, o);
        s += lane >= o ? y : 0;
    }
    *total = __shfl_sync(0xffffffffu, s, 31);
    return x - v + __shfl_sync(0xffffffffu, s - own, warp);
}

// One cluster per KV head, a contiguous slice of the slots per CTA. The key of the
// n_keep-th slot is found in three radix steps of 11, 11 and 10 bits: each CTA counts a
// digit over its keys that share the digits found so far and adds the counts that are
// not 0 (few: weights share few exponents) to every CTA's sums, in which each
// CTA then finds the digit. One cluster barrier a step, as each step has sums of its
// own. The kept slots are then placed in order, a warp taking consecutive slots (the
// slice stays in L1 between the passes). Protected slots are counted, not sorted: they would
// all meet in one bin.
// Measured (B200, 8 heads): 65536 slots 19 us, of which the barriers and remote additions take a
// third; 2100 slots 6.6 us (one CTA a head). One CTA a head with 8-bit digits took 192 us for 65536.
__global__ void __launch_bounds__(KEV_THREADS) kv8_select_kernel(Kv8EvictArgs a)
{
    __shared__ int hist[KEV_BINS], sums[3][KEV_BINS];
    __shared__ int warp_sums[KEV_WARPS];
    __shared__ int found[2];              // digit, and how many keys of it are kept
    __shared__ int counts[2][KEV_MAXC];   // keys above and equal to the n_keep-th, of every CTA
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)gridDim.x, rank = (int)blockIdx.x, g = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    const float *acc = a.acc_src + (size_t)g * a.src.cap;
    float *acc_dst = a.acc_dst + (size_t)g * a.dst.cap;
    const int recent = a.n - a.n_recent, per = (a.n + C - 1) / C;
    const int i0 = min(a.n, rank * per), i1 = min(a.n, i0 + per);
    for (int i = a.n_keep + rank * KEV_THREADS + tid; i < a.dst.cap; i += C * KEV_THREADS)
        acc_dst[i] = 0.f;
    if (a.n_keep == 0)
        return; // every CTA of every cluster
    for (int i = tid; i < KEV_BINS; i += KEV_THREADS)
        hist[i] = sums[0][i] = sums[1][i] = sums[2][i] = 0;
    if (C > 1) // the sums are 0 before another CTA adds to them: waited for before the first addition
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    uint32_t prefix = 0, known = 0;              // digits found, and the bits that they cover
    int need = a.n_keep - a.n_sink - a.n_recent; // of the keys equal to the prefix (so far), how many are kept
    if (need == 0)
        prefix = 0xFFFFFFFFu; // above every key
    if (need == 0 && C > 1)
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int lo = max(i0, a.n_sink), hi_end = min(i1, recent);
#pragma unroll 1
    for (int step = 0; step < 3 && need > 0; step++)
    {
        const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, bins = step < 2 ? 2048 : 1024;
        int *mine = C > 1 ? hist : sums[step];
        __syncthreads();
#pragma unroll 4
        for (int i = lo + tid; i < hi_end; i += KEV_THREADS)
        {
            const uint32_t key = evict_key(__ldg(acc + i));
            if ((key & known) == prefix)
                atomicAdd(&mine[(key >> shift) & (bins - 1)], 1);
        }
        __syncthreads();
        if (C > 1)
        {
            if (step == 0)
                asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            for (int i = tid; i < bins; i += KEV_THREADS)
            {
                const int v = hist[i];
                hist[i] = 0;
                if (v)
                    for (int c = 0; c < C; c++)
                        atomicAdd(cl.map_shared_rank(&sums[step][i], c), v);
            }
            cl.sync();
        }
        // thread t looks at the bins from the top: bins - 1 - 2t and the next one below
        const int hi = bins - 1 - 2 * tid;
        const int n1 = hi > 0 ? sums[step][hi] : 0, n0 = hi > 0 ? sums[step][hi - 1] : 0;
        int all;
        const int above = kev_scan(n0 + n1, warp_sums, &all);
        if (hi > 0 && above < need && above + n1 + n0 >= need)
        {
            const bool upper = above + n1 >= need;
            found[0] = upper ? hi : hi - 1;
            found[1] = need - above - (upper ? 0 : n1);
        }
        __syncthreads();
        prefix |= (uint32_t)found[0] << shift;
        known |= (uint32_t)(bins - 1) << shift;
        need = found[1];
    }

    // kept: key > prefix, and the first `need` of key == prefix. A warp takes consecutive slots.
    const int each = ((i1 - i0 + KEV_WARPS - 1) / KEV_WARPS + 31) / 32 * 32;
    const int w0 = min(i1, i0 + warp * each), w1 = min(i1, w0 + each);
    auto look = [&](int i, float &x, bool &more, bool &same) {
        x = i < w1 ? __ldg(acc + i) : 0.f;
        const bool held = i < a.n_sink || i >= recent;
        const uint32_t key = evict_key(x);
        more = i < w1 && (held || key > prefix);
        same = i < w1 && !held && key == prefix;
    };
    int gt = 0, eq = 0;
#pragma unroll 4
    for (int i = w0 + lane; i - lane < w1; i += 32)
    {
        float x;
        bool more, same;
        look(i, x, more, same);
        gt += more;
        eq += same;
    }
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    int gt_all, eq_all;
    gt = __shfl_sync(0xffffffffu, kev_scan(lane == 0 ? gt : 0, warp_sums, &gt_all), 0);
    eq = __shfl_sync(0xffffffffu, kev_scan(lane == 0 ? eq : 0, warp_sums, &eq_all), 0);
    if (C > 1)
    {
        if (tid < C)
        {
            *cl.map_shared_rank(&counts[0][rank], tid) = gt_all;
            *cl.map_shared_rank(&counts[1][rank], tid) = eq_all;
        }
        cl.sync();
        for (int c = 0; c < rank; c++)
        {
            gt += counts[0][c];
            eq += counts[1][c];
        }
    }
    const uint32_t below = (1u << lane) - 1u;
#pragma unroll 4
    for (int i = w0 + lane; i - lane < w1; i += 32)
    {
        float x;
        bool more, same;
        look(i, x, more, same);
        const uint32_t mg = __ballot_sync(0xffffffffu, more), me = __ballot_sync(0xffffffffu, same);
        const int eq_at = eq + __popc(me & below);
        if (more || (same && eq_at < need))
        {
            const int at = gt + __popc(mg & below) + min(eq_at, need);
            a.kept[(size_t)g * a.n_keep + at] = i;
            acc_dst[at] = x;
        }
        gt += __popc(mg);
        eq += __popc(me);
    }
}

// One CTA per (128 destination slots, KV head, K or V), whole blocks: a block's scale is the
// largest of its tokens' old scales, and a token whose old block had a smaller
// one is rescaled to it. Eight threads move a token's 128 codes, which are on
// their way before the scales are known. Launched as a programmatic dependent of the
// selection. Measured (B200): 40000 of 65536 slots, 8 heads, 82 MB in and 82 MB out, 24 us at every
// block size (26 under the profiler, which saw 84 MB read from DRAM and 34 MB written: the other writes were
// still in L2, so the memory is at 55 % of its rate meanwhile). It waits for loads and at its barriers.
// A CTA per block took 30 us with blocks of 64 and 80 us with blocks of 16.
constexpr int KEV_MOVE = 128; // the largest block
template <int FMT> __global__ void __launch_bounds__(256) kv8_move_kernel(Kv8EvictArgs a)
{
    __shared__ int from[KEV_MOVE];
    __shared__ float old[KEV_MOVE], seg[KEV_MOVE / 16], top[KEV_MOVE / 16]; // per 16 tokens: the largest; of their block
    const bool is_v = blockIdx.z != 0;
    const int g = blockIdx.y, lo = (int)blockIdx.x * KEV_MOVE, tid = threadIdx.x;
    const int block = a.src.block, shift = 31 - __clz(block), m = min(KEV_MOVE, a.n_keep - lo);
    const size_t src_blocks = (a.src.cap + block - 1) >> shift, dst_blocks = (a.dst.cap + block - 1) >> shift;
    const float *src_scale = (is_v ? a.src.v_scale : a.src.k_scale) + g * src_blocks;
    const uint8_t *src = (is_v ? a.src.v : a.src.k) + (size_t)g * a.src.cap * YLM_HEAD_DIM;
    uint8_t *dst = (is_v ? a.dst.v : a.dst.k) + ((size_t)g * a.dst.cap + lo) * YLM_HEAD_DIM;
    pdl_wait();
    int f = 0;
    if (tid < m)
        from[tid] = f = a.kept[(size_t)g * a.n_keep + lo + tid];
    __syncthreads();
    uint4 x[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
    {
        const int i = (tid >> 3) + 32 * k;
        if (i < m)
            x[k] = *reinterpret_cast<const uint4 *>(src + (size_t)from[i] * YLM_HEAD_DIM + (tid & 7) * 16);
    }
    if (tid < KEV_MOVE)
    {
        float s = tid < m ? src_scale[f >> shift] : 0.f;
        old[tid] = s;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
            s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, o));
        if ((tid & 15) == 0)
            seg[tid >> 4] = s;
    }
    __syncthreads();
    if (tid < KEV_MOVE / 16)
    {
        const int s0 = tid >> (shift - 4) << (shift - 4); // the block's first 16 tokens
        float t = seg[s0];
        for (int k = 1; k < block / 16; k++)
            t = fmaxf(t, seg[s0 + k]);
        top[tid] = t;
        if (s0 == tid && tid * 16 < m)
            ((is_v ? a.dst.v_scale : a.dst.k_scale) + g * dst_blocks)[(lo + tid * 16) >> shift] = t;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; k++)
    {
        const int i = (tid >> 3) + 32 * k;
        if (i >= m)
            continue;
        const float now = top[i >> 4];
        if (old[i] != now)
        {
            const float ratio = now > 0.f ? old[i] / now : 1.f;
            x[k].x = kv8_rescale4<FMT>(x[k].x, ratio);
            x[k].y = kv8_rescale4<FMT>(x[k].y, ratio);
            x[k].z = kv8_rescale4<FMT>(x[k].z, ratio);
            x[k].w = kv8_rescale4<FMT>(x[k].w, ratio);
        }
        *reinterpret_cast<uint4 *>(dst + (size_t)i * YLM_HEAD_DIM + (tid & 7) * 16) = x[k];
    }
}

cudaError_t kv8_evict_launch(const Kv8EvictArgs &a, cudaStream_t s)
{
    const int C = a.n <= KEV_ALONE ? 1 : KEV_MAXC;
    cudaLaunchAttribute at[1];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)C, (unsigned)a.src.hkv);
    cfg.blockDim = dim3(KEV_THREADS);
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kv8_select_kernel, a);
    if (e != cudaSuccess || a.n_keep == 0)
        return e;
    cfg.gridDim = dim3((unsigned)((a.n_keep + KEV_MOVE - 1) / KEV_MOVE), (unsigned)a.src.hkv, 2);
    cfg.blockDim = dim3(256);
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    return a.src.format == KV8_E4M3 ? cudaLaunchKernelEx(&cfg, kv8_move_kernel<KV8_E4M3>, a)
                                    : cudaLaunchKernelEx(&cfg, kv8_move_kernel<KV8_INT8>, a);
}

} // namespace ylm
