// Log probabilities of rows of FP16 logits: of one given id per row, the
// row's entropy, and its most likely ids.
//   m = max x, z = sum over the others of e^(x - m), ln Z = m + ln(1 + z)
//   logprob = (x_id - m) - log1p(z)
//   entropy = log1p(z) + sum e^(x - m) (m - x) / (1 + z)
// The maximum's own term is left out of z, so a nearly certain row keeps its
// small log probabilities (log1p(z) where 1 + z would round to 1), and the
// entropy is a sum of terms of one sign.
//
// A row is read once, by the C CTAs of a cluster (1 for many rows, 8 for few),
// each on a contiguous part of it, 16 bytes a load. The maximum that the
// terms refer to is shared by a warp, so that it moves seldom.
//
// The alternatives need no second pass over the row: each thread also keeps the
// largest value it saw. With T the n_top-th largest of these, at least n_top ids have
// a value >= T, so every alternative does, and only the threads whose largest is >= T
// (n_top and a few) have any: their warps read those threads' parts again (L1 or
// L2), collect the ids >= T, and rank them by counting. Where that collects
// more than LGP_CAP (many equal values, or the largest ones all in one thread's
// part) or the row has a NaN, a radix select over the part takes its place.
#include "ylm_common.cuh"
#include <algorithm>
#include <cooperative_groups.h>

namespace ylm {

namespace cg = cooperative_groups;

constexpr int LGP_THREADS = 512;
constexpr int LGP_WARPS = LGP_THREADS / 32;
constexpr int LGP_U = 4;      // 16-byte loads in flight per thread
constexpr int LGP_CAP = 512;  // collected candidates per CTA
constexpr int LGP_TOP = 64;   // largest n_top
constexpr uint32_t LGP_LOWEST = 0x0400u; // ord16 of the lowest finite value: what lies below is -inf

// Running (max, z, w): z = sum e^(x - m) without one maximal element, w = sum e^(x - m) (m - x).
struct LseState
{
    float m, z, w;
};

__device__ __forceinline__ LseState lse_merge(LseState a, LseState b)
{
    if (b.m > a.m)
    {
        const LseState t = a;
        a = b;
        b = t;
    }
    if (b.m == -INFINITY)
    {
        a.z += b.z; // 0, or NaN
        return a;
    }
    // b's terms relative to a.m: e^(x - a.m) = e^(x - b.m) f, a.m - x = (b.m - x) + d
    const float d = a.m - b.m, f = expf(-d), zb = 1.f + b.z;
    a.z += zb * f;
    a.w += (b.w + zb * d) * f;
    return a;
}

__device__ __forceinline__ float lgp_ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Key of an alternative: NaN above everything, then the value (-0 as +0), then the lower id.
__device__ __forceinline__ uint32_t lgp_ord(uint32_t u)
{
    if ((u & 0x7FFFu) > 0x7C00u)
        u = 0x7FFFu;
    if (u == 0x8000u)
        u = 0u;
    return ord16(u);
}

// The part of a row that a CTA works on, as 16-byte vectors at 16-byte aligned
// addresses: vector v holds ids [8 v - off, 8 v - off + 8). Ids outside the row
// and masked ones read as -inf.
struct LgpRow
{
    const __half *x;
    const uint32_t *bits;
    int vocab, off;

    __device__ __forceinline__ uint4 load(int v) const
    {
        const int i0 = 8 * v - off;
        uint4 r;
        if (i0 >= 0 && i0 + 8 <= vocab)
            r = __ldg(reinterpret_cast<const uint4 *>(x + i0));
        else
        {
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                h[i] = i0 + i >= 0 && i0 + i < vocab ? __half_as_ushort(x[i0 + i]) : 0xFC00u;
            r = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        }
        if (bits)
        {
            const int last = (vocab - 1) >> 5, w = max(i0, 0) >> 5;
            const uint64_t two = (uint64_t)bits[w] | (uint64_t)bits[min(w + 1, last)] << 32;
            const uint32_t b = i0 >= 0 ? (uint32_t)(two >> (i0 & 31)) : (uint32_t)two << -i0;
            uint32_t *p = reinterpret_cast<uint32_t *>(&r);
#pragma unroll
            for (int i = 0; i < 4; i++)
            {
                if (b >> (2 * i) & 1u)
                    p[i] = (p[i] & 0xFFFF0000u) | 0xFC00u;
                if (b >> (2 * i + 1) & 1u)
                    p[i] = (p[i] & 0xFFFFu) | 0xFC000000u;
            }
        }
        return r;
    }
};

struct LgpShared
{
    LseState st[LGP_WARPS];
    LseState part;            // this CTA's
    int n_top;                // candidates in top
    int count;                // collected
    int scan[LGP_WARPS];
    int hist[256];
    int sel[2];
    uint64_t top[LGP_TOP];    // this CTA's best, best first
    uint64_t cand[LGP_CAP];   // collected; in rank 0 of a cluster, later every CTA's best
};

// sh.cand[0, m) ranked into sh.top[0, min(m, n)): a key's place is the number of larger ones (keys are distinct)
__device__ __forceinline__ void lgp_rank(LgpShared &sh, int m, int n)
{
    for (int i = threadIdx.x; i < m; i += LGP_THREADS)
    {
        const uint64_t k = sh.cand[i];
        int r = 0;
        for (int j = 0; j < m; j++)
            r += sh.cand[j] > k;
        if (r < n)
            sh.top[r] = k;
    }
    if (threadIdx.x == 0)
        sh.n_top = min(m, n);
}

// The n best of vectors [v0, v1) by two 8-bit radix steps, whatever their
// values: sh.cand gets those above the n-th value T in any order, then the first of
// those equal to T by id.
__device__ void lgp_select(const LgpRow &row, int v0, int v1, int n, LgpShared &sh)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t prefix = 0;
    int need = n;
    for (int step = 0; step < 2; step++)
    {
        __syncthreads();
        for (int i = tid; i < 256; i += LGP_THREADS)
            sh.hist[i] = 0;
        __syncthreads();
        for (int v = v0 + tid; v < v1; v += LGP_THREADS)
        {
            const uint4 r = row.load(v);
            const uint32_t *p = reinterpret_cast<const uint32_t *>(&r);
            for (int i = 0; i < 8; i++)
            {
                const uint32_t o = lgp_ord(p[i >> 1] >> (16 * (i & 1)) & 0xFFFFu);
                if (o >= LGP_LOWEST && (step == 0 || o >> 8 == prefix))
                    atomicAdd(&sh.hist[step == 0 ? o >> 8 : o & 255u], 1);
            }
        }
        __syncthreads();
        if (tid == 0)
        {
            int b = 255;
            while (b > 0 && need > sh.hist[b])
                need -= sh.hist[b--];
            sh.sel[0] = b;
            sh.sel[1] = need;
            sh.count = 0;
        }
        __syncthreads();
        prefix = prefix << 8 | (uint32_t)sh.sel[0];
        need = sh.sel[1];
    }
    int taken = 0; // of those equal to T
    for (int base = v0; base < v1; base += LGP_THREADS)
    {
        uint4 r = make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);
        if (base + tid < v1)
            r = row.load(base + tid);
        const uint32_t *p = reinterpret_cast<const uint32_t *>(&r);
        const uint32_t id0 = (uint32_t)(8 * (base + tid) - row.off);
        int eq = 0;
        for (int i = 0; i < 8; i++)
        {
            const uint32_t o = lgp_ord(p[i >> 1] >> (16 * (i & 1)) & 0xFFFFu);
            eq += o == prefix && o >= LGP_LOWEST;
            if (o > prefix && o >= LGP_LOWEST)
                sh.cand[atomicAdd(&sh.count, 1)] = make_key(o, id0 + i);
        }
        int before = eq;
        for (int o = 1; o < 32; o <<= 1)
        {
            const int y = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o)
                before += y;
        }
        if (lane == 31)
            sh.scan[warp] = before;
        __syncthreads();
        int at = taken + before - eq;
        for (int w = 0; w < LGP_WARPS; w++)
        {
            at += w < warp ? sh.scan[w] : 0;
            taken += sh.scan[w];
        }
        for (int i = 0; i < 8; i++)
        {
            const uint32_t o = lgp_ord(p[i >> 1] >> (16 * (i & 1)) & 0xFFFFu);
            if (o == prefix && o >= LGP_LOWEST && at++ < need)
                sh.cand[atomicAdd(&sh.count, 1)] = make_key(o, id0 + i);
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(LGP_THREADS, 2) logprobs_kernel(LogprobArgs a)
{
    __shared__ LgpShared sh;
    const int C = (int)gridDim.x, rank = (int)blockIdx.x;
    const int64_t ri = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (ri >= a.rows) // the whole cluster: blockIdx.x is the rank in it
        return;
    LgpRow row;
    row.x = a.logits + ri * a.ld;
    row.bits = a.mask_bits;
    row.vocab = (int)a.vocab;
    row.off = (int)(reinterpret_cast<uintptr_t>(row.x) >> 1 & 7u);
    const int nv = (int)((a.vocab + row.off + 7) / 8), per = (nv + C - 1) / C;
    const int v0 = min(nv, rank * per), v1 = min(nv, v0 + per);

    // ---- one pass: the warp's reference m, this thread's z, w and largest value
    LseState s = {-INFINITY, 0.f, 0.f};
    float ref = 0.f; // m, or 0 while there is none
    __half2 tmax2 = __half2half2(__ushort_as_half(0xFC00u));
    for (int v = v0 + tid; v - lane < v1; v += LGP_THREADS * LGP_U)
    {
        uint4 r[LGP_U];
#pragma unroll
        for (int u = 0; u < LGP_U; u++)
            r[u] = v + u * LGP_THREADS < v1 ? row.load(v + u * LGP_THREADS)
                                            : make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);
        const __half2 *h = reinterpret_cast<const __half2 *>(r);
        __half2 um = h[0];
#pragma unroll
        for (int i = 1; i < 4 * LGP_U; i++)
            um = __hmax2(um, h[i]);
        um = __hmax2(um, __half2half2(__ushort_as_half(0xFC00u))); // NaN only: -inf
        tmax2 = __hmax2(tmax2, um);
        const uint32_t mine = ord16(__half_as_ushort(__hmax(__low2half(um), __high2half(um))));
        const float top = h2f(__ushort_as_half((unsigned short)unord16(__reduce_max_sync(0xffffffffu, mine))));
        bool skip = false; // this lane leaves out one element equal to the new maximum
        if (top > s.m)
        {
            const uint32_t has = __ballot_sync(0xffffffffu, unord16(mine) == __half_as_ushort(__float2half_rn(top)));
            skip = lane == __ffs(has) - 1;
            // what was summed so far, with the former maximum, which lane `owner` alone counts
            const bool counted = s.m != -INFINITY && lane == 0;
            const float d = top - (s.m == -INFINITY ? top : s.m), f = lgp_ex2(-d * 1.4426950408889634f);
            const float zo = s.z + (counted ? 1.f : 0.f);
            s.w = (s.w + zo * d) * f;
            s.z = zo * f;
            s.m = ref = top;
        }
        if (skip)
        {
#pragma unroll
            for (int i = 0; i < 4 * LGP_U; i++)
            {
                const float2 f = __half22float2(h[i]);
#pragma unroll
                for (int j = 0; j < 2; j++)
                {
                    const float x = j ? f.y : f.x;
                    if (skip && x == top)
                    {
                        skip = false;
                        continue;
                    }
                    const float d = x - ref, e = lgp_ex2(d * 1.4426950408889634f);
                    s.z += e;
                    s.w -= e * fmaxf(d, -200.f);
                }
            }
        }
        else
        {
#pragma unroll
            for (int i = 0; i < 4 * LGP_U; i++)
            {
                const float2 f = __half22float2(h[i]);
                // d: -inf, far below any e > 0, would make 0 * -inf of the entropy's term
                const float d0 = f.x - ref, d1 = f.y - ref;
                const float e0 = lgp_ex2(d0 * 1.4426950408889634f), e1 = lgp_ex2(d1 * 1.4426950408889634f);
                s.z += e0 + e1;
                s.w -= e0 * fmaxf(d0, -200.f) + e1 * fmaxf(d1, -200.f);
            }
        }
    }
    // the warp's sum (its one left-out maximum stays out), then the CTA's
    for (int o = 16; o > 0; o >>= 1)
    {
        s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
        s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
    }
    if (lane == 0)
        sh.st[warp] = s;
    if (tid == 0)
        sh.count = 0;
    const bool nan = __syncthreads_or(s.z != s.z);
    if (warp == 0)
    {
        LseState t = lane < LGP_WARPS ? sh.st[lane] : LseState{-INFINITY, 0.f, 0.f};
        for (int o = LGP_WARPS / 2; o > 0; o >>= 1)
            t = lse_merge(t, LseState{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.z, o),
                                      __shfl_xor_sync(0xffffffffu, t.w, o)});
        if (lane == 0)
            sh.part = t;
    }

    // ---- this CTA's best ids
    if (a.n_top)
    {
        const uint32_t mine = lgp_ord(__half_as_ushort(__hmax(__low2half(tmax2), __high2half(tmax2))));
        uint32_t T = 0;
        bool whole = nan;
        if (!whole)
        {
#pragma unroll 1
            for (int b = 15; b >= 0; b--) // the largest T that n_top threads reach
                if (__syncthreads_count(mine >= (T | 1u << b)) >= a.n_top)
                    T |= 1u << b;
            T = max(T, LGP_LOWEST);
            for (uint32_t left = __ballot_sync(0xffffffffu, mine >= T); left; left &= left - 1)
            {
                const int owner = warp * 32 + __ffs(left) - 1;
                for (int v = v0 + owner + lane * LGP_THREADS; v < v1; v += 32 * LGP_THREADS)
                {
                    const uint4 r = row.load(v);
                    const uint32_t *p = reinterpret_cast<const uint32_t *>(&r);
#pragma unroll
                    for (int i = 0; i < 8; i++)
                    {
                        const uint32_t o = lgp_ord(p[i >> 1] >> (16 * (i & 1)) & 0xFFFFu);
                        if (o >= T)
                        {
                            const int at = atomicAdd(&sh.count, 1);
                            if (at < LGP_CAP)
                                sh.cand[at] = make_key(o, (uint32_t)(8 * v - row.off + i));
                        }
                    }
                }
            }
            __syncthreads();
            whole = sh.count > LGP_CAP;
        }
        if (whole) // uniform over the CTA
            lgp_select(row, v0, v1, a.n_top, sh);
        __syncthreads();
        lgp_rank(sh, sh.count, a.n_top);
    }
    __syncthreads();

    // ---- rank 0 joins the parts and writes the row
    cg::cluster_group cl = cg::this_cluster();
    if (C > 1)
        cl.sync();
    if (rank == 0)
    {
        LseState t = sh.part;
        for (int c = 1; c < C; c++)
            t = lse_merge(t, *cl.map_shared_rank(&sh.part, c));
        const bool bad = t.z != t.z || t.m == INFINITY;
        const bool none = t.m == -INFINITY && !bad;
        const float lz = bad ? NAN : log1pf(t.z);
        if (tid == 0 && a.logprob)
        {
            const int64_t id = a.ids[ri];
            float lp = -INFINITY;
            if (id >= 0 && id < a.vocab && !(a.mask_bits && (a.mask_bits[id >> 5] >> (id & 31) & 1u)))
            {
                const float x = h2f(row.x[id]);
                lp = bad ? NAN : x == -INFINITY ? -INFINITY : (x - t.m) - lz;
            }
            a.logprob[ri] = lp;
        }
        if (tid == 0 && a.entropy)
            a.entropy[ri] = bad ? NAN : none ? 0.f : lz + t.w / (1.f + t.z);
        if (a.n_top)
        {
            if (C > 1)
            {
                // the parts' lists side by side (at most 8 x 64), ranked again
                int m = 0;
                for (int c = 0; c < C; c++)
                {
                    const int k = *cl.map_shared_rank(&sh.n_top, c);
                    const uint64_t *from = cl.map_shared_rank(&sh.top[0], c);
                    for (int i = tid; i < k; i += LGP_THREADS)
                        sh.cand[m + i] = from[i];
                    m += k;
                }
                __syncthreads();
                lgp_rank(sh, m, a.n_top);
                __syncthreads();
            }
            if (tid < a.n_top)
            {
                const bool is = tid < sh.n_top;
                const uint64_t key = is ? sh.top[tid] : 0;
                const float x = h2f(__ushort_as_half((unsigned short)unord16((uint32_t)(key >> 32))));
                a.top_ids[ri * a.n_top + tid] = is ? (int64_t)key_idx(key) : -1;
                a.top_logprobs[ri * a.n_top + tid] = !is ? -INFINITY : bad ? NAN : (x - t.m) - lz;
            }
        }
    }
    if (C > 1)
        cl.sync(); // the parts stay until rank 0 has read them
}

cudaError_t logprobs_launch(const LogprobArgs &a, int num_sms, cudaStream_t s)
{
    if (a.rows <= 0)
        return cudaSuccess;
    int C = 8;
    while (C > 1 && (int64_t)a.rows * (C / 2) >= 4 * num_sms)
        C /= 2;
    cudaLaunchConfig_t cfg = {};
    const unsigned y = (unsigned)std::min(a.rows, 32768);
    cfg.gridDim = dim3((unsigned)C, y, (unsigned)((a.rows + (int64_t)y - 1) / y));
    cfg.blockDim = dim3(LGP_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel, a);
}

cudaError_t logprobs_prepare() { return cudaSuccess; }

} // namespace ylm
