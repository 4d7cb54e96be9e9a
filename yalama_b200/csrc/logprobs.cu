// Log probabilities of rows of FP16 logits: of one given id per row, the
// row's entropy, and its most likely ids.
//   m = max x, z = sum over the others of e^(x - m), ln Z = m + ln(1 + z)
//   logprob = (x_id - m) - log1p(z)
//   entropy = log1p(z) + sum e^(x - m) (m - x) / (1 + z)
// The maximum's own term is left out of z, so a nearly certain row keeps its
// small log probabilities (log1p(z) where 1 + z would round to 1), and the
// entropy is a sum of terms of one sign. The sums are FP32: a thread adds vocab / (512 C)
// terms one after another to each of its two, which bounds their error at
// vocab / 512 steps of 2^-24 for the longest rows (rounding both ways keeps it near the square root).
//
// A row is read once, by the C CTAs of a cluster (1 for many rows, 8 for few),
// each on a contiguous part of it, 16 bytes a load. The maximum that the
// terms refer to is shared by a warp, so that it moves seldom.
//
// The alternatives need no second pass over the row: each thread also keeps the
// largest value it saw in each half of its vectors. With T the n_top-th largest of the threads'
// values, at least n_top ids have a value >= T, so every alternative does, and only the halves
// whose largest is >= T (n_top and a few) have any: the CTA reads those again,
// dealt out over all its threads, collects the ids >= T, and ranks them by
// counting. Where that collects more than LGP_CAP (many equal values, or the largest
// ones all in one thread's part) or the row has a NaN, a radix select over the part
// takes its place. Rank 0 of the cluster joins the CTAs' sums and lists.
//
// Measured (B200): 600 rows of 151936 ids 45.9 us, with 8 alternatives 51.2 us = 3.6 TB/s (of DRAM also the halves
// read again, a tenth of the row). Without any arithmetic
// the same loads take 36 us (all CTAs start and end together, and 8 SMs have five rows where the others
// have four); the exponentials and sums add the rest (about nine instructions an id, one of them ex2). One row of
// 128256 ids with 20 alternatives 9.5 us, with 64 11.4 us: a chain of latencies (2.5 us the pass, about 1 us each the sums, the threshold,
// the candidates, the cluster barrier and the join). Packed FP32 pairs, two loads in flight instead of four,
// and the next loads issued before the current sums gave the same or longer times; a pass per alternative (the
// first version) 1301 us and 543 us. Five CTAs an SM hold the kernel to 48 registers, for which it spills 12 bytes
// a thread. A mask puts every vector on the checked path: one row of 128256 ids 7.8 us against 6.1.
#include "ylm_common.cuh"
#include <cooperative_groups.h>

namespace ylm {

namespace cg = cooperative_groups;

constexpr int LGP_THREADS = 256;
constexpr int LGP_WARPS = LGP_THREADS / 32;
constexpr int LGP_U = 4;      // 16-byte loads in flight per thread: a unit, of two halves
static_assert(LGP_U == 4, "a half is two vectors");
constexpr int LGP_CAP = 512;  // collected candidates per CTA
constexpr int LGP_TOP = 64;   // largest n_top
constexpr int LGP_MAXC = 8;   // largest cluster (the portable size)
// CTAs per row: halved from LGP_MAXC while that leaves LGP_FILL CTAs per SM or parts
// are shorter than LGP_PART ids. Measured, us for 1 / 2 / 4 / 8 CTAs a row (8 alternatives): 151936 ids, 16 rows
// 22.5 / 17.8 / 13.7 / 12.7, 74 rows 23.2 / 18.7 / 16.7 / 18.7, 200 rows 34.1 / 27.3 / 33.9 / 41.2,
// 450 rows 43.6 / 50.2 / 57.0 / 79.9; 32768 ids, 16 rows 10.5 / 9.9 / 9.1 / 9.8, 200 rows 12.1 / 12.0 / 16.8 / 26.0.
constexpr int LGP_FILL = 2;
constexpr int LGP_PART = 8192;
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
    LseState parts[LGP_MAXC]; // rank 0: every CTA's
    int n_top;                // keys in top
    int counts[LGP_MAXC];     // rank 0: keys in every CTA's top
    int count;                // keys in cand
    int scan[LGP_WARPS];
    int hist[256];
    int sel[2];
    uint32_t T;
    bool nan, low;
    uint16_t most[LGP_THREADS];         // each thread's largest value (ord16)
    uint64_t top[LGP_TOP];              // the best, best first
    alignas(16) uint64_t cand[LGP_CAP]; // collected keys
    alignas(16) uint64_t lists[LGP_MAXC * LGP_TOP]; // rank 0: every CTA's best, 0 behind its last
    uint16_t owners[LGP_THREADS * 2]; // halves of threads' vectors with candidates
    int n_owners;
};

// sh.cand[0, m) ranked into sh.top[0, n): a key's place is the number of larger ones (the
// keys are distinct; where m is odd, sh.cand[m] is 0). One copy of the code for both
// calls: the second one finds it in the instruction cache, worth 1.3 us of one row's 11.1
// (a merge by bisection, fewer steps, took that longer).
__device__ __noinline__ void lgp_rank(LgpShared &sh, int m, int n)
{
    const int pairs = (m + 1) / 2;
    const ulonglong2 *two = reinterpret_cast<const ulonglong2 *>(sh.cand);
    for (int i = threadIdx.x; i < m; i += LGP_THREADS)
    {
        const uint64_t k = sh.cand[i];
        int r = 0;
#pragma unroll 4
        for (int j = 0; j < pairs; j++)
        {
            const ulonglong2 t = two[j];
            r += (t.x > k) + (t.y > k);
        }
        if (r < n)
            sh.top[r] = k;
    }
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

// The warps' states joined (in warp 0, which sh.nan and sh.low describe to all).
__device__ __forceinline__ LseState lgp_block(LseState s, LgpShared &sh)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0)
        sh.st[warp] = s;
    __syncthreads();
    if (warp == 0)
    {
        s = lane < LGP_WARPS ? sh.st[lane] : LseState{-INFINITY, 0.f, 0.f};
        for (int o = LGP_WARPS / 2; o > 0; o >>= 1)
            s = lse_merge(s, LseState{__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.z, o),
                                      __shfl_xor_sync(0xffffffffu, s.w, o)});
        if (lane == 0)
        {
            sh.nan = s.z != s.z;
            sh.low = s.m < -65000.f;
        }
    }
    __syncthreads();
    return s;
}

__global__ void __launch_bounds__(LGP_THREADS, 5) logprobs_kernel(LogprobArgs a)
{
    __shared__ LgpShared sh;
    const int C = (int)gridDim.x, rank = (int)blockIdx.x;
    const int64_t ri = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (ri >= a.rows) // the whole cluster: blockIdx.x is the rank in it
        return;
    // the other CTAs write into rank 0's shared memory once all have started:
    // arrive now, wait before the first such write
    if (C > 1)
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    LgpRow row;
    row.x = a.logits + ri * a.ld;
    row.bits = a.mask_bits;
    row.vocab = (int)a.vocab;
    row.off = (int)(reinterpret_cast<uintptr_t>(row.x) >> 1 & 7u);
    const int nv = (int)((a.vocab + row.off + 7) / 8), per = (nv + C - 1) / C;
    const int v0 = min(nv, rank * per), v1 = min(nv, v0 + per);

    // the given id's logit, early: two dependent loads
    bool has_given = false;
    float given = 0.f;
    if (rank == 0 && tid == 0 && a.logprob)
    {
        const int64_t id = a.ids[ri];
        has_given = id >= 0 && id < a.vocab && !(a.mask_bits && (a.mask_bits[id >> 5] >> (id & 31) & 1u));
        given = has_given ? h2f(row.x[id]) : 0.f;
    }

    // ---- one pass. Terms are 2^t, t = x L - c with L = log2 e and c = m L rounded
    // (one multiply-add an element, whatever the size of m); c's rounding error
    // d = m L - c, the t of the maximum itself, is taken out at the end. Per
    // thread z' = sum 2^t and w' = sum 2^t t, per warp m. Logits below the lowest
    // finite one count as that here: their terms vanish unless m is as low.
    constexpr float L = 1.4426950408889634f;
    const __half2 lowest = __half2half2(__ushort_as_half(0xFBFFu));
    float m = -INFINITY, c = 0.f, delta = 0.f;
    float2 z = make_float2(0.f, 0.f), w = z; // two of each, for the two halves of a pair
    __half2 tmax2[2] = {lowest, lowest}; // the largest values seen in the first and second half of this thread's units
    const int inner = min(v1, nv - 1); // vectors (0, inner) lie in the row whole
    for (int v = v0 + tid; v - lane < v1; v += LGP_THREADS * LGP_U)
    {
        uint4 r[LGP_U];
        const int first = v - lane, last = first + 31 + (LGP_U - 1) * LGP_THREADS; // the warp's vectors
        if (!row.bits && first > 0 && last < inner)
        {
#pragma unroll
            for (int u = 0; u < LGP_U; u++)
                r[u] = __ldg(reinterpret_cast<const uint4 *>(row.x + (8 * v - row.off)) + u * LGP_THREADS);
        }
        else
        {
#pragma unroll
            for (int u = 0; u < LGP_U; u++)
                r[u] = v + u * LGP_THREADS < v1 ? row.load(v + u * LGP_THREADS)
                                                : make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);
        }
        __half2 *h = reinterpret_cast<__half2 *>(r);
        __half2 um;
#pragma unroll
        for (int u = 0; u < LGP_U; u++)
        {
#pragma unroll
            for (int i = 4 * u; i < 4 * u + 4; i++)
            {
                h[i] = __hmax2_nan(h[i], lowest);
                tmax2[u >> 1] = __hmax2(tmax2[u >> 1], h[i]);
            }
        }
        um = __hmax2(tmax2[0], tmax2[1]);
        const uint32_t mine = ord16(__half_as_ushort(__hmax(__low2half(um), __high2half(um))));
        const uint32_t most = __reduce_max_sync(0xffffffffu, mine);
        const float top = h2f(__ushort_as_half((unsigned short)unord16(most)));
        if (top > m)
        {
            // the former maximum, which lane 0 counts, joins the sums, in the new unit
            const float cn = top * L, dn = fmaf(top, L, -cn);
            if (m > -INFINITY)
            {
                const float own = lane == 0 ? lgp_ex2(delta) : 0.f, shift = c - cn, f = lgp_ex2(shift);
                z.x += own;
                w.x = (w.x + own * delta + z.x * shift) * f;
                w.y = (w.y + z.y * shift) * f;
                z.x *= f;
                z.y *= f;
            }
            m = top;
            c = cn;
            delta = dn;
            // one element equal to the new one is left out: it becomes the lowest value
            if (lane == __ffs(__ballot_sync(0xffffffffu, mine == most)) - 1)
            {
                const __half th = __float2half_rn(top), low = __ushort_as_half(0xFBFFu);
                bool open = true;
#pragma unroll
                for (int i = 0; i < 4 * LGP_U; i++)
                {
                    const bool x = open && __heq(__low2half(h[i]), th), y = open && !x && __heq(__high2half(h[i]), th);
                    h[i] = __halves2half2(x ? low : __low2half(h[i]), y ? low : __high2half(h[i]));
                    open = open && !x && !y;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4 * LGP_U; i++)
        {
            const float2 x = __half22float2(h[i]);
            const float t0 = fmaf(x.x, L, -c), t1 = fmaf(x.y, L, -c), e0 = lgp_ex2(t0), e1 = lgp_ex2(t1);
            z.x += e0;
            z.y += e1;
            w.x = fmaf(e0, t0, w.x);
            w.y = fmaf(e1, t1, w.y);
        }
    }
    LseState s;
    {
        const float zs = warp_sum(z.x + z.y), ws = warp_sum(w.x + w.y), f = lgp_ex2(-delta);
        s = LseState{m, zs * f, -0.69314718055994531f * (ws - delta * zs) * f};
    }
    s = lgp_block(s, sh);
    if (tid == 0)
        sh.count = 0;
    const bool nan = sh.nan;
    if (sh.low) // uniform: an empty part, or one whose logits are as low as what stood in for -inf
    {
        LseState t = {-INFINITY, 0.f, 0.f};
        for (int v = v0 + tid; v < v1; v += LGP_THREADS)
        {
            const uint4 r = row.load(v);
            const __half2 *h = reinterpret_cast<const __half2 *>(&r);
#pragma unroll 1
            for (int i = 0; i < 8; i++)
            {
                const float x = h2f(i & 1 ? __high2half(h[i >> 1]) : __low2half(h[i >> 1]));
                t = x != x ? LseState{t.m, x, x} : x > -INFINITY ? lse_merge(t, LseState{x, 0.f, 0.f}) : t;
            }
        }
        for (int o = 16; o > 0; o >>= 1)
            t = lse_merge(t, LseState{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.z, o),
                                      __shfl_xor_sync(0xffffffffu, t.w, o)});
        s = lgp_block(t, sh);
    }

    // ---- this CTA's best ids
    if (a.n_top)
    {
        bool whole = nan;
        if (!whole)
        {
            uint32_t mine[2], most = 0;
#pragma unroll
            for (int u = 0; u < 2; u++)
            {
                mine[u] = lgp_ord(__half_as_ushort(__hmax(__low2half(tmax2[u]), __high2half(tmax2[u]))));
                most = max(most, mine[u]);
            }
            // the largest T that n_top threads reach, bit by bit, by one warp
            sh.most[tid] = (uint16_t)most;
            __syncthreads();
            if (warp == 0)
            {
                uint32_t v[LGP_WARPS];
#pragma unroll
                for (int i = 0; i < LGP_WARPS; i++)
                    v[i] = sh.most[i * 32 + lane];
                uint32_t T = 0;
                // to 12 bits: a lower T only lets a few more candidates in
#pragma unroll 1
                for (int b = 15; b >= 4; b--)
                {
                    int n = 0;
#pragma unroll
                    for (int i = 0; i < LGP_WARPS; i++)
                        n += v[i] >= (T | 1u << b);
                    if (__reduce_add_sync(0xffffffffu, n) >= a.n_top)
                        T |= 1u << b;
                }
                if (lane == 0)
                {
                    sh.T = max(T, LGP_LOWEST);
                    sh.n_owners = 0;
                }
            }
            __syncthreads();
            const uint32_t T = sh.T;
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (mine[u] >= T)
                    sh.owners[atomicAdd(&sh.n_owners, 1)] = (uint16_t)(u * (LGP_U / 2) * LGP_THREADS + tid);
            __syncthreads();
            // the owners' vectors again, dealt out over the CTA: consecutive threads take consecutive owners
            constexpr int STEP = LGP_THREADS * LGP_U;
            const int n_owners = sh.n_owners, total = n_owners * (LGP_U / 2) * ((v1 - v0 + STEP - 1) / STEP);
            for (int i = tid; i < total; i += LGP_THREADS)
            {
                const int k = i / n_owners; // unit k / 2, vector k % 2 of the owner's half
                const int v = v0 + (k >> 1) * STEP + (k & 1) * LGP_THREADS + sh.owners[i - k * n_owners];
                if (v >= v1)
                    continue;
                const uint4 r = row.load(v);
                const uint32_t *p = reinterpret_cast<const uint32_t *>(&r);
#pragma unroll
                for (int j = 0; j < 8; j++)
                {
                    const uint32_t o = lgp_ord(p[j >> 1] >> (16 * (j & 1)) & 0xFFFFu);
                    if (o >= T)
                    {
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < LGP_CAP)
                            sh.cand[at] = make_key(o, (uint32_t)(8 * v - row.off + j));
                    }
                }
            }
            __syncthreads();
            whole = sh.count > LGP_CAP;
        }
        if (whole) // uniform over the CTA
            lgp_select(row, v0, v1, a.n_top, sh);
        __syncthreads();
        if (tid == 0)
        {
            sh.n_top = min(sh.count, a.n_top);
            if (sh.count & 1)
                sh.cand[sh.count] = 0;
        }
        __syncthreads();
        lgp_rank(sh, sh.count, a.n_top);
    }

    // ---- rank 0 joins the parts and writes the row
    cg::cluster_group cl = cg::this_cluster();
    __syncthreads();
    if (C > 1)
    {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (tid == 0)
        {
            sh.count = 0;
            *cl.map_shared_rank(&sh.parts[rank], 0) = s;
            *cl.map_shared_rank(&sh.counts[rank], 0) = a.n_top ? sh.n_top : 0;
        }
        if (tid < a.n_top)
            *cl.map_shared_rank(&sh.lists[rank * a.n_top + tid], 0) = tid < sh.n_top ? sh.top[tid] : 0ull;
        cl.sync();
        if (rank != 0)
            return;
        if (a.n_top)
        {
            // every list has ceil(n / C) keys that reach its own ceil(n / C)-th: the smallest of these is reached by
            // n keys, and what lies below it is not among the n best
            const int part = (a.n_top + C - 1) / C - 1;
            uint64_t least = ~0ull;
            for (int c = 0; c < C; c++)
                least = min(least, sh.lists[c * a.n_top + part]);
            for (int i = tid; i < C * a.n_top; i += LGP_THREADS)
            {
                const uint64_t k = sh.lists[i];
                if (k && k >= least)
                    sh.cand[atomicAdd(&sh.count, 1)] = k;
            }
            __syncthreads();
            if (tid == 0 && (sh.count & 1))
                sh.cand[sh.count] = 0;
            __syncthreads();
            lgp_rank(sh, sh.count, a.n_top);
            __syncthreads();
        }
    }
    else
    {
        if (tid == 0)
        {
            sh.parts[0] = s;
            sh.counts[0] = sh.n_top;
        }
        __syncthreads();
    }
    if (warp < 2) // the row's state, and a lane for each alternative
    {
        LseState t = lane < C ? sh.parts[lane] : LseState{-INFINITY, 0.f, 0.f};
        int found = lane < C ? sh.counts[lane] : 0;
#pragma unroll
        for (int o = LGP_MAXC / 2; o > 0; o >>= 1)
        {
            t = lse_merge(t, LseState{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.z, o),
                                      __shfl_xor_sync(0xffffffffu, t.w, o)});
            found += __shfl_xor_sync(0xffffffffu, found, o);
        }
        // lanes 0..7 hold the join, which every lane takes from lane 0
        t.m = __shfl_sync(0xffffffffu, t.m, 0);
        t.z = __shfl_sync(0xffffffffu, t.z, 0);
        t.w = __shfl_sync(0xffffffffu, t.w, 0);
        found = __shfl_sync(0xffffffffu, found, 0);
        const bool bad = t.z != t.z || t.m == INFINITY;
        const float lz = bad ? NAN : log1pf(t.z);
        if (tid == 0 && a.logprob)
        {
            const float x = given;
            a.logprob[ri] = !has_given ? -INFINITY : bad ? NAN : x == -INFINITY ? -INFINITY : (x - t.m) - lz;
        }
        if (tid == 0 && a.entropy)
            a.entropy[ri] = bad ? NAN : lz + t.w / (1.f + t.z); // no id at all: 0
        if (tid < a.n_top)
        {
            const bool is = tid < found;
            const uint64_t key = is ? sh.top[tid] : 0;
            const float x = h2f(__ushort_as_half((unsigned short)unord16((uint32_t)(key >> 32))));
            a.top_ids[ri * a.n_top + tid] = is ? (int64_t)key_idx(key) : -1;
            a.top_logprobs[ri * a.n_top + tid] = !is ? -INFINITY : bad ? NAN : (x - t.m) - lz;
        }
    }
}

cudaError_t logprobs_launch(const LogprobArgs &a, int num_sms, cudaStream_t s)
{
    if (a.rows <= 0)
        return cudaSuccess;
    int C = LGP_MAXC;
    while (C > 1 && ((int64_t)a.rows * (C / 2) >= LGP_FILL * num_sms || a.vocab < C * LGP_PART))
        C /= 2;
    cudaLaunchConfig_t cfg = {};
    const int64_t z = ((int64_t)a.rows + 65534) / 65535; // a grid's y and z end at 65535
    cfg.gridDim = dim3((unsigned)C, (unsigned)((a.rows + z - 1) / z), (unsigned)z);
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

} // namespace ylm
