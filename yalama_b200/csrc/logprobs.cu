// Log probabilities of rows of FP16 logits: of one given id per row, the
// row's entropy, and its most likely ids.
//   m = max x, z = sum over the others of e^(x - m), ln Z = m + ln(1 + z)
//   logprob = (x_id - m) - log1p(z)
//   entropy = log1p(z) + sum e^(x - m) (m - x) / (1 + z)
// The maximum's own term is left out of z, so a nearly certain row keeps its
// small log probabilities (log1p(z) where 1 + z would round to 1), and the
// entropy is a sum of terms of one sign.
#include "ylm_common.cuh"

namespace ylm {

constexpr int LGP_THREADS = 512;

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
        return a;
    // b's terms relative to a.m: e^(x - a.m) = e^(x - b.m) f, a.m - x = (b.m - x) + d
    const float d = a.m - b.m, f = expf(-d), zb = 1.f + b.z;
    a.z += zb * f;
    a.w += (b.w + zb * d) * f;
    return a;
}

__device__ __forceinline__ void lse_add(LseState &s, float x)
{
    if (x == -INFINITY)
        return;
    s = lse_merge(s, LseState{x, 0.f, 0.f});
}

__device__ __forceinline__ bool lgp_masked(const uint32_t *bits, int64_t i)
{
    return bits && (bits[i >> 5] >> (i & 31) & 1u);
}

// Key of an alternative: NaN above everything, then the value (-0 as +0), then the lower id.
__device__ __forceinline__ uint64_t lgp_key(__half x, int64_t i)
{
    uint32_t u = __half_as_ushort(x);
    if ((u & 0x7FFFu) > 0x7C00u)
        u = 0x7FFFu;
    if (u == 0x8000u)
        u = 0u;
    return make_key(ord16(u), (uint32_t)i);
}

// One CTA per row: the row's state in one pass, then one pass per alternative
// (the largest key below the last one).
__global__ void __launch_bounds__(LGP_THREADS) logprobs_kernel(LogprobArgs a)
{
    __shared__ LseState st[LGP_THREADS / 32];
    __shared__ uint64_t best[LGP_THREADS / 32];
    const int64_t row = blockIdx.x;
    const __half *x = a.logits + row * a.ld;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    LseState s = {-INFINITY, 0.f, 0.f};
    bool nan = false;
    for (int64_t i = tid; i < a.vocab; i += LGP_THREADS)
    {
        if (lgp_masked(a.mask_bits, i))
            continue;
        const float v = h2f(x[i]);
        nan |= v != v || v == INFINITY;
        if (v == v && v != INFINITY)
            lse_add(s, v);
    }
    for (int o = 16; o > 0; o >>= 1)
    {
        const LseState t = {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.z, o),
                            __shfl_xor_sync(0xffffffffu, s.w, o)};
        s = lse_merge(s, t);
    }
    if (lane == 0)
        st[warp] = s;
    nan = __syncthreads_or(nan);
    s = st[0];
    for (int w = 1; w < LGP_THREADS / 32; w++)
        s = lse_merge(s, st[w]);
    const float lz = nan ? NAN : log1pf(s.z);
    if (tid == 0)
    {
        if (a.logprob)
        {
            const int64_t id = a.ids[row];
            float lp = -INFINITY;
            if (id >= 0 && id < a.vocab && !lgp_masked(a.mask_bits, id) && (nan || h2f(x[id]) > -INFINITY))
                lp = nan ? NAN : (h2f(x[id]) - s.m) - lz;
            a.logprob[row] = lp;
        }
        if (a.entropy)
            a.entropy[row] = nan ? NAN : lz + s.w / (1.f + s.z);
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.n_top; k++)
    {
        uint64_t mine = 0;
        for (int64_t i = tid; i < a.vocab; i += LGP_THREADS)
        {
            const __half h = x[i];
            if (lgp_masked(a.mask_bits, i) || __half_as_ushort(h) == 0xFC00u)
                continue;
            const uint64_t key = lgp_key(h, i);
            if (key < last && key > mine)
                mine = key;
        }
        mine = warp_max_u64(mine);
        __syncthreads();
        if (lane == 0)
            best[warp] = mine;
        __syncthreads();
        for (int w = 0; w < LGP_THREADS / 32; w++)
            mine = best[w] > mine ? best[w] : mine;
        last = mine;
        if (tid == 0)
        {
            const int64_t id = mine ? (int64_t)key_idx(mine) : -1;
            a.top_ids[row * a.n_top + k] = id;
            a.top_logprobs[row * a.n_top + k] = id < 0 ? -INFINITY : nan ? NAN : (h2f(x[id]) - s.m) - lz;
        }
        if (!mine)
            last = 0; // no more: the rest of the list stays empty
    }
}

cudaError_t logprobs_launch(const LogprobArgs &a, int num_sms, cudaStream_t s)
{
    (void)num_sms;
    if (a.rows <= 0)
        return cudaSuccess;
    logprobs_kernel<<<(unsigned)a.rows, LGP_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t logprobs_prepare() { return cudaSuccess; }

} // namespace ylm
