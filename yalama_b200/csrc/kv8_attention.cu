// Attention of the last t tokens over the 8-bit K/V cache (formats: kv8.cuh).
//
//   x_rj = q_r . (code_j * ks_j) / sqrt(128), -inf for hidden j
//   o_r  = sum_j softmax(x_r)_j * code_j * vs_j,  0 where every slot is hidden
//   acc[head][j] += sum of softmax(x_r)_j over the rows r of the KV head
// Row r = i * G + h of a KV head is query head h of its group, token i; token i
// sees slots [0, n - t + i]. Scores are kept in base 2 (x * log2 e).
#include "kv8.cuh"
#include <algorithm>

namespace ylm {

constexpr int KVA_THREADS = 128;
constexpr int KVA_ACC_TILE = 256; // slots per CTA of the accumulation

struct Kv8Plan
{
    int G, rows;     // query heads per KV head, rows per KV head of a pass (G * tokens)
    int splits, len; // splits of the slots and slots per split (a multiple of 64)
    size_t part_off, ml_off, score_off, bytes;
};

// Tokens of one pass. The accumulated weight keeps a pass's scores in the
// workspace ([rows][n] FP32 per KV head), so a pass takes at most 128 rows;
// without it 4096, which bounds the workspace and the grid.
static int pass_tokens(int G, int t, bool acc) { return std::min(t, std::max(1, (acc ? 128 : 4096) / G)); }

static Kv8Plan kv8_plan(int hkv, int hq, int t, int n, bool acc, int num_sms)
{
    Kv8Plan p;
    p.G = hq / hkv;
    p.rows = p.G * t;
    const int64_t groups = (int64_t)hkv * p.rows;
    const int want = (int)std::max<int64_t>(1, (num_sms * 8 + groups - 1) / groups);
    p.len = std::max(64, ((n + want - 1) / want + 63) / 64 * 64);
    p.splits = (n + p.len - 1) / p.len;
    // room for the most splits that any length up to n takes, so that a
    // workspace for n serves every smaller length
    const size_t heads_rows = (size_t)hkv * p.rows, most = heads_rows * std::min(want, (n + 63) / 64);
    p.part_off = 0;
    p.ml_off = p.part_off + most * YLM_HEAD_DIM * sizeof(float);
    p.score_off = p.ml_off + (most * 2 * sizeof(float) + 255) / 256 * 256;
    p.bytes = p.score_off + (acc ? heads_rows * n * sizeof(float) : 0);
    return p;
}

size_t kv8_attn_workspace(int hkv, int hq, int t, int n, bool acc, int num_sms)
{
    // passes see at most n slots; a pass over fewer slots never needs more
    if (t <= 0)
        return 0;
    size_t most = 0;
    const int per = pass_tokens(hq / hkv, t, acc);
    for (int i0 = 0; i0 < t; i0 += per)
        most = std::max(most, kv8_plan(hkv, hq, std::min(per, t - i0), n - t + std::min(t, i0 + per), acc, num_sms).bytes);
    return most;
}

struct Kv8Pass
{
    Kv8AttnArgs a;
    Kv8Plan p;
    float *part, *ml, *scores;
};

// One warp per slot in turn, lane l holding dimensions [4l, 4l + 4).
template <int FMT> __global__ void __launch_bounds__(KVA_THREADS) kv8_attn_kernel(Kv8Pass w)
{
    __shared__ float om[KVA_THREADS / 32][YLM_HEAD_DIM], mm[KVA_THREADS / 32], lm[KVA_THREADS / 32];
    const Kv8AttnArgs &a = w.a;
    const int G = w.p.G, sp = blockIdx.x, r = blockIdx.y, g = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int token = r / G, h = r % G;
    const int see = a.n - a.t + token + 1;
    const int j1 = min(see, (sp + 1) * w.p.len);
    const int nb = (a.c.cap + a.c.block - 1) / a.c.block;
    const float *ks = a.c.k_scale + (size_t)g * nb, *vs = a.c.v_scale + (size_t)g * nb;
    const __half *q = a.q + token * a.q_stride + (size_t)(g * G + h) * YLM_HEAD_DIM + lane * 4;
    float qf[4];
    for (int i = 0; i < 4; i++)
        qf[i] = h2f(q[i]);
    float M = -INFINITY, L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    float *score = w.scores + ((size_t)g * w.p.rows + r) * a.n;
    for (int j = sp * w.p.len + warp; j < min(a.n, (sp + 1) * w.p.len); j += KVA_THREADS / 32)
    {
        float x = -INFINITY;
        const bool hidden = j >= j1 || (a.mask && (a.mask[j >> 5] >> (j & 31) & 1u));
        const size_t at = ((size_t)g * a.c.cap + j) * YLM_HEAD_DIM + lane * 4;
        if (!hidden)
        {
            const uint32_t kc = *reinterpret_cast<const uint32_t *>(a.c.k + at);
            const uint32_t d0 = kv8_decode2<FMT>(kc), d1 = kv8_decode2<FMT>(kc >> 16);
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&d0));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&d1));
            x = warp_sum(qf[0] * f0.x + qf[1] * f0.y + qf[2] * f1.x + qf[3] * f1.y) * ks[j / a.c.block] *
                (float)(1.4426950408889634 / 11.313708498984760);
        }
        if (w.a.acc && lane == 0)
            score[j] = x;
        if (x == -INFINITY)
            continue;
        const float Mn = fmaxf(M, x), f = exp2f(M - Mn), p = exp2f(x - Mn);
        const uint32_t vc = *reinterpret_cast<const uint32_t *>(a.c.v + at);
        const uint32_t d0 = kv8_decode2<FMT>(vc), d1 = kv8_decode2<FMT>(vc >> 16);
        const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&d0));
        const float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&d1));
        const float pv = p * vs[j / a.c.block];
        M = Mn;
        L = L * f + p;
        o[0] = o[0] * f + pv * f0.x;
        o[1] = o[1] * f + pv * f0.y;
        o[2] = o[2] * f + pv * f1.x;
        o[3] = o[3] * f + pv * f1.y;
    }
    for (int i = 0; i < 4; i++)
        om[warp][lane * 4 + i] = o[i];
    if (lane == 0)
    {
        mm[warp] = M;
        lm[warp] = L;
    }
    __syncthreads();
    M = mm[0];
    for (int i = 1; i < KVA_THREADS / 32; i++)
        M = fmaxf(M, mm[i]);
    L = 0.f;
    float O = 0.f;
    for (int i = 0; i < KVA_THREADS / 32; i++)
    {
        const float f = mm[i] == -INFINITY ? 0.f : exp2f(mm[i] - M);
        L += lm[i] * f;
        O += om[i][tid] * f;
    }
    const size_t row = ((size_t)g * w.p.rows + r) * w.p.splits + sp;
    w.part[row * YLM_HEAD_DIM + tid] = O;
    if (tid == 0)
    {
        w.ml[2 * row] = M;
        w.ml[2 * row + 1] = L;
    }
}

// M and 1 / L of one row over its splits (0 and 0 where every slot is hidden)
__device__ __forceinline__ float2 kv8_row_state(const float *ml, int splits)
{
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < splits; s++)
        M = fmaxf(M, ml[2 * s]);
    if (M == -INFINITY)
        return make_float2(0.f, 0.f);
    for (int s = 0; s < splits; s++)
        L += ml[2 * s + 1] * exp2f(ml[2 * s] - M);
    return make_float2(M, 1.f / L);
}

// Joins the splits: CTAs [0, hkv * rows) write one output row each, the others
// add the weights of KVA_ACC_TILE slots of one KV head to acc.
__global__ void __launch_bounds__(KVA_THREADS) kv8_join_kernel(Kv8Pass w)
{
    const Kv8AttnArgs &a = w.a;
    const int G = w.p.G, R = w.p.rows, S = w.p.splits, tid = threadIdx.x;
    const int rows = a.c.hkv * R;
    int b = blockIdx.x;
    if (b < rows)
    {
        const int g = b / R, r = b % R;
        const float *ml = w.ml + (size_t)b * S * 2;
        const float2 st = kv8_row_state(ml, S);
        float O = 0.f;
        for (int s = 0; s < S; s++)
            if (ml[2 * s] != -INFINITY)
                O += w.part[((size_t)b * S + s) * YLM_HEAD_DIM + tid] * exp2f(ml[2 * s] - st.x);
        a.out[(r / G) * a.out_stride + (size_t)(g * G + r % G) * YLM_HEAD_DIM + tid] = f2h(O * st.y);
        return;
    }
    __shared__ float2 state[128];
    b -= rows;
    const int tiles = (a.n + KVA_ACC_TILE - 1) / KVA_ACC_TILE;
    const int g = b / tiles, j0 = b % tiles * KVA_ACC_TILE;
    if (tid < R)
        state[tid] = kv8_row_state(w.ml + ((size_t)g * R + tid) * S * 2, S);
    __syncthreads();
    for (int j = j0 + tid; j < min(a.n, j0 + KVA_ACC_TILE); j += KVA_THREADS)
    {
        float sum = 0.f;
        for (int r = 0; r < R; r++)
            sum += exp2f(w.scores[((size_t)g * R + r) * a.n + j] - state[r].x) * state[r].y;
        a.acc[(size_t)g * a.c.cap + j] += sum;
    }
}

cudaError_t kv8_attn_launch(const Kv8AttnArgs &args, void *ws, int num_sms, cudaStream_t s)
{
    const int G = args.hq / args.c.hkv, per = pass_tokens(G, args.t, args.acc != nullptr);
    for (int i0 = 0; i0 < args.t; i0 += per)
    {
        Kv8Pass w;
        w.a = args;
        w.a.t = std::min(per, args.t - i0);
        w.a.n = args.n - args.t + i0 + w.a.t;
        w.a.q = args.q + i0 * args.q_stride;
        w.a.out = args.out + i0 * args.out_stride;
        w.p = kv8_plan(args.c.hkv, args.hq, w.a.t, w.a.n, args.acc != nullptr, num_sms);
        w.part = reinterpret_cast<float *>(static_cast<char *>(ws) + w.p.part_off);
        w.ml = reinterpret_cast<float *>(static_cast<char *>(ws) + w.p.ml_off);
        w.scores = reinterpret_cast<float *>(static_cast<char *>(ws) + w.p.score_off);
        const dim3 grid((unsigned)w.p.splits, (unsigned)w.p.rows, (unsigned)args.c.hkv);
        if (args.c.format == KV8_E4M3)
            kv8_attn_kernel<KV8_E4M3><<<grid, KVA_THREADS, 0, s>>>(w);
        else
            kv8_attn_kernel<KV8_INT8><<<grid, KVA_THREADS, 0, s>>>(w);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess)
            return e;
        const int tiles = args.acc ? (w.a.n + KVA_ACC_TILE - 1) / KVA_ACC_TILE : 0;
        kv8_join_kernel<<<(unsigned)(args.c.hkv * (w.p.rows + tiles)), KVA_THREADS, 0, s>>>(w);
        e = cudaGetLastError();
        if (e != cudaSuccess)
            return e;
    }
    return cudaSuccess;
}

cudaError_t kv8_prepare() { return cudaSuccess; }

} // namespace ylm
