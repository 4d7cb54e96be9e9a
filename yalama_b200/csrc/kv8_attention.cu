// Attention of the last t tokens over the 8-bit K/V cache (formats: kv8.cuh).
//
//   x_rj = q_r . (code_j * ks_j) / sqrt(128), -inf for hidden j
//   o_r  = sum_j softmax(x_r)_j * code_j * vs_j,  0 where every slot is hidden
//   acc[head][j] += sum of softmax(x_r)_j over the rows r of the KV head
// Row r = i * G + h of a KV head is query head h of its group, token i; token i
// sees slots [0, n - t + i]. Scores are kept in base 2 (x * log2 e).
//
// kv8_attn_kernel splits the slots over CTAs (a decode step has too few rows to
// fill the GPU otherwise), which leaves sums (M, l, O) per split and row. Up to
// KVA_ALONE slots the splits of a KV head are one cluster, which joins them through
// distributed shared memory and adds the weights from scores kept there: one launch, no
// workspace. Beyond (and where weights are kept of more than 16 rows a KV head), sums and
// scores go through the workspace, and kv8_join_kernel joins the splits and turns the
// scores into weights.
#include "kv8.cuh"
#include <algorithm>
#include <cooperative_groups.h>
#include <type_traits>

namespace ylm {

constexpr int KVA_THREADS = 128;
constexpr int KVA_WARPS = KVA_THREADS / 32;
constexpr int KVA_CHUNK = 32;     // slots a warp takes at a time
constexpr int KVA_BUF = KVA_CHUNK * YLM_HEAD_DIM; // bytes of a chunk's K or V
constexpr int KVA_RING = 4 * KVA_BUF;             // a warp's two K and two V chunks
constexpr int KVA_SMEM = KVA_WARPS * KVA_RING;
constexpr int KVA_JOIN = 256;     // threads of the joining CTAs
// FP16 weights: the largest score seen weighs 2^KVA_LEAD when the reference is set, and the reference moves when one
// passes 2^KVA_MOST (FP16 ends at 2^16). A higher lead keeps more of the small weights, and moves the reference more
// often: 8 x 4099 (64 / 8 heads) 1 % longer at a lead of 11 than at 9, 3 % at 12; one row the same at all.
constexpr float KVA_LEAD = 11.f, KVA_MOST = 15.9f;
// Octaves below the largest value scale from which weights are lifted: above it, slots of equal softmax weight stay 15
// octaves clear of FP16's smallest normal number.
constexpr float KVA_LIFT = 10.f;
constexpr int KVA_CLUSTER = 8;    // most splits of a cluster (the portable size)
// Slots up to which the splits of a KV head are one cluster. One launch against two, us of device time (8 heads of
// 4 query heads; with kept weights): 100 slots 4.3 / 5.2 (5.5 / 6.2), 611 slots 5.0 / 5.3 (6.2 / 7.0), 1000 slots
// 5.7 / 5.5 (6.9 / 7.4), 2000 slots 6.5 / 5.5 (8.2 / 7.7). Without weights two launches are the faster already at 1000
// slots, by 0.2 us in a captured graph; a caller that launches each step saves more than that with the second launch.
constexpr int KVA_ALONE = 1024;
constexpr int KVA_ALONE_LEN = KVA_ALONE / KVA_CLUSTER;
static_assert(KVA_ALONE_LEN % (KVA_CHUNK * KVA_WARPS) == 0, "a split is whole rounds of its warps");

struct Kv8Plan
{
    int G, rows;      // query heads per KV head, rows per KV head of a pass (G * tokens)
    int nt;           // 8-row tiles per CTA, 1 or 2
    int zblocks;      // CTAs over the rows of a KV head
    int cluster;      // 1: the splits are one cluster
    int splits, len;  // splits of the slots and slots per split
    int pad;          // rows, rounded up to a multiple of 4: stride of the kept scores and of (M, l)
    int lps;          // lanes that share a slot's rows in the accumulation, four rows a load
    int tile;         // slots per CTA of the accumulation
    size_t ml_off, score_off, bytes;
};

// Tokens of one pass. The accumulated weight keeps a pass's scores in the
// workspace ([n][rows] FP32 per KV head), so a pass takes at most 128 rows;
// without it 4096, which bounds the workspace and the grid.
static int pass_tokens(int G, int t, bool acc) { return std::min(t, std::max(1, (acc ? 128 : 4096) / G)); }

static Kv8Plan kv8_plan(int hkv, int hq, int t, int n, bool acc, int num_sms)
{
    Kv8Plan p;
    p.G = hq / hkv;
    p.rows = p.G * t;
    p.nt = p.rows <= 8 ? 1 : 2;
    p.zblocks = (p.rows + 8 * p.nt - 1) / (8 * p.nt);
    const int unit = KVA_CHUNK * KVA_WARPS; // slots of one round of a CTA's warps
    // one wave of CTAs: as many as the SMs hold
    const int64_t groups = (int64_t)hkv * p.zblocks;
    // (rows of several CTAs would meet in acc: they go the other way)
    p.cluster = n <= KVA_ALONE && (!acc || p.zblocks == 1);
    const int want = p.cluster ? KVA_CLUSTER
                               : (int)std::max<int64_t>(1, (int64_t)num_sms * (p.nt == 1 ? 3 : 2) / groups);
    p.len = std::max(1, ((n + want - 1) / want + unit - 1) / unit) * unit;
    p.splits = (n + p.len - 1) / p.len;
    // room for the most splits that any length up to n takes, so that a
    // workspace for n serves every smaller length
    const size_t most = (size_t)hkv * std::min(want, (n + unit - 1) / unit);
    p.pad = (p.rows + 3) / 4 * 4;
    p.ml_off = most * p.rows * YLM_HEAD_DIM * sizeof(float);
    p.score_off = p.ml_off + (most * p.pad * 2 * sizeof(float) + 255) / 256 * 256;
    // slots per accumulating CTA: about four CTAs per SM, each of which finds every row's state first
    p.lps = !acc || p.pad < 8 ? 1 : p.pad < 32 ? 2 : p.pad < 64 ? 8 : 16; // at most pad / 4
    const int round = 4 * KVA_JOIN / p.lps;
    p.tile = std::max(1, (int)(((int64_t)hkv * n / (num_sms * 4) + round - 1) / round)) * round;
    p.bytes = p.cluster ? 0 : p.score_off + (acc ? (size_t)hkv * n * p.pad * sizeof(float) : 0);
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
    float *part, *ml, *scores; // [hkv][rows][split][128], [hkv][split][pad][2], [hkv][n][pad]
};

__device__ __forceinline__ float kva_ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// D += A B, m16n8k16, FP16 operands, FP32 accumulation
__device__ __forceinline__ void kva_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the 8 x 8 matrix of 16-bit values held two to a lane, transposed
__device__ __forceinline__ uint32_t kva_transpose(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t kva_word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// 2^lv is a value block's scale (a block of zeros: the clamp's 2^-64 does as well)
__device__ __forceinline__ float kva_log_scale(float s)
{
    return (float)max(-64, min(64, (int)(__float_as_uint(s) >> 23 & 255u) - 127));
}

// 2^e, exactly, for a whole e of at most 126 either way
__device__ __forceinline__ float kva_pow2(float e) { return __uint_as_float((uint32_t)(127 + (int)e) << 23); }

// Both products run on the tensor cores with the slots as rows of the A operand,
// so that 8 query rows fill the N dimension: S^T = K Q^T and O^T = V^T P^T
// (m16n8k16; NT tiles of 8 query rows share each decoded fragment; more rows
// than 16 go to CTAs of their own, which read the codes from L2 again). Lane
// (g, c) = (lane / 4, lane % 4).
//  S^T: the head dimension is summed in a permuted order in which every A
//    fragment comes from 16-byte reads of code rows: lane (g, c) reads
//    dimensions [16c, 16c + 16) and 64 + [16c, 16c + 16) of slots g and g + 8, and k-step
//    j takes word j % 4 of piece j / 4; Q's fragments are in the same order.
//  O^T: lane (g, c) reads dimensions [16g, 16g + 16) of slots 2c, 2c + 1, 2c + 8
//    and 2c + 9; one byte permute pairs the codes of two slots of a dimension into a
//    fragment's halves, and M-tile i holds dimension 16g + 2i in row g, 16g + 2i + 1 in row
//    g + 8. P^T is S^T's accumulator packed to FP16 and transposed 8 x 8 at a time.
// Each warp streams its own chunks of 32 slots through a ring of two K and two V
// buffers (cp.async, no barrier between warps): while it works on one chunk the next
// one's K and V are in flight.
//
// Scales: ks multiplies the scores. vs enters the exponent: the PV weight of score x is
// w = 2^((x - mx) + (log2 vs + cx)) and the softmax sum takes w / vs (exact: vs is a power of two). The
// reference is the score mx of a slot that had the largest vs 2^x, with cx = KVA_LEAD less its own log2 vs,
// and moves only when some w would pass 2^KVA_MOST. It is kept as a score and a small whole number
// because x - mx is exact where it matters: scores of 2^24 and beyond step by octaves, and mx less the lead in one
// number was off by as many. w enters P V
// rounded to FP16, the matrix unit's operand: off by 2^-11 of itself at most down to 2^-25 of the
// largest (2^-14, FP16's smallest normal number), and by 2^-36 of the largest below (2^-25, half its
// smallest step). That is the size of the result's own rounding to FP16; what a second product with the
// weights' next 11 bits would add took 2 to 9 % longer at one row and 13 to 26 % with more. The
// reference, l, the scores and both accumulators are FP32; a split's (M, l, O) leave in units of 2^(x - mx), M = mx.
// Slots whose values have a scale far below the largest have small w however large their softmax weight, and may
// alone reach a dimension: their weights are lifted for the product (KVA_LIFT).
//
// Measured (B200, E4M3, 8 KV heads of 4 query heads, decode step without kept weights): 131071 slots 48.8 us =
// 5.50 TB/s in both launches (INT8 49.7 us), and 6.4 TB/s for each slot more: bound by HBM behind about 7 us of
// start, tail and join; 8200 slots 8.3 us, bound by the two launches' latency; 611 slots 5.2 us in one launch, bound by
// the latency of one chunk a warp and of the cluster's join. Eight tokens of 64 / 8 heads over 4099 slots 13.4 us:
// bound by the instructions that decode every code once per 16 rows.
// Registers as the buffers instead of the ring: 131071 slots 52 us, 611 slots 7.2 us (with the join of that
// time); three CTAs an SM (NT = 1) at 168 registers; without the decode (wrong values) 131071 slots take 1 us less.
template <int FMT, int NT, bool CLUSTER>
__global__ void __launch_bounds__(KVA_THREADS, NT == 1 ? 3 : 2) kv8_attn_kernel(const Kv8Pass w)
{
    extern __shared__ __align__(128) uint8_t ring[]; // a warp's two K and two V chunks; at the end the sums O
    float(*om)[8 * NT][YLM_HEAD_DIM + 8] = reinterpret_cast<float(*)[8 * NT][YLM_HEAD_DIM + 8]>(ring);
    static_assert(sizeof(float) * 8 * NT * (YLM_HEAD_DIM + 8) <= KVA_RING, "a warp's O fits its ring");
    __shared__ float mm[KVA_WARPS][8 * NT], lm[KVA_WARPS][8 * NT];
    float *kept = reinterpret_cast<float *>(ring + KVA_SMEM); // CLUSTER: scores [slot of the split][8 * NT]
    if (!CLUSTER)
        pdl_launch_dependents(); // the joining CTAs may start; they wait for this grid's end
    const Kv8AttnArgs &a = w.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int sp = blockIdx.x, kvh = blockIdx.y;
    const int R = w.p.rows, G = w.p.G;
    const int row0 = (int)blockIdx.z * 8 * NT; // first of this CTA's rows
    const int n = a.n, first = n - a.t;                           // slots >= first are hidden from some row
    const int j_end = min(n, (sp + 1) * w.p.len);
    const int nb = (a.c.cap + a.c.block - 1) / a.c.block, bshift = 31 - __clz(a.c.block);
    const uint8_t *kc = a.c.k + (size_t)kvh * a.c.cap * YLM_HEAD_DIM;
    const uint8_t *vc = a.c.v + (size_t)kvh * a.c.cap * YLM_HEAD_DIM;
    const float *ksp = a.c.k_scale + (size_t)kvh * nb, *vsp = a.c.v_scale + (size_t)kvh * nb;

    // Q fragments and, for the accumulator's columns 2c and 2c + 1 of each tile, the last slot their token sees
    uint32_t q[NT][8][2];
    int see[NT][2];
#pragma unroll
    for (int t = 0; t < NT; t++)
    {
        const int r = row0 + 8 * t + g;
        const bool is = r < R;
        const __half *src = a.q + (is ? r / G : 0) * a.q_stride + (size_t)(kvh * G + (is ? r % G : 0)) * YLM_HEAD_DIM + c * 16;
#pragma unroll
        for (int p = 0; p < 2; p++)
        {
            uint4 x = make_uint4(0, 0, 0, 0), y = x;
            if (is)
            {
                x = *reinterpret_cast<const uint4 *>(src + p * 64);
                y = *reinterpret_cast<const uint4 *>(src + p * 64 + 8);
            }
            q[t][4 * p][0] = x.x, q[t][4 * p][1] = x.y, q[t][4 * p + 1][0] = x.z, q[t][4 * p + 1][1] = x.w;
            q[t][4 * p + 2][0] = y.x, q[t][4 * p + 2][1] = y.y, q[t][4 * p + 3][0] = y.z, q[t][4 * p + 3][1] = y.w;
        }
        for (int i = 0; i < 2; i++)
            see[t][i] = first + (row0 + 8 * t + 2 * c + i) / G;
    }

    // ---- the warp's ring: chunk (row r, 16-byte piece q) at r * 128 + (q ^ f(r)) * 16 with
    // f(r) = 2 ((r / 2) % 4) ^ 4 (r % 2), which spreads the pieces that eight lanes read
    // together (K: four pieces of two rows; V: two pieces of four even or four odd rows) over all banks
    uint8_t *mine = ring + warp * KVA_RING;
    const uint32_t ring_at = smem_u32(mine);
    // this lane copies piece lane % 8 of rows 4 i + lane / 8: f there for even i, and for odd i
    const uint32_t dst_even = (lane >> 3) * 128 + (((lane & 7) ^ (((lane >> 4) & 1) << 1) ^ ((lane >> 3 & 1) << 2)) << 4);
    const uint32_t dst_odd = (lane >> 3) * 128 + (((lane & 7) ^ ((2 + ((lane >> 4) & 1)) << 1) ^ ((lane >> 3 & 1) << 2)) << 4);
    // A decode step reads the codes once, and what it writes for the join should stay in L2: 131071 slots with kept
    // weights 61.1 us against 62.4 with the normal policy, 32000 slots 17.6 against 18.2. The CTAs of more than 16 rows
    // read the same codes at about the same time and find them in L2 under either policy: 8 tokens of 64 / 8 heads
    // over 60000 and 131071 slots, 64 tokens over 30000, and several passes over 60000 differ by 0.5 % at most.
    const uint64_t policy = l2_policy_evict_first();
    auto copy = [&](const uint8_t *src, int j0, uint32_t at) {
        const int r0 = j0 + (lane >> 3);
        const uint8_t *p = src + (size_t)r0 * YLM_HEAD_DIM + (lane & 7) * 16;
        if (j0 + KVA_CHUNK <= n)
        {
#pragma unroll
            for (int i = 0; i < 8; i++)
                asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(
                                 at + i * 512 + (i & 1 ? dst_odd : dst_even)),
                             "l"(p + i * 512), "l"(policy)
                             : "memory");
        }
        else
        {
            // rows behind the last slot are not read and arrive as zeros
#pragma unroll
            for (int i = 0; i < 8; i++)
            {
                const bool in = r0 + 4 * i < n;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                 at + i * 512 + (i & 1 ? dst_odd : dst_even)),
                             "l"(in ? p + i * 512 : src), "r"(in ? 16 : 0)
                             : "memory");
            }
        }
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    // the lane's reads: K pieces c and 4 + c of row g (+ 8 k, same f), V piece g of rows 2c (+ 8) and 2c + 1 (+ 8)
    const uint32_t fg = ((g >> 1 & 3) << 1) ^ ((g & 1) << 2), fc = c << 1;
    const uint32_t k_lo = g * 128 + ((c ^ fg) << 4), k_hi = g * 128 + (((4 + c) ^ fg) << 4);
    const uint32_t v_even = c * 256 + ((g ^ fc) << 4), v_odd = c * 256 + 128 + ((g ^ fc ^ 4) << 4);
    float ks[2], vs[2], ks_next[2], vs_next[2];
    auto load_scales = [&](int j0) {
#pragma unroll
        for (int s = 0; s < 2; s++)
        {
            const int b = min(j0 + 16 * s, n - 1) >> bshift;
            ks_next[s] = ksp[b];
            vs_next[s] = vsp[b];
        }
    };

    float O[NT][8][4], l[NT][2];
    float mx[NT][2], cx[NT][2]; // the reference score (-inf: nothing seen), and the lead less its value scale
#pragma unroll
    for (int t = 0; t < NT; t++)
    {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                O[t][i][e] = 0.f;
        mx[t][0] = mx[t][1] = -INFINITY;
        cx[t][0] = cx[t][1] = l[t][0] = l[t][1] = 0.f;
    }
    float vs_top = -INFINITY; // largest value scale so far of a half with a slot that is not masked
    constexpr int step = KVA_CHUNK * KVA_WARPS;
    int j0 = sp * w.p.len + warp * KVA_CHUNK;
    int phase = 0; // the buffers of this round: 0 or 1
    if (j0 < j_end)
    {
        load_scales(j0);
#pragma unroll
        for (int i = 0; i < 2; i++)
        {
            if (j0 + i * step < j_end)
                copy(kc, j0 + i * step, ring_at + i * KVA_BUF);
            commit();
            if (j0 + i * step < j_end)
                copy(vc, j0 + i * step, ring_at + (2 + i) * KVA_BUF);
            commit();
        }
    }
    for (; j0 < j_end; j0 += step, phase ^= 1)
    {
        // in flight: this round's K and V, the next one's K and V
        asm volatile("cp.async.wait_group 3;" ::: "memory");
        __syncwarp();
        const uint8_t *kb = mine + phase * KVA_BUF, *vb = mine + (2 + phase) * KVA_BUF;
        // ---- S^T
        float S[2][NT][4];
#pragma unroll
        for (int s = 0; s < 2; s++)
        {
            ks[s] = ks_next[s];
            vs[s] = kva_log_scale(vs_next[s]);
            uint4 K[4];
            K[0] = *reinterpret_cast<const uint4 *>(kb + s * 2048 + k_lo);
            K[1] = *reinterpret_cast<const uint4 *>(kb + s * 2048 + k_hi);
            K[2] = *reinterpret_cast<const uint4 *>(kb + s * 2048 + 1024 + k_lo);
            K[3] = *reinterpret_cast<const uint4 *>(kb + s * 2048 + 1024 + k_hi);
#pragma unroll
            for (int t = 0; t < NT; t++)
                S[s][t][0] = S[s][t][1] = S[s][t][2] = S[s][t][3] = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++)
            {
                uint32_t a0, a1, a2, a3;
                kv8_decode4<FMT>(kva_word(K[j >> 2], j & 3), a0, a2);
                kv8_decode4<FMT>(kva_word(K[2 + (j >> 2)], j & 3), a1, a3);
#pragma unroll
                for (int t = 0; t < NT; t++)
                    kva_mma(S[s][t], a0, a1, a2, a3, q[t][j][0], q[t][j][1]);
            }
        }
        __syncwarp(); // every lane has read this K
        if (j0 + 2 * step < j_end)
            copy(kc, j0 + 2 * step, ring_at + phase * KVA_BUF);
        commit();
        if (j0 + step < j_end)
            load_scales(j0 + step);
        // ---- scores in base 2, hidden slots -inf
        bool edge[2]; // some row does not see some slot of the half
        uint32_t off[2];
        float grow = -INFINITY;
#pragma unroll
        for (int s = 0; s < 2; s++)
        {
            const int js = j0 + 16 * s;
            const float f = ks[s] * (float)(1.4426950408889634 / 11.313708498984760);
            off[s] = js + 16 <= n ? 0u : js >= n ? 0xFFFFu : 0xFFFFu << (n - js) & 0xFFFFu;
            if (a.mask && js < n)
                off[s] |= a.mask[js >> 5] >> (js & 16) & 0xFFFFu;
            edge[s] = js + 15 > first;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    S[s][t][e] *= f;
            if (off[s] || edge[s])
            {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                    {
                        const int k = g + 8 * (e >> 1);
                        if (off[s] >> k & 1u || js + k > see[t][e & 1])
                            S[s][t][e] = -INFINITY;
                    }
            }
            if (a.acc)
            {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        if (CLUSTER)
                            *reinterpret_cast<float2 *>(kept + (js - sp * w.p.len + g + 8 * i) * 8 * NT + 8 * t + 2 * c) =
                                make_float2(S[s][t][2 * i], S[s][t][2 * i + 1]);
                        else if (js + g + 8 * i < n && row0 + 8 * t + 2 * c < w.p.pad)
                            *reinterpret_cast<float2 *>(w.scores + ((size_t)kvh * n + js + g + 8 * i) * w.p.pad + row0 +
                                                        8 * t + 2 * c) = make_float2(S[s][t][2 * i], S[s][t][2 * i + 1]);
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    grow = fmaxf(grow, (S[s][t][e] - mx[t][e & 1]) + (vs[s] + cx[t][e & 1]));
        }
        // ---- the reference follows where a weight would pass 2^KVA_MOST. mx = -inf makes grow +inf, or NaN
        // (kept out by fmaxf) where the score is -inf, too
        if (__any_sync(0xffffffffu, grow > KVA_MOST))
        {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                {
                    float m[2];
#pragma unroll
                    for (int s = 0; s < 2; s++)
                    {
                        m[s] = fmaxf(S[s][t][i], S[s][t][i + 2]);
                        m[s] = fmaxf(m[s], __shfl_xor_sync(0xffffffffu, m[s], 4));
                        m[s] = fmaxf(m[s], __shfl_xor_sync(0xffffffffu, m[s], 8));
                        m[s] = fmaxf(m[s], __shfl_xor_sync(0xffffffffu, m[s], 16));
                    }
                    const bool second = (m[1] - m[0]) + (vs[1] - vs[0]) > 0.f;
                    const float top = second ? m[1] : m[0], v = second ? vs[1] : vs[0];
                    if ((top - mx[t][i]) + (v + cx[t][i]) > KVA_LEAD)
                    {
                        const float f = kva_ex2((mx[t][i] - top) + (KVA_LEAD - v - cx[t][i]));
                        mx[t][i] = top;
                        cx[t][i] = KVA_LEAD - v;
                        l[t][i] *= f;
#pragma unroll
                        for (int k = 0; k < 8; k++)
                        {
                            O[t][k][i] *= f;
                            O[t][k][i + 2] *= f;
                        }
                    }
                }
        }
        // ---- O^T
        asm volatile("cp.async.wait_group 3;" ::: "memory");
        __syncwarp();
        const auto weigh = [&](auto far_values) {
            constexpr bool FAR = decltype(far_values)::value;
#pragma unroll
            for (int s = 0; s < 2; s++)
            {
                uint4 V[4];
                V[0] = *reinterpret_cast<const uint4 *>(vb + s * 2048 + v_even);
                V[1] = *reinterpret_cast<const uint4 *>(vb + s * 2048 + v_odd);
                V[2] = *reinterpret_cast<const uint4 *>(vb + s * 2048 + 1024 + v_even);
                V[3] = *reinterpret_cast<const uint4 *>(vb + s * 2048 + 1024 + v_odd);
                float lift[NT][2];
                if (FAR)
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 2; i++)
                        {
                            float m = fmaxf(S[s][t][i], S[s][t][i + 2]);
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                            // -inf (or NaN) where the row sees none of these slots: no weight, any lift
                            lift[t][i] = fminf(fmaxf(floorf(KVA_LEAD - ((m - mx[t][i]) + (vs[s] + cx[t][i]))), 0.f), 64.f);
#pragma unroll
                            for (int k = 0; k < 8; k++)
                            {
                                O[t][k][i] *= kva_pow2(lift[t][i]);
                                O[t][k][i + 2] *= kva_pow2(lift[t][i]);
                            }
                        }
                uint32_t P[NT][2];
                const float unscale = kva_pow2(-vs[s]);
#pragma unroll
                for (int t = 0; t < NT; t++)
                {
                    // nothing seen so far: mx = -inf, and every weight 0
                    const float ref[2] = {mx[t][0] == -INFINITY ? 0.f : mx[t][0], mx[t][1] == -INFINITY ? 0.f : mx[t][1]};
                    const float shift[2] = {vs[s] + cx[t][0], vs[s] + cx[t][1]};
                    float e4[4];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                    {
                        e4[e] = kva_ex2((S[s][t][e] - ref[e & 1]) + shift[e & 1]);
                    }
                    l[t][0] += (e4[0] + e4[2]) * unscale;
                    l[t][1] += (e4[1] + e4[3]) * unscale;
                    if (FAR)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            e4[e] = kva_ex2((S[s][t][e] - ref[e & 1]) + (shift[e & 1] + lift[t][e & 1]));
                    const __half2 lo = __floats2half2_rn(e4[0], e4[1]), hi = __floats2half2_rn(e4[2], e4[3]);
                    P[t][0] = kva_transpose(*reinterpret_cast<const uint32_t *>(&lo));
                    P[t][1] = kva_transpose(*reinterpret_cast<const uint32_t *>(&hi));
                }
                // hidden slots may hold anything, NaN codes too: 0 x NaN must not arise
                if (off[s])
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (off[s] >> (2 * c + (i & 1) + 8 * (i >> 1)) & 1u)
                            V[i] = make_uint4(0, 0, 0, 0);
                if (FMT == KV8_E4M3 && edge[s] && a.t > 1)
                {
                    // a slot that some rows do not see: its NaN codes are taken out and put
                    // back as NaN into the rows that do see it
                    uint32_t nan = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            nan |= (kva_word(V[i], k) & 0x7F7F7F7Fu) + 0x01010101u;
                    if (__any_sync(0xffffffffu, nan & 0x80808080u))
                    {
                        uint32_t seen[NT][2];
#pragma unroll
                        for (int t = 0; t < NT; t++)
#pragma unroll
                            for (int i = 0; i < 2; i++)
                                seen[t][i] = kva_transpose((S[s][t][2 * i] == -INFINITY ? 0u : 0x3C00u) |
                                                           (S[s][t][2 * i + 1] == -INFINITY ? 0u : 0x3C000000u));
                        uint32_t *v = reinterpret_cast<uint32_t *>(&V[0]);
                        uint32_t flag[16]; // 1 (0x38 in E4M3) where a code is NaN
#pragma unroll
                        for (int k = 0; k < 16; k++)
                        {
                            const uint32_t hit = ((v[k] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                            flag[k] = (hit >> 7) * 0x38u;
                            v[k] &= ~((hit >> 7) * 0xFFu);
                        }
#pragma unroll
                        for (int i = 0; i < 8; i++)
                        {
                            const uint32_t sel = i & 1 ? 0x7362 : 0x5140;
                            const uint32_t x = __byte_perm(flag[i >> 1], flag[4 + (i >> 1)], sel);
                            const uint32_t y = __byte_perm(flag[8 + (i >> 1)], flag[12 + (i >> 1)], sel);
                            uint32_t a0, a1, a2, a3;
                            kv8_decode4<FMT>(x, a0, a1);
                            kv8_decode4<FMT>(y, a2, a3);
#pragma unroll
                            for (int t = 0; t < NT; t++)
                            {
                                float d[4] = {0.f, 0.f, 0.f, 0.f};
                                kva_mma(d, a0, a1, a2, a3, seen[t][0], seen[t][1]);
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    if (d[e] > 0.f)
                                        O[t][i][e] = NAN;
                            }
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; i++)
                {
                    const uint32_t sel = i & 1 ? 0x7362 : 0x5140;
                    const uint32_t x = __byte_perm(kva_word(V[0], i >> 1), kva_word(V[1], i >> 1), sel);
                    const uint32_t y = __byte_perm(kva_word(V[2], i >> 1), kva_word(V[3], i >> 1), sel);
                    uint32_t a0, a1, a2, a3;
                    kv8_decode4<FMT>(x, a0, a1);
                    kv8_decode4<FMT>(y, a2, a3);
#pragma unroll
                    for (int t = 0; t < NT; t++)
                    {
                        kva_mma(O[t][i], a0, a1, a2, a3, P[t][0], P[t][1]);
                    }
                }
                if (FAR)
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int k = 0; k < 8; k++)
                            {
                                O[t][k][i] *= kva_pow2(-lift[t][i]);
                                O[t][k][i + 2] *= kva_pow2(-lift[t][i]);
                            }
            }
        };
        // Values of a scale far below the largest so far: their weights would lose digits to FP16's range, although
        // nothing else may reach their dimensions. Each row's are lifted by a power of two of its own while they
        // are added, and the row's sums with them.
#pragma unroll
        for (int s = 0; s < 2; s++)
            if (off[s] != 0xFFFFu)
                vs_top = fmaxf(vs_top, vs[s]);
        if (fminf(vs[0], vs[1]) < vs_top - KVA_LIFT) // uniform over the warp
            weigh(std::true_type{});
        else
            weigh(std::false_type{});
        __syncwarp(); // every lane has read this V
        if (j0 + 2 * step < j_end)
            copy(vc, j0 + 2 * step, ring_at + (2 + phase) * KVA_BUF);
        commit();
    }
    __syncthreads(); // the rings become the warps' sums

    // ---- join the warps that share rows, and leave the split's sums
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 2; i++)
        {
            float s = l[t][i];
            s += __shfl_xor_sync(0xffffffffu, s, 4);
            s += __shfl_xor_sync(0xffffffffu, s, 8);
            s += __shfl_xor_sync(0xffffffffu, s, 16);
            // to 2^(score - mx), without the lead and the reference's value scale
            const float own = kva_pow2(-cx[t][i]);
            if (g == 0)
            {
                mm[warp][8 * t + 2 * c + i] = mx[t][i];
                lm[warp][8 * t + 2 * c + i] = s * own;
            }
#pragma unroll
            for (int k = 0; k < 8; k++)
                *reinterpret_cast<float2 *>(&om[warp][8 * t + 2 * c + i][16 * g + 2 * k]) =
                    make_float2(O[t][k][i] * own, O[t][k][i + 2] * own);
        }
    __syncthreads();
    // the warps' sums, joined: a warp per row in turn, lane = 4 dimensions
    for (int r = warp; r < 8 * NT && row0 + r < R; r += KVA_WARPS)
    {
        float m = mm[0][r], L = 0.f;
#pragma unroll
        for (int s = 1; s < KVA_WARPS; s++)
            m = fmaxf(m, mm[s][r]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int s = 0; s < KVA_WARPS; s++)
        {
            const float ms = mm[s][r], f = ms == -INFINITY ? 0.f : kva_ex2(ms - m);
            const float4 x = *reinterpret_cast<const float4 *>(&om[s][r][lane * 4]);
            L += lm[s][r] * f;
            o.x += x.x * f;
            o.y += x.y * f;
            o.z += x.z * f;
            o.w += x.w * f;
        }
        if (CLUSTER)
        {
            // in place: a lane's own four dimensions, and the row's M and l by the lane that read them last
            *reinterpret_cast<float4 *>(&om[0][r][lane * 4]) = o;
            __syncwarp();
            if (lane == 0)
            {
                mm[0][r] = m;
                lm[0][r] = L;
            }
            continue;
        }
        *reinterpret_cast<float4 *>(w.part + (((size_t)kvh * R + row0 + r) * w.p.splits + sp) * YLM_HEAD_DIM + lane * 4) = o;
        if (lane == 0)
            *reinterpret_cast<float2 *>(w.ml + 2 * (((size_t)kvh * w.p.splits + sp) * w.p.pad + row0 + r)) = make_float2(m, L);
    }
    if constexpr (CLUSTER)
    {
        // ---- the splits, joined: row r by warp r % 4 of rank r / 4 % C
        namespace cg = cooperative_groups;
        cg::cluster_group cl = cg::this_cluster();
        __shared__ float2 state[8 * NT];
        const int C = (int)gridDim.x;
        cl.sync();
        for (int r = sp * KVA_WARPS + warp; r < 8 * NT && row0 + r < R; r += C * KVA_WARPS)
        {
            float m[KVA_CLUSTER], M = -INFINITY, L = 0.f;
#pragma unroll
            for (int s = 0; s < KVA_CLUSTER; s++)
            {
                m[s] = s < C ? *cl.map_shared_rank(&mm[0][r], s) : -INFINITY;
                M = fmaxf(M, m[s]);
            }
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int s = 0; s < KVA_CLUSTER; s++)
            {
                if (s >= C)
                    break;
                const float f = m[s] == -INFINITY ? 0.f : kva_ex2(m[s] - M);
                const float4 x = *reinterpret_cast<const float4 *>(cl.map_shared_rank(&om[0][r][lane * 4], s));
                L += *cl.map_shared_rank(&lm[0][r], s) * f;
                o.x += x.x * f;
                o.y += x.y * f;
                o.z += x.z * f;
                o.w += x.w * f;
            }
            const float inv = M == -INFINITY ? 1.f : 1.f / L; // no slot seen: 0
            const int row = row0 + r;
            const __half2 lo = __floats2half2_rn(o.x * inv, o.y * inv), hi = __floats2half2_rn(o.z * inv, o.w * inv);
            *reinterpret_cast<uint2 *>(a.out + (row / G) * a.out_stride + (size_t)(kvh * G + row % G) * YLM_HEAD_DIM + lane * 4) =
                make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
        }
        if (a.acc) // all rows are this CTA's: the plan sees to it
        {
            if (tid < 8 * NT)
            {
                float m[KVA_CLUSTER], M = -INFINITY, L = 0.f;
#pragma unroll
                for (int s = 0; s < KVA_CLUSTER; s++)
                {
                    m[s] = s < C ? *cl.map_shared_rank(&mm[0][tid], s) : -INFINITY;
                    M = fmaxf(M, m[s]);
                }
#pragma unroll
                for (int s = 0; s < KVA_CLUSTER; s++)
                    if (s < C && m[s] != -INFINITY)
                        L += *cl.map_shared_rank(&lm[0][tid], s) * kva_ex2(m[s] - M);
                // a row that sees nothing weighs nothing
                state[tid] = M == -INFINITY ? make_float2(0.f, 0.f) : make_float2(M, 1.f / L);
            }
            __syncthreads();
            float *acc = a.acc + (size_t)kvh * a.c.cap;
            for (int j = sp * w.p.len + tid; j < j_end; j += KVA_THREADS)
            {
                const float4 *x = reinterpret_cast<const float4 *>(kept + (j - sp * w.p.len) * 8 * NT);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * NT; i++)
                {
                    const float4 v = x[i];
                    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int k = 0; k < 4; k++)
                    {
                        const float2 st = state[4 * i + k];
                        if (4 * i + k < R) // rows that are not there must not count
                            sum += kva_ex2(e[k] - st.x) * st.y;
                    }
                }
                acc[j] += sum;
            }
        }
        cl.sync(); // the sums stay until every CTA has read them
    }
}

// Launched as a programmatic dependent: its CTAs are resident when the first
// launch ends (-1.2 us a step).
// Joins the splits. CTAs [0, hkv * rows) write one output row each: every warp
// finds the row's M and l from the splits' (a lane each), then takes every eighth
// split's O, four dimensions a lane. The others add the weights of p.tile
// slots of one KV head to acc: first the M and 1 / l of every row, by all threads,
// then the slots, each by the LPS lanes (a power of two) that share its rows.
template <int LPS> __global__ void __launch_bounds__(KVA_JOIN) kv8_join_kernel(const Kv8Pass w)
{
    constexpr int WARPS = KVA_JOIN / 32;
    const Kv8AttnArgs &a = w.a;
    const int G = w.p.G, R = w.p.rows, S = w.p.splits, pad = w.p.pad;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.c.hkv * R;
    int b = blockIdx.x;
    pdl_wait();
    if (b < rows)
    {
        __shared__ float4 om[WARPS][32];
        const int g = b / R, r = b % R;
        const float2 *ml = reinterpret_cast<const float2 *>(w.ml) + (size_t)g * S * pad + r;
        const float4 *part = reinterpret_cast<const float4 *>(w.part) + (size_t)b * S * (YLM_HEAD_DIM / 4) + lane;
        float M = -INFINITY, L = 0.f;
        for (int s = lane; s < S; s += 32)
            M = fmaxf(M, ml[(size_t)s * pad].x);
        M = warp_max(M);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < S; s0 += 32)
        {
            const float2 x = s0 + lane < S ? ml[(size_t)(s0 + lane) * pad] : make_float2(-INFINITY, 0.f);
            const float f = x.x == -INFINITY ? 0.f : kva_ex2(x.x - M);
            L += x.y * f;
#pragma unroll
            for (int k = 0; k < 32 / WARPS; k++)
            {
                const int s = s0 + WARPS * k + warp;
                const float fs = __shfl_sync(0xffffffffu, f, WARPS * k + warp);
                if (s < S)
                {
                    const float4 v = part[(size_t)s * (YLM_HEAD_DIM / 4)];
                    o.x += v.x * fs;
                    o.y += v.y * fs;
                    o.z += v.z * fs;
                    o.w += v.w * fs;
                }
            }
        }
        L = warp_sum(L);
        om[warp][lane] = o;
        __syncthreads();
        if (tid < YLM_HEAD_DIM)
        {
            const float *of = reinterpret_cast<const float *>(om);
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < WARPS; k++)
                sum += of[k * YLM_HEAD_DIM + tid];
            a.out[(r / G) * a.out_stride + (size_t)(g * G + r % G) * YLM_HEAD_DIM + tid] =
                f2h(M == -INFINITY ? sum : sum / L); // no slot seen: 0
        }
        return;
    }
    __shared__ __align__(16) float2 state[128];
    __shared__ float2 join[KVA_JOIN];
    b -= rows;
    const int tiles = (a.n + w.p.tile - 1) / w.p.tile;
    const int g = b / tiles, j0 = b % tiles * w.p.tile, j1 = min(a.n, j0 + w.p.tile);
    float *acc = a.acc + (size_t)g * a.c.cap;
    const float4 *x = reinterpret_cast<const float4 *>(w.scores) + (size_t)g * a.n * (pad / 4);
    constexpr int U = 4, PER = KVA_JOIN / LPS; // slots in flight per thread, slots per round of the CTA
    const int l = tid % LPS;
    // the first scores are on their way while the state is found
    float4 v[U];
    auto load = [&](int j, int i) {
#pragma unroll
        for (int u = 0; u < U; u++)
            v[u] = x[(size_t)min(j + u * PER, j1 - 1) * (pad / 4) + i];
    };
    load(j0 + tid / LPS, l);
    const int parts = min(16, KVA_JOIN / pad), part = tid / pad, r = tid % pad;
    if (part < parts)
    {
        const float2 *ml = reinterpret_cast<const float2 *>(w.ml) + (size_t)g * S * pad + r;
        float M = -INFINITY, L = 0.f;
        if (r < R)
#pragma unroll 4
            for (int s = part; s < S; s += parts)
            {
                const float2 x = ml[(size_t)s * pad];
                const float m = fmaxf(M, x.x), ref = m == -INFINITY ? 0.f : m;
                L = L * kva_ex2(M - ref) + x.y * kva_ex2(x.x - ref);
                M = m;
            }
        join[tid] = make_float2(M, L);
    }
    __syncthreads();
    if (tid < pad)
    {
        float M = -INFINITY, L = 0.f;
        for (int p = 0; p < parts; p++)
            M = fmaxf(M, join[p * pad + tid].x);
        const float ref = M == -INFINITY ? 0.f : M;
        for (int p = 0; p < parts; p++)
            L += join[p * pad + tid].y * kva_ex2(join[p * pad + tid].x - ref);
        // a row that sees nothing weighs nothing
        state[tid] = M == -INFINITY ? make_float2(0.f, 0.f) : make_float2(M, 1.f / L);
    }
    __syncthreads();
    const float4 *st = reinterpret_cast<const float4 *>(state); // two rows each
    for (int jb = j0; jb < j1; jb += PER * U)
    {
        const int j = jb + tid / LPS;
        float sum[U] = {};
        for (int i = l; i < pad / 4; i += LPS)
        {
            if (jb > j0 || i > l)
                load(j, i);
            const float4 s0 = st[2 * i], s1 = st[2 * i + 1];
#pragma unroll
            for (int u = 0; u < U; u++)
            {
                sum[u] += kva_ex2(v[u].x - s0.x) * s0.y;
                // rows that are not there: whatever their scores hold must not count
                if (4 * i + 1 < R)
                    sum[u] += kva_ex2(v[u].y - s0.z) * s0.w;
                if (4 * i + 2 < R)
                    sum[u] += kva_ex2(v[u].z - s1.x) * s1.y;
                if (4 * i + 3 < R)
                    sum[u] += kva_ex2(v[u].w - s1.z) * s1.w;
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
        {
#pragma unroll
            for (int o = 1; o < LPS; o <<= 1)
                sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
            if (l == 0 && j + u * PER < j1)
                acc[j + u * PER] += sum[u];
        }
    }
}

// Dynamic shared memory: the rings, and for a cluster the scores of a split
static constexpr int kva_smem(int nt, bool cluster)
{
    return KVA_SMEM + (cluster ? KVA_ALONE_LEN * 8 * nt * (int)sizeof(float) : 0);
}

template <int FMT, int NT, bool CLUSTER> static cudaError_t attn_launch(const Kv8Pass &w, cudaStream_t s)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)w.p.splits, (unsigned)w.a.c.hkv, (unsigned)w.p.zblocks);
    cfg.blockDim = dim3(KVA_THREADS);
    cfg.dynamicSmemBytes = kva_smem(NT, CLUSTER);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CLUSTER ? (unsigned)w.p.splits : 1;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CLUSTER ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kv8_attn_kernel<FMT, NT, CLUSTER>, w);
}

template <int FMT> static cudaError_t attn_launch_fmt(const Kv8Pass &w, cudaStream_t s)
{
    if (w.p.nt == 1)
        return w.p.cluster ? attn_launch<FMT, 1, true>(w, s) : attn_launch<FMT, 1, false>(w, s);
    return w.p.cluster ? attn_launch<FMT, 2, true>(w, s) : attn_launch<FMT, 2, false>(w, s);
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
        w.part = static_cast<float *>(ws);
        w.ml = reinterpret_cast<float *>(static_cast<char *>(ws) + w.p.ml_off);
        w.scores = reinterpret_cast<float *>(static_cast<char *>(ws) + w.p.score_off);
        cudaError_t e = args.c.format == KV8_E4M3 ? attn_launch_fmt<KV8_E4M3>(w, s) : attn_launch_fmt<KV8_INT8>(w, s);
        if (e != cudaSuccess)
            return e;
        if (w.p.cluster)
            continue;
        const int tiles = args.acc ? (w.a.n + w.p.tile - 1) / w.p.tile : 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(args.c.hkv * (w.p.rows + tiles)));
        cfg.blockDim = dim3(KVA_JOIN);
        cfg.stream = s;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        e = w.p.lps == 1   ? cudaLaunchKernelEx(&cfg, kv8_join_kernel<1>, w)
            : w.p.lps == 2 ? cudaLaunchKernelEx(&cfg, kv8_join_kernel<2>, w)
            : w.p.lps == 8 ? cudaLaunchKernelEx(&cfg, kv8_join_kernel<8>, w)
                           : cudaLaunchKernelEx(&cfg, kv8_join_kernel<16>, w);
        if (e != cudaSuccess)
            return e;
    }
    return cudaSuccess;
}

template <int FMT> static cudaError_t prepare_fmt()
{
    const auto opt_in = [](const void *f, int bytes) {
        return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    cudaError_t e = opt_in((const void *)kv8_attn_kernel<FMT, 1, false>, kva_smem(1, false));
    if (e == cudaSuccess)
        e = opt_in((const void *)kv8_attn_kernel<FMT, 2, false>, kva_smem(2, false));
    if (e == cudaSuccess)
        e = opt_in((const void *)kv8_attn_kernel<FMT, 1, true>, kva_smem(1, true));
    if (e == cudaSuccess)
        e = opt_in((const void *)kv8_attn_kernel<FMT, 2, true>, kva_smem(2, true));
    return e;
}

cudaError_t kv8_prepare()
{
    const cudaError_t e = prepare_fmt<KV8_E4M3>();
    return e == cudaSuccess ? prepare_fmt<KV8_INT8>() : e;
}

} // namespace ylm
