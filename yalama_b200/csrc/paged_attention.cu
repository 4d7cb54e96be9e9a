// Attention of a step's rows over the paged cache (device rules: paged.cuh).
//
//   x_rj = q_r . k_j / sqrt(128) for the slots j < n + t of the row's request that row i sees: j < n, and
//          the slots n + d of its ancestors d and of itself (without a tree: d <= i)
//   o_r  = sum_j softmax(x_r)_j v_j,  0 where the row sees no slot
//
// An item is a request's KV head and up to tpi of its tokens: their G query heads each are the rows of one or two
// tiles of 128 (row i * G + h). It has a unit for each 128 slots its tokens see. The units of all items, in order, are
// dealt evenly to one CTA per SM, so that requests of any lengths keep all SMs busy to the end; an item that
// a CTA border cuts leaves sums (M, l, O) per CTA, which paged_join_kernel joins.
//
// Both products run on the 5th-generation tensor cores, from two streams that take turns, so that one stream's softmax
// runs while the other's products do: with more than 128 rows the item's two row tiles on the same slots, else even and
// odd units of the one tile, joined at the end. Warps: 0 K tiles by TMA, 2 Q and V tiles, 3 cleans V (below), 1
// issues S_w = Q K^T and O_w += P_w V, 4-7 and 8-11 the softmax of streams 0 and 1, a row a thread. TMEM: S_0, S_1
// (P_w over the first half of S_w), O_0, O_1.
//
// Softmax: weights 2^((x - mr) / sqrt(128) log2 e + PX_LEAD) with a reference score mr per row and stream, which moves
// only when a weight would pass 2^PX_MOST. They enter P V rounded to FP16, the matrix unit's operand: off by 2^-11
// of themselves at most down to 2^-25 of the row's largest, by 2^-36 of the largest below. The sums are FP32.
//
// A hidden slot's weight is 0, but 0 x NaN is not: where some row of an item does not see some slot (the last
// units), warp 3 sets what is not finite in those rows of V to 0 before the product, and says so where the slot is one of the
// step's; the rows that do see it then get it added at the end. Scores of hidden slots are replaced, whatever they are.
#include "paged.cuh"
#include "ylm_tc.cuh"
#include <algorithm>

namespace ylm {

constexpr int PX_TILE = 128 * 128 * 2; // a tile of 128 rows or slots: two halves of 64 dimensions
constexpr int PX_THREADS = 384;
constexpr int PX_KST = 3;
constexpr int PX_CONTROL = 3072; // barriers, the streams' (M, l)
constexpr int PX_SMEM = 7 * PX_TILE + PX_CONTROL;
constexpr float PX_SCALE = (float)(1.4426950408889634 / 11.313708498984760); // log2(e) / sqrt(128)
// FP16 weights end at 2^16; a higher lead keeps more of the small ones and moves the reference more often
constexpr float PX_LEAD = 11.f, PX_MOST = 15.9f;
constexpr float PX_RISE = (PX_MOST - PX_LEAD) / PX_SCALE; // in scores

struct PagedPlan
{
    int G, tpt, tpi; // query heads per KV head, tokens per 128-row tile and per item
    int pair;        // 1: items of two tiles (some request may have more than tpt rows)
    int cap;         // most rows of an item
    int ctas;
    size_t ml_off, o_off, bytes;
};

static PagedPlan paged_plan(const PagedAttnArgs &a, int num_sms)
{
    PagedPlan p;
    p.G = a.hq / a.c.hkv;
    p.tpt = 128 / p.G;
    p.pair = a.st.max_rows > p.tpt;
    p.tpi = p.pair ? 2 * p.tpt : p.tpt;
    p.cap = std::max(1, std::min(p.tpi, a.st.max_rows)) * p.G;
    p.ctas = num_sms;
    p.ml_off = ((size_t)p.ctas * 64 + 255) / 256 * 256;
    p.o_off = p.ml_off + ((size_t)p.ctas * 2 * p.cap * sizeof(float2) + 255) / 256 * 256;
    p.bytes = p.o_off + (size_t)p.ctas * 2 * p.cap * YLM_HEAD_DIM * sizeof(float);
    return p;
}

size_t paged_attn_workspace(const PagedAttnArgs &a, int num_sms) { return paged_plan(a, num_sms).bytes; }

// Where a CTA's share starts; left in the workspace for the join.
struct PagedCut
{
    long long u0, u1;
    int s, qp, kvh, tile0, kt;
    int cut; // the share starts inside an item
};
static_assert(sizeof(PagedCut) <= 64, "64 bytes a CTA");

struct PagedPass
{
    PagedAttnArgs a;
    PagedPlan p;
    PagedCut *cuts;
    float2 *ml; // [cta][2][cap]: (M, l) of the item that the share starts inside of, and of the one it ends inside of
    float *o;   // [cta][2][cap][128]
};

// ------------------------------------------------------------------ units
// units of the item with tokens [qp * tpi, ...) of a request: its last token sees slots below n + min(t, ...)
__device__ __forceinline__ int px_units(int n, int t, int qp, int tpi) { return (n + min(t, (qp + 1) * tpi) + 127) >> 7; }

// sum of ceil((n + i * tpi) / 128) over i = 1..k: each is (x + r) / 128 with r = -x mod 128, whose
// values repeat after 128 / g and then are those that are congruent to -n mod g, for g the power of two in tpi
__device__ __forceinline__ long long px_before(int n, int k, int tpi)
{
    if (k <= 0)
        return 0;
    const int g = min(tpi & -tpi, 128), period = 128 / g;
    long long sum = (long long)k * n + (long long)tpi * k * (k + 1) / 2;
    sum += (long long)(k / period) * ((long long)period * (-n & (g - 1)) + (long long)g * period * (period - 1) / 2);
    for (int i = 1; i <= k % period; i++)
        sum += -(n + i * tpi) & 127;
    return sum >> 7;
}

__device__ __forceinline__ long long px_request_units(const PagedRequest &r, int tpi, int hkv)
{
    const int items = (r.t + tpi - 1) / tpi;
    return hkv * (px_before(r.n, items - 1, tpi) + px_units(r.n, r.t, items - 1, tpi));
}

// A CTA's way through its share: one item, or a part of one, after another. Every warp role walks it alike.
struct PagedItem
{
    int s, qp, kvh, tile0, tiles, seq; // seq: its number among the CTA's items
    PagedRequest r;
    long long left; // units of the share from here on

    __device__ __forceinline__ bool start(const PagedPass &w, const PagedCut &c)
    {
        s = c.s, qp = c.qp, kvh = c.kvh, tile0 = c.tile0;
        left = c.u1 - c.u0;
        seq = 0;
        if (left <= 0)
            return false;
        bool bad;
        paged_request(w.a.st, w.a.c.page, s, r, bad);
        tiles = (int)min((long long)(c.kt - tile0), left);
        return true;
    }
    __device__ __forceinline__ bool next(const PagedPass &w)
    {
        left -= tiles;
        if (left <= 0)
            return false;
        seq++;
        tile0 = 0;
        if (++kvh == w.a.c.hkv)
        {
            kvh = 0;
            if (++qp * w.p.tpi >= r.t)
            {
                qp = 0;
                bool bad;
                do
                {
                    if (++s >= w.a.st.n_seq)
                        return false;
                } while (!paged_request(w.a.st, w.a.c.page, s, r, bad));
            }
        }
        tiles = (int)min((long long)units(w), left);
        return true;
    }
    __device__ __forceinline__ int units(const PagedPass &w) const { return px_units(r.n, r.t, qp, w.p.tpi); }
    __device__ __forceinline__ int first(const PagedPass &w) const { return qp * w.p.tpi; } // its first token
    // slots below are seen by every row of the item
    __device__ __forceinline__ int open(const PagedPass &w) const
    {
        return r.n + (w.a.st.parent ? (r.t == 1 ? 1 : 0) : first(w) + 1);
    }
    __device__ __forceinline__ bool two(const PagedPass &w) const { return r.t - first(w) > w.p.tpt; }
};

// ------------------------------------------------------------------ waits
// Bounded: after 2 s, or once another warp gave up, *abort is set and the caller unwinds.
__device__ __forceinline__ bool px_wait(uint64_t *bar, uint32_t parity, volatile int *abort)
{
    if (mbar_try_wait(bar, parity))
        return true;
    const uint64_t t0 = globaltimer_ns();
    for (;;)
    {
        for (int i = 0; i < 64; i++)
            if (mbar_try_wait(bar, parity))
                return true;
        if (*abort || globaltimer_ns() - t0 > YLM_WAIT_LIMIT_NS)
        {
            *abort = 1;
            return false;
        }
    }
}
// The same, all lanes of a warp leaving alike.
__device__ __forceinline__ bool px_wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort)
{
    return __all_sync(0xffffffffu, px_wait(bar, parity, abort));
}

// For copies and products that are on their way and need nobody else: whatever happened, they end first.
__device__ __forceinline__ void px_drain(uint64_t *bar, uint32_t parity)
{
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 <= YLM_WAIT_LIMIT_NS)
        ;
}

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z,
                                            int32_t u, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                     smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(u), "r"(smem_u32(bar))
                 : "memory");
}

// One unit's K or V into a stage: a warp, a page's half of the dimensions a lane. Pages behind the request's
// last slot, and pages that are not in the pool, arrive as zeros (coordinate -1).
__device__ __forceinline__ void px_load(uint8_t *dst, const CUtensorMap *map, const PagedPass &w, const PagedItem &it,
                                        int tile, uint64_t *bar, int lane)
{
    const int pages = 128 >> w.a.c.page_shift, k = lane >> 1, half = lane & 1;
    if (lane == 0)
        mbar_arrive_expect_tx(bar, PX_TILE);
    __syncwarp();
    if (k < pages)
    {
        const int slot = tile * 128 + k * w.a.c.page;
        const int page = slot < it.r.n + it.r.t ? paged_page(w.a.st, w.a.c, it.s, slot) : -1;
        tma_load_4d(dst + half * (PX_TILE / 2) + k * w.a.c.page * 128, map, half * 64, 0, it.kvh, page, bar);
    }
}

template <bool PAIR>
__global__ void __launch_bounds__(PX_THREADS, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedPass w)
{
    constexpr int KST = PX_KST, QT = PAIR ? 2 : 1, VST = 7 - KST - QT;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *sq = smem, *sk = sq + QT * PX_TILE, *sv = sk + KST * PX_TILE;
    uint8_t *control = smem + 7 * PX_TILE;
    uint64_t *bars = reinterpret_cast<uint64_t *>(control);
    uint64_t *k_full = bars, *k_empty = k_full + KST, *v_full = k_empty + KST, *v_empty = v_full + VST,
             *v_clean = v_empty + VST, *q_full = v_clean + VST, *q_empty = q_full + 1, *s_full = q_empty + 1,
             *p_full = s_full + 2, *o_done = p_full + 2, *joined = o_done + 2, *parted = joined + 1, *done = parted + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(control + 256);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(control + 260);
    volatile int *special = reinterpret_cast<volatile int *>(control + 264); // [8]: 1 + the item that had one, by its number mod 8
    PagedCut *mine = reinterpret_cast<PagedCut *>(control + 320);
    long long *sums = reinterpret_cast<long long *>(control + 384); // [12]
    float2 *state = reinterpret_cast<float2 *>(control + 1024);     // [2][128]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PagedAttnArgs &a = w.a;
    const PagedStep &st = a.st;

    pdl_launch_dependents(); // the joining CTAs may start; they wait for this grid's end
    if (tid == 0)
    {
        for (int i = 0; i < KST; i++)
        {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < VST; i++)
        {
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&v_clean[i], 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int i = 0; i < 2; i++)
        {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(joined, 8);
        mbar_init(parted, 8);
        mbar_init(done, 1);
        *abort_flag = 0;
        for (int i = 0; i < 8; i++)
            special[i] = 0;
        mine->u0 = mine->u1 = 0;
        mine->cut = 0;
        fence_mbar_init();
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&kmap);
        prefetch_tensormap(&vmap);
    }
    if (warp == 1)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    // ---- this CTA's share: requests in runs of `run` a thread, their units summed over the threads
    const int run = (st.n_seq + PX_THREADS - 1) / PX_THREADS;
    long long own = 0;
    for (int s = tid * run; s < min(st.n_seq, (tid + 1) * run); s++)
    {
        PagedRequest r;
        bool bad;
        if (paged_request(st, a.c.page, s, r, bad))
            own += px_request_units(r, w.p.tpi, a.c.hkv);
        else if (bad && blockIdx.x == 0)
            paged_fault(st, PAGED_BAD_REQUEST);
    }
    long long incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        incl += lane >= o ? x : 0;
    }
    if (lane == 31)
        sums[warp] = incl;
    __syncthreads();
    long long total = 0, before = incl - own;
#pragma unroll
    for (int i = 0; i < PX_THREADS / 32; i++)
    {
        total += sums[i];
        before += i < warp ? sums[i] : 0;
    }
    const long long ctas = min((long long)gridDim.x, total);
    if (blockIdx.x < ctas)
    {
        const long long u0 = total * blockIdx.x / ctas, u1 = total * (blockIdx.x + 1) / ctas;
        if (u0 >= before && u0 < before + own)
        {
            long long rest = u0 - before;
            int s = tid * run;
            PagedRequest r;
            bool bad;
            for (;; s++)
            {
                if (!paged_request(st, a.c.page, s, r, bad))
                    continue;
                const long long u = px_request_units(r, w.p.tpi, a.c.hkv);
                if (rest < u)
                    break;
                rest -= u;
            }
            // the last item row whose units before it do not pass `rest`
            int lo = 0, hi = (r.t + w.p.tpi - 1) / w.p.tpi;
            while (hi - lo > 1)
            {
                const int mid = (lo + hi) / 2;
                if (a.c.hkv * px_before(r.n, mid, w.p.tpi) <= rest)
                    lo = mid;
                else
                    hi = mid;
            }
            rest -= a.c.hkv * px_before(r.n, lo, w.p.tpi);
            PagedCut c;
            c.u0 = u0;
            c.u1 = u1;
            c.s = s;
            c.qp = lo;
            c.kt = px_units(r.n, r.t, lo, w.p.tpi);
            c.kvh = (int)(rest / c.kt);
            c.tile0 = (int)(rest % c.kt);
            c.cut = c.tile0 > 0;
            *mine = c;
            w.cuts[blockIdx.x] = c;
        }
    }
    else if (tid == 0)
    {
        PagedCut c = {};
        c.u0 = c.u1 = total;
        w.cuts[blockIdx.x] = c;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const PagedCut cut = *mine;
    const int G = w.p.G, tpt = w.p.tpt;
    PagedItem it;
    bool more = it.start(w, cut);

    if (warp == 0)
    {
        // ---- K tiles
        int kc = 0;
        for (bool ok = true; more && ok; more = it.next(w))
            for (int t = 0; t < it.tiles; t++, kc++)
            {
                const int s = kc % KST;
                if (*abort_flag || (kc >= KST && !px_wait_warp(&k_empty[s], (kc / KST - 1) & 1, abort_flag)))
                {
                    ok = false;
                    break;
                }
                px_load(sk + s * PX_TILE, &kmap, w, it, it.tile0 + t, &k_full[s], lane);
            }
        // every copy has landed before the CTA can end
        for (int j = max(0, kc - KST); j < kc; j++)
            px_drain(&k_full[j % KST], (j / KST) & 1);
    }
    else if (warp == 2)
    {
        // ---- the items' Q, and V tiles
        int vc = 0, items = 0;
        for (bool ok = true; more && ok; more = it.next(w), items++)
        {
            if (*abort_flag || (items && !px_wait_warp(q_empty, (items - 1) & 1, abort_flag)))
                break;
            if (lane == 0)
            {
                const int tiles = PAIR && it.two(w) ? 2 : 1, row = it.r.row0 + it.first(w);
                mbar_arrive_expect_tx(q_full, (uint32_t)(tiles * tpt * G * 256));
                for (int i = 0; i < tiles; i++)
                {
                    tma_load_3d(sq + i * PX_TILE, &qmap, 0, it.kvh * G, row + i * tpt, q_full);
                    tma_load_3d(sq + i * PX_TILE + PX_TILE / 2, &qmap, 64, it.kvh * G, row + i * tpt, q_full);
                }
            }
            __syncwarp();
            for (int t = 0; t < it.tiles; t++, vc++)
            {
                const int s = vc % VST;
                if (*abort_flag || (vc >= VST && !px_wait_warp(&v_empty[s], (vc / VST - 1) & 1, abort_flag)))
                {
                    items++; // its Q is on the way
                    ok = false;
                    break;
                }
                px_load(sv + s * PX_TILE, &vmap, w, it, it.tile0 + t, &v_full[s], lane);
            }
            if (!ok)
                break;
        }
        if (items)
            px_drain(q_full, (items - 1) & 1);
        for (int j = max(0, vc - VST); j < vc; j++)
            px_drain(&v_full[j % VST], (j / VST) & 1);
    }
    else if (warp == 3)
    {
        // ---- V without what is not finite in slots that some row does not see
        int vc = 0;
        for (bool ok = true; more && ok; more = it.next(w))
            for (int t = 0; t < it.tiles; t++, vc++)
            {
                const int s = vc % VST, k0 = (it.tile0 + t) * 128, n = it.r.n + it.r.t;
                if (!px_wait_warp(&v_full[s], (vc / VST) & 1, abort_flag))
                {
                    ok = false;
                    break;
                }
                // (pages behind the last slot's are zeros)
                const int lo = max(0, it.open(w) - k0), hi = min(128, ((n + a.c.page - 1) & -a.c.page) - k0);
                if (lo < hi)
                {
                    bool found = false;
                    for (int i = lo * 16 + lane; i < hi * 16; i += 32)
                    {
                        // row i / 16's 16-byte pieces, in whatever order the swizzle has them
                        uint4 *p = reinterpret_cast<uint4 *>(sv + s * PX_TILE + (i & 8 ? PX_TILE / 2 : 0) + (i >> 4) * 128 +
                                                             (i & 7) * 16);
                        uint4 v = *p;
                        // an exponent of ones carries into the sign's place
                        uint32_t f[4] = {v.x, v.y, v.z, v.w}, any = 0;
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            any |= (f[k] & 0x7C007C00u) + 0x04000400u;
                        if (any & 0x80008000u)
                        {
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                f[k] &= ~((((f[k] & 0x7C007C00u) + 0x04000400u & 0x80008000u) >> 15) * 0xFFFFu);
                            *p = make_uint4(f[0], f[1], f[2], f[3]);
                            found |= k0 + (i >> 4) < n;
                        }
                    }
                    if (found)
                        special[it.seq & 7] = it.seq + 1;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if (lane == 0)
                    mbar_arrive(&v_clean[s]);
            }
    }
    else if (warp == 1)
    {
        // ---- the products
        if (lane == 0)
        {
            const uint32_t idesc_s = tc_idesc(128, 128);
            const uint32_t idesc_o = tc_idesc(128, 128) | (1u << 16); // B (V) MN-major
            int kc = 0, items = 0, np[2] = {0, 0};
            bool ok = true;
            for (; more && ok; more = it.next(w), items++)
            {
                const bool two = PAIR && it.two(w);
                const int tasks = two ? 2 * it.tiles : it.tiles;
                ok = px_wait(q_full, items & 1, abort_flag);
                // task i: stream i & 1 on unit i (two streams of one tile), or on unit i / 2 (a tile each)
                const auto scores = [&](int i) {
                    const int unit = two ? i >> 1 : i, st_ = (kc + unit) % KST, s = i & 1;
                    if (!px_wait(&k_full[st_], ((kc + unit) / KST) & 1, abort_flag))
                        return false;
                    tc_fence_after();
                    const uint32_t q0 = smem_u32(sq + (two ? s * PX_TILE : 0)), k0 = smem_u32(sk + st_ * PX_TILE);
#pragma unroll
                    for (int kk = 0; kk < 8; kk++)
                    {
                        const uint32_t off = (uint32_t)((kk >> 2) * (PX_TILE / 2) + (kk & 3) * 32);
                        tc_mma(tmem + 128u * s, smem_desc_k128(q0 + off), smem_desc_k128(k0 + off), idesc_s, kk ? 1u : 0u);
                    }
                    tc_commit(&s_full[s]);
                    if (!two || s)
                        tc_commit(&k_empty[st_]);
                    if (i == tasks - 1)
                        tc_commit(q_empty);
                    return true;
                };
                ok = ok && scores(0) && (tasks < 2 || scores(1));
                for (int i = 0; ok && i < tasks; i++)
                {
                    const int unit = two ? i >> 1 : i, st_ = (kc + unit) % VST, s = i & 1;
                    if (!px_wait(&p_full[s], np[s] & 1, abort_flag) ||
                        !px_wait(&v_clean[st_], ((kc + unit) / VST) & 1, abort_flag))
                    {
                        ok = false;
                        break;
                    }
                    np[s]++;
                    tc_fence_after();
                    const uint32_t v0 = smem_u32(sv + st_ * PX_TILE);
#pragma unroll
                    for (int kk = 0; kk < 8; kk++)
                        tc_mma_ts(tmem + 256u + 128u * s, tmem + 128u * s + 8u * kk,
                                  smem_desc_mn128(v0 + kk * 2048, PX_TILE / 2, 1024), idesc_o, (i > 1 || kk) ? 1u : 0u);
                    tc_commit(&o_done[s]);
                    if (!two || s)
                        tc_commit(&v_empty[st_]);
                    if (i + 2 < tasks)
                        ok = scores(i + 2);
                }
                kc += it.tiles;
            }
            if (!ok)
                *abort_flag = 1;
            // all products are complete before TMEM is given back
            tc_commit(done);
            px_drain(done, 0);
        }
        __syncwarp();
    }
    else
    {
        // ---- softmax: stream ws, row `row` of its tile
        const int ws = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16), tS = trow + 128u * ws, tO = trow + 256u;
        int nt[2] = {0, 0}; // tasks of the streams so far
        int meets = 0;
        bool ok = true;
        for (; more && ok; more = it.next(w))
        {
            const bool two = PAIR && it.two(w);
            const int n = it.r.n, t = it.r.t;
            const int tok0 = it.first(w) + (two ? ws * tpt : 0);  // first token of this stream's tile
            const int rows = min(tpt, t - tok0) * G;              // rows of the tile
            const int mine_t = two ? it.tiles : (it.tiles + 1 - ws) >> 1;
            const int i = tok0 + row / G; // this row's token (one of the request's where row < rows)
            const bool works = quad * 32 < rows;
            const int clear = it.open(w);
            uint32_t anc[4] = {0, 0, 0, 0};
            if (st.parent && works)
            {
                PagedTree tree;
                if (tree.load(st, it.r, lane))
                    paged_fault(st, PAGED_BAD_PARENT);
                int cur = i < t && row < rows ? i : -1;
                while (__any_sync(0xffffffffu, cur >= 0))
                {
                    const int from = max(cur, 0), k = from >> 5;
                    if (cur >= 0)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            anc[j] |= j == k ? 1u << (from & 31) : 0u;
                    int p[4];
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        p[j] = __shfl_sync(0xffffffffu, tree.p[j], from & 31);
                    cur = cur < 0 ? -1 : k == 0 ? p[0] : k == 1 ? p[1] : k == 2 ? p[2] : p[3];
                }
            }
            // bits of the slots k .. k + 31 that this row sees
            const auto seen = [&](int k) -> uint32_t {
                const int c = (st.parent ? n : n + i + 1) - k; // so many of them from the first on
                uint32_t bits = c >= 32 ? 0xFFFFFFFFu : c <= 0 ? 0u : (1u << c) - 1u;
                if (st.parent)
                {
                    const int d = k - n; // the first one's row
                    if (d > -32 && d < 0)
                        bits |= anc[0] << -d;
                    else if (d >= 0 && d < 128)
                    {
                        const int q = d >> 5;
                        const uint32_t lo = q == 0 ? anc[0] : q == 1 ? anc[1] : q == 2 ? anc[2] : anc[3];
                        const uint32_t hi = q == 0 ? anc[1] : q == 1 ? anc[2] : q == 2 ? anc[3] : 0u;
                        bits = __funnelshift_r(lo, hi, d & 31);
                    }
                }
                return bits;
            };
            float mr = -INFINITY, l = 0.f;
            for (int u = 0; u < mine_t; u++)
            {
                const int k0 = (it.tile0 + (two ? u : 2 * u + ws)) * 128;
                uint32_t bad = 0; // sixteens of slots that are not in the pool
                if (works)
                {
                    const int slot = k0 + lane * 16;
                    const bool out = lane < 8 && slot < n + t && paged_page(st, a.c, it.s, slot) < 0;
                    bad = __ballot_sync(0xffffffffu, out);
                    if (out)
                        paged_fault(st, PAGED_BAD_PAGE);
                }
                // (the product before this one is complete, too, long since: nobody falls two phases of o_done behind,
                // where a parity would say nothing)
                if (!px_wait_warp(&s_full[ws], nt[ws] & 1, abort_flag) ||
                    (u && !px_wait_warp(&o_done[ws], (nt[ws] - 1) & 1, abort_flag)))
                {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (works)
                {
                    const bool edge = bad || k0 + 128 > clear;
                    const auto load = [&](int c, float(&v)[32]) {
                        tmem_ld32(tS + 32u * c, v);
                        if (edge)
                        {
                            uint32_t bits = seen(k0 + 32 * c);
                            if (bad >> (2 * c) & 1u)
                                bits &= 0xFFFF0000u;
                            if (bad >> (2 * c) & 2u)
                                bits &= 0x0000FFFFu;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                v[j] = bits >> j & 1u ? v[j] : -INFINITY;
                        }
                    };
                    float mx = -INFINITY;
#pragma unroll
                    for (int c = 0; c < 4; c++)
                    {
                        float v[32];
                        load(c, v);
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            mx = fmaxf(mx, v[j]);
                    }
                    if (u == 0)
                        mr = mx;
                    else if (__any_sync(0xffffffffu, mx > mr + PX_RISE))
                    {
                        // the sums so far in units of the new reference
                        float f = 1.f;
                        if (mx > mr + PX_RISE)
                        {
                            f = ex2_ftz((mr - mx) * PX_SCALE);
                            mr = mx;
                        }
                        l *= f;
#pragma unroll
                        for (int c = 0; c < 4; c++)
                        {
                            float v[32];
                            tmem_ld32(tO + 128u * ws + 32u * c, v);
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                v[j] *= f;
                            tmem_st32(tO + 128u * ws + 32u * c, v);
                        }
                    }
                    const float ref = mr == -INFINITY ? 0.f : mr; // nothing seen: every weight 0
                    float sum[2] = {0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 4; c += 2)
                    {
                        uint32_t pk[32];
#pragma unroll
                        for (int h = 0; h < 2; h++)
                        {
                            float v[32];
                            load(c + h, v);
#pragma unroll
                            for (int j = 0; j < 32; j += 2)
                            {
                                const float x = ex2_ftz(fmaf(v[j] - ref, PX_SCALE, PX_LEAD));
                                const float y = ex2_ftz(fmaf(v[j + 1] - ref, PX_SCALE, PX_LEAD));
                                sum[0] += x;
                                sum[1] += y;
                                const __half2 p = __floats2half2_rn(x, y);
                                pk[16 * h + (j >> 1)] = *reinterpret_cast<const uint32_t *>(&p);
                            }
                        }
                        tmem_st32(tS + 16u * c, reinterpret_cast<const float *>(pk));
                    }
                    l += sum[0] + sum[1];
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&p_full[ws]);
                nt[ws]++;
            }
            nt[ws ^ 1] += two ? it.tiles : (it.tiles + ws) >> 1;
            if (!ok)
                break;
            // ---- the item's rows: whole, or this share's part
            const bool whole = it.tile0 == 0 && it.tiles == it.units(w);
            const int slot = it.tile0 ? 0 : 1;
            const int rho = (two ? ws * tpt * G : 0) + row; // the row's number in the item
            float M = mr, L = l, f0 = ws ? 0.f : 1.f, f1 = ws ? 1.f : 0.f;
            int c0 = 0, c1 = 4; // this thread's share of the dimensions, 32 each
            if (!two)
            {
                // the streams' sums are of the same rows: half of the dimensions each
                state[ws * 128 + row] = make_float2(mr, l);
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(joined);
                if (!px_wait_warp(joined, meets & 1, abort_flag))
                {
                    ok = false;
                    break;
                }
                const float2 x = state[row], y = state[128 + row];
                M = fmaxf(x.x, y.x);
                f0 = x.x == -INFINITY ? 0.f : ex2_ftz((x.x - M) * PX_SCALE);
                f1 = y.x == -INFINITY ? 0.f : ex2_ftz((y.x - M) * PX_SCALE);
                L = x.y * f0 + y.y * f1;
                c0 = 2 * ws;
                c1 = c0 + 2;
            }
            // every product of the item is in the sums
            bool in = true;
#pragma unroll
            for (int s = 0; s < 2; s++)
                if (!two || s == ws)
                    in = in && (nt[s] == 0 || px_wait_warp(&o_done[s], (nt[s] - 1) & 1, abort_flag));
            if (!in)
            {
                ok = false;
                break;
            }
            tc_fence_after();
            if (works)
            {
                const bool both = !two && it.tiles > 1; // stream 1 of a single unit has no sums
                const bool odd = special[it.seq & 7] == it.seq + 1;
                const float inv = M == -INFINITY ? 0.f : 1.f / L;
                const int64_t r = it.r.row0 + i;
                for (int c = c0; c < c1; c++)
                {
                    __syncwarp();
                    float v[32];
                    if (two)
                        tmem_ld32(tO + 128u * ws + 32u * c, v);
                    else
                    {
                        tmem_ld32(tO + 32u * c, v);
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            v[j] *= f0;
                        if (both)
                        {
                            float y[32];
                            tmem_ld32(tO + 128u + 32u * c, y);
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                v[j] = f1 == 0.f ? v[j] : fmaf(y[j], f1, v[j]);
                        }
                    }
                    if (odd && row < rows)
                    {
                        // what was taken out of the values that this row sees
                        const int lo = max(clear, it.tile0 * 128), hi = min(n + t, (it.tile0 + it.tiles) * 128);
                        for (int k = lo; k < hi; k++)
                        {
                            const int page = seen(k) & 1u ? paged_page(st, a.c, it.s, k) : -1;
                            if (page < 0)
                                continue;
                            const __half *src = a.c.v + paged_offset(a.c, page, k) +
                                                (size_t)it.kvh * a.c.page * YLM_HEAD_DIM + 32 * c;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                            {
                                const float x = h2f(src[j]);
                                v[j] += x - x != 0.f ? x : 0.f; // (x - x is NaN)
                            }
                        }
                    }
                    if (row < rows)
                    {
                        if (whole)
                        {
                            uint4 *dst = reinterpret_cast<uint4 *>(a.out + r * a.out_stride +
                                                                   (it.kvh * G + row % G) * YLM_HEAD_DIM + 32 * c);
#pragma unroll
                            for (int j = 0; j < 4; j++)
                            {
                                __half2 h[4];
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    h[e] = __floats2half2_rn(v[8 * j + 2 * e] * inv, v[8 * j + 2 * e + 1] * inv);
                                dst[j] = *reinterpret_cast<const uint4 *>(h);
                            }
                        }
                        else
                        {
                            float4 *dst = reinterpret_cast<float4 *>(
                                w.o + (((size_t)blockIdx.x * 2 + slot) * w.p.cap + rho) * YLM_HEAD_DIM + 32 * c);
#pragma unroll
                            for (int j = 0; j < 8; j++)
                                dst[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                        }
                    }
                }
                if (!whole && row < rows && c0 == 0)
                    w.ml[((size_t)blockIdx.x * 2 + slot) * w.p.cap + rho] = make_float2(M, L);
            }
            if (!two)
            {
                // the other stream's sums and state have been read: they may change
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(parted);
                if (!px_wait_warp(parted, meets & 1, abort_flag))
                    ok = false;
                meets++;
            }
        }
        if (!ok)
            *abort_flag = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
    {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (tid == 0 && *abort_flag)
        paged_fault(st, PAGED_TIMEOUT);
}

// ------------------------------------------------------------------ join
// CTA b, for the item that share b starts inside of, where share b - 1 holds its start: rows blockIdx.y * 8 + warp, four
// dimensions a lane. Launched as a programmatic dependent.
constexpr int PJ_WARPS = 8;

__global__ void __launch_bounds__(32 * PJ_WARPS) paged_join_kernel(const __grid_constant__ PagedPass w)
{
    const int lane = threadIdx.x & 31, b = blockIdx.x + 1;
    pdl_wait();
    const PagedCut c = w.cuts[b];
    if (!c.cut || c.tile0 > c.u0 - w.cuts[b - 1].u0)
        return;
    const PagedAttnArgs &a = w.a;
    PagedRequest r;
    bool bad;
    paged_request(a.st, a.c.page, c.s, r, bad);
    const int tok0 = c.qp * w.p.tpi, rows = min(w.p.tpi, r.t - tok0) * w.p.G;
    const int rho = blockIdx.y * PJ_WARPS + (threadIdx.x >> 5);
    if (rho >= rows)
        return;
    // part 0 is share b - 1's end, part k the start of share b - 1 + k
    const long long end = c.u0 - c.tile0 + c.kt;
    int parts = 2;
    while (b + parts - 1 < (int)gridDim.x + 1 && w.cuts[b + parts - 1].u0 < end)
        parts++;
    const auto at = [&](int k) { return (size_t)((b - 1 + k) * 2 + (k == 0)) * w.p.cap + rho; };
    float M = -INFINITY, L = 0.f;
    for (int k = lane; k < parts; k += 32)
        M = fmaxf(M, w.ml[at(k)].x);
    M = warp_max(M);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < parts; k++)
    {
        const float2 ml = w.ml[at(k)];
        const float f = ml.x == -INFINITY ? 0.f : ex2_ftz((ml.x - M) * PX_SCALE);
        const float4 x = *reinterpret_cast<const float4 *>(w.o + at(k) * YLM_HEAD_DIM + lane * 4);
        L += ml.y * f;
        o.x += x.x * f;
        o.y += x.y * f;
        o.z += x.z * f;
        o.w += x.w * f;
    }
    const float inv = M == -INFINITY ? 0.f : 1.f / L;
    __half2 h[2] = {__floats2half2_rn(o.x * inv, o.y * inv), __floats2half2_rn(o.z * inv, o.w * inv)};
    *reinterpret_cast<uint2 *>(a.out + (int64_t)(r.row0 + tok0 + rho / w.p.G) * a.out_stride +
                               (c.kvh * w.p.G + rho % w.p.G) * YLM_HEAD_DIM + lane * 4) = *reinterpret_cast<const uint2 *>(h);
}

// ------------------------------------------------------------------ host side
// The pool as [n_pages][hkv][page][128], a page's head and half of its dimensions a box.
static bool px_pool_map(CUtensorMap *map, const __half *p, const PagedCache &c)
{
    auto enc = encoder();
    if (!enc)
        return false;
    cuuint64_t dims[4] = {128, (cuuint64_t)c.page, (cuuint64_t)c.hkv, (cuuint64_t)c.n_pages};
    cuuint64_t strides[3] = {256, (cuuint64_t)c.page * 256, (cuuint64_t)c.page * 256 * c.hkv};
    cuuint32_t box[4] = {64, (cuuint32_t)c.page, 1, 1}, estr[4] = {1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half *>(p), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Q as [rows][hq][128], the G heads of tpt tokens and half of their dimensions a box: rows i * G + h of a tile.
static bool px_q_map(CUtensorMap *map, const PagedAttnArgs &a, const PagedPlan &p)
{
    auto enc = encoder();
    if (!enc)
        return false;
    cuuint64_t dims[3] = {128, (cuuint64_t)a.hq, (cuuint64_t)a.st.rows};
    cuuint64_t strides[2] = {256, (cuuint64_t)a.q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)p.G, (cuuint32_t)p.tpt}, estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half *>(a.q), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t paged_attn_launch(const PagedAttnArgs &a, void *ws, int num_sms, cudaStream_t s)
{
    if (a.st.rows <= 0 || a.st.n_seq <= 0 || a.st.max_rows <= 0)
        return cudaSuccess;
    PagedPass w;
    w.a = a;
    w.p = paged_plan(a, num_sms);
    char *base = static_cast<char *>(ws);
    w.cuts = reinterpret_cast<PagedCut *>(base);
    w.ml = reinterpret_cast<float2 *>(base + w.p.ml_off);
    w.o = reinterpret_cast<float *>(base + w.p.o_off);
    CUtensorMap qm, km, vm;
    if (!px_q_map(&qm, a, w.p) || !px_pool_map(&km, a.c.k, a.c) || !px_pool_map(&vm, a.c.v, a.c))
        return cudaErrorNotSupported;
    if (w.p.pair)
        paged_attn_kernel<true><<<w.p.ctas, PX_THREADS, PX_SMEM, s>>>(qm, km, vm, w);
    else
        paged_attn_kernel<false><<<w.p.ctas, PX_THREADS, PX_SMEM, s>>>(qm, km, vm, w);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || w.p.ctas < 2)
        return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)w.p.ctas - 1, (unsigned)((w.p.cap + PJ_WARPS - 1) / PJ_WARPS));
    cfg.blockDim = dim3(32 * PJ_WARPS);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_join_kernel, w);
}

cudaError_t paged_prepare()
{
    const cudaError_t e = cudaFuncSetAttribute((const void *)paged_attn_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM);
    return e != cudaSuccess ? e
                            : cudaFuncSetAttribute((const void *)paged_attn_kernel<false>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM);
}

} // namespace ylm
