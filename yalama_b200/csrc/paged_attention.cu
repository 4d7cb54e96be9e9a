// Attention of a step's rows over the paged cache (device rules: paged.cuh).
//
//   x_rj = q_r . k_j / sqrt(128) for the slots j < n + t of the row's request that row i sees: j < n, and
//          the slots n + d of its ancestors d and of itself (without a tree: d <= i)
//   o_r  = sum_j softmax(x_r)_j v_j,  0 where the row sees no slot
//
// An item is a request's KV head and up to tpi of its tokens: their G query heads each are the rows of one or two
// tiles of 128 (row i * G + h). It has a unit for each 128 slots its tokens see. The units of all items, in order, are
// dealt evenly, by what they cost, to one CTA per SM, so that requests of any lengths keep all SMs busy to the end; an item that
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
//
// Measured (B200, 32 / 8 heads but where noted, device time in a captured graph that is repeated without pause, join
// included; the card's power limit lowers the clock of the long cases, which is given with them):
//   one token over 131071 slots: 98 us = 5.4 TB/s at 1540 MHz (95 after a pause). The CTAs end after 74 to 89 us, as HBM
//   serves them.
//   48 requests of 20 to 9000 slots (28 / 4 heads) 37 us, 32 trees of 9 to 45 tokens over 300 to 5000 slots 65 us at 1850 MHz: a
//   unit of one tile takes 2050 cycles, one of two 3870, and an item some 5500 beside its units.
//   a tree of 64 tokens over 8200 slots: 30 us, the attention's CTAs ending after 14 to 20; partial sums of 19 MB are joined.
//   2049 rows behind 6145 slots: 281 us = 857 TFLOP/s at 1740 MHz (263 = 915 after a pause). A stream's unit is 2000 cycles of
//   softmax (a quarter of it maxima) and 1900 of hand-over and products, with the other stream's in between: tensor pipe
//   48 %, exponential unit 47 % of the time.
//   611 slots: 12.2 us, one unit a CTA: in a CTA's 15800 cycles the share takes 4100, the item and its first
//   loads 3500, S 900, the weights 2800, the product 1200, the way out 3200. The rest is the join. That is this kernel's
//   set-up, not the case: the 8-bit cache's attention, a kernel for few rows, takes 5 us for as many slots.
// Tried and slower, the 2049 rows (after a pause): all 128 scores of a row unrolled (380 us, registers spilled), the reference taken from the
// tile before (342, code beyond the instruction cache), two threads a row (271 against 259: an SM quarter's two warps
// share its exponential unit), a quarter or half of the exponentials by polynomial (263 and 281 against 261), units of 64 slots with two S a
// stream (358: twice the commits and waits of the issuing warp).
#include "paged.cuh"
#include "ylm_tc.cuh"
#include <algorithm>

namespace ylm {

constexpr int PX_TILE = 128 * 128 * 2; // a tile of 128 rows or slots: two halves of 64 dimensions
constexpr int PX_THREADS = 384;
constexpr int PX_KST = 3;
constexpr int PX_CONTROL = 3 * 1024; // barriers, the streams' (M, l)
constexpr int PX_SMEM = 7 * PX_TILE + PX_CONTROL;
constexpr int PX_CUT = 128; // bytes of a PagedCut
constexpr float PX_SCALE = (float)(1.4426950408889634 / 11.313708498984760); // log2(e) / sqrt(128)
// FP16 weights end at 2^16; a higher lead keeps more of the small ones and moves the reference more often
constexpr float PX_LEAD = 11.f, PX_MOST = 15.9f;
constexpr float PX_RISE = (PX_MOST - PX_LEAD) / PX_SCALE; // in scores

struct PagedPlan
{
    int G, tpt, tpi; // query heads per KV head, tokens per 128-row tile and per item
    int over_g;      // r / G = r * over_g >> 16 for the rows of a tile (r G < 2^16)
    int pair;        // 1: items of two tiles (some request may have more than tpt rows)
    int box;         // tokens of a tile that are loaded: tpt, or fewer where no request has so many
    int cap;         // most rows of an item
    int item;        // what an item costs beside its units, for the dealing
    int ctas;
    size_t ml_off, o_off, bytes;
};

static PagedPlan paged_plan(const PagedAttnArgs &a, int num_sms)
{
    PagedPlan p;
    p.G = a.hq / a.c.hkv;
    p.tpt = 128 / p.G;
    p.over_g = 65536 / p.G + 1;
    p.pair = a.st.max_rows > p.tpt;
    p.tpi = p.pair ? 2 * p.tpt : p.tpt;
    p.box = std::max(1, std::min(p.tpt, a.st.max_rows));
    p.cap = std::max(1, std::min(p.tpi, a.st.max_rows)) * p.G;
    // An item's first loads and its sums' way out, where a unit of one tile costs 1 and a unit of two tiles 2 (2050 and
    // 3870 cycles). Few rows, with 0, 1, 2, 3, 4: 48 requests of 20 to 9000 slots 57, 47, 41, 39.5, 40 us. More rows, with 3,
    // 4, 5, 6: 32 trees 71, 67, 66, 64 us. All requests alike in rows, with 3, 4, 6: 4 rows an item 64, 61, 66 us (48 requests of 20
    // to 9000 slots) and 64, 66, 70 (100 of 50 to 2000); 64 rows 74, 70, 71 and 73, 72, 75; 180 rows 130, 121, 117 and 125,
    // 118, 116. So the turn belongs between 64 and 180 rows, and 4 would be 1 to 5 % faster from 16 to 64.
    p.item = p.cap <= 32 ? 3 : 6;
    p.ctas = num_sms;
    p.ml_off = (size_t)p.ctas * PX_CUT;
    p.o_off = p.ml_off + ((size_t)p.ctas * 2 * p.cap * sizeof(float2) + 255) / 256 * 256;
    p.bytes = p.o_off + (size_t)p.ctas * 2 * p.cap * YLM_HEAD_DIM * sizeof(float);
    return p;
}

size_t paged_attn_workspace(const PagedAttnArgs &a, int num_sms) { return paged_plan(a, num_sms).bytes; }

// A part of an item, as a share has it.
struct PagedItem
{
    int s, row0, t, n;  // the request
    int first, kvh;     // the item's first token, its KV head
    int tile0, tiles;   // units [tile0, tile0 + tiles) are the share's; tiles = 0: the share's end
    int units;          // units of the item
};

// A CTA's share and its first item; left in the workspace for the join. Places are what the items and units in front of
// them cost together: unit k of an item lies at zero + k * px_cost, and is the share's in which that is.
struct PagedCut
{
    long long each, more; // every share is `each` long, the first `more` of them one more; the rest are empty
    long long left;       // what is behind its part of the first item
    long long zero;       // where the first item's unit 0 lies
    PagedItem it;
    int cut;              // the share starts inside an item
};
static_assert(sizeof(PagedCut) <= PX_CUT, "the workspace's layout");

struct PagedPass
{
    PagedAttnArgs a;
    PagedPlan p;
    PagedCut *cuts;
    float2 *ml; // [cta][2][cap]: (M, l) of the item that the share starts inside of, and of the one it ends inside of
    float4 *o;  // [cta][2][32][cap]: four dimensions of every row after one another
};

// ------------------------------------------------------------------ units
// units of the item with tokens [qp * tpi, ...) of a request: its last token sees slots below n + min(t, ...)
__device__ __forceinline__ int px_units(int n, int t, int qp, int tpi) { return (n + min(t, (qp + 1) * tpi) + 127) >> 7; }

// sum of ceil((n + i * tpi) / 128) over i = 1..k: each is (x + r) / 128 with r = -x mod 128, whose
// values repeat after 128 / g and then are those that are congruent to -n mod g, for g the power of two in tpi
__device__ __noinline__ long long px_before(int n, int k, int tpi)
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

// what a request's items and their units cost in front of token group k, for one KV head: all of its groups are full
__device__ __forceinline__ long long px_front(int n, int k, const PagedPlan &p)
{
    const int cost = p.pair ? 2 : 1;
    return cost * px_before(n, k, p.tpi) + (long long)p.item * k;
}

__device__ __forceinline__ long long px_request_cost(const PagedRequest &r, const PagedPlan &p, int hkv)
{
    const int last = r.t <= p.tpi ? 0 : (r.t - 1) / p.tpi;
    const int cost = r.t - last * p.tpi > p.tpt ? 2 : 1;
    return hkv * (px_front(r.n, last, p) + p.item + cost * px_units(r.n, r.t, last, p.tpi));
}

// slots below are seen by every row of the item
__device__ __forceinline__ int px_open(const PagedPass &w, const PagedItem &it)
{
    return it.n + (w.a.st.parent ? (it.t == 1 ? 1 : 0) : it.first + 1);
}
__device__ __forceinline__ bool px_two(const PagedPass &w, const PagedItem &it) { return it.t - it.first > w.p.tpt; }

__device__ __forceinline__ int px_cost(const PagedPass &w, const PagedItem &it) { return w.p.pair && px_two(w, it) ? 2 : 1; }

// a / b for b > 0; nearly every step's numbers have 32 bits
__device__ __forceinline__ long long px_div(long long a, int b)
{
    return a >> 31 == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// Warp 0's way through the share, an item after another. The next requests, a lane each, are loaded ahead of their turn.
struct PagedWalk
{
    PagedItem it;
    long long left; // what of the share is behind this item
    int base;       // ahead: requests base + lane
    PagedRequest ahead;
    bool there;

    __device__ __forceinline__ void look(const PagedPass &w, int from, int lane)
    {
        base = from;
        bool bad;
        there = from + lane < w.a.st.n_seq && paged_request(w.a.st, w.a.c.page, from + lane, ahead, bad);
    }
    __device__ __forceinline__ void start(const PagedPass &w, const PagedCut &c, int lane)
    {
        left = c.left;
        it = c.it;
        base = -1; // not yet looked ahead
        if (it.tiles == 0)
            next(w, lane);
    }
    __device__ __forceinline__ void next(const PagedPass &w, int lane)
    {
        it.tiles = 0;
        if (left <= 0) // (where the item goes on in the next share, left is below 0)
            return;
        it.tile0 = 0;
        if (++it.kvh == w.a.c.hkv)
        {
            it.kvh = 0;
            it.first += w.p.tpi;
            if (it.first >= it.t)
            {
                it.first = 0;
                unsigned hit;
                if (base < 0)
                    look(w, it.s + 1, lane);
                while (!(hit = __ballot_sync(0xffffffffu, there && base + lane > it.s)))
                {
                    if (base + 32 >= w.a.st.n_seq)
                        return;
                    look(w, base + 32, lane);
                }
                const int k = __ffs(hit) - 1;
                it.s = base + k;
                it.row0 = __shfl_sync(0xffffffffu, ahead.row0, k);
                it.t = __shfl_sync(0xffffffffu, ahead.t, k);
                it.n = __shfl_sync(0xffffffffu, ahead.n, k);
            }
        }
        it.units = (it.n + min(it.t, it.first + w.p.tpi) + 127) >> 7;
        const int cost = px_cost(w, it);
        left -= w.p.item;
        it.tiles = left <= 0 ? 0 : (int)min((long long)it.units, (left + cost - 1) / cost);
        left -= (long long)cost * it.units;
    }
};

// ------------------------------------------------------------------ arithmetic of two values an instruction
__device__ __forceinline__ float2 px_add2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\t"
        "mov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 px_fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, u;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 u, x, y, z;\n\tmov.b64 {%0, %1}, u;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
// Two results to FP16. A row's weights sum to one before they are rounded for the product, after it to 1 + 2^-11 at most:
// a finite result that rounds to infinity is FP16's largest value, where the values that it is made of end; rounded towards
// zero it stops there, and an infinite one stays. (48 requests of 20 to 9000 slots: 0.1 us; clamped in FP32 0.7 us.)
__device__ __forceinline__ __half2 px_result(float x, float y)
{
    const __half2 h = __floats2half2_rn(x, y);
    const uint32_t inf = __heq2_mask(__habs2(h), __half2half2(__ushort_as_half(0x7C00)));
    uint32_t down;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(down) : "f"(y), "f"(x));
    const uint32_t r = (*reinterpret_cast<const uint32_t *>(&h) & ~inf) | (down & inf);
    return *reinterpret_cast<const __half2 *>(&r);
}

// Between lanes 2 i and 2 i + 1: the lower one gets (x, the other's x), the upper one (the other's y, y).
__device__ __forceinline__ void px_trade(uint4 &x, uint4 &y, int lane)
{
    const bool up = lane & 1;
    uint4 give = up ? x : y;
    give.x = __shfl_xor_sync(0xffffffffu, give.x, 1);
    give.y = __shfl_xor_sync(0xffffffffu, give.y, 1);
    give.z = __shfl_xor_sync(0xffffffffu, give.z, 1);
    give.w = __shfl_xor_sync(0xffffffffu, give.w, 1);
    if (up)
        x = give;
    else
        y = give;
}

// ------------------------------------------------------------------ waits
// Bounded: after 2 s, or once another warp gave up, *abort is set and the caller unwinds.
__device__ __forceinline__ bool px_wait(uint64_t *bar, uint32_t parity, volatile int *abort)
{
    for (int i = 0; i < 16; i++)
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

// One lane of a converged warp, the same every time.
__device__ __forceinline__ bool px_elect()
{
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}

__device__ __forceinline__ bool px_stopped(volatile int *abort) { return __any_sync(0xffffffffu, *abort != 0); }

// For copies and products that are on their way and need nobody else: whatever happened, they end first.
__device__ __forceinline__ void px_drain(uint64_t *bar, uint32_t parity)
{
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 <= YLM_WAIT_LIMIT_NS)
        ;
}

__device__ __forceinline__ void tma_load_4d_hint(void *dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z,
                                                 int32_t u, uint64_t *bar, uint64_t policy)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(
                     smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(u), "r"(smem_u32(bar)), "l"(policy)
                 : "memory");
}

// Lane 2 p + h's page of a unit's slots (half h of its dimensions): page p of them; -1 behind the request's last slot,
// and where it is not in the pool (bad).
__device__ __forceinline__ int px_page(const PagedPass &w, const PagedItem &it, int tile, int lane, bool &bad)
{
    const int k = lane >> 1, slot = tile * 128 + k * w.a.c.page;
    bad = false;
    if (k >= 128 >> w.a.c.page_shift || slot >= it.n + it.t)
        return -1;
    const int page = paged_page(w.a.st, w.a.c, it.s, slot);
    bad = page < 0;
    return page;
}

// A unit's K or V into a stage, from the pages that px_page gave (-1: zeros). Warp-wide.
__device__ __forceinline__ void px_load(uint8_t *dst, const CUtensorMap *map, const PagedPass &w, int kvh, int page,
                                        uint64_t *bar, uint64_t policy, int lane)
{
    if (lane == 0)
        mbar_arrive_expect_tx(bar, PX_TILE);
    __syncwarp();
    if (lane >> 1 < 128 >> w.a.c.page_shift)
        tma_load_4d_hint(dst + (lane & 1) * (PX_TILE / 2) + (lane >> 1) * w.a.c.page * 128, map, (lane & 1) * 64, 0, kvh, page,
                         bar, policy);
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
             *v_clean = v_empty + VST, *q_full = v_clean + VST, *q_empty = q_full + 2, *s_full = q_empty + 2,
             *p_most = s_full + 2, *p_full = p_most + 2, *o_done = p_full + 2, *joined = o_done + 2, *parted = joined + 1, *done = parted + 1,
             *item_full = done + 1; // [8]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(control + 320);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(control + 324);
    volatile int *special = reinterpret_cast<volatile int *>(control + 328); // [8]: 1 + the item that had one, by its number mod 8
    PagedCut *mine = reinterpret_cast<PagedCut *>(control + 384);
    long long *sums = reinterpret_cast<long long *>(control + 512);          // [12]
    // Rings of 8: warp 0 is never more than six items or units ahead of any other warp, since a K stage comes free by
    // products that waited for everybody else's work on the items before.
    PagedItem *items = reinterpret_cast<PagedItem *>(control + 640);
    volatile uint32_t *lost = reinterpret_cast<volatile uint32_t *>(control + 960); // a unit's sixteens of slots that are not in the pool
    float2 *state = reinterpret_cast<float2 *>(control + 1024);                     // [2][128]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PagedAttnArgs &a = w.a;
    const PagedStep &st = a.st;

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
        for (int i = 0; i < 2; i++)
        {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_most[i], 4);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(joined, 8);
        mbar_init(parted, 8);
        mbar_init(done, 1);
        *abort_flag = 0;
        for (int i = 0; i < 8; i++)
        {
            mbar_init(&item_full[i], 1);
            special[i] = 0;
        }
        mine->left = 0; // an empty share
        mine->it.tiles = 0;
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

    // (launched as a programmatic dependent: what comes before this grid in the stream may have run until here)
    pdl_wait();
    pdl_launch_dependents(); // the joining CTAs may start; they wait for this grid's end
    // ---- this CTA's share: requests in runs of `run` a thread, their units summed over the threads
    const int run = st.n_seq <= PX_THREADS ? 1 : (st.n_seq + PX_THREADS - 1) / PX_THREADS;
    const int s_end = min(st.n_seq, (tid + 1) * run);
    long long own = 0;
    PagedRequest req; // the run's last (of a run of one: the request)
    for (int s = tid * run; s < s_end; s++)
    {
        bool bad;
        if (paged_request(st, a.c.page, s, req, bad))
            own += px_request_cost(req, w.p, a.c.hkv);
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
    // share b: [b * each + min(b, more), + each + (b < more)); none so short that a unit of two tiles is longer
    const int b = blockIdx.x;
    const int shares = PAIR ? (int)max(1ll, min((long long)gridDim.x, total / 2)) : (int)gridDim.x;
    const long long each = px_div(total, shares), over = total - each * shares;
    const long long u0 = b < shares ? b * each + min((long long)b, over) : total;
    const long long u1 = b < shares ? u0 + each + (b < over) : total;
    if (u0 >= before && u0 < before + own && u1 > u0)
    {
        long long rest = u0 - before;
        int s = tid * run;
        if (run > 1)
            for (;; s++)
            {
                bool bad;
                if (!paged_request(st, a.c.page, s, req, bad))
                    continue;
                const long long u = px_request_cost(req, w.p, a.c.hkv);
                if (rest < u)
                    break;
                rest -= u;
            }
        // the last of the request's token groups whose units before it do not pass `rest`
        int lo = 0, hi = req.t <= w.p.tpi ? 1 : (req.t + w.p.tpi - 1) / w.p.tpi;
        while (hi - lo > 1)
        {
            const int mid = (lo + hi) / 2;
            if (a.c.hkv * px_front(req.n, mid, w.p) <= rest)
                lo = mid;
            else
                hi = mid;
        }
        rest -= a.c.hkv * px_front(req.n, lo, w.p);
        PagedCut c;
        c.each = each;
        c.more = over;
        c.it.s = s;
        c.it.row0 = req.row0;
        c.it.t = req.t;
        c.it.n = req.n;
        c.it.first = lo * w.p.tpi;
        c.it.units = px_units(req.n, req.t, lo, w.p.tpi);
        const int cost = px_cost(w, c.it), all = w.p.item + cost * c.it.units;
        c.it.kvh = (int)px_div(rest, all);
        const int from = (int)(rest - (long long)c.it.kvh * all) - w.p.item; // from unit 0 to the share's start
        const long long to = u1 - u0 + from;
        c.zero = u0 - from;
        c.it.tile0 = from <= 0 ? 0 : (from + cost - 1) / cost;
        c.it.tiles = to <= 0 ? 0 : (int)min((long long)c.it.units, (to + cost - 1) / cost) - c.it.tile0;
        c.left = to - (long long)cost * c.it.units;
        c.cut = c.it.tile0 > 0 && c.it.tiles > 0;
        *mine = c;
        w.cuts[b] = c;
    }
    else if (u0 == u1 && tid == 0)
        w.cuts[b] = PagedCut{};
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int G = w.p.G, tpt = w.p.tpt;
    // item number j, once warp 0 has left it; tiles = 0 after the last, or where a wait ran out
    const auto fetch = [&](int j) {
        PagedItem it;
        if (px_wait(&item_full[j & 7], (j >> 3) & 1, abort_flag))
            it = items[j & 7];
        else
            it.tiles = 0;
        return it;
    };

    // Two places for Q, so that the next item's is there in time: an item of one tile takes the other one than the last
    // item's, an item of two tiles both. With one tile in shared memory the places are its halves of 64 rows,
    // where no item has more (the products read 128 rows from there on, and nobody reads what comes of the others), or one.
    const int q_places = PAIR || w.p.cap <= 64 ? 2 : 1;
    const uint32_t q_step = PAIR ? PX_TILE : PX_TILE / 4;
    // Where every request is one item a KV head, K and V on pages of its own are read once, and the sums should stay in L2
    // instead: 48 requests of 20 to 9000 slots 57.3 us against 63.5 with the normal policy (L2 full of other data before),
    // 32 trees 90 against 94, 131071 slots 115 against 121. Pages that requests share are read by
    // each of them, and leave L2 early for it: 48 requests behind a common prefix of 4096 or 8192 slots 77.5 and 137.2 against
    // 75.8 and 137.0, 64 with 4000 slots of their own behind one of 8192 (1.1 GB) 414 against 391, the most that was met.
    uint64_t policy;
    if (st.max_rows <= w.p.tpi)
        policy = l2_policy_evict_first();
    else
        asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));

    if (warp == 0)
    {
        // ---- the share's items, and K tiles
        PagedWalk walk;
        walk.start(w, *mine, lane);
        int kc = 0;
        for (int j = 0;; j++)
        {
            if (lane == 0)
            {
                items[j & 7] = walk.it;
                mbar_arrive(&item_full[j & 7]);
            }
            const PagedItem it = walk.it;
            bool bad, ok = true;
            int page = it.tiles ? px_page(w, it, it.tile0, lane, bad) : -1;
            for (int t = 0; t < it.tiles; t++, kc++)
            {
                const int s = kc % KST;
                if (px_stopped(abort_flag) || (kc >= KST && !px_wait_warp(&k_empty[s], (kc / KST - 1) & 1, abort_flag)))
                {
                    ok = false;
                    break;
                }
                // a page covers page / 16 sixteens
                const uint32_t bits = bad ? (0xFFu >> (8 - (a.c.page >> 4))) << ((lane >> 1) * (a.c.page >> 4)) : 0u;
                const uint32_t all = __reduce_or_sync(0xffffffffu, bits);
                if (lane == 0)
                {
                    lost[kc & 7] = all;
                    if (all)
                        paged_fault(st, PAGED_BAD_PAGE);
                }
                px_load(sk + s * PX_TILE, &kmap, w, it.kvh, page, &k_full[s], policy, lane);
                page = px_page(w, it, it.tile0 + t + 1, lane, bad); // on its way while the next stage comes free
                if (walk.base < 0)
                    walk.look(w, it.s + 1, lane);
            }
            if (!ok || it.tiles == 0)
                break;
            walk.next(w, lane);
        }
        // every copy has landed before the CTA can end
        for (int j = max(0, kc - KST); j < kc; j++)
            px_drain(&k_full[j % KST], (j / KST) & 1);
    }
    else if (warp == 2)
    {
        // ---- the items' Q, and V tiles
        int vc = 0, place = 0, used[2] = {0, 0}; // the next item's place for Q; items that had each
        bool ok = true;
        for (int j = 0; ok; j++)
        {
            const PagedItem it = fetch(j);
            if (!__all_sync(0xffffffffu, it.tiles != 0) || px_stopped(abort_flag))
                break;
            const bool two = PAIR && px_two(w, it);
            if (two)
                place = 0;
#pragma unroll
            for (int i = 0; i < 2; i++)
                if ((two || i == place) && ok)
                {
                    if (used[i] && !px_wait_warp(&q_empty[i], (used[i] - 1) & 1, abort_flag))
                        ok = false;
                    else
                    {
                        if (lane == 0)
                        {
                            const int row = it.row0 + it.first + (two ? i * tpt : 0);
                            uint8_t *dst = sq + i * q_step;
                            mbar_arrive_expect_tx(&q_full[i], (uint32_t)(w.p.box * G * 256));
                            tma_load_3d(dst, &qmap, 0, it.kvh * G, row, &q_full[i]);
                            tma_load_3d(dst + PX_TILE / 2, &qmap, 64, it.kvh * G, row, &q_full[i]);
                        }
                        used[i]++;
                    }
                }
            if (!ok)
                break;
            place = two ? 0 : q_places == 2 ? place ^ 1 : 0;
            __syncwarp();
            bool bad;
            int page = px_page(w, it, it.tile0, lane, bad);
            for (int t = 0; t < it.tiles; t++, vc++)
            {
                const int s = vc % VST;
                if (px_stopped(abort_flag) || (vc >= VST && !px_wait_warp(&v_empty[s], (vc / VST - 1) & 1, abort_flag)))
                {
                    ok = false;
                    break;
                }
                px_load(sv + s * PX_TILE, &vmap, w, it.kvh, page, &v_full[s], policy, lane);
                page = px_page(w, it, it.tile0 + t + 1, lane, bad);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (used[i])
                px_drain(&q_full[i], (used[i] - 1) & 1);
        for (int i = max(0, vc - VST); i < vc; i++)
            px_drain(&v_full[i % VST], (i / VST) & 1);
    }
    else if (warp == 3)
    {
        // ---- V without what is not finite in slots that some row does not see
        int vc = 0;
        bool ok = true;
        for (int j = 0; ok; j++)
        {
            const PagedItem it = fetch(j);
            if (!__all_sync(0xffffffffu, it.tiles != 0))
                break;
            for (int t = 0; t < it.tiles; t++, vc++)
            {
                const int s = vc % VST, k0 = (it.tile0 + t) * 128, n = it.n + it.t;
                if (!px_wait_warp(&v_full[s], (vc / VST) & 1, abort_flag))
                {
                    ok = false;
                    break;
                }
                // (pages behind the last slot's are zeros)
                const int lo = max(0, px_open(w, it) - k0), hi = min(128, ((n + a.c.page - 1) & -a.c.page) - k0);
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
                        special[j & 7] = j + 1;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if (lane == 0)
                    mbar_arrive(&v_clean[s]);
            }
        }
    }
    else if (warp == 1)
    {
        // ---- the products: every lane walks along, one issues
        const uint32_t idesc_s = tc_idesc(128, 128);
        const uint32_t idesc_o = tc_idesc(128, 128) | (1u << 16); // B (V) MN-major
        const uint64_t dq = smem_desc_k128(smem_u32(sq)), dk = smem_desc_k128(smem_u32(sk)),
                       dv = smem_desc_mn128(smem_u32(sv), PX_TILE / 2, 1024);
        int ks = 0, kp = 0, vs = 0, vp = 0, place = 0; // stages and their phases, the item's place for Q
        uint32_t pp = 0, qp = 0; // bit s: the phase of p_full[s] and of q_full[s]
        bool ok = true;
        for (int j = 0; ok; j++)
        {
            const PagedItem it = fetch(j);
            if (!__all_sync(0xffffffffu, it.tiles != 0))
                break;
            const bool two = PAIR && px_two(w, it);
            const int tasks = two ? 2 * it.tiles : it.tiles;
            if (two)
                place = 0;
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (two || i == place)
                {
                    ok = ok && px_wait_warp(&q_full[i], qp >> i & 1, abort_flag);
                    qp ^= 1u << i;
                }
            // Task i: stream i & 1 on unit i (two streams of one tile), or on unit i / 2 (a tile each). S of a stream's next
            // task follows O += P V of this one, which reads P where that S goes.
            for (int i = -2; i < tasks; i++)
            {
                const int s = i & 1;
                if (i >= 0)
                {
                    // the first three quarters of the slots while the softmax has the last one in work
                    if (!px_wait_warp(&v_clean[vs], vp, abort_flag) || !px_wait_warp(&p_most[s], pp >> s & 1, abort_flag))
                    {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const bool last = !two || s;
                    const uint64_t v0 = dv + (uint32_t)vs * (PX_TILE >> 4);
                    if (px_elect())
                    {
#pragma unroll
                        for (int kk = 0; kk < 6; kk++)
                            tc_mma_ts(tmem + 256u + 128u * s, tmem + 128u * s + 8u * kk, v0 + kk * (2048 >> 4), idesc_o,
                                      (i > 1 || kk) ? 1u : 0u);
                    }
                    __syncwarp();
                    if (!px_wait_warp(&p_full[s], pp >> s & 1, abort_flag))
                    {
                        ok = false;
                        break;
                    }
                    pp ^= 1u << s;
                    tc_fence_after();
                    if (px_elect())
                    {
#pragma unroll
                        for (int kk = 6; kk < 8; kk++)
                            tc_mma_ts(tmem + 256u + 128u * s, tmem + 128u * s + 8u * kk, v0 + kk * (2048 >> 4), idesc_o, 1u);
                        tc_commit(&o_done[s]);
                        if (last)
                            tc_commit(&v_empty[vs]);
                    }
                    __syncwarp();
                    if (last && ++vs == VST)
                    {
                        vs = 0;
                        vp ^= 1;
                    }
                }
                if (i + 2 >= tasks)
                    continue;
                if (!px_wait_warp(&k_full[ks], kp, abort_flag))
                {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const bool last = !two || s; // of the unit
                if (px_elect())
                {
                    const uint64_t q0 = dq + (uint32_t)(two ? s : place) * (q_step >> 4), k0 = dk + (uint32_t)ks * (PX_TILE >> 4);
#pragma unroll
                    for (int kk = 0; kk < 8; kk++)
                    {
                        const uint32_t off = (uint32_t)((kk >> 2) * (PX_TILE / 2) + (kk & 3) * 32) >> 4;
                        tc_mma(tmem + 128u * s, q0 + off, k0 + off, idesc_s, kk ? 1u : 0u);
                    }
                    tc_commit(&s_full[s]);
                    if (last)
                        tc_commit(&k_empty[ks]);
                    if (two ? i >= tasks - 4 : i == tasks - 3)
                        tc_commit(&q_empty[two ? s : place]);
                }
                if (last && ++ks == KST)
                {
                    ks = 0;
                    kp ^= 1;
                }
            }
            place = two ? 0 : q_places == 2 ? place ^ 1 : 0;
        }
        if (!ok)
            *abort_flag = 1;
        // all products are complete before TMEM is given back
        if (px_elect())
            tc_commit(done);
        px_drain(done, 0);
        __syncwarp();
    }
    else
    {
        // ---- softmax: stream ws, row `row` of its tile
        const int ws = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16), tS = trow + 128u * ws, tO = trow + 256u;
        uint32_t nt = 0; // bit s: whether stream s has had an odd number of tasks
        int meets = 0, kc = 0;
        bool ok = true;
        for (int j = 0; ok; j++)
        {
            const PagedItem it = fetch(j);
            if (!__all_sync(0xffffffffu, it.tiles != 0))
                break;
            const bool two = PAIR && px_two(w, it);
            const int n = it.n, t = it.t;
            const int tok0 = it.first + (two ? ws * tpt : 0); // first token of this stream's tile
            const int rows = min(tpt, t - tok0) * G;          // rows of the tile
            const int mine_t = two ? it.tiles : (it.tiles + 1 - ws) >> 1;
            const int i = tok0 + (row * w.p.over_g >> 16); // this row's token (one of the request's where row < rows)
            const bool works = quad * 32 < rows;
            const int clear = px_open(w, it);
            uint32_t anc[4] = {0, 0, 0, 0};
            if (st.parent && works)
            {
                PagedTree tree;
                if (tree.load(st, PagedRequest{it.row0, t, n}, lane))
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
                const int unit = two ? u : 2 * u + ws, k0 = (it.tile0 + unit) * 128;
                // (the product before this one is complete, too, long since: nobody falls two phases of o_done behind,
                // where a parity would say nothing)
                if (!px_wait_warp(&s_full[ws], nt >> ws & 1, abort_flag) ||
                    (u && !px_wait_warp(&o_done[ws], ~nt >> ws & 1, abort_flag)))
                {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (works)
                {
                    const uint32_t bad = lost[(kc + unit) & 7];
                    if (__builtin_expect(bad || k0 + 128 > clear, 0))
                    {
                        // scores of hidden slots become -inf
#pragma unroll 1
                        for (int c = 0; c < 4; c++)
                        {
                            uint32_t bits = seen(k0 + 32 * c);
                            if (bad >> (2 * c) & 1u)
                                bits &= 0xFFFF0000u;
                            if (bad >> (2 * c) & 2u)
                                bits &= 0x0000FFFFu;
                            float v[32];
                            tmem_ld32(tS + 32u * c, v);
#pragma unroll
                            for (int e = 0; e < 32; e++)
                                v[e] = bits >> e & 1u ? v[e] : -INFINITY;
                            tmem_st32(tS + 32u * c, v);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                    float mx;
                    {
                        float v[128];
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            tmem_ld32_async(tS + 32u * c, v + 32 * c);
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            tmem_wait_ld32(v + 32 * c);
                        float most[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                        for (int e = 4; e < 128; e++)
                            most[e & 3] = fmaxf(most[e & 3], v[e]);
                        mx = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
                    }
                    if (u == 0)
                        mr = mx;
                    // (by the difference, which is exact for scores so near: mr + PX_RISE could round past the next score)
                    else if (__builtin_expect(__any_sync(0xffffffffu, mx - mr > PX_RISE), 0))
                    {
                        // the sums so far in units of the new reference
                        float f = 1.f;
                        if (mx - mr > PX_RISE)
                        {
                            f = ex2_ftz((mr - mx) * PX_SCALE);
                            mr = mx;
                        }
                        l *= f;
#pragma unroll 1
                        for (int c = 0; c < 8; c++)
                        {
                            float y[16];
                            tmem_ld16(tO + 128u * ws + 16u * c, y);
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                y[e] *= f;
                            tmem_st16(tO + 128u * ws + 16u * c, y);
                        }
                    }
                    // The weights. A loop whose code stays in the instruction cache: unrolled over all 128
                    // scores it took half as long again.
                    const float ref = mr == -INFINITY ? 0.f : mr; // nothing seen: every weight 0
                    const float2 less = make_float2(-ref, -ref), scale = make_float2(PX_SCALE, PX_SCALE),
                                 lead = make_float2(PX_LEAD, PX_LEAD);
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    const auto weights = [&](const float(&v)[32], uint32_t at) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2)
                        {
                            float2 x = px_fma2(px_add2(make_float2(v[e], v[e + 1]), less), scale, lead);
                            x = make_float2(ex2_ftz(x.x), ex2_ftz(x.y));
                            sum[e >> 1 & 1] = px_add2(sum[e >> 1 & 1], x);
                            const __half2 p = __floats2half2_rn(x.x, x.y);
                            pk[e >> 1] = *reinterpret_cast<const uint32_t *>(&p);
                        }
                        tmem_st16(at, reinterpret_cast<const float *>(pk));
                    };
                    // (32 weights take the place of 16 scores: those are always read by then)
                    float v0[32], v1[32];
                    tmem_ld32_async(tS, v0);
#pragma unroll 1
                    for (int c = 0; c < 4; c += 2)
                    {
                        tmem_wait_ld32(v0);
                        tmem_ld32_async(tS + 32u * (c + 1), v1);
                        weights(v0, tS + 16u * c);
                        if (c == 2)
                        {
                            // all but the last 32 are there
                            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0)
                                mbar_arrive(&p_most[ws]);
                        }
                        tmem_wait_ld32(v1);
                        if (c == 0)
                            tmem_ld32_async(tS + 64u, v0);
                        weights(v1, tS + 16u * (c + 1));
                    }
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0)
                {
                    if (!works)
                        mbar_arrive(&p_most[ws]);
                    mbar_arrive(&p_full[ws]);
                }
                nt ^= 1u << ws;
            }
            nt ^= (uint32_t)((two ? it.tiles : (it.tiles + ws) >> 1) & 1) << (ws ^ 1);
            kc += it.tiles;
            if (!ok)
                break;
            // ---- the item's rows: whole, or this share's part
            const bool whole = it.tiles == it.units;
            const int slot = it.tile0 ? 0 : 1;
            const int rho = (two ? ws * tpt * G : 0) + row; // the row's number in the item
            float M = mr, L = l, f0 = ws ? 0.f : 1.f, f1 = ws ? 1.f : 0.f;
            int c0 = 0, c1 = 8; // this thread's share of the dimensions, 16 each
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
                c0 = 4 * ws;
                c1 = c0 + 4;
            }
            // every product of the item is in the sums
            bool in = true;
#pragma unroll
            for (int s = 0; s < 2; s++)
                if (!two || s == ws)
                    in = in && px_wait_warp(&o_done[s], ~nt >> s & 1, abort_flag); // (before its first task: at once)
            if (!in)
            {
                ok = false;
                break;
            }
            tc_fence_after();
            if (works)
            {
                const bool both = !two && it.tiles > 1; // stream 1 of a single unit has no sums
                const bool odd = special[j & 7] == j + 1;
                const float inv = M == -INFINITY ? 0.f : 1.f / L;
                int64_t to[2]; // where the two rows start whose pieces this lane stores
#pragma unroll
                for (int e = 0; e < 2; e++)
                {
                    const int r = quad * 32 + (lane & ~1) + e, token = r * w.p.over_g >> 16;
                    to[e] = r < rows ? (int64_t)(it.row0 + tok0 + token) * a.out_stride + (it.kvh * G + r - token * G) * YLM_HEAD_DIM : -1;
                }
#pragma unroll 1
                for (int c = c0; c < c1; c++) // 16 dimensions
                {
                    __syncwarp();
                    float v[16], y[16];
                    tmem_ld16_async(tO + (two ? 128u * ws : 0u) + 16u * c, v);
                    if (both)
                        tmem_ld16_async(tO + 128u + 16u * c, y);
                    tmem_wait_ld16(v);
                    if (!two)
                    {
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            v[e] *= f0;
                        if (both)
                        {
                            tmem_wait_ld16(y);
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                v[e] = fmaf(y[e], f1, v[e]); // (a sum that is not finite stays in, whatever its factor)
                        }
                    }
                    if (__builtin_expect(odd && row < rows, 0))
                    {
                        // what was taken out of the values that this row sees
                        const int lo = max(clear, it.tile0 * 128), hi = min(n + t, (it.tile0 + it.tiles) * 128);
#pragma unroll 1
                        for (int k = lo; k < hi; k++)
                        {
                            const int page = seen(k) & 1u ? paged_page(st, a.c, it.s, k) : -1;
                            if (page < 0)
                                continue;
                            const __half *src = a.c.v + paged_offset(a.c, page, k) +
                                                (size_t)it.kvh * a.c.page * YLM_HEAD_DIM + 16 * c;
#pragma unroll
                            for (int e = 0; e < 16; e++)
                            {
                                const float x = h2f(src[e]);
                                v[e] += x - x != 0.f ? x : 0.f; // (x - x is NaN)
                            }
                        }
                    }
                    if (whole)
                    {
                        // a row's 16 values are two 16-byte pieces; two lanes trade theirs, so that each stores its piece of
                        // two rows and a store covers whole sectors
                        uint4 x[2];
#pragma unroll
                        for (int e = 0; e < 2; e++)
                        {
                            __half2 h[4];
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                h[k] = px_result(v[8 * e + 2 * k] * inv, v[8 * e + 2 * k + 1] * inv);
                            x[e] = *reinterpret_cast<const uint4 *>(h);
                        }
                        px_trade(x[0], x[1], lane);
#pragma unroll
                        for (int e = 0; e < 2; e++)
                            if (to[e] >= 0)
                                *reinterpret_cast<uint4 *>(a.out + to[e] + 16 * c + 8 * (lane & 1)) = x[e];
                    }
                    else if (row < rows)
                    {
                        float4 *dst = w.o + (((size_t)blockIdx.x * 2 + slot) * 32 + 4 * c) * w.p.cap + rho;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            dst[(size_t)e * w.p.cap] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
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
// A task is 32 rows (fewer where items have fewer: then the lanes' upper bits count parts), a row a lane, by PER times 32
// dimensions, four a warp at a time. An item of few parts has tasks of 128 dimensions, one of many parts of 32, so that
// about as many loads are under way. CTA x is at the border between shares x and x + 1; the CTAs at the borders inside
// an item share its tasks. Launched as a programmatic dependent.
constexpr int PJ_WARPS = 8, PJ_ROWS = 32;
constexpr int PJ_FEW = 4; // parts

template <int PER, int BATCH>
__device__ __forceinline__ void px_join(const PagedPass &w, const PagedItem &it, int first, int parts, int rows, int task,
                                        int rows_log, __half (*tile)[YLM_HEAD_DIM + 8])
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = lane & ((1 << rows_log) - 1), group = lane >> rows_log, groups = 32 >> rows_log;
    const int row0 = task / (4 / PER) * PJ_ROWS, d0 = task % (4 / PER) * 32;
    const int in = min(row0 + row, rows - 1); // (lanes without a row read another one's)
    // part 0 is share `first`'s end, part k the start of share first + k
    const auto at = [&](int k) { return (size_t)(first + k) * 2 + (k == 0); };
    float M = -INFINITY, L = 0.f;
    float4 o[PER];
#pragma unroll
    for (int d = 0; d < PER; d++)
        o[d] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = group; k0 < parts; k0 += groups * BATCH)
    {
        float2 ml[BATCH];
        float4 x[BATCH][PER];
#pragma unroll
        for (int i = 0; i < BATCH; i++)
        {
            ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int d = 0; d < PER; d++)
                x[i][d] = make_float4(0.f, 0.f, 0.f, 0.f);
            const int k = k0 + i * groups;
            if (k < parts)
            {
                ml[i] = w.ml[at(k) * w.p.cap + in];
#pragma unroll
                for (int d = 0; d < PER; d++)
                    x[i][d] = w.o[(at(k) * 32 + d0 / 4 + warp + PJ_WARPS * d) * w.p.cap + in];
            }
        }
        float m = M;
#pragma unroll
        for (int i = 0; i < BATCH; i++)
            m = fmaxf(m, ml[i].x);
        float f = M == -INFINITY ? 0.f : ex2_ftz((M - m) * PX_SCALE);
        M = m;
        L *= f;
#pragma unroll
        for (int d = 0; d < PER; d++)
            o[d] = make_float4(o[d].x * f, o[d].y * f, o[d].z * f, o[d].w * f);
#pragma unroll
        for (int i = 0; i < BATCH; i++)
        {
            // (a part without a score above -inf counts nothing, but one that is NaN, or has such values, stays)
            f = ml[i].x == -INFINITY ? 0.f : ex2_ftz((ml[i].x - M) * PX_SCALE);
            L += ml[i].y * f;
#pragma unroll
            for (int d = 0; d < PER; d++)
            {
                o[d].x += x[i][d].x * f;
                o[d].y += x[i][d].y * f;
                o[d].z += x[i][d].z * f;
                o[d].w += x[i][d].w * f;
            }
        }
    }
    for (int s = 1 << rows_log; s < 32; s <<= 1)
    {
        const float m = __shfl_xor_sync(0xffffffffu, M, s), top = fmaxf(M, m);
        const float f = M == -INFINITY ? 0.f : ex2_ftz((M - top) * PX_SCALE);
        const float g = m == -INFINITY ? 0.f : ex2_ftz((m - top) * PX_SCALE);
        M = top;
        L = L * f + __shfl_xor_sync(0xffffffffu, L, s) * g;
#pragma unroll
        for (int d = 0; d < PER; d++)
        {
            o[d].x = o[d].x * f + __shfl_xor_sync(0xffffffffu, o[d].x, s) * g;
            o[d].y = o[d].y * f + __shfl_xor_sync(0xffffffffu, o[d].y, s) * g;
            o[d].z = o[d].z * f + __shfl_xor_sync(0xffffffffu, o[d].z, s) * g;
            o[d].w = o[d].w * f + __shfl_xor_sync(0xffffffffu, o[d].w, s) * g;
        }
    }
    const float inv = M == -INFINITY ? 0.f : 1.f / L;
    if (group == 0)
#pragma unroll
        for (int d = 0; d < PER; d++)
        {
            const __half2 h[2] = {px_result(o[d].x * inv, o[d].y * inv), px_result(o[d].z * inv, o[d].w * inv)};
            *reinterpret_cast<uint2 *>(&tile[row][4 * (warp + PJ_WARPS * d)]) = *reinterpret_cast<const uint2 *>(h);
        }
    __syncthreads();
    // 4 PER lanes a row
    const int G = w.p.G;
    for (int i = threadIdx.x; i < min(1 << rows_log, rows - row0) * 4 * PER; i += 32 * PJ_WARPS)
    {
        const int r = i / (4 * PER), p = i % (4 * PER), y = row0 + r;
        *reinterpret_cast<uint4 *>(w.a.out + (int64_t)(it.row0 + it.first + y / G) * w.a.out_stride +
                                   (it.kvh * G + y % G) * YLM_HEAD_DIM + d0 + p * 8) =
            *reinterpret_cast<const uint4 *>(&tile[r][p * 8]);
    }
    __syncthreads();
}

__global__ void __launch_bounds__(32 * PJ_WARPS) paged_join_kernel(const __grid_constant__ PagedPass w, const int rows_log)
{
    __shared__ __align__(16) __half tile[PJ_ROWS][YLM_HEAD_DIM + 8];
    const int b = blockIdx.x + 1;
    pdl_wait();
    pdl_launch_dependents(); // a next call's CTAs may set themselves up beside these
    const PagedCut &c = w.cuts[b];
    const long long each = c.each, more = c.more;
    const PagedItem it = c.it;
    if (!c.cut)
        return;
    // the shares with the item's first and last units
    const auto share = [&](long long u) {
        const long long big = more * (each + 1);
        return (int)(u < big ? px_div(u, (int)(each + 1)) : more + px_div(u - big, (int)each));
    };
    const int first = share(c.zero), parts = share(c.zero + (long long)px_cost(w, it) * (it.units - 1)) - first + 1;
    const int rows = min(w.p.tpi, it.t - it.first) * w.p.G, blocks = (rows + PJ_ROWS - 1) / PJ_ROWS;
    const int mine = b - first - 1 + (parts - 1) * blockIdx.y, step = (parts - 1) * gridDim.y;
    if (parts <= PJ_FEW)
        for (int task = mine; task < blocks; task += step)
            px_join<4, 2>(w, it, first, parts, rows, task, rows_log, tile);
    else
        for (int task = mine; task < 4 * blocks; task += step)
            px_join<1, 8>(w, it, first, parts, rows, task, rows_log, tile);
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

// Q as [rows][hq][128], the G heads of a tile's tokens and half of their dimensions a box: rows i * G + h of a tile.
static bool px_q_map(CUtensorMap *map, const PagedAttnArgs &a, const PagedPlan &p)
{
    auto enc = encoder();
    if (!enc)
        return false;
    cuuint64_t dims[3] = {128, (cuuint64_t)a.hq, (cuuint64_t)a.st.rows};
    cuuint64_t strides[2] = {256, (cuuint64_t)a.q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)p.G, (cuuint32_t)p.box}, estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half *>(a.q), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t paged_attn_launch(const PagedAttnArgs &a, void *ws, int num_sms, cudaStream_t s)
{
    if (a.st.rows <= 0 || a.st.n_seq <= 0)
        return cudaSuccess;
    PagedPass w;
    w.a = a;
    w.p = paged_plan(a, num_sms);
    char *base = static_cast<char *>(ws);
    w.cuts = reinterpret_cast<PagedCut *>(base);
    w.ml = reinterpret_cast<float2 *>(base + w.p.ml_off);
    w.o = reinterpret_cast<float4 *>(base + w.p.o_off);
    CUtensorMap qm, km, vm;
    if (!px_q_map(&qm, a, w.p) || !px_pool_map(&km, a.c.k, a.c) || !px_pool_map(&vm, a.c.v, a.c))
        return cudaErrorNotSupported;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)w.p.ctas);
    cfg.blockDim = dim3(PX_THREADS);
    cfg.dynamicSmemBytes = PX_SMEM;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = w.p.pair ? cudaLaunchKernelEx(&cfg, paged_attn_kernel<true>, qm, km, vm, w)
                                   : cudaLaunchKernelEx(&cfg, paged_attn_kernel<false>, qm, km, vm, w);
    if (e != cudaSuccess || w.p.ctas < 2)
        return e;
    int rows_log = 0;
    while (1 << rows_log < std::min(w.p.cap, PJ_ROWS))
        rows_log++;
    // (a task of an item of few parts a CTA; 8 a border at most)
    cfg.gridDim = dim3((unsigned)w.p.ctas - 1, (unsigned)((w.p.cap + PJ_ROWS - 1) / PJ_ROWS));
    cfg.blockDim = dim3(32 * PJ_WARPS);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, paged_join_kernel, w, rows_log);
}

cudaError_t paged_prepare()
{
    const cudaError_t e = cudaFuncSetAttribute((const void *)paged_attn_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM);
    return e != cudaSuccess ? e
                            : cudaFuncSetAttribute((const void *)paged_attn_kernel<false>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM);
}

} // namespace ylm
