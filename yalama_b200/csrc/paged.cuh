// What the kernels of a step on the paged cache share: which request a row belongs to, whether the request
// can be served, where a slot lies, and how deep a row is in its tree.
//
// The step's arrays are on the device, so that a captured graph serves steps of other lengths; the host cannot
// check them, and every kernel does, by the same rules: a request whose rows or slots do not fit is left out as a
// whole, a page that is not in the pool keeps its slots out, a parent that is no earlier row counts as none. *fault
// collects which of these were met.
#pragma once
#include "ylm_common.cuh"

namespace ylm {

constexpr int PAGED_BAD_REQUEST = 1, PAGED_BAD_PAGE = 2, PAGED_BAD_PARENT = 4, PAGED_BAD_POSITION = 8, PAGED_TIMEOUT = 16;
constexpr int PAGED_TREE = 128; // most rows of a request in a tree

__device__ __forceinline__ void paged_fault(const PagedStep &st, int bit)
{
    if (st.fault)
        atomicOr(st.fault, bit);
}

struct PagedRequest
{
    int row0, t, n; // its rows [row0, row0 + t), and its tokens cached before the step
};

// The request's rows and length; false where it has no rows or is left out (bad: the latter).
__device__ __forceinline__ bool paged_request(const PagedStep &st, int page, int s, PagedRequest &r, bool &bad)
{
    const int a = st.row_start[s], b = st.row_start[s + 1];
    r.row0 = a;
    r.t = b - a;
    r.n = st.length[s];
    bad = false;
    if (a >= 0 && b == a)
        return false;
    bad = a < 0 || b < a || b > st.rows || b - a > st.max_rows || r.n < 0 ||
          (int64_t)r.n + (b - a) > (int64_t)st.table_ld * page;
    return !bad;
}

// Warp-wide: the last request that starts at or before row r, by 32-way search; -1: none. (With a row_start
// that decreases the result is any request; paged_request and the caller's range check decide.)
__device__ __forceinline__ int paged_find(const PagedStep &st, int r, int lane)
{
    int lo = 0, hi = st.n_seq;
    for (;;)
    {
        const int span = (hi - lo + 31) / 32, at = lo + lane * span;
        const int hit = __popc(__ballot_sync(0xffffffffu, at < hi && st.row_start[at] <= r));
        if (hit == 0)
            return -1;
        lo += (hit - 1) * span;
        hi = min(hi, lo + span);
        if (span == 1)
            return lo;
    }
}

// Warp-wide: the request that row r belongs to, and what it has; -1: none, or one that is left out. Up to 32
// requests are looked at in one round of loads.
__device__ __forceinline__ int paged_row(const PagedStep &st, int page, int r, int lane, PagedRequest &q)
{
    bool bad;
    if (st.n_seq <= 32)
    {
        q.row0 = q.t = q.n = 0;
        const bool mine = lane < st.n_seq && paged_request(st, page, lane, q, bad) && r >= q.row0 && r < q.row0 + q.t;
        // (requests that share rows, as none should: the last one)
        const int s = 31 - __clz(__ballot_sync(0xffffffffu, mine));
        q.row0 = __shfl_sync(0xffffffffu, q.row0, max(s, 0));
        q.t = __shfl_sync(0xffffffffu, q.t, max(s, 0));
        q.n = __shfl_sync(0xffffffffu, q.n, max(s, 0));
        return s;
    }
    const int s = paged_find(st, r, lane);
    return s >= 0 && paged_request(st, page, s, q, bad) && r >= q.row0 && r < q.row0 + q.t ? s : -1;
}

// The page of slot j, or -1 where the table names none of the pool.
__device__ __forceinline__ int paged_page(const PagedStep &st, const PagedCache &c, int s, int j)
{
    const int p = st.table[(size_t)s * st.table_ld + (j >> c.page_shift)];
    return p >= 0 && p < c.n_pages ? p : -1;
}

// Halves from the pool's start to slot j of KV head 0 on page p; a head is c.page * 128 halves further.
__device__ __forceinline__ size_t paged_offset(const PagedCache &c, int p, int j)
{
    return ((size_t)p * c.hkv * c.page + (j & (c.page - 1))) * YLM_HEAD_DIM;
}

// A tree's parents, row lane + 32 k in p[k] of each lane, -1 where there is none (before the first row, behind the
// last, and for a parent that is no earlier row; bad: one such).
struct PagedTree
{
    int p[PAGED_TREE / 32];

    __device__ __forceinline__ bool load(const PagedStep &st, const PagedRequest &r, int lane)
    {
        bool bad = false;
#pragma unroll
        for (int k = 0; k < PAGED_TREE / 32; k++)
        {
            const int i = lane + 32 * k;
            p[k] = i < r.t ? st.parent[r.row0 + i] : -1;
            if (p[k] < -1 || p[k] >= i)
            {
                bad = true;
                p[k] = -1;
            }
        }
        return bad;
    }
    // row i's parent; every lane of the warp calls it with the same i >= 0
    __device__ __forceinline__ int of(int i) const
    {
        const int k = i >> 5;
        return __shfl_sync(0xffffffffu, k == 0 ? p[0] : k == 1 ? p[1] : k == 2 ? p[2] : p[3], i & 31);
    }
};
static_assert(PAGED_TREE == 128, "PagedTree::of picks from four words");

} // namespace ylm
