// Attention of a step's rows over the paged cache (device rules: paged.cuh).
//
//   x_rj = q_r . k_j / sqrt(128) for the slots j < n + t of the row's request that row i sees: j < n, and
//          the slots n + d of its ancestors d and of itself (without a tree: d <= i)
//   o_r  = sum_j softmax(x_r)_j v_j,  0 where the row sees no slot
//
// A warp per row and query head, slot by slot.
#include "paged.cuh"

namespace ylm {

constexpr int PT_WARPS = 8;

__global__ void __launch_bounds__(32 * PT_WARPS) paged_attn_rows_kernel(const PagedAttnArgs a)
{
    const int lane = threadIdx.x & 31;
    const PagedStep &st = a.st;
    const int r = blockIdx.x, h = blockIdx.y * PT_WARPS + (threadIdx.x >> 5);
    const int s = paged_find(st, r, lane);
    PagedRequest q;
    bool bad = false;
    if (h >= a.hq || s < 0)
        return;
    const bool is = paged_request(st, a.c.page, s, q, bad);
    if (bad)
        paged_fault(st, PAGED_BAD_REQUEST);
    if (!is || r < q.row0 || r >= q.row0 + q.t)
        return;
    const int i = r - q.row0, g = h / (a.hq / a.c.hkv);
    unsigned see[PAGED_TREE / 32] = {};
    if (st.parent)
    {
        PagedTree tree;
        if (tree.load(st, q, lane))
            paged_fault(st, PAGED_BAD_PARENT);
        for (int p = i; p >= 0; p = tree.of(p))
#pragma unroll
            for (int k = 0; k < PAGED_TREE / 32; k++)
                see[k] |= p >> 5 == k ? 1u << (p & 31) : 0u;
    }
    float x[4], o[4] = {}, m = -INFINITY, z = 0.f;
    {
        const __half2 *src = reinterpret_cast<const __half2 *>(a.q + (int64_t)r * a.q_stride + h * YLM_HEAD_DIM + lane * 4);
        const float2 u = __half22float2(src[0]), v = __half22float2(src[1]);
        x[0] = u.x, x[1] = u.y, x[2] = v.x, x[3] = v.y;
    }
    for (int j = 0; j <= q.n + i; j++)
    {
        const int d = j - q.n;
        if (d >= 0 && st.parent &&
            !((d < 32 ? see[0] : d < 64 ? see[1] : d < 96 ? see[2] : see[3]) >> (d & 31) & 1u))
            continue;
        const int page = paged_page(st, a.c, s, j);
        if (page < 0)
        {
            paged_fault(st, PAGED_BAD_PAGE);
            continue;
        }
        const size_t at = paged_offset(a.c, page, j) + (size_t)g * a.c.page * YLM_HEAD_DIM + lane * 4;
        const __half2 *kp = reinterpret_cast<const __half2 *>(a.c.k + at), *vp = reinterpret_cast<const __half2 *>(a.c.v + at);
        const float2 k0 = __half22float2(kp[0]), k1 = __half22float2(kp[1]);
        const float2 v0 = __half22float2(vp[0]), v1 = __half22float2(vp[1]);
        const float sc = warp_sum(x[0] * k0.x + x[1] * k0.y + x[2] * k1.x + x[3] * k1.y) * 0.08838834764831845f;
        if (sc == -INFINITY) // no weight
            continue;
        const float mn = fmaxf(m, sc), c = m == -INFINITY ? 0.f : expf(m - mn), p = expf(sc - mn);
        z = z * c + p;
        o[0] = o[0] * c + p * v0.x;
        o[1] = o[1] * c + p * v0.y;
        o[2] = o[2] * c + p * v1.x;
        o[3] = o[3] * c + p * v1.y;
        m = mn;
    }
    const float inv = z > 0.f || z != z ? 1.f / z : 0.f;
    __half2 *dst = reinterpret_cast<__half2 *>(a.out + (int64_t)r * a.out_stride + h * YLM_HEAD_DIM + lane * 4);
    dst[0] = __floats2half2_rn(o[0] * inv, o[1] * inv);
    dst[1] = __floats2half2_rn(o[2] * inv, o[3] * inv);
}

size_t paged_attn_workspace(const PagedAttnArgs &, int) { return 0; }

cudaError_t paged_attn_launch(const PagedAttnArgs &a, void *, int, cudaStream_t s)
{
    if (a.st.rows <= 0 || a.st.n_seq <= 0)
        return cudaSuccess;
    paged_attn_rows_kernel<<<dim3((unsigned)a.st.rows, (unsigned)((a.hq + PT_WARPS - 1) / PT_WARPS)), 32 * PT_WARPS, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t paged_prepare() { return cudaSuccess; }

} // namespace ylm
