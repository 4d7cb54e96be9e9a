// Paged K/V cache of several requests: a step's rows appended (with q/k-norm and rotation on the way), and its
// drafted tokens accepted (their keys and values moved to consecutive slots). Device rules: paged.cuh.
#include "paged.cuh"
#include <algorithm>

namespace ylm {

// Launched as programmatic dependents: they wait for what comes before them in the stream first thing.
template <typename A>
static cudaError_t paged_launch(void (*kernel)(const A), dim3 grid, int threads, cudaStream_t s, const A &a)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// ------------------------------------------------------------------ append
//   x' = x * rsqrt(mean(x^2) + eps) * w   (where there is a norm)
//   y_d = x'_d cos_d - x'_{d+64} sin_d,  y_{d+64} = x'_{d+64} cos_d + x'_d sin_d   for d < 64
// in FP32, rounded to FP16 once.
constexpr int PA_THREADS = 128;
constexpr int PA_HEADS = PA_THREADS / 8; // a pass: 8 lanes a head, 8 dimensions d and their partners d + 64 each

// A CTA takes every gridDim.y-th pass of one row; the loads of BATCH passes are under way while the request is looked up.
// With a dimension and its partner in one lane the rotation needs no exchange. Bound by HBM behind the lookup's chain of
// loads, which eight CTAs an SM cover: 4522 rows of 80 heads 33.9 us = 5.5 TB/s (256 threads, four CTAs an SM 37.6 us; five
// passes at a time, and fewer CTAs, 36 to 41 us; 16 lanes a head, with shuffles for the partners, 41 us). The price of
// eight CTAs is 64 registers a thread: of the three passes' state 84 bytes are spilled and 160 loaded back (of two 24 and
// 24). One row of 48 heads 2.1 us: the chain's latency.
template <int BATCH>
__global__ void __launch_bounds__(PA_THREADS, 8) paged_append_kernel(const __grid_constant__ PagedAppendArgs a)
{
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, l = threadIdx.x & 7, at_head = threadIdx.x >> 3;
    const int r = blockIdx.x, heads = a.hq + 2 * a.c.hkv;
    const PagedStep &st = a.st;
    uint4 w[BATCH][2];
    // head h of the row: query heads, then keys, then values
    const auto load = [&](int h, uint4(&x)[2]) {
        const __half *src = h < a.hq             ? a.q + (int64_t)r * a.q_stride + h * YLM_HEAD_DIM
                            : h < a.hq + a.c.hkv ? a.k + (int64_t)r * a.k_stride + (h - a.hq) * YLM_HEAD_DIM
                                                 : a.v + (int64_t)r * a.v_stride + (h - a.hq - a.c.hkv) * YLM_HEAD_DIM;
        x[0] = x[1] = make_uint4(0, 0, 0, 0);
        if (h < heads)
        {
            x[0] = *reinterpret_cast<const uint4 *>(src + l * 8);
            x[1] = *reinterpret_cast<const uint4 *>(src + 64 + l * 8);
        }
    };
#pragma unroll
    for (int k = 0; k < BATCH; k++)
        load((blockIdx.y + k * gridDim.y) * PA_HEADS + at_head, w[k]);

    if (st.fault && blockIdx.y == 0)
        for (int64_t s = (int64_t)r * PA_THREADS + threadIdx.x; s < st.n_seq; s += (int64_t)gridDim.x * PA_THREADS)
        {
            PagedRequest q;
            bool bad;
            paged_request(st, a.c.page, (int)s, q, bad);
            if (bad)
                paged_fault(st, PAGED_BAD_REQUEST);
        }
    PagedRequest q;
    const int s = paged_row(st, a.c.page, r, lane, q);
    if (s < 0)
        return;
    const int i = r - q.row0, slot = q.n + i;
    int pos = slot;
    if (st.parent)
    {
        PagedTree tree;
        if (tree.load(st, q, lane))
            paged_fault(st, PAGED_BAD_PARENT);
        pos = q.n;
        for (int p = tree.of(i); p >= 0; p = tree.of(p))
            pos++;
    }
    if (a.rope_cos && pos >= a.max_pos)
    {
        paged_fault(st, PAGED_BAD_POSITION);
        return;
    }
    const int page = paged_page(st, a.c, s, slot);
    if (page < 0)
        paged_fault(st, PAGED_BAD_PAGE);
    const size_t at = page < 0 ? 0 : paged_offset(a.c, page, slot);
    uint4 cw = make_uint4(0, 0, 0, 0), sw = cw;
    if (a.rope_cos)
    {
        const int64_t t = (int64_t)pos * 64 + l * 8;
        cw = *reinterpret_cast<const uint4 *>(a.rope_cos + t);
        sw = *reinterpret_cast<const uint4 *>(a.rope_sin + t);
    }
    for (int p0 = blockIdx.y; p0 * PA_HEADS < heads; p0 += BATCH * gridDim.y)
    {
        if (p0 != blockIdx.y)
#pragma unroll
            for (int k = 0; k < BATCH; k++)
                load((p0 + k * gridDim.y) * PA_HEADS + at_head, w[k]);
#pragma unroll
        for (int k = 0; k < BATCH; k++)
        {
            const int h = (p0 + k * gridDim.y) * PA_HEADS + at_head;
            const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.c.hkv;
            const __half *norm = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
            const bool turn = a.rope_cos && (is_q || is_k);
            // (every lane takes part in the shuffles, whatever its head is)
            const bool any_norm = __any_sync(0xffffffffu, norm != nullptr);
            if (any_norm || turn)
            {
                float x[8], y[8];
                unpack8(w[k][0], x);
                unpack8(w[k][1], y);
                if (any_norm)
                {
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
                    for (int o = 4; o > 0; o >>= 1)
                        ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    if (norm)
                    {
                        float nx[8], ny[8];
                        unpack8(*reinterpret_cast<const uint4 *>(norm + l * 8), nx);
                        unpack8(*reinterpret_cast<const uint4 *>(norm + 64 + l * 8), ny);
                        const float d = rsqrtf(ss * (1.0f / YLM_HEAD_DIM) + a.eps);
#pragma unroll
                        for (int e = 0; e < 8; e++)
                        {
                            x[e] = x[e] * d * nx[e];
                            y[e] = y[e] * d * ny[e];
                        }
                    }
                }
                if (turn)
                {
                    float c[8], sn[8];
                    unpack8(cw, c);
                    unpack8(sw, sn);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                    {
                        const float u = x[e];
                        x[e] = fmaf(u, c[e], -y[e] * sn[e]);
                        y[e] = fmaf(y[e], c[e], u * sn[e]);
                    }
                }
                if (norm || turn)
                {
                    __half2 *ox = reinterpret_cast<__half2 *>(&w[k][0]), *oy = reinterpret_cast<__half2 *>(&w[k][1]);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                    {
                        ox[e] = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
                        oy[e] = __floats2half2_rn(y[2 * e], y[2 * e + 1]);
                    }
                }
            }
            __half *dst = nullptr;
            if (is_q)
                dst = a.q_out + (int64_t)r * a.q_out_stride + h * YLM_HEAD_DIM;
            else if (h < heads && page >= 0)
                dst = (is_k ? a.c.k : a.c.v) + at + (size_t)(is_k ? h - a.hq : h - a.hq - a.c.hkv) * a.c.page * YLM_HEAD_DIM;
            if (dst)
            {
                *reinterpret_cast<uint4 *>(dst + l * 8) = w[k][0];
                *reinterpret_cast<uint4 *>(dst + 64 + l * 8) = w[k][1];
            }
        }
    }
}

cudaError_t paged_append_launch(const PagedAppendArgs &a, int num_sms, cudaStream_t s)
{
    if (a.st.rows <= 0 || a.st.n_seq <= 0)
        return cudaSuccess;
    const int passes = (a.hq + 2 * a.c.hkv + PA_HEADS - 1) / PA_HEADS;
    // few rows: a CTA a pass, so that more SMs take part
    const int y = a.st.rows < num_sms ? std::min(passes, 65535) : 1;
    const dim3 grid((unsigned)a.st.rows, (unsigned)y);
    const int batch = (passes + y - 1) / y;
    return batch <= 1   ? paged_launch(paged_append_kernel<1>, grid, PA_THREADS, s, a)
           : batch == 2 ? paged_launch(paged_append_kernel<2>, grid, PA_THREADS, s, a)
                        : paged_launch(paged_append_kernel<3>, grid, PA_THREADS, s, a);
}

// ------------------------------------------------------------------ accept
// The walk: from row 0, to the lowest child whose token is the row's pick, until there is none. The rows of the
// path only rise, so path[j] >= j: moved in order, no slot is overwritten before it has been read.
// Each CTA of a request walks for itself (a warp, a shuffle and four ballots a step) and then moves its share of the
// 2 * layers * hkv rows of 256 bytes that an accepted token has, 16 lanes each.
// 60 trees of 50 to 64 tokens, 32 layers of 8 heads: 11.8 us = 3.4 TB/s: 2.6 when no draft is accepted, 3.9 with the moves
// of one layer, so most of it is the moves, rows of 256 bytes apart from one another. 28 layers of 4 heads, one tree of 8: 3.5 us, of
// which 2.3 are there without an accepted draft. CTAs an SM by threads, 60 trees: 8 x 128 11.9 us, 4 x 128 15.2, 16 x 128 12.6,
// 4 x 256 12.1, 8 x 256 12.7, 16 x 64 12.4.
constexpr int AC_THREADS = 128;
constexpr int AC_HALF = AC_THREADS / 16;
constexpr int AC_BATCH = 8; // rows in flight per 16 lanes

__global__ void __launch_bounds__(AC_THREADS) paged_accept_kernel(const __grid_constant__ PagedAcceptArgs a)
{
    __shared__ int path[PAGED_TREE];
    __shared__ int64_t from[PAGED_TREE], to[PAGED_TREE], picks[PAGED_TREE];
    __shared__ int count_s;
    pdl_wait();
    pdl_launch_dependents();
    const PagedStep &st = a.st;
    const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const bool writes = blockIdx.x == 0;
    PagedRequest q;
    bool bad;
    const bool is = paged_request(st, a.c.page, s, q, bad);
    int count = 0, last = 0;
    if (!is)
    {
        if (bad && writes && tid == 0)
            paged_fault(st, PAGED_BAD_REQUEST);
    }
    else if (!st.parent)
    {
        // a chain: the rows up to the first whose token is not the pick before it; they are in place already
        __shared__ int first;
        if (tid == 0)
            first = q.t;
        __syncthreads();
        for (int i = 1 + tid; i < q.t; i += AC_THREADS)
            if (a.tokens[q.row0 + i] != a.picks[q.row0 + i - 1])
            {
                atomicMin(&first, i);
                break;
            }
        __syncthreads();
        count = first;
        last = count - 1;
    }
    else
    {
        if (tid < 32)
        {
            PagedTree tree;
            if (tree.load(st, q, lane) && writes)
                paged_fault(st, PAGED_BAD_PARENT);
            int64_t token[PAGED_TREE / 32];
#pragma unroll
            for (int k = 0; k < PAGED_TREE / 32; k++)
            {
                const int i = lane + 32 * k;
                token[k] = i < q.t ? a.tokens[q.row0 + i] : 0;
                if (i < q.t)
                    picks[i] = a.picks[q.row0 + i];
            }
            __syncwarp();
            int cur = 0, m = 0;
            for (;;)
            {
                if (lane == 0)
                    path[m] = cur;
                m++;
                const int64_t pick = picks[cur];
                int next = -1;
#pragma unroll
                for (int k = PAGED_TREE / 32 - 1; k >= 0; k--)
                {
                    // (rows behind the last have no parent)
                    const unsigned hit = __ballot_sync(0xffffffffu, tree.p[k] == cur && token[k] == pick);
                    if (hit)
                        next = 32 * k + __ffs(hit) - 1;
                }
                if (next < 0)
                    break;
                cur = next; // > its parent: at most t steps
            }
            __syncwarp();
            for (int j = lane; j < m; j += 32)
            {
                const int x = q.n + path[j], y = q.n + j;
                const int px = paged_page(st, a.c, s, x), py = paged_page(st, a.c, s, y);
                if ((px < 0 || py < 0) && writes)
                    paged_fault(st, PAGED_BAD_PAGE);
                from[j] = px < 0 || py < 0 || x == y ? -1 : (int64_t)paged_offset(a.c, px, x);
                to[j] = px < 0 || py < 0 || x == y ? -1 : (int64_t)paged_offset(a.c, py, y);
            }
            if (lane == 0)
                count_s = m;
        }
        __syncthreads();
        count = count_s;
        last = path[count - 1];
        // this half warp's heads of the layers' keys and values
        const int l = tid & 15, rows = 2 * a.layers * a.c.hkv;
        for (int h = blockIdx.x * AC_HALF + (tid >> 4); h < rows; h += gridDim.x * AC_HALF)
        {
            const int layer = h / (2 * a.c.hkv), g = h % (2 * a.c.hkv);
            __half *pool = (g < a.c.hkv ? a.c.k : a.c.v) + (int64_t)layer * a.layer_stride +
                           (size_t)(g < a.c.hkv ? g : g - a.c.hkv) * a.c.page * YLM_HEAD_DIM + l * 8;
            for (int j0 = 1; j0 < count; j0 += AC_BATCH)
            {
                uint4 x[AC_BATCH];
#pragma unroll
                for (int u = 0; u < AC_BATCH; u++)
                    if (j0 + u < count && from[j0 + u] >= 0)
                        x[u] = *reinterpret_cast<const uint4 *>(pool + from[j0 + u]);
#pragma unroll
                for (int u = 0; u < AC_BATCH; u++)
                    if (j0 + u < count && from[j0 + u] >= 0)
                        *reinterpret_cast<uint4 *>(pool + to[j0 + u]) = x[u];
            }
        }
    }
    if (!writes)
        return;
    int32_t *acc = a.accepted + (size_t)s * a.accepted_ld;
    for (int j = tid; j < a.accepted_ld; j += AC_THREADS)
        acc[j] = j < count ? (st.parent ? path[j] : j) : -1;
    if (tid == 0)
    {
        a.n_accepted[s] = count;
        a.next_token[s] = count ? a.picks[q.row0 + last] : -1;
        a.new_length[s] = q.n + count; // of a request that is left out: as it was
    }
}

cudaError_t paged_accept_launch(const PagedAcceptArgs &a, int num_sms, cudaStream_t s)
{
    if (a.st.n_seq <= 0)
        return cudaSuccess;
    // about eight CTAs an SM at most, each with at least one round of moves
    const int64_t rounds = a.st.parent ? ((int64_t)2 * a.layers * a.c.hkv + AC_HALF - 1) / AC_HALF : 1;
    const int64_t slices = std::max<int64_t>(1, std::min<int64_t>(rounds, (int64_t)num_sms * 8 / a.st.n_seq));
    return paged_launch(paged_accept_kernel, dim3((unsigned)slices, (unsigned)a.st.n_seq), AC_THREADS, s, a);
}

} // namespace ylm
