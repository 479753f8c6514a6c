// Attention of new tokens over a paged cache (paged.cuh).  A warp takes a (token, head) and walks the positions up to its own, 32 at a time: a lane scores a
// position, and the running maximum and sum of the softmax are joined once per 32.
#include "paged_attention.cuh"

#include <type_traits>

namespace bpdq {

template <typename A, typename K>
__global__ void __launch_bounds__(128) k_paged_attn_plain(const PagedArgs p, int* err)
{
    __shared__ float s_q[4][kPagedMaxDim];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int item = blockIdx.x * 4 + warp;
    pdl_launch_dependents();
    pdl_wait();
    if (item >= p.n_tokens * p.heads) return;
    const int t = item / p.heads, h = item % p.heads, g = h / (p.heads / p.kv_heads);
    int seq = -1, pos = 0;
    for (int b0 = 0; b0 < p.batch && seq < 0; b0 += 32) {
        const int b = b0 + lane;
        PagedSpan s = {0, 0, 0};
        if (b < p.batch) s = paged_span(p.seq_start, p.length, b, p.n_tokens, p.max_pages * p.page, err);
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, s.count > 0 && s.first <= t && t < s.first + s.count);
        if (hit) {
            const int src = __ffs(hit) - 1;
            seq = b0 + src;
            pos = __shfl_sync(0xFFFFFFFFu, s.held + t - s.first, src);
        }
    }
    if (seq < 0) return;
    const A* q = static_cast<const A*>(p.q) + (size_t)t * p.ld_q + h * p.dim;
    for (int d = lane; d < p.dim; d += 32) s_q[warp][d] = ActOf<A>::get(q[d]);
    __syncwarp();
    float m = -INFINITY, sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j0 = 0; j0 <= pos; j0 += 32) {
        const int j = j0 + lane;
        float x = -INFINITY;
        long at = -1;
        if (j <= pos) {
            const int page = p.table[(size_t)seq * p.max_pages + j / p.page];
            if (page >= 0 && page < p.n_pages) {
                at = (long)((size_t)page * p.page_stride + ((size_t)g * p.page + j % p.page) * p.dim);
                const K* k = static_cast<const K*>(p.k_pool) + at;
                float s = 0.0f;
                for (int d = 0; d < p.dim; d++) s = fmaf(s_q[warp][d], ActOf<K>::get(k[d]), s);
                x = s * p.scale;
                if (p.cap > 0.0f) x = p.cap * tanhf(x / p.cap);
            } else {
                report(err, 82);
            }
        }
        const float top = fmaxf(m, warp_max(x)), base = top == -INFINITY ? 0.0f : top;
        const float down = expf(m - base), w = at < 0 ? 0.0f : expf(x - base);
        sum = sum * down + warp_sum(w);
        m = top;
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] *= down;
        for (int l = 0; l < 32; l++) {
            const float wl = __shfl_sync(0xFFFFFFFFu, w, l);
            const long al = __shfl_sync(0xFFFFFFFFu, at, l);
            if (al < 0) continue;
            const K* v = static_cast<const K*>(p.v_pool) + al;
            for (int i = 0; i < 4; i++)
                if (32 * i + lane < p.dim) acc[i] = fmaf(wl, ActOf<K>::get(v[32 * i + lane]), acc[i]);
        }
    }
    A* o = static_cast<A*>(p.o) + (size_t)t * p.ld_o + h * p.dim;
    for (int i = 0; i < 4; i++)
        if (32 * i + lane < p.dim) o[32 * i + lane] = ActOf<A>::put(sum > 0.0f ? acc[i] / sum : 0.0f);
}

static int check_groups(const bpdq_paged_kv* kv, const bpdq_paged_groups* g)
{
    return g && (g->n < 0 || g->n > kv->batch || (g->n && (!g->start || !g->pages))) ? latch(BPDQ_ERR_ARG) : 0;
}

// Adds up the parts of rows that the kernels ahead have left in scratch memory: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.  A warp per row, or four of
// them where there are few rows.
template <typename A, int DP, int TEAM>
__global__ void __launch_bounds__(128) k_paged_join(const PagedArgs p)
{
    constexpr int kCols = DP / 32;
    __shared__ float s_o[4][DP];
    __shared__ float2 s_ml[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, member = TEAM > 1 ? warp : 0;
    const long rows = (long)p.n_tokens * p.heads, teams = (long)gridDim.x * (4 / TEAM), team = TEAM > 1 ? (long)blockIdx.x : (long)blockIdx.x * 4 + warp;
    pdl_wait();
    pdl_launch_dependents();
    for (long base = team; base < rows; base += 32 * teams) {
        // the descriptors of the team's next 32 rows at once
        const long mine = base + lane * teams;
        int4 d = make_int4(0, 0, 0, 0);
        if (mine < rows) d = p.own[mine];
        unsigned todo = __ballot_sync(0xFFFFFFFFu, d.y > 1 || (d.y == 1 && (d.w & kJoinPrefix)));
        while (todo) {
            const int src = __ffs(todo) - 1;
            todo &= todo - 1;
            const long row = base + src * teams;
            const int4 own = make_int4(__shfl_sync(0xFFFFFFFFu, d.x, src), __shfl_sync(0xFFFFFFFFu, d.y, src), __shfl_sync(0xFFFFFFFFu, d.z, src), __shfl_sync(0xFFFFFFFFu, d.w, src));
            int4 pre = make_int4(0, 0, 0, 0);
            if (own.w & kJoinPrefix) pre = p.prefix[row];
            // part i of the row: its own positions' first, then the prefix's
            const int n = own.y + pre.y;
            auto place = [&](int i, const float*& o, const float2*& ml) {
                const bool mine = i < own.y;
                const int4 e = mine ? own : pre;
                const int k = mine ? i : i - own.y;
                size_t at;
                if (e.y == 1) {
                    at = (size_t)row;
                    o = mine ? p.own_o : p.prefix_o;
                    ml = mine ? p.own_ml : p.prefix_ml;
                } else {
                    at = (size_t)(2 * (e.x + k) + (k == 0)) * (e.w & kJoinTile ? kTileRows : kSplitRows) + e.z;
                    o = e.w & kJoinTile ? p.tile_o : p.split_o;
                    ml = e.w & kJoinTile ? p.tile_ml : p.split_ml;
                }
                o += at * DP;
                ml += at;
            };
            float most = -INFINITY, l = 0.0f, acc[kCols];
#pragma unroll
            for (int c = 0; c < kCols; c++) acc[c] = 0.0f;
            for (int i0 = 32 * member; i0 < n; i0 += 32 * TEAM) {
                // maxima and sums of up to 32 parts, a lane each
                const float *o = nullptr;
                const float2* ml = nullptr;
                float2 v = make_float2(-INFINITY, 0.0f);
                if (i0 + lane < n) {
                    place(i0 + lane, o, ml);
                    v = *ml;
                }
                const float top = fmaxf(most, warp_max(v.x)), ref = top == -INFINITY ? 0.0f : top, down = ex2(most - ref);
                const float w = ex2(v.x - ref);
                l = l * down + warp_sum(w * v.y);
                most = top;
#pragma unroll
                for (int c = 0; c < kCols; c++) acc[c] *= down;
                const int here = n - i0 < 32 ? n - i0 : 32;
#pragma unroll 4
                for (int i = 0; i < here; i++) {
                    const float wi = __shfl_sync(0xFFFFFFFFu, w, i);
                    const float* from = reinterpret_cast<const float*>(__shfl_sync(0xFFFFFFFFu, (unsigned long long)o, i)) + kCols * lane;
                    if (kCols == 4) {
                        const float4 x = *reinterpret_cast<const float4*>(from);
                        acc[0] = fmaf(wi, x.x, acc[0]);
                        acc[1] = fmaf(wi, x.y, acc[1]);
                        acc[kCols - 2] = fmaf(wi, x.z, acc[kCols - 2]);
                        acc[kCols - 1] = fmaf(wi, x.w, acc[kCols - 1]);
                    } else {
                        const float2 x = *reinterpret_cast<const float2*>(from);
                        acc[0] = fmaf(wi, x.x, acc[0]);
                        acc[1] = fmaf(wi, x.y, acc[1]);
                    }
                }
            }
            if (TEAM > 1) {
                __syncthreads();                    // (what the row before was read from)
                if (lane == 0) s_ml[warp] = make_float2(most, l);
#pragma unroll
                for (int c = 0; c < kCols; c++) s_o[warp][kCols * lane + c] = acc[c];
                __syncthreads();
                if (warp > 0) continue;
                float top = -INFINITY;
                for (int i = 0; i < TEAM; i++) top = fmaxf(top, s_ml[i].x);
                const float ref = top == -INFINITY ? 0.0f : top;
                l = 0.0f;
#pragma unroll
                for (int c = 0; c < kCols; c++) acc[c] = 0.0f;
                for (int i = 0; i < TEAM; i++) {
                    const float w = ex2(s_ml[i].x - ref);
                    l = fmaf(w, s_ml[i].y, l);
#pragma unroll
                    for (int c = 0; c < kCols; c++) acc[c] = fmaf(w, s_o[i][kCols * lane + c], acc[c]);
                }
            }
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            A* out = static_cast<A*>(p.o) + (size_t)(row / p.heads) * p.ld_o + (int)(row % p.heads) * p.dim;
#pragma unroll
            for (int c = 0; c < kCols; c++)
                if (kCols * lane + c < p.dim) out[kCols * lane + c] = ActOf<A>::put(acc[c] * inv);
        }
    }
}

template <typename A, int DP>
static int launch_join(const PagedArgs& p, cudaStream_t s)
{
    const long rows = (long)p.n_tokens * p.heads, room = 8L * sm_count();
    if (rows <= room) return launch_ordered(k_paged_join<A, DP, 4>, dim3((unsigned)rows), 128, 0, s, p);
    const long ctas = (rows + 3) / 4;
    return launch_ordered(k_paged_join<A, DP, 1>, dim3((unsigned)(ctas < room ? ctas : room)), 128, 0, s, p);
}

// Scratch of a call, carved out of `base` (null: sizes alone); returns its bytes.
static size_t carve(PagedArgs& a, uint8_t* base, int ctas, bool tiles)
{
    size_t at = 0;
    auto take = [&](auto*& p, size_t n) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
        at += (n * sizeof(*p) + 255) / 256 * 256;
    };
    const size_t rows = (size_t)a.n_tokens * a.heads, pad = a.dim > 64 ? 128 : 64;
    take(a.own, rows);
    take(a.split_o, (size_t)2 * ctas * kSplitRows * pad);
    take(a.split_ml, (size_t)2 * ctas * kSplitRows);
    take(a.head_o, (size_t)kSplitWarps * ctas * kSplitRows * pad);
    take(a.head_ml, (size_t)kSplitWarps * ctas * kSplitRows);
    if (tiles) {
        take(a.tile_o, (size_t)2 * ctas * kTileRows * pad);
        take(a.tile_ml, (size_t)2 * ctas * kTileRows);
    }
    if (a.groups) {
        take(a.prefix, rows);
        take(a.own_o, rows * pad);
        take(a.own_ml, rows);
        take(a.prefix_o, rows * pad);
        take(a.prefix_ml, rows);
    }
    return at;
}

static int attention_check(const bpdq_paged_kv* kv, int n_tokens, const bpdq_paged_groups* groups)
{
    int rc = paged_check(kv, n_tokens);
    if (rc || (rc = check_groups(kv, groups))) return rc;
    // units of work are counted in 32 bits
    return (double)kv->batch * kv->kv_heads * kv->max_pages * kv->page > 8589934592.0 ? latch(BPDQ_ERR_RANGE) : 0;
}

static PagedArgs arguments(const bpdq_paged_kv& kv, int n_tokens, const bpdq_paged_groups* groups)
{
    PagedArgs p = {};
    p.n_tokens = n_tokens; p.batch = kv.batch; p.heads = kv.heads; p.kv_heads = kv.kv_heads; p.share = kv.heads / kv.kv_heads; p.dim = kv.dim;
    p.page = kv.page; p.max_pages = kv.max_pages; p.n_pages = kv.n_pages; p.page_stride = paged_stride(kv);
    while ((1 << p.log_page) < p.page) p.log_page++;
    p.seq_start = kv.seq_start; p.length = kv.length; p.table = kv.page_table;
    if (groups && groups->n) { p.groups = groups->n; p.group_start = groups->start; p.group_pages = groups->pages; }
    return p;
}

static int paged_attention(const bpdq_paged_kv* kv, const void* q, int ld_q, void* o, int ld_o, int n_tokens, float scale, float cap, const bpdq_paged_groups* groups,
                           Workspace* ws, cudaStream_t s)
{
    int rc = attention_check(kv, n_tokens, groups);
    if (rc) return rc;
    const int width = kv->heads * kv->dim;
    if (!q || !o || ld_q < width || ld_o < width || !(cap >= 0.0f) || !isfinite(cap) || !isfinite(scale)) return latch(BPDQ_ERR_ARG);
    const int unit = kv->act_type == BPDQ_TYPE_F32 ? 4 : 8;
    if ((((uintptr_t)q | (uintptr_t)o) & 15) || ld_q % unit || ld_o % unit) return latch(BPDQ_ERR_ALIGN);
    if (n_tokens == 0 || kv->batch == 0) return 0;
    PagedArgs p = arguments(*kv, n_tokens, groups);
    p.k_pool = kv->k; p.v_pool = kv->v; p.q = q; p.o = o; p.ld_q = ld_q; p.ld_o = ld_o; p.scale = scale; p.cap = cap;
    const int ctas = sm_count();
    if (!kv->seq_start && p.share <= kSplitRows && !p.groups) {
        uint8_t* mem = scratch_take(ws, kScratchPaged, carve(p, nullptr, ctas, false), s, &rc);
        if (!mem) return rc;
        carve(p, mem, ctas, false);
        p.split_rows = p.share;
        p.mark = 1;
        if ((rc = paged_split(p, *kv, ctas, s))) return rc;
        const bool wide = kv->dim > 64;
        if (kv->act_type == BPDQ_TYPE_F32) return wide ? launch_join<float, 128>(p, s) : launch_join<float, 64>(p, s);
        if (kv->act_type == BPDQ_TYPE_F16) return wide ? launch_join<__half, 128>(p, s) : launch_join<__half, 64>(p, s);
        return wide ? launch_join<bf16, 128>(p, s) : launch_join<bf16, 64>(p, s);
    }
    const dim3 grid((unsigned)((n_tokens * kv->heads + 3) / 4));
    if (kv->act_type == BPDQ_TYPE_F32) return launch_ordered(k_paged_attn_plain<float, __half>, grid, 128, 0, s, p, device_error_flag());
    if (kv->act_type == BPDQ_TYPE_F16) return launch_ordered(k_paged_attn_plain<__half, __half>, grid, 128, 0, s, p, device_error_flag());
    return launch_ordered(k_paged_attn_plain<bf16, bf16>, grid, 128, 0, s, p, device_error_flag());
}

}  // namespace bpdq

using namespace bpdq;

extern "C" {

int bpd_paged_attention_cuda(const bpdq_paged_kv* kv, const void* q, int ld_q, void* o, int ld_o, int n_tokens, float scale, float cap,
                             const bpdq_paged_groups* groups, void* stream)
{
    return paged_attention(kv, q, ld_q, o, ld_o, n_tokens, scale, cap, groups, nullptr, (cudaStream_t)stream);
}

size_t bpdq_paged_attention_workspace_bytes(const bpdq_paged_kv* kv, int n_tokens, const bpdq_paged_groups* groups)
{
    if (attention_check(kv, n_tokens, groups)) return 0;
    PagedArgs p = arguments(*kv, n_tokens, groups);
    return carve(p, nullptr, sm_count(), false) + 256;
}

int bpd_paged_attention_ws_cuda(const bpdq_paged_kv* kv, const void* q, int ld_q, void* o, int ld_o, int n_tokens, float scale, float cap,
                                const bpdq_paged_groups* groups, void* workspace, size_t workspace_bytes, void* stream)
{
    Workspace ws = {(uint8_t*)workspace, workspace_bytes, 0};
    if (!workspace) return latch(BPDQ_ERR_ARG);
    return paged_attention(kv, q, ld_q, o, ld_o, n_tokens, scale, cap, groups, &ws, (cudaStream_t)stream);
}

}  // extern "C"
