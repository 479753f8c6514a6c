// Attention of new tokens over a paged cache (paged_attention.cuh): which kernels a call takes, their scratch memory, and how parts are joined.
#include "paged_attention.cuh"

#include <type_traits>

namespace bpdq {

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
            // the member's parts: member, member + TEAM, ..; their maxima and sums a lane each, their outputs eight at a time
            for (int i0 = 0; i0 * TEAM + member < n; i0 += 32) {
                const int i = (i0 + lane) * TEAM + member;
                const float* o = p.own_o;
                const float2* ml = nullptr;
                float2 v = make_float2(-INFINITY, 0.0f);
                if (i < n) {
                    place(i, o, ml);
                    v = *ml;
                }
                const float top = fmaxf(most, warp_max(v.x)), ref = top == -INFINITY ? 0.0f : top, down = ex2(most - ref);
                const float w = ex2(v.x - ref);
                l = l * down + warp_sum(w * v.y);
                most = top;
#pragma unroll
                for (int c = 0; c < kCols; c++) acc[c] *= down;
                const int here = min(32, (n - member + TEAM - 1) / TEAM - i0);
                for (int k0 = 0; k0 < here; k0 += 8) {
                    float x[8][kCols];
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const float* from = reinterpret_cast<const float*>(__shfl_sync(0xFFFFFFFFu, (unsigned long long)o, k0 + k)) + kCols * lane;
#pragma unroll
                        for (int c = 0; c < kCols; c++) x[k][c] = 0.0f;
                        if (k0 + k < here) {
                            if constexpr (kCols == 4) *reinterpret_cast<float4*>(x[k]) = *reinterpret_cast<const float4*>(from);
                            else *reinterpret_cast<float2*>(x[k]) = *reinterpret_cast<const float2*>(from);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const float wk = __shfl_sync(0xFFFFFFFFu, w, k0 + k);
#pragma unroll
                        for (int c = 0; c < kCols; c++) acc[c] = fmaf(wk, x[k][c], acc[c]);
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
    // a tile of rows holds a token's at least; units of work are counted in 32 bits
    if (kv->heads / kv->kv_heads > 128 || kv->batch + (groups ? groups->n : 0) > kPagedMaxJobs) return latch(BPDQ_ERR_RANGE);
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

// Which kernels a call needs.  The host does not know lengths or bounds: where a job may have more rows than k_paged_split takes, both are launched, and each passes over the
// other's jobs.
struct Kernels {
    int split_rows;         // jobs of up to so many rows go to k_paged_split; 0: it is not launched
    bool tile;
};
static Kernels kernels(const PagedArgs& p)
{
    Kernels k;
    k.split_rows = p.share > kSplitRows ? 0 : (p.share <= 8 && !p.seq_start ? 8 : kSplitRows);
    k.tile = p.seq_start || p.groups || !k.split_rows;
    return k;
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
    p.q = q; p.o = o; p.ld_q = ld_q; p.ld_o = ld_o; p.scale = scale; p.cap = cap;
    const int ctas = sm_count();
    const Kernels run = kernels(p);
    uint8_t* mem = scratch_take(ws, kScratchPaged, carve(p, nullptr, ctas, run.tile), s, &rc);
    if (!mem) return rc;
    carve(p, mem, ctas, run.tile);
    p.split_rows = run.split_rows;
    if (run.tile) {
        p.mark = !run.split_rows;
        if ((rc = paged_tile(p, *kv, ctas, s))) return rc;
    }
    if (run.split_rows) {
        p.mark = 1;
        if ((rc = paged_split(p, *kv, ctas, s))) return rc;
    }
    const bool wide = kv->dim > 64;
    if (kv->act_type == BPDQ_TYPE_F32) return wide ? launch_join<float, 128>(p, s) : launch_join<float, 64>(p, s);
    if (kv->act_type == BPDQ_TYPE_F16) return wide ? launch_join<__half, 128>(p, s) : launch_join<__half, 64>(p, s);
    return wide ? launch_join<bf16, 128>(p, s) : launch_join<bf16, 64>(p, s);
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
    return carve(p, nullptr, sm_count(), kernels(p).tile) + 256;
}

int bpd_paged_attention_ws_cuda(const bpdq_paged_kv* kv, const void* q, int ld_q, void* o, int ld_o, int n_tokens, float scale, float cap,
                                const bpdq_paged_groups* groups, void* workspace, size_t workspace_bytes, void* stream)
{
    Workspace ws = {(uint8_t*)workspace, workspace_bytes, 0};
    if (!workspace) return latch(BPDQ_ERR_ARG);
    return paged_attention(kv, q, ld_q, o, ld_o, n_tokens, scale, cap, groups, &ws, (cudaStream_t)stream);
}

}  // extern "C"
