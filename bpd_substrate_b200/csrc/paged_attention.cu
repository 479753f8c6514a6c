// Attention of new tokens over a paged cache (paged_attention.cuh): which kernels a call takes, their scratch memory, and how parts are joined.
#include "paged_attention.cuh"

#include <type_traits>

namespace bpdq {

static int check_groups(const bpdq_paged_kv* kv, const bpdq_paged_groups* g)
{
    return g && (g->n < 0 || g->n > kv->batch || (g->n && (!g->start || !g->pages))) ? latch(BPDQ_ERR_ARG) : 0;
}

// Adds up the parts of rows that the kernels ahead have left in scratch memory: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.  Eight threads walk through the
// parts of a row; or, where there are few rows, a CTA has one row and eight threads every sixteenth part.  (192000 rows, a fifth of them in two parts: 14 us.  A
// call of 2048 rows with a prefix: 53 us with a CTA per row, 64 with eight threads; of 2048 without: 49.0 and 48.4.)
constexpr int kJoinThreads = 128, kJoinGroups = kJoinThreads / 8;

template <typename A, int DP, bool kFew>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(const PagedArgs p)
{
    constexpr int kUnits = DP / 32;
    __shared__ float s_o[kFew ? kJoinGroups : 1][DP];
    __shared__ float2 s_ml[kJoinGroups];
    const int l8 = threadIdx.x & 7, group = threadIdx.x >> 3;
    const long rows = (long)p.n_tokens * p.heads, stride = kFew ? (long)gridDim.x : (long)gridDim.x * kJoinGroups;
    pdl_wait();
    pdl_launch_dependents();
    // (where bounds run backwards, a row may have no job in its group, or several)
    auto sane = [&](const int4& e) { return e.x >= 0 && e.y >= 0 && e.x <= p.ctas - e.y && e.z >= 0 && e.z < (e.w & kJoinTile ? kTileRows : kSplitRows); };
    long row = kFew ? (long)blockIdx.x : (long)blockIdx.x * kJoinGroups + group;
    int4 next = row < rows ? p.own[row] : make_int4(0, 0, 0, 0);
    for (; row < rows; row += stride) {
        const int4 own = next;
        if (row + stride < rows) next = p.own[row + stride];
        if (own.y == 0 || (own.y == 1 && !(own.w & kJoinPrefix)) || !sane(own)) continue;
        int4 pre = make_int4(0, 0, 0, 0);
        if (own.w & kJoinPrefix) {
            pre = p.prefix[row];
            if (!sane(pre)) pre.y = 0;
        }
        // part i of the row: its own positions' first, then the prefix's
        const int n = own.y + pre.y;
        auto place = [&](int i, const float*& o, const float2*& ml) {
            const bool mine = i < own.y;
            const int4 e = mine ? own : pre;
            const int k = mine ? i : i - own.y;
            size_t at = (size_t)row;
            if (e.y == 1) {
                o = mine ? p.own_o : p.prefix_o;
                ml = mine ? p.own_ml : p.prefix_ml;
            } else {
                at = (size_t)(2 * (e.x + k) + (k == 0)) * (e.w & kJoinTile ? kTileRows : kSplitRows) + e.z;
                o = e.w & kJoinTile ? p.tile_o : p.split_o;
                ml = e.w & kJoinTile ? p.tile_ml : p.split_ml;
            }
            o += at * DP + 4 * l8;
            ml += at;
        };
        float top = -INFINITY, l = 0.0f;
        float4 acc[kUnits];
#pragma unroll
        for (int c = 0; c < kUnits; c++) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        // two parts at a time
        constexpr int step = kFew ? kJoinGroups : 1;
#pragma unroll 1
        for (int i = kFew ? group : 0; i < n; i += 2 * step) {
            const float* o[2];
            const float2* ml[2];
            float2 v[2];
            float4 x[2][kUnits];
            const bool two = i + step < n;
            place(i, o[0], ml[0]);
            place(two ? i + step : i, o[1], ml[1]);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                v[k] = *ml[k];
#pragma unroll
                for (int c = 0; c < kUnits; c++) x[k][c] = *reinterpret_cast<const float4*>(o[k] + 32 * c);
            }
            if (!two) v[1] = make_float2(-INFINITY, 0.0f);
            const float now = fmaxf(top, fmaxf(v[0].x, v[1].x)), zero = now == -INFINITY ? 0.0f : now;
            const float down = ex2(top - zero), w0 = ex2(v[0].x - zero), w1 = ex2(v[1].x - zero);
            l = fmaf(w1, v[1].y, fmaf(w0, v[0].y, l * down));
            top = now;
#pragma unroll
            for (int c = 0; c < kUnits; c++) {
                acc[c].x = fmaf(w1, x[1][c].x, fmaf(w0, x[0][c].x, acc[c].x * down));
                acc[c].y = fmaf(w1, x[1][c].y, fmaf(w0, x[0][c].y, acc[c].y * down));
                acc[c].z = fmaf(w1, x[1][c].z, fmaf(w0, x[0][c].z, acc[c].z * down));
                acc[c].w = fmaf(w1, x[1][c].w, fmaf(w0, x[0][c].w, acc[c].w * down));
            }
        }
        A* out = static_cast<A*>(p.o) + (size_t)(row / p.heads) * p.ld_o + (int)(row % p.heads) * p.dim;
        if (kFew) {
            __syncthreads();                    // (what the row before was read from)
            if (l8 == 0) s_ml[group] = make_float2(top, l);
#pragma unroll
            for (int c = 0; c < kUnits; c++) *reinterpret_cast<float4*>(&s_o[kFew ? group : 0][32 * c + 4 * l8]) = acc[c];
            __syncthreads();
            const int d = threadIdx.x;
            if (d < p.dim) {
                const int used = n < kJoinGroups ? n : kJoinGroups;
                float most = -INFINITY, sum = 0.0f, o = 0.0f;
                for (int i = 0; i < used; i++) most = fmaxf(most, s_ml[i].x);
                const float zero = most == -INFINITY ? 0.0f : most;
                for (int i = 0; i < used; i++) {
                    const float w = ex2(s_ml[i].x - zero);
                    sum = fmaf(w, s_ml[i].y, sum);
                    o = fmaf(w, s_o[kFew ? i : 0][d], o);
                }
                out[d] = ActOf<A>::put(sum != 0.0f ? o / sum : 0.0f);
            }
            continue;
        }
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int c = 0; c < kUnits; c++)
            if (32 * c + 4 * l8 < p.dim) {
                A* at = out + 32 * c + 4 * l8;
                at[0] = ActOf<A>::put(acc[c].x * inv);
                at[1] = ActOf<A>::put(acc[c].y * inv);
                at[2] = ActOf<A>::put(acc[c].z * inv);
                at[3] = ActOf<A>::put(acc[c].w * inv);
            }
    }
}

template <typename A, int DP>
static int launch_join(const PagedArgs& p, cudaStream_t s)
{
    const long rows = (long)p.n_tokens * p.heads;
    // a CTA per row: few rows have many parts, and so may rows with a prefix
    if (rows <= (p.groups ? 16L : 4L) * sm_count()) return launch_ordered(k_paged_join<A, DP, true>, dim3((unsigned)rows), kJoinThreads, 0, s, p);
    const long ctas = (rows + kJoinGroups - 1) / kJoinGroups, room = 12L * sm_count();
    return launch_ordered(k_paged_join<A, DP, false>, dim3((unsigned)(ctas < room ? ctas : room)), kJoinThreads, 0, s, p);
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
        if (a.f32) take(a.tile_sums, (size_t)ctas * kTileRows * pad);
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
    const double capacity = (double)kv->max_pages * kv->page, tiles = 2.0 * n_tokens / (128 / (kv->heads / kv->kv_heads)) + 2.0 * kv->batch;
    return kv->batch * kv->kv_heads * capacity > 8589934592.0 || tiles * kv->kv_heads * (capacity / 128 + 3) > 2147483647.0 ? latch(BPDQ_ERR_RANGE) : 0;
}

static PagedArgs arguments(const bpdq_paged_kv& kv, int n_tokens, const bpdq_paged_groups* groups)
{
    PagedArgs p = {};
    p.n_tokens = n_tokens; p.batch = kv.batch; p.heads = kv.heads; p.kv_heads = kv.kv_heads; p.share = kv.heads / kv.kv_heads; p.dim = kv.dim;
    p.page = kv.page; p.max_pages = kv.max_pages; p.n_pages = kv.n_pages; p.page_stride = paged_stride(kv);
    while ((1 << p.log_page) < p.page) p.log_page++;
    p.seq_start = kv.seq_start; p.length = kv.length; p.table = kv.page_table; p.f32 = kv.act_type == BPDQ_TYPE_F32;
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
    // k_paged_split's products of 8 rows or of 16, or k_paged_tile, for 9 to 16 rows: where query heads on a key head are more than 8, or a few tokens per sequence.
    // fp32, 16 rows: 16 sequences of 2000 positions 35 us in k_paged_split and 51 in k_paged_tile, 64 of them 83 and 123.  16-bit types, sixteen heads: 1 of 4000 20.5 and
    // 19.0, 16 of 2000 34.7 and 32.0, 64 103 and 80; four tokens of four heads: 4 of 4000 24.5 and 27.8, 16 of 2000 39.5 and 43.5, 64 107 and 87 (8 key heads of 128).
    const long average = p.seq_start && p.batch ? ((long)p.n_tokens * p.share + p.batch - 1) / p.batch : p.share;
    Kernels k;
    const bool few = p.f32 || (p.share <= 8 && (long)p.batch * p.kv_heads <= 2L * sm_count());
    k.split_rows = p.share <= 8 ? 8 : 0;
    if (few && p.share <= kSplitRows && (p.share > 8 || (average > 8 && average <= kSplitRows))) k.split_rows = kSplitRows;
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
    if (q == o && ld_q != ld_o && n_tokens > 1) return latch(BPDQ_ERR_ARG);         // (rows would lie over others that are yet to be read)
    if (n_tokens == 0 || kv->batch == 0) return 0;
    PagedArgs p = arguments(*kv, n_tokens, groups);
    const int ctas = sm_count();
    p.q = q; p.o = o; p.ld_q = ld_q; p.ld_o = ld_o; p.scale = scale; p.cap = cap; p.ctas = ctas; p.cap_kind = cap_kind(cap, p.f32);
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
