// Attention of new tokens over a paged cache (paged.cuh).  A warp takes a (token, head) and walks the positions up to its own, 32 at a time: a lane scores a
// position, and the running maximum and sum of the softmax are joined once per 32.
#include "paged.cuh"

namespace bpdq {

struct PagedArgs {
    const void *q, *k_pool, *v_pool;
    void* o;
    int ld_q, ld_o;
    int n_tokens, batch, heads, kv_heads, dim, page, max_pages, n_pages;
    size_t page_stride;
    const int *seq_start, *length, *table;
    float scale, cap;
};

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
                atomicCAS(err, 0, 82);
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

static int paged_attention(const bpdq_paged_kv* kv, const void* q, int ld_q, void* o, int ld_o, int n_tokens, float scale, float cap, const bpdq_paged_groups* groups,
                           Workspace*, cudaStream_t s)
{
    int rc = paged_check(kv, n_tokens);
    if (rc) return rc;
    const int width = kv->heads * kv->dim;
    if (!q || !o || ld_q < width || ld_o < width || !(cap >= 0.0f) || !isfinite(cap) || !isfinite(scale)) return latch(BPDQ_ERR_ARG);
    if ((rc = check_groups(kv, groups))) return rc;
    const int unit = kv->act_type == BPDQ_TYPE_F32 ? 4 : 8;
    if ((((uintptr_t)q | (uintptr_t)o) & 15) || ld_q % unit || ld_o % unit) return latch(BPDQ_ERR_ALIGN);
    if (n_tokens == 0 || kv->batch == 0) return 0;
    PagedArgs p = {};
    p.q = q; p.o = o; p.k_pool = kv->k; p.v_pool = kv->v; p.ld_q = ld_q; p.ld_o = ld_o;
    p.n_tokens = n_tokens; p.batch = kv->batch; p.heads = kv->heads; p.kv_heads = kv->kv_heads; p.dim = kv->dim; p.page = kv->page;
    p.max_pages = kv->max_pages; p.n_pages = kv->n_pages; p.page_stride = paged_stride(*kv);
    p.seq_start = kv->seq_start; p.length = kv->length; p.table = kv->page_table; p.scale = scale; p.cap = cap;
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
    return paged_check(kv, n_tokens) || check_groups(kv, groups) ? 0 : 16;
}

int bpd_paged_attention_ws_cuda(const bpdq_paged_kv* kv, const void* q, int ld_q, void* o, int ld_o, int n_tokens, float scale, float cap,
                                const bpdq_paged_groups* groups, void* workspace, size_t workspace_bytes, void* stream)
{
    Workspace ws = {(uint8_t*)workspace, workspace_bytes, 0};
    if (!workspace) return latch(BPDQ_ERR_ARG);
    return paged_attention(kv, q, ld_q, o, ld_o, n_tokens, scale, cap, groups, &ws, (cudaStream_t)stream);
}

}  // extern "C"
