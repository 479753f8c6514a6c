// Attention over a paged cache: what its kernels share.  A call's work is cut into jobs, a set of rows (row = (token, query head of a key head)) against
// a range of positions: every sequence's new tokens against its own positions, and every group's tokens against the pages that the group shares.  A
// job has an item per key head.  Items are laid end to end in units of keys and dealt to the CTAs in equal portions, whatever the lengths; an item
// that several CTAs have parts of, or that has a prefix, leaves its parts in scratch memory, and k_paged_join adds them up.
#pragma once
#include "paged.cuh"
#include "tensor_map.cuh"

namespace bpdq {

struct PagedArgs {
    const void* q;
    void* o;
    int ld_q, ld_o;
    int n_tokens, batch, heads, kv_heads, share, dim, page, log_page, max_pages, n_pages;
    size_t page_stride;
    const int *seq_start, *length, *table;
    int groups;
    const int *group_start, *group_pages;
    float scale, cap;
    int split_rows;             // jobs of up to so many rows are k_paged_split's, the others k_paged_tile's
    int both;                   // this launch's requests bring both halves of 128 dimensions
    int f32;                    // activations
    int cap_kind;               // CapKind
    int ctas;                   // of a grid, at most
    int mark;                   // this launch says which tokens belong to no sequence
    // scratch
    int4* own;                  // [tokens][heads]: what k_paged_join finds of a row's own positions
    int4* prefix;               // the same of its group's
    float *own_o, *prefix_o;    // [tokens * heads][dim_pad]: parts that are whole, unnormalised
    float2 *own_ml, *prefix_ml; // what their sums count from (maxima, in units of log2, less the kernel's shift) and sums of weights
    float *split_o, *tile_o;    // parts of items that several CTAs share: [2 * CTA + which][rows][dim_pad]
    float2 *split_ml, *tile_ml;
    float* tile_sums;           // k_paged_tile of fp32: what a stream has put aside, [2 * CTA + stream][dim_pad / 4][rows of a stream][4]
    float* head_o;              // k_paged_split: a warp's first part, when it has two
    float2* head_ml;
};

// A row's descriptor: x the CTA with the first part, y the number of parts (0: the row belongs to no sequence; 1: all in one CTA), z the row within the
// parts, w: flags
constexpr int kJoinTile = 1;            // parts are k_paged_tile's
constexpr int kJoinPrefix = 2;          // (own) the row has a prefix as well
constexpr int kSplitRows = 16, kTileRows = 256;
constexpr int kPagedMaxJobs = 1280;      // sequences and groups of a call: 20 to 24 bytes of shared memory each

// Tiles of a pool in the 128-byte swizzle: up to `rows` positions of a head of a page, 64 dimensions wide, or (paged_both) both halves of 128 dimensions,
// one behind the other, in one request.  Dimensions beyond the head's read as zeros.
static inline bool paged_both(const bpdq_paged_kv& kv, int rows) { return kv.dim == 128 && kv.page >= rows; }
static inline int paged_map(CUtensorMap* map, const void* pool, const bpdq_paged_kv& kv, int rows)
{
    const bool both = paged_both(kv, rows);
    const cuuint64_t row = (cuuint64_t)kv.dim * 2;
    const cuuint64_t dims[5] = {(cuuint64_t)(both ? 64 : kv.dim), (cuuint64_t)kv.page, (cuuint64_t)(both ? 2 : 1), (cuuint64_t)kv.kv_heads, (cuuint64_t)kv.n_pages};
    const cuuint64_t strides[4] = {row, both ? 128 : row, row * kv.page, (cuuint64_t)paged_stride(kv) * 2};
    const cuuint32_t box[5] = {64, (cuuint32_t)(kv.page < rows ? kv.page : rows), (cuuint32_t)(both ? 2 : 1), 1, 1};
    return swizzled_map(map, pool, 5, dims, strides, box);
}

// paged_split.cu, paged_tile.cu
int paged_split(const PagedArgs& a, const bpdq_paged_kv& kv, int ctas, cudaStream_t s);
int paged_tile(const PagedArgs& a, const bpdq_paged_kv& kv, int ctas, cudaStream_t s);
constexpr int kSplitWarps = 8;

#ifdef __CUDACC__

// Rows of a page from dimension d (a multiple of 64) on; where both halves come in one request d is 0.
__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, int d, int row, int head, int page, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(map), "r"(d), "r"(row), "r"(0), "r"(head), "r"(page), "r"(bar)
        : "memory");
}

// cap tanh(x / cap): of fp32 results by CUDA's function, of rounded ones by 1 - 2 / (1 + e^(2 x / cap)), off by 2^-22 of the cap.  That shows in the weights where the cap is far
// above the scores, and the approximate divisions have an end of their own: of such caps scores are off by 2^-20 of themselves, below 0.3 caps by the first five terms of tanh's series
// (the sixth: 2^-24).  (A bf16 prompt of 2000, 32 heads on 8 of 128: cap 30 117 us, 200 145.)
enum CapKind { kCapNone = 0, kCapNear = 1, kCapFar = 2 };
static inline CapKind cap_kind(float cap, bool f32) { return cap > 0.0f ? (f32 || (cap >= 1.0f / 1048576.0f && cap <= 64.0f) ? kCapNear : kCapFar) : kCapNone; }
template <bool f32, int kCap> __device__ __forceinline__ float capped(float x, float cap)
{
    if (f32) return cap * tanhf(x / cap);
    if (kCap == kCapNear) return cap - __fdividef(2.0f * cap, 1.0f + ex2(2.88539008177792681f * __fdividef(x, cap)));
    cap = fmaxf(cap, 1e-30f);           // (below it all scores are alike)
    const float t = x * (1.0f / cap), t2 = t * t;
    float p = fmaf(t2, 62.0f / 2835.0f, -17.0f / 315.0f);
    p = fmaf(t2, p, 2.0f / 15.0f);
    p = fmaf(t2, p, -1.0f / 3.0f);
    p = fmaf(t2, p, 1.0f);
    return fabsf(t) < 0.3f ? x * p : cap * (1.0f - __fdividef(2.0f, 1.0f + ex2(2.88539008177792681f * t)));
}

// The jobs of a call, as every CTA works them out for itself.  cum[j]: units ahead of job j; jobs 0 .. batch - 1 are the sequences', the groups' follow.
struct PagedJob {
    int first, count, rows;         // tokens, rows
    int from, to;                   // positions
    int seq;                        // whose row of the page table
    bool prefix, joined;            // a group's job; rows that k_paged_join meets in any case
};
struct PagedPlan {
    int* cum;                       // shared, [jobs + 1]
    int* group_len;                 // shared, [groups]: positions that a group shares
    int4* spans;                    // shared, [jobs]: first token, number of tokens, positions from, to; of a group's job, which starts at 0, the sequence whose pages are read instead
    int jobs;

    __host__ __device__ static int size(const PagedArgs& p) { return 16 * (p.batch + p.groups) + 4 * (p.batch + 2 * p.groups + 1); }
    // The group of a sequence, or -1.
    __device__ static int group_of(const PagedArgs& p, int b)
    {
        int lo = 0, hi = p.groups;                      // start[lo] <= b < start[hi]
        if (!p.groups || b < p.group_start[0] || b >= p.group_start[p.groups]) return -1;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.group_start[mid] <= b) lo = mid;
            else hi = mid;
        }
        return lo;
    }
    __device__ static PagedSpan span(const PagedArgs& p, int b, int* err)
    {
        return paged_span(p.seq_start, p.length, b, p.n_tokens, p.max_pages * p.page, err);
    }
    __device__ static void members(const PagedArgs& p, int g, int& s0, int& s1)
    {
        s0 = min(max(p.group_start[g], 0), p.batch);
        s1 = min(max(p.group_start[g + 1], s0), p.batch);
    }
    __device__ PagedJob job(const PagedArgs& p, int j, int* err) const
    {
        PagedJob r;
        r.prefix = j >= p.batch;
        if (!r.prefix) {
            const PagedSpan s = span(p, j, err);
            const int g = group_of(p, j);
            r.first = s.first; r.count = s.count; r.seq = j;
            r.from = g >= 0 ? group_len[g] : 0;
            r.to = s.held + s.count;
            r.joined = r.from > 0;
        } else {
            int s0, s1;
            members(p, j - p.batch, s0, s1);
            // a group's tokens lie side by side: its sequences do
            const int a = p.seq_start ? p.seq_start[s0] : s0, b = p.seq_start ? p.seq_start[s1] : s1;
            r.first = min(max(a, 0), p.n_tokens);
            r.count = min(max(b, r.first), p.n_tokens) - r.first;
            r.seq = spans[j].z;
            r.from = 0;
            r.to = group_len[j - p.batch];
            r.joined = true;
            if (r.to <= 0) r.count = 0;
        }
        r.rows = r.count * p.share;
        return r;
    }
    __device__ __forceinline__ void keep(const PagedArgs& p, int j, const PagedJob& r)
    {
        if (p.mark && blockIdx.x == 0 && !p.seq_start && !r.prefix && r.count == 0)
            for (int h = 0; h < p.heads; h++) p.own[(size_t)j * p.heads + h] = make_int4(0, 0, 0, 0);
        spans[j] = make_int4(r.first, r.count, r.prefix ? r.seq : r.from, r.to);
    }
    // Job j, once the plan is built.
    __device__ __forceinline__ PagedJob known(const PagedArgs& p, int j) const
    {
        const int4 s = spans[j];
        PagedJob r;
        r.prefix = j >= p.batch;
        r.first = s.x; r.count = s.y; r.from = r.prefix ? 0 : s.z; r.to = s.w;
        r.rows = r.count * p.share;
        r.joined = r.prefix || r.from > 0;
        r.seq = r.prefix ? s.z : j;
        return r;
    }
    // units(job): those of one of its items, 0 for a job that is not this kernel's.  All threads of the CTA; returns the units in all.
    template <int kThreads, class Units>
    __device__ int build(const PagedArgs& p, int* shared, int* err, Units units)
    {
        __shared__ int s_warp[kThreads / 32], s_total;
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        jobs = p.batch + p.groups;
        spans = reinterpret_cast<int4*>(shared);
        cum = shared + 4 * jobs;
        group_len = cum + jobs + 1;
        if (p.groups) {
            // What a group shares is its members' that bring tokens: their least length, the first one's pages.  (Another's row of the table may name anything.)
            for (int g = tid; g < p.groups; g += kThreads) {
                group_len[g] = min(max(p.group_pages[g], 0), p.max_pages) * p.page;
                spans[p.batch + g].z = p.batch;
            }
            __syncthreads();
            for (int b = tid; b < p.batch; b += kThreads) {
                const int g = group_of(p, b);
                if (g < 0) continue;
                const PagedSpan s = span(p, b, err);
                if (s.count > 0) {
                    atomicMin(&group_len[g], s.held);
                    atomicMin(&spans[p.batch + g].z, b);
                }
            }
            __syncthreads();
            for (int g = tid; g < p.groups; g += kThreads) {
                int s0, s1;
                members(p, g, s0, s1);
                group_len[g] = s1 - s0 > 1 && spans[p.batch + g].z < p.batch ? group_len[g] / p.page * p.page : 0;
            }
            __syncthreads();
        }
        int run = 0;
#pragma unroll 1
        for (int j0 = 0; j0 < jobs; j0 += kThreads) {
            const int j = j0 + tid;
            int n = 0;
            if (j < jobs) {
                const PagedJob r = job(p, j, err);
                keep(p, j, r);
                if (r.rows > 0 && r.to > r.from) n = units(r) * p.kv_heads;
            }
            int up = n;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int v = __shfl_up_sync(0xFFFFFFFFu, up, o);
                if (lane >= o) up += v;
            }
            if (lane == 31) s_warp[warp] = up;
            __syncthreads();
            int before = run;
            for (int w = 0; w < warp; w++) before += s_warp[w];
            if (j < jobs) cum[j] = before + up - n;
            if (tid == kThreads - 1) s_total = before + up;
            __syncthreads();
            run = s_total;
        }
        if (tid == 0) cum[jobs] = run;
        __syncthreads();
        return run;
    }
    // The job that unit u belongs to.
    __device__ __forceinline__ int find(int u) const
    {
        int lo = 0, hi = jobs;                          // cum[lo] <= u < cum[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (cum[mid] <= u) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};

// Units dealt to CTAs in equal runs, the first ones a unit longer where they do not come out even.
struct PagedDeal {
    int each, longer;               // units of a run; how many runs have one more
    __device__ __forceinline__ PagedDeal(int total, int ctas) : each(total / ctas), longer(total - total / ctas * ctas) {}
    __device__ __forceinline__ int first(int cta) const { return cta * each + min(cta, longer); }
    __device__ __forceinline__ int cta_of(int u) const { return u < longer * (each + 1) ? u / (each + 1) : longer + (u - longer * (each + 1)) / each; }
};

// The tokens that belong to no sequence, strided over `lanes` threads of every CTA: k_paged_join passes them over.  (Where every sequence brings one token, PagedPlan::build has
// seen to sequences that are skipped.)
__device__ __forceinline__ void mark_tokens(const PagedArgs& p, int lane, int lanes, int* err)
{
    for (int t = (p.seq_start ? 0 : p.batch) + blockIdx.x * lanes + lane; t < p.n_tokens; t += gridDim.x * lanes) {
        bool mine = false;
        if (p.seq_start) {
            int lo = 0, hi = p.batch;                   // the last sequence that starts at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (p.seq_start[mid] <= t) lo = mid;
                else hi = mid;
            }
            const PagedSpan s = PagedPlan::span(p, lo, err);
            mine = s.count > 0 && s.first <= t && t < s.first + s.count;
        }
        if (!mine)
            for (int h = 0; h < p.heads; h++) p.own[(size_t)t * p.heads + h] = make_int4(0, 0, 0, 0);
    }
}

#endif
}  // namespace bpdq
