// Attention over a paged cache for jobs of many rows (paged_attention.cuh), on tcgen05: portions of prompts, and prefixes that many sequences share.
//
// An item is up to 256 rows of a key head (two tiles of 128, whole tokens each; row = (token, query head)) against blocks of 128 keys; CTAs take equal runs
// of blocks of all items.  Two streams of work alternate on the tensor pipe, so that one's products run under the other's softmax: the item's two tiles, or, of an
// item with one, its even and odd blocks, whose sums meet at the end.
//   warp 0      tiled bulk copies of queries, and of keys and values page by page, into 128-byte-swizzled shared memory
//   warp 1      tensor memory, MMAs: after a step's O += P V its stream's next scores S = Q K^T
//   warps 4-11  softmax, four per stream, a thread per row; weights go back to tensor memory over the scores they came from.  (The tensor pipe works
//               its products off in the order in which they are issued: scores do not overtake the product that reads the weights beneath them.)
// O stays in tensor memory and is rescaled only when a row's maximum has grown by more than 2^8 since the last time.  Weights are rounded to the cache's type: half
// a step (2^-9 of a bf16 weight on average) of each, which the sum over keys averages to below the result's own rounding.  fp32 activations bring queries and weights as two
// fp16 numbers each: four products where 16 bits take two, and one tile per item.
#include "paged_attention.cuh"
#include "tcgen05_device.cuh"
#include "mma_device.cuh"

#include <type_traits>

namespace bpdq {

constexpr int kPtRows = 128, kPtKeys = 128, kPtPiece = 128 * 64 * 2;        // rows of a tile, keys of a block, bytes of 128 rows x 64 columns
constexpr int kPtWarps = 8, kPtThreads = 32 * (4 + kPtWarps);          // three groups of four warps, which have registers of their own size
constexpr float kPtGrowth = 8.0f;

template <int DP> struct PtShape {
    static constexpr int halves = DP / 64, depth = DP == 64 ? 4 : 2;        // blocks of keys (and of values) in shared memory
    static constexpr int q = 0, k = 2 * halves * kPtPiece, v = k + depth * halves * kPtPiece, end = v + depth * halves * kPtPiece;
};

__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, float* v)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
          "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]),
          "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename K> __device__ __forceinline__ uint32_t pack_16(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_16<bf16>(float a, float b) { return pack_bf16(a, b); }
template <> __device__ __forceinline__ uint32_t pack_16<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void split_f16(float v0, float v1, uint32_t& hi, uint32_t& lo)
{
    const __half2 h = __floats2half2_rn(v0, v1);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_16<__half>(v0 - f.x, v1 - f.y);
}

// An item: a key head's rows of some tokens of a job.
struct PtItem {
    PagedJob job;
    int j, head, begin, end;            // units: its blocks of keys
    int t0, tokens;                     // the first token, within the job, and how many
    int from, blocks;                   // position of the first key
};

template <typename A, typename K, int DP>
__global__ void __launch_bounds__(kPtThreads, 1)
k_paged_tile(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const PagedArgs p, int* err)
{
    using Shape = PtShape<DP>;
    constexpr bool f32 = sizeof(A) == 4;
    constexpr int kHalves = Shape::halves, kDepth = Shape::depth;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t q_full, q_empty, k_full[kDepth], k_empty[kDepth], v_full[kDepth], v_empty[kDepth], s_full[2], p_full[2], o_done[2], ml_ready, o1_free;
    __shared__ uint32_t tmem_slot;
    __shared__ unsigned short s_missing[8];             // of a block: groups of eight keys without a page; softmax is two blocks behind the copies' kDepth at most
    __shared__ float2 s_ml[kPtRows];
    __shared__ float s_factor[kPtRows];
    uint8_t* base = raw + (((smem_addr(raw) + 1023) & ~1023u) - smem_addr(raw));
    uint8_t *sq = base + Shape::q, *sk = base + Shape::k, *sv = base + Shape::v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        mbar_init(&q_full, f32 ? kPtWarps : 1);
        mbar_init(&q_empty, 1);
        for (int i = 0; i < kDepth; i++) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
        for (int i = 0; i < 2; i++) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_done[i], 1); }
        mbar_init(&ml_ready, 4);
        mbar_init(&o1_free, 4);
        mbar_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;                    // scores of stream s in columns 128 s on, its sums in columns 256 + 128 s on
    pdl_wait();
    pdl_launch_dependents();

    const int tile_tokens = kPtRows / p.share, item_tokens = f32 ? tile_tokens : 2 * tile_tokens;
    // blocks of the item that starts with token t0 of a job
    auto blocks_of = [&](const PagedJob& r, int t0) {
        const int to = r.prefix ? r.to : r.to - r.count + min(t0 + item_tokens, r.count);
        return (to - r.from + kPtKeys - 1) / kPtKeys;
    };
    PagedPlan plan = {};
    const int total = plan.build<kPtThreads>(p, reinterpret_cast<int*>(base + Shape::end), err, [&](const PagedJob& r) {
        if (r.rows <= p.split_rows) return 0;
        int n = 0;
        for (int t = 0; t < r.count; t += item_tokens) n += blocks_of(r, t);
        return n;
    });
    const int ctas = max(1, min((int)gridDim.x, total)), cta = blockIdx.x;
    const PagedDeal deal(total, ctas);
    const int u0 = cta < ctas ? deal.first(cta) : total, u1 = cta < ctas ? deal.first(cta + 1) : total;
    auto open = [&](PtItem& it, int u, bool again) {
        if (!again || u >= plan.cum[it.j + 1]) {
            it.j = plan.find(u);
            it.job = plan.known(p, it.j);
        }
        const int per = (plan.cum[it.j + 1] - plan.cum[it.j]) / p.kv_heads;
        int at = u - plan.cum[it.j];
        it.head = at / per;
        at -= it.head * per;
        it.t0 = 0;
        int n = blocks_of(it.job, 0);
        while (at >= n) {
            at -= n;
            it.t0 += item_tokens;
            n = blocks_of(it.job, it.t0);
        }
        it.begin = u - at;
        it.end = it.begin + n;
        it.tokens = min(item_tokens, it.job.count - it.t0);
        it.from = it.job.from + at * kPtKeys;
        it.blocks = min(it.end, u1) - u;
    };
    // two tiles, each against every block; or one, its blocks in turn
    auto is_dual = [&](const PtItem& it) { return !f32 && it.tokens > tile_tokens; };

    // of 168 registers a thread at launch: 4 * 56 + 8 * 224 = 12 * 168
    if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---------------- softmax
        const int s = (warp - 4) >> 2, quarter = warp & 3, r = 32 * quarter + lane;
        const uint32_t lanes = (uint32_t)(32 * quarter) << 16, ts = tmem + lanes + 128 * s, to_ = tmem + lanes + 256;
        PtItem it = {};
        int nk = 0, steps = 0, items = 0, meets = 0;
        bool ok = true;
        for (int u = u0; ok && u < u1; u += it.blocks, items++) {
            open(it, u, u != u0);
            const bool dual = is_dual(it);
            const int n_steps = dual ? 2 * it.blocks : it.blocks;
            const int mine = (dual ? s * tile_tokens : 0) + r / p.share;            // the row's token, within the item
            const bool live = r < tile_tokens * p.share && mine < it.tokens;
            const int tok = it.job.first + it.t0 + mine, h = it.head * p.share + r % p.share;
            // positions below `limit` are the row's to see
            const int limit = it.job.prefix ? it.job.to : it.job.to - it.job.count + (live ? it.t0 + mine : it.job.count - 1) + 1;
            float f = p.scale * 1.44269504088896341f;
            if constexpr (f32) {
                // queries as two fp16 numbers: a power of two brings a row's largest entry to 1 .. 2; two neighbouring threads per row
                const int i = tid - 128, row = i >> 1, part = i & 1, m = row / p.share;
                const bool there = row < tile_tokens * p.share && m < it.tokens;
                const float* q = static_cast<const float*>(p.q) + (size_t)(it.job.first + it.t0 + (there ? m : 0)) * p.ld_q + (it.head * p.share + (there ? row % p.share : 0)) * p.dim;
                float big = 0.0f;
                for (int d = part * 4; d < p.dim; d += 8) {
                    const float4 x = there ? *reinterpret_cast<const float4*>(q + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    big = fmaxf(fmaxf(big, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
                }
                big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
                const int e = big > 0.0f && big < INFINITY ? min(max(ilogbf(big), -100), 100) : 0;
                const float down = __int_as_float((127 - e) << 23);
                if (part == 0) s_factor[row] = __int_as_float((127 + e) << 23);
                for (int d = part * 8; d < DP; d += 16) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float4 x = there && d + 4 * j < p.dim ? *reinterpret_cast<const float4*>(q + d + 4 * j) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        split_f16(x.x * down, x.y * down, hi[2 * j], lo[2 * j]);
                        split_f16(x.z * down, x.w * down, hi[2 * j + 1], lo[2 * j + 1]);
                    }
                    uint8_t* at = sq + (d >> 6) * kPtPiece + row * 128 + ((((d >> 3) & 7) ^ (row & 7)) << 4);
                    *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(at + kHalves * kPtPiece) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full);
                // all factors are written
                if (!mbar_wait_bounded(&q_full, (uint32_t)items & 1u, err, 91)) { ok = false; break; }
                f *= s_factor[r];
            }
            const float sign = f < 0.0f ? -1.0f : 1.0f;
            f = fabsf(f);
            float top = -INFINITY, sum = 0.0f;          // in units of log2
            int n = s;
            for (; n < n_steps; n += 2, steps++) {
                const int b = dual ? n >> 1 : n, key = it.from + b * kPtKeys;
                if (!mbar_wait_bounded(&s_full[s], (uint32_t)steps & 1u, err, 92)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float v[128];
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld_32(ts + 32 * c, v + 32 * c);
                tmem_loaded();
                const unsigned missing = s_missing[(nk + b) & 7];
                const bool edge = __any_sync(0xFFFFFFFFu, key + kPtKeys > limit || missing);
                float ff = f;
                if (p.cap > 0.0f) {
                    const float in = sign * f * 0.69314718055994531f;
#pragma unroll
                    for (int j = 0; j < 128; j++) v[j] = capped<f32>(v[j] * in, p.cap) * 1.44269504088896341f;
                    ff = 1.0f;
                } else if (sign < 0.0f) {
#pragma unroll
                    for (int j = 0; j < 128; j++) v[j] = -v[j];
                }
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 128; j++) v[j] = key + j < limit && !(missing >> (j >> 3) & 1u) ? v[j] * ff : -INFINITY;
                    ff = 1.0f;
                }
                float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int j = 4; j < 128; j++) m4[j & 3] = fmaxf(m4[j & 3], v[j]);
                const float now = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * ff;
                const bool grown = now > top + kPtGrowth;
                if (n > 1 && __any_sync(0xFFFFFFFFu, grown)) {
                    if (!mbar_wait_bounded(&o_done[s], (uint32_t)(steps - 1) & 1u, err, 93)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const float down = grown ? ex2(top - now) : 1.0f;
                    sum *= down;
#pragma unroll
                    for (int c = 0; c < DP; c += 16) {
                        int ov[16];
                        tmem_ld(to_ + 128 * s + c, ov);
                        tmem_loaded();
                        uint32_t st[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) st[j] = __float_as_uint(__int_as_float(ov[j]) * down);
                        tmem_st(to_ + 128 * s + c, st);
                    }
                }
                if (grown) top = now;
                const float zero = top == -INFINITY ? 0.0f : top;
                float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < 4; c++) {
#pragma unroll
                    for (int j = 32 * c; j < 32 * c + 32; j++) {
                        v[j] = ex2(fmaf(v[j], ff, -zero));
                        part[j & 3] += v[j];
                    }
                    uint32_t hi[16];
                    if constexpr (f32) {
                        uint32_t lo[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) split_f16(v[32 * c + 2 * j], v[32 * c + 2 * j + 1], hi[j], lo[j]);
                        tmem_st(ts + 64 + 16 * c, lo);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j++) hi[j] = pack_16<K>(v[32 * c + 2 * j], v[32 * c + 2 * j + 1]);
                    }
                    tmem_st(ts + 16 * c, hi);
                }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
                if (key + kPtKeys > it.job.to || missing) {
                    // whatever lies in places that hold no position must not meet a weight, not even one of 0: a thread per key
                    const int slot = (nk + b) % kDepth;
                    if (!mbar_wait_bounded(&v_full[slot], (uint32_t)((nk + b) / kDepth) & 1u, err, 94)) { ok = false; break; }
                    if (key + r >= it.job.to || (missing >> (r >> 3) & 1u))
#pragma unroll
                        for (int c = 0; c < kHalves * 8; c++)
                            *reinterpret_cast<uint4*>(sv + (slot * kHalves + (c >> 3)) * kPtPiece + r * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                tmem_stored();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[s]);
            }
            if (!ok) break;
            nk += it.blocks;
            // ---- the item's sums, or this CTA's part of them
            const bool any = n_steps > s;               // (a single block has no odd ones)
            if (any && !mbar_wait_bounded(&o_done[s], (uint32_t)(steps - 1) & 1u, err, 95)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float w0 = 1.0f, w1 = 0.0f;
            const bool both = !dual && n_steps > 1;
            if (!dual) {
                if (s == 1) s_ml[r] = make_float2(top, sum);
                __syncwarp();
                if (s == 1) {
                    if (lane == 0) mbar_arrive(&ml_ready);
                    // its sums are read by the other stream's threads
                    if (!mbar_wait_bounded(&o1_free, (uint32_t)meets & 1u, err, 96)) { ok = false; break; }
                    meets++;
                    continue;
                }
                if (!mbar_wait_bounded(&ml_ready, (uint32_t)meets & 1u, err, 97)) { ok = false; break; }
                meets++;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (both) {
                    const float2 odd = s_ml[r];
                    const float most = fmaxf(top, odd.x), zero = most == -INFINITY ? 0.0f : most;
                    w0 = ex2(top - zero);
                    w1 = ex2(odd.x - zero);
                    sum = w0 * sum + w1 * odd.y;
                    top = most;
                }
            }
            const bool starts = it.begin >= u0, all = starts && it.end <= u1;
            const size_t row = (size_t)tok * p.heads + h;
            const int in_part = (dual ? s * kPtRows : 0) + r;
            const size_t at = all ? row : (size_t)(2 * cta + starts) * kTileRows + in_part;
            const bool direct = all && !it.job.joined;
            float* dst = (!all ? p.tile_o : (it.job.prefix ? p.prefix_o : p.own_o)) + at * DP;
            A* o = static_cast<A*>(p.o) + (size_t)tok * p.ld_o + h * p.dim;
            if (direct) {
                const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
                w0 *= inv;
                w1 *= inv;
            }
#pragma unroll
            for (int c = 0; c < DP; c += 16) {
                int ov[16];
                float x[16];
                tmem_ld(to_ + 128 * s + c, ov);
                tmem_loaded();
#pragma unroll
                for (int j = 0; j < 16; j++) x[j] = __int_as_float(ov[j]) * w0;
                if (both) {
                    tmem_ld(to_ + 128 + c, ov);
                    tmem_loaded();
#pragma unroll
                    for (int j = 0; j < 16; j++) x[j] = fmaf(__int_as_float(ov[j]), w1, x[j]);
                }
                if (!live) continue;
                if (!direct) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(dst + c + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                } else if constexpr (f32) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4)
                        if (c + j < p.dim) *reinterpret_cast<float4*>(o + c + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; j += 8)
                        if (c + j < p.dim)
                            *reinterpret_cast<uint4*>(o + c + j) = make_uint4(pack_16<K>(x[j], x[j + 1]), pack_16<K>(x[j + 2], x[j + 3]), pack_16<K>(x[j + 4], x[j + 5]),
                                                                              pack_16<K>(x[j + 6], x[j + 7]));
                }
            }
            if (live) {
                if (!direct) (!all ? p.tile_ml : (it.job.prefix ? p.prefix_ml : p.own_ml))[at] = make_float2(top, sum);
                if (starts) {
                    const int end = all ? cta : deal.cta_of(it.end - 1);
                    (it.job.prefix ? p.prefix : p.own)[row] = make_int4(cta, end - cta + 1, in_part, kJoinTile | (it.job.joined && !it.job.prefix ? kJoinPrefix : 0));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (!dual && lane == 0) mbar_arrive(&o1_free);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
        // ---------------- copies
        PtItem it = {};
        int nk = 0, items = 0;
        bool ok = true;
        for (int u = u0; ok && u < u1; u += it.blocks, items++) {
            open(it, u, u != u0);
            const bool dual = is_dual(it);
            if (!f32) {
                if (items && !mbar_wait_bounded(&q_empty, (uint32_t)(items - 1) & 1u, err, 84)) break;
                if (lane == 0) {
                    mbar_expect_tx(&q_full, (uint32_t)((dual ? 2 : 1) * kHalves * tile_tokens * p.share * 128));
                    for (int s = 0; s < (dual ? 2 : 1); s++)
#pragma unroll
                        for (int h = 0; h < kHalves; h++) tma_rows_3d(sq + (s * kHalves + h) * kPtPiece, &qmap, 64 * h, it.head * p.share, it.job.first + it.t0 + s * tile_tokens, &q_full);
                }
            }
            // a lane per page (box) of a block
            const int box_rows = p.page < kPtKeys ? p.page : kPtKeys, boxes = kPtKeys / box_rows;
            const int* table = p.table + (size_t)it.job.seq * p.max_pages;
            auto entry_of = [&](int b) {
                const int key = it.from + b * kPtKeys + lane * box_rows;
                return lane < boxes && key < it.job.to ? table[key >> p.log_page] : -2;
            };
            int entry = entry_of(0);
            for (int b = 0; b < it.blocks; b++, nk++) {
                const int slot = nk % kDepth, now = entry;
                if (b + 1 < it.blocks) entry = entry_of(b + 1);
                const bool have = now >= 0 && now < p.n_pages;
                if (now != -2 && !have) report(err, 82);
                const unsigned who = __ballot_sync(0xFFFFFFFFu, have);
                const uint32_t bytes = (uint32_t)(__popc(who) * box_rows * 128 * kHalves);
                if (nk >= kDepth && !mbar_wait_bounded(&k_empty[slot], (uint32_t)(nk / kDepth - 1) & 1u, err, 85)) { ok = false; break; }
                if (lane == 0) {
                    unsigned missing = 0;
                    for (int g = 0; g < 16; g++)
                        if (!(who >> (g * 8 / box_rows) & 1u)) missing |= 1u << g;
                    s_missing[nk & 7] = (unsigned short)missing;
                    mbar_expect_tx(&k_full[slot], bytes);
                }
                __syncwarp();
                const int row = (it.from + b * kPtKeys + lane * box_rows) & (p.page - 1);
                if (have)
                    for (int h = 0; h < (p.both ? 1 : kHalves); h++)
                        tma_page(smem_addr(sk + (slot * kHalves + h) * kPtPiece + lane * box_rows * 128), &kmap, 64 * h, row, it.head, now, smem_addr(&k_full[slot]));
                if (nk >= kDepth && !mbar_wait_bounded(&v_empty[slot], (uint32_t)(nk / kDepth - 1) & 1u, err, 86)) { ok = false; break; }
                if (lane == 0) mbar_expect_tx(&v_full[slot], bytes);
                __syncwarp();
                if (have)
                    for (int h = 0; h < (p.both ? 1 : kHalves); h++)
                        tma_page(smem_addr(sv + (slot * kHalves + h) * kPtPiece + lane * box_rows * 128), &vmap, 64 * h, row, it.head, now, smem_addr(&v_full[slot]));
            }
        }
        } else if (warp == 1) {
        // ---------------- MMAs
        if (elect_one()) {
            constexpr uint32_t kind = sizeof(K) == 2 && std::is_same<K, bf16>::value ? 1u : 0u;
            constexpr uint32_t fmt = (1u << 4) | (kind << 7) | (kind << 10) | ((uint32_t)(kPtRows >> 4) << 24);
            constexpr uint32_t idesc_s = fmt | ((uint32_t)(kPtKeys >> 3) << 17), idesc_o = fmt | (1u << 16) | ((uint32_t)(DP >> 3) << 17);
            PtItem it = {};
            int nk = 0, items = 0, steps[2] = {0, 0};
            bool ok = true;
            for (int u = u0; ok && u < u1; u += it.blocks, items++) {
                open(it, u, u != u0);
                const bool dual = is_dual(it);
                const int n_steps = dual ? 2 * it.blocks : it.blocks;
                auto block_of = [&](int n) { return dual ? n >> 1 : n; };
                if (!(ok = mbar_wait_bounded(&q_full, (uint32_t)items & 1u, err, 87))) break;
                auto scores = [&](int n) {
                    const int s = n & 1, at = nk + block_of(n), slot = at % kDepth;
                    if (!mbar_wait_bounded(&k_full[slot], (uint32_t)(at / kDepth) & 1u, err, 88)) return false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t qd = swizzled_desc(smem_addr(sq + (dual ? s : 0) * kHalves * kPtPiece)), kd = swizzled_desc(smem_addr(sk + slot * kHalves * kPtPiece));
#pragma unroll
                    for (int part = 0; part < (f32 ? 2 : 1); part++)
#pragma unroll
                        for (int h = 0; h < kHalves; h++)
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                umma_bf16_ss(tmem + 128 * s, qd + (uint64_t)((part * kHalves + h) * (kPtPiece >> 4) + 2 * k), kd + (uint64_t)(h * (kPtPiece >> 4) + 2 * k), idesc_s,
                                             part | h | k ? 1u : 0u);
                    umma_commit(&s_full[s]);
                    if (!dual || s == 1) umma_commit(&k_empty[slot]);
                    if (n == n_steps - 1) umma_commit(&q_empty);
                    return true;
                };
                ok = scores(0) && (n_steps < 2 || scores(1));
                for (int n = 0; ok && n < n_steps; n++) {
                    const int s = n & 1, at = nk + block_of(n), slot = at % kDepth;
                    if (!(ok = mbar_wait_bounded(&v_full[slot], (uint32_t)(at / kDepth) & 1u, err, 89) && mbar_wait_bounded(&p_full[s], (uint32_t)steps[s] & 1u, err, 90))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t vd = swizzled_desc_mn(smem_addr(sv + slot * kHalves * kPtPiece), kPtPiece);
                    const uint32_t o = tmem + 256 + 128 * s, w = tmem + 128 * s;
#pragma unroll
                    for (int k = 0; k < kPtKeys / 16; k++) {
                        if (f32) umma_bf16_ts(o, w + 64 + 8 * k, vd + (uint64_t)(k * 128), idesc_o, (n > 1) | k ? 1u : 0u);
                        umma_bf16_ts(o, w + 8 * k, vd + (uint64_t)(k * 128), idesc_o, f32 || (n > 1) | k ? 1u : 0u);
                    }
                    umma_commit(&o_done[s]);
                    if (!dual || s == 1) umma_commit(&v_empty[slot]);
                    steps[s]++;
                    if (n + 2 < n_steps) ok = scores(n + 2);
                }
                nk += it.blocks;
            }
        }
        __syncwarp();
        }
    }
    if (p.mark && warp < 4) mark_tokens(p, tid, 128, err);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <typename A, typename K, int DP>
static int launch_tile(PagedArgs a, const bpdq_paged_kv& kv, int ctas, cudaStream_t s)
{
    CUtensorMap qmap, kmap, vmap;
    int rc;
    if ((rc = paged_map(&kmap, kv.k, kv, kPtKeys)) || (rc = paged_map(&vmap, kv.v, kv, kPtKeys))) return rc;
    a.both = paged_both(kv, kPtKeys);
    qmap = kmap;                // (of fp32 queries: not used)
    if (sizeof(A) == 2) {
        const int tokens = kPtRows / a.share;
        if ((rc = bf16_map(&qmap, a.q, a.dim, a.heads, a.dim, a.share, a.n_tokens, a.ld_q, tokens))) return rc;
    }
    if ((rc = allow_smem<k_paged_tile<A, K, DP>>(221 * 1024))) return rc;
    const size_t smem = 1024 + PtShape<DP>::end + PagedPlan::size(a);
    return launch_ordered(k_paged_tile<A, K, DP>, dim3((unsigned)ctas), kPtThreads, smem, s, qmap, kmap, vmap, a, device_error_flag());
}

int paged_tile(const PagedArgs& a, const bpdq_paged_kv& kv, int ctas, cudaStream_t s)
{
    const bool wide = a.dim > 64;
    if (kv.act_type == BPDQ_TYPE_F32) return wide ? launch_tile<float, __half, 128>(a, kv, ctas, s) : launch_tile<float, __half, 64>(a, kv, ctas, s);
    if (kv.kv_type == BPDQ_TYPE_F16) return wide ? launch_tile<__half, __half, 128>(a, kv, ctas, s) : launch_tile<__half, __half, 64>(a, kv, ctas, s);
    return wide ? launch_tile<bf16, bf16, 128>(a, kv, ctas, s) : launch_tile<bf16, bf16, 64>(a, kv, ctas, s);
}

}  // namespace bpdq
