// Attention over a paged cache for jobs of many rows (paged_attention.cuh), on tcgen05: portions of prompts, and prefixes that many sequences share.
//
// An item is up to 256 rows of a key head (two tiles of 128, whole tokens each; row = (token, query head)) against blocks of 128 keys; CTAs take equal runs
// of blocks of all items.  Two streams of work share the tensor pipe: the item's two tiles, or, of an item with one, the halves of every block, whose sums meet at the
// end.  A step is 64 keys; a stream has two sets of scores, so that products run under the softmax of the step before.
//   warps 0, 2  tiled bulk copies of queries and keys, and of values, page by page, into 128-byte-swizzled shared memory
//   warps 1, 3  tensor memory, MMAs of a stream each: after a step's O += P V the scores S = Q K^T of the step after next
//   warps 4-11  softmax, four per stream, a thread per row; weights go back to tensor memory over the scores they came from.  (The tensor pipe works
//               its products off in the order in which they are issued: scores do not overtake the product that reads the weights beneath them.)
// (Every barrier of a stream's steps comes twice, for even and odd ones: a role may be two steps ahead of another.)
// The streams take their exponentials in turns, the next one from the middle of the other's on: both at once would wait for the special function unit together and leave it
// idle together.  (One prompt of 8000 tokens: 522 us, one whole step after the other 524, no turns 560; every eighth, fourth or second pair by a polynomial instead of
// that unit 530, 550, 603: instructions are scarcer; the scores of a block's 128 keys in one product, into both sets, once both are free 627.)
// O stays in tensor memory and is rescaled only when a row's maximum has grown by much since the last time.  Weights are rounded to the cache's type: half
// a step (2^-9 of a bf16 weight on average) of each, which the sum over keys averages to below the result's own rounding.  fp32 activations bring queries and weights as two
// fp16 numbers each: four products where 16 bits take two, and one tile per item.
// One prompt of 8000 tokens, 32 heads on 8 of 128 in bf16: 526 us with the launches behind it, 997 TFLOP/s of a measured 1688; three portions of 2000 after up to 2000: 136 us, 14 of it
// the join and 4 the kernel for few rows, which has nothing to do.  Bound by what
// the streams and the tensor pipe hand to each other: some 2400 cycles for a step of both streams, 1024 of them products.  64 tokens on a prefix of 16000 (8 items on 148
// CTAs): 40 us, half of it until the first scores.
#include "paged_attention.cuh"
#include "tcgen05_device.cuh"
#include "mma_device.cuh"

#include <type_traits>

namespace bpdq {

constexpr int kPtRows = 128, kPtKeys = 128, kPtStep = 64, kPtPiece = 128 * 64 * 2;     // rows of a tile, keys of a block and of a step, bytes of 128 rows x 64 columns
constexpr int kPtWarps = 8, kPtThreads = 32 * (4 + kPtWarps);          // three groups of four warps, which have registers of their own size
// By activations.  O is rescaled when a row's maximum has grown by more than 2^growth since the last time.  fp16 ends at 2^16 and rounds what is below 2^-25 to 0: fp16 weights are
// held 2^shift times as large, growth + shift < 16, so that each is off by 2^(-25 - shift) of the largest at most, or by its rounding.  (Growth, shift 4, 11 for 8, 7: three fp16 prompts of
// 2000 after 2000, 32 heads on 8 of 128, 139.1 us for 132.2, of fp32 ones of 1000 156.7 for 155.6; 0, 15: 159.2 and 159.5.)
template <typename A> constexpr float kPtGrowth = 8.0f;
template <> constexpr float kPtGrowth<float> = 4.0f;
template <typename A> constexpr float kPtShift = 0.0f;
template <> constexpr float kPtShift<__half> = 7.0f;
template <> constexpr float kPtShift<float> = 11.0f;
// The tensor pipe cuts off what does not fit fp32 of each of its sums, always toward zero: 6000 keys in one go are 4e-6 short.  With fp32 activations a stream
// puts its sums aside every so many steps, added to the last ones as fp32 numbers round, and begins anew.  (Prompts of 1500 after 4000, error against 64 bits, us: every two
// steps 0.9e-6, 253; four 1.1e-6, 229; eight 1.6e-6, 213.  Elementary operations in fp32: 1.1e-6.)
constexpr int kPtFold = 4;

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

// Two fp32 numbers at once.
__device__ __forceinline__ float2 fma_two(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add_two(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// An item: a key head's rows of some tokens of a job.
struct PtItem {
    PagedJob job;
    int head, begin, end;               // units: its blocks of keys
    int t0, tokens;                     // the first token, within the job, and how many
    int from, blocks;                   // this CTA's part of it: position of the first key, blocks (0: there are no more items)
    bool starts;                        // it has the item's first block
};
constexpr int kPtItems = 4;             // a warp finds the items and puts them here; the others take them
constexpr int kPtTakers = 1 + 2 + 8;
// An item's beginning and end (queries, a pipe that runs empty, results) take about as long as two blocks: it counts two units more than it has blocks, its first ones.
// (One prompt of 8000 tokens, 32 heads on 8 of 128: none 692 us, one 595, two 555, three 555, eight 592, all with a polynomial for every fourth pair of exponentials.)
constexpr int kPtExtra = 2;

template <typename A, typename K, int DP, int kCap>
__global__ void __launch_bounds__(kPtThreads, 1)
k_paged_tile(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const PagedArgs p, int* err)
{
    using Shape = PtShape<DP>;
    constexpr bool f32 = sizeof(A) == 4;
    constexpr int kHalves = Shape::halves, kDepth = Shape::depth;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t q_full, q_empty, k_full[kDepth], k_empty[kDepth], v_full[kDepth], v_empty[kDepth], s_full[2][2], p_full[2][2], o_done[2][2], ml_ready, o1_free, turn[2], idle[2];
    __shared__ uint64_t item_full[kPtItems], item_empty[kPtItems];
    __shared__ PtItem items[kPtItems];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;                             // a role has
    __shared__ unsigned short s_missing[8];             // of a block: groups of eight keys without a page; softmax is two blocks behind the copies' kDepth at most
    __shared__ float2 s_ml[kPtRows];
    __shared__ uint8_t* s_row[2][kPtRows];              // where rows go; null: nowhere
    __shared__ float s_factor[kPtRows], s_aside[kPtRows];
    uint8_t* base = raw + (((smem_addr(raw) + 1023) & ~1023u) - smem_addr(raw));
    uint8_t *sq = base + Shape::q, *sk = base + Shape::k, *sv = base + Shape::v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
        if (!f32) asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
    }
    if (tid == 0) {
        gave_up = 0;
        mbar_init(&q_full, f32 ? kPtWarps : 1);
        mbar_init(&q_empty, kPtWarps);
        for (int i = 0; i < kDepth; i++) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 2); mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 2); }
        for (int i = 0; i < 2; i++) { mbar_init(&s_full[0][i], 1); mbar_init(&s_full[1][i], 1); mbar_init(&p_full[0][i], 4); mbar_init(&p_full[1][i], 4); mbar_init(&o_done[0][i], 1); mbar_init(&o_done[1][i], 1); }
        for (int i = 0; i < kPtItems; i++) { mbar_init(&item_full[i], 1); mbar_init(&item_empty[i], kPtTakers); }
        mbar_init(&ml_ready, 4);
        mbar_init(&o1_free, 4);
        mbar_init(&turn[0], 4); mbar_init(&turn[1], 4);
        mbar_init(&idle[0], 1); mbar_init(&idle[1], 1);
        mbar_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp >= 8 && lane == 0) mbar_arrive(&turn[0]);          // the first stream begins
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;                    // scores of stream s in columns 128 s and 128 s + 64 on, its sums in columns 256 + 128 s on
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
        for (int t = 0; t < r.count; t += item_tokens) n += blocks_of(r, t) + kPtExtra;
        return n;
    });
    const int ctas = max(1, min((int)gridDim.x, total)), cta = blockIdx.x;
    const PagedDeal deal(total, ctas);
    const int u0 = cta < ctas ? deal.first(cta) : total, u1 = cta < ctas ? deal.first(cta + 1) : total;
    // Item n of this CTA, by a warp (or the thread that issues products).
    auto take = [&](PtItem& it, int n, bool one) {
        const int slot = n % kPtItems;
        if (!mbar_wait_bounded(&item_full[slot], (uint32_t)(n / kPtItems) & 1u, err, 100)) return false;
        it = items[slot];
        if (!one) __syncwarp();
        if (one || lane == 0) mbar_arrive(&item_empty[slot]);
        return it.blocks > 0;
    };
    // Two tiles, each against every block, step t against half t % 2 of block t / 2; or one, stream s against half s of block t.
    auto is_dual = [&](const PtItem& it) { return !f32 && it.tokens > tile_tokens; };

    // of 168 registers a thread at launch: 4 * 56 + 8 * 224 = 12 * 168
    if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---------------- softmax
        const int s = (warp - 4) >> 2, quarter = warp & 3, r = 32 * quarter + lane;
        const uint32_t lanes = (uint32_t)(32 * quarter) << 16, to_ = tmem + lanes + 256;
        PtItem it = {};
        int nk = 0, steps = 0, taken = 0, meets = 0;
        bool ok = true;
        while (ok && take(it, taken, false)) {
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
                if (!mbar_wait_bounded(&q_full, (uint32_t)taken & 1u, err, 91)) { ok = false; break; }
                f *= s_factor[r];
            }
            const int least = __reduce_min_sync(0xFFFFFFFFu, limit);
            const bool negative = p.scale < 0.0f;
            float top = -INFINITY, sum = 0.0f;          // in units of log2
            float aside_top = -INFINITY;                // of the sums put aside
            float4* aside = f32 ? reinterpret_cast<float4*>(p.tile_sums) + ((size_t)(2 * cta + s) * (DP / 4)) * kPtRows + r : nullptr;
            for (int t = 0; t < n_steps; t++, steps++) {
                const int b = dual ? t >> 1 : t, half = dual ? t & 1 : s, key = it.from + b * kPtKeys + half * kPtStep;
                const uint32_t ts = tmem + lanes + 128 * s + 64 * (steps & 1);
                if (!mbar_wait_bounded(&s_full[s][steps & 1], (uint32_t)(steps >> 1) & 1u, err, 92)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float v[64];
                tmem_ld_32(ts, v);
                tmem_ld_32(ts + 32, v + 32);
                tmem_loaded();
                const unsigned missing = s_missing[(nk + b) & 7] >> (8 * half) & 0xFFu;
                // (where the scale is negative the largest score is the least product)
                const bool edge = key + kPtStep > least || missing || (!kCap && negative);
                float ff = f;
                if (kCap) {
                    const float in = f * 0.69314718055994531f;
#pragma unroll
                    for (int j = 0; j < 64; j++) v[j] = capped<f32, kCap>(v[j] * in, p.cap) * 1.44269504088896341f;
                    ff = 1.0f;
                }
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 64; j++) v[j] = key + j < limit && !(missing >> (j >> 3) & 1u) ? v[j] * ff : -INFINITY;
                    ff = 1.0f;
                }
                float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int j = 4; j < 64; j += 8) {
#pragma unroll
                    for (int i = 0; i < 4; i++) m4[i] = j + 4 < 64 ? fmaxf(fmaxf(m4[i], v[j + i]), v[(j + 4 + i) & 63]) : fmaxf(m4[i], v[j + i]);
                }
                const float now = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * ff;
                const bool grown = now > top + kPtGrowth<A>;
                const bool fold = f32 && t > 0 && t % kPtFold == 0;
                if (fold) {
                    if (!mbar_wait_bounded(&o_done[s][(steps - 1) & 1], (uint32_t)((steps - 1) >> 1) & 1u, err, 93)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const float down = aside_top == -INFINITY ? 0.0f : ex2(aside_top - top);
                    // (loads run a piece ahead)
                    float4 x[8] = {}, next[8];
                    auto last = [&](float4* x, int c) {
#pragma unroll
                        for (int j = 0; j < 8; j++) x[j] = __ldcg(aside + (c / 4 + j) * kPtRows);
                    };
                    if (t > kPtFold) last(x, 0);
#pragma unroll 1
                    for (int c = 0; c < DP; c += 32) {
                        float o[32];
                        tmem_ld_32(to_ + 128 * s + c, o);
                        if (t > kPtFold && c + 32 < DP) last(next, c + 32);
                        tmem_loaded();
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            __stcg(aside + (c / 4 + j) * kPtRows,
                                   make_float4(fmaf(x[j].x, down, o[4 * j]), fmaf(x[j].y, down, o[4 * j + 1]), fmaf(x[j].z, down, o[4 * j + 2]), fmaf(x[j].w, down, o[4 * j + 3])));
                        if (t > kPtFold)
#pragma unroll
                            for (int j = 0; j < 8; j++) x[j] = next[j];
                    }
                    aside_top = top;
                    if (grown) sum *= ex2(top - now);
                } else if (t > 0 && __any_sync(0xFFFFFFFFu, grown)) {
                    if (!mbar_wait_bounded(&o_done[s][(steps - 1) & 1], (uint32_t)((steps - 1) >> 1) & 1u, err, 93)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const float down = grown ? ex2(top - now) : 1.0f;
                    sum *= down;
#pragma unroll 1
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
                const float zero = top == -INFINITY ? 0.0f : top - kPtShift<A>;
                if (!mbar_wait_bounded(&turn[s], (uint32_t)steps & 1u, err, 98)) { ok = false; break; }
                const float2 f2 = make_float2(ff, ff), zero2 = make_float2(-zero, -zero);
                float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c = 0; c < 2; c++) {
#pragma unroll
                    for (int j = 32 * c; j < 32 * c + 32; j += 2) {
                        float2 x = fma_two(make_float2(v[j], v[j + 1]), f2, zero2);
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        part[(j >> 1) & 1] = add_two(part[(j >> 1) & 1], x);
                        v[j] = x.x;
                        v[j + 1] = x.y;
                    }
                    uint32_t hi[16];
                    if constexpr (f32) {
                        uint32_t lo[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) split_f16(v[32 * c + 2 * j], v[32 * c + 2 * j + 1], hi[j], lo[j]);
                        tmem_st(ts + 32 + 16 * c, lo);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j++) hi[j] = pack_16<K>(v[32 * c + 2 * j], v[32 * c + 2 * j + 1]);
                    }
                    tmem_st(ts + 16 * c, hi);
                    if (c == 0 && lane == 0) mbar_arrive(&turn[1 - s]);
                }
                sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
                if (key + kPtStep > it.job.to || missing) {
                    // whatever lies in places that hold no position must not meet a weight, not even one of 0: two threads per key
                    const int slot = (nk + b) % kDepth, mine = r >> 1;
                    if (!mbar_wait_bounded(&v_full[slot], (uint32_t)((nk + b) / kDepth) & 1u, err, 94)) { ok = false; break; }
                    if (key + mine >= it.job.to || (missing >> (mine >> 3) & 1u))
#pragma unroll
                        for (int c = 0; c < kHalves * 4; c++)
                            *reinterpret_cast<uint4*>(sv + (slot * kHalves + (c >> 2)) * kPtPiece + (half * kPtStep + mine) * 128 + ((c & 3) * 2 + (r & 1)) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                tmem_stored();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[s][steps & 1]);
            }
            if (!ok) break;
            nk += it.blocks;
            // ---- the item's sums, or this CTA's part of them
            if (!mbar_wait_bounded(&o_done[s][(steps - 1) & 1], (uint32_t)((steps - 1) >> 1) & 1u, err, 95)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float w0 = 1.0f, w1 = 0.0f, a0 = 0.0f, a1 = 0.0f;       // what the streams' sums count, and those put aside
            if (!dual) {
                if (s == 1) {
                    s_ml[r] = make_float2(top, sum);
                    s_aside[r] = aside_top;
                }
                __syncwarp();
                if (s == 1) {
                    if (lane == 0) mbar_arrive(&ml_ready);
                    // its sums are read by the other stream's threads
                    if (!mbar_wait_bounded(&o1_free, (uint32_t)meets & 1u, err, 96)) { ok = false; break; }
                    meets++;
                    taken++;
                    if (lane == 0) mbar_arrive(&q_empty);
                    continue;
                }
                if (!mbar_wait_bounded(&ml_ready, (uint32_t)meets & 1u, err, 97)) { ok = false; break; }
                meets++;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                {
                    const float2 odd = s_ml[r];
                    const float most = fmaxf(top, odd.x), zero = most == -INFINITY ? 0.0f : most;
                    w0 = ex2(top - zero);
                    w1 = ex2(odd.x - zero);
                    a0 = ex2(aside_top - zero);
                    a1 = ex2(s_aside[r] - zero);
                    sum = w0 * sum + w1 * odd.y;
                    top = most;
                }
            }
            const bool starts = it.starts, all = starts && it.end <= u1;
            const size_t row = (size_t)tok * p.heads + h;
            const int in_part = (dual ? s * kPtRows : 0) + r;
            const size_t at = all ? row : (size_t)(2 * cta + starts) * kTileRows + in_part;
            const bool direct = all && !it.job.joined;
            if (direct) {
                const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
                w0 *= inv;
                w1 *= inv;
                a0 *= inv;
                a1 *= inv;
            }
            // Rows pass through the room of the item's queries, of which a warp has an eighth, so that whole lines of them are stored: DP * 2 bytes of a row at a time, 16-byte
            // units turned by the row.
            constexpr int kUnits = DP / 8;
            uint8_t *room = sq + (s * 4 + quarter) * (32 * DP * 2), *mine_room = room + lane * DP * 2;
            uint8_t* dst = direct ? reinterpret_cast<uint8_t*>(static_cast<A*>(p.o) + (size_t)tok * p.ld_o + h * p.dim)
                                  : reinterpret_cast<uint8_t*>((!all ? p.tile_o : (it.job.prefix ? p.prefix_o : p.own_o)) + at * DP);
            const bool narrow = direct && !f32;             // 16-bit results
            const int row_bytes = direct ? p.dim * (int)sizeof(A) : DP * 4, pass = narrow ? DP : DP / 2;
            s_row[s][r] = live ? dst : nullptr;
#pragma unroll 1
            for (int c0 = 0; c0 < DP; c0 += pass) {
#pragma unroll 1
                for (int c = c0; c < c0 + pass; c += 16) {
                    int x[16], y[16];
                    tmem_ld(to_ + 128 * s + c, x);
                    if (!dual) tmem_ld(to_ + 128 + c, y);
                    tmem_loaded();
                    float o[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        o[j] = __int_as_float(x[j]) * w0;
                        if (!dual) o[j] = fmaf(__int_as_float(y[j]), w1, o[j]);
                    }
                    if (f32 && n_steps > kPtFold) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float4 u = __ldcg(aside + (c / 4 + j) * kPtRows), v = __ldcg(aside + (DP / 4 + c / 4 + j) * kPtRows);
                            o[4 * j] += fmaf(u.x, a0, v.x * a1);
                            o[4 * j + 1] += fmaf(u.y, a0, v.y * a1);
                            o[4 * j + 2] += fmaf(u.z, a0, v.z * a1);
                            o[4 * j + 3] += fmaf(u.w, a0, v.w * a1);
                        }
                    }
                    if (narrow) {
#pragma unroll
                        for (int j = 0; j < 2; j++)
                            *reinterpret_cast<uint4*>(mine_room + (((((c - c0) >> 3) + j) ^ (lane & (kUnits - 1))) << 4)) =
                                make_uint4(pack_16<K>(o[8 * j], o[8 * j + 1]), pack_16<K>(o[8 * j + 2], o[8 * j + 3]), pack_16<K>(o[8 * j + 4], o[8 * j + 5]), pack_16<K>(o[8 * j + 6], o[8 * j + 7]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            *reinterpret_cast<float4*>(mine_room + (((((c - c0) >> 2) + j) ^ (lane & (kUnits - 1))) << 4)) = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                    }
                }
                __syncwarp();
                const int unit = lane & (kUnits - 1), byte = c0 * (narrow ? 2 : 4) + 16 * unit;
#pragma unroll 4
                for (int i = 0; i < kUnits; i++) {
                    const int from = i * (32 / kUnits) + lane / kUnits;
                    uint8_t* to = s_row[s][32 * quarter + from];
                    const uint4 x = *reinterpret_cast<const uint4*>(room + from * DP * 2 + ((unit ^ (from & (kUnits - 1))) << 4));
                    if (to && byte < row_bytes) *reinterpret_cast<uint4*>(to + byte) = x;
                }
                __syncwarp();
            }
            if (live) {
                if (!direct) (!all ? p.tile_ml : (it.job.prefix ? p.prefix_ml : p.own_ml))[at] = make_float2(top - kPtShift<A>, sum);
                if (starts) {
                    const int end = all ? cta : deal.cta_of(it.end - 1);
                    (it.job.prefix ? p.prefix : p.own)[row] = make_int4(cta, end - cta + 1, in_part, kJoinTile | (it.job.joined && !it.job.prefix ? kJoinPrefix : 0));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // (the next queries are copied there)
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_empty);
            if (!dual && lane == 0) mbar_arrive(&o1_free);
            // the stream's other warps may still read where this one will put queries
            if (f32 && !mbar_wait_bounded(&o1_free, (uint32_t)(meets - 1) & 1u, err, 99)) { ok = false; break; }
            taken++;
        }
        if (!ok) {
            tmem_stored();
            gave_up = 1;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0 || warp == 2) {
            // ---------------- copies: queries and keys, or values.  (Scores run ahead of sums, so neither may wait for the other's room.)
            const bool keys = warp == 0;
            const CUtensorMap* map = keys ? &kmap : &vmap;
            uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
            uint8_t* room = keys ? sk : sv;
            PtItem it = {};
            int nk = 0, n_items = 0, asked = 0, u = u0;         // blocks, items; whose queries have been requested
            bool ok = true;
            while (ok) {
                if (keys) {
                    // the CTA's next item that it has blocks of
                    it.blocks = 0;
                    while (u < u1 && it.blocks <= 0) {
                        int at = 0;
                        if (u == u0) {
                            const int j = plan.find(u), per = (plan.cum[j + 1] - plan.cum[j]) / p.kv_heads;
                            it.job = plan.known(p, j);
                            at = u - plan.cum[j];
                            it.head = at / per;
                            at -= it.head * per;
                            it.t0 = 0;
                            for (int n = blocks_of(it.job, 0) + kPtExtra; at >= n; n = blocks_of(it.job, it.t0) + kPtExtra) {
                                at -= n;
                                it.t0 += item_tokens;
                            }
                        } else if (it.t0 + item_tokens < it.job.count) {
                            it.t0 += item_tokens;
                        } else {
                            it.t0 = 0;
                            if (++it.head == p.kv_heads) {
                                it.job = plan.known(p, plan.find(u));
                                it.head = 0;
                            }
                        }
                        it.begin = u - at;
                        it.end = it.begin + blocks_of(it.job, it.t0) + kPtExtra;
                        it.tokens = min(item_tokens, it.job.count - it.t0);
                        const int block = max(at - kPtExtra, 0);
                        it.from = it.job.from + block * kPtKeys;
                        it.blocks = min(it.end, u1) - it.begin - kPtExtra - block;          // (none: the next CTA has the first one)
                        it.starts = block == 0;
                        u = it.end;
                    }
                    const int slot = n_items % kPtItems;
                    if (n_items >= kPtItems && !mbar_wait_bounded(&item_empty[slot], (uint32_t)(n_items / kPtItems - 1) & 1u, err, 101)) { ok = false; break; }
                    if (lane == 0) {
                        items[slot] = it;
                        mbar_arrive(&item_full[slot]);
                    }
                    __syncwarp();
                    if (it.blocks <= 0) break;
                } else if (!take(it, n_items, false)) {
                    ok = it.blocks <= 0;
                    break;
                }
                // Queries, once the room of the last item's is free, which is while this one's first keys come.  (The first item's need not wait for any, and the first products wait for them.)
                auto queries = [&] {
                    const int tiles = is_dual(it) ? 2 : 1;
                    if (n_items && !mbar_wait_bounded(&q_empty, (uint32_t)(n_items - 1) & 1u, err, 84)) return false;
                    if (lane == 0) {
                        mbar_expect_tx(&q_full, (uint32_t)(tiles * kHalves * tile_tokens * p.share * 128));
                        for (int s = 0; s < tiles; s++)
#pragma unroll
                            for (int h = 0; h < kHalves; h++)
                                tma_rows_3d(sq + (s * kHalves + h) * kPtPiece, &qmap, 64 * h, it.head * p.share, it.job.first + it.t0 + s * tile_tokens, &q_full);
                    }
                    asked++;
                    return true;
                };
                // a lane per page (box) of a block
                const int box_rows = p.page < kPtKeys ? p.page : kPtKeys, boxes = kPtKeys / box_rows;
                const int* table = p.table + (size_t)it.job.seq * p.max_pages;
                auto needed = [&](int b) { return lane < boxes && it.from + b * kPtKeys + lane * box_rows < it.job.to; };
                // (on its way while the block before is requested: nothing is made of it here)
                auto entry_of = [&](int b) { return needed(b) ? table[(it.from + b * kPtKeys + lane * box_rows) >> p.log_page] : -1; };
                int entry = entry_of(0);
                for (int b = 0; b <= it.blocks; b++) {
                    if (!f32 && keys && b == (n_items ? min(kDepth, it.blocks) : 0) && !(ok = queries())) break;
                    if (b == it.blocks) break;
                    const int slot = nk % kDepth, now = entry;
                    if (b + 1 < it.blocks) entry = entry_of(b + 1);
                    const bool have = now >= 0 && now < p.n_pages;
                    if (!have && needed(b)) report(err, 82);
                    const unsigned who = __ballot_sync(0xFFFFFFFFu, have);
                    if (nk >= kDepth && !mbar_wait_bounded(&empty[slot], (uint32_t)(nk / kDepth - 1) & 1u, err, 85 + !keys)) { ok = false; break; }
                    if (lane == 0) {
                        if (keys) {
                            unsigned missing = 0;
                            for (int g = 0; g < 16; g++)
                                if (!(who >> (g * 8 / box_rows) & 1u)) missing |= 1u << g;
                            s_missing[nk & 7] = (unsigned short)missing;
                        }
                        mbar_expect_tx(&full[slot], (uint32_t)(__popc(who) * box_rows * 128 * kHalves));
                    }
                    __syncwarp();
                    const int row = (it.from + b * kPtKeys + lane * box_rows) & (p.page - 1);
                    if (have)
                        for (int h = 0; h < (p.both ? 1 : kHalves); h++)
                            tma_page(smem_addr(room + (slot * kHalves + h) * kPtPiece + lane * box_rows * 128), map, 64 * h, row, it.head, now, smem_addr(&full[slot]));
                    nk++;
                }
                n_items++;
            }
            // Where this role has given up, no copy is left under way when the CTA leaves.  (Else the products have waited for all of them.)
            if (!ok) {
                gave_up = 1;
                for (int b = max(nk - kDepth, 0); b < nk; b++) mbar_wait_bounded(&full[b % kDepth], (uint32_t)(b / kDepth) & 1u, err, 102);
                if (asked) mbar_wait_bounded(&q_full, (uint32_t)(asked - 1) & 1u, err, 103);
            }
        } else {
            // ---------------- MMAs.  (What this thread computes between two products is a chain that nothing covers: addresses and descriptors are ready ahead.)
            const int s = warp >> 1;
            if (elect_one()) {
                constexpr uint32_t kind = std::is_same<K, bf16>::value ? 1u : 0u;
                constexpr uint32_t fmt = (1u << 4) | (kind << 7) | (kind << 10) | ((uint32_t)(kPtRows >> 4) << 24);
                constexpr uint32_t idesc_s = fmt | ((uint32_t)(kPtStep >> 3) << 17), idesc_o = fmt | (1u << 16) | ((uint32_t)(DP >> 3) << 17);
                constexpr uint32_t block = kHalves * kPtPiece >> 4, half_block = kPtStep * 128 >> 4;       // in a descriptor's units
                const uint32_t o = tmem + 256 + 128 * s, scores_at = tmem + 128 * s;
                const uint32_t b_s = smem_addr(s_full[s]), b_p = smem_addr(p_full[s]), b_o = smem_addr(o_done[s]), b_kf = smem_addr(k_full), b_ke = smem_addr(k_empty),
                               b_vf = smem_addr(v_full), b_ve = smem_addr(v_empty);
                const uint64_t kd0 = swizzled_desc(smem_addr(sk)), vd0 = swizzled_desc_mn(smem_addr(sv), kPtPiece);
                PtItem it = {};
                int taken = 0;
                uint32_t ks = 0, kp = 0, vs = 0, vp = 0;        // the next blocks of keys and values: slots and phases
                uint32_t si = 0, pi = 0;                        // steps so far: scores, sums
                bool ok = true;
                while (ok && take(it, taken, true)) {
                    const bool dual = is_dual(it);
                    const int steps = dual ? 2 * it.blocks : it.blocks;
                    const uint64_t qd = swizzled_desc(smem_addr(sq + (dual ? s : 0) * kHalves * kPtPiece));
                    if (!(ok = mbar_wait_bounded(&q_full, (uint32_t)taken & 1u, err, 87))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    // step t reads half `h` of a block; `first` and `last` of this stream's steps on it
                    auto scores = [&](int t) {
                        const int h = dual ? t & 1 : s;
                        const bool first = !dual || !(t & 1), last = !dual || (t & 1);
                        if (first && !mbar_wait_at(b_kf + 8 * ks, kp, err, 88)) return false;
                        const uint64_t kd = kd0 + ks * block + h * half_block;
                        const uint32_t to = scores_at + 64 * (si & 1);
#pragma unroll
                        for (int part = f32 ? 1 : 0; part >= 0; part--)         // (the small parts first: the sum is cut off at its own last bit)
#pragma unroll
                            for (int c = 0; c < kHalves; c++)
#pragma unroll
                                for (int k = 0; k < 4; k++)
                                    umma_bf16_ss(to, qd + (uint64_t)((part * kHalves + c) * (kPtPiece >> 4) + 2 * k), kd + (uint64_t)(c * (kPtPiece >> 4) + 2 * k), idesc_s,
                                                 (f32 && part == 0) | c | k ? 1u : 0u);
                        umma_commit_at(b_s + 8 * (si & 1));
                        if (last) {
                            umma_commit_at(b_ke + 8 * ks);
                            if (++ks == kDepth) { ks = 0; kp ^= 1; }
                        }
                        si++;
                        return true;
                    };
                    ok = scores(0) && (steps < 2 || scores(1));
#pragma unroll 1
                    for (int t = 0; ok && t < steps; t++) {
                        const int h = dual ? t & 1 : s;
                        const bool first = !dual || !(t & 1), last = !dual || (t & 1);
                        if (first && !(ok = mbar_wait_at(b_vf + 8 * vs, vp, err, 89))) break;
                        if (!(ok = mbar_wait_at(b_p + 8 * (pi & 1), (pi >> 1) & 1u, err, 90))) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t vd = vd0 + vs * block + h * half_block;
                        const uint32_t w = scores_at + 64 * (pi & 1);
#pragma unroll
                        for (int k = 0; k < kPtStep / 16; k++) {
                            if (f32) umma_bf16_ts(o, w + 32 + 8 * k, vd + (uint64_t)(k * 128), idesc_o, t % kPtFold | k ? 1u : 0u);
                            umma_bf16_ts(o, w + 8 * k, vd + (uint64_t)(k * 128), idesc_o, f32 || (t | k) ? 1u : 0u);
                        }
                        umma_commit_at(b_o + 8 * (pi & 1));
                        if (last) {
                            umma_commit_at(b_ve + 8 * vs);
                            if (++vs == kDepth) { vs = 0; vp ^= 1; }
                        }
                        pi++;
                        if (t + 2 < steps) ok = scores(t + 2);
                    }
                    taken++;
                }
                if (!ok) gave_up = 1;
            }
        __syncwarp();
        }
    }
    if (p.mark && warp < 4) mark_tokens(p, tid, 128, err);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (gave_up) {                      // no product is left under way, either, when tensor memory is given back: the threads that have issued them wait
        if ((warp == 1 || warp == 3) && elect_one()) {
            umma_commit(&idle[warp >> 1]);
            mbar_wait_bounded(&idle[warp >> 1], 0, err, 104);
        }
        __syncthreads();
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <typename A, typename K, int DP, int kCap>
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
    if ((rc = allow_smem<k_paged_tile<A, K, DP, kCap>>(221 * 1024))) return rc;
    const size_t smem = 1024 + PtShape<DP>::end + PagedPlan::size(a);
    return launch_ordered(k_paged_tile<A, K, DP, kCap>, dim3((unsigned)ctas), kPtThreads, smem, s, qmap, kmap, vmap, a, device_error_flag());
}

template <typename A, typename K>
static int launch_kind(const PagedArgs& a, const bpdq_paged_kv& kv, int ctas, cudaStream_t s)
{
    const bool wide = a.dim > 64;
    if (a.cap_kind == kCapNone) return wide ? launch_tile<A, K, 128, kCapNone>(a, kv, ctas, s) : launch_tile<A, K, 64, kCapNone>(a, kv, ctas, s);
    if constexpr (sizeof(A) == 2)
        if (a.cap_kind == kCapFar) return wide ? launch_tile<A, K, 128, kCapFar>(a, kv, ctas, s) : launch_tile<A, K, 64, kCapFar>(a, kv, ctas, s);
    return wide ? launch_tile<A, K, 128, kCapNear>(a, kv, ctas, s) : launch_tile<A, K, 64, kCapNear>(a, kv, ctas, s);
}

int paged_tile(const PagedArgs& a, const bpdq_paged_kv& kv, int ctas, cudaStream_t s)
{
    if (kv.act_type == BPDQ_TYPE_F32) return launch_kind<float, __half>(a, kv, ctas, s);
    return kv.kv_type == BPDQ_TYPE_F16 ? launch_kind<__half, __half>(a, kv, ctas, s) : launch_kind<bf16, bf16>(a, kv, ctas, s);
}

}  // namespace bpdq
