// Attention over a paged cache for jobs of few rows (paged_attention.cuh): decoding, where every key and value is read for a handful of query heads.
//
// The keys of all items lie end to end in tiles of 16; every CTA takes an equal run of them and every warp an equal run of its CTA's, so that lengths
// do not matter and no warp waits for another before the end.  A warp fills its own ring of tiles (keys and values, tiled bulk copies straight from the
// pages), and has running maxima, sums and outputs of its rows in registers.  Eight rows fill half of an m16n8k16 product: the other half is the small
// part of what does not fit 16 bits, of softmax weights (w = hi + lo) and of fp32 queries, so it costs nothing.
// fp16 ends at 2^16 and rounds what is below 2^-25 to 0.  Weights may reach 2^8 (kPsGrowth), so fp16 ones are held 2^7 times as large, and their small parts, whose
// products have sums of their own, another 2^11 times: a weight is off by 2^-43 of the largest at most, or by 2^-23 of itself.
// 64 sequences of up to 8000 positions (8 key heads of 128 in bf16, 796 MB): 136 us with the join, 5.9 TB/s, bound by memory.  One of 4000: 13.8 us, a chain of the plan, the
// first copies, three tiles a warp and two joins.
#include "paged_attention.cuh"
#include "tcgen05_device.cuh"
#include "mma_device.cuh"

namespace bpdq {

constexpr int kPsWarps = kSplitWarps, kPsThreads = 32 * kPsWarps, kPsKeys = 16, kPsRing = 24576;        // bytes of a warp's ring
constexpr int kPsItems = 8;                         // more than copies can be ahead (six tiles)
constexpr float kPsGrowth = 8.0f;                   // log2 of how far weights may exceed 1 before outputs are rescaled
template <typename K> constexpr float kPsShift = 0.0f;                  // log2 of what weights are multiplied by on their way to the tensor cores
template <> constexpr float kPsShift<__half> = 7.0f;
template <typename K> constexpr float kPsLow = 1.0f;                    // and of their small parts' products: what they are divided by again
template <> constexpr float kPsLow<__half> = 1.0f / 2048.0f;

template <typename K> __device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16<bf16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename K> __device__ __forceinline__ void split_weights(float v0, float v1, uint32_t& hi, uint32_t& lo) { split_bf16(v0, v1, hi, lo); }
template <> __device__ __forceinline__ void split_weights<__half>(float v0, float v1, uint32_t& hi, uint32_t& lo) { split_f16(v0, v1, hi, lo, 1.0f / kPsLow<__half>); }
__device__ __forceinline__ void ldsm4_at(uint32_t (&r)[4], uint32_t p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void ldsm4_t_at(uint32_t (&r)[4], uint32_t p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ float quad_max(float v)
{
    v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v)
{
    v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
    return v + __shfl_xor_sync(0xFFFFFFFFu, v, 2);
}
template <typename A> __device__ __forceinline__ void store_two(A* p, float a, float b);
template <> __device__ __forceinline__ void store_two<float>(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
template <> __device__ __forceinline__ void store_two<__half>(__half* p, float a, float b) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b); }
template <> __device__ __forceinline__ void store_two<bf16>(bf16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }

// An item, and the unit of it that is next.
struct PsItem {
    PagedJob job;
    int tiles, head, begin, end, key;   // units of an item of the job, key head, its units, position of the next unit's first key
};
// What a warp leaves of an item that it has not all of.
struct PsPart {
    int begin, end, first, rows, head, joined, prefix, valid;
};

template <typename A, typename K, int DP, int MT>
__global__ void __launch_bounds__(kPsThreads, 1)
k_paged_split(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const PagedArgs p, int* err)
{
    constexpr int kHalves = DP / 64, kTile = kPsKeys * DP * 2, kStages = kPsRing / (2 * kTile), kSteps = DP / 16, kOut = DP / 8;
    constexpr bool f32 = sizeof(A) == 4;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t bars[kPsWarps][kStages];
    __shared__ PsPart parts[kPsWarps][2];
    __shared__ PsItem items[kPsWarps][kPsItems];        // as copies meet them, for the sums behind
    const uint32_t ring_all = (smem_addr(raw) + 1023) & ~1023u;
    uint8_t* ring_ptr = raw + (ring_all - smem_addr(raw));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = ring_all + warp * kPsRing;
    if (lane == 0) {
        for (int i = 0; i < kStages; i++) mbar_init(&bars[warp][i], 1);
        mbar_init_fence();
    }
    if (lane < 2) parts[warp][lane].valid = 0;
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    }
    int row_tok[MT], row_head[MT];      // of the thread's rows: token within the job, query head within the key head's
#pragma unroll
    for (int m = 0; m < MT; m++) {
        row_tok[m] = (8 * m + g) / p.share;
        row_head[m] = 8 * m + g - row_tok[m] * p.share;
    }
    // (Behind k_paged_tile too: only a wait makes visible to this grid what launches before that one have written.)
    pdl_wait();
    pdl_launch_dependents();

    PagedPlan plan = {};
    const int total = plan.build<kPsThreads>(p, reinterpret_cast<int*>(ring_ptr + kPsWarps * kPsRing), err,
                                             [&](const PagedJob& r) { return r.rows <= p.split_rows ? (r.to - r.from + kPsKeys - 1) / kPsKeys : 0; });
    // A tile per warp at least: fewer CTAs have fewer parts to join.
    const int most = (total + kPsWarps - 1) / kPsWarps, ctas = max(1, min((int)gridDim.x, most)), cta = blockIdx.x;
    const PagedDeal deal(total, ctas);
    const int u0 = cta < ctas ? deal.first(cta) : total, u1 = cta < ctas ? deal.first(cta + 1) : total;
    const int a0 = u0 + (u1 - u0) * warp / kPsWarps, a1 = u0 + (u1 - u0) * (warp + 1) / kPsWarps;

    // ---- copies: the warp's tiles in order, kStages ahead.  (Code that runs once waits for its instructions: what follows is laid out so that nothing stands
    // in it twice.)
    PsItem src = {};
    src.end = a0;
    int src_u = a0, entry = 0, entry_base = 0, opened = 0;
    uint32_t missing = 0;               // two bits per stage: its first eight, its last eight positions have no page
    const bool small = p.page == 8;
    auto request = [&](int stage) {
        if (src_u == src.end) {
            if (opened && src.head + 1 < p.kv_heads) {
                src.head++;
                src.begin = src.end;
            } else {
                const int j = plan.find(src_u), at = src_u - plan.cum[j];
                src.job = plan.known(p, j);
                src.tiles = (src.job.to - src.job.from + kPsKeys - 1) / kPsKeys;
                src.head = at / src.tiles;
                src.begin = plan.cum[j] + src.head * src.tiles;
            }
            src.end = src.begin + src.tiles;
            src.key = src.job.from + (src_u - src.begin) * kPsKeys;
            if (lane == 0) items[warp][opened % kPsItems] = src;
            opened++;
            entry_base = -32;
        }
        const int e = src.key >> p.log_page;
        if (e + 1 >= entry_base + 32) {
            entry_base = e;
            entry = e + lane < p.max_pages ? p.table[(size_t)src.job.seq * p.max_pages + e + lane] : -1;
        }
        const int page0 = __shfl_sync(0xFFFFFFFFu, entry, e - entry_base), page1 = __shfl_sync(0xFFFFFFFFu, entry, e - entry_base + 1);
        const bool ok0 = page0 >= 0 && page0 < p.n_pages, need1 = small && src.key + 8 < src.job.to, ok1 = need1 ? page1 >= 0 && page1 < p.n_pages : !small && ok0;
        if (lane == 0) {
            const uint32_t bar = smem_addr(&bars[warp][stage]), at = ring + stage * 2 * kTile;
            const uint32_t box = (uint32_t)((small ? 8 : kPsKeys) * 128 * kHalves * 2), n = small ? (ok0 ? 1u : 0u) + (ok1 ? 1u : 0u) : (ok0 ? 1u : 0u);
            mbar_expect_tx_at(bar, n * box);
            const int row = src.key & (p.page - 1);
            for (int h = 0; h < (p.both ? 1 : kHalves); h++) {
                if (ok0) {
                    tma_page(at + h * (kPsKeys * 128), &kmap, 64 * h, row, src.head, page0, bar);
                    tma_page(at + kTile + h * (kPsKeys * 128), &vmap, 64 * h, row, src.head, page0, bar);
                }
                if (small && ok1) {
                    tma_page(at + h * (kPsKeys * 128) + 1024, &kmap, 64 * h, 0, src.head, page1, bar);
                    tma_page(at + kTile + h * (kPsKeys * 128) + 1024, &vmap, 64 * h, 0, src.head, page1, bar);
                }
            }
            if (!ok0 || (need1 && !ok1)) report(err, 82);
        }
        missing = (missing & ~(3u << (2 * stage))) | ((ok0 ? 0u : 1u) | (ok1 ? 0u : 2u)) << (2 * stage);
        src_u++;
        src.key += kPsKeys;
    };
    PsItem it = {};
    uint32_t qf[MT][kSteps][f32 ? 4 : 2];           // queries: rows' (and their small parts') fragments
    float factor[MT];
    int limit[MT];
    auto queries = [&] {
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const bool live = 8 * m + g < it.job.rows;
            const int tok = it.job.first + (live ? row_tok[m] : 0), h = it.head * p.share + (live ? row_head[m] : 0);
            limit[m] = it.job.prefix ? it.job.to : it.job.to - it.job.count + (live ? row_tok[m] : 0) + 1;
            const A* q = static_cast<const A*>(p.q) + (size_t)tok * p.ld_q + h * p.dim;
            factor[m] = p.scale;
            if constexpr (f32) {
                float2 x[kSteps][2];
                float big = 0.0f;
#pragma unroll
                for (int s = 0; s < kSteps; s++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const int d = 16 * s + 8 * c + 2 * t4;
                        x[s][c] = live && d < p.dim ? *reinterpret_cast<const float2*>(q + d) : make_float2(0.0f, 0.0f);
                        big = fmaxf(big, fmaxf(fabsf(x[s][c].x), fabsf(x[s][c].y)));
                    }
                // a power of two brings the row's largest entry to 1 .. 2: both parts are then fp16 numbers, off by 2^-22 of it
                big = quad_max(big);
                const int e = big > 0.0f && big < INFINITY ? min(max(ilogbf(big), -100), 100) : 0;
                const float down = __int_as_float((127 - e) << 23);
                factor[m] *= __int_as_float((127 + e) << 23);
#pragma unroll
                for (int s = 0; s < kSteps; s++)
#pragma unroll
                    for (int c = 0; c < 2; c++) split_f16(x[s][c].x * down, x[s][c].y * down, qf[m][s][2 * c], qf[m][s][2 * c + 1]);
            } else {
#pragma unroll
                for (int s = 0; s < kSteps; s++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const int d = 16 * s + 8 * c + 2 * t4;
                        qf[m][s][c] = live && d < p.dim ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
                    }
            }
        }
    };

    // ---- sums
    // (The tensor pipe cuts off what does not fit fp32 of each of its sums, always toward zero: with fp32 activations a tile's products start from 0 and are added here.)
    constexpr int kSums = f32 ? 2 : 4;
    float out[MT][kOut][kSums], top[MT], sum[MT];
    auto result = [&](int m, int i, int c) {
        if constexpr (f32) return out[m][i][c];
        else return fmaf(out[m][i][c + 2], kPsLow<K>, out[m][i][c]);
    };
    auto product = [&](int m, int i, uint32_t b0, uint32_t b1, const uint32_t (&w)[4]) {
        if constexpr (f32) {
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma_16<K>(d, w, b0, b1);
            out[m][i][0] += fmaf(d[2], kPsLow<K>, d[0]);
            out[m][i][1] += fmaf(d[3], kPsLow<K>, d[1]);
        } else {
            mma_16<K>(out[m][i], w, b0, b1);
        }
    };
    int began = a0, taken = 0;          // the unit with which the warp's part of the item began; items so far
    // tile n is used, then the copy of tile n + kStages requested into its place
#pragma unroll 1
    for (int u = a0 - kStages, stage = 0, phase = 0; u < a1; u++) {
      if (u >= a0) {
        if (u == a0 || u == it.end) {
            __syncwarp();
            it = items[warp][taken++ % kPsItems];
            queries();
            began = u;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                top[m] = -INFINITY;
                sum[m] = 0.0f;
#pragma unroll
                for (int i = 0; i < kOut; i++)
#pragma unroll
                    for (int c = 0; c < kSums; c++) out[m][i][c] = 0.0f;
            }
        }
        if (!mbar_wait_bounded(&bars[warp][stage], (uint32_t)phase, err, 83)) {
            // no copy is left under way
#pragma unroll 1
            for (int v = u; v < src_u; v++) mbar_wait_bounded(&bars[warp][(v - a0) % kStages], (uint32_t)((v - a0) / kStages) & 1u, err, 83);
            break;
        }
        const uint32_t kt = ring + stage * 2 * kTile, vt = kt + kTile;
        const int have = min(kPsKeys, it.job.to - it.key);
        const uint32_t gone = missing >> (2 * stage) & 3u, valid = ((1u << have) - 1u) & ~((gone & 1u ? 0xFFu : 0u) | (gone & 2u ? 0xFF00u : 0u));
        const bool whole = valid == 0xFFFFu;
        if (!whole) {
            // whatever lies in places that hold no position must not meet a weight, not even one of 0
            for (int i = lane; i < kPsKeys * DP / 8; i += 32) {
                const int r = i / (DP / 8), c = i % (DP / 8);
                if (!(valid >> r & 1u)) asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vt + (c >> 3) * (kPsKeys * 128) + r * 128 + (c & 7) * 16), "r"(0u) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        }
        // two chains of products per eight keys, fragments of four steps at a time
        float sc[MT][2][4], sc2[MT][2][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < 8; i++) sc[m][i >> 2][i & 3] = sc2[m][i >> 2][i & 3] = 0.0f;
        {
            const int r = (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
#pragma unroll
            for (int s0 = 0; s0 < kSteps; s0 += 4) {
                uint32_t b[4][4];
#pragma unroll
                for (int s = 0; s < 4; s++) ldsm4_at(b[s], kt + (s0 >> 2) * (kPsKeys * 128) + r * 128 + (((2 * s + c) ^ (r & 7)) << 4));
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        uint32_t a[4];
                        const int q = s0 + s;
                        if constexpr (f32) { a[0] = qf[m][q][0]; a[1] = qf[m][q][1]; a[2] = qf[m][q][2]; a[3] = qf[m][q][3]; }
                        else { a[0] = qf[m][q][0]; a[1] = 0; a[2] = qf[m][q][1]; a[3] = 0; }
                        mma_16<K>(s & 1 ? sc2[m][0] : sc[m][0], a, b[s][0], b[s][1]);
                        mma_16<K>(s & 1 ? sc2[m][1] : sc[m][1], a, b[s][2], b[s][3]);
                    }
            }
        }
        uint32_t w[MT][4];
        bool grown = false;
        float now[MT];
#pragma unroll
        for (int m = 0; m < MT; m++) {
            // in units of log2
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = sc[m][i >> 1][i & 1] + sc2[m][i >> 1][i & 1];
                if constexpr (f32) x[i] += sc[m][i >> 1][2 + (i & 1)] + sc2[m][i >> 1][2 + (i & 1)];
                x[i] *= factor[m];
                if (p.cap_kind == kCapNear) x[i] = capped<f32, kCapNear>(x[i], p.cap);
                else if (p.cap_kind == kCapFar) x[i] = capped<f32, kCapFar>(x[i], p.cap);
                x[i] *= 1.44269504088896341f;
            }
            if (!whole || it.key + kPsKeys > limit[m]) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int c = 8 * (i >> 1) + 2 * t4 + (i & 1);
                    if (it.key + c >= limit[m] || !(valid >> c & 1u)) x[i] = -INFINITY;
                }
            }
            now[m] = quad_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
            grown = grown || now[m] > top[m] + kPsGrowth;
#pragma unroll
            for (int i = 0; i < 4; i++) sc[m][i >> 1][i & 1] = x[i];
        }
        if (__any_sync(0xFFFFFFFFu, grown)) {
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const float to = fmaxf(top[m], now[m]), down = to == -INFINITY ? 1.0f : ex2(top[m] - to);
                top[m] = to;
                if (u == began) continue;           // (there is nothing yet)
                sum[m] *= down;
#pragma unroll
                for (int i = 0; i < kOut; i++)
#pragma unroll
                    for (int c = 0; c < kSums; c++) out[m][i][c] *= down;
            }
        }
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float base = top[m] == -INFINITY ? 0.0f : top[m] - kPsShift<K>;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = ex2(sc[m][i >> 1][i & 1] - base);
            sum[m] += (x[0] + x[1]) + (x[2] + x[3]);
            split_weights<K>(x[0], x[1], w[m][0], w[m][1]);
            split_weights<K>(x[2], x[3], w[m][2], w[m][3]);
        }
        {
            const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = lane >> 4;
#pragma unroll
            for (int i0 = 0; i0 < kOut / 2; i0 += 4) {
                uint32_t b[4][4];
#pragma unroll
                for (int i = 0; i < 4; i++) ldsm4_t_at(b[i], vt + (i0 >> 2) * (kPsKeys * 128) + r * 128 + (((2 * i + c) ^ (r & 7)) << 4));
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        product(m, 2 * (i0 + i), b[i][0], b[i][1], w[m]);
                        product(m, 2 * (i0 + i) + 1, b[i][2], b[i][3], w[m]);
                    }
            }
        }
        it.key += kPsKeys;
        if (u + 1 == it.end || u + 1 == a1) {
        // ---- the warp's part of the item is complete
        const bool all = began == it.begin && u + 1 == it.end, tail = u + 1 == a1;
        if (!all) {
            if (lane == 0) parts[warp][tail] = {it.begin, it.end, it.job.first, it.job.rows, it.head, it.job.joined, it.job.prefix, 1};
        }
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float l = quad_sum(sum[m]), most = top[m] - kPsShift<K>;      // (the maximum that the sums count from)
            const int r = 8 * m + g;
            if (r >= it.job.rows) continue;
            const int tok = it.job.first + row_tok[m], h = it.head * p.share + row_head[m];
            const size_t row = (size_t)tok * p.heads + h;
            float* dst = nullptr;
            if (all && !it.job.joined) {
                const float inv = l != 0.0f ? 1.0f / l : 0.0f;
                A* o = static_cast<A*>(p.o) + (size_t)tok * p.ld_o + h * p.dim;
#pragma unroll
                for (int i = 0; i < kOut; i++)
                    if (8 * i + 2 * t4 < p.dim) store_two<A>(o + 8 * i + 2 * t4, result(m, i, 0) * inv, result(m, i, 1) * inv);
            } else if (all) {
                dst = (it.job.prefix ? p.prefix_o : p.own_o) + row * DP;
                if (t4 == 0) (it.job.prefix ? p.prefix_ml : p.own_ml)[row] = make_float2(most, l);
            } else if (tail) {
                float* mine = reinterpret_cast<float*>(ring_ptr + warp * kPsRing);
                dst = mine + r * DP;
                if (t4 == 0) reinterpret_cast<float2*>(mine + kSplitRows * DP)[r] = make_float2(most, l);
            } else {
                const size_t at = (size_t)(cta * kPsWarps + warp) * kSplitRows + r;
                dst = p.head_o + at * DP;
                if (t4 == 0) p.head_ml[at] = make_float2(most, l);
            }
            if (all && t4 == 0) (it.job.prefix ? p.prefix : p.own)[row] = make_int4(cta, 1, 0, it.job.joined && !it.job.prefix ? kJoinPrefix : 0);
            if (dst)
#pragma unroll
                for (int i = 0; i < kOut; i++) store_two<float>(dst + 8 * i + 2 * t4, result(m, i, 0), result(m, i, 1));
        }
        }
        __syncwarp();
      }
      if (src_u < a1) request(stage);
      if (++stage == kStages) { stage = 0; phase ^= u >= a0; }
    }
    if (p.mark && warp == kPsWarps - 1) mark_tokens(p, lane, 32, err);
    __syncthreads();

    // ---- items that several warps have parts of, eight threads per row.  Part e is the first (e even) or last part of warp e / 2.
    const PsPart* of_lane = &parts[(lane & 15) >> 1][lane & 1];
    const unsigned exist = __ballot_sync(0xFFFFFFFFu, lane < 2 * kPsWarps && of_lane->valid);
    const int begins = of_lane->begin, before = exist & ((1u << lane) - 1) ? 31 - __clz(exist & ((1u << lane) - 1)) : lane;
    const int begins_before = __shfl_sync(0xFFFFFFFFu, begins, before);
    unsigned heads = __ballot_sync(0xFFFFFFFFu, (exist >> lane & 1u) && (before == lane || begins_before != begins));        // the items' first parts
    const int l8 = tid & 7;
    int turn = tid >> 3;                // the rows, item by item, that are still to be passed over
#pragma unroll 1
    while (heads) {
        const int e = __ffs(heads) - 1;
        heads &= heads - 1;
        const PsPart item = parts[e >> 1][e & 1];
        if (turn >= item.rows) { turn -= item.rows; continue; }
        const unsigned members = exist & ~((1u << e) - 1) & (heads ? (1u << (__ffs(heads) - 1)) - 1 : ~0u);
        const bool starts = item.begin >= u0, all = starts && item.end <= u1;
        const int r = turn;
        turn += kPsThreads / 8 - item.rows;         // (an item has fewer rows than there are groups of threads)
        float top = -INFINITY, l = 0.0f;
        float4 acc[kHalves * 2];
#pragma unroll
        for (int c = 0; c < kHalves * 2; c++) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        // two parts at a time
#pragma unroll 1
        for (unsigned rest = members; rest;) {
            float2 v[2];
            float4 x[2][kHalves * 2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int i = rest ? __ffs(rest) - 1 : e;
                const size_t at = (size_t)(cta * kPsWarps + (i >> 1)) * kSplitRows;
                const float* ring_part = reinterpret_cast<const float*>(ring_ptr + (i >> 1) * kPsRing);
                const float* from = (i & 1 ? ring_part : p.head_o + at * DP) + r * DP + 4 * l8;
                v[k] = i & 1 ? reinterpret_cast<const float2*>(ring_part + kSplitRows * DP)[r] : p.head_ml[at + r];
#pragma unroll
                for (int c = 0; c < kHalves * 2; c++) x[k][c] = *reinterpret_cast<const float4*>(from + 32 * c);
                if (!rest) v[k] = make_float2(-INFINITY, 0.0f);
                rest &= rest - 1;
            }
            const float now = fmaxf(top, fmaxf(v[0].x, v[1].x)), zero = now == -INFINITY ? 0.0f : now;
            const float down = ex2(top - zero), w0 = ex2(v[0].x - zero), w1 = ex2(v[1].x - zero);
            l = fmaf(w1, v[1].y, fmaf(w0, v[0].y, l * down));
            top = now;
#pragma unroll
            for (int c = 0; c < kHalves * 2; c++) {
                acc[c].x = fmaf(w1, x[1][c].x, fmaf(w0, x[0][c].x, acc[c].x * down));
                acc[c].y = fmaf(w1, x[1][c].y, fmaf(w0, x[0][c].y, acc[c].y * down));
                acc[c].z = fmaf(w1, x[1][c].z, fmaf(w0, x[0][c].z, acc[c].z * down));
                acc[c].w = fmaf(w1, x[1][c].w, fmaf(w0, x[0][c].w, acc[c].w * down));
            }
        }
        const int t = r / p.share, tok = item.first + t, h = item.head * p.share + r - t * p.share;
        const size_t row = (size_t)tok * p.heads + h;
        if (all && !item.joined) {
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            A* out_row = static_cast<A*>(p.o) + (size_t)tok * p.ld_o + h * p.dim + 4 * l8;
#pragma unroll
            for (int c = 0; c < kHalves * 2; c++)
                if (32 * c + 4 * l8 < p.dim) {
                    store_two<A>(out_row + 32 * c, acc[c].x * inv, acc[c].y * inv);
                    store_two<A>(out_row + 32 * c + 2, acc[c].z * inv, acc[c].w * inv);
                }
        } else {
            const size_t at = all ? row : (size_t)(2 * cta + starts) * kSplitRows + r;
            float* dst = (!all ? p.split_o : (item.prefix ? p.prefix_o : p.own_o)) + at * DP + 4 * l8;
#pragma unroll
            for (int c = 0; c < kHalves * 2; c++) *reinterpret_cast<float4*>(dst + 32 * c) = acc[c];
            if (l8 == 0) (!all ? p.split_ml : (item.prefix ? p.prefix_ml : p.own_ml))[at] = make_float2(top, l);
        }
        if (l8 == 0 && starts) {
            // the CTA with the item's last unit
            const int end = all ? cta : deal.cta_of(item.end - 1);
            (item.prefix ? p.prefix : p.own)[row] = make_int4(cta, end - cta + 1, r, item.joined && !item.prefix ? kJoinPrefix : 0);
        }
    }
}

template <typename A, typename K, int DP, int MT>
static int launch_split(PagedArgs a, const bpdq_paged_kv& kv, int ctas, cudaStream_t s)
{
    CUtensorMap kmap, vmap;
    int rc;
    if ((rc = paged_map(&kmap, kv.k, kv, kPsKeys)) || (rc = paged_map(&vmap, kv.v, kv, kPsKeys))) return rc;
    a.both = paged_both(kv, kPsKeys);
    if ((rc = allow_smem<k_paged_split<A, K, DP, MT>>(221 * 1024))) return rc;
    const size_t smem = 1024 + kPsWarps * kPsRing + PagedPlan::size(a);
    return launch_ordered(k_paged_split<A, K, DP, MT>, dim3((unsigned)ctas), kPsThreads, smem, s, kmap, vmap, a, device_error_flag());
}

int paged_split(const PagedArgs& a, const bpdq_paged_kv& kv, int ctas, cudaStream_t s)
{
    // Rows of a job go to one product of eight, or two.
    const bool wide = a.dim > 64, two = a.split_rows > 8;
    if (kv.act_type == BPDQ_TYPE_F32) {
        if (wide) return two ? launch_split<float, __half, 128, 2>(a, kv, ctas, s) : launch_split<float, __half, 128, 1>(a, kv, ctas, s);
        return two ? launch_split<float, __half, 64, 2>(a, kv, ctas, s) : launch_split<float, __half, 64, 1>(a, kv, ctas, s);
    }
    if (kv.kv_type == BPDQ_TYPE_F16) {
        if (wide) return two ? launch_split<__half, __half, 128, 2>(a, kv, ctas, s) : launch_split<__half, __half, 128, 1>(a, kv, ctas, s);
        return two ? launch_split<__half, __half, 64, 2>(a, kv, ctas, s) : launch_split<__half, __half, 64, 1>(a, kv, ctas, s);
    }
    if (wide) return two ? launch_split<bf16, bf16, 128, 2>(a, kv, ctas, s) : launch_split<bf16, bf16, 128, 1>(a, kv, ctas, s);
    return two ? launch_split<bf16, bf16, 64, 2>(a, kv, ctas, s) : launch_split<bf16, bf16, 64, 1>(a, kv, ctas, s);
}

}  // namespace bpdq
