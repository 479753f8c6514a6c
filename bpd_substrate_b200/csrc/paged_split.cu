// Attention over a paged cache for jobs of few rows (paged_attention.cuh): decoding, where every key and value is read for a handful of query heads.
//
// The keys of all items lie end to end in tiles of 16; every CTA takes an equal run of them and every warp an equal run of its CTA's, so that lengths
// do not matter and no warp waits for another before the end.  A warp fills its own ring of tiles (keys and values, tiled bulk copies straight from the
// pages), and has running maxima, sums and outputs of its rows in registers.  Eight rows fill half of an m16n8k16 product: the other half is the small
// part of what does not fit 16 bits, of softmax weights (w = hi + lo) and of fp32 queries, so it costs nothing.
#include "paged_attention.cuh"
#include "tcgen05_device.cuh"
#include "mma_device.cuh"

namespace bpdq {

constexpr int kPsWarps = kSplitWarps, kPsThreads = 32 * kPsWarps, kPsKeys = 16, kPsRing = 24576;        // bytes of a warp's ring
constexpr float kPsGrowth = 8.0f;                   // log2 of how far weights may exceed 1 before outputs are rescaled

template <typename K> __device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16<bf16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { mma_bf16(d, a, b0, b1); }
template <> __device__ __forceinline__ void mma_16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename K> __device__ __forceinline__ void split_16(float v0, float v1, uint32_t& hi, uint32_t& lo);
template <> __device__ __forceinline__ void split_16<bf16>(float v0, float v1, uint32_t& hi, uint32_t& lo) { split_bf16(v0, v1, hi, lo); }
template <> __device__ __forceinline__ void split_16<__half>(float v0, float v1, uint32_t& hi, uint32_t& lo)
{
    const __half2 h = __floats2half2_rn(v0, v1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(v0 - f.x, v1 - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
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
    int j, head, begin, end, key;       // job, key head, its units, position of the next unit's first key
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
    const uint32_t ring_all = (smem_addr(raw) + 1023) & ~1023u;
    uint8_t* ring_ptr = raw + (ring_all - smem_addr(raw));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = ring_all + warp * kPsRing;
    if (lane == 0) {
        for (int i = 0; i < kStages; i++) mbar_init(&bars[warp][i], 1);
        mbar_init_fence();
    }
    if (lane < 2) parts[warp][lane].valid = 0;
    pdl_wait();
    pdl_launch_dependents();

    PagedPlan plan = {};
    const int total = plan.build<kPsThreads>(p, reinterpret_cast<int*>(ring_ptr + kPsWarps * kPsRing), err,
                                             [&](const PagedJob& r) { return r.rows <= p.split_rows ? (r.to - r.from + kPsKeys - 1) / kPsKeys : 0; });
    // A tile per warp at least: fewer CTAs have fewer parts to join.
    const int most = (total + kPsWarps - 1) / kPsWarps, ctas = max(1, min((int)gridDim.x, most)), cta = blockIdx.x;
    const int u0 = cta < ctas ? (int)((long long)total * cta / ctas) : total, u1 = cta < ctas ? (int)((long long)total * (cta + 1) / ctas) : total;
    const int a0 = u0 + (u1 - u0) * warp / kPsWarps, a1 = u0 + (u1 - u0) * (warp + 1) / kPsWarps;

    auto open = [&](PsItem& it, int u, bool again) {
        if (!again || u >= plan.cum[it.j + 1]) {
            it.j = plan.find(u);
            it.job = plan.job(p, it.j, err);
        }
        const int tiles = (it.job.to - it.job.from + kPsKeys - 1) / kPsKeys, at = u - plan.cum[it.j];
        it.head = at / tiles;
        it.begin = plan.cum[it.j] + it.head * tiles;
        it.end = it.begin + tiles;
        it.key = it.job.from + (u - it.begin) * kPsKeys;
    };

    // ---- copies: the warp's tiles in order, kStages ahead
    PsItem src = {};
    int src_u = a0, entry = 0, entry_base = -1;
    uint32_t missing = 0;               // two bits per stage: its first eight, its last eight positions have no page
    const bool small = p.page == 8;
    auto request = [&](int stage) {
        if (src_u == a0 || src_u >= src.end) {
            open(src, src_u, src_u != a0);
            entry_base = -1;
        }
        const int e = src.key >> p.log_page;
        if (entry_base < 0 || e + 1 >= entry_base + 32) {
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
#pragma unroll
            for (int h = 0; h < kHalves; h++) {
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
    for (int i = 0; i < kStages; i++)
        if (src_u < a1) request(i);

    // ---- sums
    PsItem it = {};
    uint32_t qf[MT][kSteps][f32 ? 4 : 2];           // queries: rows' (and their small parts') fragments
    float out[MT][kOut][4], top[MT], sum[MT], factor[MT];
    int limit[MT];
    bool alive = true;
    int began = a0;                     // the unit with which the warp's part of the item began
    for (int u = a0, n = 0; u < a1 && alive; u++, n++) {
        const int stage = n % kStages;
        if (u == a0 || u >= it.end) {
            open(it, u, u != a0);
            began = u;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const int r = 8 * m + g;
                const bool live = r < it.job.rows;
                const int tok = it.job.first + (live ? r / p.share : 0), h = it.head * p.share + (live ? r % p.share : 0);
                limit[m] = it.job.prefix ? it.job.to : it.job.to - it.job.count + (live ? r / p.share : 0) + 1;
                const A* q = static_cast<const A*>(p.q) + (size_t)tok * p.ld_q + h * p.dim;
                top[m] = -INFINITY;
                sum[m] = 0.0f;
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
                        for (int c = 0; c < 2; c++) split_16<K>(x[s][c].x * down, x[s][c].y * down, qf[m][s][2 * c], qf[m][s][2 * c + 1]);
                } else {
#pragma unroll
                    for (int s = 0; s < kSteps; s++)
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const int d = 16 * s + 8 * c + 2 * t4;
                            qf[m][s][c] = live && d < p.dim ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
                        }
                }
#pragma unroll
                for (int i = 0; i < kOut; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) out[m][i][c] = 0.0f;
            }
        }
        if (!mbar_wait_bounded(&bars[warp][stage], (uint32_t)(n / kStages) & 1u, err, 83)) { alive = false; break; }
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
        float sc[MT][2][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < 8; i++) sc[m][i >> 2][i & 3] = 0.0f;
        {
            const int r = (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                uint32_t b[4];
                ldsm4_at(b, kt + (s >> 2) * (kPsKeys * 128) + r * 128 + (((2 * (s & 3) + c) ^ (r & 7)) << 4));
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    uint32_t a[4];
                    if constexpr (f32) { a[0] = qf[m][s][0]; a[1] = qf[m][s][1]; a[2] = qf[m][s][2]; a[3] = qf[m][s][3]; }
                    else { a[0] = qf[m][s][0]; a[1] = 0; a[2] = qf[m][s][1]; a[3] = 0; }
                    mma_16<K>(sc[m][0], a, b[0], b[1]);
                    mma_16<K>(sc[m][1], a, b[2], b[3]);
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
                x[i] = sc[m][i >> 1][i & 1];
                if constexpr (f32) x[i] += sc[m][i >> 1][2 + (i & 1)];
                x[i] *= factor[m];
                if (p.cap > 0.0f) x[i] = capped<f32>(x[i], p.cap);
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
                sum[m] *= down;
#pragma unroll
                for (int i = 0; i < kOut; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) out[m][i][c] *= down;
            }
        }
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float base = top[m] == -INFINITY ? 0.0f : top[m];
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = ex2(sc[m][i >> 1][i & 1] - base);
            sum[m] += (x[0] + x[1]) + (x[2] + x[3]);
            split_16<K>(x[0], x[1], w[m][0], w[m][1]);
            split_16<K>(x[2], x[3], w[m][2], w[m][3]);
        }
        {
            const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = lane >> 4;
#pragma unroll
            for (int i = 0; i < kOut / 2; i++) {
                uint32_t b[4];
                ldsm4_t_at(b, vt + (i >> 2) * (kPsKeys * 128) + r * 128 + (((2 * (i & 3) + c) ^ (r & 7)) << 4));
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    mma_16<K>(out[m][2 * i], w[m], b[0], b[1]);
                    mma_16<K>(out[m][2 * i + 1], w[m], b[2], b[3]);
                }
            }
        }
        it.key += kPsKeys;
        __syncwarp();
        if (src_u < a1) request(stage);

        if (u + 1 < it.end && u + 1 < a1) continue;
        // ---- the warp's part of the item is complete
        const bool all = began == it.begin && u + 1 == it.end, tail = u + 1 == a1;
        if (!all) {
            if (lane == 0) parts[warp][tail] = {it.begin, it.end, it.job.first, it.job.rows, it.head, it.job.joined, it.job.prefix, 1};
        }
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float l = quad_sum(sum[m]);
            const int r = 8 * m + g;
            if (r >= it.job.rows) continue;
            const int tok = it.job.first + r / p.share, h = it.head * p.share + r % p.share;
            const size_t row = (size_t)tok * p.heads + h;
            float* dst = nullptr;
            if (all && !it.job.joined) {
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
                A* o = static_cast<A*>(p.o) + (size_t)tok * p.ld_o + h * p.dim;
#pragma unroll
                for (int i = 0; i < kOut; i++)
                    if (8 * i + 2 * t4 < p.dim) store_two<A>(o + 8 * i + 2 * t4, (out[m][i][0] + out[m][i][2]) * inv, (out[m][i][1] + out[m][i][3]) * inv);
            } else if (all) {
                dst = (it.job.prefix ? p.prefix_o : p.own_o) + row * DP;
                if (t4 == 0) (it.job.prefix ? p.prefix_ml : p.own_ml)[row] = make_float2(top[m], l);
            } else if (tail) {
                float* mine = reinterpret_cast<float*>(ring_ptr + warp * kPsRing);
                dst = mine + r * DP;
                if (t4 == 0) reinterpret_cast<float2*>(mine + kSplitRows * DP)[r] = make_float2(top[m], l);
            } else {
                const size_t at = (size_t)(cta * kPsWarps + warp) * kSplitRows + r;
                dst = p.head_o + at * DP;
                if (t4 == 0) p.head_ml[at] = make_float2(top[m], l);
            }
            if (all && t4 == 0) (it.job.prefix ? p.prefix : p.own)[row] = make_int4(cta, 1, 0, it.job.joined && !it.job.prefix ? kJoinPrefix : 0);
            if (dst)
#pragma unroll
                for (int i = 0; i < kOut; i++) store_two<float>(dst + 8 * i + 2 * t4, out[m][i][0] + out[m][i][2], out[m][i][1] + out[m][i][3]);
        }
    }
    __syncthreads();

    // ---- items that several warps have parts of
    constexpr int kCols = DP / 32;
    int turn = 0;
    for (int e = 0; e < 2 * kPsWarps;) {
        const PsPart part = parts[e >> 1][e & 1];
        if (!part.valid) { e++; continue; }
        int last = e;                   // entries e .. last: the item's
        for (int f = e + 1; f < 2 * kPsWarps; f++) {
            const PsPart& next = parts[f >> 1][f & 1];
            if (!next.valid) continue;
            if (next.begin != part.begin) break;
            last = f;
        }
        const bool starts = part.begin >= u0, all = starts && part.end <= u1;
        for (int r = 0; r < part.rows; r++) {
            if (turn++ % kPsWarps != warp) continue;
            float most = -INFINITY;
            auto ml = [&](int f) {
                return f & 1 ? reinterpret_cast<const float2*>(reinterpret_cast<const float*>(ring_ptr + (f >> 1) * kPsRing) + kSplitRows * DP)[r]
                             : p.head_ml[(size_t)(cta * kPsWarps + (f >> 1)) * kSplitRows + r];
            };
            for (int f = e; f <= last; f++)
                if (parts[f >> 1][f & 1].valid) most = fmaxf(most, ml(f).x);
            const float base = most == -INFINITY ? 0.0f : most;
            float acc[kCols], l = 0.0f;
#pragma unroll
            for (int c = 0; c < kCols; c++) acc[c] = 0.0f;
            for (int f = e; f <= last; f++) {
                if (!parts[f >> 1][f & 1].valid) continue;
                const float2 v = ml(f);
                const float w = ex2(v.x - base);
                l = fmaf(w, v.y, l);
                const float* o = (f & 1 ? reinterpret_cast<const float*>(ring_ptr + (f >> 1) * kPsRing) : p.head_o + (size_t)(cta * kPsWarps + (f >> 1)) * kSplitRows * DP) + r * DP;
#pragma unroll
                for (int c = 0; c < kCols; c++) acc[c] = fmaf(w, o[kCols * lane + c], acc[c]);
            }
            const int tok = part.first + r / p.share, h = part.head * p.share + r % p.share;
            const size_t row = (size_t)tok * p.heads + h;
            float* dst = nullptr;
            float2* dst_ml = nullptr;
            if (all && !part.joined) {
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
                A* o = static_cast<A*>(p.o) + (size_t)tok * p.ld_o + h * p.dim;
#pragma unroll
                for (int c = 0; c < kCols; c++)
                    if (kCols * lane + c < p.dim) o[kCols * lane + c] = ActOf<A>::put(acc[c] * inv);
            } else {
                const size_t at = all ? row : (size_t)(2 * cta + starts) * kSplitRows + r;
                dst = (!all ? p.split_o : (part.prefix ? p.prefix_o : p.own_o)) + at * DP;
                dst_ml = (!all ? p.split_ml : (part.prefix ? p.prefix_ml : p.own_ml)) + at;
            }
            if (dst) {
#pragma unroll
                for (int c = 0; c < kCols; c++) dst[kCols * lane + c] = acc[c];
                if (lane == 0) *dst_ml = make_float2(most, l);
            }
            if (lane == 0 && starts) {
                // the CTA with the item's last unit
                const int end = all ? cta : (int)(((long long)part.end * ctas - 1) / total);
                (part.prefix ? p.prefix : p.own)[row] = make_int4(cta, end - cta + 1, r, part.joined && !part.prefix ? kJoinPrefix : 0);
            }
        }
        e = last + 1;
    }
    if (p.mark) mark_tokens<kPsThreads>(p, err);
}

template <typename A, typename K, int DP, int MT>
static int launch_split(const PagedArgs& a, const bpdq_paged_kv& kv, int ctas, cudaStream_t s)
{
    CUtensorMap kmap, vmap;
    int rc;
    if ((rc = paged_map(&kmap, kv.k, kv, kPsKeys)) || (rc = paged_map(&vmap, kv.v, kv, kPsKeys))) return rc;
    if ((rc = allow_smem<k_paged_split<A, K, DP, MT>>(224 * 1024))) return rc;
    const size_t smem = 1024 + kPsWarps * kPsRing + (size_t)(a.batch + 2 * a.groups + 2) * 4;
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
