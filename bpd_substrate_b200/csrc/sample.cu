// A token per row of logits by temperature, top-k, top-p and min-p from a given random number (the rules stand in bpdq.h).
//
// The CTAs of a cluster hold a row between them in shared memory, each a range of the vocabulary, so that it is read once.  A weight
// w = 2^((x - max) log2(e) / T) is a whole number of 2^-44 (worked out in 64 bits, to 1e-12): sums of 2^18 of them fit 64 bits, are exact, and depend on
// no order, so neither do the cuts and the choice.  What is kept is always a beginning of the row's order (by value, then by index), hence one
// place (value, index), the cut.  It is found by a histogram over octaves of weight (32 bins each): the bins that certainly lie above are settled, the few
// elements of the bin that holds the cut are sorted.  Where those are too many (flat rows, equal values) the bin is halved by exact sums until
// they are not.
#include "cluster_device.cuh"
#include "launch.cuh"
#include "paged.cuh"

namespace bpdq {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048, kSampleOctave = 32;       // bins, bins per octave of weight: 64 octaves, far more than a weight has bits
constexpr int kSampleOctaves = kSampleBins / kSampleOctave;
constexpr int kSampleList = 1024;                           // elements that are sorted
constexpr int kSampleCounted = 256;                         // elements that are compared with each other instead
constexpr int kSampleBits = 44;
constexpr int kSampleMaxVocab = 1 << 18;
constexpr double kLog2e = 1.4426950408889634074;
typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    int ld, vocab, slice, chunk;                            // elements of a CTA, a multiple of 8; of a warp, a multiple of 128
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    long long* token;
    float* logprob;
};

struct SampleShared {
    u64 list[kSampleList];                                  // places
    u64 weight[kSampleList];
    unsigned hist[kSampleBins];
    double octave[kSampleOctaves];
    u64 red[2][2], warp_red[kSampleWarps][2], warp_sum[kSampleWarps];
    unsigned exp_lo[32], exp_hi[32];
    unsigned list_n, found[4], least, most;
    double before;
    u64 answer[3];
};

__device__ __forceinline__ unsigned order_of(float x)
{
    const unsigned b = __float_as_uint(x);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
// Larger: earlier in the row's order.
__device__ __forceinline__ u64 place_of(float x, int i) { return (u64)order_of(x) << 32 | (unsigned)~i; }
__device__ __forceinline__ float place_value(u64 p) { return value_of((unsigned)(p >> 32)); }
__device__ __forceinline__ int place_index(u64 p) { return (int)~(unsigned)p; }

__device__ __forceinline__ u64 peer_u64(const u64* p, uint32_t rank)
{
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ unsigned peer_u32(const unsigned* p, uint32_t rank)
{
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ double peer_f64(const double* p, uint32_t rank) { return __longlong_as_double((long long)peer_u64(reinterpret_cast<const u64*>(p), rank)); }
__device__ __forceinline__ unsigned peer_add(unsigned* p, uint32_t rank, unsigned v)
{
    unsigned old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(peer_addr(p, rank)), "r"(v) : "memory");
    return old;
}
__device__ __forceinline__ void peer_store_u64(u64* p, uint32_t rank, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(peer_addr(p, rank)), "l"(v) : "memory"); }
__device__ __forceinline__ void cluster_meet() { cluster_arrive(); cluster_wait(); }

template <typename T> struct RowLoad;
template <> struct RowLoad<float> {
    static constexpr int unit = 4;
    static __device__ __forceinline__ void get(const float* p, float (&x)[4]) { const float4 v = *reinterpret_cast<const float4*>(p); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
};
template <> struct RowLoad<__half> {
    static constexpr int unit = 8;
    static __device__ __forceinline__ void get(const __half* p, float (&x)[8])
    {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; i++) { const float2 f = __half22float2(h[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    }
};
template <> struct RowLoad<bf16> {
    static constexpr int unit = 8;
    static __device__ __forceinline__ void get(const bf16* p, float (&x)[8]) { act_load_group(p, x); }
};

__device__ __forceinline__ u64 warp_total(u64 v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
template <typename T> __device__ __forceinline__ T warp_scan(T v, int lane)
{
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const T t = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

// Sorts the first n (padded to a power of two, up to the whole list) places, the largest first.  All threads.
__device__ __noinline__ void sort_list(u64* list, int n, int tid)
{
    int size = 32;
    while (size < n) size *= 2;
#pragma unroll 1
    for (int i = n + tid; i < size; i += kSampleThreads) list[i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int k = 2; k <= size; k *= 2)
#pragma unroll 1
        for (int j = k / 2; j > 0; j /= 2) {
#pragma unroll 1
            for (int t = tid; t < size / 2; t += kSampleThreads) {
                const int i = 2 * t - (t & (j - 1)), l = i + j;
                const u64 a = list[i], b = list[l];
                if ((a < b) == ((i & k) == 0)) { list[i] = b; list[l] = a; }
            }
            __syncthreads();
        }
}

struct Sampler {
    SampleShared& s;
    const float* x;                 // this CTA's elements, -inf behind the last one
    int base, chunk;                // the first one's index; elements of a warp, a multiple of 128
    int tid, lane, warp;
    uint32_t rank, ranks;
    float top, rate;                // the largest logit; log2(e) / T
    double top64, rate64;
    u64 cut;                        // places >= cut are kept
    int meetings;

    // In octaves below the largest; falls with x.
    __device__ __forceinline__ float octaves(float v) const { return v == top ? 0.0f : (top - v) * rate; }
    __device__ __forceinline__ int bin_of(float v) const { return (int)fminf(octaves(v) * (float)kSampleOctave, (float)(kSampleBins - 1)); }
    // 2^44 2^y, y = (v - top) log2(e) / T: y = j / 32 + f, |f| <= 1/64, a table for j and the Taylor polynomial of degree 5 of 2^f (remainder 3e-15).  Without branches: several
    // of them run side by side.
    __device__ __forceinline__ u64 weight(float v) const
    {
        const double y = fmax(((double)v - top64) * rate64, -60.0);         // (NaN, beside infinity: nothing)
        const double shift = 6755399441055744.0 / 32.0;             // 1.5 2^52 / 32: the sum's last bit is 1/32
        const double k = y + shift, f = y - (k - shift);
        const int j = __double2loint(k);
        double p = 0.0013333558146428443;
        p = fma(p, f, 0.0096181291076284772);
        p = fma(p, f, 0.055504108664821580);
        p = fma(p, f, 0.24022650695910071);
        p = fma(p, f, 0.69314718055994531);
        p = fma(p, f, 1.0);
        const double t = __hiloint2double((int)s.exp_hi[j & 31] + ((j >> 5) + kSampleBits) * (1 << 20), (int)s.exp_lo[j & 31]);      // 2^44 2^(j / 32)
        const u64 w = (u64)(__double_as_longlong(fma(p, t, 4503599627370496.0)) & 0xFFFFFFFFFFFFFll);       // to the nearest whole number
        return v == top ? 1ull << kSampleBits : w;
    }
    __device__ __forceinline__ bool kept(float v, int i) const { return place_of(v, i) >= cut; }
    // f(four neighbouring values, index of the first) for the warp's elements, 128 at a time in the order of the vocabulary, all lanes together.
    template <class F> __device__ __forceinline__ void each(F f) const
    {
#pragma unroll 1
        for (int i = warp * chunk + 4 * lane, n = 0; n < chunk; i += 128, n += 128) {
            const float4 v = *reinterpret_cast<const float4*>(x + i);
            const float a[4] = {v.x, v.y, v.z, v.w};
            f(a, base + i);
        }
    }

    // Sums over the cluster, in every thread.  The slots alternate, so that one is read while the next is written.
    __device__ __forceinline__ void total(u64& a, u64& b)
    {
        a = warp_total(a);
        b = warp_total(b);
        if (lane == 0) { s.warp_red[warp][0] = a; s.warp_red[warp][1] = b; }
        __syncthreads();
        u64* red = s.red[meetings & 1];
        if (warp < 2) {
            const u64 v = warp_total(lane < kSampleWarps ? s.warp_red[lane][warp] : 0);
            if (lane == 0) red[warp] = v;
        }
        cluster_meet();
        a = b = 0;
#pragma unroll 1
        for (uint32_t r = 0; r < ranks; r++) { a += peer_u64(&red[0], r); b += peer_u64(&red[1], r); }
        meetings++;
    }

    // Of the histogram's octaves, the sums of this CTA (of weights: in units of theirs).
    __device__ __forceinline__ void sum_octaves(bool mass)
    {
        __syncthreads();
        static_assert(kSampleThreads * 4 == kSampleBins && kSampleOctave == 32, "eight threads per octave");
        const uint4 h = reinterpret_cast<const uint4*>(s.hist)[tid];
        u64 v = (u64)h.x + h.y + h.z + h.w;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
        if ((tid & 7) == 0) s.octave[tid >> 3] = (double)v * (mass ? unit_of(tid >> 3) : 1.0);
    }
    // The histogram's weights are multiples of 2^-16 of their octave's largest.
    static __device__ __forceinline__ double unit_of(int octave) { return __hiloint2double((1023 + kSampleBits - 16 - octave) << 20, 0); }
    // Walks the merged histogram, octave by octave and then bin by bin (warp 0; after a meeting): the first bin b for which reached(sum up to b, sum of all) holds, or
    // kSampleBins; the sum ahead of it.
    template <class R> __device__ __forceinline__ int first_bin(bool mass, R reached, double& before) const
    {
        double o[2] = {0.0, 0.0};
#pragma unroll 1
        for (uint32_t r = 0; r < ranks; r++)
#pragma unroll
            for (int i = 0; i < 2; i++) o[i] += peer_f64(&s.octave[2 * lane + i], r);
        const double up = warp_scan(o[0] + o[1], lane), all = __shfl_sync(0xFFFFFFFFu, up, 31);
        const unsigned who0 = __ballot_sync(0xFFFFFFFFu, reached(up - o[1], all)), who1 = __ballot_sync(0xFFFFFFFFu, reached(up, all));
        before = all;
        if (!(who0 | who1)) return kSampleBins;
        // octave 2 l is reached first where lane l is the first in who0 and none ahead of it is in who1
        const int l0 = who0 ? __ffs(who0) - 1 : 32, l1 = who1 ? __ffs(who1) - 1 : 32, lead = min(l0, l1);
        const int octave = 2 * lead + (l0 <= l1 ? 0 : 1);
        const double ahead = __shfl_sync(0xFFFFFFFFu, up - o[1] - (l0 <= l1 ? o[0] : 0.0), lead);
        u64 h = 0;
#pragma unroll 1
        for (uint32_t r = 0; r < ranks; r++) h += peer_u32(&s.hist[32 * octave + lane], r);
        const double mine = (double)h * (mass ? unit_of(octave) : 1.0), run = ahead + warp_scan(mine, lane);
        const unsigned who = __ballot_sync(0xFFFFFFFFu, reached(run, all));
        const int b = who ? __ffs(who) - 1 : 31;
        before = __shfl_sync(0xFFFFFFFFu, run - mine, b);
        return 32 * octave + b;
    }

    // Puts the place where `yes` holds into rank 0's list, while there is room; list_n counts them all.
    __device__ __forceinline__ void list_if(bool yes, u64 place) const
    {
        const unsigned who = __ballot_sync(0xFFFFFFFFu, yes);
        if (!who) return;
        unsigned at = 0;
        if (lane == 0) at = peer_add(&s.list_n, 0, __popc(who));
        at = __shfl_sync(0xFFFFFFFFu, at, 0) + __popc(who & ((1u << lane) - 1));
        if (yes && at < kSampleList) peer_store_u64(&s.list[at], 0, place);
    }

    // s.weight[i] = sum of f(0) .. f(i), i < n <= 1024.
    template <class F> __device__ __forceinline__ void scan_weights(int n, F f)
    {
        const u64 a = 2 * tid < n ? f(2 * tid) : 0, b = 2 * tid + 1 < n ? f(2 * tid + 1) : 0, sum = warp_scan(a + b, lane);
        if (lane == 31) s.warp_sum[warp] = sum;
        __syncthreads();
        u64 before = sum - a - b;
#pragma unroll 1
        for (int w = 0; w < warp; w++) before += s.warp_sum[w];
        if (2 * tid < n) s.weight[2 * tid] = before + a;
        if (2 * tid + 1 < n) s.weight[2 * tid + 1] = before + a + b;
        __syncthreads();
    }
    // The first i < n with s.weight[i] >= want; n if there is none.
    __device__ __forceinline__ int first_reaching(int n, u64 want)
    {
        if (tid == 0) s.found[0] = n;
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < n; i += kSampleThreads)
            if (s.weight[i] >= want && (i == 0 || s.weight[i - 1] < want)) s.found[0] = i;
        __syncthreads();
        const int i = s.found[0];
        __syncthreads();
        return i;
    }
    // Sum over the CTA, in every thread.
    __device__ __forceinline__ u64 cta_total(u64 v)
    {
        v = warp_total(v);
        if (lane == 0) s.warp_sum[warp] = v;
        __syncthreads();
        v = warp_total(lane < kSampleWarps ? s.warp_sum[lane] : 0);
        __syncthreads();
        return v;
    }

    // Sums of this thread's warp's and CTA's predecessors, in the vocabulary's order, over the cluster; sum: of the warp.  One meeting.
    __device__ __forceinline__ u64 ahead_of_warp(u64 mine, u64& sum)
    {
        sum = warp_total(mine);
        if (lane == 0) s.warp_sum[warp] = sum;
        __syncthreads();
        u64 before = 0, cta = 0;
#pragma unroll 1
        for (int w = 0; w < kSampleWarps; w++) {
            if (w < warp) before += s.warp_sum[w];
            cta += s.warp_sum[w];
        }
        if (tid == 0) s.answer[0] = cta;
        cluster_meet();
#pragma unroll 1
        for (uint32_t r = 0; r < rank; r++) before += peer_u64(&s.answer[0], r);
        return before;
    }
    // found(place) in the lane that holds the first element at which the sum of f, `run` ahead of the warp, reaches want.
    template <class F, class G> __device__ __forceinline__ void walk(u64 run, u64 want, F f, G found)
    {
        bool done = false;
        each([&](const float (&v)[4], int i) {
            if (done) return;
            u64 a[4], mine = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) { a[j] = f(v[j], i + j); mine += a[j]; }
            const u64 up = warp_scan(mine, lane);
            const unsigned who = __ballot_sync(0xFFFFFFFFu, run + up >= want);
            if (who) {
                done = true;
                if (lane == __ffs(who) - 1) {
                    u64 at = run + up - mine;
                    bool yet = true;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        at += a[j];
                        if (yet && at >= want) { yet = false; found(place_of(v[j], i + j)); }
                    }
                }
            }
            run += __shfl_sync(0xFFFFFFFFu, up, 31);
        });
    }
};

// Keys (order_of) between which the cut lies, how many kept elements have them, the sum above them, and the sum at which it is.
struct Border {
    unsigned lo, hi;
    u64 count, above, want;
};
// More elements than are sorted: the range of keys is halved by exact sums until there are not; equal values are told apart by their index.  True: the cut is
// known; false: the border's elements are few.  All threads of the cluster.
template <bool kMass>
__device__ __forceinline__ bool narrow(Sampler& w, Border& b)
{
    auto one = [&](float v) -> u64 { return kMass ? w.weight(v) : 1; };
    while (b.count > kSampleList && b.lo < b.hi) {
        const unsigned mid = b.lo + (b.hi - b.lo) / 2;
        u64 upper = 0, count = 0;
        w.each([&](const float (&v)[4], int i) {
#pragma unroll 1
            for (int j = 0; j < 4; j++) {
                const unsigned k = order_of(v[j]);
                if (k > mid && k <= b.hi && w.kept(v[j], i + j)) { upper += one(v[j]); count++; }
            }
        });
        w.total(upper, count);
        if (b.above + upper >= b.want) { b.lo = mid + 1; b.count = count; }
        else { b.hi = mid; b.above += upper; b.count -= count; }
    }
    if (b.lo < b.hi) return false;
    const float v = value_of(b.lo);
    const u64 each_one = one(v), nth = each_one ? (b.want - b.above + each_one - 1) / each_one : 1;
    auto equal = [&](float a, int i) -> u64 { return a == v && w.kept(a, i); };
    u64 mine = 0, sum;
    w.each([&](const float (&a)[4], int i) {
#pragma unroll 1
        for (int j = 0; j < 4; j++) mine += equal(a[j], i + j);
    });
    const u64 run = w.ahead_of_warp(mine, sum);
    if (run < nth && nth <= run + sum)
        w.walk(run, nth, equal, [&](u64 place) {
#pragma unroll 1
            for (uint32_t r = 0; r < w.ranks; r++) peer_store_u64(&w.s.answer[2], r, place);
        });
    cluster_meet();
    w.cut = w.s.answer[2];
    return true;
}

// The cut among the border's elements, which are listed in rank 0.  All threads of the cluster.
template <bool kMass>
__device__ __forceinline__ void cut_in_list(Sampler& w, const Border& b)
{
    if (w.rank == 0) {
        const int n = (int)b.count;
        sort_list(w.s.list, n, w.tid);
        w.scan_weights(n, [&](int i) -> u64 { return kMass ? w.weight(place_value(w.s.list[i])) : 1; });
        const int at = w.first_reaching(n, b.want - b.above);
        if (w.tid < (int)w.ranks) peer_store_u64(&w.s.answer[2], (uint32_t)w.tid, w.s.list[at < n ? at : n - 1]);
        if (w.tid == 0) w.s.list_n = 0;
    }
    cluster_meet();
    w.cut = w.s.answer[2];
}
// Lists the border's elements (list_n is 0), then as above.
template <bool kMass>
__device__ __noinline__ u64 cut_at_border(Sampler w, Border b, int& meetings)
{
    const bool known = narrow<kMass>(w, b);
    meetings = w.meetings;
    if (known) return w.cut;
    w.each([&](const float (&v)[4], int i) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned k = order_of(v[j]);
            w.list_if(k >= b.lo && k <= b.hi && w.kept(v[j], i + j), place_of(v[j], i + j));
        }
    });
    cluster_meet();
    cut_in_list<kMass>(w, b);
    return w.cut;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) k_sample(const SampleArgs p)
{
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ SampleShared s;
    float* x = reinterpret_cast<float*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x;
    Sampler w{s, x};
    w.tid = tid; w.lane = lane; w.warp = warp;
    w.rank = cluster_rank(); w.ranks = cluster_size();
    w.base = (int)w.rank * p.slice;
    const int n = max(0, min(p.vocab - w.base, p.slice));
    w.chunk = p.chunk;
    w.meetings = 0;
    if (tid < 32) {
        const double t = exp2((double)tid / 32.0);
        s.exp_lo[tid] = (unsigned)__double2loint(t);
        s.exp_hi[tid] = (unsigned)__double2hiint(t);
    }
    if (tid == 0) { s.list_n = 0; s.least = 0xFFFFFFFFu; s.most = 0; }
    reinterpret_cast<uint4*>(s.hist)[tid] = make_uint4(0, 0, 0, 0);
    pdl_wait();
    pdl_launch_dependents();

    // ---- the row, and its first place
    const float temperature = p.temperature ? p.temperature[row] : 1.0f;
    const int k = p.top_k ? p.top_k[row] : 0;
    const float part = p.top_p ? p.top_p[row] : 1.0f, least = p.min_p ? fminf(p.min_p[row], 1.0f) : 0.0f;
    const double u = fmin(fmax((double)p.u[row], 0.0), 1.0 - 1.0 / 16777216.0);
    float best = -INFINITY;
    int best_at = 0x7FFFFFFF;
    auto take = [&](int i, float v) {
        if (!(v > -INFINITY)) v = -INFINITY;                     // NaN too
        if (v > best) { best = v; best_at = i; }                 // (a thread's indices rise)
        return v;
    };
    const T* from = static_cast<const T*>(p.logits) + (size_t)row * p.ld + w.base;
    constexpr int unit = RowLoad<T>::unit;
    const int units = ((uintptr_t)from & 15) == 0 ? n / unit : 0;
#pragma unroll 4
    for (int i = tid; i < units; i += kSampleThreads) {
        float v[unit];
        RowLoad<T>::get(from + i * unit, v);
#pragma unroll
        for (int j = 0; j < unit; j++) v[j] = take(i * unit + j, v[j]);
#pragma unroll
        for (int j = 0; j < unit; j += 4) *reinterpret_cast<float4*>(x + i * unit + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
#pragma unroll 1
    for (int i = units * unit + tid; i < n; i += kSampleThreads) x[i] = take(i, ActOf<T>::get(from[i]));
#pragma unroll 1
    for (int i = n + tid; i < kSampleWarps * w.chunk; i += kSampleThreads) x[i] = -INFINITY;
    u64 first = place_of(best, w.base + best_at);
    if (best == -INFINITY) first = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xFFFFFFFFu, first, o);
        if (other > first) first = other;
    }
    if (lane == 0) s.warp_sum[warp] = first;
    __syncthreads();
    if (warp == 0) {
        first = s.warp_sum[lane & (kSampleWarps - 1)];
#pragma unroll
        for (int o = kSampleWarps / 2; o > 0; o >>= 1) {
            const u64 other = __shfl_xor_sync(0xFFFFFFFFu, first, o);
            if (other > first) first = other;
        }
        if (lane == 0) s.answer[1] = first;
    }
    cluster_meet();
    first = 0;
#pragma unroll 1
    for (uint32_t r = 0; r < w.ranks; r++) {
        const u64 other = peer_u64(&s.answer[1], r);
        if (other > first) first = other;
    }
    cluster_arrive();                                            // (answer[1] is not written again; nobody leaves before all have read)
    const bool lead = w.rank == 0 && tid == 0, none = first == 0;
    if (none || !(temperature > 0.0f)) {
        if (lead) {
            p.token[row] = none ? -1 : (long long)place_index(first);
            if (p.logprob) p.logprob[row] = none ? -INFINITY : 0.0f;
        }
        cluster_wait();
        return;
    }
    w.top = place_value(first);
    w.top64 = (double)w.top;
    w.rate64 = kLog2e / (double)temperature;
    w.rate = (float)w.rate64;
    w.cut = place_of(-INFINITY, -1) + 1;                         // everything but -inf
    const bool cut_k = k > 0 && k < p.vocab, cut_p = part < 1.0f, cut_m = least > 0.0f;
    // the least logit with w >= min_p, w rounded to 64 bits (1 - 2^-54 is 1)
    float floor_m = -INFINITY;
    if (cut_m && w.top < INFINITY && w.rate64 > 0.0) {           // (otherwise weights are 1 and 0, or all 1)
        floor_m = __double2float_ru(w.top64 + (log2((double)least) - kLog2e / 18014398509481984.0) / w.rate64);
        if (!(floor_m <= w.top)) floor_m = w.top;
    }
    auto answer = [&](float v, int i, u64 all) {
        p.token[row] = i;
        if (p.logprob) p.logprob[row] = (float)((v == w.top ? 0.0 : ((double)v - w.top64) / (double)temperature) - log((double)all * (1.0 / (double)(1ull << kSampleBits))));
    };
    cluster_wait();

    if (cut_k) {
        w.each([&](const float (&v)[4], int) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (v[j] > -INFINITY) atomicAdd(&s.hist[w.bin_of(v[j])], 1u);
        });
        w.sum_octaves(false);
        cluster_meet();
        if (warp == 0) {
            double before;
            const int b = w.first_bin(false, [&](double up, double) { return up >= (double)k; }, before);
            // elements in bins up to it (all, where there are fewer than k)
            unsigned in_bin = 0;
            if (b < kSampleBins)
#pragma unroll 1
                for (uint32_t r = 0; r < w.ranks; r++) in_bin += peer_u32(&s.hist[b], r);
            if (lane == 0) { s.found[1] = (unsigned)b; s.found[2] = (unsigned)before; s.found[3] = in_bin; }
        }
        __syncthreads();
        const int b = (int)s.found[1], above = (int)s.found[2], in_bin = (int)s.found[3];
        if (above + in_bin <= kSampleList) {
            // ---- few enough for one CTA to finish
            w.each([&](const float (&v)[4], int i) {
                // one vote for four: most have none
                const bool any = (v[0] > -INFINITY && w.bin_of(v[0]) <= b) || (v[1] > -INFINITY && w.bin_of(v[1]) <= b) || (v[2] > -INFINITY && w.bin_of(v[2]) <= b) ||
                                 (v[3] > -INFINITY && w.bin_of(v[3]) <= b);
                if (!__any_sync(0xFFFFFFFFu, any)) return;
#pragma unroll
                for (int j = 0; j < 4; j++) w.list_if(v[j] > -INFINITY && w.bin_of(v[j]) <= b, place_of(v[j], i + j));
            });
            cluster_meet();
            if (w.rank != 0) return;
            const int n = above + in_bin;
            if (n <= kSampleCounted) {
                // An element is kept if fewer than k and less than the share of top_p lie ahead of it: both counted from the list as it is.
                const u64 mine = tid < n ? s.list[tid] : 0, wt = tid < n ? w.weight(place_value(mine)) : 0;
                if (tid < n) s.weight[tid] = wt;
                __syncthreads();
                int ahead = 0;
                u64 mass = 0;
                if (tid < n)
#pragma unroll 4
                    for (int i = 0; i < n; i++)
                        if (s.list[i] > mine) { ahead++; mass += s.weight[i]; }
                const bool in_k = tid < n && ahead < k;
                const u64 all_k = w.cta_total(in_k ? wt : 0);
                const u64 want = cut_p ? (u64)fmax(ceil((double)part * (double)all_k), 1.0) : ~0ull;
                const bool keep = in_k && mass < want && place_value(mine) >= floor_m;
                if (tid < n) s.weight[tid] = keep ? wt : 0;
                const u64 sum = w.cta_total(keep ? wt : 0), goal = (u64)(u * (double)sum) + 1;
                u64 upto = 0;
                if (keep) {
#pragma unroll 4
                    for (int i = 0; i < n; i++)
                        if ((unsigned)s.list[i] >= (unsigned)mine) upto += s.weight[i];           // indices up to its own
                    if (upto >= goal && upto - wt < goal) answer(place_value(mine), place_index(mine), sum);
                }
                return;
            }
            sort_list(s.list, n, tid);
            int keep = n < k ? n : k;
            w.scan_weights(keep, [&](int i) { return w.weight(place_value(s.list[i])); });
            if (cut_p) {
                const int at = w.first_reaching(keep, (u64)fmax(ceil((double)part * (double)s.weight[keep - 1]), 1.0));
                keep = at < keep ? at + 1 : keep;
            }
            if (cut_m) {
                if (tid == 0) s.found[0] = 0;
                __syncthreads();
#pragma unroll 1
                for (int i = tid; i < keep; i += kSampleThreads)
                    if (place_value(s.list[i]) >= floor_m && (i + 1 == keep || place_value(s.list[i + 1]) < floor_m)) s.found[0] = i + 1;
                __syncthreads();
                keep = (int)s.found[0];
                __syncthreads();
            }
            // in the order of the vocabulary: the largest ~index first
            u64 mine[2];
            for (int j = 0; j < 2; j++) {
                const int i = tid + j * kSampleThreads;
                mine[j] = i < keep ? s.list[i] << 32 | s.list[i] >> 32 : 0;
            }
            __syncthreads();
            for (int j = 0; j < 2; j++)
                if (tid + j * kSampleThreads < keep) s.list[tid + j * kSampleThreads] = mine[j];
            __syncthreads();
            sort_list(s.list, keep, tid);
            w.scan_weights(keep, [&](int i) { return w.weight(value_of((unsigned)s.list[i])); });
            const u64 sum = s.weight[keep - 1];
            const int at = w.first_reaching(keep, (u64)(u * (double)sum) + 1);
            if (tid == 0) {
                const u64 e = s.list[at < keep ? at : keep - 1];
                answer(value_of((unsigned)e), (int)~(unsigned)(e >> 32), sum);
            }
            return;
        }
        if (b < kSampleBins) {
            // the bin's keys, then its elements
            unsigned lo = 0xFFFFFFFFu, hi = 0;
            w.each([&](const float (&v)[4], int) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (v[j] > -INFINITY && w.bin_of(v[j]) == b) { lo = min(lo, order_of(v[j])); hi = max(hi, order_of(v[j])); }
            });
            lo = __reduce_min_sync(0xFFFFFFFFu, lo);
            hi = __reduce_max_sync(0xFFFFFFFFu, hi);
            if (lane == 0) { atomicMin(&s.least, lo); atomicMax(&s.most, hi); }
            cluster_meet();
#pragma unroll 1
            for (uint32_t r = 0; r < w.ranks; r++) { lo = min(lo, peer_u32(&s.least, r)); hi = max(hi, peer_u32(&s.most, r)); }
            int meetings;
            w.cut = cut_at_border<false>(w, Border{lo, hi, (u64)in_bin, (u64)above, (u64)k}, meetings);
            w.meetings = meetings;
        }
        if (cut_p) {
            cluster_meet();                                      // (the histogram and the bounds are still being read)
            reinterpret_cast<uint4*>(s.hist)[tid] = make_uint4(0, 0, 0, 0);
            if (tid == 0) { s.least = 0xFFFFFFFFu; s.most = 0; }
            __syncthreads();
        }
    }
    // what the choice is made by, as far as it is known: places above the bins with the cut
    u64 mine = 0;
    unsigned lo = 0, hi = 0xFFFFFFFFu;                           // keys of elements that are not in it yet
    if (cut_p) {
        u64 sum = 0, nothing = 0;
        // per bin, the weights as multiples of 2^-16 of its octave's, rounded up: within 2^-14 of the bin's sum, errors of fp32 octaves included
        w.each([&](const float (&v)[4], int i) {
            bool in[4];
            u64 wt[4];
#pragma unroll
            for (int j = 0; j < 4; j++) { in[j] = w.kept(v[j], i + j); wt[j] = w.weight(v[j]); }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float d = w.octaves(v[j]);
                if (in[j]) sum += wt[j];
                if (in[j] && d < (float)kSampleOctaves) atomicAdd(&s.hist[(int)(d * (float)kSampleOctave)], (unsigned)(ex2(floorf(d) - d) * 65536.0f) + 1u);
            }
        });
        w.sum_octaves(true);
        w.total(sum, nothing);
        const u64 want = (u64)fmax(ceil((double)part * (double)sum), 1.0);
        if (warp == 0) {
            // the sum up to a bin from either side: whichever is less is known better
            const double m = (double)sum, goal = (double)want, slack = (double)p.vocab, err = 1.0 / 16384.0;
            double before;
            const int b1 = w.first_bin(true, [&](double up, double all) { return fmin(up * (1.0 + err), m - fmax(all - up, 0.0) * (1.0 - err)) + slack >= goal; }, before);
            const int b2 = w.first_bin(true, [&](double up, double all) { return fmax(up * (1.0 - err), m - fmax(all - up, 0.0) * (1.0 + err)) - slack >= goal; }, before);
            if (lane == 0) { s.found[1] = (unsigned)min(b1, kSampleBins - 1); s.found[2] = (unsigned)min(b2, kSampleBins - 1); }
        }
        __syncthreads();
        const int b1 = (int)s.found[1], b2 = (int)s.found[2];
        // the exact sum above, and the elements of the bins with the cut
        u64 above = 0;
        lo = 0xFFFFFFFFu;
        hi = 0;
        w.each([&](const float (&v)[4], int i) {
            bool over[4], in[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int b = w.bin_of(v[j]);
                const bool yes = w.kept(v[j], i + j);
                over[j] = yes && b < b1;
                in[j] = yes && b >= b1 && b <= b2;
            }
            if (__any_sync(0xFFFFFFFFu, over[0] || over[1] || over[2] || over[3])) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const u64 wt = w.weight(v[j]);
                    if (over[j]) { above += wt; if (v[j] >= floor_m) mine += wt; }
                }
            }
            if (__any_sync(0xFFFFFFFFu, in[0] || in[1] || in[2] || in[3])) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (in[j]) { lo = min(lo, order_of(v[j])); hi = max(hi, order_of(v[j])); }
                    w.list_if(in[j], place_of(v[j], i + j));
                }
            }
        });
        lo = __reduce_min_sync(0xFFFFFFFFu, lo);
        hi = __reduce_max_sync(0xFFFFFFFFu, hi);
        if (lane == 0) { atomicMin(&s.least, lo); atomicMax(&s.most, hi); }
        w.total(above, nothing);
        Border b = {0xFFFFFFFFu, 0, (u64)peer_u32(&s.list_n, 0), above, want};
#pragma unroll 1
        for (uint32_t r = 0; r < w.ranks; r++) { b.lo = min(b.lo, peer_u32(&s.least, r)); b.hi = max(b.hi, peer_u32(&s.most, r)); }
        lo = b.lo;
        hi = b.hi;
        if (b.count > 0 && b.count <= kSampleList) {
            cut_in_list<true>(w, b);
        } else if (b.count > kSampleList) {
            cluster_meet();                                      // (everyone has read their number)
            if (w.rank == 0 && tid == 0) s.list_n = 0;
            cluster_meet();
            int meetings;
            w.cut = cut_at_border<true>(w, b, meetings);
        }
    }
    // ---- the choice
    auto share = [&](float v, int i) -> u64 { return w.kept(v, i) && v >= floor_m ? w.weight(v) : 0; };
    w.each([&](const float (&v)[4], int i) {
        bool in[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned key = order_of(v[j]);
            in[j] = key >= lo && key <= hi && w.kept(v[j], i + j) && v[j] >= floor_m;
        }
        if (!__any_sync(0xFFFFFFFFu, in[0] || in[1] || in[2] || in[3])) return;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const u64 wt = w.weight(v[j]);
            if (in[j]) mine += wt;
        }
    });
    u64 sum;
    const u64 run = w.ahead_of_warp(mine, sum);
    u64 all = 0;
#pragma unroll 1
    for (uint32_t r = 0; r < w.ranks; r++) all += peer_u64(&s.answer[0], r);
    cluster_arrive();                                            // nobody leaves before all have read
    const u64 goal = (u64)(u * (double)all) + 1;
    if (run < goal && goal <= run + sum) w.walk(run, goal, share, [&](u64 e) { answer(place_value(e), place_index(e), all); });
    cluster_wait();
}

// CTAs of a cluster: as many as hold a row in 64 KB of shared memory each (two such fit an SM), more while the rows leave SMs idle.
static int sample_ctas(int rows, int vocab)
{
    int n = 1;
    while (n < 8 && (vocab + n - 1) / n * 4 > 64 * 1024) n *= 2;
    while (n < 8 && rows * n * 2 <= sm_count() && vocab / n > 4096) n *= 2;
    return n;
}

template <typename T>
static int launch_sample(SampleArgs p, int rows, cudaStream_t s)
{
    const int n = sample_ctas(rows, p.vocab);
    p.slice = ((p.vocab + n - 1) / n + 7) / 8 * 8;
    p.chunk = (p.slice + 128 * kSampleWarps - 1) / (128 * kSampleWarps) * 128;
    int rc = allow_smem<k_sample<T>>(160 * 1024);
    if (rc) return rc;
    return launch_cluster(k_sample<T>, dim3((unsigned)rows, (unsigned)n), dim3(1, (unsigned)n), kSampleThreads, (size_t)p.chunk * kSampleWarps * 4, s, p);
}

}  // namespace bpdq

using namespace bpdq;

extern "C" int bpd_sample_cuda(const void* logits, int logits_type, int ld, int rows, int vocab, const float* temperature, const int32_t* top_k, const float* top_p,
                               const float* min_p, const float* u, long long* token, float* logprob, void* stream)
{
    if (!logits || !u || !token || rows < 0 || vocab < 1 || ld < vocab || logits_type < BPDQ_TYPE_F32 || logits_type > BPDQ_TYPE_BF16) return latch(BPDQ_ERR_ARG);
    if (vocab > kSampleMaxVocab) return latch(BPDQ_ERR_RANGE);
    if ((uintptr_t)logits & (logits_type == BPDQ_TYPE_F32 ? 3 : 1)) return latch(BPDQ_ERR_ALIGN);
    if (rows == 0) return 0;
    SampleArgs p = {};
    p.logits = logits; p.ld = ld; p.vocab = vocab; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p; p.u = u;
    p.token = token; p.logprob = logprob;
    cudaStream_t s = (cudaStream_t)stream;
    if (logits_type == BPDQ_TYPE_F32) return launch_sample<float>(p, rows, s);
    return logits_type == BPDQ_TYPE_F16 ? launch_sample<__half>(p, rows, s) : launch_sample<bf16>(p, rows, s);
}
