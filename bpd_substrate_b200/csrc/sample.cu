// A token per row of logits by temperature, top-k, top-p and min-p from a given random number (the rules stand in bpdq.h).
//
// The CTAs of a cluster hold a row between them in shared memory, each a range of the vocabulary, so that it is read once.  A weight
// w = 2^((x - max) log2(e) / T) is a whole number of 2^-44 (worked out in 64 bits, to 1e-12): sums of 2^18 of them fit 64 bits, are exact, and depend on
// no order, so neither do the cuts and the choice.  What is kept is always a beginning of the row's order (by value, then by index), hence one
// place (value, index), the cut.  It is found by a histogram, of numbers over octaves of fp32 weights or of weights over their own leading bits (exact: three
// numbers of 15 bits a weight, as shared memory adds 32): the bins above are settled, the few elements of the bin that holds the cut are listed in one
// CTA and compared with each other.  Where those are too many (flat rows, equal values) the bin is halved by exact sums until they are not.  Its own
// histogram tells a CTA what it holds of the kept weights, so only the one with the chosen token walks through them.
// Bound by the steps that follow one another, each with a meeting of the cluster, and by barriers in them: a row of 32000 11 to 14 us, 64 rows of 128256 57 (their
// bytes: 5), 300 rows of 32000 in bf16 76, two full waves and a third of four rows.
#include "cluster_device.cuh"
#include "launch.cuh"
#include "paged.cuh"

namespace bpdq {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kCountBins = 2048, kCountOctave = 32;         // numbers: bins, bins per octave of weight
constexpr int kMassBins = 1472;                             // weights: 32 per octave for the 46 octaves down to 2^-45
constexpr int kSampleList = 1024;                           // elements that are sorted
constexpr int kSampleCounted = 256;                         // elements that are compared with each other instead
constexpr int kSampleBits = 44;
constexpr int kSampleMaxVocab = 1 << 18;
constexpr int kSampleSteps = kSampleMaxVocab / 8 / 128;     // of 128 elements, in a CTA's largest range
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
    ulonglong2 pair[kSampleCounted];                        // place, weight
    unsigned hist[3 * kMassBins];
    u64 octave[64], octaves[64], bin[32];
    u64 step[kSampleSteps];
    u64 red[2][2], warp_red[kSampleWarps][2], warp_sum[kSampleWarps];
    unsigned exp_lo[32], exp_hi[32];
    unsigned list_n, found[4], least, most;
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
__device__ __forceinline__ u64 warp_most(u64 v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 t = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        if (t > v) v = t;
    }
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
    bool whole;                     // they all are
    int meetings;

    // fp32 octaves below the largest, as bins; rise as v falls.
    __device__ __forceinline__ int bin_of(float v) const { return (int)fminf((top - v) * rate * (float)kCountOctave, (float)(kCountBins - 1)); }
    // 2^44 2^y, y = (v - top) log2(e) / T = j / 32 + f, |f| <= 1/64: a table for j and the Taylor polynomial of degree 5 of 2^f (remainder 3e-15).  Without branches: several
    // of them run side by side.
    __device__ __forceinline__ double scaled(float v) const
    {
        const double d = ((double)v - top64) * rate64, y = d > -60.0 ? d : -60.0;         // (weights have long been 0 there)
        const double shift = 6755399441055744.0 / 32.0;             // 1.5 2^52 / 32: the sum's last bit is 1/32
        const double k = y + shift, f = y - (k - shift);
        const int j = __double2loint(k);
        double p = 0.0013333558146428443;
        p = fma(p, f, 0.0096181291076284772);
        p = fma(p, f, 0.055504108664821580);
        p = fma(p, f, 0.24022650695910071);
        p = fma(p, f, 0.69314718055994531);
        p = fma(p, f, 1.0);
        return p * __hiloint2double((int)s.exp_hi[j & 31] + ((j >> 5) + kSampleBits) * (1 << 20), (int)s.exp_lo[j & 31]);      // 2^44 2^(j / 32)
    }
    // To the nearest whole number.
    static __device__ __forceinline__ u64 whole_of(double z) { return (u64)(__double_as_longlong(z + 4503599627370496.0) & 0xFFFFFFFFFFFFFll); }
    __device__ __forceinline__ u64 weight(float v) const { return whole_of(scaled(v)); }
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
        a = warp_total(lane < ranks ? peer_u64(&red[0], lane) : 0);
        b = warp_total(lane < ranks ? peer_u64(&red[1], lane) : 0);
        meetings++;
    }

    static __device__ __forceinline__ u64 share_of(float part, u64 all) { return (u64)fmax(ceil((double)part * (double)all), 1.0); }
    // Bin of a weight 2^44 2^y: by its exponent and its first five bits; rises as it falls.  (At or beyond kMassBins: it rounds to 0.)
    static __device__ __forceinline__ int mass_bin(double z) { return ((1023 + kSampleBits) << 5) + 31 - (__double2hiint(z) >> 15); }
    // What this CTA's histogram holds in a bin.
    template <bool kMass> __device__ __forceinline__ u64 in_bin(int b, uint32_t r) const
    {
        if (!kMass) return peer_u32(&s.hist[b], r);
        return peer_u32(&s.hist[b], r) + ((u64)peer_u32(&s.hist[kMassBins + b], r) << 15) + ((u64)peer_u32(&s.hist[2 * kMassBins + b], r) << 30);
    }
    // The first bin, in the histogram of the cluster, up to which the sum reaches `want`, part of the sum of all or (of numbers) k; -1: none; the sum ahead of it and
    // what it holds.  All threads; one meeting.
    template <bool kMass> __device__ __forceinline__ int first_bin(float part, int k, u64& before, u64& holds, u64& want)
    {
        __syncthreads();
        for (int o = warp; o < 64; o += kSampleWarps) {
            u64 v = 0;
            const int i = 32 * o + lane;
            if (kMass && o < kMassBins / 32) v = warp_total(s.hist[i] + ((u64)s.hist[kMassBins + i] << 15) + ((u64)s.hist[2 * kMassBins + i] << 30));
            if (!kMass) v = __reduce_add_sync(0xFFFFFFFFu, s.hist[i]);
            if (lane == 0) s.octave[o] = v;
        }
        cluster_meet();
        // eight threads per octave, a rank each
        auto eight = [&](u64 v) {
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
            return v;
        };
        const uint32_t r = tid & 7;
        const u64 octave_sum = eight(r < ranks ? peer_u64(&s.octave[tid >> 3], r) : 0);
        if (r == 0) s.octaves[tid >> 3] = octave_sum;
        __syncthreads();
        const u64 two0 = s.octaves[2 * lane], two1 = s.octaves[2 * lane + 1], up = warp_scan(two0 + two1, lane);
        want = (u64)k;
        if (kMass) want = share_of(part, __shfl_sync(0xFFFFFFFFu, up, 31));
        const unsigned who0 = __ballot_sync(0xFFFFFFFFu, up - two1 >= want), who1 = __ballot_sync(0xFFFFFFFFu, up >= want);
        if (!who1) {
            before = __shfl_sync(0xFFFFFFFFu, up, 31);
            holds = 0;
            return -1;
        }
        const int l0 = who0 ? __ffs(who0) - 1 : 32, lead = min(l0, __ffs(who1) - 1), octave = 2 * lead + (l0 == lead ? 0 : 1);
        const u64 ahead = __shfl_sync(0xFFFFFFFFu, up - two1 - (l0 == lead ? two0 : 0), lead);
        const u64 bin_sum = eight(tid < 256 && r < ranks ? in_bin<kMass>(32 * octave + (tid >> 3), r) : 0);
        if (tid < 256 && r == 0) s.bin[tid >> 3] = bin_sum;
        __syncthreads();
        const u64 mine = s.bin[lane], run = ahead + warp_scan(mine, lane);
        const int l = __ffs(__ballot_sync(0xFFFFFFFFu, run >= want)) - 1;
        before = __shfl_sync(0xFFFFFFFFu, run - mine, l);
        holds = __shfl_sync(0xFFFFFFFFu, mine, l);
        return 32 * octave + l;
    }
    // f(whether it is a kept one of the bin, value, index) for what fp32 does not tell from this CTA's elements of bin b of weights; all lanes together.
    template <class F> __device__ __forceinline__ void each_in_bin(int bin, F f) const
    {
        const int sub = 31 - (bin & 31);
        // octaves below the largest, and 10^-4 beyond: more than fp32 is off by
        const float least = (float)(bin >> 5) - log2f(1.0f + (float)(sub + 1) / 32.0f) - 1e-4f, most = (float)(bin >> 5) - log2f(1.0f + (float)sub / 32.0f) + 1e-4f;
        each([&](const float (&v)[4], int i) {
            unsigned maybe = 0, sure = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float d = (top - v[j]) * rate;
                if (d >= least && d <= most && (whole || kept(v[j], i + j))) {
                    maybe |= 1u << j;
                    if (d > least + 2e-4f && d < most - 2e-4f) sure |= 1u << j;
                }
            }
            if (!__any_sync(0xFFFFFFFFu, maybe)) return;
            // at the bin's ends the weight itself tells
            if (__any_sync(0xFFFFFFFFu, maybe != sure)) {
#pragma unroll 1
                for (int j = 0; j < 4; j++) {
                    const float a = j == 0 ? v[0] : (j == 1 ? v[1] : (j == 2 ? v[2] : v[3]));
                    if (mass_bin(scaled(a)) == bin) sure |= maybe & 1u << j;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) f((sure >> j & 1u) != 0, v[j], i + j);
        });
    }

    // Puts the place where `yes` holds into this CTA's list, while there is room; list_n counts them all.
    __device__ __forceinline__ void list_if(bool yes, u64 place) const
    {
        const unsigned who = __ballot_sync(0xFFFFFFFFu, yes);
        if (!who) return;
        unsigned at = 0;
        if (lane == 0) at = atomicAdd(&s.list_n, __popc(who));
        at = __shfl_sync(0xFFFFFFFFu, at, 0) + __popc(who & ((1u << lane) - 1));
        if (yes && at < kSampleList) s.list[at] = place;
    }
    // Of the CTAs' lists (after a meeting): how many places they hold.
    __device__ __forceinline__ unsigned listed() const { return __reduce_add_sync(0xFFFFFFFFu, lane < ranks ? peer_u32(&s.list_n, lane) : 0u); }
    // Rank 0 appends the others' lists to its own; up to kSampleList places in all.
    __device__ __forceinline__ void collect()
    {
        const unsigned n = lane < ranks ? peer_u32(&s.list_n, lane) : 0u, ahead = warp_scan(n, lane) - n;
        const uint32_t r = (uint32_t)warp & (ranks - 1);
        const unsigned from = __shfl_sync(0xFFFFFFFFu, ahead, r), count = __shfl_sync(0xFFFFFFFFu, n, r);
        if (r > 0)
            for (unsigned i = 32 * (warp / ranks) + lane; i < count; i += 32 * (kSampleWarps / ranks)) s.list[from + i] = peer_u64(&s.list[i], r);
        __syncthreads();
    }
    // For element tid / parts of the n <= kSampleCounted in s.pair: how many of the others lie ahead of it, and the sum of their weights; in all of its threads, of
    // which there are `parts`, neighbours.
    __device__ __forceinline__ void counted(int n, int parts, u64 mine, int& ahead, u64& mass) const
    {
        ahead = 0;
        mass = 0;
        if (tid / parts < n) {
            for (int i = tid & (parts - 1); i < n; i += parts) {
                const ulonglong2 e = s.pair[i];
                if (e.x > mine) { ahead++; mass += e.y; }
            }
        }
        for (int o = parts / 2; o > 0; o >>= 1) {
            ahead += __shfl_xor_sync(0xFFFFFFFFu, ahead, o);
            mass += __shfl_xor_sync(0xFFFFFFFFu, mass, o);
        }
    }
    static __device__ __forceinline__ int parts_for(int n)
    {
        int parts = 2;
        while (parts < 32 && 2 * parts * n <= kSampleThreads) parts *= 2;
        return parts;
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

    // Sums of this thread's warp's and CTA's predecessors, in the vocabulary's order, over the cluster; sum: of the warp; all: of the cluster.  One meeting.
    __device__ __forceinline__ u64 ahead_of_warp(u64 mine, u64& sum, u64& all)
    {
        sum = warp_total(mine);
        if (lane == 0) s.warp_sum[warp] = sum;
        __syncthreads();
        const u64 of = lane < kSampleWarps ? s.warp_sum[lane] : 0;
        u64 before = warp_total(lane < warp ? of : 0);
        const u64 cta = warp_total(of);
        if (tid == 0) s.answer[0] = cta;
        cluster_meet();
        const u64 peer = lane < ranks ? peer_u64(&s.answer[0], lane) : 0;
        before += warp_total(lane < rank ? peer : 0);
        all = warp_total(peer);
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
    u64 mine = 0, sum, all;
    w.each([&](const float (&a)[4], int i) {
#pragma unroll 1
        for (int j = 0; j < 4; j++) mine += equal(a[j], i + j);
    });
    const u64 run = w.ahead_of_warp(mine, sum, all);
    if (run < nth && nth <= run + sum)
        w.walk(run, nth, equal, [&](u64 place) {
#pragma unroll 1
            for (uint32_t r = 0; r < w.ranks; r++) peer_store_u64(&w.s.answer[2], r, place);
        });
    cluster_meet();
    w.cut = w.s.answer[2];
    return true;
}

// The cut among the border's elements, which the CTAs have listed (after a meeting).  All threads of the cluster.
template <bool kMass>
__device__ __forceinline__ void cut_in_list(Sampler& w, const Border& b)
{
    if (w.rank == 0) {
        const int n = (int)b.count;
        SampleShared& s = w.s;
        w.collect();
        auto one = [&](u64 place) -> u64 { return kMass ? w.weight(place_value(place)) : 1; };
        if (n <= kSampleCounted) {
            if (w.tid < n) s.pair[w.tid] = make_ulonglong2(s.list[w.tid], one(s.list[w.tid]));
            __syncthreads();
            const int parts = Sampler::parts_for(n), j = w.tid / parts;
            ulonglong2 mine = make_ulonglong2(0, 0);
            if (j < n) mine = s.pair[j];
            int ahead;
            u64 mass;
            w.counted(n, parts, mine.x, ahead, mass);
            // the element that reaches the sum (the last one, should none)
            if (j < n && b.above + mass < b.want && (b.above + mass + mine.y >= b.want || ahead == n - 1))
                for (int r = w.tid & (parts - 1); r < (int)w.ranks; r += parts) peer_store_u64(&s.answer[2], (uint32_t)r, mine.x);
        } else {
            sort_list(s.list, n, w.tid);
            w.scan_weights(n, [&](int i) -> u64 { return one(s.list[i]); });
            const int at = w.first_reaching(n, b.want - b.above);
            if (w.tid < (int)w.ranks) peer_store_u64(&s.answer[2], (uint32_t)w.tid, s.list[at < n ? at : n - 1]);
        }
    }
    cluster_meet();
    w.cut = w.s.answer[2];
    w.whole = false;
}
// The same of any number of elements, the kept ones whose bin of the histogram is b (count of them).
template <bool kMass>
__device__ __noinline__ u64 cut_in_bin(Sampler w, int bin, u64 count, u64 above, u64 want)
{
    SampleShared& s = w.s;
    auto in = [&](float v, int i) { return v > -INFINITY && w.kept(v, i) && (kMass ? Sampler::mass_bin(w.scaled(v)) : w.bin_of(v)) == bin; };
    unsigned lo = 0xFFFFFFFFu, hi = 0;
    w.each([&](const float (&v)[4], int i) {
#pragma unroll 1
        for (int j = 0; j < 4; j++)
            if (in(v[j], i + j)) { lo = min(lo, order_of(v[j])); hi = max(hi, order_of(v[j])); }
    });
    lo = __reduce_min_sync(0xFFFFFFFFu, lo);
    hi = __reduce_max_sync(0xFFFFFFFFu, hi);
    if (w.tid == 0) { s.least = 0xFFFFFFFFu; s.most = 0; s.list_n = 0; }
    __syncthreads();
    if (w.lane == 0) { atomicMin(&s.least, lo); atomicMax(&s.most, hi); }
    cluster_meet();
    Border b = {__reduce_min_sync(0xFFFFFFFFu, w.lane < w.ranks ? peer_u32(&s.least, w.lane) : 0xFFFFFFFFu),
                __reduce_max_sync(0xFFFFFFFFu, w.lane < w.ranks ? peer_u32(&s.most, w.lane) : 0u), count, above, want};
    if (narrow<kMass>(w, b)) return w.cut;
    w.each([&](const float (&v)[4], int i) {
#pragma unroll 1
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
    if (tid == 0) s.list_n = 0;
    for (int i = tid; i < 3 * kMassBins / 4; i += kSampleThreads) reinterpret_cast<uint4*>(s.hist)[i] = make_uint4(0, 0, 0, 0);
    pdl_wait();
    pdl_launch_dependents();

    // ---- the row, and its first place
    const float temperature = p.temperature ? p.temperature[row] : 1.0f;
    const int k = p.top_k ? p.top_k[row] : 0;
    const float part = p.top_p ? p.top_p[row] : 1.0f, least = p.min_p && p.min_p[row] > 0.0f ? fminf(p.min_p[row], 1.0f) : 0.0f;       // (a setting that is NaN is none)
    const double u = fmin(fmax((double)p.u[row], 0.0), 1.0 - 1.0 / 16777216.0);
    float best = -INFINITY;
    int best_at = 0x7FFFFFFF;
    auto take = [&](int i, float v) {
        v = v > -INFINITY ? v + 0.0f : -INFINITY;                // NaN too; -0 becomes 0, which it is equal to, so that equal numbers have one place by value
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
    first = warp_most(first);
    if (lane == 0) s.warp_sum[warp] = first;
    __syncthreads();
    if (warp == 0) {
        first = warp_most(lane < kSampleWarps ? s.warp_sum[lane] : 0);
        if (lane == 0) s.answer[1] = first;
    }
    cluster_meet();
    first = warp_most(lane < w.ranks ? peer_u64(&s.answer[1], lane) : 0);
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
    if (w.top == INFINITY) {
        // infinite logits share everything: as 0 beside -inf
        for (int i = tid; i < kSampleWarps * w.chunk; i += kSampleThreads) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
        w.top = 0.0f;
        __syncthreads();
    }
    // beyond this temperature all logits but the lowest numbers of fp32 weigh the same
    const float warm = fminf(temperature, 8e36f);
    w.top64 = (double)w.top;
    w.rate64 = kLog2e / (double)warm;
    w.rate = fminf((float)w.rate64, 3e38f);
    w.cut = place_of(-INFINITY, -1) + 1;                         // everything but -inf
    w.whole = true;
    const bool cut_k = k > 0 && k < p.vocab, cut_p = part < 1.0f, cut_m = least > 0.0f;
    // the least logit with w >= min_p, w rounded to 64 bits (1 - 2^-54 is 1)
    float floor_m = -INFINITY;
    if (cut_m) {
        floor_m = __double2float_ru(w.top64 + (log2((double)least) - kLog2e / 18014398509481984.0) / w.rate64);
        if (!(floor_m <= w.top)) floor_m = w.top;
    }
    auto answer = [&](float v, int i, u64 all) {
        p.token[row] = i;
        if (p.logprob) p.logprob[row] = (float)(((double)v - w.top64) / (double)warm - log((double)all * (1.0 / (double)(1ull << kSampleBits))));
    };
    cluster_wait();

    if (cut_k) {
        w.each([&](const float (&v)[4], int) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (v[j] > -INFINITY) atomicAdd(&s.hist[w.bin_of(v[j])], 1u);
        });
        u64 before, holds, want;
        const int found = w.first_bin<false>(0.0f, k, before, holds, want);
        const int b = found < 0 ? kCountBins : found, above = (int)before, in_bin = (int)holds;      // (all, where there are fewer than k)
        if (above + in_bin <= kSampleList) {
            // ---- few enough for one CTA to finish
            w.each([&](const float (&v)[4], int i) {
                bool in[4];
#pragma unroll
                for (int j = 0; j < 4; j++) in[j] = v[j] > -INFINITY && w.bin_of(v[j]) <= b;
                if (!__any_sync(0xFFFFFFFFu, in[0] || in[1] || in[2] || in[3])) return;
#pragma unroll 1
                for (int j = 0; j < 4; j++) w.list_if(in[j], place_of(v[j], i + j));
            });
            cluster_meet();
            if (w.rank != 0) {
                cluster_meet();                                  // until rank 0 has the list
                return;
            }
            w.collect();
            cluster_meet();
            const int n = above + in_bin;
            if (n <= kSampleCounted) {
                // An element is kept if fewer than k and less than the share of top_p lie ahead of it: both counted from the list as it is.
                const int parts = Sampler::parts_for(n), j = tid / parts;
                if (tid < n) s.pair[tid] = make_ulonglong2(s.list[tid], w.weight(place_value(s.list[tid])));
                __syncthreads();
                ulonglong2 mine = make_ulonglong2(0, 0);
                if (j < n) mine = s.pair[j];
                int ahead;
                u64 mass;
                w.counted(n, parts, mine.x, ahead, mass);
                const bool lead = (tid & (parts - 1)) == 0, in_k = j < n && ahead < k;
                const u64 all_k = w.cta_total(lead && in_k ? mine.y : 0);
                const u64 want = cut_p ? Sampler::share_of(part, all_k) : ~0ull;
                const bool keep = in_k && mass < want && place_value(mine.x) >= floor_m;
                if (lead && j < n && !keep) s.pair[j].y = 0;
                const u64 sum = w.cta_total(lead && keep ? mine.y : 0), goal = (u64)(u * (double)sum) + 1;
                u64 upto = 0;                                    // of indices up to its own
                if (keep)
#pragma unroll 4
                    for (int i = tid & (parts - 1); i < n; i += parts) {
                        const ulonglong2 e = s.pair[i];
                        if ((unsigned)e.x >= (unsigned)mine.x) upto += e.y;
                    }
                for (int o = parts / 2; o > 0; o >>= 1) upto += __shfl_xor_sync(0xFFFFFFFFu, upto, o);
                if (lead && keep && upto >= goal && upto - mine.y < goal) answer(place_value(mine.x), place_index(mine.x), sum);
                return;
            }
            sort_list(s.list, n, tid);
            int keep = n < k ? n : k;
            w.scan_weights(keep, [&](int i) { return w.weight(place_value(s.list[i])); });
            if (cut_p) {
                const int at = w.first_reaching(keep, Sampler::share_of(part, s.weight[keep - 1]));
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
        if (b < kCountBins) {
            w.cut = cut_in_bin<false>(w, b, (u64)in_bin, (u64)above, (u64)k);
            w.whole = false;
        }
        if (cut_p) {
            cluster_meet();                                      // (the histogram is still being read)
            for (int i = tid; i < 3 * kMassBins / 4; i += kSampleThreads) reinterpret_cast<uint4*>(s.hist)[i] = make_uint4(0, 0, 0, 0);
            if (tid == 0) s.list_n = 0;
            __syncthreads();
        }
    }
    // ---- what this CTA holds of the kept weights
    u64 mine = 0;
    if (cut_p) {
        w.each([&](const float (&v)[4], int i) {
            double z[4];
#pragma unroll
            for (int j = 0; j < 4; j++) z[j] = w.scaled(v[j]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (!w.whole && !w.kept(v[j], i + j)) z[j] = 0.0;
                const int b = Sampler::mass_bin(z[j]);
                const u64 wt = Sampler::whole_of(z[j]);
                if (b < kMassBins) {
                    atomicAdd(&s.hist[b], (unsigned)wt & 0x7FFFu);
                    const unsigned middle = (unsigned)(wt >> 15) & 0x7FFFu, upper = (unsigned)(wt >> 30);
                    if (middle) atomicAdd(&s.hist[kMassBins + b], middle);
                    if (upper) atomicAdd(&s.hist[2 * kMassBins + b], upper);
                }
            }
        });
        bool in_list = false;                                    // the elements of the cut's bin are this CTA's list
        u64 above, holds, want;
        const int b = w.first_bin<true>(part, 0, above, holds, want);
        if (b >= 0) {
            w.each_in_bin(b, [&](bool yes, float v, int i) { w.list_if(yes, place_of(v, i)); });
            cluster_meet();
            const u64 count = w.listed();
            if (count <= kSampleList) {
                Border border;
                border.lo = border.hi = 0;
                border.count = count;
                border.above = above;
                border.want = want;
                cut_in_list<true>(w, border);
                in_list = w.rank != 0 || count <= kSampleCounted;        // (longer ones have been sorted there, with the others')
            } else {
                cluster_meet();                                  // (everyone has read the number)
                w.cut = cut_in_bin<true>(w, b, count, above, want);
                w.whole = false;
            }
        }
        const u64 floor_place = (u64)order_of(floor_m) << 32;
        if (floor_m > -INFINITY && floor_place > w.cut) { w.cut = floor_place; w.whole = in_list = false; }
        // the bins above the cut's, by the CTA's own histogram, and of that bin the elements from the cut on
        int last = kMassBins;
        if (!w.whole) {
            const int of_cut = Sampler::mass_bin(w.scaled(place_value(w.cut)));
            if (of_cut < last) last = of_cut;
        }
        for (int i = tid; i < last; i += kSampleThreads) mine += s.hist[i] + ((u64)s.hist[kMassBins + i] << 15) + ((u64)s.hist[2 * kMassBins + i] << 30);
        if (in_list) {
            const int own = (int)s.list_n;
            for (int i = tid; i < own; i += kSampleThreads)
                if (s.list[i] >= w.cut) mine += w.weight(place_value(s.list[i]));
        } else if (last < kMassBins) w.each_in_bin(last, [&](bool yes, float v, int) { if (yes) mine += w.weight(v); });
    } else {
        const u64 floor_place = (u64)order_of(floor_m) << 32;
        if (floor_m > -INFINITY && floor_place > w.cut) { w.cut = floor_place; w.whole = false; }
        w.each([&](const float (&v)[4], int i) {
            bool in[4];
#pragma unroll
            for (int j = 0; j < 4; j++) in[j] = w.whole || w.kept(v[j], i + j);
            if (!__any_sync(0xFFFFFFFFu, in[0] || in[1] || in[2] || in[3])) return;
            u64 wt[4];
#pragma unroll
            for (int j = 0; j < 4; j++) wt[j] = w.weight(v[j]);
#pragma unroll
            for (int j = 0; j < 4; j++) mine += in[j] ? wt[j] : 0;
        });
    }
    // ---- the choice: the CTA, then the step of 128 elements, then the element
    const u64 held = w.cta_total(mine);
    if (tid == 0) s.answer[0] = held;
    cluster_meet();
    const u64 peer = lane < w.ranks ? peer_u64(&s.answer[0], lane) : 0, all = warp_total(peer);
    u64 run = warp_total(lane < w.rank ? peer : 0);
    cluster_arrive();                                            // nobody leaves before all have read
    const u64 goal = (u64)(u * (double)all) + 1;
    if (run < goal && goal <= run + held) {
        auto share = [&](const float (&v)[4], int i, u64 (&wt)[4]) {
#pragma unroll
            for (int j = 0; j < 4; j++) wt[j] = w.weight(v[j]);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (!w.whole && !w.kept(v[j], i + j)) wt[j] = 0;
        };
        int at = warp * (w.chunk / 128);
        w.each([&](const float (&v)[4], int i) {
            u64 wt[4];
            share(v, i, wt);
            const u64 sum = warp_total(wt[0] + wt[1] + wt[2] + wt[3]);
            if (lane == 0) s.step[at] = sum;
            at++;
        });
        __syncthreads();
        if (warp == 0) {
            const int steps = kSampleWarps * w.chunk / 128;
            for (int i0 = 0; i0 < steps; i0 += 32) {
                const u64 up = run + warp_scan(i0 + lane < steps ? s.step[i0 + lane] : 0, lane);
                const unsigned who = __ballot_sync(0xFFFFFFFFu, up >= goal);
                if (!who) {
                    run = __shfl_sync(0xFFFFFFFFu, up, 31);
                    continue;
                }
                const int l = __ffs(who) - 1, i = 128 * (i0 + l) + 4 * lane;
                if (l > 0) run = __shfl_sync(0xFFFFFFFFu, up, l - 1);
                const float4 f = *reinterpret_cast<const float4*>(x + i);
                const float v[4] = {f.x, f.y, f.z, f.w};
                u64 wt[4];
                share(v, w.base + i, wt);
                u64 sum = run + warp_scan(wt[0] + wt[1] + wt[2] + wt[3], lane);
                const unsigned in = __ballot_sync(0xFFFFFFFFu, sum >= goal);
                if (lane == __ffs(in) - 1) {
                    // its last element at which the sum is still there without those behind it
                    float value = v[3];
                    int index = w.base + i + 3;
#pragma unroll
                    for (int j = 3; j > 0; j--) {
                        sum -= wt[j];
                        if (sum >= goal) { value = v[j - 1]; index = w.base + i + j - 1; }
                    }
                    answer(value, index, all);
                }
                break;
            }
        }
    }
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
