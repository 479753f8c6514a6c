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
constexpr int kSampleList = 1024;                           // elements that are sorted
constexpr int kSampleBits = 44;
constexpr int kSampleMaxVocab = 1 << 18;
constexpr double kLog2e = 1.4426950408889634074;
typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    int ld, vocab, slice;                                   // slice: elements of a CTA, a multiple of 8
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    long long* token;
    float* logprob;
};

struct SampleShared {
    u64 list[kSampleList];
    union {
        u64 weight[kSampleList];
        double merged[kSampleBins];
    };
    unsigned hist[kSampleBins];
    double part[kSampleWarps][2];
    u64 red[2][2], warp_red[kSampleWarps][2], warp_sum[kSampleWarps];
    unsigned exp_lo[32], exp_hi[32];
    unsigned list_n, found[4];
    u64 answer[3];
};

__device__ __forceinline__ unsigned order_of(float x)
{
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
// Larger: earlier in the row's order.
__device__ __forceinline__ u64 place_of(float x, int i) { return (u64)order_of(x) << 32 | (unsigned)~i; }

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

struct Sampler {
    SampleShared& s;
    const float* x;                 // this CTA's elements, -inf behind the last one
    int n, base, chunk;             // their number, the first one's index, elements of a warp
    int tid, lane, warp;
    uint32_t rank, ranks;
    float top, rate;                // the largest logit; log2(e) / T
    double rate64;
    u64 cut;                        // places >= cut are kept
    int meetings;

    // In octaves below the largest; falls with x.
    __device__ __forceinline__ float octaves(float v) const { return v == top ? 0.0f : (top - v) * rate; }
    // 2^44 2^y, y = (v - top) log2(e) / T: y = j / 32 + f, |f| <= 1/64, a table for j and the Taylor polynomial of degree 5 of 2^f (remainder 3e-15).
    __device__ __forceinline__ u64 weight(float v) const
    {
        if (v == top) return 1ull << kSampleBits;
        const double y = ((double)v - (double)top) * rate64;
        if (!(y > -(kSampleBits + 1.0))) return 0;
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
        return (u64)(__double_as_longlong(fma(p, t, 4503599627370496.0)) & 0xFFFFFFFFFFFFFll);       // to the nearest whole number
    }
    __device__ __forceinline__ bool kept(float v, int i) const { return place_of(v, i) >= cut; }
    // f(value, index) for the warp's elements in the order of the vocabulary, 32 at a time, all lanes together (-inf behind the last one).
    template <class F> __device__ __forceinline__ void each(F f) const
    {
        const int from = warp * chunk, to = from + chunk < n ? from + chunk : n;
        for (int i = from + lane; i - lane < to; i += 32) f(i < to ? x[i] : -INFINITY, base + i);
    }

    __device__ __forceinline__ u64 warp_total(u64 v) const
    {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
        return v;
    }
    // Sums over the cluster, in every thread.  The slots alternate, so that one is read while the next is written.
    __device__ __forceinline__ void total(u64& a, u64& b)
    {
        a = warp_total(a);
        b = warp_total(b);
        if (lane == 0) { s.warp_red[warp][0] = a; s.warp_red[warp][1] = b; }
        __syncthreads();
        u64* red = s.red[meetings & 1];
        if (tid < 2) {
            u64 v = 0;
            for (int w = 0; w < kSampleWarps; w++) v += s.warp_red[w][tid];
            red[tid] = v;
        }
        cluster_meet();
        a = b = 0;
        for (uint32_t r = 0; r < ranks; r++) { a += peer_u64(&red[0], r); b += peer_u64(&red[1], r); }
        meetings++;
    }

    // The histogram summed over the cluster, each bin times 2^-octave for weights.
    __device__ void merge_bins(bool mass)
    {
        cluster_meet();
        const int share = kSampleBins / ranks, from = share * rank;
        for (int b = tid; b < share; b += kSampleThreads) {
            u64 v = 0;
            for (uint32_t r = 0; r < ranks; r++) v += peer_u32(&s.hist[from + b], r);
            double m = (double)v;
            if (mass) m *= __hiloint2double((1023 + kSampleBits - 16 - (from + b) / kSampleOctave) << 20, 0);
            s.merged[from + b] = m;
        }
        cluster_meet();
        for (int b = tid; b < kSampleBins; b += kSampleThreads)
            if (b < from || b >= from + share) s.merged[b] = peer_f64(&s.merged[b], b / share);
        __syncthreads();
    }
    // Sums of merged bins ahead of this thread's four and in all.
    __device__ void scan_bins(double& before, double& all)
    {
        double mine = 0.0;
        for (int i = 0; i < 4; i++) mine += s.merged[4 * tid + i];
        double sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const double v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) s.part[warp][0] = sum;
        __syncthreads();
        before = 0.0;
        all = 0.0;
        for (int w = 0; w < kSampleWarps; w++) {
            if (w < warp) before += s.part[w][0];
            all += s.part[w][0];
        }
        before += sum - mine;
        __syncthreads();
    }

    // Elements that want(value, index) picks, in rank 0's list, up to its size; the number that there are.
    template <class F> __device__ unsigned gather(F want)
    {
        if (tid == 0) s.list_n = 0;
        cluster_meet();
        each([&](float v, int i) {
            const bool yes = want(v, i);
            const unsigned who = __ballot_sync(0xFFFFFFFFu, yes);
            if (!who) return;
            unsigned at = 0;
            if (lane == 0) at = peer_add(&s.list_n, 0, __popc(who));
            at = __shfl_sync(0xFFFFFFFFu, at, 0) + __popc(who & ((1u << lane) - 1));
            if (yes && at < kSampleList) peer_store_u64(&s.list[at], 0, place_of(v, i));
        });
        cluster_meet();
        return peer_u32(&s.list_n, 0);
    }
    // Sorts the first n (padded to a power of two) of the list, the largest first.
    __device__ void sort_list(int n)
    {
        int size = 32;
        while (size < n) size *= 2;
        for (int i = n + tid; i < size; i += kSampleThreads) s.list[i] = 0;
        __syncthreads();
        for (int k = 2; k <= size; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                for (int t = tid; t < size / 2; t += kSampleThreads) {
                    const int i = 2 * t - (t & (j - 1)), l = i + j;
                    const u64 a = s.list[i], b = s.list[l];
                    if ((a < b) == ((i & k) == 0)) { s.list[i] = b; s.list[l] = a; }
                }
                __syncthreads();
            }
    }
    // s.weight[i] = sum of f(0) .. f(i), i < n <= 1024.
    template <class F> __device__ void scan_weights(int n, F f)
    {
        u64 a = 2 * tid < n ? f(2 * tid) : 0, b = 2 * tid + 1 < n ? f(2 * tid + 1) : 0, sum = a + b;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const u64 v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) s.warp_sum[warp] = sum;
        __syncthreads();
        u64 before = 0;
        for (int w = 0; w < warp; w++) before += s.warp_sum[w];
        before += sum - a - b;
        if (2 * tid < n) s.weight[2 * tid] = before + a;
        if (2 * tid + 1 < n) s.weight[2 * tid + 1] = before + a + b;
        __syncthreads();
    }
    // The first i < n with s.weight[i] >= want; n if there is none.
    __device__ int first_reaching(int n, u64 want)
    {
        if (tid == 0) s.found[0] = n;
        __syncthreads();
        for (int i = tid; i < n; i += kSampleThreads)
            if (s.weight[i] >= want && (i == 0 || s.weight[i - 1] < want)) s.found[0] = i;
        __syncthreads();
        const int i = s.found[0];
        __syncthreads();
        return i;
    }
    __device__ __forceinline__ float list_value(int i) const { return value_of((unsigned)(s.list[i] >> 32)); }
    __device__ __forceinline__ int list_index(int i) const { return (int)~(unsigned)s.list[i]; }

    // Of the kept elements equal to v the one with `nth` (from 1) of them up to it, in the vocabulary's order; its place, everywhere.
    __device__ u64 nth_equal(float v, u64 nth)
    {
        u64 mine = 0;
        each([&](float w, int i) { mine += w == v && kept(w, i); });
        return locate(mine, nth, [&](float w, int i) -> u64 { return w == v && kept(w, i); });
    }
    // The place of the first element, in the vocabulary's order, at which the sum of f reaches want; mine: what this thread adds to it.
    template <class F> __device__ u64 locate(u64 mine, u64 want, F f)
    {
        const u64 sum = warp_total(mine);
        if (lane == 0) s.warp_sum[warp] = sum;
        __syncthreads();
        u64 before = 0, cta = 0;
        for (int w = 0; w < kSampleWarps; w++) {
            if (w < warp) before += s.warp_sum[w];
            cta += s.warp_sum[w];
        }
        if (tid == 0) s.answer[0] = cta;
        cluster_meet();
        for (uint32_t r = 0; r < rank; r++) before += peer_u64(&s.answer[0], r);
        if (before < want && want <= before + sum) {
            u64 run = before;
            bool done = false;
            each([&](float v, int i) {
                if (done) return;
                const u64 a = f(v, i);
                u64 up = a;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const u64 t = __shfl_up_sync(0xFFFFFFFFu, up, o);
                    if (lane >= o) up += t;
                }
                const unsigned who = __ballot_sync(0xFFFFFFFFu, run + up >= want);
                if (who) {
                    done = true;
                    if (lane == __ffs(who) - 1)
                        for (uint32_t r = 0; r < ranks; r++) peer_store_u64(&s.answer[1], r, place_of(v, i));
                }
                run += __shfl_sync(0xFFFFFFFFu, up, 31);
            });
        }
        cluster_meet();
        return s.answer[1];
    }

    // Moves the cut to the first place at which the kept elements' f, in the row's order, reaches `want`, which all of them do; the place is known to
    // lie among those with keys lo .. hi (order_of), c of them, and those above add up to `above`.
    template <class F> __device__ void narrow(unsigned lo, unsigned hi, u64 c, u64 above, u64 want, F f)
    {
        if (c == 0) return;
        while (c > kSampleList && lo < hi) {
            const unsigned mid = lo + (hi - lo) / 2;
            u64 upper = 0, count = 0;
            each([&](float v, int i) {
                const unsigned k = order_of(v);
                if (k > mid && k <= hi && kept(v, i)) { upper += f(v); count++; }
            });
            total(upper, count);
            if (above + upper >= want) { lo = mid + 1; c = count; }
            else { hi = mid; above += upper; c -= count; }
        }
        if (lo == hi) {
            const float v = value_of(lo);
            const u64 one = f(v), each_one = one ? one : 1;
            cut = nth_equal(v, (want - above + each_one - 1) / each_one);
            return;
        }
        const int got = (int)gather([&](float v, int i) { const unsigned k = order_of(v); return k >= lo && k <= hi && kept(v, i); });
        if (rank == 0) {
            sort_list(got);
            scan_weights(got, [&](int i) { return f(list_value(i)); });
            const int at = first_reaching(got, want - above);
            if (tid < (int)ranks) peer_store_u64(&s.answer[2], (uint32_t)tid, s.list[at < got ? at : got - 1]);
        }
        cluster_meet();
        cut = s.answer[2];
    }
    __device__ __forceinline__ int bin_of(float v) const { return (int)fminf(octaves(v) * (float)kSampleOctave, (float)(kSampleBins - 1)); }
    // Keys of the kept elements in bins b1 .. b2, their number, and the sum of f above them.
    template <class F> __device__ void bounds(int b1, int b2, unsigned& lo, unsigned& hi, u64& c, u64& above, F f)
    {
        u64 sum = 0, count = 0;
        unsigned least = 0xFFFFFFFFu, most = 0;
        each([&](float v, int i) {
            if (!kept(v, i)) return;
            const int b = bin_of(v);
            if (b < b1) sum += f(v);
            else if (b <= b2) { const unsigned k = order_of(v); count++; least = min(least, k); most = max(most, k); }
        });
        least = __reduce_min_sync(0xFFFFFFFFu, least);
        most = __reduce_max_sync(0xFFFFFFFFu, most);
        if (tid == 0) { s.found[1] = 0xFFFFFFFFu; s.found[2] = 0; }
        __syncthreads();
        if (lane == 0) { atomicMin(&s.found[1], least); atomicMax(&s.found[2], most); }
        total(sum, count);
        lo = 0xFFFFFFFFu;
        hi = 0;
        for (uint32_t r = 0; r < ranks; r++) { lo = min(lo, peer_u32(&s.found[1], r)); hi = max(hi, peer_u32(&s.found[2], r)); }
        c = count;
        above = sum;
        cluster_meet();
    }
};

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) k_sample(const SampleArgs p)
{
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ SampleShared s;
    float* x = reinterpret_cast<float*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x;
    pdl_launch_dependents();
    if (tid < 32) {
        const double t = exp2((double)tid / 32.0);
        s.exp_lo[tid] = (unsigned)__double2loint(t);
        s.exp_hi[tid] = (unsigned)__double2hiint(t);
    }
    Sampler w{s, x};
    w.tid = tid; w.lane = lane; w.warp = warp;
    w.rank = cluster_rank(); w.ranks = cluster_size();
    w.base = (int)w.rank * p.slice;
    w.n = p.vocab - w.base < p.slice ? p.vocab - w.base : p.slice;
    if (w.n < 0) w.n = 0;
    w.chunk = (w.n + kSampleThreads - 1) / kSampleThreads * 32;
    w.meetings = 0;
    pdl_wait();

    // ---- the row, and its first place
    u64 best = 0;
    auto take = [&](int i, float v) {
        if (!(v > -INFINITY)) v = -INFINITY;                     // NaN too
        x[i] = v;
        const u64 k = place_of(v, w.base + i);
        if (k > best) best = k;
    };
    const T* from = static_cast<const T*>(p.logits) + (size_t)row * p.ld + w.base;
    constexpr int unit = RowLoad<T>::unit;
    int done = 0;
    if (((uintptr_t)from & 15) == 0) {
        done = w.n / unit * unit;
#pragma unroll 4
        for (int i = tid * unit; i < done; i += kSampleThreads * unit) {
            float v[unit];
            RowLoad<T>::get(from + i, v);
#pragma unroll
            for (int j = 0; j < unit; j++) take(i + j, v[j]);
        }
    }
    for (int i = done + tid; i < w.n; i += kSampleThreads) take(i, ActOf<T>::get(from[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xFFFFFFFFu, best, o);
        if (other > best) best = other;
    }
    if (lane == 0) s.warp_sum[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kSampleWarps; i++)
            if (s.warp_sum[i] > best) best = s.warp_sum[i];
        s.answer[2] = best;
    }
    cluster_meet();
    best = 0;
    for (uint32_t r = 0; r < w.ranks; r++) {
        const u64 other = peer_u64(&s.answer[2], r);
        if (other > best) best = other;
    }
    cluster_meet();
    w.top = value_of((unsigned)(best >> 32));

    const float temperature = p.temperature ? p.temperature[row] : 1.0f;
    const bool lead = w.rank == 0 && tid == 0;
    if (w.top == -INFINITY || !(temperature > 0.0f)) {
        if (lead) {
            p.token[row] = w.top == -INFINITY ? -1 : (long long)~(unsigned)best;
            if (p.logprob) p.logprob[row] = w.top == -INFINITY ? -INFINITY : 0.0f;
        }
        return;
    }
    w.rate64 = kLog2e / (double)temperature;
    w.rate = (float)w.rate64;
    w.cut = place_of(-INFINITY, -1) + 1;                         // everything but -inf
    const int k = p.top_k ? p.top_k[row] : 0;
    const float part = p.top_p ? p.top_p[row] : 1.0f, least = p.min_p ? fminf(p.min_p[row], 1.0f) : 0.0f;
    const bool cut_k = k > 0 && k < p.vocab, cut_p = part < 1.0f, cut_m = least > 0.0f;
    // the least logit with w >= min_p, w rounded to 64 bits (1 - 2^-54 is 1)
    float floor_m = cut_m ? __double2float_ru((double)w.top + (log2((double)least) - kLog2e / 18014398509481984.0) / w.rate64) : -INFINITY;
    if (!(floor_m <= w.top)) floor_m = w.top;
    if (w.top == INFINITY || w.rate64 == 0.0) floor_m = -INFINITY;       // weights are 1 and 0, or all 1
    const double u = fmin(fmax((double)p.u[row], 0.0), 1.0 - 1.0 / 16777216.0);

    auto one = [](float) -> u64 { return 1; };
    auto mass = [&](float v) { return w.weight(v); };
    auto answer = [&](float v, int i, u64 all) {
        p.token[row] = i;
        if (p.logprob) p.logprob[row] = (float)((v == w.top ? 0.0 : ((double)v - (double)w.top) / (double)temperature) - log((double)all * exp2(-(double)kSampleBits)));
    };

    if (cut_k) {
        for (int b = tid; b < kSampleBins; b += kSampleThreads) s.hist[b] = 0;
        __syncthreads();
        w.each([&](float v, int) {
            if (v > -INFINITY) atomicAdd(&s.hist[w.bin_of(v)], 1u);
        });
        w.merge_bins(false);
        double before, all;
        w.scan_bins(before, all);
        if (tid == 0) s.found[3] = kSampleBins;
        __syncthreads();
        for (int i = 0; i < 4; i++) {
            const double up = before + s.merged[4 * tid + i];
            if (before < k && up >= k) { s.found[3] = 4 * tid + i; s.part[0][0] = up; }
            before = up;
        }
        __syncthreads();
        const int b = (int)s.found[3];
        const int top_bins = b < kSampleBins ? (int)s.part[0][0] : (int)all;                // elements in bins up to b
        if (top_bins <= kSampleList) {
            // ---- few enough for one CTA to finish
            const int n = (int)w.gather([&](float v, int) { return v > -INFINITY && w.bin_of(v) <= b; });
            cluster_arrive();                                    // rank 0 stays until the others have read the number
            if (w.rank == 0) {
                w.sort_list(n);
                int keep = n < k ? n : k;
                w.scan_weights(keep, [&](int i) { return w.weight(w.list_value(i)); });
                if (cut_p) {
                    const u64 want = (u64)fmax(ceil((double)part * (double)s.weight[keep - 1]), 1.0);
                    const int at = w.first_reaching(keep, want);
                    keep = at < keep ? at + 1 : keep;
                }
                if (cut_m) {
                    if (tid == 0) s.found[0] = 0;
                    __syncthreads();
                    for (int i = tid; i < keep; i += kSampleThreads)
                        if (w.list_value(i) >= floor_m && (i + 1 == keep || w.list_value(i + 1) < floor_m)) s.found[0] = i + 1;
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
                w.sort_list(keep);
                w.scan_weights(keep, [&](int i) { return w.weight(value_of((unsigned)s.list[i])); });
                const u64 sum = s.weight[keep - 1];
                const int at = w.first_reaching(keep, (u64)(u * (double)sum) + 1);
                if (tid == 0) {
                    const u64 e = s.list[at < keep ? at : keep - 1];
                    answer(value_of((unsigned)e), (int)~(unsigned)(e >> 32), sum);
                }
            }
            cluster_wait();
            return;
        }
        if (b < kSampleBins) {
            unsigned lo, hi;
            u64 c, above;
            w.bounds(b, b, lo, hi, c, above, one);
            w.narrow(lo, hi, c, above, (u64)k, one);
        }
    }
    if (cut_p) {
        u64 sum = 0, nothing = 0;
        for (int b = tid; b < kSampleBins; b += kSampleThreads) s.hist[b] = 0;
        __syncthreads();
        // per bin, the weights as multiples of 2^-16 of its octave's, rounded up: within 2^-14 of the bin's sum, errors of fp32 octaves included
        w.each([&](float v, int i) {
            if (!w.kept(v, i)) return;
            sum += w.weight(v);
            const float d = w.octaves(v);
            if (d < (float)(kSampleBins / kSampleOctave)) {
                const int b = w.bin_of(v);
                atomicAdd(&s.hist[b], (unsigned)(ex2((float)(b / kSampleOctave) - d) * 65536.0f) + 1u);
            }
        });
        w.total(sum, nothing);
        w.merge_bins(true);
        const u64 want = (u64)fmax(ceil((double)part * (double)sum), 1.0);
        double before, all;
        w.scan_bins(before, all);
        if (tid == 0) { s.found[0] = kSampleBins; s.found[3] = kSampleBins; }
        __syncthreads();
        const double m = (double)sum, goal = (double)want, slack = (double)p.vocab, err = 1.0 / 16384.0;
        for (int i = 0; i < 4; i++) {
            // the sum up to this bin from either side: whichever is less is known better
            const double up = before + s.merged[4 * tid + i], rest = fmax(all - up, 0.0);
            const double most = fmin(up * (1.0 + err), m - rest * (1.0 - err)) + slack, sure = fmax(up * (1.0 - err), m - rest * (1.0 + err)) - slack;
            if (most >= goal) atomicMin(&s.found[0], (unsigned)(4 * tid + i));
            if (sure >= goal) atomicMin(&s.found[3], (unsigned)(4 * tid + i));
            before = up;
        }
        __syncthreads();
        const int b1 = min((int)s.found[0], kSampleBins - 1), b2 = min((int)s.found[3], kSampleBins - 1);
        unsigned lo, hi;
        u64 c, above;
        w.bounds(b1, b2, lo, hi, c, above, mass);
        w.narrow(lo, hi, c, above, want, mass);
    }
    // ---- the choice
    auto share = [&](float v, int i) -> u64 { return w.kept(v, i) && v >= floor_m ? w.weight(v) : 0; };
    u64 mine = 0, nothing = 0;
    w.each([&](float v, int i) { mine += share(v, i); });
    u64 sum = mine;
    w.total(sum, nothing);
    const u64 e = w.locate(mine, (u64)(u * (double)sum) + 1, share);
    if (lead) answer(value_of((unsigned)(e >> 32)), (int)~(unsigned)e, sum);
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
    int rc = allow_smem<k_sample<T>>(160 * 1024);
    if (rc) return rc;
    return launch_cluster(k_sample<T>, dim3((unsigned)rows, (unsigned)n), dim3(1, (unsigned)n), kSampleThreads, (size_t)p.slice * 4, s, p);
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
