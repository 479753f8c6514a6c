// New tokens' queries, keys and values on their way to attention over a paged cache (paged.cuh): queries and keys turned by their positions, keys and
// values rounded to the cache's type and stored in their sequences' pages.
//
// Pair (x, y) with frequency f at position p becomes (x cos a - y sin a, x sin a + y cos a), a = p f.  The angle is formed and reduced to half
// turns in 64 bits: fp32 would lose 2^-24 p f of it.
// Bound by the launch where there are few tokens: 16 of fp32 2.6 us.  Many: 7683 of 32 heads on 8 of 128 in bf16 (189 MB) 42 us, 4.5 TB/s, 70 % of the measured copy rate: a
// CTA's loads wait for its token's sequence, the page's number and the angles, three steps that follow one another.  (Four tokens per CTA, the next loads ahead of the stores: 43; two: 46; 16-byte units: 41 to 54.)
#include "paged.cuh"

namespace bpdq {

constexpr int kAppendThreads = 256;

struct AppendArgs {
    const void *q, *k, *v;
    void *q_out, *k_pool, *v_pool;
    int ld_q, ld_q_out, ld_k, ld_v;
    int n_tokens, batch, heads, kv_heads, dim, page, max_pages, n_pages, rot;
    size_t page_stride;
    const int *seq_start, *length, *table;
    const float* freq;
};

// V neighbouring elements of type T as fp32 numbers, in units of up to 16 bytes.
template <typename T, int V> __device__ __forceinline__ void load_unit(const T* p, float (&x)[V])
{
    if constexpr (V == 1) {
        x[0] = ActOf<T>::get(*p);
    } else {
        alignas(16) T raw[V];
        constexpr int words = (int)(V * sizeof(T) / 8);
        if constexpr (words >= 2) {
#pragma unroll
            for (int i = 0; i < words / 2; i++) reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
            *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
        }
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = ActOf<T>::get(raw[i]);
    }
}
template <typename T, int V> __device__ __forceinline__ void store_unit(T* p, const float (&x)[V])
{
    if constexpr (V == 1) {
        *p = ActOf<T>::put(x[0]);
    } else {
        alignas(16) T raw[V];
#pragma unroll
        for (int i = 0; i < V; i++) raw[i] = ActOf<T>::put(x[i]);
        constexpr int words = (int)(V * sizeof(T) / 8);
        if constexpr (words >= 2) {
#pragma unroll
            for (int i = 0; i < words / 2; i++) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(raw)[i];
        } else {
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(raw);
        }
    }
}

// A CTA takes a token (blockIdx.x) or, of few tokens, a part of its heads (blockIdx.y).  A unit is V pairs, or 2 V dimensions that do not turn.
template <typename A, typename K, int V, bool kNeighbours>
__global__ void __launch_bounds__(kAppendThreads) k_paged_append(const AppendArgs p, int* err)
{
    __shared__ float s_cos[kPagedMaxDim / 2], s_sin[kPagedMaxDim / 2];
    __shared__ int s_seq, s_held, s_page;
    const int tid = threadIdx.x, t = blockIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0) s_seq = -1;
    __syncthreads();
    if (p.seq_start) {
        for (int b = tid; b < p.batch; b += kAppendThreads) {
            const int from = p.seq_start[b], to = p.seq_start[b + 1];
            if (from <= t && t < to) {
                const PagedSpan s = paged_span(p.seq_start, p.length, b, p.n_tokens, p.max_pages * p.page, err);
                if (s.count > 0) { s_seq = b; s_held = s.held + t - s.first; }
            }
        }
    } else if (tid == 0 && t < p.batch) {
        const PagedSpan s = paged_span(nullptr, p.length, t, p.n_tokens, p.max_pages * p.page, err);
        if (s.count > 0) { s_seq = t; s_held = s.held; }
    }
    __syncthreads();
    if (s_seq < 0) return;
    const int pos = s_held, half = p.rot / 2;
    if (tid == 0) {
        const int page = p.table[(size_t)s_seq * p.max_pages + pos / p.page];
        s_page = page >= 0 && page < p.n_pages ? page : -1;
        if (s_page < 0) report(err, 82);
    }
    if (tid < half) {
        // in half turns: a / pi, less the nearest even number
        const double turns = (double)pos * (double)p.freq[tid] * 0.31830988618379067154;
        sincospif((float)(turns - 2.0 * rint(0.5 * turns)), &s_sin[tid], &s_cos[tid]);
    }
    __syncthreads();

    const int turning = half / V, units = turning + (p.dim - p.rot) / (2 * V), kv_units = p.kv_heads * units;
    const int q_units = p.q ? p.heads * units : 0;
    const size_t row = (size_t)(s_page < 0 ? 0 : s_page) * p.page_stride + (size_t)(pos % p.page) * p.dim;
    const A* q = static_cast<const A*>(p.q) + (size_t)t * p.ld_q;
    A* q_out = static_cast<A*>(p.q_out) + (size_t)t * p.ld_q_out;
    const A *k = static_cast<const A*>(p.k) + (size_t)t * p.ld_k, *v = static_cast<const A*>(p.v) + (size_t)t * p.ld_v;
    for (int u = blockIdx.y * kAppendThreads + tid; u < q_units + 2 * kv_units; u += gridDim.y * kAppendThreads) {
        const int kind = u < q_units ? 0 : (u < q_units + kv_units ? 1 : 2);         // query, key, value
        const int w = u - (kind == 0 ? 0 : (kind == 1 ? q_units : q_units + kv_units)), head = w / units, i = w % units;
        const A* src = (kind == 0 ? q : (kind == 1 ? k : v)) + head * p.dim;
        const bool turns = i < turning;
        // elements a[] and b[]: the two sides of V pairs in halves, or 2 V neighbours
        const int at = !turns ? p.rot + 2 * V * (i - turning) : (kNeighbours ? 2 * V * i : V * i), step = turns && !kNeighbours ? half : V;
        float a[V], b[V];
        load_unit<A, V>(src + at, a);
        load_unit<A, V>(src + at + step, b);
        if (turns && kind < 2) {
            if (kNeighbours) {
                if constexpr (V == 1) {
                    const float c = s_cos[i], s = s_sin[i], x = a[0], y = b[0];
                    a[0] = x * c - y * s;
                    b[0] = x * s + y * c;
                } else {
#pragma unroll
                    for (int j = 0; j < V / 2; j++) {
                        const float c0 = s_cos[V * i + j], s0 = s_sin[V * i + j], c1 = s_cos[V * i + V / 2 + j], s1 = s_sin[V * i + V / 2 + j];
                        const float x0 = a[2 * j], y0 = a[2 * j + 1], x1 = b[2 * j], y1 = b[2 * j + 1];
                        a[2 * j] = x0 * c0 - y0 * s0;
                        a[2 * j + 1] = x0 * s0 + y0 * c0;
                        b[2 * j] = x1 * c1 - y1 * s1;
                        b[2 * j + 1] = x1 * s1 + y1 * c1;
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float c = s_cos[V * i + j], s = s_sin[V * i + j], x = a[j], y = b[j];
                    a[j] = x * c - y * s;
                    b[j] = x * s + y * c;
                }
            }
        }
        if (kind == 0) {
            store_unit<A, V>(q_out + head * p.dim + at, a);
            store_unit<A, V>(q_out + head * p.dim + at + step, b);
        } else if (s_page >= 0) {
            K* dst = static_cast<K*>(kind == 1 ? p.k_pool : p.v_pool) + row + (size_t)head * p.page * p.dim;
            store_unit<K, V>(dst + at, a);
            store_unit<K, V>(dst + at + step, b);
        }
    }
}

template <typename A, typename K>
static int launch_append(const AppendArgs& p, bool neighbours, bool wide, cudaStream_t s)
{
    const int units = (p.heads * (p.q ? 1 : 0) + 2 * p.kv_heads) * (p.dim / (wide ? 8 : 2)), parts = (units + kAppendThreads - 1) / kAppendThreads;
    const int room = 2 * sm_count() / p.n_tokens, y = room < 1 ? 1 : (room < parts ? room : parts);
    const dim3 grid((unsigned)p.n_tokens, (unsigned)y);
    if (wide) return neighbours ? launch_ordered(k_paged_append<A, K, 4, true>, grid, kAppendThreads, 0, s, p, device_error_flag())
                                : launch_ordered(k_paged_append<A, K, 4, false>, grid, kAppendThreads, 0, s, p, device_error_flag());
    return neighbours ? launch_ordered(k_paged_append<A, K, 1, true>, grid, kAppendThreads, 0, s, p, device_error_flag())
                      : launch_ordered(k_paged_append<A, K, 1, false>, grid, kAppendThreads, 0, s, p, device_error_flag());
}

}  // namespace bpdq

using namespace bpdq;

extern "C" int bpd_paged_append_cuda(const bpdq_paged_kv* kv, const void* q, int ld_q, void* q_out, int ld_q_out, const void* k, int ld_k, const void* v, int ld_v,
                                     int n_tokens, int rot_dims, int neighbours, const float* rot_freq, void* stream)
{
    int rc = paged_check(kv, n_tokens);
    if (rc) return rc;
    const int width = kv->heads * kv->dim, kv_width = kv->kv_heads * kv->dim;
    if (!k || !v || !q != !q_out || rot_dims < 0 || rot_dims > kv->dim || rot_dims % 2 || (rot_dims && !rot_freq)) return latch(BPDQ_ERR_ARG);
    if (ld_k < kv_width || ld_v < kv_width || (q && (ld_q < width || ld_q_out < width))) return latch(BPDQ_ERR_ARG);
    if (n_tokens == 0 || kv->batch == 0) return 0;
    const bool f32 = kv->act_type == BPDQ_TYPE_F32;
    const uintptr_t places = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v;
    if (places & (f32 ? 3 : 1)) return latch(BPDQ_ERR_ALIGN);
    if (q && q == q_out && ld_q != ld_q_out && n_tokens > 1) return latch(BPDQ_ERR_ARG);       // (rows would lie over others that are yet to be read)
    // Four pairs per thread where rows and halves allow loads of four elements (8 bytes, or 16 of fp32).
    const int unit = f32 ? 15 : 7;
    const bool wide = !(places & unit) && !((ld_k | ld_v | (q ? ld_q | ld_q_out : 0)) & 3) && rot_dims % 8 == 0;
    AppendArgs p = {};
    p.q = q; p.k = k; p.v = v; p.q_out = q_out; p.k_pool = kv->k; p.v_pool = kv->v;
    p.ld_q = ld_q; p.ld_q_out = ld_q_out; p.ld_k = ld_k; p.ld_v = ld_v;
    p.n_tokens = n_tokens; p.batch = kv->batch; p.heads = kv->heads; p.kv_heads = kv->kv_heads; p.dim = kv->dim; p.page = kv->page;
    p.max_pages = kv->max_pages; p.n_pages = kv->n_pages; p.rot = rot_dims;
    p.page_stride = paged_stride(*kv);
    p.seq_start = kv->seq_start; p.length = kv->length; p.table = kv->page_table; p.freq = rot_freq;
    cudaStream_t s = (cudaStream_t)stream;
    if (f32) return launch_append<float, __half>(p, neighbours, wide, s);
    return kv->kv_type == BPDQ_TYPE_F16 ? launch_append<__half, __half>(p, neighbours, wide, s) : launch_append<bf16, bf16>(p, neighbours, wide, s);
}
