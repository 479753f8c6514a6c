// A KV cache in pages that many sequences share: what the kernels that fill and read it have in common.
#pragma once
#include "decoder_device.cuh"
#include "launch.cuh"
#include "../../include/bpdq.h"

#include <cuda_fp16.h>

namespace bpdq {

constexpr int kPagedMaxBatch = 2048;        // sequences of a call: bounds the tables that a CTA keeps of them
constexpr int kPagedMaxDim = 128;

// Status of a descriptor, without touching the device.
static inline int paged_check(const bpdq_paged_kv* kv, int n_tokens)
{
    if (!kv || n_tokens < 0 || !kv->k || !kv->v || !kv->page_table || !kv->length) return latch(BPDQ_ERR_ARG);
    if (kv->heads < 1 || kv->kv_heads < 1 || kv->heads % kv->kv_heads || kv->dim < 1 || kv->batch < 0 || kv->max_pages < 1 || kv->n_pages < 1) return latch(BPDQ_ERR_ARG);
    const bool types = (kv->act_type == BPDQ_TYPE_F32 && kv->kv_type == BPDQ_TYPE_F16) ||
                       (kv->act_type == kv->kv_type && (kv->kv_type == BPDQ_TYPE_F16 || kv->kv_type == BPDQ_TYPE_BF16));
    if (!types) return latch(BPDQ_ERR_ARG);
    if (kv->page < 8 || kv->page > 256 || (kv->page & (kv->page - 1)) || kv->dim % 8 || kv->dim > kPagedMaxDim || kv->batch > kPagedMaxBatch || kv->heads > 65535 ||
        (long long)kv->max_pages * kv->page > (1 << 30) || (long long)n_tokens * kv->heads > (1 << 30))
        return latch(BPDQ_ERR_RANGE);
    const size_t dense = (size_t)kv->kv_heads * kv->page * kv->dim;
    if (kv->page_stride && kv->page_stride < dense) return latch(BPDQ_ERR_ARG);
    if (((uintptr_t)kv->k | (uintptr_t)kv->v) & 15 || (kv->page_stride & 7)) return latch(BPDQ_ERR_ALIGN);
    if (!kv->seq_start && n_tokens < kv->batch) return latch(BPDQ_ERR_ARG);
    return 0;
}

static inline size_t paged_stride(const bpdq_paged_kv& kv) { return kv.page_stride ? kv.page_stride : (size_t)kv.kv_heads * kv.page * kv.dim; }

#ifdef __CUDACC__

__device__ __forceinline__ void report(int* err, int code)
{
    if (err) atomicCAS(err, 0, code);
}

// What a sequence brings to a call.  A sequence whose numbers make no sense (a negative length, more tokens than its row of the page table holds,
// bounds that run backwards or beyond the call's tokens) brings nothing, and the error word says so.
struct PagedSpan {
    int first, count, held;         // its tokens among the call's, positions before them
};
__device__ __forceinline__ PagedSpan paged_span(const int* __restrict__ seq_start, const int* __restrict__ length, int b, int n_tokens, int capacity, int* err)
{
    PagedSpan s;
    s.first = seq_start ? seq_start[b] : b;
    s.count = seq_start ? seq_start[b + 1] - s.first : 1;
    s.held = length[b];
    if (s.count == 0) return s;
    if (s.first < 0 || s.count < 0 || s.count > n_tokens || s.first > n_tokens - s.count || s.held < 0 || s.held > capacity - s.count) {
        report(err, 81);
        s.count = 0;
    }
    return s;
}

template <typename A> struct ActOf;
template <> struct ActOf<float> { static __device__ float get(float v) { return v; } static __device__ float put(float v) { return v; } };
template <> struct ActOf<__half> { static __device__ float get(__half v) { return __half2float(v); } static __device__ __half put(float v) { return __float2half_rn(v); } };
template <> struct ActOf<bf16> { static __device__ float get(bf16 v) { return __bfloat162float(v); } static __device__ bf16 put(float v) { return __float2bfloat16_rn(v); } };

#endif
}  // namespace bpdq
