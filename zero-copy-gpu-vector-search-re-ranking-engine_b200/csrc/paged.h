// Host-side checks and device-side addressing shared by the operators over the paged key/value
// cache (kv_append.cu, paged_attention.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <string>

#include "host_common.h"
#include "zcgvs_sm100.h"

namespace zc {
namespace paged {

constexpr int kMaxHeadDim = 128;

// The parts of the cache and of the step that kernels read, by value in their parameters.
struct View {
    uint8_t* keys;
    uint8_t* values;
    long long page_stride, slot_stride, head_stride;  // elements
    long long pages;
    const int* starts;
    const int* lengths;
    const int* table;
    long long table_stride;
    int table_cols;
    int page_size;
    int page_shift;  // log2 of page_size, or -1 when it is no power of two
    int kv_heads;
    int head_dim;
    int sequences;
    int tokens;
};

inline bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline int invalid(const char* what, const char* why) {
    return fail(ZCGVS_ERR_INVALID_ARG, std::string(what) + ": " + why);
}

// Checks a cache and a step description and fills the kernels' view of them. Nothing on the
// device is read.
inline int make_view(const char* what, const zcgvs_paged_cache* cache, const zcgvs_step_batch* batch, View& v) {
    if (cache->dtype != ZCGVS_DTYPE_F16 && cache->dtype != ZCGVS_DTYPE_BF16) {
        return invalid(what, "the cache's dtype must be F16 or BF16");
    }
    if (cache->page_size <= 0 || cache->kv_heads <= 0) return invalid(what, "page_size and kv_heads must be positive");
    if (cache->head_dim <= 0 || cache->head_dim % 8 != 0) return invalid(what, "head_dim must be a positive multiple of 8");
    if (cache->head_dim > kMaxHeadDim) return fail(ZCGVS_ERR_UNSUPPORTED, std::string(what) + ": head_dim exceeds 128");
    if (cache->pages < 0 || cache->pages > INT_MAX) return invalid(what, "pages out of range");
    if (cache->keys == nullptr || cache->values == nullptr) return invalid(what, "null cache pointer");
    if (!aligned_to(cache->keys, 16) || !aligned_to(cache->values, 16)) {
        return invalid(what, "keys and values must be 16-byte aligned");
    }
    if (cache->page_stride % 8 != 0 || cache->slot_stride % 8 != 0 || cache->head_stride % 8 != 0) {
        return invalid(what, "the cache's strides must be multiples of 8 elements");
    }
    if (cache->page_stride < 0 || cache->slot_stride < 0 || cache->head_stride < 0) {
        return invalid(what, "the cache's strides must not be negative");
    }
    if (batch->query_starts == nullptr || batch->kv_lengths == nullptr || batch->page_table == nullptr) {
        return invalid(what, "null query_starts, kv_lengths or page_table");
    }
    if (batch->pages_per_sequence <= 0 || batch->page_table_stride < batch->pages_per_sequence) {
        return invalid(what, "page_table_stride is smaller than pages_per_sequence, or that is not positive");
    }
    if (static_cast<long long>(batch->pages_per_sequence) * cache->page_size > INT_MAX - 1024) {
        return invalid(what, "pages_per_sequence * page_size exceeds 2^31 - 1025 positions");
    }
    v.keys = static_cast<uint8_t*>(cache->keys);
    v.values = static_cast<uint8_t*>(cache->values);
    v.page_stride = cache->page_stride;
    v.slot_stride = cache->slot_stride;
    v.head_stride = cache->head_stride;
    v.pages = cache->pages;
    v.starts = batch->query_starts;
    v.lengths = batch->kv_lengths;
    v.table = batch->page_table;
    v.table_stride = batch->page_table_stride;
    v.table_cols = batch->pages_per_sequence;
    v.page_size = cache->page_size;
    v.page_shift = -1;
    for (int s = 0; s < 31; ++s) {
        if ((1 << s) == cache->page_size) v.page_shift = s;
    }
    v.kv_heads = cache->kv_heads;
    v.head_dim = cache->head_dim;
    v.sequences = batch->sequences;
    v.tokens = batch->tokens;
    return ZCGVS_OK;
}

// A [tokens, heads, head_dim] operand of the cache's type.
inline int check_rows(const char* what, const char* name, const void* p, int64_t token_stride, int64_t head_stride) {
    if (!aligned_to(p, 16)) return invalid(what, (std::string(name) + " must be 16-byte aligned").c_str());
    if (token_stride < 0 || head_stride < 0 || token_stride % 8 != 0 || head_stride % 8 != 0) {
        return invalid(what, (std::string(name) + "'s strides must be multiples of 8 elements and not negative").c_str());
    }
    return ZCGVS_OK;
}

#ifdef __CUDACC__

__device__ __forceinline__ int page_column(const View& v, int position) {
    return v.page_shift >= 0 ? position >> v.page_shift : position / v.page_size;
}

// Element offset of a position's slot (head 0) in keys or values, or -1 when the position has no
// page of the cache.
__device__ __forceinline__ long long slot_offset(const View& v, int sequence, int position) {
    if (position < 0) return -1;
    const int column = page_column(v, position);
    if (column >= v.table_cols) return -1;
    const int page = __ldg(v.table + sequence * v.table_stride + column);
    if (page < 0 || page >= v.pages) return -1;
    return page * v.page_stride + (position - column * v.page_size) * v.slot_stride;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

#endif  // __CUDACC__

}  // namespace paged
}  // namespace zc
