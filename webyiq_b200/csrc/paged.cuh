// The paged KV cache and the step's batch, as the paged operators' kernels see them,
// and the argument checks that their entry points share.
//
// The cache is k, v [pages, KVH, page, D] with strides of its own (unit inner
// stride); sequence b of the batch has the new tokens q_start[b] .. q_start[b + 1]
// and kv_len[b] slots, the new tokens' own among them (the last ones); slot j is row
// j % page of page table[b, j / page].  New token i of n sees slots 0 ..
// kv_len - n + i: nothing where that is negative.
//
// The arrays of the batch are read on the device, so what they hold cannot be
// checked before a launch.  The kernels bound every index they take from them
// instead: a start to the token count, a length to the table's row, a page to the
// cache.  A wrong entry gives wrong values and no access out of range.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace w4a8 {

struct PagedCache {
    void* k;
    void* v;
    int dtype;           // W4A8_F16 or W4A8_BF16
    int pages, page;
    size_t page_stride;  // in elements
    int head_stride, row_stride;
};

struct PagedBatch {
    const uint32_t* q_start;  // [batch + 1]
    const uint32_t* kv_len;   // [batch]
    const uint32_t* table;    // [batch, table_stride]
    int batch, table_stride, tokens;
};

constexpr int kMaxHeadDim = 256;

w4a8_status check_heads(const char* what, int H, int KVH, int D);
w4a8_status check_cache(const char* what, const PagedCache& c, int KVH, int D);
w4a8_status check_batch(const char* what, const PagedBatch& b);

struct SeqSpan {
    int t0, n;  // first new token, new tokens
    int len;    // cached slots
};

__device__ __forceinline__ SeqSpan seq_span(const PagedBatch& b, const PagedCache& c, int seq) {
    const uint32_t tokens = static_cast<uint32_t>(b.tokens);
    const uint32_t s = min(ld_dep(b.q_start + seq), tokens), e = min(ld_dep(b.q_start + seq + 1), tokens);
    // table_stride * page fits 31 bits (checked by the host)
    const uint32_t cap = static_cast<uint32_t>(b.table_stride) * static_cast<uint32_t>(c.page);
    return SeqSpan{static_cast<int>(s), e > s ? static_cast<int>(e - s) : 0,
                   static_cast<int>(min(ld_dep(b.kv_len + seq), cap))};
}

__device__ __forceinline__ uint32_t page_of(const PagedBatch& b, const PagedCache& c, int seq, int index) {
    return min(ld_dep(b.table + static_cast<size_t>(seq) * b.table_stride + index), static_cast<uint32_t>(c.pages - 1));
}

// Element offset of slot j of a sequence (0 <= j < len) for one kv head.
__device__ __forceinline__ size_t slot_offset(const PagedBatch& b, const PagedCache& c, int seq, int kh, int j) {
    const int pi = j / c.page;
    return page_of(b, c, seq, pi) * c.page_stride + static_cast<size_t>(kh) * c.head_stride +
           static_cast<size_t>(j - pi * c.page) * c.row_stride;
}

// The 16-bit element types: conversion of pairs, rounding to nearest even.  f16
// results saturate at its largest finite value: an infinity in the cache would turn
// every later token's output into NaN, and a value past 65504 is still the largest
// one of its row.  NaN stays NaN.
template <typename T>
struct Elem;
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float sat(float x) { return x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x; }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float sat(float x) { return x; }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) {
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
};

}  // namespace w4a8
