// Paged 8-bit KV cache: what its kernels share.
//
// Layout (include/vault_b200.h, v3g_kv_cache_t): codes [layer][page][kv head][page token][head_dim], one byte each,
// biased by 128; scales [layer][page][kv head][page / 16], fp32.  The 16 consecutive tokens of a block share a
// scale, so a block of one head is 16 head_dim consecutive bytes, 16-byte aligned.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/vault_b200.h"
#include "v3g.cuh"

namespace v3g {

constexpr int KV_BLOCK = 16;
constexpr float KV_SCALE_MIN = 7.52316385e-37f;   // 2^-120: smaller scales are stored as zero (1 / scale stays finite)

// one layer of a cache and the batch that uses it, as the kernels see them
struct KvView {
    uint8_t *k, *v;              // the layer's first page
    float *ks, *vs;
    int n_pages, heads, page, page_shift;
    const int32_t *table;        // [batch][table_ld]
    int64_t table_ld;
    int max_pages, batch, n_tokens;
    const int32_t *kv_len, *q_start;

    // the stored length, never past what the table can name
    __device__ __forceinline__ int len(int b) const {
        const int cap = (int)min((int64_t)max_pages << page_shift, (int64_t)0x7FFFFF00);
        return min(max(kv_len[b], 0), cap);
    }
    // the length as the positions count it (a length past the table's capacity keeps its positions)
    __device__ __forceinline__ int end(int b) const { return min(max(kv_len[b], -(1 << 29)), 0x7FFFFF00); }
    // packed tokens [first, first + n) of sequence b, inside [0, n_tokens) whatever q_start holds
    __device__ __forceinline__ int tokens(int b, int &first) const {
        first = min(max(q_start[b], 0), n_tokens);
        return max(min(q_start[b + 1], n_tokens) - first, 0);
    }
    // packed rows that belong to no sequence, before the first and after the last: how many; row(i): the i-th of them
    __device__ __forceinline__ int loose(int &before, int &after) const {
        before = min(max(q_start[0], 0), n_tokens);
        after = min(max(q_start[batch], 0), n_tokens);
        return before + n_tokens - after;
    }
    // page that holds position pos of sequence b, -1 where there is none
    __device__ __forceinline__ int page_of(int b, int pos) const {
        const int i = pos >> page_shift;
        if (pos < 0 || i >= max_pages) return -1;
        const int p = table[(int64_t)b * table_ld + i];
        return p < n_pages ? p : -1;
    }
    // index of the 16-token block at position pos of (page, head): codes at 16 D times it, scales at it
    __device__ __forceinline__ int64_t block(int pg, int head, int pos) const {
        return (((int64_t)pg * heads + head) << (page_shift - 4)) + ((pos & (page - 1)) >> 4);
    }
};

// Sequence whose items hold index i, where sequence b owns the items [f(b), f(b + 1)), f(b) = q_start[b] / unit + extra b:
// an upper bound on the units that its tokens touch, known without a pass over the lengths.
__device__ __forceinline__ int kv_find(const int32_t *q_start, int batch, int n_tokens, int unit, int mul, int extra, int64_t i,
                                       int64_t &base) {
    int lo = 0, hi = batch;   // f(lo) <= i < f(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const int64_t f = (int64_t)min(max(q_start[mid], 0), n_tokens) * mul / unit + (int64_t)extra * mid;
        if (f <= i) lo = mid;
        else hi = mid;
    }
    base = (int64_t)min(max(q_start[lo], 0), n_tokens) * mul / unit + (int64_t)extra * lo;
    return lo;
}

// four values from memory, 4 elements wide where `vec`
template <typename T>
__device__ __forceinline__ float4 kv_load4(const T *p, bool vec);
template <>
__device__ __forceinline__ float4 kv_load4<float>(const float *p, bool vec) {
    if (vec) return *reinterpret_cast<const float4 *>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
template <>
__device__ __forceinline__ float4 kv_load4<__half>(const __half *p, bool vec) {
    if (!vec) return make_float4(__half2float(p[0]), __half2float(p[1]), __half2float(p[2]), __half2float(p[3]));
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 kv_load4<__nv_bfloat16>(const __nv_bfloat16 *p, bool vec) {
    if (!vec)
        return make_float4(__bfloat162float(p[0]), __bfloat162float(p[1]), __bfloat162float(p[2]), __bfloat162float(p[3]));
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xFFFF0000u));
}
// the same to memory (contiguous rows of this library's own layout: always aligned)
__device__ __forceinline__ void kv_store4(float *p, float4 x) { *reinterpret_cast<float4 *>(p) = x; }
__device__ __forceinline__ void kv_store4(__half *p, float4 x) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void kv_store4(__nv_bfloat16 *p, float4 x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// Zeros to the rows of out [n_tokens][heads][D] that belong to no sequence, and -inf to their lse (may be null): the share of
// worker `w` of `workers`.
template <typename T, int D>
__device__ __forceinline__ void kv_clear_loose(const KvView &c, T *out, float *lse, int heads, int64_t w, int64_t workers) {
    constexpr int PIECES = D * sizeof(T) / 16;
    int before, after;
    const int rows = c.loose(before, after);
    for (int64_t i = w; i < (int64_t)rows * heads * PIECES; i += workers) {
        const int64_t head = i / PIECES, at = head + (head < (int64_t)before * heads ? 0 : (int64_t)(after - before) * heads);
        reinterpret_cast<uint4 *>(out + at * D)[i % PIECES] = make_uint4(0u, 0u, 0u, 0u);
        if (lse && i % PIECES == 0) lse[at] = -INFINITY;
    }
}

// host: argument checks shared by the entry points; fills the kernels' view of `layer`
int kv_view(const char *who, const v3g_kv_cache_t *c, uint32_t layer, const v3g_kv_batch_t *b, KvView *out);

}  // namespace v3g
