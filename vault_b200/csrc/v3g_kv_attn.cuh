// What the attention kernels over the paged 8-bit cache share: arguments, visibility, operand scaling.
#pragma once
#include <type_traits>

#include "v3g_kv.cuh"

namespace v3g {

struct KvAttnArgs {
    KvView c;
    const void *q;
    int64_t q_tok, q_head;     // strides in elements
    bool q_vec, q_vec8;        // four- and eight-element loads of q are aligned
    int group;                 // query heads per KV head
    float scale_log2;          // scale x log2(e)
    int window, n_sink;        // window 0: every earlier key
    void *out;                 // [tokens][query heads][D]
    float *lse;                // [tokens][query heads], or null
    // sequences of at most max_rows rows (tokens x group) are the few-row kernel's, the others the many-row kernel's
    int max_rows;
    int splits, row_tiles;     // few rows: key shares of a sequence at most, row tiles in the grid
    int units;                 // few rows: shares of the whole batch, given out by the sequences' lengths; 0: `splits` each
    int pf_items, pf_splits;   // many rows: units of 256 rows that a head has room for, key shares
    bool after_few;            // the many-row kernel starts while the few-row kernel runs, and ends after it
    int part_stride;           // shares that a row has room for
    float2 *part_ml;           // [row][share] maximum (log2 units) and sum
    float *part_o;             // [row][share][D]
    int32_t *status;           // V3G_STATUS_TIMEOUT when a bounded wait ran out, or null
};

// a row at position p sees key j; negative positions see nothing
__device__ __forceinline__ bool kv_sees(const KvAttnArgs &a, int p, int j) {
    return j <= p && (a.window == 0 || j > p - a.window || j < a.n_sink);
}

// Key blocks of `unit` keys that rows at positions pmin..pmax can see: [0, sinks) and [first, first + count - sinks);
// returns count.  Keys past the page table's reach do not exist.
__device__ __forceinline__ int kv_visible(const KvAttnArgs &a, int pmin, int pmax, int unit, int &sinks, int &first) {
    const int64_t cap = (int64_t)a.c.max_pages << a.c.page_shift;
    const int end = (int)min((int64_t)pmax + 1, cap);
    sinks = first = 0;
    if (end <= 0) return 0;
    const int last = (end + unit - 1) / unit;
    if (a.window == 0) return last;
    first = min(max(pmin - a.window + 1, 0) / unit, last);
    sinks = (min(a.n_sink, end) + unit - 1) / unit;
    if (first <= sinks) {
        sinks = first = 0;
        return last;
    }
    return sinks + last - first;
}

// power of two that brings a row of largest magnitude top into fp16's range without losing bits (fp16 rows: 1)
template <typename T>
__device__ __forceinline__ int kv_row_exponent(float top) {
    if constexpr (sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value) return 0;
    const int e = (int)((__float_as_uint(top) >> 23) & 255u) - 127;
    return min(13 - e, 100);
}

constexpr int PF_ROWS = 256;   // rows of a many-row CTA

// the many-row kernel over every sequence of at least min_rows rows (v3g_kv_prefill.cu)
cudaError_t launch_kv_prefill(const KvAttnArgs &a, int dtype, int head_dim, int min_rows, cudaStream_t st);

}  // namespace v3g
