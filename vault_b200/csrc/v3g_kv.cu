// Paged 8-bit KV cache: append with the position rotation, read-back, and reordering for beam search.
//
// All three move bytes and are bound by HBM at large sizes and by launch latency at small ones.
#include <cfloat>
#include <type_traits>

#include "v3g_internal.h"
#include "v3g_kv.cuh"

namespace v3g {

// ------------------------------------------------------------------------------------------------------- append
// One CTA takes the new tokens of one 16-token block of one sequence (all heads, or the blockIdx.y-th share of
// them), because a scale belongs to a block: the CTA's warps are its only writers, so there are no atomics and the
// codes are the same every time.  The rotation's cosines and sines of the block's tokens are staged once in shared
// memory and serve every head.  A warp holds the block's rows of one head in registers between the two uses (the
// largest magnitude, then the rounding), so each input is read once.  HBM bounds it at large sizes, the chain of
// look-ups at small ones.
//
// x' = rotation of x (pairs i, i + D/2; fp32, each product and sum rounded by itself), s = max(s_old, max |x'| / 127),
// code = rint(x' * (1 / s)).  A larger s moves the block's earlier codes to rint(code * (s_old / s)).
// 11,247 tokens with 32/8 heads of 128 take 46 us in bf16 (254 MB, 5.5 TB/s; 59 while the rows were held as fp32 and fewer
// CTAs had room) and 122 us in fp32 (483 MB); 16 single fp32 tokens with 12/2 heads 3.6 us.
constexpr int APPEND_WARPS = 4;

struct AppendArgs {
    KvView c;
    const void *k, *v, *q;
    int64_t k_tok, k_head, v_tok, v_head, q_tok, q_head;   // strides in elements
    void *q_out;                                           // [tokens][q_heads][D]
    int q_heads, rope_rows;
    const float *rope;                                     // [rope_rows][D / 2 cos | D / 2 sin], null: no rotation
    int32_t *status;
    bool vec;                                              // every row starts on a multiple of four elements
};

// A lane's elements of a row: H consecutive ones of the first half and their rotation partners, D / 2 further on, so that a
// pair is in one lane
template <int D>
struct Piece {
    static constexpr int H = 4, LR = D / 2 / H;   // elements of each half; lanes of a row
    float x[2][H];
    // x1 c - x2 s; x2 c + x1 s, every product and sum rounded by itself
    __device__ __forceinline__ void rotate(const float *cs, int l) {
        float c[H], s[H];
        *reinterpret_cast<float4 *>(c) = *reinterpret_cast<const float4 *>(cs + H * l);
        *reinterpret_cast<float4 *>(s) = *reinterpret_cast<const float4 *>(cs + D / 2 + H * l);
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const float a = x[0][i], b = x[1][i];
            x[0][i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
            x[1][i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
        }
    }
};

// The same elements as they came: for 16-bit types half the registers, so that more warps have their loads in flight
template <typename T, int D>
struct alignas(16) Raw {
    typedef Piece<D> P;
    T e[2][P::H];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 2 * P::H; ++i) e[i / P::H][i % P::H] = (T)0.f;
    }
    template <bool VEC>
    __device__ __forceinline__ void load(const T *p) {   // p: the lane's first element
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if constexpr (!VEC)
#pragma unroll
                for (int i = 0; i < P::H; ++i) e[k][i] = p[k * (D / 2) + i];
            else if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(e[k]) = ldg_stream16(p + k * (D / 2));
            else *reinterpret_cast<uint2 *>(e[k]) = ldg_stream8(p + k * (D / 2));
        }
    }
    __device__ __forceinline__ P values() const {
        P r;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < P::H; ++i) {
                if constexpr (std::is_same<T, float>::value) r.x[k][i] = e[k][i];
                else if constexpr (std::is_same<T, __half>::value) r.x[k][i] = __half2float(e[k][i]);
                else r.x[k][i] = __bfloat162float(e[k][i]);
            }
        return r;
    }
    // keeps the compiler from carrying what it computed from 16-bit elements past this point
    __device__ __forceinline__ void forget() {
        uint32_t *w = reinterpret_cast<uint32_t *>(e);
        asm volatile("" : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3]));
    }
};

__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN wins
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// rint(x inv) + 128 in the low byte: adding 1.5 x 2^23 rounds to the nearest even integer.  |x inv| is at most 127 and a few
// 2^-24 of it, so no clamp is needed.
__device__ __forceinline__ uint32_t code_bits(float x, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f + 128.f)); }
__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x0040u); }

__device__ __forceinline__ uint32_t moved_code(uint32_t c, float ratio) {
    return (uint32_t)((int)rintf(__fmul_rn((float)((int)c - 128), ratio)) + 128);
}

// one head's rows [s0, s1) of a block: the rounding described above.  cs: the rotation's rows, from row s0's on
template <typename T, int D, bool VEC>
__device__ __forceinline__ void append_rows(const T *src, int64_t tok_ld, const float *cs, bool turn, int s0, int s1,
                                            uint8_t *codes, float *scale, int lane) {
    typedef Piece<D> P;
    constexpr int H = P::H, RP = 32 / P::LR, NP = KV_BLOCK / RP;   // rows of a pass, passes
    const int l = lane % P::LR, sub = lane / P::LR;
    const float s_old = s0 > 0 ? *scale : 0.f;
    constexpr bool AGAIN = sizeof(T) == 2;                         // rotated for the magnitude and again for the codes
    Raw<T, D> x[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int r = s0 + i * RP + sub;
        x[i].zero();
        if (r < s1) x[i].template load<VEC>(src + (int64_t)(r - s0) * tok_ld + H * l);
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int r = s0 + i * RP + sub;
        if (s0 + i * RP >= s1) break;   // uniform over the warp
        P y = x[i].values();
        if (turn && r < s1) y.rotate(cs + (r - s0) * D, l);
#pragma unroll
        for (int k = 0; k < H; ++k) top = max_nan(max_nan(top, fabsf(y.x[0][k])), fabsf(y.x[1][k]));
        if constexpr (AGAIN) x[i].forget();
        else
#pragma unroll
            for (int k = 0; k < 2 * H; ++k) x[i].e[k / H][k % H] = y.x[k / H][k % H];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool bad = !(top <= FLT_MAX) || s_old != s_old;
    float s = fmaxf(s_old, __fmul_rn(top, 1.f / 127.f));
    if (s < KV_SCALE_MIN) s = 0.f;
    if (bad) s = __int_as_float(0x7FC00000);   // the block holds a NaN or an infinity: it reads as NaN
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    if (s0 > 0 && s != s_old) {
        const float ratio = s > 0.f ? __fdiv_rn(s_old, s) : 0.f;
        for (int i = lane; i < s0 * D / 4; i += 32) {
            uint32_t *p = reinterpret_cast<uint32_t *>(codes) + i;
            const uint32_t w = *p;
            *p = moved_code(w & 255u, ratio) | moved_code(w >> 8 & 255u, ratio) << 8 | moved_code(w >> 16 & 255u, ratio) << 16 |
                 moved_code(w >> 24, ratio) << 24;
        }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int r = s0 + i * RP + sub;
        if (r < s1) {
            P all = x[i].values();
            if (AGAIN && turn) all.rotate(cs + (r - s0) * D, l);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float *y = all.x[k];
                uint8_t *p = codes + r * D + k * (D / 2) + H * l;
                const uint32_t lo = pack_bytes(code_bits(y[0], inv), code_bits(y[1], inv));
                const uint32_t hi = pack_bytes(code_bits(y[2], inv), code_bits(y[3], inv));
                *reinterpret_cast<uint32_t *>(p) = bad ? 0x80808080u : __byte_perm(lo, hi, 0x5410u);
            }
        }
    }
    __syncwarp();
    if (lane == 0) *scale = s;
}

// one query head's rows of a block, rotated and not rounded further than their own type; rows past `placed` become zero
template <typename T, int D, bool VEC>
__device__ __forceinline__ void turn_rows(const T *src, int64_t tok_ld, const float *cs, bool turn, int rows, int placed, T *out,
                                          int64_t out_ld, int lane) {
    typedef Piece<D> P;
    constexpr int RP = 32 / P::LR, NP = KV_BLOCK / RP;
    const int l = lane % P::LR, sub = lane / P::LR;
    Raw<T, D> x[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        x[i].zero();
        if (i * RP + sub < placed) x[i].template load<VEC>(src + (int64_t)(i * RP + sub) * tok_ld + P::H * l);
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int r = i * RP + sub;
        P y = x[i].values();
        if (turn && r < placed) y.rotate(cs + r * D, l);
        if (r < rows)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                kv_store4(out + r * out_ld + k * (D / 2) + P::H * l, make_float4(y.x[k][0], y.x[k][1], y.x[k][2], y.x[k][3]));
    }
}

// CTAs of an SM: what the rows in flight leave registers for
template <typename T, int D, bool VEC>
constexpr int append_ctas() { return D * sizeof(T) >= 512 ? (VEC ? 5 : 4) : (VEC ? 7 : 5); }
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(32 * APPEND_WARPS, append_ctas<T, D, VEC>()) k_kv_append(const __grid_constant__ AppendArgs a) {
    __shared__ __align__(16) float cs[KV_BLOCK * D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int64_t base;
    const int b = kv_find(a.c.q_start, a.c.batch, a.c.n_tokens, KV_BLOCK, 1, 2, blockIdx.x, base);
    int first;
    const int n = a.c.tokens(b, first);
    const int p0 = a.c.end(b) - n;                                        // position of the first new token
    const int blk = (p0 >> 4) + (int)(blockIdx.x - base);                 // arithmetic shift: p0 may be negative
    const int lo = max(blk * KV_BLOCK, p0), hi = min(blk * KV_BLOCK + KV_BLOCK, p0 + n);
    if (lo >= hi) {
        // past the last sequence's blocks: the queries of no sequence (the grid has one such CTA at least)
        const int idle = (int)(blockIdx.x - base) - (n > 0 ? ((p0 + n - 1) >> 4) - (p0 >> 4) + 1 : 0);
        if (a.q && b == a.c.batch - 1 && idle >= 0) {
            const int64_t cta = (int64_t)idle * gridDim.y + blockIdx.y, ctas = (int64_t)(gridDim.x - blockIdx.x + idle) * gridDim.y;
            kv_clear_loose<T, D>(a.c, static_cast<T *>(a.q_out), nullptr, a.q_heads, cta * (32 * APPEND_WARPS) + threadIdx.x,
                                 ctas * (32 * APPEND_WARPS));
        }
        return;
    }
    const int t0 = first + (lo - p0), nt = hi - lo;                       // the block's packed tokens
    const int s0 = lo - blk * KV_BLOCK;
    const bool turn = a.rope != nullptr;
    const int page = a.c.page_of(b, lo);
    // tokens that the rotation table reaches; the others have no place, and their queries become zero
    const int placed = lo < 0 ? 0 : (turn ? max(min(a.rope_rows - lo, nt), 0) : nt);
    if (threadIdx.x == 0 && (page < 0 || placed < nt) && a.status) atomicOr(a.status, STATUS_BOUNDS);
    if (turn) {
        const float4 *src = reinterpret_cast<const float4 *>(a.rope + (int64_t)lo * D);
        for (int i = threadIdx.x; i < placed * D / 4; i += 32 * APPEND_WARPS) reinterpret_cast<float4 *>(cs)[i] = __ldg(src + i);
        __syncthreads();
    }
    // a warp takes the block's rows of one head at a time: the query heads, then K, then V
    const int heads = a.c.heads, step = APPEND_WARPS * gridDim.y;
    for (int t = blockIdx.y * APPEND_WARPS + warp; t < a.q_heads + 2 * heads; t += step) {
        if (t < a.q_heads) {
            turn_rows<T, D, VEC>(static_cast<const T *>(a.q) + (int64_t)t0 * a.q_tok + (int64_t)t * a.q_head, a.q_tok, cs, turn, nt, placed,
                            static_cast<T *>(a.q_out) + ((int64_t)t0 * a.q_heads + t) * D, (int64_t)a.q_heads * D, lane);
            continue;
        }
        if (page < 0 || placed == 0) continue;
        const int kind = t - a.q_heads >= heads, h = t - a.q_heads - kind * heads;
        const int64_t at = a.c.block(page, h, lo);
        const T *src = kind ? static_cast<const T *>(a.v) + (int64_t)t0 * a.v_tok + (int64_t)h * a.v_head
                            : static_cast<const T *>(a.k) + (int64_t)t0 * a.k_tok + (int64_t)h * a.k_head;
        append_rows<T, D, VEC>(src, kind ? a.v_tok : a.k_tok, cs, turn && !kind, s0, s0 + placed,
                          (kind ? a.c.v : a.c.k) + at * (KV_BLOCK * D), (kind ? a.c.vs : a.c.ks) + at, lane);
    }
}

// --------------------------------------------------------------------------------------------------------- read
// Values of tokens [first[b], kv_len[b]) of every sequence, of `layers` layers: row row_start[b] + i is token
// first[b] + i.  A thread takes sixteen dims of one row of one head, so that finding the row weighs half as much, U layers in
// flight; rows without a page read as zero.  HBM bounds it, D codes in and D values out per row and head: 192 rows of 63 tokens,
// 28 layers, 2 heads of 128 to bf16 (174 MB in, 347 MB out) take 86 us, 6.1 TB/s; 11,247 tokens, one layer, 8 heads (69 MB)
// 11.4 us (17.2 with eight dims, 64-bit divisions and integer conversions).
struct ReadArgs {
    KvView c;                     // layer 0 of the call; q_start holds row_start, n_tokens the rows
    const int32_t *first;
    int64_t layer_codes, layer_scales;
    int layers;
    void *k, *v;                  // [layers][rows][heads][D]
};

__device__ __forceinline__ void read8(uint2 w, float s, float4 &lo, float4 &hi) {
    // 2^23 + code as a float, less 2^23 + 128: exact
    auto f = [&](uint32_t u, int i) { return __fmul_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + i)) - 8388736.f, s); };
    lo = make_float4(f(w.x, 0), f(w.x, 1), f(w.x, 2), f(w.x, 3));
    hi = make_float4(f(w.y, 0), f(w.y, 1), f(w.y, 2), f(w.y, 3));
}

// A thread takes two pieces of 8 values of a row, D / 2 apart, in U layers at a time
template <typename T, int D, int U>
__global__ void __launch_bounds__(256) k_kv_read(const __grid_constant__ ReadArgs a) {
    constexpr int P = 2, LR = D / 8 / P;   // lanes of a row
    const uint32_t pair = blockIdx.x * (256 / LR) + threadIdx.x / LR, row = pair / a.c.heads;
    if (row >= a.c.n_tokens) return;
    const int h = (int)(pair - row * a.c.heads), d = threadIdx.x % LR * 8;
    int64_t base;
    const int b = kv_find(a.c.q_start, a.c.batch, a.c.n_tokens, 1, 1, 0, row, base);
    const int pos = a.first[b] + (int)((int64_t)row - base);
    const bool in = base <= row && (int64_t)row < a.c.q_start[b + 1] && pos >= 0 && pos < a.c.len(b);
    const int page = in ? a.c.page_of(b, pos) : -1;
    const int64_t at = page >= 0 ? a.c.block(page, h, pos) : 0;
    const int64_t src = (at * KV_BLOCK + (pos & 15)) * D + d, dst = ((int64_t)row * a.c.heads + h) * D + d, layer_out = (int64_t)a.c.n_tokens * a.c.heads * D;
    for (int l0 = blockIdx.y; l0 < a.layers; l0 += U * gridDim.y) {
        uint2 w[U][2][P];
        float s[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int l = l0 + u * gridDim.y;
#pragma unroll
            for (int kind = 0; kind < 2; ++kind) {
#pragma unroll
                for (int k = 0; k < P; ++k) w[u][kind][k] = make_uint2(0x80808080u, 0x80808080u);
                s[u][kind] = 0.f;
                if (page >= 0 && l < a.layers) {
#pragma unroll
                    for (int k = 0; k < P; ++k) w[u][kind][k] = ldg_stream8((kind ? a.c.v : a.c.k) + l * a.layer_codes + src + k * (D / P));
                    s[u][kind] = (kind ? a.c.vs : a.c.ks)[l * a.layer_scales + at];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int l = l0 + u * gridDim.y;
            if (l < a.layers)
#pragma unroll
                for (int kind = 0; kind < 2; ++kind)
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        float4 lo, hi;
                        read8(w[u][kind][k], s[u][kind], lo, hi);
                        T *out = static_cast<T *>(kind ? a.v : a.k) + l * layer_out + dst + k * (D / P);
                        if constexpr (sizeof(T) == 2) {
                            uint4 r;
                            kv_store4(reinterpret_cast<T *>(&r), lo);
                            kv_store4(reinterpret_cast<T *>(&r) + 4, hi);
                            __stcs(reinterpret_cast<uint4 *>(out), r);
                        } else {
                            kv_store4(out, lo);
                            kv_store4(out + 4, hi);
                        }
                    }
        }
    }
}

// ------------------------------------------------------------------------------------------------------ reorder
// Beam j of a group continues beam parents[j]: full pages are shared through the table, the page still being
// filled is copied (codes and scales of its tokens, every layer).  A thread owns one 16-byte unit of the page and
// reads it from all of the group's parents before it writes any of the children, so a child's page may be another
// child's source; groups share no page that is still being filled.  Bytes bound it: 24 groups of 8 beams, 63 tokens of a page of
// 64, 28 layers (348 MB moved) take 54 us, 6.4 TB/s, the copy rate.
struct ReorderArgs {
    KvView c;
    int64_t layer_codes, layer_scales;
    int layers, beams;
    const int32_t *parents, *dst;
    int32_t *out;
    int64_t out_ld;
    int32_t *status;
};

template <int KB, int D>
__global__ void __launch_bounds__(256) k_kv_reorder(const __grid_constant__ ReorderArgs a) {
    __shared__ int src_s[KB], dst_s[KB], par_s[KB];
    const int g = blockIdx.y, r0 = g * a.beams;
    const int len = a.c.len(r0), full = len >> a.c.page_shift, tail = len & (a.c.page - 1);
    if (threadIdx.x < KB) {
        const int j = threadIdx.x;
        int par = -1, src = -1, dst = -1;
        if (j < a.beams) {
            par = a.parents[r0 + j];
            if (par < 0 || par >= a.beams) par = -1;
            if (par >= 0 && tail) {
                src = a.c.page_of(r0 + par, len);
                dst = a.dst ? a.dst[r0 + j] : a.c.page_of(r0 + j, len);
                if (dst >= a.c.n_pages) dst = -1;
            }
            if (tail && (src < 0 || dst < 0)) par = src = -1;   // the row stays as it is
            if (par < 0 && blockIdx.x == 0 && a.status) atomicOr(a.status, STATUS_BOUNDS);
        }
        par_s[j] = par;
        src_s[j] = src == dst || dst < 0 ? -1 : src;
        dst_s[j] = dst;
    }
    __syncthreads();
    // the table: a column at a time, as the beams' rows of it are exchanged
    for (int col = blockIdx.x * 256 + threadIdx.x; col < a.c.max_pages; col += gridDim.x * 256)
#pragma unroll
        for (int j = 0; j < KB; ++j)
            if (j < a.beams) {
                int from = r0 + j;
                if (col < full && par_s[j] >= 0) from = r0 + par_s[j];
                int32_t e = a.c.table[(int64_t)from * a.c.table_ld + col];
                if (col == full && tail && par_s[j] >= 0 && dst_s[j] >= 0) e = dst_s[j];
                a.out[(int64_t)(r0 + j) * a.out_ld + col] = e;
            }
    if (!tail) return;
    const int upr = tail * (D / 16), blocks = (tail + 15) >> 4;   // 16-byte units and scales of one head's part of the page
    const int64_t per_head = 2 * (int64_t)(upr + blocks), total = per_head * a.c.heads * a.layers;
    const int64_t page_codes = (int64_t)a.c.heads * a.c.page * D, page_scales = (int64_t)a.c.heads * a.c.page / 16;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t lh = i / per_head;
        int u = (int)(i - lh * per_head);
        const int layer = (int)(lh / a.c.heads), h = (int)(lh - (int64_t)layer * a.c.heads);
        const bool is_v = u >= upr + blocks;
        if (is_v) u -= upr + blocks;
        if (u < upr) {
            uint8_t *p = (is_v ? a.c.v : a.c.k) + layer * a.layer_codes + (int64_t)h * a.c.page * D + (int64_t)u * 16;
            uint4 x[KB];
#pragma unroll
            for (int j = 0; j < KB; ++j)
                if (src_s[j] >= 0) x[j] = *reinterpret_cast<const uint4 *>(p + src_s[j] * page_codes);
#pragma unroll
            for (int j = 0; j < KB; ++j)
                if (src_s[j] >= 0) *reinterpret_cast<uint4 *>(p + dst_s[j] * page_codes) = x[j];
        } else {
            float *p = (is_v ? a.c.vs : a.c.ks) + layer * a.layer_scales + (int64_t)h * (a.c.page / 16) + (u - upr);
            float x[KB];
#pragma unroll
            for (int j = 0; j < KB; ++j)
                if (src_s[j] >= 0) x[j] = p[src_s[j] * page_scales];
#pragma unroll
            for (int j = 0; j < KB; ++j)
                if (src_s[j] >= 0) p[dst_s[j] * page_scales] = x[j];
        }
    }
}

// --------------------------------------------------------------------------------------------------------- host
static bool aligned_to(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int kv_view(const char *who, const v3g_kv_cache_t *c, uint32_t layer, const v3g_kv_batch_t *b, KvView *out) {
    const std::string w = who;
    if (!c || !b) return v3g_fail(V3G_E_ARG, w + ": null cache or batch");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !b->page_table || !b->kv_len || !b->q_start)
        return v3g_fail(V3G_E_ARG, w + ": null pointer");
    if (c->head_dim != 64 && c->head_dim != 128) return v3g_fail(V3G_E_UNSUPPORTED, w + ": head_dim must be 64 or 128");
    if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)))
        return v3g_fail(V3G_E_UNSUPPORTED, w + ": the page must hold 16, 32, 64, 128 or 256 tokens");
    if (c->n_layers == 0 || c->n_pages == 0 || c->n_kv_heads == 0 || c->n_pages > 0x7FFFFFFFu || c->n_kv_heads > 65535u ||
        c->n_layers > 65535u)
        return v3g_fail(V3G_E_ARG, w + ": layers, pages and heads must be positive");
    if (layer >= c->n_layers) return v3g_fail(V3G_E_ARG, w + ": no such layer");
    if (b->max_pages == 0 || b->table_ld < b->max_pages || b->max_pages > 0x7FFFFFFFu / 256)
        return v3g_fail(V3G_E_ARG, w + ": the page table needs at least one column and table_ld >= max_pages");
    if (b->batch > 65535u || b->n_tokens > 0x7FFFFFFFu / 64) return v3g_fail(V3G_E_LIMIT, w + ": at most 65535 sequences and 2^25 tokens");
    if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16) || !aligned_to(c->k_scale, 4) || !aligned_to(c->v_scale, 4) ||
        !aligned_to(b->page_table, 4) || !aligned_to(b->kv_len, 4) || !aligned_to(b->q_start, 4))
        return v3g_fail(V3G_E_ALIGN, w + ": codes need 16-byte alignment");
    const int64_t scales = (int64_t)c->n_pages * c->n_kv_heads * (c->page / 16), codes = scales * 16 * c->head_dim;
    out->k = c->k + layer * codes;
    out->v = c->v + layer * codes;
    out->ks = c->k_scale + layer * scales;
    out->vs = c->v_scale + layer * scales;
    out->n_pages = (int)c->n_pages;
    out->heads = (int)c->n_kv_heads;
    out->page = (int)c->page;
    out->page_shift = 31 - __builtin_clz(c->page);
    out->table = b->page_table;
    out->table_ld = (int64_t)b->table_ld;
    out->max_pages = (int)b->max_pages;
    out->batch = (int)b->batch;
    out->n_tokens = (int)b->n_tokens;
    out->kv_len = b->kv_len;
    out->q_start = b->q_start;
    return V3G_OK;
}

static int launched(const char *who) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? V3G_OK : v3g_fail(V3G_E_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

static size_t dtype_bytes(int t) { return t == V3G_F32 ? 4 : 2; }

// loads of four elements: the base and both strides keep that alignment
static bool rows_vec(const v3g_rows_t &r, int dtype) {
    return aligned_to(r.data, 4 * dtype_bytes(dtype)) && r.tok_stride % 4 == 0 && r.head_stride % 4 == 0;
}

template <typename T>
static void launch_append(const AppendArgs &a, int D, dim3 grid, cudaStream_t st) {
    if (a.vec) {
        if (D == 64) k_kv_append<T, 64, true><<<grid, 32 * APPEND_WARPS, 0, st>>>(a);
        else k_kv_append<T, 128, true><<<grid, 32 * APPEND_WARPS, 0, st>>>(a);
    } else {
        if (D == 64) k_kv_append<T, 64, false><<<grid, 32 * APPEND_WARPS, 0, st>>>(a);
        else k_kv_append<T, 128, false><<<grid, 32 * APPEND_WARPS, 0, st>>>(a);
    }
}

template <typename T>
static void launch_read(const ReadArgs &a, int D, dim3 grid, cudaStream_t st) {
    if ((int)grid.y >= a.layers) {
        if (D == 64) k_kv_read<T, 64, 1><<<grid, 256, 0, st>>>(a);
        else k_kv_read<T, 128, 1><<<grid, 256, 0, st>>>(a);
    } else {
        if (D == 64) k_kv_read<T, 64, 2><<<grid, 256, 0, st>>>(a);
        else k_kv_read<T, 128, 2><<<grid, 256, 0, st>>>(a);
    }
}

template <int KB>
static void launch_reorder(const ReorderArgs &a, int D, dim3 grid, cudaStream_t st) {
    if (D == 64) k_kv_reorder<KB, 64><<<grid, 256, 0, st>>>(a);
    else k_kv_reorder<KB, 128><<<grid, 256, 0, st>>>(a);
}

}  // namespace v3g

using namespace v3g;

extern "C" int v3g_kv_append(const v3g_kv_cache_t *cache, uint32_t layer, const v3g_kv_batch_t *batch, int dtype, const v3g_rows_t *k,
                             const v3g_rows_t *v, const v3g_rows_t *q, uint32_t n_q_heads, void *q_out, const float *rope,
                             uint32_t rope_rows, int32_t *dev_status, void *stream) {
    AppendArgs a = {};
    const int rc = kv_view("v3g_kv_append", cache, layer, batch, &a.c);
    if (rc != V3G_OK) return rc;
    if (dtype != V3G_F32 && dtype != V3G_F16 && dtype != V3G_BF16) return v3g_fail(V3G_E_DTYPE, "v3g_kv_append: fp32, fp16 or bf16 rows");
    if (!k || !v || !k->data || !v->data) return v3g_fail(V3G_E_ARG, "v3g_kv_append: null rows");
    if (q && (!q->data || !q_out || n_q_heads == 0 || n_q_heads > 65535u)) return v3g_fail(V3G_E_ARG, "v3g_kv_append: q needs heads and q_out");
    if ((rope && rope_rows == 0) || rope_rows > 0x7FFFFFFFu) return v3g_fail(V3G_E_ARG, "v3g_kv_append: an empty rotation table");
    const size_t e = dtype_bytes(dtype);
    if (!aligned_to(k->data, e) || !aligned_to(v->data, e) || (q && (!aligned_to(q->data, e) || !aligned_to(q_out, 16))) ||
        (rope && !aligned_to(rope, 16)) || !aligned_to(dev_status, 4))
        return v3g_fail(V3G_E_ALIGN, "v3g_kv_append: q_out and the rotation table need 16-byte alignment, rows that of their type");
    if (batch->batch == 0 || batch->n_tokens == 0) return V3G_OK;
    a.k = k->data;
    a.v = v->data;
    a.k_tok = k->tok_stride;
    a.k_head = k->head_stride;
    a.v_tok = v->tok_stride;
    a.v_head = v->head_stride;
    a.vec = rows_vec(*k, dtype) && rows_vec(*v, dtype) && (!q || rows_vec(*q, dtype));
    if (q) {
        a.q = q->data;
        a.q_tok = q->tok_stride;
        a.q_head = q->head_stride;
        a.q_heads = (int)n_q_heads;
        a.q_out = q_out;
    }
    a.rope = rope;
    a.rope_rows = (int)rope_rows;
    a.status = dev_status;
    const uint32_t items = batch->n_tokens / KV_BLOCK + 2 * batch->batch + 1;
    // A block's heads are shared out over CTAs while the blocks are few (8 sequences of up to 200 tokens, 32/8 heads: one CTA a
    // block 15.5 us, shared out 10.0 us), and further so that the last round of CTAs is a small part of all (11,247 bf16 tokens: 32
    // CTAs an SM in all 46.5 us, 8 of them 56.4); past one pass of the warps over the heads there is nothing left to share.
    const uint32_t passes = (2 * cache->n_kv_heads + (q ? n_q_heads : 0) + APPEND_WARPS - 1) / APPEND_WARPS;
    uint32_t ny = (148 * 32 + items - 1) / items;
    ny = ny > passes ? passes : ny;
    const dim3 grid(items, ny);
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == V3G_F32) launch_append<float>(a, (int)cache->head_dim, grid, st);
    else if (dtype == V3G_F16) launch_append<__half>(a, (int)cache->head_dim, grid, st);
    else launch_append<__nv_bfloat16>(a, (int)cache->head_dim, grid, st);
    return launched("v3g_kv_append");
}

extern "C" int v3g_kv_read(const v3g_kv_cache_t *cache, uint32_t layer, uint32_t n_layers, const v3g_kv_batch_t *batch,
                           const int32_t *dev_first, int dtype, void *k_out, void *v_out, void *stream) {
    ReadArgs a = {};
    const int rc = kv_view("v3g_kv_read", cache, layer, batch, &a.c);
    if (rc != V3G_OK) return rc;
    if (dtype != V3G_F32 && dtype != V3G_F16 && dtype != V3G_BF16) return v3g_fail(V3G_E_DTYPE, "v3g_kv_read: fp32, fp16 or bf16 values");
    if (!dev_first) return v3g_fail(V3G_E_ARG, "v3g_kv_read: null pointer");
    if (n_layers == 0 || n_layers > cache->n_layers - layer) return v3g_fail(V3G_E_ARG, "v3g_kv_read: no such layers");
    if (batch->batch == 0 || batch->n_tokens == 0) return V3G_OK;
    if (!k_out || !v_out) return v3g_fail(V3G_E_ARG, "v3g_kv_read: null pointer");
    if (!aligned_to(k_out, 16) || !aligned_to(v_out, 16) || !aligned_to(dev_first, 4))
        return v3g_fail(V3G_E_ALIGN, "v3g_kv_read: outputs need 16-byte alignment");
    a.first = dev_first;
    a.layer_scales = (int64_t)cache->n_pages * cache->n_kv_heads * (cache->page / 16);
    a.layer_codes = a.layer_scales * 16 * cache->head_dim;
    a.layers = (int)n_layers;
    a.k = k_out;
    a.v = v_out;
    const int64_t rows = (int64_t)batch->n_tokens * cache->n_kv_heads;
    if (rows > 0x7FFFFFFF) return v3g_fail(V3G_E_LIMIT, "v3g_kv_read: too many values");
    // a thread that takes several layers looks its page up once; few rows spread their layers over the GPU
    const int64_t gx = (rows * (cache->head_dim / 16) + 255) / 256;
    int64_t gy = 4096 / gx;
    gy = gy < 1 ? 1 : (gy > n_layers ? n_layers : gy);
    const dim3 grid((uint32_t)gx, (uint32_t)gy);
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == V3G_F32) launch_read<float>(a, (int)cache->head_dim, grid, st);
    else if (dtype == V3G_F16) launch_read<__half>(a, (int)cache->head_dim, grid, st);
    else launch_read<__nv_bfloat16>(a, (int)cache->head_dim, grid, st);
    return launched("v3g_kv_read");
}

extern "C" int v3g_kv_reorder(const v3g_kv_cache_t *cache, const v3g_kv_batch_t *batch, uint32_t beams, const int32_t *dev_parents,
                              const int32_t *dev_dst_page, int32_t *table_out, uint64_t table_out_ld, int32_t *dev_status, void *stream) {
    ReorderArgs a = {};
    v3g_kv_batch_t rows;
    if (batch) {
        rows = *batch;
        rows.q_start = rows.kv_len;   // a reorder has no new tokens: any readable array stands for q_start
        rows.n_tokens = 0;
    }
    const int rc = kv_view("v3g_kv_reorder", cache, 0, batch ? &rows : nullptr, &a.c);
    if (rc != V3G_OK) return rc;
    if (beams == 0 || beams > V3G_BEAM_MAX) return v3g_fail(V3G_E_LIMIT, "v3g_kv_reorder: 1 to 32 beams");
    if (batch->batch % beams) return v3g_fail(V3G_E_ARG, "v3g_kv_reorder: the rows are not whole groups of beams");
    if (batch->batch == 0) return V3G_OK;
    if (!dev_parents || !table_out) return v3g_fail(V3G_E_ARG, "v3g_kv_reorder: null pointer");
    if (table_out_ld < batch->max_pages) return v3g_fail(V3G_E_ARG, "v3g_kv_reorder: table_out_ld < max_pages");
    if (!aligned_to(dev_parents, 4) || !aligned_to(dev_dst_page, 4) || !aligned_to(table_out, 4) || !aligned_to(dev_status, 4))
        return v3g_fail(V3G_E_ALIGN, "v3g_kv_reorder: misaligned pointer");
    if (table_out == batch->page_table) return v3g_fail(V3G_E_ARG, "v3g_kv_reorder: table_out must be another buffer than the page table");
    a.layer_scales = (int64_t)cache->n_pages * cache->n_kv_heads * (cache->page / 16);
    a.layer_codes = a.layer_scales * 16 * cache->head_dim;
    a.layers = (int)cache->n_layers;
    a.beams = (int)beams;
    a.parents = dev_parents;
    a.dst = dev_dst_page;
    a.out = table_out;
    a.out_ld = (int64_t)table_out_ld;
    a.status = dev_status;
    const uint32_t groups = batch->batch / beams;
    // 16-byte units of a whole page; the part that is filled is known on the device only
    const int64_t units = (int64_t)cache->n_layers * cache->n_kv_heads * 2 * cache->page * (cache->head_dim / 16);
    int64_t gx = (units + 255) / 256;
    const int64_t most = (148 * 8 + groups - 1) / groups;
    gx = gx > most ? most : gx;
    const dim3 grid((uint32_t)gx, groups);
    const cudaStream_t st = (cudaStream_t)stream;
    const int D = (int)cache->head_dim;
    if (beams <= 4) launch_reorder<4>(a, D, grid, st);
    else if (beams <= 8) launch_reorder<8>(a, D, grid, st);
    else if (beams <= 16) launch_reorder<16>(a, D, grid, st);
    else launch_reorder<32>(a, D, grid, st);
    return launched("v3g_kv_reorder");
}
