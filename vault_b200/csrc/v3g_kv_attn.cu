// Attention over the paged 8-bit cache: few query rows per KV head (decode steps, short chunks).
//
// o_r = sum_j softmax_j(scale q_r . k_j) v_j over the visible keys of row r.  A decode step reads every visible key and
// value once, 2 D bytes per key and KV head against 4 D G flops (G query heads share them), so HBM bounds it; the
// kernel's work is to keep loads in flight and to spread one sequence over many SMs.
//
// * A CTA (4 warps) takes up to 8 NT rows (token, query head of one KV head) and a contiguous share of the visible
//   16-key blocks; each warp takes every fourth of them with its own running maximum and sum, so the loop has no
//   barrier.  A block of one head is 16 D consecutive bytes of codes; a warp loads K and V straight to registers, the
//   next block's while it computes.
// * S^T[key, row] = K Q^T on mma.sync m16n8k16 with the 16 keys as M: a lane's bytes of a key row are its fragment when
//   the head dims are taken in that order (the contraction does not care), so no shared memory is used.  Codes become
//   fp16 integers exactly (byte permute to 1024 + c, minus 1152).  fp16 queries enter as they are, bf16 queries as fp16
//   after an exact power of two per row that puts the largest magnitude in [2^13, 2^14).
// * The K scale of the block multiplies the scores, the V scale enters the exponent of the operand: P' = 2^(s + log2 vs - M)
//   with an offset M of the row's own, which follows the largest of its terms p vs as m follows its largest score.  So P'
//   keeps fp16's 11 bits whatever the scales are, and no block that the row does not see, or gives no weight, costs it any.
//   For fp16 outputs P' enters as two fp16 parts, since the rounding of one would be as large as that of the output itself.
//   Sums, maxima and the accumulators are fp32.  m and M are raised only when a score or a term exceeds them by 8 (P' then
//   stays below 2^8).
// * O^T[d, row] = V^T P'^T: V's bytes of four keys are interleaved into fragments, P' is transposed with movmatrix.
//   Splits of one row are joined by a second kernel in split order, so results do not depend on timing.
//
// 4 sequences of 100,000 keys, 32/8 heads (819 MB): 136 us, 6.0 TB/s; 64 of 1,411-4,608 keys, 12/2 heads (93 MB): 26 us, of
// which about 8 are the launch, the chain length -> page -> codes and the join; one of 1,545 keys: 8 us, all latency.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "v3g_internal.h"
#include "v3g_kv.cuh"
#include "v3g_kv_attn.cuh"

namespace v3g {

constexpr int DEC_WARPS = 4;
constexpr int DEC_MIN_BLOCKS = 2 * DEC_WARPS;   // blocks of a split at least: fewer leave warps idle

__device__ __forceinline__ uint32_t magic_half2(uint32_t w, uint32_t sel) {   // two code bytes -> fp16 integers
    const uint32_t v = __byte_perm(w, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&v), __float2half2_rn(1152.f));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float ex2(float x) {   // 2^x, 0 for -inf
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

template <int BYTES>
struct Bytes;
template <>
struct Bytes<16> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const uint8_t *p) {
        const uint4 u = ldg_stream16(p);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    }
};
template <>
struct Bytes<8> {
    uint32_t w[2];
    __device__ __forceinline__ void load(const uint8_t *p) {
        const uint2 u = ldg_stream8(p);
        w[0] = u.x, w[1] = u.y;
    }
};

// Unit u of the a.units in which the key blocks of the whole batch are shared out: its sequence (-1: none), which of the
// sequence's `shares` it is.  One warp works it out from the lengths (nb: place for them, a lane touches its own entries): the
// smallest share size, to a sixteenth, whose shares fit the units.
constexpr int BALANCE_MAX = 256;   // sequences
__device__ __forceinline__ int kv_share(const KvAttnArgs &a, int u, int *nb, int &split, int &shares) {
    const int lane = threadIdx.x & 31, to = (a.c.batch + 31) / 32 * 32 + lane;
    int total = 0, top = 0;
#pragma unroll 2
    for (int b = lane; b < to; b += 32) {
        const int at = min(b, a.c.batch - 1);   // the loads wait for one another nowhere
        int first, x, y, n = a.c.tokens(at, first);
        const int p0 = a.c.end(at) - n, seen = min(max(kv_visible(a, p0, p0 + n - 1, KV_BLOCK, x, y), 1), 1 << 22);
        n = b < a.c.batch && n > 0 && n * a.group <= a.max_rows ? seen : 0;
        nb[b] = n;
        total += n;
        top = max(top, n);
    }
    total = __reduce_add_sync(0xffffffffu, total);
    top = __reduce_max_sync(0xffffffffu, top);
    auto parts = [](int n, float inv) { return __float2int_ru(n * inv); };   // one at least; a whole multiple is not rounded up
    int lo = max((total + a.units - 1) / a.units, DEC_MIN_BLOCKS), per = max(lo, top);   // per: one share each, which fits
    while (per - lo > lo / 16) {
        const int mid = (lo + per) / 2;
        const float inv = 0.999999f / mid;
        int need = 0;
#pragma unroll 2
        for (int b = lane; b < to; b += 32) need += parts(nb[b], inv);
        if ((int)__reduce_add_sync(0xffffffffu, need) <= a.units) per = mid;
        else lo = mid + 1;
    }
    const float inv = 0.999999f / per;
    int before = 0;
#pragma unroll 1
    for (int b = lane; b < to; b += 32) {
        const int mine = min(parts(nb[b], inv), a.splits);
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, u < before + upto);
        if (past) {
            const int l = __ffs(past) - 1;
            shares = __shfl_sync(0xffffffffu, mine, l);
            split = u - before - __shfl_sync(0xffffffffu, upto - mine, l);
            return b - lane + l;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return -1;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * DEC_WARPS, NT == 1 ? 4 : 2) k_kv_decode(const __grid_constant__ KvAttnArgs a) {
    constexpr int ROWS = 8 * NT, NCH = D / 64, VB = D / 8, MT = D / 16, OS = D + 4;
    constexpr bool TWO = std::is_same<T, __half>::value;
    __shared__ int sm_share[3];
    __shared__ float sm_m[DEC_WARPS][ROWS], sm_l[DEC_WARPS][ROWS];
    __shared__ __align__(16) float sm_o[DEC_WARPS][ROWS][OS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    int idx = blockIdx.x;
    const int rt0 = idx % a.row_tiles;
    idx /= a.row_tiles;
    int h, b, split, shares = a.splits;
    auto clear = [&]() {
        kv_clear_loose<T, D>(a.c, static_cast<T *>(a.out), a.lse, a.c.heads * a.group, (int64_t)blockIdx.x * (32 * DEC_WARPS) + threadIdx.x,
                             (int64_t)gridDim.x * (32 * DEC_WARPS));
    };
    griddep_launch();
    if (a.units) {
        h = idx % a.c.heads;
        if (warp == 0) {
            b = kv_share(a, idx / a.c.heads, reinterpret_cast<int *>(sm_o), split, shares);
            if (lane == 0) sm_share[0] = b, sm_share[1] = split, sm_share[2] = shares;
        }
        __syncthreads();
        b = sm_share[0], split = sm_share[1], shares = sm_share[2];
        if (b < 0) {
            clear();
            return;
        }
    } else {
        split = idx % a.splits;
        idx /= a.splits;
        h = idx % a.c.heads;
        b = idx / a.c.heads;
    }
    int first;
    const int n = a.c.tokens(b, first);
    const int rows = n * a.group > a.max_rows ? 0 : n * a.group;             // else they are the many-row kernel's
    const int p0 = a.c.end(b) - n;
    for (int rt = rt0; rt * ROWS < rows; rt += a.row_tiles) {
        const int r0 = rt * ROWS, rn = min(rows - r0, ROWS);
        const int pmin = p0 + r0 / a.group, pmax = p0 + (r0 + rn - 1) / a.group;
        int sb, ws;                                                          // blocks [0, sb) and [ws, ws + nb - sb)
        const int nb = kv_visible(a, pmin, pmax, KV_BLOCK, sb, ws);
        const int per = max((nb + shares - 1) / shares, DEC_MIN_BLOCKS);
        const int lo = split * per, hi = min(nb, lo + per);

        auto row_of = [&](int r) {
            const int rr = r0 + r, tok = rr / a.group;
            return (int64_t)(first + tok) * a.c.heads * a.group + h * a.group + rr - tok * a.group;
        };
        if (split == shares - 1)                                             // shares that the sequence does not have
            for (int i = threadIdx.x; i < rn * (a.splits - shares); i += 32 * DEC_WARPS)
                a.part_ml[row_of(i % rn) * a.part_stride + shares + i / rn] = make_float2(-INFINITY, 0.f);
        if (lo >= hi && a.splits > 1) {                                      // no share for this CTA
            if (threadIdx.x < rn) a.part_ml[row_of(threadIdx.x) * a.part_stride + split] = make_float2(-INFINITY, 0.f);
            continue;
        }
        // lane i looks up the i-th of the warp's next 32 blocks: its page, then its place and scales
        int64_t my_at, at;
        float my_ks, my_lv;                                                  // K scale, log2 of the V scale
        auto position = [&](int base) {
            const int vi = base + DEC_WARPS * lane;
            return vi < hi ? (vi < sb ? vi : vi - sb + ws) * KV_BLOCK : -1;
        };
        auto place = [&](int pos, int pg) {
            my_at = -1;
            my_ks = my_lv = 0.f;
            if (pg >= 0) {
                my_at = a.c.block(pg, h, pos);
                my_ks = a.c.ks[my_at];
                my_lv = log2f(a.c.vs[my_at]);
            }
        };
        Bytes<16> kr[NCH][2];
        Bytes<VB> vr[4];
        auto load_k = [&](int64_t at) {
            if (at < 0) return;
            const uint8_t *p = a.c.k + at * (KV_BLOCK * D) + g * D + 16 * t;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                kr[c][0].load(p + 64 * c);
                kr[c][1].load(p + 8 * D + 64 * c);
            }
        };
        auto load_v = [&](int64_t at) {
            if (at < 0) return;
            const uint8_t *p = a.c.v + at * (KV_BLOCK * D) + 2 * t * D + g * VB;
            vr[0].load(p);
            vr[1].load(p + D);
            vr[2].load(p + 8 * D);
            vr[3].load(p + 9 * D);
        };
        const int pos0 = position(lo + warp), pg0 = a.c.page_of(b, pos0);   // on its way while the queries are laid out
        // queries: row g of each n tile, dims 64 c + 16 t .. + 15
        uint32_t qf[NT][NCH][8];
        float qs[NT][2], m[NT][2], M[NT][2], l[NT][2];
        int rpos[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = r0 + 8 * nt + g, tok = r / a.group, qh = h * a.group + r - tok * a.group;
            float x[NCH][16], top = 0.f;
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (8 * nt + g < rn)
                        v = kv_load4<T>(static_cast<const T *>(a.q) + (int64_t)(first + tok) * a.q_tok + (int64_t)qh * a.q_head + 64 * c +
                                            16 * t + 4 * i, a.q_vec);
                    x[c][4 * i] = v.x, x[c][4 * i + 1] = v.y, x[c][4 * i + 2] = v.z, x[c][4 * i + 3] = v.w;
                    top = fmaxf(fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int up = kv_row_exponent<T>(top);
            const float f = __int_as_float((up + 127) << 23), fi = __int_as_float((127 - up) << 23) * a.scale_log2;
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) qf[nt][c][i] = pack_half2(x[c][2 * i] * f, x[c][2 * i + 1] * f);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                qs[nt][i] = __shfl_sync(0xffffffffu, fi, (2 * t + i) * 4);
                const int rr = 8 * nt + 2 * t + i;
                rpos[nt][i] = rr < rn ? p0 + (r0 + rr) / a.group : -1;
                m[nt][i] = M[nt][i] = -INFINITY;
                l[nt][i] = 0.f;
            }
        }
        place(pos0, pg0);
        at = __shfl_sync(0xffffffffu, my_at, 0);
        load_k(at);
        load_v(at);
        float acc[MT][NT][4];
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j][nt][i] = 0.f;

        for (int base = lo + warp; base < hi; base += 32 * DEC_WARPS) {
            const int cnt = min(32, (hi - base + DEC_WARPS - 1) / DEC_WARPS);
            if (base != lo + warp) {
                const int pos = position(base);
                place(pos, a.c.page_of(b, pos));
                at = __shfl_sync(0xffffffffu, my_at, 0);
                load_k(at);
                load_v(at);
            }
            for (int it = 0; it < cnt; ++it) {
                const int64_t next = it + 1 < cnt ? __shfl_sync(0xffffffffu, my_at, it + 1) : -1;
                const float ks = __shfl_sync(0xffffffffu, my_ks, it), lv = __shfl_sync(0xffffffffu, my_lv, it);
                if (at < 0) {   // no page: no key is visible
                    load_k(next);
                    load_v(next);
                    at = next;
                    continue;
                }
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
                for (int c = 0; c < NCH; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t a0 = magic_half2(kr[c][0].w[i], 0x4140u), a2 = magic_half2(kr[c][0].w[i], 0x4342u);
                        const uint32_t a1 = magic_half2(kr[c][1].w[i], 0x4140u), a3 = magic_half2(kr[c][1].w[i], 0x4342u);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16816(s[nt], a0, a1, a2, a3, qf[nt][c][2 * i], qf[nt][c][2 * i + 1]);
                    }
                load_k(next);
                const int vi = base + DEC_WARPS * it, j0 = (vi < sb ? vi : vi - sb + ws) * KV_BLOCK;
                const bool whole = j0 + KV_BLOCK - 1 <= pmin &&
                                   (a.window == 0 || j0 > pmax - a.window || j0 + KV_BLOCK - 1 < a.n_sink);
                bool raise = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float f = ks * qs[nt][i];
                        s[nt][i] *= f;
                        s[nt][2 + i] *= f;
                        if (!whole) {
                            if (!kv_sees(a, rpos[nt][i], j0 + g)) s[nt][i] = -INFINITY;
                            if (!kv_sees(a, rpos[nt][i], j0 + g + 8)) s[nt][2 + i] = -INFINITY;
                        }
                        const float mx = fmaxf(s[nt][i], s[nt][2 + i]);
                        raise |= mx > m[nt][i] + 8.f || mx + lv > M[nt][i] + 8.f;
                    }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float mx = fmaxf(s[nt][i], s[nt][2 + i]);
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                            const float t = fmaxf(mx + lv, M[nt][i]), al = ex2(M[nt][i] - (t == -INFINITY ? 0.f : t));
                            mx = fmaxf(mx, m[nt][i]);
                            l[nt][i] *= ex2(m[nt][i] - (mx == -INFINITY ? 0.f : mx));
                            m[nt][i] = mx;
                            M[nt][i] = t;
#pragma unroll
                            for (int j = 0; j < MT; ++j) {
                                acc[j][nt][i] *= al;
                                acc[j][nt][2 + i] *= al;
                            }
                        }
                }
                uint32_t pb[NT][2], pl[NT][2];   // P' as fp16, and for fp16 outputs what that rounding left
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float pw[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float mi = m[nt][i & 1], ti = M[nt][i & 1];
                        l[nt][i & 1] += ex2(s[nt][i] - (mi == -INFINITY ? 0.f : mi));
                        const float p = ex2((s[nt][i] - (ti == -INFINITY ? 0.f : ti)) + lv);
                        pw[i] = s[nt][i] == -INFINITY ? 0.f : p;   // a hidden key counts for nothing, whatever its block's scale
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t hi = pack_half2(pw[2 * i], pw[2 * i + 1]);
                        if constexpr (TWO) {
                            const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                            pl[nt][i] = movmatrix(pack_half2(pw[2 * i] - r.x, pw[2 * i + 1] - r.y));
                        }
                        pb[nt][i] = movmatrix(hi);
                    }
                }
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    const uint32_t sel = j & 1 ? 0x7362u : 0x5140u;
                    const uint32_t x = __byte_perm(vr[0].w[j / 2], vr[1].w[j / 2], sel), y = __byte_perm(vr[2].w[j / 2], vr[3].w[j / 2], sel);
                    const uint32_t a0 = magic_half2(x, 0x4140u), a1 = magic_half2(x, 0x4342u);
                    const uint32_t a2 = magic_half2(y, 0x4140u), a3 = magic_half2(y, 0x4342u);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16816(acc[j][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                        if constexpr (TWO) mma16816(acc[j][nt], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
                    }
                }
                load_v(next);
                at = next;
            }
        }
        // join the warps: rows' maxima first, then the scaled accumulators in warp order
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], o);
                if (g == 0) {
                    sm_m[warp][8 * nt + 2 * t + i] = m[nt][i];
                    sm_l[warp][8 * nt + 2 * t + i] = l[nt][i];
                }
            }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 8 * nt + 2 * t + i;
                float mx = sm_m[0][r];
#pragma unroll
                for (int w = 1; w < DEC_WARPS; ++w) mx = fmaxf(mx, sm_m[w][r]);
                const float f = exp2f(M[nt][i] - (mx == -INFINITY ? 0.f : mx));   // from units of 2^M to the maximum's
#pragma unroll
                for (int j = 0; j < MT; ++j)
                    *reinterpret_cast<float2 *>(&sm_o[warp][r][VB * g + 2 * j]) = make_float2(acc[j][nt][i] * f, acc[j][nt][2 + i] * f);
            }
        __syncthreads();
        for (int i = threadIdx.x; i < rn * (D / 4); i += 32 * DEC_WARPS) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float mx = sm_m[0][r], ls = 0.f;
#pragma unroll
            for (int w = 1; w < DEC_WARPS; ++w) mx = fmaxf(mx, sm_m[w][r]);
            const float mu = mx == -INFINITY ? 0.f : mx;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < DEC_WARPS; ++w) {
                ls += sm_l[w][r] * exp2f(sm_m[w][r] - mu);
                const float4 x = *reinterpret_cast<const float4 *>(&sm_o[w][r][d]);
                o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
            }
            const int64_t row = row_of(r);
            if (a.splits > 1) {
                if (d == 0) a.part_ml[row * a.part_stride + split] = make_float2(mx, ls);
                if (lo < hi) *reinterpret_cast<float4 *>(a.part_o + (row * a.part_stride + split) * D + d) = o;
            } else {
                const float inv = ls == 0.f ? 0.f : 1.f / ls;   // no visible key: zeros
                kv_store4(static_cast<T *>(a.out) + row * D + d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
                if (a.lse && d == 0) a.lse[row] = ls == 0.f ? -INFINITY : (mx + log2f(ls)) * 0.69314718f;
            }
        }
        __syncthreads();
    }
    clear();
}

// Joins the shares of a row: WR warps take every WR-th share each, in order, and are added in order.  Latency bounds it (5 us
// alone for 768 rows of 4 shares); it starts under the kernel before it and finds its row's sequence meanwhile.
template <typename T, int D, int WR>
__global__ void __launch_bounds__(128) k_kv_join(const __grid_constant__ KvAttnArgs a) {
    constexpr int W = D / 32, ROWS = 4 / WR;
    __shared__ float sm_o[4][D], sm_l[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, qh = a.c.heads * a.group, w0 = warp % WR;
    const int64_t row = (int64_t)blockIdx.x * ROWS + warp / WR;
    int shares = 0;
    if (row < (int64_t)a.c.n_tokens * qh) {
        const int tok = (int)(row / qh);
        int64_t base;
        const int b = kv_find(a.c.q_start, a.c.batch, a.c.n_tokens, 1, 1, 0, tok, base);
        int first;
        const int n = a.c.tokens(b, first);
        if (tok >= first && tok < first + n) shares = n * a.group > a.max_rows ? a.pf_splits : a.splits;
    }
    // Every CTA waits, one without work too: this grid's end stands for the end of the kernels before it.
    griddep_wait();
    if (WR == 4 && shares <= 1) return;            // no sequence's row, or a finished one
    const float2 *ml = a.part_ml + row * a.part_stride;
    float mx = -INFINITY, ls = 0.f, o[W];
#pragma unroll
    for (int i = 0; i < W; ++i) o[i] = 0.f;
    if (shares > 1) {
        int used = 0;                              // places past the sequence's shares hold (-inf, 0), nothing was written for them
        for (int s = lane; s < shares; s += 32) {
            const float2 x = ml[s];
            mx = fmaxf(mx, x.x);
            if (!(x.x == -INFINITY && x.y == 0.f)) used = s + 1;
        }
        mx = warp_max(mx);
        used = __reduce_max_sync(0xffffffffu, used);
        const float mu = mx == -INFINITY ? 0.f : mx;
#pragma unroll 4
        for (int s = w0; s < used; s += WR) {
            const float2 x = ml[s];
            const float f = ex2(x.x - mu);         // 0 for a share without a visible key, whose part was not written
            const float *p = a.part_o + (row * a.part_stride + s) * D + W * lane;
            ls += x.y * f;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float v = p[i];
                o[i] += x.x == -INFINITY ? 0.f : f * v;
            }
        }
    }
    if constexpr (WR > 1) {
#pragma unroll
        for (int i = 0; i < W; ++i) sm_o[warp][W * lane + i] = o[i];
        if (lane == 0) sm_l[warp] = ls;
        __syncthreads();
        if (w0 > 0) return;
        for (int k = 1; k < WR; ++k) {             // a NaN in any share stays one
            ls += sm_l[warp + k];
#pragma unroll
            for (int i = 0; i < W; ++i) o[i] += sm_o[warp + k][W * lane + i];
        }
    }
    if (shares <= 1) return;
    const float inv = ls == 0.f ? 0.f : 1.f / ls;
    T *out = static_cast<T *>(a.out) + row * D + W * lane;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if constexpr (std::is_same<T, __half>::value) out[i] = __float2half_rn(o[i] * inv);
        else out[i] = __float2bfloat16_rn(o[i] * inv);
    }
    if (a.lse && lane == 0) a.lse[row] = ls == 0.f ? -INFINITY : (mx + log2f(ls)) * 0.69314718f;
}

// ----------------------------------------------------------------------------------------------------------- host
// Sequences of at most this many rows go to the few-row kernel when a batch has longer ones too.
constexpr int DEC_MAX_ROWS = 64;
constexpr size_t PART_BYTES_MAX = (size_t)64 << 20;   // partial results stay in L2

struct KvAttnPlan {
    bool few, many;              // kernels that run
    int nt, row_tiles, splits, units, pf_items, pf_splits, part_stride, max_rows;
    size_t part_o, bytes;
};

static KvAttnPlan kv_plan(const v3g_kv_cache_t *c, const v3g_kv_batch_t *b, uint32_t q_heads, uint32_t max_q, uint32_t max_kv,
                          uint32_t window, uint32_t n_sink) {
    KvAttnPlan p = {};
    const uint64_t group = q_heads / c->n_kv_heads, seq = (uint64_t)b->batch * c->n_kv_heads;
    const uint64_t mean = (b->n_tokens + b->batch - 1) / b->batch;
    uint64_t longest = max_q && max_q < b->n_tokens ? max_q : b->n_tokens;   // as the host knows it: a hint
    if (longest < mean) longest = mean;
    p.few = true;
    p.max_rows = 0x7FFFFFFF;
    if (longest * group > DEC_MAX_ROWS) {
        p.many = true;
        p.few = longest * b->batch > b->n_tokens;                            // else all are of that length
        p.max_rows = p.few ? DEC_MAX_ROWS : 0;
    }
    uint64_t keys = (uint64_t)b->max_pages * c->page;
    if (max_kv && max_kv < keys) keys = max_kv;
    auto seen = [&](uint64_t tokens) {
        const uint64_t w = (uint64_t)window + n_sink + tokens + 2 * KV_BLOCK;
        return window && w < keys ? w : keys;
    };
    const uint64_t room = PART_BYTES_MAX / (((uint64_t)b->n_tokens * q_heads) * (c->head_dim + 2) * 4);
    p.splits = p.pf_splits = p.row_tiles = 1;
    if (p.few) {
        const uint64_t tokens = p.many ? (longest * group < DEC_MAX_ROWS ? longest : (DEC_MAX_ROWS + group - 1) / group) : longest;
        const uint64_t rows = tokens * group;
        p.nt = rows > 8 ? 2 : 1;
        uint64_t tiles = (rows + 8 * p.nt - 1) / (8 * p.nt);
        while (tiles > 1 && tiles * seq > 0x1000000u) tiles = (tiles + 1) / 2;   // a tile loop serves the rest
        p.row_tiles = (int)tiles;
        const uint64_t blocks = (seen(tokens) + KV_BLOCK - 1) / KV_BLOCK, most = (blocks + DEC_MIN_BLOCKS - 1) / DEC_MIN_BLOCKS;
        // Every CTA slot (4 per SM) gets a share, none less than DEC_MIN_BLOCKS blocks; beside the many-row kernel, whose
        // sequences take no shares here, twice as many.  Where a sequence's shares would be few (1 to 7), they are given out by
        // the lengths instead: 64 sequences of 1,411-4,608 keys take 26.3 us instead of 29.1, 128 of them 45.6 instead of
        // 51.9, for 2 us of one warp's work per CTA that equal lengths pay for nothing (64 of 3,000: 27.2 instead of 25.3).
        // With more shares each, or more units than slots, nothing is won.
        const uint64_t slots = (p.many ? 148 * 8 : 148 * 4) / (c->n_kv_heads * tiles);
        uint64_t s = slots / b->batch;
        if (!p.many && b->batch > 1 && b->batch <= BALANCE_MAX && slots > b->batch && slots < 8 * (uint64_t)b->batch) {
            p.units = (int)slots;
            s = slots - b->batch + 1 < 4 * s + 4 ? slots - b->batch + 1 : 4 * s + 4;
        }
        s = s > most ? most : s;
        s = s > room ? room : s;
        p.splits = s < 1 ? 1 : (s > 128 ? 128 : (int)s);
        if (p.splits == 1) p.units = 0;
    }
    if (p.many) {
        // Units that have room in the grid, and about how many of them hold rows: sequences end within one.  Fewer than
        // half the SMs: shares of the keys fill the others, eight key tiles each at least.  (Splitting what is left after whole
        // rounds of the SMs was no gain: 216 units on 148 SMs, 78 us whole, 70 us and 6 us for the join with the last 68 in
        // two.)
        const uint64_t items = (uint64_t)b->n_tokens * group / PF_ROWS + b->batch, live = (items - b->batch / 2) * c->n_kv_heads;
        const uint64_t most = (seen(longest) + 1023) / 1024;
        uint64_t s = 148 / live;
        s = s > most ? most : s;
        s = s > room ? room : s;
        p.pf_items = (int)items + 1;   // one that is never a sequence's
        p.pf_splits = s < 1 ? 1 : (s > 128 ? 128 : (int)s);
    }
    p.part_stride = p.splits > p.pf_splits ? p.splits : p.pf_splits;
    if (p.part_stride > 1) {
        const size_t n = (size_t)b->n_tokens * q_heads * p.part_stride;
        p.part_o = (n * sizeof(float2) + 255) & ~(size_t)255;
        p.bytes = p.part_o + n * c->head_dim * sizeof(float);
    }
    return p;
}

template <typename T, int D>
static cudaError_t launch_attention_kernels(const KvAttnArgs &a, const KvAttnPlan &p, int dtype, cudaStream_t st) {
    cudaError_t e = cudaSuccess;
    if (p.few) {
        const dim3 grid((uint32_t)((a.units ? (uint64_t)a.units : (uint64_t)a.c.batch * a.splits) * a.c.heads * a.row_tiles));
        if (p.nt == 1) e = launch_k(false, k_kv_decode<T, D, 1>, grid, 32 * DEC_WARPS, 0, st, a);
        else e = launch_k(false, k_kv_decode<T, D, 2>, grid, 32 * DEC_WARPS, 0, st, a);
    }
    if (e == cudaSuccess && p.many) e = launch_kv_prefill(a, dtype, D, a.max_rows + 1, st);
    if (e != cudaSuccess || a.part_stride == 1) return e;
    // four warps a row while rows are few
    const int64_t rows = (int64_t)a.c.n_tokens * a.c.heads * a.group;
    if (rows <= 148 * 16) return launch_k(true, k_kv_join<T, D, 4>, dim3((uint32_t)rows), 128, 0, st, a);
    return launch_k(true, k_kv_join<T, D, 1>, dim3((uint32_t)((rows + 3) / 4)), 128, 0, st, a);
}

}  // namespace v3g

using namespace v3g;

static bool attention_shape(const v3g_kv_cache_t *c, const v3g_kv_batch_t *b, uint32_t q_heads) {
    return c && b && c->n_kv_heads && q_heads && q_heads % c->n_kv_heads == 0 && q_heads <= 65535u && b->batch && b->n_tokens &&
           b->max_pages && c->page >= 16;
}

extern "C" size_t v3g_kv_attention_work_size(const v3g_kv_cache_t *cache, const v3g_kv_batch_t *batch, uint32_t n_q_heads,
                                             uint32_t max_q, uint32_t max_kv, uint32_t window, uint32_t n_sink) {
    if (!attention_shape(cache, batch, n_q_heads)) return 0;
    return kv_plan(cache, batch, n_q_heads, max_q, max_kv, window, n_sink).bytes;
}

extern "C" int v3g_kv_attention(const v3g_kv_cache_t *cache, uint32_t layer, const v3g_kv_batch_t *batch, int dtype, const v3g_rows_t *q,
                                uint32_t n_q_heads, float scale, uint32_t window, uint32_t n_sink, uint32_t max_q, uint32_t max_kv,
                                void *out, float *lse, int32_t *dev_status, void *dev_work, size_t work_bytes, void *stream) {
    KvAttnArgs a = {};
    const int rc = kv_view("v3g_kv_attention", cache, layer, batch, &a.c);
    if (rc != V3G_OK) return rc;
    if (dtype != V3G_F16 && dtype != V3G_BF16) return v3g_fail(V3G_E_DTYPE, "v3g_kv_attention: fp16 or bf16 queries");
    if (n_q_heads == 0 || n_q_heads % cache->n_kv_heads || n_q_heads > 65535u)
        return v3g_fail(V3G_E_ARG, "v3g_kv_attention: the query heads must be a multiple of the KV heads");
    if (!std::isfinite(scale)) return v3g_fail(V3G_E_ARG, "v3g_kv_attention: scale must be finite");
    if (batch->batch == 0 || batch->n_tokens == 0) return V3G_OK;
    if (!q || !q->data || !out) return v3g_fail(V3G_E_ARG, "v3g_kv_attention: null pointer");
    if (reinterpret_cast<uintptr_t>(q->data) % 2 || reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(lse) % 4 ||
        reinterpret_cast<uintptr_t>(dev_status) % 4)
        return v3g_fail(V3G_E_ALIGN, "v3g_kv_attention: out needs 16-byte alignment");
    if ((uint64_t)batch->n_tokens * n_q_heads > 0x7FFFFFFFu) return v3g_fail(V3G_E_LIMIT, "v3g_kv_attention: too many query rows");
    if (window > 0x40000000u) window = 0;   // past every position
    if (n_sink > 0x40000000u) n_sink = 0x40000000u;
    const KvAttnPlan p = kv_plan(cache, batch, n_q_heads, max_q, max_kv, window, n_sink);
    if (p.bytes && (!dev_work || work_bytes < p.bytes)) return v3g_fail(V3G_E_SIZE, "v3g_kv_attention: workspace too small");
    if (p.bytes && reinterpret_cast<uintptr_t>(dev_work) % 256) return v3g_fail(V3G_E_ALIGN, "v3g_kv_attention: the workspace needs 256-byte alignment");
    if ((uint64_t)batch->batch * cache->n_kv_heads * p.splits * p.row_tiles > 0x7FFFFFFFu ||
        (uint64_t)p.pf_items * cache->n_kv_heads * p.pf_splits > 0x7FFFFFFFu)
        return v3g_fail(V3G_E_LIMIT, "v3g_kv_attention: too many sequences and heads");
    a.q = q->data;
    a.q_tok = q->tok_stride;
    a.q_head = q->head_stride;
    a.q_vec = reinterpret_cast<uintptr_t>(q->data) % 8 == 0 && q->tok_stride % 4 == 0 && q->head_stride % 4 == 0;
    a.q_vec8 = reinterpret_cast<uintptr_t>(q->data) % 16 == 0 && q->tok_stride % 8 == 0 && q->head_stride % 8 == 0;
    a.group = (int)(n_q_heads / cache->n_kv_heads);
    a.scale_log2 = scale * 1.44269504f;
    a.window = (int)window;
    a.n_sink = (int)n_sink;
    a.out = out;
    a.lse = lse;
    a.splits = p.splits;
    a.units = p.units;
    a.row_tiles = p.row_tiles;
    a.max_rows = p.max_rows;
    a.pf_items = p.pf_items;
    a.pf_splits = p.pf_splits;
    a.after_few = p.many && p.few;
    a.part_stride = p.part_stride;
    a.status = dev_status;
    a.part_ml = static_cast<float2 *>(dev_work);
    a.part_o = reinterpret_cast<float *>(static_cast<uint8_t *>(dev_work) + p.part_o);
    const cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (dtype == V3G_F16)
        e = cache->head_dim == 64 ? launch_attention_kernels<__half, 64>(a, p, dtype, st) : launch_attention_kernels<__half, 128>(a, p, dtype, st);
    else
        e = cache->head_dim == 64 ? launch_attention_kernels<__nv_bfloat16, 64>(a, p, dtype, st)
                                  : launch_attention_kernels<__nv_bfloat16, 128>(a, p, dtype, st);
    return e == cudaSuccess ? V3G_OK : v3g_fail(V3G_E_CUDA, std::string("v3g_kv_attention: ") + cudaGetErrorString(e));
}
