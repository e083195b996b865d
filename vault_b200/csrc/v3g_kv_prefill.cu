// Attention over the paged 8-bit cache: many query rows per KV head (prompts, long chunks), on tcgen05.
//
// 4 D flops per visible (row, key) against 2 D bytes of codes per key and 256 rows: the tensor cores and the
// exponentials bound it.  A CTA takes 256 rows (token, query head) of one KV head of one sequence as two M = 128 tiles and
// walks the visible keys in tiles of 128:
//
//   warps 0-3, 4-7   softmax of tile 0 / 1, one row per thread: scores from tensor memory, P' back to it (fp16, over the
//                    scores' own columns), and the final division
//   warps 8-11       converters: codes from their pages to fp16 operands (exact: permute to 1024 + c, minus 1152), two
//                    stages each of K and V.  Both are stored [key][d] with the 128-byte swizzle, K read as a K-major
//                    operand, V as an MN-major one, so neither is transposed
//   warp 12          tensor memory and the MMAs: S = Q K^T (128 x 128), O += P' V (P' from tensor memory)
//
// The two tiles alternate, so one tile's softmax runs under the other's MMAs: in issue order PV0(j), QK0(j+1), PV1(j),
// QK1(j+1).  tcgen05 operations of one thread run in order, so QK(j+1) may overwrite P'(j), and a full S(j) says that
// PV(j-1) is done: a row whose maximum grew by more than 8 (else its old one stays; P' is then below 2^12) rescales its
// O in tensor memory right there.
//
// K scales multiply the scores; a V scale vs enters the exponent, P' = 2^(s - m + log2(vs / ref)), ref a power of two
// that follows the largest vs, and the row sum takes P' ref / vs.  vs / ref is held at or above 2^-40, where P' rounds to
// zero in fp16 whatever p is: a block with scale 0 adds nothing to O and its full weight to the sum.
#include <atomic>
#include <cfloat>

#include "v3g_internal.h"
#include "v3g_kv.cuh"
#include "v3g_kv_attn.cuh"
#include "v3g_tc.cuh"

namespace v3g {

constexpr int PF_ROWS = 256, PF_KEYS = 128, PF_THREADS = 512;
constexpr int PF_SCALES = 4;   // ring of scale sets: the converters are at most two tiles ahead of the softmax

template <int D>
struct PfSmem {
    static constexpr int OP = 128 * D * 2;                      // one 128 x D fp16 operand
    static constexpr int Q = 0, K = 2 * OP, V = 4 * OP, SC = 6 * OP, BAR = SC + PF_SCALES * 128, END = BAR + 192, BYTES = END + 1024;
};

struct PfScales {   // of one key tile: per 16-key block
    float ks[8], lv[8], iv[8];   // K scale, log2 of the V scale, its inverse
    uint32_t valid, pad[7];      // bit i: block i has a page
};
static_assert(sizeof(PfScales) == 128, "scale ring slot");

#define TC_REGS8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define TC_IN8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : TC_REGS8(r, 0), TC_REGS8(r, 8), TC_REGS8(r, 16), TC_REGS8(r, 24)
        : "r"(a));
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::TC_IN8(r, 0),
        TC_IN8(r, 8), TC_IN8(r, 16), TC_IN8(r, 24), "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::TC_IN8(r, 0),
        TC_IN8(r, 8), "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem, fp16 pairs] * B[smem desc]
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// V as the MN-major B operand: 64 d (128 swizzled bytes) x 8 keys per 1024-byte atom; key groups 1024 bytes apart (stride
// offset), the second 64 d one half operand apart (leading offset)
template <int D>
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(16384u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1u << 46) |
           ((uint64_t)2u << 61);
}
__device__ __forceinline__ float pf_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pf_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint4 pf_convert8(uint32_t a, uint32_t b) {   // eight codes -> eight fp16
    uint4 r;
    uint32_t *o = &r.x;
    const __half2 z = __float2half2_rn(1152.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = __byte_perm(i < 2 ? a : b, 0x64646464u, i & 1 ? 0x4342u : 0x4140u);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&v), z);
        o[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return r;
}

// a whole warp's bounded wait: one answer for all its lanes
__device__ __forceinline__ bool pf_wait(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity)); }

// visible keys of 32 consecutive ones from kb, as a bit mask, for a row at position p
__device__ __forceinline__ uint32_t pf_mask(const KvAttnArgs &a, int p, int kb, uint32_t pages) {
    auto below = [](int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u); };   // the first n bits
    uint32_t m = below(p - kb + 1);
    if (a.window) m &= ~below(p - a.window + 1 - kb) | below(a.n_sink - kb);
    return m & ((pages & 1u ? 0xFFFFu : 0u) | (pages & 2u ? 0xFFFF0000u : 0u));
}

template <typename T, int D>
__global__ void __launch_bounds__(PF_THREADS, 1) k_kv_prefill(const __grid_constant__ KvAttnArgs a, int min_rows) {
    typedef PfSmem<D> SM;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (tc::smem_addr(smem_raw) & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the rows of this CTA; late tiles see the most keys and go first
    int64_t base;
    const int64_t item = gridDim.x - 1 - blockIdx.x;
    const int b = kv_find(a.c.q_start, a.c.batch, a.c.n_tokens, PF_ROWS, a.group, 1, item, base);
    const int h = blockIdx.y;
    int first;
    const int n = a.c.tokens(b, first);
    const int64_t off = (item - base) * PF_ROWS;
    if (off < 0 || off >= (int64_t)n * a.group || n * a.group < min_rows) return;
    const int r0 = (int)off, rn = min(n * a.group - r0, PF_ROWS), tiles = rn > 128 ? 2 : 1;
    const int p0 = a.c.end(b) - n;
    int sb, ws;
    const int plo = p0 + r0 / a.group, phi = p0 + (r0 + rn - 1) / a.group;
    const int all = kv_visible(a, plo, phi, PF_KEYS, sb, ws);
    // this CTA's share of the key tiles
    const int per = (all + a.pf_splits - 1) / a.pf_splits, jlo = min((int)blockIdx.z * per, all), nk = min(per, all - jlo);
    auto key0 = [&](int j) { return (j + jlo < sb ? j + jlo : j + jlo - sb + ws) * PF_KEYS; };

    const uint32_t bars = tc::smem_addr(smem + SM::BAR);
    // barrier slots
    auto QFULL = bars;
    auto KFULL = [&](int s) { return bars + 8u * (1 + s); };
    auto KEMPTY = [&](int s) { return bars + 8u * (3 + s); };
    auto VFULL = [&](int s) { return bars + 8u * (5 + s); };
    auto VEMPTY = [&](int s) { return bars + 8u * (7 + s); };
    auto SFULL = [&](int t) { return bars + 8u * (9 + t); };
    auto PFULL = [&](int t) { return bars + 8u * (11 + t); };
    auto OFULL = [&](int t) { return bars + 8u * (13 + t); };
    auto SCFULL = [&](int s) { return bars + 8u * (15 + s); };
    const uint32_t DRAIN = bars + 8u * 19;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + SM::BAR + 160);
    PfScales *scales = reinterpret_cast<PfScales *>(smem + SM::SC);
    if (threadIdx.x == 0) {
        tc::mbar_init(QFULL, 4 * tiles);
        for (int s = 0; s < 2; ++s) {
            tc::mbar_init(KFULL(s), 4);
            tc::mbar_init(KEMPTY(s), 1);
            tc::mbar_init(VFULL(s), 4);
            tc::mbar_init(VEMPTY(s), 1);
            tc::mbar_init(SFULL(s), 1);
            tc::mbar_init(PFULL(s), 4);
            tc::mbar_init(OFULL(s), 1);
        }
        for (int s = 0; s < PF_SCALES; ++s) tc::mbar_init(SCFULL(s), 1);
        tc::mbar_init(DRAIN, 1);
        tc::mbar_fence_init();
    }
    if (warp == 12) tc::tmem_alloc(tc::smem_addr(tmem_slot), 512);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp < 8) {   // ------------------------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int tile = warp >> 2, row = 32 * (warp & 3) + lane;
        const int r = r0 + 128 * tile + row, tok = r / a.group;
        const bool live = 128 * tile + row < rn;
        const int qh = h * a.group + r - tok * a.group;
        const uint32_t lane_tm = tmem + ((uint32_t)(32 * (warp & 3)) << 16), tS = lane_tm + 128u * tile, tO = lane_tm + 256u + 128u * tile;
        if (tile < tiles) {
            // the row's query: a power of two brings it into fp16 (sign of the scale with it), 128-byte swizzled halves
            float qf;
            {
                const T *src = static_cast<const T *>(a.q) + (int64_t)(first + tok) * a.q_tok + (int64_t)qh * a.q_head;
                float top = 0.f;
                if (live)
                    for (int i = 0; i < D; i += 4) {
                        const float4 v = kv_load4<T>(src + i, a.q_vec);
                        top = fmaxf(fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
                    }
                const int up = kv_row_exponent<T>(top);
                const float f = __int_as_float((up + 127) << 23) * (a.scale_log2 < 0.f ? -1.f : 1.f);
                qf = __int_as_float((127 - up) << 23) * fabsf(a.scale_log2);
                uint8_t *dst = smem + SM::Q + tile * SM::OP + row * 128;
#pragma unroll 4
                for (int c = 0; c < D / 8; ++c) {
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
                    if (live) {
                        x = kv_load4<T>(src + 8 * c, a.q_vec);
                        y = kv_load4<T>(src + 8 * c + 4, a.q_vec);
                    }
                    *reinterpret_cast<uint4 *>(dst + (c >> 3) * 16384 + (((c & 7) ^ (row & 7)) << 4)) =
                        make_uint4(pf_half2(x.x * f, x.y * f), pf_half2(x.z * f, x.w * f), pf_half2(y.x * f, y.y * f), pf_half2(y.z * f, y.w * f));
                }
                tc::fence_proxy_async();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(QFULL);
            }
            const int p = live ? p0 + tok : -1;
            const int tn = min(rn - 128 * tile, 128);
            const int pmin = p0 + (r0 + 128 * tile) / a.group, pmax = p0 + (r0 + 128 * tile + tn - 1) / a.group;
            float m = -INFINITY, l = 0.f, eref = -126.f;   // eref: log2 of ref
            for (int j = 0; j < nk && ok; ++j) {
                ok = pf_wait(SCFULL(j & (PF_SCALES - 1)), (j / PF_SCALES) & 1) && pf_wait(SFULL(tile), j & 1);
                if (!ok) break;
                tc::tc_fence_after();
                uint32_t s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(tS + 32 * c, s + 32 * c);
                const PfScales &sc = scales[j & (PF_SCALES - 1)];
                const int k0 = key0(j);
                const uint32_t valid = sc.valid;
                const bool whole = valid == 0xFFu && k0 + PF_KEYS - 1 <= pmin &&
                                   (a.window == 0 || k0 > pmax - a.window || k0 + PF_KEYS - 1 < a.n_sink);
                float f[8], lv[8];
                float vmax = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    f[i] = sc.ks[i] * qf;
                    lv[i] = sc.lv[i];
                    vmax = fmaxf(vmax, lv[i]);
                }
                tc::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 128; ++i) asm volatile("" : "+r"(s[i]));   // no use moves above the wait
                if (!whole)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t see = pf_mask(a, p, k0 + 32 * c, valid >> (2 * c));
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(see >> i & 1u)) s[32 * c + i] = 0xFF800000u;
                    }
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float g = __uint_as_float(s[16 * i]);
#pragma unroll
                    for (int e = 1; e < 16; ++e) g = fmaxf(g, __uint_as_float(s[16 * i + e]));
                    mx = fmaxf(mx, g * f[i]);
                }
                float al = 1.f;
                bool change = false;
                if (mx > m + 8.f) {
                    al = pf_ex2(m - mx);
                    m = mx;
                    l *= al;
                    change = true;
                }
                if (vmax > eref + 4.f) {   // the same in every thread of the CTA
                    const float e = fminf(fmaxf(ceilf(vmax), -120.f), 120.f);
                    al *= pf_ex2(eref - e);
                    change = true;
                    eref = e;
                }
                if (__any_sync(0xffffffffu, change) && j > 0) {
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tc::tmem_ld16(tO + 16 * c, o);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(o[i]));
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                        tmem_st16(tO + 16 * c, o);
                    }
                }
                const float mu = m == -INFINITY ? 0.f : m, ref = pf_ex2(eref);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pk[16], see = ~0u;
                    if (!whole) see = pf_mask(a, p, k0 + 32 * c, valid >> (2 * c));
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int i = 2 * c + u;
                        const float w = lv[i] - eref, cw = (w < -40.f ? -40.f : w) - mu;   // a NaN scale stays one
                        float sum = 0.f;
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            float x = pf_ex2(fmaf(__uint_as_float(s[16 * i + e]), f[i], cw));
                            float y = pf_ex2(fmaf(__uint_as_float(s[16 * i + e + 1]), f[i], cw));
                            if (!whole) {
                                x = see >> (16 * u + e) & 1u ? x : 0.f;
                                y = see >> (16 * u + e + 1) & 1u ? y : 0.f;
                            }
                            sum += x + y;
                            pk[8 * u + e / 2] = pf_half2(x, y);
                        }
                        l = fmaf(sum, fminf(sc.iv[i] * ref, 0x1p40f), l);
                    }
                    tmem_st16(tS + 16 * c, pk);
                }
                tmem_st_wait();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(PFULL(tile));
            }
            const int64_t out_row = (int64_t)(first + tok) * a.c.heads * a.group + qh;
            float inv = 0.f;
            if (nk > 0 && ok) {
                ok = pf_wait(OFULL(tile), 0);
                tc::tc_fence_after();
                inv = a.pf_splits > 1 ? pf_ex2(eref) : (l == 0.f ? 0.f : pf_ex2(eref) / l);
            }
            const int64_t part = out_row * a.part_stride + blockIdx.z;
            if (ok && (nk > 0 || a.pf_splits == 1))   // an empty share has no accumulator
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = 0u;
                    if (nk > 0) {
                        tc::tmem_ld16(tO + 16 * c, o);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(o[i]));
                    }
                    if (live)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const float4 v = make_float4(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv,
                                                         __uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                            if (a.pf_splits > 1) kv_store4(a.part_o + part * D + 16 * c + i, v);
                            else kv_store4(static_cast<T *>(a.out) + out_row * D + 16 * c + i, v);
                        }
                }
            if (live && ok) {
                if (a.pf_splits > 1) a.part_ml[part] = make_float2(m, l);
                else if (a.lse) a.lse[out_row] = l == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m) + log2f(l)) * 0.69314718f;
            }
        }
    } else if (warp < 12) {   // ----------------------------------------------------------------------- converters
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        constexpr int CH = D / 16, RP = 128 / CH, NL = 128 / RP;   // 16-byte pieces of a key, keys of a pass, passes
        const int ct = threadIdx.x - 256, ch = ct % CH, kr = ct / CH;
        uint4 x[NL];
        uint32_t valid = 0;
        // item i: K of tile i / 2 when i is even, V when odd; its codes to registers
        auto load = [&](int i) {
            const int k0 = key0(i >> 1);
            const uint8_t *codes = i & 1 ? a.c.v : a.c.k;
            int pg = -1;
            if (lane < 8) {   // blocks that no row of the CTA sees count as blocks without a page
                const int kb = k0 + 16 * lane;
                if (kb <= phi && (a.window == 0 || kb + 15 > plo - a.window || kb < a.n_sink)) pg = a.c.page_of(b, kb);
            }
            valid = __ballot_sync(0xffffffffu, pg >= 0) & 0xFFu;
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                const int key = u * RP + kr, pos = k0 + key;
                const int page = __shfl_sync(0xffffffffu, pg, key >> 4);
                x[u] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                if (page >= 0) x[u] = ldg_stream16(codes + (a.c.block(page, h, pos) * KV_BLOCK + (pos & 15)) * D + 16 * ch);
            }
            if (!(i & 1) && warp == 8 && lane < 8) {   // the tile's scales travel with its K
                PfScales &sc = scales[(i >> 1) & (PF_SCALES - 1)];
                float ks = 0.f, vs = 0.f;
                if (pg >= 0) {
                    const int64_t at = a.c.block(pg, h, k0 + 16 * lane);
                    ks = a.c.ks[at];
                    vs = a.c.vs[at];
                }
                sc.ks[lane] = ks;
                sc.lv[lane] = log2f(vs);
                sc.iv[lane] = 1.f / vs;
                if (lane == 0) sc.valid = valid;
            }
            if (!(i & 1) && warp == 8) {
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(SCFULL((i >> 1) & (PF_SCALES - 1)));
            }
        };
        if (nk > 0) load(0);
        for (int i = 0; i < 2 * nk && ok; ++i) {
            const int j = i >> 1, s = j & 1;
            if (j >= 2 && !(ok = pf_wait(i & 1 ? VEMPTY(s) : KEMPTY(s), ((j >> 1) - 1) & 1))) break;
            uint8_t *op = smem + (i & 1 ? SM::V : SM::K) + s * SM::OP;
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                const int key = u * RP + kr;
                uint8_t *d = op + (ch >> 2) * 16384 + key * 128;
                const uint4 lo = pf_convert8(x[u].x, x[u].y), hi = pf_convert8(x[u].z, x[u].w);
                const int c0 = (ch & 3) * 2, sw = key & 7;
                // lanes of the second half store their upper piece first, so that eight lanes fill all banks
                const bool swap = ch & 4;
                *reinterpret_cast<uint4 *>(d + (((c0 + swap) ^ sw) << 4)) = swap ? hi : lo;
                *reinterpret_cast<uint4 *>(d + (((c0 + !swap) ^ sw) << 4)) = swap ? lo : hi;
            }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(i & 1 ? VFULL(s) : KFULL(s));
            if (i + 1 < 2 * nk) load(i + 1);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 12 && nk > 0) {   // ------------------------------------------------------------- MMA issuer
            constexpr uint32_t id_qk = tc::idesc_f16(128, PF_KEYS), id_pv = tc::idesc_f16(128, D) | (1u << 16);
            auto qk = [&](int t, int j) {
                if (lane == 0) {
                    const uint32_t sq = tc::smem_addr(smem + SM::Q + t * SM::OP), sk = tc::smem_addr(smem + SM::K + (j & 1) * SM::OP);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t o = (k >> 2) * 16384 + (k & 3) * 32;
                        tc::mma_f16(tmem + 128u * t, tc::sw128_desc(sq + o), tc::sw128_desc(sk + o), id_qk, k > 0);
                    }
                    tc::mma_commit(SFULL(t));
                }
                __syncwarp();
            };
            ok = pf_wait(QFULL, 0) && pf_wait(KFULL(0), 0);
            tc::tc_fence_after();
            if (ok) {
                for (int t = 0; t < tiles; ++t) qk(t, 0);
                if (lane == 0) tc::mma_commit(KEMPTY(0));
                __syncwarp();
            }
            for (int j = 0; j < nk && ok; ++j) {
                for (int t = 0; t < tiles && ok; ++t) {
                    ok = pf_wait(PFULL(t), j & 1) && (t > 0 || pf_wait(VFULL(j & 1), (j >> 1) & 1));
                    if (!ok) break;
                    tc::tc_fence_after();
                    if (lane == 0) {
                        const uint32_t sv = tc::smem_addr(smem + SM::V + (j & 1) * SM::OP);
#pragma unroll
                        for (int k = 0; k < PF_KEYS / 16; ++k)
                            mma_f16_ts(tmem + 256u + 128u * t, tmem + 128u * t + 8u * k, v_desc<D>(sv + 2048u * k), id_pv, j > 0 || k > 0);
                        if (t == tiles - 1) tc::mma_commit(VEMPTY(j & 1));
                        if (j == nk - 1) tc::mma_commit(OFULL(t));
                    }
                    __syncwarp();
                    if (j + 1 < nk) {
                        if (t == 0 && !(ok = pf_wait(KFULL((j + 1) & 1), ((j + 1) >> 1) & 1))) break;
                        tc::tc_fence_after();
                        qk(t, j + 1);
                        if (t == tiles - 1 && lane == 0) tc::mma_commit(KEMPTY((j + 1) & 1));
                        __syncwarp();
                    }
                }
            }
            // nothing of this CTA is in flight when tensor memory is given back
            if (lane == 0) tc::mma_commit(DRAIN);
            __syncwarp();
            ok = pf_wait(DRAIN, 0) && ok;
        }
    }
    if (!ok && a.status) atomicOr(a.status, STATUS_TIMEOUT);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == 12) tc::tmem_dealloc(tmem, 512);
}

template <typename T, int D>
static cudaError_t launch_pf(const KvAttnArgs &a, int min_rows, cudaStream_t st) {
    auto kern = k_kv_prefill<T, D>;
    // Once per device: room for the operands, and the check that the launch brings the 512 x 128 registers that the warps'
    // shares (setmaxnreg) add up to; with fewer they would wait for good.
    static std::atomic<uint64_t> ready{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !(ready.load() >> dev & 1u)) {
        cudaFuncAttributes at;
        e = cudaFuncGetAttributes(&at, kern);
        if (e == cudaSuccess && at.numRegs != 128) e = cudaErrorInvalidConfiguration;
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PfSmem<D>::BYTES);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) ready.fetch_or(1ull << dev);
    }
    const int64_t items = (int64_t)a.c.n_tokens * a.group / PF_ROWS + a.c.batch;
    return launch_k(false, kern, dim3((uint32_t)items, a.c.heads, a.pf_splits), PF_THREADS, PfSmem<D>::BYTES, st, a, min_rows);
}

cudaError_t launch_kv_prefill(const KvAttnArgs &a, int dtype, int head_dim, int min_rows, cudaStream_t st) {
    if (dtype == V3G_F16) return head_dim == 64 ? launch_pf<__half, 64>(a, min_rows, st) : launch_pf<__half, 128>(a, min_rows, st);
    return head_dim == 64 ? launch_pf<__nv_bfloat16, 64>(a, min_rows, st) : launch_pf<__nv_bfloat16, 128>(a, min_rows, st);
}

}  // namespace v3g
