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
//   warps 12, 13     the MMAs of tile 0 / 1: S = Q K^T, O += P' V (P' from tensor memory); warp 12 holds tensor memory
//   warp 14          the tiles' pages and scales
//
// A step is 64 keys of one tile: S = Q K^T into one of the tile's two score buffers, softmax, P' over the same columns,
// O += P' V.  A tile's issuer runs PV(u), QK(u + 2): while these run, the tile's softmax works on the other buffer, so neither
// waits for a round trip.  tcgen05 operations of one thread run in order, so QK(u + 2) may overwrite P'(u).  Each tile has
// an issuer in another quarter of the SM, because an issuing warp slows the softmax warps of its quarter (one issuer for
// both tiles: 718 us for the 8,192-token prompt, 32/8 heads; two: 693).  The offset m of a row's exponents is its maximum
// when m was set, plus 3; it stays until a score passes it by 11 (P' is then below 2^11).  Only then the warp rescales its O
// in tensor memory, after a wait for PV(u - 1): with a margin of 8 from the maximum itself, some row of the 32 did so at every
// second step on scores of standard deviation 3.
//
// K scales multiply the scores; a V scale vs enters the exponent, P' = 2^(s + log2 vs - M), with a second offset M of the
// row's own that follows the largest of its terms p vs as m follows its largest score, so that no block which the row does
// not see, or gives no weight, can push its P' into the range where fp16 has fewer bits.  O stands in units of 2^M, the row
// sum takes P' 2^(M - m) / vs.  P' is held at or above 2^(s - m - 40), where it rounds to zero in fp16 whatever s is: a block
// with scale 0 adds nothing to O and its full weight to the sum.  So does one whose V scale is NaN or infinite, since V is no
// matter of the sum; the warp that looks up the scales notes which rows see such a block, and those have no output.
//
// 8,192 tokens, 32/8 heads of 128, every earlier key: 602 us, 913 TFLOP/s (530 us in a burst, before the clock falls); 4,608
// tokens under a window of 1,024, 12/2 heads: 68 us, of which each of the two rounds of CTAs spends a quarter on its start and
// end.
#include <atomic>
#include <cfloat>

#include "v3g_internal.h"
#include "v3g_kv.cuh"
#include "v3g_kv_attn.cuh"
#include "v3g_tc.cuh"

namespace v3g {

constexpr int PF_KEYS = 128, PF_THREADS = 512;
// Ring of the tiles' places and scales.  Its writer is at most PF_AHEAD tiles past the converters' loads; they load tile t + 1
// after tile t - 2's PV, which needed every softmax warp to be through with that tile's scales, so a slot is written again
// only after its last reader.
constexpr int PF_RING = 8, PF_AHEAD = 5;

template <int D>
struct PfSmem {
    static constexpr int OP = 128 * D * 2;                      // one 128 x D fp16 operand
    static constexpr int Q = 0, K = 2 * OP, V = 4 * OP, SC = 6 * OP, BAR = SC + PF_RING * 192, QF = BAR + 384, BYTES = QF + 1024 + 1024;
};

struct alignas(16) PfPlaces {   // of one key tile, per 16-key block
    float ks[8], lv[8], iv[8];   // K scale, log2 of vs, 1 / vs
    int64_t at[8];               // index of the block in the layer
    int k0;                      // first key
    uint32_t valid, whole;       // bit i: block i has a page and some row sees it; bit 2 tile + half: every key of the half is visible
    uint32_t pad[5];
};
static_assert(sizeof(PfPlaces) == 192, "ring slot");

#define TC_REGS8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define TC_IN8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 64 consecutive columns of the warp's 32 lanes; the values are there after tmem_ld64_done
__device__ __forceinline__ void tmem_ld64(uint32_t a, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,"
        "%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
        : TC_REGS8(r, 0), TC_REGS8(r, 8), TC_REGS8(r, 16), TC_REGS8(r, 24), TC_REGS8(r, 32), TC_REGS8(r, 40), TC_REGS8(r, 48), TC_REGS8(r, 56)
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_ld64_done(uint32_t (&r)[64]) {
    tc::tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 64; ++i) asm volatile("" : "+r"(r[i]));   // no use moves above the wait
}
__device__ __forceinline__ void tmem_ld16_wait(uint32_t a, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : TC_REGS8(r, 0), TC_REGS8(r, 8)
        : "r"(a)
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
__device__ __forceinline__ bool elect_one() {   // one lane of the converged warp
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p;
}
// two fp32 operations at once
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t x, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {   // NaN operands are passed over, as by fmaxf
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
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
__device__ __forceinline__ bool pf_wait(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < tc::WAIT_LIMIT; ++i) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (__all_sync(0xffffffffu, done)) return true;
    }
    return false;
}
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
    griddep_launch();
    // the rows of this CTA, and its share of their keys; late rows see the most keys and go first
    const int shares = a.pf_splits, share = blockIdx.x % shares, unit = blockIdx.x / shares;
    const int64_t item = a.pf_items - 1 - unit / a.c.heads;
    const int h = unit % a.c.heads;
    int64_t base;
    const int b = kv_find(a.c.q_start, a.c.batch, a.c.n_tokens, PF_ROWS, a.group, 1, item, base);
    int first;
    const int n = a.c.tokens(b, first);
    const int64_t off = (item - base) * PF_ROWS;
    if (off < 0 || off >= (int64_t)n * a.group || n * a.group < min_rows) {
        // past the last sequence's units (one for each head at least): the rows of no sequence, unless the few-row kernel runs
        const int64_t idle = item - base - ((int64_t)n * a.group + PF_ROWS - 1) / PF_ROWS, per = (int64_t)a.c.heads * shares;
        if (a.after_few) griddep_wait();
        else if (b == a.c.batch - 1 && idle >= 0)
            kv_clear_loose<T, D>(a.c, static_cast<T *>(a.out), a.lse, a.c.heads * a.group,
                                 (idle * per + h * shares + share) * PF_THREADS + threadIdx.x, (a.pf_items - item + idle) * per * PF_THREADS);
        return;
    }
    const int r0 = (int)off, rn = min(n * a.group - r0, PF_ROWS), tiles = rn > 128 ? 2 : 1;
    const int p0 = a.c.end(b) - n;
    int sb, ws;
    const int plo = p0 + r0 / a.group, phi = p0 + (r0 + rn - 1) / a.group;
    const int all = kv_visible(a, plo, phi, PF_KEYS, sb, ws);
    // this CTA's share of the key tiles
    const int per = (all + shares - 1) / shares, jlo = min(share * per, all), nk = min(per, all - jlo);
    auto key0 = [&](int j) { return (j + jlo < sb ? j + jlo : j + jlo - sb + ws) * PF_KEYS; };

    // The softmax warps' 32 query rows each, LPR lanes to a row so that reads are whole lines, on their way while the barriers
    // are set up
    constexpr int LPR = D / 8, RPI = 32 / LPR;
    const int row_w = 32 * warp, pc = lane % LPR, pr = lane / LPR;   // the warp's first row; this lane's piece, its row in a pass
    uint4 xq[LPR];
    // f(pass, row, its token, its head in the group), for this lane's rows
    auto rows_of = [&](auto f) {
        const int dt = RPI / a.group, dg = RPI - dt * a.group;
        int tk = (r0 + row_w + pr) / a.group, g = r0 + row_w + pr - tk * a.group;
#pragma unroll
        for (int i = 0; i < LPR; ++i) {
            f(i, row_w + i * RPI + pr, tk, g);
            tk += dt, g += dg;
            if (g >= a.group) ++tk, g -= a.group;
        }
    };
    if (warp < 8)
        rows_of([&](int i, int rr, int tk, int g) {
            xq[i] = make_uint4(0u, 0u, 0u, 0u);
            if (rr < rn) {
                const T *src = static_cast<const T *>(a.q) + (int64_t)(first + tk) * a.q_tok + (int64_t)(h * a.group + g) * a.q_head + 8 * pc;
                if (a.q_vec8) xq[i] = ldg_stream16(src);
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e) reinterpret_cast<T *>(&xq[i])[e] = src[e];
            }
        });

    const uint32_t bars = tc::smem_addr(smem + SM::BAR);
    // barrier slots
    auto QFULL = bars;
    auto KFULL = [&](int s) { return bars + 8u * (1 + s); };
    auto KEMPTY = [&](int s) { return bars + 8u * (3 + s); };
    auto VFULL = [&](int s) { return bars + 8u * (5 + s); };
    auto VEMPTY = [&](int s) { return bars + 8u * (7 + s); };
    auto SFULL = [&](int t, int half) { return bars + 8u * (9 + 2 * t + half); };
    auto PFULL = [&](int t, int half) { return bars + 8u * (13 + 2 * t + half); };
    auto ODONE = [&](int t) { return bars + 8u * (17 + t); };
    auto OFULL = [&](int t) { return bars + 8u * (19 + t); };
    auto ATFULL = [&](int s) { return bars + 8u * (21 + s); };
    auto ATEMPTY = [&](int s) { return bars + 8u * (29 + s); };
    const uint32_t DRAIN = bars + 8u * 37;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + SM::BAR + 8 * 38);
    uint32_t *spoilt = tmem_slot + 2;   // a bit for each row: it sees a V scale that is NaN or infinite
    PfPlaces *places = reinterpret_cast<PfPlaces *>(smem + SM::SC);
    if (threadIdx.x == 0) {
        tc::mbar_init(QFULL, 4 * tiles);
        for (int s = 0; s < 2; ++s) {
            tc::mbar_init(KFULL(s), 4);
            tc::mbar_init(KEMPTY(s), tiles);
            tc::mbar_init(VFULL(s), 4);
            tc::mbar_init(VEMPTY(s), tiles);
            for (int half = 0; half < 2; ++half) {
                tc::mbar_init(SFULL(s, half), 1);
                tc::mbar_init(PFULL(s, half), 4);
            }
            tc::mbar_init(ODONE(s), 1);
            tc::mbar_init(OFULL(s), 1);
        }
        for (int s = 0; s < PF_RING; ++s) {
            tc::mbar_init(ATFULL(s), 1);
            tc::mbar_init(ATEMPTY(s), 4);
        }
        tc::mbar_init(DRAIN, tiles);
        for (int i = 0; i < PF_ROWS / 32; ++i) spoilt[i] = 0u;
        tc::mbar_fence_init();
    }
    if (warp == 12) tc::tmem_alloc(tc::smem_addr(tmem_slot), 512);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    constexpr uint32_t tmem = 0;   // all 512 columns are this CTA's: S0 0, S1 128, O0 256, O1 384
    bool ok = *tmem_slot == tmem;

    if (warp < 8) {   // ------------------------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        const int tile = warp >> 2, row = 32 * (warp & 3) + lane;
        const int r = r0 + 128 * tile + row, tok = r / a.group;
        const bool live = 128 * tile + row < rn;
        const int qh = h * a.group + r - tok * a.group;
        const uint32_t lane_tm = tmem + ((uint32_t)(32 * (warp & 3)) << 16), tS = lane_tm + 128u * tile, tO = lane_tm + 256u + 128u * tile;
        if (tile < tiles) {
            // a power of two brings a row into fp16 (the sign of the scale with it), in 128-byte swizzled halves
            float *qfac = reinterpret_cast<float *>(smem + SM::QF);
            uint8_t *piece = smem + SM::Q + tile * SM::OP + (pc >> 3) * 16384;   // rows of 128 bytes, piece pc & 7
            {
#pragma unroll
                for (int i = 0; i < LPR; ++i) {
                    float y[8], top = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        const float4 v = kv_load4<T>(reinterpret_cast<const T *>(&xq[i]) + e, true);
                        y[e] = v.x, y[e + 1] = v.y, y[e + 2] = v.z, y[e + 3] = v.w;
                        top = fmaxf(fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
                    }
#pragma unroll
                    for (int o = 1; o < LPR; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const int up = kv_row_exponent<T>(top), rl = 32 * (warp & 3) + i * RPI + pr;
                    const float f = __int_as_float((up + 127) << 23) * (a.scale_log2 < 0.f ? -1.f : 1.f);
                    *reinterpret_cast<uint4 *>(piece + rl * 128 + (((pc & 7) ^ (rl & 7)) << 4)) =
                        make_uint4(pf_half2(y[0] * f, y[1] * f), pf_half2(y[2] * f, y[3] * f), pf_half2(y[4] * f, y[5] * f), pf_half2(y[6] * f, y[7] * f));
                    if (pc == 0) qfac[128 * tile + rl] = __int_as_float((127 - up) << 23) * fabsf(a.scale_log2);
                }
                tc::fence_proxy_async();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(QFULL);
            }
            const float qf = qfac[128 * tile + row];
            const int p = live ? p0 + tok : -1;
            float m = -INFINITY, M = -INFINITY, l = 0.f, lr = 0.f;   // lr: the sum as the rounded P' have it (fp16 outputs)
            float root = 0.f;   // of 2^(M - m): as two factors it stays in range; 0 while there is no M
            // Warps w of the two tiles share a quarter of the SM and its exponential unit, so they take turns at it (named
            // barriers 1 + w and 5 + w, equal step counts): together they took 1,250 clocks for 64 keys each, in turn 750.
            bool had_turn = false, gave_turn = false;
            auto turn = [&](int id, bool wait) {
                if (tiles == 1) return;
                if (wait) asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory");
                else asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory");
            };
            auto my_turn = [&]() {
                turn(1 + 4 * tile + (warp & 3), true);
                had_turn = true;
            };
            auto turn_over = [&](int u) {
                if (tile == 0 || u + 1 < 2 * nk) turn(5 - 4 * tile + (warp & 3), false);
                gave_turn = true;
            };
            auto step = [&](int u) {
                const int j = u >> 1, half = u & 1;
                if (!(ok = pf_wait(SFULL(tile, half), j & 1))) return;
                tc::tc_fence_after();
                uint32_t s[64];
                tmem_ld64(tS + 64 * half, s);
                // the tile's scales were written before the K that the scores come from
                const PfPlaces &at = places[j & (PF_RING - 1)];
                const float4 k4 = *reinterpret_cast<const float4 *>(at.ks + 4 * half), w4 = *reinterpret_cast<const float4 *>(at.lv + 4 * half),
                             i4 = *reinterpret_cast<const float4 *>(at.iv + 4 * half);
                float f[4] = {k4.x * qf, k4.y * qf, k4.z * qf, k4.w * qf};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (f[i] < 0x1p-100f) f[i] = 0x1p-100f;   // hidden keys' -inf stays -inf in a block of scale 0; a NaN stays one
                float wv[4] = {w4.x, w4.y, w4.z, w4.w}, iw[4] = {i4.x, i4.y, i4.z, i4.w};
                const bool whole = at.whole >> (2 * tile + half) & 1u;
                tmem_ld64_done(s);
                if (!whole) {   // hide keys; a block that the row does not see at all loses its scales
                    const int k0 = at.k0 + 64 * half;
                    const uint32_t valid = at.valid >> (4 * half);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t see = pf_mask(a, p, k0 + 32 * c, valid >> (2 * c));
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(see >> i & 1u)) s[32 * c + i] = 0xFF800000u;
#pragma unroll
                        for (int h2 = 0; h2 < 2; ++h2)
                            if (!(see >> (16 * h2) & 0xFFFFu)) {
                                f[2 * c + h2] = 1.f;
                                wv[2 * c + h2] = 0.f;
                                iw[2 * c + h2] = 0.f;
                            }
                    }
                }
                float mx = -INFINITY, tx = -INFINITY;   // largest score, largest term
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float g = __uint_as_float(s[16 * i]);
#pragma unroll
                    for (int e = 1; e < 15; e += 2) g = max3(g, __uint_as_float(s[16 * i + e]), __uint_as_float(s[16 * i + e + 1]));
                    g = fmaxf(g, __uint_as_float(s[16 * i + 15])) * f[i];
                    mx = fmaxf(mx, g);
                    tx = fmaxf(tx, g + wv[i]);
                }
                float al = 1.f;
                if (mx > m + 11.f || tx > M + 11.f) {
                    const float m1 = fmaxf(m, mx + 3.f), M1 = fmaxf(M, tx + 3.f), f = pf_ex2(m - m1);
                    l *= f;
                    lr *= f;
                    m = m1;
                    if (M1 > -INFINITY) {
                        al = pf_ex2(M - M1);
                        M = M1;
                        root = pf_ex2(0.5f * (M - m));
                    }
                }
                if (__any_sync(0xffffffffu, al != 1.f) && u > 0) {   // O as it stands after the step before this one
                    if (!(ok = pf_wait(ODONE(tile), (u - 1) & 1))) return;
                    tc::tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld16_wait(tO + 16 * c, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                        tmem_st16(tO + 16 * c, o);
                    }
                }
                const float mu = m == -INFINITY ? 0.f : m, Mu = M == -INFINITY ? 0.f : M, least = -40.f - mu;
                bool weigh[4];   // fp16 outputs: the sum of the rounded P' takes part
                uint32_t pa[32];
                float exact[4];
                my_turn();
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t *pk = pa + 16 * c;
#pragma unroll
                    for (int h2 = 0; h2 < 2; ++h2) {
                        const int i = 2 * c + h2;
                        float cw = wv[i] - Mu;
                        weigh[i] = cw >= -4.f - mu;
                        iw[i] = root * iw[i] * root;
                        if (cw < least) cw = least, iw[i] = 0x1p40f;
                        const uint64_t f2 = f2_pack(f[i], f[i]), c2 = f2_pack(cw, cw);
                        uint64_t sum2 = 0;   // two zeros
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            float x, y;
                            f2_unpack(f2_fma(f2_pack(__uint_as_float(s[16 * i + e]), __uint_as_float(s[16 * i + e + 1])), f2, c2), x, y);
                            x = pf_ex2(x);
                            y = pf_ex2(y);
                            sum2 = f2_add(sum2, f2_pack(x, y));
                            pk[8 * h2 + e / 2] = pf_half2(x, y);
                        }
                        float sum, odd;
                        f2_unpack(sum2, sum, odd);
                        if constexpr (std::is_same<T, __half>::value) exact[i] = sum + odd;
                        l = fmaf(sum + odd, iw[i], l);
                    }
                    tmem_st16(tS + 64 * half + 16 * c, pk);
                }
                turn_over(u);
                tmem_st_wait();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(PFULL(tile, half));
                // fp16 outputs show what P' loses when it is rounded, so they are divided by the sum of the rounded P', whose error is
                // in part the same (one key that outweighs the others: all of it).  Not where vs is small beside the row's others: there
                // P' may be 0.
                if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float s0 = exact[i], s1 = 0.f;
                        if (weigh[i]) {
                            uint64_t r2 = 0;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&pa[8 * i + e]));
                                r2 = f2_add(r2, f2_pack(r.x, r.y));
                            }
                            f2_unpack(r2, s0, s1);
                        }
                        lr = fmaf(s0 + s1, iw[i], lr);
                    }
                }
            };
            if (tile == 1) turn(1 + (warp & 3), false);
            for (int u = 0; u < 2 * nk; ++u) {
                if (ok) step(u);
                if (!ok) {   // a wait ran out: the partner must not wait for this warp's turns
                    if (!had_turn) my_turn();
                    if (!gave_turn) turn_over(u);
                }
                had_turn = gave_turn = false;
            }
            const int64_t out_row = (int64_t)(first + tok) * a.c.heads * a.group + qh;
            float inv = 0.f;
            if (nk > 0 && ok) {
                ok = pf_wait(OFULL(tile), 0);
                tc::tc_fence_after();
                // O to units of 2^m, over the sum where this CTA has all of it
                float sum = shares == 1 ? l : 1.f;
                if constexpr (std::is_same<T, __half>::value) sum = shares == 1 ? lr : lr / l;
                inv = l == 0.f ? 0.f : root / sum * root;
                if (spoilt[warp] >> lane & 1u) inv = NAN;
            }
            const int64_t part = out_row * a.part_stride + share;
            if (ok && shares > 1 && nk > 0) {   // (an empty share has no accumulator)
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16_wait(tO + 16 * c, o);
                    if (live)
#pragma unroll
                        for (int i = 0; i < 16; i += 4)
                            kv_store4(a.part_o + part * D + 16 * c + i, make_float4(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv,
                                                                                    __uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv));
                }
            } else if (ok && shares == 1) {   // rows through the query's place in shared memory (no MMA reads it any more), out in whole lines
                uint8_t *mine = smem + SM::Q + tile * SM::OP + row * 128;
#pragma unroll 2
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = 0u;
                    if (nk > 0) tmem_ld16_wait(tO + 16 * c, o);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint4 w;
#pragma unroll
                        for (int i = 0; i < 8; i += 4)
                            kv_store4(reinterpret_cast<T *>(&w) + i,
                                      make_float4(__uint_as_float(o[8 * k + i]) * inv, __uint_as_float(o[8 * k + i + 1]) * inv,
                                                  __uint_as_float(o[8 * k + i + 2]) * inv, __uint_as_float(o[8 * k + i + 3]) * inv));
                        const int pcs = 2 * c + k;
                        *reinterpret_cast<uint4 *>(mine + (pcs >> 3) * 16384 + (((pcs & 7) ^ (row & 7)) << 4)) = w;
                    }
                }
                __syncwarp();
                rows_of([&](int, int rr, int tk, int g) {
                    const int rl = rr & 127;
                    if (rr < rn)
                        *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + ((int64_t)(first + tk) * a.c.heads * a.group + h * a.group + g) * D + 8 * pc) =
                            *reinterpret_cast<const uint4 *>(piece + rl * 128 + (((pc & 7) ^ (rl & 7)) << 4));
                });
            }
            if (live && ok) {
                if (shares > 1) a.part_ml[part] = make_float2(m, l);
                else if (a.lse) a.lse[out_row] = l == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m) + log2f(l)) * 0.69314718f;
            }
        }
    } else if (warp < 12) {   // ----------------------------------------------------------------------- converters
        asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
        // A thread takes 16 codes of a key at a time: 32 keys and 64 dims a pass.  Eight lanes then hold two keys, whose swizzled
        // rows fill all banks.
        constexpr int HV = D / 64, NL = 4 * HV;   // halves of the dims, passes
        const int ct = threadIdx.x - 256, ch = ct & 3, kr = ct >> 2, sw = kr & 7;
        const uint8_t *kc = a.c.k + (kr & 15) * D + 16 * ch, *vc = a.c.v + (kr & 15) * D + 16 * ch;
        const int d0 = kr * 128 + ((2 * ch ^ sw) << 4), d1 = kr * 128 + (((2 * ch + 1) ^ sw) << 4);
        uint4 xk[NL], xv[NL];   // a tile's codes, a tile ahead of their conversion
        auto load = [&](uint4 *x, const uint8_t *codes, int j) {
            const PfPlaces &at = places[j & (PF_RING - 1)];
            const uint32_t valid = at.valid >> (kr >> 4);
            const int64_t *where = at.at + (kr >> 4);
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                const int blk = u / HV * 2;
                x[u] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                if (valid >> blk & 1u) x[u] = ldg_stream16(codes + where[blk] * (KV_BLOCK * D) + u % HV * 64);
            }
        };
        auto store = [&](const uint4 *x, uint8_t *op) {
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                uint8_t *d = op + u % HV * 16384 + u / HV * 4096;
                *reinterpret_cast<uint4 *>(d + d0) = pf_convert8(x[u].x, x[u].y);
                *reinterpret_cast<uint4 *>(d + d1) = pf_convert8(x[u].z, x[u].w);
            }
            tc::fence_proxy_async();
            __syncwarp();
        };
        if (nk > 0 && (ok = pf_wait(ATFULL(0), 0))) {
            load(xk, kc, 0);
            load(xv, vc, 0);
            if (lane == 0) tc::mbar_arrive(ATEMPTY(0));
        }
        for (int j = 0; j < nk && ok; ++j) {
            const int s = j & 1, t = (j + 1) & (PF_RING - 1);
            if (j >= 2 && !(ok = pf_wait(KEMPTY(s), ((j >> 1) - 1) & 1))) break;
            store(xk, smem + SM::K + s * SM::OP);
            if (lane == 0) tc::mbar_arrive(KFULL(s));
            if (j + 1 < nk) {
                if (!(ok = pf_wait(ATFULL(t), ((j + 1) / PF_RING) & 1))) break;
                load(xk, kc, j + 1);
            }
            if (j >= 2 && !(ok = pf_wait(VEMPTY(s), ((j >> 1) - 1) & 1))) break;
            store(xv, smem + SM::V + s * SM::OP);
            if (lane == 0) tc::mbar_arrive(VFULL(s));
            if (j + 1 < nk) {
                load(xv, vc, j + 1);
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(ATEMPTY(t));
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 14) {   // ------------------------------------------------------ pages, some tiles ahead
            // first and last position of each tile's rows
            const int lo1 = p0 + (r0 + 128) / a.group, hi0 = tiles > 1 ? p0 + (r0 + 127) / a.group : phi;
            for (int j = 0; j < nk && ok; ++j) {
                const int s = j & (PF_RING - 1), k0 = key0(j), kb = k0 + 16 * lane;
                int pg = -1;
                // blocks that no row of the CTA sees count as blocks without a page
                if (lane < 8 && kb <= phi && (a.window == 0 || kb + 15 > plo - a.window || kb < a.n_sink)) pg = a.c.page_of(b, kb);
                const uint32_t valid = __ballot_sync(0xffffffffu, pg >= 0);
                float ks = 0.f, vs = 0.f;
                int64_t at = 0;
                if (pg >= 0) {
                    at = a.c.block(pg, h, kb);
                    ks = a.c.ks[at];
                    vs = a.c.vs[at];
                }
                const bool proper = vs <= FLT_MAX;
                for (uint32_t bad = __ballot_sync(0xffffffffu, !proper); bad; bad &= bad - 1)
#pragma unroll 1
                    for (int w = 0; w < PF_ROWS / 32; ++w) {
                        const uint32_t see = __ballot_sync(0xffffffffu, pf_mask(a, p0 + (r0 + 32 * w + lane) / a.group, k0 + 16 * (__ffs(bad) - 1), 1u));
                        if (lane == 0) spoilt[w] |= see;
                    }
                uint32_t whole = 0;
                if (lane < 4) {
                    const int t = lane >> 1, k = k0 + 64 * (lane & 1), lo = t ? lo1 : plo, hi = t ? phi : hi0;
                    whole = (valid >> (4 * (lane & 1)) & 15u) == 15u && k + 63 <= lo && (a.window == 0 || k > hi - a.window || k + 63 < a.n_sink);
                }
                whole = __ballot_sync(0xffffffffu, whole);
                if (j >= PF_AHEAD && !(ok = pf_wait(ATEMPTY((j - PF_AHEAD) & (PF_RING - 1)), ((j - PF_AHEAD) / PF_RING) & 1))) break;
                if (lane < 8) {
                    places[s].ks[lane] = ks;
                    places[s].lv[lane] = proper ? log2f(vs) : -INFINITY;
                    places[s].iv[lane] = 1.f / vs;
                    places[s].at[lane] = at;
                }
                if (lane == 8) {
                    places[s].k0 = k0;
                    places[s].valid = valid;
                    places[s].whole = whole;
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(ATFULL(s));
            }
        } else if (warp < 12 + tiles && nk > 0) {   // ------------------------------------------------- MMA issuers
            constexpr uint32_t id_qk = tc::idesc_f16(128, 64), id_pv = tc::idesc_f16(128, D) | (1u << 16);
            constexpr uint32_t OPD = SM::OP >> 4;   // one operand further in a descriptor
            const int t = warp - 12;
            const uint64_t dq = tc::sw128_desc(tc::smem_addr(smem + SM::Q + t * SM::OP)), dk = tc::sw128_desc(tc::smem_addr(smem + SM::K)),
                           dv = v_desc<D>(tc::smem_addr(smem + SM::V));
            const bool one = elect_one();
            auto qk = [&](int j, int half) {   // scores of 64 keys
                if (one) {
                    const uint64_t k = dk + (j & 1) * OPD + half * 512;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        tc::mma_f16(128u * t + 64u * half, dq + (i >> 2) * 1024 + (i & 3) * 2, k + (i >> 2) * 1024 + (i & 3) * 2, id_qk, i > 0);
                    tc::mma_commit(SFULL(t, half));
                    if (half) tc::mma_commit(KEMPTY(j & 1));   // the last of this tile to read it
                }
                __syncwarp();
            };
            ok = pf_wait(QFULL, 0) && pf_wait(KFULL(0), 0);
            tc::tc_fence_after();
            if (ok) {
                qk(0, 0);
                qk(0, 1);
            }
            for (int u = 0; u < 2 * nk && ok; ++u) {
                const int j = u >> 1, half = u & 1;
                if (half == 0)
                    ok = (j + 1 == nk || pf_wait(KFULL((j + 1) & 1), ((j + 1) >> 1) & 1)) && pf_wait(VFULL(j & 1), (j >> 1) & 1);
                if (!(ok = ok && pf_wait(PFULL(t, half), j & 1))) break;
                tc::tc_fence_after();
                if (one) {
                    const uint64_t v = dv + (j & 1) * OPD + half * 512;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma_f16_ts(256u + 128u * t, 128u * t + 64u * half + 8u * i, v + 128 * i, id_pv, u > 0 || i > 0);
                    tc::mma_commit(ODONE(t));
                    if (half) tc::mma_commit(VEMPTY(j & 1));
                    if (u == 2 * nk - 1) tc::mma_commit(OFULL(t));
                }
                __syncwarp();
                if (j + 1 < nk) qk(j + 1, half);
            }
            // nothing of this CTA is in flight when tensor memory is given back
            if (one) tc::mma_commit(DRAIN);
            __syncwarp();
            ok = pf_wait(DRAIN, 0) && ok;
        }
    }
    if (!ok && a.status) atomicOr(a.status, STATUS_TIMEOUT);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == 12) tc::tmem_dealloc(tmem, 512);
    if (a.after_few) griddep_wait();   // whoever waits for this kernel's end waits for both
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
    return launch_k(a.after_few, kern, dim3((uint32_t)((uint64_t)a.pf_items * a.c.heads * a.pf_splits)), PF_THREADS, PfSmem<D>::BYTES, st, a, min_rows);
}

cudaError_t launch_kv_prefill(const KvAttnArgs &a, int dtype, int head_dim, int min_rows, cudaStream_t st) {
    if (dtype == V3G_F16) return head_dim == 64 ? launch_pf<__half, 64>(a, min_rows, st) : launch_pf<__half, 128>(a, min_rows, st);
    return head_dim == 64 ? launch_pf<__nv_bfloat16, 64>(a, min_rows, st) : launch_pf<__nv_bfloat16, 128>(a, min_rows, st);
}

}  // namespace v3g
