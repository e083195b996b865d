// Beam search selection: of each group's beams x vocab continuations, the `beams` best.
//
//   score(k, t) = (logit[k][t] - lse_k) + scores[k],   lse_k = max + log(sum exp(logit - max))
//
// The logits are read once (4 bytes and an exponential per element: HBM bounds it).  Inside a beam the order of the
// scores is the order of the logits, so the first kernel needs no lse: a CTA streams a slice of one beam's logits, each
// thread keeping the maximum and the sum of exponentials of its own, and writes the slice's `beams` best as 64-bit keys
// (value, then lower index).  The second kernel joins the sums of a beam, scores the beams x slices x beams keys and
// selects again.  Both selections are exact: the `beams`-th largest of some group maxima bounds the answer from below; the few
// threads whose maximum reaches it read their logits again, and what is at or above it is collected and ranked by
// counting; where too much is (long ties, sorted logits), `beams` rounds of a block maximum take its place.
#include <cfloat>

#include "v3g_internal.h"
#include "v3g_kv.cuh"

namespace v3g {

constexpr int BEAM_THREADS = 256;
constexpr int BEAM_BUF = 256;   // collected keys that are ranked by counting

typedef unsigned long long u64;

__device__ __forceinline__ float key_float(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

__device__ __forceinline__ u64 u64_max(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 shfl_xor64(u64 x, int o) { return __shfl_xor_sync(0xffffffffu, x, o); }

struct BeamShared {
    u64 buf[BEAM_BUF];
    u64 red[BEAM_THREADS / 32];
    float group[32];
    u64 best;
    int count;
};

// The `beams`-th largest of the maxima of G groups of threads, G = 8, 16 or 32 >= beams: at least `beams` values of the
// block are at or above it.
__device__ __forceinline__ int beam_groups(int beams) { return beams <= 8 ? 8 : (beams <= 16 ? 16 : 32); }
__device__ __forceinline__ float beam_bound(BeamShared &sm, float v, int beams) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = beam_groups(beams), per = groups / 8;   // groups of a warp
    for (int o = 1; o < 32 / per; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (threadIdx.x == 0) sm.count = 0;
    if (lane % (32 / per) == 0) sm.group[warp * per + lane / (32 / per)] = v;
    __syncthreads();
    v = lane < groups ? sm.group[lane] : -INFINITY;
    int rank = 0;
    for (int k = 0; k < groups; k += 8)
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float o = __shfl_sync(0xffffffffu, v, k + u);
            rank += o > v || (o == v && k + u < lane);
        }
    const uint32_t at = __ballot_sync(0xffffffffu, lane < groups && rank == beams - 1);
    return __shfl_sync(0xffffffffu, v, __ffs(at) - 1);
}

// the block's largest key, to every thread
__device__ __forceinline__ u64 beam_block_max(BeamShared &sm, u64 k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) k = u64_max(k, shfl_xor64(k, o));
    if ((threadIdx.x & 31) == 0) sm.red[threadIdx.x >> 5] = k;
    __syncthreads();
    k = sm.red[0];
#pragma unroll
    for (int w = 1; w < BEAM_THREADS / 32; ++w) k = u64_max(k, sm.red[w]);
    __syncthreads();
    return k;
}

// The `beams` largest of the keys that each(f) hands to f (distinct keys, the same ones at every call), in order, to
// emit(rank, key); missing ones are emitted as 0.  bound: a value that at least `beams` of the keys reach, or the
// block holds fewer.
template <class Each, class Emit>
__device__ __forceinline__ void beam_best(BeamShared &sm, int beams, uint32_t bound, Each each, Emit emit) {
    each([&](u64 k) {
        if ((uint32_t)(k >> 32) >= bound) {
            const int at = atomicAdd(&sm.count, 1);
            if (at < BEAM_BUF) sm.buf[at] = k;
        }
    });
    __syncthreads();
    const int n = sm.count;
    if (n <= BEAM_BUF) {
        if ((int)threadIdx.x < n) {
            const u64 k = sm.buf[threadIdx.x];
            int rank = 0;
#pragma unroll 8
            for (int i = 0; i < n; ++i) rank += sm.buf[i] > k;
            if (rank < beams) emit(rank, k);
        }
        if ((int)threadIdx.x >= n && (int)threadIdx.x < beams) emit((int)threadIdx.x, 0ull);
        return;
    }
    u64 last = ~0ull;
    for (int j = 0; j < beams; ++j) {
        u64 k = 0;
        each([&](u64 x) {
            if (x < last) k = u64_max(k, x);
        });
        last = beam_block_max(sm, k);
        if (threadIdx.x == 0) emit(j, last);
        if (last == 0) last = 1;   // keys are larger than 1: the rest stays empty
    }
}

template <typename T>
__device__ __forceinline__ float beam_value(T x);
template <>
__device__ __forceinline__ float beam_value<float>(float x) { return x; }
template <>
__device__ __forceinline__ float beam_value<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float beam_value<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ float beam_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// `slice` consecutive logits of a beam (a multiple of BEAM_STEP): the threads' running maxima and sums, then the best
constexpr int BEAM_EPT = 16, BEAM_STEP = BEAM_THREADS * BEAM_EPT;
template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 6) k_beam_slice(const T *logits, int64_t ld, int vocab, int slice, int beams, bool vec, u64 *keys,
                                                               float2 *sums) {
    __shared__ BeamShared sm;
    __shared__ float red[BEAM_THREADS / 32];
    griddep_launch();
    constexpr int W = 16 / sizeof(T), NL = BEAM_EPT / W;          // elements of a 16-byte load, loads of a step
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.y;
    const int i0 = blockIdx.x * slice, steps = (min(slice, vocab - i0) + BEAM_STEP - 1) / BEAM_STEP;
    const T *p = logits + row * ld;
    // element e of the thread's share of a step: 16-byte pieces where the step is whole and aligned, else every 256th
    auto whole = [&](int step) { return vec && i0 + (step + 1) * BEAM_STEP <= vocab; };
    auto index = [&](int step, int e) {
        return i0 + step * BEAM_STEP + (whole(step) ? (e / W) * (BEAM_THREADS * W) + tid * W + e % W : e * BEAM_THREADS + tid);
    };
    auto load = [&](int step, float(&x)[BEAM_EPT]) {
        if (whole(step)) {
            uint4 u[NL];
#pragma unroll
            for (int i = 0; i < NL; ++i) u[i] = ldg_stream16(p + (i0 + step * BEAM_STEP + i * (BEAM_THREADS * W) + tid * W));
#pragma unroll
            for (int e = 0; e < BEAM_EPT; ++e) x[e] = beam_value(reinterpret_cast<const T *>(&u[e / W])[e % W]);
        } else {
#pragma unroll
            for (int e = 0; e < BEAM_EPT; ++e) {
                const int i = i0 + step * BEAM_STEP + e * BEAM_THREADS + tid;
                x[e] = i < vocab ? beam_value(p[i]) : -INFINITY;
            }
        }
    };
    // a power that ends at 2^-200 = 0 where the difference is no number: hidden logits, NaN, an infinite maximum
    auto power = [](float a, float b) { return beam_ex2(fmaxf((a - b) * 1.44269504f, -200.f)); };
    float mine = -INFINITY, sum = 0.f;                            // of the thread's logits: maximum, sum of e^(x - maximum)
    for (int step = 0; step < steps; ++step) {
        float x[BEAM_EPT];
        load(step, x);
        float m = mine;
#pragma unroll
        for (int e = 0; e < BEAM_EPT; ++e) m = fmaxf(m, x[e]);    // NaN logits are passed over
        // in one product where that stays in range (logits at the type's lowest value would leave it) and no NaN came in
        float add = 0.f;
        const bool plain = fabsf(m) < 1e38f;
        if (plain) {
            const float shift = -m * 1.44269504f;
#pragma unroll
            for (int e = 0; e < BEAM_EPT; ++e) add += beam_ex2(fmaf(x[e], 1.44269504f, shift));
        }
        if (!plain || add != add) {
            add = 0.f;
#pragma unroll
            for (int e = 0; e < BEAM_EPT; ++e) add += power(x[e], m);
        }
        sum = sum * power(mine, m) + add;
        mine = m;
    }
    const float bound = beam_bound(sm, mine, beams);
    float top = sm.group[lane];
    if (lane >= beam_groups(beams)) top = -INFINITY;
    top = warp_max(top);                                          // the slice's maximum
    sum = warp_sum(sum * power(mine, top));
    if (lane == 0) red[warp] = sum;
    const int64_t at = row * gridDim.x + blockIdx.x;
    const float lo = fmaxf(bound, -FLT_MAX);                      // finite ones only
    beam_best(
        sm, beams, float_key(bound),
        [&](auto f) {   // few threads hold one of the best: they read theirs again
            if (mine >= lo)
                for (int step = 0; step < steps; ++step) {
                    float x[BEAM_EPT];
                    load(step, x);
#pragma unroll
                    for (int e = 0; e < BEAM_EPT; ++e)
                        if (x[e] >= lo && x[e] <= FLT_MAX) f(((u64)float_key(x[e]) << 32) | (0xFFFFFFFFu - (uint32_t)index(step, e)));
                }
        },
        [&](int rank, u64 k) { keys[at * beams + rank] = k; });
    if (tid == 0) {   // red was written before beam_best's barrier
        sum = red[0];
        for (int w = 1; w < BEAM_THREADS / 32; ++w) sum += red[w];
        sums[at] = make_float2(top, sum);
    }
}

struct BeamArgs {
    u64 *keys;          // the slices' best; the join scores them in place
    const float2 *sums;
    const float *scores;
    const uint8_t *finished;
    int beams, slices, vocab, eos;
    int32_t *tokens, *parents;
    float *scores_out;
    uint8_t *finished_out;
};

__global__ void __launch_bounds__(BEAM_THREADS) k_beam_join(const __grid_constant__ BeamArgs a) {
    __shared__ BeamShared sm;
    __shared__ u64 only[V3G_BEAM_MAX];
    __shared__ bool done[V3G_BEAM_MAX];
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, K = a.beams, per = a.slices * K;
    const int64_t g0 = (int64_t)blockIdx.x * K;
    // a warp takes a beam: its logsumexp, then the scores of its slices' best
    uint32_t top = 0;
    for (int k = warp; k < K; k += BEAM_THREADS / 32) {
        const float2 *p = a.sums + (g0 + k) * a.slices;
        u64 *keys = a.keys + (g0 + k) * per;
        const float run_k = a.scores[g0 + k];
        const bool done_k = a.finished && a.finished[g0 + k];
        u64 ahead[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ahead[i] = lane + 32 * i < per ? keys[lane + 32 * i] : 0ull;
        float m = -INFINITY;
        for (int i = lane; i < a.slices; i += 32) m = fmaxf(m, p[i].x);
        m = warp_max(m);
        float s = 0.f;
        for (int i = lane; i < a.slices; i += 32) {
            const float2 v = p[i];
            if (v.x > -INFINITY) s += v.y * beam_ex2((v.x - m) * 1.44269504f);
        }
        const float lse = m + logf(warp_sum(s));
        auto score = [&](u64 key) -> u64 {
            const float y = (key_float((uint32_t)(key >> 32)) - lse) + run_k;
            if (done_k || !key || !(y > -INFINITY && y < INFINITY)) return 0ull;
            return ((u64)float_key(y) << 32) | (0xFFFFFFFFu - ((uint32_t)k * (uint32_t)a.vocab + (0xFFFFFFFFu - (uint32_t)key)));
        };
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32 * i < per) {
                const u64 y = score(ahead[i]);
                keys[lane + 32 * i] = y;
                top = max(top, (uint32_t)(y >> 32));
            }
        for (int i = lane + 128; i < per; i += 32) {
            const u64 y = score(keys[i]);
            keys[i] = y;
            top = max(top, (uint32_t)(y >> 32));
        }
        // a finished beam's one continuation
        const bool goes_on = done_k && a.eos >= 0 && run_k > -INFINITY && run_k < INFINITY;
        if (lane == 0) {
            done[k] = done_k;
            only[k] = goes_on ? ((u64)float_key(run_k) << 32) | (0xFFFFFFFFu - ((uint32_t)k * (uint32_t)a.vocab + (uint32_t)a.eos)) : 0ull;
            if (goes_on) top = max(top, float_key(run_k));
        }
    }
    auto each = [&](auto f) {   // every thread its own keys again
        for (int k = warp; k < K; k += BEAM_THREADS / 32) {
            const u64 *keys = a.keys + (g0 + k) * per;
            for (int i = lane; i < per; i += 32) {
                const u64 y = keys[i];
                if (y) f(y);
            }
            if (lane == 0 && only[k]) f(only[k]);
        }
    };
    const float bound = beam_bound(sm, top ? key_float(top) : -INFINITY, K);
    beam_best(sm, K, float_key(bound), each, [&](int rank, u64 k) {
        const int64_t at = g0 + rank;
        if (k) {
            const uint32_t flat = 0xFFFFFFFFu - (uint32_t)k;
            const int parent = (int)(flat / (uint32_t)a.vocab), token = (int)(flat % (uint32_t)a.vocab);
            a.tokens[at] = token;
            a.parents[at] = parent;
            a.scores_out[at] = key_float((uint32_t)(k >> 32));
            a.finished_out[at] = done[parent] || token == a.eos;
        } else {
            a.tokens[at] = a.eos < 0 ? 0 : a.eos;
            a.parents[at] = rank;
            a.scores_out[at] = -INFINITY;
            a.finished_out[at] = 1;
        }
    });
}

struct BeamPlan {
    int slice, slices;
    size_t keys, bytes;
};
// Long slices cost less beside their data, short ones spread small steps over the SMs: the shortest that leaves at most 32
// CTAs an SM.
static BeamPlan beam_plan(uint64_t rows, uint32_t beams, uint32_t vocab) {
    BeamPlan p;
    p.slice = BEAM_STEP;
    while (p.slice < 8 * BEAM_STEP && rows * ((vocab + p.slice - 1) / p.slice) > 148 * 32) p.slice *= 2;
    p.slices = (int)(((uint64_t)vocab + p.slice - 1) / p.slice);
    p.keys = (rows * p.slices * sizeof(float2) + 255) & ~(size_t)255;
    p.bytes = p.keys + rows * p.slices * beams * sizeof(u64);
    return p;
}

template <typename T>
static cudaError_t launch_slices(const void *logits, int64_t ld, int vocab, int beams, const BeamPlan &p, uint32_t rows, u64 *keys,
                                 float2 *sums, cudaStream_t st) {
    const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld * sizeof(T) % 16 == 0;
    return launch_k(false, k_beam_slice<T>, dim3(p.slices, rows), BEAM_THREADS, 0, st, static_cast<const T *>(logits), ld, vocab, p.slice,
                    beams, vec, keys, sums);
}

}  // namespace v3g

using namespace v3g;

extern "C" size_t v3g_beam_select_work_size(uint32_t groups, uint32_t beams, uint32_t vocab) {
    if (groups == 0 || beams == 0 || beams > V3G_BEAM_MAX || vocab == 0) return 0;
    return beam_plan((uint64_t)groups * beams, beams, vocab).bytes;
}

extern "C" int v3g_beam_select(const void *dev_logits, int dtype, uint32_t groups, uint32_t beams, uint32_t vocab, uint64_t ld,
                               const float *dev_scores, const uint8_t *dev_finished, int32_t eos_id, int32_t *tokens, int32_t *parents,
                               float *scores_out, uint8_t *finished_out, void *dev_work, size_t work_bytes, void *stream) {
    if (dtype != V3G_F32 && dtype != V3G_F16 && dtype != V3G_BF16) return v3g_fail(V3G_E_DTYPE, "v3g_beam_select: fp32, fp16 or bf16 logits");
    if (beams == 0 || beams > V3G_BEAM_MAX) return v3g_fail(V3G_E_LIMIT, "v3g_beam_select: 1 to 32 beams");
    if (vocab == 0 || ld < vocab || (int64_t)vocab <= eos_id) return v3g_fail(V3G_E_ARG, "v3g_beam_select: vocab must be > 0, <= ld and > eos_id");
    if (vocab > 0x40000000u / beams) return v3g_fail(V3G_E_LIMIT, "v3g_beam_select: beams x vocab must stay within 2^30");
    if (groups == 0) return V3G_OK;
    if ((uint64_t)groups * beams > 65535u) return v3g_fail(V3G_E_LIMIT, "v3g_beam_select: at most 65535 beams in all");
    if (!dev_logits || !dev_scores || !tokens || !parents || !scores_out || !finished_out)
        return v3g_fail(V3G_E_ARG, "v3g_beam_select: null pointer");
    if (reinterpret_cast<uintptr_t>(dev_logits) % (dtype == V3G_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(dev_scores) % 4 ||
        reinterpret_cast<uintptr_t>(tokens) % 4 || reinterpret_cast<uintptr_t>(parents) % 4 || reinterpret_cast<uintptr_t>(scores_out) % 4)
        return v3g_fail(V3G_E_ALIGN, "v3g_beam_select: misaligned pointer");
    const uint32_t rows = groups * beams;
    const BeamPlan p = beam_plan(rows, beams, vocab);
    if (!dev_work || work_bytes < p.bytes) return v3g_fail(V3G_E_SIZE, "v3g_beam_select: workspace too small");
    if (reinterpret_cast<uintptr_t>(dev_work) % 256) return v3g_fail(V3G_E_ALIGN, "v3g_beam_select: the workspace needs 256-byte alignment");
    BeamArgs a = {};
    float2 *sums = static_cast<float2 *>(dev_work);
    u64 *keys = reinterpret_cast<u64 *>(static_cast<uint8_t *>(dev_work) + p.keys);
    a.keys = keys;
    a.sums = sums;
    a.scores = dev_scores;
    a.finished = dev_finished;
    a.beams = (int)beams;
    a.slices = p.slices;
    a.vocab = (int)vocab;
    a.eos = eos_id;
    a.tokens = tokens;
    a.parents = parents;
    a.scores_out = scores_out;
    a.finished_out = finished_out;
    const cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (dtype == V3G_F32) e = launch_slices<float>(dev_logits, (int64_t)ld, (int)vocab, (int)beams, p, rows, keys, sums, st);
    else if (dtype == V3G_F16) e = launch_slices<__half>(dev_logits, (int64_t)ld, (int)vocab, (int)beams, p, rows, keys, sums, st);
    else e = launch_slices<__nv_bfloat16>(dev_logits, (int64_t)ld, (int)vocab, (int)beams, p, rows, keys, sums, st);
    if (e == cudaSuccess) e = launch_k(true, k_beam_join, dim3(groups), BEAM_THREADS, 0, st, a);
    return e == cudaSuccess ? V3G_OK : v3g_fail(V3G_E_CUDA, std::string("v3g_beam_select: ") + cudaGetErrorString(e));
}
