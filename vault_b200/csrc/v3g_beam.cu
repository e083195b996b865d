// Beam search selection: of each group's beams x vocab continuations, the `beams` best.
//
//   score(k, t) = (logit[k][t] - lse_k) + scores[k],   lse_k = max + log(sum exp(logit - max))
//
// The logits are read once (4 bytes and an exponential per element: HBM bounds it).  Inside a beam the order of the
// scores is the order of the logits, so the first kernel needs no lse: a CTA streams a slice of one beam's logits, each
// thread keeping the maximum and the sum of exponentials of its own, and writes the slice's `beams` best as 64-bit keys
// (value, then lower index) and the largest logit that it leaves out.  The second kernel joins the sums of a beam and selects
// among the slices' best, reading only those of the slices whose maximum can be among the answers.  Both selections are exact:
// the `beams`-th largest of 64 group maxima bounds the answer from below; the few threads whose maximum reaches it have their
// logits read again, and what is at or above it is collected and ranked by counting; where too much is (long ties), `beams`
// rounds of a block maximum take its place.
//
// Equal scores go to the lower index, but different logits may round to one score, and a slice chose by logit.  What it left
// out scores at most what the last place is worth, so only places of that score can be wrong, and only if a left-out logit has
// it too.  Then those places are given out again, over the logits themselves in the order of their indices.
//
// 48 x 8 beams over 151,936 logits (233 MB) take 44 us in fp32 (5.3 TB/s; the join starts under the slices) and
// 35 us in bf16, where loads and powers of a CTA alternate; one request of 4 beams 7.0 us.
#include <cfloat>

#include "v3g_internal.h"
#include "v3g_kv.cuh"

namespace v3g {

constexpr int BEAM_THREADS = 256;
constexpr int BEAM_BUF = 256;    // collected keys that are ranked by counting
constexpr int BEAM_GROUPS = 64;  // groups of threads whose maxima give the bound: more than V3G_BEAM_MAX
constexpr int BEAM_LIST = 512;   // slices the join picks its keys from

typedef unsigned long long u64;

__device__ __forceinline__ float key_float(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

__device__ __forceinline__ u64 u64_max(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 shfl_xor64(u64 x, int o) { return __shfl_xor_sync(0xffffffffu, x, o); }

struct BeamShared {
    u64 buf[BEAM_BUF];
    u64 red[BEAM_THREADS / 32];
    float4 group[BEAM_GROUPS / 4];
    float bound, next;           // next: what the best leave out
    int count, listed;
};

// The `beams`-th largest of the maxima of the block's groups of threads: at least `beams` values of the block are at or
// above it.  With 64 groups few others are: 8 beams find 9 values in a slice on average, where 8 groups (one needed of
// each) let 22 through.
__device__ __forceinline__ float beam_bound(BeamShared &sm, float v, int beams) {
    constexpr int PER = BEAM_THREADS / BEAM_GROUPS, SHARE = BEAM_GROUPS / PER;
    const int tid = threadIdx.x, mine = tid / PER, first = tid % PER * SHARE;
#pragma unroll
    for (int o = 1; o < PER; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (tid == 0) sm.count = sm.listed = 0;
    if (first == 0) reinterpret_cast<float *>(sm.group)[mine] = v;
    __syncthreads();
    // the rank of the group's maximum, its comparisons shared out over the group; equal ones rank by place
    int rank = 0;
#pragma unroll
    for (int k = 0; k < SHARE; k += 4) {
        const float4 o = sm.group[(first + k) / 4];
        rank += o.x > v || (o.x == v && first + k < mine);
        rank += o.y > v || (o.y == v && first + k + 1 < mine);
        rank += o.z > v || (o.z == v && first + k + 2 < mine);
        rank += o.w > v || (o.w == v && first + k + 3 < mine);
    }
#pragma unroll
    for (int o = 1; o < PER; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (rank == beams - 1) sm.bound = v;
    __syncthreads();
    return sm.bound;
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
constexpr int BEAM_EPT = 32, BEAM_STEP = BEAM_THREADS * BEAM_EPT;
template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 4) k_beam_slice(const T *logits, int64_t ld, int vocab, int slice, int beams, bool vec, u64 *keys,
                                                               float4 *sums) {
    __shared__ BeamShared sm;
    __shared__ float red[BEAM_THREADS / 32];
    __shared__ uint32_t list[BEAM_THREADS];
    griddep_launch();
    constexpr int W = 16 / sizeof(T), NL = BEAM_EPT / W;          // elements of a 16-byte load, loads of a step
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.y;
    const int i0 = blockIdx.x * slice, steps = (min(slice, vocab - i0) + BEAM_STEP - 1) / BEAM_STEP;
    const T *p = logits + row * ld;
    // element e of thread t's share of a step: 16-byte pieces where the step is whole and aligned, else every 256th
    auto whole = [&](int step) { return vec && i0 + (step + 1) * BEAM_STEP <= vocab; };
    auto index = [&](int step, int t, int e) {
        return i0 + step * BEAM_STEP + (whole(step) ? (e / W) * (BEAM_THREADS * W) + t * W + e % W : e * BEAM_THREADS + t);
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
    // of the thread's logits: their maximum, the step that has it, the other steps' maximum, the sum of e^(x - maximum)
    float mine = -INFINITY, others = -INFINITY, sum = 0.f;
    int best = 0;
    for (int step = 0; step < steps; ++step) {
        float x[BEAM_EPT];
        load(step, x);
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < BEAM_EPT; ++e) m = fmaxf(m, x[e]);    // NaN logits are passed over
        others = fmaxf(others, fminf(mine, m));
        if (m > mine) best = step;
        m = fmaxf(mine, m);
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
    const float bound = beam_bound(sm, mine, beams + 1);
    const float *group = reinterpret_cast<const float *>(sm.group);
    float top = fmaxf(group[lane], group[lane + 32]);
    top = warp_max(top);                                          // the slice's maximum
    sum = warp_sum(sum * power(mine, top));
    if (lane == 0) red[warp] = sum;
    const int64_t at = row * gridDim.x + blockIdx.x;
    const float lo = fmaxf(bound, -FLT_MAX);                      // finite ones only
    // The threads that hold one of the best, with the step to look at, or all of them (the sign bit).  A warp reads such a
    // share again: were each thread to read its own, most warps would go through 32 elements a step for one thread's sake.
    if (mine >= lo) list[atomicAdd(&sm.listed, 1)] = (others >= lo ? 0x80000000u : (uint32_t)best << 8) | tid;
    __syncthreads();
    const int listed = sm.listed;
    beam_best(
        sm, beams + 1, float_key(bound),
        [&](auto f) {
            for (int k = tid / BEAM_EPT; k < listed; k += BEAM_THREADS / BEAM_EPT) {
                const uint32_t l = list[k];
                const int first = (int)(l >> 31 ? 0 : l >> 8), last = l >> 31 ? steps : first + 1;
                for (int step = first; step < last; ++step) {
                    const int i = index(step, l & 255, tid % BEAM_EPT);
                    const float x = i < vocab ? beam_value(p[i]) : -INFINITY;
                    if (x >= lo && x <= FLT_MAX) f(((u64)float_key(x) << 32) | (0xFFFFFFFFu - (uint32_t)i));
                }
            }
        },
        [&](int rank, u64 k) {
            if (rank < beams) keys[at * beams + rank] = k;
            else sm.next = k ? key_float((uint32_t)(k >> 32)) : -INFINITY;
        });
    __syncthreads();
    if (tid == 0) {   // red was written before beam_best's barrier
        sum = red[0];
        for (int w = 1; w < BEAM_THREADS / 32; ++w) sum += red[w];
        sums[at] = make_float4(top, sum, sm.next, 0.f);
    }
}

struct BeamArgs {
    const void *logits;
    int64_t ld;
    const u64 *keys;    // the slices' best, largest first
    const float4 *sums; // their largest logit, sum, and the largest logit that is not among the best
    const float *scores;
    const uint8_t *finished;
    int beams, slice, slices, vocab, eos;
    int32_t *tokens, *parents;
    float *scores_out;
    uint8_t *finished_out;
};

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS) k_beam_join(const __grid_constant__ BeamArgs a) {
    __shared__ BeamShared sm;
    __shared__ u64 only[V3G_BEAM_MAX];
    __shared__ float lse[V3G_BEAM_MAX], run[V3G_BEAM_MAX], given[V3G_BEAM_MAX];
    __shared__ bool done[V3G_BEAM_MAX];
    __shared__ int list[BEAM_LIST], found[BEAM_THREADS / 32];
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, K = a.beams, n = a.slices * K;
    const int64_t g0 = (int64_t)blockIdx.x * K;
    const float4 *sums = a.sums + g0 * a.slices;
    const u64 *keys = a.keys + g0 * a.slices * K;
    const bool few = n * K <= 4 * BEAM_THREADS;   // every key fits the threads' registers
    u64 ahead[4];
    if (few)
#pragma unroll
        for (int i = 0; i < 4; ++i) ahead[i] = tid + BEAM_THREADS * i < n * K ? keys[tid + BEAM_THREADS * i] : 0ull;
    // a warp takes a beam: its logsumexp
    for (int k = warp; k < K; k += BEAM_THREADS / 32) {
        const float4 *p = sums + (int64_t)k * a.slices;
        const float run_k = a.scores[g0 + k];
        const bool done_k = a.finished && a.finished[g0 + k];
        float m = -INFINITY;
        for (int i = lane; i < a.slices; i += 32) m = fmaxf(m, p[i].x);
        m = warp_max(m);
        float s = 0.f;
        for (int i = lane; i < a.slices; i += 32) {
            const float4 v = p[i];
            if (v.x > -INFINITY) s += v.y * beam_ex2((v.x - m) * 1.44269504f);
        }
        s = m + logf(warp_sum(s));
        if (lane == 0) {
            // a finished beam has one continuation
            const bool goes_on = done_k && a.eos >= 0 && run_k > -INFINITY && run_k < INFINITY;
            done[k] = done_k;
            run[k] = run_k;
            lse[k] = done_k ? NAN : s;   // and no others
            only[k] = goes_on ? ((u64)float_key(run_k) << 32) | (0xFFFFFFFFu - ((uint32_t)k * (uint32_t)a.vocab + (uint32_t)a.eos)) : 0ull;
        }
    }
    __syncthreads();
    // Scores that are no number or infinite stand for nothing.  A slice's best key comes first, and its value is the
    // slice's maximum (if that is finite): the bound needs no keys.
    auto score = [&](int k, float x) -> float {
        const float y = (x - lse[k]) + run[k];
        return y > -INFINITY && y < INFINITY ? y : -INFINITY;
    };
    // consecutive slices go to different groups of the bound: often one beam alone has candidates
    const int mine = tid % (BEAM_THREADS / BEAM_GROUPS) * BEAM_GROUPS + tid / (BEAM_THREADS / BEAM_GROUPS);
    float top = tid < K && only[tid] ? run[tid] : -INFINITY;
    float left = -INFINITY;   // the best score that a slice left out
    for (int i = mine; i < n; i += BEAM_THREADS) {
        const float4 v = sums[i];
        top = fmaxf(top, score(i / a.slices, v.x));
        left = fmaxf(left, score(i / a.slices, v.z));
    }
    const float bound = beam_bound(sm, top, K), lo = fmaxf(bound, -FLT_MAX);
    if (!few && top >= lo)
        for (int i = mine; i < n; i += BEAM_THREADS)
            if (score(i / a.slices, sums[i].x) >= lo) {
                const int at = atomicAdd(&sm.listed, 1);
                if (at < BEAM_LIST) list[at] = i;
            }
    if (!few) __syncthreads();
    const bool all = sm.listed > BEAM_LIST;   // long ties: every slice
    const int picked = few ? 0 : (all ? n : sm.listed);
    auto each = [&](auto f) {
        auto pick = [&](int k, u64 key) {
            const float y = key ? score(k, key_float((uint32_t)(key >> 32))) : -INFINITY;
            if (y >= lo) f(((u64)float_key(y) << 32) | (0xFFFFFFFFu - ((uint32_t)k * (uint32_t)a.vocab + (0xFFFFFFFFu - (uint32_t)key))));
        };
        if (few)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (ahead[i]) pick((tid + BEAM_THREADS * i) / (a.slices * K), ahead[i]);
        for (int64_t i = tid; i < (int64_t)picked * K; i += BEAM_THREADS) {
            const int at = all ? (int)(i / K) : list[(int)i / K];
            pick(at / a.slices, keys[(int64_t)at * K + i % K]);
        }
        if (tid < K && only[tid]) f(only[tid]);
    };
    auto put = [&](int rank, int parent, int token, float y) {
        const int64_t at = g0 + rank;
        a.tokens[at] = token;
        a.parents[at] = parent;
        a.scores_out[at] = y;
        a.finished_out[at] = done[parent] || token == a.eos;
    };
    beam_best(sm, K, float_key(bound), each, [&](int rank, u64 k) {
        const int64_t at = g0 + rank;
        given[rank] = k ? key_float((uint32_t)(k >> 32)) : INFINITY;   // an empty place: nothing was left out
        if (k) {
            const uint32_t flat = 0xFFFFFFFFu - (uint32_t)k;
            put(rank, (int)(flat / (uint32_t)a.vocab), (int)(flat % (uint32_t)a.vocab), given[rank]);
        } else {
            a.tokens[at] = a.eos < 0 ? 0 : a.eos;
            a.parents[at] = rank;
            a.scores_out[at] = -INFINITY;
            a.finished_out[at] = 1;
        }
    });
    __syncthreads();
    const float last = given[K - 1];
    if (!__syncthreads_or(left >= last)) return;
    // The places worth `last`, to the lowest indices that have this score.  A thread looks at PER consecutive logits at a time.
    constexpr int PER = 16;
    int rank = 0;
    while (given[rank] > last) ++rank;
    for (int k = 0; k < K && rank < K; ++k) {
        if (done[k]) {
            if (only[k] && run[k] == last) {
                if (tid == 0) put(rank, k, a.eos, last);
                ++rank;
            }
            continue;
        }
        const T *p = static_cast<const T *>(a.logits) + (g0 + k) * a.ld;
        for (int s = 0; s < a.slices && rank < K; ++s) {
            if (!(score(k, sums[k * a.slices + s].x) >= last)) continue;
            const int end = min((s + 1) * a.slice, a.vocab);
            for (int i0 = s * a.slice; i0 < end && rank < K; i0 += BEAM_THREADS * PER) {
                const int first = i0 + tid * PER;
                uint32_t has = 0;
                for (int e = 0; e < PER; ++e)
                    if (first + e < end && score(k, beam_value(p[first + e])) == last) has |= 1u << e;
                int upto = __popc(has);
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                if (lane == 31) found[warp] = upto;
                __syncthreads();
                int at = rank + upto - __popc(has);
                for (int w = 0; w < BEAM_THREADS / 32; ++w) {
                    at += w < warp ? found[w] : 0;
                    rank += found[w];
                }
                for (; has && at < K; has &= has - 1) put(at++, k, first + __ffs(has) - 1, last);
                __syncthreads();
            }
        }
    }
}

struct BeamPlan {
    int slice, slices;
    size_t keys, bytes;
};
// Long slices cost less beside their data, short ones spread small steps over the SMs: as many slices as make two rounds
// of the 4 CTAs that fit an SM (48 x 8 beams over 151,936 fp32 logits: one round 47 us, two 43, four 45; 8 x 16 beams 24.5,
// 24.6, 26.5).
constexpr uint64_t BEAM_SLICES = 2 * 148 * 4;
static BeamPlan beam_plan(uint64_t rows, uint32_t beams, uint32_t vocab) {
    BeamPlan p;
    const uint64_t steps = ((uint64_t)vocab + BEAM_STEP - 1) / BEAM_STEP, want = std::max<uint64_t>(BEAM_SLICES / rows, 1);
    const uint64_t each = (steps + want - 1) / want;
    p.slice = (int)(each * BEAM_STEP);
    p.slices = (int)((steps + each - 1) / each);
    p.keys = (rows * p.slices * sizeof(float4) + 255) & ~(size_t)255;
    p.bytes = p.keys + rows * p.slices * beams * sizeof(u64);
    return p;
}

template <typename T>
static cudaError_t launch_slices(const void *logits, int64_t ld, int vocab, int beams, const BeamPlan &p, uint32_t rows, u64 *keys,
                                 float4 *sums, cudaStream_t st) {
    const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld * sizeof(T) % 16 == 0;
    return launch_k(false, k_beam_slice<T>, dim3(p.slices, rows), BEAM_THREADS, 0, st, static_cast<const T *>(logits), ld, vocab, p.slice,
                    beams, vec, keys, sums);
}

template <typename T>
static cudaError_t launch_beam(const BeamArgs &a, const BeamPlan &p, uint32_t groups, u64 *keys, float4 *sums, cudaStream_t st) {
    const cudaError_t e = launch_slices<T>(a.logits, a.ld, a.vocab, a.beams, p, groups * a.beams, keys, sums, st);
    return e == cudaSuccess ? launch_k(true, k_beam_join<T>, dim3(groups), BEAM_THREADS, 0, st, a) : e;
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
    float4 *sums = static_cast<float4 *>(dev_work);
    u64 *keys = reinterpret_cast<u64 *>(static_cast<uint8_t *>(dev_work) + p.keys);
    a.logits = dev_logits;
    a.ld = (int64_t)ld;
    a.keys = keys;
    a.sums = sums;
    a.scores = dev_scores;
    a.finished = dev_finished;
    a.beams = (int)beams;
    a.slice = p.slice;
    a.slices = p.slices;
    a.vocab = (int)vocab;
    a.eos = eos_id;
    a.tokens = tokens;
    a.parents = parents;
    a.scores_out = scores_out;
    a.finished_out = finished_out;
    const cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (dtype == V3G_F32) e = launch_beam<float>(a, p, groups, keys, sums, st);
    else if (dtype == V3G_F16) e = launch_beam<__half>(a, p, groups, keys, sums, st);
    else e = launch_beam<__nv_bfloat16>(a, p, groups, keys, sums, st);
    return e == cudaSuccess ? V3G_OK : v3g_fail(V3G_E_CUDA, std::string("v3g_beam_select: ") + cudaGetErrorString(e));
}
