// Log probabilities of given tokens, their ranks, the entropy and the
// likeliest alternatives of every row of logits (chn_token_logprobs).
//
// With x = (l - l_max) / T and S = sum exp x: log p = x - log S and the
// entropy is log S - sum(x exp x) / S, two sums of terms of one sign, so
// nothing cancels.  Two launches:
//  1 k_logprob_sums reads the row once, a wave per stretch of 2048 values in
//    registers: their largest, both sums against it, how many tokens come
//    before the given one, and the largest of every block of 256;
//  2 k_logprob_rows, a workgroup per row, joins the stretches.  The n_top
//    blocks with the largest maxima hold the n_top largest tokens: they are
//    read again, and what reaches the least of those maxima is ranked.
#include "chn_internal.h"

#include <cmath>

namespace chn {

typedef float f4l __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kScoreMaxV = 1u << 20;
constexpr uint32_t kScoreStretch = 2048, kScoreBlock = 256;
constexpr uint32_t kScoreTop = 64;
constexpr uint32_t kScoreThreads = 1024;
constexpr uint32_t kScoreRows = 1024;        // rows that share the workspace
constexpr uint32_t kBlockBits = 12;
static_assert(kScoreMaxV / kScoreBlock == 1u << kBlockBits, "a block's number");
constexpr uint32_t kScoreKeys = (1u << kBlockBits) / kScoreThreads;      // of a thread

struct LogProbs {
    const float *logits;
    uint32_t V, ld;
    const uint32_t *targets;
    const float *temperature;
    float cap;
    uint32_t n_top;
    float *logp, *entropy;
    uint32_t *ranks, *ids;
    float *tops;
    // workspace, per row: block maxima and, per stretch, maxima (orderable, 0: nothing allowed), the two sums, the count
    uint32_t blocks, stretches;
    uint32_t *bmax, *smax, *ahead;
    float *sum, *xsum;
};

__device__ __forceinline__ bool scored(float v) { return v > -3.4028234663852886e38f; }      // not NaN either
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);                               // -0 orders as +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return __builtin_bit_cast(float, (o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

// cap tanh(l / cap) from exp(-2 |l / cap|), off by about two steps of fp32:
// the sums average it out, and what is returned of single tokens is formed in
// 64 bits.
template <bool CAP>
__device__ __forceinline__ float capped(float l, float cap, float inv_cap) {
    if (!CAP) return l;
    const float t = __builtin_amdgcn_exp2f(-2.8853900817779268f * fabsf(l * inv_cap));
    return copysignf(cap * ((1.0f - t) / (1.0f + t)), l);
}
template <bool CAP>
__device__ __forceinline__ double capped64(float l, float cap) {
    return CAP ? (double)cap * tanh((double)l / (double)cap) : (double)l;
}
// a temperature that takes the largest only
__device__ __forceinline__ float powers_of(const LogProbs &a, uint32_t row, bool &greedy) {
    const float T = a.temperature ? a.temperature[row] : 1.0f;
    greedy = !(T > 0.0f);
    return greedy ? 0.0f : 1.4426950408889634f / T;
}
// The distance of two values in powers of two; at least -200, where a weight is nothing.
__device__ __forceinline__ float distance(float v, float top, float powers) {
    return v == top ? 0.0f : fmaxf((v - top) * powers, -200.0f);
}

template <bool CAP>
__global__ __launch_bounds__(256) void k_logprob_sums(LogProbs a) {
    const uint32_t row = blockIdx.y, s = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (s >= a.stretches) return;
    const float *x = a.logits + (size_t)row * a.ld;
    const uint32_t i0 = s * kScoreStretch + 4 * lane;
    f4l v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t i = i0 + 256 * j;
        if (i + 4 <= a.V) v[j] = *(const f4l *)(x + i);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = i + e < a.V ? x[i + e] : __builtin_nanf("");
    }
    const uint32_t target = a.targets[row];
    const float mine = target < a.V ? x[target] : __builtin_nanf("");
    bool greedy;
    const float powers = powers_of(a, row, greedy), cap = a.cap, inv_cap = 1.0f / cap;
    float top = -__builtin_inff();
    uint32_t before = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float m = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t i = i0 + 256 * j + e;
            before += scored(v[j][e]) && (v[j][e] > mine || (v[j][e] == mine && i < target));
            m = fmaxf(m, scored(v[j][e]) ? v[j][e] : -__builtin_inff());
        }
        if (a.n_top) {
            const float b = wave_max64(m);
            const uint32_t block = s * (kScoreStretch / kScoreBlock) + j;
            if (lane == 0 && block < a.blocks) a.bmax[(size_t)row * a.blocks + block] = scored(b) ? ordered(b) : 0u;
        }
        top = fmaxf(top, m);
    }
    top = wave_max64(top);
    before = (uint32_t)wave_sum_u64(before);
    float S = 0.0f, X = 0.0f;
    if (scored(top) && !greedy) {
        const float ref = capped<CAP>(top, cap, inv_cap);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float d = distance(capped<CAP>(v[j][e], cap, inv_cap), ref, powers);
                const float p = scored(v[j][e]) ? __builtin_amdgcn_exp2f(d) : 0.0f;
                S += p;
                X = scored(v[j][e]) ? fmaf(p, d, X) : X;
            }
        S = wave_sum64(S);
        X = wave_sum64(X);
    }
    if (lane == 0) {
        const size_t at = (size_t)row * a.stretches + s;
        a.smax[at] = scored(top) ? ordered(top) : 0u;
        a.ahead[at] = before;
        a.sum[at] = S;
        a.xsum[at] = X;
    }
}

// Sums and maxima over the workgroup, the same bits for every thread.
struct RowSums {
    float part[kScoreThreads / 64];
    uint32_t count[kScoreThreads / 64];
    uint64_t counts[2][kScoreThreads / 64];
};
__device__ __forceinline__ float group_sum(RowSums &sh, float v) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    return row16_sum(sh.part[threadIdx.x & 15]);
}
__device__ __forceinline__ uint32_t group_sum(RowSums &sh, uint32_t v) {
    v = (uint32_t)wave_sum_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.count[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t t = 0;
#pragma unroll
    for (uint32_t i = 0; i < kScoreThreads / 64; ++i) t += sh.count[i];
    return t;
}
__device__ __forceinline__ uint32_t group_max(RowSums &sh, uint32_t v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.count[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t t = 0;
#pragma unroll
    for (uint32_t i = 0; i < kScoreThreads / 64; ++i) t = max(t, sh.count[i]);
    return t;
}

// The n-th largest of unique keys below 2^BITS (0: none), from the top bits
// down, two at a time: each(f) calls f(key) for the thread's keys.  0 where
// there are fewer than n.
template <int BITS, typename F>
__device__ __forceinline__ uint64_t nth_largest(RowSums &sh, uint32_t n, F &&each) {
    uint64_t least = 0;
    for (int bit = BITS - 2, turn = 0; bit >= 0; bit -= 2, turn ^= 1) {
        const uint64_t step = 1ull << bit;
        uint64_t mine = 0;                                     // three counts of 20 bits
        each([&](uint64_t key) {
            mine += (uint64_t)(key >= least + step) + ((uint64_t)(key >= least + 2 * step) << 20) +
                    ((uint64_t)(key >= least + 3 * step) << 40);
        });
        mine = wave_sum_u64(mine);
        if ((threadIdx.x & 63) == 0) sh.counts[turn][threadIdx.x >> 6] = mine;
        __syncthreads();
        const uint64_t all = lane64(row16_scan_u64(sh.counts[turn][threadIdx.x & 15]), 15);
        const uint32_t c1 = (uint32_t)all & 0xFFFFF, c2 = (uint32_t)(all >> 20) & 0xFFFFF, c3 = (uint32_t)(all >> 40);
        least += (c3 >= n ? 3 : c2 >= n ? 2 : c1 >= n ? 1 : 0) * step;
    }
    return least;
}

constexpr uint32_t kScoreFew = 512;          // keys that are ranked by counting

template <bool CAP>
__global__ __launch_bounds__(kScoreThreads) void k_logprob_rows(LogProbs a) {
    extern __shared__ uint64_t list[];                          // n_top * kScoreBlock keys
    __shared__ RowSums sh;
    __shared__ uint64_t few[kScoreTop];
    __shared__ uint32_t chosen[kScoreTop], n_chosen, n_list, n_few;
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const int lane = tid & 63, wave = tid >> 6;
    const float *x = a.logits + (size_t)row * a.ld;
    const uint32_t target = a.targets[row];
    const float mine = target < a.V ? x[target] : __builtin_nanf("");
    bool greedy;
    const float powers = powers_of(a, row, greedy), inv_cap = 1.0f / a.cap;
    if (tid == 0) n_chosen = n_list = n_few = 0;

    // the stretches: at most 512, a thread each
    uint32_t m = 0, before = 0;
    float S = 0.0f, X = 0.0f;
    if (tid < a.stretches) {
        const size_t at = (size_t)row * a.stretches + tid;
        m = a.smax[at];
        before = a.ahead[at];
        S = a.sum[at];
        X = a.xsum[at];
    }
    const uint32_t most = group_max(sh, m);
    const float top = unordered(most);
    if (most && m) {
        const float d = distance(capped<CAP>(unordered(m), a.cap, inv_cap), capped<CAP>(top, a.cap, inv_cap), powers);
        const float f = __builtin_amdgcn_exp2f(d);
        X = f * (X + d * S);
        S *= f;
    }
    S = group_sum(sh, S);
    X = group_sum(sh, X);
    before = group_sum(sh, before);
    const double log_sum = greedy ? 0.0 : log((double)S);
    // of an allowed logit that `first` tokens come before
    const auto logp = [&](float l, bool first) {
        if (greedy) return first ? 0.0f : -__builtin_inff();
        const double T = a.temperature ? (double)a.temperature[row] : 1.0;
        return (float)((l == top ? 0.0 : (capped64<CAP>(l, a.cap) - capped64<CAP>(top, a.cap)) / T) - log_sum);
    };
    if (tid == 0) {
        const bool given = target < a.V, ok = most && scored(mine);
        a.logp[row] = !given ? 0.0f : ok ? logp(mine, before == 0) : -__builtin_inff();
        if (a.entropy) a.entropy[row] = most && !greedy ? (float)(log_sum - 0.69314718055994531 * (double)X / (double)S) : 0.0f;
        if (a.ranks) a.ranks[row] = ok ? before : CHN_NO_TOKEN;
    }
    if (!a.n_top) return;

    // the blocks with the largest maxima, equal ones by lower number
    const uint32_t *bmax = a.bmax + (size_t)row * a.blocks;
    uint64_t key[kScoreKeys];
#pragma unroll
    for (uint32_t k = 0; k < kScoreKeys; ++k) {
        const uint32_t b = tid + kScoreThreads * k, o = b < a.blocks ? bmax[b] : 0u;
        key[k] = o ? (uint64_t)o << kBlockBits | ((1u << kBlockBits) - 1 - b) : 0;
    }
    const uint64_t least = nth_largest<32 + kBlockBits>(sh, a.n_top, [&](auto &&f) {
#pragma unroll
        for (uint32_t k = 0; k < kScoreKeys; ++k) f(key[k]);
    });
#pragma unroll
    for (uint32_t k = 0; k < kScoreKeys; ++k)
        if (key[k] && key[k] >= least) chosen[atomicAdd(&n_chosen, 1u)] = tid + kScoreThreads * k;
    __syncthreads();
    const uint32_t floor_key = (uint32_t)(least >> kBlockBits);
    for (uint32_t c = wave; c < n_chosen; c += kScoreThreads / 64) {
        const uint32_t i0 = chosen[c] * kScoreBlock + 4 * lane;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t i = i0 + e;
            const float v = x[min(i, a.V - 1)];
            if (i < a.V && scored(v) && ordered(v) >= floor_key)
                list[atomicAdd(&n_list, 1u)] = (uint64_t)ordered(v) << 32 | (0xFFFFFFFFu - i);
        }
    }
    __syncthreads();
    const uint64_t *keys = list;
    uint32_t n = n_list;
    if (n > kScoreFew) {
        const uint64_t last = nth_largest<64>(sh, a.n_top, [&](auto &&f) {
            for (uint32_t i = tid; i < n; i += kScoreThreads) f(list[i]);
        });
        for (uint32_t i = tid; i < n; i += kScoreThreads)
            if (list[i] >= last) few[atomicAdd(&n_few, 1u)] = list[i];       // n_top of them
        __syncthreads();
        keys = few;
        n = n_few;
    }
    uint32_t *ids = a.ids + (size_t)row * a.n_top;
    float *tops = a.tops + (size_t)row * a.n_top;
    if (tid < n) {
        const uint64_t k = keys[tid];
        uint32_t rank = 0;
        for (uint32_t i = 0; i < n; ++i) rank += keys[i] > k;
        if (rank < a.n_top) {
            ids[rank] = 0xFFFFFFFFu - (uint32_t)k;
            tops[rank] = logp(unordered((uint32_t)(k >> 32)), rank == 0);
        }
    }
    if (tid >= n && tid < a.n_top) {                             // fewer tokens than n_top
        ids[tid] = CHN_NO_TOKEN;
        tops[tid] = -__builtin_inff();
    }
}

template <bool CAP>
static void launch_scores(chn_ctx *ctx, const LogProbs &a, uint32_t n) {
    k_logprob_sums<CAP><<<dim3((a.stretches + 3) / 4, n), 256, 0, ctx->stream>>>(a);
    k_logprob_rows<CAP><<<n, kScoreThreads, (size_t)a.n_top * kScoreBlock * 8, ctx->stream>>>(a);
}

}  // namespace chn

using namespace chn;

extern "C" int chn_token_logprobs(chn_ctx *ctx, const float *logits, uint32_t n_rows, uint32_t V, uint32_t ld,
                                  const uint32_t *targets, const float *temperature, float softcap, uint32_t n_top,
                                  float *logprobs, float *entropy, uint32_t *ranks, uint32_t *top_ids,
                                  float *top_logprobs) {
    CHN_REQUIRE(ctx, logits && targets && logprobs, "NULL argument");
    CHN_REQUIRE(ctx, n_top <= kScoreTop, "n_top %u exceeds %u", n_top, kScoreTop);
    CHN_REQUIRE(ctx, !n_top || (top_ids && top_logprobs), "NULL top_ids or top_logprobs");
    CHN_REQUIRE(ctx, V > 0 && V <= kScoreMaxV, "V=%u must be in 1..%u", V, kScoreMaxV);
    CHN_REQUIRE(ctx, ld >= V, "ld=%u is below V=%u", ld, V);
    CHN_REQUIRE(ctx, softcap >= 0.0f && std::isfinite(softcap), "softcap must be finite and not negative");
    CHN_REQUIRE(ctx, n_rows <= 65535, "n_rows=%u exceeds 65535", n_rows);
    CHN_REQUIRE(ctx, ctx, "ctx is NULL");
    if (!n_rows) return CHN_OK;
    DeviceGuard dev(ctx);
    LogProbs a{};
    a.V = V;
    a.ld = ld;
    a.cap = softcap;
    a.n_top = n_top;
    a.blocks = (V + kScoreBlock - 1) / kScoreBlock;
    a.stretches = (V + kScoreStretch - 1) / kScoreStretch;
    const size_t rows = std::min(n_rows, kScoreRows);
    int rc = ensure_workspace(ctx, rows * ((size_t)a.blocks + 4 * (size_t)a.stretches) * 4);
    if (rc) return rc;
    a.bmax = (uint32_t *)ctx->ws;
    a.smax = a.bmax + rows * a.blocks;
    a.ahead = a.smax + rows * a.stretches;
    a.sum = (float *)(a.ahead + rows * a.stretches);
    a.xsum = a.sum + rows * a.stretches;
    for (uint32_t r0 = 0; r0 < n_rows; r0 += kScoreRows) {
        a.logits = logits + (size_t)r0 * ld;
        a.targets = targets + r0;
        a.temperature = temperature ? temperature + r0 : nullptr;
        a.logp = logprobs + r0;
        a.entropy = entropy ? entropy + r0 : nullptr;
        a.ranks = ranks ? ranks + r0 : nullptr;
        a.ids = n_top ? top_ids + (size_t)r0 * n_top : nullptr;
        a.tops = n_top ? top_logprobs + (size_t)r0 * n_top : nullptr;
        const uint32_t n = std::min(n_rows - r0, kScoreRows);
        softcap > 0.0f ? launch_scores<true>(ctx, a, n) : launch_scores<false>(ctx, a, n);
        CHN_LAUNCHED(ctx, "k_logprob");
    }
    return CHN_OK;
}
