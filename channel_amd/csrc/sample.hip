// The next token of every row of logits: temperature, top-k, top-p and min-p
// from given random numbers (chn_sample).
//
// Tokens are ordered by the 64-bit key orderable(logit) << 32 | ~index
// (unique; descending: larger logits first, equal ones by lower index); every
// filter keeps a prefix of that order, so a row's kept tokens are those at or
// above one key.  A token's weight is exp((l - l_max) / T) as an integer in
// units of 2^-43: integer sums do not depend on their order, so the borders
// that top-p and the draw look for are the same whichever thread adds first.
// 43 bits: 2^20 weights of at most 2^43 fit 64, and the 2^-44 a rounding
// costs is far below what 32-bit sums would lose (a flat row of 2^18 tokens
// has its borders 2^-18 of the sum apart).
#include "chn_internal.h"

#include <cmath>

namespace chn {

constexpr uint32_t kSampleMaxV = 1u << 20;
constexpr int kWeightBits = 43;
constexpr uint32_t kRowThreads = 1024;

struct Sample {
    const float *logits;
    uint32_t V, ld;
    const float *temperature;
    const uint32_t *top_k;
    const float *top_p, *min_p, *u;
    float softcap;
    uint32_t *tokens;
    float *probs;
};

__device__ __forceinline__ bool allowed(float v) { return v > -3.4028234663852886e38f; }   // not NaN either
__device__ __forceinline__ uint32_t orderable(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);                             // -0 orders as +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t token_key(float v, uint32_t i) {
    return ((uint64_t)orderable(v) << 32) | (0xFFFFFFFFu - i);
}

// Weights of a row: cap * tanh(l / cap) relative to the row's largest.
struct Weigh {
    double cap, inv_cap, top, inv_t;
    float raw_top;
    __device__ __forceinline__ double capped(float l) const { return cap > 0.0 ? cap * tanh((double)l * inv_cap) : (double)l; }
    __device__ __forceinline__ double weight(float l) const {                              // 2^kWeightBits exp(..)
        if (l == raw_top) return (double)(1ull << kWeightBits);
        const double x = (capped(l) - top) * inv_t;
        return x > -64.0 ? exp(x) * (double)(1ull << kWeightBits) : 0.0;                  // below: rounds to zero anyway
    }
    __device__ __forceinline__ uint64_t units(float l) const { return (uint64_t)(weight(l) + 0.5); }
};

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += (uint64_t)__shfl_xor((unsigned long long)v, o, 64);
    return v;
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t w = (uint64_t)__shfl_xor((unsigned long long)v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}

// One workgroup per row.
__global__ __launch_bounds__(kRowThreads) void k_sample_row(Sample a) {
    constexpr int NW = kRowThreads / 64;
    __shared__ uint64_t part[NW];
    __shared__ uint64_t hist_w[256];
    __shared__ uint32_t hist_n[256];
    __shared__ uint64_t found[3];
    const uint32_t tid = threadIdx.x, row = blockIdx.x;
    const int lane = tid & 63, wave = tid >> 6;
    const float *x = a.logits + (size_t)row * a.ld;

    auto block_sum = [&](uint64_t v) {
        v = wave_sum_u64(v);
        __syncthreads();
        if (lane == 0) part[wave] = v;
        __syncthreads();
        uint64_t t = 0;
        for (int w = 0; w < NW; ++w) t += part[w];
        return t;
    };

    uint64_t top = 0;
    for (uint32_t i = tid; i < a.V; i += kRowThreads) {
        const float v = x[i];
        const uint64_t k = allowed(v) ? token_key(v, i) : 0;
        top = k > top ? k : top;
    }
    top = wave_max_u64(top);
    if (lane == 0) part[wave] = top;
    __syncthreads();
    for (int w = 0; w < NW; ++w) top = part[w] > top ? part[w] : top;
    const float T = a.temperature ? a.temperature[row] : 1.0f;
    if (top == 0 || !(T > 0.0f)) {
        if (tid == 0) {
            a.tokens[row] = top ? 0xFFFFFFFFu - (uint32_t)top : CHN_NO_TOKEN;
            if (a.probs) a.probs[row] = top ? 1.0f : 0.0f;
        }
        return;
    }
    Weigh wg;
    wg.cap = a.softcap;
    wg.inv_cap = 1.0 / (double)a.softcap;
    wg.raw_top = x[0xFFFFFFFFu - (uint32_t)top];
    wg.top = wg.capped(wg.raw_top);
    wg.inv_t = 1.0 / (double)T;

    // The key of the last token of the order, from the tokens at or above
    // `above`, that the running count (or sum of weights) needs to reach
    // `goal`: eight bits of the key at a time, until the bin is wanted whole.
    auto last_key = [&](uint64_t above, bool by_weight, uint64_t goal) {
        uint64_t prefix = 0;
        for (int shift = 56;; shift -= 8) {
            __syncthreads();
            if (tid < 256) {
                hist_n[tid] = 0;
                hist_w[tid] = 0;
            }
            __syncthreads();
            for (uint32_t i = tid; i < a.V; i += kRowThreads) {
                const float v = x[i];
                if (!allowed(v)) continue;
                const uint64_t k = token_key(v, i);
                if (k < above || (shift < 56 && (k >> (shift + 8)) != prefix)) continue;
                const uint32_t bin = (uint32_t)(k >> shift) & 255u;
                atomicAdd(&hist_n[bin], 1u);
                if (by_weight) atomicAdd((unsigned long long *)&hist_w[bin], (unsigned long long)wg.units(v));
            }
            __syncthreads();
            if (tid == 0) {
                uint64_t sum = 0;
                int bin = 255, last = -1;
                for (; bin >= 0; --bin) {
                    const uint64_t c = by_weight ? hist_w[bin] : hist_n[bin];
                    if (hist_n[bin]) last = bin;
                    if (sum + c >= goal) break;
                    sum += c;
                }
                if (bin < 0) bin = last;                       // fewer than wanted: the last token there is
                found[0] = bin;
                found[1] = sum;
                found[2] = shift == 0 || hist_n[bin] == 1 || (!by_weight && sum + hist_n[bin] == goal);
            }
            __syncthreads();
            prefix = (prefix << 8) | found[0];
            goal -= found[1] < goal ? found[1] : goal;
            if (found[2]) {
                const uint64_t key = prefix << shift;          // the bin's lower end: it may reach below `above`
                return key > above ? key : above;
            }
        }
    };
    auto mass = [&](uint64_t above, uint64_t least) {
        uint64_t s = 0;
        for (uint32_t i = tid; i < a.V; i += kRowThreads) {
            const float v = x[i];
            if (!allowed(v) || token_key(v, i) < above) continue;
            const uint64_t w = wg.units(v);
            s += w >= least ? w : 0;
        }
        return block_sum(s);
    };

    uint64_t above = 1;
    const uint32_t k = a.top_k ? a.top_k[row] : 0;
    if (k && k < a.V) {
        uint64_t n = 0;
        for (uint32_t i = tid; i < a.V; i += kRowThreads) n += allowed(x[i]) ? 1 : 0;
        if (block_sum(n) > k) above = last_key(1, false, k);
    }
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    if (p < 1.0f) {
        const uint64_t Z = mass(above, 0);
        // kept while the mass before is below p Z: the last one is the first whose running sum reaches ceil(p Z)
        const double goal = ceil((p > 0.0f ? (double)p : 0.0) * (double)Z);
        const uint64_t g = goal < 1.0 ? 1 : (uint64_t)goal;
        above = last_key(above, true, g < Z ? g : Z);
    }
    const float m = a.min_p ? a.min_p[row] : 0.0f;
    const uint64_t least = m > 0.0f ? (uint64_t)ceil(fmin((double)m, 1.0) * (double)(1ull << kWeightBits)) : 0;
    const uint64_t Z = mass(above, least);
    const float uf = a.u[row];
    const double want = (uf > 0.0f ? (double)uf : 0.0) * (double)Z;
    uint64_t target = want >= (double)Z ? Z - 1 : (uint64_t)want;
    target = target < Z ? target : Z - 1;

    // the first index whose running sum exceeds target: a range of indexes in
    // as many parts as there are waves, then that part again, until a thread
    // each is left
    uint32_t lo = 0, n = a.V;
    for (;;) {
        const uint32_t len = (n + NW - 1) / NW;               // per wave
        const uint32_t b = lo + wave * len, e = min(b + len, lo + n);
        uint64_t s = 0, run = 0;
        for (uint32_t i = b + lane; i < e; i += 64) {
            const float v = x[i];
            if (!allowed(v) || token_key(v, i) < above) continue;
            const uint64_t w = wg.units(v);
            s += w >= least ? w : 0;
        }
        run = s;
        s = wave_sum_u64(s);
        __syncthreads();
        if (lane == 0) part[wave] = s;
        __syncthreads();
        uint64_t before = 0;
        int at = 0;
        for (; at < NW - 1 && before + part[at] <= target; ++at) before += part[at];
        target -= before;
        if (len <= 64) {
            // one value per lane of wave `at`
            if (wave == at) {
                const uint64_t own = run;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const uint64_t w = (uint64_t)__shfl_up((unsigned long long)run, o, 64);
                    if (lane >= o) run += w;
                }
                if (own && run > target && run - own <= target) {
                    const uint32_t i = b + lane;
                    a.tokens[row] = i;
                    if (a.probs) a.probs[row] = (float)(wg.weight(x[i]) / (double)Z);
                }
            }
            return;
        }
        lo += at * len;
        n = min(len, a.V - lo);
    }
}

}  // namespace chn

using namespace chn;

extern "C" int chn_sample(chn_ctx *ctx, const float *logits, uint32_t n_rows, uint32_t V, uint32_t ld,
                          const float *temperature, const uint32_t *top_k, const float *top_p, const float *min_p,
                          const float *u, float softcap, uint32_t *tokens, float *probs) {
    CHN_REQUIRE(ctx, logits && u && tokens, "NULL argument");
    CHN_REQUIRE(ctx, V > 0 && V <= kSampleMaxV, "V=%u must be in 1..%u", V, kSampleMaxV);
    CHN_REQUIRE(ctx, ld >= V, "ld=%u is below V=%u", ld, V);
    CHN_REQUIRE(ctx, softcap >= 0.0f && std::isfinite(softcap), "softcap must be finite and not negative");
    CHN_REQUIRE(ctx, n_rows <= 65535, "n_rows=%u exceeds 65535", n_rows);
    CHN_REQUIRE(ctx, ctx, "ctx is NULL");
    if (!n_rows) return CHN_OK;
    DeviceGuard dev(ctx);
    k_sample_row<<<n_rows, kRowThreads, 0, ctx->stream>>>(
        Sample{logits, V, ld, temperature, top_k, top_p, min_p, u, softcap, tokens, probs});
    CHN_LAUNCHED(ctx, "k_sample_row");
    return CHN_OK;
}
