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
constexpr uint32_t kScoreThreads = 256;
constexpr uint32_t kScoreRows = 1024;        // rows that share the workspace
constexpr uint32_t kBlockBits = 12;
static_assert(kScoreMaxV / kScoreBlock == 1u << kBlockBits, "a block's number");

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
    // (16 bits) and, with a softcap, how many equal the maximum (above them; the sums are then without those)
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

// CAP: 0 no softcap, 1 and 2 cap tanh(l / cap) from exp(-2 |l / cap|), off by
// about two steps of fp32 of the cap: the sums average it out, and what is
// returned of single tokens is formed in 64 bits.  A cap that is large beside
// the logits would take their digits, so 2 has the series of tanh below a quarter
// of the cap, off by steps of the logit (its next term is 2^-27 of it).  Caps
// up to kStepCap take 1: 500 rows of 262144 in 124 us, with 2 143.
constexpr float kStepCap = 64.0f;
template <int CAP>
__device__ __forceinline__ float capped(float l, float cap, float inv_cap) {
    if (!CAP) return l;
    const float x = l * inv_cap, t = __builtin_amdgcn_exp2f(-2.8853900817779268f * fabsf(x));
    const float y = copysignf(cap * ((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t)), l);
    if (CAP == 1) return y;
    const float z = x * x, series = fmaf(fmaf(fmaf(62.0f / 2835, z, -17.0f / 315), z, 2.0f / 15), z, -1.0f / 3);
    return fabsf(x) < 0.25f ? fmaf(l * z, series, l) : y;
}
// of denormal caps no infinity, whose product with zero is none
__device__ __forceinline__ float inverse_of(float cap) { return fminf(1.0f / cap, 3.4028235e38f); }
template <int CAP>
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
// the larger; m if v is NaN
__device__ __forceinline__ float larger_of(float v, float m) { return __builtin_amdgcn_fmed3f(v, m, __builtin_inff()); }
template <int CTRL>
__device__ __forceinline__ float max_row(float v) {
    return larger_of(__builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true)), v);
}
// Exchanges halves (rows) of two registers; an empty asm keeps this compiler from taking the second result for the first.
__device__ __forceinline__ float max_of_halves(float x, float y) {       // low half: x's, high half: y's
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
    uint32_t a = r[0], b = r[1];
    __asm__("" : "+v"(a), "+v"(b));
    return larger_of(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float max_of_rows(float x, float y) {         // even rows: x's, odd rows: y's
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
    uint32_t a = r[0], b = r[1];
    __asm__("" : "+v"(a), "+v"(b));
    return larger_of(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
// The largest of each of eight values over the wave: lanes 8 i .. 8 i + 7 get that of v[order(i)].
__device__ __forceinline__ float wave_max8(const float (&v)[8], int lane) {
    float h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = max_of_halves(v[i], v[i + 4]);                    // halves: i, i + 4
    const float a = max_of_rows(h[0], h[1]), b = max_of_rows(h[2], h[3]);              // rows: 0 1 4 5, 2 3 6 7
    const float keep = lane & 8 ? b : a, give = lane & 8 ? a : b;
    float m = larger_of(__builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, give), 0x128, 0xF, 0xF, true)), keep);
    m = max_row<0xB1>(m);                                                              // quad_perm [1,0,3,2], [2,3,0,1]
    m = max_row<0x4E>(m);
    return max_row<0x141>(m);                                                          // row_half_mirror
}
__device__ __forceinline__ int max8_order(int i) {                       // the value whose maximum lanes 8 i hold
    return (i >> 2) * 4 + (i & 1) * 2 + (i >> 1 & 1);
}

// A wave's 2048 values: 256 a load, four of them a lane, all eight loads under
// way at once.  Bound by memory where there are many rows: 500 rows of 262144,
// 524 MB, in 85-90 us (5.8-6.2 TB/s); softcapped 98-109, memory and issue; one
// row is a latency, 4.6 us.
template <int CAP>
__global__ __launch_bounds__(256) void k_logprob_sums(LogProbs a) {
    const uint32_t row = blockIdx.y, s = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (s >= a.stretches) return;
    const float *x = a.logits + (size_t)row * a.ld;
    const uint32_t i0 = s * kScoreStretch + 4 * lane;
    f4l v[8];
    if ((s + 1) * kScoreStretch <= a.V) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = *(const f4l *)(x + i0 + 256 * j);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t i = i0 + 256 * j + e;
                const float l = x[min(i, a.V - 1)];
                v[j][e] = i < a.V ? l : __builtin_nanf("");
            }
    }
    const uint32_t target = a.targets[row];
    const float mine = target < a.V ? x[target] : __builtin_nanf("");
    bool greedy;
    const float powers = powers_of(a, row, greedy), cap = a.cap, inv_cap = inverse_of(cap);
    float m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = larger_of(v[j][3], larger_of(v[j][2], larger_of(v[j][1], larger_of(v[j][0], -__builtin_inff()))));
    const float most = wave_max8(m, lane);
    const size_t at = (size_t)row * a.stretches + s;
    if (a.n_top && (lane & 7) == 0) {
        const uint32_t block = s * (kScoreStretch / kScoreBlock) + max8_order(lane >> 3);
        if (block < a.blocks) a.bmax[(size_t)row * a.blocks + block] = scored(most) ? ordered(most) : 0u;
    }
    const float top = wave_max64(most);
    // NaN compares false, and what is barred lies below a given token that is not
    uint32_t before = 0;
    if (scored(mine)) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) before += (uint32_t)__popcll(__ballot(v[j][e] > mine));
        uint32_t same = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) same += v[j][e] == mine && i0 + 256 * j + e < target;
        if (__any(same)) before += (uint32_t)wave_sum_u64(same);
    }
    float S = 0.0f, X = 0.0f;
    uint32_t ties = 0;
    if (scored(top) && !greedy) {
        const float ref = capped<CAP>(top, cap, inv_cap);
        if (fabsf(ref) <= 1e30f && powers >= 1e-6f && powers <= 1e30f) {
            // barred values lie 200 powers below and more, NaN is taken for that
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float d = larger_of((capped<CAP>(v[j][e], cap, inv_cap) - ref) * powers, -200.0f);
                    float p = __builtin_amdgcn_exp2f(d);
                    if (CAP) {
                        const bool tie = v[j][e] == top;
                        ties += tie;
                        p = scored(v[j][e]) && !tie ? p : 0.0f;           // -inf is capped too
                    }
                    S += p;
                    X = fmaf(p, d, X);
                }
        } else {
            for (int j = 0; j < 8; ++j)
                for (int e = 0; e < 4; ++e) {
                    const float d = distance(capped<CAP>(v[j][e], cap, inv_cap), ref, powers);
                    const bool tie = CAP && v[j][e] == top;
                    ties += tie;
                    const float p = scored(v[j][e]) && !tie ? __builtin_amdgcn_exp2f(d) : 0.0f;
                    S += p;
                    X += scored(v[j][e]) && !tie ? p * d : 0.0f;
                }
        }
        S = wave_sum64(S);
        X = wave_sum64(X);
        if (CAP) ties = __any(ties > 1) ? (uint32_t)wave_sum_u64(ties) : (uint32_t)__popcll(__ballot(ties));
    }
    if (lane == 0) {
        a.smax[at] = scored(top) ? ordered(top) : 0u;
        a.ahead[at] = before | ties << 16;
        a.sum[at] = S;
        a.xsum[at] = X;
    }
}

// What a row's workgroup exchanges.
constexpr int kScoreWaves = kScoreThreads / 64;
struct RowSums {
    float sum[kScoreWaves], xsum[kScoreWaves];
    uint32_t most[kScoreWaves], before[kScoreWaves];
    float ties[kScoreWaves];
    uint32_t counts[2][kScoreWaves][4];
};

// The n-th largest of unique keys below 2^BITS (0: none), or any bound that n
// of them reach, from the top bits down, two at a time: each(f) calls f(key)
// for the thread's keys, the same number of times in every lane.  0 where there
// are fewer than n.
template <int BITS, typename F>
__device__ __forceinline__ uint64_t nth_largest(RowSums &sh, uint32_t n, F &&each) {
    uint64_t least = 0;
    for (int bit = BITS - 2, turn = 0; bit >= 0; bit -= 2, turn ^= 1) {
        const uint64_t step = 1ull << bit;
        uint32_t c[3] = {0, 0, 0};
        each([&](uint64_t key) {
#pragma unroll
            for (int i = 0; i < 3; ++i) c[i] += (uint32_t)__popcll(__ballot(key >= least + (i + 1) * step));
        });
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < 3; ++i) sh.counts[turn][threadIdx.x >> 6][i] = c[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            c[i] = 0;
#pragma unroll
            for (int w = 0; w < kScoreWaves; ++w) c[i] += sh.counts[turn][w][i];
        }
        const int take = c[2] >= n ? 3 : c[1] >= n ? 2 : c[0] >= n ? 1 : 0;
        least += take * step;
        if (take && c[take - 1] == n) break;
    }
    return least;
}

constexpr uint32_t kScoreFew = 256;          // keys that are ranked by counting

// Bound by its chain of latencies, the same for one row and for hundreds: the
// sums, the bound on the block maxima two bits at a time, the chosen blocks,
// their ranks.  500 rows with 5 alternatives 10.5 us, softcapped 15.8; one with
// 20, softcapped, 11.8.  KEYS: block maxima of a thread (4 up to 262144 values, else 16).
template <int CAP, int KEYS>
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
    const float powers = powers_of(a, row, greedy), inv_cap = inverse_of(a.cap);
    if (tid == 0) n_chosen = n_list = n_few = 0;

    // the stretches: at most 512, two a thread; the blocks' maxima
    uint32_t m[2], ahead[2];
    float S[2], X[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t s = tid + kScoreThreads * i;
        const size_t at = (size_t)row * a.stretches + min(s, a.stretches - 1);
        const bool there = s < a.stretches;
        m[i] = there ? a.smax[at] : 0u;
        ahead[i] = there ? a.ahead[at] : 0u;
        S[i] = a.sum[at];
        X[i] = a.xsum[at];
    }
    uint64_t key[KEYS];
    if (a.n_top) {
        const uint32_t *bmax = a.bmax + (size_t)row * a.blocks;
#pragma unroll
        for (uint32_t k = 0; k < KEYS; ++k) {
            const uint32_t b = tid + kScoreThreads * k, o = b < a.blocks ? bmax[b] : 0u;
            key[k] = o ? (uint64_t)o << kBlockBits | ((1u << kBlockBits) - 1 - b) : 0;
        }
    }
    uint32_t most = max(m[0], m[1]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) most = max(most, (uint32_t)__shfl_xor(most, o, 64));
    if (lane == 0) sh.most[wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScoreWaves; ++w) most = max(most, sh.most[w]);
    const float top = unordered(most);
    float sum = 0.0f, xsum = 0.0f;
    uint32_t before = 0;
    float ties = 0.0f;                                          // of the row's largest: at most 2^20
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float same = (float)(ahead[i] >> 16);
        before += ahead[i] & 0xFFFFu;
        if (CAP && m[i] == most) ties += same;
        else if (CAP) S[i] += same;
        if (m[i]) {
            const float d = distance(capped<CAP>(unordered(m[i]), a.cap, inv_cap), capped<CAP>(top, a.cap, inv_cap), powers);
            const float f = __builtin_amdgcn_exp2f(d);
            xsum += f * (X[i] + d * S[i]);
            sum += f * S[i];
        }
    }
    sum = wave_sum64(sum);
    xsum = wave_sum64(xsum);
    before = (uint32_t)wave_sum_u64(before);
    if (CAP) ties = wave_sum64(ties);
    if (lane == 0) {
        sh.sum[wave] = sum;
        sh.xsum[wave] = xsum;
        sh.before[wave] = before;
        if (CAP) sh.ties[wave] = ties;
    }
    __syncthreads();
    sum = xsum = ties = 0.0f;
    before = 0;
#pragma unroll
    for (int w = 0; w < kScoreWaves; ++w) {
        sum += sh.sum[w];
        xsum += sh.xsum[w];
        before += sh.before[w];
        if (CAP) ties += sh.ties[w];
    }
    const double T = a.temperature ? (double)a.temperature[row] : 1.0;
    // With a softcap the sums are those of the other tokens, relative to the largest capped in fp32: its rounding is taken
    // out of them again, theirs go both ways.  Where that is much of an exponent (T near a step of fp32's of the cap, and
    // below) it is left in: a token's weight is then one at most.
    double all = (double)sum, mean = 0.69314718055994531 * (double)xsum;
    if (CAP && !greedy) {
        double off = ((double)capped<CAP>(top, a.cap, inv_cap) - capped64<CAP>(top, a.cap)) / T;
        if (!(fabs(off) <= 0.5)) off = 0.0;
        const double f = exp(off), others = all;
        mean = f * (mean + others * off);
        all = (double)ties + others * f;
    }
    const double log_sum = greedy ? 0.0 : log(all);
    // of an allowed logit; `first`: no token comes before it
    const auto logp = [&](float l, bool first) {
        if (greedy) return first ? 0.0f : -__builtin_inff();
        return (float)((l == top ? 0.0 : (capped64<CAP>(l, a.cap) - capped64<CAP>(top, a.cap)) / T) - log_sum);
    };
    if (wave == kScoreWaves - 1 && lane == 0) {
        const bool given = target < a.V, ok = most && scored(mine);
        a.logp[row] = !given ? 0.0f : ok ? logp(mine, before == 0) : -__builtin_inff();
        if (a.entropy) a.entropy[row] = most && !greedy ? (float)(log_sum - mean / all) : 0.0f;
        if (a.ranks) a.ranks[row] = ok ? before : CHN_NO_TOKEN;
    }
    if (!a.n_top) return;

    // the blocks with the largest maxima, equal ones by lower number
    const uint64_t least = nth_largest<32 + kBlockBits>(sh, a.n_top, [&](auto &&f) {
#pragma unroll
        for (int k = 0; k < KEYS; ++k) f(key[k]);
    });
#pragma unroll
    for (int k = 0; k < KEYS; ++k)
        if (key[k] && key[k] >= least) chosen[atomicAdd(&n_chosen, 1u)] = tid + kScoreThreads * k;
    __syncthreads();
    // the bound's bits above the block's number: of the n_top values that reach it, none is below
    const uint32_t floor_key = (uint32_t)(least >> kBlockBits);
    for (uint32_t c = wave; c < n_chosen; c += 2 * kScoreWaves) {
        // two blocks in flight
        float v[2][4];
        uint32_t i0[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i0[h] = chosen[min(c + kScoreWaves * h, n_chosen - 1)] * kScoreBlock + 4 * lane;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[h][e] = x[min(i0[h] + e, a.V - 1)];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t i = i0[h] + e;
                if (c + kScoreWaves * h < n_chosen && i < a.V && scored(v[h][e]) && ordered(v[h][e]) >= floor_key)
                    list[atomicAdd(&n_list, 1u)] = (uint64_t)ordered(v[h][e]) << 32 | (0xFFFFFFFFu - i);
            }
    }
    __syncthreads();
    const uint64_t *keys = list;
    uint32_t n = n_list;
    if (n > kScoreFew) {
        const uint64_t last = nth_largest<64>(sh, a.n_top, [&](auto &&f) {
            for (uint32_t i = tid; i < (n + kScoreThreads - 1) / kScoreThreads * kScoreThreads; i += kScoreThreads) f(i < n ? list[i] : 0);
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

template <int CAP>
static void launch_scores(chn_ctx *ctx, const LogProbs &a, uint32_t n) {
    k_logprob_sums<CAP><<<dim3((a.stretches + 3) / 4, n), 256, 0, ctx->stream>>>(a);
    const size_t lds = (size_t)a.n_top * kScoreBlock * 8;
    if (a.blocks <= 4 * kScoreThreads) k_logprob_rows<CAP, 4><<<n, kScoreThreads, lds, ctx->stream>>>(a);
    else k_logprob_rows<CAP, (1 << kBlockBits) / kScoreThreads><<<n, kScoreThreads, lds, ctx->stream>>>(a);
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
    const size_t n_all = n_rows, n_tops = n_all * n_top;
    const Span outs[] = {{logprobs, n_all}, {entropy, n_all}, {ranks, n_all}, {top_ids, n_tops}, {top_logprobs, n_tops}};
    const Span ins[] = {{logits, n_all ? (n_all - 1) * ld + V : 0}, {targets, n_all}, {temperature, n_all}};
    for (const Span &o : outs) {
        for (const Span &i : ins) CHN_REQUIRE(ctx, !overlap(i, o), "an output overlaps an input");
        for (const Span &p : outs) CHN_REQUIRE(ctx, &p == &o || !overlap(p, o), "two outputs overlap");
    }
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
        if (softcap > kStepCap) launch_scores<2>(ctx, a, n);
        else if (softcap > 0.0f) launch_scores<1>(ctx, a, n);
        else launch_scores<0>(ctx, a, n);
        CHN_LAUNCHED(ctx, "k_logprob");
    }
    return CHN_OK;
}
