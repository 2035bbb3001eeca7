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
//
// Four launches; what a row needs of them depends on its settings, which only
// the device knows:
//  1 k_sample_max: the largest logit of every block of 64, and of every 2048;
//  2 k_sample_mass (rows without top-k): with top-p a histogram of the weights
//    over their distance from the largest, else the sums of 2048 at a time;
//  3 k_sample_border (rows with top-p and without top-k): the bin that holds
//    the border goes into a list, the weights above it are summed;
//  4 k_sample_draw: a workgroup per row.  With top-k, the k-th largest block
//    maximum bounds the k-th largest logit from below, and only blocks whose
//    maximum reaches it can hold a kept token: the row is read once, and k
//    blocks of it again.  Otherwise the border is found in the list, and the
//    draw reads the one stretch of 2048 that it falls into.
// Rows that fit none of this (top-k above kMaxK, a border among more equal or
// near equal logits than the list holds) take k_sample_draw's walk over the
// whole row.  Rows of up to kSmallV take one launch, k_sample_small.
//
// Measured: one row of 262144 with top-k 64 and top-p: 18 us, of which the
// draw's single workgroup takes 11, step after step.  32 rows of 32 users,
// softcapped: 49 us.  128 rows (134 MB) by top-p: 130 us; the first pass takes
// 28 (4.7 TB/s), the second and third are bound by issuing their 64-bit
// arithmetic (the second 51, 38 without it).  50 rows of 10007 in one launch:
// 25 us.  The walk costs a pass over the row by one workgroup for every round:
// a row of 262144 with top-k 1025 takes 213 us (1024: 91), with top-k 5000 and
// top-p 424, by top-p over equal values or quarters 715 to 720 (distinct ones:
// 29); 32 such rows 296, 517 and 808 to 835.
#include "chn_internal.h"

#include <cmath>

namespace chn {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kSampleMaxV = 1u << 20;
constexpr int kWeightBits = 43;
constexpr uint32_t kStretch = 2048;         // values of a wave: one sum, 32 blocks
constexpr uint32_t kBins = 2048;            // of 2^-6 powers of two each: 32 powers, the rest (2^-32 of the largest) in the last
constexpr uint32_t kList = 4096;            // tokens of a row's list: 32 KB of LDS
constexpr uint32_t kMaxK = 1024;            // top-k by block maxima: a thread per kept token
constexpr uint32_t kDrawThreads = 1024;
// Two waves per stretch, as a wave's values are one chain of 64-bit arithmetic (one wave: 57 us instead of 50 at 32 users);
// 4 stretches a workgroup, which share a histogram: 256, 512 and 1024 threads take 182, 130 and 131 us at 128 rows by
// top-p (histograms merged more or less often), 51, 50 and 55 at 32 users
constexpr uint32_t kPassThreads = 512, kPassStretches = kPassThreads / 128;
constexpr uint32_t kRowsAtOnce = 1024;      // rows that share the workspace (64 KB a row at 262144)

struct Sample {
    const float *logits;
    uint32_t V, ld;
    const float *temperature;
    const uint32_t *top_k;
    const float *top_p, *min_p, *u;
    float softcap;
    uint32_t *tokens;
    float *probs;
    // workspace, per row: block maxima and stretch maxima (orderable, 0: nothing allowed), sums of stretches, the
    // histogram, the list and its length
    uint32_t blocks, stretches;
    uint32_t *bmax, *smax;
    uint64_t *sums, *hist, *list;
    uint32_t *listed;
};

__device__ __forceinline__ bool allowed(float v) { return v > -3.4028234663852886e38f; }   // not NaN either
__device__ __forceinline__ uint32_t orderable(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);                             // -0 orders as +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
    return __builtin_bit_cast(float, (o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ uint64_t token_key(float v, uint32_t i) {
    return ((uint64_t)orderable(v) << 32) | (0xFFFFFFFFu - i);
}

// a b + c, c in scalar registers (otherwise it is moved into vector registers
// before every use)
__device__ __forceinline__ double fma_s(double a, double b, double c) {
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
    return d;
}
// exp on half a power of two either way: x = n ln 2 + r, and (exp(r) - 1) by
// its series (the 13th term is below 2^-52 of the first).
struct Exp {
    double em1, n;
    __device__ __forceinline__ explicit Exp(double x) {
        const double t = x * 1.4426950408889634074;
        n = rint(t);
        const double r = (t - n) * 0.69314718055994530942;
        double p = fma(1.0 / 479001600.0, r, 1.0 / 39916800.0);
        p = fma_s(p, r, 1.0 / 3628800.0);
        p = fma_s(p, r, 1.0 / 362880.0);
        p = fma_s(p, r, 1.0 / 40320.0);
        p = fma_s(p, r, 1.0 / 5040.0);
        p = fma_s(p, r, 1.0 / 720.0);
        p = fma_s(p, r, 1.0 / 120.0);
        p = fma_s(p, r, 1.0 / 24.0);
        p = fma_s(p, r, 1.0 / 6.0);
        p = fma(p, r, 0.5);
        p = fma(p, r, 1.0);
        em1 = p * r;
    }
};
// 2^t for -1000 < t < 900 as part * scale, scale a power of two times
// 2^kWeightBits: 2^f on half a power of two either way by its series, whose
// 12th term is 2^-47 of the first: a sixteenth of a weight's unit.
struct Pow2 {
    double part, scale;
    __device__ __forceinline__ explicit Pow2(double t) {
        constexpr double L = 0.69314718055994530942, c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5,
                         c6 = c5 * L / 6, c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9, c10 = c9 * L / 10,
                         c11 = c10 * L / 11;
        const double n = rint(t), f = t - n;
        double p = fma_s(f, c11, c10);
        p = fma_s(p, f, c9);
        p = fma_s(p, f, c8);
        p = fma_s(p, f, c7);
        p = fma_s(p, f, c6);
        p = fma_s(p, f, c5);
        p = fma_s(p, f, c4);
        p = fma_s(p, f, c3);
        p = fma_s(p, f, c2);
        p = fma_s(p, f, L);
        part = fma(p, f, 1.0);
        scale = __builtin_bit_cast(double, (uint64_t)(uint32_t)(((int)n + kWeightBits + 1023) << 20) << 32);
    }
};
// tanh(y) from exp(-2 |y|) - 1, which keeps its digits near 0
__device__ __forceinline__ double tanh_of(double y) {
    const Exp e(fmax(-2.0 * fabs(y), -64.0));
    const double s = ldexp(1.0, (int)e.n), m = fma(s, e.em1, s - 1.0);
    return copysign(-m / (2.0 + m), y);
}

// A row's settings and the weights of its tokens: cap * tanh(l / cap) (or l)
// relative to the row's largest.
template <bool CAP>
struct Row {
    double cap, inv_cap, top, powers;   // powers: log2(e) / T
    float raw_top, bin_scale;
    uint64_t least;                // min_p, as a weight
    uint32_t k;                    // 0: no top-k
    float p;                       // 1: no top-p
    bool some, greedy;             // a token is allowed; the largest is taken

    __device__ __forceinline__ Row(const Sample &a, uint32_t row, uint32_t largest) {
        const float T = a.temperature ? a.temperature[row] : 1.0f;
        some = largest != 0;
        greedy = !(T > 0.0f);
        raw_top = value_of(largest);
        cap = a.softcap;
        inv_cap = 1.0 / cap;
        powers = 1.4426950408889634074 / (double)T;
        top = capped(raw_top);
        // 64 bins per power of two of the weight where the cap does not flatten it
        bin_scale = fminf((float)(64.0 * powers), 1e30f);
        const uint32_t kk = a.top_k ? a.top_k[row] : 0u;
        k = kk < a.V ? kk : 0u;
        const float pp = a.top_p ? a.top_p[row] : 1.0f, mm = a.min_p ? a.min_p[row] : 0.0f;
        p = pp < 1.0f ? fmaxf(pp, 0.0f) : 1.0f;
        least = mm > 0.0f ? (uint64_t)ceil(fmin((double)mm, 1.0) * (double)(1ull << kWeightBits)) : 0;
    }
    __device__ __forceinline__ double capped(float l) const {
        return CAP ? cap * tanh_of((double)l * inv_cap) : (double)l;
    }
    // a token's weight: no branch, so that several run side by side.  Below 2^-90 it is zero units anyway; a NaN (of
    // infinities) ends there too
    __device__ __forceinline__ Pow2 power(float l) const {
        double x = fmax((capped(l) - top) * powers, -90.0);
        if (CAP) x = fmin(x, 0.0);                                     // tanh need not grow in its last bit
        return Pow2(l == raw_top ? 0.0 : x);
    }
    __device__ __forceinline__ double weight(float l) const {                              // 2^kWeightBits exp(..)
        const Pow2 w = power(l);
        return w.part * w.scale;
    }
    // 2^52 added leaves the rounded weight in the low bits
    __device__ __forceinline__ uint64_t units(float l) const {
        const Pow2 w = power(l);
        return __builtin_bit_cast(uint64_t, fma(w.part, w.scale, 4503599627370496.0)) & ((1ull << 52) - 1);
    }
    __device__ __forceinline__ uint64_t units_if_allowed(float l) const {
        const uint64_t w = units(l);
        return allowed(l) ? w : 0;
    }
    __device__ __forceinline__ uint64_t kept(uint64_t w) const { return w >= least ? w : 0; }
    // the bin of an allowed logit: larger logits never lie in a later one
    __device__ __forceinline__ uint32_t bin(float l) const {
        return (uint32_t)fminf((raw_top - l) * bin_scale, (float)(kBins - 1));     // all in the last, if the largest is infinite
    }
    // the running sum at which top-p ends, of a mass Z: kept while the mass before is below p Z, so the last one is
    // the first whose running sum reaches ceil(p Z)
    __device__ __forceinline__ uint64_t goal(uint64_t Z) const {
        const double g = ceil((double)p * (double)Z);
        const uint64_t n = g < 1.0 ? 1 : (uint64_t)g;
        return n < Z ? n : Z;
    }
};

__device__ __forceinline__ uint64_t wave_min_u64(uint64_t v) {
    v = min(v, dpp64<0x111, 0xF>(v, v));
    v = min(v, dpp64<0x112, 0xF>(v, v));
    v = min(v, dpp64<0x114, 0xF>(v, v));
    v = min(v, dpp64<0x118, 0xF>(v, v));
    v = min(v, dpp64<0x142, 0xA>(v, v));
    return lane64(min(v, dpp64<0x143, 0xC>(v, v)), 63);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor(v, o, 64));
    return v;
}

// A wave's stretch of 2048 values, four per lane and load (rows start at any
// 4-byte address), half of it in registers at a time; NaN behind the row's end.
struct Stretch {
    f4u v[4];

    __device__ __forceinline__ void load(const Sample &a, const float *x, uint32_t s, int j, f4u &d) {
        const uint32_t i = s * kStretch + 4 * (threadIdx.x & 63) + 256 * j;
        if (i + 4 <= a.V) d = *(const f4u *)(x + i);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = i + e < a.V ? x[i + e] : __builtin_nanf("");
    }
    __device__ __forceinline__ void start(const Sample &a, const float *x, uint32_t s, int h) {
#pragma unroll
        for (int j = 0; j < 4; ++j) load(a, x, s, 4 * h + j, v[j]);
    }
    // f(index of the first, four values, number of the load) for the half of stretch s that is here
    template <typename F>
    __device__ __forceinline__ void half(uint32_t s, int h, F &&f) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f(s * kStretch + 4 * (threadIdx.x & 63) + 256 * (4 * h + j), v[j], 4 * h + j);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};
// f over both halves
template <typename F>
__device__ __forceinline__ void stretch(const Sample &a, const float *x, uint32_t s, F &&f) {
    Stretch v[2];
    v[0].start(a, x, s, 0);
    v[1].start(a, x, s, 1);
    v[0].half(s, 0, f);
    v[1].half(s, 1, f);
}

// the row's largest logit, by every wave
__device__ __forceinline__ uint32_t row_top(const Sample &a, uint32_t row) {
    uint32_t m = 0;
    for (uint32_t i = threadIdx.x & 63; i < a.stretches; i += 64) m = max(m, a.smax[(size_t)row * a.stretches + i]);
    return wave_max_u32(m);
}

// Rows whose weights k_sample_mass sums: neither greedy nor with top-k.
__device__ __forceinline__ bool by_mass(const Sample &a, uint32_t row) {
    return (!a.temperature || a.temperature[row] > 0.0f) && (!a.top_k || a.top_k[row] == 0 || a.top_k[row] >= a.V);
}

// A wave per stretch: maxima of 64 (16 lanes of a load) and of all.  The
// row's first workgroup clears its histogram.
__global__ __launch_bounds__(256) void k_sample_max(Sample a) {
    const uint32_t row = blockIdx.y, s = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (blockIdx.x == 0) {
        for (uint32_t i = threadIdx.x; i < kBins; i += 256) a.hist[(size_t)row * kBins + i] = 0;
        if (threadIdx.x == 0) a.listed[row] = 0;
    }
    if (s >= a.stretches) return;
    float most = -__builtin_inff();
    stretch(a, a.logits + (size_t)row * a.ld, s,
            [&](uint32_t, const f4u &v, int j) {
                float m = -__builtin_inff();
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, allowed(v[e]) ? v[e] : -__builtin_inff());
                m = row16_max(m);
                const uint32_t b = s * 32 + 4 * j + (lane >> 4);
                if ((lane & 15) == 0 && b < a.blocks) a.bmax[(size_t)row * a.blocks + b] = allowed(m) ? orderable(m) : 0u;
                most = fmaxf(most, m);
            });
    most = wave_max64(most);
    if (lane == 0) a.smax[(size_t)row * a.stretches + s] = allowed(most) ? orderable(most) : 0u;
}

// The sums of the stretches from the waves' (two waves take a stretch); all
// threads, part: a word per wave.
__device__ __forceinline__ void put_sums(const Sample &a, uint32_t row, uint64_t sum, uint64_t *part) {
    sum = wave_sum_u64(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    const uint32_t t = threadIdx.x, s = blockIdx.x * kPassStretches + t;
    if (t < kPassStretches && s < a.stretches) a.sums[(size_t)row * a.stretches + s] = part[2 * t] + part[2 * t + 1];
}

// Rows without top-k: the histogram of the weights (with top-p), or the sums of
// the stretches.
template <bool CAP>
__global__ __launch_bounds__(kPassThreads) void k_sample_mass(Sample a) {
    __shared__ uint64_t hist[kBins];
    const uint32_t row = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t s = blockIdx.x * kPassStretches + wave / 2;
    if (!by_mass(a, row)) return;                                    // the whole workgroup
    const float *x = a.logits + (size_t)row * a.ld;
    Stretch v;
    if (s < a.stretches) v.start(a, x, s, wave % 2);                            // while the row's settings and bins are prepared
    __builtin_amdgcn_sched_barrier(0);
    const Row<CAP> r(a, row, row_top(a, row));
    if (r.p < 1.0f) {
        for (uint32_t i = threadIdx.x; i < kBins; i += blockDim.x) hist[i] = 0;
        __syncthreads();
        if (s < a.stretches)
            v.half(s, wave % 2,
                   [&](uint32_t, const f4u &l, int) {
                       uint64_t w[4];
#pragma unroll
                       for (int e = 0; e < 4; ++e) w[e] = r.units(l[e]);
#pragma unroll
                       for (int e = 0; e < 4; ++e)
                           if (w[e] && allowed(l[e])) atomicAdd((unsigned long long *)&hist[r.bin(l[e])], (unsigned long long)w[e]);
                   });
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kBins; i += blockDim.x)
            if (hist[i]) atomicAdd((unsigned long long *)&a.hist[(size_t)row * kBins + i], (unsigned long long)hist[i]);
    } else {
        uint64_t sum = 0;
        if (s < a.stretches)
            v.half(s, wave % 2, [&](uint32_t, const f4u &l, int) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += r.kept(r.units_if_allowed(l[e]));
                asm volatile("" : "+v"(sum));                          // summed here, not kept apart until the end
            });
        put_sums(a, row, sum, hist);
    }
}

// The bin in which a row's running sum reaches its goal, and the goal's rest
// there.  All threads; sh: 20 words.
template <bool CAP>
__device__ __forceinline__ uint32_t border_bin(const Sample &a, const Row<CAP> &r, uint32_t row, uint64_t *sh, uint64_t &rest) {
    const uint32_t tid = threadIdx.x, nt = blockDim.x, per = kBins / nt;       // 512 or 1024 threads: 4 or 2 bins
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = nt >> 6;
    const uint64_t *h = a.hist + (size_t)row * kBins + tid * per;
    uint64_t own = 0;
    for (uint32_t i = 0; i < per; ++i) own += h[i];
    const uint64_t incl = wave_scan_u64(own);
    if (lane == 63) sh[wave] = incl;
    __syncthreads();
    const uint64_t waves = row16_scan_u64((lane & 15) < nw ? sh[lane & 15] : 0), Z = lane64(waves, 15);
    uint64_t before = incl - own + (wave ? lane64(waves, wave - 1) : 0);
    const uint64_t g = r.goal(Z);
    if (before < g && before + own >= g) {
        uint32_t b = tid * per;
        for (; before + *h < g; ++h, ++b) before += *h;
        sh[18] = b;
        sh[19] = g - before;
    }
    __syncthreads();
    rest = sh[19];
    return (uint32_t)sh[18];
}

// Rows with top-p and without top-k: the tokens of the border's bin into the
// list, the kept weights above it summed by stretch.  A tenth to a half of a
// row's tokens lie above: they are queued, and their weights (64-bit
// arithmetic) formed by full waves.
template <bool CAP>
__global__ __launch_bounds__(kPassThreads) void k_sample_border(Sample a) {
    constexpr uint32_t kMine = 1024;                                     // the workgroup's share of the list
    __shared__ uint64_t sh[20], found[kMine];
    __shared__ float queue[kPassThreads / 64][512];
    __shared__ uint32_t nfound, at0;
    const uint32_t row = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t s = blockIdx.x * kPassStretches + wave / 2;
    const int lane = threadIdx.x & 63;
    if (!by_mass(a, row) || !(a.top_p[row] < 1.0f)) return;
    const float *x = a.logits + (size_t)row * a.ld;
    Stretch v;
    if (s < a.stretches) v.start(a, x, s, wave % 2);
    __builtin_amdgcn_sched_barrier(0);
    const Row<CAP> r(a, row, row_top(a, row));
    if (!r.some) return;
    uint64_t rest;
    const uint32_t border = border_bin(a, r, row, sh, rest);
    if (threadIdx.x == 0) nfound = 0;
    __syncthreads();
    float *q = queue[threadIdx.x >> 6];
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    auto fence = [] {                                                    // the wave reads what it wrote
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    uint64_t sum = 0;
    if (s < a.stretches) {
        uint32_t n = 0;                                                  // queued, below 256 between steps
        v.half(s, wave % 2, [&](uint32_t i, const f4u &l, int) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t b = allowed(l[e]) ? r.bin(l[e]) : kBins;
                const uint64_t over = __ballot(b < border), in = __ballot(b == border);
                if (b < border) q[n + __popcll(over & below)] = l[e];
                n += __popcll(over);
                if (in) {                                                // one atomic for the wave's
                    const int first = __ffsll((unsigned long long)in) - 1;
                    uint32_t at = 0;
                    if (lane == first) at = atomicAdd(&nfound, (uint32_t)__popcll(in));
                    at = __shfl(at, first, 64) + (uint32_t)__popcll(in & below);
                    if (b == border && at < kMine) found[at] = token_key(l[e], i + e);
                }
            }
            if (n >= 256) {                                              // four a lane, side by side
                fence();
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += r.kept(r.units(q[64 * e + lane]));
                asm volatile("" : "+v"(sum));
                n -= 256;
                float tail[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) tail[e] = q[256 + 64 * e + lane];
                fence();
#pragma unroll
                for (int e = 0; e < 4; ++e) q[64 * e + lane] = tail[e];
            }
        });
        fence();
        for (uint32_t e = lane; e < n; e += 64) sum += r.kept(r.units(q[e]));
    }
    put_sums(a, row, sum, sh);
    __syncthreads();
    // more than its share: the row's list counts as full
    if (threadIdx.x == 0 && nfound) at0 = atomicAdd(&a.listed[row], nfound <= kMine ? nfound : kList + 1);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < min(nfound, kMine); i += blockDim.x)
        if (at0 + i < kList) a.list[(size_t)row * kList + at0 + i] = found[i];
}

// LDS and steps of a workgroup of kDrawThreads that looks for a row's border.
constexpr uint32_t kDigits = 2 * kDrawThreads;
struct Group {
    static constexpr int NW = kDrawThreads / 64;
    static_assert(NW == 16, "the waves' parts are a row of 16 lanes");
    uint64_t hist_w[kDigits], part[NW], part2[NW], found[4];
    uint32_t hist_n[kDigits], n, hit;

    __device__ __forceinline__ uint64_t sum(uint64_t v) {
        v = wave_sum_u64(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        return lane64(row16_scan_u64(part[threadIdx.x & 15]), 15);
    }
    __device__ __forceinline__ uint64_t least(uint64_t v) {
        v = wave_min_u64(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        return wave_min_u64(part[threadIdx.x & 15]);
    }
    // the largest and the smallest
    __device__ __forceinline__ void ends(uint64_t &hi, uint64_t &lo) {
        hi = wave_min_u64(~hi);
        lo = wave_min_u64(lo);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            part[threadIdx.x >> 6] = hi;
            part2[threadIdx.x >> 6] = lo;
        }
        __syncthreads();
        hi = ~wave_min_u64(part[threadIdx.x & 15]);
        lo = wave_min_u64(part2[threadIdx.x & 15]);
    }
    // inclusive running sum over the threads, and the whole sum
    __device__ __forceinline__ uint64_t scan(uint64_t v, uint64_t &total) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        v = wave_scan_u64(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 63) part[wave] = v;
        __syncthreads();
        const uint64_t waves = row16_scan_u64(part[threadIdx.x & 15]);
        total = lane64(waves, 15);
        return v + (wave ? lane64(waves, wave - 1) : 0);
    }
    // every(f): f(key, weight()) for all tokens looked through.  The key of the last token of the order, from those in
    // [lo, hi], that the running count (or sum of weights) needs to reach `goal`: the range in up to 2048 parts, then the
    // part that holds it, until that is wanted whole.
    template <typename F>
    __device__ __forceinline__ uint64_t last_key(F &&every, uint64_t lo, uint64_t hi, bool by_weight, uint64_t goal) {
        const uint32_t tid = threadIdx.x;
        // each round leaves at most 2^-10 of the range: six at most
        for (int round = 0; round < 7; ++round) {
            const int bits = 64 - __clzll((long long)(hi - lo)), shift = hi == lo ? 0 : max(bits - 11, 0);
            __syncthreads();
            for (uint32_t i = tid; i < kDigits; i += kDrawThreads) {
                hist_n[i] = 0;
                hist_w[i] = 0;
            }
            __syncthreads();
            every([&](uint64_t key, auto &&weight) {
                if (key < lo || key > hi) return;
                const uint32_t d = (uint32_t)((key - lo) >> shift);
                atomicAdd(&hist_n[d], 1u);
                if (by_weight) atomicAdd((unsigned long long *)&hist_w[d], (unsigned long long)weight());
            });
            __syncthreads();
            // thread 0 has the two largest parts
            const uint32_t d = kDigits - 1 - 2 * tid;
            const uint64_t c0 = by_weight ? hist_w[d] : hist_n[d], c1 = by_weight ? hist_w[d - 1] : hist_n[d - 1];
            uint64_t total;
            uint64_t before = scan(c0 + c1, total) - c0 - c1;
            if (before < goal && before + c0 + c1 >= goal) {
                const bool second = before + c0 < goal;
                before += second ? c0 : 0;
                const uint32_t cnt = hist_n[d - second];
                found[0] = d - second;
                found[1] = before;
                found[2] = shift == 0 || cnt == 1 || (!by_weight && before + cnt == goal);
            }
            __syncthreads();
            lo += found[0] << shift;
            // (one type on both sides: min of unsigned long and unsigned long long is the one for doubles)
            hi = min(hi, lo + (((uint64_t)1 << shift) - 1));
            goal -= found[1];
            if (found[2]) break;
        }
        return lo;
    }
};

// What the draw looks for in a sum of Z: a running sum above this.
__device__ __forceinline__ uint64_t target_of(float u, uint64_t Z) {
    const double want = (u > 0.0f ? (double)u : 0.0) * (double)Z;
    const uint64_t t = want >= (double)Z ? Z - 1 : (uint64_t)want;
    return t < Z ? t : Z - 1;
}

// The draw of a row with top-k from a list of n tokens that holds its k <= kMaxK
// largest.  sorted: kMaxK words.
template <bool CAP, typename F>
__device__ __forceinline__ void draw_listed(const Row<CAP> &r, Group &sh, uint64_t *list, uint64_t *sorted, uint32_t n, float u,
                                            F &&finish) {
    const uint32_t tid = threadIdx.x;
    if (tid == 0 && n % 2) list[n] = 0;                                // below every key
    __syncthreads();
    // the k largest, in order: a thread counts what is larger than its key
    for (uint32_t i = tid; i < n; i += kDrawThreads) {
        const uint64_t key = list[i];
        uint32_t rank = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < n; j += 2) {                          // two a read
            const ulonglong2 o = *(const ulonglong2 *)(list + j);
            rank += (o.x > key ? 1u : 0u) + (o.y > key ? 1u : 0u);
        }
        if (rank < r.k) sorted[rank] = key;
    }
    __syncthreads();
    const uint32_t k = min(n, r.k);
    const uint64_t key = tid < k ? sorted[tid] : 0;
    const uint64_t w = tid < k ? r.units(value_of(key >> 32)) : 0;
    uint64_t Z, total;
    const uint64_t incl = sh.scan(w, Z);
    bool in = tid < k;
    if (r.p < 1.0f) in = in && incl - w < r.goal(Z);
    const uint64_t kw = in ? r.kept(w) : 0;
    (void)sh.scan(kw, total);
    const uint64_t target = target_of(u, total);
    // the draw goes by index: a kept token sums the kept ones before it, which are among the first of the order
    list[tid] = kw;
    const uint32_t first = __syncthreads_count(in);
    if (kw) {
        uint64_t before = 0;
        const uint32_t mine = (uint32_t)key;                           // ~index: larger for lower indexes
#pragma unroll 8
        for (uint32_t j = 0; j < first; ++j) {
            const uint64_t other = list[j];                          // read either way: no branch, so reads overlap
            before += (uint32_t)sorted[j] > mine ? other : 0;
        }
        if (before <= target && before + kw > target)
            finish(0xFFFFFFFFu - mine, (float)(r.weight(value_of(key >> 32)) / (double)total));
    }
}

// Rows of up to kSmallV: one launch, a workgroup per row, which holds the row in
// registers (thread t: values J t .. J t + J - 1; J as few as V needs: 50 rows
// of 10007 take 25 us with J = 12 and 35 with 16).  One workgroup's steps are
// latency after latency, but fewer than those of four launches: 50 rows of
// 10007 25 us and 47; one and 128 rows of 16000 with top-k 14 and 17 against 18
// and 20.  By top-p alone, which only the device knows of a row, it is nearly
// even there: 1, 20, 50 and 128 rows of 16000 28.5, 30, 30.5 and 32 us against
// 26, 28.5, 31 and 33.  J = 16 spills already (26 registers, softcapped 54), and
// with more values the rows would not stay in registers.
constexpr uint32_t kSmallV = 16 * kDrawThreads;
template <int J, bool CAP>
__global__ __launch_bounds__(kDrawThreads) void k_sample_small(Sample a) {
    constexpr uint32_t kShort = 2048;                                  // a list of the largest
    __shared__ Group sh;
    __shared__ __align__(16) uint64_t list[kShort];
    __shared__ uint64_t sorted[kMaxK];
    const uint32_t tid = threadIdx.x, row = blockIdx.x, i0 = tid * J;
    const float *x = a.logits + (size_t)row * a.ld;
    float v[J];
#pragma unroll
    for (int j = 0; j < J; j += 4) {
        if (i0 + j + 4 <= a.V) {
            const f4u y = *(const f4u *)(x + i0 + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j + e] = y[e];
        } else
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j + e] = i0 + j + e < a.V ? x[i0 + j + e] : __builtin_nanf("");
    }
    const float u = a.u[row];
    if (tid == 0) sh.n = 0;
    for (uint32_t i = tid; i < kDigits; i += kDrawThreads) sh.hist_n[i] = 0;
    uint64_t hi = 0, lo = ~0ull;
    auto key_of = [&](int j) { return allowed(v[j]) ? token_key(v[j], i0 + j) : 0; };
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const uint64_t key = key_of(j);
        hi = max(hi, key);
        lo = key ? min(lo, key) : lo;
    }
    sh.ends(hi, lo);
    const Row<CAP> r(a, row, (uint32_t)(hi >> 32));
    auto finish = [&](uint32_t token, float prob) {
        a.tokens[row] = token;
        if (a.probs) a.probs[row] = prob;
    };
    if (!r.some || r.greedy) {
        if (tid == 0) finish(r.some ? 0xFFFFFFFFu - (uint32_t)hi : CHN_NO_TOKEN, r.some ? 1.0f : 0.0f);
        return;
    }
    if (r.k) {
        // the logits in up to 2048 parts between the smallest and the largest: where the running count from the top reaches
        // k, k tokens are that large
        const uint32_t least = (uint32_t)(lo >> 32), range = (uint32_t)(hi >> 32) - least;
        const int shift = max(32 - __clz(range) - 11, 0);              // range 0: 0
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (allowed(v[j])) atomicAdd(&sh.hist_n[(orderable(v[j]) - least) >> shift], 1u);
        __syncthreads();
        const uint32_t e = kDigits - 1 - 2 * tid, c0 = sh.hist_n[e], c1 = sh.hist_n[e - 1];
        uint64_t n;
        const uint64_t before = sh.scan(c0 + c1, n) - c0 - c1;
        if (n > r.k) {
            if (before < r.k && before + c0 + c1 >= r.k) sh.found[0] = e - (before + c0 < r.k);
            __syncthreads();
            const uint32_t floor_key = least + ((uint32_t)sh.found[0] << shift);
            if (r.k <= kMaxK) {
#pragma unroll
                for (int j = 0; j < J; ++j)
                    if (allowed(v[j]) && orderable(v[j]) >= floor_key) {
                        const uint32_t at = atomicAdd(&sh.n, 1u);
                        if (at < kShort) list[at] = token_key(v[j], i0 + j);
                    }
                __syncthreads();
                if (sh.n <= kShort) {
                    draw_listed(r, sh, list, sorted, sh.n, u, finish);
                    return;
                }
            }
            // many equal or near equal ones, or many wanted: key by key
            lo = sh.last_key(
                [&](auto &&f) {
#pragma unroll
                    for (int j = 0; j < J; ++j) f(key_of(j), [] { return (uint64_t)1; });   // key 0 is below lo
                },
                lo, hi, false, r.k);
        }
    }
    uint64_t w[J], Z = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        w[j] = 0;
        if (key_of(j) >= lo) w[j] = r.units(v[j]);
        Z += w[j];
        if (j % 2) __builtin_amdgcn_sched_barrier(0);                  // two at a time: the registers are full
    }
    if (r.p < 1.0f) {
        Z = sh.sum(Z);
        lo = sh.last_key(
            [&](auto &&f) {
#pragma unroll
                for (int j = 0; j < J; ++j) f(key_of(j), [&] { return w[j]; });
            },
            lo, hi, true, r.goal(Z));
    }
    uint64_t own = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        w[j] = key_of(j) >= lo ? r.kept(w[j]) : 0;
        own += w[j];
    }
    const uint64_t incl = sh.scan(own, Z), target = target_of(u, Z);
    if (own && incl > target && incl - own <= target) {                // one thread
        uint64_t run = incl - own;
        uint32_t token = 0;
        float l = 0.0f;
        bool hit = false;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            run += w[j];
            if (!hit && run > target) {
                hit = true;
                token = i0 + j;
                l = v[j];
            }
        }
        finish(token, (float)(r.weight(l) / (double)Z));
    }
}

// LDS of k_sample_draw.
struct Draw {
    __align__(16) uint64_t list[kList];
    Group g;
};

// A workgroup per row: the kept tokens' last key, then the draw.
template <bool CAP>
__global__ __launch_bounds__(kDrawThreads) void k_sample_draw(Sample a) {
    extern __shared__ __align__(16) uint64_t lds[];
    constexpr int NW = Group::NW;
    Draw &d = *(Draw *)lds;
    Group &sh = d.g;
    uint32_t *spare = (uint32_t *)(lds + sizeof(Draw) / 8);          // block maxima, then blocks; or sums of stretches
    const uint32_t tid = threadIdx.x, row = blockIdx.x;
    const int lane = tid & 63, wave = tid >> 6;
    const float *x = a.logits + (size_t)row * a.ld;
    const uint32_t *bmax = a.bmax + (size_t)row * a.blocks;
    const float u = a.u[row];
    // the first block maxima, on their way while the settings are looked at
    uint32_t first[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) first[e] = bmax[min(tid + e * kDrawThreads, a.blocks - 1)];
    __builtin_amdgcn_sched_barrier(0);
    const Row<CAP> r(a, row, row_top(a, row));

    auto finish = [&](uint32_t token, float prob) {
        a.tokens[row] = token;
        if (a.probs) a.probs[row] = prob;
    };
    if (!r.some) {
        if (tid == 0) finish(CHN_NO_TOKEN, 0.0f);
        return;
    }
    if (r.greedy) {
        // the first block that holds the largest logit, and its first place there
        if (tid == 0) sh.hit = 0xFFFFFFFFu;
        __syncthreads();
        const uint32_t want = orderable(r.raw_top);
        for (uint32_t b = tid; b < a.blocks; b += kDrawThreads)
            if (bmax[b] == want) {
                atomicMin(&sh.hit, b);
                break;
            }
        __syncthreads();
        if (wave == 0) {
            const uint32_t i = sh.hit * 64 + lane;
            const uint64_t at = __ballot(i < a.V && x[i < a.V ? i : a.V - 1] == r.raw_top);
            if (lane == 0) finish(sh.hit * 64 + __ffsll((unsigned long long)at) - 1, 1.0f);
        }
        return;
    }
    auto whole_row = [&](auto &&f) __attribute__((always_inline)) {
        for (uint32_t i = tid; i < a.V; i += kDrawThreads) {
            const float v = x[i];
            if (allowed(v)) f(token_key(v, i), [&] { return r.units(v); });
        }
    };
    // The draw from the kept tokens of a row given the sums of its stretches (n of them, in LDS).
    auto draw_stretch = [&](uint64_t above, const uint64_t *sums) __attribute__((always_inline)) {
        uint64_t Z, own = 0;
        const uint32_t n = a.stretches;                               // at most kSampleMaxV / kStretch = 512
        own = tid < n ? sums[tid] : 0;
        const uint64_t incl = sh.scan(own, Z), target = target_of(u, Z);
        if (own && incl > target && incl - own <= target) {
            sh.hit = tid;
            sh.found[0] = target - (incl - own);
        }
        __syncthreads();
        const uint32_t i = sh.hit * kStretch + 2 * tid;
        const uint64_t rest = sh.found[0];
        float v[2];
        uint64_t w[2], total;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            v[e] = i + e < a.V ? x[i + e] : __builtin_nanf("");
            w[e] = allowed(v[e]) && token_key(v[e], i + e) >= above ? r.kept(r.units(v[e])) : 0;
        }
        uint64_t run = sh.scan(w[0] + w[1], total) - w[0] - w[1];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (w[e] && run <= rest && run + w[e] > rest) finish(i + e, (float)(r.weight(v[e]) / (double)Z));
            run += w[e];
        }
    };
    // The sums of the stretches, formed here.
    auto draw_whole = [&](uint64_t above) __attribute__((always_inline)) {
        uint64_t *sums = (uint64_t *)spare;
        for (uint32_t s = wave; s < a.stretches; s += NW) {
            uint64_t sum = 0;
            stretch(a, x, s, [&](uint32_t i, const f4u &v, int) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (allowed(v[e]) && token_key(v[e], i + e) >= above) sum += r.kept(r.units(v[e]));
            });
            sum = wave_sum_u64(sum);
            if (lane == 0) sums[s] = sum;
        }
        __syncthreads();
        draw_stretch(above, sums);
    };
    const uint64_t top_key = ((uint64_t)orderable(r.raw_top) << 32) | 0xFFFFFFFFu;
    auto least_key = [&](uint64_t &n) __attribute__((always_inline)) {                              // the row's, and how many are allowed
        uint64_t m = ~0ull;
        n = 0;
        whole_row([&](uint64_t key, auto &&) {
            m = min(m, key);
            ++n;
        });
        n = sh.sum(n);
        return sh.least(m);
    };
    auto walk = [&]() __attribute__((always_inline)) {
        uint64_t n, above = least_key(n), Z = 0;
        if (r.k && n > r.k) above = sh.last_key(whole_row, above, top_key, false, r.k);
        if (r.p < 1.0f) {
            whole_row([&](uint64_t key, auto &&weight) { Z += key >= above ? weight() : 0; });
            Z = sh.sum(Z);
            above = sh.last_key(whole_row, above, top_key, true, r.goal(Z));
        }
        draw_whole(above);
    };

    if (r.k == 0) {
        uint64_t *sums = (uint64_t *)spare;
        if (!(r.p < 1.0f)) {
            draw_stretch(1, a.sums + (size_t)row * a.stretches);
            return;
        }
        const uint32_t n = a.listed[row];
        if (n > kList) {
            walk();
            return;
        }
        uint64_t rest;
        border_bin(a, r, row, sh.hist_w, rest);
        __syncthreads();
        for (uint32_t i = tid; i < a.stretches; i += kDrawThreads) sums[i] = a.sums[(size_t)row * a.stretches + i];
        uint64_t lo = ~0ull, hi = 0;
        for (uint32_t i = tid; i < n; i += kDrawThreads) {
            const uint64_t key = a.list[(size_t)row * kList + i];
            d.list[i] = key;
            lo = min(lo, key);
            hi = max(hi, key);
        }
        lo = sh.least(lo);
        hi = ~sh.least(~hi);
        auto listed = [&](auto &&f) __attribute__((always_inline)) {
            for (uint32_t i = tid; i < n; i += kDrawThreads) {
                const uint64_t key = d.list[i];
                f(key, [&] { return r.units(value_of(key >> 32)); });
            }
        };
        // a key at or below the wanted token's and above the next listed one's; it is not below the list's smallest, so no
        // token of a later bin reaches it
        const uint64_t above = sh.last_key(listed, lo, hi, true, rest);
        listed([&](uint64_t key, auto &&weight) {
            const uint64_t w = key >= above ? r.kept(weight()) : 0;
            if (w) atomicAdd((unsigned long long *)&sums[(0xFFFFFFFFu - (uint32_t)key) / kStretch], (unsigned long long)w);
        });
        __syncthreads();
        draw_stretch(above, sums);
        return;
    }
    if (r.k > kMaxK) {
        walk();
        return;
    }
    // top-k: the tokens that can be among the k largest into the list.  The blocks' maxima in up to 2048 parts between the
    // smallest and the largest: where the running count from the top reaches k, k tokens are that large.
    if (tid == 0) sh.n = sh.hit = 0;
    bool bounded = r.k <= a.blocks;
    uint32_t floor_key = 1;
    if (bounded) {
        uint32_t least = 0xFFFFFFFFu;
        uint64_t some = 0;
        for (uint32_t b0 = tid; b0 < a.blocks; b0 += 4 * kDrawThreads) {
            uint32_t m[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const uint32_t b = b0 + e * kDrawThreads;
                m[e] = b >= a.blocks ? 0 : b0 == tid ? first[e] : bmax[b];
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                if (b0 + e * kDrawThreads < a.blocks) spare[b0 + e * kDrawThreads] = m[e];
                least = m[e] ? min(least, m[e]) : least;
                some += m[e] ? 1 : 0;
            }
        }
        for (uint32_t i = tid; i < kDigits; i += kDrawThreads) sh.hist_n[i] = 0;
        some = sh.sum(some);
        least = (uint32_t)sh.least(least);
        if (some >= r.k) {
            const uint32_t range = orderable(r.raw_top) - least;
            const int shift = max(32 - __clz(range) - 11, 0);                 // range 0: 0
            for (uint32_t b0 = tid; b0 < a.blocks; b0 += 4 * kDrawThreads) {
                uint32_t m[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) m[e] = b0 + e * kDrawThreads < a.blocks ? spare[b0 + e * kDrawThreads] : 0;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (m[e]) atomicAdd(&sh.hist_n[(m[e] - least) >> shift], 1u);
            }
            __syncthreads();
            const uint32_t e = kDigits - 1 - 2 * tid, c0 = sh.hist_n[e], c1 = sh.hist_n[e - 1];
            uint64_t total;
            const uint64_t before = sh.scan(c0 + c1, total) - c0 - c1;
            if (before < r.k && before + c0 + c1 >= r.k) sh.found[0] = e - (before + c0 < r.k);
            __syncthreads();
            floor_key = least + ((uint32_t)sh.found[0] << shift);
        }
        // those blocks' numbers, in place of the maxima: every round writes only where it and earlier ones have read
        for (uint32_t b0 = 0; b0 < a.blocks; b0 += 4 * kDrawThreads) {
            bool in[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const uint32_t b = b0 + e * kDrawThreads + tid;
                in[e] = b < a.blocks && spare[b] >= floor_key;
            }
            __syncthreads();
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (in[e]) spare[atomicAdd(&sh.hit, 1u)] = b0 + e * kDrawThreads + tid;
            __syncthreads();
        }
        const uint32_t nb = sh.hit;
        // their tokens at or above the bound
        for (uint32_t q = wave; q < nb; q += 8 * NW) {
            float v[8];
            uint32_t i[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                i[e] = spare[min(q + e * NW, nb - 1)] * 64 + lane;
                v[e] = x[min(i[e], a.V - 1)];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (q + e * NW < nb && i[e] < a.V && allowed(v[e]) && orderable(v[e]) >= floor_key) {
                    const uint32_t at = atomicAdd(&sh.n, 1u);
                    if (at < kList) d.list[at] = token_key(v[e], i[e]);
                }
        }
        __syncthreads();
        bounded = sh.n <= kList;
    }
    if (!bounded) {
        // more tokens than the list holds, or fewer blocks than k: the exact bound
        uint64_t m;
        uint64_t above = least_key(m);
        if (m > r.k) above = sh.last_key(whole_row, above, top_key, false, r.k);
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        whole_row([&](uint64_t key, auto &&) {
            if (key >= above) d.list[atomicAdd(&sh.n, 1u)] = key;         // at most k
        });
        __syncthreads();
    }
    draw_listed(r, sh, d.list, (uint64_t *)spare, sh.n, u, finish);
}

template <bool CAP>
static int launch_small(chn_ctx *ctx, const Sample &a, uint32_t n) {
    if (a.V <= 4 * kDrawThreads) k_sample_small<4, CAP><<<n, kDrawThreads, 0, ctx->stream>>>(a);
    else if (a.V <= 8 * kDrawThreads) k_sample_small<8, CAP><<<n, kDrawThreads, 0, ctx->stream>>>(a);
    else if (a.V <= 12 * kDrawThreads) k_sample_small<12, CAP><<<n, kDrawThreads, 0, ctx->stream>>>(a);
    else k_sample_small<16, CAP><<<n, kDrawThreads, 0, ctx->stream>>>(a);
    CHN_LAUNCHED(ctx, "k_sample_small");
    return CHN_OK;
}

template <bool CAP>
static void launch_rows(chn_ctx *ctx, const Sample &a, uint32_t n, size_t lds) {
    const dim3 wide((a.stretches + kPassStretches - 1) / kPassStretches, n);
    k_sample_max<<<dim3((a.stretches + 3) / 4, n), 256, 0, ctx->stream>>>(a);
    k_sample_mass<CAP><<<wide, kPassThreads, 0, ctx->stream>>>(a);
    if (a.top_p) k_sample_border<CAP><<<wide, kPassThreads, 0, ctx->stream>>>(a);
    k_sample_draw<CAP><<<n, kDrawThreads, lds, ctx->stream>>>(a);
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
    Sample a{};
    a.V = V;
    a.ld = ld;
    a.softcap = softcap;
    auto rows_from = [&](uint32_t r0) {
        a.logits = logits + (size_t)r0 * ld;
        a.temperature = temperature ? temperature + r0 : nullptr;
        a.top_k = top_k ? top_k + r0 : nullptr;
        a.top_p = top_p ? top_p + r0 : nullptr;
        a.min_p = min_p ? min_p + r0 : nullptr;
        a.u = u + r0;
        a.tokens = tokens + r0;
        a.probs = probs ? probs + r0 : nullptr;
    };
    if (V <= kSmallV) {
        rows_from(0);
        return softcap > 0.0f ? launch_small<true>(ctx, a, n_rows) : launch_small<false>(ctx, a, n_rows);
    }
    const uint32_t blocks = (V + 63) / 64, stretches = (V + kStretch - 1) / kStretch;
    const size_t rows = std::min(n_rows, kRowsAtOnce);
    const size_t row_bytes = (size_t)(stretches + kBins + kList) * 8 + (size_t)(blocks + stretches + 1) * 4;
    int rc = ensure_workspace(ctx, rows * row_bytes);
    if (rc) return rc;
    a.blocks = blocks;
    a.stretches = stretches;
    a.sums = (uint64_t *)ctx->ws;
    a.hist = a.sums + rows * stretches;
    a.list = a.hist + rows * kBins;
    a.bmax = (uint32_t *)(a.list + rows * kList);
    a.smax = a.bmax + rows * blocks;
    a.listed = a.smax + rows * stretches;
    // k_sample_draw's spare LDS: block maxima, kMaxK sorted keys, or the stretches' sums
    const size_t lds = sizeof(Draw) + std::max<size_t>({(size_t)blocks * 4, (size_t)kMaxK * 8, (size_t)stretches * 8});
    for (uint32_t r0 = 0; r0 < n_rows; r0 += kRowsAtOnce) {
        const uint32_t n = std::min(n_rows - r0, kRowsAtOnce);
        rows_from(r0);
        softcap > 0.0f ? launch_rows<true>(ctx, a, n, lds) : launch_rows<false>(ctx, a, n, lds);
        CHN_LAUNCHED(ctx, "k_sample");
    }
    return CHN_OK;
}
