// Decode attention of a batch of requests over a paged KV cache whose first
// blocks all requests share (chn_prefix_decode_attn).
//
// The query rows of one KV head - n_req * gqa of them over the prefix, gqa
// over a request's own tokens - times its keys are matrix products, on the
// fp32 matrix instructions (operands and sums in fp32, as the caches are).
// One pass over the keys: scores, weights against a running reference, the
// weighted sum of V, in registers throughout.  A launch holds two kinds of
// workgroups: prefix items (KV head, some rows, a range of keys; the prefix is
// read once per 64 or 32 rows) and own items (KV head, request, a range of its
// keys).  A second launch joins the items' partial results.
//
// Few rows (own items, and prefixes with few rows) are bound by reading the
// caches: struct Quads, 4x4x1 instructions straight from the registers the
// keys are loaded into.  Many rows over a prefix are bound by the matrix
// instructions (157 TFLOP/s in fp32): struct Rows, 16x16x4 instructions, keys
// shared through LDS.
//
// The running reference is kept per row and only moved when a score passes it
// by more than kSlack (in powers of two): weights then lie below 2^kSlack,
// which fp32 holds as exactly as those below one, and a group of keys seldom
// pays for rescaling the sums (1 us of 64 with heads of 512; nothing where
// memory bounds it).
//
// Measured (fp32, one decode step, both launches): 8 requests of up to 96
// tokens behind 512, heads of 256: 13 us, most of it the two launches and
// the block-table, key, weight and join latencies one after another.  64
// requests of up to 480 tokens behind 3968: 78 us; the prefix alone takes 57 (28
// at the matrix rate), the requests' own keys share the chip with it.  33
// requests of up to 333 behind 1488, heads of 512: 44 us, the prefix alone 38.
// 12 requests of up to 20000 tokens, no prefix: 135 us where the lengths drawn
// come to 0.81 GB, 277 where to 1.77: 6.0 to 6.4 TB/s.
#include "chn_internal.h"

#include <cmath>
#include <type_traits>

namespace chn {

typedef float f4a __attribute__((ext_vector_type(4)));

constexpr uint32_t kBadSlot = 0xFFFFFFFFu;
constexpr float kSlack = 8.0f;
constexpr float kNone = -__builtin_inff();
// 16-key groups per own item at least: one per wave, or two where items of four would not all be resident at once (12
// groups cost every case below).  Four against eight: one request of up to 4096 tokens 13.0 and 16.2 us, four of 2048
// 17.1 and 18.9; 64 of up to 500 46.5 and 42.8, 33 of 333 with heads of 512 28.9 and 24.0
constexpr uint32_t kOwnMinGroups = 4, kOwnMoreGroups = 8;

struct PrefixAttn {
    const float *q, *kc, *vc;
    const uint32_t *prefix, *tables, *lens;
    uint32_t npb, n_req, max_blocks, shift, n_blocks, num_q, num_kv, kv_dim, gqa;
    float exp_hi, exp_lo;      // scale * log2(e) in two parts
    float *out;
    // prefix items: unit u = (KV head, key range), `tiles` tiles of rows each
    uint32_t splits, split_keys, tiles, prefix_wgs, quads;
    // own items: at most own_cap + n_req of them per KV head, of which own_fit run at once
    uint32_t own_cap, own_fit;
    // partial results, [splits][n_req][num_q] of the prefix and then [own item][num_q]: sums of D values, references
    // and denominators; own_start[n_req + 1]: the first own item of each request
    float *o, *m, *l;
    uint32_t *own_start;
};

// 16-key groups of request r's own tokens.
__device__ __forceinline__ uint32_t own_groups(const PrefixAttn &a, uint32_t r) {
    const uint32_t P = a.npb << a.shift, len = min(a.lens[r], a.max_blocks << a.shift);
    return len > P ? (len - P + 15) / 16 : 0u;
}

// The own items: every request's groups are cut into ranges of `per` groups,
// per the smallest that leaves at most own_cap + n_req items.  Every wave works
// this out by itself.
__device__ __forceinline__ uint32_t own_per(const PrefixAttn &a, int lane) {
    uint64_t sum = 0;
    for (uint32_t r = lane; r < a.n_req; r += 64) sum += own_groups(a, r);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += (uint64_t)__shfl_xor((unsigned long long)sum, o, 64);
    const uint64_t per = (sum + a.own_cap - 1) / a.own_cap;
    const uint32_t least = sum / kOwnMinGroups + a.n_req / 2 > a.own_fit ? kOwnMoreGroups : kOwnMinGroups;
    return (uint32_t)min(max(per, (uint64_t)least), (uint64_t)1 << 27);           // 2^31 positions at most
}

__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v, int lane) {      // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t w = __shfl_up(v, o, 64);
        if (lane >= o) v += w;
    }
    return v;
}

// Keys [begin, end) of a list of positions that `blocks` maps, in groups of
// 16.  Key c of the group at kb has no slot if it lies past the end or its
// block is bad.
struct Keys {
    const uint32_t *blocks;
    uint32_t begin, end, kvh;
    __device__ __forceinline__ uint32_t block(const PrefixAttn &a, uint32_t kb, int c) const {
        return blocks[min(kb + c, end - 1) >> a.shift];
    }
    __device__ __forceinline__ uint32_t slot(const PrefixAttn &a, uint32_t kb, int c, uint32_t b) const {
        const uint32_t k = kb + c;
        return k < end && b < a.n_blocks ? (b << a.shift) + (k & ((1u << a.shift) - 1)) : kBadSlot;
    }
};
// What is read where a key has no slot.
static __device__ __align__(16) const float zero_row[512] = {};
// A slot's row of one KV head.
template <int D>
__device__ __forceinline__ const float *cache_row(const PrefixAttn &a, const float *cache, uint32_t slot, uint32_t kvh) {
    return slot == kBadSlot ? zero_row : cache + (size_t)slot * a.kv_dim + (size_t)kvh * D;
}

// The weight of a score against a reference: the exponent's rounding is that
// of its distance to the reference, not of the score.  A score of -inf has the
// weight zero; exp_lo, of either sign, would make its distance inf - inf.  The
// reference itself is a rounded product; from 2^24 on its half step passes a
// power of two (and the exponential's range from 2^32 on), so there the
// distance is that of the rounded products, zero for the largest.
__device__ __forceinline__ float weight(const PrefixAttn &a, float s, float ref) {
#pragma clang fp contract(off)
    const float d = s * a.exp_hi - ref;
    float e = fmaf(s, a.exp_hi, -ref);
    e = e == kNone ? e : fmaf(s, a.exp_lo, e);
    return __builtin_amdgcn_exp2f(fabsf(ref) < 16777216.0f ? e : d);
}

// 16 query rows of a wave over 256 dims, on v_mfma_f32_16x16x4_f32.  Lane l =
// 16 g + c.  Scores are formed transposed, S^T = K Q^T: as A operand lane l
// holds key c's dims 16 s + 4 g + j (one 16-byte read per s), as B operand row
// c's same dims.  The result register i of lane l is key 4 g + i of row c,
// which is the A operand of step i of P V (row c, key 4 g + i); the B operand
// of that step is V[key 4 g + i][dim 64 m + 4 c + j], again one 16-byte read.
// So nothing is exchanged between lanes but the rare rescaling.
//
// Kept here: the weighted sums (lane 16 g + c,
// element i of o[n][j]: row 4 g + i, dim 64 n + 4 c + j), and row c's reference
// and this lane's part of its denominator.  lim: how many positions row c may
// see.
struct Rows {
    f4a o[4][4];
    float m, l;
    uint32_t lim, full;

    // Rows that see no key of the range are dead: computed along, dropped in
    // end().  Groups below `full` are seen whole by every other row; behind
    // it (requests shorter than the prefix) rows see parts of them.
    __device__ __forceinline__ void start(uint32_t limit, const Keys &k) {
        m = kNone;
        l = 0.0f;
        lim = limit;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][j] = f4a{0, 0, 0, 0};
        uint32_t least = lim > k.begin ? min(lim, k.end) : k.end;
#pragma unroll
        for (int x = 8; x >= 1; x >>= 1) least = min(least, (uint32_t)__shfl_xor(least, x, 64));
        least = __builtin_amdgcn_readfirstlane(least);
        full = least >= k.end ? k.end : k.begin + (least - k.begin) / 16 * 16;
    }
    __device__ __forceinline__ void end(const Keys &k) {
        if (lim <= k.begin) {
            m = kNone;
            l = 0.0f;
        }
    }
    // The scores of a group to weights: element i is key 4 g + i of row c;
    // seen(i): whether the row sees it.
    template <typename F>
    __device__ __forceinline__ f4a softmax(const PrefixAttn &a, f4a s, F &&seen) {
        const int g = (threadIdx.x & 63) >> 4;
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = seen(i) ? s[i] * a.exp_hi : kNone;
        const float mx = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        if (__any(mx > m + kSlack)) {
            const float mn = fmaxf(m, rows4_max(mx));
            const float f = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float fr = __shfl(f, 4 * g + i, 64);
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[n][j][i] *= fr;
            }
        }
        const float ref = m == kNone ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float w = weight(a, s[i], ref);
            s[i] = seen(i) ? w : 0.0f;
        }
        l += (s[0] + s[1]) + (s[2] + s[3]);
        return s;
    }
    // Weights times V of a group that some row sees a part of, key by key: a
    // weight of zero does not keep an infinity or NaN of an unseen V row out
    // of a product, so that row is left out.  v(k): key k's V row.
    template <typename F>
    __device__ __forceinline__ void weigh_part(const f4a &s, uint32_t kb, F &&v) {
        const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
        uint32_t rl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) rl[i] = __shfl(lim, 4 * g + i, 64);
#pragma unroll 1
        for (int kg = 0; kg < 4; ++kg)
#pragma unroll
            for (int ki = 0; ki < 4; ++ki) {
                const uint32_t key = kb + 4 * kg + ki;
                const float *row = v(4 * kg + ki);
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = __shfl(s[ki], 16 * kg + 4 * g + i, 64);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const f4a x = *(const f4a *)(row + 64 * n + 4 * c);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[n][j][i] = key < rl[i] ? fmaf(p[i], x[j], o[n][j][i]) : o[n][j][i];
                }
            }
    }
};

// Nothing may move across: the loads before it are issued ahead of the
// products behind it, which run while they are under way.
__device__ __forceinline__ void issue_fence() { __builtin_amdgcn_sched_barrier(0); }

// --- few rows (RQ quads of four): the four waves take a group of 16 keys each
// in turn, on v_mfma_f32_4x4x1_16b_f32, whose 16 blocks multiply 4 x 1 by 1 x
// 4.  Lane l = 4 b + r belongs to block b.
// Scores: the blocks share out the dims (block b: 64 m + 4 b + j), A is K[key 4
// kq + r], B is q[row r]; a transposed sum over the blocks leaves lane 4 b + r
// with the score of key b and row r, one register for the whole group.
// V: every block has dims of its own (4 l + j), A is one key's weights,
// broadcast from the block that holds them, B the lane's V value.
// So K is read 256 bytes and V a whole row at a time, straight into the
// registers they are multiplied from (two buffers of 64), and four rows cost a
// quarter of what a 16-row tile would.  The query rows come from LDS (stride D
// + 16).  ONCE: the keys are a request's own, which nothing else reads:
// non-temporal loads (12 requests of up to 20000 tokens: 231 -> 207 us).
template <int D, int RQ, bool ONCE>
struct Quads {
    static constexpr int H = D / 256;
    static __device__ __forceinline__ f4a fetch(const float *p) {
        return ONCE ? __builtin_nontemporal_load((const f4a *)p) : *(const f4a *)p;
    }
    f4a o[RQ][H][4];               // element i of o[.][h][j]: row i, dim 256 h + 4 l + j
    float m[RQ], l[RQ];            // row r's reference, and this lane's part of its denominator
    uint32_t lim[RQ];              // how many positions row r may see

    // limit(row): how many positions row `row` may see.  stage() puts the query rows into LDS, for all waves, once the
    // first keys are on their way.
    template <typename F, typename G>
    __device__ __forceinline__ void run(const PrefixAttn &a, const float *sq, const Keys &k, F &&limit, G &&stage) {
        const int lane = threadIdx.x & 63, b = lane >> 2, r = lane & 3;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        uint32_t least = k.end;
#pragma unroll
        for (int x = 0; x < RQ; ++x) {
            m[x] = kNone;
            l[x] = 0.0f;
            lim[x] = limit(4 * x + r);
            if (lim[x] > k.begin) least = min(least, lim[x]);
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[x][h][j] = f4a{0, 0, 0, 0};
        }
        least = min(least, (uint32_t)__shfl_xor(least, 1, 64));
        least = min(least, (uint32_t)__shfl_xor(least, 2, 64));
        least = __builtin_amdgcn_readfirstlane(least);
        // rows that see none of these keys are dead: computed along, dropped at the end.  Up to `full` every other row
        // sees every key; behind it (requests shorter than the prefix) rows see parts of the groups
        const uint32_t full = least >= k.end ? k.end : k.begin + (least - k.begin) / 16 * 16;

        f4a A[16], B[16];
        auto load_k = [&](f4a (&d)[16], uint32_t slot, int h) {
#pragma unroll
            for (int kq = 0; kq < 4; ++kq) {
                const float *x = cache_row<D>(a, a.kc, __shfl(slot, 16 * kq + 4 * r, 64), k.kvh) + 256 * h + 4 * b;
#pragma unroll
                for (int n = 0; n < 4; ++n) d[4 * kq + n] = fetch(x + 64 * n);
            }
        };
        auto load_v = [&](f4a (&d)[16], uint32_t slot, int h) {
#pragma unroll
            for (int y = 0; y < 16; ++y)
                d[y] = fetch(cache_row<D>(a, a.vc, __builtin_amdgcn_readlane(slot, 4 * y), k.kvh) + 256 * h + 4 * lane);
        };
        // the transposed sum: lane 4 b + r gets key b's score of row r
        auto total = [&](const f4a (&c)[4]) {
            float v[8], y[4], z[2];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = swap_add32(c[i >> 2][i & 3], c[2 + (i >> 2)][i & 3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = swap_add16(v[i], v[4 + i]);
            const bool h8 = lane & 8, h4 = lane & 4;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float keep = h8 ? y[2 + i] : y[i], send = h8 ? y[i] : y[2 + i];
                z[i] = keep + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, send), 0x128, 0xF,
                                                                                 0xF, true));        // row_ror:8
            }
            const float keep = h4 ? z[1] : z[0], send = h4 ? z[0] : z[1];
            return keep + __shfl_xor(send, 4, 64);
        };
        // adds a half's scores, quad by quad
        auto scores = [&](float (&s)[RQ], const f4a (&d)[16], int h) {
#pragma unroll
            for (int x = 0; x < RQ; ++x) {
                f4a part[4];
#pragma unroll
                for (int kq = 0; kq < 4; ++kq) part[kq] = f4a{0, 0, 0, 0};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const f4a q = *(const f4a *)(sq + (4 * x + r) * (D + 16) + 256 * h + 64 * n + 4 * b);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int kq = 0; kq < 4; ++kq)
                            part[kq] = __builtin_amdgcn_mfma_f32_4x4x1f32(d[4 * kq + n][j], q[j], part[kq], 0, 0, 0);
                }
                s[x] = h ? s[x] + total(part) : total(part);
                if (RQ > 1) issue_fence();
            }
        };
        // scores to weights, in place; seen(x): whether row r of quad x sees key b
        auto softmax = [&](float (&s)[RQ], auto &&seen) {
            float t[RQ];
            bool up = false;
#pragma unroll
            for (int x = 0; x < RQ; ++x) {
                t[x] = seen(x) ? s[x] * a.exp_hi : kNone;
                up = up || t[x] > m[x] + kSlack;
            }
            if (__any(up)) {
#pragma unroll
                for (int x = 0; x < RQ; ++x) {
                    float mn = fmaxf(m[x], t[x]);
#pragma unroll
                    for (int y = 4; y <= 32; y <<= 1) mn = fmaxf(mn, __shfl_xor(mn, y, 64));
                    const float f = mn == m[x] ? 1.0f : __builtin_amdgcn_exp2f(m[x] - mn);
                    m[x] = mn;
                    l[x] *= f;
                    const f4a fr = {lane_f(f, 0), lane_f(f, 1), lane_f(f, 2), lane_f(f, 3)};
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[x][h][j] *= fr;
                }
            }
#pragma unroll
            for (int x = 0; x < RQ; ++x) {
                const float ref = m[x] == kNone ? 0.0f : m[x];
                const float w = weight(a, s[x], ref);
                s[x] = seen(x) ? w : 0.0f;
                l[x] += s[x];
            }
        };
        auto weigh = [&](const float (&s)[RQ], const f4a (&d)[16], int h) {
            static_for<16>([&](auto key) {
#pragma unroll
                for (int x = 0; x < RQ; ++x)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        o[x][h][j] = __builtin_amdgcn_mfma_f32_4x4x1f32(s[x], d[key][j], o[x][h][j], 4, key, 0);
            });
        };

        uint32_t kb = k.begin + 16 * wave;
        uint32_t slot = k.slot(a, kb, b, k.block(a, kb, b)), nextb = k.block(a, kb + 64, b);
        load_k(A, slot, 0);                        // past the end: the row of zeros, not used
        issue_fence();
        stage();
        if (kb < k.end) {
            float s[RQ];
            if (kb < full) {
                for (;;) {
                    const uint32_t next = k.slot(a, kb + 64, b, nextb);
                    nextb = k.block(a, kb + 128, b);
                    if constexpr (H == 1) {
                        load_v(B, slot, 0);
                        issue_fence();
                        scores(s, A, 0);
                    } else {
                        load_k(B, slot, 1);
                        issue_fence();
                        scores(s, A, 0);
                        issue_fence();
                        load_v(A, slot, 0);
                        issue_fence();
                        scores(s, B, 1);
                        issue_fence();
                        load_v(B, slot, 1);
                        issue_fence();
                    }
                    softmax(s, [&](int) { return slot != kBadSlot; });
                    slot = next;
                    issue_fence();
                    if constexpr (H == 1) {
                        load_k(A, slot, 0);        // past the end: the row of zeros, not used
                        issue_fence();
                        weigh(s, B, 0);
                    } else {
                        weigh(s, A, 0);
                        issue_fence();
                        load_k(A, slot, 0);
                        issue_fence();
                        weigh(s, B, 1);
                    }
                    issue_fence();
                    kb += 64;
                    if (kb >= full) break;
                }
            }
            // Groups that some row sees a part of: the weighted sum key by key, as a weight of zero does not keep an
            // infinity or NaN of an unseen V row out of a product.
#pragma unroll 1
            for (; kb < k.end; kb += 64) {
                slot = k.slot(a, kb, b, k.block(a, kb, b));
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    load_k(A, slot, h);
                    scores(s, A, h);
                }
                softmax(s, [&](int x) { return slot != kBadSlot && kb + b < lim[x]; });
#pragma unroll 1
                for (int key = 0; key < 16; ++key) {
                    const float *v = cache_row<D>(a, a.vc, __builtin_amdgcn_readlane(slot, 4 * key), k.kvh) + 4 * lane;
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const f4a y = *(const f4a *)(v + 256 * h);
#pragma unroll
                        for (int x = 0; x < RQ; ++x)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float w = lane_f(s[x], 4 * key + i);
                                if (kb + key < (uint32_t)__builtin_amdgcn_readlane(lim[x], i))
#pragma unroll
                                    for (int j = 0; j < 4; ++j) o[x][h][j][i] = fmaf(w, y[j], o[x][h][j][i]);
                            }
                    }
                }
            }
        }
#pragma unroll
        for (int x = 0; x < RQ; ++x) {
#pragma unroll
            for (int y = 4; y <= 32; y <<= 1) l[x] += __shfl_xor(l[x], y, 64);
            if (lim[x] <= k.begin) {
                m[x] = kNone;
                l[x] = 0.0f;
            }
        }
    }

    // The four waves' sums of the n first rows joined: a row's sum of D
    // values, reference and denominator as the partial result where(row).  A
    // wave without keys for a row is one whose denominator is zero: NaN scores
    // do not move the reference, but the denominator.
    template <typename F>
    __device__ __forceinline__ void join(const PrefixAttn &a, float *sh, uint32_t n, F &&where) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 3;
        constexpr int R = 4 * RQ;
        float *so = sh, *sm = sh + 4 * R * D, *sl = sm + 4 * R;
#pragma unroll
        for (int x = 0; x < RQ; ++x)
            if (lane < 4) {
                sm[wave * R + 4 * x + r] = m[x];
                sl[wave * R + 4 * x + r] = l[x];
            }
        __syncthreads();                           // and the query rows have been read
#pragma unroll
        for (int x = 0; x < RQ; ++x) {
            const float *mr = sm + 4 * x + r;
            const float M = fmaxf(fmaxf(mr[0], mr[R]), fmaxf(mr[2 * R], mr[3 * R]));
            const float f = l[x] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m[x] - M);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (4 * x + i >= (int)n) continue;
                const float fr = lane_f(f, i);
                const bool none = lane_f(l[x], i) == 0.0f;
#pragma unroll
                for (int h = 0; h < H; ++h)
                    *(f4a *)(so + (wave * R + 4 * x + i) * D + 256 * h + 4 * lane) =
                        none ? f4a{0, 0, 0, 0} : f4a{o[x][h][0][i], o[x][h][1][i], o[x][h][2][i], o[x][h][3][i]} * fr;
            }
        }
        __syncthreads();
        if (tid < (int)n) {
            const float *mr = sm + tid;
            const float M = fmaxf(fmaxf(mr[0], mr[R]), fmaxf(mr[2 * R], mr[3 * R]));
            float L = 0.0f;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const float ly = sl[y * R + tid];
                L += ly == 0.0f ? 0.0f : ly * __builtin_amdgcn_exp2f(mr[y * R] - M);
            }
            const size_t at = where(tid);
            a.m[at] = M;
            a.l[at] = L;
        }
        for (int e = tid; e < (int)n * D / 4; e += 256) {
            const int row = e / (D / 4), d = (e % (D / 4)) * 4;
            const float *s = so + row * D + d;
            *(f4a *)(a.o + where(row) * D + d) = (*(const f4a *)s + *(const f4a *)(s + R * D)) +
                                                 (*(const f4a *)(s + 2 * R * D) + *(const f4a *)(s + 3 * R * D));
        }
    }
};

// --- many rows: a wave takes 16 rows and 256 dims (of heads of 512, two waves
// the halves, whose scores they exchange) and all waves share the keys, whose K
// and V rows go through LDS, 16 at a time: the next group's loads are issued
// between the products of the scores and stored between those of the weighted
// sum (before and behind them they cost 1300 of 6900 cycles a group, of which the
// products take 4100), into a second buffer where the heads leave room for two.  (With one buffer for heads of 512, two
// workgroups fit a CU: 33 requests of up to 333 behind 1488: 60 -> 45 us.
// Another group on its way would need registers: with spills 95 -> 116 us.)  The
// query rows stay in registers.  A K row's stride of D + 4 floats spreads the 16 rows that a read
// takes over the banks.
template <int D>
struct Shared {
    static constexpr int NB = D == 512 ? 1 : 2;    // buffers
    f4a k[NB][16][D / 4 + 1], v[NB][16][D / 4], s[D == 512 ? 4 : 1][64];
    uint32_t slot[NB][16], full;
};
constexpr uint32_t rows_wg(uint32_t D) { return 64 / (D / 256); }     // rows of a workgroup
// q: row c of this wave's 16, its 256 dims; n: how many rows the workgroup has
template <int D, typename F>
__device__ __forceinline__ void run_rows(const PrefixAttn &a, Rows &w, const f4a (&q)[16], Shared<D> &sh, const Keys &k,
                                         uint32_t n, F &&where) {
    constexpr int H = D / 256, RG = 4 / H, NB = Shared<D>::NB;
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rows = wave % RG, half = wave / RG;
    f4a sk[4][H], sv[4][H];                        // keys wave, wave + 4, ..: this lane's dims 4 lane + 256 h
    auto load = [&](int x, uint32_t slot) {        // key wave + 4 x of the group
        const uint32_t s = __builtin_amdgcn_readlane(slot, wave + 4 * x);
        const float *kr = cache_row<D>(a, a.kc, s, k.kvh) + 4 * lane, *vr = cache_row<D>(a, a.vc, s, k.kvh) + 4 * lane;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            sk[x][h] = *(const f4a *)(kr + 256 * h);
            sv[x][h] = *(const f4a *)(vr + 256 * h);
        }
    };
    auto store_k = [&](int x, int b) {
#pragma unroll
        for (int h = 0; h < H; ++h) sh.k[b][wave + 4 * x][64 * h + lane] = sk[x][h];
    };
    auto store_v = [&](int x, int b) {
#pragma unroll
        for (int h = 0; h < H; ++h) sh.v[b][wave + 4 * x][64 * h + lane] = sv[x][h];
    };
    auto load_all = [&](uint32_t slot) {
#pragma unroll
        for (int x = 0; x < 4; ++x) load(x, slot);
    };
    auto store_all = [&](int b, uint32_t slot) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            store_k(x, b);
            store_v(x, b);
        }
        if (threadIdx.x < 16) sh.slot[b][threadIdx.x] = slot;
    };
    constexpr int X = 2;                           // LDS reads ahead of the products, no more: the registers are full
    f4a x[2][X];
    // beside(s): what the wave does while its products run, in eight portions
    auto scores = [&](int b, auto &&beside) {
        f4a part[4];                               // four chains: shorter sums round less
        auto read = [&](int s) {
#pragma unroll
            for (int y = 0; y < X; ++y) x[s & 1][y] = sh.k[b][c][64 * half + 4 * (X * s + y) + g];
        };
#pragma unroll
        for (int j = 0; j < 4; ++j) part[j] = f4a{0, 0, 0, 0};
        read(0);
#pragma unroll
        for (int s = 0; s < 16 / X; ++s) {
            if (s + 1 < 16 / X) read(s + 1);
            issue_fence();
#pragma unroll
            for (int y = 0; y < X; ++y)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    part[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[s & 1][y][j], q[X * s + y][j], part[j], 0, 0, 0);
            beside(s);
            issue_fence();
        }
        return (part[0] + part[1]) + (part[2] + part[3]);
    };
    // the whole heads' scores: both waves of a pair add them in the same order
    auto whole = [&](f4a s) {
        if constexpr (H == 2) {
            sh.s[wave][lane] = s;
            __syncthreads();
            const f4a o = sh.s[wave ^ RG][lane];
            s = half ? o + s : s + o;
        }
        return s;
    };
    // the i-th X of the V reads, four a key
    auto read_v = [&](int i, int b) {
#pragma unroll
        for (int y = 0; y < X; ++y) x[i & 1][y] = sh.v[b][4 * g + i * X / 4][64 * half + 16 * (i * X % 4 + y) + c];
    };
    // after read_v(0)
    auto weigh = [&](const f4a &s, int b, auto &&beside) {
#pragma unroll
        for (int i = 0; i < 16 / X; ++i) {
            if (i + 1 < 16 / X) read_v(i + 1, b);
            issue_fence();
#pragma unroll
            for (int y = 0; y < X; ++y)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f4a &o = w.o[i * X % 4 + y][j];
                    o = __builtin_amdgcn_mfma_f32_16x16x4f32(s[i * X / 4], x[i & 1][y][j], o, 0, 0, 0);
                }
            beside(i);
            issue_fence();
        }
    };
    // the groups that every row of the workgroup sees whole, then the others
    if (threadIdx.x == 0) sh.full = k.end;
    __syncthreads();
    if (lane == 0) atomicMin(&sh.full, w.full);
    uint32_t slot = k.slot(a, k.begin, c, k.block(a, k.begin, c)), nextb = k.block(a, k.begin + 16, c);
    load_all(slot);
    store_all(0, slot);
    __syncthreads();
    const uint32_t full = __builtin_amdgcn_readfirstlane(sh.full);
    uint32_t kb = k.begin;
    int b = 0;
#pragma unroll 1
    for (; kb < full; kb += 16, b ^= NB - 1) {
        slot = k.slot(a, kb + 16, c, nextb);
        nextb = k.block(a, kb + 32, c);
        const int to = b ^ (NB - 1);
        // past the end: the row of zeros, not used
        f4a s = whole(scores(b, [&](int i) {
            if (i < 4) load(i, slot);
        }));
        uint32_t vs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[i] = sh.slot[b][4 * g + i];
        read_v(0, b);
        s = w.softmax(a, s, [&](int i) { return vs[i] != kBadSlot; });
        // The next keys into the other buffer, which was last read before the barrier of the round before; with one, its K
        // part was last read before the barrier in whole()
        weigh(s, b, [&](int i) {
            if (i < 4) return;
            store_k(i - 4, to);
            if constexpr (NB == 2) store_v(i - 4, to);
        });
        if constexpr (NB == 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) store_v(i, to);
        }
        if (threadIdx.x < 16) sh.slot[to][threadIdx.x] = slot;
        __syncthreads();
    }
#pragma unroll 1
    for (; kb < k.end; kb += 16, b ^= NB - 1) {
        slot = k.slot(a, kb + 16, c, k.block(a, kb + 16, c));
        f4a s = whole(scores(b, [](int) {}));
        s = w.softmax(a, s, [&](int i) { return sh.slot[b][4 * g + i] != kBadSlot && kb + 4 * g + i < w.lim; });
        w.weigh_part(s, kb, [&](int key) { return (const float *)&sh.v[b][key][64 * half]; });
        load_all(slot);
        if constexpr (NB == 1) __syncthreads();
        store_all(b ^ (NB - 1), slot);
        __syncthreads();
    }
    w.end(k);
    const float lt = rows4_sum(w.l);
    if (half == 0 && g == 0 && rows * 16 + c < (int)n) {
        const size_t at = where(rows * 16 + c);
        a.m[at] = w.m;
        a.l[at] = lt;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t row = rows * 16 + 4 * g + i;
        if (row >= n) continue;
        float *out = a.o + where(row) * D + 256 * half + 4 * c;
#pragma unroll
        for (int y = 0; y < 4; ++y) *(f4a *)(out + 64 * y) = f4a{w.o[y][0][i], w.o[y][1][i], w.o[y][2][i], w.o[y][3][i]};
    }
}

// LDS bytes of an item: the waves' sums (the query rows take less), or the
// keys that they share.
template <int D, int RQ, bool ROWS>
constexpr size_t lds_bytes() {
    const size_t own = (4 * 4 * RQ * (D + 2)) * 4, prefix = ROWS ? sizeof(Shared<D>) : D == 256 ? (4 * 8 * (D + 2)) * 4 : 0;
    return own > prefix ? own : prefix;
}

// RQ: quads of rows of own items.  ROWS: whether prefix items hold rows_wg
// rows, 16 a wave, or one or two quads that the waves share (heads of 256).
// Two workgroups per CU where the registers can be held to 256.
template <int D, int RQ, bool ROWS>
__global__ __launch_bounds__(256, D == 256 || RQ == 1 ? 2 : 1) void k_prefix_attn(PrefixAttn a) {
    extern __shared__ f4a sh4[];
    float *const sh = (float *)sh4;
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t P = a.npb << a.shift;
    // a KV head's row: (request, head in the group)
    auto q_row = [&](uint32_t kvh, uint32_t row) {
        const uint32_t r = row / a.gqa, h = row - r * a.gqa;
        return a.q + ((size_t)r * a.num_q + kvh * a.gqa + h) * D;
    };
    // rows from `from` on into LDS, zeros behind the n that there are
    auto load_q = [&](uint32_t kvh, uint32_t from, uint32_t n, int rows) {
        for (int e = tid; e < rows * (D / 4); e += 256) {
            const uint32_t row = e / (D / 4), d = (e % (D / 4)) * 4;
            *(f4a *)(sh + row * (D + 16) + d) = row < n ? *(const f4a *)(q_row(kvh, from + row) + d) : f4a{0, 0, 0, 0};
        }
        __syncthreads();
    };
    if (blockIdx.x < a.prefix_wgs) {
        // the row tiles of one unit run on one XCD (workgroup i runs on XCD i % 8) and share its keys there
        const uint32_t R = ROWS ? rows_wg(D) : 4 * a.quads;
        const uint32_t b = blockIdx.x, tile = (b >> 3) % a.tiles, u = (b >> 3) / a.tiles * 8 + (b & 7);
        if (u >= a.num_kv * a.splits) return;
        const uint32_t kvh = u % a.num_kv, split = u / a.num_kv, begin = split * a.split_keys;
        const Keys k{a.prefix, begin, min(begin + a.split_keys, P), kvh};
        const uint32_t row0 = tile * R, n = min(a.n_req * a.gqa - row0, R);
        auto where = [&](uint32_t row) {
            const uint32_t r = (row0 + row) / a.gqa, h = (row0 + row) - r * a.gqa;
            return ((size_t)split * a.n_req + r) * a.num_q + kvh * a.gqa + h;
        };
        auto limit = [&](uint32_t row) { return row < n ? a.lens[(row0 + row) / a.gqa] : 0u; };
        if constexpr (ROWS) {
            const uint32_t mine = (tid >> 6) * 16 % R + (lane & 15);
            Rows w;
            w.start(limit(mine), k);
            f4a q[16];
            const float *x = q_row(kvh, row0 + (mine < n ? mine : 0u)) + (tid >> 6) * 16 / R * 256 + 4 * (lane >> 4);
#pragma unroll
            for (int s = 0; s < 16; ++s) q[s] = *(const f4a *)(x + 16 * s);
            run_rows<D>(a, w, q, *(Shared<D> *)sh4, k, n, where);
        } else if constexpr (D == 256) {               // heads of 512 always share
            auto quads = [&](auto Q) {
                Quads<D, Q, false> w;
                w.run(a, sh, k, limit, [&] { load_q(kvh, row0, n, 4 * Q); });
                w.join(a, sh, n, where);
            };
            if (a.quads == 1) quads(std::integral_constant<int, 1>{});
            else quads(std::integral_constant<int, 2>{});
        }
        return;
    }
    // an own item
    const uint32_t b = blockIdx.x - a.prefix_wgs, kvh = b % a.num_kv, item = b / a.num_kv;
    const uint32_t per = own_per(a, lane);
    uint32_t req = kBadSlot, first = 0, start = 0;
    for (uint32_t r0 = 0; r0 < a.n_req && (req == kBadSlot || b == 0); r0 += 64) {
        const uint32_t r = r0 + lane, n = r < a.n_req ? (own_groups(a, r) + per - 1) / per : 0u;
        const uint32_t incl = start + wave_scan_u32(n, lane);
        const uint64_t mine = __ballot(n && item >= incl - n && item < incl);
        if (mine) {
            const int x = __ffsll((unsigned long long)mine) - 1;
            req = r0 + x;
            first = item - __shfl(incl - n, x, 64);
        }
        if (b == 0 && tid < 64 && r < a.n_req) {       // for the launch that joins
            a.own_start[r] = incl - n;
            if (r == a.n_req - 1) a.own_start[a.n_req] = incl;
        }
        start = __shfl(incl, 63, 64);
    }
    if (req == kBadSlot) return;
    const uint32_t len = min(a.lens[req], a.max_blocks << a.shift), begin = P + first * per * 16;
    const Keys k{a.tables + (size_t)req * a.max_blocks, begin,
                 (uint32_t)min((uint64_t)len, (uint64_t)begin + (uint64_t)per * 16), kvh};
    Quads<D, RQ, true> w;
    w.run(a, sh, k, [&](uint32_t row) { return row < a.gqa ? k.end : 0u; },
          [&] { load_q(kvh, req * a.gqa, a.gqa, 4 * RQ); });
    w.join(a, sh, a.gqa, [&](uint32_t row) {
        return ((size_t)a.splits * a.n_req + item) * a.num_q + kvh * a.gqa + row;
    });
}

// Joins a query row's partial results: a workgroup per row, its waves take
// every fourth part, a lane four values per 256 dims.  The parts' weights are
// formed a lane each, 64 parts at a time, so the sums' loads wait for nothing
// but one another's queue.
template <int D>
__global__ __launch_bounds__(256) void k_prefix_join(PrefixAttn a) {
    __shared__ f4a sh[4][D / 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t row = blockIdx.x, r = row / a.num_q, h = row - r * a.num_q, stride = a.n_req * a.num_q;
    const uint32_t o0 = a.own_start ? a.own_start[r] : 0u, parts = a.splits + (a.own_start ? a.own_start[r + 1] - o0 : 0u);
    // part p's place; the prefix's arrays lie before the own items'
    auto at = [&](uint32_t p) {
        return p < a.splits ? (size_t)p * stride + row : (size_t)a.splits * stride + (size_t)(o0 + p - a.splits) * a.num_q + h;
    };
    float M = kNone;
    for (uint32_t p = lane; p < parts; p += 64) M = fmaxf(M, a.m[at(p)]);
    M = wave_max64(M);
    f4a acc[D / 256];
#pragma unroll
    for (int k = 0; k < D / 256; ++k) acc[k] = f4a{0, 0, 0, 0};
    float L = 0.0f;
    for (uint32_t p0 = 0; p0 < parts; p0 += 64) {
        const uint32_t n = min(parts - p0, 64u);
        float w = 0.0f, l = 0.0f;
        if ((uint32_t)lane < n) {
            const size_t i = at(p0 + lane);
            const float m = a.m[i], part = a.l[i];
            if (part != 0.0f) {                                  // NaN: whatever its reference is
                w = __builtin_amdgcn_exp2f(m - M);
                l = w * part;
            }
        }
        L += wave_sum64(l);
        constexpr int U = 4;                                     // loads in flight
        for (uint32_t p = wave; p < n; p += 4 * U) {
            f4a v[U][D / 256];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float *o = a.o + at(p0 + min(p + 4 * u, n - 1)) * D + 4 * lane;
#pragma unroll
                for (int k = 0; k < D / 256; ++k) v[u][k] = *(const f4a *)(o + 256 * k);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t q = min(p + 4 * u, n - 1);
                const float wq = lane_f(w, q);
                const bool some = p + 4 * u < n && lane_f(l, q) != 0.0f;     // a part without keys holds nothing
#pragma unroll
                for (int k = 0; k < D / 256; ++k) acc[k] += some ? wq * v[u][k] : f4a{0, 0, 0, 0};
            }
        }
    }
#pragma unroll
    for (int k = 0; k < D / 256; ++k) sh[wave][64 * k + lane] = acc[k];
    __syncthreads();
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;               // no token: zeros
    for (int e = tid; e < D / 4; e += 256)
        *(f4a *)(a.out + (size_t)row * D + 4 * e) = ((sh[0][e] + sh[1][e]) + (sh[2][e] + sh[3][e])) * inv;
}

// Own items per KV head at most: no request has more than its table has room for (`slots` of them).
static uint64_t most_own(uint32_t cap, uint32_t n_req, uint64_t slots) {
    const uint64_t groups = (slots + 15) / 16;
    return std::min<uint64_t>((uint64_t)cap + n_req, n_req * ((groups + kOwnMinGroups - 1) / kOwnMinGroups));
}

template <int D, int RQ, bool ROWS>
static void launch_items(hipStream_t st, const PrefixAttn &a, uint32_t grid) {
    constexpr size_t lds = lds_bytes<D, RQ, ROWS>();
    static_assert(lds <= 160 * 1024, "LDS per workgroup");
    k_prefix_attn<D, RQ, ROWS><<<grid, 256, lds, st>>>(a);
}

template <int D>
static int launch_prefix(chn_ctx *ctx, const PrefixAttn &a, uint32_t grid, bool rows) {
    if (grid) {
        // as few quads as the heads of a group need: 12 requests of up to 20000 tokens with 8 query heads to each of 2 KV
        // heads take 72 us with two and 90 with four, heads of 512 148 and 178.  With four the registers do not hold all
        // (15 to 21 spill): 16 query heads to one KV head of 256 take 61 us for 164 MB, 34 at a copy's rate
        if (a.gqa <= 4) rows ? launch_items<D, 1, true>(ctx->stream, a, grid) : launch_items<D, 1, false>(ctx->stream, a, grid);
        else if (a.gqa <= 8) rows ? launch_items<D, 2, true>(ctx->stream, a, grid) : launch_items<D, 2, false>(ctx->stream, a, grid);
        else rows ? launch_items<D, 4, true>(ctx->stream, a, grid) : launch_items<D, 4, false>(ctx->stream, a, grid);
        CHN_LAUNCHED(ctx, "k_prefix_attn");
    }
    k_prefix_join<D><<<a.n_req * a.num_q, 256, 0, ctx->stream>>>(a);
    CHN_LAUNCHED(ctx, "k_prefix_join");
    return CHN_OK;
}

}  // namespace chn

using namespace chn;

extern "C" int chn_prefix_decode_attn(chn_ctx *ctx, const float *q, const float *k_cache, const float *v_cache,
                                      const uint32_t *prefix_blocks, uint32_t n_prefix_blocks,
                                      const uint32_t *tables, const uint32_t *lens, uint32_t n_req,
                                      uint32_t max_blocks, uint32_t block_size, uint32_t n_blocks,
                                      uint32_t num_q_heads, uint32_t head_dim, uint32_t kv_dim, uint32_t gqa_ratio,
                                      float scale, float *out) {
    CHN_REQUIRE(ctx, q && k_cache && v_cache && tables && lens && out, "NULL argument");
    CHN_REQUIRE(ctx, !n_prefix_blocks || prefix_blocks, "NULL prefix_blocks");
    CHN_REQUIRE(ctx, head_dim == 256 || head_dim == 512, "head_dim %u must be 256 or 512", head_dim);
    CHN_REQUIRE(ctx, gqa_ratio > 0 && gqa_ratio <= 16 && num_q_heads % gqa_ratio == 0,
                "num_q_heads %u, gqa ratio %u: a ratio of 1..16 that divides the heads", num_q_heads, gqa_ratio);
    CHN_REQUIRE(ctx, num_q_heads <= 4096, "num_q_heads %u exceeds 4096", num_q_heads);
    CHN_REQUIRE(ctx, kv_dim >= (num_q_heads / gqa_ratio) * head_dim && kv_dim % 4 == 0,
                "kv_dim %u too small for %u kv heads of %u", kv_dim, num_q_heads / gqa_ratio, head_dim);
    CHN_REQUIRE(ctx, aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16),
                "q, caches and out must be 16-byte aligned");
    int rc = check_blocks(ctx, block_size, n_blocks, max_blocks);
    if (rc) return rc;
    CHN_REQUIRE(ctx, n_prefix_blocks <= max_blocks, "%u prefix blocks in tables of %u", n_prefix_blocks, max_blocks);
    CHN_REQUIRE(ctx, n_req <= 65536, "n_req %u exceeds 65536", n_req);
    if ((uint64_t)n_req * num_q_heads > kMaxGrid256)               // the joining launch's workgroups
        return set_err(ctx, CHN_E_UNSUPPORTED, "%u requests of %u heads are too many for one call", n_req, num_q_heads);
    CHN_REQUIRE(ctx, ctx, "ctx is NULL");
    if (!n_req || !num_q_heads) return CHN_OK;
    DeviceGuard dev(ctx);
    PrefixAttn a{};
    a.q = q;
    a.kc = k_cache;
    a.vc = v_cache;
    a.prefix = prefix_blocks;
    a.tables = tables;
    a.lens = lens;
    a.npb = n_prefix_blocks;
    a.n_req = n_req;
    a.max_blocks = max_blocks;
    a.shift = (uint32_t)__builtin_ctz(block_size);
    a.n_blocks = n_blocks;
    a.num_q = num_q_heads;
    a.num_kv = num_q_heads / gqa_ratio;
    a.kv_dim = kv_dim;
    a.gqa = gqa_ratio;
    const double e = (double)scale * 1.4426950408889634;
    a.exp_hi = (float)e;
    a.exp_lo = std::isfinite(a.exp_hi) ? (float)(e - a.exp_hi) : 0.0f;
    a.out = out;
    const uint32_t P = n_prefix_blocks << a.shift, M = n_req * gqa_ratio;
    // Few rows or little work with heads of 256: every workgroup of 4 or 8 rows reads the prefix for itself and its waves
    // split the keys.  Otherwise 64 (of heads of 512: 32) rows share what is read.  The one way and the other, rows x keys
    // x KV heads of 256: 16 x 512 x 8 13.5 and 18.9 us, 16 x 3968 x 8 25.4 and 32.2, 32 x 1024 x 8 19.4 and 22.5, 48 x
    // 1024 x 8 25.6 and 24.7, 24 x 2048 x 8 24.5 and 23.5, 64 x 512 x 8 25.7 and 24.0, 128 x 3968 x 8 110 and 58, 64 x
    // 3968 x 2 25.7 and 25.8; 4 of 512: 4 x 256 19.7 and 19.4, 32 x 4000 49 and 34
    const uint64_t work = (uint64_t)M * P * (num_q_heads / gqa_ratio);
    const bool by_rows = P && (head_dim == 512 || (M > 16 && work >= (M >= 64 ? 1u << 18 : 3u << 17)));
    if (P) {
        // 4 rows behind 512 and 20000 keys take 11.8 and 65 us with one quad, 14.7 and 81 with four; 16 rows 13.6 and 90
        // with twice two, 16.9 and 85 with four
        a.quads = M > 4 ? 2 : 1;
        const uint32_t R = by_rows ? rows_wg(head_dim) : 4 * a.quads;
        a.tiles = (M + R - 1) / R;
        // about one workgroup per CU, 64 keys (16 per wave) at least.  128 rows on 3968 keys with own tokens beside them:
        // 99 us with half as many workgroups, 78 so, 95 with twice as many (and twice the partial results); 132 rows of
        // heads of 512 on 1488 keys 64, 44 and 62
        const uint32_t want = std::max(1u, 256 / std::max(1u, a.tiles * a.num_kv));
        a.split_keys = ((P + want - 1) / want + 63) / 64 * 64;
        a.splits = (P + a.split_keys - 1) / a.split_keys;
        // about 256, or below 2^21: 2^24 rows by at least 32 (quads only where rows times keys are few)
        a.prefix_wgs = (a.num_kv * a.splits + 7) / 8 * 8 * a.tiles;
    }
    uint64_t grid = a.prefix_wgs, items = 0;
    if (max_blocks > n_prefix_blocks) {
        // at most about eight own items per CU: 12 requests of up to 20000 tokens take 228, 216, 205 and 211 us with
        // 512, 1024, 2048 and 4096 items; with few tokens the least groups per item decide
        a.own_cap = std::max(1u, 2048 / a.num_kv);
        // two workgroups per CU, or one (of heads of 512 another is the prefix's, or fills the registers)
        a.own_fit = (head_dim == 256 || (!P && gqa_ratio <= 4) ? 512 : 256) / a.num_kv;
        items = most_own(a.own_cap, n_req, (uint64_t)(max_blocks - n_prefix_blocks) << a.shift);
        grid += items * a.num_kv;
    }
    if (grid > kMaxGrid256) return set_err(ctx, CHN_E_UNSUPPORTED, "too many requests and heads for one call");
    const size_t rows = ((size_t)a.splits * n_req + (size_t)items) * num_q_heads;
    // What any call of these heads with no more requests and no wider tables needs, whatever its prefix, so that one at the
    // largest size readies the workspace for recordings of all.  splits * n_req falls at every new tile of rows: splits <=
    // 256 / (tiles * num_kv), tiles >= n_req * gqa / rows of a workgroup
    const uint64_t prefix_parts = std::max<uint64_t>(
        n_req, std::min<uint64_t>((uint64_t)n_req * (256 / a.num_kv), 256 * rows_wg(head_dim) / num_q_heads));
    const uint64_t own_parts = most_own(std::max(1u, 2048 / a.num_kv), n_req, (uint64_t)max_blocks << a.shift);
    rc = ensure_workspace(ctx, (size_t)(prefix_parts + own_parts) * num_q_heads * (head_dim + 2) * 4 + ((size_t)n_req + 1) * 4);
    if (rc) return rc;
    a.o = (float *)ctx->ws;
    a.m = a.o + rows * head_dim;
    a.l = a.m + rows;
    a.own_start = items ? (uint32_t *)(a.l + rows) : nullptr;
    return head_dim == 256 ? launch_prefix<256>(ctx, a, (uint32_t)grid, by_rows)
                           : launch_prefix<512>(ctx, a, (uint32_t)grid, by_rows);
}
