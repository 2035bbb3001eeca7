// Attention of several tokens per request over a paged KV cache: packed
// prompts, causal (chn_paged_causal_attn), and trees of drafted tokens
// (chn_paged_tree_attn); and the trees' masks and clocks (chn_draft_trees).
//
// Work is a list of tiles: (request, KV head, a stretch of the request's new
// tokens with all query heads of the KV head).  Laid end to end - a tile as
// long as the keys it walks and a constant for its beginning and end - they
// are cut into equal shares, one per workgroup, wherever a cut falls: a tile
// that is cut leaves parts (the sums, their reference and denominator per
// row), which a second launch joins.  Every workgroup finds its share itself
// from the lengths, so nothing is planned on the host and no workgroup waits
// for another.
//
// A row's result is sum_k 2^(c (s_k - m)) v_k / sum_k 2^(c (s_k - m)), s = q.k,
// c = |scale| log2 e, for any reference m: one pass over the keys, the
// reference moved when a score passes it.  Both products run on the fp16 matrix
// instructions with every fp32 operand split in two halves (three products of
// the four): 409 TFLOP/s at the rate that a large fp16 product reaches (1227
// TFLOP/s), against 154 of the fp32 instructions.
//
// Measured (us, first launch + second, least and mean of 30 calls under a
// profiler) and what bounds it: 8 trees of up to 16 tokens behind up to 700 17-18 +
// 7-8, a chain of latencies, the second launch's among them; 64 trees on a sliding
// layer 164-183 + 11-12, and 5 trees of up to 64 behind up to 60000 300-362 + 9-11,
// K and V from memory (0.77 and 1.65 GB); 64 requests of one token on a sliding
// layer 178-201 + 6, the same (0.92 GB); 13 trees of 512-wide heads 115-120 + 12, a
// chunk's latencies, the share of a tile per CU; a prompt of 24 tokens 12-13 + 1-4,
// a tile's beginning and end, and a launch with nothing to do; 48 prompts on a
// sliding layer 1090-1213 + 18, LDS reads, products and issue, and 12 tiles'
// beginnings and ends per CU; 2000 tokens behind 30000 3172-3373 + 18, the same (905
// TFLOP/s of fp16 products at the latter); 9 prompts of 512-wide heads 199-216 + 17,
// two latencies a chunk: K and V take turns in the same registers.
#include "chn_internal.h"

#include <cmath>

namespace chn {

typedef float f4q __attribute__((ext_vector_type(4)));

constexpr uint32_t kPackedRequests = 8192;
constexpr uint32_t kPackedRows = 1u << 24;
constexpr uint32_t kMaskWords = 8;          // drafted tokens of a request: 256
constexpr int kShareLog = 8;
constexpr uint32_t kShares = 1u << kShareLog;   // workgroups: one per CU
constexpr int kThreads = 512;
// A key is 2 units, or 3 where both waves of a SIMD have rows (a chunk of 32 keys takes 2.9 and 4.1 us).  A tile costs
// kTileCost besides its keys, its beginning and end (heads of 256 14 us; heads of 512 16, where a chunk takes 5.4).  A
// cut that would fall within kNearEnd of a tile's end is moved there; a share has kShareUnits or more, twice that, so
// that no share of a tile that is cut is empty.  A tile below kShortTile, three chunks, is not worth the join.
constexpr int64_t kTileCost = 320, kNearEnd = 96, kShareUnits = 2 * kNearEnd, kShortTile = 512;
constexpr float kNoScore = -__builtin_inff();

// Rows of a tile: tokens x query heads of the KV head.
constexpr uint32_t tile_rows(uint32_t D) { return D == 256 ? 128 : 64; }

// A tile whose last part a workgroup made: the join's work.
struct Joined {
    uint32_t first, last;      // the shares that made its parts
    uint32_t row, rows, kvh;   // the tile's first batch row, its rows (0: no such tile)
};

struct Packed {
    const float *q, *kc, *vc;
    const uint32_t *tables, *row_start, *lens, *masks;
    uint32_t mask_words;       // 0: causal
    uint32_t n_req, n_rows, max_blocks, shift, n_blocks, num_q, num_kv, kv_dim, gqa, tokens;   // tokens per tile
    uint32_t per_gqa, per_tokens;             // their inverses: 2^16 / gqa, 2^32 / tokens, rounded up
    int window;
    float c, sign;             // |scale| log2(e), the scale's sign
    float *out;
    float *po, *pm, *pl;       // parts: [2 * kShares][rows of a tile](D sums, divided by the denominator; reference; denominator)
    Joined *joined;
};

// The new tokens of request r: batch rows row .. row + n - 1, at positions
// have .. of len.  Row starts that are no sum of counts give other rows, none
// outside the batch.
struct Seq {
    uint32_t row;
    int n, have, len;
};
__device__ __forceinline__ Seq seq_of(const Packed &a, uint32_t r) {
    const uint32_t s = min(a.row_start[r], a.n_rows), e = min(a.row_start[r + 1], a.n_rows);
    Seq q;
    q.row = s;
    q.n = e > s ? (int)(e - s) : 0;
    q.len = (int)min(a.lens[r], a.max_blocks << a.shift);
    q.have = q.len - q.n;
    return q;
}

// row of a tile -> token
__device__ __forceinline__ uint32_t token_of(const Packed &a, uint32_t row) { return row * a.per_gqa >> 16; }

// What the tiles of a request and KV head cost: tile t walks keys lo(t) ..
// hi(t) - 1, both linear in t (the last tile's end is the work's, not the
// cost's, matter).
struct TileKeys {
    int64_t T, hi0, lo0;               // hi = hi0 + t T, lo = max(0, lo0 + t T); T is 0 where all tiles see the same keys
    uint32_t tiles, s0;                // the first tile whose lo is above 0
    bool full, last_full;              // whether a tile's rows, and the last one's, are more than half of a tile's
    template <int D>
    static __device__ __forceinline__ TileKeys of(const Packed &a, const Seq &s) {
        TileKeys k;
        k.tiles = __umulhi((uint32_t)s.n + a.tokens - 1, a.per_tokens);
        k.s0 = k.tiles;
        k.full = a.tokens * a.gqa > tile_rows(D) / 2;
        // of many tiles the last counts as the others: shares then begin at the same keys of neighbouring tiles, which the
        // workgroups of an XCD walk together (as itself / as the others: 2000 tokens behind 30000, whose tiles are as many as
        // the shares, 3560-3815 us / 3390; 2500 behind 20000, 40 tiles per head, 3350 / 3170; 1500 behind 12000 1110 / 1080;
        // 600 of 512-wide heads 840 / 748; 600 behind 8000, 4100 behind 10000 and 7000 alone within 2 %; two to eight tiles
        // within 4 % either way)
        k.last_full = k.tiles > 8 ? k.full : (s.n - (k.tiles - 1) * a.tokens) * a.gqa > tile_rows(D) / 2;
        if (a.mask_words) {
            k.T = 0;
            k.hi0 = max(0, s.have + min(s.n, (int)(32 * a.mask_words)));      // no sum passes the length
            k.lo0 = a.window && s.have > a.window ? s.have - a.window : 0;
        } else {
            k.T = a.tokens;
            k.hi0 = max(s.have, 0) + k.T;
            k.lo0 = 0;
            if (a.window) {
                k.lo0 = (int64_t)s.have + 1 - a.window;
                k.s0 = k.lo0 > 0 ? 0 : (uint32_t)-k.lo0 / a.tokens + 1;
            }
        }
        return k;
    }
    __device__ __forceinline__ int64_t hi(uint32_t t) const { return hi0 + t * T; }
    __device__ __forceinline__ int64_t lo(uint32_t t) const { return T && t < s0 ? 0 : lo0 + t * T; }
    __device__ __forceinline__ bool is_full(uint32_t t) const { return t + 1 < tiles ? full : last_full; }
    static __device__ __forceinline__ int64_t weighed(int64_t keys, bool full) { return keys * (full ? 3 : 2); }
    __device__ __forceinline__ int64_t cost(uint32_t t) const { return kTileCost + weighed(hi(t) - lo(t), is_full(t)); }
    // of the tiles before t, which are not the last
    __device__ __forceinline__ int64_t before(uint32_t t) const {
        const int64_t pairs = (int64_t)t * t - t, n = t > s0 ? t - s0 : 0;
        int64_t keys = t * hi0 + (T * pairs >> 1);
        keys -= T ? n * lo0 + (T * n * ((int64_t)s0 + t - 1) >> 1) : t * lo0;
        return t * kTileCost + weighed(keys, full);
    }
    __device__ __forceinline__ int64_t all() const { return tiles ? before(tiles - 1) + cost(tiles - 1) : 0; }
    // units behind a tile's begin -> keys behind its first
    __device__ __forceinline__ int64_t keys_at(uint32_t t, int64_t units) const {
        const int64_t u = max(units - kTileCost / 2, (int64_t)0);
        return is_full(t) ? (int64_t)__umul64hi((uint64_t)u, 0x5555555555555556ull) : u >> 1;
    }
};
__device__ __forceinline__ int64_t snapped(int64_t at, int64_t cost, bool whole) {
    if (whole && cost < kShortTile) return 2 * at < cost ? 0 : cost;
    return at < kNearEnd ? 0 : (at + kNearEnd > cost ? cost : at);
}

// One tile's share: rows, and keys key0 .. key1 - 1 (key0 a multiple of 32, or no keys).
struct Work {
    Seq s;
    const uint32_t *table;
    uint32_t kvh, tile_row, rows;      // the tile's first batch row; rows (tokens x heads)
    int token, key0, key1;             // its first token's index
    int part;                          // -1: the whole tile
};

// What a row sees: cached keys lo .. hi - 1, and by its mask drafted ones.
struct Seen {
    int lo, hi;
    const uint32_t *mask;
};
__device__ __forceinline__ Seen seen_by(const Packed &a, const Work &w, int token) {
    Seen s;
    s.mask = nullptr;
    if (a.mask_words) {
        s.mask = a.masks + (size_t)(w.s.row + token) * a.mask_words;
        s.hi = max(w.s.have, 0);
        s.lo = 0;
        if (a.window) {
            int ones = 0;
            for (uint32_t i = 0; i < a.mask_words; ++i) ones += __popc(s.mask[i]);
            s.lo = w.s.have > a.window - ones ? w.s.have - (a.window - ones) : 0;      // a window is no shorter than a mask
        }
    } else {
        s.hi = w.s.have + token + 1;
        s.lo = a.window && s.hi > a.window ? s.hi - a.window : 0;
    }
    return s;
}

__device__ __forceinline__ uint32_t slot_of(const Packed &a, const uint32_t *table, uint32_t pos) {
    const uint32_t b = table[pos >> a.shift];
    return b < a.n_blocks ? (b << a.shift) + (pos & ((1u << a.shift) - 1)) : CHN_NO_SLOT;
}

// A row's result, in lane's dims 4 lane + 256 k .. + 3: to the batch's row, or as a part.
template <int D>
__device__ __forceinline__ float *row_out(const Packed &a, const Work &w, uint32_t row) {
    if (w.part >= 0) return a.po + ((size_t)w.part * tile_rows(D) + row) * D;
    const uint32_t token = token_of(a, row);
    return a.out + ((size_t)(w.tile_row + token) * a.num_q + w.kvh * a.gqa + row - token * a.gqa) * D;
}

// A row per wave, a key at a time: scores in plain fp32, what any of them do,
// infinities and NaN among them; sums in 64 bits, which no values pass and
// which keep the digits of long lists.  Every row reads its keys for itself: a
// prompt of 24 tokens 58 us instead of 15, 64 requests of one token on a sliding
// layer 2.2 ms instead of 0.2, 16 prompts of 200 14.0 instead of 0.18, 2000 tokens
// behind 30000 471 instead of 3.4, and 372 with one NaN in one head's first keys.
template <int D>
__device__ __forceinline__ void rows_plain(const Packed &a, const Work &w) {
    constexpr int N = D / 256;
    // made again here: what follows from it would be held over the tiles, all the others' time (a prompt of 24 14.7 us, 14.5)
    const uint32_t thread = opaque_u32(threadIdx.x);
    const int lane = thread & 63;
    for (uint32_t row = __builtin_amdgcn_readfirstlane(thread >> 6); row < w.rows; row += kThreads / 64) {
        const int token = w.token + (int)token_of(a, row);
        const Seen s = seen_by(a, w, token);
        const float *qr = a.q + ((size_t)(w.s.row + token) * a.num_q + w.kvh * a.gqa + row - token_of(a, row) * a.gqa) * D;
        f4q q[N];
        double o[N][4];
        for (int k = 0; k < N; ++k) {
            q[k] = *(const f4q *)(qr + 4 * lane + 256 * k) * a.sign;
            for (int e = 0; e < 4; ++e) o[k][e] = 0.0;
        }
        float m = kNoScore;
        double l = 0.0;
        for (int pos = w.key0; pos < w.key1; ++pos) {
            bool ok = pos >= s.lo && pos < s.hi;
            const int node = pos - w.s.have;
            if (s.mask && node >= 0) ok = (s.mask[node >> 5] >> (node & 31)) & 1;          // key1 is below 32 mask_words of them
            const uint32_t slot = ok ? slot_of(a, w.table, pos) : CHN_NO_SLOT;
            if (slot == CHN_NO_SLOT) continue;
            const size_t at = (size_t)slot * a.kv_dim + (size_t)w.kvh * D + 4 * lane;
            float sum = 0.0f;
            for (int k = 0; k < N; ++k) {
                const f4q x = *(const f4q *)(a.kc + at + 256 * k);
                for (int e = 0; e < 4; ++e) sum = fmaf(x[e], q[k][e], sum);
            }
            sum = wave_sum64(sum);
            if (sum == kNoScore) continue;                                                // no weight, whatever its V
            if (sum > m) {
                const double old = m == kNoScore ? 0.0 : (double)__builtin_amdgcn_exp2f((m - sum) * a.c);
                m = sum;
                l *= old;
                for (int k = 0; k < N; ++k)
                    for (int e = 0; e < 4; ++e) o[k][e] *= old;
            }
            // of a NaN score, or of two infinite ones, NaN
            const double p = __builtin_amdgcn_exp2f((sum - (m == kNoScore ? 0.0f : m)) * a.c);
            l += p;
            for (int k = 0; k < N; ++k) {
                const f4q x = *(const f4q *)(a.vc + at + 256 * k);
                for (int e = 0; e < 4; ++e) o[k][e] = fma(p, (double)x[e], o[k][e]);
            }
        }
        const double inv = l != 0.0 ? 1.0 / l : 0.0;
        float *to = row_out<D>(a, w, row);
        for (int k = 0; k < N; ++k)
            *(f4q *)(to + 4 * lane + 256 * k) = f4q{(float)(o[k][0] * inv), (float)(o[k][1] * inv), (float)(o[k][2] * inv), (float)(o[k][3] * inv)};
        if (w.part >= 0 && lane == 0) {
            a.pm[(size_t)w.part * tile_rows(D) + row] = m;
            a.pl[(size_t)w.part * tile_rows(D) + row] = (float)l;
        }
    }
}

// ---------------------------------------------------------------------
// Tiles on matrix instructions.
// ---------------------------------------------------------------------
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

// What keys that are nobody's read.
static __device__ __align__(16) const float no_key[512] = {};

// x * scale (scale a power of two) as fp16 halves hi + lo of 11 bits each:
// |x scale - hi - lo| <= 2^-22 |x scale|.  The products hi hi, hi lo and lo hi
// are exact in fp32, where the instructions sum them; lo lo (2^-22 of a
// product) is dropped.
// Two values together.  ONCE: an empty asm keeps the compiler from making the
// second one's hi twice, once to be packed and once to be subtracted (prompts of
// 256-wide heads 1195 -> 1140 us for 48, one of 24 16.1 -> 14.7).  512-wide heads
// have no register for it but at V: 131 -> 137 us with all, in 13 trees' step.
template <bool ONCE, typename V>
__device__ __forceinline__ void halves(float x0, float scale0, float x1, float scale1, V &hi, V &lo, int at) {
    h2 h = {(_Float16)fmaf(x0, scale0, 0.0f), (_Float16)fmaf(x1, scale1, 0.0f)};
    if (ONCE) __asm__("" : "+v"(h));
    hi[at] = h[0];
    hi[at + 1] = h[1];
    lo[at] = (_Float16)fmaf(x0, scale0, -(float)h[0]);
    lo[at + 1] = (_Float16)fmaf(x1, scale1, -(float)h[1]);
}

// The power of two that brings values of magnitude `top` (its bits) below
// 2^15, and its inverse: fp16 then holds what is 2^-39 of the largest and
// more.  At most 2^126, so that the inverse is no denormal; what is rounded
// then lies below the type's least value.
__device__ __forceinline__ float scale_for(uint32_t top, float &inverse) {
    const uint32_t f = min(0x86000000u - (top & 0x7F800000u), 253u << 23);
    inverse = __builtin_bit_cast(float, (254u << 23) - f);
    return __builtin_bit_cast(float, f);
}
// Magnitudes of q and K from here on, 2^56 (infinities and NaN among them), are left to fp32: below it none of their
// products, in units of either's scale or of both, passes the type's range.  Of V's only infinities and NaN are.
constexpr uint32_t kPlain = (127u + 56) << 23, kNotFinite = 0x7F800000u;
// NaN if either is
__device__ __forceinline__ float largest(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// the bits of the largest magnitude of N values, as unsigned words ordered as the values are
template <int N, typename F>
__device__ __forceinline__ uint32_t magnitude(F &&at) {
    float top = largest(fabsf(at(0)), fabsf(at(1)));
#pragma unroll
    for (int i = 2; i < N; ++i) top = largest(top, fabsf(at(i)));
    return __builtin_bit_cast(uint32_t, top);
}
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t row16_top(uint32_t v) {
    v = max_dpp<0xB1>(v);                              // quad_perm [1,0,3,2], [2,3,0,1], row_ror:4, row_ror:8
    v = max_dpp<0x4E>(v);
    v = max_dpp<0x124>(v);
    return max_dpp<0x128>(v);
}
// The results of a swap pass through an empty asm: this compiler otherwise takes the second for the first.
__device__ __forceinline__ void swap16(uint32_t &a, uint32_t &b) {           // rows a0 b0 a2 b2, a1 b1 a3 b3
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
    __asm__("" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ void swap32(uint32_t &a, uint32_t &b) {           // halves a0 b0, a1 b1
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
    __asm__("" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ uint32_t swap_max16(uint32_t a, uint32_t b) {
    swap16(a, b);
    return max(a, b);
}
__device__ __forceinline__ uint32_t swap_max32(uint32_t a, uint32_t b) {
    swap32(a, b);
    return max(a, b);
}
// Four values over the wave, row by row: lanes 16 i of the result hold v[i]'s.
__device__ __forceinline__ uint32_t wave_top4(const uint32_t (&v)[4]) {
    return row16_top(swap_max16(swap_max32(v[0], v[2]), swap_max32(v[1], v[3])));
}
// over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float rows4_top(float v) {
    uint32_t a = __builtin_bit_cast(uint32_t, v), b = a;
    swap16(a, b);
    a = b = __builtin_bit_cast(uint32_t, largest(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
    swap32(a, b);
    return largest(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// Addresses known to be memory's: flat loads would count as LDS operations,
// and the barriers below wait for those.
typedef const __attribute__((address_space(1))) float *mem_t;
__device__ __forceinline__ f4q load4(mem_t p) { return *(const __attribute__((address_space(1))) f4q *)p; }

// LDS of a workgroup: 32 keys in the order in which the instructions read
// them, and their scales' inverses.
//  K: [tile of 16 keys][step of 32 dims][hi, lo][64 lanes][8 dims]; lane 16 g +
//     key holds dims 4 g .. + 3 and 16 + 4 g .. + 3 of the step (the query's
//     lanes then load 64 bytes of a row together), at place key ^ (4 (step % 4)
//     + g), so that neighbouring lanes of a store fill 256 bytes
//  V: [16 dims][hi, lo][64 lanes][8 keys]; lane 16 g + c holds keys 4 g .. + 3
//     and 16 + 4 g .. + 3, the keys whose weights lane 16 g + row has after the
//     score's product; of 64 dims, tile e holds dims e, 4 + e, 8 + e .. in the
//     order in which a result's lanes store 64 bytes of a row together
template <int D>
struct TileLds {
    static constexpr int kKeyBytes = 32 * D * 4, kBuffers = D == 256 ? 2 : 1;      // of chunks in turn
    unsigned char k[kBuffers][kKeyBytes], v[kBuffers][kKeyBytes];
    float kinv[kBuffers][32], vinv[kBuffers][32];
    float half[D == 512 ? 8 * 64 * 8 : 4];            // scores of the other half of the dims
    uint32_t plain;                                   // what is left to fp32 was met
};

// By address: the places of a lane are one register and constants, and the
// register is made opaque where the compiler would rather keep every sum.
template <typename T>
__device__ __forceinline__ T lds_load(uint32_t at) { return *(const __attribute__((address_space(3))) T *)(uintptr_t)at; }
template <typename T>
__device__ __forceinline__ void lds_store(uint32_t at, T v) { *(__attribute__((address_space(3))) T *)(uintptr_t)at = v; }

// All waves: what was stored in LDS before is visible behind it.  Loads from
// memory stay in flight, and nothing moves across.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The end of a step of six products: other work stands between them, so that
// the SIMD issues it while the matrix unit is busy.
__device__ __forceinline__ void end_step() {
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);        // a product
        __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);        // vector operations
    }
    __builtin_amdgcn_sched_barrier(0);
}

// Weights are relative to a reference that is moved when a score passes it by
// more than this, in powers of two.
constexpr float kLead = 2.0f;
// A row's sums are kept relative to the largest weight times V scale of the keys that it sees (a power of two, vref):
// whatever its other keys' slots hold, and whatever lies under weights of nothing, takes no digits from them.  The
// halves of those products are relative to it, 2^kWeightLog for one, so what is below 2^-36 of it is rounded to that;
// it is raised when a product passes it by more than kRoom, which keeps them at or below 2^15.  A reference of all keys
// walked, known before the scores, is 3 us less for 64 trees (174) and 0.5 for a prompt of 24 (14.0), and wrong.
// The inverses of V's scales, 2^-126 to 2^113, are held times 2^kValueLog, so that weights times the least of them keep
// their digits and times the greatest stay below 2^127.
constexpr int kWeightLog = 12, kValueLog = 11;
constexpr float kRoom = 8.0f, kLeastRef = 0x1p-115f;

// A tile's walk over its keys, 32 at a time.  A chunk has two phases:
//   1  the scores of chunk c + 1, beside them the weights of chunk c and a V
//      into LDS: that of chunk c + 1, with heads of 512 chunk c's;
//   2  the sums of chunk c, beside them K of chunk c + 2 into LDS.
// Each is 48 products of the matrix unit, interleaved in eight steps with the
// other work, which two waves of a SIMD issue meanwhile.  What a wave loads of
// K and V (four keys of each) is under way for a phase or two.  Heads of 256
// have two LDS buffers of each in turn, and one barrier a chunk; heads of 512
// have room for one, and a barrier ahead of each phase (with heads of 256 that
// is 3.46 against 3.37 ms for 2000 tokens behind 30000).
//
// The sums and the query's halves of 16 rows stay in a wave's registers, 128 of
// its 256 with heads of 256, so every wave reads every key's halves from LDS:
// 512 KB a chunk and CU, 4100 of its 8000 cycles at 128 B a cycle, beside 3070
// of products and 2550 of vector instructions.  Measured and not taken: products' operands
// asked for a step ahead (spills, 48 prompts 1470 us), four waves a workgroup
// and two workgroups a CU (1575), keys shared by no waves, each with chunks of
// its own (64 trees 280 us, 191 shared).
template <int D>
struct Tile {
    static constexpr int H = D / 256, RT = 8 / H;     // waves that share 16 rows (256 dims each), tiles of 16 rows
    static constexpr int S = D / 32;                  // steps
    // heads of 512 have no registers for K and V at once: K is loaded a chunk later, after V has gone to LDS
    static constexpr bool kBoth = D == 256;
    static constexpr int kBuffers = TileLds<D>::kBuffers;
    static constexpr uint32_t kBuffer = TileLds<D>::kKeyBytes;
    const Packed &a;
    const Work &w;
    TileLds<D> &lds;
    int lane, wave, rt, half, q, g, keys;             // keys: the first of the four that the wave converts
    f4q kr[4][H], vr_[kBoth ? 4 : 1][H];              // their dims 4 lane + 256 h .. + 3
    uint32_t next_block;                              // of 64 keys, a lane each: the next ones' blocks,
    mem_t ka, va, vnow;                               // these ones' rows (V is loaded later than K)
    uint64_t unheld;                                  // and which of them are nobody's
    uint32_t worst;                                   // the largest magnitude met
    uint32_t k_to, v_to;                              // where the lane's values go in LDS
    uint32_t k_at, v_at;                              // and where it takes its operands

    __device__ __forceinline__ Tile(const Packed &a_, const Work &w_, TileLds<D> &l) : a(a_), w(w_), lds(l) {
        // made again for every tile: held over the tiles, what follows from them would be spilled
        const uint32_t thread = opaque_u32(threadIdx.x);
        lane = thread & 63;
        wave = __builtin_amdgcn_readfirstlane(thread >> 6);
        // the halves of a row's dims on neighbouring SIMDs, so that half of a tile's rows keep all four busy
        rt = wave / H;
        half = wave % H;
        q = lane & 15;
        g = lane >> 4;
        keys = 4 * (wave >> 1) + 16 * (wave & 1);
        worst = 0;
        const int quad = 4 * (lane >> 3) + (lane & 3);
        k_to = lds_addr(lds.k) + (((wave & 1) * S + (lane >> 3)) * 2) * 1024 + (lane & 3) * 256 + (((keys ^ quad) & 15) * 16) + (lane >> 2 & 1) * 8;
        k_at = lds_addr(lds.k) + half * 16384 + g * 256 + (q ^ g) * 16;
        v_at = lds_addr(lds.v) + half * 32768 + lane * 16;
        v_to = lds_addr(lds.v) + 4 * (lane >> 4) * 2048 + ((wave >> 1) * 16 + (4 * (lane & 3) + (lane >> 2 & 3))) * 16 + (wave & 1) * 8;
    }
    __device__ __forceinline__ f4q (&vr())[4][H] {
        if constexpr (kBoth) return vr_;
        else return kr;
    }

    // chunks come in pairs, 64 keys, a lane each
    __device__ __forceinline__ uint32_t block_of(int pair) const {
        return w.table[min((uint32_t)w.key0 + 64u * pair + lane, (uint32_t)w.key1 - 1) >> a.shift];
    }
    __device__ __forceinline__ void take_pair(int pair) {
        const uint32_t pos = (uint32_t)w.key0 + 64u * pair + lane, b = next_block;      // unsigned: up to 2^31 and a pair
        const bool held = pos < (uint32_t)w.key1 && b < a.n_blocks;
        const size_t at = (size_t)((b << a.shift) + (pos & ((1u << a.shift) - 1))) * a.kv_dim + (size_t)w.kvh * D;
        ka = held ? (mem_t)a.kc + at : (mem_t)no_key;
        va = held ? (mem_t)a.vc + at : (mem_t)no_key;
        unheld = ~__ballot(held);
        next_block = block_of(pair + 1);
    }
    // chunks behind the last are nobody's
    __device__ __forceinline__ void load(f4q (&to)[4][H], mem_t rows, int chunk) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const mem_t row = (mem_t)lane64((uint64_t)rows, 32 * (chunk & 1) + keys + i);
#pragma unroll
            for (int h = 0; h < H; ++h) to[i][h] = load4(row + 4 * lane + 256 * h);
        }
    }
    __device__ __forceinline__ uint32_t load_k(int chunk) {
        if (!(chunk & 1)) take_pair(chunk >> 1);
        load(kr, ka, chunk);
        return (uint32_t)(unheld >> (32 * (chunk & 1)));
    }
    // the four keys' scales, and their inverses: K's, or V's times 2^kValueLog
    template <bool VALUES = false>
    __device__ __forceinline__ void scales(const f4q (&of)[4][H], float (&scale)[4], float *inverses) {
        uint32_t top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            top[i] = magnitude<4 * H>([&](int e) { return of[i][e / 4][e % 4]; });
        }
        const uint32_t here = max(max(top[0], top[1]), max(top[2], top[3]));
        worst = max(worst, VALUES ? __builtin_elementwise_sub_sat(here, kNotFinite - kPlain) : here);
        const uint32_t most = wave_top4(top);
        f4q inverse;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float inv;
            scale[i] = scale_for(__builtin_amdgcn_readlane(most, 16 * i), inv);
            inverse[i] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, inv) + (VALUES ? kValueLog << 23 : 0));
        }
        if (lane == 0) *(f4q *)(inverses + keys) = inverse;
    }
    // key i of the wave's
    __device__ __forceinline__ void store_k(int i, float scale) {
        const uint32_t at = opaque_u32(k_to) ^ (i * 16);
#pragma unroll
        for (int h = 0; h < H; ++h) {
            h4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                halves<D == 256>(kr[i][h][e], scale, kr[i][h][e + 1], scale, hi, lo, e);
            }
            lds_store(at + 16384 * h, hi);
            lds_store(at + 16384 * h + 1024, lo);
        }
    }
    // dims 256 h + 4 lane + e: column lane % 16 of 16 dims
    __device__ __forceinline__ void store_v(int e, const float (&scale)[4]) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            h4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                halves<true>(vr()[i][h][e], scale[i], vr()[i + 1][h][e], scale[i + 1], hi, lo, i);
            }
            lds_store(v_to + (16 * h + e) * 2048, hi);
            lds_store(v_to + (16 * h + e) * 2048 + 1024, lo);
        }
    }

    __device__ __forceinline__ void run() {
        const uint32_t row = rt * 16 + q;
        const bool valid = row < w.rows, active = (uint32_t)(rt * 16) < w.rows;
        const int chunks = w.key1 > w.key0 ? (int)(((uint32_t)(w.key1 - w.key0) + 31) / 32) : 0;
        uint32_t none0 = 0, none1 = 0, none2 = 0, none3 = 0;      // keys that are nobody's, of chunks c ..
        if (chunks) next_block = block_of(0);
        const uint32_t of_tile = valid ? token_of(a, row) : 0;
        const int token = w.token + (int)of_tile;
        h8 qh[8], ql[8];
        float qinv = 0.0f;
        {
            // asked for before K and V, whose addresses wait for the table
            const mem_t from = (mem_t)a.q + ((size_t)(w.s.row + token) * a.num_q + w.kvh * a.gqa + (valid ? row : 0) - of_tile * a.gqa) * D + 256 * half + 4 * g;
            f4q x[8][2];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) x[i][e] = load4(from + 32 * i + 16 * e);
            __builtin_amdgcn_sched_barrier(0);
            if (chunks) {
                none0 = load_k(0);
                if (kBoth) load(vr(), va, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            uint32_t top = magnitude<64>([&](int e) { return x[e / 8][e / 4 % 2][e % 4]; });
            worst = max(worst, top);
            top = swap_max16(top, top);
            top = swap_max32(top, top);
            const float scale = scale_for(top, qinv) * a.sign;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    halves<D == 256>(x[i][e / 4][e % 4], scale, x[i][e / 4][e % 4 + 1], scale, qh[i], ql[i], e);
                }
        }
        // rows of no token see everything, so that they never stand in a chunk's way
        Seen s = seen_by(a, w, token);
        if (!valid) {
            s.lo = 0;
            s.hi = 0x7FFFFFFF;
        }
        f4q o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = f4q{0, 0, 0, 0};
        // Scores stay in units of the row's q scale, whose inverse goes into the exponent's factor; the halves of heads of
        // 512 have scales of their own.  A factor of zero would make NaN of hidden keys' -inf; the least normal one keeps
        // all weights at one as well.  One that is too large is no number: fp32 computes the tile.
        const float unit_q = kBoth ? 1.0f : qinv, factor = kBoth ? fmaxf(a.c * qinv, 0x1p-126f) : a.c;
        if (factor > 3.4028235e38f) worst = kPlain;
        float m = kNoScore, l = 0.0f, vref = kLeastRef;
        bool moved = false;                                       // a row's m, and with it vref, which is no power of two then
        f4q sc[2];
        h8 ph, pl;
        float p[8], vscale[4];
        const auto weights = [&](const float *vinv) {             // p times the keys' V scales, as halves
            float top = 0.0f;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const f4q vi = *(const f4q *)(vinv + 16 * t + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[4 * t + e] *= vi[e];
                    top = largest(top, p[4 * t + e]);
                }
            }
            top = rows4_top(top);
            if (moved || __any(top > kRoom * vref)) {
                const float to = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, fmaxf(fmaxf(vref, top), kLeastRef)) & 0x7F800000u);
                const float f = vref * __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, to));
                vref = to;
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= f;
            }
            const float unit = __builtin_bit_cast(float, ((254u + kWeightLog) << 23) - __builtin_bit_cast(uint32_t, vref));
#pragma unroll
            for (int e = 0; e < 8; e += 2) halves<D == 256>(p[e], unit, p[e + 1], unit, ph, pl, e);
        };
        h8 fr[4];
        const auto fetch_k = [&](int i) {                         // both tiles' step i
            const uint32_t place = i & 3 ? opaque_u32(k_at) ^ ((i & 3) * 64) : k_at;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t at = place + (t * S + i) * 2048;
                fr[2 * t] = lds_load<h8>(at);
                fr[2 * t + 1] = lds_load<h8>(at + 1024);
            }
        };
        const auto fetch_v = [&](int i) {                         // dims 32 i .. + 31
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                fr[2 * t] = lds_load<h8>(v_at + (2 * i + t) * 2048);
                fr[2 * t + 1] = lds_load<h8>(v_at + (2 * i + t) * 2048 + 1024);
            }
        };
        f4q next[2], low[2];
        // four sums, so that no product waits for the one before
        const auto score_step = [&](int i) {
            low[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[1], qh[i], low[0], 0, 0, 0);
            low[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[3], qh[i], low[1], 0, 0, 0);
            next[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[0], qh[i], next[0], 0, 0, 0);
            next[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[2], qh[i], next[1], 0, 0, 0);
            low[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[0], ql[i], low[0], 0, 0, 0);
            low[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[2], ql[i], low[1], 0, 0, 0);
        };
        const auto begin_scores = [&] {
#pragma unroll
            for (int t = 0; t < 2; ++t) next[t] = low[t] = f4q{0, 0, 0, 0};
        };
        const auto end_scores = [&](int c) {                      // of chunk c
            const float *kinv = lds.kinv[kBoth ? c & 1 : 0];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                sc[t] = (next[t] + low[t]) * *(const f4q *)(kinv + 16 * t + 4 * g);
                if (!kBoth) {
                    sc[t] *= unit_q;
                    *(f4q *)(lds.half + ((wave * 2 + t) * 64 + lane) * 4) = sc[t];
                }
            }
        };
        const auto add_half = [&] {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                // the same order of the halves in both waves
                const f4q other = *(const f4q *)(lds.half + (((wave ^ 1) * 2 + t) * 64 + lane) * 4);
                sc[t] = half ? other + sc[t] : sc[t] + other;
            }
        };
        const auto all_k = [&](int c) {                           // chunk c
            float scale[4];
            scales(kr, scale, lds.kinv[kBoth ? c & 1 : 0]);
#pragma unroll
            for (int i = 0; i < 4; ++i) store_k(i, scale[i]);
        };
        if (chunks) {
            all_k(0);
            if (kBoth) {
                scales<true>(vr(), vscale, lds.vinv[0]);
#pragma unroll
                for (int e = 0; e < 4; ++e) store_v(e, vscale);
            }
            if (chunks > 1) {
                none1 = load_k(1);
                if (kBoth) load(vr(), va, 1);
            }
            vnow = va;
            lds_barrier();
            if (threadIdx.x == 0) lds.plain = 0;
            if (active) {
                begin_scores();
                static_for<8>([&](auto step) {
                    fetch_k(decltype(step)::value);
                    score_step(decltype(step)::value);
                });
                end_scores(0);
            }
            if (kBoth) {
                k_to += kBuffer;
                if (chunks > 1) {
                    all_k(1);
                    none2 = load_k(2);
                }
                k_to -= kBuffer;
                k_at += kBuffer;
                v_to += kBuffer;
            } else {
                lds_barrier();
                if (chunks > 1) all_k(1);
                if (active) add_half();
                load(vr(), vnow, 0);
            }
        }
        // the last chunk has no next one
        const auto walk = [&](int c, auto more) {
            constexpr bool kMore = decltype(more)::value;
            const float *vinv = lds.vinv[kBoth ? c & 1 : 0];
            if (!kBoth && (c & 1)) vnow = va;
            lds_barrier();
            // ---- phase 1

            if (!kBoth) {
                // the registers hold V of chunk c: to LDS first
                scales<true>(vr(), vscale, lds.vinv[0]);
#pragma unroll
                for (int e = 0; e < 4; ++e) store_v(e, vscale);
                if (kMore) none2 = load_k(c + 2);
            }
            if (active) {
                if constexpr (kMore) {
                    begin_scores();
                    fetch_k(0);
                }
                static_for<8>([&](auto step) {
                    constexpr int i = decltype(step)::value;
                    if constexpr (kMore) {
                        score_step(i);
                        if constexpr (i < 7) fetch_k(i + 1);
                    }
                    if constexpr (i == 0) {
                        const int k0 = w.key0 + 32 * c;
                        if (none0 || !__all(s.lo <= k0 && s.hi - k0 >= 32)) {
                            // bit k: the row sees key k0 + k
                            uint32_t ok = 0xFFFFFFFFu;
                            const int from = min(max(s.lo - k0, 0), 32), to = min(max(s.hi - k0, 0), 32);
                            if (valid) ok = to > from ? (0xFFFFFFFFu >> (32 - (to - from))) << from : 0u;
                            const int node = k0 - w.s.have;
                            if (node > -32 && node < (int)(32 * a.mask_words) && valid) {
                                const uint32_t *mask = a.masks + (size_t)(w.s.row + opaque_u32(token)) * a.mask_words;
                                const int n = node >> 5;
                                const uint32_t w0 = n >= 0 ? mask[n] : 0u, w1 = n + 1 < (int)a.mask_words ? mask[n + 1] : 0u;
                                ok |= (uint32_t)(((uint64_t)w1 << 32 | w0) >> (node & 31));
                            }
                            ok = (ok & ~none0) >> (4 * g);
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                sc[e / 4][e % 4] = ok >> (16 * (e / 4) + e % 4) & 1 ? sc[e / 4][e % 4] : kNoScore;
                        }
                    }
                    if constexpr (i == 1) {
                        float top = kNoScore;
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = largest(top, sc[e / 4][e % 4]);
                        top = rows4_top(top);
                        const bool up = (top - m) * factor > kLead;
                        moved = __any(up);
                        const float old = up ? __builtin_amdgcn_exp2f((m - top) * factor) : 1.0f;
                        m = up ? top : m;
                        l *= old;
                        vref *= old;                              // and the sums are in its units
                    }
                    if constexpr (i == 2 || i == 3) {
                        const float ref = m == kNoScore ? 0.0f : m;
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[4 * (i - 2) + e] = __builtin_amdgcn_exp2f((sc[i - 2][e] - ref) * factor);
                    }
                    if constexpr (i == 4) {
                        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                        if (kBoth) weights(vinv);
                    }
                    if constexpr (i == 3 && kBoth && kMore) scales<true>(vr(), vscale, lds.vinv[(c + 1) & (kBuffers - 1)]);
                    if constexpr (i >= 4 && kBoth && kMore) store_v(i - 4, vscale);
                    if constexpr (kMore) end_step();
                });
                if constexpr (kMore) end_scores(c + 1);
            } else if (kBoth && kMore) {
                scales<true>(vr(), vscale, lds.vinv[(c + 1) & (kBuffers - 1)]);
#pragma unroll
                for (int e = 0; e < 4; ++e) store_v(e, vscale);
            }
            if (kBoth) {
                if (kMore) load(vr(), va, c + 2);
            } else {
                lds_barrier();
            }
            // ---- phase 2
            if (active) {
                if (!kBoth) weights(vinv);
                float scale[4];
                fetch_v(0);
                static_for<8>([&](auto step) {
                    constexpr int i = decltype(step)::value;
                    o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[1], ph, o[2 * i], 0, 0, 0);
                    o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[3], ph, o[2 * i + 1], 0, 0, 0);
                    o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[0], pl, o[2 * i], 0, 0, 0);
                    o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[2], pl, o[2 * i + 1], 0, 0, 0);
                    o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[0], ph, o[2 * i], 0, 0, 0);
                    o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[2], ph, o[2 * i + 1], 0, 0, 0);
                    if constexpr (i < 7) fetch_v(i + 1);
                    if constexpr (kMore) {
                        if constexpr (i == 2) scales(kr, scale, lds.kinv[kBoth ? c & 1 : 0]);
                        if constexpr (i >= 3 && i < 7) store_k(i - 3, scale[i - 3]);
                        if constexpr (!kBoth && i == 7) load(vr(), vnow, c + 1);
                    }
                    end_step();
                });
                if (!kBoth && kMore) add_half();
            } else if (kMore) {
                all_k(c);
                if (!kBoth) load(vr(), vnow, c + 1);
            }
            if constexpr (kMore) {
                if (kBoth) {
                    none3 = load_k(c + 3);
                    const uint32_t turn = c & 1 ? kBuffer : -kBuffer;
                    k_at += turn;
                    v_to += turn;
                    k_to -= turn;
                    v_at -= turn;
                }
                none0 = none1;
                none1 = none2;
                none2 = none3;
            }
        };
        for (int c = 0; c + 1 < chunks; ++c) walk(c, std::true_type());
        if (chunks) walk(chunks - 1, std::false_type());
        if (chunks) {
            if (__any(worst >= kPlain) && lane == 0) lds.plain = 1;
            lds_barrier();
            if (lds.plain) {
                rows_plain<D>(a, w);
                return;
            }
        }
        l = rows4_sum(l);
        if (!valid) return;
        const float inv = l != 0.0f ? 1.0f / l : 0.0f, unit = vref * (1.0f / (1ull << (kWeightLog + kValueLog)));
        float *to = row_out<D>(a, w, row) + 256 * half + 4 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(f4q *)(to + 64 * j + 16 * i) =
                    f4q{o[4 * j][i] * inv * unit, o[4 * j + 1][i] * inv * unit, o[4 * j + 2][i] * inv * unit, o[4 * j + 3][i] * inv * unit};
        if (w.part >= 0 && g == 0 && half == 0) {
            a.pm[(size_t)w.part * tile_rows(D) + row] = kBoth ? m * (factor / a.c) : m;       // qinv again, not held over the walk
            a.pl[(size_t)w.part * tile_rows(D) + row] = l;
        }
    }
};

// The workgroup's share: f(work) for each of its tiles or parts of tiles.
template <int D, typename F>
__device__ __forceinline__ void each_work(const Packed &a, F &&f) {
    __shared__ int64_t sums[kThreads / 64], found_base;
    __shared__ Seq found_seq, seqs[kThreads / 64];             // every wave's request: a load from there, not from memory, for each tile
    __shared__ uint32_t found, tile_sums[kThreads / 64];
    const uint32_t tid = threadIdx.x, per = (a.n_req + kThreads - 1) / kThreads;
    const int lane = tid & 63, wave = tid >> 6;
    // every request's units; a thread sums its neighbours
    const uint32_t r0 = min(tid * per, a.n_req), r1 = min(r0 + per, a.n_req);
    int64_t mine = 0;
    uint32_t tiles = 0;                                        // of a request at most one more than there are shares
    for (uint32_t r = r0; r < r1; ++r) {
        const TileKeys k = TileKeys::of<D>(a, seq_of(a, r));
        mine += k.all() * a.num_kv;
        tiles += min(min(k.tiles, kShares + 1) * a.num_kv, kShares + 1);
    }
    const int64_t upto = (int64_t)wave_scan_u64((uint64_t)mine);
    tiles = (uint32_t)wave_sum_u64(tiles);
    if (lane == 63) {
        sums[wave] = upto;
        tile_sums[wave] = tiles;
    }
    if (tid == 0) {
        found = 0xFFFFFFFFu;
        a.joined[blockIdx.x].rows = 0;
    }
    __syncthreads();
    int64_t total = 0, base = upto - mine;
    tiles = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) {
        base += i < wave ? sums[i] : 0;
        total += sums[i];
        tiles += tile_sums[i];
    }
    total = (int64_t)lane64((uint64_t)total, 0);
    // As many shares as there are CUs; of the least size where there is less work (8 trees 27 us, 32 with a power of two of
    // larger ones).  Where there are no more tiles than CUs, short ones stay whole and need no join (a prompt of 24 tokens
    // 14.7 us, cut 16.7; 20 of up to 30 21.4, cut 26.7).
    const bool much = total >= kShareUnits << kShareLog;
    const int bits = much ? kShareLog : 0;
    const int64_t size = much ? total : kShareUnits;           // of 2^bits shares
    const uint32_t n = much ? kShares : max((uint32_t)total / (uint32_t)kShareUnits, 1u);
    const bool whole = __builtin_amdgcn_readfirstlane(tiles) <= kShares;
    // neighbours, which read the same keys, run on one XCD (workgroup i on XCD i % 8)
    const uint32_t each = (n + 7) / 8, share = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= each || share >= n) return;      // the whole workgroup
    const auto cut = [&](uint32_t w) { return size * w >> bits; };
    const int64_t u0 = cut(share), u1 = share + 1 == n ? total : cut(share + 1);
    if (u0 >= base && u0 < base + mine) {                     // one thread, or none
        uint32_t r = r0;
        for (; r + 1 < r1; ++r) {
            const int64_t units = TileKeys::of<D>(a, seq_of(a, r)).all() * a.num_kv;
            if (u0 < base + units) break;
            base += units;
        }
        found = r;
        found_base = base;
        found_seq = seq_of(a, r);
    }
    __syncthreads();
    uint32_t r = __builtin_amdgcn_readfirstlane(found), kvh = 0, t = 0;
    if (r >= a.n_req) return;
    int64_t u = (int64_t)lane64((uint64_t)found_base, 0);
    const auto uniform = [](const Seq &of) {
        Seq s;
        s.row = __builtin_amdgcn_readfirstlane(of.row);
        s.n = __builtin_amdgcn_readfirstlane(of.n);
        s.have = __builtin_amdgcn_readfirstlane(of.have);
        s.len = __builtin_amdgcn_readfirstlane(of.len);
        return s;
    };
    seqs[wave] = found_seq;
    {
        // the KV head, then the tile, that u0 falls into
        const TileKeys k = TileKeys::of<D>(a, uniform(found_seq));
        const int64_t head = k.all();
        uint32_t hi = a.num_kv;
        while (hi - kvh > 1) {
            const uint32_t mid = (kvh + hi) / 2;
            if (u + mid * head <= u0) kvh = mid;
            else hi = mid;
        }
        u += kvh * head;
        hi = k.tiles;
        while (hi - t > 1) {
            const uint32_t mid = (t + hi) / 2;
            if (u + k.before(mid) <= u0) t = mid;
            else hi = mid;
        }
        u += k.before(t);
    }
    while (u < u1) {
        // made again for every tile, so that little is held in registers meanwhile
        Work w;
        w.s = uniform(seqs[wave]);
        const TileKeys k = TileKeys::of<D>(a, w.s);
        const int64_t cost = k.cost(t);
        const int64_t from = u < u0 ? snapped(u0 - u, cost, whole) : 0, to = u1 - u < cost ? snapped(u1 - u, cost, whole) : cost;
        if (from < to) {
            w.table = a.tables + (size_t)r * a.max_blocks;
            w.kvh = kvh;
            w.token = (int)(t * a.tokens);
            w.tile_row = w.s.row + w.token;
            const int tokens = min(w.s.n - w.token, (int)a.tokens), lo = (int)k.lo(t);
            w.rows = (uint32_t)tokens * a.gqa;
            const int limit = a.mask_words ? (int)k.hi(t) : max(0, w.s.have + w.token + tokens);
            // cuts at whole chunks of 32 keys, none behind the last
            const auto chunk_at = [&](int64_t units) { return (int)min((lo + k.keys_at(t, units) + 31) >> 5 << 5, (int64_t)limit); };
            w.key0 = from ? chunk_at(from) : lo >> 5 << 5;
            w.key1 = to < cost ? chunk_at(to) : limit;
            w.part = from ? (int)(2 * share) : (to < cost ? (int)(2 * share + 1) : -1);
            if (from && to == cost && tid == 0) {
                // the share that begins this tile: the last whose first cut is at or before it
                uint32_t first = share;
                while (first && cut(first) > u && snapped(cut(first) - u, cost, whole)) --first;
                a.joined[blockIdx.x] = Joined{first, share, w.tile_row, w.rows, kvh};
            }
            f(w);
        }
        u += cost;
        if (++t < k.tiles) continue;
        t = 0;
        if (++kvh < a.num_kv) continue;
        kvh = 0;
        // the next request that takes tokens: 64 looked at together
        for (++r; r < a.n_req; r += 64) {
            const uint64_t takes = __ballot(r + lane < a.n_req && seq_of(a, min(r + lane, a.n_req - 1)).n > 0);
            if (takes) {
                r += __builtin_ctzll(takes);
                break;
            }
        }
        if (r >= a.n_req) break;
        seqs[wave] = seq_of(a, r);
    }
}

template <int D>
__global__ __launch_bounds__(kThreads) void k_packed_attn(Packed a) {
    extern __shared__ __align__(1024) unsigned char sh[];
    each_work<D>(a, [&](const Work &w) { Tile<D>(a, w, *(TileLds<D> *)sh).run(); });
}

// Joins the parts of the tiles that were cut.  A wave takes four rows
// together: 16 lanes hold the references and denominators of one row's parts,
// up to 16 of them at a time, and the sums (a lane four values per 256 dims) of
// four parts are under way while those become weights.  Bound by three
// latencies one after another (the tile, its references, nothing else where
// there are up to four parts).
constexpr uint32_t kJoinRows = 16;
template <int D>
__global__ __launch_bounds__(256) void k_packed_join(Packed a) {
    constexpr uint32_t R = tile_rows(D);
    constexpr int N = D / 256, P = 4;
    const int lane = threadIdx.x & 63;
    const Joined j = a.joined[blockIdx.x / (R / kJoinRows)];
    const uint32_t row0 = blockIdx.x % (R / kJoinRows) * kJoinRows + 4 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row0 >= j.rows) return;                                  // a whole wave
    const uint32_t rows = min(j.rows - row0, 4u), mine = row0 + min((uint32_t)lane >> 4, rows - 1);
    // the first part is its share's last tile, the others are their shares' first
    const auto at = [&](uint32_t p, uint32_t row) { return (size_t)(p == j.first ? 2 * p + 1 : 2 * p) * R + row; };
    f4q o[4][N], v[P][4][N];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) o[i][k] = f4q{0, 0, 0, 0};
    const auto fetch = [&](uint32_t p0) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < N; ++k)
                    v[p][i][k] = *(const f4q *)(a.po + at(min(p0 + p, j.last), row0 + min((uint32_t)i, rows - 1)) * D + 4 * lane + 256 * k);
    };
    float M = kNoScore, L = 0.0f;
    for (uint32_t p0 = j.first; p0 <= j.last; p0 += 16) {
        const uint32_t n = min(j.last + 1 - p0, 16u), p = min((uint32_t)lane & 15, n - 1);
        const size_t where = at(p0 + p, mine);
        float m = a.pm[where], part = a.pl[where];
        __builtin_amdgcn_sched_barrier(0);
        fetch(p0);
        __builtin_amdgcn_sched_barrier(0);
        if (p != ((uint32_t)lane & 15)) part = 0.0f;
        if (part == 0.0f) m = kNoScore;                          // a part without keys has none
        const float top = fmaxf(M, row16_max(m)), ref = top == kNoScore ? 0.0f : top;
        // NaN: whatever its reference is
        const float old = M == kNoScore ? 0.0f : __builtin_amdgcn_exp2f((M - ref) * a.c);
        const float w = part != 0.0f ? __builtin_amdgcn_exp2f((m - ref) * a.c) * part : 0.0f;
        M = top;
        // divided as they are added: a denominator times values near the type's largest would pass it
        const float sum = L * old + row16_sum(w), inv = sum != 0.0f ? 1.0f / sum : 0.0f, share = w * inv;
        if (p0 != j.first)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < N; ++k) o[i][k] *= lane_f(L * old * inv, 16 * i);
        L = sum;
        for (uint32_t q = 0; q < n; q += P) {
            if (q) fetch(p0 + q);
#pragma unroll
            for (int e = 0; e < P; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float wi = q + e < n ? lane_f(share, 16 * i + min(q + e, 15u)) : 0.0f;
#pragma unroll
                    for (int k = 0; k < N; ++k) o[i][k] += wi != 0.0f ? wi * v[e][i][k] : f4q{0, 0, 0, 0};
                }
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        if (i >= rows) break;
        const uint32_t row = row0 + i, token = token_of(a, row);
        float *to = a.out + ((size_t)(j.row + token) * a.num_q + j.kvh * a.gqa + row - token * a.gqa) * D + 4 * lane;
#pragma unroll
        for (int k = 0; k < N; ++k) *(f4q *)(to + 256 * k) = o[i][k];
    }
}

template <int D>
static int launch_packed(chn_ctx *ctx, const Packed &a) {
    static_assert(sizeof(TileLds<D>) <= 159 * 1024, "LDS per workgroup");
    k_packed_attn<D><<<kShares, kThreads, sizeof(TileLds<D>), ctx->stream>>>(a);
    CHN_LAUNCHED(ctx, "k_packed_attn");
    k_packed_join<D><<<kShares * (tile_rows(D) / kJoinRows), 256, 0, ctx->stream>>>(a);
    CHN_LAUNCHED(ctx, "k_packed_join");
    return CHN_OK;
}

// Both entries: mask_words 0 is the causal one.
static int packed_attn(chn_ctx *ctx, const float *q, const float *k_cache, const float *v_cache, const uint32_t *tables,
                       const uint32_t *row_start, const uint32_t *lens, const uint32_t *masks, uint32_t mask_words,
                       uint32_t n_req, uint32_t n_rows, uint32_t max_blocks, uint32_t block_size, uint32_t n_blocks,
                       uint32_t num_q_heads, uint32_t head_dim, uint32_t kv_dim, uint32_t gqa_ratio, float scale,
                       uint32_t window, float *out) {
    CHN_REQUIRE(ctx, q && k_cache && v_cache && tables && row_start && lens && out, "NULL argument");
    CHN_REQUIRE(ctx, head_dim == 256 || head_dim == 512, "head_dim %u must be 256 or 512", head_dim);
    CHN_REQUIRE(ctx, gqa_ratio > 0 && gqa_ratio <= 16 && num_q_heads && num_q_heads % gqa_ratio == 0,
                "num_q_heads %u, gqa ratio %u: a ratio of 1..16 that divides the heads", num_q_heads, gqa_ratio);
    CHN_REQUIRE(ctx, num_q_heads <= 4096, "num_q_heads %u exceeds 4096", num_q_heads);
    CHN_REQUIRE(ctx, kv_dim >= (num_q_heads / gqa_ratio) * head_dim && kv_dim % 4 == 0,
                "kv_dim %u too small for %u kv heads of %u", kv_dim, num_q_heads / gqa_ratio, head_dim);
    CHN_REQUIRE(ctx, aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16),
                "q, caches and out must be 16-byte aligned");
    int rc = check_blocks(ctx, block_size, n_blocks, max_blocks);
    if (rc) return rc;
    const double c = std::fabs((double)scale) * 1.4426950408889634;
    CHN_REQUIRE(ctx, c >= 1e-37 && c <= 1e37, "scale %g must be finite and not zero", (double)scale);
    if (n_req > kPackedRequests) return set_err(ctx, CHN_E_UNSUPPORTED, "n_req %u exceeds %u", n_req, kPackedRequests);
    if (n_rows > kPackedRows) return set_err(ctx, CHN_E_UNSUPPORTED, "n_rows %u exceeds %u", n_rows, kPackedRows);
    const size_t words = (size_t)n_rows * num_q_heads * head_dim, cache = (size_t)n_blocks * block_size * kv_dim;
    const Span ins[] = {{q, words}, {k_cache, cache}, {v_cache, cache}, {tables, (size_t)n_req * max_blocks},
                        {row_start, (size_t)n_req + 1}, {lens, n_req}, {masks, (size_t)n_rows * mask_words}};
    for (const Span &i : ins) CHN_REQUIRE(ctx, !overlap(i, Span{out, words}), "out overlaps an input");
    CHN_REQUIRE(ctx, ctx, "ctx is NULL");
    if (!n_req || !n_rows) return CHN_OK;
    DeviceGuard dev(ctx);
    Packed a{};
    a.q = q;
    a.kc = k_cache;
    a.vc = v_cache;
    a.tables = tables;
    a.row_start = row_start;
    a.lens = lens;
    a.masks = masks;
    a.mask_words = mask_words;
    a.n_req = n_req;
    a.n_rows = n_rows;
    a.max_blocks = max_blocks;
    a.shift = (uint32_t)__builtin_ctz(block_size);
    a.n_blocks = n_blocks;
    a.num_q = num_q_heads;
    a.num_kv = num_q_heads / gqa_ratio;
    a.kv_dim = kv_dim;
    a.gqa = gqa_ratio;
    a.tokens = tile_rows(head_dim) / gqa_ratio;
    a.per_gqa = 65536 / gqa_ratio + 1;
    a.per_tokens = (uint32_t)((1ull << 32) / a.tokens) + 1;      // exact for the up to 2^24 rows
    // no list is longer than 2^31 - 1
    a.window = (int)std::min(window, 0x7FFFFFFFu);
    a.c = (float)c;
    a.sign = scale < 0.0f ? -1.0f : 1.0f;
    a.out = out;
    // one size for every call of a head_dim, whatever the batch
    const size_t rows = (size_t)2 * kShares * tile_rows(head_dim);
    rc = ensure_workspace(ctx, rows * (head_dim + 2) * 4 + kShares * sizeof(Joined));
    if (rc) return rc;
    a.po = (float *)ctx->ws;
    a.pm = a.po + rows * head_dim;
    a.pl = a.pm + rows;
    a.joined = (Joined *)(a.pl + rows);
    return head_dim == 256 ? launch_packed<256>(ctx, a) : launch_packed<512>(ctx, a);
}

// ---------------------------------------------------------------------
// Masks and clocks of drafted trees.
// ---------------------------------------------------------------------
struct Drafts {
    const uint32_t *parents, *row_start, *lens;
    uint32_t n_rows, words;
    uint32_t *masks, *clocks;
};

// A workgroup per request, a thread per node: node i's mask is its own bit and
// its parent's mask, found by doubling - every round takes over what the node
// that its path has reached has gathered, and that node's reach, so a path of
// depth d takes log2 d rounds.  A parent that is no earlier node ends a path,
// so every path ends.  A launch's latency: 3.5 us for 8 requests, 7 for 500 of up
// to 256 nodes (a walk up the path, node by node, would be 256 dependent reads).
constexpr uint32_t kNodes = 32 * kMaskWords;
template <int W>
__global__ __launch_bounds__(kNodes) void k_draft_trees(Drafts a) {
    __shared__ uint32_t mask[kNodes][W], reach[kNodes];
    const uint32_t r = blockIdx.x, i = threadIdx.x;
    const uint32_t s = min(a.row_start[r], a.n_rows), e = min(a.row_start[r + 1], a.n_rows), len = a.lens[r];
    const uint32_t n = e > s ? e - s : 0, nodes = min(n, 32 * a.words), have = len > n ? len - n : 0;
    if (!n) return;
    uint32_t m[W], to = kNodes;
    if (i < nodes) {
        const uint32_t p = a.parents[s + i];
        if (p < i) to = p;
    }
#pragma unroll
    for (int w = 0; w < W; ++w) m[w] = i < nodes && i / 32 == (uint32_t)w ? 1u << (i % 32) : 0u;
    while (__syncthreads_or(to < kNodes)) {
        reach[i] = to;
#pragma unroll
        for (int w = 0; w < W; ++w) mask[i][w] = m[w];
        __syncthreads();
        if (to < kNodes) {
#pragma unroll
            for (int w = 0; w < W; ++w) m[w] |= mask[to][w];
            to = reach[to];
        }
    }
    if (i < nodes) {
        uint32_t depth = 0;
#pragma unroll
        for (int w = 0; w < W; ++w)
            if ((uint32_t)w < a.words) {
                a.masks[(size_t)(s + i) * a.words + w] = m[w];
                depth += __popc(m[w]);
            }
        a.clocks[s + i] = have + depth - 1;
    }
    for (uint32_t j = nodes + i; j < n; j += kNodes) {          // more rows than the masks have bits
        for (uint32_t w = 0; w < a.words; ++w) a.masks[(size_t)(s + j) * a.words + w] = 0;
        a.clocks[s + j] = have;
    }
}

}  // namespace chn

using namespace chn;

extern "C" int chn_paged_causal_attn(chn_ctx *ctx, const float *q, const float *k_cache, const float *v_cache,
                                     const uint32_t *tables, const uint32_t *row_start, const uint32_t *lens,
                                     uint32_t n_req, uint32_t n_rows, uint32_t max_blocks, uint32_t block_size,
                                     uint32_t n_blocks, uint32_t num_q_heads, uint32_t head_dim, uint32_t kv_dim,
                                     uint32_t gqa_ratio, float scale, uint32_t window, float *out) {
    return packed_attn(ctx, q, k_cache, v_cache, tables, row_start, lens, nullptr, 0, n_req, n_rows, max_blocks, block_size,
                       n_blocks, num_q_heads, head_dim, kv_dim, gqa_ratio, scale, window, out);
}

extern "C" int chn_paged_tree_attn(chn_ctx *ctx, const float *q, const float *k_cache, const float *v_cache,
                                   const uint32_t *tables, const uint32_t *row_start, const uint32_t *lens,
                                   const uint32_t *masks, uint32_t mask_words, uint32_t n_req, uint32_t n_rows,
                                   uint32_t max_blocks, uint32_t block_size, uint32_t n_blocks, uint32_t num_q_heads,
                                   uint32_t head_dim, uint32_t kv_dim, uint32_t gqa_ratio, float scale, uint32_t window,
                                   float *out) {
    CHN_REQUIRE(ctx, masks, "NULL masks");
    CHN_REQUIRE(ctx, mask_words && mask_words <= kMaskWords, "mask_words %u must be in 1..%u", mask_words, kMaskWords);
    CHN_REQUIRE(ctx, !window || window >= 32 * mask_words, "a window of %u is shorter than %u drafted tokens", window,
                32 * mask_words);
    return packed_attn(ctx, q, k_cache, v_cache, tables, row_start, lens, masks, mask_words, n_req, n_rows, max_blocks,
                       block_size, n_blocks, num_q_heads, head_dim, kv_dim, gqa_ratio, scale, window, out);
}

extern "C" int chn_draft_trees(chn_ctx *ctx, const uint32_t *parents, const uint32_t *row_start, const uint32_t *lens,
                               uint32_t n_req, uint32_t n_rows, uint32_t mask_words, uint32_t *masks, uint32_t *clocks) {
    CHN_REQUIRE(ctx, parents && row_start && lens && masks && clocks, "NULL argument");
    CHN_REQUIRE(ctx, mask_words && mask_words <= kMaskWords, "mask_words %u must be in 1..%u", mask_words, kMaskWords);
    if (n_req > kPackedRequests) return set_err(ctx, CHN_E_UNSUPPORTED, "n_req %u exceeds %u", n_req, kPackedRequests);
    if (n_rows > kPackedRows) return set_err(ctx, CHN_E_UNSUPPORTED, "n_rows %u exceeds %u", n_rows, kPackedRows);
    const Span outs[] = {{masks, (size_t)n_rows * mask_words}, {clocks, n_rows}};
    const Span ins[] = {{parents, n_rows}, {row_start, (size_t)n_req + 1}, {lens, n_req}};
    for (const Span &o : outs)
        for (const Span &i : ins) CHN_REQUIRE(ctx, !overlap(o, i), "an output overlaps an input");
    CHN_REQUIRE(ctx, !overlap(outs[0], outs[1]), "masks and clocks overlap");
    CHN_REQUIRE(ctx, ctx, "ctx is NULL");
    if (!n_req || !n_rows) return CHN_OK;
    DeviceGuard dev(ctx);
    const Drafts a{parents, row_start, lens, n_rows, mask_words, masks, clocks};
    if (mask_words == 1) k_draft_trees<1><<<n_req, kNodes, 0, ctx->stream>>>(a);
    else if (mask_words == 2) k_draft_trees<2><<<n_req, kNodes, 0, ctx->stream>>>(a);
    else if (mask_words <= 4) k_draft_trees<4><<<n_req, kNodes, 0, ctx->stream>>>(a);
    else k_draft_trees<8><<<n_req, kNodes, 0, ctx->stream>>>(a);
    CHN_LAUNCHED(ctx, "k_draft_trees");
    return CHN_OK;
}
