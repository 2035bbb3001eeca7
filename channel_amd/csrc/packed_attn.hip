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
#include "chn_internal.h"

#include <cmath>

namespace chn {

typedef float f4q __attribute__((ext_vector_type(4)));

constexpr uint32_t kPackedRequests = 8192;
constexpr uint32_t kPackedRows = 1u << 24;
constexpr uint32_t kMaskWords = 8;          // drafted tokens of a request: 256
constexpr uint32_t kShares = 256;           // workgroups: one per CU
constexpr int kThreads = 512;
// Units are keys.  A tile costs kTileCost besides its keys; a share has kLeastShare units or more, and a cut that
// would fall within kTileCost of a tile's end is moved there.
constexpr int64_t kTileCost = 64, kLeastShare = 192;
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

// What the tiles of a request and KV head cost: tile t walks keys lo(t) ..
// hi(t) - 1, both linear in t (the last tile's end is the work's, not the
// cost's, matter).
struct TileKeys {
    int64_t tiles, T, hi0, lo0;        // hi = hi0 + t T, lo = max(0, lo0 + t T); T is 0 where all tiles see the same keys
    __device__ __forceinline__ TileKeys(const Packed &a, const Seq &s) {
        tiles = (s.n + (int64_t)a.tokens - 1) / a.tokens;
        if (a.mask_words) {
            T = 0;
            hi0 = max(0, min(s.len, s.have + (int)(32 * a.mask_words)));
            lo0 = a.window ? min(max(0, s.have - a.window), (int)hi0) : 0;
        } else {
            T = a.tokens;
            hi0 = max(s.have, 0) + T;
            lo0 = a.window ? (int64_t)s.have + 1 - a.window : -(tiles + 1) * T;
        }
    }
    __device__ __forceinline__ int64_t hi(int64_t t) const { return hi0 + t * T; }
    __device__ __forceinline__ int64_t lo(int64_t t) const { return max((int64_t)0, lo0 + t * T); }
    __device__ __forceinline__ int64_t cost(int64_t t) const { return kTileCost + hi(t) - lo(t); }
    // of all tiles before t
    __device__ __forceinline__ int64_t before(int64_t t) const {
        int64_t sum = t * (kTileCost + hi0) + T * (t * (t - 1) / 2);
        if (!T) return sum - t * max((int64_t)0, lo0);
        const int64_t s0 = lo0 > 0 ? 0 : -lo0 / T + 1;      // the first tile whose lo is above 0
        if (t > s0) sum -= (t - s0) * lo0 + T * ((t - s0) * (s0 + t - 1) / 2);
        return sum;
    }
};
__device__ __forceinline__ int64_t snapped(int64_t at, int64_t cost) {
    return at < kTileCost ? 0 : (at + kTileCost > cost ? cost : at);
}

// One tile's share: rows, and keys key0 .. key1 - 1 (key0 a multiple of 32).
struct Work {
    Seq s;
    const uint32_t *table;
    uint32_t kvh, tile_row, rows;      // the tile's first batch row; rows (tokens x heads)
    int token, key0, key1, limit;      // its first token's index; limit: keys from here on are nobody's
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
            s.lo = max(0, w.s.have + ones - a.window);
        }
    } else {
        s.hi = w.s.have + token + 1;
        s.lo = a.window ? max(0, s.hi - a.window) : 0;
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
    return a.out + ((size_t)(w.tile_row + row / a.gqa) * a.num_q + w.kvh * a.gqa + row % a.gqa) * D;
}

// A row per wave, a key at a time, in plain fp32: what any scores and values
// do, infinities and NaN among them.
template <int D>
__device__ __forceinline__ void rows_plain(const Packed &a, const Work &w) {
    constexpr int N = D / 256;
    const int lane = threadIdx.x & 63;
    for (uint32_t row = threadIdx.x >> 6; row < w.rows; row += kThreads / 64) {
        const int token = w.token + (int)(row / a.gqa);
        const Seen s = seen_by(a, w, token);
        const float *qr = a.q + ((size_t)(w.s.row + token) * a.num_q + w.kvh * a.gqa + row % a.gqa) * D;
        f4q q[N], o[N];
        for (int k = 0; k < N; ++k) {
            q[k] = *(const f4q *)(qr + 4 * lane + 256 * k) * a.sign;
            o[k] = f4q{0, 0, 0, 0};
        }
        float m = kNoScore, l = 0.0f;
        for (int pos = w.key0; pos < w.key1; ++pos) {
            bool ok = pos >= s.lo && pos < s.hi;
            const int node = pos - w.s.have;
            if (s.mask && node >= 0) ok = (s.mask[node >> 5] >> (node & 31)) & 1;      // key1 is below 32 mask_words of them
            const uint32_t slot = ok ? slot_of(a, w.table, pos) : CHN_NO_SLOT;
            if (slot == CHN_NO_SLOT) continue;
            const size_t at = (size_t)slot * a.kv_dim + (size_t)w.kvh * D + 4 * lane;
            float sum = 0.0f;
            for (int k = 0; k < N; ++k) {
                const f4q x = *(const f4q *)(a.kc + at + 256 * k);
                for (int e = 0; e < 4; ++e) sum = fmaf(x[e], q[k][e], sum);
            }
            sum = wave_sum64(sum);
            const float top = fmaxf(m, sum), ref = top == kNoScore ? 0.0f : top;
            const float old = __builtin_amdgcn_exp2f((m - ref) * a.c), p = __builtin_amdgcn_exp2f((sum - ref) * a.c);
            const bool none = sum == kNoScore;                                       // no weight, whatever its V
            m = top;
            l = none ? l : l * old + p;
            for (int k = 0; k < N; ++k) {
                const f4q x = *(const f4q *)(a.vc + at + 256 * k);
                if (!none) o[k] = o[k] * old + p * x;
            }
        }
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        float *to = row_out<D>(a, w, row);
        for (int k = 0; k < N; ++k) *(f4q *)(to + 4 * lane + 256 * k) = o[k] * inv;
        if (w.part >= 0 && lane == 0) {
            a.pm[(size_t)w.part * tile_rows(D) + row] = m;
            a.pl[(size_t)w.part * tile_rows(D) + row] = l;
        }
    }
}

// ---------------------------------------------------------------------
// Tiles on matrix instructions.
// ---------------------------------------------------------------------
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef uint32_t u2q __attribute__((ext_vector_type(2)));
typedef uint32_t u4q __attribute__((ext_vector_type(4)));

// What keys that are nobody's read.
static __device__ __align__(16) const float no_key[512] = {};

// Two fp32 values as fp16 halves hi + lo of 11 bits each: |x - hi - lo| <=
// 2^-22 |x|.  The products hi hi, hi lo and lo hi are exact in fp32, where the
// instructions sum them; lo lo (2^-22 of a product) is dropped.
__device__ __forceinline__ void halves(float a, float b, uint32_t &hi, uint32_t &lo) {
    float ra, rb;
    asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(hi) : "v"(a), "v"(b));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hi), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(hi), "v"(b));
    asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(lo) : "v"(ra), "v"(rb));
}

// The power of two that brings values of magnitude `top` (its bits) below
// 2^15, and its inverse: fp16 then holds what is 2^-39 of the largest and
// more.  At most 2^100.
__device__ __forceinline__ float scale_for(uint32_t top, float &inverse) {
    const uint32_t f = min(0x86000000u - (top & 0x7F800000u), 227u << 23);
    inverse = __builtin_bit_cast(float, (254u << 23) - f);
    return __builtin_bit_cast(float, f);
}
constexpr uint32_t kNotFinite = 0x7F800000u;           // magnitudes from here on are infinities and NaN
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
//     key holds dims 8 g .. + 7 of the step, at place key ^ (4 (step % 4) + g),
//     so that 16 neighbouring lanes of the store fill 256 bytes
//  V: [16 dims][hi, lo][64 lanes][8 keys]; lane 16 g + c holds keys 4 g .. + 3
//     and 16 + 4 g .. + 3, the keys whose weights lane 16 g + row has after the
//     score's product
template <int D>
struct TileLds {
    static constexpr int kKeyBytes = 32 * D * 4;
    unsigned char k[kKeyBytes], v[kKeyBytes];
    float kinv[32], vinv[32];
    float half[D == 512 ? 8 * 64 * 8 : 4];            // scores of the other half of the dims
};

// All waves: what was stored in LDS before is visible behind it.  Loads from
// memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

// Weights are relative to a reference that is moved when a score passes it by
// more than this, in powers of two.
constexpr float kLead = 2.0f;
constexpr float kWeightScale = 8192.0f;               // 2^13: weights of at most 2^kLead stay at or below 2^15

template <int D>
struct Tile {
    static constexpr int H = D / 256, RT = 8 / H;     // waves that share 16 rows (256 dims each), tiles of 16 rows
    static constexpr int S = D / 32;                  // steps
    static constexpr int KR = D == 256 ? 2 : 4;       // keys a lane loads dims of, K
    const Packed &a;
    const Work &w;
    TileLds<D> &lds;
    int lane, wave, rt, half, q, g;
    f4q kr[KR][2], vr[4][H];
    uint32_t ids[2], slots, unheld;                   // of 64 keys: the next ones' blocks, these ones' slots
    bool bad;                                         // an infinity or NaN was met

    __device__ __forceinline__ Tile(const Packed &a_, const Work &w_, TileLds<D> &l) : a(a_), w(w_), lds(l) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        rt = wave % RT;
        half = wave / RT;
        q = lane & 15;
        g = lane >> 4;
        bad = false;
    }

    // chunks come in pairs, 64 keys, a lane each
    __device__ __forceinline__ uint32_t block_of(int pair) const {
        return w.table[min(w.key0 + 64 * pair + lane, w.key1 - 1) >> a.shift];
    }
    __device__ __forceinline__ void take_pair(int pair) {
        const int pos = w.key0 + 64 * pair + lane;
        const uint32_t b = ids[0];
        slots = pos < w.key1 && b < a.n_blocks ? (b << a.shift) + (pos & ((1u << a.shift) - 1)) : CHN_NO_SLOT;
        ids[0] = ids[1];
        ids[1] = block_of(pair + 2);
    }
    __device__ __forceinline__ mem_t row_at(const float *cache, uint32_t slot) const {
        return slot == CHN_NO_SLOT ? (mem_t)no_key : (mem_t)cache + ((size_t)slot * a.kv_dim + (size_t)w.kvh * D);
    }

    __device__ __forceinline__ void load_k(int chunk) {
#pragma unroll
        for (int i = 0; i < KR; ++i) {
            const int key = 32 * (chunk & 1) + (D == 256 ? 16 * i + 2 * wave : 8 * i + wave);
            mem_t p = row_at(a.kc, __builtin_amdgcn_readlane(slots, key));
            if (D == 256) {
                const mem_t p1 = row_at(a.kc, __builtin_amdgcn_readlane(slots, key + 1));
                p = lane & 32 ? p1 : p;
            }
            const mem_t x = p + 8 * (lane & (D / 8 - 1));
            kr[i][0] = load4(x);
            kr[i][1] = load4(x + 4);
        }
    }
    __device__ __forceinline__ void store_k() {
        uint32_t top[KR], most;
#pragma unroll
        for (int i = 0; i < KR; ++i) {
            top[i] = magnitude<8>([&](int e) { return kr[i][e / 4][e % 4]; });
            bad |= top[i] >= kNotFinite;
        }
        if constexpr (D == 256) most = row16_top(swap_max16(top[0], top[1]));      // rows: keys 0, 16, 1, 17 of the wave's
        else most = wave_top4(top);
#pragma unroll
        for (int i = 0; i < KR; ++i) {
            const int key = D == 256 ? 16 * i + 2 * wave + (lane >> 5) : 8 * i + wave, gd = lane & (D / 8 - 1);
            const uint32_t t0 = __builtin_amdgcn_readlane(most, 16 * i), t1 = D == 256 ? __builtin_amdgcn_readlane(most, 32 + 16 * i) : t0;
            float inverse;
            const float scale = scale_for(lane & 32 ? t1 : t0, inverse);
            u4q hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t h, l;
                halves(kr[i][e / 2][2 * (e % 2)] * scale, kr[i][e / 2][2 * (e % 2) + 1] * scale, h, l);
                hi[e] = h;
                lo[e] = l;
            }
            unsigned char *to = lds.k + (((key >> 4) * S + (gd >> 2)) * 2) * 1024 + (gd & 3) * 256 + (((key ^ gd) & 15) * 16);
            *(u4q *)to = hi;
            *(u4q *)(to + 1024) = lo;
            if (gd == 0) lds.kinv[key] = inverse;
        }
    }
    // the wave's four keys: 4 (wave / 2) + 16 (wave % 2) .. + 3
    __device__ __forceinline__ void load_v(int chunk) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const mem_t p = row_at(a.vc, __builtin_amdgcn_readlane(slots, 32 * (chunk & 1) + 4 * (wave >> 1) + 16 * (wave & 1) + i));
#pragma unroll
            for (int h = 0; h < H; ++h) vr[i][h] = load4(p + 4 * lane + 256 * h);
        }
    }
    __device__ __forceinline__ void store_v() {
        uint32_t top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            top[i] = magnitude<4 * H>([&](int e) { return vr[i][e / 4][e % 4]; });
            bad |= top[i] >= kNotFinite;
        }
        const uint32_t most = wave_top4(top);
        f4q inverse;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float inv;
            const float scale = scale_for(__builtin_amdgcn_readlane(most, 16 * i), inv);
            inverse[i] = inv;
#pragma unroll
            for (int h = 0; h < H; ++h) vr[i][h] *= scale;
        }
        if (lane == 0) *(f4q *)(lds.vinv + 4 * (wave >> 1) + 16 * (wave & 1)) = inverse;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t h0, h1, l0, l1;
                halves(vr[0][h][e], vr[1][h][e], h0, l0);
                halves(vr[2][h][e], vr[3][h][e], h1, l1);
                // dim 256 h + 4 lane + e is column lane % 16 of 16 dims
                unsigned char *to = lds.v + ((16 * h + 4 * (lane >> 4) + e) * 2) * 1024 + ((wave >> 1) * 16 + (lane & 15)) * 16 + (wave & 1) * 8;
                *(u2q *)to = u2q{h0, h1};
                *(u2q *)(to + 1024) = u2q{l0, l1};
            }
    }

    __device__ __forceinline__ void run() {
        const uint32_t row = rt * 16 + q;
        const bool valid = row < w.rows, active = (uint32_t)(rt * 16) < w.rows;
        const int chunks = w.key1 > w.key0 ? (w.key1 - w.key0 + 31) / 32 : 0;
        // rows of no token see everything, so that they never stand in a chunk's way
        const int token = w.token + (int)((valid ? row : 0) / a.gqa);
        Seen s = seen_by(a, w, token);
        if (!valid) {
            s.lo = -0x7FFFFFFF;
            s.hi = 0x7FFFFFFF;
        }
        if (chunks) {
            ids[0] = block_of(0);
            ids[1] = block_of(1);
            take_pair(0);
            load_k(0);
            load_v(0);
        }
        u4q qh[8], ql[8];
        float qinv = 0.0f;
        {
            const float *p = a.q + ((size_t)(w.s.row + token) * a.num_q + w.kvh * a.gqa + (valid ? row : 0) % a.gqa) * D + 256 * half + 8 * g;
            f4q x[8][2];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) x[i][e] = load4((mem_t)p + 32 * i + 4 * e);
            uint32_t top = magnitude<64>([&](int e) { return x[e / 8][e / 4 % 2][e % 4]; });
            bad |= top >= kNotFinite;
            top = swap_max16(top, top);
            top = swap_max32(top, top);
            const float scale = scale_for(top, qinv) * a.sign;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t h, l;
                    halves(x[i][e / 2][2 * (e % 2)] * scale, x[i][e / 2][2 * (e % 2) + 1] * scale, h, l);
                    qh[i][e] = h;
                    ql[i][e] = l;
                }
        }
        f4q o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = f4q{0, 0, 0, 0};
        float m = kNoScore, l = 0.0f, vref = 0.0f;
        const unsigned char *kat[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) kat[i] = lds.k + half * 16384 + g * 256 + ((q ^ (4 * i + g)) * 16);
        const unsigned char *vat = lds.v + half * 32768 + lane * 16;
        if (chunks) {
            unheld = (uint32_t)__ballot(slots == CHN_NO_SLOT);
            store_k();
        }
        for (int c = 0; c < chunks; ++c) {
            const int k0 = w.key0 + 32 * c;
            const uint32_t none = unheld;                         // keys of the chunk that are nobody's
            lds_barrier();
            if (c + 1 < chunks) {
                if (c & 1) take_pair((c + 1) >> 1);
                unheld = (uint32_t)(__ballot(slots == CHN_NO_SLOT) >> (c & 1 ? 0 : 32));
                load_k(c + 1);
            }
            // bit k: the row sees key k0 + k
            uint32_t ok = 0xFFFFFFFFu;
            const bool all = !none && __all(s.lo <= k0 && k0 + 32 <= s.hi);
            if (!all) {
                const int from = min(max(s.lo - k0, 0), 32), to = min(max(s.hi - k0, 0), 32);
                if (valid) ok = to > from ? (0xFFFFFFFFu >> (32 - (to - from))) << from : 0u;
                const int node = k0 - w.s.have;
                if (valid && s.mask && node > -32 && node < (int)(32 * a.mask_words)) {
                    const int i = node >> 5;
                    const uint32_t w0 = i >= 0 ? s.mask[i] : 0u, w1 = i + 1 < (int)a.mask_words ? s.mask[i + 1] : 0u;
                    ok |= (uint32_t)(((uint64_t)w1 << 32 | w0) >> (node & 31));
                }
                ok &= ~none;
            }
            const bool some = active && __any(ok != 0 && valid);
            f4q sc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
            if (some) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const unsigned char *p = kat[i & 3] + (t * S + i) * 2048;
                        const h8 kh = *(const h8 *)p, kl = *(const h8 *)(p + 1024);
                        const h8 bh = __builtin_bit_cast(h8, qh[i]), bl = __builtin_bit_cast(h8, ql[i]);
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, bh, sc[t], 0, 0, 0);
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, bl, sc[t], 0, 0, 0);
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, bh, sc[t], 0, 0, 0);
                    }
#pragma unroll
                for (int t = 0; t < 2; ++t) sc[t] = (sc[t] * *(const f4q *)(lds.kinv + 16 * t + 4 * g)) * qinv;
                if (D == 512)
#pragma unroll
                    for (int t = 0; t < 2; ++t) *(f4q *)(lds.half + ((wave * 2 + t) * 64 + lane) * 4) = sc[t];
            }
            store_v();
            lds_barrier();
            if (c + 1 < chunks) load_v(c + 1);
            if (some) {
                if (D == 512)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        // the same order of the halves in both waves
                        const f4q other = *(const f4q *)(lds.half + (((wave ^ RT) * 2 + t) * 64 + lane) * 4);
                        sc[t] = half ? other + sc[t] : sc[t] + other;
                    }
                f4q vi[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) vi[t] = *(const f4q *)(lds.vinv + 16 * t + 4 * g);
                float top = kNoScore, vtop = 0.0f;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (!all) sc[t][i] = (ok >> (16 * t + 4 * g + i)) & 1 ? sc[t][i] : kNoScore;
                        top = largest(top, sc[t][i]);
                        vtop = largest(vtop, vi[t][i]);
                    }
                top = rows4_top(top);
                vtop = lane_f(rows4_top(vtop), 0);
                const bool up = (top - m) * a.c > kLead;
                if (__any(up) || vtop > vref) {
                    const float to = up ? top : m, old = up ? __builtin_amdgcn_exp2f((m - to) * a.c) : 1.0f;
                    const float vto = fmaxf(vtop, vref), f = old * (vref / vto);
                    m = to;
                    vref = vto;
                    l *= old;
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] *= f;
                }
                const float ref = m == kNoScore ? 0.0f : m;
                const float unit = __builtin_bit_cast(float, (267u << 23) - __builtin_bit_cast(uint32_t, vref));      // 2^13 / vref
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f((sc[e / 4][e % 4] - ref) * a.c);
                l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] *= vi[e / 4][e % 4] * unit;
                u4q ph, pl;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t h, lo;
                    halves(p[2 * e], p[2 * e + 1], h, lo);
                    ph[e] = h;
                    pl[e] = lo;
                }
                const h8 bh = __builtin_bit_cast(h8, ph), bl = __builtin_bit_cast(h8, pl);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const h8 vh = *(const h8 *)(vat + i * 2048), vl = *(const h8 *)(vat + i * 2048 + 1024);
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, bh, o[i], 0, 0, 0);
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, bl, o[i], 0, 0, 0);
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, bh, o[i], 0, 0, 0);
                }
            }
            if (c + 1 < chunks) store_k();
        }
        if (__syncthreads_or(bad)) {
            rows_plain<D>(a, w);
            return;
        }
        l = rows4_sum(l);
        if (!valid) return;
        const float inv = l != 0.0f ? 1.0f / l : 0.0f, unit = vref * (1.0f / kWeightScale);
        float *to = row_out<D>(a, w, row) + 256 * half + 16 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(f4q *)(to + 64 * j + 4 * i) =
                    f4q{o[4 * j][i] * inv * unit, o[4 * j + 1][i] * inv * unit, o[4 * j + 2][i] * inv * unit, o[4 * j + 3][i] * inv * unit};
        if (w.part >= 0 && g == 0 && half == 0) {
            a.pm[(size_t)w.part * tile_rows(D) + row] = m;
            a.pl[(size_t)w.part * tile_rows(D) + row] = l;
        }
    }
};

// The workgroup's share: f(work) for each of its tiles or parts of tiles.
template <int D, typename F>
__device__ __forceinline__ void each_work(const Packed &a, F &&f) {
    __shared__ int64_t sums[kThreads / 64];
    __shared__ int64_t found_base;
    __shared__ uint32_t found;
    const uint32_t tid = threadIdx.x, per = (a.n_req + kThreads - 1) / kThreads;
    const int lane = tid & 63, wave = tid >> 6;
    // every request's units; a thread sums its neighbours
    const uint32_t r0 = min(tid * per, a.n_req), r1 = min(r0 + per, a.n_req);
    int64_t mine = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const TileKeys s(a, seq_of(a, r));
        mine += s.before(s.tiles) * a.num_kv;
    }
    const int64_t upto = (int64_t)wave_scan_u64((uint64_t)mine);
    if (lane == 63) sums[wave] = upto;
    if (tid == 0) found = 0xFFFFFFFFu;
    __syncthreads();
    int64_t total = 0, base = upto - mine;
    for (int i = 0; i < kThreads / 64; ++i) {
        base += i < wave ? sums[i] : 0;
        total += sums[i];
    }
    // neighbouring shares, which read the same keys, run on one XCD (workgroup i on XCD i % 8)
    const uint32_t n = (uint32_t)max((int64_t)1, min((int64_t)kShares, total / kLeastShare)), each = (n + 7) / 8;
    const uint32_t share = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    const bool some = (blockIdx.x >> 3) < each && share < n;
    const auto cut = [&](uint32_t w) { return total / n * w + total % n * w / n; };
    if (tid == 0) a.joined[blockIdx.x].rows = 0;      // of share `share`, or of none
    if (!some) return;                                // the whole workgroup
    const int64_t u0 = cut(share), u1 = cut(share + 1);
    if (u0 >= base && u0 < base + mine) {             // one thread, or none
        uint32_t r = r0;
        for (; r + 1 < r1; ++r) {
            const TileKeys s(a, seq_of(a, r));
            const int64_t units = s.before(s.tiles) * a.num_kv;
            if (u0 < base + units) break;
            base += units;
        }
        found = r;
        found_base = base;
    }
    __syncthreads();
    uint32_t r = __builtin_amdgcn_readfirstlane(found);
    if (r >= a.n_req) return;
    Seq s = seq_of(a, r);
    TileKeys sp(a, s);
    int64_t rbase = found_base, head = sp.before(sp.tiles);       // of the request; units of one KV head
    uint32_t kvh = (uint32_t)((u0 - rbase) / head);
    int64_t t = 0;
    {
        const int64_t in = (u0 - rbase) - kvh * head;
        int64_t lo = 0, hi = sp.tiles;                // before(lo) <= in < before(hi)
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (sp.before(mid) <= in) lo = mid;
            else hi = mid;
        }
        t = lo;
    }
    int64_t u = rbase + kvh * head + sp.before(t);
    while (u < u1) {
        const int64_t cost = sp.cost(t);
        const int64_t from = u < u0 ? snapped(u0 - u, cost) : 0, to = u1 - u < cost ? snapped(u1 - u, cost) : cost;
        if (from < to) {
            Work w;
            w.s = s;
            w.table = a.tables + (size_t)r * a.max_blocks;
            w.kvh = kvh;
            w.token = (int)(t * a.tokens);
            w.tile_row = s.row + w.token;
            const int tokens = min(s.n - w.token, (int)a.tokens);
            w.rows = (uint32_t)tokens * a.gqa;
            const int lo = (int)sp.lo(t);
            w.limit = a.mask_words ? (int)sp.hi(t) : max(0, s.have + w.token + tokens);
            // cuts at whole chunks of 32 keys
            w.key0 = from ? (int)((lo + (from - kTileCost / 2) + 31) / 32 * 32) : lo / 32 * 32;
            w.key1 = to < cost ? min((int)((lo + (to - kTileCost / 2) + 31) / 32 * 32), w.limit) : w.limit;
            w.part = from ? 2 * share : (to < cost ? 2 * share + 1 : -1);
            if (from && to == cost && tid == 0) {
                // the share that begins this tile: the last whose first cut is at or before it
                uint32_t first = share;
                while (first && cut(first) > u && snapped(cut(first) - u, cost)) --first;
                a.joined[blockIdx.x] = Joined{first, share, w.tile_row, w.rows, kvh};
            }
            f(w);
        }
        u += cost;
        if (++t < sp.tiles) continue;
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
        s = seq_of(a, r);
        sp = TileKeys(a, s);
    }
}

template <int D>
__global__ __launch_bounds__(kThreads) void k_packed_attn(Packed a) {
    extern __shared__ __align__(16) unsigned char sh[];
    each_work<D>(a, [&](const Work &w) { Tile<D>(a, w, *(TileLds<D> *)sh).run(); });
}

// Joins the parts of the tiles that were cut: a wave takes a row at a time, a
// lane four values per 256 dims.
constexpr uint32_t kJoinRows = 16;
template <int D>
__global__ __launch_bounds__(256) void k_packed_join(Packed a) {
    constexpr uint32_t R = tile_rows(D);
    constexpr int N = D / 256;
    const int lane = threadIdx.x & 63;
    const Joined j = a.joined[blockIdx.x / (R / kJoinRows)];
    const uint32_t row0 = blockIdx.x % (R / kJoinRows) * kJoinRows;
    for (uint32_t row = row0 + (threadIdx.x >> 6); row < min(row0 + kJoinRows, j.rows); row += 4) {
        // the first part is its share's last tile, the others are their shares' first
        const auto at = [&](uint32_t p) { return (size_t)(p == j.first ? 2 * p + 1 : 2 * p) * R + row; };
        float M = kNoScore;
        for (uint32_t p = j.first + lane; p <= j.last; p += 64) M = fmaxf(M, a.pm[at(p)]);
        M = wave_max64(M);
        const float ref = M == kNoScore ? 0.0f : M;
        float L = 0.0f;
        f4q o[N];
        for (int k = 0; k < N; ++k) o[k] = f4q{0, 0, 0, 0};
        for (uint32_t p0 = j.first; p0 <= j.last; p0 += 64) {
            const uint32_t n = min(j.last + 1 - p0, 64u);
            float w = 0.0f;
            if ((uint32_t)lane < n) {
                const size_t i = at(p0 + lane);
                const float part = a.pl[i];
                if (part != 0.0f) w = __builtin_amdgcn_exp2f((a.pm[i] - ref) * a.c) * part;      // NaN: whatever its reference is
            }
            L += wave_sum64(w);
            for (uint32_t i = 0; i < n; ++i) {
                const float wi = lane_f(w, i);
                const float *v = a.po + at(p0 + i) * D + 4 * lane;
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const f4q x = *(const f4q *)(v + 256 * k);
                    if (wi != 0.0f) o[k] += wi * x;                // a part without keys holds nothing
                }
            }
        }
        const float inv = L != 0.0f ? 1.0f / L : 0.0f;
        float *to = a.out + ((size_t)(j.row + row / a.gqa) * a.num_q + j.kvh * a.gqa + row % a.gqa) * D + 4 * lane;
#pragma unroll
        for (int k = 0; k < N; ++k) *(f4q *)(to + 256 * k) = o[k] * inv;
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
    const size_t words = (size_t)n_rows * num_q_heads * head_dim;
    CHN_REQUIRE(ctx, !overlap(chn::Span{q, words}, chn::Span{out, words}), "out overlaps q");
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
// so every path ends.
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
