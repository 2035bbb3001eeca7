// Decode attention of a batch of requests over a paged KV cache whose first
// blocks all requests share (chn_prefix_decode_attn).
//
// The query rows of one KV head - n_req * gqa of them over the prefix, gqa
// over a request's own tokens - times its keys are matrix products, on
// v_mfma_f32_16x16x4_f32 (operands and sums in fp32, as the caches are).  A
// launch holds two kinds of workgroups: prefix items (KV head, RT tiles of 16
// rows, a range of keys) and own items (KV head, request, a range of its
// keys); a second launch joins the items' partial results.  In an item the
// four waves take 16 keys each in turn; a wave multiplies straight from the
// registers it loaded a key's row into (no key is used by two waves), the
// query rows come from LDS.
//
// Lane l = 16 g + c of a wave.  Scores are formed transposed, S^T = K Q^T: as
// A operand lane l holds key c's dims 16 s + 4 g + j (one 16-byte load per s),
// as B operand row c's same dims.  The result register i of lane l is key 4 g +
// i of row c, which is the A operand of step i of P V (row c, key 4 g + i); the
// B operand of that step is V[key 4 g + i][dim 64 m + 4 c + j], again one
// 16-byte load.  So nothing is exchanged between lanes but the rare rescaling.
//
// The running maximum is kept per row and only moved when a score passes it by
// more than kSlack (in powers of two): weights then lie below 2^kSlack, which
// fp32 holds as exactly as those below one.
#include "chn_internal.h"

#include <cmath>

namespace chn {

typedef float f4a __attribute__((ext_vector_type(4)));

constexpr uint32_t kBadSlot = 0xFFFFFFFFu;
constexpr float kSlack = 8.0f;
constexpr float kNone = -__builtin_inff();
constexpr uint32_t kOwnMinGroups = 4;       // 16-key groups per own item at least: one per wave

struct PrefixAttn {
    const float *q, *kc, *vc;
    const uint32_t *prefix, *tables, *lens;
    uint32_t npb, n_req, max_blocks, shift, n_blocks, num_q, num_kv, kv_dim, gqa;
    float exp_hi, exp_lo;      // scale * log2(e) in two parts
    float *out;
    // prefix items: unit u = (KV head, key range), `tiles` row tiles each; see decode_item
    uint32_t splits, split_keys, tiles, prefix_wgs;
    // own items: at most own_cap + n_req of them per KV head
    uint32_t own_cap;
    // partial results: [splits][n_req][num_q] of the prefix, then [own item][num_q]; sums [..][D], then maxima and
    // denominators; own_start[n_req + 1]: the first own item of each request
    float *po, *pm, *pl, *oo, *om, *ol;
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
    return per > kOwnMinGroups ? (uint32_t)per : kOwnMinGroups;
}

__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v, int lane) {      // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t w = __shfl_up(v, o, 64);
        if (lane >= o) v += w;
    }
    return v;
}

// RT tiles of 16 rows over keys [begin, end) of the positions that `blocks`
// maps.  The rows' q lie in LDS (sq, row stride D + 4 floats); lim[rt] is how
// many positions this lane's row c of tile rt may see.
template <int D, int RT>
struct Tile {
    static constexpr int H = D / 256;
    f4a o[RT][D / 64][4];
    float m[RT], l[RT];        // this row's reference, and this lane's part of its denominator

    __device__ __forceinline__ void run(const PrefixAttn &a, const float *sq, const uint32_t *blocks, uint32_t kvh,
                                        uint32_t begin, uint32_t end, const uint32_t (&lim)[RT]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
        const uint32_t mask = (1u << a.shift) - 1;
        // Rows that see none of these keys are dead: computed along, dropped at the end.  Up to `full` every other row
        // sees every key; behind it (a request shorter than the prefix) rows see parts of the groups.
        uint32_t least = end;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = kNone;
            l[rt] = 0.0f;
            if (lim[rt] > begin) least = min(least, lim[rt]);
#pragma unroll
            for (int n = 0; n < D / 64; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[rt][n][j] = f4a{0, 0, 0, 0};
        }
#pragma unroll
        for (int x = 8; x >= 1; x >>= 1) least = min(least, (uint32_t)__shfl_xor(least, x, 64));   // the 16 rows
        least = __builtin_amdgcn_readfirstlane(least);
        const uint32_t full = least >= end ? end : begin + (least - begin) / 16 * 16;

        // key c of the group at kb; a key past the end, or of a bad block, has no slot
        auto block_of = [&](uint32_t kb) { return blocks[min(kb + c, end - 1) >> a.shift]; };
        auto slot_of = [&](uint32_t kb, uint32_t b) {
            const uint32_t k = kb + c;
            return k < end && b < a.n_blocks ? (b << a.shift) + (k & mask) : kBadSlot;
        };
        auto row_of = [&](const float *cache, uint32_t slot) {
            return cache + (size_t)(slot == kBadSlot ? 0u : slot) * a.kv_dim + (size_t)kvh * D;
        };
        f4a A[16], B[16];
        auto load_k = [&](f4a (&d)[16], uint32_t slot, int h) {
            const float *k = row_of(a.kc, slot) + 256 * h + 4 * g;
#pragma unroll
            for (int s = 0; s < 16; ++s) d[s] = *(const f4a *)(k + 16 * s);
        };
        uint32_t vs[4];                            // keys 4 g + i of the group
        auto load_v = [&](f4a (&d)[16], int h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float *v = row_of(a.vc, vs[i]) + 256 * h + 4 * c;
#pragma unroll
                for (int n = 0; n < 4; ++n) d[4 * i + n] = *(const f4a *)(v + 64 * n);
            }
        };
        f4a S[RT], part[RT][4];                    // a score's sum in four chains: shorter ones round less
        auto scores = [&](const f4a (&d)[16], int h) {
#pragma unroll
            for (int s = 0; s < 16; ++s)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const f4a q = *(const f4a *)(sq + (rt * 16 + c) * (D + 4) + 256 * h + 16 * s + 4 * g);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        part[rt][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(d[s][j], q[j], part[rt][j], 0, 0, 0);
                }
        };
        auto clear = [&] {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[rt][j] = f4a{0, 0, 0, 0};
        };
        // scores to weights; seen(rt, i): whether row c of tile rt sees key 4 g + i
        auto softmax = [&](auto &&seen) {
            bool up = false;
            float mx[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                S[rt] = (part[rt][0] + part[rt][1]) + (part[rt][2] + part[rt][3]);
                float t[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) t[i] = seen(rt, i) ? S[rt][i] * a.exp_hi : kNone;
                mx[rt] = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
                up = up || mx[rt] > m[rt] + kSlack;
            }
            if (__any(up)) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const float mn = fmaxf(m[rt], rows4_max(mx[rt]));
                    const float f = mn == m[rt] ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mn);
                    m[rt] = mn;
                    l[rt] *= f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float fr = __shfl(f, 4 * g + i, 64);
#pragma unroll
                        for (int n = 0; n < D / 64; ++n)
#pragma unroll
                            for (int j = 0; j < 4; ++j) o[rt][n][j][i] *= fr;
                    }
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float ref = m[rt] == kNone ? 0.0f : m[rt];
                // the exponent's rounding is that of its distance to the reference, not of the score
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(S[rt][i], a.exp_lo, fmaf(S[rt][i], a.exp_hi, -ref)));
                    S[rt][i] = seen(rt, i) ? w : 0.0f;
                }
                l[rt] += (S[rt][0] + S[rt][1]) + (S[rt][2] + S[rt][3]);
            }
        };
        auto weigh_v = [&](const f4a (&d)[16], int h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t vm = opaque_mask(vs[i] != kBadSlot);
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float v = mask_f(d[4 * i + n][j], vm);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
                            o[rt][4 * h + n][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(S[rt][i], v, o[rt][4 * h + n][j], 0, 0, 0);
                    }
            }
        };
        // Loads are issued ahead of the products they run beside, one buffer of 64 registers each way, and stay there.
        auto fence = [] { __builtin_amdgcn_sched_barrier(0); };

        uint32_t kb = begin + 16 * wave;
        if (kb >= end) return;                     // a whole wave
        uint32_t slot = slot_of(kb, block_of(kb)), nextb = block_of(kb + 64);
        if (kb < full) {
            load_k(A, slot, 0);
            for (;;) {
#pragma unroll
                for (int i = 0; i < 4; ++i) vs[i] = __shfl(slot, 4 * g + i, 64);
                const uint32_t next = slot_of(kb + 64, nextb);
                nextb = block_of(kb + 128);
                clear();
                if constexpr (H == 1) {
                    load_v(B, 0);
                    fence();
                    scores(A, 0);
                } else {
                    load_k(B, slot, 1);
                    fence();
                    scores(A, 0);
                    fence();
                    load_v(A, 0);
                    fence();
                    scores(B, 1);
                    fence();
                    load_v(B, 1);
                    fence();
                }
                softmax([&](int, int i) { return vs[i] != kBadSlot; });
                slot = next;
                fence();
                if constexpr (H == 1) {
                    load_k(A, slot, 0);            // past the end: slot 0, not used
                    fence();
                    weigh_v(B, 0);
                } else {
                    weigh_v(A, 0);
                    fence();
                    load_k(A, slot, 0);
                    fence();
                    weigh_v(B, 1);
                }
                fence();
                kb += 64;
                if (kb >= full) break;
            }
        }
        // Groups that some row sees a part of: the weighted sum key by key, as a weight of zero does not keep an
        // infinity or NaN of an unseen V row out of a product.
#pragma unroll 1
        for (; kb < end; kb += 64) {
            slot = slot_of(kb, block_of(kb));
            clear();
#pragma unroll
            for (int h = 0; h < H; ++h) {
                load_k(A, slot, h);
                scores(A, h);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) vs[i] = __shfl(slot, 4 * g + i, 64);
            softmax([&](int rt, int i) { return vs[i] != kBadSlot && kb + 4 * g + i < lim[rt]; });
            uint32_t rlim[RT][4];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int i = 0; i < 4; ++i) rlim[rt][i] = __shfl(lim[rt], 4 * g + i, 64);
#pragma unroll 1
            for (int kg = 0; kg < 4; ++kg)
#pragma unroll
                for (int ki = 0; ki < 4; ++ki) {
                    const uint32_t key = kb + 4 * kg + ki, ks = __shfl(slot, 4 * kg + ki, 64);
                    if (ks == kBadSlot) continue;  // the whole wave
                    const float *v = row_of(a.vc, ks) + 4 * c;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float p = __shfl(S[rt][ki], 16 * kg + 4 * g + i, 64);
                            if (key < rlim[rt][i])
#pragma unroll
                                for (int n = 0; n < D / 64; ++n) {
                                    const f4a x = *(const f4a *)(v + 64 * n);
#pragma unroll
                                    for (int j = 0; j < 4; ++j) o[rt][n][j][i] = fmaf(p, x[j], o[rt][n][j][i]);
                                }
                        }
                }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
            if (lim[rt] <= begin) {
                m[rt] = kNone;
                l[rt] = 0.0f;
            }
    }

    // The waves' states joined, tile by tile: row c's sum of D values,
    // reference and denominator to where(row) (NULL: no such row).
    template <typename F>
    __device__ __forceinline__ void join(float *sh, F &&where) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15, tid = threadIdx.x;
        float *so = sh, *sm = sh + 4 * 16 * D, *sl = sm + 4 * 16;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float lt = rows4_sum(l[rt]);
            __syncthreads();                       // q, or the tile before, has been read
            if (g == 0) {
                sm[wave * 16 + c] = m[rt];
                sl[wave * 16 + c] = lt;
            }
            __syncthreads();
            const float M = fmaxf(fmaxf(sm[c], sm[16 + c]), fmaxf(sm[32 + c], sm[48 + c]));
            const float f = m[rt] == kNone ? 0.0f : __builtin_amdgcn_exp2f(m[rt] - M);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float fr = __shfl(f, 4 * g + i, 64);
                const bool none = __shfl(m[rt], 4 * g + i, 64) == kNone;
#pragma unroll
                for (int n = 0; n < D / 64; ++n)
                    *(f4a *)(so + ((size_t)wave * 16 + 4 * g + i) * D + 64 * n + 4 * c) =
                        none ? f4a{0, 0, 0, 0} : f4a{o[rt][n][0][i], o[rt][n][1][i], o[rt][n][2][i], o[rt][n][3][i]} * fr;
            }
            __syncthreads();
            if (tid < 16) {
                float L = 0.0f;
                const float Mr = fmaxf(fmaxf(sm[tid], sm[16 + tid]), fmaxf(sm[32 + tid], sm[48 + tid]));
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float mw = sm[w * 16 + tid];
                    L += mw == kNone ? 0.0f : sl[w * 16 + tid] * __builtin_amdgcn_exp2f(mw - Mr);
                }
                float *po, *pm, *pl;
                if (where(rt * 16 + tid, po, pm, pl)) {
                    *pm = Mr;
                    *pl = L;
                }
            }
            for (int e = tid; e < 16 * D / 4; e += 256) {
                const int row = e / (D / 4), d = (e % (D / 4)) * 4;
                float *po, *pm, *pl;
                if (!where(rt * 16 + row, po, pm, pl)) continue;
                const float *s = so + (size_t)row * D + d;
                *(f4a *)(po + d) = (*(const f4a *)s + *(const f4a *)(s + 16 * D)) +
                                   (*(const f4a *)(s + 32 * D) + *(const f4a *)(s + 48 * D));
            }
        }
    }
};

// LDS floats of an item: the query rows, or the four waves' sums of a tile.
template <int D, int RT>
constexpr int lds_floats() {
    const int q = RT * 16 * (D + 4), j = 4 * 16 * D + 2 * 4 * 16;
    return q > j ? q : j;
}

template <int D, int RT>
__global__ __launch_bounds__(256, RT == 1 && D == 256 ? 2 : 1) void k_prefix_attn(PrefixAttn a) {
    extern __shared__ float sh[];
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t P = a.npb << a.shift;
    // rows from..from + n of the (request, head-in-group) rows of a KV head into LDS, zeros behind them
    auto load_q = [&](uint32_t kvh, uint32_t from, uint32_t n, int rows) {
        for (int e = tid; e < rows * (D / 4); e += 256) {
            const uint32_t row = e / (D / 4), d = (e % (D / 4)) * 4;
            f4a v = {0, 0, 0, 0};
            if (row < n) {
                const uint32_t r = (from + row) / a.gqa, h = (from + row) - r * a.gqa;
                v = *(const f4a *)(a.q + ((size_t)r * a.num_q + kvh * a.gqa + h) * D + d);
            }
            *(f4a *)(sh + row * (D + 4) + d) = v;
        }
        __syncthreads();
    };
    if (blockIdx.x < a.prefix_wgs) {
        // the row tiles of one unit run on one XCD (workgroup i runs on XCD i % 8) and share its keys there
        const uint32_t b = blockIdx.x, tile = (b >> 3) % a.tiles, u = (b >> 3) / a.tiles * 8 + (b & 7);
        if (u >= a.num_kv * a.splits) return;
        const uint32_t kvh = u % a.num_kv, split = u / a.num_kv;
        const uint32_t begin = split * a.split_keys, end = min(begin + a.split_keys, P);
        const uint32_t M = a.n_req * a.gqa, row0 = tile * (RT * 16), n = min(M - row0, (uint32_t)RT * 16);
        uint32_t lim[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint32_t row = rt * 16 + (lane & 15);
            lim[rt] = row < n ? a.lens[(row0 + row) / a.gqa] : 0u;
        }
        load_q(kvh, row0, n, RT * 16);
        Tile<D, RT> t;
        t.run(a, sh, a.prefix, kvh, begin, end, lim);
        t.join(sh, [&](uint32_t row, float *&po, float *&pm, float *&pl) {
            if (row >= n) return false;
            const uint32_t r = (row0 + row) / a.gqa, h = (row0 + row) - r * a.gqa;
            const size_t at = ((size_t)split * a.n_req + r) * a.num_q + kvh * a.gqa + h;
            po = a.po + at * D;
            pm = a.pm + at;
            pl = a.pl + at;
            return true;
        });
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
            const int w = __ffsll((unsigned long long)mine) - 1;
            req = r0 + w;
            first = item - __shfl(incl - n, w, 64);
        }
        if (b == 0 && tid < 64 && r < a.n_req) {       // for the launch that joins
            a.own_start[r] = incl - n;
            if (r == a.n_req - 1) a.own_start[a.n_req] = incl;
        }
        start = __shfl(incl, 63, 64);
    }
    if (req == kBadSlot) return;
    const uint32_t len = min(a.lens[req], a.max_blocks << a.shift);
    const uint32_t begin = P + first * per * 16, end = (uint32_t)min((uint64_t)len, (uint64_t)begin + (uint64_t)per * 16);
    const uint32_t lim[1] = {(uint32_t)(lane & 15) < a.gqa ? end : 0u};
    load_q(kvh, req * a.gqa, a.gqa, 16);
    Tile<D, 1> t;
    t.run(a, sh, a.tables + (size_t)req * a.max_blocks, kvh, begin, end, lim);
    t.join(sh, [&](uint32_t row, float *&po, float *&pm, float *&pl) {
        if (row >= a.gqa) return false;
        const size_t at = (size_t)item * a.num_q + kvh * a.gqa + row;
        po = a.oo + at * D;
        pm = a.om + at;
        pl = a.ol + at;
        return true;
    });
}

// Joins a query row's partial results: a wave per row, four values per lane
// and 256 dims.
template <int D>
__global__ __launch_bounds__(256) void k_prefix_join(PrefixAttn a) {
    const int lane = threadIdx.x & 63;
    const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.n_req * a.num_q) return;
    const uint32_t r = row / a.num_q, h = row - r * a.num_q, stride = a.n_req * a.num_q;
    const bool own = a.own_start != nullptr;
    const uint32_t o0 = own ? a.own_start[r] : 0u, no = own ? a.own_start[r + 1] - o0 : 0u;
    const uint32_t parts = a.splits + no;
    auto at = [&](uint32_t p, bool &prefix) {
        prefix = p < a.splits;
        return prefix ? (size_t)p * stride + row : (size_t)(o0 + p - a.splits) * a.num_q + h;
    };
    float M = kNone;
    for (uint32_t p = lane; p < parts; p += 64) {
        bool pre;
        const size_t i = at(p, pre);
        M = fmaxf(M, pre ? a.pm[i] : a.om[i]);
    }
    M = wave_max64(M);
    f4a acc[D / 256];
#pragma unroll
    for (int k = 0; k < D / 256; ++k) acc[k] = f4a{0, 0, 0, 0};
    float L = 0.0f;
    for (uint32_t p = 0; p < parts; ++p) {
        bool pre;
        const size_t i = at(p, pre);
        const float m = pre ? a.pm[i] : a.om[i];
        if (m == kNone) continue;
        const float w = __builtin_amdgcn_exp2f(m - M);
        const float *o = (pre ? a.po : a.oo) + i * D;
        L += w * (pre ? a.pl[i] : a.ol[i]);
#pragma unroll
        for (int k = 0; k < D / 256; ++k) acc[k] += w * *(const f4a *)(o + 256 * k + 4 * lane);
    }
    const float inv = parts && L != 0.0f ? 1.0f / L : 0.0f;      // no token: zeros
#pragma unroll
    for (int k = 0; k < D / 256; ++k) *(f4a *)(a.out + (size_t)row * D + 256 * k + 4 * lane) = acc[k] * inv;
}

template <int D, int RT>
static int launch_items(chn_ctx *ctx, const PrefixAttn &a, uint32_t grid) {
    constexpr size_t lds = lds_floats<D, RT>() * sizeof(float);
    static_assert(lds <= 160 * 1024, "LDS per workgroup");
    if (grid) {
        k_prefix_attn<D, RT><<<grid, 256, lds, ctx->stream>>>(a);
        CHN_LAUNCHED(ctx, "k_prefix_attn");
    }
    k_prefix_join<D><<<(a.n_req * a.num_q + 3) / 4, 256, 0, ctx->stream>>>(a);
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
    const uint32_t rt_most = head_dim == 256 ? 2 : 1;
    uint32_t rt = 1;
    while (rt < rt_most && M > rt * 16) rt *= 2;
    if (!P) rt = 1;
    if (P) {
        a.tiles = (M + rt * 16 - 1) / (rt * 16);
        // about one workgroup per CU, 64 keys (16 per wave) at least
        const uint32_t want = std::max(1u, 256 / std::max(1u, a.tiles * a.num_kv));
        a.split_keys = ((P + want - 1) / want + 63) / 64 * 64;
        a.splits = (P + a.split_keys - 1) / a.split_keys;
        const uint64_t wgs = (uint64_t)(a.num_kv * a.splits + 7) / 8 * 8 * a.tiles;
        if (wgs > 0x7FFFFFFF) return set_err(ctx, CHN_E_UNSUPPORTED, "too many query rows for one call");
        a.prefix_wgs = (uint32_t)wgs;
    }
    uint64_t grid = a.prefix_wgs, items = 0;
    if (max_blocks > n_prefix_blocks) {
        a.own_cap = std::max(1u, 1024 / a.num_kv);
        items = a.own_cap + n_req;
        grid += items * a.num_kv;
    }
    if (grid > 0x7FFFFFFF) return set_err(ctx, CHN_E_UNSUPPORTED, "too many requests and heads for one call");
    const size_t prow = (size_t)a.splits * n_req * num_q_heads, orow = (size_t)items * num_q_heads;
    rc = ensure_workspace(ctx, (prow + orow) * (head_dim + 2) * 4 + ((size_t)n_req + 1) * 4);
    if (rc) return rc;
    a.po = (float *)ctx->ws;
    a.oo = a.po + prow * head_dim;
    a.pm = a.oo + orow * head_dim;
    a.pl = a.pm + prow;
    a.om = a.pl + prow;
    a.ol = a.om + orow;
    a.own_start = items ? (uint32_t *)(a.ol + orow) : nullptr;
    if (head_dim == 256) {
        if (rt == 1) return launch_items<256, 1>(ctx, a, (uint32_t)grid);
        return launch_items<256, 2>(ctx, a, (uint32_t)grid);
    }
    return launch_items<512, 1>(ctx, a, (uint32_t)grid);
}
