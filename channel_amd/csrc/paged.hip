// A batch of requests over one paged KV cache: block tables and slot maps
// from the requests' lengths, and q/k norm + RoPE + K/V write of tokens at
// clocks and slots of their own.  (The attention that reads such a cache is
// in prefix_attn.hip, the choice of the next tokens in sample.hip.)
#include "chn_internal.h"

#include <cmath>

namespace chn {

// ---------------------------------------------------------------------
// Block tables and slot maps.
// ---------------------------------------------------------------------
constexpr uint32_t kMaxRequests = 8192;     // two words of LDS each
constexpr uint32_t kTabThreads = 1024;
static_assert(kTabThreads / 64 == 16, "the waves' sums are a row of 16 lanes");

struct Tables {
    const uint32_t *lens, *n_new, *prefix, *free_blocks, *taken;
    uint32_t n_req, npb, n_free, n_blocks, shift, max_blocks, max_tokens;
    uint32_t *tables, *lens_out, *row_start, *slots, *clocks, *status;
};

// What request r does: its first new token's position, and the blocks that
// hold its tokens before and after.  64-bit: the lengths are the caller's.
struct Grow {
    uint64_t begin, first, last;
    bool fresh;
};
__device__ __forceinline__ Grow grow_of(const Tables &a, uint32_t len, uint32_t n_new) {
    const uint64_t P = (uint64_t)a.npb << a.shift, mask = (1ull << a.shift) - 1;
    Grow g;
    g.fresh = n_new && len < P;
    g.begin = g.fresh ? P : len;
    g.first = (g.begin + mask) >> a.shift;
    g.last = (g.begin + n_new + mask) >> a.shift;
    return g;
}

// One launch, no order between its workgroups: each of them sums all
// requests' rows and blocks by itself (n_req <= 8192: at most eight rounds of
// one block scan, the lengths from L2), so each knows whether the call holds
// and where its own share lies, and none waits for another.  A thread then
// takes a row of the batch (its request by bisection of the starts in LDS);
// the thread of a block's first token enters the block.  Bound by the launch
// and by three latencies (lengths, table entries, writes): 32 requests of one
// token 3.9 us, 1024 requests of 131072 tokens in all, with 300 new prefixes,
// 5.1 us.
__global__ __launch_bounds__(kTabThreads) void k_block_tables(Tables a) {
    extern __shared__ uint32_t sh[];
    uint32_t *row0 = sh, *blk0 = sh + a.n_req;         // first row, first of the handed-out blocks
    __shared__ uint64_t wsum[2][kTabThreads / 64];
    __shared__ uint32_t bad;
    const uint32_t tid = threadIdx.x, nth = gridDim.x * kTabThreads, gid = blockIdx.x * kTabThreads + tid;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid == 0) bad = 0;
    __syncthreads();
    uint64_t rows = 0, blocks = 0;
    uint32_t flags = 0;
    for (uint32_t base = 0; base < a.n_req; base += kTabThreads) {
        const uint32_t r = base + tid;
        const uint32_t n = r < a.n_req ? a.n_new[r] : 0u;
        const Grow g = grow_of(a, r < a.n_req ? a.lens[r] : 0u, n);
        const uint64_t need = n ? g.last - g.first : 0;
        if (n && g.last > a.max_blocks) flags = CHN_TABLES_TOO_LONG;
        const uint64_t sn = wave_scan_u64(n), sb = wave_scan_u64(need);
        if (lane == 63) {
            wsum[0][wave] = sn;
            wsum[1][wave] = sb;
        }
        __syncthreads();
        const uint64_t vn = row16_scan_u64(wsum[0][lane & 15]), vb = row16_scan_u64(wsum[1][lane & 15]);
        const uint64_t bn = rows + (wave ? lane64(vn, wave - 1) : 0), bb = blocks + (wave ? lane64(vb, wave - 1) : 0);
        rows += lane64(vn, 15);
        blocks += lane64(vb, 15);
        if (r < a.n_req) {
            // beyond 32 bits only where the call is refused below
            row0[r] = (uint32_t)(bn + sn - n);
            blk0[r] = (uint32_t)(bb + sb - need);
        }
        __syncthreads();
    }
    const uint64_t taken = a.taken ? *a.taken : 0u;
    if (flags) atomicOr(&bad, flags);
    __syncthreads();
    flags = bad;
    if (taken + blocks > a.n_free) flags |= CHN_TABLES_NO_BLOCKS;
    if (rows > a.max_tokens) flags |= CHN_TABLES_TOO_MANY;
    if (gid == 0) {
        const uint64_t t = taken + blocks;
        a.status[0] = flags;
        a.status[1] = t > 0xFFFFFFFFull ? 0xFFFFFFFFu : (uint32_t)t;
        a.status[2] = rows > 0xFFFFFFFFull ? 0xFFFFFFFFu : (uint32_t)rows;
    }
    if (flags) return;

    const uint32_t bmask = (1u << a.shift) - 1;
    for (uint32_t r = gid; r <= a.n_req; r += nth) {
        if (r == a.n_req) {
            a.row_start[r] = (uint32_t)rows;
            break;
        }
        const uint32_t n = a.n_new[r];
        a.row_start[r] = row0[r];
        a.lens_out[r] = (uint32_t)(grow_of(a, a.lens[r], n).begin + n);
    }
    for (uint64_t t64 = gid; t64 < rows; t64 += nth) {      // up to 2^32 - 1 rows
        const uint32_t t = (uint32_t)t64;
        uint32_t lo = 0, hi = a.n_req;                  // the last request whose first row is <= t
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (row0[mid] <= t) lo = mid;
            else hi = mid;
        }
        const Grow g = grow_of(a, a.lens[lo], a.n_new[lo]);
        const uint32_t pos = (uint32_t)g.begin + (t - row0[lo]), j = pos >> a.shift;
        uint32_t *entry = a.tables + (size_t)lo * a.max_blocks + j;
        uint32_t b;
        if (j >= g.first) {
            b = a.free_blocks[taken + blk0[lo] + (j - (uint32_t)g.first)];
            if ((pos & bmask) == 0) *entry = b;
        } else {
            b = *entry;                                 // a block that it already held: written by nobody here
        }
        a.slots[t] = b < a.n_blocks ? (b << a.shift) + (pos & bmask) : CHN_NO_SLOT;
        a.clocks[t] = pos;
    }
    // the prefix's entries of new requests
    const uint64_t np = (uint64_t)a.n_req * a.npb;
    for (uint64_t i = gid; i < np; i += nth) {
        const uint32_t r = (uint32_t)(i / a.npb), j = (uint32_t)(i - (uint64_t)r * a.npb);
        if (grow_of(a, a.lens[r], a.n_new[r]).fresh) a.tables[(size_t)r * a.max_blocks + j] = a.prefix[j];
    }
}

// ---------------------------------------------------------------------
// q/k norm + RoPE + K/V write at given clocks and slots.
// ---------------------------------------------------------------------
struct RopeAt {
    const float *q_in, *k_in, *v_in, *qw, *kw;   // v_in: k_in where V is the raw K
    float *q_out, *kc, *vc;
    const uint32_t *clocks, *slots;
    uint32_t n_slots, num_q, num_kv, D, rot, groups;
    double log2_theta;
    float eps;
};

// (cos, sin) of clock * theta^(-2d / rot): the turns are formed in 64 bits
// and only their fraction is rounded to 32, so the angle is off by 2^-25 of a
// half turn (the turns' own roundings, 2^-51 or so of at most clock / 6.28,
// reach that at clocks of 2^28, and 2^-22 at the last).
__device__ __forceinline__ float2 rope_angle(const RopeAt &a, uint32_t clock, uint32_t d) {
    const double freq = exp2(-(2.0 * d / a.rot) * a.log2_theta);
    const double turns = (double)clock * freq * 0.15915494309189535;      // 1 / (2 pi)
    const float half = (float)(2.0 * (turns - rint(turns)));
    float s, c;
    sincospif(half, &s, &c);
    return float2{c, s};
}

// RMSNorm * w, then RoPE on pairs (d, d + rot / 2), for query and key heads;
// unit RMSNorm for V.  Any head_dim up to 64 * DPL, any even rot, any
// alignment.  A workgroup takes four rows of one token, one per wave; the
// token's angles are evaluated once, one per thread, and handed round in LDS.
// 1500 tokens of 16 and 8 heads of 128: 18 us (49 MB, 10 at a copy's rate); of
// 256 with 100 of them rotated 27 (the form below: 20), of 16 and 4 heads of 512
// with 500 38 (30): loads of 4 bytes, one row per wave, angles for four rows.
template <int DPL>
__global__ __launch_bounds__(256) void k_rope_at(RopeAt a) {
    __shared__ float2 cs[256];
    __shared__ float buf[4][64 * DPL];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t t = blockIdx.x / a.groups, row = (blockIdx.x - t * a.groups) * 4 + wave;
    const uint32_t D = a.D, half = a.rot / 2, nrow = a.num_q + 2 * a.num_kv;
    const size_t q_dim = (size_t)a.num_q * D, kv_dim = (size_t)a.num_kv * D;
    if ((uint32_t)tid < half) cs[tid] = rope_angle(a, a.clocks[t], tid);
    __syncthreads();
    if (row >= nrow) return;                            // a whole wave; no barrier follows
    const bool q = row < a.num_q, k = !q && row < a.num_q + a.num_kv;
    const uint32_t h = q ? row : (k ? row - a.num_q : row - a.num_q - a.num_kv);
    const float *in = (q ? a.q_in + t * q_dim : (k ? a.k_in : a.v_in) + t * kv_dim) + (size_t)h * D;
    float v[DPL], ss = 0.0f;
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
        const uint32_t d = lane + 64u * j;
        v[j] = d < D ? in[d] : 0.0f;
        ss += v[j] * v[j];
    }
    const float inv = 1.0f / sqrtf(wave_sum64(ss) / (float)D + a.eps);
    const uint32_t slot = a.slots[t];
    if (!q && slot >= a.n_slots) return;
    if (!q && !k) {
        float *o = a.vc + (size_t)slot * kv_dim + (size_t)h * D;
#pragma unroll
        for (int j = 0; j < DPL; ++j)
            if (lane + 64u * j < D) o[lane + 64 * j] = v[j] * inv;
        return;
    }
    const float *nw = q ? a.qw : a.kw;
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
        const uint32_t d = lane + 64u * j;
        v[j] = d < D ? (v[j] * inv) * nw[d] : 0.0f;
        buf[wave][d] = v[j];
    }
    // the wave reads only what it wrote itself
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float *o = q ? a.q_out + t * q_dim + (size_t)h * D : a.kc + (size_t)slot * kv_dim + (size_t)h * D;
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
        const uint32_t d = lane + 64u * j;
        if (d >= D) continue;
        float r = v[j];
        if (d < half) r = r * cs[d].x - buf[wave][d + half] * cs[d].y;
        else if (d < a.rot) r = buf[wave][d - half] * cs[d - half].y + r * cs[d - half].x;
        o[d] = r;
    }
}

// The same for head_dim 256 * N, rows of 16-byte aligned values and rot a
// multiple of 8: lane l holds dims 4 l + 256 j .. + 3, and the row's partner
// values come as 16 bytes from the wave's own LDS row.  A workgroup takes 8
// rows of one token, a wave two of them with all their loads in flight, so
// the angles are evaluated once per 8 rows, while those loads are under way.
// Bound by memory: 1500 tokens of 16 query and 4 KV heads of 512 (135 MB)
// take 27 us, 5.0 TB/s (27 with one row per wave, 31 with four); with 16 and 8
// heads of 256 18.4 (20.5 and 18.6).  24 tokens of those take 4: the launch,
// then loads, a sum and writes behind one another.
typedef float f4p __attribute__((ext_vector_type(4)));
template <int N>
__global__ __launch_bounds__(256) void k_rope_at4(RopeAt a) {
    constexpr uint32_t D = 256 * N, HPW = 2;
    __shared__ float2 cs[D / 2];
    __shared__ f4p buf[4][D / 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t t = blockIdx.x / a.groups, row0 = ((blockIdx.x - t * a.groups) * 4 + wave) * HPW;
    const uint32_t half = a.rot / 2, nrow = a.num_q + 2 * a.num_kv, nk = a.num_q + a.num_kv;
    const uint32_t slot = a.slots[t], clock = a.clocks[t];
    f4p v[HPW][N], wq[N], wk[N];
#pragma unroll
    for (uint32_t i = 0; i < HPW; ++i) {
        const uint32_t row = min(row0 + i, nrow - 1);                // past the last: it again, left out below
        const float *in = row < a.num_q ? a.q_in + ((size_t)t * a.num_q + row) * D
                          : row < nk    ? a.k_in + ((size_t)t * a.num_kv + row - a.num_q) * D
                                        : a.v_in + ((size_t)t * a.num_kv + row - nk) * D;
#pragma unroll
        for (int j = 0; j < N; ++j) v[i][j] = *(const f4p *)(in + 256 * j + 4 * lane);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        wq[j] = *(const f4p *)(a.qw + 256 * j + 4 * lane);
        wk[j] = *(const f4p *)(a.kw + 256 * j + 4 * lane);
    }
    if ((uint32_t)tid < half) cs[tid] = rope_angle(a, clock, tid);
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < HPW; ++i) {
        const uint32_t row = row0 + i;
        if (row >= nrow) return;                                     // a whole wave; no barrier follows
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) ss += (v[i][j].x * v[i][j].x + v[i][j].y * v[i][j].y) + (v[i][j].z * v[i][j].z + v[i][j].w * v[i][j].w);
        const float inv = 1.0f / sqrtf(wave_sum64(ss) / (float)D + a.eps);
        if (row >= a.num_q && slot >= a.n_slots) continue;
        if (row >= nk) {
            float *o = a.vc + ((size_t)slot * a.num_kv + row - nk) * D;
#pragma unroll
            for (int j = 0; j < N; ++j) *(f4p *)(o + 256 * j + 4 * lane) = v[i][j] * inv;
            continue;
        }
        const bool q = row < a.num_q;
        float *o = q ? a.q_out + ((size_t)t * a.num_q + row) * D : a.kc + ((size_t)slot * a.num_kv + row - a.num_q) * D;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[i][j] = (v[i][j] * inv) * (q ? wq[j] : wk[j]);
            buf[wave][64 * j + lane] = v[i][j];
        }
        // the wave reads only what it wrote itself
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t d = 256 * j + 4 * lane;
            f4p r = v[i][j];
            if (d < a.rot) {
                const bool lo = d < half;
                const uint32_t at = lo ? d : d - half;
                const f4p p = buf[wave][(lo ? d + half : d - half) / 4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 x = cs[at + e];
                    r[e] = lo ? r[e] * x.x - p[e] * x.y : p[e] * x.y + r[e] * x.x;
                }
            }
            *(f4p *)(o + d) = r;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();                             // before the next row overwrites buf
    }
}

}  // namespace chn

using namespace chn;

extern "C" int chn_block_tables(chn_ctx *ctx, const uint32_t *lens, const uint32_t *n_new, uint32_t n_req,
                                const uint32_t *prefix_blocks, uint32_t n_prefix_blocks,
                                const uint32_t *free_blocks, uint32_t n_free, const uint32_t *taken,
                                uint32_t n_blocks, uint32_t block_size, uint32_t max_blocks, uint32_t max_tokens,
                                uint32_t *tables, uint32_t *lens_out, uint32_t *row_start, uint32_t *slots,
                                uint32_t *clocks, uint32_t *status) {
    CHN_REQUIRE(ctx, row_start && status, "NULL argument");
    CHN_REQUIRE(ctx, !n_req || (lens && n_new && tables && lens_out), "NULL argument");
    CHN_REQUIRE(ctx, !max_tokens || (slots && clocks), "NULL argument");
    CHN_REQUIRE(ctx, (!n_prefix_blocks || prefix_blocks) && (!n_free || free_blocks), "NULL argument");
    int rc = check_blocks(ctx, block_size, n_blocks, max_blocks);
    if (rc) return rc;
    CHN_REQUIRE(ctx, n_prefix_blocks <= max_blocks, "%u prefix blocks in tables of %u", n_prefix_blocks, max_blocks);
    if (n_req > kMaxRequests)
        return set_err(ctx, CHN_E_UNSUPPORTED, "n_req %u exceeds %u", n_req, kMaxRequests);
    // no workgroup waits for another, so what all read must not be written
    const Span in[] = {{lens, n_req}, {n_new, n_req}, {prefix_blocks, n_prefix_blocks}, {free_blocks, n_free},
                       {taken, taken ? 1u : 0u}};
    const Span out[] = {{tables, (size_t)n_req * max_blocks}, {lens_out, n_req}, {row_start, (size_t)n_req + 1},
                        {slots, max_tokens}, {clocks, max_tokens}, {status, 3}};
    for (const Span &o : out) {
        for (const Span &i : in) CHN_REQUIRE(ctx, !overlap(i, o), "an input overlaps an output");
        for (const Span &p : out) CHN_REQUIRE(ctx, &p == &o || !overlap(p, o), "two outputs overlap");
    }
    CHN_REQUIRE(ctx, ctx, "ctx is NULL");
    DeviceGuard dev(ctx);
    const uint64_t most = std::max<uint64_t>(max_tokens, (uint64_t)n_req * n_prefix_blocks);
    const uint32_t grid = (uint32_t)std::min<uint64_t>(std::max<uint64_t>((most + kTabThreads - 1) / kTabThreads, 1), 256);
    k_block_tables<<<grid, kTabThreads, (size_t)n_req * 8, ctx->stream>>>(
        Tables{lens, n_new, prefix_blocks, free_blocks, taken, n_req, n_prefix_blocks, n_free, n_blocks,
               (uint32_t)__builtin_ctz(block_size), max_blocks, max_tokens, tables, lens_out, row_start, slots, clocks,
               status});
    CHN_LAUNCHED(ctx, "k_block_tables");
    return CHN_OK;
}

extern "C" int chn_batch_qkv_rope_at(chn_ctx *ctx, const float *q_in, const float *k_in, const float *v_in,
                                     const float *q_norm_w, const float *k_norm_w, float *q_out, float *k_cache,
                                     float *v_cache, const uint32_t *clocks, const uint32_t *slots, uint32_t n_tok,
                                     uint32_t n_slots, uint32_t num_q_heads, uint32_t num_kv_heads,
                                     uint32_t head_dim, uint32_t rotary_dim, int k_eq_v, float theta, float eps) {
    CHN_REQUIRE(ctx, q_in && k_in && (v_in || k_eq_v) && q_norm_w && k_norm_w && q_out && k_cache && v_cache && clocks &&
                    slots, "NULL argument");
    CHN_REQUIRE(ctx, head_dim > 0 && head_dim <= 512, "head_dim %u must be in 1..512", head_dim);
    CHN_REQUIRE(ctx, rotary_dim <= head_dim && rotary_dim % 2 == 0, "rotary_dim %u must be even and <= head_dim",
                rotary_dim);
    CHN_REQUIRE(ctx, theta > 0.0f && std::isfinite(theta), "theta must be positive and finite");
    CHN_REQUIRE(ctx, num_q_heads <= 65536 && num_kv_heads <= 65536, "too many heads");
    if (k_eq_v) v_in = k_in;
    bool wide = (head_dim == 256 || head_dim == 512) && rotary_dim % 8 == 0;
    for (const void *p : {(const void *)q_in, (const void *)k_in, (const void *)v_in, (const void *)q_norm_w,
                          (const void *)k_norm_w, (const void *)q_out, (const void *)k_cache, (const void *)v_cache})
        wide = wide && aligned(p, 16);
    const uint32_t per = wide ? 8 : 4, groups = (num_q_heads + 2 * num_kv_heads + per - 1) / per;
    CHN_REQUIRE(ctx, (uint64_t)groups * n_tok <= kMaxGrid256, "%u tokens of %u heads are too many for one call", n_tok,
                num_q_heads);
    CHN_REQUIRE(ctx, ctx, "ctx is NULL");
    if (!n_tok || !groups) return CHN_OK;
    DeviceGuard dev(ctx);
    const RopeAt a{q_in, k_in, v_in, q_norm_w, k_norm_w, q_out, k_cache, v_cache, clocks, slots, n_slots, num_q_heads,
                   num_kv_heads, head_dim, rotary_dim, groups, std::log2((double)theta), eps};
    const uint32_t grid = groups * n_tok;
    if (wide) {
        if (head_dim == 256) k_rope_at4<1><<<grid, 256, 0, ctx->stream>>>(a);
        else k_rope_at4<2><<<grid, 256, 0, ctx->stream>>>(a);
    } else if (head_dim > 256) k_rope_at<8><<<grid, 256, 0, ctx->stream>>>(a);
    else k_rope_at<4><<<grid, 256, 0, ctx->stream>>>(a);
    CHN_LAUNCHED(ctx, "k_rope_at");
    return CHN_OK;
}
