// Decode attention of a batch of requests over a paged KV cache whose first
// blocks all requests share (chn_prefix_decode_attn).
#include "chn_internal.h"

namespace chn {

constexpr float kNoScore = -__builtin_inff();

struct PrefixAttn {
    const float *q, *kc, *vc;
    const uint32_t *prefix, *tables, *lens;
    uint32_t npb, n_req, max_blocks, shift, n_blocks, num_q, kv_dim, gqa;
    float scale;
    float *out;
};

// One workgroup per (request, query head): each wave takes every fourth key
// and keeps a running maximum, sum and weighted V row; the waves' states are
// joined in LDS.
template <int D>
__global__ __launch_bounds__(256) void k_prefix_attn(PrefixAttn a) {
    constexpr int N = D / 64;
    __shared__ float sh_o[4][D], sh_m[4], sh_l[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t r = blockIdx.x / a.num_q, h = blockIdx.x - r * a.num_q, kvh = h / a.gqa;
    const uint32_t *table = a.tables + (size_t)r * a.max_blocks;
    const uint32_t len = min(a.lens[r], a.max_blocks << a.shift), mask = (1u << a.shift) - 1;
    const float *q = a.q + ((size_t)r * a.num_q + h) * D;
    float qv[N], o[N], m = kNoScore, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        qv[i] = q[lane + 64 * i];
        o[i] = 0.0f;
    }
    for (uint32_t t = wave; t < len; t += 4) {
        const uint32_t j = t >> a.shift, b = j < a.npb ? a.prefix[j] : table[j];
        if (b >= a.n_blocks) continue;
        const size_t at = (((size_t)b << a.shift) + (t & mask)) * a.kv_dim + (size_t)kvh * D;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(qv[i], a.kc[at + lane + 64 * i], s);
        s = wave_sum64(s) * a.scale;
        const float mn = fmaxf(m, s);
        const float c = m == kNoScore ? 0.0f : expf(m - mn), p = expf(s - mn);
        l = l * c + p;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = o[i] * c + p * a.vc[at + lane + 64 * i];
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) sh_o[wave][lane + 64 * i] = o[i];
    if (lane == 0) {
        sh_m[wave] = m;
        sh_l[wave] = l;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
    float c[4], L = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        c[w] = sh_l[w] > 0.0f ? expf(sh_m[w] - M) : 0.0f;
        L += c[w] * sh_l[w];
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    for (uint32_t d = threadIdx.x; d < (uint32_t)D; d += 256)
        a.out[((size_t)r * a.num_q + h) * D + d] =
            ((c[0] * sh_o[0][d] + c[1] * sh_o[1][d]) + (c[2] * sh_o[2][d] + c[3] * sh_o[3][d])) * inv;
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
    const PrefixAttn a{q, k_cache, v_cache, prefix_blocks, tables, lens, n_prefix_blocks, n_req, max_blocks,
                       (uint32_t)__builtin_ctz(block_size), n_blocks, num_q_heads, kv_dim, gqa_ratio, scale, out};
    if (head_dim == 256) k_prefix_attn<256><<<n_req * num_q_heads, 256, 0, ctx->stream>>>(a);
    else k_prefix_attn<512><<<n_req * num_q_heads, 256, 0, ctx->stream>>>(a);
    CHN_LAUNCHED(ctx, "k_prefix_attn");
    return CHN_OK;
}
