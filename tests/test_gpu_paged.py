"""Block tables, RoPE at own clocks and shared-prefix attention on the GPU,
against the 64-bit oracle (oracle/paged.py).

Tolerances (u = 2^-24, half a step of fp32):
 * RoPE rows: the mean square sums D terms in any order, so 1 / rms is off by
   at most (D + 4) u / 2 + u; two products and the rotation (three roundings)
   follow, the angle is off by at most 2^-24 pi and its sine and cosine by two
   steps: every value within ((D + 4) / 2 + 16) u of the sum of the magnitudes
   it is formed from.
 * Attention: a score sums D products, off by at most D u sum|q k| (any order)
   plus two roundings, and the exponential and the weighted sums of L keys add
   (L + 8) u: every value within (2 (D + 2) u max sum|q k| + 2 (L + 8) u)
   max|v|.  Over a row roundings go both ways: a sum of D terms is off by about
   u sqrt(D) max|s|, so the norm of the difference stays within 8 u (sqrt(D)
   max|s| + sqrt(L)) of the norm of the row (8: for the longest of many rows).
"""
import numpy as np
import pytest

import channel_amd as ca
from gpu_util import say
from oracle import paged

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def up32(ctx, a):
    return ctx.upload(np.asarray(a, np.int64).astype(np.uint32))


def down32(ctx, buf, n):
    return ctx.download(buf, np.uint32, n).astype(np.int64)


# ---------------------------------------------------------------------------
# block tables
# ---------------------------------------------------------------------------
class Tables:
    def __init__(self, ctx, lens, n_new, prefix, free, taken, n_blocks, bs, max_tokens, table):
        self.ctx, self.n, self.table = ctx, len(lens), np.asarray(table, np.int64)
        self.args = (list(lens), list(n_new), list(prefix), list(free), taken, n_blocks, bs, max_tokens)
        self.ins = [up32(ctx, a if len(a) else [0]) for a in (lens, n_new, prefix, free, [taken])]
        self.old = [self.table, np.full(self.n, 11), np.full(self.n + 1, 12), np.full(max_tokens + 3, 13),
                    np.full(max_tokens + 3, 14)]
        self.outs = [up32(ctx, a) for a in self.old] + [up32(ctx, [9, 9, 9])]

    def call(self):
        lens, _, prefix, free, _, n_blocks, bs, max_tokens = self.args
        i, o = self.ins, self.outs
        self.ctx.call("chn_block_tables", i[0], i[1], self.n, i[2], len(prefix), i[3], len(free), i[4], n_blocks, bs,
                      self.table.shape[1], max_tokens, *o)

    def got(self):
        return [down32(self.ctx, b, a.size).reshape(a.shape) for b, a in zip(self.outs, self.old)] + [
            down32(self.ctx, self.outs[5], 3)]

    def check(self):
        lens, n_new, prefix, free, taken, n_blocks, bs, max_tokens = self.args
        want = paged.block_tables(lens, n_new, prefix, free, taken, n_blocks, bs, max_tokens, *self.old)
        for name, g, w in zip(("tables", "lens_out", "row_start", "slots", "clocks", "status"), self.got(), want):
            assert np.array_equal(g, np.asarray(w)), name


def random_tables(ctx, seed, n, bs, npb, have, most_new, idle=0.2, fresh=0.3, short=0, slack=5):
    rng = np.random.default_rng(seed)
    new = rng.integers(0, most_new + 1, n)
    new[rng.random(n) < idle] = 0
    lens = npb * bs + rng.integers(0, have + 1, n)
    lens[rng.random(n) < fresh] = 0
    begin = np.maximum(lens, npb * bs)
    width = int((-(-(begin + new) // bs)).max()) + 2
    need = int(sum(-(-(b + m) // bs) - -(-b // bs) for b, m in zip(begin, new) if m))
    n_blocks = need + n * width + 50
    ids = rng.permutation(n_blocks)
    taken = 7
    free = ids[:taken + need + slack - short]
    table = rng.integers(0, n_blocks, (n, width))
    return Tables(ctx, lens, new, ids[-npb:] if npb else [], free, taken, n_blocks, bs, int(new.sum()) + 9, table)


@pytest.mark.parametrize("n,bs,npb,have,most_new", [
    (1, 16, 0, 0, 1), (1, 1, 3, 5, 7), (3, 16, 2, 100, 40), (64, 16, 32, 700, 1), (200, 32, 5, 300, 500),
    (1024, 16, 4, 60, 3), (1025, 8, 1, 20, 20), (8192, 16, 2, 40, 2), (33, 1024, 1, 5000, 3000), (5, 128, 0, 1000, 20000),
])
def test_tables(ctx, n, bs, npb, have, most_new):
    t = random_tables(ctx, n * 7 + bs, n, bs, npb, have, most_new)
    say(f"block_tables n={n} bs={bs} npb={npb} have={have} new<={most_new}")
    t.call()
    t.check()
    t.call()                                          # the same inputs again: the same tables
    t.check()


def test_tables_no_requests(ctx):
    t = Tables(ctx, [], [], [4], [1, 2], 1, 10, 16, 5, np.zeros((0, 3)))
    t.call()
    assert [g.tolist() for g in t.got()[1:]] == [[], [0], [13] * 8, [14] * 8, [0, 1, 0]]


def test_tables_without_taken_or_lists(ctx):
    t = Tables(ctx, [3], [1], [], [], 0, 10, 4, 2, [[6]])
    ctx.call("chn_block_tables", t.ins[0], t.ins[1], 1, 0, 0, 0, 0, 0, 10, 4, 1, 2, *t.outs)
    t.check()


@pytest.mark.parametrize("short,width,tokens,flag", [(6, 0, 0, 1), (0, 1, 0, 2), (0, 0, 1, 4), (6, 1, 1, 7)])
def test_tables_refused_whole(ctx, short, width, tokens, flag):
    """Too few blocks, a table too narrow, too many rows: only the status is written."""
    t = random_tables(ctx, 5, 40, 16, 2, 200, 90, short=short)
    lens, new, prefix, free, taken, n_blocks, bs, max_tokens = t.args
    if width or tokens:
        table = t.table[:, :2 + 2] if width else t.table
        t = Tables(ctx, lens, new, prefix, free, taken, n_blocks, bs, sum(new) - 1 if tokens else max_tokens, table)
    t.call()
    t.check()
    assert t.got()[5][0] == flag


def test_tables_wild_lengths_are_refused(ctx):
    """Lengths and counts near 2^32 sum in 64 bits and are refused, not wrapped."""
    big = 0xFFFFFFFF
    for lens, new in (([big], [big]), ([big, 0], [1, 5]), ([5] * 9, [big] * 9), ([0], [1 << 31])):
        t = Tables(ctx, lens, new, [1], [2, 3], 0, 10, 16, 20, np.zeros((len(lens), 4)))
        t.call()
        t.check()
        assert t.got()[5][0] & 2


def test_tables_bad_blocks(ctx):
    t = Tables(ctx, [2, 0], [9, 3], [], [70, 4, 5], 0, 70, 4, 20, [[99, 8, 8, 8], [8, 8, 8, 8]])
    t.call()
    t.check()
    assert t.got()[3][:2].tolist() == [paged.NO_SLOT] * 2


def test_tables_alternate_in_a_loop(ctx):
    """Steps that feed each other: lens_out and status of one call are the next one's lens and taken."""
    n, bs = 5, 4
    lens, new = np.array([0, 3, 8, 0, 5]), np.array([1, 2, 1, 0, 3])
    prefix, free = [9], list(range(10, 60))
    table = np.zeros((n, 16), np.int64)
    table[[1, 2, 4], 0], table[2, 1], table[4, 1] = 9, 1, 2
    lens[1] = 4
    t = Tables(ctx, lens, new, prefix, free, 0, 100, bs, 40, table)
    other = up32(ctx, np.zeros(n)), up32(ctx, [0, 0, 0])
    want_table, want_len, taken = table, lens, 0
    a = [t.ins[0], t.ins[4], t.outs[1], t.outs[5]]
    b = [t.outs[1], ctx_word(t.outs[5], 1), other[0], other[1]]
    c = [other[0], ctx_word(other[1], 1), t.outs[1], t.outs[5]]
    for step, (ln, tk, lo, st) in enumerate([a, b, c, b, c]):
        ctx.call("chn_block_tables", ln, t.ins[1], n, t.ins[2], 1, t.ins[3], len(free), tk, 100, bs, 16, 40, t.outs[0], lo,
                 t.outs[2], t.outs[3], t.outs[4], st)
        w = paged.block_tables(want_len, new, prefix, free, taken, 100, bs, 40, want_table, want_len, [0] * (n + 1),
                               [13] * 43, [14] * 43)
        want_table, want_len, taken = w[0], w[1], w[5][1]
        assert np.array_equal(down32(ctx, t.outs[0], n * 16).reshape(n, 16), want_table), step
        assert np.array_equal(down32(ctx, lo, n), want_len)
        assert down32(ctx, st, 3).tolist() == w[5]
        rows = w[5][2]
        assert np.array_equal(down32(ctx, t.outs[3], rows), w[3][:rows])


def ctx_word(buf, i):
    return buf.offset(4 * i)


# ---------------------------------------------------------------------------
# RoPE at own clocks and slots
# ---------------------------------------------------------------------------
def rope_case(ctx, n, D, nq, nkv, rot, far, k_eq_v=0, theta=1e6, bad=0.2, shift=0):
    rng = np.random.default_rng(n * 31 + D + rot)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    q, k, v = f(n, nq, D), f(n, nkv, D), f(n, nkv, D)
    qw, kw = 1 + 0.2 * f(D), 1 + 0.2 * f(D)
    n_slots = n + 9
    slots = rng.permutation(n_slots)[:n].astype(np.int64)
    out = rng.random(n) < bad
    slots[out] = rng.choice([paged.NO_SLOT, n_slots, n_slots + 5], out.sum())
    clocks = rng.integers(0, far + 1, n)
    kc, vc = f(n_slots, nkv * D), f(n_slots, nkv * D)

    def put(a):                                       # at `shift` bytes past 256-byte alignment
        b = ctx.alloc(a.nbytes + shift)
        ctx._check("chn_upload", ca.lib.chn_upload(ctx.handle, b.offset(shift), np.ascontiguousarray(a).ctypes.data,
                                                   a.nbytes))
        return b.offset(shift)
    dq, dk, dv, dqw, dkw, dkc, dvc = (put(a) for a in (q, k, v, qw, kw, kc, vc))
    dout = put(np.full((n, nq, D), 3, np.float32))
    say(f"rope_at n={n} D={D} nq={nq} nkv={nkv} rot={rot} far={far} shift={shift}")
    ctx.call("chn_batch_qkv_rope_at", dq, dk, None if k_eq_v else dv, dqw, dkw, dout, dkc, dvc, up32(ctx, clocks),
             up32(ctx, slots), n, n_slots, nq, nkv, D, rot, k_eq_v, theta, 1e-6)
    wq, wk, wv = paged.rope_at(q, k, k if k_eq_v else v, qw, kw, kc, vc, clocks, slots, rot, theta, 1e-6)
    tol = ((D + 4) / 2 + 16) * U

    def within(got, want):
        # a rotated value is formed from its pair: |a| + |b| <= sqrt(2) |pair|
        size = np.abs(want)
        half = rot // 2
        pair = np.sqrt(want[..., :half] ** 2 + want[..., half:rot] ** 2)
        size[..., :half] = size[..., half:rot] = 2 ** 0.5 * pair
        assert np.all(np.abs(got - want) <= tol * size + 1e-30)
    get = lambda p, a: ctx.download(p, np.float32, a.size).reshape(a.shape).astype(np.float64)  # noqa: E731
    within(get(dout, q), wq)
    hit = np.zeros(n_slots, bool)
    hit[slots[slots < n_slots]] = True
    gk, gv = get(dkc, kc), get(dvc, vc)
    assert np.array_equal(gk[~hit], kc[~hit]) and np.array_equal(gv[~hit], vc[~hit])
    rows = (int(hit.sum()), nkv, D)
    within(gk[hit].reshape(rows), wk[hit].reshape(rows))
    assert np.all(np.abs(gv - wv) <= tol * np.abs(wv) + 1e-30)


@pytest.mark.parametrize("n,D,nq,nkv,rot,far", [
    (1, 256, 16, 8, 256, 0), (24, 256, 16, 8, 256, 5000), (7, 256, 2, 1, 128, 100), (300, 256, 16, 8, 256, 4000000000),
    (5, 512, 16, 4, 512, 120000), (65, 512, 8, 1, 256, 3000), (3, 512, 1, 1, 0, 9), (9, 64, 3, 1, 32, 50),
    (4, 100, 2, 2, 74, 1000), (2, 1, 1, 1, 0, 3), (6, 258, 4, 2, 258, 70000), (1100, 256, 8, 2, 256, 9000),
    (700, 512, 8, 4, 512, 9000), (11, 256, 0, 3, 256, 20), (12, 256, 3, 0, 256, 20), (5, 256, 4, 4, 20, 900),
    (5, 512, 4, 4, 508, 900), (130, 256, 5, 3, 64, 77), (130, 512, 5, 3, 16, 77),
])
def test_rope_at(ctx, n, D, nq, nkv, rot, far):
    rope_case(ctx, n, D, nq, nkv, rot, far)


@pytest.mark.parametrize("D,shift", [(256, 4), (512, 8), (256, 16)])
def test_rope_at_any_alignment(ctx, D, shift):
    rope_case(ctx, 20, D, 4, 2, D, 500, shift=shift)


def test_rope_at_v_is_raw_k(ctx):
    rope_case(ctx, 20, 256, 4, 2, 256, 500, k_eq_v=1)
    rope_case(ctx, 20, 512, 4, 2, 512, 500, k_eq_v=1)


def test_rope_at_every_token_without_a_slot(ctx):
    rope_case(ctx, 20, 256, 4, 2, 256, 500, bad=1.1)


def test_rope_at_nothing(ctx):
    b = ctx.alloc(4096)
    ctx.call("chn_batch_qkv_rope_at", b, b, b, b, b, b, b, b, b, b, 0, 4, 4, 2, 256, 256, 0, 1e4, 1e-6)
    ctx.call("chn_batch_qkv_rope_at", b, b, b, b, b, b, b, b, b, b, 3, 4, 0, 0, 256, 256, 0, 1e4, 1e-6)


# ---------------------------------------------------------------------------
# attention over a shared prefix and own blocks
# ---------------------------------------------------------------------------
def attn_case(ctx, n, D, nq, gqa, bs, npb, own, seed=0, extra=0, scale=1.0, bad=0.0, junk=True, lens=None, qs=None,
              width=None, recorded=False):
    """own: the requests' own lengths, or (lo, hi) to draw them from."""
    rng = np.random.default_rng(seed * 977 + n * 13 + D + npb)
    nkv = nq // gqa
    kv_dim = nkv * D + extra
    if lens is None:
        mine = rng.integers(own[0], own[1] + 1, n) if isinstance(own, tuple) else np.asarray(own)
        lens = npb * bs + mine
    lens = np.asarray(lens, np.int64)
    blocks = np.maximum(-(-lens // bs) - npb, 0)
    width = width or npb + int(blocks.max(initial=0)) + 1
    blocks = np.minimum(blocks, width - npb)
    n_blocks = npb + int(blocks.sum()) + 3
    ids = rng.permutation(n_blocks)
    tables = rng.integers(0, 1 << 32, (n, width))               # entries that hold nothing: anything
    at = npb
    for r in range(n):
        tables[r, npb:npb + blocks[r]] = ids[at:at + blocks[r]]
        at += blocks[r]
    prefix = ids[:npb].copy()
    if bad:
        for r in range(n):
            hit = rng.random(blocks[r]) < bad
            tables[r, npb:npb + blocks[r]][hit] = rng.choice([n_blocks, 0xFFFFFFFF, n_blocks + 1], hit.sum())
        prefix[rng.random(npb) < bad] = 0xFFFFFFFF
    kc = rng.standard_normal((n_blocks * bs, kv_dim)).astype(np.float32)
    vc = rng.standard_normal((n_blocks * bs, kv_dim)).astype(np.float32)
    q = (rng.standard_normal((n, nq * D)) * (qs or 3 / np.sqrt(D))).astype(np.float32)
    seen = [paged.request_slots(lens[r], prefix, tables[r], bs, n_blocks) for r in range(n)]
    if junk:                                                     # what no token occupies is never used
        free = np.setdiff1d(np.arange(n_blocks * bs), np.concatenate(seen + [np.zeros(0, np.int64)]))
        kc[free], vc[free] = np.nan, np.inf
        if extra:
            kc[:, nkv * D:], vc[:, nkv * D:] = np.nan, np.nan
    out = ctx.upload(np.full(n * nq * D, 7, np.float32))
    args = (ctx.upload(q), ctx.upload(kc), ctx.upload(vc), up32(ctx, prefix if npb else [0]), npb, up32(ctx, tables),
            up32(ctx, lens), n, width, bs, n_blocks, nq, D, kv_dim, gqa, scale, out)
    say(f"prefix_attn n={n} D={D} nq={nq} gqa={gqa} bs={bs} npb={npb} lens={lens.tolist()[:6]} bad={bad}")
    ctx.call("chn_prefix_decode_attn", *args)
    got = ctx.download(out, np.float32, n * nq * D).reshape(n, nq, D).astype(np.float64)
    if not junk or not extra:
        kc, vc = np.nan_to_num(kc, posinf=0), np.nan_to_num(vc, posinf=0)
    want, big, absum = paged.prefix_attn(q, kc, vc, prefix, tables, lens, bs, n_blocks, nq, D, gqa, scale)
    want = want.reshape(n, nq, D)
    L = max((len(s) for s in seen), default=0)
    vmax = max((float(np.abs(vc[s][:, :nkv * D]).max()) for s in seen if len(s)), default=0.0)
    assert np.all(np.isfinite(got))
    diff = np.abs(got - want)
    assert diff.max() <= (2 * (D + 2) * U * absum + 2 * (L + 8) * U) * vmax + 1e-30
    norm = np.linalg.norm(want, axis=2)
    rel = np.linalg.norm(got - want, axis=2) / np.maximum(norm, 1e-30)
    bound = 8 * U * (np.sqrt(D) * max(big, 1.0) + np.sqrt(L))
    assert np.all(rel[norm > 0] <= bound), (rel.max(), bound)
    for r in range(n):
        if not len(seen[r]):
            assert not got[r].any()
    for b in args:
        if isinstance(b, ca.Buffer):
            b.free()
    return got


@pytest.mark.parametrize("D", [256, 512])
@pytest.mark.parametrize("n,nq,gqa,bs,npb,own", [
    (1, 16, 2, 16, 0, (1, 1)), (1, 2, 1, 16, 1, (0, 0)), (3, 4, 4, 16, 2, (1, 40)), (8, 16, 2, 16, 32, (1, 96)),
    (5, 8, 8, 8, 9, (0, 70)), (33, 16, 16, 32, 3, (1, 50)), (70, 2, 1, 16, 5, (0, 20)), (4, 3, 3, 1, 37, (0, 33)),
    (2, 5, 5, 64, 0, (1000, 3000)), (17, 4, 1, 128, 4, (0, 300)), (9, 24, 12, 4, 11, (0, 30)), (2, 2, 2, 1024, 1, (0, 1500)),
])
def test_prefix_attn(ctx, D, n, nq, gqa, bs, npb, own):
    attn_case(ctx, n, D, nq, gqa, bs, npb, own)


@pytest.mark.parametrize("edge", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513])
def test_prefix_attn_lengths(ctx, edge):
    """Own lengths and prefixes at the edges of chunks and tiles."""
    attn_case(ctx, 3, 256, 4, 2, 1, edge, [0, 1, edge], seed=edge)
    attn_case(ctx, 2, 512, 2, 1, 1, edge, [edge, 3], seed=edge)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 129])
def test_prefix_attn_requests(ctx, n):
    """Request counts at the edges of the row tiles."""
    attn_case(ctx, n, 256, 4, 2, 16, 6, (0, 40), seed=n)
    attn_case(ctx, n, 512, 3, 1, 16, 3, (0, 20), seed=n)


def test_prefix_attn_lengths_inside_the_prefix(ctx):
    """A request that has not reached the prefix's end sees its first tokens only; one without tokens gets zeros."""
    lens = [0, 1, 5, 16, 17, 63, 64, 65, 100, 0, 64]
    attn_case(ctx, len(lens), 256, 8, 2, 16, 4, None, lens=lens)
    attn_case(ctx, len(lens), 512, 4, 4, 16, 4, None, lens=lens)


def test_prefix_attn_no_tokens_at_all(ctx):
    attn_case(ctx, 5, 256, 4, 2, 16, 0, [0] * 5)
    attn_case(ctx, 5, 256, 4, 2, 16, 2, None, lens=[0] * 5)


@pytest.mark.parametrize("D,gqa", [(256, 2), (512, 4), (256, 16)])
def test_prefix_attn_bad_blocks(ctx, D, gqa):
    """Block ids that are out of range take their tokens out, in the prefix too."""
    attn_case(ctx, 9, D, 16, gqa, 8, 12, (0, 90), bad=0.4)
    attn_case(ctx, 3, D, 16, gqa, 16, 2, (0, 20), bad=1.1)


def test_prefix_attn_lengths_beyond_the_table(ctx):
    """A length past the table's end counts as the table's."""
    attn_case(ctx, 3, 256, 4, 2, 16, 1, None, lens=[80, 81, 0xFFFFFFFF], width=5)


def test_prefix_attn_wide_rows_and_scale(ctx):
    attn_case(ctx, 6, 256, 4, 2, 16, 3, (0, 60), extra=256, scale=0.25, qs=1.0)
    attn_case(ctx, 6, 512, 4, 2, 16, 3, (0, 60), extra=4, scale=-0.5)


def test_prefix_attn_peaked_scores(ctx):
    """Scores of deviation 16 (unit q and k, scale 1): one key takes most."""
    attn_case(ctx, 6, 256, 8, 2, 16, 20, (0, 200), qs=1.0)


def test_prefix_attn_long(ctx):
    attn_case(ctx, 3, 256, 2, 2, 64, 40, [9000, 1, 4097])
    attn_case(ctx, 2, 512, 2, 1, 32, 200, [7000, 12])


def test_prefix_attn_many_requests(ctx):
    attn_case(ctx, 600, 256, 2, 2, 16, 2, (0, 9))


def test_prefix_attn_cache_past_four_gib(ctx):
    """Slots whose byte offsets pass 2^32: the tokens sit in the last blocks of a 4.5 GiB cache."""
    D, nq, bs, n = 512, 16, 64, 3
    kv_dim, n_blocks = 16 * D, 2304                            # 32 KiB a slot, 2 MiB a block
    K, V = ctx.alloc(n_blocks * bs * kv_dim * 4), ctx.alloc(n_blocks * bs * kv_dim * 4)
    rng = np.random.default_rng(3)
    prefix, tables = np.array([2303, 5]), np.array([[0, 0, 2302, 2299], [0, 0, 2301, 1], [0, 0, 2300, 0]])
    lens = np.array([128 + 64 + 7, 128 + 30, 128 + 1])
    used = sorted(set(prefix.tolist()) | {int(tables[r, j]) for r in range(n) for j in (2, 3)})
    small = {b: i for i, b in enumerate(used)}
    kc = rng.standard_normal((len(used) * bs, kv_dim)).astype(np.float32)
    vc = rng.standard_normal((len(used) * bs, kv_dim)).astype(np.float32)
    for b in used:
        for buf, a in ((K, kc), (V, vc)):
            part = np.ascontiguousarray(a[small[b] * bs:(small[b] + 1) * bs])
            ctx._check("chn_upload", ca.lib.chn_upload(ctx.handle, buf.offset(b * bs * kv_dim * 4), part.ctypes.data,
                                                       part.nbytes))
    q = (rng.standard_normal((n, nq * D)) * 0.1).astype(np.float32)
    out = ctx.alloc(n * nq * D * 4)
    say("prefix_attn over a 4.5 GiB cache")
    ctx.call("chn_prefix_decode_attn", ctx.upload(q), K, V, up32(ctx, prefix), 2, up32(ctx, tables), up32(ctx, lens), n, 4,
             bs, n_blocks, nq, D, kv_dim, 1, 1.0, out)
    got = ctx.download(out, np.float32, n * nq * D).reshape(n, -1)
    near = np.vectorize(lambda b: small.get(int(b), 0))
    want, big, absum = paged.prefix_attn(q, kc, vc, near(prefix), near(tables), lens, bs, len(used), nq, D, 1, 1.0)
    assert np.abs(got - want).max() <= (2 * (D + 2) * U * absum + 2 * (200 + 8) * U) * np.abs(vc).max()
    K.free()
    V.free()


def test_prefix_attn_nothing(ctx):
    b = ctx.alloc(4096)
    ctx.call("chn_prefix_decode_attn", b, b, b, b, 0, b, b, 0, 4, 16, 4, 4, 256, 512, 2, 1.0, b)
    ctx.call("chn_prefix_decode_attn", b, b, b, b, 0, b, b, 3, 4, 16, 4, 0, 256, 512, 2, 1.0, b)


def test_prefix_attn_agrees_with_decode_attn(ctx):
    """One request without a prefix and blocks of one slot is chn_decode_attn's slot list."""
    D, nq, gqa, S = 256, 16, 2, 700
    rng = np.random.default_rng(8)
    kc, vc = (ctx.upload(rng.standard_normal((4096, 8 * D)).astype(np.float32)) for _ in range(2))
    q = ctx.upload((rng.standard_normal(nq * D) * 0.2).astype(np.float32))
    slots = up32(ctx, rng.permutation(4096)[:S])
    a, b = ctx.alloc(nq * D * 4), ctx.alloc(nq * D * 4)
    ctx.call("chn_decode_attn", q, kc, vc, slots, up32(ctx, [S]), S, nq, D, 8 * D, gqa, 1.0, a)
    ctx.call("chn_prefix_decode_attn", q, kc, vc, 0, 0, slots, up32(ctx, [S]), 1, S, 1, 4096, nq, D, 8 * D, gqa, 1.0, b)
    x, y = ctx.download(a, np.float32, nq * D), ctx.download(b, np.float32, nq * D)
    assert np.linalg.norm(x - y) <= 2e-5 * np.linalg.norm(x)
