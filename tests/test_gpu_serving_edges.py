"""The batched step's calls as the documentation allows them and a single case
does not make them: two contexts at once, recordings that share a workspace,
more rows than share one, one slot named twice, and both sides of the rules
that choose a launch."""
import numpy as np
import pytest

import channel_amd as ca
from gpu_util import say
from oracle import paged
from test_gpu_paged import attn_case, up32
from test_gpu_sample import check, rows, sample

pytestmark = pytest.mark.gpu


class Draws:
    """n rows of V on a context of their own settings; call() enqueues, result() waits."""

    def __init__(self, ctx, seed, n, V):
        self.ctx, self.n, self.V = ctx, n, V
        self.x, self.u = rows(seed, n, V)
        rng = np.random.default_rng(seed)
        self.T, self.k = rng.choice([0, 0.7, 1.3], n).astype(np.float32), rng.choice([0, 0, 5, 64, 900, 2000], n)
        self.p = rng.choice([1, 0.6, 0.95], n).astype(np.float32)
        self.dev = [ctx.upload(a) for a in (self.x, self.T, self.k.astype(np.uint32), self.p, self.u)]
        self.tok, self.prob = ctx.alloc(n * 4), ctx.alloc(n * 4)

    def call(self):
        x, T, k, p, u = self.dev
        self.ctx.call("chn_sample", x, self.n, self.V, self.V, T, k, p, None, u, 0.0, self.tok, self.prob)

    def result(self):
        return self.ctx.download(self.tok, np.uint32, self.n), self.ctx.download(self.prob, np.float32, self.n)

    def verify(self, got=None):
        tok, prob = got or self.result()
        for r in range(self.n):
            want, wp, margin = paged.sample_row(self.x[r], float(self.T[r]), int(self.k[r]), float(self.p[r]), 0.0,
                                                float(self.u[r]), 0.0)
            assert margin > 2.0 ** -32
            assert tok[r] == want and abs(prob[r] - wp) <= 2.0 ** -22 * wp, (r, tok[r], want)


def test_two_contexts_at_once(ctx):
    """Each context has its own stream and workspace: calls of two that run side by side do not meet."""
    say("sampling on two contexts")
    with ca.Context(0) as other:
        a, b = Draws(ctx, 3, 24, 40000), Draws(other, 4, 30, 50001)
        for _ in range(5):
            a.call()
            b.call()
        a.verify()
        b.verify()


def test_recordings_share_a_workspace(ctx):
    """Two recordings and eager calls of other shapes in turn, on one context."""
    say("recorded sampling and attention")
    n, D, nq, gqa, bs, npb, width = 9, 256, 8, 2, 16, 6, 12
    rng = np.random.default_rng(1)
    nb = 80
    kc, vc = (rng.standard_normal((nb * bs, nq // gqa * D)).astype(np.float32) for _ in range(2))
    prefix, tables = rng.permutation(nb)[:npb], rng.integers(0, nb, (n, width))
    q = (rng.standard_normal((n, nq * D)) * 0.2).astype(np.float32)
    dev = dict(q=ctx.upload(q), kc=ctx.upload(kc), vc=ctx.upload(vc), prefix=up32(ctx, prefix), tables=up32(ctx, tables),
               lens=ctx.alloc(n * 4), out=ctx.alloc(n * nq * D * 4))

    def attend():
        ctx.call("chn_prefix_decode_attn", dev["q"], dev["kc"], dev["vc"], dev["prefix"], npb, dev["tables"], dev["lens"], n,
                 width, bs, nb, nq, D, nq // gqa * D, gqa, 1.0, dev["out"])

    def put_lens(lens):
        ctx.upload(np.asarray(lens, np.uint32), dev["lens"])

    draws, more = Draws(ctx, 7, 12, 30000), Draws(ctx, 8, 20, 30000)
    put_lens([0] * n)
    more.call()                                                # the larger shape: the workspace has its size
    attend()
    recs = []
    for call in (draws.call, attend):
        ctx.record_begin()
        call()
        recs.append(ctx.record_end())
    for i in range(4):
        lens = rng.integers(0, width * bs + 1, n)
        put_lens(lens)
        recs[1].submit()
        recs[0].submit()
        got = ctx.download(dev["out"], np.float32, n * nq * D)
        tok = draws.result()
        more.call()
        attend()                                               # the same call outside a recording
        assert np.array_equal(got, ctx.download(dev["out"], np.float32, n * nq * D))
        want, big, absum = paged.prefix_attn(q, kc, vc, prefix, tables, lens, bs, nb, nq, D, gqa, 1.0)
        # sums of at most 192 weighted values and of 256 products, as for every shape
        bound = 2.0 ** -24 * (2 * (D + 2) * absum + 2 * (width * bs + 8)) * np.abs(vc).max()
        assert np.abs(got.reshape(n, -1) - want.reshape(n, -1)).max() <= bound
        if i == 0:
            draws.verify(tok)
            first = tok
        assert np.array_equal(tok[0], first[0]) and np.array_equal(tok[1], first[1])
    more.verify()
    for r in recs:
        r.free()
        ctx._recs.remove(r)


def test_more_rows_than_share_the_workspace(ctx):
    n, V = 1060, 17001
    x, u = rows(5, n, V)
    rng = np.random.default_rng(2)
    check(ctx, x, u, T=rng.choice([0, 0.7, 1], n), k=rng.choice([0, 1, 40, 64], n), p=rng.choice([1, 0.5, 0.95], n),
          m=rng.choice([0, 0, 0.05], n))


@pytest.mark.parametrize("V", [4096, 4097, 8192, 8193, 12288, 12289, 16384, 16385])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_row_widths(ctx, V, cap):
    x, u = rows(V, 8, V)
    x[:, V - 1] += 8
    check(ctx, x, u, T=0.9, k=[0, 0, 0, 0, 60, 60, V - 1, 3000], p=[1, 0.9, 0.5, 0.99, 1, 0.9, 0.9, 0.99],
          m=[0, 0, 0.1, 0, 0, 0.01, 0, 0.001], cap=cap)


@pytest.mark.parametrize("V", [500, 40000])
def test_infinite_largest(ctx, V):
    """+inf: its tokens share the draw; the weights of the others are zero, or finite under a softcap."""
    x, _ = rows(6, 6, V)
    x[:, [3, 77, 400]] = np.inf
    u = [0.1, 0.5, 0.9, 0.1, 0.5, 0.9]
    for kw in (dict(), dict(p=0.999), dict(T=0.01), dict(k=200), dict(k=200, p=0.999), dict(m=0.5, p=0.999)):
        tok, prob = sample(ctx, x, u, **kw)
        assert tok.tolist() == [3, 77, 400] * 2 and np.allclose(prob, 1 / 3), kw
    for kw in (dict(), dict(p=0.9), dict(k=100), dict(m=0.3, p=0.7)):
        check(ctx, x, u, cap=30.0, **kw)


def test_odd_settings_of_long_rows(ctx):
    V = 20000
    x, _ = rows(2, 8, V)
    nan, inf = np.nan, np.inf
    order = np.argsort(-x, axis=1, kind="stable")
    tok, _ = sample(ctx, x, [0.5] * 8, p=[0, -1, nan, 2, 1, 0, 0, 0], k=[0, 0, 1, 1, 1, 9, 0xFFFFFFFF, V + 1])
    assert (tok == order[:, 0]).all()
    check(ctx, x, [0, -1, nan, 1, 7, inf, -inf, 0.5], k=6)
    check(ctx, x, [0, -1, nan, 1, 7, inf, -inf, 0.5], p=0.9)
    check(ctx, x, 0.5, m=[nan, -1, 1, 7, inf, 0.5, 0, 1e-30])
    check(ctx, x, 0.37, T=[1e-30, 1e-3, 10, 1e-40, 1e3, 0.01, 100, 1e-10], p=0.9, m=0.01)
    tok, prob = sample(ctx, x, [0.5] * 8, T=inf)
    assert (tok == V // 2).all() and np.allclose(prob, 1 / V)
    tok, prob = sample(ctx, x, [0.5] * 8, T=inf, p=0.5)        # the half with the largest logits
    for r in range(8):
        kept = np.sort(order[r, :V // 2])
        assert tok[r] == kept[V // 4] and abs(prob[r] * (V // 2) - 1) < 1e-6


@pytest.mark.parametrize("n,own,D,nq,gqa", [
    (1, (4000, 4096), 256, 16, 2),         # few items: the least groups per item
    (64, (0, 500), 256, 16, 2),            # more items than run at once
    (33, (0, 333), 512, 16, 4),
    (70, (0, 300), 512, 8, 8),
    (2, (9000, 12000), 256, 32, 4),        # groups per item by the sum of the lengths
])
def test_own_items(ctx, n, own, D, nq, gqa):
    attn_case(ctx, n, D, nq, gqa, 16, 0, own)


def test_results_do_not_depend_on_the_run(ctx):
    a = attn_case(ctx, 40, 256, 16, 2, 16, 20, (0, 200))
    b = attn_case(ctx, 40, 256, 16, 2, 16, 20, (0, 200))
    assert np.array_equal(a, b)


def test_one_slot_named_twice(ctx):
    """Two tokens with one slot leave either's values there, and their neighbours' slots as they should be."""
    say("rope_at: one slot for two tokens")
    D, nq, nkv, n = 256, 4, 2, 6
    rng = np.random.default_rng(4)
    q, k, v = (rng.standard_normal((n, h, D)).astype(np.float32) for h in (nq, nkv, nkv))
    w = np.ones(D, np.float32)
    clocks, slots = np.array([5, 9, 1, 2, 3, 4]), np.array([7, 7, 0, 1, 2, 3])

    def run(rows_):
        kc, vc = ctx.upload(np.zeros((8, nkv * D), np.float32)), ctx.upload(np.zeros((8, nkv * D), np.float32))
        ctx.call("chn_batch_qkv_rope_at", ctx.upload(q[rows_]), ctx.upload(k[rows_]), ctx.upload(v[rows_]), ctx.upload(w),
                 ctx.upload(w), ctx.alloc(len(rows_) * nq * D * 4), kc, vc, up32(ctx, clocks[rows_]), up32(ctx, slots[rows_]),
                 len(rows_), 8, nq, nkv, D, D, 0, 1e4, 1e-6)
        return [ctx.download(c, np.float32, 8 * nkv * D).reshape(8, -1) for c in (kc, vc)]

    both, first, second = run(np.arange(n)), run(np.array([0])), run(np.array([1]))
    rest = run(np.arange(2, n))
    for c in range(2):
        assert np.all((both[c][7] == first[c][7]) | (both[c][7] == second[c][7]))
        assert np.array_equal(both[c][:4], rest[c][:4]) and not both[c][4:7].any()


@pytest.mark.parametrize("D", [256, 512])
@pytest.mark.parametrize("gqa,n,npb", [(4, 3, 0), (5, 3, 0), (8, 3, 0), (9, 3, 0), (5, 9, 64), (8, 2, 64), (9, 5, 70),
                                       (16, 1, 64), (16, 2, 63), (1, 16, 64), (1, 17, 63), (1, 17, 64), (1, 32, 63),
                                       (1, 33, 63)])
def test_rows_on_both_sides_of_the_rules(ctx, D, gqa, n, npb):
    """Query heads per KV head at the edges of the quads, rows at the edges of quads and tiles."""
    attn_case(ctx, n, D, 2 * gqa, gqa, 16, npb, (0, 90))


@pytest.mark.parametrize("D", [256, 512])
def test_lengths_inside_a_shared_prefix(ctx, D):
    """Rows that see none, a part and all of a prefix whose keys are shared through LDS; the others hold NaN."""
    lens = [0, 1, 15, 16, 17, 100, 640, 641, 1023, 1024, 1025, 1100, 31, 32, 33, 999, 1024, 2]
    attn_case(ctx, len(lens), D, 2, 1, 16, 64, None, lens=lens)
    attn_case(ctx, 6, D, 16, 8, 16, 64, None, lens=lens[2:8], bad=0.2)


@pytest.mark.parametrize("n,nq,gqa,npb,own", [
    (40, 16, 2, 32, (0, 60)),              # 80 rows, keys shared
    (63, 8, 1, 33, (0, 40)),               # 63 and 64 rows on the two sides of sharing
    (64, 8, 1, 32, (0, 40)),
    (32, 8, 1, 94, (0, 40)),               # 32 and 33 rows behind 1504 keys
    (33, 8, 1, 94, (0, 40)),
    (9, 16, 8, 130, (0, 50)),              # a last tile of 8 rows
    (17, 64, 16, 64, (0, 30)),             # 272 rows
])
def test_shared_keys(ctx, n, nq, gqa, npb, own):
    attn_case(ctx, n, 256, nq, gqa, 16, npb, own)


@pytest.mark.parametrize("bad", [0.0, 0.2])
def test_lengths_inside_a_prefix_of_many_rows(ctx, bad):
    """72 rows of heads of 256 share keys of which they see none, a part or all; the others hold NaN."""
    lens = [0, 1, 15, 16, 17, 100, 640, 641, 1023, 1024, 1025, 1100, 31, 32, 33, 999, 1024, 2]
    attn_case(ctx, len(lens), 256, 16, 4, 16, 64, None, lens=lens, bad=bad)
    attn_case(ctx, len(lens), 256, 16, 4, 4, 256, None, lens=lens[::-1], bad=bad)
