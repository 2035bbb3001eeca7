"""Attention of packed prompts and of drafted trees over a paged cache, and the
trees' masks and clocks, on the GPU against the 64-bit oracle
(oracle/packed.py).

Tolerance of the attention (u = 2^-24, half a step of fp32): a score sums D
products, off by at most D u sum|q k| in any order plus two roundings; the
operands are split into two halves of 11 bits, which leaves at most 2^-22 of an
operand and drops the product of the low halves, another 2^-22 of a product: 12
u of sum|q k| in all.  The exponential and the weighted sums of L keys add (L +
8) u, their split operands 12 u: every value within (2 (D + 14) u max sum|q k|
+ 2 (L + 20) u) max|v|.  Over a row roundings go both ways: a sum of D terms is
off by about u sqrt(D) max|s|, so the norm of the difference stays within 8 u
(sqrt(D) max|s| + sqrt(L) + 12) of the norm of the row.
"""
import numpy as np
import pytest

import channel_amd as ca
from gpu_util import say
from oracle import packed
from test_gpu_paged import down32, up32

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BAD = 0xFFFFFFFF


def chain_masks(counts, words):
    """Each drafted token sees all before it."""
    return [[((1 << (i + 1)) - 1) >> (32 * w) & 0xFFFFFFFF for w in range(words)] for n in counts for i in range(n)]


def random_trees(rng, counts):
    return [int(rng.integers(max(i - 6, -1), i)) & BAD if i else BAD for n in counts for i in range(n)]


class Batch:
    """A batch's device state; new and have tokens per request."""

    def __init__(self, ctx, seed, new, have, D=256, nq=4, gqa=2, bs=16, window=0, words=0, scale=1.0, spare=3, width=None,
                 kv_pad=0, sigma=4.0):
        rng = np.random.default_rng(seed)
        self.ctx, self.D, self.nq, self.gqa, self.bs, self.window, self.words, self.scale = ctx, D, nq, gqa, bs, window, words, scale
        new, have = np.asarray(new), np.asarray(have)
        self.n = len(new)
        self.row_start = np.concatenate([[0], np.cumsum(new)])
        self.rows = int(self.row_start[-1]) + spare
        self.lens = have + new
        blocks = -(-self.lens // bs)
        self.width = width or max(int(blocks.max()), 1) + 1
        self.nb = int(blocks.sum()) + 3
        pool = rng.permutation(self.nb)
        self.tables = np.full((self.n, self.width), BAD)
        at = 0
        for r in range(self.n):
            k = min(int(blocks[r]), self.width)
            self.tables[r, :k] = pool[at:at + k]
            at += int(blocks[r])
        self.kv_dim = nq // gqa * D + kv_pad
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.q = f(self.rows, nq * D) * np.float32(sigma / np.sqrt(D))
        self.kc, self.vc = f(self.nb * bs, self.kv_dim), f(self.nb * bs, self.kv_dim)
        self.old = f(self.rows, nq * D)
        self.parents = random_trees(rng, new) + [7] * spare
        self.masks = None
        if words:
            self.masks, _ = packed.draft_trees(self.parents, self.row_start, self.lens, self.rows, words,
                                               np.zeros((self.rows, words)), np.zeros(self.rows))
        self.dev = {}

    def up(self):
        c = self.ctx
        self.dev = dict(q=c.upload(self.q), kc=c.upload(self.kc), vc=c.upload(self.vc), tables=up32(c, self.tables),
                        row_start=up32(c, self.row_start), lens=up32(c, self.lens), out=c.upload(self.old))
        if self.words:
            self.dev["masks"] = up32(c, self.masks)
        return self

    def args(self):
        d = self.dev
        shape = (self.n, self.rows, self.width, self.bs, self.nb, self.nq, self.D, self.kv_dim, self.gqa, self.scale, self.window,
                 d["out"])
        first = (d["q"], d["kc"], d["vc"], d["tables"], d["row_start"], d["lens"])
        if self.words:
            return ("chn_paged_tree_attn", *first, d["masks"], self.words, *shape)
        return ("chn_paged_causal_attn", *first, *shape)

    def call(self):
        self.ctx.call(*self.args())

    def got(self):
        return self.ctx.download(self.dev["out"], np.float32, self.rows * self.nq * self.D).reshape(self.rows, -1)

    def run(self):
        self.up().call()
        out = self.got()
        for b in self.dev.values():
            b.free()
            self.ctx._bufs.remove(b)
        return out

    def want(self):
        return packed.packed_attn(self.q, self.kc, self.vc, self.tables, self.row_start, self.lens, self.bs, self.nb, self.nq,
                                  self.D, self.gqa, self.scale, self.window, self.masks, self.old)

    def check(self, out=None):
        out = self.run() if out is None else out
        want, big, absum, L = self.want()
        D = self.D
        fine = np.isfinite(want)
        assert np.array_equal(fine, np.isfinite(out)), np.argwhere(fine != np.isfinite(out))[:4]
        assert np.array_equal(np.isnan(want), np.isnan(out))
        assert np.array_equal(want[~fine & ~np.isnan(want)], out[~fine & ~np.isnan(want)])
        vmax = float(np.abs(self.vc[np.isfinite(self.vc)]).max())
        bound = (2 * (D + 14) * U * absum + 2 * (L + 20) * U) * vmax
        taken = int(min(self.row_start[-1], self.rows))
        off = np.abs(np.where(fine, out, 0.0) - np.where(fine, want, 0.0))
        say(f"  max error {off[:taken].max(initial=0):.3g} of {bound:.3g}; L {L} max|s| {big:.3g}")
        assert off[:taken].max(initial=0) <= bound
        assert np.array_equal(out[taken:], self.old[taken:])               # rows of no request
        rowfine = fine.all(1)
        norm = np.linalg.norm(want[rowfine][:taken].reshape(-1, D), axis=1)
        diff = np.linalg.norm(out[rowfine][:taken].reshape(-1, D) - want[rowfine][:taken].reshape(-1, D), axis=1)
        some = norm > 0
        limit = 8 * U * (np.sqrt(D) * big + np.sqrt(L) + 12)
        assert (diff[some] <= limit * norm[some]).all(), (diff[some] / norm[some]).max()


# tokens per tile: 128 / gqa with heads of 256, 64 / gqa with heads of 512; chunks of 32 keys
CAUSAL = [
    dict(new=[1], have=[0]), dict(new=[1], have=[40]), dict(new=[24], have=[0]), dict(new=[33], have=[31]),
    dict(new=[63, 64, 65, 129], have=[0, 1, 31, 32]), dict(new=[0, 5, 0, 0, 7, 0], have=[9, 0, 0, 3, 100, 1]),
    dict(new=[0, 0], have=[4, 0]), dict(new=[3] * 70, have=list(range(70))),
    dict(new=[40, 100], have=[70, 5], window=1), dict(new=[40, 100], have=[70, 5], window=31),
    dict(new=[150, 1, 200], have=[90, 300, 0], window=64), dict(new=[50], have=[50], window=1 << 31),
    dict(new=[20, 70], have=[50, 3], bs=1), dict(new=[20, 70], have=[50, 3], bs=8), dict(new=[20, 70], have=[50, 1030], bs=1024),
    dict(new=[100, 30], have=[9, 80], nq=3, gqa=1), dict(new=[100, 30], have=[9, 80], nq=6, gqa=3),
    dict(new=[50, 30], have=[9, 80], nq=16, gqa=8), dict(new=[30, 9], have=[9, 80], nq=16, gqa=16),
    dict(new=[30, 9], have=[9, 80], nq=13, gqa=13), dict(new=[40], have=[500], nq=1, gqa=1, kv_pad=36),
    dict(new=[30, 45], have=[60, 0], scale=-0.37), dict(new=[30], have=[60], scale=3e-20, sigma=4e20),
    dict(new=[5], have=[3000], nq=2), dict(new=[300], have=[900], nq=2),
]


@pytest.mark.parametrize("D", [256, 512])
@pytest.mark.parametrize("i", range(len(CAUSAL)))
def test_causal(ctx, i, D):
    say("causal", CAUSAL[i], D)
    Batch(ctx, 100 + i, D=D, **CAUSAL[i]).check()


TREES = [
    dict(new=[1], have=[0], words=1), dict(new=[8], have=[20], words=1), dict(new=[32, 5, 0, 17], have=[0, 31, 9, 640], words=1),
    dict(new=[64, 33], have=[7, 100], words=2), dict(new=[100, 3], have=[45, 2], words=4), dict(new=[256, 200], have=[33, 0], words=8),
    dict(new=[30, 9, 1], have=[100, 20, 64], words=1, window=32), dict(new=[60, 9], have=[300, 20], words=2, window=70),
    dict(new=[7] * 40, have=list(range(0, 400, 10)), words=1, bs=8), dict(new=[40], have=[10], words=1),
    dict(new=[20, 31], have=[90, 3], nq=16, gqa=16, words=1), dict(new=[20, 31], have=[90, 3], nq=5, gqa=5, words=1),
    dict(new=[16, 4], have=[2500, 90], nq=2, words=1),
]


@pytest.mark.parametrize("D", [256, 512])
@pytest.mark.parametrize("i", range(len(TREES)))
def test_trees(ctx, i, D):
    say("tree", TREES[i], D)
    Batch(ctx, 200 + i, D=D, **TREES[i]).check()


@pytest.mark.parametrize("D", [256, 512])
def test_any_mask(ctx, D):
    """Masks that are no tree's: none, not itself, later tokens, bits of tokens that are not there."""
    say("any mask", D)
    b = Batch(ctx, 5, [30, 40, 3, 5], [0, 77, 64, 0], D=D, words=2)
    rng = np.random.default_rng(1)
    b.masks = rng.integers(0, 1 << 32, (b.rows, 2))
    b.masks[::5] = 0
    b.masks[3::7] = BAD
    b.check()


def test_chain_equals_causal(ctx):
    """A chain of drafted tokens is a prompt's chunk: the two entries agree."""
    say("chain")
    new, have = [20, 1, 32], [100, 0, 31]
    a, b = Batch(ctx, 6, new, have), Batch(ctx, 6, new, have, words=1)
    b.masks = np.array(chain_masks(new, 1) + [[0]] * 3)
    b.check()
    assert np.abs(a.run() - b.run()).max() <= 1e-5


@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("D", [256, 512])
def test_unusual_batches(ctx, D, words):
    """Bad blocks, more rows than tokens, rows beyond the batch, starts that fall, lengths beyond the tables."""
    say("unusual", D, words)
    b = Batch(ctx, 7, [30, 20, 9, 12], [40, 60, 50, 8], D=D, words=words)
    b.tables[0, 1] = b.nb
    b.tables[1, :] = BAD
    b.tables[3, 0] = BAD
    b.check()
    b = Batch(ctx, 8, [30, 20, 9], [0, 3, 50], D=D, words=words)
    b.lens = np.array([7, 10, 2])
    b.check()
    b = Batch(ctx, 9, [10, 20, 9], [0, 3, 50], D=D, words=words, spare=0)
    b.rows -= 15                                                        # the second is cut, the third has no row
    b.q, b.old, b.parents = b.q[:b.rows], b.old[:b.rows], b.parents[:b.rows]
    b.masks = None if b.masks is None else b.masks[:b.rows]
    b.check()
    b = Batch(ctx, 10, [10, 20, 9], [5, 3, 50], D=D, words=words, width=3)
    b.check()                                                           # 48 tokens fit the third's table
    b = Batch(ctx, 11, [10, 20, 9], [5, 3, 50], D=D, words=words)
    b.row_start = np.array([4, 1, 1, 10])                               # 9 rows of the last request alone
    out, (want, _, _, _) = b.run(), b.want()
    assert np.abs(out - want)[1:10].max() <= 1e-4
    assert np.array_equal(out[:1], b.old[:1]) and np.array_equal(out[10:], b.old[10:])


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("D", [256, 512])
def test_unseen_slots_hold_anything(ctx, D, what):
    """Slots of no token, of later tokens, of tokens outside the window, of other requests' blocks."""
    say("unseen", D, what)
    b = Batch(ctx, 12, [30, 70, 4], [41, 0, 200], D=D, window=48)
    seen = np.zeros(len(b.kc), bool)
    for r in range(b.n):
        n, length = int(b.row_start[r + 1] - b.row_start[r]), int(b.lens[r])
        pos = np.arange(max(0, length - n + 1 - 48), length)
        seen[b.tables[r, pos // b.bs] * b.bs + pos % b.bs] = True
    b.kc[~seen] = what
    b.vc[~seen] = what
    b.check()


@pytest.mark.parametrize("words", [0, 2])
@pytest.mark.parametrize("which", ["k", "v", "kv", "q"])
@pytest.mark.parametrize("D", [256, 512])
def test_nonfinite_values_stay_where_they_are_seen(ctx, D, which, words):
    """Infinities and NaN in tokens that some rows of a tile see and others do not, in one KV head of two."""
    say("nonfinite", D, which, words)
    b = Batch(ctx, 13, [50, 40, 20], [20, 0, 90], D=D, words=words)
    rng = np.random.default_rng(2)
    for r, what in enumerate([np.nan, np.inf, -np.inf]):
        pos = int(b.lens[r]) - 7
        slot = b.tables[r, pos // b.bs] * b.bs + pos % b.bs
        for name in which if which != "q" else "":
            (b.kc if name == "k" else b.vc)[slot, int(rng.integers(0, D))] = what
        if which == "q":
            b.q[b.row_start[r] + 3, int(rng.integers(0, D))] = what
    if which == "q":
        # an infinite query component makes each score infinite, of either sign: its row is NaN or has the keys of the
        # other sign only, which the fp32 and the 64-bit definition share
        out, (want, _, _, _) = b.run(), b.want()
        assert np.array_equal(np.isnan(out), np.isnan(want))
        fine = np.isfinite(want)
        assert np.abs(out - want)[fine].max() <= 1e-4
    else:
        b.check()


@pytest.mark.parametrize("D", [256, 512])
def test_scores_and_values_of_any_size(ctx, D):
    """Rows of K and V from 2^-100 to 2^100, zeros, a row with one large component; equal scores."""
    say("any size", D)
    b = Batch(ctx, 14, [40, 9], [60, 200], D=D)
    rng = np.random.default_rng(3)
    b.kc *= 2.0 ** rng.integers(-100, 2, (len(b.kc), 1))
    b.kc[::9] = 0
    b.q[::11] = 0
    out, (want, _, _, L) = b.run(), b.want()
    assert np.abs(out - want).max() <= 1e-4
    b = Batch(ctx, 15, [40, 9], [60, 200], D=D)
    b.vc *= np.float32(2.0 ** 90)
    b.check()
    b = Batch(ctx, 16, [40, 9], [60, 200], D=D)
    b.vc *= (2.0 ** rng.integers(-60, 60, (len(b.vc), 1))).astype(np.float32)
    out, (want, _, _, L) = b.run(), b.want()
    # each value within the bound of the largest value of its own row's keys, which the weights may have made small
    assert (np.abs(out - want) <= (600 * U) * np.abs(b.vc).max()).all()
    b = Batch(ctx, 17, [40, 9], [60, 200], D=D, sigma=400.0)
    out, (want, big, absum, L) = b.run(), b.want()
    # scores of thousands: the weights follow their differences to 2 (D + 14) u sum|q k|
    bound = (2 * (D + 14) * U * absum + 2 * (L + 20) * U) * np.abs(b.vc).max()
    assert np.abs(out - want).max() <= bound


def test_small_values_beside_large_ones(ctx):
    """Columns of V 2^18 apart: the small ones keep 2^-17 of their own size at least."""
    say("columns")
    b = Batch(ctx, 18, [40], [60])
    b.vc[:, ::2] *= np.float32(2.0 ** 18)
    out, (want, _, _, L) = b.run(), b.want()
    small = np.abs(out - want)[:, 1::2]
    assert small.max() <= 2.0 ** -17 * np.abs(b.vc[:, 1::2]).max()


def test_long_rows_beside_a_nan_keep_their_digits(ctx):
    """Rows of a tile that meets a NaN are recomputed key by key: they stay as exact as the others."""
    say("long rows, NaN")
    b = Batch(ctx, 19, [2], [20000], nq=2, bs=64)
    b.q[1, 3] = np.nan                                                   # the second row alone
    out, (want, _, _, _) = b.run(), b.want()
    assert np.isnan(out[1, :256]).all() and np.isfinite(out[0]).all()
    assert np.linalg.norm(out[0] - want[0]) <= 4e-6 * np.linalg.norm(want[0])


@pytest.mark.parametrize("seed", range(16))
def test_random_batches(ctx, seed):
    """Batches of any shape: heads, groups, block sizes, windows, masks, empty and new requests, bad blocks."""
    rng = np.random.default_rng(1000 + seed)
    D, gqa, words = int(rng.choice([256, 512])), int(rng.integers(1, 17)), int(rng.choice([0, 0, 1, 2, 4]))
    n = int(np.exp(rng.uniform(0, np.log(20))))
    new = rng.integers(0, min(32 * words if words else 150, 900 // n) + 1, n)
    have = np.where(rng.random(n) < 0.3, 0, rng.integers(0, 900 // n + 2, n))
    window = int(rng.choice([0, 0, 128, int(rng.integers(128, 400))])) if words else int(rng.choice([0, 0, 1, 40, int(rng.integers(1, 400))]))
    shape = dict(D=D, gqa=gqa, nq=gqa * int(rng.integers(1, 3)), bs=int(2 ** rng.integers(0, 8)), words=words, window=window)
    say("random", seed, shape, new.tolist(), have.tolist())
    b = Batch(ctx, 2000 + seed, new, have, **shape)
    if seed % 4 == 3:
        b.tables[rng.random(b.tables.shape) < 0.1] = BAD
    b.check()


DRAFTS = [([1], 1), ([32, 0, 5], 1), ([33, 40], 1), ([64, 1, 2, 3], 2), ([100, 70, 65], 3), ([128], 4), ([256, 255, 31], 8),
          ([300, 600], 8), ([5] * 600, 1), ([0, 0], 2)]


@pytest.mark.parametrize("i", range(len(DRAFTS)))
@pytest.mark.parametrize("shape", ["random", "chain", "star"])
def test_draft_trees(ctx, i, shape):
    new, words = DRAFTS[i]
    say("drafts", new[:6], words, shape)
    rng = np.random.default_rng(i)
    n, start = len(new), np.concatenate([[0], np.cumsum(new)])
    rows = int(start[-1]) + 2
    parents = random_trees(rng, new)
    if shape == "chain":
        parents = [(j - 1) & BAD for k in new for j in range(k)]
    elif shape == "star":
        parents = [0 if j else int(rng.integers(0, 1 << 32)) for k in new for j in range(k)]
        parents = [p if k % 3 else BAD for k, p in enumerate(parents)]
    parents += [3, 3]
    lens = start[1:] - start[:-1] + rng.integers(0, 1 << 30, n)
    lens[::4] = 2                                                        # fewer tokens than rows
    old_m, old_c = np.full((rows, words), 21), np.full(rows, 22)
    bufs = [up32(ctx, a) for a in (parents, start, lens, old_m, old_c)]
    ctx.call("chn_draft_trees", bufs[0], bufs[1], bufs[2], n, rows, words, bufs[3], bufs[4])
    m, c = packed.draft_trees(parents, start, lens, rows, words, old_m, old_c)
    assert np.array_equal(down32(ctx, bufs[3], rows * words).reshape(rows, words), m)
    assert np.array_equal(down32(ctx, bufs[4], rows), c)


def test_large_offsets(ctx):
    """A cache above 4 GiB whose last block is used."""
    say("large offsets")
    D, bs, kv_dim, new, have = 256, 1024, 2048, 40, 100
    nb = (5 << 30) // (bs * kv_dim * 4)
    rng = np.random.default_rng(4)
    kc, vc = ctx.zeros(nb * bs * kv_dim * 4), ctx.zeros(nb * bs * kv_dim * 4)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    k, v, q = f(new + have, kv_dim), f(new + have, kv_dim), f(new, 16 * D) / 4
    for buf, a in ((kc, k), (vc, v)):
        ctx._check("chn_upload", ca.lib.chn_upload(ctx.handle, buf.offset((nb - 1) * bs * kv_dim * 4), a.ctypes.data, a.nbytes))
    out = ctx.zeros(q.nbytes)
    ctx.call("chn_paged_causal_attn", ctx.upload(q), kc, vc, up32(ctx, [nb - 1]), up32(ctx, [0, new]), up32(ctx, [new + have]), 1, new,
             1, bs, nb, 16, D, kv_dim, 2, 1.0, 0, out)
    want, _, _, _ = packed.packed_attn(q, k, v, [[0]], [0, new], [new + have], bs, 1, 16, D, 2, 1.0, 0)
    assert np.abs(ctx.download(out, np.float32, q.size).reshape(q.shape) - want).max() <= 1e-4
    kc.free()
    vc.free()
