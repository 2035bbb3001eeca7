"""Log probabilities of given tokens, ranks, entropy and alternatives on the
GPU against the 64-bit oracle (oracle/packed.py).

Tolerances (u = 2^-24): x = (l - l_max) / T is off by three roundings of its
own size and, with a softcap, by 8 u cap / T (tanh from an exponential that is
off by a step, a quotient, products; what is returned of a single token is
formed in 64 bits and rounded once).  A weight's relative error is that of its
exponent, at most e = 3 u |x| + 8 u cap / T, and two steps of the exponential.
Under the weights |x| has a mean of at most the entropy H, and the sums add u
log2 V, so log S is off by 4 u H + 8 u cap / T + u (4 + 2 log2 V) at most.  The
entropy doubles it, and is rounded.  Ranks and ids are equal."""
import numpy as np
import pytest

import channel_amd as ca
from gpu_util import say
from oracle import packed
from test_gpu_paged import down32, up32

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NONE = 0xFFFFFFFF


def run(ctx, logits, targets, T=None, cap=0.0, n_top=0, V=None, optional=True):
    n, ld = logits.shape
    V = V or ld
    top = max(n_top, 1)
    f = lambda *s: ctx.upload(np.full(s, 7.0, np.float32))  # noqa: E731
    lp, ent, tops, ranks, ids = f(n), f(n), f(n, top), up32(ctx, [7] * n), up32(ctx, [[7] * top] * n)
    ins = [ctx.upload(logits), up32(ctx, targets), ctx.upload(np.asarray(T, np.float32)) if T is not None else None]
    ctx.call("chn_token_logprobs", ins[0], n, V, ld, ins[1], ins[2], cap, n_top, lp, ent if optional else None,
             ranks if optional else None, ids if n_top else None, tops if n_top else None)
    out = (ctx.download(lp, np.float32, n), ctx.download(ent, np.float32, n), down32(ctx, ranks, n),
           down32(ctx, ids, n * top).reshape(n, top), ctx.download(tops, np.float32, n * top).reshape(n, top))
    for b in [lp, ent, tops, ranks, ids] + [b for b in ins if b]:
        b.free()
        ctx._bufs.remove(b)
    return out


def near(got, want, bound):
    if not abs(want) < 2.0 ** 128 * (1 - 2.0 ** -25):        # rounds to an infinity in fp32 (half a step above its largest)
        return got == np.sign(want) * np.inf
    return abs(float(got) - want) <= bound + 2 * U * abs(want)


def check(ctx, logits, targets, T=None, cap=0.0, n_top=0, V=None):
    lp, ent, ranks, ids, tops = run(ctx, logits, targets, T, cap, n_top, V)
    V = V or logits.shape[1]
    for r in range(len(logits)):
        t = float(np.float32(T[r])) if T is not None else 1.0
        w = packed.logprob_row(logits[r, :V], int(targets[r]), t, cap, n_top)
        bound = 4 * U * w[1] + (8 * U * cap / t if t > 0 else 0) + U * (4 + 2 * np.log2(V))
        assert near(lp[r], w[0], bound), (r, lp[r], w[0], bound)
        assert near(ent[r], w[1], 2 * bound), (r, ent[r], w[1], bound)
        assert ranks[r] == w[2], (r, ranks[r], w[2])
        if n_top:
            assert ids[r].tolist() == w[3], (r, ids[r], w[3])
            assert all(near(g, x, bound) for g, x in zip(tops[r], w[4])), (r, tops[r], w[4])


def model_rows(seed, n, V, ld=None):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, ld or V)) * 2.5
    for r in range(n):
        at = rng.integers(0, V, 12)
        x[r, at] += rng.uniform(4, 10, 12)
    return x.astype(np.float32), rng


@pytest.mark.parametrize("V,pad", [(1, 0), (2, 1), (63, 0), (255, 3), (256, 0), (257, 0), (2047, 5), (2048, 0), (2049, 1),
                                   (10007, 9), (262144, 0), ((1 << 20) - 1, 1), (1 << 20, 0)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_sizes(ctx, V, pad, cap):
    say("logprobs", V, pad, cap)
    n = 5 if V < 100000 else 2
    x, rng = model_rows(V, n, V, V + pad)
    x[:, V:] = np.inf                                                    # what lies behind a row is not read
    targets = rng.integers(0, V, n)
    targets[0] = int(np.argmax(x[0, :V]))
    check(ctx, x, targets, None, cap, 5, V)
    check(ctx, x, targets, rng.uniform(0.3, 2, n), cap, 64, V)


@pytest.mark.parametrize("n_top", [0, 1, 2, 20, 63, 64])
def test_settings_per_row(ctx, n_top):
    say("settings", n_top)
    x, rng = model_rows(n_top, 12, 5000)
    T = [1, 0.0, -1, np.nan, 0.5, 1e-3, 3, 1e-38, 1, 1, 100, np.inf]
    targets = rng.integers(0, 5000, 12)
    targets[1] = np.argmax(x[1])
    targets[8], targets[9] = NONE, 5000
    check(ctx, x, targets, T, 0.0, n_top)
    check(ctx, x, targets, T[:11] + [1], 12.0, n_top)


def test_barred_tokens(ctx):
    """Rows under a grammar, rows that bar everything, fewer tokens than asked for, NaN, the lowest value."""
    say("barred")
    V = 3000
    x, rng = model_rows(3, 9, V)
    x[0, rng.random(V) < 0.9] = -np.inf
    x[1] = -np.inf
    x[2] = np.finfo(np.float32).min
    x[3, 7:] = np.nan
    x[4, :] = np.nan
    x[5, :2999] = -np.inf
    x[6, 100:200] = -np.inf
    targets = [int(np.argmax(x[0])), 5, 6, 3, 8, 2999, 150, NONE, 0]
    for T in (None, [1, 1, 1, 0.7, 1, 0, 0, 0, 0]):
        check(ctx, x, targets, T, 0.0, 20)
    check(ctx, x, targets, None, 30.0, 64)


def test_infinite_logits(ctx):
    say("infinite")
    x, _ = model_rows(4, 4, 4100)
    x[0, [3, 4000]] = np.inf
    x[1, 9] = np.inf
    x[2, :] = np.inf
    check(ctx, x, [4000, 5, 17, 3], None, 0.0, 5)
    check(ctx, x, [4000, 9, 17, 3], None, 30.0, 5)


@pytest.mark.parametrize("n_top", [1, 5, 64])
def test_equal_values_go_by_index(ctx, n_top):
    """Constant rows, a few distinct values, 16-bit values, the border of the alternatives inside equal ones."""
    say("equal", n_top)
    V = 20000
    x, rng = model_rows(5, 6, V)
    x[0] = 1.5
    x[1] = rng.integers(0, 3, V)
    x[2] = np.float32(np.float16(x[2]))
    x[3] = -0.0
    x[3, ::3] = 0.0
    x[4] = np.sort(x[4])[::-1]                                            # the largest lie in one block
    x[5] = np.sort(x[5])
    check(ctx, x, [777, 19999, int(np.argmax(x[2])), 4, 63, 19999], None, 0.0, n_top)
    check(ctx, x, [0, 1, 2, 3, 4, 5], [1, 0, 0, 0, 0.5, 0], 0.0, n_top)


def test_extreme_logits(ctx):
    """Values up to the type's largest: differences pass 2^127 and weights vanish."""
    say("extreme")
    x, _ = model_rows(6, 4, 2500)
    x[0] *= np.float32(1e37)
    x[1] = np.float32(-3e38)
    x[1, 40] = np.float32(3e38)
    x[2] *= np.float32(1e-40)
    x[3] *= np.float32(1e4)
    lp, ent, ranks, ids, _ = run(ctx, x, [5, 40, 6, 7], None, 0.0, 3)
    for r in range(4):
        w = packed.logprob_row(x[r], [5, 40, 6, 7][r], 1.0, 0.0, 3)
        assert ranks[r] == w[2] and ids[r].tolist() == w[3]
        assert near(lp[r], w[0], 1e-5) and near(ent[r], w[1], 1e-5), (r, lp[r], w[:2])


def test_optional_outputs_and_many_rows(ctx):
    """NULL entropy, ranks and alternatives; more rows than share the workspace."""
    say("many rows")
    x, rng = model_rows(7, 2100, 300)
    targets = rng.integers(0, 300, 2100)
    a = run(ctx, x, targets, None, 0.0, 3)
    b = run(ctx, x, targets, None, 0.0, 0, optional=False)
    assert np.array_equal(a[0], b[0]) and (b[1] == 7).all() and (b[2] == 7).all()
    for r in (0, 1023, 1024, 2047, 2048, 2099):
        w = packed.logprob_row(x[r], int(targets[r]), 1.0, 0.0, 3)
        assert ids_equal(a, r, w)


def ids_equal(got, r, w):
    return got[2][r] == w[2] and got[3][r].tolist() == w[3] and near(got[0][r], w[0], 1e-6)


def test_agrees_with_the_sampled_token(ctx):
    """What chn_sample draws at temperature 0 is the alternative of rank 0, and its probability is the one drawn with."""
    say("sampled")
    x, rng = model_rows(8, 6, 9000)
    u = rng.random(6).astype(np.float32)
    d = dict(x=ctx.upload(x), u=ctx.upload(u), tok=up32(ctx, [0] * 6), pr=ctx.zeros(24), lp=ctx.zeros(24))
    ctx.call("chn_sample", d["x"], 6, 9000, 9000, None, None, None, None, d["u"], 30.0, d["tok"], d["pr"])
    ctx.call("chn_token_logprobs", d["x"], 6, 9000, 9000, d["tok"], None, 30.0, 0, d["lp"], None, None, None, None)
    lp, pr = ctx.download(d["lp"], np.float32, 6), ctx.download(d["pr"], np.float32, 6)
    assert np.abs(np.exp(lp.astype(np.float64)) - pr).max() <= 1e-5
    tok = down32(ctx, d["tok"], 6)
    for r in range(6):
        assert near(lp[r], packed.logprob_row(x[r], int(tok[r]), 1.0, 30.0)[0], 1e-5)


def test_is_recorded(ctx):
    """A recording replayed with other logits and the program's own work between: equal to a call."""
    say("recorded")
    with ca.Context(0) as c:
        V = 30000
        rows = [model_rows(s, 3, V)[0] for s in (9, 10, 11)]
        t = up32(c, [5, 6, 7])
        buf, lp, ids, tops = c.alloc(3 * V * 4), c.zeros(12), up32(c, [0] * 15), c.zeros(60)
        args = ("chn_token_logprobs", buf, 3, V, V, t, None, 0.0, 5, lp, None, None, ids, tops)
        c.upload(rows[0], buf)
        c.call(*args)
        c.record_begin()
        c.call(*args)
        rec = c.record_end()
        for x in rows + rows[:1]:
            c.upload(x, buf)
            rec.submit()
            got = c.download(lp, np.float32, 3), down32(c, ids, 15), c.download(tops, np.float32, 15)
            c.fill_u32(ids, 0, 15)
            c.call(*args)
            again = c.download(lp, np.float32, 3), down32(c, ids, 15), c.download(tops, np.float32, 15)
            assert all(np.array_equal(a, b) for a, b in zip(got, again))
            for r in range(3):
                assert again[1][5 * r:5 * r + 5].tolist() == packed.logprob_row(x[r], 0, n_top=5)[3]
