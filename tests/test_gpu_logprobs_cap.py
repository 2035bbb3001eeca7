"""Log probabilities of softcapped rows, against the 64-bit oracle, by bounds
that count what fp32 forms in fewer digits by its share of the row.

Tolerance (u = 2^-24; as in test_gpu_logprobs.py, but for the softcap): a
capped logit that is not the row's largest is off by 8 u cap at most.  With P
the probability of the tokens that equal the largest, which are one each, the
others are a share 1 - P of the sum, so log S is off by (1 - P) 8 u cap / T
besides 4 u H + u (4 + 2 log2 V).  The entropy has that twice, and in its
second sum the others' exponents, of mean size x, once more: (1 - P) 8 u cap / T
(2 + x).  Ranks and ids are equal."""
import numpy as np
import pytest

from gpu_util import say
from oracle import packed
from test_gpu_logprobs import U, model_rows, near, run

pytestmark = pytest.mark.gpu


def check_capped(ctx, logits, targets, T, cap, n_top=3):
    lp, ent, ranks, ids, tops = run(ctx, logits, targets, T, cap, n_top)
    V = logits.shape[1]
    for r in range(len(logits)):
        t = float(np.float32(T[r]))
        w = packed.logprob_row(logits[r], int(targets[r]), t, cap, n_top)
        row = np.sort(logits[r][logits[r] > packed.LOWEST].astype(np.float64))[::-1]
        c = cap * np.tanh(row / cap)
        x = (c - c[0]) / t
        x[row == row[0]] = 0
        p = np.exp(x)
        p /= p.sum()
        other = row != row[0]
        share = p[other].sum()
        mean = -(p[other] * x[other]).sum() / share if share else 0.0
        sums = 4 * U * w[1] + U * (4 + 2 * np.log2(V))
        bound = sums + 8 * U * cap / t * share
        say(f"  row {r} T {t:g}: log p {lp[r]:.7g} off {abs(lp[r] - w[0]):.2g} of {bound + 2 * U * abs(w[0]):.2g}, "
            f"entropy off {abs(ent[r] - w[1]):.2g}")
        assert near(lp[r], w[0], bound), (r, lp[r], w[0], bound)
        assert near(ent[r], w[1], 2 * sums + 8 * U * cap / t * share * (2 + mean)), (r, ent[r], w[1], bound)
        assert ranks[r] == w[2] and ids[r].tolist() == w[3]
        assert all(near(g, x, bound) for g, x in zip(tops[r], w[4])), (r, tops[r], w[4])


@pytest.mark.parametrize("T", [1.0, 0.01, 1e-5, 1e-7])
@pytest.mark.parametrize("V", [70, 5000, 70000])
@pytest.mark.parametrize("cap", [30.0, 5.0, 50.0])
def test_equal_largest_logits(ctx, cap, V, T):
    """One, two, three, some and all tokens share the largest logit, in one stretch of a row or in many."""
    say("equal largest", cap, V, T)
    rng = np.random.default_rng(1)
    rows, targets = [], []
    for top in (25.0, 3.3, 300.0, -7.0, 0.0):
        for ties in (1, 2, 3, 40, V):
            x = np.float32(top) - 2 - np.abs(rng.standard_normal(V) * 8).astype(np.float32)
            at = rng.permutation(V)[:ties]
            x[at] = top
            rows.append(x)
            targets.append(int(at[-1]) if len(rows) % 3 else int(rng.integers(0, V)))
    check_capped(ctx, np.array(rows, np.float32), targets, [T] * len(rows), cap)


@pytest.mark.parametrize("cap", [30.0, 5.0])
def test_sixteen_bit_logits(ctx, cap):
    """Rows of bfloat16's values, many of them equal, the largest ones among them."""
    say("16-bit", cap)
    x, rng = model_rows(21, 12, 20000)
    x = (x.view(np.uint32) & 0xFFFF0000).view(np.float32).copy()
    x[:, :3] = np.sort(x, 1)[:, -1:]
    T = [1, 0.7, 0.3, 0.1, 0.01, 1e-3, 1, 0.5, 2, 1e-4, 1e-6, 5]
    check_capped(ctx, x, rng.integers(0, 20000, 12), T, cap)


def test_a_dominant_token(ctx):
    """One token far above the rest: what is left to the softcap's rounding is the rest's share, far below 1e-7."""
    say("dominant")
    x, rng = model_rows(22, 8, 30000)
    at = rng.integers(0, 30000, 8)
    x[np.arange(8), at] = rng.uniform(27, 60, 8).astype(np.float32)
    check_capped(ctx, x, at, [1.0] * 8, 50.0)


@pytest.mark.parametrize("cap", [65.0, 100.0, 1e3, 1e4, 1e6, 1e15, 3e38])
def test_softcaps_far_above_the_logits(ctx, cap):
    """Softcaps that hardly bend the logits: with the capped logit off by 8 u of its own size, and not of the cap's, log S
    is off by 8 u max|l| / T and the rest of it as without a softcap."""
    say("large softcaps", cap)
    x, rng = model_rows(23, 6, 9000)
    x[3] *= 4
    x[4, ::7] = -np.inf
    x[5, ::5] = np.float32(-1e30)                                          # at the cap's other end
    T = [1, 0.5, 2, 1, 1, 1]
    targets = rng.integers(0, 9000, 6) // 7 * 7 + 1
    lp, ent, ranks, ids, tops = run(ctx, x, targets, T, cap, 5)
    for r in range(6):
        w = packed.logprob_row(x[r], int(targets[r]), T[r], cap, 5)
        size = np.abs(x[r][np.abs(x[r]) < 1e20]).max()
        bound = 4 * U * w[1] + U * (4 + 2 * np.log2(9000)) + 8 * U * size / T[r]
        say(f"  {abs(lp[r] - w[0]):.2g} {abs(ent[r] - w[1]):.2g} of {bound:.2g}")
        assert near(lp[r], w[0], bound) and near(ent[r], w[1], 2 * bound), (r, lp[r], w[:2], ent[r])
        assert ranks[r] == w[2] and ids[r].tolist() == w[3]
        assert all(near(g, v, bound) for g, v in zip(tops[r], w[4]))


@pytest.mark.parametrize("cap", [1e-45, 1e-40, 1e-30, 1e-3])
def test_softcaps_of_nothing(ctx, cap):
    """All logits capped to nothing beside the temperature, zeros among them: every token alike."""
    say("small softcaps", cap)
    x, rng = model_rows(24, 3, 5000)
    x[1, ::3] = 0
    x[2] = 0
    targets = rng.integers(0, 5000, 3)
    T = 1e3
    lp, ent, ranks, ids, _ = run(ctx, x, targets, [T] * 3, cap, 5)
    for r in range(3):
        w = packed.logprob_row(x[r], int(targets[r]), T, cap, 5)
        bound = 4 * U * w[1] + U * (4 + 2 * np.log2(5000)) + 8 * U * cap / T
        assert near(lp[r], w[0], bound) and near(ent[r], w[1], 2 * bound), (r, lp[r], w[:2])
        assert ranks[r] == w[2] and ids[r].tolist() == w[3]
