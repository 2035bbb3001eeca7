"""Sampling on the GPU against the 64-bit oracle: the tokens equal, the
probabilities within 2^-22 (their weights are exact to 2^-43 of the largest,
the quotient is rounded to fp32 once).

The oracle tells how near a row's nearest other decision was (margin, relative
to the sum in question).  Weights are held to 2^-44 of the largest, so sums of
n of them to n 2^-44 of a sum that is at least one: decisions further than
2^20 2^-44 = 2^-24 apart cannot differ, nor, as roundings go both ways, those
further than 2^-32.  Rows nearer than that are not compared; at most one row
in a hundred may be."""
import numpy as np
import pytest

import channel_amd as ca
from gpu_util import say
from oracle import paged

pytestmark = pytest.mark.gpu

NEAR = 2.0 ** -32


def sample(ctx, logits, u, T=None, k=None, p=None, m=None, cap=0.0, V=None, probs=True, shift=0):
    logits = np.ascontiguousarray(logits, np.float32)
    n, ld = logits.shape
    V = V or ld
    up = lambda a, t: None if a is None else ctx.upload(np.broadcast_to(np.asarray(a, t), (n,)).copy())  # noqa: E731
    buf = ctx.alloc(logits.nbytes + 64)
    ctx._check("chn_upload", ca.lib.chn_upload(ctx.handle, buf.offset(shift), logits.ctypes.data, logits.nbytes))
    tok, prob = ctx.upload(np.full(n + 2, 77, np.uint32)), ctx.upload(np.full(n + 2, 77, np.float32))
    ctx.call("chn_sample", buf.offset(shift), n, V, ld, up(T, np.float32), up(k, np.uint32), up(p, np.float32),
             up(m, np.float32), up(u, np.float32), cap, tok, prob if probs else None)
    t, pr = ctx.download(tok, np.uint32, n + 2), ctx.download(prob, np.float32, n + 2)
    assert t[n:].tolist() == [77, 77] and pr[n:].tolist() == [77, 77]
    return t[:n].astype(np.int64), pr[:n]


def check(ctx, logits, u, T=1.0, k=0, p=1.0, m=0.0, cap=0.0, V=None, ties=0, **kw):
    logits = np.asarray(logits, np.float32)
    n = logits.shape[0]
    V = V or logits.shape[1]
    col = lambda a, t: np.broadcast_to(np.asarray(a, t), (n,)).copy()  # noqa: E731
    u, T, p, m, k = col(u, np.float32), col(T, np.float32), col(p, np.float32), col(m, np.float32), col(k, np.uint32)
    say(f"sample n={n} V={V} ld={logits.shape[1]} cap={cap} T={T[:3]} k={k[:3]} p={p[:3]} m={m[:3]}")
    tok, prob = sample(ctx, logits, u, T, k, p, m, cap, V, **kw)
    near = 0
    for r in range(n):
        want, wp, margin = paged.sample_row(logits[r, :V], float(T[r]), int(k[r]), float(p[r]), float(m[r]), float(u[r]), cap)
        if margin < NEAR:
            near += 1
            continue
        assert tok[r] == want, (r, int(tok[r]), want, margin)
        assert abs(prob[r] - wp) <= 2.0 ** -22 * wp, (r, prob[r], wp)
    assert near <= max(1, n // 100, ties), near
    return tok, prob


def rows(seed, n, V, sigma=2.5, peaks=20):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, V)) * sigma
    for r in range(n):
        at = rng.integers(0, V, peaks)
        x[r, at] += 3 + 6 * rng.random(peaks)
    return x.astype(np.float32), rng.random(n).astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 1025, 4095, 4096, 4097, 8193, 10007, 65537, 262144])
def test_plain_temperature(ctx, V):
    x, u = rows(V, 6, V)
    check(ctx, x, u, T=[0.3, 0.7, 1.0, 1.0, 1.7, 5.0])


@pytest.mark.parametrize("V", [5, 100, 5000, 32771, 262144])
@pytest.mark.parametrize("k", [1, 2, 63, 64, 65, 1000, 2048, 5000])
def test_top_k(ctx, V, k):
    x, u = rows(V + k, 5, V)
    check(ctx, x, u, T=[0.8, 1.0, 1.0, 1.2, 3.0], k=k)
    check(ctx, x, u[::-1].copy(), T=[0.8, 1.0, 1.0, 1.2, 3.0], k=k, p=[1.0, 0.95, 0.5, 0.9, 0.2], m=[0, 0, 0, 0.02, 0.1], cap=30.0)


@pytest.mark.parametrize("V", [7, 1000, 32771, 262144])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_top_p_and_min_p(ctx, V, cap):
    x, u = rows(V, 12, V)
    p = [0.01, 0.3, 0.5, 0.8, 0.9, 0.95, 0.99, 0.999, 1.0, 1.0, 0.9, 0.999999]
    m = [0, 0, 0, 0, 0, 0, 0, 0, 0.01, 0.3, 0.05, 1e-6]
    check(ctx, x, u, T=[1, 0.7, 1, 1, 1.3, 1, 1, 2.0, 1, 1, 1, 1], p=p, m=m, cap=cap)


def test_flat_rows(ctx):
    """All tokens equal: the order is the index's, the sums are whole numbers, borders fall on tokens exactly."""
    for V in (10, 1000, 5000, 262144):
        x = np.full((8, V), 1.25, np.float32)
        u = np.array([0, 0.5, 0.25, 0.999, 0.5, 0.75, 0.1, 0.9], np.float32)
        p = np.array([1, 1, 0.5, 0.5, 0.3, 1, 1, 0.7], np.float32)
        k = np.array([0, 0, 0, 0, 0, V // 2, 3, V - 1], np.uint32)
        say(f"flat V={V}")
        tok, prob = sample(ctx, x, u, None, k, p)
        for r in range(8):
            kept = V if k[r] == 0 else int(k[r])
            if p[r] < 1:                                        # ranks below p * kept
                kept = int(np.ceil(float(p[r]) * kept))
            assert tok[r] == int(np.floor(float(u[r]) * kept)), (V, r)
            assert abs(prob[r] * kept - 1) < 1e-6


def test_few_distinct_values(ctx):
    """Logits of a 16-bit head: thousands of tokens share the border's value."""
    for V in (5000, 262144):
        x, u = rows(V + 1, 10, V, sigma=1.0, peaks=3)
        x = (np.round(x * 4) / 4).astype(np.float32)
        check(ctx, x, u, T=1.0, p=[0.3, 0.5, 0.7, 0.9, 0.99, 1, 1, 1, 0.8, 0.9], k=[0, 0, 0, 0, 0, 50, 700, 3000, 100, 2000])


def test_barred_tokens(ctx):
    V = 3001
    x, u = rows(4, 9, V)
    rng = np.random.default_rng(9)
    barred = [-np.inf, np.nan, np.finfo(np.float32).min]
    for r in range(9):
        x[r, rng.random(V) < (0.1, 0.9, 0.999)[r // 3]] = barred[r % 3]
    x[8] = barred[2]
    x[8, 1234] = -1e30
    tok, _ = check(ctx, x, u, T=1.0, p=0.9, k=[0, 40, 0] * 3)
    assert tok[8] == 1234
    tok, _ = check(ctx, x, u, T=0.0, cap=30.0)
    assert all(np.isfinite(x[r, t]) for r, t in enumerate(tok))


@pytest.mark.parametrize("V", [1, 100, 5000, 262144])
def test_rows_that_bar_everything(ctx, V):
    x = np.zeros((4, V), np.float32)
    x[0], x[1], x[2] = -np.inf, np.nan, np.finfo(np.float32).min
    for kw in (dict(), dict(T=0.0), dict(k=3, p=0.5), dict(p=0.9, m=0.1, cap=30.0)):
        tok, prob = sample(ctx, x, np.full(4, 0.5), **kw)
        assert tok[:3].tolist() == [paged.NO_TOKEN] * 3 and prob[:3].tolist() == [0, 0, 0]
        assert tok[3] != paged.NO_TOKEN


def test_infinite_logits(ctx):
    x = np.zeros((3, 500), np.float32)
    x[:, 3], x[:, 77], x[:, 400] = np.inf, np.inf, np.inf
    tok, prob = sample(ctx, x, [0.1, 0.5, 0.9])
    assert tok.tolist() == [3, 77, 400] and np.allclose(prob, 1 / 3)
    tok, _ = sample(ctx, x, [0.1, 0.5, 0.9], k=2)
    assert tok.tolist() == [3, 77, 77]
    check(ctx, x, [0.1, 0.5, 0.9], cap=30.0)


def test_greedy_takes_the_lowest_of_equals(ctx):
    x, u = rows(1, 5, 9000)
    x[:, [8000, 4000, 4500]] = 50.0
    tok, prob = check(ctx, x, u, T=[0.0, -1.0, np.nan, 0.0, -0.0], k=5, p=0.3)
    assert (tok == 4000).all() and (prob == 1).all()
    x[:, :] = 0.0
    x[:, 5:] = -0.0                                            # equal to +0: index order
    tok, _ = sample(ctx, x, u, T=0.0)
    assert (tok == 0).all()
    tok, _ = sample(ctx, x, [0, 0.3, 0.5, 0.9, 0.99], k=10)
    assert tok.tolist() == [0, 3, 5, 8, 9]                     # 0.9 in fp32 lies below nine tenths


def test_odd_settings(ctx):
    """Settings out of range: documented meanings, no faults."""
    x, _ = rows(2, 8, 5000)
    nan, inf = np.nan, np.inf
    order = np.argsort(-x, axis=1, kind="stable")
    tok, _ = sample(ctx, x, [0.5] * 8, p=[0, -1, nan, 2, 1, 0, 0, 0], k=[0, 0, 1, 1, 1, 9, 0xFFFFFFFF, 5001])
    assert (tok == order[:, 0]).all()
    check(ctx, x, [0, -1, nan, 1, 7, inf, -inf, 0.5], k=6)
    check(ctx, x, 0.5, m=[nan, -1, 1, 7, inf, 0.5, 0, 1e-30])
    # at 1e30 and 3e38 every weight is exactly one, 4500 are kept, and half of that is a whole number: on a border
    check(ctx, x, 0.5, T=[1e-30, 1e-3, 1e30, 1e-40, 1e3, 0.01, 3e38, 1e-10], p=0.9, ties=2)
    tok, prob = sample(ctx, x, [0.5] * 8, T=inf)
    assert (tok == 2500).all() and np.allclose(prob, 1 / 5000)


def test_wide_ranges(ctx):
    """Weights over the whole range of the exponent, and logits of any size."""
    rng = np.random.default_rng(12)
    x = np.stack([rng.uniform(-60, 0, 30000), rng.uniform(-3e38, 3e38, 30000), rng.uniform(-1e-30, 1e-30, 30000),
                  -np.abs(rng.standard_cauchy(30000)) * 10, rng.uniform(-600, 600, 30000)]).astype(np.float32)
    for cap in (0.0, 30.0, 1e-3, 1e30):
        check(ctx, x, rng.random(5), T=1.0, cap=cap)
        check(ctx, x, rng.random(5), T=1.0, cap=cap, p=0.9, k=[0, 0, 500, 0, 100])


def test_padded_rows_and_alignment(ctx):
    """ld past V holds anything; rows may start at any 4-byte address."""
    for V, pad, shift in ((1000, 1, 0), (4099, 13, 4), (10007, 9, 8), (4096, 4, 12), (70001, 2, 4)):
        x, u = rows(V, 7, V + pad)
        x[:, V:] = 1e30
        check(ctx, x, u, T=0.9, p=0.9, k=[0, 0, 0, 50, 50, 1, 2000], V=V, shift=shift)


def test_defaults(ctx):
    x, u = rows(3, 6, 2000)
    a = sample(ctx, x, u)
    b = sample(ctx, x, u, T=1.0, k=0, p=1.0, m=0.0)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    c = sample(ctx, x, u, probs=False)
    assert np.array_equal(a[0], c[0]) and (c[1] == 77).all()


def test_largest_vocabulary(ctx):
    x, u = rows(6, 3, 1 << 20, sigma=1.0, peaks=0)
    check(ctx, x, u, T=[1.0, 0.7, 1.0], p=[1.0, 0.9, 0.95], k=[0, 0, 2000])


def test_many_rows(ctx):
    x, u = rows(7, 700, 1500)
    rng = np.random.default_rng(1)
    check(ctx, x, u, T=rng.choice([0, 0.7, 1, 1.5], 700), k=rng.choice([0, 1, 40, 64, 1400], 700),
          p=rng.choice([1, 0.5, 0.9, 0.95], 700), m=rng.choice([0, 0, 0.05], 700), cap=30.0)


def test_draws_follow_the_distribution(ctx):
    """4096 evenly spread u over one row draw every kept token in proportion, to one draw each way."""
    V, n = 600, 4096
    x, _ = rows(10, 1, V, sigma=1.0, peaks=4)
    u = (np.arange(n, dtype=np.float32) + 0.5) / n
    tok, _ = sample(ctx, np.repeat(x, n, 0), u, T=0.8, k=30, p=0.9)
    order = np.argsort(-x[0], kind="stable")[:30]
    w = np.exp((x[0, order].astype(np.float64) - x[0, order[0]]) / np.float32(0.8))
    keep = np.cumsum(w) - w < np.float32(0.9) * w.sum()
    order, w = order[keep], w[keep]
    for t, share in zip(order, w / w.sum()):
        assert abs((tok == t).sum() - share * n) <= 1.0 + 1e-6
    assert set(tok.tolist()) <= set(order.tolist())
