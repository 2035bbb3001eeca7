"""Shared-prefix attention where scores are infinite, NaN or far from one: what
the softmax of the definition gives, on every path of the kernels (few rows,
many rows of heads of 256 and of 512, a request's own keys).

A key whose score is -inf has the weight zero, so the row is the softmax over
the others; a NaN among a row's scores makes its output NaN; of finite scores
that lie further apart than the exponential reaches only the largest counts.
Tolerances as in test_gpu_paged.py: every value within (2 (D + 2) u max sum|q
k| + 2 (L + 8) u) max|v| of the 64-bit result, u = 2^-24, over the keys that
count."""
import numpy as np
import pytest

from gpu_util import say
from oracle import paged
from test_gpu_paged import U, up32

pytestmark = pytest.mark.gpu

BS = 16
# n, D, query heads, gqa, prefix blocks, own tokens: the paths of the kernels
PATHS = {
    "own": (3, 256, 4, 2, 0, 200),
    "own512": (3, 512, 8, 8, 0, 200),
    "few": (3, 256, 4, 2, 8, 40),
    "rows": (18, 256, 16, 4, 64, 20),
    "rows512": (9, 512, 8, 4, 12, 20),
}


class Attn:
    """Requests over random keys; change q, k and v, then run()."""

    def __init__(self, path, seed=0, short=False):
        self.n, self.D, self.nq, self.gqa, self.npb, own = PATHS[path]
        rng = np.random.default_rng(seed + 100 * self.n + self.D)
        n, D, npb = self.n, self.D, self.npb
        self.nkv = self.nq // self.gqa
        self.lens = npb * BS + rng.integers(own // 2, own + 1, n)
        if short and npb:                                        # some end inside the prefix
            self.lens[::3] = rng.integers(npb * BS // 2, npb * BS, len(self.lens[::3]))
        blocks = np.maximum(-(-self.lens // BS) - npb, 0)
        self.width = npb + int(blocks.max()) + 1
        self.nb = npb + int(blocks.sum()) + 2
        ids = rng.permutation(self.nb)
        self.prefix, self.tables = ids[:npb], np.full((n, self.width), 0xFFFFFFFF)
        at = npb
        for r in range(n):
            self.tables[r, npb:npb + blocks[r]] = ids[at:at + blocks[r]]
            at += blocks[r]
        self.k, self.v = (rng.standard_normal((self.nb * BS, self.nkv * D)).astype(np.float32) for _ in range(2))
        self.q = (rng.standard_normal((n, self.nq, D)) * 3 / np.sqrt(D)).astype(np.float32)

    def slots(self, r):
        return paged.request_slots(self.lens[r], self.prefix, self.tables[r], BS, self.nb)

    def run(self, ctx, scale=1.0):
        say(f"prefix_attn n={self.n} D={self.D} nq={self.nq} gqa={self.gqa} npb={self.npb} scale={scale}")
        out = ctx.upload(np.full(self.q.shape, 7, np.float32))
        bufs = [ctx.upload(self.q), ctx.upload(self.k), ctx.upload(self.v), up32(ctx, self.prefix if self.npb else [0]),
                up32(ctx, self.tables), up32(ctx, self.lens)]
        ctx.call("chn_prefix_decode_attn", *bufs[:4], self.npb, *bufs[4:], self.n, self.width, BS, self.nb, self.nq, self.D,
                 self.nkv * self.D, self.gqa, scale, out)
        got = ctx.download(out, np.float32, out.nbytes // 4).reshape(self.q.shape)
        for b in bufs + [out]:
            b.free()
        return got

    def check(self, got, scale, rows=None):
        """got against the definition over the keys of finite scores."""
        for r in range(self.n):
            at = self.slots(r)
            for h in range(self.nq):
                if rows is not None and not rows[r, h]:
                    continue
                c = slice(h // self.gqa * self.D, (h // self.gqa + 1) * self.D)
                k, v, q = (a.astype(np.float64) for a in (self.k[at, c], self.v[at, c], self.q[r, h]))
                with np.errstate(invalid="ignore"):
                    s = k @ q * scale
                live = np.isfinite(s)
                if not live.any():
                    assert not got[r, h].any()
                    continue
                k, v, s = k[live], v[live], s[live]
                p = np.exp(s - s.max())
                absum = (np.abs(k) @ np.abs(q)).max() * abs(scale)
                bound = (2 * (self.D + 2) * U * absum + 2 * (len(at) + 8) * U) * np.abs(v).max()
                assert np.abs(got[r, h] - p @ v / p.sum()).max() <= bound, (r, h)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("scale", [1.0, 0.0625, 0.1, 512 ** -0.5, -0.1, 0.3])
def test_scores_of_minus_infinity(ctx, path, scale):
    """Keys with an infinity on the side that a row's query takes down: no weight, for scales of any rounding."""
    a = Attn(path, short=True)
    a.q[..., 5] = np.abs(a.q[..., 5]) + 0.1
    rng = np.random.default_rng(3)
    hit = rng.random(len(a.k)) < 0.2
    for h in range(a.nkv):
        a.k[hit, h * a.D + 5] = -np.inf if scale > 0 else np.inf
    a.check(a.run(ctx, scale), scale)


@pytest.mark.parametrize("path", PATHS)
def test_every_score_minus_infinity(ctx, path):
    """No key with any weight: zeros, as a request without tokens."""
    a = Attn(path)
    a.q[..., 0] = 1.0
    a.k[:, ::a.D] = -np.inf
    assert not a.run(ctx).any()


# scores of the j-th key: a (j + 1), exactly apart: rounding cannot change their order, and the next one lies a below
@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("a_", [3e6, 1.37e8, 3.3e9, -7.7e9, 1.1e12, 2.9e20, -1.3e30, 1.7e35])
def test_scores_far_beyond_the_exponential(ctx, path, a_):
    """Finite scores of any size: the largest one's value, without overflow on the way."""
    a = Attn(path, short=True)
    a.q[:] = 0
    a.q[..., 3] = a_
    for r in range(a.n):
        at = a.slots(r)
        for h in range(a.nkv):
            a.k[at, h * a.D + 3] = np.arange(1, len(at) + 1)
    got = a.run(ctx)
    for r in range(a.n):
        at = a.slots(r)
        best = at[-1] if a_ > 0 else at[0]
        for h in range(a.nq):
            want = a.v[best, h // a.gqa * a.D:(h // a.gqa + 1) * a.D]
            assert np.abs(got[r, h] - want).max() <= 2 * (len(at) + 8) * U * np.abs(want).max(), (r, h)


@pytest.mark.parametrize("path", PATHS)
def test_nan_query(ctx, path):
    """A NaN in a head's query: that head's output is NaN, the others hold to the definition.  (Not bit for bit to a run
    without it: the references of a wave's rows move together, when one of them must.  Weights
    against another reference differ by a factor of the row, which the quotient takes out, and one rounding each, so both
    runs lie within the bound.)"""
    a = Attn(path, short=True)
    bad = np.zeros((a.n, a.nq), bool)
    bad[0, 1] = bad[a.n - 1, 0] = bad[1, a.nq - 1] = True
    a.q[bad, 7] = np.nan
    got = a.run(ctx)
    assert np.isnan(got[bad]).all()
    a.check(got, 1.0, ~bad)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("first,last", [(0, 1), (0, 16), (16, 32), (0, 64), (64, 128), (5, 90), (0, 100000)])
def test_nan_keys(ctx, path, first, last):
    """NaN among the keys at positions first .. last - 1, a group of 16, a part of the work or all: whoever sees one
    gets NaN, wherever the borders of the parts lie."""
    a = Attn(path, short=True)
    seen = np.zeros((a.n, a.nq), bool)
    for r in (range(a.n) if a.npb else (1,)):                   # the prefix is everybody's
        at = a.slots(r)[first:last]
        a.k[at, a.D - 1] = np.nan                               # KV head 0
        seen[r, :a.gqa] = len(at) > 0
    got = a.run(ctx)
    assert np.isnan(got[seen]).all()
    a.check(got, 1.0, ~seen)


@pytest.mark.parametrize("path", PATHS)
def test_infinite_score(ctx, path):
    """A score of +inf: inf - inf in the definition's softmax."""
    a = Attn(path)
    a.q[..., 0] = np.abs(a.q[..., 0]) + 0.1
    a.k[a.slots(0)[-1], 0] = np.inf
    got = a.run(ctx)
    assert np.isnan(got[0, :a.gqa]).all() and np.isfinite(got[0, a.gqa:]).all()
