"""The batched step as the documentation composes it, where a step does not
place every row: the tables refuse it while the rest is already enqueued, or
it has fewer tokens than the fixed number of rows of a recorded step.  Rows
without a place write no K/V, and a refused step can be made again."""
import numpy as np
import pytest

from gpu_util import say
from oracle import paged
from test_gpu_paged import U, down32, up32

pytestmark = pytest.mark.gpu

D, NQ, NKV, BS, NPB, WIDTH, THETA, EPS = 256, 4, 2, 4, 3, 12, 1e4, 1e-6
P, H, KV, NB = NPB * BS, NQ * D, NKV * D, 80


class Batch:
    """n requests on the device with their state in 64 bits beside it; step() enqueues one step of max_tokens rows."""

    def __init__(self, ctx, lens, max_tokens, seed=0):
        self.ctx, self.n, self.rows = ctx, len(lens), max_tokens
        rng = self.rng = np.random.default_rng(seed)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        ids = rng.permutation(NB)
        self.prefix, self.free = ids[:NPB], ids[NPB:]
        self.lens, self.table, self.taken = np.asarray(lens, np.int64), np.full((self.n, WIDTH), 0xFFFFFFFF), 0
        for r, ln in enumerate(lens):
            if ln:
                own = -(-(ln - P) // BS)
                self.table[r, :NPB], self.table[r, NPB:NPB + own] = self.prefix, self.free[self.taken:self.taken + own]
                self.taken += own
        self.kc, self.vc = f(NB * BS, KV), f(NB * BS, KV)
        self.qw, self.kw = (0.2 * (1 + 0.1 * f(D))).astype(np.float32), 1 + 0.1 * f(D)
        u = lambda a: up32(ctx, a)  # noqa: E731
        self.dev = dict(prefix=u(self.prefix), free=u(self.free), tables=u(self.table), n_new=u([0] * self.n),
                        lens0=u(lens), st0=u([0, self.taken, 0]), lens1=u([0] * self.n), st1=u([0] * 3),
                        row_start=u([0] * (self.n + 1)), slots=u([0] * max_tokens), clocks=u([0] * max_tokens),
                        kc=ctx.upload(self.kc), vc=ctx.upload(self.vc), qw=ctx.upload(self.qw), kw=ctx.upload(self.kw),
                        q=ctx.zeros(max_tokens * H * 4), k=ctx.zeros(max_tokens * KV * 4), v=ctx.zeros(max_tokens * KV * 4),
                        qr=ctx.zeros(max_tokens * H * 4), qa=ctx.zeros(self.n * H * 4), o=ctx.zeros(self.n * H * 4))
        self.now = 0

    def feed(self, new):
        """The step's tokens: their rows of q, k and v."""
        self.new, f = np.asarray(new), lambda w: self.rng.standard_normal((self.rows, w)).astype(np.float32)
        self.q, self.k, self.v = f(H), f(KV), f(KV)
        self.ctx.upload(self.new.astype(np.uint32), self.dev["n_new"])
        for name in "qkv":
            self.ctx.upload(getattr(self, name), self.dev[name])

    def step(self, n_free=None, last_rows=None):
        """The documented calls.  last_rows: {request: row of its last new token}, where rows are not requests."""
        d, c = self.dev, self.ctx.call
        a, b = str(self.now), str(1 - self.now)
        c("chn_fill_u32", d["slots"], 0xFFFFFFFF, self.rows)
        c("chn_copy", d["lens" + b], d["lens" + a], 4 * self.n)
        c("chn_block_tables", d["lens" + a], d["n_new"], self.n, d["prefix"], NPB, d["free"],
          len(self.free) if n_free is None else n_free, d["st" + a].offset(4), NB, BS, WIDTH, self.rows, d["tables"],
          d["lens" + b], d["row_start"], d["slots"], d["clocks"], d["st" + b])
        c("chn_batch_qkv_rope_at", d["q"], d["k"], d["v"], d["qw"], d["kw"], d["qr"], d["kc"], d["vc"], d["clocks"],
          d["slots"], self.rows, NB * BS, NQ, NKV, D, D, 0, THETA, EPS)
        qa = d["qr"]
        if last_rows is not None:
            qa = d["qa"]
            for r, row in last_rows.items():
                c("chn_copy", qa.offset(r * H * 4), d["qr"].offset(row * H * 4), H * 4)
        c("chn_prefix_decode_attn", qa, d["kc"], d["vc"], d["prefix"], NPB, d["tables"], d["lens" + b], self.n, WIDTH, BS, NB,
          NQ, D, KV, NQ // NKV, 1.0, d["o"])

    def caches(self):
        return [self.ctx.download(self.dev[x], np.float32, NB * BS * KV).reshape(-1, KV) for x in ("kc", "vc")]

    def status(self):
        return down32(self.ctx, self.dev["st%d" % (1 - self.now)], 3).tolist()

    def lens_out(self):
        return down32(self.ctx, self.dev["lens%d" % (1 - self.now)], self.n)

    def verify(self):
        """The step that was enqueued, against the oracle; the batch moves on."""
        w = paged.block_tables(self.lens, self.new, self.prefix, self.free, self.taken, NB, BS, self.rows, self.table,
                               self.lens, [0] * (self.n + 1), [paged.NO_SLOT] * self.rows, [0] * self.rows)
        assert self.status() == w[5] and w[5][0] == 0
        self.table, self.lens, starts, slots, clocks, self.taken = w[0], w[1], w[2], w[3], w[4], w[5][1]
        assert np.array_equal(self.lens_out(), self.lens)
        assert np.array_equal(down32(self.ctx, self.dev["tables"], self.n * WIDTH), self.table.ravel())
        before = self.kc, self.vc
        q, self.kc, self.vc = paged.rope_at(self.q.reshape(-1, NQ, D), self.k.reshape(-1, NKV, D), self.v.reshape(-1, NKV, D),
                                            self.qw, self.kw, self.kc, self.vc, clocks, slots, D, THETA, EPS)
        hit = np.zeros(NB * BS, bool)
        hit[slots[slots < NB * BS]] = True
        for got, want, old in zip(self.caches(), (self.kc, self.vc), before):
            # RoPE rows: ((D + 4) / 2 + 16) u of the magnitudes a value is formed from, at most twice the largest
            assert np.array_equal(got[~hit], old[~hit].astype(np.float32))
            assert np.abs(got[hit] - want[hit]).max(initial=0) <= ((D + 4) / 2 + 16) * U * 2 * np.abs(want[hit]).max(initial=0)
            want[hit] = got[hit]                                 # a step's error stays the step's
        took = np.nonzero(self.new)[0]
        qa = np.zeros((self.n, H))
        qa[took] = q.reshape(-1, H)[starts[took + 1] - 1]
        want, big, absum = paged.prefix_attn(qa, self.kc, self.vc, self.prefix, self.table, self.lens, BS, NB, NQ, D, NQ // NKV,
                                             1.0)
        got = self.ctx.download(self.dev["o"], np.float32, self.n * H).reshape(self.n, H)
        # attention rows: (2 (D + 2) u sum|q k| + 2 (L + 8) u) max|v|, and the scores of a query that is off by
        # ((D + 4) / 2 + 16) u of its magnitude
        bound = U * ((2 * (D + 2) + (D + 4) + 32) * absum + 2 * (WIDTH * BS + 8)) * np.abs(self.vc).max()
        assert np.abs(got[took] - want[took]).max(initial=0) <= bound
        self.now = 1 - self.now


LENS = [0, P + 3, P + 4, 0, P + 9, P, P + 1]


def test_refused_step_leaves_the_caches(ctx):
    """Too few blocks, seen only after the whole step was enqueued: caches, tables and lengths are as they were, and the
    step made again with more blocks is the step."""
    say("serving step refused for want of blocks")
    b = Batch(ctx, LENS, len(LENS), 3)
    for _ in range(3):
        b.feed([1] * b.n)
        b.step()
        b.verify()
    b.feed([BS] * 2 + [0] * (b.n - 2))                          # eight rows where seven fit
    kc, vc = b.caches()
    b.step()
    assert b.status()[0] == 4 and all(np.array_equal(x, y) for x, y in zip(b.caches(), (kc, vc)))
    b.feed([1] * b.n)
    table = down32(ctx, b.dev["tables"], b.n * WIDTH)
    for n_free in (b.taken, 0):
        b.step(n_free)
        assert b.status()[0] == 1
        assert all(np.array_equal(x, y) for x, y in zip(b.caches(), (kc, vc)))
        assert np.array_equal(down32(ctx, b.dev["tables"], b.n * WIDTH), table)
        assert np.array_equal(b.lens_out(), b.lens)
        assert np.isfinite(ctx.download(b.dev["o"], np.float32, b.n * H)).all()
    b.step()
    b.verify()
    b.feed([1] * b.n)
    b.step()
    b.verify()


def test_refused_step_recorded(ctx):
    """The same of a recorded step: its replay is refused when its blocks run out, and writes nothing."""
    say("recorded serving step refused")
    b = Batch(ctx, LENS, len(LENS), 4)
    Batch(ctx, LENS, len(LENS), 5).step()                         # the workspace has its size
    recs = []
    for i in range(2):
        b.now = i
        ctx.record_begin()
        b.step(n_free=b.taken + 11)
        recs.append(ctx.record_end())
    b.now, refused = 0, False
    for i in range(8):
        b.feed([1] * b.n)
        kc, vc = b.caches()
        recs[b.now].submit()
        if b.status()[0]:
            refused = True
            assert b.status()[0] == 1 and all(np.array_equal(x, y) for x, y in zip(b.caches(), (kc, vc)))
            assert np.array_equal(b.lens_out(), b.lens)
            b.step()                                             # the same step, with the whole free list
        b.verify()
    assert refused
    for r in recs:
        r.free()
        ctx._recs.remove(r)


def last_rows(new):
    ends = np.cumsum(new)
    return {r: int(ends[r]) - 1 for r in range(len(new)) if new[r]}


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_requests_of_no_and_of_several_tokens(ctx, seed):
    """The tables pack rows by token, the attention takes a row per request: with each request's last row copied to its
    place, idle requests and admitted prompts leave the others' results what they are."""
    say("serving step with idle and growing requests")
    b = Batch(ctx, LENS, 24, 10 + seed)
    for new in ([0, 1, 1, 0, 0, 1, 1], [5, 0, 1, 3, 1, 1, 0], [1] * 7, [0] * 7, [0, 4, 0, 0, 0, 1, 6], [0, 0, 0, 0, 0, 0, 1]):
        b.feed(new)
        b.step(last_rows=last_rows(new))
        b.verify()


def test_idle_requests_behind_the_others_recorded(ctx):
    """A recorded step of fixed rows whose requests end one after another, those that go on kept in front: their rows are
    the requests', and the rows behind them write nothing."""
    say("recorded serving step with idle requests")
    b = Batch(ctx, LENS, len(LENS), 20)
    Batch(ctx, LENS, len(LENS), 21).step()                        # the workspace has its size
    recs = []
    for i in range(2):
        b.now = i
        ctx.record_begin()
        b.step()
        recs.append(ctx.record_end())
    b.now = 0
    for live in (7, 7, 5, 4, 4, 1, 0, 2):
        b.feed([1] * live + [0] * (b.n - live))
        recs[b.now].submit()
        b.verify()
    for r in recs:
        r.free()
        ctx._recs.remove(r)
