"""One decode step of several requests, as they would be served: block tables,
RoPE + K/V write at their slots, attention over the shared prefix and their own
blocks, logits and sampling; run directly and as one recording replayed with
the program's own work between the replays, against the oracle step by step."""
import numpy as np
import pytest

import channel_amd as ca
import oracle
from gpu_util import say, synth_normal_dev
from oracle import paged

pytestmark = pytest.mark.gpu

N, D, NQ, NKV, BS, NPB, WIDTH, V, STEPS = 7, 256, 4, 2, 4, 3, 12, 2048, 6
P, H, NB = NPB * BS, NQ * D, 64
THETA, EPS = 1e4, 1e-6


class Step:
    """The device state of the batch and the calls of one step: x -> q, k, v -> attention -> logits -> token."""

    def __init__(self, ctx, seed):
        self.ctx, rng = ctx, np.random.default_rng(seed)
        self.prefix, self.free = rng.permutation(NB)[:NPB], None
        ids = np.setdiff1d(np.arange(NB), self.prefix)
        rng.shuffle(ids)
        self.free = ids
        up = lambda a: ctx.upload(np.asarray(a, np.int64).astype(np.uint32))  # noqa: E731
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.kc, self.vc = f(NB * BS, NKV * D), f(NB * BS, NKV * D)
        self.embed = f(V, (NQ + 2 * NKV) * D)                   # a token's raw q, k and v
        self.qw, self.kw = (0.2 * (1 + 0.1 * f(D))).astype(np.float32), 1 + 0.1 * f(D)
        self.Wq8 = ctx.alloc(ca.q8_bytes(V, H))
        ctx.call("chn_synth_q8", self.Wq8, V, H, seed, 0.002, 0.004)
        self.head = oracle.dequant_q8(ctx.download(self.Wq8, np.uint32, V * (H // 32) * 9), V, H)
        self.u = rng.random((STEPS, N)).astype(np.float32)
        self.T = np.array([1, 0.7, 0, 1, 1.2, 1, 0.9], np.float32)
        self.k = np.array([0, 50, 0, 1, 0, 300, 0], np.uint32)
        self.p = np.array([1, 0.9, 1, 1, 0.8, 0.95, 0.9], np.float32)
        self.lens = np.array([0, P + 3, P + 4, 0, P + 9, P, P + 1])
        self.table = np.full((N, WIDTH), 0xFFFFFFFF)
        t = 0
        for r in range(N):
            own = -(-max(self.lens[r] - P, 0) // BS)
            if self.lens[r]:
                self.table[r, :NPB] = self.prefix
                self.table[r, NPB:NPB + own] = self.free[t:t + own]
                t += own
        self.taken = t
        d = self.dev = {k: up(v) for k, v in dict(prefix=self.prefix, free=self.free, tables=self.table, n_new=[1] * N,
                                                  lens0=self.lens, st0=[0, t, 0], lens1=[0] * N, st1=[0] * 3,
                                                  row_start=[0] * (N + 1), slots=[0] * N, clocks=[0] * N, tokens=[0] * N,
                                                  k=self.k).items()}
        d.update(kc=ctx.upload(self.kc), vc=ctx.upload(self.vc), q=ctx.alloc(N * H * 4), kk=ctx.alloc(N * NKV * D * 4),
                 vv=ctx.alloc(N * NKV * D * 4), qr=ctx.alloc(N * H * 4), o=ctx.alloc(N * H * 4), lg=ctx.alloc(N * V * 4),
                 qw=ctx.upload(self.qw), kw=ctx.upload(self.kw), T=ctx.upload(self.T), p=ctx.upload(self.p),
                 u=ctx.alloc(N * 4), probs=ctx.alloc(N * 4))

    def calls(self, i):
        """Step i's calls; lengths and status alternate between two sets."""
        d, c = self.dev, self.ctx.call
        a, b = ("0", "1") if i % 2 == 0 else ("1", "0")
        c("chn_block_tables", d["lens" + a], d["n_new"], N, d["prefix"], NPB, d["free"], len(self.free),
          d["st" + a].offset(4), NB, BS, WIDTH, N, d["tables"], d["lens" + b], d["row_start"], d["slots"], d["clocks"],
          d["st" + b])
        c("chn_batch_qkv_rope_at", d["q"], d["kk"], d["vv"], d["qw"], d["kw"], d["qr"], d["kc"], d["vc"], d["clocks"],
          d["slots"], N, NB * BS, NQ, NKV, D, D, 0, THETA, EPS)
        c("chn_prefix_decode_attn", d["qr"], d["kc"], d["vc"], d["prefix"], NPB, d["tables"], d["lens" + b], N, WIDTH, BS, NB,
          NQ, D, NKV * D, NQ // NKV, 1.0, d["o"])
        for r in range(N):
            c("chn_gemv_q8", self.Wq8, d["o"].offset(r * H * 4), d["lg"].offset(r * V * 4), V, H)
        c("chn_sample", d["lg"], N, V, V, d["T"], d["k"], d["p"], None, d["u"], 30.0, d["tokens"], d["probs"])

    def put(self, name, a):
        self.ctx.upload(np.ascontiguousarray(a), self.dev[name])

    def feed(self, i, tokens):
        e = self.embed[tokens]
        self.put("q", e[:, :H])
        self.put("kk", e[:, H:H + NKV * D])
        self.put("vv", e[:, H + NKV * D:])
        self.put("u", self.u[i])

    def oracle_step(self, i, tokens, got_logits):
        """The step in 64 bits; the draw on the logits the device had."""
        w = paged.block_tables(self.lens, [1] * N, self.prefix, self.free, self.taken, NB, BS, N, self.table, self.lens,
                               [0] * (N + 1), [0] * N, [0] * N)
        self.table, self.lens, slots, clocks, self.taken = w[0], w[1], w[3], w[4], w[5][1]
        e = self.embed[tokens].astype(np.float64)
        q, kc, vc = paged.rope_at(e[:, :H].reshape(N, NQ, D), e[:, H:H + NKV * D].reshape(N, NKV, D),
                                  e[:, H + NKV * D:].reshape(N, NKV, D), self.qw, self.kw, self.kc, self.vc, clocks, slots,
                                  D, THETA, EPS)
        self.kc, self.vc = kc, vc
        o, _, _ = paged.prefix_attn(q.reshape(N, H), kc, vc, self.prefix, self.table, self.lens, BS, NB, NQ, D, NQ // NKV, 1.0)
        logits = o @ self.head.astype(np.float64).T
        # fp32 rows of at most 40 keys through a Q8 matvec on 22-bit activations: the framework's fp32 bar
        assert np.abs(got_logits - logits).max() <= 1e-3 * np.abs(logits).max()
        out = []
        for r in range(N):
            t, pr, margin = paged.sample_row(got_logits[r], float(self.T[r]), int(self.k[r]), float(self.p[r]), 0.0,
                                             float(self.u[i, r]), 30.0)
            assert margin > 2.0 ** -32
            out.append(t)
        return np.array(out)


def run(ctx, seed, recorded):
    s = Step(ctx, seed)
    recs = []
    if recorded:
        # one unrecorded call of the shapes on a batch of its own, so that the workspace has its size
        Step(ctx, seed + 1).calls(0)
        for i in range(2):
            ctx.record_begin()
            s.calls(i)
            recs.append(ctx.record_end())
    tokens, seen = np.arange(N) * 11 % V, []
    other = synth_normal_dev(ctx, 5000, 3)
    for i in range(STEPS):
        s.feed(i, tokens)
        if recorded:
            recs[i % 2].submit()
        else:
            s.calls(i)
        got = ctx.download(s.dev["tokens"], np.uint32, N).astype(np.int64)
        logits = ctx.download(s.dev["lg"], np.float32, N * V).reshape(N, V)
        want = s.oracle_step(i, tokens, logits)
        assert np.array_equal(got, want), (i, got, want)
        assert np.array_equal(ctx.download(s.dev["slots"], np.uint32, N) < NB * BS, np.ones(N, bool))
        # the program's own work between the steps: a norm, and a sampling call that shares the workspace
        ctx.call("chn_rmsnorm", other, other, s.dev["o"], 512, 1e-6)
        ctx.call("chn_sample", other, 2, 2500, 2500, None, None, None, None, s.dev["u"], 0.0, s.dev["row_start"], None)
        ctx.sync()
        seen.append(logits.copy())
        tokens = got
    for r in recs:
        r.free()
        ctx._recs.remove(r)
    return np.array(seen)


def test_step_against_the_oracle(ctx):
    say("serving step, direct")
    run(ctx, 40, False)


def test_recorded_step_equals_the_direct_one(ctx):
    say("serving step, recorded")
    a = run(ctx, 41, False)
    b = run(ctx, 41, True)
    assert np.array_equal(a, b)
