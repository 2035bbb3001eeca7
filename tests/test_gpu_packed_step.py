"""Steps in which requests take several tokens, as they would be served: packed
prompts (block tables, RoPE + K/V write, causal attention, logits, the prompts'
log probabilities), then drafted trees (masks and clocks, RoPE at those, tree
attention, each node's likeliest token), the accepted paths' K/V moved behind
the cached tokens, and a decode step over them; directly and recorded, against
the oracles in 64 bits."""
import numpy as np
import pytest

import channel_amd as ca
import oracle
from gpu_util import say, synth_normal_dev
from oracle import packed, paged

pytestmark = pytest.mark.gpu

D, NQ, NKV, BS, V, WIDTH, NB = 256, 4, 2, 4, 2048, 24, 80
H, KV = NQ * D, NKV * D
THETA, EPS = 1e4, 1e-6
NONE = 0xFFFFFFFF
PROMPTS, DRAFTS = [21, 1, 0, 38, 9], [7, 3, 0, 12, 5]
N, WORDS = len(PROMPTS), 1
ROWS = sum(PROMPTS) + 3                              # the batch has room for a few more


class Serving:
    def __init__(self, ctx, seed, window):
        self.ctx, self.window, rng = ctx, window, np.random.default_rng(seed)
        self.rng = rng
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        up = lambda a: ctx.upload(np.asarray(a, np.int64).astype(np.uint32))  # noqa: E731
        self.embed = f(V, H + 2 * KV)
        self.qw, self.kw = (0.2 * (1 + 0.1 * f(D))).astype(np.float32), 1 + 0.1 * f(D)
        self.kc, self.vc = f(NB * BS, KV), f(NB * BS, KV)
        self.free = rng.permutation(NB)
        self.table, self.lens, self.taken = np.full((N, WIDTH), NONE), np.zeros(N, np.int64), 0
        self.Wq8 = ctx.alloc(ca.q8_bytes(V, H))
        ctx.call("chn_synth_q8", self.Wq8, V, H, seed, 0.002, 0.004)
        self.head = oracle.dequant_q8(ctx.download(self.Wq8, np.uint32, V * (H // 32) * 9), V, H).astype(np.float64)
        self.dev = {k: up(v) for k, v in dict(
            lens=self.lens, n_new=[0] * N, free=self.free, tables=self.table, lens_out=[0] * N, row_start=[0] * (N + 1),
            slots=[0] * ROWS, clocks=[0] * ROWS, tree_clocks=[0] * ROWS, status=[0] * 3, taken=[0], parents=[NONE] * ROWS,
            masks=[0] * ROWS * WORDS, targets=[NONE] * ROWS, ids=[0] * ROWS, ranks=[0] * ROWS).items()}
        alloc = lambda n: ctx.alloc(n * 4)  # noqa: E731
        self.dev.update(q=alloc(ROWS * H), k=alloc(ROWS * KV), v=alloc(ROWS * KV), qr=alloc(ROWS * H), o=alloc(ROWS * H),
                        lg=alloc(ROWS * V), lp=alloc(ROWS), ent=alloc(ROWS), tops=alloc(ROWS), qw=ctx.upload(self.qw),
                        kw=ctx.upload(self.kw), kc=ctx.upload(self.kc), vc=ctx.upload(self.vc))

    def put(self, name, a):
        a = np.ascontiguousarray(a)
        self.ctx.upload(a if a.dtype == np.float32 else a.astype(np.int64).astype(np.uint32), self.dev[name])

    def feed(self, tokens, n_new, parents=None, targets=None):
        """A step's inputs: the rows' tokens, how many each request takes."""
        e = np.zeros((ROWS, H + 2 * KV), np.float32)
        e[:len(tokens)] = self.embed[tokens]
        self.put("q", e[:, :H])
        self.put("k", e[:, H:H + KV])
        self.put("v", e[:, H + KV:])
        self.put("lens", self.lens)
        self.put("n_new", n_new)
        self.put("taken", [self.taken])
        pad = lambda a: list(a) + [NONE] * (ROWS - len(a))  # noqa: E731
        self.put("parents", pad([] if parents is None else parents))
        self.put("targets", pad([] if targets is None else targets))

    def calls(self, tree, rows):
        d, c = self.dev, self.ctx.call
        # what a refused or shorter step leaves behind is no slot and the old length
        self.ctx.fill_u32(d["slots"], NONE, ROWS)
        c("chn_copy", d["lens_out"], d["lens"], N * 4)
        c("chn_block_tables", d["lens"], d["n_new"], N, None, 0, d["free"], NB, d["taken"], NB, BS, WIDTH, ROWS, d["tables"],
          d["lens_out"], d["row_start"], d["slots"], d["clocks"], d["status"])
        clocks = d["clocks"]
        if tree:
            c("chn_draft_trees", d["parents"], d["row_start"], d["lens_out"], N, ROWS, WORDS, d["masks"], d["tree_clocks"])
            clocks = d["tree_clocks"]
        c("chn_batch_qkv_rope_at", d["q"], d["k"], d["v"], d["qw"], d["kw"], d["qr"], d["kc"], d["vc"], clocks, d["slots"], ROWS,
          NB * BS, NQ, NKV, D, D, 0, THETA, EPS)
        shape = (N, ROWS, WIDTH, BS, NB, NQ, D, KV, NQ // NKV, 1.0, self.window, d["o"])
        first = (d["qr"], d["kc"], d["vc"], d["tables"], d["row_start"], d["lens_out"])
        if tree:
            c("chn_paged_tree_attn", *first, d["masks"], WORDS, *shape)
        else:
            c("chn_paged_causal_attn", *first, *shape)
        for r in range(rows):
            c("chn_gemv_q8", self.Wq8, d["o"].offset(r * H * 4), d["lg"].offset(r * V * 4), V, H)
        c("chn_token_logprobs", d["lg"], rows, V, V, d["targets"], None, 30.0, 1, d["lp"], d["ent"], d["ranks"], d["ids"], d["tops"])

    def outputs(self, rows):
        g, d = self.ctx.download, self.dev
        return [g(d["o"], np.float32, ROWS * H).reshape(ROWS, H)[:rows], g(d["lg"], np.float32, rows * V).reshape(rows, V),
                g(d["lp"], np.float32, rows), g(d["ent"], np.float32, rows), g(d["ranks"], np.uint32, rows).astype(np.int64),
                g(d["ids"], np.uint32, rows).astype(np.int64), g(d["kc"], np.float32, NB * BS * KV).reshape(-1, KV),
                g(d["slots"], np.uint32, ROWS).astype(np.int64)]

    def check(self, tokens, n_new, parents, targets, got):
        """The step in 64 bits; tables, lengths and caches go on from it."""
        rows = len(tokens)
        w = paged.block_tables(self.lens, n_new, [], self.free, self.taken, NB, BS, ROWS, self.table, self.lens, [0] * (N + 1),
                               [NONE] * ROWS, [0] * ROWS)
        self.table, self.lens, start, slots, clocks, self.taken = w[0], w[1], w[2], w[3], w[4], w[5][1]
        masks = None
        if parents is not None:
            masks, clocks = packed.draft_trees(parents, start, self.lens, ROWS, WORDS, np.zeros((ROWS, WORDS)), np.zeros(ROWS))
        e = self.embed[tokens].astype(np.float64)
        q, kc, vc = paged.rope_at(e[:, :H].reshape(rows, NQ, D), e[:, H:H + KV].reshape(rows, NKV, D), e[:, H + KV:].reshape(rows, NKV, D),
                                  self.qw, self.kw, self.kc, self.vc, clocks[:rows], slots[:rows], D, THETA, EPS)
        self.kc, self.vc = kc, vc
        o, _, _, _ = packed.packed_attn(q.reshape(rows, H), kc, vc, self.table, start, self.lens, BS, NB, NQ, D, NQ // NKV, 1.0,
                                        self.window, masks)
        logits = o @ self.head.T
        assert np.array_equal(got[7], slots)
        assert np.abs(got[6] - kc).max() <= 1e-4
        # the framework's fp32 bar: the attention through a Q8 matvec on 22-bit activations
        assert np.abs(got[0] - o).max() <= 1e-4 * np.abs(o).max()
        assert np.abs(got[1] - logits).max() <= 1e-3 * np.abs(logits).max()
        for r in range(rows):
            lp, ent, rank, ids, _ = packed.logprob_row(got[1][r], targets[r], 1.0, 30.0, 1)
            assert (abs(got[2][r] - lp) <= 1e-4 or got[2][r] == lp) and abs(got[3][r] - ent) <= 1e-4
            assert got[4][r] == rank and [got[5][r]] == ids

    def step(self, tokens, n_new, parents=None, targets=None, recorded=False):
        targets = [NONE] * len(tokens) if targets is None else targets
        self.feed(tokens, n_new, parents, targets)
        rows, tree = len(tokens), parents is not None
        before = self.dev["tables"], self.ctx.download(self.dev["tables"], np.uint32, N * WIDTH)
        self.calls(tree, rows)
        got = self.outputs(rows)
        if recorded:
            other = synth_normal_dev(self.ctx, 5000, 3)
            self.ctx.record_begin()
            self.calls(tree, rows)
            rec = self.ctx.record_end()
            for _ in range(3):
                # the program's own work between the replays, some of it in the same workspace
                self.ctx.call("chn_sample", other, 2, 2500, 2500, None, None, None, None, other, 0.0, self.dev["ids"], None)
                self.ctx.upload(before[1], before[0])
                self.ctx.fill_u32(self.dev["o"], 0, ROWS * H)
                self.ctx.sync()
                rec.submit()
                again = self.outputs(rows)
                assert all(np.array_equal(a, b) for a, b in zip(got, again))
            rec.free()
            self.ctx._recs.remove(rec)
        self.check(tokens, n_new, parents, targets, got)
        return got


def pos_slot(table, pos):
    return int(table[pos // BS]) * BS + pos % BS


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("window", [0, 32])
def test_prompts_drafts_and_decode(ctx, window, recorded):
    say("packed step", window, recorded)
    s = Serving(ctx, 70 + window, window)
    rng = s.rng
    prompt = rng.integers(0, V, sum(PROMPTS))
    ends = np.cumsum(PROMPTS)
    targets = np.append(prompt[1:], NONE)
    targets[ends[np.array(PROMPTS) > 0] - 1] = NONE                      # what follows a prompt is not known
    s.step(prompt, PROMPTS, targets=targets, recorded=recorded)

    drafts = rng.integers(0, V, sum(DRAFTS))
    parents = [NONE if i == 0 else int(rng.integers(max(i - 4, 0), i)) for n in DRAFTS for i in range(n)]
    parents[1] = NONE                                                    # two roots
    held, taken = s.lens.copy(), s.taken
    s.step(drafts, DRAFTS, parents=parents, targets=drafts, recorded=recorded)

    # the deepest node's path is accepted: its K/V behind the cached tokens, ancestors first
    at = 0
    for r, n in enumerate(DRAFTS):
        paths = []
        for i in range(n):
            path = [i]
            while parents[at + path[-1]] < path[-1]:
                path.append(parents[at + path[-1]])
            paths.append(path[::-1])
        path = max(paths, key=len) if paths else []
        for i, node in enumerate(path):
            to, src = pos_slot(s.table[r], held[r] + i), pos_slot(s.table[r], held[r] + node)
            if to != src:
                for name in ("kc", "vc"):
                    ctx.call("chn_copy", s.dev[name].offset(to * KV * 4), s.dev[name].offset(src * KV * 4), KV * 4)
            # what the token's K and V are at its position, from the definition
            e = s.embed[drafts[at + node]][None].astype(np.float64)
            _, s.kc, s.vc = paged.rope_at(e[:, :H].reshape(1, NQ, D), e[:, H:H + KV].reshape(1, NKV, D), e[:, H + KV:].reshape(1, NKV, D),
                                          s.qw, s.kw, s.kc, s.vc, [held[r] + i], [to], D, THETA, EPS)
        s.lens[r] = held[r] + len(path)
        at += n
    assert taken < s.taken and (s.lens[np.array(DRAFTS) > 0] > held[np.array(DRAFTS) > 0]).all()

    # blocks that the rejected tokens opened stay in the tables: hand the next step new ones only behind them
    last = s.step(rng.integers(0, V, N), [1] * N, targets=[5] * N)
    if not window:
        # the decode step's own attention over the same caches
        d = s.dev
        ctx.call("chn_prefix_decode_attn", d["qr"], d["kc"], d["vc"], None, 0, d["tables"], d["lens_out"], N, WIDTH, BS, NB, NQ, D, KV,
                 NQ // NKV, 1.0, d["o"])
        assert np.abs(ctx.download(d["o"], np.float32, N * H).reshape(N, H) - last[0]).max() <= 1e-5 * np.abs(last[0]).max()


def test_two_contexts_at_once(ctx):
    """Two contexts' streams run packed attention side by side, each in its own workspace."""
    say("two contexts")
    from test_gpu_packed import Batch
    with ca.Context(0) as other:
        a, b = Batch(ctx, 31, [70, 9, 130], [300, 0, 77]).up(), Batch(other, 32, [60, 40], [20, 900], D=512, words=2).up()
        for _ in range(4):
            a.call()
            b.call()
        a.check(a.got())
        b.check(b.got())


def test_one_workspace_serves_every_batch(ctx):
    """One call of any size is enough for recordings of all others of its head_dim."""
    say("workspace")
    from test_gpu_packed import Batch
    with ca.Context(0) as c:
        Batch(c, 33, [1], [0], D=512).run()
        Batch(c, 33, [1], [0]).run()
        batches = [Batch(c, 34, [200, 3], [50, 700]).up(), Batch(c, 35, [20, 30], [400, 7], words=1).up(),
                   Batch(c, 36, [90], [333], D=512).up()]
        recs = []
        for b in batches:
            c.record_begin()
            b.call()
            recs.append(c.record_end())
        for _ in range(2):
            for b, rec in zip(batches, recs):
                rec.submit()
            for b in batches:
                b.check(b.got())
