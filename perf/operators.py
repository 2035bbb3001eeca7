"""Performance cases of the batched decode step over a paged KV cache.

One step of several requests calls four operators, each a "kind" here:

  tables   block tables and slot maps from the requests' lengths
           (chn_block_tables): blocks of the free list for the new tokens,
           and the slot and clock of each of them
  rope     q/k norm + RoPE + K/V write of tokens at clocks and slots of
           their own (chn_batch_qkv_rope_at)
  attn     attention of one token per request over a prefix that all
           requests share and over each request's own blocks
           (chn_prefix_decode_attn)
  sample   the next token of every row of logits by temperature, top-k,
           top-p and min-p from given random numbers (chn_sample)

Where `own` is false, run() computes them in their plain form.  Sizes: the
12B-class model of bench.py (16 query / 8 KV heads of 256, vocabulary
262144), heads of 512, the ring's 4096 and 3968 slots, and generic ones.
Unsigned 32-bit values are held in int32 tensors: -1 is "no slot", "no
token" and, in a table, "no block".
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e6
LOWEST = torch.finfo(torch.float32).min


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a decode step of 32 conversations with one system prompt: every request gains one token, a few a block
        dict(name="tables_decode_32", kind="tables", n=32, tokens=32, fresh=0, have=700, prefix=512, bs=16),
        # a step that admits prompts: a thousand requests, some new, most decoding, 131072 new tokens in all
        dict(name="tables_admit_1024", kind="tables", n=1024, tokens=131072, fresh=300, have=4000, prefix=1024, bs=32),
        # a decode step of 24 requests of the 12B model
        dict(name="rope_decode_24", kind="rope", n=24, D=256, nq=16, nkv=8, rot=256, far=5000, kv=0),
        # prompts of several requests together, 512-wide heads whose V is the raw K, far positions
        dict(name="rope_prompts_1500", kind="rope", n=1500, D=512, nq=16, nkv=4, rot=512, far=120000, kv=1),
        # eight answers to one question, some way in
        dict(name="attn_best_of_8", kind="attn", n=8, D=256, nq=16, nkv=8, prefix=512, own=96, bs=16),
        # 64 conversations with one long system prompt that fills a ring's window
        dict(name="attn_shared_64", kind="attn", n=64, D=256, nq=16, nkv=8, prefix=3968, own=480, bs=16),
        # 512-wide heads, an odd number of requests, a ragged prefix
        dict(name="attn_d512_33", kind="attn", n=33, D=512, nq=16, nkv=4, prefix=1488, own=333, bs=16),
        # long documents of their own: no common prefix at all
        dict(name="attn_own_12", kind="attn", n=12, D=256, nq=16, nkv=8, prefix=0, own=20000, bs=64),
        # one user: the 12B vocabulary, top-k 64 and top-p 0.95
        dict(name="sample_one", kind="sample", n=1, V=262144, pad=0, mix="chat"),
        # 32 users with settings of their own, softcapped logits
        dict(name="sample_users_32", kind="sample", n=32, V=262144, pad=0, mix="users"),
        # 128 answers drawn by top-p or min-p alone, over the whole vocabulary
        dict(name="sample_nucleus_128", kind="sample", n=128, V=262144, pad=0, mix="nucleus"),
        # a smaller model's odd vocabulary in padded rows
        dict(name="sample_odd_50", kind="sample", n=50, V=10007, pad=9, mix="users"),
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer between lo and hi, even over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["tables", "rope", "attn", "attn", "sample", "sample"])
    if kind == "tables":
        n, bs = _log_int(rng, 1, 1024), rng.choice([1, 8, 16, 32, 64, 128])
        return dict(kind=kind, n=n, tokens=n * _log_int(rng, 1, 128), fresh=rng.choice([0, rng.randint((n + 3) // 4, n)]),
                    have=_log_int(rng, 1, 4096), prefix=bs * rng.randint(0, 1024 // bs), bs=bs)
    if kind == "rope":
        D, nkv = rng.choice([256, 256, 512]), rng.choice([1, 2, 4, 8])
        return dict(kind=kind, n=_log_int(rng, 1, 1024), D=D, nq=nkv * rng.choice([1, 2, 4]), nkv=nkv,
                    rot=rng.choice([D, D, D // 2]), far=_log_int(rng, 1, 200000), kv=rng.randint(0, 1))
    if kind == "attn":
        D, nkv, bs = rng.choice([256, 256, 512]), rng.choice([1, 2, 4, 8]), rng.choice([8, 16, 16, 32, 64])
        n, own_most = _log_int(rng, 1, 64), _log_int(rng, 1, 8192)
        prefix = bs * rng.choice([0, rng.randint(1, 3968 // bs), rng.randint(1, 3968 // bs)])
        # at most the work of attn_shared_64
        while n > 1 and n * (prefix + own_most) * nkv * D > 64 * 4448 * 8 * 256:
            n -= 1
        return dict(kind=kind, n=n, D=D, nq=nkv * rng.choice([1, 2, 4]), nkv=nkv, prefix=prefix, own=own_most, bs=bs)
    n, V = _log_int(rng, 1, 128), _log_int(rng, 1000, 262144)
    return dict(kind=kind, n=n, V=V, pad=rng.choice([0, 0, rng.randint(1, 64)]),
                mix=rng.choice(["chat", "users", "nucleus"]))


def work(case):
    n = case["n"]
    if case["kind"] == "tables":
        blocks = case["tokens"] / case["bs"] + case["fresh"] * case["prefix"] / case["bs"]
        return {"bytes": n * 16 + blocks * 8 + case["tokens"] * 8, "flops": 0}
    if case["kind"] == "rope":
        rows = n * (case["nq"] + 2 * case["nkv"])
        read = n * (case["nq"] + (1 if case["kv"] else 2) * case["nkv"])
        return {"bytes": (rows + read) * case["D"] * 4 + n * 8, "flops": 8.0 * rows * case["D"]}
    if case["kind"] == "attn":
        mean = (case["own"] + 2) / 3                          # of the lengths that prepare() draws
        keys = case["prefix"] + n * mean
        return {"bytes": keys * case["nkv"] * case["D"] * 8 + 2 * n * case["nq"] * case["D"] * 4,
                "flops": 4.0 * n * (case["prefix"] + mean) * case["nq"] * case["D"]}
    return {"bytes": n * (case["V"] * 4 + 28), "flops": 4.0 * n * case["V"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int64).astype(np.uint32).view(np.int32), device="cuda")


def _lengths(rng, n, most):
    """n lengths from 1 to about `most`, short ones more often; their mean is (most + 2) / 3."""
    return 1 + np.floor(rng.random(n) ** 2 * most).astype(np.int64)


def _table_width(case):
    """Blocks that the longest request can need: a taker of new tokens gets at most three times the mean."""
    takers = case["fresh"] or case["n"]
    return -(-(case["prefix"] + case["have"] + 3 * (case["tokens"] // takers) + 4) // case["bs"]) + 1


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    s = {"case": dict(case)}
    n = case["n"]
    if case["kind"] == "tables":
        bs, npb = case["bs"], case["prefix"] // case["bs"]
        # every request gains a token; the rest are dealt to the new ones (or to all)
        fresh = np.zeros(n, bool)
        fresh[rng.permutation(n)[:case["fresh"]]] = True
        new = np.ones(n, np.int64)
        takers = np.nonzero(fresh)[0] if fresh.any() else np.arange(n)
        share = rng.random(len(takers)) + 0.5
        more = np.floor(share / share.sum() * (case["tokens"] - n)).astype(np.int64)
        more[:case["tokens"] - n - more.sum()] += 1
        new[takers] += more
        lens = np.where(fresh, 0, npb * bs + _lengths(rng, n, case["have"]))
        begin = np.maximum(lens, npb * bs)
        held = -(-lens // bs)
        need = -(-(begin + new) // bs) - -(-begin // bs)
        width = _table_width(case)
        pool = rng.permutation(npb + int(held.sum() + need.sum()) + 64)      # blocks in any order
        prefix, free = pool[:npb], pool[npb + int(held.sum()):]
        tables = np.full((n, width), -1, np.int64)
        at = npb
        for r in np.nonzero(~fresh)[0]:
            tables[r, :npb] = prefix
            tables[r, npb:held[r]] = pool[at:at + held[r] - npb]
            at += held[r] - npb
        s.update(lens=_i32(lens), n_new=_i32(new), prefix=_i32(prefix), free=_i32(free), taken=_i32([0]),
                 n_blocks=len(pool), max_blocks=width, max_tokens=case["tokens"] + 100, tables=_i32(tables),
                 lens_out=_i32([0] * n), row_start=_i32([0] * (n + 1)), slots=_i32([-1] * (case["tokens"] + 100)),
                 clocks=_i32([-1] * (case["tokens"] + 100)), status=_i32([0] * 3))
    elif case["kind"] == "rope":
        D, nq, nkv = case["D"], case["nq"], case["nkv"]
        n_slots = n + 64
        s.update(q=normal(n, nq * D), k=normal(n, nkv * D), v=normal(n, nkv * D), qw=1 + 0.1 * normal(D),
                 kw=1 + 0.1 * normal(D), clocks=_i32(rng.integers(0, case["far"], n)),
                 slots=_i32(rng.permutation(n_slots)[:n]), n_slots=n_slots, kc=normal(n_slots, nkv * D),
                 vc=normal(n_slots, nkv * D), q_out=torch.zeros((n, nq * D), device="cuda"))
    elif case["kind"] == "attn":
        D, nq, nkv, bs, npb = case["D"], case["nq"], case["nkv"], case["bs"], case["prefix"] // case["bs"]
        mine = _lengths(rng, n, case["own"])
        blocks = -(-mine // bs)
        width = npb + -(-(case["own"] + 1) // bs)
        pool = rng.permutation(npb + int(blocks.sum()) + 16)
        tables = np.full((n, width), -1, np.int64)
        tables[:, :npb] = pool[:npb]
        at = npb
        for r in range(n):
            tables[r, npb:npb + blocks[r]] = pool[at:at + blocks[r]]
            at += blocks[r]
        # keys leave the q/k norm with a mean square of one; the scores' deviation is about 4, their scale 1 as the
        # model's is
        s.update(q=normal(n, nq * D) * (4 / math.sqrt(D)), kc=normal(len(pool) * bs, nkv * D),
                 vc=normal(len(pool) * bs, nkv * D), prefix=_i32(pool[:npb]), tables=_i32(tables),
                 lens=_i32(npb * bs + mine), max_blocks=width, n_blocks=len(pool),
                 out=torch.zeros((n, nq * D), device="cuda"))
    else:
        V, ld, mix = case["V"], case["V"] + case["pad"], case["mix"]
        logits = normal(n, ld) * 2.5
        # a few likely tokens per row, as a model's logits have
        at = torch.randint(0, V, (n, 40), generator=gen, device="cuda")
        logits.scatter_add_(1, at, 4 + 6 * torch.rand((n, 40), generator=gen, device="cuda"))
        rows = torch.arange(n, device="cuda")
        if mix == "users":
            # some rows come from a 16-bit head (many equal values), some under a grammar (most tokens barred), and a
            # row in 25 belongs to nobody (all barred)
            coarse = logits.bfloat16().float()
            logits = torch.where((rows % 3 == 1)[:, None], coarse, logits)
            barred = torch.rand((n, ld), generator=gen, device="cuda") < 0.9
            logits = torch.where((rows % 5 == 2)[:, None] & barred, torch.full_like(logits, -math.inf), logits)
            logits = torch.where((rows % 25 == 23)[:, None], torch.full_like(logits, -math.inf), logits)
        pick = lambda values: np.asarray(values)[rng.integers(0, len(values), n)]  # noqa: E731
        if mix == "chat":
            T, k, p, m = [1.0] * n, [64] * n, [0.95] * n, [0.0] * n
        elif mix == "users":
            T, k = pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3]), pick([0, 1, 20, 40, 64, 64, 200])
            p, m = pick([1.0, 0.8, 0.9, 0.95, 0.95]), pick([0.0, 0.0, 0.05, 0.1])
        else:
            T, k, p, m = pick([0.7, 0.9, 1.0, 1.2]), [0] * n, pick([1.0, 0.9, 0.95, 0.99]), pick([0.0, 0.0, 0.02])
        f32 = lambda x: torch.as_tensor(np.asarray(x, np.float32), device="cuda")  # noqa: E731
        s.update(logits=logits.contiguous(), T=f32(T), k=_i32(k), p=f32(p), m=f32(m),
                 u=torch.rand(n, generator=gen, device="cuda"), cap=30.0 if mix == "users" else 0.0,
                 tokens=_i32([0] * n), probs=torch.zeros(n, device="cuda"))
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_tables(s):
    bs, npb = s["case"]["bs"], s["prefix"].numel()
    lens, new = s["lens"].long(), s["n_new"].long()
    begin = torch.where(new > 0, lens.clamp(min=npb * bs), lens)
    first, last = (begin + bs - 1) // bs, (begin + new + bs - 1) // bs
    need = last - first
    blocks, total = need.sum(), new.sum()
    taken = s["taken"].long()[0]
    flags = ((taken + blocks > s["free"].numel()) * 1 + (last.max() > s["max_blocks"]) * 2
             + (total > s["max_tokens"]) * 4)
    ok = flags == 0
    col = torch.arange(s["max_blocks"], device="cuda")
    at = taken + (need.cumsum(0) - need)[:, None] + col - first[:, None]
    grown = (col >= first[:, None]) & (col < last[:, None])
    tables = torch.where(grown, s["free"].long()[at.clamp(0, s["free"].numel() - 1)], s["tables"].long())
    if npb:
        head = (col < npb) & ((new > 0) & (lens < npb * bs))[:, None]
        tables = torch.where(head, s["prefix"].long()[col.clamp(max=npb - 1)], tables)
    ends = new.cumsum(0)
    t = torch.arange(s["max_tokens"], device="cuda")
    req = torch.searchsorted(ends, t, right=True).clamp(max=lens.numel() - 1)
    pos = begin[req] + t - (ends - new)[req]
    block = tables[req, (pos // bs).clamp(0, s["max_blocks"] - 1)]
    slot = torch.where((block >= 0) & (block < s["n_blocks"]), block * bs + pos % bs, -1)
    there = ok & (t < total)
    keep = lambda cond, new_, old: torch.where(cond, new_, old.long()).int()  # noqa: E731
    return [keep(ok, tables, s["tables"]), keep(ok, begin + new, s["lens_out"]),
            keep(ok, torch.cat([ends.new_zeros(1), ends]), s["row_start"]), keep(there, slot, s["slots"]),
            keep(there, pos, s["clocks"]), torch.stack([flags, taken + blocks, total]).int()]


def _plain_norm(x):
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()


def _plain_rotate(x, clocks, rot):
    """Pairs (d, d + rot / 2) of [tokens][heads][D]; the angles in 64 bits."""
    d = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    angle = clocks.double()[:, None, None] * THETA ** (-2 * d / rot)
    c, sn = angle.cos().float(), angle.sin().float()
    a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
    return torch.cat([a * c - b * sn, a * sn + b * c, rest], -1)


def _plain_rope(s):
    c = s["case"]
    D, nq, nkv, n = c["D"], c["nq"], c["nkv"], c["n"]
    q, k, v = s["q"].view(n, nq, D), s["k"].view(n, nkv, D), s["v"].view(n, nkv, D)
    v = k if c["kv"] else v
    at = s["slots"].long()
    kc, vc = s["kc"].clone(), s["vc"].clone()
    kc[at] = _plain_rotate(_plain_norm(k) * s["kw"], s["clocks"], c["rot"]).flatten(1)
    vc[at] = _plain_norm(v).flatten(1)
    return [_plain_rotate(_plain_norm(q) * s["qw"], s["clocks"], c["rot"]).flatten(1), kc, vc]


def _plain_attn(s):
    c = s["case"]
    D, nq, nkv, n, bs = c["D"], c["nq"], c["nkv"], c["n"], c["bs"]
    pos = torch.arange(c["prefix"] + c["own"], device="cuda")
    block = s["tables"].long()[:, pos // bs]
    seen = (pos < s["lens"].long()[:, None]) & (block >= 0) & (block < s["n_blocks"])
    slot = torch.where(seen, block * bs + pos % bs, 0)
    k = s["kc"][slot].view(n, -1, nkv, D).permute(0, 2, 3, 1).contiguous()
    v = torch.where(seen[:, :, None], s["vc"][slot], 0.0).view(n, -1, nkv, D).permute(0, 2, 1, 3).contiguous()
    score = s["q"].view(n, nkv, nq // nkv, D) @ k
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    return [torch.where(total > 0, p @ v / total, 0.0).reshape(n, nq * D)]


def _plain_sample(s):
    V, cap = s["case"]["V"], s["cap"]
    raw = s["logits"][:, :V]
    raw = torch.where(raw > LOWEST, raw, -math.inf)                       # barred: NaN, -inf and the lowest value
    raw, order = raw.sort(dim=1, descending=True, stable=True)               # equal values: the lower index first
    barred = raw == -math.inf
    x = raw.double()
    x = cap * (x / cap).tanh() if cap else x
    T, p, m = s["T"].double()[:, None], s["p"].double()[:, None], s["m"].double()[:, None]
    greedy = ~(T > 0)
    x = torch.where(x == x[:, :1], 0.0, (x - x[:, :1]) / torch.where(greedy, 1.0, T))
    w = torch.where(barred, 0.0, x.exp())
    rank = torch.arange(V, device="cuda")
    k = s["k"].long()[:, None]
    w = torch.where((k == 0) | (rank < k), w, 0.0)
    before = w.cumsum(1) - w
    kept = ~(p < 1) | (before < p * w.sum(1, keepdim=True))
    kept &= ~(m > 0) | (w >= m)
    kept &= ~greedy
    kept |= rank == 0
    w = torch.where(kept, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)                         # back in the order of the indices
    mass = w.cumsum(1)
    total = mass[:, -1:]
    token = (mass <= s["u"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=V - 1)
    some = total > 0
    prob = torch.where(some, w.gather(1, token) / total, 0.0)
    return [torch.where(some, token, -1).int().flatten(), prob.float().flatten()]


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
_contexts = {}


def _context():
    """The process's context on the current device."""
    import channel_amd as ca
    at = torch.cuda.current_device()
    if at not in _contexts:
        _contexts[at] = ca.Context(at)
    return _contexts[at]


def _call(s):
    """The case's call with its arguments converted once, as a serving loop keeps it."""
    c, n = s["case"], s["case"]["n"]
    a = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    bind = _context().bind
    if c["kind"] == "tables":
        return bind("chn_block_tables", a["lens"], a["n_new"], n, a["prefix"], s["prefix"].numel(), a["free"],
                    s["free"].numel(), a["taken"], s["n_blocks"], c["bs"], s["max_blocks"], s["max_tokens"],
                    a["tables"], a["lens_out"], a["row_start"], a["slots"], a["clocks"], a["status"])
    if c["kind"] == "rope":
        return bind("chn_batch_qkv_rope_at", a["q"], a["k"], a["v"], a["qw"], a["kw"], a["q_out"], a["kc"], a["vc"],
                    a["clocks"], a["slots"], n, s["n_slots"], c["nq"], c["nkv"], c["D"], c["rot"], c["kv"], THETA, EPS)
    if c["kind"] == "attn":
        return bind("chn_prefix_decode_attn", a["q"], a["kc"], a["vc"], a["prefix"], s["prefix"].numel(), a["tables"],
                    a["lens"], n, s["max_blocks"], c["bs"], s["n_blocks"], c["nq"], c["D"], c["nkv"] * c["D"],
                    c["nq"] // c["nkv"], 1.0, a["out"])
    return bind("chn_sample", a["logits"], n, c["V"], c["V"] + c["pad"], a["T"], a["k"], a["p"], a["m"], a["u"],
                s["cap"], a["tokens"], a["probs"])


_OUTPUTS = {"tables": ("tables", "lens_out", "row_start", "slots", "clocks", "status"), "rope": ("q_out", "kc", "vc"),
            "attn": ("out",), "sample": ("tokens", "probs")}
_PLAIN = {"tables": _plain_tables, "rope": _plain_rope, "attn": _plain_attn, "sample": _plain_sample}


def run(state):
    kind = state["case"]["kind"]
    if own:
        call = state.get("call") or state.setdefault("call", _call(state))
        call()
        return [state[name] for name in _OUTPUTS[kind]]
    return _PLAIN[kind](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _u32(t):
    return t.cpu().numpy().view(np.uint32).astype(np.int64)


def _exact_tables(s):
    bs, prefix, free = s["case"]["bs"], _u32(s["prefix"]), _u32(s["free"])
    lens, new = _u32(s["lens"]), _u32(s["n_new"])
    tables = s["tables"].cpu().numpy().astype(np.int64)
    slots, clocks = (s[k].cpu().numpy().astype(np.int64) for k in ("slots", "clocks"))
    lens_out, row_start, taken, row = [], [0], int(_u32(s["taken"])[0]), 0
    for r in range(len(lens)):
        length = int(lens[r])
        if new[r] and length < len(prefix) * bs:
            tables[r, :len(prefix)] = prefix
            length = len(prefix) * bs
        for _ in range(int(new[r])):
            if length % bs == 0:
                tables[r, length // bs] = free[taken]
                taken += 1
            slots[row], clocks[row] = tables[r, length // bs] * bs + length % bs, length
            row, length = row + 1, length + 1
        lens_out.append(length)
        row_start.append(row)
    return [tables, np.array(lens_out), np.array(row_start), slots, clocks, np.array([0, taken, row])]


def _exact_rope(s):
    c = s["case"]
    n, rot = c["n"], c["rot"]

    def rows(x, weight, turn):
        x = x.double().cpu().numpy().reshape(n, -1, c["D"])
        x = x / np.sqrt(np.mean(x * x, axis=2, keepdims=True) + EPS)
        if weight is not None:
            x = x * weight.double().cpu().numpy()
        if turn:
            z = x[..., :rot // 2] + 1j * x[..., rot // 2:rot]
            angle = np.outer(_u32(s["clocks"]), THETA ** (-np.arange(0, rot, 2) / rot))
            z = z * np.exp(1j * angle)[:, None]
            x = np.concatenate([z.real, z.imag, x[..., rot:]], 2)
        return x.reshape(n, -1)
    at = _u32(s["slots"])
    kc, vc = s["kc"].double().cpu().numpy(), s["vc"].double().cpu().numpy()
    kc[at], vc[at] = rows(s["k"], s["kw"], True), rows(s["k"] if c["kv"] else s["v"], None, False)
    return [rows(s["q"], s["qw"], True), kc, vc]


def _exact_attn(s):
    c = s["case"]
    D, nkv, bs = c["D"], c["nkv"], c["bs"]
    out = torch.zeros((c["n"], c["nq"] * D), dtype=torch.float64, device="cuda")
    for r, length in enumerate(_u32(s["lens"])):
        pos = torch.arange(int(length), device="cuda")
        at = s["tables"][r].long()[pos // bs] * bs + pos % bs
        k, v = (s[x][at].double().view(-1, nkv, D).transpose(0, 1).contiguous() for x in ("kc", "vc"))
        p = torch.softmax(torch.bmm(s["q"][r].double().view(nkv, -1, D), k.transpose(1, 2).contiguous()), 2)
        out[r] = torch.bmm(p, v).flatten()
    return [out]


def _exact_sample(s):
    V, cap = s["case"]["V"], s["cap"]
    tokens, probs = [], []
    logits, u, T, p, m = (s[k].double().cpu().numpy() for k in ("logits", "u", "T", "p", "m"))
    for r in range(s["case"]["n"]):
        row = logits[r, :V]
        allowed = np.nonzero(row > LOWEST)[0]
        allowed = allowed[np.argsort(-row[allowed], kind="stable")]
        if not len(allowed):
            tokens.append(-1)
            probs.append(0.0)
            continue
        if not T[r] > 0:
            allowed = allowed[:1]
        elif s["k"][r]:
            allowed = allowed[:int(s["k"][r])]
        value = row[allowed]
        value = cap * np.tanh(value / cap) if cap else value
        weight = np.exp((value - value[0]) / T[r]) if T[r] > 0 else np.ones(1)
        if p[r] < 1:
            mass = np.concatenate([[0.0], np.cumsum(weight)])
            last = max(1, int(np.searchsorted(mass[:-1], p[r] * mass[-1], side="left")))
            allowed, weight = allowed[:last], weight[:last]
        if m[r] > 0:
            stay = weight >= min(m[r], 1.0)
            allowed, weight = allowed[stay], weight[stay]
        by_index = np.argsort(allowed)
        allowed, weight = allowed[by_index], weight[by_index]
        mass = np.cumsum(weight)
        at = min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), len(mass) - 1)
        tokens.append(int(allowed[at]))
        probs.append(weight[at] / mass[-1])
    return [np.array(tokens), np.array(probs)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "rope": _exact_rope, "attn": _exact_attn, "sample": _exact_sample}[case["kind"]](s)
