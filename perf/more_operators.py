"""Performance cases of steps in which a request takes several tokens, over a paged KV cache.

Prompts, drafted trees and their scoring, four operators, each a "kind" here:

  drafts    ancestor masks and clocks of the requests' drafted trees from the
            nodes' parents (chn_draft_trees)
  tree      attention of the drafted tokens: each sees its request's cached
            tokens and its own ancestors (chn_paged_tree_attn)
  prompt    causal attention of packed prompts (or chunks of them) of
            different lengths, with or without a window
            (chn_paged_causal_attn)
  logprobs  log probabilities of given tokens, their ranks, the entropy and
            the likeliest alternatives of every row of logits
            (chn_token_logprobs)

Where `own` is false, run() computes them in their plain form.  Sizes: the
12B-class model of bench.py (16 query / 8 KV heads of 256, vocabulary 262144,
window 512 and the prefill's 1024), heads of 512, and generic ones.  Unsigned
32-bit values are held in int32 tensors: -1 is "no parent", "no token" and, in
a table, "no block".
"""
import math

import numpy as np
import torch

own = False

LOWEST = torch.finfo(torch.float32).min


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a step that drafts small trees for a few conversations
        dict(name="drafts_8", kind="drafts", n=8, new=32, have=700, words=1),
        # the largest such step: hundreds of requests, trees of up to 256 nodes, chains among them
        dict(name="drafts_500", kind="drafts", n=500, new=256, have=4000, words=8),
        # a few conversations, trees of up to 16 nodes: latency
        dict(name="tree_chat_8", kind="tree", n=8, new=16, have=700, words=1, D=256, nq=16, nkv=8, window=0, bs=16),
        # many users, some way into theirs, on a sliding layer
        dict(name="tree_users_64", kind="tree", n=64, new=32, have=4000, words=1, D=256, nq=16, nkv=8, window=1024, bs=16),
        # large trees behind long documents
        dict(name="tree_long_5", kind="tree", n=5, new=64, have=60000, words=2, D=256, nq=16, nkv=8, window=0, bs=64),
        # 512-wide heads, an odd number of requests, trees of up to 100 nodes
        dict(name="tree_d512_13", kind="tree", n=13, new=100, have=3000, words=4, D=512, nq=16, nkv=4, window=0, bs=16),
        # one short question: latency
        dict(name="prompt_one_24", kind="prompt", n=1, new=24, have=0, D=256, nq=16, nkv=8, window=0, bs=16),
        # a burst of prompts of different lengths on a sliding layer, some behind earlier turns
        dict(name="prompt_burst_48", kind="prompt", n=48, new=1500, have=500, D=256, nq=16, nkv=8, window=1024, bs=16),
        # one chunk of a long document behind what is cached of it
        dict(name="prompt_chunk_2000", kind="prompt", n=1, new=2000, have=30000, D=256, nq=16, nkv=8, window=0, bs=32),
        # 512-wide heads, an odd number of prompts
        dict(name="prompt_d512_9", kind="prompt", n=9, new=1111, have=0, D=512, nq=16, nkv=4, window=0, bs=16),
        # the answer's next token, for a user who asks for its alternatives
        dict(name="logprobs_one", kind="logprobs", n=1, V=262144, pad=0, top=20, cap=30.0, mix="chat"),
        # a prompt's tokens scored under the whole vocabulary
        dict(name="logprobs_prompt_500", kind="logprobs", n=500, V=262144, pad=0, top=5, cap=0.0, mix="prompt"),
    ]


def _log_int(rng, lo, hi):
    """An integer between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _pairs(case):
    """Query rows times keys, as prepare() draws them in the mean."""
    new = _mean(case["n"], case["new"])
    have = _mean(case["n"], case["have"]) if case["have"] else 0
    seen = have + (new if case["kind"] == "tree" else new / 2)
    if case["window"]:
        seen = min(seen, case["window"])
    return case["n"] * new * seen


def draw(rng):
    kind = rng.choice(["drafts", "tree", "tree", "prompt", "prompt", "logprobs", "logprobs"])
    if kind == "drafts":
        words = rng.choice([1, 2, 3, 4, 8])
        return dict(kind=kind, n=_log_int(rng, 1, 500), new=rng.randint(1, 32 * words), have=_log_int(rng, 1, 100000),
                    words=words)
    if kind == "logprobs":
        n, V = _log_int(rng, 1, 500), _log_int(rng, 1000, 262144)
        return dict(kind=kind, n=n, V=V, pad=rng.choice([0, 0, rng.randint(1, 64)]), top=rng.choice([0, 1, 5, 20, 64]),
                    cap=rng.choice([0.0, 30.0]), mix=rng.choice(["chat", "prompt", "users"]))
    D, nkv = rng.choice([256, 256, 512]), rng.choice([1, 2, 4, 8])
    case = dict(kind=kind, D=D, nq=nkv * rng.choice([1, 2, 2, 4, 8]), nkv=nkv, bs=rng.choice([8, 16, 16, 32, 64]))
    if kind == "tree":
        words = rng.choice([1, 1, 2, 4])
        case.update(n=_log_int(rng, 1, 64), new=rng.randint(1, 32 * words), have=_log_int(rng, 1, 30000), words=words,
                    window=rng.choice([0, 0, 512, 1024]))
    else:
        case.update(n=_log_int(rng, 1, 48), new=_log_int(rng, 1, 2000), have=rng.choice([0, 0, _log_int(rng, 1, 30000)]),
                    window=rng.choice([0, 0, 512, 1024]))
    # at most the work of prompt_burst_48, of its keys and of the plain form's scores
    while case["n"] > 1 and (_pairs(case) * case["nq"] * D > 4.5e10 or case["n"] * (case["have"] + case["new"]) * nkv * D > 2.5e8
                             or case["n"] * case["new"] * (case["have"] + case["new"]) * case["nq"] > 1.5e9):
        case["n"] -= 1
    if case["new"] * (case["have"] + case["new"]) * case["nq"] > 1.1e9:
        case["have"] = int(1.1e9 / (case["new"] * case["nq"])) - case["new"]
    return case


def work(case):
    n = case["n"]
    if case["kind"] == "drafts":
        rows = n * _mean(n, case["new"])
        return {"bytes": rows * (8 + 4 * case["words"]) + n * 8, "flops": 0}
    if case["kind"] == "logprobs":
        return {"bytes": n * (case["V"] * 4 + 24 + 8 * case["top"]), "flops": 5.0 * n * case["V"]}
    rows = n * _mean(n, case["new"])
    keys = _mean(n, case["new"]) + (_mean(n, case["have"]) if case["have"] else 0)
    if case["window"]:
        keys = min(keys, case["window"] + _mean(n, case["new"]))
    return {"bytes": n * keys * case["nkv"] * case["D"] * 8 + 2 * rows * case["nq"] * case["D"] * 4,
            "flops": 4.0 * _pairs(case) * case["nq"] * case["D"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int64).astype(np.uint32).view(np.int32), device="cuda")


def _lengths(rng, n, most):
    """n lengths from 1 to `most`, short ones more often, of the same sum for every seed; one alone has the most."""
    if n == 1:
        return np.array([most])
    some = 1 + np.floor(rng.random(n) ** 2 * most).astype(np.int64)
    while (short := round(n * _mean(n, most)) - int(some.sum())):
        can = np.nonzero(some < most if short > 0 else some > 1)[0]
        some[rng.permutation(can)[:abs(short)]] += 1 if short > 0 else -1
    return some


def _mean(n, most):
    return most if n == 1 else (most + 2) / 3


def _trees(rng, new):
    """The parents of packed trees (index in the request, -1: none): most nodes hang on a recent one, some chains."""
    parents = []
    for n in new:
        i = np.arange(n)
        back = 1 + np.floor(rng.random(n) ** 2 * min(8, n)).astype(np.int64)
        back = np.where(rng.random() < 0.2, 1, back)
        parents.append(np.maximum(i - back, -1))
    return np.concatenate(parents) if len(parents) else np.zeros(0, np.int64)


def _ancestors(new, parents, words):
    """Packed ancestor-or-self masks, [rows][words]."""
    masks, at = np.zeros((len(parents), words), np.uint32), 0
    for n in new:
        for i in range(int(n)):
            p = parents[at + i]
            if p >= 0:
                masks[at + i] = masks[at + p]
            masks[at + i, i // 32] |= np.uint32(1 << (i % 32))
        at += n
    return masks


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    s = {"case": dict(case)}
    n = case["n"]
    if case["kind"] == "logprobs":
        V, ld = case["V"], case["V"] + case["pad"]
        logits = normal(n, ld) * 2.5
        # a few likely tokens per row, as a model's logits have
        at = torch.randint(0, V, (n, 40), generator=gen, device="cuda")
        logits.scatter_add_(1, at, 4 + 6 * torch.rand((n, 40), generator=gen, device="cuda"))
        rows = torch.arange(n, device="cuda")
        targets = at[:, 0].clone()
        T = np.ones(n, np.float32)
        if case["mix"] == "prompt":
            # a prompt's tokens are not always likely ones; its first has no row before it
            targets = torch.where(rows % 3 == 1, torch.randint(0, V, (n,), generator=gen, device="cuda"), targets)
            targets[-1] = -1
        elif case["mix"] == "users":
            # some rows come from a 16-bit head (many equal values), some under a grammar (most tokens barred), a row in
            # 25 belongs to nobody (all barred); temperatures differ
            coarse = logits.bfloat16().float()
            logits = torch.where((rows % 3 == 1)[:, None], coarse, logits)
            barred = torch.rand((n, ld), generator=gen, device="cuda") < 0.9
            logits = torch.where((rows % 5 == 2)[:, None] & barred, torch.full_like(logits, -math.inf), logits)
            logits = torch.where((rows % 25 == 23)[:, None], torch.full_like(logits, LOWEST), logits)
            T = np.asarray([0.0, 0.6, 0.8, 1.0, 1.0, 1.3], np.float32)[rng.integers(0, 6, n)]
        top = max(case["top"], 1)
        s.update(logits=logits.contiguous(), targets=targets.int(), T=torch.as_tensor(T, device="cuda"),
                 logp=torch.zeros(n, device="cuda"), entropy=torch.zeros(n, device="cuda"), ranks=_i32([0] * n),
                 top_ids=_i32([[0] * top] * n), top_logp=torch.zeros((n, top), device="cuda"))
        torch.cuda.synchronize()
        return s

    new = _lengths(rng, n, case["new"])
    have = _lengths(rng, n, case["have"]) if case["have"] else np.zeros(n, np.int64)
    if n >= 8:                                            # a request that takes nothing, one that has nothing yet
        new, have[5] = np.insert(_lengths(rng, n - 1, case["new"]), 3, 0), 0
    starts = np.concatenate([[0], np.cumsum(new)])
    rows = int(starts[-1]) + 7                            # a batch is a little larger than what fills it
    s.update(row_start=_i32(starts), lens=_i32(have + new), rows=rows, most_new=int(new.max()), longest=int((have + new).max()))
    if case["kind"] != "prompt":
        parents = _trees(rng, new)
        if case["kind"] == "drafts":
            s.update(parents=_i32(np.concatenate([parents, np.full(7, -1)])), masks=_i32(np.zeros((rows, case["words"]))),
                     clocks=_i32([-1] * rows))
            torch.cuda.synchronize()
            return s
        masks = _ancestors(new, parents, case["words"])
        if n >= 8 and new[5]:
            masks[starts[6] - 1] = 0                      # a drafted token that was dropped: it sees nothing
        s["masks"] = _i32(np.concatenate([masks, np.zeros((7, case["words"]), np.uint32)]))
    D, nq, nkv, bs = case["D"], case["nq"], case["nkv"], case["bs"]
    blocks = -(-(have + new) // bs)
    width = -(-(case["have"] + case["new"] + 2) // bs)
    pool = rng.permutation(int(blocks.sum()) + 16)        # blocks in any order
    tables, at = np.full((n, width), -1, np.int64), 0
    for r in range(n):
        tables[r, :blocks[r]] = pool[at:at + blocks[r]]
        at += blocks[r]
    # keys leave the q/k norm with a mean square of one; the scores' deviation is about 4, their scale 1 as the model's is
    s.update(q=normal(rows, nq * D) * (4 / math.sqrt(D)), kc=normal(len(pool) * bs, nkv * D),
             vc=normal(len(pool) * bs, nkv * D), tables=_i32(tables), max_blocks=width, n_blocks=len(pool),
             out=torch.zeros((rows, nq * D), device="cuda"))
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_drafts(s):
    c = s["case"]
    N, W, n, rows = s["most_new"], c["words"], c["n"], s["rows"]
    start, lens = s["row_start"].long(), s["lens"].long()
    new = start[1:] - start[:-1]
    i = torch.arange(N, device="cuda")
    there = i < new[:, None]
    row = torch.where(there, start[:-1, None] + i, rows)
    parent = torch.where(there, s["parents"].long()[row.clamp(max=rows - 1)], -1)
    # reach[r][a][b]: b is a or an ancestor of a; the paths double in length
    reach = ((parent[:, :, None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, (N - 1).bit_length())):
        reach = (reach @ reach > 0).float()
    depth = reach.sum(-1).long() - 1
    bits = torch.nn.functional.pad(reach, (0, W * 32 - N)).view(n, N, W, 32).long()
    words = (bits << torch.arange(32, device="cuda")).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).int()
    clock = (lens - new)[:, None] + depth
    masks = torch.cat([s["masks"], s["masks"].new_zeros(1, W)])          # one more row, for what is not there
    clocks = torch.cat([s["clocks"], s["clocks"].new_zeros(1)])
    masks[row.flatten()] = words.flatten(0, 1)
    clocks[row.flatten()] = clock.flatten().int()
    return [masks[:rows], clocks[:rows]]


def _plain_attn(s):
    c = s["case"]
    D, nq, nkv, n, bs, N, L, rows = (c["D"], c["nq"], c["nkv"], c["n"], c["bs"], s["most_new"], s["longest"], s["rows"])
    G = nq // nkv
    start, lens = s["row_start"].long(), s["lens"].long()
    new = start[1:] - start[:-1]
    i, pos = torch.arange(N, device="cuda"), torch.arange(L, device="cuda")
    there = i < new[:, None]
    row = torch.where(there, start[:-1, None] + i, rows)
    block = s["tables"].long()[:, pos // bs]
    held = (pos < lens[:, None]) & (block >= 0) & (block < s["n_blocks"])
    slot = torch.where(held, block * bs + pos % bs, 0)
    have = lens - new
    if c["kind"] == "tree":
        mask = s["masks"].long()[row.clamp(max=rows - 1)]
        node = pos - have[:, None]                                       # [n][L], negative: a cached token
        at = node.clamp(0, 32 * c["words"] - 1)
        word = mask.gather(2, (at // 32)[:, None].expand(n, N, L))
        drafted = ((word >> (at % 32)[:, None]) & 1).bool() & (node < 32 * c["words"])[:, None]
        ones = ((mask[..., None] >> torch.arange(32, device="cuda")) & 1).sum((2, 3))
        first = (have[:, None] + ones - c["window"]) if c["window"] else torch.zeros_like(ones)
        seen = torch.where(node[:, None] < 0, pos >= first[:, :, None], drafted)
    else:
        mine = have[:, None] + i
        seen = pos <= mine[:, :, None]
        if c["window"]:
            seen &= pos > (mine - c["window"])[:, :, None]
    seen = (seen & held[:, None] & there[:, :, None])[:, None, None]     # [n][1][1][N][L]
    q = s["q"][row.clamp(max=rows - 1)].view(n, N, nkv, G, D).permute(0, 2, 3, 1, 4).reshape(n, nkv, G * N, D)
    k = s["kc"][slot].view(n, L, nkv, D).permute(0, 2, 3, 1).contiguous()
    v = torch.where(held[:, :, None], s["vc"][slot], 0.0).view(n, L, nkv, D).permute(0, 2, 1, 3).contiguous()
    score = torch.where(seen, (q @ k).view(n, nkv, G, N, L), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1).view(n, nkv, G * N, 1)
    o = torch.where(total > 0, p.view(n, nkv, G * N, L) @ v / total, 0.0)
    out = torch.cat([s["out"], s["out"].new_zeros(1, nq * D)])
    out[row.flatten()] = o.view(n, nkv, G, N, D).permute(0, 3, 1, 2, 4).reshape(n * N, nq * D)
    return [out[:rows]]


def _plain_logprobs(s):
    c = s["case"]
    V, K = c["V"], c["top"]
    raw = s["logits"][:, :V]
    barred = ~(raw > LOWEST)                                              # NaN, -inf and the lowest value
    raw = torch.where(barred, -math.inf, raw)
    some = ~barred.all(1)
    x = c["cap"] * (raw / c["cap"]).tanh() if c["cap"] else raw
    T = s["T"][:, None]
    top = raw.argmax(1, keepdim=True)                                     # a row's largest values differ, or T > 0
    first = (raw == raw.gather(1, top)).int().argmax(1, keepdim=True)
    x = torch.where(raw == raw.gather(1, top), 0.0, (x - x.gather(1, top)) / torch.where(T > 0, T, 1.0))
    index = torch.arange(V, device="cuda")
    x = torch.where(barred | (~(T > 0) & (index != first)), -math.inf, x)
    e = x.exp()
    total = e.sum(1, keepdim=True)
    logp = x - total.log()
    entropy = total.log()[:, 0] - torch.where(e > 0, e * x, 0.0).sum(1) / total[:, 0]
    target = s["targets"].long()[:, None]
    given = (target >= 0) & (target < V)
    t = torch.where(given, target, 0)
    mine = raw.gather(1, t)
    ahead = (raw > mine) | ((raw == mine) & (index < t) & ~barred)
    ranked = given & some[:, None] & ~barred.gather(1, t)
    rank = torch.where(ranked, ahead.sum(1, keepdim=True), -1)
    value = torch.where(given, torch.where(some[:, None], logp.gather(1, t), -math.inf), 0.0)
    outputs = [value[:, 0], torch.where(some, entropy, 0.0), rank[:, 0].int()]
    if K:
        # equal values: the lower index first
        bits = (raw + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 20) + (V - 1 - index)
        order = key.topk(K, dim=1)[1]
        off = barred.gather(1, order)
        outputs += [torch.where(off, -1, order).int(), torch.where(off, -math.inf, logp.gather(1, order))]
    return outputs


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
    if c["kind"] == "drafts":
        return bind("chn_draft_trees", a["parents"], a["row_start"], a["lens"], n, s["rows"], c["words"], a["masks"],
                    a["clocks"])
    if c["kind"] == "logprobs":
        return bind("chn_token_logprobs", a["logits"], n, c["V"], c["V"] + c["pad"], a["targets"], a["T"], c["cap"],
                    c["top"], a["logp"], a["entropy"], a["ranks"], a["top_ids"] if c["top"] else None,
                    a["top_logp"] if c["top"] else None)
    shape = (n, s["rows"], s["max_blocks"], c["bs"], s["n_blocks"], c["nq"], c["D"], c["nkv"] * c["D"], c["nq"] // c["nkv"],
             1.0, c["window"], a["out"])
    if c["kind"] == "tree":
        return bind("chn_paged_tree_attn", a["q"], a["kc"], a["vc"], a["tables"], a["row_start"], a["lens"], a["masks"],
                    c["words"], *shape)
    return bind("chn_paged_causal_attn", a["q"], a["kc"], a["vc"], a["tables"], a["row_start"], a["lens"], *shape)


_OUTPUTS = {"drafts": ("masks", "clocks"), "tree": ("out",), "prompt": ("out",),
            "logprobs": ("logp", "entropy", "ranks", "top_ids", "top_logp")}
_PLAIN = {"drafts": _plain_drafts, "tree": _plain_attn, "prompt": _plain_attn, "logprobs": _plain_logprobs}


def run(state):
    c = state["case"]
    if own:
        call = state.get("call") or state.setdefault("call", _call(state))
        call()
        return [state[name] for name in _OUTPUTS[c["kind"]][:3 if c.get("top") == 0 else 5]]
    return _PLAIN[c["kind"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _u32(t):
    return t.cpu().numpy().view(np.uint32).astype(np.int64)


def _exact_drafts(s):
    start, lens, parents = _u32(s["row_start"]), _u32(s["lens"]), s["parents"].cpu().numpy()
    masks, clocks = s["masks"].cpu().numpy().view(np.uint32).copy(), s["clocks"].cpu().numpy().copy()
    for r in range(len(lens)):
        n = start[r + 1] - start[r]
        for i in range(n):
            bits, node = 0, i
            while node >= 0:
                bits |= 1 << int(node)
                node = parents[start[r] + node]
            masks[start[r] + i] = [(bits >> (32 * w)) & 0xFFFFFFFF for w in range(masks.shape[1])]
            clocks[start[r] + i] = lens[r] - n + bits.bit_count() - 1 if hasattr(bits, "bit_count") else (
                lens[r] - n + bin(bits).count("1") - 1)
    return [masks.view(np.int32), clocks]


def _exact_attn(s):
    c = s["case"]
    D, nkv, bs = c["D"], c["nkv"], c["bs"]
    G = c["nq"] // nkv
    start, lens = _u32(s["row_start"]), _u32(s["lens"])
    out = s["out"].double()
    bit = None
    if c["kind"] == "tree":
        words = s["masks"].cpu().numpy().view(np.uint32)
        bit = np.unpackbits(words.astype("<u4").view(np.uint8), axis=1, bitorder="little").astype(bool)
    for r, length in enumerate(lens):
        a, b = int(start[r]), int(start[r + 1])
        if a == b or not length:
            continue
        have = int(length) - (b - a)
        pos = torch.arange(int(length), device="cuda")
        at = s["tables"][r].long()[pos // bs] * bs + pos % bs
        hidden = torch.zeros((b - a, int(length)), dtype=torch.bool)
        if bit is not None:
            hidden[:, have:] = ~torch.from_numpy(bit[a:b, :b - a])
            if c["window"]:
                for i in range(b - a):
                    hidden[i, :max(0, min(have, have + int(bit[a + i].sum()) - c["window"]))] = True
        else:
            for i in range(b - a):
                hidden[i, have + i + 1:] = True
                if c["window"]:
                    hidden[i, :max(0, have + i + 1 - c["window"])] = True
        hidden = hidden.cuda()
        nothing = hidden.all(1)
        for h in range(nkv):
            k, v = (s[x][at, h * D:(h + 1) * D].double() for x in ("kc", "vc"))
            kt = k.t().contiguous()
            for g in range(G):
                col = slice((h * G + g) * D, (h * G + g + 1) * D)
                score = (s["q"][a:b, col].double() @ kt).masked_fill_(hidden, -math.inf)
                o = torch.softmax(score, 1) @ v
                out[a:b, col] = torch.where(nothing[:, None], 0.0, o)
    return [out]


def _exact_logprobs(s):
    c = s["case"]
    V, K, cap = c["V"], c["top"], c["cap"]
    logp, entropy, ranks, ids, tops = [], [], [], [], []
    for r in range(c["n"]):
        row, t, T = s["logits"][r, :V].double().cpu().numpy(), int(s["targets"][r]), float(s["T"][r])
        allowed = np.nonzero(row > LOWEST)[0]
        given = 0 <= t < V
        if not len(allowed):
            logp.append(-math.inf if given else 0.0)
            entropy.append(0.0)
            ranks.append(-1)
            ids.append([-1] * K)
            tops.append([-math.inf] * K)
            continue
        value = row[allowed]
        best = int(np.argmax(value))
        x = cap * np.tanh(value / cap) if cap else value
        if T > 0:
            x = (x - x[best]) / T
            lp = x - np.log(np.exp(x).sum())
        else:
            lp = np.full(len(x), -math.inf)
            lp[best] = 0.0
        p = np.exp(lp)
        entropy.append(-(p[p > 0] * lp[p > 0]).sum())
        place = int(np.searchsorted(allowed, t)) if given else 0
        if given and place < len(allowed) and allowed[place] == t:
            logp.append(lp[place])
            ranks.append(int((value > value[place]).sum() + (value[:place] == value[place]).sum()))
        else:
            logp.append(-math.inf if given else 0.0)
            ranks.append(-1)
        if K:
            border = np.partition(value, -min(K, len(value)))[-min(K, len(value))]
            few = np.nonzero(value >= border)[0]
            few = few[np.argsort(-value[few], kind="stable")][:K]
            short = K - len(few)
            ids.append([int(i) for i in allowed[few]] + [-1] * short)
            tops.append([float(v) for v in lp[few]] + [-math.inf] * short)
    outputs = [np.array(logp), np.array(entropy), np.array(ranks)]
    return outputs + ([np.array(ids), np.array(tops)] if K else [])


def exact(case, seed):
    s = prepare(case, seed)
    return {"drafts": _exact_drafts, "tree": _exact_attn, "prompt": _exact_attn, "logprobs": _exact_logprobs}[case["kind"]](s)
