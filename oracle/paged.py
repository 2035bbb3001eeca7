"""Plain 64-bit restatement of the batched decode step over a paged KV cache
(chn_block_tables, chn_batch_qkv_rope_at, chn_prefix_decode_attn,
chn_sample): one request, token or row at a time, from the definitions in
channel_hip.h.

TEST INFRASTRUCTURE ONLY, like the rest of this package.
"""
import numpy as np

NO_SLOT = NO_TOKEN = 0xFFFFFFFF
NO_BLOCKS, TOO_LONG, TOO_MANY = 1, 2, 4
LOWEST = float(np.finfo(np.float32).min)


def block_tables(lens, n_new, prefix, free, taken, n_blocks, bs, max_tokens, tables, lens_out, row_start, slots,
                 clocks):
    """The written buffers (copies) and the three status words."""
    tables, lens_out, row_start, slots, clocks = (np.array(a, np.int64) for a in
                                                  (tables, lens_out, row_start, slots, clocks))
    P = len(prefix) * bs
    begin = [max(int(ln), P) if n else int(ln) for ln, n in zip(lens, n_new)]
    ceil = lambda v: -(-v // bs)  # noqa: E731
    need = [ceil(b + int(n)) - ceil(b) if n else 0 for b, n in zip(begin, n_new)]
    rows = sum(int(n) for n in n_new)
    status = [0, min(taken + sum(need), 0xFFFFFFFF), min(rows, 0xFFFFFFFF)]
    if taken + sum(need) > len(free):
        status[0] |= NO_BLOCKS
    if any(n and ceil(b + int(n)) > tables.shape[1] for b, n in zip(begin, n_new)):
        status[0] |= TOO_LONG
    if rows > max_tokens:
        status[0] |= TOO_MANY
    if status[0]:
        return tables, lens_out, row_start, slots, clocks, status
    row = 0
    for r, n in enumerate(n_new):
        if n and lens[r] < P:
            tables[r, :len(prefix)] = prefix
        row_start[r] = row
        for pos in range(begin[r], begin[r] + int(n)):
            if pos % bs == 0:
                tables[r, pos // bs] = free[taken]
                taken += 1
            b = int(tables[r, pos // bs])
            slots[row] = b * bs + pos % bs if b < n_blocks else NO_SLOT
            clocks[row] = pos
            row += 1
        lens_out[r] = begin[r] + int(n)
    row_start[len(n_new)] = row
    return tables, lens_out, row_start, slots, clocks, status


def rope_at(q, k, v, qw, kw, kc, vc, clocks, slots, rot, theta, eps):
    """q [n][nq][D], k / v [n][nkv][D], caches [n_slots][nkv * D]: (q_out, kc, vc)."""
    q, k, v, qw, kw = (np.asarray(a, np.float64) for a in (q, k, v, qw, kw))
    kc, vc = np.array(kc, np.float64), np.array(vc, np.float64)
    norm = lambda x: x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)  # noqa: E731
    half = rot // 2
    freq = float(np.float32(theta)) ** (-2.0 * np.arange(half) / rot) if half else np.zeros(0)

    def turn(x, clock):
        a, b = x[:, :half], x[:, half:rot]
        c, s = np.cos(clock * freq), np.sin(clock * freq)
        return np.concatenate([a * c - b * s, a * s + b * c, x[:, rot:]], 1)
    out = np.zeros_like(q)
    for t, (clock, slot) in enumerate(zip(clocks, slots)):
        out[t] = turn(norm(q[t]) * qw, float(clock))
        if slot < len(kc):
            kc[slot] = turn(norm(k[t]) * kw, float(clock)).ravel()
            vc[slot] = norm(v[t]).ravel()
    return out, kc, vc


def request_slots(length, prefix, table, bs, n_blocks):
    """The cache slots of a request's tokens, without those of bad blocks."""
    out = []
    for pos in range(min(int(length), len(table) * bs)):
        j = pos // bs
        b = int(prefix[j]) if j < len(prefix) else int(table[j])
        if b < n_blocks:
            out.append(b * bs + pos % bs)
    return np.array(out, np.int64)


def prefix_attn(q, kc, vc, prefix, tables, lens, bs, n_blocks, num_q, D, gqa, scale):
    """q [n][num_q * D], caches [slots][kv_dim]: (out, the largest |score|,
    the largest sum of |q k| products)."""
    n = len(lens)
    out, big, absum = np.zeros((n, num_q, D)), 0.0, 0.0
    for r in range(n):
        at = request_slots(lens[r], prefix, tables[r], bs, n_blocks)
        if not len(at):
            continue
        for h in range(num_q):
            c = slice(h // gqa * D, h // gqa * D + D)
            k, v = kc[at, c].astype(np.float64), vc[at, c].astype(np.float64)
            qv = q[r, h * D:(h + 1) * D].astype(np.float64)
            s = k @ qv * scale
            p = np.exp(s - s.max())
            out[r, h] = p @ v / p.sum()
            big = max(big, float(np.abs(s).max()))
            absum = max(absum, float((np.abs(k) @ np.abs(qv)).max() * abs(scale)))
    return out.reshape(n, -1), big, absum


def sample_row(row, T=1.0, k=0, p=1.0, m=0.0, u=0.0, cap=0.0):
    """(token, probability, margin): margin is how far, relative to the sum of
    the weights in question, the nearest other decision of top-p or of the
    draw lies."""
    row = np.asarray(row, np.float64)
    order = np.nonzero(row > LOWEST)[0]
    order = order[np.argsort(-row[order], kind="stable")]
    if not len(order):
        return NO_TOKEN, 0.0, 1.0
    if not T > 0:
        return int(order[0]), 1.0, 1.0
    if k:
        order = order[:k]
    x = row[order]
    with np.errstate(invalid="ignore", over="ignore"):
        x = cap * np.tanh(x / cap) if cap else x
        w = np.where(x == x[0], 1.0, np.exp((x - x[0]) / T))
    w = np.where(np.isnan(w), 0.0, w)
    margin = 1.0
    if p < 1:
        before = np.cumsum(w) - w
        goal = max(p, 0.0) * w.sum()
        keep = before < goal
        keep[0] = True
        if p > 0:
            margin = min(margin, float(np.abs(before[1:] - goal).min(initial=w.sum()) / w.sum()))
        order, w = order[keep], w[keep]
    if m > 0:
        stay = w >= min(m, 1.0)
        order, w = order[stay], w[stay]
    by = np.argsort(order)
    order, w = order[by], w[by]
    mass = np.cumsum(w)
    target = (u if u > 0 else 0.0) * mass[-1]
    at = int(np.searchsorted(mass, target, side="right"))
    if at >= len(mass):
        at = int(np.nonzero(w)[0][-1])
    if 0 < u < 1:
        margin = min(margin, float(np.abs(mass[:-1] - target).min(initial=mass[-1]) / mass[-1]))
    return int(order[at]), float(w[at] / mass[-1]), margin
