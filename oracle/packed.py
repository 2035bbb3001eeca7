"""Plain 64-bit restatement of the steps in which a request takes several
tokens over a paged KV cache (chn_draft_trees, chn_paged_causal_attn,
chn_paged_tree_attn, chn_token_logprobs): one row at a time, from the
definitions in channel_hip.h.

TEST INFRASTRUCTURE ONLY, like the rest of this package.
"""
import numpy as np

NO_TOKEN = 0xFFFFFFFF
LOWEST = float(np.finfo(np.float32).min)


def rows_of(row_start, r, n_rows):
    """(first, number) of the batch rows of request r."""
    s, e = min(int(row_start[r]), n_rows), min(int(row_start[r + 1]), n_rows)
    return s, max(e - s, 0)


def draft_trees(parents, row_start, lens, n_rows, words, masks, clocks):
    """The written masks [n_rows][words] and clocks (copies)."""
    masks, clocks = np.array(masks, np.int64), np.array(clocks, np.int64)
    for r, length in enumerate(lens):
        s, n = rows_of(row_start, r, n_rows)
        have = max(int(length) - n, 0)
        for i in range(n):
            path, node = [], i
            while i < 32 * words:
                path.append(node)
                if parents[s + node] >= node:
                    break
                node = int(parents[s + node])
            masks[s + i] = [sum(1 << (j % 32) for j in path if j // 32 == w) for w in range(words)]
            clocks[s + i] = have + max(len(path) - 1, 0)
    return masks, clocks


def seen_by(i, n, length, window, mask=None):
    """The positions that row i of n sees, of a request of `length` tokens with them."""
    have = length - n
    if mask is None:
        return np.arange(max(0, have + i + 1 - window if window else 0), max(0, have + i + 1))
    bits = [32 * w + b for w in range(len(mask)) for b in range(32) if int(mask[w]) >> b & 1]
    first = max(0, have + len(bits) - window) if window else 0
    drafted = [have + j for j in bits if j < n and have + j >= 0]
    return np.array(list(range(first, max(0, have))) + drafted, np.int64)


def packed_attn(q, kc, vc, tables, row_start, lens, bs, n_blocks, num_q, D, gqa, scale, window, masks=None, out=None,
                sizes=None):
    """q [n_rows][num_q * D], caches [slots][kv_dim]: (out, the largest |score|, the largest sum of |q k|
    products, the most keys of a row).  sizes ([n_rows][num_q][3], or None) receives for each row and head the sum of
    weight times largest |v| over the keys that it sees, its largest sum of |q k| products, and its keys."""
    n_rows = len(q)
    out = np.zeros((n_rows, num_q * D)) if out is None else np.array(out, np.float64)
    big = absum = 0.0
    most = 0
    for r in range(len(lens)):
        s, n = rows_of(row_start, r, n_rows)
        table = np.asarray(tables[r], np.int64)
        length = min(int(lens[r]), len(table) * bs)
        for i in range(n):
            pos = seen_by(i, n, length, window, None if masks is None else masks[s + i])
            block = table[pos // bs] if len(pos) else pos
            at = (block * bs + pos % bs)[block < n_blocks]
            most = max(most, len(at))
            for h in range(num_q):
                o = out[s + i, h * D:(h + 1) * D]
                c = slice(h // gqa * D, h // gqa * D + D)
                k, v = kc[at, c].astype(np.float64), vc[at, c].astype(np.float64)
                qv = q[s + i, h * D:(h + 1) * D].astype(np.float64)
                with np.errstate(all="ignore"):
                    score = k @ qv * scale
                    keep = score != -np.inf
                    if not keep.any():
                        o[:] = 0
                        continue
                    v, score = v[keep], score[keep]
                    p = np.exp(score - score.max())
                    o[:] = p @ v / p.sum()
                    if not np.isfinite(score).all():
                        o[:] = np.nan
                if np.isfinite(score).all():
                    big = max(big, float(np.abs(score).max()))
                    mine = float((np.abs(k[keep]) @ np.abs(qv)).max() * abs(scale))
                    absum = max(absum, mine)
                    if sizes is not None:
                        sizes[s + i, h] = p @ np.abs(v).max(1) / p.sum(), mine, len(at)
    return out, big, absum, most


def logprob_row(row, target, T=1.0, cap=0.0, n_top=0):
    """(log p of target, entropy, rank, ids, their log p) of one row."""
    row = np.asarray(row, np.float64)
    order = np.nonzero(row > LOWEST)[0]
    order = order[np.argsort(-row[order], kind="stable")]
    given = target < len(row)
    if not len(order):
        return (-np.inf if given else 0.0), 0.0, NO_TOKEN, [NO_TOKEN] * n_top, [-np.inf] * n_top
    x = row[order]
    lp = np.full(len(x), -np.inf)
    if T > 0:
        with np.errstate(all="ignore"):
            top = x == x[0]
            x = cap * np.tanh(x / cap) if cap else x
            x = np.where(top, 0.0, (x - x[0]) / T)
            lp = x - np.log(np.exp(x).sum())
    else:
        lp[0] = 0.0
    p = np.exp(lp)
    entropy = float(-(p[p > 0] * lp[p > 0]).sum())
    at = np.nonzero(order == target)[0]
    value = float(lp[at[0]]) if len(at) else (-np.inf if given else 0.0)
    short = max(n_top - len(order), 0)
    return (value, entropy, int(at[0]) if len(at) else NO_TOKEN, [int(i) for i in order[:n_top]] + [NO_TOKEN] * short,
            [float(v) for v in lp[:n_top]] + [-np.inf] * short)
