"""Attention of packed prompts and of drafted trees where operands differ widely
in size: what a row does not see, and what lies under weights of nothing, takes
no digits from what it sees.

Tolerance, for each row and head by the keys that IT sees (u = 2^-24): a score
is off by (D + 14) u S at most, S its largest sum of |q k| (see
test_gpu_packed.py), which moves a weight by twice that of its own; the
exponential, the sums of L keys and the split operands move it by 2 (L + 20) u.
With w_k the exact weights and v_k the keys' values, no value is off by more
than (2 (D + 14) u S + 2 (L + 20) u) sum_k w_k max|v_k|.  The halves of a
weight times V scale leave 2^-36 of the largest such product, and V's own 2^-39
of the key's largest value: L times both is below what the second term has
for the L keys."""
import numpy as np
import pytest

import channel_amd as ca
from gpu_util import say
from oracle import packed
from test_gpu_packed import U, Batch
from test_gpu_paged import up32

pytestmark = pytest.mark.gpu


def check_rows(b, out=None, but=()):
    """All rows but the ones named."""
    out = b.run() if out is None else out
    sizes = np.zeros((b.rows, b.nq, 3))
    want, _, _, _ = packed.packed_attn(b.q, b.kc, b.vc, b.tables, b.row_start, b.lens, b.bs, b.nb, b.nq, b.D, b.gqa, b.scale,
                                       b.window, b.masks, b.old, sizes)
    A, S, L = sizes[..., 0], sizes[..., 1], sizes[..., 2]
    bound = (2 * (b.D + 14) * U * S + 2 * (L + 20) * U) * A
    out, want = out.copy(), want.copy()
    out[list(but)] = want[list(but)] = 0
    assert np.isfinite(out).all()
    off = np.abs(out - want).reshape(b.rows, b.nq, b.D).max(2)
    taken = int(min(b.row_start[-1], b.rows))
    worst = (off[:taken] / np.maximum(bound[:taken], 1e-300)).max()
    say(f"  {worst:.3g} of the bound; relative {(off[:taken] / np.maximum(A[:taken], 1e-300)).max():.3g}")
    assert (off <= bound).all(), np.argwhere(off > bound)[:4]
    assert np.array_equal(out[taken:], b.old[taken:])


def slots_of(b, r, positions):
    positions = np.asarray(positions)
    return b.tables[r, positions // b.bs] * b.bs + positions % b.bs


@pytest.mark.parametrize("what", [1e6, 1e12, 1e16])
@pytest.mark.parametrize("D", [256, 512])
def test_finite_values_in_unseen_slots(ctx, D, what):
    """Slots of no token, of tokens outside the window, of other requests' blocks."""
    say("finite unseen", D, what)
    b = Batch(ctx, 12, [30, 70, 4], [41, 0, 200], D=D, window=48)
    seen = np.zeros(len(b.kc), bool)
    for r in range(b.n):
        n, length = int(b.row_start[r + 1] - b.row_start[r]), int(b.lens[r])
        seen[slots_of(b, r, np.arange(max(0, length - n + 1 - 48), length))] = True
    b.kc[~seen] *= np.float32(what)
    b.vc[~seen] *= np.float32(what)
    check_rows(b)


@pytest.mark.parametrize("log", [16, 24, 40, 52])
@pytest.mark.parametrize("D", [256, 512])
def test_large_values_of_later_tokens(ctx, D, log):
    """The prompts' last tokens' V is larger by a power of two: the rows before them do not see it."""
    say("later tokens", D, log)
    b = Batch(ctx, 60, [7, 90, 33], [0, 31, 300], D=D)
    for r in range(b.n):
        b.vc[slots_of(b, r, [b.lens[r] - 1])] *= np.float32(2.0 ** log)
    check_rows(b)


@pytest.mark.parametrize("log", [24, 45])
@pytest.mark.parametrize("D", [256, 512])
def test_large_values_of_other_branches(ctx, D, log):
    """Every third drafted token's V is large: its descendants see it, the other branches do not."""
    say("branches", D, log)
    b = Batch(ctx, 61, [40, 64, 9], [70, 3, 0], D=D, words=2)
    for r in range(b.n):
        b.vc[slots_of(b, r, np.arange(b.lens[r] - 1, b.lens[r] - (b.row_start[r + 1] - b.row_start[r]), -3))] *= np.float32(2.0 ** log)
    check_rows(b)


@pytest.mark.parametrize("at", [0, 31, 64, 150, 199])
@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("D", [256, 512])
def test_large_values_under_weights_of_nothing(ctx, D, words, at):
    """A cached token 85 powers of two below the others' scores has a V 2^45 times theirs: 2^-40 of the result."""
    say("weights of nothing", D, words, at)
    b = Batch(ctx, 62, [20], [200], D=D, words=words, nq=2, sigma=0.25)
    common = np.random.default_rng(1).standard_normal(D).astype(np.float32) / np.float32(np.sqrt(D))
    b.q += np.tile(common, 2)                                             # every query's product with it: about one
    slot = slots_of(b, 0, [at])
    b.kc[slot] = -59.0 * common
    b.vc[slot] *= np.float32(2.0 ** 45)
    check_rows(b)


@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("D", [256, 512])
def test_scores_that_rise_as_values_fall(ctx, D, order):
    """Along 300 keys scores rise (or fall) by 60 powers of two and V's sizes fall (or rise) by as many, so that every
    key adds alike; and V's alone by 50, so that the last (or first) keys' results remain."""
    say("rise and fall", D, order)
    for fall in (60, 50):
        b = Batch(ctx, 63, [30], [300], D=D, nq=2, sigma=0.25)
        common = np.random.default_rng(2).standard_normal(D).astype(np.float32)
        common /= np.linalg.norm(common)
        b.q = np.float32(0.01) * b.q + np.tile(common, 2)
        pos = np.arange(330)
        part = pos / 330.0 * order
        slot = slots_of(b, 0, pos)
        b.kc[slot] = np.float32(0.1) * b.kc[slot] + ((60 * np.log(2) * part)[:, None] * common).astype(np.float32)
        b.vc[slot] *= (2.0 ** (-fall * part))[:, None].astype(np.float32)
        check_rows(b)


@pytest.mark.parametrize("words", [0, 2])
@pytest.mark.parametrize("D", [256, 512])
def test_values_of_any_size_by_what_a_row_sees(ctx, D, words):
    """V's rows from 2^-50 to 2^50, cut tiles among them."""
    say("any size by row", D, words)
    b = Batch(ctx, 64, [40, 9, 60], [60, 200, 2500], D=D, words=words)
    b.vc *= (2.0 ** np.random.default_rng(3).integers(-50, 50, (len(b.vc), 1))).astype(np.float32)
    check_rows(b)


@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("D", [256, 512])
def test_rows_of_zeros_under_any_scale(ctx, D, words):
    """Queries of zeros and of tiny values under scales from 1e-36 up: every key that a row sees weighs alike, no other
    does."""
    say("zeros", D, words)
    for scale in (1e-36, 1e-20, 1e-6, 1.0, 1e20):
        b = Batch(ctx, 65, [30, 9], [40, 900], D=D, words=words, scale=scale, sigma=4.0 * min(1.0, 1.0 / scale))
        b.q[::3] = 0
        b.q[1::3] *= np.float32(1e-18)
        check_rows(b)


@pytest.mark.parametrize("what,log", [("q", -115), ("q", -100), ("k", -115), ("k", -104), ("v", -100), ("v", -108), ("v", -118)])
@pytest.mark.parametrize("D", [256, 512])
def test_tiny_operands(ctx, D, what, log):
    """Queries, K or V far below one, the scale making the scores ordinary ones; a row of V of zeros."""
    say("tiny", D, what, log)
    b = Batch(ctx, 67, [30, 9], [40, 900], D=D, scale=2.0 ** -log if what != "v" else 1.0)
    {"q": b.q, "k": b.kc, "v": b.vc}[what][:] *= np.float32(2.0 ** log)
    b.vc[slots_of(b, 0, [3])] = 0
    check_rows(b)


@pytest.mark.parametrize("D", [256, 512])
def test_tiny_values_beside_ordinary_ones(ctx, D):
    """Cached V near 2^-110, a new token's near one: rows before it keep their digits, those behind see both."""
    say("tiny beside", D)
    b = Batch(ctx, 68, [30], [40], D=D)
    b.vc[slots_of(b, 0, np.arange(60))] *= np.float32(2.0 ** -110)
    check_rows(b)


@pytest.mark.parametrize("D", [256, 512])
def test_factors_beyond_the_type(ctx, D):
    """Scale times the queries' largest component passes 2^128, their products with K are of ordinary size: no key has
    anything where the query is large."""
    say("factors", D)
    b = Batch(ctx, 66, [30, 9], [40, 900], D=D, scale=2.0 ** 122)
    b.q[:, ::D] = 2.0 ** 24
    b.kc *= np.float32(2.0 ** -122)
    b.kc[:, ::D] = 0
    check_rows(b)


@pytest.mark.parametrize("k,q", [(60, -60), (104, -104), (112, -112), (124, -124), (-60, 60), (-104, 104), (-112, 112)])
@pytest.mark.parametrize("D", [256, 512])
def test_large_keys_and_queries(ctx, D, k, q):
    """K or queries up to 2^124, the other as small: ordinary scores."""
    say("large", D, k, q)
    b = Batch(ctx, 69, [30, 9], [40, 900], D=D)
    b.kc *= np.float32(2.0 ** k)
    b.q *= np.float32(2.0 ** q)
    check_rows(b)


@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("log", [55, 57, 100, 120])
@pytest.mark.parametrize("D", [256, 512])
def test_large_values(ctx, D, log, words):
    """All of V large; one cached token's, which all rows see; one drafted or later token's."""
    say("large V", D, log, words)
    for at in (slice(None), 5, 950):
        b = Batch(ctx, 70, [30, 20], [40, 940], D=D, words=words)
        b.vc[at if isinstance(at, slice) else slots_of(b, 1, [at])] *= np.float32(2.0 ** log)
        check_rows(b)


@pytest.mark.parametrize("what", [1e18, 1e30])
@pytest.mark.parametrize("D", [256, 512])
def test_huge_values_in_unseen_slots(ctx, D, what):
    say("huge unseen", D, what)
    b = Batch(ctx, 71, [30, 70], [41, 0], D=D, window=48)
    seen = np.zeros(len(b.kc), bool)
    for r in range(b.n):
        n, length = int(b.row_start[r + 1] - b.row_start[r]), int(b.lens[r])
        seen[slots_of(b, r, np.arange(max(0, length - n + 1 - 48), length))] = True
    b.kc[~seen] *= np.float32(what)
    b.vc[~seen] *= np.float32(what)
    check_rows(b)


@pytest.mark.parametrize("plain", [False, True])
@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("D", [256, 512])
def test_lengths_at_the_end_of_their_range(ctx, D, words, plain):
    """A request of 2^31 - 16 tokens on a sliding layer, the last block of its table full: the same as one of 128 tokens
    whose table is that table's end.  plain: a row's query is NaN, so that its tile is computed in plain fp32."""
    say("long end", D, words, plain)
    width, small = (1 << 27) - 1, 8
    b = Batch(ctx, 72, [5], [small * 16 - 5], D=D, words=words, window=64, width=small, spare=0)
    if plain:
        b.q[3, 7] = np.nan
    b.up()
    table = ctx.zeros(width * 4)
    end = np.ascontiguousarray(b.tables, np.uint32)
    ctx._check("chn_upload", ca.lib.chn_upload(ctx.handle, table.offset((width - small) * 4), end.ctypes.data, end.nbytes))
    b.dev.update(tables=table, lens=up32(ctx, [width * 16]))
    b.width = width
    b.call()
    out = b.got()
    table.free()
    b.width = small
    if plain:
        assert np.isnan(out[3, :D]).all()
    check_rows(b, out, [3] if plain else [])


@pytest.mark.parametrize("window", [0, 128, (1 << 31) - 2, (1 << 31) - 1, (1 << 32) - 1])
@pytest.mark.parametrize("words", [0, 1, 2])
def test_windows_longer_than_any_request(ctx, words, window):
    """Windows up to 2^32 - 1 where requests hold fewer tokens than they have rows, as many, and more."""
    say("long windows", words, window)
    b = Batch(ctx, 73, [30, 9, 60, 20, 8, 64], [0, 0, 0, 100, 3, 0], words=words, window=window)
    b.lens = np.array([12, 9, 50, 120, 5, 63])
    check_rows(b)


def largest_values(b, log):
    """V's rows as large as the type allows, or 2^log times what they were: many of one sign in every column."""
    b.vc = np.float32(2.0 ** log) * (np.float32(1.0) + np.float32(0.9) * np.abs(np.tanh(b.vc)))
    b.vc[:, 1::2] *= -1
    b.q[::2] = 0                                                          # every key alike: hundreds of them sum up
    return b


@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("log", [60, 112, 127])
@pytest.mark.parametrize("D", [256, 512])
def test_values_whose_sums_pass_the_type(ctx, D, words, log):
    """Up to 50 keys of equal weight whose V is near the type's largest: their mean is no larger."""
    say("largest V", D, words, log)
    check_rows(largest_values(Batch(ctx, 75, [30], [20], D=D, words=words), log))


@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("have", [60, 700, 2500, 9000])
@pytest.mark.parametrize("D", [256, 512])
def test_parts_whose_sums_pass_the_type(ctx, D, words, have):
    """The same in tiles that are cut, into a few parts and into more than the join takes at a time."""
    say("largest V in parts", D, words, have)
    check_rows(largest_values(Batch(ctx, 74, [5, 30], [have, 60], D=D, words=words), 127))


@pytest.mark.parametrize("have", [60, 2500])
@pytest.mark.parametrize("D", [256, 512])
def test_plain_sums_pass_the_type(ctx, D, have):
    """The same where a NaN in one row's query leaves its tile to plain fp32."""
    say("largest V, plain", D, have)
    b = largest_values(Batch(ctx, 76, [5, 30], [have, 60], D=D), 127)
    b.q[[3, 9], ::D] = np.nan
    check_rows(b, but=[3, 9])


@pytest.mark.parametrize("seed", range(16))
def test_random_batches_of_any_size(ctx, seed):
    """Batches of any shape whose rows of q, K and V have sizes of their own, V's up to 2^120 apart."""
    rng = np.random.default_rng(3000 + seed)
    D, gqa, words = int(rng.choice([256, 512])), int(rng.integers(1, 17)), int(rng.choice([0, 0, 1, 2, 4]))
    n = int(np.exp(rng.uniform(0, np.log(12))))
    new = rng.integers(0, min(32 * words if words else 100, 400 // n) + 1, n)
    have = np.where(rng.random(n) < 0.3, 0, rng.integers(0, 1500 // n + 2, n))
    window = int(rng.choice([0, 0, 128, int(rng.integers(128, 400))]))
    shape = dict(D=D, gqa=gqa, nq=gqa * int(rng.integers(1, 3)), bs=int(2 ** rng.integers(0, 8)), words=words, window=window)
    say("random sizes", seed, shape, new.tolist(), have.tolist())
    b = Batch(ctx, 4000 + seed, new, have, **shape)
    size = lambda x, lo, hi: (2.0 ** rng.integers(lo, hi, (len(x), 1))).astype(np.float32)  # noqa: E731
    b.vc *= size(b.vc, -60, 61)
    b.kc *= size(b.kc, -8, 3)
    b.q *= size(b.q, -8, 2)
    check_rows(b)
