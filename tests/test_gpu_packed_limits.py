"""Steps of several tokens per request at the ends of their ranges: the most
requests, rows and logits behind 4 GiB, heads by the hundred, the same call
again.  Tolerances as in test_gpu_packed.py; log probabilities of equal logits
are log V, rounded once."""
import numpy as np
import pytest

import channel_amd as ca
from gpu_util import say
from oracle import packed
from test_gpu_packed import Batch
from test_gpu_paged import down32, up32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("words", [0, 1])
def test_the_most_requests(ctx, words):
    """8192 requests of up to two tokens, most of them of none in one half."""
    say("most requests", words)
    rng = np.random.default_rng(41)
    new = rng.integers(0, 3, 8192)
    new[2000:6000] = rng.random(4000) < 0.01
    Batch(ctx, 42, new, rng.integers(0, 6, 8192), nq=2, bs=4, words=words, sigma=2.0).check()


def test_requests_beyond_the_most_are_refused(ctx):
    b = Batch(ctx, 43, [1], [2]).up()
    args = list(b.args())
    args[7] = 8193
    with pytest.raises(ca.ChannelError):
        ctx.call(*args)


@pytest.mark.parametrize("D,nq,gqa", [(256, 256, 1), (512, 160, 10)])
def test_many_heads(ctx, D, nq, gqa):
    say("many heads", D, nq, gqa)
    Batch(ctx, 44, [5, 30], [40, 3], D=D, nq=nq, gqa=gqa).check()


@pytest.mark.parametrize("words", [0, 2])
def test_the_same_call_gives_the_same_bits(ctx, words):
    """Whatever call ran between and left its parts in the workspace."""
    say("same bits", words)
    b = Batch(ctx, 45, [40, 64, 3], [900, 0, 2100], words=words).up()
    b.call()
    first = b.got()
    Batch(ctx, 46, [300, 9], [50, 4000], D=512).run()
    Batch(ctx, 47, [1], [70]).run()
    b.call()
    assert np.array_equal(first, b.got())
    b.check(first)


@pytest.mark.parametrize("new,have", [
    ([3] * 32, [5] * 32), ([3] * 33, [5] * 33), ([3] * 31 + [60], [5] * 31 + [1500]), ([60] + [3] * 31, [1500] + [5] * 31),
    ([2, 60, 2, 64, 1], [0, 700, 3, 100, 90]), ([1] * 20, [95, 96, 97, 98] * 5), ([64] * 8, [0, 31, 32, 33, 63, 64, 65, 95]),
    ([65] * 6, [40] * 6), ([1], [192 * 128]), ([5] * 40, [150] * 40),
])
@pytest.mark.parametrize("words", [0, 2])
def test_shares_of_short_and_long_tiles(ctx, new, have, words):
    """As many tiles as CUs and one more, tiles on both sides of those that are cut, short ones beside long ones."""
    say("shares", new, have, words)
    Batch(ctx, 50, [min(n, 64) for n in new] if words else new, have, nq=16, words=words).check()


def test_rows_behind_4_gib(ctx):
    """A request whose rows of q and out lie behind 4 GiB."""
    say("rows behind 4 GiB")
    b = Batch(ctx, 48, [40], [100], nq=16, spare=0)
    width, first = 16 * 256, 270000
    q, out = ctx.zeros((first + 40) * width * 4), ctx.zeros((first + 40) * width * 4)
    ctx._check("chn_upload", ca.lib.chn_upload(ctx.handle, q.offset(first * width * 4), b.q.ctypes.data, b.q.nbytes))
    ctx.call("chn_paged_causal_attn", q, ctx.upload(b.kc), ctx.upload(b.vc), up32(ctx, b.tables), up32(ctx, [first, first + 40]),
             up32(ctx, b.lens), 1, first + 40, b.width, b.bs, b.nb, 16, 256, b.kv_dim, 2, 1.0, 0, out)
    got = np.empty((41, width), np.float32)
    ctx._check("chn_download", ca.lib.chn_download(ctx.handle, got.ctypes.data, out.offset((first - 1) * width * 4), got.nbytes))
    assert not got[0].any()
    b.check(got[1:])
    q.free()
    out.free()


def test_logits_behind_4_gib(ctx):
    say("logits behind 4 GiB")
    n, V = 4200, 262144
    x = ctx.zeros(n * V * 4)
    rng = np.random.default_rng(49)
    targets = rng.integers(0, V, n)
    last = rng.standard_normal(V).astype(np.float32)
    ctx._check("chn_upload", ca.lib.chn_upload(ctx.handle, x.offset((n - 1) * V * 4), last.ctypes.data, last.nbytes))
    lp, ranks, ids, tops = ctx.zeros(n * 4), ctx.zeros(n * 4), ctx.zeros(n * 8), ctx.zeros(n * 8)
    ctx.call("chn_token_logprobs", x, n, V, V, up32(ctx, targets), None, 0.0, 2, lp, None, ranks, ids, tops)
    got, log_v = ctx.download(lp, np.float32, n), np.log(V)
    # equal logits: 2^18 terms of one, an exact sum
    assert np.abs(got[:-1] + log_v).max() <= 2.0 ** -24 * log_v
    assert np.array_equal(down32(ctx, ranks, n)[:-1], targets[:-1])
    assert (down32(ctx, ids, 2 * n).reshape(n, 2)[:-1] == [0, 1]).all()
    w = packed.logprob_row(last, int(targets[-1]), 1.0, 0.0, 2)
    # 4 u H + u (4 + 2 log2 V), as in test_gpu_logprobs.py, and a rounding
    assert abs(got[-1] - w[0]) <= 2.0 ** -24 * (4 * w[1] + 40 + abs(w[0])) and down32(ctx, ranks, n)[-1] == w[2]
    assert down32(ctx, ids, 2 * n)[-2:].tolist() == w[3]
    x.free()
