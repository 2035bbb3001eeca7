"""The context's workspace under the batched step: one call at the largest size
is enough for recordings of smaller ones, and does not grow under them."""
import numpy as np
import pytest

import channel_amd as ca
from gpu_util import say
from test_gpu_paged import up32

pytestmark = pytest.mark.gpu


class Step:
    """Attention of up to n requests over zeroed caches."""

    def __init__(self, ctx, n, D, nq, gqa, npb, width, bs):
        self.ctx, self.nq, self.npb, self.width, self.bs = ctx, nq, npb, width, bs
        self.D, self.gqa, self.nb = D, gqa, npb + 8
        kv_dim = nq // gqa * D
        self.kc, self.vc = ctx.zeros(self.nb * bs * kv_dim * 4), ctx.zeros(self.nb * bs * kv_dim * 4)
        self.q, self.out = ctx.zeros(n * nq * D * 4), ctx.zeros(n * nq * D * 4)
        self.prefix, self.tables = up32(ctx, np.arange(npb)), up32(ctx, np.full((n, width), npb))
        self.lens = up32(ctx, npb * bs + np.arange(n) % 5)

    def call(self, n, npb=None, width=None):
        self.ctx.call("chn_prefix_decode_attn", self.q, self.kc, self.vc, self.prefix, self.npb if npb is None else npb,
                      self.tables, self.lens, n, width or self.width, self.bs, self.nb, self.nq, self.D,
                      self.nq // self.gqa * self.D, self.gqa, 1.0, self.out)


@pytest.mark.parametrize("most,D,nq,gqa,npb,width", [
    (40, 256, 16, 2, 248, 400), (65, 256, 16, 2, 248, 400), (33, 512, 16, 4, 93, 200), (70, 256, 4, 4, 60, 61),
    (9, 512, 8, 8, 500, 500),
])
def test_the_largest_call_is_enough(most, D, nq, gqa, npb, width):
    """Warm once at the largest batch, then record every smaller one, with the whole prefix, a part of it and none."""
    say(f"workspace: most={most} D={D} nq={nq} gqa={gqa} npb={npb} width={width}")
    with ca.Context(0) as ctx:
        s = Step(ctx, most, D, nq, gqa, npb, width, 16)
        s.call(most)
        ctx.record_begin()
        s.call(most)
        first = ctx.record_end()
        for n in range(1, most + 1):
            for part in (npb, npb // 3, 0):
                ctx.record_begin()
                s.call(n, part)                                  # refused if the workspace would have to grow
                ctx.record_end()
            s.call(n)
        s.call(1, 0, width // 2)
        first.submit()                                           # refused if it had grown since
        ctx.sync()
