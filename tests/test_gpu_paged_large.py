"""Block tables of as many rows as 32 bits count: every row is placed once and
the call ends."""
import numpy as np
import pytest

from gpu_util import say
from test_gpu_paged import down32, up32

pytestmark = pytest.mark.gpu


def test_tables_of_nearly_two_to_the_32_rows(ctx):
    bs, width, n_blocks = 1024, (1 << 21) - 1, 4000000
    new = np.array([width * bs - 7, width * bs - 1000, 2990])      # past 2^32 - 2^18 rows
    rows = int(new.sum())
    assert 2 ** 32 - 2 ** 18 < rows < 2 ** 32
    need = -(-new // bs)
    rng = np.random.default_rng(1)
    free = rng.integers(0, n_blocks, int(need.sum()))            # blocks may repeat: nothing is read from them
    say(f"block_tables of {rows} rows")
    tables, slots, clocks = ctx.alloc(3 * width * 4), ctx.alloc((rows + 2) * 4), ctx.alloc((rows + 2) * 4)
    lens_out, row_start, status = up32(ctx, [9] * 3), up32(ctx, [9] * 4), up32(ctx, [9] * 3)
    for b in (slots, clocks):
        ctx.fill_u32(b, 77, rows + 2)
    ctx.call("chn_block_tables", up32(ctx, [0] * 3), up32(ctx, new), 3, 0, 0, up32(ctx, free), len(free), 0, n_blocks, bs,
             width, rows, tables, lens_out, row_start, slots, clocks, status)
    assert down32(ctx, status, 3).tolist() == [0, int(need.sum()), rows]
    assert down32(ctx, lens_out, 3).tolist() == new.tolist()
    start = np.concatenate([[0], np.cumsum(new)])
    assert np.array_equal(down32(ctx, row_start, 4), start)
    first = np.concatenate([[0], np.cumsum(need)])
    for at in (0, start[1] - 300, start[1], start[2] - 300, start[2], 2 ** 31 - 100, 2 ** 32 - 2 ** 18 - 100, rows - 300):
        t = np.arange(at, min(at + 300, rows))
        r = np.searchsorted(start, t, side="right") - 1
        pos = t - start[r]
        want = free[first[r] + pos // bs] * bs + pos % bs
        assert np.array_equal(ctx.download(slots, np.uint32, len(t), 4 * int(at)).astype(np.int64), want), at
        assert np.array_equal(ctx.download(clocks, np.uint32, len(t), 4 * int(at)).astype(np.int64), pos), at
    for b in (slots, clocks):
        assert ctx.download(b, np.uint32, 2, 4 * rows).tolist() == [77, 77]
        b.free()
    for r in range(3):
        got = ctx.download(tables, np.uint32, int(need[r]), 4 * r * width).astype(np.int64)
        assert np.array_equal(got, free[first[r]:first[r + 1]])
    tables.free()
