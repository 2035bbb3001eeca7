"""The batched decode step over a paged cache on the CPU: what its entries
refuse (they check their arguments before they need a device), and hand-worked
cases of the oracle that the GPU tests compare with: bad blocks, a prefix,
lengths of zero, ties, barred rows, filters that leave one token."""
import numpy as np
import pytest

import channel_amd as ca
from oracle import paged

A = [(i + 1) << 32 for i in range(24)]        # addresses far apart; nothing is read before a check fails


def refused(fn, args, code=-1):
    rc = getattr(ca.lib, fn)(None, *args)
    assert rc == code, (fn, args, rc)
    return ca.lib.chn_last_error(None).decode()


def with_(args, **kw):
    args = list(args)
    for i, v in kw.items():
        args[int(i[1:])] = v
    return args


# lens n_new n_req prefix npb free n_free taken n_blocks bs max_blocks max_tokens tables lens_out row_start slots clocks status
TABLES = [A[0], A[1], 4, A[2], 2, A[3], 64, A[4], 100, 16, 32, 64, A[5], A[6], A[7], A[8], A[9], A[10]]
# q k v qw kw q_out kc vc clocks slots n_tok n_slots nq nkv D rot k_eq_v theta eps
ROPE = [A[0], A[1], A[2], A[3], A[4], A[5], A[6], A[7], A[8], A[9], 8, 64, 4, 2, 256, 256, 0, 1e4, 1e-6]
# q kc vc prefix npb tables lens n_req max_blocks bs n_blocks nq D kv_dim gqa scale out
ATTN = [A[0], A[1], A[2], A[3], 2, A[4], A[5], 4, 32, 16, 100, 4, 256, 512, 2, 1.0, A[6]]
# logits n V ld T k p m u cap tokens probs
SAMPLE = [A[0], 4, 1000, 1000, A[1], A[2], A[3], A[4], A[5], 30.0, A[6], A[7]]


@pytest.mark.parametrize("fn,args", [("chn_block_tables", TABLES), ("chn_batch_qkv_rope_at", ROPE),
                                     ("chn_prefix_decode_attn", ATTN), ("chn_sample", SAMPLE)])
def test_sound_calls_only_lack_the_context(fn, args):
    assert refused(fn, args) == "ctx is NULL"


@pytest.mark.parametrize("change,text", [
    (dict(_0=None), "NULL"), (dict(_1=None), "NULL"), (dict(_3=None), "NULL"), (dict(_5=None), "NULL"),
    (dict(_12=None), "NULL"), (dict(_13=None), "NULL"), (dict(_14=None), "NULL"), (dict(_15=None), "NULL"),
    (dict(_16=None), "NULL"), (dict(_17=None), "NULL"),
    (dict(_9=0), "block_size"), (dict(_9=24), "block_size"), (dict(_9=2048), "block_size"), (dict(_8=0), "blocks"),
    (dict(_8=1 << 28), "blocks"), (dict(_10=0), "tables"), (dict(_10=1 << 27), "tables"), (dict(_4=33), "prefix"),
    (dict(_13=A[0]), "overlaps"), (dict(_13=A[0] + 12), "overlaps"), (dict(_17=A[4] - 4), "overlaps"),
    (dict(_15=A[8], _16=A[8] + 4 * 63), "overlap"), (dict(_12=A[3] + 64), "overlaps"),
])
def test_block_tables_refusals(change, text):
    assert text in refused("chn_block_tables", with_(TABLES, **change))


def test_block_tables_refuses_too_many_requests():
    assert "n_req" in refused("chn_block_tables", with_(TABLES, _2=8193), -6)


@pytest.mark.parametrize("change,text", [
    (dict(_0=None), "NULL"), (dict(_2=None), "NULL"), (dict(_8=None), "NULL"), (dict(_9=None), "NULL"),
    (dict(_14=0), "head_dim"), (dict(_14=513), "head_dim"), (dict(_15=257), "rotary_dim"), (dict(_15=258), "rotary_dim"),
    (dict(_17=0.0), "theta"), (dict(_17=float("nan")), "theta"), (dict(_10=1 << 30), "too many"), (dict(_12=65537), "heads"),
])
def test_rope_at_refusals(change, text):
    assert text in refused("chn_batch_qkv_rope_at", with_(ROPE, **change))


def test_rope_at_takes_no_v_where_v_is_k():
    assert refused("chn_batch_qkv_rope_at", with_(ROPE, _2=None, _16=1)) == "ctx is NULL"


@pytest.mark.parametrize("change,text", [
    (dict(_0=None), "NULL"), (dict(_3=None), "NULL"), (dict(_5=None), "NULL"), (dict(_6=None), "NULL"),
    (dict(_16=None), "NULL"), (dict(_12=128), "head_dim"), (dict(_14=0), "ratio"), (dict(_14=3), "ratio"),
    (dict(_14=32, _11=32), "ratio"), (dict(_13=508), "kv_dim"), (dict(_13=514), "kv_dim"), (dict(_0=A[0] + 4), "aligned"),
    (dict(_16=A[6] + 8), "aligned"), (dict(_9=3), "block_size"), (dict(_4=33), "prefix"), (dict(_7=65537), "n_req"),
    (dict(_10=1 << 28), "blocks"), (dict(_8=1 << 27), "tables"),
])
def test_prefix_attn_refusals(change, text):
    assert text in refused("chn_prefix_decode_attn", with_(ATTN, **change))


@pytest.mark.parametrize("change,text", [
    (dict(_0=None), "NULL"), (dict(_8=None), "NULL"), (dict(_10=None), "NULL"), (dict(_2=0), "V="),
    (dict(_2=(1 << 20) + 1, _3=1 << 21), "V="), (dict(_3=999), "ld"), (dict(_9=-1.0), "softcap"),
    (dict(_9=float("inf")), "softcap"), (dict(_9=float("nan")), "softcap"), (dict(_1=65536), "n_rows"),
])
def test_sample_refusals(change, text):
    assert text in refused("chn_sample", with_(SAMPLE, **change))


def test_sample_settings_are_optional():
    assert refused("chn_sample", with_(SAMPLE, _4=None, _5=None, _6=None, _7=None, _11=None)) == "ctx is NULL"


# ---- the oracle, by hand
def tables_of(lens, n_new, prefix=(), free=(), taken=0, n_blocks=100, bs=4, max_tokens=16, width=6, table=None):
    n = len(lens)
    t = np.full((n, width), 77) if table is None else np.array(table)
    return paged.block_tables(lens, n_new, list(prefix), list(free), taken, n_blocks, bs, max_tokens, t, [0] * n,
                              [0] * (n + 1), [55] * max_tokens, [55] * max_tokens)


def test_tables_by_hand():
    # a new request behind a prefix of two blocks, one that gains nothing, one that fills its block and opens another
    t, ln, rs, sl, ck, st = tables_of([0, 9, 11], [3, 0, 2], prefix=[7, 3], free=[40, 41, 42], taken=1,
                                      table=[[77] * 6, [7, 3, 20, 77, 77, 77], [7, 3, 21, 77, 77, 77]])
    assert st == [0, 3, 5]
    assert t.tolist() == [[7, 3, 41, 77, 77, 77], [7, 3, 20, 77, 77, 77], [7, 3, 21, 42, 77, 77]]
    assert ln.tolist() == [11, 9, 13] and rs.tolist() == [0, 3, 3, 5]
    assert sl.tolist() == [164, 165, 166, 21 * 4 + 3, 168] + [55] * 11
    assert ck.tolist() == [8, 9, 10, 11, 12] + [55] * 11


@pytest.mark.parametrize("kw,flag", [(dict(free=[1]), 1), (dict(free=list(range(9)), width=2), 2),
                                     (dict(free=list(range(9)), max_tokens=8), 4)])
def test_tables_refuse_whole(kw, flag):
    t, ln, rs, sl, ck, st = tables_of([0], [9], **kw)
    assert st == [flag, 3, 9]
    assert (t == 77).all() and not ln.any() and not rs.any() and (sl == 55).all() and (ck == 55).all()


def test_tables_bad_block_has_no_slot():
    t, _, _, sl, _, st = tables_of([0], [5], free=[100, 2])
    assert st[0] == 0 and t[0, :2].tolist() == [100, 2]
    assert sl[:5].tolist() == [paged.NO_SLOT] * 4 + [8]


def test_request_slots_leave_bad_blocks_out():
    assert paged.request_slots(11, [2], [99, 100, 1], 4, 100).tolist() == [8, 9, 10, 11, 4, 5, 6]
    assert paged.request_slots(0, [2], [0, 1, 1], 4, 100).tolist() == []
    assert paged.request_slots(10 ** 9, [], [1, 0], 2, 100).tolist() == [2, 3, 0, 1]


def test_sample_by_hand():
    inf = float("inf")
    row = [0.0, 2.0, 1.0, 2.0, -inf, float("nan"), float(np.finfo(np.float32).min)]
    assert paged.sample_row(row, T=0.0)[:2] == (1, 1.0)
    assert paged.sample_row(row, k=1, u=0.99)[:2] == (1, 1.0)                # of equal logits the lower index
    assert paged.sample_row(row, k=2, u=0.5)[:2] == (3, 0.5)
    assert paged.sample_row(row, p=0.0, u=0.9)[0] == 1
    assert paged.sample_row(row, m=1.0, u=0.4)[:2] == (1, 0.5)
    w = np.exp([-2.0, 0.0, -1.0, 0.0])
    c = np.cumsum(w) / w.sum()
    for u, want in ((0.0, 0), (c[0] * 0.99, 0), (c[0] * 1.01, 1), (c[1] * 1.01, 2), (c[2] * 1.01, 3), (1.0, 3), (7.0, 3)):
        assert paged.sample_row(row, u=u)[0] == want
    assert paged.sample_row([-inf, -inf])[:2] == (paged.NO_TOKEN, 0.0)
    assert paged.sample_row([1.0, inf, 0.0, inf], u=0.6)[:2] == (3, 0.5)
    assert paged.sample_row([5.0], p=0.1, k=3, m=0.5, u=0.9)[:2] == (0, 1.0)
