"""Steps in which a request takes several tokens, on the CPU: what the entries
refuse (they check their arguments before they need a device), and hand-worked
cases of the oracle that the GPU tests compare with."""
import math

import numpy as np
import pytest

from oracle import packed
from test_paged import A, refused, with_

# parents row_start lens n_req n_rows mask_words masks clocks
TREES = [A[0], A[1], A[2], 4, 64, 2, A[3], A[4]]
# q kc vc tables row_start lens n_req n_rows max_blocks bs n_blocks nq D kv_dim gqa scale window out
CAUSAL = [A[0], A[1], A[2], A[3], A[4], A[5], 4, 64, 32, 16, 100, 4, 256, 512, 2, 1.0, 0, A[6]]
# .. lens masks mask_words n_req ..
TREE = CAUSAL[:6] + [A[7], 2] + CAUSAL[6:]
# logits n V ld targets T cap n_top logp entropy ranks ids tops
SCORES = [A[0], 4, 1000, 1000, A[1], A[2], 30.0, 20, A[3], A[4], A[5], A[6], A[7]]


@pytest.mark.parametrize("fn,args", [("chn_draft_trees", TREES), ("chn_paged_causal_attn", CAUSAL),
                                     ("chn_paged_tree_attn", TREE), ("chn_token_logprobs", SCORES)])
def test_sound_calls_only_lack_the_context(fn, args):
    assert refused(fn, args) == "ctx is NULL"


@pytest.mark.parametrize("change,text", [
    (dict(_0=None), "NULL"), (dict(_1=None), "NULL"), (dict(_2=None), "NULL"), (dict(_6=None), "NULL"), (dict(_7=None), "NULL"),
    (dict(_5=0), "mask_words"), (dict(_5=9), "mask_words"), (dict(_6=A[0]), "overlaps"), (dict(_6=A[0] - 4), "overlaps"),
    (dict(_7=A[2] + 12), "overlaps"), (dict(_7=A[3] + 4 * 127), "overlap"),
])
def test_draft_trees_refusals(change, text):
    assert text in refused("chn_draft_trees", with_(TREES, **change))


@pytest.mark.parametrize("change,text", [(dict(_3=8193), "n_req"), (dict(_4=(1 << 24) + 1), "n_rows")])
def test_draft_trees_refuses_too_many(change, text):
    assert text in refused("chn_draft_trees", with_(TREES, **change), -6)


@pytest.mark.parametrize("change,text", [
    (dict(_0=None), "NULL"), (dict(_1=None), "NULL"), (dict(_2=None), "NULL"), (dict(_3=None), "NULL"), (dict(_4=None), "NULL"),
    (dict(_5=None), "NULL"), (dict(_17=None), "NULL"), (dict(_12=128), "head_dim"), (dict(_14=0), "ratio"),
    (dict(_14=3), "ratio"), (dict(_14=32, _11=32), "ratio"), (dict(_11=0), "ratio"), (dict(_11=4100, _13=1 << 20), "4096"),
    (dict(_13=508), "kv_dim"), (dict(_13=514), "kv_dim"), (dict(_0=A[0] + 4), "aligned"), (dict(_17=A[6] + 8), "aligned"),
    (dict(_9=3), "block_size"), (dict(_10=1 << 28), "blocks"), (dict(_8=1 << 27), "tables"), (dict(_15=0.0), "scale"),
    (dict(_15=math.nan), "scale"), (dict(_15=math.inf), "scale"), (dict(_17=A[0]), "overlaps"),
    (dict(_17=A[0] + 63 * 4096), "overlaps"),
])
def test_causal_attn_refusals(change, text):
    assert text in refused("chn_paged_causal_attn", with_(CAUSAL, **change))


@pytest.mark.parametrize("change,text", [(dict(_6=8193), "n_req"), (dict(_7=(1 << 24) + 1), "n_rows")])
def test_causal_attn_refuses_too_many(change, text):
    assert text in refused("chn_paged_causal_attn", with_(CAUSAL, **change), -6)


@pytest.mark.parametrize("change,text", [
    (dict(_6=None), "NULL"), (dict(_7=0), "mask_words"), (dict(_7=9), "mask_words"), (dict(_18=63), "window"),
    (dict(_0=None), "NULL"), (dict(_14=100), "head_dim"), (dict(_19=A[0]), "overlaps"),
])
def test_tree_attn_refusals(change, text):
    assert text in refused("chn_paged_tree_attn", with_(TREE, **change))


def test_tree_attn_takes_a_window_of_the_largest_tree():
    assert refused("chn_paged_tree_attn", with_(TREE, _18=64)) == "ctx is NULL"


@pytest.mark.parametrize("change,text", [
    (dict(_0=None), "NULL"), (dict(_4=None), "NULL"), (dict(_8=None), "NULL"), (dict(_11=None), "top_ids"),
    (dict(_12=None), "top_ids"), (dict(_7=65), "n_top"), (dict(_2=0), "V="), (dict(_2=(1 << 20) + 1, _3=1 << 21), "V="),
    (dict(_3=999), "ld="), (dict(_6=-1.0), "softcap"), (dict(_6=math.nan), "softcap"), (dict(_1=65536), "n_rows"),
])
def test_token_logprobs_refusals(change, text):
    assert text in refused("chn_token_logprobs", with_(SCORES, **change))


@pytest.mark.parametrize("change", [dict(_5=None), dict(_9=None), dict(_10=None), dict(_7=0, _11=None, _12=None), dict(_1=0)])
def test_token_logprobs_optional_arguments(change):
    assert refused("chn_token_logprobs", with_(SCORES, **change)) == "ctx is NULL"


@pytest.mark.parametrize("at", [A[1], A[2], A[3], A[4], A[5], A[1] + 100 * 16 * 512 * 4 - 16, A[3] + 4 * (4 * 32 - 4), A[4] + 16])
def test_attention_into_an_input_is_refused(at):
    assert "overlaps" in refused("chn_paged_causal_attn", with_(CAUSAL, _17=at))
    assert "overlaps" in refused("chn_paged_tree_attn", with_(TREE, _19=at))


def test_attention_into_its_masks_is_refused():
    assert "overlaps" in refused("chn_paged_tree_attn", with_(TREE, _19=A[7] + 4 * (64 * 2 - 4)))


@pytest.mark.parametrize("change", [dict(_8=A[0] + 4 * 3999), dict(_9=A[1] + 12), dict(_10=A[2]), dict(_11=A[0]), dict(_12=A[1]),
                                    dict(_8=A[4]), dict(_10=A[6] + 4 * 79), dict(_12=A[6] + 16)])
def test_scores_into_an_input_or_each_other_are_refused(change):
    assert "overlap" in refused("chn_token_logprobs", with_(SCORES, **change))


def test_scores_behind_the_logits_are_taken():
    # ld counts between rows: behind the last one lies nothing that is read
    assert refused("chn_token_logprobs", with_(SCORES, _3=2000, _8=A[0] + 4 * 7000)) == "ctx is NULL"


def test_oracle_trees():
    none = packed.NO_TOKEN
    #       0 1 2 3     4 (two requests, then one without rows; 0 <- 1 <- 3, 0 <- 2; 5 names itself, 6 a later one)
    parents = [none, 0, 0, 1, none, 1, 5]
    m, c = packed.draft_trees(parents, [0, 4, 7, 7], [10, 3, 9], 8, 1, np.full((8, 1), 77), np.full(8, 88))
    assert m[:, 0].tolist() == [1, 0b11, 0b101, 0b1011, 1, 0b10, 0b100, 77]
    assert c.tolist() == [6, 7, 7, 8, 0, 0, 0, 88]


def test_oracle_trees_longer_than_their_masks():
    n = 40
    m, c = packed.draft_trees([packed.NO_TOKEN] + list(range(n - 1)), [0, n], [50], n, 1, np.zeros((n, 1)), np.zeros(n))
    assert m[31, 0] == 0xFFFFFFFF and c[31] == 41
    assert (m[32:] == 0).all() and (c[32:] == 10).all()


def test_oracle_seen():
    see = lambda *a, **k: packed.seen_by(*a, **k).tolist()  # noqa: E731
    assert see(1, 3, 7, 0) == [0, 1, 2, 3, 4, 5]
    assert see(1, 3, 7, 2) == [4, 5]
    assert see(0, 3, 2, 0) == [] and see(1, 3, 2, 0) == [0]              # more rows than tokens
    assert see(2, 3, 7, 0, mask=[0b101]) == [0, 1, 2, 3, 4, 6]
    assert see(2, 3, 7, 3, mask=[0b101]) == [3, 4, 6]                    # two of its window of three are drafted
    assert see(2, 3, 7, 0, mask=[0b1001]) == [0, 1, 2, 3, 4]             # no fourth drafted token
    assert see(0, 3, 3, 0, mask=[0]) == []


def test_oracle_attention():
    D, rng = 4, np.random.default_rng(0)
    q, kc, vc = rng.standard_normal((5, 2 * D)), rng.standard_normal((16, D)), rng.standard_normal((16, D))
    out, _, _, most = packed.packed_attn(q, kc, vc, [[3, 9], [1, 0]], [0, 1, 4], [1, 6], 4, 4, 2, D, 2, 1.0, 0)
    assert np.allclose(out[0, :D], vc[12]) and np.allclose(out[0, D:], vc[12])           # one key, both heads
    at = [4, 5, 6, 7]
    p = np.exp(kc[at] @ q[1, :D])
    assert np.allclose(out[1, :D], p @ vc[at] / p.sum())                                 # row 1: positions 0 .. 3
    assert (out[4] == 0).all() and most == 6
    bad, _, _, _ = packed.packed_attn(q, kc, vc, [[9, 9], [1, 9]], [0, 1, 4], [1, 6], 4, 4, 2, D, 2, 1.0, 0)
    assert (bad[0] == 0).all() and np.allclose(bad[3, :D], np.exp(kc[at] @ q[3, :D]) @ vc[at] / np.exp(kc[at] @ q[3, :D]).sum())


def test_oracle_logprobs():
    row = [math.log(1), math.log(2), -math.inf, math.log(1), math.nan, packed.LOWEST]
    lp, ent, rank, ids, tops = packed.logprob_row(row, 3, n_top=4)
    assert math.isclose(lp, math.log(0.25)) and rank == 2 and ids == [1, 0, 3, packed.NO_TOKEN]
    assert math.isclose(ent, 1.5 * math.log(2)) and tops[3] == -math.inf and math.isclose(tops[0], math.log(0.5))
    assert packed.logprob_row(row, 2)[0] == -math.inf and packed.logprob_row(row, 2)[2] == packed.NO_TOKEN
    assert packed.logprob_row(row, 6)[:3] == (0.0, ent, packed.NO_TOKEN)
    assert packed.logprob_row(row, 1, T=0.0)[:3] == (0.0, 0.0, 0) and packed.logprob_row(row, 0, T=0.0)[0] == -math.inf
    assert math.isclose(packed.logprob_row(row, 0, T=0.5)[0], math.log(1 / 6))
    assert packed.logprob_row([-math.inf] * 3, 1, n_top=1) == (-math.inf, 0.0, packed.NO_TOKEN, [packed.NO_TOKEN], [-math.inf])
    two = packed.logprob_row([math.inf, 1.0, math.inf], 2, n_top=3)
    assert math.isclose(two[0], math.log(0.5)) and two[3] == [0, 2, 1] and two[4][2] == -math.inf
