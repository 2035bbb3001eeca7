"""Hand-worked cases of the oracle's RoPE at own clocks and of its attention
over a prefix and own blocks (CPU)."""
import numpy as np
import pytest

from oracle import paged


# ---- RoPE: heads of 8, 4 of them rotated in pairs (0, 2) and (1, 3), theta 16: a pair turns by clock and clock / 4
def test_rope_turns_pairs_by_their_angles():
    q = np.zeros((1, 1, 8))
    q[0, 0, 0], q[0, 0, 1] = 2.0, 2.0                            # mean square 1, norm (eps 0) leaves it
    w = np.array([1.0, 3.0, 1, 1, 1, 1, 1, 1])
    out, _, _ = paged.rope_at(q, np.ones((1, 1, 8)), np.ones((1, 1, 8)), w, np.ones(8), np.zeros((2, 8)), np.zeros((2, 8)),
                              [2], [0], 4, 16.0, 0.0)
    # the weight comes before the turn
    want = [2 * np.cos(2), 6 * np.cos(0.5), 2 * np.sin(2), 6 * np.sin(0.5), 0, 0, 0, 0]
    assert np.allclose(out[0, 0], want, rtol=0, atol=1e-15)


def test_rope_second_of_a_pair_turns_back():
    q = np.zeros((1, 1, 4))
    q[0, 0, 2] = 2.0
    out, _, _ = paged.rope_at(q, np.ones((1, 1, 4)), np.ones((1, 1, 4)), np.ones(4), np.ones(4), np.zeros((1, 4)),
                              np.zeros((1, 4)), [1], [0], 4, 100.0, 0.0)
    assert np.allclose(out[0, 0], [-2 * np.sin(1), 0, 2 * np.cos(1), 0], rtol=0, atol=1e-15)


def test_rope_writes_k_and_v_at_the_slots_only():
    k = np.array([[[3.0, 4.0]], [[1.0, 1.0]], [[5.0, 0.0]]])
    v = np.array([[[6.0, 8.0]], [[2.0, 2.0]], [[7.0, 0.0]]])
    old = np.full((3, 2), 9.0)
    _, kc, vc = paged.rope_at(np.ones((3, 1, 2)), k, v, np.ones(2), np.array([2.0, 1.0]), old, old, [0, 5, 6], [2, 3, 0xFFFFFFFF],
                              0, 1e4, 0.0)
    rms = np.sqrt(12.5)
    assert np.allclose(kc, [[9, 9], [9, 9], [6 / rms, 4 / rms]], rtol=1e-15)
    assert np.allclose(vc, [[9, 9], [9, 9], [6 / 50 ** 0.5, 8 / 50 ** 0.5]], rtol=1e-15)      # unit norm, no weight
    assert (old == 9).all()


def test_rope_far_clocks_keep_their_turn():
    # theta 1 turns the pair by the clock itself
    q = np.ones((2, 1, 2))
    clocks = [355, 103993 * 2]                                    # near 113 pi and 2 * 33102 pi
    out, _, _ = paged.rope_at(q, q, q, np.ones(2), np.ones(2), np.zeros((2, 2)), np.zeros((2, 2)), clocks, [0, 1], 2, 1.0, 0.0)
    assert np.allclose(out[0, 0], [-1, -1], atol=4e-5) and np.allclose(out[1, 0], [1, 1], atol=5e-5)


def test_rope_norm_has_its_epsilon():
    out, _, _ = paged.rope_at(np.full((1, 1, 2), 3.0), np.ones((1, 1, 2)), np.ones((1, 1, 2)), np.ones(2), np.ones(2),
                              np.zeros((1, 2)), np.zeros((1, 2)), [0], [0], 2, 1e4, 16.0)
    assert np.allclose(out, 3 / 5.0)


# ---- attention: heads of 2, blocks of 2 slots
def attend(q, kc, vc, prefix, tables, lens, num_q, gqa, scale=1.0, n_blocks=None):
    kc = np.asarray(kc, np.float64)
    return paged.prefix_attn(np.asarray(q, np.float64), kc, np.asarray(vc, np.float64), prefix, tables, lens, 2,
                             n_blocks or len(kc) // 2, num_q, 2, gqa, scale)


KC = [[1, 0], [0, 1], [2, 0], [0, 2], [1, 1], [-1, -1]]
VC = [[1, 2], [3, 4], [5, 6], [7, 8], [9, 10], [11, 12]]


def test_attention_of_one_key_is_its_value():
    out, big, absum = attend([[2.0, -1.0]], KC, VC, [], [[2, 0]], [1], 1, 1)
    assert np.array_equal(out, [[9, 10]]) and big == 1 and absum == 3


def test_attention_of_none_is_zero():
    out, big, absum = attend([[2.0, 1.0], [1.0, 1.0]], KC, VC, [1], [[1, 0], [1, 0]], [0, 1], 1, 1)
    assert np.array_equal(out, [[0, 0], [5, 6]])
    out, _, _ = attend([[2.0, 1.0]], KC, VC, [], [[9]], [2], 1, 1)           # a bad block holds no key
    assert np.array_equal(out, [[0, 0]])


def test_attention_of_equal_scores_is_the_mean():
    out, _, _ = attend([[0.0, 0.0]], KC, VC, [], [[0, 2]], [3], 1, 1)
    assert np.allclose(out, [[(1 + 3 + 9) / 3, (2 + 4 + 10) / 3]])


@pytest.mark.parametrize("scale", [1.0, 0.5, -2.0])
def test_attention_weights_prefix_and_own_keys(scale):
    # prefix: block 2 (keys 4 and 5); the request's own: block 0 (key 0); the table's first entry is not read
    q = [1.0, 3.0]
    s = scale * np.array([4.0, -4.0, 1.0])
    w = np.exp(s) / np.exp(s).sum()
    out, big, absum = attend([q], KC, VC, [2], [[77, 0]], [3], 1, 1, scale)
    assert np.allclose(out, [w @ np.array([[9, 10], [11, 12], [1, 2]], float)])
    assert big == 4 * abs(scale) and absum == 4 * abs(scale)


def test_query_heads_read_their_groups_kv_head():
    kc = np.arange(16.0).reshape(2, 8)                           # one block, two KV heads behind each other, and padding
    vc = 100 + np.arange(16.0).reshape(2, 8)
    out, _, _ = attend(np.zeros((1, 8)), kc, vc, [], [[0]], [2], 4, 2)
    h0, h1 = vc[:, 0:2].mean(0), vc[:, 2:4].mean(0)
    assert np.allclose(out, [np.concatenate([h0, h0, h1, h1])])
