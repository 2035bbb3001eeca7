"""The largest batches that one launch of the batched step takes, refused before
a device is needed: a launch has fewer than 2^32 threads."""
import pytest

from test_paged import ATTN, ROPE, refused, with_

MOST = (1 << 24) - 1


# 4 query and 2 KV heads: 8 rows a token, one workgroup of the 16-byte form, two of the other
@pytest.mark.parametrize("change,fits", [
    (dict(_10=MOST), True), (dict(_10=MOST + 1), False), (dict(_10=(1 << 32) - 1), False),
    (dict(_10=MOST // 2, _15=30), True), (dict(_10=MOST // 2 + 1, _15=30), False),
    (dict(_10=MOST // 2, _14=100, _15=100), True), (dict(_10=MOST // 2 + 1, _14=100, _15=100), False),
])
def test_rope_tokens(change, fits):
    text = refused("chn_batch_qkv_rope_at", with_(ROPE, **change))
    assert ("ctx is NULL" if fits else "too many") in text


# n_req and query heads; one query head per KV head keeps kv_dim beside them
@pytest.mark.parametrize("n,heads,fits", [(65536, 255, True), (65536, 256, False), (4096, 4095, True), (4096, 4096, False),
                                          (1, 4096, True)])
def test_attention_rows(n, heads, fits):
    args = with_(ATTN, _7=n, _11=heads, _13=heads * 256, _14=1)
    if fits:
        assert refused("chn_prefix_decode_attn", args) == "ctx is NULL"
    else:
        assert "too many" in refused("chn_prefix_decode_attn", args, -6)
