"""Sizes and numbers that the encoder blocks' kernels do not take are refused when the blocks are made, before anything is
allocated; without a GPU."""

import numpy as np
import pytest

from test_embedder_order import recorded  # noqa: F401
from test_encoder_order import _block, _encoder, with_blocks  # noqa: F401


def _heads(head_dim):
    return dict(out=np.ones((8, 4 * head_dim), np.float32), qkv=np.ones((8 * head_dim, 8), np.float32))


@pytest.mark.parametrize("block,more,match", [
    (_heads(129), {}, "at most 128 values, not 129"),
    (dict(distance_bias=np.ones((4, 1027), np.float32)), {}, "at most 512"),
    ({}, dict(eps=-1e-6), "eps and cap"),
    ({}, dict(eps=float("nan")), "eps and cap"),
    ({}, dict(cap=-1.0), "eps and cap"),
    ({}, dict(cap=float("inf")), "eps and cap"),
    ({}, dict(activation=3), "unknown activation"),
    ({}, dict(heads=1028, kv_heads=4), "lie in .1, 1024. and be a multiple of kv_heads"),
])
def test_refused_when_made(capi, with_blocks, block, more, match):  # noqa: F811
    with pytest.raises(ValueError, match=match):
        _encoder(capi, _block(**block), **more)
    assert not with_blocks.made


def test_rows_wider_than_the_norm_takes(capi, with_blocks):  # noqa: F811
    from zcgvs_amd.encoder import EncoderBlocks
    with pytest.raises(ValueError, match="1 to 16384 values"):
        EncoderBlocks([], np.ones(16385, np.float32), heads=4, dtype=capi.F32)
    assert not with_blocks.made


def test_the_largest_are_taken(capi, with_blocks):  # noqa: F811
    _encoder(capi, _block(**_heads(128), distance_bias=np.ones((4, 1025), np.float32)), cap=50.0, eps=0.0,
             activation=capi.ACT_GELU)


@pytest.mark.parametrize("texts,rows,heads", [(1 << 24, 1 << 24, 1), (1, 1 << 28, 1024)])
def test_attention_of_more_workgroups_than_a_launch_takes(capi, texts, rows, heads):
    at = 1 << 20  # an address that nothing reads here
    desc = capi.attention_desc(at, at, at, texts, rows, rows, heads, 8, capi.F16)
    with pytest.raises(ValueError, match="more texts and rows than one launch"):
        capi.attention(desc, at, at, 1 << 50)
    with pytest.raises(ValueError, match="more texts and rows than one launch"):
        capi.attention_gradient(desc, at, at, at, at, at, at, at, 1 << 60)
