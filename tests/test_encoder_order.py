"""The order of an embedder's calls over streams with encoder blocks, and what the blocks refuse, without a GPU: the
library's calls are recorded instead of made."""

import numpy as np
import pytest

import test_embedder_order
from test_embedder_order import GRADIENT, IDS, OFFSETS, Stream, _calls, _weights, recorded  # noqa: F401


@pytest.fixture
def with_blocks(capi, recorded, monkeypatch):  # noqa: F811
    """The recorder with the blocks' operators among the kernels."""
    monkeypatch.setattr(test_embedder_order, "KERNELS", test_embedder_order.KERNELS + (
        "zcgvs_residual_norm", "zcgvs_linear", "zcgvs_attention", "zcgvs_residual_norm_gradient", "zcgvs_linear_gradient",
        "zcgvs_attention_gradient"))
    return recorded


def _block(**change):
    shapes = dict(norm1=8, qkv=(32, 8), out=(8, 16), norm2=8, gate=(12, 8), up=(12, 8), down=(8, 12))
    block = {name: np.ones(shape, np.float32) for name, shape in shapes.items()}
    return dict(block, **change)


def _encoder(capi, *blocks, **more):
    from zcgvs_amd.encoder import EncoderBlocks
    return EncoderBlocks(blocks, np.ones(8, np.float32), **dict(dict(heads=4, kv_heads=2, dtype=capi.F32), **more))


def _model(capi, encoder):
    from zcgvs_amd.embedder import DeviceEmbedder
    adapters = dict(down=np.ones((3, 4, 12), np.float32), up=np.ones((3, 10, 4), np.float32))
    return DeviceEmbedder(*_weights().values(), dtype=capi.F32, padding_id=5, adapters=adapters, encoder=encoder)


@pytest.mark.parametrize("streams", [(7, 7), (7, 9), (None, 7), (7, None)])
def test_calls_follow_each_other_without_a_wait(capi, with_blocks, streams):
    model = _model(capi, _encoder(capi, _block(), _block(qkv_bias=np.ones(32, np.float32),
                                                         distance_bias=np.ones((4, 7), np.float32))))
    first, second = (None if s is None else Stream(s) for s in streams)
    for a in range(4):
        for b in range(4):
            _calls(model, first)[a]()
            _calls(model, second)[b]()
    made = with_blocks.made
    assert made.count("zcgvs_attention") == 2 * made.count("zcgvs_gated_projection") // 3 > 0
    assert made.count("zcgvs_attention_gradient") > 0


def test_a_text_takes_its_own_tokens_alone(capi, with_blocks):
    model = _model(capi, _encoder(capi, _block()))
    ids, offsets = model._without_padding(np.array([9, 5, 1, 2, 5, -1, 50, 3, 4, 8], np.int32), np.array([1, 4, 4, 7, 9]))
    assert ids.tolist() == [1, 2, 3, 4] and offsets.tolist() == [0, 2, 2, 2, 4]
    with_blocks.made.clear()
    model.embed([5, 5], [0, 1, 2])  # no token at all: the plain lookup gives rows of zeros
    assert "zcgvs_attention" not in with_blocks.made and "zcgvs_adapted_projection" in with_blocks.made
    model.gradient([5, 5], [0, 1, 2], GRADIENT)
    assert model.embed([], [0]).shape == (0, 10)


@pytest.mark.parametrize("change,match", [
    (dict(qkv=None), "without .'qkv'"),
    (dict(query=np.ones(8, np.float32)), "block's .'query'"),
    (dict(norm1=np.ones(9, np.float32)), "norm1 has shape"),
    (dict(qkv=np.ones((33, 8), np.float32)), "qkv has shape"),
    (dict(out=np.ones((8, 18), np.float32)), "heads . head_dim columns"),
    (dict(out=np.ones((8, 0), np.float32)), "heads . head_dim columns"),
    (dict(gate=np.ones((12, 8), np.float16)), "gate must hold float32"),
    (dict(up=np.ones((11, 8), np.float32)), "up has shape"),
    (dict(down=np.ones((8, 13), np.float32)), "down has shape"),
    (dict(qkv_bias=np.ones(31, np.float32)), "qkv_bias has shape"),
    (dict(distance_bias=np.ones((3, 7), np.float32)), "distance_bias has shape"),
    (dict(distance_bias=np.ones((4, 6), np.float32)), "2 max_distance . 1"),
])
def test_blocks_that_do_not_fit(capi, with_blocks, change, match):
    with pytest.raises(ValueError, match=match):
        _encoder(capi, _block(**change))
    assert not with_blocks.made  # refused before anything is allocated


def test_encoders_that_do_not_fit(capi, with_blocks):
    with pytest.raises(ValueError, match="F32, F16 or BF16"):
        _encoder(capi, _block(), dtype=capi.I8)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        _encoder(capi, _block(), kv_heads=3)
    with pytest.raises(ValueError, match="one head_dim"):
        _encoder(capi, _block(), _block(out=np.ones((8, 32), np.float32), qkv=np.ones((64, 8), np.float32)))
    with pytest.raises(ValueError, match="slopes has shape"):
        _encoder(capi, _block(), slopes=np.ones(3, np.float32))
    from zcgvs_amd.embedder import DeviceEmbedder
    weights = _weights()
    weights.update(table=np.ones((50, 6), np.float32), gate=np.ones((12, 6), np.float32), up=np.ones((12, 6), np.float32))
    with pytest.raises(ValueError, match="encoder's rows"):
        DeviceEmbedder(*weights.values(), dtype=capi.F32, encoder=_encoder(capi, _block()))
