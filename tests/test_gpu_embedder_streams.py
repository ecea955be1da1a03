"""Calls of one DeviceEmbedder behind each other, without a wait, on one stream and on changing ones."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _batch(rng, vocab, texts, hidden):
    offsets = np.concatenate([[0], np.cumsum(rng.integers(0, 60, texts))]).astype(np.int64)
    return (rng.integers(0, vocab, offsets[-1]).astype(np.int32), offsets,
            (rng.standard_normal((texts, hidden)) * 0.1).astype(np.float16))


@pytest.mark.parametrize("streams", [1, 2])
def test_calls_without_a_wait_between(gpu, streams):
    """The bits of the same calls on the null stream, each waited for."""
    from zcgvs_amd.embedder import DeviceEmbedder
    capi = gpu
    rng = np.random.default_rng(41)
    vocab, dim, hidden, width = 20_000, 384, 1024, 256
    weights = [(rng.standard_normal(s) * 0.1).astype(np.float16) for s in
               ((vocab, dim), (hidden, dim), (hidden, dim), (width, hidden))]
    model = DeviceEmbedder(*weights, dtype=capi.F16, padding_id=0)
    batches = [_batch(rng, vocab, texts, hidden) for texts in (2000, 1500, 2000)]
    expected = []
    for ids, offsets, d in batches:
        grads = model.gradient(ids, offsets, d)
        capi.synchronize()
        expected.append({name: g.to_host() for name, g in grads.items()})
    on = [capi.Stream() for _ in range(streams)]
    for _ in range(3):
        got = []
        for i, (ids, offsets, d) in enumerate(batches):
            got.append(model.gradient(ids, offsets, d, stream=on[i % streams]))
            model.embed(*batches[0][:2], stream=on[i % streams])
        capi.synchronize()
        for e, g in zip(expected, got):
            assert all(np.array_equal(g[name].to_host(), e[name]) for name in e)
