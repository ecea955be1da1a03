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


def test_queries_on_the_host(gpu):
    """to_host() of what embed returns: float32 [texts, width], also after a larger call."""
    from zcgvs_amd.embedder import DeviceEmbedder
    capi = gpu
    rng = np.random.default_rng(42)
    weights = [rng.integers(-2, 3, s).astype(np.float32) for s in ((20, 8), (8, 8), (8, 8), (5, 8))]
    weights[1][:] = 100.0 * np.eye(8)  # silu(g) = g or 0 to float32's last digit
    model = DeviceEmbedder(*weights, dtype=capi.F32)
    table, gate, up, projection = (w.astype(np.float64) for w in weights)
    for texts in (7, 2):
        ids = rng.integers(0, 20, texts)
        got = model.embed(ids, np.arange(texts + 1)).to_host()
        hidden = np.maximum(table[ids] @ gate.T, 0.0) * (table[ids] @ up.T)
        assert got.shape == (texts, 5) and got.dtype == np.float32
        # values below 2^17 of at most 8 terms, each a few float32 roundings
        assert np.all(np.abs(got - hidden @ projection.T) <= 2.0 ** -18 * (np.abs(hidden) @ np.abs(projection).T) + 1e-30)
