"""The embedding model on the device: token ids to hits, a training step, and replay from a graph."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _model(rng, vocab=500, dim=64, hidden=96, width=128, adapters=5, rank=8):
    return dict(table=rng.standard_normal((vocab, dim)), gate=rng.standard_normal((hidden, dim)),
                up=rng.standard_normal((hidden, dim)), projection=rng.standard_normal((width, hidden)) / math.sqrt(hidden),
                down=rng.standard_normal((adapters, rank, hidden)) / math.sqrt(hidden),
                adapter_up=rng.standard_normal((adapters, width, rank)))


def _texts(rng, vocab, texts):
    lengths = rng.integers(0, 40, texts)
    lengths[0], lengths[-1] = 0, 1
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    return rng.integers(0, vocab, offsets[-1]).astype(np.int32), offsets


def _hidden(m, ids, offsets):
    rows = np.zeros((len(offsets) - 1, m["table"].shape[1]))
    for t in range(len(rows)):
        part = [i for i in ids[offsets[t]:offsets[t + 1]] if i != 0]
        if part:
            rows[t] = m["table"][part].mean(axis=0)
    g = rows @ m["gate"].T
    return rows, g / (1.0 + np.exp(-g)) * (rows @ m["up"].T)


def _queries(m, ids, offsets, adapter_ids):
    _, hidden = _hidden(m, ids, offsets)
    queries = hidden @ m["projection"].T
    for t, a in enumerate(adapter_ids):
        if a >= 0:
            queries[t] += hidden[t] @ m["down"][a].T @ m["adapter_up"][a].T
    return queries


def _embedder(capi, m, kind, code):
    from zcgvs_amd.embedder import DeviceEmbedder
    stored = {k: v.astype(kind) for k, v in m.items()}
    model = DeviceEmbedder(stored["table"], stored["gate"], stored["up"], stored["projection"], dtype=code, padding_id=0,
                           adapters=dict(down=stored["down"], up=stored["adapter_up"]))
    return model, {k: v.astype(np.float64) for k, v in stored.items()}


@pytest.mark.parametrize("kind", ["float16", "float32"])
def test_token_ids_to_hits(gpu, kind):
    """The queries that the model leaves on the device find what the formula's queries find."""
    capi = gpu
    rng = np.random.default_rng(21)
    model, m = _embedder(capi, _model(rng), kind, capi.F16 if kind == "float16" else capi.F32)
    corpus = rng.standard_normal((3000, 128)).astype(np.float32)
    d_corpus = capi.DeviceArray.from_host(corpus)
    for texts in (5, 40):  # the larger call grows the model's buffers
        ids, offsets = _texts(rng, 500, texts)
        adapter_ids = rng.integers(-1, 5, texts)
        queries = model.embed(ids, offsets, adapter_ids)
        desc = capi.search_desc(capi.store_desc(d_corpus, 3000, 128, capi.F32), queries, texts, 10, capi.DOT)
        idx, val, _ = capi.search(desc)
        expected = _queries(m, ids, offsets, adapter_ids)
        scores = expected @ corpus.astype(np.float64).T
        # hidden rows of float16 carry 2^-11 each; float32's own sums are far below that
        unit = 2.0 ** -11 if kind == "float16" else 2.0 ** -18
        size = np.abs(expected).max(axis=1, keepdims=True) * np.abs(corpus).sum(axis=1) + 1e-30
        for t in range(texts):
            tolerance = 4 * unit * size[t] + 1e-6
            assert np.all(np.abs(val[t] - scores[t, idx[t]]) <= tolerance[idx[t]])
            if offsets[t + 1] > offsets[t]:
                best = np.sort(scores[t])[::-1][:10]
                assert np.all(np.abs(val[t] - best) <= tolerance.max())


def test_training_step(gpu):
    """A step against the gradients lowers the loss by what they promise."""
    capi = gpu
    rng = np.random.default_rng(22)
    weights = _model(rng, vocab=60, dim=32, hidden=40)
    ids, offsets = _texts(rng, 60, 50)
    target = rng.standard_normal((50, 40))
    model, m = _embedder(capi, weights, "float32", capi.F32)

    def loss(parts):
        return 0.5 * ((_hidden(parts, ids, offsets)[1] - target) ** 2).sum()

    hidden = model.hidden_rows(ids, offsets)
    grads = model.gradient(ids, offsets, (hidden - target).astype(np.float32))
    capi.synchronize()
    grads = {k: v.to_host().astype(np.float64) for k, v in grads.items()}
    slope = sum((g ** 2).sum() for g in grads.values())
    assert np.all(grads["table"][0] == 0.0)  # the padding learns nothing
    # central differences along the gradient: the step's third order and the losses' rounding stay below
    # a thousandth of the slope
    step = 1e-4 / math.sqrt(slope)
    moved = [loss({k: v + sign * step * grads.get(k, 0.0) for k, v in m.items()}) for sign in (1, -1)]
    assert abs((moved[0] - moved[1]) / (2 * step) - slope) <= 1e-3 * slope


def test_graph_replays(gpu):
    """The three operators and both gradients recorded into a graph give the eager call's bits every time."""
    capi = gpu
    rng = np.random.default_rng(23)
    texts, vocab, dim, hidden, width = 300, 9000, 64, 128, 96
    ids, offsets = _texts(rng, vocab, texts)
    host = [rng.standard_normal(s).astype(np.float16) * np.float16(0.1) for s in
            ((vocab, dim), (hidden, dim), (hidden, dim), (width, hidden), (7, 16, hidden), (7, width, 16), (texts, hidden))]
    table, gate, up, projection, down, adapter_up, d_hidden = (capi.DeviceArray.from_host(a) for a in host)
    d_ids, d_offsets = capi.DeviceArray.from_host(ids), capi.DeviceArray.from_host(offsets)
    adapter_ids = capi.DeviceArray.from_host(rng.integers(-1, 7, texts).astype(np.int32))
    rows, out = capi.DeviceArray((texts, dim), np.float16), capi.DeviceArray((texts, hidden), np.float16)
    queries = capi.DeviceArray((texts, width), np.float32)
    lookup = capi.embedding_desc(table, vocab, dim, capi.F16, d_ids, len(ids), bag_offsets=d_offsets, bag_count=texts,
                                 reduce=capi.EMBEDDING_MEAN)
    gated = capi.gated_desc(rows, texts, dim, gate, up, hidden, capi.F16, capi.ACT_GELU)
    adapted = capi.adapted_desc(out, texts, hidden, projection, width, capi.F16, down=down, up=adapter_up,
                                adapter_count=7, max_rank=16, adapter_ids=adapter_ids)
    sizes = [capi.adapted_projection_workspace_bytes(adapted), capi.gated_gradient_workspace_bytes(gated),
             capi.embedding_gradient_workspace_bytes(lookup)]
    spaces = [capi.DeviceArray(s, np.uint8) for s in sizes]
    grads = [capi.DeviceArray(s, np.float16) for s in ((texts, dim), (hidden, dim), (hidden, dim))]
    table_grad = capi.DeviceArray((vocab, dim), np.float32)
    results = [rows, out, queries, *grads, table_grad]

    def record(stream):
        capi.embedding_lookup(lookup, rows, capi.F16, stream=stream)
        capi.gated_projection(gated, out, stream=stream)
        capi.adapted_projection(adapted, queries, capi.F32, spaces[0], sizes[0], stream=stream)
        capi.gated_gradient(gated, d_hidden, *grads, spaces[1], sizes[1], stream=stream)
        capi.embedding_gradient(lookup, grads[0], capi.F16, table_grad, capi.F32, spaces[2], sizes[2], stream=stream)

    record(None)
    capi.synchronize()
    expected = [r.to_host() for r in results]
    assert all(np.all(np.isfinite(e)) for e in expected)
    stream = capi.Stream()
    graph = capi.Graph(stream, lambda: record(stream))
    for _ in range(4):
        for r in results:  # the program's own work between the replays
            capi.call("zcgvs_fill_u32", r.ptr, 0x7FC07FC0, r.nbytes // 4, None)
        capi.synchronize()
        graph.launch(stream)
        stream.synchronize()
        assert all(np.array_equal(r.to_host(), e) for r, e in zip(results, expected))
