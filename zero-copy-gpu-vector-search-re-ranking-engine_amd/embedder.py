"""A small text-embedding model on the device, from token ids to the queries of a search.

    rows    = mean over each text's tokens of table[id], times `scale`     (embedding_lookup)
    hidden  = act(rows gate^T) * (rows up^T)                               (gated_projection)
    queries = hidden projection^T + the text's low-rank adapter            (adapted_projection)

`queries` is float32 [texts, width] on the device: a SearchDesc takes its address as it is, so nothing
travels to the host between the token ids and the hits:

    model = DeviceEmbedder(table, gate, up, projection, dtype=capi.F16, padding_id=0)
    queries = model.embed(ids, offsets, adapter_ids)
    desc = capi.search_desc(corpus, queries, len(offsets) - 1, k, capi.DOT)

With `stream`, a call's copies and kernels run on that stream (the caller waits for it before another stream reads
what the call returns); calls may follow each other without a wait, also on changing streams.

The reference's QueryEmbedder (include/zcgvs/embed/query_embedder.hpp:8-15) returns one text's vector on
the host instead. `gradient` gives what training the table and the gated block needs.
"""

from __future__ import annotations

import numpy as np

from . import capi


class DeviceEmbedder:
    """Weights and work buffers of the model; host arrays in, device arrays out.

    table [vocab, dim], gate and up [hidden, dim] and projection [width, hidden] hold `dtype` (bfloat16 as
    uint16 bit patterns). adapters: None, or a dict with down [n, rank, hidden], up [n, width, rank] and
    optionally ranks [n] and scales [n]."""

    def __init__(self, table, gate, up, projection, *, dtype, scale=1.0, padding_id=-1, activation=capi.ACT_SILU,
                 adapters=None):
        self.dtype, self.scale, self.padding_id, self.activation = dtype, scale, padding_id, activation
        self.vocab, self.dim = table.shape
        self.hidden, self.width = gate.shape[0], projection.shape[0]
        if gate.shape != up.shape or gate.shape[1] != self.dim or projection.shape[1] != self.hidden:
            raise ValueError("zcgvs embedder: the weights' shapes do not match")
        self._element = table.dtype
        self.table, self.gate, self.up, self.projection = map(capi.DeviceArray.from_host, (table, gate, up, projection))
        self._adapters = {}
        if adapters is not None:
            count, rank = adapters["down"].shape[:2]
            if adapters["down"].shape[2] != self.hidden or adapters["up"].shape != (count, self.width, rank):
                raise ValueError("zcgvs embedder: the adapters' shapes do not match")
            self._adapters = dict(adapter_count=count, max_rank=rank)
            for name, kind in (("down", None), ("up", None), ("ranks", np.int32), ("scales", np.float32)):
                if adapters.get(name) is not None:
                    values = adapters[name] if kind is None else np.asarray(adapters[name], kind)
                    self._adapters[name] = capi.DeviceArray.from_host(values)
        self._buffers = {}
        self._stream = None  # of the last call
        self._host = []      # arrays whose copies may be on their way

    def _enter(self, stream):
        """A call's copies and kernels go to its stream, in order behind those of the calls before it on that
        stream. The buffers are shared by all calls, so one on another stream waits for the last one's."""
        if getattr(stream, "handle", stream) != getattr(self._stream, "handle", self._stream):
            capi.synchronize()
        self._stream = stream  # kept: a destroyed stream's handle could come back as another stream's

    def _buffer(self, name, shape, kind):
        """A work buffer that grows and is kept; `shape` of it is used."""
        need = int(np.prod(shape, dtype=np.int64)) * np.dtype(kind).itemsize
        held = self._buffers.get(name)
        if held is None or held.nbytes < need:
            capi.synchronize()  # earlier calls may still use the smaller one
            held = self._buffers[name] = capi.DeviceArray(max(need, 1), np.uint8)
        return held

    def _lookup_desc(self, ids, offsets, texts, tokens):
        return capi.embedding_desc(self.table, self.vocab, self.dim, self.dtype, ids, tokens, bag_offsets=offsets,
                                   bag_count=texts, reduce=capi.EMBEDDING_MEAN, padding_id=self.padding_id,
                                   scale=self.scale)

    def _upload(self, name, values, kind):
        """Starts the copy of a host array on the call's stream; _settle() waits for it."""
        values = np.ascontiguousarray(values, dtype=kind)
        buffer = self._buffer(name, values.shape, kind)
        if values.nbytes:
            self._host.append(values)
            capi.call("zcgvs_memcpy_h2d", buffer.ptr, values.ctypes.data, values.nbytes,
                      getattr(self._stream, "handle", self._stream))
        return buffer

    def _settle(self):
        """Waits for the call's stream alone."""
        capi.call("zcgvs_stream_synchronize", getattr(self._stream, "handle", self._stream))
        self._host.clear()

    def _forward(self, ids, offsets, stream, **more):
        """The lookup and the gated block; `more`: further host arrays of the call, name=(values, type), copied
        beside the ids."""
        texts, tokens = len(offsets) - 1, len(ids)
        self._enter(stream)
        d_ids, d_offsets = self._upload("ids", ids, np.int32), self._upload("offsets", offsets, np.int64)
        uploaded = {name: self._upload(name, *values) for name, values in more.items()}
        self._settle()
        lookup = self._lookup_desc(d_ids, d_offsets, texts, tokens)
        rows = self._buffer("rows", (texts, self.dim), self._element)
        hidden = self._buffer("hidden", (texts, self.hidden), self._element)
        capi.embedding_lookup(lookup, rows, self.dtype, stream=stream)
        gated = capi.gated_desc(rows, texts, self.dim, self.gate, self.up, self.hidden, self.dtype, self.activation)
        capi.gated_projection(gated, hidden, stream=stream)
        return lookup, gated, hidden, uploaded

    def embed(self, ids, offsets, adapter_ids=None, stream=None) -> capi.DeviceArray:
        """Queries of the texts ids[offsets[t]:offsets[t + 1]], each through adapter adapter_ids[t] (-1: none).
        The array belongs to the model and holds until the next call."""
        texts = len(offsets) - 1
        more = {}
        if adapter_ids is not None:
            if not self._adapters:
                raise ValueError("zcgvs embedder: the model has no adapters")
            if len(adapter_ids) != texts:
                raise ValueError("zcgvs embedder: one adapter id per text")
            more = dict(adapter_ids=(adapter_ids, np.int32))
        _, _, hidden, uploaded = self._forward(ids, offsets, stream, **more)
        extra = dict(self._adapters, **uploaded) if uploaded else {}
        desc = capi.adapted_desc(hidden, texts, self.hidden, self.projection, self.width, self.dtype, **extra)
        size = capi.adapted_projection_workspace_bytes(desc)
        workspace = self._buffer("workspace", (size,), np.uint8)
        queries = self._buffer("queries", (texts, self.width), np.float32)
        capi.adapted_projection(desc, queries, capi.F32, workspace, size, stream=stream)
        return queries

    def hidden_rows(self, ids, offsets, stream=None) -> np.ndarray:
        """The hidden rows on the host, as stored (for training, where a loss is formed from them)."""
        _, _, hidden, _ = self._forward(ids, offsets, stream)
        out = np.empty((len(offsets) - 1, self.hidden), dtype=self._element)
        if out.nbytes:
            capi.call("zcgvs_memcpy_d2h", out.ctypes.data, hidden.ptr, out.nbytes, getattr(stream, "handle", stream))
        self._settle()
        return out

    def gradient(self, ids, offsets, hidden_gradient, stream=None) -> dict:
        """The gradients of the table (float32) and of gate and up (their type), as device arrays, from the
        gradient of the hidden rows (host, of the model's type)."""
        texts, tokens = len(offsets) - 1, len(ids)
        lookup, gated, _, uploaded = self._forward(ids, offsets, stream, hidden_gradient=(hidden_gradient, self._element))
        d_hidden = uploaded["hidden_gradient"]
        rows = self._buffer("rows_gradient", (texts, self.dim), self._element)
        gate, up = (capi.DeviceArray((self.hidden, self.dim), self._element) for _ in range(2))
        size = capi.gated_gradient_workspace_bytes(gated)
        capi.gated_gradient(gated, d_hidden, rows, gate, up, self._buffer("gated_workspace", (size,), np.uint8), size,
                            stream=stream)
        table = capi.DeviceArray((self.vocab, self.dim), np.float32)
        size = capi.embedding_gradient_workspace_bytes(lookup)
        capi.embedding_gradient(lookup, rows, self.dtype, table, capi.F32,
                                self._buffer("table_workspace", (size,), np.uint8), size, stream=stream)
        return dict(table=table, gate=gate, up=up)
