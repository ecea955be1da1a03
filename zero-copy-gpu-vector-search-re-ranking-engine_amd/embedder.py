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

With `encoder`, an EncoderBlocks, each token's row (table[id] times `scale`) goes through its blocks, where it meets the
other tokens of its text, before the mean is taken; padding and ids out of range are left out of the texts first.
"""

from __future__ import annotations

import numpy as np

from . import capi

_STORAGE = {capi.F32: np.dtype(np.float32), capi.F16: np.dtype(np.float16), capi.BF16: np.dtype(np.uint16)}


def _refuse(message):
    raise ValueError(f"zcgvs embedder: {message}")


def _matrix(name, values, shape, element):
    """A host array whose address goes to the kernels: its shape (None: any length) and type have to be right."""
    values = np.asarray(values)
    if values.dtype != element:
        _refuse(f"{name} must hold {element}, not {values.dtype}")
    if values.ndim != len(shape) or any(want is not None and have != want for have, want in zip(values.shape, shape)):
        _refuse(f"{name} has shape {values.shape}, not {shape}")
    return values


def _whole(name, values, kind):
    """A list of whole numbers as an array of `kind`; none of them may change on the way."""
    values = np.asarray(values)
    if values.ndim != 1 or (values.size and values.dtype.kind not in "iu"):
        _refuse(f"{name} must be a list of whole numbers")
    limits = np.iinfo(kind)
    if values.size and (values.min() < limits.min or values.max() > limits.max):
        _refuse(f"{name} must fit {np.dtype(kind)}")
    return values.astype(kind)


class DeviceEmbedder:
    """Weights and work buffers of the model; host arrays in, device arrays out.

    table [vocab, dim], gate and up [hidden, dim] and projection [width, hidden] hold `dtype` (bfloat16 as
    uint16 bit patterns); arrays of other types, shapes or sizes are refused. adapters: None, or a dict with down [n, rank, hidden], up [n, width, rank] and
    optionally ranks [n] and scales [n]."""

    def __init__(self, table, gate, up, projection, *, dtype, scale=1.0, padding_id=-1, activation=capi.ACT_SILU,
                 adapters=None, encoder=None):
        self.dtype, self.scale, self.padding_id, self.activation = dtype, scale, padding_id, activation
        if dtype not in _STORAGE:
            _refuse("dtype must be F32, F16 or BF16")
        self._element = element = _STORAGE[dtype]
        table = _matrix("table", table, (None, None), element)
        self.vocab, self.dim = table.shape
        gate = _matrix("gate", gate, (None, self.dim), element)
        self.hidden = gate.shape[0]
        up = _matrix("up", up, (self.hidden, self.dim), element)
        projection = _matrix("projection", projection, (None, self.hidden), element)
        self.width = projection.shape[0]
        if encoder is not None and (encoder.dim != self.dim or encoder.dtype != dtype):
            _refuse(f"the encoder's rows are [{encoder.dim}] of dtype {encoder.dtype}, not [{self.dim}] of {dtype}")
        self.encoder = encoder
        parts = {}
        if adapters is not None:
            if adapters.get("down") is None or adapters.get("up") is None:
                _refuse("adapters need down and up")
            parts["down"] = _matrix("down", adapters["down"], (None, None, self.hidden), element)
            count, rank = parts["down"].shape[:2]
            parts["up"] = _matrix("the adapters' up", adapters["up"], (count, self.width, rank), element)
            if adapters.get("ranks") is not None:
                parts["ranks"] = _whole("ranks", adapters["ranks"], np.int32)
            if adapters.get("scales") is not None:
                parts["scales"] = np.asarray(adapters["scales"], np.float32)
            for name in ("ranks", "scales"):
                if name in parts and parts[name].shape != (count,):
                    _refuse(f"one of {name} for each adapter")
        self.table, self.gate, self.up, self.projection = map(capi.DeviceArray.from_host, (table, gate, up, projection))
        self._adapters = {name: capi.DeviceArray.from_host(values) for name, values in parts.items()}
        if parts:
            self._adapters.update(adapter_count=count, max_rank=rank)
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
        """A work buffer that grows and is kept, as an array of `shape` and `kind`."""
        need = int(np.prod(shape, dtype=np.int64)) * np.dtype(kind).itemsize
        held = self._buffers.get(name)
        if held is None or held.nbytes < need:
            capi.synchronize()  # earlier calls may still use the smaller one
            held = self._buffers[name] = capi.DeviceArray(max(need, 1), np.uint8)
        return held.view(shape, kind)

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

    @staticmethod
    def _lists(ids, offsets):
        """The checked ids and offsets: texts follow each other within the ids."""
        ids, offsets = _whole("ids", ids, np.int32), _whole("offsets", offsets, np.int64)
        if offsets.size == 0 or offsets[0] < 0 or offsets[-1] > ids.size or np.any(offsets[1:] < offsets[:-1]):
            _refuse("offsets must ascend from 0 or more to at most the number of ids")
        return ids, offsets

    def _without_padding(self, ids, offsets):
        """The tokens of the texts that count, one text directly behind the other."""
        ids, offsets = ids[offsets[0]:offsets[-1]], offsets - offsets[0]
        held = (ids >= 0) & (ids < self.vocab) & (ids != self.padding_id)
        return ids[held], np.concatenate([[0], np.cumsum(held, dtype=np.int64)])[offsets]

    def _encode(self, d_ids, d_offsets, d_order, texts, tokens, stream, keep):
        """The token rows through the encoder, and the descriptors of their lookup and of their mean by text."""
        lookup = capi.embedding_desc(self.table, self.vocab, self.dim, self.dtype, d_ids, tokens, scale=self.scale)
        x = self._buffer("token rows", (tokens, self.dim), self._element)
        capi.embedding_lookup(lookup, x, self.dtype, stream=stream)
        encoded, kept = self.encoder.forward(self._buffer, x, d_offsets, texts, tokens, stream, keep)
        pooled = capi.embedding_desc(encoded, tokens, self.dim, self.dtype, d_order, tokens, bag_offsets=d_offsets,
                                     bag_count=texts, reduce=capi.EMBEDDING_MEAN)
        return pooled, dict(lookup=lookup, kept=kept, tokens=tokens)

    def _forward(self, ids, offsets, stream, keep=False, **more):
        """The lookup (with an encoder: the mean of its rows) and the gated block; `more`: further host arrays of the
        call, name=(values, type), copied beside the ids."""
        if self.encoder is not None:
            ids, offsets = self._without_padding(ids, offsets)
            more = dict(more, order=(np.arange(len(ids)), np.int32))
        texts, tokens = len(offsets) - 1, len(ids)
        self._enter(stream)
        d_ids, d_offsets = self._upload("ids", ids, np.int32), self._upload("offsets", offsets, np.int64)
        uploaded = {name: self._upload(name, *values) for name, values in more.items()}
        self._settle()
        encoded = None
        if self.encoder is not None and tokens:
            lookup, encoded = self._encode(d_ids, d_offsets, uploaded["order"], texts, tokens, stream, keep)
        else:
            lookup = self._lookup_desc(d_ids, d_offsets, texts, tokens)
        rows = self._buffer("rows", (texts, self.dim), self._element)
        hidden = self._buffer("hidden", (texts, self.hidden), self._element)
        capi.embedding_lookup(lookup, rows, self.dtype, stream=stream)
        gated = capi.gated_desc(rows, texts, self.dim, self.gate, self.up, self.hidden, self.dtype, self.activation)
        capi.gated_projection(gated, hidden, stream=stream)
        return lookup, gated, hidden, dict(uploaded, encoded=encoded)

    def embed(self, ids, offsets, adapter_ids=None, stream=None) -> capi.DeviceArray:
        """Queries of the texts ids[offsets[t]:offsets[t + 1]], each through adapter adapter_ids[t] (-1: none):
        float32 [texts, width]. The array belongs to the model and holds until the next call."""
        ids, offsets = self._lists(ids, offsets)
        texts = len(offsets) - 1
        more = {}
        if adapter_ids is not None:
            if not self._adapters:
                _refuse("the model has no adapters")
            adapter_ids = _whole("adapter_ids", adapter_ids, np.int32)
            if len(adapter_ids) != texts:
                _refuse("one adapter id per text")
            more = dict(adapter_ids=(adapter_ids, np.int32))
        _, _, hidden, uploaded = self._forward(ids, offsets, stream, **more)
        extra = dict(self._adapters, adapter_ids=uploaded["adapter_ids"]) if more else {}
        desc = capi.adapted_desc(hidden, texts, self.hidden, self.projection, self.width, self.dtype, **extra)
        size = capi.adapted_projection_workspace_bytes(desc)
        workspace = self._buffer("workspace", (size,), np.uint8)
        queries = self._buffer("queries", (texts, self.width), np.float32)
        capi.adapted_projection(desc, queries, capi.F32, workspace, size, stream=stream)
        return queries

    def hidden_rows(self, ids, offsets, stream=None) -> np.ndarray:
        """The hidden rows on the host, as stored (for training, where a loss is formed from them)."""
        ids, offsets = self._lists(ids, offsets)
        _, _, hidden, _ = self._forward(ids, offsets, stream)
        out = np.empty((len(offsets) - 1, self.hidden), dtype=self._element)
        if out.nbytes:
            capi.call("zcgvs_memcpy_d2h", out.ctypes.data, hidden.ptr, out.nbytes, getattr(stream, "handle", stream))
        self._settle()
        return out

    def gradient(self, ids, offsets, hidden_gradient, stream=None) -> dict:
        """The gradients of the table (float32) and of gate and up (their type), as device arrays, from the
        gradient of the hidden rows (host [texts, hidden], of the model's type: no other is converted). With an
        encoder also `encoder`: dict(blocks=[{name: array}], final_norm=array), None where no text has a token."""
        ids, offsets = self._lists(ids, offsets)
        texts = len(offsets) - 1
        hidden_gradient = _matrix("hidden_gradient", hidden_gradient, (texts, self.hidden), self._element)
        lookup, gated, _, uploaded = self._forward(ids, offsets, stream, keep=True,
                                                   hidden_gradient=(hidden_gradient, self._element))
        d_hidden = uploaded["hidden_gradient"]
        rows = self._buffer("rows_gradient", (texts, self.dim), self._element)
        gate, up = (capi.DeviceArray((self.hidden, self.dim), self._element) for _ in range(2))
        size = capi.gated_gradient_workspace_bytes(gated)
        capi.gated_gradient(gated, d_hidden, rows, gate, up, self._buffer("gated_workspace", (size,), np.uint8), size,
                            stream=stream)
        table, more = capi.DeviceArray((self.vocab, self.dim), np.float32), {}
        if self.encoder is not None:
            more = dict(encoder=None)
        if uploaded["encoded"] is not None:
            saved, tokens = uploaded["encoded"], uploaded["encoded"]["tokens"]
            mean = self._buffer("encoded gradient", (tokens, self.dim), self._element)
            size = capi.embedding_gradient_workspace_bytes(lookup)
            capi.embedding_gradient(lookup, rows, self.dtype, mean, self.dtype,
                                    self._buffer("mean workspace", (size,), np.uint8), size, stream=stream)
            rows, more["encoder"] = self.encoder.gradient(self._buffer, saved["kept"], mean, tokens, stream)
            lookup = saved["lookup"]
        size = capi.embedding_gradient_workspace_bytes(lookup)
        capi.embedding_gradient(lookup, rows, self.dtype, table, capi.F32,
                                self._buffer("table_workspace", (size,), np.uint8), size, stream=stream)
        return dict(table=table, gate=gate, up=up, **more)
