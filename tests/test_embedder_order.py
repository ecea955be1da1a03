"""The order of a DeviceEmbedder's copies and kernels over streams, and what it refuses, without a GPU: the
library's calls are recorded instead of made."""

import itertools

import numpy as np
import pytest

KERNELS = ("zcgvs_embedding_lookup", "zcgvs_gated_projection", "zcgvs_adapted_projection", "zcgvs_gated_gradient",
           "zcgvs_embedding_gradient")


class Stream:
    def __init__(self, handle):
        self.handle = handle


class Recorder:
    """Stands in for capi.call. The streams of it do not wait for each other and the null stream for none of them:
    whatever touches the model's buffers while work is pending on another stream is a race."""

    def __init__(self):
        self.addresses = itertools.count(1 << 20, 1 << 20)
        self.pending, self.made, self.device_waits = set(), [], 0

    def __call__(self, name, *args):
        self.made.append(name)
        if name == "zcgvs_malloc":
            args[0]._obj.value = next(self.addresses)
        elif name == "zcgvs_device_synchronize":
            self.pending.clear()
            self.device_waits += 1
        elif name == "zcgvs_stream_synchronize":
            self.pending.discard(args[0])
        elif name in KERNELS or name.startswith("zcgvs_memcpy"):
            stream = args[-1]
            assert self.pending <= {stream}, f"{name} on {stream} beside work on {self.pending}"
            self.pending.add(stream)
        else:
            assert name == "zcgvs_free", name


def _weights(kind=np.float32):
    shapes = dict(table=(50, 8), gate=(12, 8), up=(12, 8), projection=(10, 12))
    return {name: np.ones(shape, kind) for name, shape in shapes.items()}


@pytest.fixture
def recorded(capi, monkeypatch):
    recorder = Recorder()
    monkeypatch.setattr(capi, "call", recorder)
    monkeypatch.setattr(capi.DeviceArray, "__del__", lambda self: None)
    return recorder


def _model(capi, adapters=True):
    from zcgvs_amd.embedder import DeviceEmbedder
    adapters = dict(down=np.ones((3, 4, 12), np.float32), up=np.ones((3, 10, 4), np.float32)) if adapters else None
    return DeviceEmbedder(*_weights().values(), dtype=capi.F32, adapters=adapters)


IDS, OFFSETS = np.arange(6, dtype=np.int32), np.array([0, 2, 6], np.int64)
GRADIENT = np.ones((2, 12), np.float32)


def _calls(model, stream):
    return [lambda: model.embed(IDS, OFFSETS, stream=stream), lambda: model.embed(IDS, OFFSETS, [1, -1], stream=stream),
            lambda: model.hidden_rows(IDS, OFFSETS, stream=stream),
            lambda: model.gradient(IDS, OFFSETS, GRADIENT, stream=stream)]


@pytest.mark.parametrize("streams", [(7, 7), (7, 9), (None, 7), (7, None)])
def test_calls_follow_each_other_without_a_wait(capi, recorded, streams):
    model = _model(capi)
    first, second = (None if s is None else Stream(s) for s in streams)
    for a, b in itertools.product(range(4), range(4)):
        _calls(model, first)[a]()
        _calls(model, second)[b]()
        _calls(model, getattr(first, "handle", None))[a]()  # the same stream by its handle


def test_calls_on_one_stream_leave_other_streams_alone(capi, recorded):
    model, stream = _model(capi), Stream(7)
    for call in _calls(model, stream):
        call()  # grows the buffers
    before = recorded.device_waits
    for call in _calls(model, stream):
        call()
    assert recorded.device_waits == before
