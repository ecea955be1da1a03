"""The gradient of attention against the formula in 64 bits and against differences: head widths, shared key heads, masks,
biases, caps, lengths of zero and one, rows of no text."""

import numpy as np
import pytest

from attention_helpers import Batch
from operator_helpers import Output, from_bits, kind_code, storage, strided, to_bits

pytestmark = pytest.mark.gpu


class Gradient:
    """One call on a batch: the output handed in is the formula's, rounded; rows of no text hold NaN."""

    def __init__(self, b, pad=0, shift=0, seed=5):
        capi = self.capi = b.capi
        self.b = b
        rng = np.random.default_rng(seed)
        width = b.heads * b.head_dim
        values = np.full((b.q_rows, width), np.nan)
        out, _, lse, _ = b.forward()
        for start, n in zip(b.q_starts, b.q_lens):
            values[start:start + n] = 0.3 * rng.standard_normal((n, width))
        self.owners = []
        owner, self.d_ptr, self.d_stride, self.g = strided(capi, values, b.kind, pad, shift)
        o_owner, self.o_ptr, self.o_stride, self.out = strided(capi, out, b.kind, pad + 3, shift)
        self.lse = capi.DeviceArray.from_host(lse.astype(np.float32))
        self.owners += [owner, o_owner]
        self.outs = dict(q=Output(capi, b.q_rows, width, b.kind, pad, shift),
                         k=Output(capi, b.k_rows, b.kv_heads * b.head_dim, b.kind, pad, shift),
                         v=Output(capi, b.k_rows, b.kv_heads * b.head_dim, b.kind, pad + 1, shift))
        self.table = Output(capi, b.heads, 2 * b.far + 1, b.kind) if b.table is not None else None
        self.size = capi.attention_gradient_workspace_bytes(b.desc)
        self.workspace = capi.DeviceArray.from_host(np.full(self.size, 0xFF, np.uint8))  # NaN everywhere

    def call(self, stream=None, table=True):
        o = self.outs
        self.capi.attention_gradient(
            self.b.desc, self.o_ptr, self.lse, self.d_ptr, o["q"].ptr, o["k"].ptr, o["v"].ptr, self.workspace, self.size,
            distance_bias_gradient=self.table.ptr if table and self.table is not None else None, out_stride=self.o_stride,
            out_gradient_stride=self.d_stride, q_gradient_stride=o["q"].stride, k_gradient_stride=o["k"].stride,
            v_gradient_stride=o["v"].stride, stream=stream)

    def read(self):
        got = {name: o.read() for name, o in self.outs.items()}
        if self.table is not None:
            got["table"] = self.table.read()
        return got


def check(b, **kw):
    grad = Gradient(b, **kw)
    grad.call()
    b.capi.synchronize()
    got = grad.read()
    for name, (expected, tolerance) in b.gradient(grad.g, grad.out).items():
        counted = ~np.isnan(expected)
        assert np.all(np.abs(got[name] - expected)[counted] <= tolerance[counted]), name
    return grad, got


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("head_dim", [1, 20, 32, 33, 64, 80, 96, 128])
def test_head_widths(gpu, kind, head_dim):
    check(Batch(gpu, kind, [5, 70, 1, 130], heads=3, head_dim=head_dim))
    check(Batch(gpu, kind, [150, 97], heads=2, kv_heads=1, head_dim=head_dim, mask="causal"))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mask", ["full", "causal", "prefix"])
@pytest.mark.parametrize("bias,cap", [(None, 0.0), ("slopes", 0.0), ("table", 0.0), (None, 2.0), ("table", 1.5), ("slopes", 30.0)])
def test_masks_and_scores(gpu, kind, mask, bias, cap):
    b = Batch(gpu, kind, [140, 1, 33, 260], heads=4, kv_heads=2, head_dim=64, mask=mask, prefix=[50, 0, 40, 7], bias=bias,
              far=19 if bias == "table" else 0, cap=cap, spread=1.5, pad=8)
    check(b, pad=4)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("far", [0, 1, 64, 128, 129, 512])
@pytest.mark.parametrize("lens", [[700, 40], [30, 20, 50]], ids=str)
def test_table_ends(gpu, kind, far, lens):
    check(Batch(gpu, kind, lens, heads=4, kv_heads=2, head_dim=32, bias="table", far=far))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 3, 0], [1] * 70, [16, 17, 63, 64, 65, 127, 128, 129], [2, 0, 1000]], ids=str)
def test_lengths(gpu, kind, lens):
    check(Batch(gpu, kind, lens, heads=2, head_dim=64, mask="causal", bias="table", far=4))


@pytest.mark.parametrize("kind,head_dim,pad,shift", [("f16", 64, 1, 0), ("bf16", 64, 0, 1), ("f32", 33, 3, 1), ("f16", 100, 8, 0),
                                                     ("bf16", 128, 5, 3), ("f32", 64, 4, 4), ("f32", 128, 1, 1)])
@pytest.mark.parametrize("lens", [[200, 90, 331], [20, 9, 31]], ids=str)
def test_strides_and_alignment(gpu, kind, head_dim, pad, shift, lens):
    check(Batch(gpu, kind, lens, heads=4, kv_heads=2, head_dim=head_dim, pad=pad, shift=shift, mask="causal"), pad=pad, shift=shift)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_rows_of_no_text_are_left_alone(gpu, kind):
    b = Batch(gpu, kind, [30, 77], heads=2, head_dim=64, lead=13, tail=21, bias="table", far=7)
    _, got = check(b)
    for name in ("q", "k", "v"):
        assert np.all(got[name][:13] == 7.0) and np.all(got[name][-21:] == 7.0)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mask", ["full", "prefix"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_padded_batches(gpu, kind, mask, head_dim):
    """Padding rows hold NaN in every operand and get zeros."""
    b = Batch(gpu, kind, [50, 0, 96, 1], heads=2, head_dim=head_dim, room=96, mask=mask, prefix=[20, 3, 0, 1], bias="table", far=9)
    _, got = check(b)
    for name in ("q", "k", "v"):
        for t, n in enumerate(b.q_lens):
            assert not got[name][96 * t + n:96 * (t + 1)].any()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("q_lens,k_lens", [([1, 1, 1], [300, 1, 0]), ([5, 0, 9], [2, 40, 900]), ([200], [70]), ([70], [200])], ids=str)
def test_queries_of_their_own(gpu, kind, last, q_lens, k_lens):
    for mask in ("full", "causal"):
        check(Batch(gpu, kind, q_lens, k_lens=k_lens, heads=4, kv_heads=2, head_dim=64, mask=mask, last=last, bias="table", far=30))


@pytest.mark.parametrize("scale", [-0.7, 0.0])
@pytest.mark.parametrize("bias", [None, "table"])
def test_scales_of_any_sign(gpu, scale, bias):
    check(Batch(gpu, "f16", [90, 20], heads=2, head_dim=32, scale=scale, bias=bias, far=5 if bias else 0, mask="causal"))


def test_long_texts(gpu):
    check(Batch(gpu, "bf16", [2100], heads=2, kv_heads=1, head_dim=64, mask="causal", bias="table", far=100))


@pytest.mark.parametrize("cap,bias,mask", [(0.0, None, "full"), (1.5, "table", "causal"), (3.0, "slopes", "prefix")])
def test_against_differences(gpu, cap, bias, mask):
    capi = gpu
    b = Batch(capi, "f32", [7, 4], heads=2, kv_heads=1, head_dim=5, cap=cap, bias=bias, far=2 if bias == "table" else 0, mask=mask,
              prefix=[3, 1])
    grad, got = check(b)
    operands = dict(q=b.q, k=b.k, v=b.v)
    if bias == "table":
        operands["table"] = b.table

    def loss():
        return np.nansum(b.forward()[0] * grad.g)

    # central differences with a step of 1e-5 in 64 bits: off by about 1e-9
    for name, values in operands.items():
        for i in range(values.shape[0]):
            for j in range(values.shape[1]):
                here = values[i, j]
                values[i, j] = here + 1e-5
                up = loss()
                values[i, j] = here - 1e-5
                down = loss()
                values[i, j] = here
                slope = (up - down) / 2e-5
                assert abs(slope - got[name][i, j]) <= 2e-5 * (1 + abs(slope)), (name, i, j)


def test_without_the_table_gradient(gpu):
    b = Batch(gpu, "bf16", [150, 80], heads=2, head_dim=64, bias="table", far=20)
    grad, got = check(b)
    again = Gradient(b)
    again.call(table=False)
    gpu.synchronize()
    other = again.read()
    assert all(np.array_equal(got[n], other[n]) for n in ("q", "k", "v")) and np.all(other["table"] == 7.0)


@pytest.mark.parametrize("which", ["queries", "keys", "texts"])
def test_nothing_to_see(gpu, which):
    """No queries, no keys or no texts: zeros where there are rows of texts, and for the table."""
    capi = gpu
    q_rows, k_rows, texts = (0, 6, 2) if which == "queries" else (6, 0, 2) if which == "keys" else (0, 0, 0)
    table = capi.DeviceArray.from_host(np.ones((2, 5), np.float32))
    desc = capi.attention_desc(1 << 20, 1 << 20, 1 << 20, texts, q_rows, k_rows, 2, 8, capi.F32, distance_bias=table, max_distance=2)
    outs = [Output(capi, n, 16, "f32", 3) for n in (max(q_rows, 1), max(k_rows, 1), max(k_rows, 1))]
    bias = Output(capi, 2, 5, "f32")
    size = capi.attention_gradient_workspace_bytes(desc)
    workspace = capi.DeviceArray(size, np.uint8)
    capi.attention_gradient(desc, 1 << 20, 1 << 20, 1 << 20, *(o.ptr for o in outs), workspace, size,
                            distance_bias_gradient=bias.ptr, q_gradient_stride=19, k_gradient_stride=19, v_gradient_stride=19)
    capi.synchronize()
    assert not bias.read().any()
    for o, n in zip(outs, (q_rows, k_rows, k_rows)):
        assert not o.read()[:n].any() and (n or np.all(o.read() == 7.0))


@pytest.mark.parametrize("lens", [[300, 64, 513], [20, 9, 31, 64]], ids=str)
def test_same_bits_and_graph_replays(gpu, lens):
    capi = gpu
    grad = Gradient(Batch(capi, "bf16", lens, heads=4, kv_heads=2, head_dim=64, mask="causal", bias="table", far=40))
    grad.call()
    capi.synchronize()
    eager = grad.read()
    stream = capi.Stream()
    graph = capi.Graph(stream, lambda: grad.call(stream))
    for replay in range(3):
        for a in [o.array for o in grad.outs.values()] + [grad.table.array, grad.workspace]:
            fill = capi.DeviceArray.from_host(np.full(a.nbytes, 0xEE, np.uint8))
            capi.call("zcgvs_memcpy_d2d", a.ptr, fill.ptr, a.nbytes, None)
        for o in list(grad.outs.values()) + [grad.table]:
            o.host.view(np.uint8)[:] = 0xEE
        capi.synchronize()
        graph.launch(stream)
        capi.synchronize()
        got = grad.read()
        assert all(np.array_equal(got[n], eager[n]) for n in eager), replay
