"""Attention over packed and padded texts against the formula in 64 bits: head widths, head groups, masks, biases,
caps, lengths of zero and one, rows of no text, split keys."""

import numpy as np
import pytest

from attention_helpers import Batch
from operator_helpers import Output, from_bits, storage, to_bits

pytestmark = pytest.mark.gpu


def run(b, pad=0, shift=0, lse=True):
    capi = b.capi
    out = Output(capi, b.q_rows, b.heads * b.head_dim, b.kind, pad, shift)
    d_lse = capi.DeviceArray.from_host(np.full((b.q_rows, b.heads), 5.0, np.float32))
    size = capi.attention_workspace_bytes(b.desc)
    workspace = capi.DeviceArray.from_host(np.full(size, 0xFF, np.uint8))  # NaN everywhere
    capi.attention(b.desc, out.ptr, workspace, size, lse=d_lse if lse else None, out_stride=out.stride)
    capi.synchronize()
    return out.read(), d_lse.to_host()


def check(b, **kw):
    got, got_lse = run(b, **kw)
    out, tolerance, lse, lse_tolerance = b.forward()
    counted = ~np.isnan(lse[:, 0])
    assert np.all(np.abs(got[counted] - out[counted]) <= tolerance[counted])
    empty = counted & np.isneginf(lse[:, 0])
    assert not got[empty].any()
    with np.errstate(invalid="ignore"):
        close = np.abs(got_lse - lse) <= lse_tolerance
    assert np.all(close[counted] | (got_lse[counted] == lse[counted]))
    return got, got_lse, counted


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("head_dim", [1, 20, 32, 33, 64, 80, 96, 128])
def test_head_widths(gpu, kind, head_dim):
    check(Batch(gpu, kind, [5, 70, 1, 130], heads=3, head_dim=head_dim))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mask", ["full", "causal", "prefix"])
@pytest.mark.parametrize("bias,cap", [(None, 0.0), ("slopes", 0.0), ("table", 0.0), (None, 2.0), ("table", 1.5), ("slopes", 30.0)])
def test_masks_and_scores(gpu, kind, mask, bias, cap):
    b = Batch(gpu, kind, [140, 1, 33, 260], heads=4, kv_heads=2, head_dim=64, mask=mask, prefix=[50, 0, 40, 7], bias=bias,
              far=19 if bias == "table" else 0, cap=cap, spread=1.5, pad=8)
    check(b, pad=4)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("far", [0, 1, 64, 129, 512])
def test_table_ends(gpu, kind, far):
    check(Batch(gpu, kind, [700, 40], heads=2, head_dim=32, bias="table", far=far))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 3, 0], [1] * 70, [16, 17, 63, 64, 65, 127, 128, 129], [4097], [2, 0, 1000]],
                         ids=str)
def test_lengths(gpu, kind, lens):
    check(Batch(gpu, kind, lens, heads=2, head_dim=64, mask="causal"))


def test_many_texts(gpu):
    rng = np.random.default_rng(9)
    check(Batch(gpu, "bf16", rng.integers(0, 9, 5000), heads=1, head_dim=32))


@pytest.mark.parametrize("kind,head_dim,pad,shift", [("f16", 64, 1, 0), ("bf16", 64, 0, 1), ("f32", 33, 3, 1), ("f16", 100, 8, 0),
                                                     ("bf16", 128, 5, 3), ("f32", 64, 4, 4)])
@pytest.mark.parametrize("rows", ["all", "one"])
def test_strides_and_alignment(gpu, kind, head_dim, pad, shift, rows):
    apart = dict(k_lens=[200, 90, 31]) if rows == "one" else {}
    b = Batch(gpu, kind, [1, 1, 1] if rows == "one" else [200, 90, 31], heads=4, kv_heads=2, head_dim=head_dim, pad=pad, shift=shift,
              mask="causal", last=rows == "one", **apart)
    check(b, pad=pad, shift=shift)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_rows_of_no_text_are_left_alone(gpu, kind):
    b = Batch(gpu, kind, [30, 77], heads=2, head_dim=64, lead=13, tail=21)
    got, lse, counted = check(b)
    assert np.all(got[~counted] == 7.0) and np.all(lse[~counted] == 5.0)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mask", ["full", "prefix"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_padded_batches(gpu, kind, mask, head_dim):
    """Padding rows hold NaN, give zeros and reach no other row."""
    b = Batch(gpu, kind, [50, 0, 96, 1], heads=2, head_dim=head_dim, room=96, mask=mask, prefix=[20, 3, 0, 1], bias="table", far=9)
    got, lse, counted = check(b)
    assert not got[~counted].any() and np.all(np.isneginf(lse[~counted]))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("q_lens,k_lens", [([1, 1, 1], [300, 1, 0]), ([5, 0, 9], [2, 40, 900]), ([200], [70]), ([70], [200])], ids=str)
def test_queries_of_their_own(gpu, kind, last, q_lens, k_lens):
    """Causal with fewer keys than queries: rows before the first key see nothing and give zeros."""
    for mask in ("full", "causal"):
        check(Batch(gpu, kind, q_lens, k_lens=k_lens, heads=4, kv_heads=2, head_dim=64, mask=mask, last=last, bias="table", far=30))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(16, 4, 128), (12, 12, 64), (8, 1, 32), (5, 1, 80), (32, 1, 64)])
@pytest.mark.parametrize("cap", [0.0, 10.0])
def test_one_query_over_long_keys(gpu, kind, heads, kv_heads, head_dim, cap):
    """Keys split over wavefronts and workgroups, and joined."""
    b = Batch(gpu, kind, [1, 1], k_lens=[6001, 3], heads=heads, kv_heads=kv_heads, head_dim=head_dim, mask="causal", last=True,
              cap=cap, spread=1.5, bias="slopes")
    assert gpu.attention_workspace_bytes(b.desc) > 256
    check(b)


def test_split_rows_of_no_text(gpu):
    b = Batch(gpu, "f16", [1, 2], k_lens=[5000, 4000], heads=4, kv_heads=2, head_dim=64, last=True, lead=2, tail=3)
    got, lse, counted = check(b)
    assert np.all(got[~counted] == 7.0) and np.all(lse[~counted] == 5.0)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_large_scores(gpu, kind):
    """Scores of hundreds, maxima late in the row: the running maximum is raised many times."""
    b = Batch(gpu, kind, [300], heads=2, head_dim=64, spread=6.0, scale=1.0)
    order = np.argsort(np.abs(b.k[:, :64]).sum(1))
    check(b)
    assert order.size == 300


@pytest.mark.parametrize("scale", [-0.7, 0.0])
@pytest.mark.parametrize("bias", [None, "table"])
def test_scales_of_any_sign(gpu, scale, bias):
    check(Batch(gpu, "f16", [90, 20], heads=2, head_dim=32, scale=scale, bias=bias, far=5 if bias else 0, mask="causal"))


def test_without_lse(gpu):
    b = Batch(gpu, "bf16", [90, 20], heads=2, head_dim=64)
    with_lse, _ = run(b)
    without, untouched = run(b, lse=False)
    assert np.array_equal(with_lse, without) and np.all(untouched == 5.0)


def test_table_of_the_lowest_value(gpu):
    """A bias of float16's lowest value leaves a distance out."""
    capi = gpu
    b = Batch(capi, "f16", [60], heads=2, head_dim=32, bias="table", far=3)
    b.table[:, 4:] = -65504.0
    stored = capi.DeviceArray.from_host(to_bits(b.table, "f16"))
    b.desc.distance_bias = stored.ptr
    check(b)


@pytest.mark.parametrize("shape", ["long", "one"])
def test_same_bits_and_graph_replays(gpu, shape):
    capi = gpu
    if shape == "long":
        b = Batch(capi, "bf16", [300, 64, 513], heads=4, kv_heads=2, head_dim=64, mask="causal", bias="table", far=40)
    else:
        b = Batch(capi, "bf16", [1], k_lens=[4001], heads=4, kv_heads=2, head_dim=64, bias="table", far=40)
    out = capi.DeviceArray((b.q_rows, b.heads * b.head_dim), np.uint16)
    lse = capi.DeviceArray((b.q_rows, b.heads), np.float32)
    size = capi.attention_workspace_bytes(b.desc)
    workspace = capi.DeviceArray(size, np.uint8)

    def step(stream):
        capi.attention(b.desc, out, workspace, size, lse=lse, stream=stream)

    step(None)
    capi.synchronize()
    eager = out.to_host(), lse.to_host()
    stream = capi.Stream()
    graph = capi.Graph(stream, lambda: step(stream))
    for replay in range(3):
        for a in (out, lse, workspace):
            fill = capi.DeviceArray.from_host(np.full(a.nbytes, 0xEE, np.uint8))
            capi.call("zcgvs_memcpy_d2d", a.ptr, fill.ptr, a.nbytes, None)
        capi.synchronize()
        graph.launch(stream)
        capi.synchronize()
        assert np.array_equal(out.to_host(), eager[0]) and np.array_equal(lse.to_host(), eager[1]), replay
